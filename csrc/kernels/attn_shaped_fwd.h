// Forward of attention with shaped scores: query tiles, and the form for few query rows (attn_shaped.h).
#pragma once
#include <algorithm>
#include "attn_shaped.h"

namespace {
// ------------------------------------------------------------------------------- forward
// NW waves of 32 rows
template <typename T, int D, int NW, typename O>
__global__ __launch_bounds__(NW * 64, D == 64 ? 4 : 2) void shaped_fwd_kernel(Shaped p) {
  constexpr bool DOCS = O::docs;
  constexpr int TB = KT * D * 2;
  typedef DeadRows<D, NW> Dead;
  __shared__ __attribute__((aligned(1024))) char smem[4 * TB];  // [slot][K | V]
  __shared__ __attribute__((aligned(256))) unsigned marks[DOCS ? 2 * Dead::WORDS : 1];
  __shared__ int range[2][NW];
  const unsigned lds = (unsigned)(size_t)(LDS_AS char*)smem, lds_marks = (unsigned)(size_t)(LDS_AS unsigned*)marks;
  const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = l >> 5;
  Offs<D> fo;
  fo.init();
  int col, rank;
  locate(p.B * p.Hk * p.heads, col, rank);
  const int inst = col / p.heads, b = inst / p.Hk, hk = inst % p.Hk;
  const int tile = col % p.heads * p.tiles + (p.causal ? p.tiles - 1 - rank : rank);
  const int r = tile * NW * 32 + w * 32 + (l & 31), g = r / p.Sqp, q = r % p.Sqp;
  const bool valid = g < p.G && q < p.Sq;
  const int head = hk * p.G + min(g, p.G - 1), qc = min(q, p.Sq - 1);
  const Mask mk(p, b);
  const Span sp = valid ? mk.of<DOCS>(q) : Span{0, 0};
  const bool sees = sp.hi > sp.lo;
  const Reach re(sp, sees);
  if (l == 0) { range[0][w] = re.ulo; range[1][w] = re.uhi; }
  __syncthreads();
  int blo = range[0][0], bhi = range[1][0];
#pragma unroll
  for (int u = 1; u < NW; ++u) { blo = min(blo, range[0][u]); bhi = max(bhi, range[1][u]); }
  blo = __builtin_amdgcn_readfirstlane(blo);
  bhi = __builtin_amdgcn_readfirstlane(bhi);
  // tiles from the first key that a row sees: keys in front of it are not read
  const int org = bhi > 0 ? blo : 0, t1 = (bhi - org + KT - 1) / KT;

  const T* Kb = (const T*)p.k + b * p.k_bs + hk * D;
  const T* Vb = (const T*)p.v + b * p.v_bs + hk * D;
  Dma<D, NW> km, vm;
  km.init(p.k_rs);
  vm.init(p.v_rs);
  auto issue = [&](int t, int slot) {
    const int k0 = org + t * KT;
    km.issue(Kb + k0 * p.k_rs, p.k_rs, bhi - k0, lds + slot * 2 * TB);
    vm.issue(Vb + k0 * p.v_rs, p.v_rs, bhi - k0, lds + slot * 2 * TB + TB);
    if constexpr (DOCS) Dead::issue(mk.docs, 8, 4, p.Sk, k0, vm, lds_marks + slot * Dead::WORDS * 4);  // a run's end; 0: in none
  };
  auto landed = [&](int slot) {
    dma_wait();
    if constexpr (DOCS) {
#pragma unroll
      for (int i = 0; i < Dead::N; ++i)
        if ((int)Dead::mark(marks + slot * Dead::WORDS, i) <= 0) {
          vm.clear(smem + slot * 2 * TB + TB, i);
        }
    }
    lds_bar();
  };
  if (t1 > 0) issue(0, 0);
  const T* Qr = (const T*)p.q + b * p.q_bs + qc * p.q_rs + head * D;
  typename Ty<T>::x8 qf[D / 16];
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) qf[kk] = frag_mem<T>(Qr, kk, sees);
  const Score<O> sc(p);
  const float slope = slope_of<O>(p, head);
  const int pos = q + mk.shift;
  const int thr = drop_thr(p.p_drop);
  constexpr bool drop = O::drop;
  const uint32_t hs = drop ? head_seed(p, b * p.H + head) : 0u;
  const int qg = (q >> 2) * p.Sk;
  constexpr float RAISE = Ty<T>::raise, UP = Ty<T>::fits ? 0.f : Ty<T>::fwd_up - RAISE;  // P is 2^UP times itself
  float m = -INFINITY, lsum = 0.f;  // lsum: this lane's half of the row
  f32x16 o[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[db][e] = 0.f;
  if (t1 > 0) landed(0);
  auto step = [&](auto slot_, int t) {
    constexpr int slot = decltype(slot_)::value, KA = slot * 2 * TB, VA = KA + TB;
    if (t + 1 < t1) issue(t + 1, slot ^ 1);
#pragma unroll
    for (int kb = 0; kb < KT / 32; ++kb) {
      const int k0 = org + t * KT + 32 * kb;
      if (!(k0 < re.uhi && k0 + 32 > re.ulo)) continue;  // wave-uniform
      f32x16 s;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) s = Ty<T>::mfma(frag_row<T, D>(smem, KA, fo, kb, kk), qf[kk], s);
      const bool part = !(k0 >= re.ilo && k0 + 32 <= re.ihi);
      if (O::bias) {
        const float d0 = (float)(pos - k0 - 4 * h);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          s[e] = fmaf(-slope, fabsf(d0 - (float)srow(e)), sc.x(s[e]));
      }
      if (part) mask_slots(s, (unsigned)(k0 + 4 * h - sp.lo), (unsigned)(sp.hi - sp.lo), -INFINITY);
      // the row maximum of the raw products (a score grows with its product; distances: of the scores)
      float mx = s[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
      mx = pair_max(mx);
      if (!O::bias) mx = !O::cap ? mx * sc.mult : mx == -INFINITY ? mx : sc.c2l * sc.r(mx);
      mx = above<T>(mx);
      // the running maximum follows only where a row outgrew it by 2^RAISE: O and the sum are rescaled
      // in few tiles, P stays below 2^RAISE
      if (__any(mx > m + RAISE)) {
        const float mnew = fmaxf(m, mx), alpha = ex2(m - (mnew == -INFINITY ? 0.f : mnew));
        lsum *= alpha;
        m = mnew;
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[db][e] *= alpha;
      }
      const float nm = m == -INFINITY ? 0.f : UP - m;
      if (O::bias) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = ex2(s[e] + nm);
      } else if (O::cap) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = ex2(fmaf(sc.r(s[e]), sc.c2l, nm));
        if (part) mask_slots(s, (unsigned)(k0 + 4 * h - sp.lo), (unsigned)(sp.hi - sp.lo), 0.f);  // a capped score has no -inf
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = ex2(fmaf(s[e], sc.mult, nm));
      }
      {
        float t0_ = s[0] + s[1], t1_ = s[2] + s[3];
#pragma unroll
        for (int e = 4; e < 16; e += 4) { t0_ += s[e] + s[e + 1]; t1_ += s[e + 2] + s[e + 3]; }
        lsum += t0_ + t1_;
      }
      if (drop) {
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const unsigned kp = keep4_rows(hs, qg, k0 + srow(e) + 4 * h, q & 3, thr);
#pragma unroll
          for (int u = 0; u < 4; ++u) s[e + u] = (kp & (1u << u)) ? s[e + u] : 0.f;
        }
      }
#pragma unroll
      for (int kc = 0; kc < 2; ++kc) {
        const typename Ty<T>::x8 pf = pack8<T>(s, kc);
#pragma unroll
        for (int db = 0; db < D / 32; ++db) o[db] = Ty<T>::mfma(frag_tr<T, D>(smem, VA, fo, 2 * kb + kc, db), pf, o[db]);
      }
    }
    if (t + 1 < t1) landed(slot ^ 1);
  };
  for (int t = 0; t < t1; t += 2) {
    step(iconst<0>{}, t);
    if (t + 1 < t1) step(iconst<1>{}, t + 1);
  }
  lsum = xor_sum<32>(lsum);
  if (valid) {
    const float keep = drop ? 256.f / (float)(256 - thr) : 1.f;
    const float inv = sees && lsum != 0.f ? keep / lsum : 0.f;
    T* Or = (T*)p.out + b * p.o_bs + q * p.o_rs + head * D + 4 * h;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        typename Ty<T>::x4 v;
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = (T)(sees ? o[db][e + u] * inv : 0.f);
        *(typename Ty<T>::x4*)(Or + db * 32 + srow(e)) = v;
      }
    if (h == 0) p.lse[((long long)b * p.H + head) * p.Sq + q] = sees && lsum != 0.f ? (m + sc.base + (__log2f(lsum) - UP)) * LN2 : INFINITY;
  }
}

// ------------------------------------------------------------------------------- few query rows
// The forward for at most 32 rows (queries x heads of a group): serving's single tokens. All waves of a
// block hold the same rows and divide the keys (8 KiB of K at a time), so the work along the cache is split
// NW ways inside a block and `splits` ways over blocks; each block takes an even share of the keys
// that its rows see (the lengths are device data). Bound by reading K and V once: K goes from memory
// straight into operand registers, V through the wave's own LDS (no block barrier in the loop). The
// waves' (m, l, O) meet in LDS, those of the blocks in shaped_few_join_kernel. B16 H32/8 D128 over caches of up to
// 16384: 157 us, 5.4 TB/s. B1 H16 D64 Sk 777: 10 us, of which 6 are a launch with no keys at all; its second tile
// costs as much as the first, a chain of dependent steps and no load (touching the tile's lines early: equal).
constexpr int FW = 8;  // waves
template <typename T, int D, typename O>
__global__ __launch_bounds__(FW * 64, 2) void shaped_few_kernel(Shaped p, int splits, float* __restrict__ part) {
  constexpr bool DOCS = O::docs;
  constexpr int KB = 128 / D, KEYS = 32 * KB;  // a wave's tile: 8 KiB of K, of V
  constexpr int VB = KEYS * D * 2;             // (the f32 accumulators take D / 64 * VB)
  __shared__ __attribute__((aligned(16))) char smem[FW * VB];
  __shared__ float ml[2][FW][32];
  const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = l >> 5, r = l & 31;
  Offs<D> fo;
  fo.init();
  const int inst = blockIdx.x / splits, split = blockIdx.x % splits;
  const int b = inst / p.Hk, hk = inst % p.Hk, R = p.G * p.Sq;
  const bool valid = r < R;
  const int g = valid ? r / p.Sq : 0, q = valid ? r % p.Sq : 0, head = hk * p.G + g;
  const Mask mk(p, b);
  const Span sp = valid ? mk.of<DOCS>(q) : Span{0, 0};
  const bool sees = sp.hi > sp.lo;
  const Reach re(sp, sees);
  const int org = re.uhi > 0 ? re.ulo : 0, an = (re.uhi - org + KEYS - 1) / KEYS, per = (an + splits - 1) / splits;
  const int t1 = min(an, (split + 1) * per);
  int t = split * per + w;

  // loads through descriptors that end behind the last key any row sees: keys past it arrive as zeros
  constexpr int NVV = KEYS * D / 8 / 64, RPI = 512 / D;  // 16-byte vectors of V a lane moves, rows of one instruction
  const T* Kb = (const T*)p.k + b * p.k_bs + hk * D;
  const T* Vb = (const T*)p.v + b * p.v_bs + hk * D;
  const int vrow = l / (D / 8), krs = (int)p.k_rs * 2, vrs = (int)p.v_rs * 2;
  const int koff = r * krs + 16 * h, voff = vrow * vrs + (l % (D / 8)) * 16;
  char* V_ = smem + w * VB;
  u32x4 kn[KB][D / 16], vn[NVV];
  bool vdead[DOCS ? NVV : 1];
  auto load = [&](int tt) {
    const int k0 = org + tt * KEYS, rows = min(re.uhi - k0, KEYS);
    const __amdgpu_buffer_rsrc_t rk = rows_rsrc(Kb + k0 * p.k_rs, krs, rows);
    const __amdgpu_buffer_rsrc_t rv = rows_rsrc(Vb + k0 * p.v_rs, vrs, rows);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
        kn[kb][kk] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, koff + kk * 32, kb * 32 * krs, 0));
#pragma unroll
    for (int i = 0; i < NVV; ++i)
      vn[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rv, voff, i * RPI * vrs, 0));
    if constexpr (DOCS) {
#pragma unroll
      for (int i = 0; i < NVV; ++i) {
        const int2 d = p.docs[(long long)b * p.Sk + min(k0 + vrow + i * RPI, p.Sk - 1)];
        vdead[i] = d.y <= d.x;
      }
    }
  };
  if (t < t1) load(t);  // (no load past the end: the block barriers behind the loop would wait for it)
  const T* Qr = (const T*)p.q + b * p.q_bs + q * p.q_rs + head * D;
  typename Ty<T>::x8 qf[D / 16];
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) qf[kk] = frag_mem<T>(Qr, kk, sees);
  const Score<O> sc(p);
  const float slope = slope_of<O>(p, head);
  const int pos = q + mk.shift;
  const float fs = O::cap || O::wide ? 1.f : sc.mult, fx = O::bias ? 1.f : fs;  // factors left to the bias, to the exponent
  constexpr float UP = Ty<T>::fwd_up;  // P is 2^UP times itself
  float m = -INFINITY, lsum = 0.f;
  f32x16 o[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[db][e] = 0.f;

  for (; t < t1; t += FW) {
    const int k0 = org + t * KEYS;
    f32x16 s[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[kb][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) s[kb] = Ty<T>::mfma(__builtin_bit_cast(typename Ty<T>::x8, kn[kb][kk]), qf[kk], s[kb]);
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < NVV; ++i) {  // rows i RPI + vrow: the swizzle of a row depends on its low 4 bits
      const int row = i * RPI + vrow;
      const u32x4 z = u32x4{0u, 0u, 0u, 0u};
      *(u32x4*)(V_ + row * 2 * D + (((l % (D / 8)) ^ swz<D>(row)) << 4)) = DOCS && vdead[i] ? z : vn[i];
    }
    __builtin_amdgcn_wave_barrier();
    if (t + FW < t1) load(t + FW);
    // (maximum of the finished scores: few rows are bound by memory, and this path is the shortest code)
    if (O::cap || O::wide) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[kb][e] = sc.x(s[kb][e]);
    }
    if (O::bias) {
      const float d0 = (float)(pos - k0 - 4 * h);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[kb][e] = fmaf(-slope, fabsf(d0 - (float)(32 * kb + srow(e))), s[kb][e] * fs);
    }
    if (!(k0 >= re.ilo && k0 + KEYS <= re.ihi)) {
      const unsigned base = (unsigned)(k0 + 4 * h - sp.lo), len = (unsigned)(sp.hi - sp.lo);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (base + (unsigned)(32 * kb + srow(e)) >= len) s[kb][e] = -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[kb][e]);
    mx = pair_max(mx);
    const float mnew = fmaxf(m, above<T>(mx * fx)), muse = mnew == -INFINITY ? 0.f : mnew, alpha = ex2(m - muse);
    float rs = 0.f;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[kb][e] = ex2(fmaf(s[kb][e], fx, UP - muse));
        rs += s[kb][e];
      }
    lsum = fmaf(lsum, alpha, xor_sum<32>(rs));
    m = mnew;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[db][e] *= alpha;
#pragma unroll
    for (int kc = 0; kc < 2 * KB; ++kc) {
      const typename Ty<T>::x8 pf = pack8<T>(s[kc >> 1], kc & 1);
#pragma unroll
      for (int db = 0; db < D / 32; ++db) o[db] = Ty<T>::mfma(frag_tr<T, D>(V_, 0, fo, kc, db), pf, o[db]);
    }
  }
  // the waves' parts: a common maximum, then the sums in a tree
  if (h == 0) { ml[0][w][r] = m; ml[1][w][r] = lsum; }
  __syncthreads();
  float M = ml[0][0][r], L = 0.f;
#pragma unroll
  for (int u = 1; u < FW; ++u) M = fmaxf(M, ml[0][u][r]);
  const float Mu = M == -INFINITY ? 0.f : M;
#pragma unroll
  for (int u = 0; u < FW; ++u) L = fmaf(ml[1][u][r], ex2(ml[0][u][r] - Mu), L);
  const float own = ex2(m - Mu);
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[db][e] *= own;
#pragma unroll
  for (int half = FW / 2; half > 0; half >>= 1) {  // waves half .. 2 half - 1 hand theirs to w - half
    f32x4* x = (f32x4*)smem + (w & (half - 1)) * (D / 8) * 64 + l;
    if (w >= half && w < 2 * half) {
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int e = 0; e < 16; e += 4) x[(db * 4 + e / 4) * 64] = f32x4{o[db][e], o[db][e + 1], o[db][e + 2], o[db][e + 3]};
    }
    __syncthreads();
    if (w < half) {
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const f32x4 y = x[(db * 4 + e / 4) * 64];
#pragma unroll
          for (int u = 0; u < 4; ++u) o[db][e + u] += y[u];
        }
    }
    __syncthreads();
  }
  if (w != 0 || !valid) return;
  if (splits > 1) {  // (a row that sees nothing went through tiles that its neighbours see whole: no part of it stays)
    float* P = part + ((long long)blockIdx.x * R + r) * D + 4 * h;
    const f32x4 none = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *(f32x4*)(P + db * 32 + srow(e)) = sees ? f32x4{o[db][e], o[db][e + 1], o[db][e + 2], o[db][e + 3]} : none;
    if (h == 0) {
      float* S = part + (long long)gridDim.x * R * D + ((long long)blockIdx.x * R + r) * 2;
      S[0] = sees ? M : -INFINITY;
      S[1] = sees ? L : 0.f;
    }
    return;
  }
  const float inv = sees && L != 0.f ? 1.f / L : 0.f;
  T* Or = (T*)p.out + b * p.o_bs + q * p.o_rs + head * D + 4 * h;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      typename Ty<T>::x4 v;
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = (T)(sees ? o[db][e + u] * inv : 0.f);
      *(typename Ty<T>::x4*)(Or + db * 32 + srow(e)) = v;
    }
  if (h == 0) p.lse[((long long)b * p.H + head) * p.Sq + q] = sees && L != 0.f ? (M + sc.base + (__log2f(L) - UP)) * LN2 : INFINITY;
}
// one wave per (instance, row): the splits' parts in order
template <typename T, int D>
__global__ __launch_bounds__(64) void shaped_few_join_kernel(Shaped p, int splits, const float* __restrict__ part) {
  const int R = p.G * p.Sq, inst = blockIdx.x / R, r = blockIdx.x % R, l = threadIdx.x;
  const float* S = part + (long long)p.B * p.Hk * splits * R * D;
  auto row = [&](int s) { return ((long long)inst * splits + s) * R + r; };
  float M = -INFINITY;
  for (int s = 0; s < splits; ++s) M = fmaxf(M, S[2 * row(s)]);
  float L = 0.f, o[D / 64];
#pragma unroll
  for (int u = 0; u < D / 64; ++u) o[u] = 0.f;
#pragma unroll 8
  for (int s = 0; s < splits; ++s) {
    const float m = S[2 * row(s)], f = m == -INFINITY ? 0.f : ex2(m - M);
    L = fmaf(S[2 * row(s) + 1], f, L);
#pragma unroll
    for (int u = 0; u < D / 64; ++u) {
      const float v = part[row(s) * D + u * 64 + l];
      o[u] = fmaf(v, f, o[u]);
    }
  }
  const int b = inst / p.Hk, head = inst % p.Hk * p.G + r / p.Sq, q = r % p.Sq;
  const float inv = L != 0.f ? 1.f / L : 0.f;
  T* Or = (T*)p.out + b * p.o_bs + q * p.o_rs + head * D;
#pragma unroll
  for (int u = 0; u < D / 64; ++u) Or[u * 64 + l] = (T)(o[u] * inv);
  if (l == 0) p.lse[((long long)b * p.H + head) * p.Sq + q] = L != 0.f ? (M + (shifted(p) ? p.cap * LOG2E : 0.f) + (__log2f(L) - Ty<T>::fwd_up)) * LN2 : INFINITY;
}

// few rows and no dropout: the split form; shares of a cache so that there are about 4 blocks for each of
// 256 CUs, none below 512 keys (one token, H32/8 D128, caches half to all full, us: B16 Sk 16384 with 2, 4 and 8 blocks a
// CU 168, 165 and 170, Sk 65536 626, 595 and 567, B64 Sk 2048 93, 97 and 114; shares from 256, 512 and 1024 keys: B1 Sk 2048
// 16, 18 and 20, Sk 16384 37, 26 and 24, B16 Sk 2048 44, 34 and 28, Sk 16384 equal)
bool few_rows(int G, int Sq, float p_drop) { return G * (long long)Sq <= 32 && p_drop == 0.f; }
int few_splits(int inst, int Sk) { return std::max(1, std::min((1024 + inst - 1) / inst, Sk / 512)); }
template <typename T, int D>
int launch_fwd(Shaped p, float* part, hipStream_t s) {
  if (few_rows(p.G, p.Sq, p.p_drop)) {
    const int inst = p.B * p.Hk, splits = few_splits(inst, p.Sk);
    with_rules(p, [&](auto o) {
      typedef decltype(o) O;
      if constexpr (!O::drop)
        hipLaunchKernelGGL((shaped_few_kernel<T, D, O>), dim3((unsigned)(inst * splits)), dim3(FW * 64), 0, s, p, splits, part);
    });
    if (splits > 1)
      hipLaunchKernelGGL((shaped_few_join_kernel<T, D>), dim3((unsigned)(inst * p.G * p.Sq)), dim3(64), 0, s, p, splits, part);
    return hipGetLastError() == hipSuccess ? 0 : -1;
  }
  const int waves = row_waves(p, D);
  row_tiles(p, waves * 32);
  const dim3 grid((unsigned)(p.tiles * p.heads * p.B * p.Hk)), block(waves * 64);
  with_rules(p, [&](auto o) {
    constexpr int MAX = max_row_waves<decltype(o)>(D);
    if (waves == MAX) hipLaunchKernelGGL((shaped_fwd_kernel<T, D, MAX, decltype(o)>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((shaped_fwd_kernel<T, D, 4, decltype(o)>), grid, block, 0, s, p);
  });
  return hipGetLastError() == hipSuccess ? 0 : -1;
}
}  // namespace
