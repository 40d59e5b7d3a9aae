// Backward of attention with shaped scores: dQ pass and dK/dV pass (attn_shaped.h).
#pragma once
#include <algorithm>
#include "attn_shaped.h"

namespace {
// ------------------------------------------------------------------------------- dQ pass
// same rows and tiles as the forward; also writes lse in log2 units (shifted, Score; f16: less bwd_up) and -delta.
// Precision: delta = sum P dP is taken as dO.O here, off by O's rounding. Beside the roundings of dS and of the
// gradients this weighs as much as they do where a row's softmax rests on few keys, 1 / n_eff of it else (974 keys
// under a slope of 1/2 gave 1.7 times the error of a float32 backward, 372 without one 1.48). So where a row of the
// wave sees at most FEW keys, or its slope of either sign leaves it about as many, sum P (dP - delta) over the row, which is that
// error, corrects the delta of the dK/dV pass, and dQ, where it stays, takes dS into its product as two 16-bit
// terms. (Everywhere: B1 H16/4 S8192 D128 dQ 417 -> 580 us, B4 H16 S2048 D64 documents 35 -> 41.)
constexpr int FEW = 128;
// (168 registers are not enough for dropout's hashes beside f16's running scale)
constexpr int dq_min_waves(int D, bool drop, bool fits) { return D == 64 && (fits || !drop) ? 3 : 2; }
template <typename T, int D, int NW, typename O>
__global__ __launch_bounds__(NW * 64, dq_min_waves(D, O::drop, Ty<T>::fits)) void shaped_dq_kernel(Shaped p) {
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
          km.clear(smem + slot * 2 * TB, i);
          vm.clear(smem + slot * 2 * TB + TB, i);
        }
    }
    lds_bar();
  };
  if (t1 > 0) issue(0, 0);
  const T* Qr = (const T*)p.q + b * p.q_bs + qc * p.q_rs + head * D;
  const long long orow = b * p.o_bs + qc * p.o_rs + head * D;
  typename Ty<T>::x8 qf[D / 16], df[D / 16];
  float dlt = 0.f;
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    qf[kk] = frag_mem<T>(Qr, kk, sees);
    df[kk] = frag_mem<T>((const T*)p.dout + orow, kk, sees);
    const typename Ty<T>::x8 of = frag_mem<T>((const T*)p.o + orow, kk, sees);
#pragma unroll
    for (int e = 0; e < 8; ++e) dlt = fmaf((float)df[kk][e], (float)of[e], dlt);
  }
  dlt = xor_sum<32>(dlt);
  const long long srow_i = ((long long)b * p.H + head) * p.Sq + qc;
  const Score<O> sc(p);
  const float lse2 = sees ? fmaf(p.lse[srow_i], LOG2E, -sc.base) : INFINITY;
  const float slope = slope_of<O>(p, head);
  const int pos = q + mk.shift;
  const int thr = drop_thr(p.p_drop);
  constexpr bool drop = O::drop;
  const float keep = drop ? 256.f / (float)(256 - thr) : 1.f;
  const uint32_t hs = drop ? head_seed(p, b * p.H + head) : 0u;
  const int qg = (q >> 2) * p.Sk;
  const bool two = __any(sees && (sp.hi - sp.lo <= FEW || (O::bias && fabsf(slope) * FEW >= 2.f * LOG2E)));  // e^-2 at FEW
  float rest = 0.f;  // this lane's half of sum P (dP - delta)
  float up = START;
  f32x16 acc[D / 32], ndl;  // -delta in every slot: dP - delta is the product's start
#pragma unroll
  for (int e = 0; e < 16; ++e) ndl[e] = -dlt;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[db][e] = 0.f;
  if (t1 > 0) landed(0);
  auto step = [&](auto slot_, int t) {
    constexpr int slot = decltype(slot_)::value, KA = slot * 2 * TB, VA = KA + TB;
    if (t + 1 < t1) issue(t + 1, slot ^ 1);
#pragma unroll
    for (int kb = 0; kb < KT / 32; ++kb) {
      const int k0 = org + t * KT + 32 * kb;
      if (!(k0 < re.uhi && k0 + 32 > re.ulo)) continue;  // wave-uniform
      f32x16 s, dp = ndl;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        s = Ty<T>::mfma(frag_row<T, D>(smem, KA, fo, kb, kk), qf[kk], s);
        dp = Ty<T>::mfma(frag_row<T, D>(smem, VA, fo, kb, kk), df[kk], dp);
      }
      if (drop) {
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const unsigned kp = keep4_rows(hs, qg, k0 + srow(e) + 4 * h, q & 3, thr);
#pragma unroll
          for (int u = 0; u < 4; ++u) dp[e + u] = fmaf((kp & (1u << u)) ? dp[e + u] + dlt : 0.f, keep, -dlt);
        }
      }
      // P (dP - delta) in s; capped: d tanh / 4 (wide: d tanh) in dp
      const float d0 = O::bias ? (float)(pos - k0 - 4 * h) : 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float r_ = O::wide ? sc.t(s[e]) : O::cap ? sc.r(s[e]) : 0.f;
        const float x = O::wide ? fmaf(r_, sc.cl, -lse2) : O::cap ? fmaf(r_, sc.c2l, -lse2) : fmaf(s[e], sc.mult, -lse2);
        s[e] = ex2(O::bias ? fmaf(-slope, fabsf(d0 - (float)srow(e)), x) : x) * dp[e];
        if (O::cap) dp[e] = fmaf(-r_, r_, r_);
        if (O::wide) dp[e] = fmaf(-r_, r_, 1.f);
      }
      if (!(k0 >= re.ilo && k0 + 32 <= re.ihi)) mask_slots(s, (unsigned)(k0 + 4 * h - sp.lo), (unsigned)(sp.hi - sp.lo), 0.f);
      if (two) {
        float a = s[0] + s[1], b_ = s[2] + s[3];
#pragma unroll
        for (int e = 4; e < 16; e += 4) { a += s[e] + s[e + 1]; b_ += s[e + 2] + s[e + 3]; }
        rest += a + b_;
      }
      if (O::cap || O::wide) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] *= dp[e];
      }
      fit<T, D>(s, up, acc);
#pragma unroll
      for (int kc = 0; kc < 2; ++kc) {
        const typename Ty<T>::x8 hi = pack8<T>(s, kc, up);
#pragma unroll
        for (int db = 0; db < D / 32; ++db) acc[db] = Ty<T>::mfma(frag_tr<T, D>(smem, KA, fo, 2 * kb + kc, db), hi, acc[db]);
        if (two) {
          const typename Ty<T>::x8 lo = pack8_rest<T>(s, kc, up, hi);
#pragma unroll
          for (int db = 0; db < D / 32; ++db) acc[db] = Ty<T>::mfma(frag_tr<T, D>(smem, KA, fo, 2 * kb + kc, db), lo, acc[db]);
        }
      }
    }
    if (t + 1 < t1) landed(slot ^ 1);
  };
  for (int t = 0; t < t1; t += 2) {
    step(iconst<0>{}, t);
    if (t + 1 < t1) step(iconst<1>{}, t + 1);
  }
  rest = xor_sum<32>(rest);
  if (valid && h == 0) {  // for the dK/dV pass
    p.delta[srow_i] = lse2 - Ty<T>::bwd_up;
    p.delta[(long long)p.B * p.H * p.Sq + srow_i] = -(dlt + rest);
  }
  if (valid) {
    const float f = (O::cap ? 4.f * p.scale : p.scale) * (Ty<T>::fits ? 1.f : down(up));
    T* dQ = (T*)p.dq + b * p.dq_bs + q * p.dq_rs + head * D + 4 * h;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        typename Ty<T>::x4 v;
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = (T)(sees ? acc[db][e + u] * f : 0.f);
        *(typename Ty<T>::x4*)(dQ + db * 32 + srow(e)) = v;
      }
  }
}

// ------------------------------------------------------------------------------- dK/dV pass
// key tiles of NW * 32 keys: 4 waves at D = 64, 8 at D = 128 (one block a CU, sharing the Q / dO tiles); with dropout's
// hashes 256 registers are not enough at D = 128
constexpr int dkv_waves(int D, bool drop) { return D == 128 && !drop ? 8 : 4; }
constexpr int dkv_min_waves(int D, bool drop) { return D == 64 ? (drop ? 2 : 3) : (drop ? 1 : 2); }
__device__ __forceinline__ float dk_scale(const Shaped& p) { return shifted(p) ? 4.f * p.scale : p.scale; }  // d tanh's 4
// NW waves of 32 keys; streams the query tiles of all G heads of the group (or, with `splits`, an even share of
// them: then f32 sums go to `part` and shaped_dkv_join_kernel adds them in order). The block's K rows stay in
// LDS instead of registers: at D = 128 the two accumulators take 128 registers, and K's 32 more made the
// compiler spill and wait out every LDS read.
template <typename T, int D, int NW, typename O>
__global__ __launch_bounds__(NW * 64, dkv_min_waves(D, O::drop)) void shaped_dkv_kernel(Shaped p, int splits, float* __restrict__ part) {
  constexpr bool DOCS = O::docs;
  constexpr int TB = KT * D * 2;
  typedef DeadRows<D, NW> Dead;
  __shared__ __attribute__((aligned(1024))) char smem[4 * TB + NW * 64 * D];  // [slot][Q | dO], K
  __shared__ __attribute__((aligned(256))) float stat[2][2][64];  // [slot][lse in log2 units, -delta]
  __shared__ __attribute__((aligned(256))) unsigned marks[DOCS ? 2 * Dead::WORDS : 1];
  __shared__ int range[2][NW];
  const unsigned lds = (unsigned)(size_t)(LDS_AS char*)smem, lds_marks = (unsigned)(size_t)(LDS_AS unsigned*)marks;
  const unsigned lds_stat = (unsigned)(size_t)(LDS_AS float*)&stat[0][0][0];
  const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = l >> 5;
  Offs<D> fo;
  fo.init();
  int col, tile;
  locate(p.B * p.Hk * splits, col, tile);
  const int split = col % splits, inst = col / splits, b = inst / p.Hk, hk = inst % p.Hk;
  const int key = tile * NW * 32 + w * 32 + (l & 31);
  const Mask mk(p, b);
  // the queries that see this lane's key: [qlo, qhi)
  const Span sb = key < p.Sk ? mk.seen_by<DOCS>(key) : Span{0, 0};
  const int qlo = (int)min(max((long long)sb.lo - mk.shift, 0ll), (long long)p.Sq);
  const int qhi = (int)min(max((long long)sb.hi - mk.shift, 0ll), (long long)p.Sq);
  const Reach re(Span{qlo, qhi}, qhi > qlo);
  const bool all_seen = __all(qhi > qlo);
  if (l == 0) { range[0][w] = re.ulo; range[1][w] = re.uhi; }
  __syncthreads();
  int blo = range[0][0], bhi = range[1][0];
#pragma unroll
  for (int u = 1; u < NW; ++u) { blo = min(blo, range[0][u]); bhi = max(bhi, range[1][u]); }
  blo = __builtin_amdgcn_readfirstlane(blo);
  bhi = __builtin_amdgcn_readfirstlane(bhi);
  // tiles from the first query that sees a key of the block (dropout hashes whole quads of queries)
  const int org = bhi > 0 ? (O::drop ? blo & ~3 : blo) : 0, nt = (bhi - org + KT - 1) / KT;
  // this block's share of the (head, tile) sequence
  const long long all = (long long)nt * p.G;
  const int i0 = (int)(all * split / splits), i1 = (int)(all * (split + 1) / splits);

  // the wave's K rows: one address, the k-slots by XOR (8 addresses more would spill)
  int krow = fo.row[0] + 4 * TB + w * 64 * D;
  Dma<D, NW> qm, om;
  qm.init(p.q_rs);
  om.init(p.o_rs);
  int g_next = i0 / max(nt, 1), t_next = i0 % max(nt, 1);  // (head, tile) of the next issue
  // without documents the rows that see nothing are those before position 0 (no prefix)
  const int qa = mk.causal && mk.prefix <= 0 ? -mk.shift : 0;
  auto issue = [&](int slot) {
    const int q0 = org + t_next * KT, head = hk * p.G + g_next, rows = min(bhi - q0, KT);
    qm.issue((const T*)p.q + b * p.q_bs + head * D + q0 * p.q_rs, p.q_rs, rows, lds + slot * 2 * TB);
    om.issue((const T*)p.dout + b * p.o_bs + head * D + q0 * p.o_rs, p.o_rs, rows, lds + slot * 2 * TB + TB);
    // row statistics as they are: lse +inf, delta 0 where a row sees nothing; zeros (with zero rows) from bhi on
    const float* st = p.delta + ((long long)b * p.H + head) * p.Sq + q0;
    const long long n = (long long)p.B * p.H * p.Sq;
    dma_b32(rows_rsrc(st + (w & 1) * n, 4, rows), lds_stat + (slot * 2 + (w & 1)) * 256, l * 4);
    if constexpr (DOCS) Dead::issue(st, 4, 0, rows, 0, qm, lds_marks + slot * Dead::WORDS * 4);
    if (++t_next == nt) {
      t_next = 0;
      ++g_next;
    }
  };
  auto landed = [&](int slot, int q0) {
    dma_wait();
    if (DOCS || q0 < qa) {
#pragma unroll
      for (int i = 0; i < Dead::N; ++i)
        if (DOCS ? Dead::mark(marks + slot * Dead::WORDS, i) == 0x7f800000u : q0 + qm.row(i) < qa) {
          qm.clear(smem + slot * 2 * TB, i);
          om.clear(smem + slot * 2 * TB + TB, i);
        }
    }
    lds_bar();
  };
  if (i0 < i1) {
    {
      Dma<D, NW> km;
      km.init(p.k_rs);
      const int kb = tile * NW * 32;
#pragma unroll
      for (int i = 0; i < NW * 32 / KT; ++i)
        km.issue((const T*)p.k + b * p.k_bs + hk * D + (long long)(kb + i * KT) * p.k_rs, p.k_rs, p.Sk - kb - i * KT,
                 lds + (4 + i) * TB);
    }
    issue(0);
  }
  const int kc_ = min(key, p.Sk - 1);
  const T* Vr = (const T*)p.v + b * p.v_bs + kc_ * p.v_rs + hk * D;
  typename Ty<T>::x8 vf[D / 16];
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    vf[kk] = frag_mem<T>(Vr, kk, true);
  }
  const Score<O> sc(p);
  const int thr = drop_thr(p.p_drop);
  constexpr bool drop = O::drop;
  const float keep = drop ? 256.f / (float)(256 - thr) : 1.f;
  f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) dk[db][e] = dv[db][e] = 0.f;
  constexpr float P_DOWN = Ty<T>::fits ? 1.f : 0x1p-8f;  // 2^-bwd_up: f16's P, and with it dS, is 2^bwd_up times itself
  static_assert(Ty<T>::fits || Ty<T>::bwd_up == 8.f, "P_DOWN");
  float up = START * P_DOWN;
  int g = i0 / max(nt, 1), t = i0 % max(nt, 1);
  if (i0 < i1) landed(0, org + t * KT);
  auto step = [&](auto slot_, int i) {
    constexpr int slot = decltype(slot_)::value, QA = slot * 2 * TB, OA = QA + TB;
    const int q0 = org + t * KT, head = hk * p.G + g;
    if (i + 1 < i1) issue(slot ^ 1);
    const float slope = slope_of<O>(p, head);
    const uint32_t hs = drop ? head_seed(p, b * p.H + head) : 0u;
    const bool full = all_seen && q0 >= re.ilo && q0 + KT <= re.ihi;
    if (q0 < re.uhi && q0 + KT > re.ulo) {  // wave-uniform
#pragma unroll
      for (int qb_ = 0; qb_ < KT / 32; ++qb_) {
          if (D == 128) __builtin_amdgcn_sched_barrier(0);  // one 32-query unit at a time: two overlapped spill
        asm volatile("" : "+v"(krow));
        f32x16 s, dp;  // dP - delta: from -delta of each row
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const f32x4 dl = *(const f32x4*)&stat[slot][1][32 * qb_ + 8 * u + 4 * h];
#pragma unroll
          for (int e = 0; e < 4; ++e) dp[4 * u + e] = dl[e];
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          s = Ty<T>::mfma(frag_row<T, D>(smem, QA, fo, qb_, kk), *(const typename Ty<T>::x8*)(smem + (krow ^ (kk << 5))), s);
          dp = Ty<T>::mfma(frag_row<T, D>(smem, OA, fo, qb_, kk), vf[kk], dp);
        }
        __builtin_amdgcn_sched_barrier(0);  // no transposed reads ahead of the element phase: they would spill
        if (drop) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const unsigned kp = keep4_cols(hs, (q0 + 32 * qb_ + 8 * u + 4 * h) >> 2, p.Sk, key, thr);
            const f32x4 dl = *(const f32x4*)&stat[slot][1][32 * qb_ + 8 * u + 4 * h];
#pragma unroll
            for (int e = 0; e < 4; ++e) dp[4 * u + e] = fmaf((kp & (1u << e)) ? dp[4 * u + e] - dl[e] : 0.f, keep, dl[e]);
          }
        }
        // P in s, dS (capped: / 4) in dp
        const float* Lr = &stat[slot][0][32 * qb_ + 4 * h];
        if (O::bias) {
          const float d0 = (float)(q0 + 32 * qb_ + 4 * h + mk.shift - key);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float x = s[e] * sc.mult;
            if (O::cap) {
              const float r_ = sc.r(s[e]);
              x = sc.c2l * r_;
              dp[e] *= fmaf(-r_, r_, r_);
            }
            if (O::wide) {
              const float t_ = sc.t(s[e]);
              x = sc.cl * t_;
              dp[e] *= fmaf(-t_, t_, 1.f);
            }
            s[e] = ex2(fmaf(-slope, fabsf(d0 + (float)srow(e)), x - Lr[srow(e)]));
            dp[e] *= s[e];
          }
        } else {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if (D == 128) __builtin_amdgcn_sched_barrier(0);  // the quads of statistics one at a time
            const f32x4 L = *(const f32x4*)(Lr + 8 * u);
#pragma unroll
            for (int e = 4 * u; e < 4 * u + 4; ++e) {
              if (O::cap) {
                const float r_ = sc.r(s[e]);
                s[e] = ex2(fmaf(r_, sc.c2l, -L[e & 3]));
                dp[e] *= fmaf(-r_, r_, r_) * s[e];
              } else {
                s[e] = ex2(fmaf(s[e], sc.mult, -L[e & 3]));
                dp[e] *= s[e];
              }
            }
          }
        }
        if (!full) {
          mask_slots(s, (unsigned)(q0 + 32 * qb_ + 4 * h - qlo), (unsigned)(qhi - qlo), 0.f);
          mask_slots(dp, (unsigned)(q0 + 32 * qb_ + 4 * h - qlo), (unsigned)(qhi - qlo), 0.f);
        }
        if (drop) {  // hashed again rather than held across the exponentials (4 registers)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const unsigned kp = keep4_cols(hs, (q0 + 32 * qb_ + 8 * u + 4 * h) >> 2, p.Sk, key, thr);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * u + e] = (kp & (1u << e)) ? s[4 * u + e] : 0.f;
          }
        }
        fit<T, D>(dp, up, dk);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kc = 0; kc < 2; ++kc) {
          const typename Ty<T>::x8 pf = pack8<T>(s, kc), sf = pack8<T>(dp, kc, up);
#pragma unroll
          for (int db = 0; db < D / 32; ++db) {
            dv[db] = Ty<T>::mfma(frag_tr<T, D>(smem, OA, fo, 2 * qb_ + kc, db), pf, dv[db]);
            dk[db] = Ty<T>::mfma(frag_tr<T, D>(smem, QA, fo, 2 * qb_ + kc, db), sf, dk[db]);
          }
        }
      }
    }
    if (++t == nt) {
      t = 0;
      ++g;
    }
    if (i + 1 < i1) landed(slot ^ 1, org + t * KT);
  };
  for (int i = i0; i < i1; i += 2) {
    step(iconst<0>{}, i);
    if (i + 1 < i1) step(iconst<1>{}, i + 1);
  }
  if constexpr (!Ty<T>::fits) {
    const float fk = down(up) * P_DOWN;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        dk[db][e] *= fk;
        dv[db][e] *= P_DOWN;
      }
  }
  if (splits > 1) {
    if (key >= p.Sk) return;
    float* P = part + ((((long long)split * p.B + b) * p.Sk + key) * p.Hk + hk) * 2 * D + 4 * h;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        *(f32x4*)(P + db * 32 + srow(e)) = f32x4{dk[db][e], dk[db][e + 1], dk[db][e + 2], dk[db][e + 3]};
        *(f32x4*)(P + D + db * 32 + srow(e)) = f32x4{dv[db][e], dv[db][e + 1], dv[db][e + 2], dv[db][e + 3]};
      }
    return;
  }
  if (key < p.Sk) {
    T* dK = (T*)p.dk + b * p.dk_bs + key * p.dk_rs + hk * D + 4 * h;
    T* dV = (T*)p.dv + b * p.dv_bs + key * p.dv_rs + hk * D + 4 * h;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        typename Ty<T>::x4 a, c;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          a[u] = (T)(dk[db][e + u] * dk_scale(p));
          c[u] = (T)(dv[db][e + u] * keep);
        }
        *(typename Ty<T>::x4*)(dK + db * 32 + srow(e)) = a;
        *(typename Ty<T>::x4*)(dV + db * 32 + srow(e)) = c;
      }
  }
}

// sums the splits' f32 parts [split][B][Sk][Hk][dk | dv] in order; a thread takes 4 columns
template <typename T, int D>
__global__ __launch_bounds__(256) void shaped_dkv_join_kernel(Shaped p, int splits, const float* __restrict__ part) {
  const long long n = (long long)p.B * p.Sk * p.Hk * (2 * D / 4), i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  f32x4 a = *(const f32x4*)(part + i * 4);
  for (int s = 1; s < splits; ++s) a += *(const f32x4*)(part + (s * n + i) * 4);
  const int c = (int)(i % (2 * D / 4)) * 4;
  const long long row = i / (2 * D / 4);  // (b Sk + key) Hk + hk
  const int hk = (int)(row % p.Hk);
  const long long bk = row / p.Hk;
  const int key = (int)(bk % p.Sk), b = (int)(bk / p.Sk);
  const bool is_k = c < D;
  const float f = is_k ? dk_scale(p) : (p.p_drop > 0.f ? 256.f / (float)(256 - drop_thr(p.p_drop)) : 1.f);
  T* d = is_k ? (T*)p.dk + b * p.dk_bs + key * p.dk_rs + hk * D + c : (T*)p.dv + b * p.dv_bs + key * p.dv_rs + hk * D + c - D;
  typename Ty<T>::x4 v;
#pragma unroll
  for (int u = 0; u < 4; ++u) v[u] = (T)(a[u] * f);
  *(typename Ty<T>::x4*)d = v;
}

// shares of a key tile's queries: about 2 blocks for each of 256 CUs (4 cost B1 H16/4 S8192 D128 50 us more, the
// join's f32 parts), none below 256 queries (forward and backward of B2 H4/1 S1459 D128: 1024 179 us, 512 148,
// 256 138; B4 H8/2 S600 D128: 117, 85, 77)
int dkv_splits(long long blocks, int G, int Sq) {
  return (int)std::max(1ll, std::min((512 + blocks - 1) / blocks, (long long)G * ((Sq + 63) / 64) / 4));
}
template <typename T, int D>
int launch_dq(Shaped p, hipStream_t s) {
  const int waves = row_waves(p, D);
  row_tiles(p, waves * 32);
  const dim3 grid((unsigned)(p.tiles * p.heads * p.B * p.Hk)), block(waves * 64);
  with_rules(p, [&](auto o) {
    constexpr int MAX = max_row_waves<decltype(o)>(D);
    if (waves == MAX) hipLaunchKernelGGL((shaped_dq_kernel<T, D, MAX, decltype(o)>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((shaped_dq_kernel<T, D, 4, decltype(o)>), grid, block, 0, s, p);
  });
  return hipGetLastError() == hipSuccess ? 0 : -1;
}
template <typename T, int D>
int launch_dkv(Shaped p, float* part, hipStream_t s) {
  const int kw = dkv_waves(D, p.p_drop > 0.f), nkt = (p.Sk + kw * 32 - 1) / (kw * 32);
  const int splits = dkv_splits((long long)nkt * p.B * p.Hk, p.G, p.Sq);
  with_rules(p, [&](auto o) {
    constexpr int KW = dkv_waves(D, decltype(o)::drop);
    hipLaunchKernelGGL((shaped_dkv_kernel<T, D, KW, decltype(o)>), dim3((unsigned)(nkt * p.B * p.Hk * splits)), dim3(KW * 64), 0,
                       s, p, splits, part);
  });
  if (splits > 1) {
    const long long n = (long long)p.B * p.Sk * p.Hk * (2 * D / 4);
    hipLaunchKernelGGL((shaped_dkv_join_kernel<T, D>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, p, splits, part);
  }
  return hipGetLastError() == hipSuccess ? 0 : -1;
}
}  // namespace
