// hipcc-flags: -Xclang -target-feature -Xclang -packed-fp32-ops
// Attention with shaped scores for gfx950: forward, dQ pass, dK/dV pass (flash style, no float atomics).
//
//   s(i, j) = cap tanh(scale q_i.k_j / cap) - slope_h |p_i - j|          (cap, slopes: optional)
//   key j is seen by query i iff lo_i <= j < hi_i;  P = softmax over the seen keys, O = P V
//
// p_i = i + q_start[b] is the query's position among the keys. Every mask here is one interval of keys
// per query: hi = min(kv_len, Sk), causal: hi <= p + 1 or, with a prefix, hi <= max(p + 1, prefix_len);
// documents: [lo, hi) also within the run of the query's document. So a block walks exactly the key
// tiles between its rows' smallest lo and largest hi, a tile that all rows of a wave see needs no mask
// arithmetic, and no [Sq, Sk] mask is read. A query that sees no key gets O = 0 and lse = +inf (its P
// and gradients vanish); rows that no query sees are zeroed on their way into the LDS, so what padding
// holds never meets a product.
//
// Heads: H query heads in Hk groups of G = H / Hk. The forward and dQ passes lay the G heads of a group
// out as G * Sqp rows (queries fastest; Sqp: Sq, padded), so few queries of many heads share one tile;
// the dK/dV pass sums a group's heads in its registers.
//
// Types bf16 / f16, head dim D = 64 / 128, any token and batch strides (multiples of 8 elements).
//
// MFMA mapping (32x32x16, wave64): mfma(X, Y) gives lane l, slot r: sum_k X[(r & 3) + 8 (r >> 2) + 4 (l >> 5)][k]
// * Y[l & 31][k], operand fragments put row (l & 31), k-slots 8 (l >> 5) .. + 7 in lane l. The streamed
// tile is X (rows of K and V, or of Q and dO in the dK/dV pass), the lane's own row is Y: a lane owns one
// query (key), row statistics are lane scalars plus one exchange with lane ^ 32. The slots of two 4-row
// groups are, packed, the k-slots of the next product's Y operand when its X operand (V^T, K^T, dO^T, Q^T)
// is read with the same row order: two ds_read_b64_tr_b16 of rows 4h.. and 8 + 4h.. of each 16.
// LDS rows are D elements, their 16-byte chunks XOR-swizzled (swz): conflict-free for both reads.
#include "common.h"
#include <algorithm>
#include <type_traits>

namespace {
typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int KT = 64;  // streamed rows of a tile

template <typename T>
struct Ty;
template <>
struct Ty<bf16> {
  typedef bf16x8 x8;
  typedef bf16x4 x4;
  static __device__ __forceinline__ f32x16 mfma(x8 x, x8 y, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
  }
  static __device__ __forceinline__ x4 tr(const char* p) { return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((LDS_AS x4*)p); }
};
template <>
struct Ty<f16> {
  typedef f16x8 x8;
  typedef f16x4 x4;
  static __device__ __forceinline__ f32x16 mfma(x8 x, x8 y, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0);
  }
  static __device__ __forceinline__ x4 tr(const char* p) {  // 16-bit elements move as they are
    return __builtin_bit_cast(x4, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((LDS_AS bf16x4*)p));
  }
};

struct Shaped {
  const void *q, *k, *v, *o, *dout;
  void *out, *dq, *dk, *dv;
  float *lse, *delta;
  long long q_bs, k_bs, v_bs, o_bs, dq_bs, dk_bs, dv_bs;  // batch strides (elements)
  long long q_rs, k_rs, v_rs, o_rs, dq_rs, dk_rs, dv_rs;  // token strides
  int B, H, Hk, G, Sq, Sk, Sqp, tiles;                    // tiles: row tiles of one (batch, key head)
  const int *kv_len, *q_start, *prefix_len;               // [B] or null
  const int2* docs;                                       // [B][Sk] document run of each position, or null
  const float* slopes;                                    // [H] or null
  float scale, cap;
  int causal, remap;
  float p_drop;
  unsigned long long seed;
  const unsigned long long* seed_key;
};

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float pair_max(float v) {  // over lanes l, l ^ 32
  float o;
  const float a = lane_swap32(v, o);
  return fmaxf(a, o);
}
// wave-wide integer extremes by DPP and permlane swaps (common.h wave_sum's butterfly)
template <int CTRL>
__device__ __forceinline__ int dpp_i(int v) {
  return __builtin_amdgcn_mov_dpp(v, CTRL, 0xf, 0xf, false);
}
__device__ __forceinline__ int wave_max_i(int v) {
  v = max(v, dpp_i<0xB1>(v));
  v = max(v, dpp_i<0x4E>(v));
  v = max(v, dpp_i<0x141>(v));
  v = max(v, dpp_i<0x140>(v));
  auto a = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);
  v = max((int)a[0], (int)a[1]);
  auto b = __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false);
  return __builtin_amdgcn_readfirstlane(max((int)b[0], (int)b[1]));
}
__device__ __forceinline__ int wave_min_i(int v) { return ~wave_max_i(~v); }
// LDS-only block barrier: the next tile's global loads stay in flight across it
__device__ __forceinline__ void lds_bar() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
template <bool B>
using bconst = std::integral_constant<bool, B>;

// ---- masks
struct Span {
  int lo, hi;  // lo >= hi: sees nothing
};
__device__ __forceinline__ int q_shift(const Shaped& p, int b) {
  return p.q_start ? min(max(p.q_start[b], -(1 << 30)), 1 << 30) : 0;
}
__device__ __forceinline__ Span span_of(const Shaped& p, int b, int q, int shift, int kvl) {
  const int pos = q + shift;
  Span s{0, kvl};
  if (p.causal) s.hi = min(s.hi, p.prefix_len ? max(pos + 1, p.prefix_len[b]) : pos + 1);
  if (p.docs) {
    if (pos >= 0 && pos < p.Sk) {
      const int2 d = p.docs[(long long)b * p.Sk + pos];
      s.lo = max(s.lo, d.x);
      s.hi = min(s.hi, d.y);
    } else {
      s.hi = 0;
    }
  }
  if (s.hi <= s.lo) s.lo = s.hi = 0;
  return s;
}
// positions that see key j: [x, y) (superset; the pair test decides)
__device__ __forceinline__ Span seen_by(const Shaped& p, int b, int j, int kvl) {
  Span s{-(1 << 30), 0x7fffffff};
  if (j >= kvl) return Span{0, 0};
  if (p.docs) {
    const int2 d = p.docs[(long long)b * p.Sk + j];
    if (d.y <= d.x) return Span{0, 0};
    s.lo = d.x;
    s.hi = d.y;
  }
  if (p.causal && !(p.prefix_len && j < p.prefix_len[b])) s.lo = max(s.lo, j);
  return s;
}

// ---- dropout: the mask bytes of attention.hip (one hash per 4 queries and key), see dropout_keep_mask
__device__ __forceinline__ uint32_t head_seed(const Shaped& p, int bh) {
  const unsigned long long s = eff_seed(p.seed, p.seed_key);
  return hash32((uint32_t)s ^ (uint32_t)(s >> 32) ^ ((uint32_t)bh * 0x9E3779B9u));
}
__device__ __forceinline__ int drop_thr(float p) {
  const int t = (int)(p * 256.f + 0.5f);
  return t > 255 ? 255 : t;
}
template <int R>
__device__ __forceinline__ uint32_t qb(uint32_t h) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)h, R * 0x55, 0xf, 0xf, false);
}
// keep bits of this lane's query with keys kb .. kb + 3; a lane quad holds the 4 queries of a group
__device__ __forceinline__ unsigned keep4_rows(uint32_t hs, int qg, int kb, int j, int thr) {
  const uint32_t h = hash32(hs ^ (uint32_t)(qg + kb + j));
  const uint32_t h0 = qb<0>(h), h1 = qb<1>(h), h2 = qb<2>(h), h3 = qb<3>(h);
  const int sh = 8 * j;
  return (((h0 >> sh) & 0xffu) >= (uint32_t)thr ? 1u : 0u) | (((h1 >> sh) & 0xffu) >= (uint32_t)thr ? 2u : 0u) |
         (((h2 >> sh) & 0xffu) >= (uint32_t)thr ? 4u : 0u) | (((h3 >> sh) & 0xffu) >= (uint32_t)thr ? 8u : 0u);
}
// keep bits of this lane's key with queries 4 qg .. + 3
__device__ __forceinline__ unsigned keep4_cols(uint32_t hs, int qg, int Sk, int key, int thr) {
  const uint32_t h = hash32(hs ^ (uint32_t)(qg * Sk + key));
  return ((h & 0xffu) >= (uint32_t)thr ? 1u : 0u) | (((h >> 8) & 0xffu) >= (uint32_t)thr ? 2u : 0u) |
         (((h >> 16) & 0xffu) >= (uint32_t)thr ? 4u : 0u) | ((h >> 24) >= (uint32_t)thr ? 8u : 0u);
}

// ---- LDS tiles: [rows][D], 16-byte chunk c of row r at chunk c ^ swz(r)
template <int D>
__device__ __forceinline__ int swz(int r) {
  return D == 64 ? (((r >> 1) & 1) << 2) | ((r >> 2) & 3) : ((r & 3) << 2) | ((r >> 2) & 3);
}
// per-lane byte offsets of the fragment reads (row blocks are immediate offsets on top)
template <int D>
struct Offs {
  int row[D / 16];     // row (l & 31), k-slots 16 kk + 8 h ..
  int tr[D / 32][2];   // column 32 db + (l & 31), rows 4 h .. and 8 + 4 h .. of a 16-row group
  __device__ __forceinline__ void init() {
    const int l = threadIdx.x & 63, h = l >> 5, r = l & 31;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) row[kk] = r * (2 * D) + (((2 * kk + h) ^ swz<D>(r)) << 4);
    const int li = l & 15, gg = (l >> 4) & 1;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int t = 8 * u + 4 * h + (li >> 2), c = 4 * db + 2 * gg + ((li & 3) >> 1);
        tr[db][u] = t * (2 * D) + ((c ^ swz<D>(t)) << 4) + (li & 1) * 8;
      }
  }
};
template <typename T, int D>
__device__ __forceinline__ typename Ty<T>::x8 frag_row(const char* lds, const Offs<D>& o, int rb, int kk) {
  return *(const typename Ty<T>::x8*)(lds + o.row[kk] + rb * 32 * 2 * D);
}
// X operand of a product over 16 tile rows (16 kc ..): column 32 db + (l & 31)
template <typename T, int D>
__device__ __forceinline__ typename Ty<T>::x8 frag_tr(const char* lds, const Offs<D>& o, int kc, int db) {
  typename Ty<T>::x8 r;
  r.lo = Ty<T>::tr(lds + o.tr[db][0] + kc * 16 * 2 * D);
  r.hi = Ty<T>::tr(lds + o.tr[db][1] + kc * 16 * 2 * D);
  return r;
}
// k-slots 16 kk + 8 h .. of a row in memory, zeros unless ok
template <typename T>
__device__ __forceinline__ typename Ty<T>::x8 frag_mem(const T* row, int kk, bool ok) {
  const int h = (threadIdx.x & 63) >> 5;
  const u32x4 v = *(const u32x4*)(row + kk * 16 + 8 * h);
  const u32x4 z = u32x4{0u, 0u, 0u, 0u};
  return __builtin_bit_cast(typename Ty<T>::x8, ok ? v : z);
}
template <typename T>
__device__ __forceinline__ typename Ty<T>::x8 pack8(const f32x16& a, int half) {
  typename Ty<T>::x8 r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = (T)a[8 * half + e];
  return r;
}

// a tile of KT rows on its way global -> registers -> LDS; rows are clamped into [0, n) for the loads
// and zeroed at the store unless ok
template <int D, int NTH>
struct Stage {
  static constexpr int N = KT * D / 8 / NTH;
  u32x4 v[N];
  bool ok[N];
  static __device__ __forceinline__ int row(int i) { return ((int)threadIdx.x + i * NTH) / (D / 8); }
  static __device__ __forceinline__ int chunk() { return (int)threadIdx.x % (D / 8); }
  template <typename T>
  __device__ __forceinline__ void load(const T* base, long long rs, int row0, int n) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = *(const u32x4*)(base + min(max(row0 + row(i), 0), n - 1) * rs + chunk() * 8);
  }
  __device__ __forceinline__ void store(char* lds) const {
    const u32x4 z = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = row(i);
      *(u32x4*)(lds + r * 2 * D + ((chunk() ^ swz<D>(r)) << 4)) = ok[i] ? v[i] : z;
    }
  }
};
// ok of the staged key rows: inside the block's keys and, with documents, in one
template <int D, int NTH>
__device__ __forceinline__ void key_ok(Stage<D, NTH>& s, const Shaped& p, int b, int row0, int lo, int hi) {
#pragma unroll
  for (int i = 0; i < Stage<D, NTH>::N; ++i) {
    const int j = row0 + s.row(i);
    s.ok[i] = j >= lo && j < hi;
    if (p.docs) {
      const int2 d = p.docs[(long long)b * p.Sk + min(max(j, 0), p.Sk - 1)];
      s.ok[i] = s.ok[i] && d.y > d.x;
    }
  }
}

// ---- scores: raw products s -> log2 units times 1 / mult
struct Score {
  float c2, capl, mult;  // 2 log2e scale / cap, cap log2e, factor left to the exponent
  bool capped, biased;
  __device__ __forceinline__ Score(const Shaped& p) {
    capped = p.cap > 0.f;
    biased = p.slopes != nullptr;
    c2 = capped ? 2.f * LOG2E * p.scale / p.cap : 0.f;
    capl = p.cap * LOG2E;
    mult = capped || biased ? 1.f : p.scale * LOG2E;
  }
  // tanh(s scale / cap) from the native exp2 and reciprocal, saturating through e = inf / 0
  __device__ __forceinline__ float th(float s) const { return 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + ex2(s * c2)); }
};
// slot r of a 32-row block: row (r & 3) + 8 (r >> 2) (+ 4 h)
__device__ __forceinline__ constexpr int srow(int r) { return (r & 3) + 8 * (r >> 2); }

// block -> (key-head instance, row tile); blocks of one instance share an XCD's L2 where there are
// enough instances, later (causal: longer) tiles first
__device__ __forceinline__ void locate(const Shaped& p, int n, bool rev, int& inst, int& tile) {
  const int id = p.remap ? xcd_remap(blockIdx.x, gridDim.x) : (int)blockIdx.x;
  inst = id / n;
  tile = id % n;
  if (rev) tile = n - 1 - tile;
}

// ------------------------------------------------------------------------------- forward
// NW waves of 32 rows
template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64, 2) void shaped_fwd_kernel(Shaped p) {
  constexpr int NTH = NW * 64, TB = KT * D * 2;
  __shared__ __attribute__((aligned(16))) char smem[4 * TB];
  __shared__ int range[2][NW];
  char *Ks = smem, *Vs = smem + 2 * TB;
  const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = l >> 5;
  Offs<D> fo;
  fo.init();
  int inst, tile;
  locate(p, p.tiles, p.causal, inst, tile);
  const int b = inst / p.Hk, hk = inst % p.Hk;
  const int r = tile * NW * 32 + w * 32 + (l & 31), g = r / p.Sqp, q = r % p.Sqp;
  const bool valid = g < p.G && q < p.Sq;
  const int head = hk * p.G + min(g, p.G - 1), qc = min(q, p.Sq - 1);
  const int shift = q_shift(p, b), kvl = min(p.kv_len ? p.kv_len[b] : p.Sk, p.Sk);
  Span sp = valid ? span_of(p, b, q, shift, kvl) : Span{0, 0};
  const bool sees = sp.hi > sp.lo;
  // what the wave's rows see: union and intersection
  const int ulo = wave_min_i(sees ? sp.lo : 0x7fffffff), uhi = wave_max_i(sees ? sp.hi : 0);
  const int ilo = wave_max_i(sees ? sp.lo : 0), ihi = wave_min_i(sees ? sp.hi : 0x7fffffff);
  if (l == 0) { range[0][w] = ulo; range[1][w] = uhi; }
  __syncthreads();
  int blo = range[0][0], bhi = range[1][0];
#pragma unroll
  for (int u = 1; u < NW; ++u) { blo = min(blo, range[0][u]); bhi = max(bhi, range[1][u]); }
  const int t0 = bhi > 0 ? blo / KT : 0, t1 = (bhi + KT - 1) / KT;

  const T* Qr = (const T*)p.q + b * p.q_bs + qc * p.q_rs + head * D;
  const T* Kb = (const T*)p.k + b * p.k_bs + hk * D;
  const T* Vb = (const T*)p.v + b * p.v_bs + hk * D;
  typename Ty<T>::x8 qf[D / 16];
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) qf[kk] = frag_mem<T>(Qr, kk, sees);
  const Score sc(p);
  const float slope = sc.biased ? p.slopes[head] * LOG2E : 0.f;
  const int pos = q + shift;
  const int thr = drop_thr(p.p_drop);
  const bool drop = p.p_drop > 0.f;
  const uint32_t hs = drop ? head_seed(p, b * p.H + head) : 0u;
  const int qg = (q >> 2) * p.Sk;
  float m = -INFINITY, lsum = 0.f;
  f32x16 o[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[db][e] = 0.f;

  Stage<D, NTH> ks, vs;
  auto load = [&](int t) {
    ks.load(Kb, p.k_rs, t * KT, p.Sk);
    vs.load(Vb, p.v_rs, t * KT, p.Sk);
    key_ok(ks, p, b, t * KT, blo, bhi);
#pragma unroll
    for (int i = 0; i < Stage<D, NTH>::N; ++i) vs.ok[i] = ks.ok[i];
  };
  load(t0);
  ks.store(Ks + (t0 & 1) * TB);
  vs.store(Vs + (t0 & 1) * TB);
  load(t0 + 1);
  lds_bar();
  for (int t = t0; t < t1; ++t) {
    const int k0 = t * KT;
    const char *K_ = Ks + (t & 1) * TB, *V_ = Vs + (t & 1) * TB;
    if (k0 < uhi && k0 + KT > ulo) {  // wave-uniform
      f32x16 s[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[kb][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) s[kb] = Ty<T>::mfma(frag_row<T, D>(K_, fo, kb, kk), qf[kk], s[kb]);
      }
      if (sc.capped) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[kb][e] = sc.capl * sc.th(s[kb][e]);
      }
      if (sc.biased) {
        const float sl = sc.capped ? 1.f : p.scale * LOG2E, d0 = (float)(pos - k0 - 4 * h);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[kb][e] = fmaf(-slope, fabsf(d0 - (float)(32 * kb + srow(e))), s[kb][e] * sl);
      }
      if (!(k0 >= ilo && k0 + KT <= ihi)) {
        const unsigned base = (unsigned)(k0 + 4 * h - sp.lo), len = (unsigned)(sp.hi - sp.lo);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (base + (unsigned)(32 * kb + srow(e)) >= len) s[kb][e] = -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[kb][e]);
      mx = pair_max(mx);
      const float mnew = fmaxf(m, mx * sc.mult);
      const float muse = mnew == -INFINITY ? 0.f : mnew;
      const float alpha = ex2(m - muse);
      float rs = 0.f;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float x = ex2(fmaf(s[kb][e], sc.mult, -muse));
          rs += x;
          s[kb][e] = x;
        }
      lsum = fmaf(lsum, alpha, xor_sum<32>(rs));
      m = mnew;
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[db][e] *= alpha;
      if (drop) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            const unsigned kp = keep4_rows(hs, qg, k0 + 32 * kb + srow(e) + 4 * h, q & 3, thr);
#pragma unroll
            for (int u = 0; u < 4; ++u) s[kb][e + u] = (kp & (1u << u)) ? s[kb][e + u] : 0.f;
          }
      }
#pragma unroll
      for (int kc = 0; kc < 4; ++kc) {
        const typename Ty<T>::x8 pf = pack8<T>(s[kc >> 1], kc & 1);
#pragma unroll
        for (int db = 0; db < D / 32; ++db) o[db] = Ty<T>::mfma(frag_tr<T, D>(V_, fo, kc, db), pf, o[db]);
      }
    }
    ks.store(Ks + ((t + 1) & 1) * TB);
    vs.store(Vs + ((t + 1) & 1) * TB);
    load(t + 2);
    lds_bar();
  }
  if (valid) {
    const float keep = drop ? 256.f / (float)(256 - thr) : 1.f;
    const bool any = sees && lsum > 0.f;
    const float inv = sees ? (lsum != 0.f ? keep / lsum : 0.f) : 0.f;
    T* O = (T*)p.out + b * p.o_bs + q * p.o_rs + head * D + 4 * h;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        typename Ty<T>::x4 v;
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = (T)(sees ? o[db][e + u] * inv : 0.f);
        *(typename Ty<T>::x4*)(O + db * 32 + srow(e)) = v;
      }
    if (h == 0) p.lse[((long long)b * p.H + head) * p.Sq + q] = any || lsum != lsum ? (m + __log2f(lsum)) * LN2 : INFINITY;
  }
}

// ------------------------------------------------------------------------------- dQ pass
// same rows and tiles as the forward; also writes delta = rowsum(dO * O) for the dK/dV pass
template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64, D == 128 ? 1 : 2) void shaped_dq_kernel(Shaped p) {
  constexpr int NTH = NW * 64, TB = KT * D * 2;
  __shared__ __attribute__((aligned(16))) char smem[4 * TB];
  __shared__ int range[2][NW];
  char *Ks = smem, *Vs = smem + 2 * TB;
  const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = l >> 5;
  Offs<D> fo;
  fo.init();
  int inst, tile;
  locate(p, p.tiles, p.causal, inst, tile);
  const int b = inst / p.Hk, hk = inst % p.Hk;
  const int r = tile * NW * 32 + w * 32 + (l & 31), g = r / p.Sqp, q = r % p.Sqp;
  const bool valid = g < p.G && q < p.Sq;
  const int head = hk * p.G + min(g, p.G - 1), qc = min(q, p.Sq - 1);
  const int shift = q_shift(p, b), kvl = min(p.kv_len ? p.kv_len[b] : p.Sk, p.Sk);
  Span sp = valid ? span_of(p, b, q, shift, kvl) : Span{0, 0};
  const bool sees = sp.hi > sp.lo;
  const int ulo = wave_min_i(sees ? sp.lo : 0x7fffffff), uhi = wave_max_i(sees ? sp.hi : 0);
  const int ilo = wave_max_i(sees ? sp.lo : 0), ihi = wave_min_i(sees ? sp.hi : 0x7fffffff);
  if (l == 0) { range[0][w] = ulo; range[1][w] = uhi; }
  __syncthreads();
  int blo = range[0][0], bhi = range[1][0];
#pragma unroll
  for (int u = 1; u < NW; ++u) { blo = min(blo, range[0][u]); bhi = max(bhi, range[1][u]); }
  const int t0 = bhi > 0 ? blo / KT : 0, t1 = (bhi + KT - 1) / KT;

  const T* Qr = (const T*)p.q + b * p.q_bs + qc * p.q_rs + head * D;
  const long long orow = b * p.o_bs + qc * p.o_rs + head * D;
  const T* Kb = (const T*)p.k + b * p.k_bs + hk * D;
  const T* Vb = (const T*)p.v + b * p.v_bs + hk * D;
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
  const float lse2 = sees ? p.lse[srow_i] * LOG2E : INFINITY;
  if (valid && h == 0) p.delta[srow_i] = dlt;
  const Score sc(p);
  const float slope = sc.biased ? p.slopes[head] * LOG2E : 0.f;
  const int pos = q + shift;
  const int thr = drop_thr(p.p_drop);
  const bool drop = p.p_drop > 0.f;
  const float keep = drop ? 256.f / (float)(256 - thr) : 1.f;
  const uint32_t hs = drop ? head_seed(p, b * p.H + head) : 0u;
  const int qg = (q >> 2) * p.Sk;
  f32x16 acc[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[db][e] = 0.f;

  Stage<D, NTH> ks, vs;
  auto load = [&](int t) {
    ks.load(Kb, p.k_rs, t * KT, p.Sk);
    vs.load(Vb, p.v_rs, t * KT, p.Sk);
    key_ok(ks, p, b, t * KT, blo, bhi);
#pragma unroll
    for (int i = 0; i < Stage<D, NTH>::N; ++i) vs.ok[i] = ks.ok[i];
  };
  load(t0);
  ks.store(Ks + (t0 & 1) * TB);
  vs.store(Vs + (t0 & 1) * TB);
  load(t0 + 1);
  lds_bar();
  for (int t = t0; t < t1; ++t) {
    const char *K_ = Ks + (t & 1) * TB, *V_ = Vs + (t & 1) * TB;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const int k0 = t * KT + 32 * kb;
      if (!(k0 < uhi && k0 + 32 > ulo)) continue;  // wave-uniform
      f32x16 s, dp;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = dp[e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        s = Ty<T>::mfma(frag_row<T, D>(K_, fo, kb, kk), qf[kk], s);
        dp = Ty<T>::mfma(frag_row<T, D>(V_, fo, kb, kk), df[kk], dp);
      }
      if (drop) {
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const unsigned kp = keep4_rows(hs, qg, k0 + srow(e) + 4 * h, q & 3, thr);
#pragma unroll
          for (int u = 0; u < 4; ++u) dp[e + u] = (kp & (1u << u)) ? dp[e + u] * keep : 0.f;
        }
      }
      if (sc.capped) {  // d tanh = 1 - t^2, folded into dP - delta
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float t_ = sc.th(s[e]);
          s[e] = sc.capl * t_;
          dp[e] = (dp[e] - dlt) * fmaf(-t_, t_, 1.f);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) dp[e] -= dlt;
      }
      if (sc.biased) {
        const float sl = sc.capped ? 1.f : p.scale * LOG2E, d0 = (float)(pos - k0 - 4 * h);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = fmaf(-slope, fabsf(d0 - (float)srow(e)), s[e] * sl);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = ex2(fmaf(s[e], sc.mult, -lse2)) * dp[e];
      if (!(k0 >= ilo && k0 + 32 <= ihi)) {
        const unsigned base = (unsigned)(k0 + 4 * h - sp.lo), len = (unsigned)(sp.hi - sp.lo);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (base + (unsigned)srow(e) >= len) s[e] = 0.f;
      }
#pragma unroll
      for (int kc = 0; kc < 2; ++kc) {
        const typename Ty<T>::x8 sf = pack8<T>(s, kc);
#pragma unroll
        for (int db = 0; db < D / 32; ++db) acc[db] = Ty<T>::mfma(frag_tr<T, D>(K_, fo, 2 * kb + kc, db), sf, acc[db]);
      }
    }
    ks.store(Ks + ((t + 1) & 1) * TB);
    vs.store(Vs + ((t + 1) & 1) * TB);
    load(t + 2);
    lds_bar();
  }
  if (valid) {
    T* dQ = (T*)p.dq + b * p.dq_bs + q * p.dq_rs + head * D + 4 * h;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        typename Ty<T>::x4 v;
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = (T)(sees ? acc[db][e + u] * p.scale : 0.f);
        *(typename Ty<T>::x4*)(dQ + db * 32 + srow(e)) = v;
      }
  }
}

// ------------------------------------------------------------------------------- dK/dV pass
// NW waves of 32 keys; streams the query tiles of all G heads of the group
template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64, D == 128 ? 1 : 2) void shaped_dkv_kernel(Shaped p) {
  constexpr int NTH = NW * 64, TB = KT * D * 2;
  __shared__ __attribute__((aligned(16))) char smem[4 * TB];
  __shared__ __attribute__((aligned(16))) float lse_s[2][KT], dlt_s[2][KT];
  __shared__ __attribute__((aligned(16))) int lo_s[2][KT], hi_s[2][KT];
  __shared__ int tile_s[2][4], range[2][NW];
  char *Qs = smem, *Ds = smem + 2 * TB;
  const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = l >> 5;
  Offs<D> fo;
  fo.init();
  const int nkt = (p.Sk + NW * 32 - 1) / (NW * 32);
  int inst, tile;
  locate(p, nkt, false, inst, tile);
  const int b = inst / p.Hk, hk = inst % p.Hk;
  const int kw = tile * NW * 32 + w * 32, key = kw + (l & 31);
  const int shift = q_shift(p, b), kvl = min(p.kv_len ? p.kv_len[b] : p.Sk, p.Sk);
  const Span sb = seen_by(p, b, key, kvl);
  const bool seen = key < p.Sk && sb.hi > sb.lo;
  {
    const int a = wave_min_i(seen ? sb.lo : 0x7fffffff), z = wave_max_i(seen ? sb.hi : -(1 << 30));
    if (l == 0) { range[0][w] = a; range[1][w] = z; }
  }
  __syncthreads();
  int plo = range[0][0], phi = range[1][0];
#pragma unroll
  for (int u = 1; u < NW; ++u) { plo = min(plo, range[0][u]); phi = max(phi, range[1][u]); }
  // queries of those positions, in tiles of KT
  const long long qlo = max((long long)plo - shift, 0ll), qhi = min((long long)phi - shift, (long long)p.Sq);
  const int t0 = qhi > qlo ? (int)(qlo / KT) : 0, nt = qhi > qlo ? (int)((qhi + KT - 1) / KT) - t0 : 0;
  const int total = nt * p.G;

  const int kc_ = min(key, p.Sk - 1);
  const T* Kr = (const T*)p.k + b * p.k_bs + kc_ * p.k_rs + hk * D;
  const T* Vr = (const T*)p.v + b * p.v_bs + kc_ * p.v_rs + hk * D;
  typename Ty<T>::x8 kf[D / 16], vf[D / 16];
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    kf[kk] = frag_mem<T>(Kr, kk, seen);
    vf[kk] = frag_mem<T>(Vr, kk, seen);
  }
  const Score sc(p);
  const int thr = drop_thr(p.p_drop);
  const bool drop = p.p_drop > 0.f;
  const float keep = drop ? 256.f / (float)(256 - thr) : 1.f;
  f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) dk[db][e] = dv[db][e] = 0.f;

  Stage<D, NTH> qs, ds_;
  float nl = 0.f, nd = 0.f;
  Span ns{0, 0};
  bool nok = false;
  // tile i of the flattened (head, query tile) loop; thread u < KT also carries query row u
  auto load = [&](int i) {
    const int g = min(i / max(nt, 1), p.G - 1), q0 = (t0 + i % max(nt, 1)) * KT, head = hk * p.G + g;
    qs.load((const T*)p.q + b * p.q_bs + head * D, p.q_rs, q0, p.Sq);
    ds_.load((const T*)p.dout + b * p.o_bs + head * D, p.o_rs, q0, p.Sq);
#pragma unroll
    for (int u = 0; u < Stage<D, NTH>::N; ++u) {
      const int q = q0 + qs.row(u);
      Span s = q < p.Sq ? span_of(p, b, q, shift, kvl) : Span{0, 0};
      qs.ok[u] = ds_.ok[u] = s.hi > s.lo;
    }
    if (threadIdx.x < KT) {
      const int q = q0 + (int)threadIdx.x;
      ns = q < p.Sq ? span_of(p, b, q, shift, kvl) : Span{0, 0};
      nok = ns.hi > ns.lo;
      const long long at = ((long long)b * p.H + head) * p.Sq + min(q, p.Sq - 1);
      nl = p.lse[at];
      nd = p.delta[at];
    }
  };
  auto store = [&](int buf) {
    qs.store(Qs + buf * TB);
    ds_.store(Ds + buf * TB);
    if (threadIdx.x < KT) {  // wave 0
      lse_s[buf][threadIdx.x] = nok ? nl * LOG2E : INFINITY;
      dlt_s[buf][threadIdx.x] = nok ? nd : 0.f;
      lo_s[buf][threadIdx.x] = ns.lo;
      hi_s[buf][threadIdx.x] = ns.hi;
      const int a = wave_min_i(nok ? ns.lo : 0x7fffffff), z = wave_max_i(nok ? ns.hi : 0);
      const int c = wave_max_i(nok ? ns.lo : 0), y = wave_min_i(nok ? ns.hi : 0x7fffffff);
      if (threadIdx.x == 0) { tile_s[buf][0] = a; tile_s[buf][1] = z; tile_s[buf][2] = c; tile_s[buf][3] = y; }
    }
  };
  load(0);
  store(0);
  load(1);
  lds_bar();
  for (int i = 0; i < total; ++i) {
    const int g = i / nt, q0 = (t0 + i % nt) * KT, buf = i & 1, head = hk * p.G + g;
    const char *Q_ = Qs + buf * TB, *D_ = Ds + buf * TB;
    const float slope = sc.biased ? p.slopes[head] * LOG2E : 0.f;
    const uint32_t hs = drop ? head_seed(p, b * p.H + head) : 0u;
    const bool any = tile_s[buf][0] < kw + 32 && tile_s[buf][1] > kw;
    const bool full = tile_s[buf][2] <= kw && tile_s[buf][3] >= kw + 32;
    if (any) {
#pragma unroll
      for (int qb_ = 0; qb_ < 2; ++qb_) {
        f32x16 s, dp;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = dp[e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          s = Ty<T>::mfma(frag_row<T, D>(Q_, fo, qb_, kk), kf[kk], s);
          dp = Ty<T>::mfma(frag_row<T, D>(D_, fo, qb_, kk), vf[kk], dp);
        }
        unsigned kp[4];
        if (drop) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            kp[u] = keep4_cols(hs, (q0 + 32 * qb_ + 8 * u + 4 * h) >> 2, p.Sk, key, thr);
#pragma unroll
            for (int e = 0; e < 4; ++e) dp[4 * u + e] = (kp[u] & (1u << e)) ? dp[4 * u + e] * keep : 0.f;
          }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const f32x4 dl = *(const f32x4*)&dlt_s[buf][32 * qb_ + 8 * u + 4 * h];
#pragma unroll
          for (int e = 0; e < 4; ++e) dp[4 * u + e] -= dl[e];
        }
        if (sc.capped) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float t_ = sc.th(s[e]);
            s[e] = sc.capl * t_;
            dp[e] *= fmaf(-t_, t_, 1.f);
          }
        }
        if (sc.biased) {
          const float sl = sc.capped ? 1.f : p.scale * LOG2E, d0 = (float)(q0 + 32 * qb_ + 4 * h + shift - key);
#pragma unroll
          for (int e = 0; e < 16; ++e) s[e] = fmaf(-slope, fabsf(d0 + (float)srow(e)), s[e] * sl);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const f32x4 L = *(const f32x4*)&lse_s[buf][32 * qb_ + 8 * u + 4 * h];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float pr = ex2(fmaf(s[4 * u + e], sc.mult, -L[e]));
            s[4 * u + e] = pr;
            dp[4 * u + e] *= pr;
          }
        }
        if (!full) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const i32x4 lo = *(const i32x4*)&lo_s[buf][32 * qb_ + 8 * u + 4 * h];
            const i32x4 hi = *(const i32x4*)&hi_s[buf][32 * qb_ + 8 * u + 4 * h];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (key < lo[e] || key >= hi[e]) s[4 * u + e] = dp[4 * u + e] = 0.f;
          }
        }
        if (drop) {
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * u + e] = (kp[u] & (1u << e)) ? s[4 * u + e] : 0.f;
        }
#pragma unroll
        for (int kc = 0; kc < 2; ++kc) {
          const typename Ty<T>::x8 pf = pack8<T>(s, kc), sf = pack8<T>(dp, kc);
#pragma unroll
          for (int db = 0; db < D / 32; ++db) {
            dv[db] = Ty<T>::mfma(frag_tr<T, D>(D_, fo, 2 * qb_ + kc, db), pf, dv[db]);
            dk[db] = Ty<T>::mfma(frag_tr<T, D>(Q_, fo, 2 * qb_ + kc, db), sf, dk[db]);
          }
        }
      }
    }
    store(buf ^ 1);
    load(i + 2);
    lds_bar();
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
          a[u] = (T)(dk[db][e + u] * p.scale);
          c[u] = (T)(dv[db][e + u] * keep);
        }
        *(typename Ty<T>::x4*)(dK + db * 32 + srow(e)) = a;
        *(typename Ty<T>::x4*)(dV + db * 32 + srow(e)) = c;
      }
  }
}

// ------------------------------------------------------------------------------- few query rows
// The forward for at most 32 rows (queries x heads of a group): serving's single tokens. All waves of a
// block hold the same rows and divide the keys (8 KiB of K at a time), so the work along the cache is split
// NW ways inside a block and `splits` ways over blocks; each block takes an even share of the keys
// that its rows see (the lengths are device data). Bound by reading K and V once: K goes from memory
// straight into operand registers, V through the wave's own LDS (no block barrier in the loop). The
// waves' (m, l, O) meet in LDS, those of the blocks in shaped_few_join_kernel.
constexpr int FW = 8;  // waves
template <typename T, int D>
__global__ __launch_bounds__(FW * 64, 2) void shaped_few_kernel(Shaped p, int splits, float* __restrict__ part) {
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
  const int shift = q_shift(p, b), kvl = min(p.kv_len ? p.kv_len[b] : p.Sk, p.Sk);
  Span sp = valid ? span_of(p, b, q, shift, kvl) : Span{0, 0};
  const bool sees = sp.hi > sp.lo;
  const int ulo = wave_min_i(sees ? sp.lo : 0x7fffffff), uhi = wave_max_i(sees ? sp.hi : 0);
  const int ilo = wave_max_i(sees ? sp.lo : 0), ihi = wave_min_i(sees ? sp.hi : 0x7fffffff);
  const int a0 = uhi > 0 ? ulo / KEYS : 0, an = (uhi + KEYS - 1) / KEYS - a0, per = (an + splits - 1) / splits;
  const int t1 = a0 + min(an, (split + 1) * per);
  int t = a0 + split * per + w;

  const T* Qr = (const T*)p.q + b * p.q_bs + q * p.q_rs + head * D;
  const T* Kb = (const T*)p.k + b * p.k_bs + hk * D + 8 * h;
  const T* Vb = (const T*)p.v + b * p.v_bs + hk * D;
  typename Ty<T>::x8 qf[D / 16];
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) qf[kk] = frag_mem<T>(Qr, kk, sees);
  const Score sc(p);
  const float slope = sc.biased ? p.slopes[head] * LOG2E : 0.f;
  const int pos = q + shift;
  float m = -INFINITY, lsum = 0.f;
  f32x16 o[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[db][e] = 0.f;

  constexpr int NVV = KEYS * D / 8 / 64;  // 16-byte vectors of V a lane moves
  char* V_ = smem + w * VB;
  u32x4 kn[KB][D / 16], vn[NVV];
  bool vok[NVV];
  auto load = [&](int tt) {
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const T* kr = Kb + min(tt * KEYS + kb * 32 + r, p.Sk - 1) * p.k_rs;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) kn[kb][kk] = *(const u32x4*)(kr + kk * 16);
    }
#pragma unroll
    for (int i = 0; i < NVV; ++i) {
      const int c = l + i * 64, j = tt * KEYS + c / (D / 8), jc = min(j, p.Sk - 1);
      vn[i] = *(const u32x4*)(Vb + jc * p.v_rs + (c % (D / 8)) * 8);
      vok[i] = j >= ulo && j < uhi;
      if (p.docs) {
        const int2 d = p.docs[(long long)b * p.Sk + jc];
        vok[i] = vok[i] && d.y > d.x;
      }
    }
  };
  if (t < t1) load(t);  // (no load past the end: the block barriers behind the loop would wait for it)
  for (; t < t1; t += FW) {
    const int k0 = t * KEYS;
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
    for (int i = 0; i < NVV; ++i) {
      const int c = l + i * 64, row = c / (D / 8);
      const u32x4 z = u32x4{0u, 0u, 0u, 0u};
      *(u32x4*)(V_ + row * 2 * D + (((c % (D / 8)) ^ swz<D>(row)) << 4)) = vok[i] ? vn[i] : z;
    }
    __builtin_amdgcn_wave_barrier();
    if (t + FW < t1) load(t + FW);
    if (sc.capped) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[kb][e] = sc.capl * sc.th(s[kb][e]);
    }
    if (sc.biased) {
      const float sl = sc.capped ? 1.f : p.scale * LOG2E, d0 = (float)(pos - k0 - 4 * h);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[kb][e] = fmaf(-slope, fabsf(d0 - (float)(32 * kb + srow(e))), s[kb][e] * sl);
    }
    if (!(k0 >= ilo && k0 + KEYS <= ihi)) {
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
    const float mnew = fmaxf(m, mx * sc.mult), muse = mnew == -INFINITY ? 0.f : mnew, alpha = ex2(m - muse);
    float rs = 0.f;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[kb][e] = ex2(fmaf(s[kb][e], sc.mult, -muse));
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
      for (int db = 0; db < D / 32; ++db) o[db] = Ty<T>::mfma(frag_tr<T, D>(V_, fo, kc, db), pf, o[db]);
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
  if (splits > 1) {
    float* P = part + ((long long)blockIdx.x * R + r) * D + 4 * h;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *(f32x4*)(P + db * 32 + srow(e)) = f32x4{o[db][e], o[db][e + 1], o[db][e + 2], o[db][e + 3]};
    if (h == 0) {
      float* S = part + (long long)gridDim.x * R * D + ((long long)blockIdx.x * R + r) * 2;
      S[0] = M;
      S[1] = L;
    }
    return;
  }
  const float inv = sees && L != 0.f ? 1.f / L : 0.f;
  T* O = (T*)p.out + b * p.o_bs + q * p.o_rs + head * D + 4 * h;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      typename Ty<T>::x4 v;
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = (T)(sees ? o[db][e + u] * inv : 0.f);
      *(typename Ty<T>::x4*)(O + db * 32 + srow(e)) = v;
    }
  if (h == 0) p.lse[((long long)b * p.H + head) * p.Sq + q] = sees && L != 0.f ? (M + __log2f(L)) * LN2 : INFINITY;
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
  T* O = (T*)p.out + b * p.o_bs + q * p.o_rs + head * D;
#pragma unroll
  for (int u = 0; u < D / 64; ++u) O[u * 64 + l] = (T)(o[u] * inv);
  if (l == 0) p.lse[((long long)b * p.H + head) * p.Sq + q] = L != 0.f ? (M + __log2f(L)) * LN2 : INFINITY;
}

// ------------------------------------------------------------------------------- document runs
// out[b][i] = [first, end) of the run of equal ids around position i; (0, 0) where the id is negative.
// One block per row: each thread scans a segment, the block scans the segments' borders.
constexpr int DT = 1024;
__global__ __launch_bounds__(DT) void doc_spans_kernel(const int* __restrict__ ids, int S, int2* __restrict__ out) {
  __shared__ int first[DT], next[DT];
  const int* x = ids + (long long)blockIdx.x * S;
  int2* y = out + (long long)blockIdx.x * S;
  const int per = (S + DT - 1) / DT, i0 = min(S, (int)threadIdx.x * per), i1 = min(S, i0 + per);
  int f = -1, n = S;  // last and first border (a position whose predecessor differs) of the segment
  for (int i = i0; i < i1; ++i)
    if (i == 0 || x[i] != x[i - 1]) {
      if (f < 0) n = i;
      f = i;
    }
  first[threadIdx.x] = f;
  next[threadIdx.x] = n;
  __syncthreads();
  for (int o = 1; o < DT; o <<= 1) {  // running max of the last borders, running min of the first ones behind
    const int a = (int)threadIdx.x >= o ? first[threadIdx.x - o] : -1;
    const int b = (int)threadIdx.x + o < DT ? next[threadIdx.x + o] : S;
    __syncthreads();
    first[threadIdx.x] = max(first[threadIdx.x], a);
    next[threadIdx.x] = min(next[threadIdx.x], b);
    __syncthreads();
  }
  int cur = threadIdx.x > 0 ? first[threadIdx.x - 1] : 0;
  for (int i = i0; i < i1; ++i) {
    if (i == 0 || x[i] != x[i - 1]) cur = i;
    y[i].x = x[i] < 0 ? 0 : cur;
  }
  int end = threadIdx.x + 1 < DT ? next[threadIdx.x + 1] : S;
  for (int i = i1 - 1; i >= i0; --i) {
    y[i].y = x[i] < 0 ? 0 : end;
    if (i == 0 || x[i] != x[i - 1]) end = i;
  }
}

// few rows and no dropout: the split form; shares of a cache so that there are about 4 blocks for each of
// 256 CUs, none below 512 keys
bool few_rows(int G, int Sq, float p_drop) { return G * (long long)Sq <= 32 && p_drop == 0.f; }
int few_splits(int inst, int Sk) { return std::max(1, std::min((1024 + inst - 1) / inst, Sk / 512)); }
template <typename T, int D>
int launch_fwd(Shaped p, float* part, hipStream_t s) {
  constexpr int NW = 4;
  if (few_rows(p.G, p.Sq, p.p_drop)) {
    const int inst = p.B * p.Hk, splits = few_splits(inst, p.Sk);
    hipLaunchKernelGGL((shaped_few_kernel<T, D>), dim3((unsigned)(inst * splits)), dim3(FW * 64), 0, s, p, splits, part);
    if (splits > 1)
      hipLaunchKernelGGL((shaped_few_join_kernel<T, D>), dim3((unsigned)(inst * p.G * p.Sq)), dim3(64), 0, s, p, splits, part);
    return hipGetLastError() == hipSuccess ? 0 : -1;
  }
  p.tiles = (p.G * p.Sqp + NW * 32 - 1) / (NW * 32);
  hipLaunchKernelGGL((shaped_fwd_kernel<T, D, NW>), dim3((unsigned)(p.tiles * p.B * p.Hk)), dim3(NW * 64), 0, s, p);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}
template <typename T, int D>
int launch_bwd(Shaped p, hipStream_t s) {
  constexpr int NW = 4;
  p.tiles = (p.G * p.Sqp + NW * 32 - 1) / (NW * 32);
  hipLaunchKernelGGL((shaped_dq_kernel<T, D, NW>), dim3((unsigned)(p.tiles * p.B * p.Hk)), dim3(NW * 64), 0, s, p);
  const int nkt = (p.Sk + NW * 32 - 1) / (NW * 32);
  hipLaunchKernelGGL((shaped_dkv_kernel<T, D, NW>), dim3((unsigned)(nkt * p.B * p.Hk)), dim3(NW * 64), 0, s, p);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}
// shape [B, H, Hk, Sq, Sk, D]; strides [q_bs, q_rs, k_bs, k_rs, v_bs, v_rs, o_bs, o_rs]
Shaped params(const long long* shape, const long long* st, const int* kv_len, const int* q_start, const int* prefix_len,
              const int* docs, const float* slopes, float scale, float cap, int causal, float p_drop,
              unsigned long long seed) {
  Shaped p{};
  p.B = (int)shape[0]; p.H = (int)shape[1]; p.Hk = (int)shape[2]; p.Sq = (int)shape[3]; p.Sk = (int)shape[4];
  p.G = p.H / p.Hk;
  p.q_bs = st[0]; p.q_rs = st[1]; p.k_bs = st[2]; p.k_rs = st[3];
  p.v_bs = st[4]; p.v_rs = st[5]; p.o_bs = st[6]; p.o_rs = st[7];
  p.kv_len = kv_len; p.q_start = q_start; p.prefix_len = prefix_len; p.docs = (const int2*)docs; p.slopes = slopes;
  p.scale = scale; p.cap = cap; p.causal = causal; p.p_drop = p_drop; p.seed = seed; p.seed_key = tfk_seed_key();
  // rows of a head: whole tiles where a head has many queries (a tile then walks one head's keys),
  // packed where it has few; dropout hashes quads of queries, so quads stay whole
  p.Sqp = p.Sq >= 64 ? (p.Sq + 127) / 128 * 128 : (p_drop > 0.f ? (p.Sq + 3) / 4 * 4 : p.Sq);
  p.remap = p.B * p.H >= 8;
  return p;
}
}  // namespace

extern "C" {
// f32 words of workspace of a forward (0: none)
long long tfk_shaped_fwd_ws(const long long* shape, float p_drop) {
  const int B = (int)shape[0], Hk = (int)shape[2], G = (int)(shape[1] / shape[2]), Sq = (int)shape[3];
  if (!few_rows(G, Sq, p_drop)) return 0;
  const int splits = few_splits(B * Hk, (int)shape[4]);
  return splits == 1 ? 0 : (long long)B * Hk * splits * G * Sq * (shape[5] + 2);
}
// f16: 0 bf16, 1 f16
int tfk_shaped_fwd(const void* q, const void* k, const void* v, void* out, float* lse, int f16_, const long long* shape,
                   const long long* strides, const int* kv_len, const int* q_start, const int* prefix_len,
                   const int* docs, const float* slopes, float scale, float cap, int causal, float p_drop,
                   unsigned long long seed, float* ws, hipStream_t s) {
  Shaped p = params(shape, strides, kv_len, q_start, prefix_len, docs, slopes, scale, cap, causal, p_drop, seed);
  p.q = q; p.k = k; p.v = v; p.out = out; p.lse = lse;
  if (shape[5] == 64) return f16_ ? launch_fwd<f16, 64>(p, ws, s) : launch_fwd<bf16, 64>(p, ws, s);
  return f16_ ? launch_fwd<f16, 128>(p, ws, s) : launch_fwd<bf16, 128>(p, ws, s);
}
// gstrides [dq_bs, dq_rs, dk_bs, dk_rs, dv_bs, dv_rs]; delta: f32 [B, H, Sq] scratch
int tfk_shaped_bwd(const void* q, const void* k, const void* v, const void* o, const void* dout, const float* lse,
                   float* delta, void* dq, void* dk, void* dv, int f16_, const long long* shape,
                   const long long* strides, const long long* gstrides, const int* kv_len, const int* q_start,
                   const int* prefix_len, const int* docs, const float* slopes, float scale, float cap, int causal,
                   float p_drop, unsigned long long seed, hipStream_t s) {
  Shaped p = params(shape, strides, kv_len, q_start, prefix_len, docs, slopes, scale, cap, causal, p_drop, seed);
  p.q = q; p.k = k; p.v = v; p.o = o; p.dout = dout; p.lse = (float*)lse; p.delta = delta;
  p.dq = dq; p.dk = dk; p.dv = dv;
  p.dq_bs = gstrides[0]; p.dq_rs = gstrides[1]; p.dk_bs = gstrides[2]; p.dk_rs = gstrides[3];
  p.dv_bs = gstrides[4]; p.dv_rs = gstrides[5];
  if (shape[5] == 64) return f16_ ? launch_bwd<f16, 64>(p, s) : launch_bwd<bf16, 64>(p, s);
  return f16_ ? launch_bwd<f16, 128>(p, s) : launch_bwd<bf16, 128>(p, s);
}
int tfk_doc_spans(const int* ids, long long B, int S, int* out, hipStream_t s) {
  if (B <= 0 || S <= 0) return 0;
  hipLaunchKernelGGL(doc_spans_kernel, dim3((unsigned)B), dim3(DT), 0, s, ids, S, (int2*)out);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}
}
