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
constexpr int KT = 64;         // streamed rows of a tile
constexpr float RAISE = 8.f;  // log2 units by which a row may outgrow its running maximum

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
  float *lse, *delta;  // delta [2][B][H][Sq]: lse in log2 units, rowsum(dO * O)
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
// one batch's mask: query i at position i + shift sees keys below min(kvl, causal: max(position + 1, prefix))
struct Mask {
  int shift, kvl, prefix;
  bool causal;
  const int2* docs;
  int Sk;
  __device__ __forceinline__ Mask(const Shaped& p, int b) {
    shift = p.q_start ? min(max(p.q_start[b], -(1 << 30)), 1 << 30) : 0;
    kvl = min(p.kv_len ? p.kv_len[b] : p.Sk, p.Sk);
    prefix = p.prefix_len ? p.prefix_len[b] : 0;
    causal = p.causal != 0;
    docs = p.docs ? p.docs + (long long)b * p.Sk : nullptr;
    Sk = p.Sk;
  }
  // d: the document run at the query's position (DOCS)
  template <bool DOCS>
  __device__ __forceinline__ Span of(int q, int2 d) const {
    const int pos = q + shift;
    Span s{0, causal ? min(kvl, max(pos + 1, prefix)) : kvl};
    if (DOCS) {
      s.lo = max(0, d.x);
      s.hi = pos >= 0 && pos < Sk ? min(s.hi, d.y) : 0;
    }
    if (s.hi <= s.lo) s.lo = s.hi = 0;
    return s;
  }
  __device__ __forceinline__ int2 doc_at(int pos) const { return docs[min(max(pos, 0), Sk - 1)]; }
  template <bool DOCS>
  __device__ __forceinline__ Span of(int q) const {
    return of<DOCS>(q, DOCS ? doc_at(q + shift) : int2{0, 0});
  }
  // positions that see key j < Sk: [lo, hi) (superset; the pair test decides)
  template <bool DOCS>
  __device__ __forceinline__ Span seen_by(int j) const {
    Span s{-(1 << 30), 0x7fffffff};
    if (j >= kvl) return Span{0, 0};
    if (DOCS) {
      const int2 d = docs[j];
      if (d.y <= d.x) return Span{0, 0};
      s.lo = d.x;
      s.hi = d.y;
    }
    if (causal && j >= prefix) s.lo = max(s.lo, j);
    return s;
  }
};

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
// Per-lane byte offsets of the fragment reads; row blocks are immediate offsets on top. The swizzle is an
// XOR of chunk bits and the compile-time parts of a chunk index (kk, db) fill bits of their own, so one
// base serves all of them through an XOR (registers: 18 fewer at D = 128 than an offset each).
template <int D>
struct Offs {
  int row;  // row (l & 31), k-slots 8 h ..
  int tr;   // column (l & 31), rows 4 h .. of a 16-row group
  __device__ __forceinline__ void init() {
    const int l = threadIdx.x & 63, h = l >> 5, r = l & 31;
    row = r * (2 * D) + ((h ^ swz<D>(r)) << 4);
    const int li = l & 15, t = 4 * h + (li >> 2), c = 2 * ((l >> 4) & 1) + ((li & 3) >> 1);
    tr = t * (2 * D) + ((c ^ swz<D>(t)) << 4) + (li & 1) * 8;
  }
  // keeps the XORs inside a loop: hoisted, each would hold a register for the whole kernel
  __device__ __forceinline__ void local() { asm volatile("" : "+v"(row), "+v"(tr)); }
};
// rows 32 rb + (l & 31), k-slots 16 kk + 8 h ..
template <typename T, int D>
__device__ __forceinline__ typename Ty<T>::x8 frag_row(const char* lds, const Offs<D>& o, int rb, int kk) {
  return *(const typename Ty<T>::x8*)(lds + (o.row ^ (kk << 5)) + rb * 32 * 2 * D);
}
// X operand of a product over 16 tile rows (16 kc ..): column 32 db + (l & 31); rows 8 + 4 h .. have swz ^ 2
template <typename T, int D>
__device__ __forceinline__ typename Ty<T>::x8 frag_tr(const char* lds, const Offs<D>& o, int kc, int db) {
  typename Ty<T>::x8 r;
  r.lo = Ty<T>::tr(lds + (o.tr ^ (db << 6)) + kc * 16 * 2 * D);
  r.hi = Ty<T>::tr(lds + (o.tr ^ (db << 6) ^ 32) + (kc * 16 + 8) * 2 * D);
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

// A tile of KT rows of D elements from memory straight into the LDS (buffer loads with LDS destination, 16
// bytes a lane): instruction i of wave w fills rows (i NW + w) RPI .. + RPI - 1, the swizzle is in the
// lanes' source addresses. Rows from `rows` on lie past the descriptor's end and arrive as zeros, as do
// rows whose lane is told so (dead). The wave waits for its loads itself (dma_wait) before a barrier
// hands the tile over.
constexpr unsigned OOB = 0x80000000u;
// descriptor of `rows` rows, rb bytes apart, from a block-uniform address
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* base, int rb, int rows) {
  const unsigned long long a = (unsigned long long)base;
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)a), hi = __builtin_amdgcn_readfirstlane((unsigned)(a >> 32));
  return __builtin_amdgcn_make_buffer_rsrc((void*)(((unsigned long long)hi << 32) | lo), (short)0,
                                           __builtin_amdgcn_readfirstlane(rows * rb), 0x00020000);
}
template <int D, int NW>
struct Dma {
  static constexpr int N = KT * D * 2 / (NW * 1024), RPI = 512 / D, STEP = NW * RPI;  // STEP % 16 == 0: one swizzle
  unsigned voff, step;  // lane's byte offset of instruction 0, bytes between instructions
  int row0;
  __device__ __forceinline__ void init(long long rs) {
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
    row0 = w * RPI + l / (D / 8);
    voff = (unsigned)(row0 * (int)rs * 2 + (((l % (D / 8)) ^ swz<D>(row0)) << 4));
    step = (unsigned)(STEP * (int)rs * 2);
  }
  __device__ __forceinline__ int row(int i) const { return row0 + i * STEP; }
  template <typename T, typename Dead>
  __device__ __forceinline__ void issue(const T* base, long long rs, int rows, unsigned lds, Dead dead) const {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const __amdgpu_buffer_rsrc_t rsrc = rows_rsrc(base, (int)rs * 2, max(min(rows, KT), 0));
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const unsigned v = dead(i) ? OOB : voff;
      const unsigned m0 = lds + (i * NW + w) * 1024;
      asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(m0), "v"(v), "s"(rsrc), "s"(__builtin_amdgcn_readfirstlane(i * step)) : "memory");
    }
  }
};
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

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

// what a wave's rows see: union [ulo, uhi) and intersection [ilo, ihi)
struct Reach {
  int ulo, uhi, ilo, ihi;
  __device__ __forceinline__ Reach(const Span& s, bool sees) {
    ulo = wave_min_i(sees ? s.lo : 0x7fffffff);
    uhi = wave_max_i(sees ? s.hi : 0);
    ilo = wave_max_i(sees ? s.lo : 0);
    ihi = wave_min_i(sees ? s.hi : 0x7fffffff);
  }
};
// with documents: which of the lane's rows of the next key tiles belong to none (loaded one tile ahead)
template <int D, int NW, bool DOCS>
struct DeadKeys {
  int2 d[DOCS ? Dma<D, NW>::N : 1];
  __device__ __forceinline__ void load(const Shaped& p, const Dma<D, NW>& m, int b, int row0) {
    if constexpr (DOCS) {
#pragma unroll
      for (int i = 0; i < Dma<D, NW>::N; ++i) d[i] = p.docs[(long long)b * p.Sk + min(row0 + m.row(i), p.Sk - 1)];
    }
  }
  __device__ __forceinline__ bool operator()(int i) const { return DOCS && d[i].y <= d[i].x; }
};

// ------------------------------------------------------------------------------- forward
// NW waves of 32 rows
template <typename T, int D, int NW, bool DOCS>
__global__ __launch_bounds__(NW * 64, 2) void shaped_fwd_kernel(Shaped p) {
  constexpr int TB = KT * D * 2;
  __shared__ __attribute__((aligned(1024))) char smem[4 * TB];
  const unsigned lds = (unsigned)(size_t)(LDS_AS char*)smem;
  __shared__ int range[2][NW];
  const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = l >> 5;
  Offs<D> fo;
  fo.init();
  int inst, tile;
  locate(p, p.tiles, p.causal, inst, tile);
  const int b = inst / p.Hk, hk = inst % p.Hk;
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
  const int t0 = bhi > 0 ? blo / KT : 0, t1 = (bhi + KT - 1) / KT;

  const T* Kb = (const T*)p.k + b * p.k_bs + hk * D;
  const T* Vb = (const T*)p.v + b * p.v_bs + hk * D;
  Dma<D, NW> km, vm;
  km.init(p.k_rs);
  vm.init(p.v_rs);
  DeadKeys<D, NW, DOCS> dead;
  auto issue = [&](int t) {
    km.issue(Kb + (long long)t * KT * p.k_rs, p.k_rs, bhi - t * KT, lds + (t & 1) * TB, [](int) { return false; });
    vm.issue(Vb + (long long)t * KT * p.v_rs, p.v_rs, bhi - t * KT, lds + (2 + (t & 1)) * TB, dead);
  };
  if (t0 < t1) {
    dead.load(p, vm, b, t0 * KT);
    issue(t0);
    dead.load(p, vm, b, (t0 + 1) * KT);
  }
  const T* Qr = (const T*)p.q + b * p.q_bs + qc * p.q_rs + head * D;
  typename Ty<T>::x8 qf[D / 16];
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) qf[kk] = frag_mem<T>(Qr, kk, sees);
  const Score sc(p);
  const float slope = sc.biased ? p.slopes[head] * LOG2E : 0.f;
  const int pos = q + mk.shift;
  const int thr = drop_thr(p.p_drop);
  const bool drop = p.p_drop > 0.f;
  const uint32_t hs = drop ? head_seed(p, b * p.H + head) : 0u;
  const int qg = (q >> 2) * p.Sk;
  float m = -INFINITY, lsum = 0.f;  // lsum: this lane's half of the row
  f32x16 o[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[db][e] = 0.f;
  dma_wait();
  lds_bar();
  for (int t = t0; t < t1; ++t) {
    if (t + 1 < t1) {
      issue(t + 1);
      dead.load(p, vm, b, (t + 2) * KT);
    }
    const int k0 = t * KT;
    const char *K_ = smem + (t & 1) * TB, *V_ = smem + (2 + (t & 1)) * TB;
    if (k0 < re.uhi && k0 + KT > re.ulo) {  // wave-uniform
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
      if (!(k0 >= re.ilo && k0 + KT <= re.ihi)) {
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
      mx = pair_max(mx) * sc.mult;
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
      const float muse = m == -INFINITY ? 0.f : m;
      float rs = 0.f;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float x = ex2(fmaf(s[kb][e], sc.mult, -muse));
          rs += x;
          s[kb][e] = x;
        }
      lsum += rs;
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
    dma_wait();
    lds_bar();
  }
  lsum = xor_sum<32>(lsum);
  if (valid) {
    const float keep = drop ? 256.f / (float)(256 - thr) : 1.f;
    const float inv = sees && lsum != 0.f ? keep / lsum : 0.f;
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
    if (h == 0) p.lse[((long long)b * p.H + head) * p.Sq + q] = sees && lsum != 0.f ? (m + __log2f(lsum)) * LN2 : INFINITY;
  }
}

// ------------------------------------------------------------------------------- dQ pass
// same rows and tiles as the forward; also writes lse in log2 units and delta = rowsum(dO * O)
template <typename T, int D, int NW, bool DOCS>
__global__ __launch_bounds__(NW * 64, 2) void shaped_dq_kernel(Shaped p) {
  constexpr int TB = KT * D * 2;
  __shared__ __attribute__((aligned(1024))) char smem[4 * TB];
  const unsigned lds = (unsigned)(size_t)(LDS_AS char*)smem;
  __shared__ int range[2][NW];
  const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = l >> 5;
  Offs<D> fo;
  fo.init();
  int inst, tile;
  locate(p, p.tiles, p.causal, inst, tile);
  const int b = inst / p.Hk, hk = inst % p.Hk;
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
  const int t0 = bhi > 0 ? blo / KT : 0, t1 = (bhi + KT - 1) / KT;

  const T* Kb = (const T*)p.k + b * p.k_bs + hk * D;
  const T* Vb = (const T*)p.v + b * p.v_bs + hk * D;
  Dma<D, NW> km, vm;
  km.init(p.k_rs);
  vm.init(p.v_rs);
  DeadKeys<D, NW, DOCS> dead;
  auto issue = [&](int t) {
    km.issue(Kb + (long long)t * KT * p.k_rs, p.k_rs, bhi - t * KT, lds + (t & 1) * TB, dead);
    vm.issue(Vb + (long long)t * KT * p.v_rs, p.v_rs, bhi - t * KT, lds + (2 + (t & 1)) * TB, dead);
  };
  if (t0 < t1) {
    dead.load(p, vm, b, t0 * KT);
    issue(t0);
    dead.load(p, vm, b, (t0 + 1) * KT);
  }
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
  const float lse2 = sees ? p.lse[srow_i] * LOG2E : INFINITY;
  if (valid && h == 0) {  // for the dK/dV pass
    p.delta[srow_i] = lse2;
    p.delta[(long long)p.B * p.H * p.Sq + srow_i] = dlt;
  }
  const Score sc(p);
  const float slope = sc.biased ? p.slopes[head] * LOG2E : 0.f;
  const int pos = q + mk.shift;
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
  dma_wait();
  lds_bar();
  for (int t = t0; t < t1; ++t) {
    if (t + 1 < t1) {
      issue(t + 1);
      dead.load(p, vm, b, (t + 2) * KT);
    }
    const char *K_ = smem + (t & 1) * TB, *V_ = smem + (2 + (t & 1)) * TB;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const int k0 = t * KT + 32 * kb;
      if (!(k0 < re.uhi && k0 + 32 > re.ulo)) continue;  // wave-uniform
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
      if (!(k0 >= re.ilo && k0 + 32 <= re.ihi)) {
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
    dma_wait();
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
// NW waves of 32 keys; streams the query tiles of all G heads of the group (or, with `splits`, an even share of
// them: then f32 sums go to `part` and shaped_dkv_join_kernel adds them in order). KL: the block's K rows
// stay in LDS instead of registers -- at D = 128 the two accumulators take 128 registers, and K's 32 more
// made the compiler spill and wait out every LDS read.
template <typename T, int D, int NW, bool DOCS, bool KL>
__global__ __launch_bounds__(NW * 64, 2) void shaped_dkv_kernel(Shaped p, int splits, float* __restrict__ part) {
  constexpr int TB = KT * D * 2;
  __shared__ __attribute__((aligned(1024))) char smem[4 * TB + (KL ? NW * 64 * D : 0)];
  const unsigned lds = (unsigned)(size_t)(LDS_AS char*)smem;
  const char* Kl = smem + 4 * TB;
  __shared__ __attribute__((aligned(256))) float stat[2][2][KT];  // [buffer][lse in log2 units, delta]
  __shared__ int range[2][NW];
  const unsigned lds_stat = (unsigned)(size_t)(LDS_AS float*)&stat[0][0][0];
  const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = l >> 5;
  Offs<D> fo;
  fo.init();
  const int nkt = (p.Sk + NW * 32 - 1) / (NW * 32);
  int inst, tile;
  locate(p, nkt * splits, false, inst, tile);
  const int split = tile % splits;
  tile /= splits;
  const int b = inst / p.Hk, hk = inst % p.Hk;
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
  const int t0 = bhi > 0 ? blo / KT : 0, nt = bhi > 0 ? (bhi + KT - 1) / KT - t0 : 0;
  // this block's share of the (head, tile) sequence
  const long long all = (long long)nt * p.G;
  const int i0 = (int)(all * split / splits), i1 = (int)(all * (split + 1) / splits);

  Dma<D, NW> qm, om;
  qm.init(p.q_rs);
  om.init(p.o_rs);
  int2 dd[DOCS ? Dma<D, NW>::N : 1];  // documents of the next tile's staged rows
  int g_next = i0 / max(nt, 1), t_next = t0 + i0 % max(nt, 1);  // (head, tile) of the next issue
  auto docs_load = [&](int t) {
    if constexpr (DOCS) {
#pragma unroll
      for (int i = 0; i < Dma<D, NW>::N; ++i) dd[i] = mk.doc_at(t * KT + qm.row(i) + mk.shift);
    }
  };
  // without documents the rows that see nothing are those before position 0 (no prefix)
  const int qa = mk.causal && mk.prefix <= 0 ? -mk.shift : 0;
  auto issue = [&](int buf) {
    const int q0 = t_next * KT, head = hk * p.G + g_next;
    auto dead = [&](int i) {  // rows that see nothing arrive as zeros
      const int q = q0 + qm.row(i);
      if (!DOCS) return q < qa;
      const Span s = mk.of<DOCS>(q, dd[i]);
      return s.hi <= s.lo;
    };
    qm.issue((const T*)p.q + b * p.q_bs + head * D + q0 * p.q_rs, p.q_rs, p.Sq - q0, lds + buf * TB, dead);
    om.issue((const T*)p.dout + b * p.o_bs + head * D + q0 * p.o_rs, p.o_rs, p.Sq - q0, lds + (2 + buf) * TB, dead);
    if (w < 2) {  // row statistics as they are: lse +inf, delta 0 where a row sees nothing; zeros (with zero rows) past Sq
      const float* row = p.delta + ((long long)w * p.B * p.H + (long long)b * p.H + head) * p.Sq + q0;
      const __amdgpu_buffer_rsrc_t rsrc = rows_rsrc(row, 4, min(p.Sq - q0, KT));
      asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds_stat + (buf * 2 + w) * KT * 4),
                   "v"(l * 4), "s"(rsrc) : "memory");
    }
    if (++t_next == t0 + nt) {
      t_next = t0;
      ++g_next;
    }
    docs_load(t_next);
  };
  if (i0 < i1) {
    docs_load(t_next);
    issue(0);
    if (KL) {
      Dma<D, NW> km;
      km.init(p.k_rs);
      const int kb = tile * NW * 32;
#pragma unroll
      for (int i = 0; i < NW / 2; ++i)
        km.issue((const T*)p.k + b * p.k_bs + hk * D + (long long)(kb + i * KT) * p.k_rs, p.k_rs, p.Sk - kb - i * KT,
                 lds + (4 + i) * TB, [](int) { return false; });
    }
  }
  const int kc_ = min(key, p.Sk - 1);
  const T* Kr = (const T*)p.k + b * p.k_bs + kc_ * p.k_rs + hk * D;
  const T* Vr = (const T*)p.v + b * p.v_bs + kc_ * p.v_rs + hk * D;
  typename Ty<T>::x8 kf[KL ? 1 : D / 16], vf[D / 16];
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    if constexpr (!KL) kf[kk] = frag_mem<T>(Kr, kk, true);
    vf[kk] = frag_mem<T>(Vr, kk, true);
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
  dma_wait();
  lds_bar();
  int g = i0 / max(nt, 1), t = t0 + i0 % max(nt, 1);
  for (int i = i0; i < i1; ++i) {
    const int buf = (i - i0) & 1, q0 = t * KT, head = hk * p.G + g;
    if (i + 1 < i1) issue(buf ^ 1);
    const char *Q_ = smem + buf * TB, *D_ = smem + (2 + buf) * TB;
    const float slope = sc.biased ? p.slopes[head] * LOG2E : 0.f;
    const uint32_t hs = drop ? head_seed(p, b * p.H + head) : 0u;
    const bool full = all_seen && q0 >= re.ilo && q0 + KT <= re.ihi;
    if (q0 < re.uhi && q0 + KT > re.ulo) {  // wave-uniform
#pragma unroll
      for (int qb_ = 0; qb_ < 2; ++qb_) {
        if (D == 128) fo.local();
        f32x16 s, dp;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = dp[e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          s = Ty<T>::mfma(frag_row<T, D>(Q_, fo, qb_, kk), KL ? frag_row<T, D>(Kl, fo, w, kk) : kf[KL ? 0 : kk], s);
          dp = Ty<T>::mfma(frag_row<T, D>(D_, fo, qb_, kk), vf[kk], dp);
        }
        if (KL) __builtin_amdgcn_sched_barrier(0);  // no transposed reads ahead of the element phase: they would spill
        if (drop) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const unsigned kp = keep4_cols(hs, (q0 + 32 * qb_ + 8 * u + 4 * h) >> 2, p.Sk, key, thr);
#pragma unroll
            for (int e = 0; e < 4; ++e) dp[4 * u + e] = (kp & (1u << e)) ? dp[4 * u + e] * keep : 0.f;
          }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const f32x4 dl = *(const f32x4*)&stat[buf][1][32 * qb_ + 8 * u + 4 * h];
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
          const float sl = sc.capped ? 1.f : p.scale * LOG2E, d0 = (float)(q0 + 32 * qb_ + 4 * h + mk.shift - key);
#pragma unroll
          for (int e = 0; e < 16; ++e) s[e] = fmaf(-slope, fabsf(d0 + (float)srow(e)), s[e] * sl);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const f32x4 L = *(const f32x4*)&stat[buf][0][32 * qb_ + 8 * u + 4 * h];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float pr = ex2(fmaf(s[4 * u + e], sc.mult, -L[e]));
            s[4 * u + e] = pr;
            dp[4 * u + e] *= pr;
          }
        }
        if (!full) {
          const unsigned base = (unsigned)(q0 + 32 * qb_ + 4 * h - qlo), len = (unsigned)(qhi - qlo);
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (base + (unsigned)srow(e) >= len) s[e] = dp[e] = 0.f;
        }
        if (drop) {  // hashed again rather than held across the exponentials (4 registers)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const unsigned kp = keep4_cols(hs, (q0 + 32 * qb_ + 8 * u + 4 * h) >> 2, p.Sk, key, thr);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * u + e] = (kp & (1u << e)) ? s[4 * u + e] : 0.f;
          }
        }
        if (KL) __builtin_amdgcn_sched_barrier(0);
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
    if (++t == t0 + nt) {
      t = t0;
      ++g;
    }
    dma_wait();
    lds_bar();
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
          a[u] = (T)(dk[db][e + u] * p.scale);
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
  const float f = is_k ? p.scale : (p.p_drop > 0.f ? 256.f / (float)(256 - drop_thr(p.p_drop)) : 1.f);
  T* d = is_k ? (T*)p.dk + b * p.dk_bs + key * p.dk_rs + hk * D + c : (T*)p.dv + b * p.dv_bs + key * p.dv_rs + hk * D + c - D;
  typename Ty<T>::x4 v;
#pragma unroll
  for (int u = 0; u < 4; ++u) v[u] = (T)(a[u] * f);
  *(typename Ty<T>::x4*)d = v;
}

// ------------------------------------------------------------------------------- few query rows
// The forward for at most 32 rows (queries x heads of a group): serving's single tokens. All waves of a
// block hold the same rows and divide the keys (8 KiB of K at a time), so the work along the cache is split
// NW ways inside a block and `splits` ways over blocks; each block takes an even share of the keys
// that its rows see (the lengths are device data). Bound by reading K and V once: K goes from memory
// straight into operand registers, V through the wave's own LDS (no block barrier in the loop). The
// waves' (m, l, O) meet in LDS, those of the blocks in shaped_few_join_kernel.
constexpr int FW = 8;  // waves
template <typename T, int D, bool DOCS>
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
  const Mask mk(p, b);
  const Span sp = valid ? mk.of<DOCS>(q) : Span{0, 0};
  const bool sees = sp.hi > sp.lo;
  const Reach re(sp, sees);
  const int a0 = re.uhi > 0 ? re.ulo / KEYS : 0, an = (re.uhi + KEYS - 1) / KEYS - a0, per = (an + splits - 1) / splits;
  const int t1 = a0 + min(an, (split + 1) * per);
  int t = a0 + split * per + w;

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
    const int rows = min(re.uhi - tt * KEYS, KEYS);
    const __amdgpu_buffer_rsrc_t rk = rows_rsrc(Kb + (long long)tt * KEYS * p.k_rs, krs, rows);
    const __amdgpu_buffer_rsrc_t rv = rows_rsrc(Vb + (long long)tt * KEYS * p.v_rs, vrs, rows);
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
        const int2 d = p.docs[(long long)b * p.Sk + min(tt * KEYS + vrow + i * RPI, p.Sk - 1)];
        vdead[i] = d.y <= d.x;
      }
    }
  };
  if (t < t1) load(t);  // (no load past the end: the block barriers behind the loop would wait for it)
  const T* Qr = (const T*)p.q + b * p.q_bs + q * p.q_rs + head * D;
  typename Ty<T>::x8 qf[D / 16];
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) qf[kk] = frag_mem<T>(Qr, kk, sees);
  const Score sc(p);
  const float slope = sc.biased ? p.slopes[head] * LOG2E : 0.f;
  const int pos = q + mk.shift;
  float m = -INFINITY, lsum = 0.f;
  f32x16 o[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[db][e] = 0.f;

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
    for (int i = 0; i < NVV; ++i) {  // rows i RPI + vrow: the swizzle of a row depends on its low 4 bits
      const int row = i * RPI + vrow;
      const u32x4 z = u32x4{0u, 0u, 0u, 0u};
      *(u32x4*)(V_ + row * 2 * D + (((l % (D / 8)) ^ swz<D>(row)) << 4)) = DOCS && vdead[i] ? z : vn[i];
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
    const dim3 gr((unsigned)(inst * splits));
    if (p.docs) hipLaunchKernelGGL((shaped_few_kernel<T, D, true>), gr, dim3(FW * 64), 0, s, p, splits, part);
    else hipLaunchKernelGGL((shaped_few_kernel<T, D, false>), gr, dim3(FW * 64), 0, s, p, splits, part);
    if (splits > 1)
      hipLaunchKernelGGL((shaped_few_join_kernel<T, D>), dim3((unsigned)(inst * p.G * p.Sq)), dim3(64), 0, s, p, splits, part);
    return hipGetLastError() == hipSuccess ? 0 : -1;
  }
  p.tiles = (p.G * p.Sqp + NW * 32 - 1) / (NW * 32);
  const dim3 gr((unsigned)(p.tiles * p.B * p.Hk));
  if (p.docs) hipLaunchKernelGGL((shaped_fwd_kernel<T, D, NW, true>), gr, dim3(NW * 64), 0, s, p);
  else hipLaunchKernelGGL((shaped_fwd_kernel<T, D, NW, false>), gr, dim3(NW * 64), 0, s, p);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}
// key tiles of NW * 32 keys: 4 waves at D = 64 (K and V in registers), 8 at D = 128 (K in LDS, shared Q / dO tiles)
constexpr int dkv_waves(int D) { return D == 128 ? 8 : 4; }
// shares of a key tile's queries: about 4 blocks for each of 256 CUs, none below 16 query tiles
int dkv_splits(long long blocks, int G, int Sq) {
  return (int)std::max(1ll, std::min((1024 + blocks - 1) / blocks, (long long)G * ((Sq + KT - 1) / KT) / 16));
}
template <typename T, int D>
int launch_bwd(Shaped p, float* part, hipStream_t s) {
  constexpr int NW = 4;
  p.tiles = (p.G * p.Sqp + NW * 32 - 1) / (NW * 32);
  constexpr int KW = dkv_waves(D);
  const int nkt = (p.Sk + KW * 32 - 1) / (KW * 32), splits = dkv_splits((long long)nkt * p.B * p.Hk, p.G, p.Sq);
  const dim3 gq((unsigned)(p.tiles * p.B * p.Hk)), gk((unsigned)(nkt * p.B * p.Hk * splits));
  if (p.docs) {
    hipLaunchKernelGGL((shaped_dq_kernel<T, D, NW, true>), gq, dim3(NW * 64), 0, s, p);
    hipLaunchKernelGGL((shaped_dkv_kernel<T, D, KW, true, D == 128>), gk, dim3(KW * 64), 0, s, p, splits, part);
  } else {
    hipLaunchKernelGGL((shaped_dq_kernel<T, D, NW, false>), gq, dim3(NW * 64), 0, s, p);
    hipLaunchKernelGGL((shaped_dkv_kernel<T, D, KW, false, D == 128>), gk, dim3(KW * 64), 0, s, p, splits, part);
  }
  if (splits > 1) {
    const long long n = (long long)p.B * p.Sk * p.Hk * (2 * D / 4);
    hipLaunchKernelGGL((shaped_dkv_join_kernel<T, D>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, p, splits, part);
  }
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
long long tfk_shaped_bwd_ws(const long long* shape) {
  const int D = (int)shape[5], kw = dkv_waves(D) * 32, G = (int)(shape[1] / shape[2]);
  const int splits = dkv_splits((shape[4] + kw - 1) / kw * shape[0] * shape[2], G, (int)shape[3]);
  return splits == 1 ? 0 : splits * shape[0] * shape[4] * shape[2] * 2 * D;
}
// gstrides [dq_bs, dq_rs, dk_bs, dk_rs, dv_bs, dv_rs]; delta: f32 [2, B, H, Sq] scratch
int tfk_shaped_bwd(const void* q, const void* k, const void* v, const void* o, const void* dout, const float* lse,
                   float* delta, void* dq, void* dk, void* dv, int f16_, const long long* shape,
                   const long long* strides, const long long* gstrides, const int* kv_len, const int* q_start,
                   const int* prefix_len, const int* docs, const float* slopes, float scale, float cap, int causal,
                   float p_drop, unsigned long long seed, float* ws, hipStream_t s) {
  Shaped p = params(shape, strides, kv_len, q_start, prefix_len, docs, slopes, scale, cap, causal, p_drop, seed);
  p.q = q; p.k = k; p.v = v; p.o = o; p.dout = dout; p.lse = (float*)lse; p.delta = delta;
  p.dq = dq; p.dk = dk; p.dv = dv;
  p.dq_bs = gstrides[0]; p.dq_rs = gstrides[1]; p.dk_bs = gstrides[2]; p.dk_rs = gstrides[3];
  p.dv_bs = gstrides[4]; p.dv_rs = gstrides[5];
  if (shape[5] == 64) return f16_ ? launch_bwd<f16, 64>(p, ws, s) : launch_bwd<bf16, 64>(p, ws, s);
  return f16_ ? launch_bwd<f16, 128>(p, ws, s) : launch_bwd<bf16, 128>(p, ws, s);
}
int tfk_doc_spans(const int* ids, long long B, int S, int* out, hipStream_t s) {
  if (B <= 0 || S <= 0) return 0;
  hipLaunchKernelGGL(doc_spans_kernel, dim3((unsigned)B), dim3(DT), 0, s, ids, S, (int2*)out);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}
}
