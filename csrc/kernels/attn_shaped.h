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
//
// Bound by arithmetic: an element costs 4 D (dQ: 6 D, dK/dV: 8 D) matrix flops and 9 to 20 vector instructions
// with one or two exponentials, and the two units overlap only between the waves of a SIMD. B1 H16/4 S8192 D128 bf16,
// causal, capped: forward 389 to 408 us (700 TFLOP/s; alone 351), dQ 477 to 505 (850), dK/dV 584 to 616 (920) and 24 of
// its join, as the clock goes; vector unit busy 60 / 54 / 47% of the CUs' busy cycles, matrix unit 34 / 42 / 46%.
// B4 H16 S2048 D64 in documents of about 512: 29, 41 and 53 us, vector unit 56 / 41 / 31%, matrix unit 20 / 23 / 22%: the
// waves wait 42 to 45% of their cycles. A block walks the tiles between its rows' first and last key, of which a wave has
// work in 74% (dK/dV works on 64 queries where 32 would do: 78% of its pairs are needed, 88% by 32).
#pragma once
#include <algorithm>
#include "common.h"
#include <type_traits>

namespace {
typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
template <bool B>
using bconst = std::integral_constant<bool, B>;
template <int I>
using iconst = std::integral_constant<int, I>;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int KT = 64;  // streamed rows of a tile: keys (forward, dQ), queries (dK/dV)

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
  static constexpr bool fits = true;  // has float's exponents
  static constexpr float fwd_up = 0.f, bwd_up = 0.f, raise = 8.f;
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
  static constexpr bool fits = false;   // 2^-14 .. 2^16
  static constexpr float fwd_up = 15.f, bwd_up = 8.f, raise = 3.f;
};

struct Shaped {
  const void *q, *k, *v, *o, *dout;
  void *out, *dq, *dk, *dv;
  float *lse, *delta;  // delta [2][B][H][Sq]: lse in log2 units, -rowsum(dO * O)
  long long q_bs, k_bs, v_bs, o_bs, dq_bs, dk_bs, dv_bs;  // batch strides (elements)
  long long q_rs, k_rs, v_rs, o_rs, dq_rs, dk_rs, dv_rs;  // token strides
  int B, H, Hk, G, Sq, Sk, Sqp;
  int tiles, heads;  // row tiles of a column, columns of one (batch, key head): G where a head fills whole tiles, else 1
  const int *kv_len, *q_start, *prefix_len;               // [B] or null
  const int2* docs;                                       // [B][Sk] document run of each position, or null
  const float* slopes;                                    // [H] or null
  float scale, cap;
  int causal;
  float p_drop;
  unsigned long long seed;
  const unsigned long long* seed_key;
};

// Caps up to here take the shifted form of a score (Score), larger ones the wide form. The shift puts the float32 step of
// cap on every score: f16, S 600, relative error of O (0.00020: rounded once) and absolute one of lse are 0.000256 and 1e-5 at
// a cap of 128, 0.000255 and 4e-5 at 512, 0.000258 and 6e-5 at 1024, 0.00049 and 7e-4 at 1e4, 0.0037 and 8e-3 at 1e5; the
// wide form's 0.000254 and 1e-6 at any cap, for up to half more time (B1 H16/4 S8192 D128 bf16: forward 351 -> 540 us,
// backward 1021 -> 1323). 128 keeps an lse near 0 to 2e-5: half a step of the shift and one of its reciprocal.
constexpr float CAP_SHIFT = 128.f;
__host__ __device__ __forceinline__ bool shifted(const Shaped& p) { return p.cap > 0.f && p.cap <= CAP_SHIFT; }

// the score rules of a call, compiled in: as runtime branches their joins cost the dK/dV pass 40 registers
enum Cap { NONE, SHIFTED, WIDE };
template <bool DOCS, Cap CAP, bool BIAS, bool DROP>
struct Rules {
  static constexpr bool docs = DOCS, cap = CAP == SHIFTED, wide = CAP == WIDE, bias = BIAS, drop = DROP;
};
template <typename F>
void with_rules(const Shaped& p, F f) {
  auto dr = [&](auto docs, auto cap, auto bias) {
    constexpr Cap C = (Cap)decltype(cap)::value;
    if (p.p_drop > 0.f) f(Rules<docs.value, C, bias.value, true>{});
    else f(Rules<docs.value, C, bias.value, false>{});
  };
  auto bi = [&](auto docs, auto cap) {
    if (p.slopes) dr(docs, cap, bconst<true>{});
    else dr(docs, cap, bconst<false>{});
  };
  auto ca = [&](auto docs) {
    if (p.cap > CAP_SHIFT) dr(docs, iconst<WIDE>{}, bconst<true>{});  // slopes: perhaps 0
    else if (p.cap > 0.f) bi(docs, iconst<SHIFTED>{});
    else bi(docs, iconst<NONE>{});
  };
  if (p.docs) ca(bconst<true>{});
  else ca(bconst<false>{});
}

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
  // positions that see key j < Sk: [lo, hi), exactly (documents: runs of document_spans, the same at both of a pair's ends)
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
// Per-lane LDS byte addresses of the fragment reads. Row blocks and the slot of a double-buffered tile are
// immediate offsets on top (the tile loops are unrolled by the slot): no address arithmetic in the loops,
// which are bound by vector instructions.
template <int D>
struct Offs {
  int row[D / 16];    // row (l & 31), k-slots 16 kk + 8 h ..
  int tr[D / 32][2];  // column 32 db + (l & 31), rows 4 h .. and 8 + 4 h .. of a 16-row group
  __device__ __forceinline__ void init() {
    const int l = threadIdx.x & 63, h = l >> 5, r = l & 31;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) row[kk] = r * (2 * D) + (((2 * kk + h) ^ swz<D>(r)) << 4);
    const int li = l & 15, t = 4 * h + (li >> 2), c = 2 * ((l >> 4) & 1) + ((li & 3) >> 1);
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int u = 0; u < 2; ++u)
        tr[db][u] = (t + 8 * u) * (2 * D) + (((4 * db + c) ^ swz<D>(t + 8 * u)) << 4) + (li & 1) * 8;
  }
};
// rows 32 rb + (l & 31), k-slots 16 kk + 8 h .. of the tile at byte `at` of `lds`
template <typename T, int D>
__device__ __forceinline__ typename Ty<T>::x8 frag_row(const char* lds, int at, const Offs<D>& o, int rb, int kk) {
  return *(const typename Ty<T>::x8*)(lds + o.row[kk] + (at + rb * 32 * 2 * D));
}
// X operand of a product over 16 tile rows (16 kc ..): column 32 db + (l & 31)
template <typename T, int D>
__device__ __forceinline__ typename Ty<T>::x8 frag_tr(const char* lds, int at, const Offs<D>& o, int kc, int db) {
  typename Ty<T>::x8 r;
  r.lo = Ty<T>::tr(lds + o.tr[db][0] + (at + kc * 16 * 2 * D));
  r.hi = Ty<T>::tr(lds + o.tr[db][1] + (at + kc * 16 * 2 * D));
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

// f16 operands. The forward's P goes into its product times 2^fwd_up and has whole digits down to 2^-29 of the row's
// maximum (unscaled: 2^-14, and a row that gives most of its weight to one key with a small V lost the rest: 16384 keys
// that share 1%, O off by 0.010 of itself, now 0.0003); less `raise` in the tiled form, the log2 units by which a row may
// outgrow its running maximum before it is rescaled. That is f16's largest, so the maximum is taken one or two steps too
// large (above): the product with the scale rounds, at scores of 1e7 by whole units. The dK/dV pass, whose P comes from
// the rounded lse and may pass 1 by as much, takes 2^bwd_up (whole digits down to 2^-22).
// dS = P (dP - delta) (1 - t^2) goes with 1 / keys and with the upstream gradient: unscaled it left f16's range on long
// rows, for gradients of 1e-3 and smaller (no digits) and of 1e4 (infinite). So a lane's row (dQ) or key (dK) has a
// power of two `up` for its dS, divided out of the f32 sums at the end: from 2^START,
// too large for nearly any row, it falls where an element of the row would pass 2^15, to 2^12 .. 2^13 for that element, and
// the sums so far fall with it. The largest |dS| of a lane's row or key so far is then above 2^12, and what lies 2^26
// below it keeps all its digits. It costs an f16 backward 5 to 11% (B1 H16/4 S8192 D128 capped 1089 -> 1143 us, B2 H16
// S2048 D64 with a bias 116 -> 130).
constexpr float START = 0x1p60f;
template <typename T, int D>
__device__ __forceinline__ void fit(const f32x16& ds, float& up, f32x16 (&acc)[D / 32]) {
  if constexpr (Ty<T>::fits) return;
  float mx = fabsf(ds[0]);
#pragma unroll
  for (int e = 1; e < 16; ++e) mx = fmaxf(mx, fabsf(ds[e]));
  mx = pair_max(mx) * up;
  if (!__any(mx > 0x1p15f)) return;
  const float f = ldexpf(1.f, mx > 0x1p15f ? min(13 - __builtin_amdgcn_frexp_expf(mx), 0) : 0);  // (inf: stays)
  up *= f;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[db][e] *= f;
}
// 1 / up, exactly
__device__ __forceinline__ float down(float up) { return __uint_as_float((254u << 23) - __float_as_uint(up)); }
template <typename T>
__device__ __forceinline__ typename Ty<T>::x8 pack8(const f32x16& a, int half, float up) {
  typename Ty<T>::x8 r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = (T)(Ty<T>::fits ? a[8 * half + e] : a[8 * half + e] * up);
  return r;
}
// what pack8 leaves of a half: a up - pack8(a, up)
template <typename T>
__device__ __forceinline__ typename Ty<T>::x8 pack8_rest(const f32x16& a, int half, float up, typename Ty<T>::x8 hi) {
  typename Ty<T>::x8 r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = (T)((Ty<T>::fits ? a[8 * half + e] : a[8 * half + e] * up) - (float)hi[e]);
  return r;
}

// A tile of KT rows of D elements from memory straight into the LDS (buffer loads with LDS destination, 16
// bytes a lane): instruction i of wave w fills rows (i NW + w) RPI .. + RPI - 1, the swizzle is in the
// lanes' source addresses. Rows from `rows` on lie past the descriptor's end and arrive as zeros.
//
// Tiles are double-buffered: tile t + 1 is issued before tile t's products, each wave waits for its own loads
// behind them (dma_wait), clears rows of its own that nothing sees (DeadRows), and a barrier hands the tile
// over. (Rings of 3 and 4 smaller tiles measured slower: B1 H16/4 S8192 D128 capped 1956 us against 1755.)
// descriptor of `rows` rows, rb bytes apart, from a block-uniform address
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* base, int rb, int rows) {
  const unsigned long long a = (unsigned long long)base;
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)a), hi = __builtin_amdgcn_readfirstlane((unsigned)(a >> 32));
  return __builtin_amdgcn_make_buffer_rsrc((void*)(((unsigned long long)hi << 32) | lo), (short)0,
                                           __builtin_amdgcn_readfirstlane(rows * rb), 0x00020000);
}
__device__ __forceinline__ void dma_b128(__amdgpu_buffer_rsrc_t r, unsigned lds, unsigned voff, unsigned soff) {
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff),
               "s"(r), "s"(__builtin_amdgcn_readfirstlane(soff)) : "memory");
}
__device__ __forceinline__ void dma_b32(__amdgpu_buffer_rsrc_t r, unsigned lds, unsigned voff) {
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(r) : "memory");
}
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
template <int D, int NW>
struct Dma {
  static constexpr int N = KT * D * 2 / (NW * 1024), RPI = 512 / D, STEP = NW * RPI;
  static_assert(N >= 1 && (N == 1 || STEP % 16 == 0), "one swizzle for all instructions of a lane");
  unsigned voff, step;  // lane's byte offset of instruction 0, bytes between instructions
  int row0;
  __device__ __forceinline__ void init(long long rs) {
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
    row0 = w * RPI + l / (D / 8);
    voff = (unsigned)(row0 * (int)rs * 2 + (((l % (D / 8)) ^ swz<D>(row0)) << 4));
    step = (unsigned)(STEP * (int)rs * 2);
  }
  __device__ __forceinline__ int row(int i) const { return row0 + i * STEP; }
  template <typename T>
  __device__ __forceinline__ void issue(const T* base, long long rs, int rows, unsigned lds) const {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const __amdgpu_buffer_rsrc_t rsrc = rows_rsrc(base, (int)rs * 2, max(min(rows, KT), 0));
#pragma unroll
    for (int i = 0; i < N; ++i) dma_b128(rsrc, lds + (i * NW + w) * 1024, voff, i * step);
  }
  // zeros over this lane's piece of instruction i
  __device__ __forceinline__ void clear(char* tile, int i) const {
    *(u32x4*)(tile + (i * NW + (int)(threadIdx.x >> 6)) * 1024 + (threadIdx.x & 63) * 16) = u32x4{0u, 0u, 0u, 0u};
  }
};

// ---- scores: raw products s -> exponents of 2
// plain: x = s scale log2e. Capped: cap tanh(u) = cap - 2 cap r with r = 1 / (1 + e^2u), u = s scale / cap; the
// constant cap shifts a whole row, so x = -2 cap log2e r, and d tanh = 1 - tanh^2 = 4 (r - r^2). Distances add
// -slope log2e |p - j|. (Row statistics between the passes are in these shifted units.)
// Wide caps: x = cap log2e t without a shift, t = tanh(u) to a few of its own steps: the Taylor series up to u^9 where
// |u| < 1/4 (the next term is below 2^-26 of it), else 1 - 2 r of |u| with u's sign.
template <typename O>
struct Score {
  float c2, c2l, mult, base;  // 2 log2e scale / cap, -2 cap log2e, scale log2e, the shift
  float cu, cl;               // wide: scale / cap, cap log2e
  __device__ __forceinline__ Score(const Shaped& p) {
    mult = p.scale * LOG2E;
    c2 = O::cap ? fminf(2.f * mult / p.cap, 3.4e38f) : 0.f;
    base = O::cap ? p.cap * LOG2E : 0.f;
    c2l = -2.f * base;
    const float wide = fminf(p.cap, 1e30f);  // (leaves any score below 1e26 alone)
    cu = O::wide ? p.scale / wide : 0.f;
    cl = O::wide ? wide * LOG2E : 0.f;
  }
  __device__ __forceinline__ float t(float s) const {
    const float u = s * cu, w = u * u;
    const float series = fmaf(w, fmaf(w, fmaf(w, fmaf(w, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
    const float far = fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + ex2(fabsf(u) * (2.f * LOG2E))), 1.f);
    return fabsf(u) < 0.25f ? u * series : copysignf(far, u);
  }
  // a score without its distance
  __device__ __forceinline__ float x(float s) const { return O::wide ? cl * t(s) : O::cap ? c2l * r(s) : s * mult; }
  // native exp2 and reciprocal: saturates through e = inf (r = 0) and e = 0 (r = 1)
  __device__ __forceinline__ float r(float s) const { return __builtin_amdgcn_rcpf(1.f + ex2(s * c2)); }
};
template <typename O>
__device__ __forceinline__ float slope_of(const Shaped& p, int head) {
  return O::bias && (!O::wide || p.slopes) ? p.slopes[head] * LOG2E : 0.f;
}
// a maximum that no score passes by rounding, where P goes up to f16's largest
template <typename T>
__device__ __forceinline__ float above(float m) {
  return Ty<T>::fits ? m : fmaf(fminf(fabsf(m), 1e30f), 0x1p-23f, m);
}
// slot r of a 32-row block: row (r & 3) + 8 (r >> 2) (+ 4 h)
__device__ __forceinline__ constexpr int srow(int r) { return (r & 3) + 8 * (r >> 2); }

// slots whose row is not in [0, len) from `base` take v. `base` is made opaque so that the compares stay inside the
// branch of the partly visible tiles (hoisted, they cost every tile 32 instructions).
__device__ __forceinline__ void mask_slots(f32x16& s, unsigned base, unsigned len, float v) {
  asm volatile("" : "+v"(base));
#pragma unroll
  for (int e = 0; e < 16; ++e) s[e] = base + (unsigned)srow(e) < len ? s[e] : v;
}

// Blocks of one launch: the tile's rank is the slow index, the columns (head instances) the fast one. Consecutive
// blocks go round the 8 XCDs, so a column stays on one XCD (8 divides their number, usually) and its K / V in
// that XCD's L2, every XCD and CU gets tiles of all ranks, and the long ones (causal: the last rows, the
// first keys) start first. (A column's tiles side by side instead: CUs were idle 57% of a packed-document
// forward, the tiles of one CU being all long or all short.)
__device__ __forceinline__ void locate(int columns, int& column, int& rank) {
  rank = (int)blockIdx.x / columns;
  column = (int)blockIdx.x % columns;
}

// waves of 32 rows in a block of the forward and of the dQ pass. 4; 8, which read each key tile once instead of twice, at
// D = 128, where a CU holds 8 waves, if their blocks are two full rounds of the 256 CUs (449 .. 512) of 3584 queries or
// more: blocks are long then, and every CU gets a long and a short one. Forward / backward in us, 4 -> 8 waves, causal bf16:
//   two rounds:   S7424 H16 238 / 804 -> 225 / 792, S8192 H16 288 / 918 -> 268 / 897 (cap 30: 366 / 1074 -> 351 / 1048),
//                 S32000 H4 1067 / 3337 -> 984 / 3252, S4096 H32 151 / 502 -> 143 / 497
//   other counts: S4096 H16 96 / 301 -> 110 / 322, S6144 163 / 565 -> 179 / 589, S10240 426 / 1450 -> 442 / 1481 (cap 30:
//                 535 / 1679 -> 582 / 1735), S12288 604 / 2036 -> 618 / 2060, S16384 within 3% either way
//   short rows:   S1024 B8 H16 52 / 201 -> 54 / 208, S2048 H64 cap 30 102 / 331 -> 104 / 335
//   documents:    S8192 H16 134 / 409 -> 140 / 411 (cap 30: 148 / 445 -> 177 / 477); cap and bias: 404 / 1175 -> 441 / 1158
// (At D = 64, with 12 to 16 waves a CU, 8 were slower: forward 27.8 -> 30.1, dQ 35.4 -> 44.5 for B4 H16 S2048 in documents
// of about 512.) Dropout's and wide caps' instances keep 4.
template <typename O>
__host__ __device__ constexpr int max_row_waves(int D) {
  return D == 128 && !O::drop && !O::docs && !O::wide && !(O::cap && O::bias) ? 8 : 4;
}
inline int row_waves(const Shaped& p, int D) {
  const bool has = D == 128 && p.p_drop == 0.f && !p.docs && p.cap <= CAP_SHIFT && !(p.cap > 0.f && p.slopes);
  const long long blocks = p.B * (long long)p.H * ((p.Sq + 255) / 256);
  return has && p.Sq >= 3584 && blocks > 448 && blocks <= 512 ? 8 : 4;
}

inline void row_tiles(Shaped& p, int rows) {
  p.heads = p.Sqp % rows == 0 ? p.G : 1;
  p.tiles = (p.G / p.heads * p.Sqp + rows - 1) / rows;
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
// With documents: one 4-byte mark for each staged row of the lane, loaded into the wave's own LDS words
// beside the tile; rows whose mark says that nothing sees them are cleared.
template <int D, int NW>
struct DeadRows {
  static constexpr int N = Dma<D, NW>::N, WORDS = N * NW * 64;  // of one slot
  // marks at base[row * stride_b bytes + at], rows outside [0, rows) read 0
  static __device__ __forceinline__ void issue(const void* base, int stride, int at, int rows, int row0, const Dma<D, NW>& m, unsigned lds) {
    const __amdgpu_buffer_rsrc_t r = rows_rsrc(base, stride, rows);
    const int w = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < N; ++i) dma_b32(r, lds + (i * NW + w) * 256, (unsigned)((row0 + m.row(i)) * stride + at));
  }
  static __device__ __forceinline__ unsigned mark(const unsigned* slot, int i) { return slot[(i * NW) * 64 + threadIdx.x]; }
};
}  // namespace
