// hipcc-flags: -Xclang -target-feature -Xclang -packed-fp32-ops
// Log probabilities of given tokens, with the entropy of each row's distribution and its k most
// probable tokens, and their gradient, for gfx950.
//
// For a row x of V logits: lse = m + ln S, S = sum e^(x - m), m = max x;
//   logp = (x[id] - m) - ln S,   entropy = lse - sum p x = ln S - Y / S with Y = sum (x - m) e^(x - m).
// m and ln S are kept apart for the backward (norm): lse alone loses ln S where |m| is large (a row whose
// logits all are a mask value).
// Gradient of the row, with the incoming gl (logp), gh (entropy) and gt[j] (the alternatives):
//   dx[v] = gl [v == id] + sum_j gt[j] [v == top[j]] - p (gl + sum_j gt[j] + gh (ln p + entropy)).
//
// Both directions read each logit once (memory bound). The forward cuts a row into parts of at most
// NT * NV 16-byte vectors; a part lives in the registers of one block, which reduces it to (m, S, Y) and
// its k best, and a second launch joins the parts of a row (a row of one part is finished at once).
// So a few long rows fill the card as many short ones do. f32 sums throughout. 8192 rows of 33708 bf16 logits:
// forward 116 to 127 us (4.5 TB/s), backward 173 to 180 us (6.2 TB/s); 1021 rows of 131072 f32 logits with 5
// alternatives 100 us (5.3 TB/s).
#include <algorithm>
#include "common.h"

namespace {
typedef _Float16 f16;
typedef unsigned long long u64;
constexpr int NT = 256, NW = NT / 64;
constexpr int NV = 8;   // 16-byte vectors a thread of the forward holds
constexpr int BNV = 2;  // and of the backward, which needs no statistics of its part: 181 -> 169 us against 8
constexpr int KMAX = 32;
constexpr float LOG2E = 1.4426950408889634f;

// 16 bytes at any element-aligned address
typedef u32x4 __attribute__((aligned(2))) u32x4_any;

template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  union {
    u32x4 raw;
    T e[N];
  };
  __device__ __forceinline__ float at(int i) const { return (float)e[i]; }
};
__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

// values and places as one sortable word: larger value first, then the lower column
__device__ __forceinline__ u64 order_key(float x, int col) {
  const unsigned u = __float_as_uint(x + 0.f);  // -0 and +0 tie
  const unsigned o = u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
  return ((u64)o << 32) | (unsigned)~col;
}
__device__ __forceinline__ int key_col(u64 k) { return (int)~(unsigned)k; }
__device__ __forceinline__ float key_val(u64 k) {
  const unsigned o = (unsigned)(k >> 32);
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ u64 wave_max64(u64 v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const u64 x = __shfl_xor(v, o, 64);
    v = x > v ? x : v;
  }
  return v;
}

struct Stat {  // m, S, Y of a set of logits (m = -inf: none)
  float m, s, y;
};
__device__ __forceinline__ Stat join(const Stat& a, const Stat& b) {
  Stat r;
  r.m = fmaxf(a.m, b.m);
  // an empty side has s = y = 0; beyond e^-1e4 a side weighs nothing (and 0 * (inf) must not arise)
  const float da = a.m == -INFINITY ? 0.f : fmaxf(a.m - r.m, -1e4f), db = b.m == -INFINITY ? 0.f : fmaxf(b.m - r.m, -1e4f);
  const float ea = ex2(da * LOG2E), eb = ex2(db * LOG2E);
  r.s = a.s * ea + b.s * eb;
  r.y = (a.y + da * a.s) * ea + (b.y + db * b.s) * eb;
  return r;
}

// all parts of a row, by one wave: a lane a part (loads in flight together), then a tree in a fixed order
__device__ __forceinline__ Stat join_parts(const Stat* ps, int parts) {
  const int l = threadIdx.x & 63;
  Stat st{-INFINITY, 0.f, 0.f};
  for (int u = l; u < parts; u += 64) st = join(st, ps[u]);
  for (int o = 1; o < min(parts, 64); o <<= 1) {
    Stat b;
    b.m = __shfl_down(st.m, o, 64);
    b.s = __shfl_down(st.s, o, 64);
    b.y = __shfl_down(st.y, o, 64);
    if (l + o < 64) st = join(st, b);
  }
  st.m = __shfl(st.m, 0, 64);
  st.s = __shfl(st.s, 0, 64);
  st.y = __shfl(st.y, 0, 64);
  return st;
}

struct FwdParams {
  const void* x;
  const int* ids;
  long long ld;
  int V, T, k, ignore, parts, per;  // per: 16-byte vectors of a part
  float *logp, *ent, *lse, *norm, *top_logp;  // norm [T][2]: m (-inf: no class), ln S
  int* top_ids;
  Stat* pstat;  // [T][parts]
  u64* pkeys;   // [T][parts][k]
};
__device__ __forceinline__ float log_p(float x, float m, float ls) { return m == -INFINITY ? -INFINITY : (x - m) - ls; }
// the given token: its column (-1: none) and, loaded ahead of the reductions, its logit. In a row of several
// parts the part with the column leaves the logit in logp for the join, whose loads then all go out at once
__device__ __forceinline__ int given(const FwdParams& p, int row) {
  const int id = p.ids[row];
  return id != p.ignore && (unsigned)id < (unsigned)p.V ? id : -1;
}
__device__ __forceinline__ void write_row(const FwdParams& p, int row, const Stat& st, int id, float x) {
  const bool any = !(st.s == 0.f);  // false: every logit is -inf
  const float ls = any ? logf(st.s) : 0.f, m = any ? st.m : -INFINITY;
  p.norm[2ll * row] = m;
  p.norm[2ll * row + 1] = ls;
  p.lse[row] = m + ls;
  p.ent[row] = any ? ls - st.y / st.s : 0.f;
  p.logp[row] = id >= 0 ? log_p(x, m, ls) : 0.f;
}
__device__ __forceinline__ void write_top(const FwdParams& p, int row, int j, u64 key, const Stat& st, float ls) {
  p.top_ids[(long long)row * p.k + j] = key_col(key);
  p.top_logp[(long long)row * p.k + j] = st.s == 0.f ? -INFINITY : log_p(key_val(key), st.m, ls);
}

template <typename T>
__device__ __forceinline__ void load_vec(Vec<T>& v, const T* x, int i, int V) {
  constexpr int N = Vec<T>::N;
  if ((i + 1) * N <= V) {
    v.raw = *(const u32x4_any*)(x + i * N);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) v.e[e] = i * N + e < V ? x[i * N + e] : (T)-INFINITY;
  }
}

// The k best of a part. Each wave finds the k-th largest of its 64 lane maxima by bisection over the bits of
// the ordered value; the largest of these over the block bounds the part's k-th best from below, so the
// few logits that are not below it hold the answer. They are listed in LDS and ranked by counting the
// larger keys. Where the list overflows (hundreds of equal logits) k rounds of a block maximum decide,
// over the part read again (its registers would cost every call occupancy: 152 VGPRs instead of 93).
constexpr int CAND = 1024;
struct TopShared {
  u64 key[CAND];
  u64 wkey[2][NW];
  float bound[NW];
  int n;
};
template <typename T, typename Put>
__device__ __forceinline__ void top_k(const Vec<T> (&v)[NV], const T* x, int V, int v0, int v1, float lane_max, int k,
                                      TopShared& sh, Put put) {
  constexpr int N = Vec<T>::N;
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int lim = min(V, v1 * N);
  const unsigned om = v0 + (int)threadIdx.x < v1 ? (unsigned)(order_key(lane_max, 0) >> 32) : 0u;
  unsigned t = 0;
#pragma unroll
  for (int bit = 31; bit >= 0; --bit) {
    const unsigned c = t | (1u << bit);
    if (__popcll(__ballot(om >= c)) >= k) t = c;
  }
  if (l == 0) sh.bound[w] = t == 0 ? -INFINITY : key_val((u64)t << 32);
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  float bound = sh.bound[0];
#pragma unroll
  for (int u = 1; u < NW; ++u) bound = fmaxf(bound, sh.bound[u]);
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    if (c * NT >= v1 - v0) break;
    float m = v[c].at(0);
#pragma unroll
    for (int e = 1; e < N; ++e) m = fmaxf(m, v[c].at(e));
    // !(x < bound): NaN counts as largest (a vector of NaN only has m = NaN)
    if (!(m < bound) || m != m) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int col = (v0 + c * NT + (int)threadIdx.x) * N + e;
        if (!(v[c].at(e) < bound) && col < lim) {
          const int at = atomicAdd(&sh.n, 1);
          if (at < CAND) sh.key[at] = order_key(v[c].at(e), col);
        }
      }
    }
  }
  __syncthreads();
  const int n = sh.n;
  if (n <= CAND) {
    for (int i = threadIdx.x; i < n; i += NT) {
      const u64 key = sh.key[i];
      int r = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) r += sh.key[j] > key ? 1 : 0;
      if (r < k) put(r, key);
    }
    for (int j = n + (int)threadIdx.x; j < k; j += NT) put(j, 0ull);  // a part shorter than k
    return;
  }
  u64 prev = ~0ull;
  for (int j = 0; j < k; ++j) {
    u64 best = 0;
    for (int i = v0 + (int)threadIdx.x; i < v1; i += NT) {
      Vec<T> y;
      load_vec<T>(y, x, i, V);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int col = i * N + e;
        const u64 key = col < lim ? order_key(y.at(e), col) : 0;
        best = key < prev && key > best ? key : best;
      }
    }
    best = wave_max64(best);
    if (l == 0) sh.wkey[j & 1][w] = best;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < NW; ++u) best = sh.wkey[j & 1][u] > best ? sh.wkey[j & 1][u] : best;
    prev = best;
    if (threadIdx.x == 0) put(j, best);
  }
}

template <typename T, bool TOP>
__global__ __launch_bounds__(NT) void logprobs_fwd_kernel(FwdParams p) {
  constexpr int N = Vec<T>::N;
  __shared__ Stat wst[NW];
  const int row = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  const T* x = (const T*)p.x + (long long)row * p.ld;
  const int nvec = (p.V + N - 1) / N, v0 = part * p.per, v1 = min(nvec, v0 + p.per);
  const int id = given(p, row);
  Vec<T> v[NV];
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    const int i = v0 + c * NT + (int)threadIdx.x;
    if (i < v1) {
      load_vec<T>(v[c], x, i, p.V);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) v[c].e[e] = (T)-INFINITY;
    }
  }
  const float xid = id >= v0 * N && id < v1 * N ? (float)x[id] : 0.f;
  float m = -INFINITY;
#pragma unroll
  for (int c = 0; c < NV; ++c)
#pragma unroll
    for (int e = 0; e < N; ++e) m = fmaxf(m, v[c].at(e));
  Stat st;
  st.m = wave_max(m);
  const float ref = st.m == -INFINITY ? 0.f : st.m;
  st.s = st.y = 0.f;
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    if (c * NT >= p.per) break;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float d = v[c].at(e) - ref;
      const float ee = ex2(d * LOG2E);
      st.s += ee;
      st.y = fmaf(fmaxf(d, -1e30f), ee, st.y);  // -inf: 0 * -1e30, not 0 * -inf
    }
  }
  st.s = wave_sum(st.s);
  st.y = wave_sum(st.y);
  if (l == 0) wst[w] = st;
  __syncthreads();
  st = wst[0];
#pragma unroll
  for (int u = 1; u < NW; ++u) st = join(st, wst[u]);
  if (threadIdx.x == 0) {
    if (p.parts == 1) {
      write_row(p, row, st, id, xid);
    } else {
      p.pstat[(long long)row * p.parts + part] = st;
      if (id >= v0 * N && id < v1 * N) p.logp[row] = xid;
    }
  }
  if constexpr (TOP) {
    __shared__ TopShared sh;
    const float ls = st.s == 0.f ? 0.f : logf(st.s);
    top_k<T>(v, x, p.V, v0, v1, m, p.k, sh, [&](int j, u64 key) {
      if (p.parts == 1) write_top(p, row, j, key, st, ls);
      else p.pkeys[((long long)row * p.parts + part) * p.k + j] = key;
    });
  }
}

// One block per row: joins its parts, and picks the k best of their parts * k candidates. The parts' lists are
// in order: where t parts have their m-th key at or above a value, t m >= k candidates are, so candidates below
// the t-th largest of the m-th keys are out (t about half the parts), and the rest, little more than k, are
// ranked by counting the larger ones (all 340 of 17 parts: 5.6 -> 11 us for 8 rows). Where more than JT stay, all
// candidates are ranked, JT at a time.
constexpr int JT = 1024;
template <typename T, bool TOP>
__global__ __launch_bounds__(TOP ? NT : 64) void logprobs_join_kernel(FwdParams p) {
  const int row = blockIdx.x;
  const int id = given(p, row);
  const float xid = p.logp[row];
  const Stat* ps = p.pstat + (long long)row * p.parts;
  if constexpr (TOP) {
    __shared__ u64 keys[JT];
    __shared__ int count;
    const int n = p.parts * p.k;
    const u64* pk = p.pkeys + (long long)row * n;
    const u64 first = (int)threadIdx.x < n ? pk[threadIdx.x] : 0;
    const int np = min(p.parts, 64), m = min(p.k, (2 * p.k + np - 1) / np), t = (p.k + m - 1) / m;
    const int l = threadIdx.x & 63;
    const u64 mine = l < np ? pk[l * p.k + m - 1] : 0;
    const Stat st = join_parts(ps, p.parts);
    int above = 0;
    for (int u = 0; u < np; ++u) above += (u64)__shfl(mine, u, 64) > mine ? 1 : 0;
    const unsigned long long at_t = __ballot(l < np && above == t - 1);  // no lane, or keys of 0: no bound
    const u64 bound = at_t ? (u64)__shfl(mine, __ffsll(at_t) - 1, 64) : 0;
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += NT) {
      const u64 key = i < NT ? first : pk[i];
      if (key != 0 && key >= bound) {
        const int at = atomicAdd(&count, 1);
        if (at < JT) keys[at] = key;
      }
    }
    if (threadIdx.x == 0) write_row(p, row, st, id, xid);
    const float ls = st.s == 0.f ? 0.f : logf(st.s);
    __syncthreads();
    const int found = count;
    if (found <= JT) {
      for (int i = threadIdx.x; i < found; i += NT) {
        const u64 key = keys[i];
        int r = 0;
#pragma unroll 4
        for (int j = 0; j < found; ++j) r += keys[j] > key ? 1 : 0;
        if (r < p.k) write_top(p, row, r, key, st, ls);
      }
      return;
    }
    for (int i0 = 0; i0 < n; i0 += NT) {
      const int i = i0 + (int)threadIdx.x;
      const u64 key = i < n ? pk[i] : 0;
      int r = 0;
      for (int j0 = 0; j0 < n; j0 += JT) {
        const int m = min(JT, n - j0);
        __syncthreads();
        for (int j = threadIdx.x; j < m; j += NT) keys[j] = pk[j0 + j];
        __syncthreads();
#pragma unroll 4
        for (int j = 0; j < m; ++j) r += keys[j] > key ? 1 : 0;
      }
      if (key != 0 && r < p.k) write_top(p, row, r, key, st, ls);
    }
  } else {
    const Stat st = join_parts(ps, p.parts);
    if (threadIdx.x == 0) write_row(p, row, st, id, xid);
  }
}

struct BwdParams {
  const void* x;
  void* dx;
  const int *ids, *top_ids;
  long long ld, ldd;
  int V, T, k, ignore, parts, per, cols;  // cols: columns of dx, V..cols-1 get zeros
  const float *norm, *ent, *dlogp, *dent, *dtop;
};
template <typename T>
__global__ __launch_bounds__(NT) void logprobs_bwd_kernel(BwdParams p) {
  constexpr int N = Vec<T>::N;
  const int row = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
  const T* x = (const T*)p.x + (long long)row * p.ld;
  T* d = (T*)p.dx + (long long)row * p.ldd;
  const int nvec = (p.cols + N - 1) / N, v0 = part * p.per, v1 = min(nvec, v0 + p.per);
  Vec<T> v[BNV];
#pragma unroll
  for (int c = 0; c < BNV; ++c) {
    const int i = v0 + c * NT + (int)threadIdx.x;
    if (i < v1 && i * N < p.V) load_vec<T>(v[c], x, i, p.V);
  }
  const int id = p.ids[row];
  const bool use = id != p.ignore && (unsigned)id < (unsigned)p.V;
  const float gl = use && p.dlogp ? p.dlogp[row] : 0.f;
  const float gh = p.dent ? p.dent[row] : 0.f;
  float tot = gl;
  for (int j = 0; j < p.k; ++j) tot += p.dtop[(long long)row * p.k + j];
  const float m = p.norm[2ll * row], ls = p.norm[2ll * row + 1], ent = p.ent[row];
  auto grad = [&](float xv) {  // the part every column has
    const float lp = fmaxf(log_p(xv, m, ls), -1e4f);  // p = 0 there
    const float pr = ex2(lp * LOG2E);
    return -pr * fmaf(gh, lp + ent, tot);
  };
#pragma unroll
  for (int c = 0; c < BNV; ++c) {
    const int i = v0 + c * NT + (int)threadIdx.x;
    if (i < v1) {
      Vec<T> o;
#pragma unroll
      for (int e = 0; e < N; ++e) o.e[e] = (T)(i * N + e < p.V ? grad(v[c].at(e)) : 0.f);
      if ((i + 1) * N <= p.cols) {
        *(u32x4_any*)(d + i * N) = o.raw;
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (i * N + e < p.cols) d[i * N + e] = o.e[e];
      }
    }
  }
  // the named columns once more, with their own terms (after this block's plain stores)
  __syncthreads();
  if ((int)threadIdx.x <= p.k) {
    const int col = threadIdx.x == 0 ? id : p.top_ids[(long long)row * p.k + threadIdx.x - 1];
    if ((threadIdx.x > 0 || use) && (unsigned)col < (unsigned)p.V && col >= v0 * N && col < v1 * N) {
      float g = use && col == id ? gl : 0.f;
      for (int j = 0; j < p.k; ++j)
        if (p.top_ids[(long long)row * p.k + j] == col) g += p.dtop[(long long)row * p.k + j];
      d[col] = (T)(g + grad((float)x[col]));
    }
  }
}

// parts of a row, in even shares: of at most NT * nv vectors, and where that leaves fewer than 256 blocks
// more of them, down to one vector a thread (8 rows of 33708 bf16 logits, k = 20: 3 -> 17 parts, 14.6 -> 11.7 us)
void cut(int vecs, long long T, int nv, int& parts, int& per) {
  const long long most = (vecs + NT - 1) / NT, least = (vecs + NT * nv - 1) / (NT * nv);
  parts = (int)std::max(least, std::min(most, 256 / std::max(T, 1ll)));
  per = (vecs + parts - 1) / parts;
}
// A launch has below 2^32 threads (beyond, the count wraps without an error): rows go out in slices of at most 2^23 blocks
constexpr int SLICE = 1 << 23;
int vecs_of(int cols, int dtype) { const int n = dtype == 2 ? 4 : 8; return (cols + n - 1) / n; }
}  // namespace

extern "C" {
int tfk_logprobs_kmax() { return KMAX; }
// bytes of workspace of a forward (0: none)
long long tfk_logprobs_ws(long long T, int V, int dtype, int k) {
  int parts, per;
  cut(vecs_of(V, dtype), T, NV, parts, per);
  return parts == 1 ? 0 : T * parts * (16 + 8ll * k);
}
// dtype: 0 bf16, 1 f16, 2 f32
int tfk_logprobs_fwd(const void* x, int dtype, const int* ids, int T, int V, long long ld, int k, int ignore, float* logp,
                     float* ent, float* lse, float* norm, float* top_logp, int* top_ids, void* ws, hipStream_t s) {
  if (T <= 0) return 0;
  FwdParams p{x, ids, ld, V, T, k, ignore, 0, 0, logp, ent, lse, norm, top_logp, top_ids, nullptr, nullptr};
  cut(vecs_of(V, dtype), T, NV, p.parts, p.per);
  p.pkeys = (u64*)ws;
  p.pstat = (Stat*)((u64*)ws + (long long)T * p.parts * k);
  const int step = SLICE / p.parts;
#define TFK_LP(T_)                                                                                              \
  if (k) hipLaunchKernelGGL((logprobs_fwd_kernel<T_, true>), g, dim3(NT), 0, s, p);                             \
  else hipLaunchKernelGGL((logprobs_fwd_kernel<T_, false>), g, dim3(NT), 0, s, p);                              \
  if (p.parts > 1 && k) hipLaunchKernelGGL((logprobs_join_kernel<T_, true>), dim3(p.T), dim3(NT), 0, s, p);     \
  else if (p.parts > 1) hipLaunchKernelGGL((logprobs_join_kernel<T_, false>), dim3(p.T), dim3(64), 0, s, p);
  for (long long r = 0; r < T; r += step) {
    p.T = (int)std::min<long long>(step, T - r);
    const dim3 g((unsigned)p.T * p.parts);
    if (dtype == 0) { TFK_LP(bf16) } else if (dtype == 1) { TFK_LP(f16) } else { TFK_LP(float) }
    if (hipGetLastError() != hipSuccess) return -1;
    p.x = (const char*)p.x + step * ld * (dtype == 2 ? 4 : 2);
    p.ids += step; p.logp += step; p.ent += step; p.lse += step; p.norm += 2ll * step;
    if (k) { p.top_logp += (long long)step * k; p.top_ids += (long long)step * k; }
    p.pkeys += (long long)step * p.parts * k; p.pstat += (long long)step * p.parts;
  }
#undef TFK_LP
  return 0;
}
// dx: cols >= V columns, row stride ldd; dlogp / dent may be null; k = 0: no alternatives
int tfk_logprobs_bwd(const void* x, int dtype, const int* ids, int T, int V, long long ld, int k, int ignore,
                     const float* norm, const float* ent, const int* top_ids, const float* dlogp, const float* dent,
                     const float* dtop, void* dx, long long ldd, int cols, hipStream_t s) {
  if (T <= 0) return 0;
  BwdParams p{x, dx, ids, top_ids, ld, ldd, V, T, k, ignore, 0, 0, cols, norm, ent, dlogp, dent, dtop};
  cut(vecs_of(cols, dtype), T, BNV, p.parts, p.per);
  const int step = SLICE / p.parts;
  for (long long r = 0; r < T; r += step) {
    p.T = (int)std::min<long long>(step, T - r);
    const dim3 g((unsigned)p.T * p.parts);
    if (dtype == 0) hipLaunchKernelGGL(logprobs_bwd_kernel<bf16>, g, dim3(NT), 0, s, p);
    else if (dtype == 1) hipLaunchKernelGGL(logprobs_bwd_kernel<f16>, g, dim3(NT), 0, s, p);
    else hipLaunchKernelGGL(logprobs_bwd_kernel<float>, g, dim3(NT), 0, s, p);
    if (hipGetLastError() != hipSuccess) return -1;
    const int e = dtype == 2 ? 4 : 2;
    p.x = (const char*)p.x + step * ld * e;
    p.dx = (char*)p.dx + step * ldd * e;
    p.ids += step; p.norm += 2ll * step; p.ent += step;
    if (p.dlogp) p.dlogp += step;
    if (p.dent) p.dent += step;
    if (k) { p.top_ids += (long long)step * k; p.dtop += (long long)step * k; }
  }
  return 0;
}
}
