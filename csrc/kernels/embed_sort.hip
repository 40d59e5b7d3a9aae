// hipcc-flags: -Xclang -target-feature -Xclang -packed-fp32-ops
// Token order and the embedding gradient summed in that order, for gfx950.
//
// Order: perm = the stable sort of the token positions by id, keys = the sorted ids; ids outside
// [0, V) (padding) take the key V, so they come last. The order is a function of the ids alone, so
// every sum below has a fixed order of its terms: no float atomics, equal bits from run to run.
//
// Gradient: dword[r] (+)= scale * sum over the positions t with ids[t] == r of dy[t], in f32. The
// sorted positions are cut into chunks (chunk_of); a group of lanes (8 columns each) walks a chunk and
// sums each run of equal keys. A run inside one chunk is written at once; the pieces of a run that
// crosses a chunk border go to a workspace (`part`: a head and a tail row per chunk) and a second
// launch adds them in chunk order, so a token that fills half the batch is summed by many groups.
// Without accumulation the rows that no token names are zeroed by extra blocks of the same launch
// (they find their rows by a search in `keys`), so the table is written once. Bound by that write and the read
// of dy: order and gradient of 8192 tokens, W 1024, V 33792 bf16 45 us (155 MB, 3.5 TB/s; the write alone 21),
// of 65536 tokens, W 768, V 131072 135 us (503 MB, 3.7 TB/s). Each further launch costs 3 to 6 us of it.
#include <algorithm>
#include "common.h"

namespace {
typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
constexpr int NT = 256;

__device__ __forceinline__ int key_of(int id, int V) { return (unsigned)id < (unsigned)V ? id : V; }

// ------------------------------------------------------------------------------- order by counting
// rank(i) = #{j : key_j < key_i} + #{j < i : key_j == key_i}, one launch. T^2 compares: a block holds 32
// positions (one a lane of each half wave), its 16 waves divide the j's, the two halves of a wave take
// alternate groups of 16 j's, and the counts meet in LDS. A wave stages its j's keys in LDS and reads
// them back four at a time, the same for all lanes of a half, so a compare is two vector instructions:
// key_j < key_i + 1 for the j's before the block's positions, key_j < key_i for those behind.
// 8192 tokens: 8 us (scalar loads of the keys, 64 positions a block: 21 us, one load's latency per 16 keys).
constexpr int STAGE = 512, OP = 32;
typedef int i32x4 __attribute__((ext_vector_type(4)));
__global__ __launch_bounds__(1024) void order_count_kernel(const int* __restrict__ ids, int T, int V,
                                                           int* __restrict__ perm, int* __restrict__ keys) {
  __shared__ int cnt[32][OP];
  __shared__ __attribute__((aligned(16))) int stage[16][STAGE];
  const int l = threadIdx.x & 63, hw = l >> 5, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i0 = blockIdx.x * OP, i = i0 + (l & 31);
  const int key = key_of(ids[min(i, T - 1)], V);
  const int per = ((T + 15) / 16 + 3) & ~3, j0 = w * per, j1 = min(T, j0 + per);
  int n = 0;
  for (int g0 = j0; g0 < j1; g0 += STAGE) {
    const int m = min(STAGE, j1 - g0);
    int v[STAGE / 64];
#pragma unroll
    for (int u = 0; u < STAGE / 64; ++u) v[u] = ids[min(g0 + u * 64 + l, T - 1)];
#pragma unroll
    for (int u = 0; u < STAGE / 64; ++u) stage[w][u * 64 + l] = u * 64 + l < m ? key_of(v[u], V) : 0x7fffffff;
    __builtin_amdgcn_wave_barrier();  // the wave's own buffer: its LDS operations are in order
#pragma unroll 2
    for (int q0 = 0; q0 < m; q0 += 32) {
      const int q = q0 + 16 * hw, j = g0 + q;
      i32x4 k[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) k[u] = *(const i32x4*)&stage[w][q + 4 * u];
      if (g0 + q0 + 32 <= i0 || g0 + q0 >= i0 + OP) {
        const int lim = key + (g0 + q0 < i0 ? 1 : 0);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) n += k[u][e] < lim ? 1 : 0;
      } else {
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) n += k[u][e] < key + (j + 4 * u + e < i ? 1 : 0) ? 1 : 0;
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  cnt[2 * w + hw][l & 31] = n;
  __syncthreads();
  if (threadIdx.x < OP && i < T) {
    int r = 0;
#pragma unroll
    for (int u = 0; u < 32; ++u) r += cnt[u][threadIdx.x];
    perm[r] = i;
    keys[r] = key;
  }
}

// ------------------------------------------------------------------------------- order by digits
// One pass of a stable least-significant-digit sort: histogram of each tile, then every tile finds
// its digits' places from all histograms and writes its items in order.
constexpr int RT = 512, RW = RT / 64;  // threads, waves of a sorting block
constexpr int RB_MAX = 10;             // digit bits
// items of a tile (each wave: consecutive ones): small tiles for more blocks, large ones because each block reads
// the histograms of all tiles (tiles of 1024 and 4096, us: 65536 items of 16 bits 18.5 and 23.0, 131072 22.1 and 24.1,
// 163840 24.4 and 28.2, 196608 26.8 and 25.6, 262144 31.8 and 26.7, 2^20 108 and 48; of 18 bits: 163840 27.4 and 30.3,
// 196608 30.5 and 27.9, 2^22 2309 and 262)
constexpr int RTILE_FEW = 1024, RTILE_MANY = 4096;
int radix_tile(long long T) { return T <= 180000 ? RTILE_FEW : RTILE_MANY; }

template <bool FIRST>
__device__ __forceinline__ int radix_key(const int* src, long long i, int V) {
  return FIRST ? key_of(src[i], V) : src[i];
}
template <bool FIRST, int RTILE>
__global__ __launch_bounds__(RT) void radix_hist_kernel(const int* __restrict__ src, int T, int V, int shift, int bits,
                                                        int* __restrict__ hist) {
  __shared__ int h[1 << RB_MAX];
  const int nd = 1 << bits;
  for (int d = threadIdx.x; d < nd; d += RT) h[d] = 0;
  __syncthreads();
  const int t0 = blockIdx.x * RTILE, t1 = min(T, t0 + RTILE);
  for (int i = t0 + threadIdx.x; i < t1; i += RT) atomicAdd(&h[(radix_key<FIRST>(src, i, V) >> shift) & (nd - 1)], 1);
  __syncthreads();
  for (int d = threadIdx.x; d < nd; d += RT) hist[(long long)blockIdx.x * nd + d] = h[d];
}
template <bool FIRST, int RTILE>
__global__ __launch_bounds__(RT) void radix_place_kernel(const int* __restrict__ src, const int* __restrict__ psrc, int T,
                                                         int V, int shift, int bits, const int* __restrict__ hist,
                                                         int* __restrict__ dst, int* __restrict__ pdst) {
  constexpr int DPT = (1 << RB_MAX) / RT, IPL = RTILE / RW / 64;  // digits of a thread, items of a lane
  __shared__ int at[RW][1 << RB_MAX];  // next place of (wave, digit)
  __shared__ int tot[RW];
  const int nd = 1 << bits, nb = gridDim.x, l = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int w0 = blockIdx.x * RTILE + w * (RTILE / RW);
  int k[IPL], v[IPL];
#pragma unroll
  for (int u = 0; u < IPL; ++u) {
    const int i = min(w0 + u * 64 + l, T - 1);
    k[u] = radix_key<FIRST>(src, i, V);
    v[u] = FIRST ? i : psrc[i];
  }
  // digits d0 .. d0 + per - 1 belong to this thread: items of smaller digits anywhere, then of equal
  // digits in earlier tiles
  const int per = (nd + RT - 1) / RT, d0 = threadIdx.x * per;
  int all[DPT], before[DPT], mine = 0;
#pragma unroll
  for (int u = 0; u < DPT; ++u) {
    all[u] = before[u] = 0;
    if (u < per && d0 + u < nd) {
#pragma unroll 16
      for (int b = 0; b < nb; ++b) {
        const int c = hist[(long long)b * nd + d0 + u];
        all[u] += c;
        before[u] += b < (int)blockIdx.x ? c : 0;
      }
      mine += all[u];
    }
  }
  for (int d = threadIdx.x; d < nd * RW; d += RT) at[d / nd][d % nd] = 0;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < IPL; ++u)
    if (w0 + u * 64 + l < T) atomicAdd(&at[w][(k[u] >> shift) & (nd - 1)], 1);
  int base = mine;  // inclusive scan over the block: within the wave, then over the waves' totals
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(base, o, 64);
    base += l >= o ? x : 0;
  }
  if (l == 63) tot[w] = base;
  __syncthreads();
  base -= mine;
  for (int u = 0; u < w; ++u) base += tot[u];
#pragma unroll
  for (int u = 0; u < DPT; ++u)
    if (u < per && d0 + u < nd) {
      int p = base + before[u];
#pragma unroll
      for (int x = 0; x < RW; ++x) {
        const int c = at[x][d0 + u];
        at[x][d0 + u] = p;
        p += c;
      }
      base += all[u];
    }
  __syncthreads();
  // items in order: equal digits of one 64-item round by a match over the digit's bits
#pragma unroll
  for (int u = 0; u < IPL; ++u) {
    const bool ok = w0 + u * 64 + l < T;
    const int d = (k[u] >> shift) & (nd - 1);
    unsigned long long same = __ballot(ok);
    for (int b = 0; b < bits; ++b) {
      const unsigned long long m = __ballot((d >> b) & 1);
      same &= ((d >> b) & 1) ? m : ~m;
    }
    const int r = __popcll(same & ((1ull << l) - 1));
    int p = 0;
    if (ok) p = at[w][d] + r;
    __builtin_amdgcn_wave_barrier();
    if (ok && r == 0) at[w][d] = p + __popcll(same);
    __builtin_amdgcn_wave_barrier();
    if (ok) {
      dst[p] = k[u];
      pdst[p] = v[u];
    }
  }
}

template <bool FIRST, int RTILE>
void radix_pass(const int* ks, const int* ps, int T, int V, int shift, int bits, int nb, int* hist, int* kd, int* pd, hipStream_t s) {
  hipLaunchKernelGGL((radix_hist_kernel<FIRST, RTILE>), dim3(nb), dim3(RT), 0, s, ks, T, V, shift, bits, hist);
  hipLaunchKernelGGL((radix_place_kernel<FIRST, RTILE>), dim3(nb), dim3(RT), 0, s, ks, ps, T, V, shift, bits, hist, kd, pd);
}

// ------------------------------------------------------------------------------- gradient
template <typename T>
__device__ __forceinline__ void load8(float (&f)[8], const T* p) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) { f[e] = a[e]; f[4 + e] = b[e]; }
  } else {
    typedef T T8 __attribute__((ext_vector_type(8)));
    const T8 a = *(const T8*)p;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (float)a[e];
  }
}
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
  *(f32x4*)p = f32x4{f[0], f[1], f[2], f[3]};
  *(f32x4*)(p + 4) = f32x4{f[4], f[5], f[6], f[7]};
}
template <bool ACC>
__device__ __forceinline__ void put_row(float* d, float (&a)[8], float scale) {
  if (ACC) {
    float o[8];
    load8<float>(o, d);
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = fmaf(a[e], scale, o[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] *= scale;
  }
  store8(d, a);
}

// first place of `keys` whose key is >= k, by one wave: 64 probes a round
__device__ __forceinline__ int lower_wave(const int* keys, int n, int k) {
  const int l = threadIdx.x & 63;
  int lo = 0, hi = n;  // the answer is in [lo, hi]
  while (hi - lo > 0) {
    const int step = (hi - lo + 63) / 64, at = lo + l * step;
    const unsigned long long m = __ballot(at < hi && keys[min(at, n - 1)] < k);  // a prefix of the lanes
    const int c = __popcll(m);
    if (c == 0) return lo;
    const int nlo = lo + (c - 1) * step + 1;
    hi = min(hi, lo + c * step);
    lo = nlo;
  }
  return lo;
}

// lpc lanes share a chunk (8 columns each, `slabs` groups across a row); blocks from `sumb` on zero
// the rows without tokens, from zrow on, ZROWS rows a block. A group loads BATCH rows at once, then adds them in order:
// one row's latency at a time was most of a short batch's 18 us.
constexpr int BATCH = 8;
constexpr int ZROWS = 8;  // of a zeroing block: many short blocks (V 33792, W 1024: 8 36.7 us, 16 37.6, 32 38.1, 64 38.8)
template <typename T, bool ACC>
__global__ __launch_bounds__(NT) void emb_sum_kernel(const int* __restrict__ keys, const int* __restrict__ perm, int n,
                                                     int V, int W, const T* __restrict__ dy, long long ldy,
                                                     float* __restrict__ dword, float* __restrict__ part, float scale,
                                                     int chunk_len, int lpc, int slabs, int sumb, int zrow) {
  if ((int)blockIdx.x >= sumb) {
    __shared__ unsigned has;
    __shared__ int range[2];
    const int r0 = zrow + ((int)blockIdx.x - sumb) * ZROWS, nr = min(ZROWS, V - r0);
    if (threadIdx.x == 0) has = 0;
    if (threadIdx.x < 128) {
      const int w = threadIdx.x >> 6, p = lower_wave(keys, n, r0 + w * nr);
      if ((threadIdx.x & 63) == 0) range[w] = p;
    }
    __syncthreads();
    for (int p = range[0] + threadIdx.x; p < range[1]; p += NT)
      if (p == range[0] || keys[p - 1] != keys[p]) atomicOr(&has, 1u << (keys[p] - r0));
    __syncthreads();
    const unsigned named = has;
    const int vpr = W >> 2;
    int r = 0, c = threadIdx.x;
    float* d = dword + (long long)r0 * W;
    while (c >= vpr) { c -= vpr; ++r; }
    for (; r < nr;) {
      if (!((named >> r) & 1)) *(f32x4*)(d + (long long)r * W + 4 * c) = f32x4{0.f, 0.f, 0.f, 0.f};
      c += NT;
      while (c >= vpr) { c -= vpr; ++r; }
    }
    return;
  }
  const unsigned gid = blockIdx.x * NT + threadIdx.x, unit = gid / lpc;
  const int chunk = (int)(unit / slabs), col = ((int)(unit % slabs) * lpc + (int)(gid % lpc)) * 8;
  const int c0 = chunk * chunk_len;
  if (c0 >= n || col >= W) return;
  const int c1 = min(n, c0 + chunk_len);
  int cur = keys[c0];
  const bool head = c0 > 0 && keys[c0 - 1] == cur;
  bool first = true;
  float acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
  float* hp = part + ((long long)chunk * 2) * W + col;
  for (int p0 = c0; p0 < c1; p0 += BATCH) {
    int k[BATCH], t[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      k[u] = p0 + u < c1 ? keys[p0 + u] : V;
      t[u] = perm[min(p0 + u, n - 1)];
    }
    typedef T T8 __attribute__((ext_vector_type(8)));
    T8 row[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) row[u] = *(const T8*)(dy + t[u] * ldy + col);
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      if (p0 + u >= c1) break;
      if (k[u] != cur) {
        if (first && head) store8(hp, acc);
        else put_row<ACC>(dword + (long long)cur * W + col, acc, scale);
        first = false;
        cur = k[u];
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = 0.f;
      }
      if (cur >= V) return;  // only padding from here on
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += (float)row[u][e];
    }
  }
  if (first && head) store8(hp, acc);
  else if (c1 < n && keys[c1] == cur) store8(hp + W, acc);
  else put_row<ACC>(dword + (long long)cur * W + col, acc, scale);
}

// the runs that begin in chunk blockIdx.x and reach past its end: tail of that chunk + heads of the
// following ones, the groups of a block taking equal parts of them
template <bool ACC>
__global__ __launch_bounds__(NT) void emb_join_kernel(const int* __restrict__ keys, int n, int V, int W,
                                                      const float* __restrict__ part, float* __restrict__ dword,
                                                      float scale, int chunk_len, int lpc) {
  __shared__ float red[NT * 8];
  const int chunk = blockIdx.x, c0 = chunk * chunk_len, c1 = c0 + chunk_len;
  if (c1 >= n) return;
  const int k = keys[c1 - 1];
  if (k >= V || keys[c1] != k || (c0 > 0 && keys[c0 - 1] == k)) return;
  const int last = (c1 + lower_wave(keys + c1, n - c1, k + 1) - 1) / chunk_len;
  const int groups = NT / lpc, g = threadIdx.x / lpc, li = threadIdx.x % lpc;
  const int col = (blockIdx.y * lpc + li) * 8;
  const int m = last - chunk, per = (m + groups - 1) / groups;
  float acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
  if (col < W) {
    if (g == 0) load8<float>(acc, part + ((long long)chunk * 2 + 1) * W + col);
    const int b = chunk + 1 + g * per, e1 = min(last + 1, b + per);
#pragma unroll 8
    for (int c = b; c < e1; ++c) {
      float f[8];
      load8<float>(f, part + ((long long)c * 2) * W + col);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += f[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) red[threadIdx.x * 8 + e] = acc[e];
  __syncthreads();
  if (g == 0 && col < W) {
    for (int u = 1; u < groups; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += red[(u * lpc + li) * 8 + e];
    put_row<ACC>(dword + (long long)k * W + col, acc, scale);
  }
}

// lanes of a chunk's group: the power of two from 8 to 64 that leaves the fewest lanes idle over a
// row's 8-column vectors, the larger one where equal
int lanes_per_chunk(int W) {
  const int nv = W / 8;
  int best = 64, waste = 1 << 30;
  for (int l = 64; l >= 8; l >>= 1) {
    const int u = (nv + l - 1) / l * l - nv;
    if (u < waste) { waste = u; best = l; }
  }
  return best;
}
// positions of a chunk, powers of two that give 512 to 2048 chunks over the middle of the range: short ones give
// a small batch more groups (accumulating, 8192 tokens of width 1024: 8 17.9 us, 16 19.2, 32 26.5), long ones cut
// fewer runs in pieces (65536 tokens of width 768: 8 94 us, 16 86, 32 83; 16384 of width 1024: 33.8, 32.5, 38.6)
int chunk_of(long long n) { return n <= 8192 ? 8 : n <= 32768 ? 16 : 32; }
template <typename T>
void emb_sum_launch(const int* keys, const int* perm, int n, int V, int W, const void* dy, long long ldy, float* dword,
                    float* part, float scale, int acc, hipStream_t s) {
  const int lpc = lanes_per_chunk(W), slabs = (W / 8 + lpc - 1) / lpc, cl = chunk_of(n);
  const long long chunks = ((long long)n + cl - 1) / cl;
  const int sumb = (int)((chunks * slabs * lpc + NT - 1) / NT), zerob = acc ? 0 : V / ZROWS + (V % ZROWS != 0);
  if (sumb + zerob == 0) return;
  // (sumb has at most 2^31 threads; a launch has below 2^32, beyond, their count wraps without an error)
  constexpr int ZMAX = 1 << 22;
  const int z = std::min(zerob, ZMAX);
  if (acc) hipLaunchKernelGGL((emb_sum_kernel<T, true>), dim3(sumb), dim3(NT), 0, s, keys, perm, n, V, W, (const T*)dy, ldy, dword, part, scale, cl, lpc, slabs, sumb, 0);
  else hipLaunchKernelGGL((emb_sum_kernel<T, false>), dim3(sumb + z), dim3(NT), 0, s, keys, perm, n, V, W, (const T*)dy, ldy, dword, part, scale, cl, lpc, slabs, sumb, 0);
  for (int z0 = z; z0 < zerob; z0 += ZMAX)
    hipLaunchKernelGGL((emb_sum_kernel<T, false>), dim3(std::min(ZMAX, zerob - z0)), dim3(NT), 0, s, keys, perm, n, V, W, (const T*)dy, ldy, dword, part, scale, cl, lpc, slabs, 0, z0 * ZROWS);
  if (chunks < 2) return;
  const dim3 g((unsigned)(chunks - 1), slabs);
  if (acc) hipLaunchKernelGGL(emb_join_kernel<true>, g, dim3(NT), 0, s, keys, n, V, W, part, dword, scale, cl, lpc);
  else hipLaunchKernelGGL(emb_join_kernel<false>, g, dim3(NT), 0, s, keys, n, V, W, part, dword, scale, cl, lpc);
}
// counting is one launch of T^2 compares (8192 tokens, a block on each CU: 8 us), digits are two launches for each 10
// bits of V: 12288 tokens 17 us against 20 for 12289 by digits, 16384 22 against 15
constexpr int COUNT_MAX = 12288;
}  // namespace

extern "C" {
// int32 words of scratch that tfk_token_order needs
long long tfk_token_order_scratch(long long T) {
  if (T <= COUNT_MAX) return 0;
  const long long tile = radix_tile(T), nb = (T + tile - 1) / tile;
  return nb * (1 << RB_MAX) + 2 * T;
}
int tfk_token_order(const int* ids, int T, int V, int* perm, int* keys, int* scratch, hipStream_t s) {
  if (T <= 0) return 0;
  if (T <= COUNT_MAX) {
    hipLaunchKernelGGL(order_count_kernel, dim3((T + OP - 1) / OP), dim3(1024), 0, s, ids, T, V, perm, keys);
    return hipGetLastError() == hipSuccess ? 0 : -1;
  }
  int total = 1;
  while (total < 31 && (V >> total)) ++total;  // bits of the largest key, V
  const int passes = (total + RB_MAX - 1) / RB_MAX, bits = (total + passes - 1) / passes;
  const int tile = radix_tile(T), nb = (T + tile - 1) / tile;
  int *hist = scratch, *k2 = scratch + (long long)nb * (1 << RB_MAX), *p2 = k2 + T;
  const int *ks = ids, *ps = nullptr;
  for (int p = 0; p < passes; ++p) {
    // the last pass writes keys / perm; the passes before it alternate
    const bool fin = ((passes - 1 - p) & 1) == 0;
    int *kd = fin ? keys : k2, *pd = fin ? perm : p2;
    if (tile == RTILE_FEW) {
      if (p == 0) radix_pass<true, RTILE_FEW>(ks, ps, T, V, 0, bits, nb, hist, kd, pd, s);
      else radix_pass<false, RTILE_FEW>(ks, ps, T, V, p * bits, bits, nb, hist, kd, pd, s);
    } else {
      if (p == 0) radix_pass<true, RTILE_MANY>(ks, ps, T, V, 0, bits, nb, hist, kd, pd, s);
      else radix_pass<false, RTILE_MANY>(ks, ps, T, V, p * bits, bits, nb, hist, kd, pd, s);
    }
    ks = kd;
    ps = pd;
  }
  return hipGetLastError() == hipSuccess ? 0 : -1;
}
// f32 words of workspace that tfk_emb_sorted needs
long long tfk_emb_sorted_part(long long T, int W) { return (T + chunk_of(T) - 1) / chunk_of(T) * 2 * W; }
// dtype: 0 bf16, 1 f16, 2 f32; W % 8 == 0, rows of dy and dword 16-B aligned
int tfk_emb_sorted(const int* keys, const int* perm, int T, int V, int W, const void* dy, int dtype, long long ldy,
                   float* dword, float* part, float scale, int acc, hipStream_t s) {
  if (dtype == 0) emb_sum_launch<bf16>(keys, perm, T, V, W, dy, ldy, dword, part, scale, acc, s);
  else if (dtype == 1) emb_sum_launch<f16>(keys, perm, T, V, W, dy, ldy, dword, part, scale, acc, s);
  else emb_sum_launch<float>(keys, perm, T, V, W, dy, ldy, dword, part, scale, acc, s);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}
}
