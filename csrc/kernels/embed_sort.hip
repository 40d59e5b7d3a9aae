// hipcc-flags: -Xclang -target-feature -Xclang -packed-fp32-ops
// Token order and the embedding gradient summed in that order, for gfx950.
//
// Order: perm = the stable sort of the token positions by id, keys = the sorted ids; ids outside
// [0, V) (padding) take the key V, so they come last. The order is a function of the ids alone, so
// every sum below has a fixed order of its terms: no float atomics, equal bits from run to run.
//
// Gradient: dword[r] (+)= scale * sum over the positions t with ids[t] == r of dy[t], in f32. The
// sorted positions are cut into chunks of CHUNK; a group of lanes (8 columns each) walks a chunk and
// sums each run of equal keys. A run inside one chunk is written at once; the pieces of a run that
// crosses a chunk border go to a workspace (`part`: a head and a tail row per chunk) and a second
// launch adds them in chunk order, so a token that fills half the batch is summed by many groups.
// Without accumulation the rows that no token names are zeroed by extra blocks of the same launch
// (they find their rows by a search in `keys`), so the table is written once.
#include "common.h"

namespace {
typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
constexpr int NT = 256;
constexpr int CHUNK = 32;

__device__ __forceinline__ int key_of(int id, int V) { return (unsigned)id < (unsigned)V ? id : V; }

// ------------------------------------------------------------------------------- order by counting
// rank(i) = #{j : key_j < key_i} + #{j < i : key_j == key_i}, one launch. T^2 compares: a wave holds
// 64 positions, the 16 waves of a block share them and divide the j's, the counts meet in LDS.
__global__ __launch_bounds__(1024) void order_count_kernel(const int* __restrict__ ids, int T, int V,
                                                           int* __restrict__ perm, int* __restrict__ keys) {
  __shared__ int cnt[16][64];
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int i = blockIdx.x * 64 + l;
  const int key = key_of(ids[min(i, T - 1)], V);
  const int per = (T + 15) / 16, j0 = w * per, j1 = min(T, j0 + per);
  int n = 0;
  for (int j = j0; j < j1; j += 64) {
    // the wave's 64 keys, broadcast lane by lane
    const int kj = j + l < j1 ? key_of(ids[j + l], V) : 0x7fffffff;
    const int m = min(64, j1 - j);
    for (int e = 0; e < m; ++e) {
      const int k = __builtin_amdgcn_readlane(kj, e);
      n += (k < key || (k == key && j + e < i)) ? 1 : 0;
    }
  }
  cnt[w][l] = n;
  __syncthreads();
  if (w == 0 && i < T) {
    int r = 0;
#pragma unroll
    for (int u = 0; u < 16; ++u) r += cnt[u][l];
    perm[r] = i;
    keys[r] = key;
  }
}

// ------------------------------------------------------------------------------- order by digits
// One pass of a stable least-significant-digit sort: histogram of each tile, then every tile finds
// its digits' places from all histograms and writes its items in order.
constexpr int RT = 512, RW = RT / 64;  // threads, waves of a sorting block
constexpr int RTILE = 2048;            // items of a tile (each wave: 256 consecutive ones)
constexpr int RB_MAX = 10;             // digit bits

template <bool FIRST>
__device__ __forceinline__ int radix_key(const int* src, long long i, int V) {
  return FIRST ? key_of(src[i], V) : src[i];
}
template <bool FIRST>
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
template <bool FIRST>
__global__ __launch_bounds__(RT) void radix_place_kernel(const int* __restrict__ src, const int* __restrict__ psrc, int T,
                                                         int V, int shift, int bits, const int* __restrict__ hist,
                                                         int* __restrict__ dst, int* __restrict__ pdst) {
  __shared__ int at[RW][1 << RB_MAX];  // next place of (wave, digit)
  __shared__ int tot[RT];
  const int nd = 1 << bits, nb = gridDim.x, l = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (int d = threadIdx.x; d < nd * RW; d += RT) at[d / nd][d % nd] = 0;
  __syncthreads();
  const int w0 = blockIdx.x * RTILE + w * (RTILE / RW), w1 = min(T, w0 + RTILE / RW);
  for (int i = w0 + l; i < w1; i += 64) atomicAdd(&at[w][(radix_key<FIRST>(src, i, V) >> shift) & (nd - 1)], 1);
  // digits d0 .. d0 + per - 1 belong to this thread: items of smaller digits anywhere, then of equal
  // digits in earlier tiles
  const int per = (nd + RT - 1) / RT, d0 = threadIdx.x * per;
  int all[(1 << RB_MAX) / RT], before[(1 << RB_MAX) / RT], mine = 0;
#pragma unroll
  for (int u = 0; u < (1 << RB_MAX) / RT; ++u) {
    all[u] = before[u] = 0;
    if (u < per && d0 + u < nd) {
      for (int b = 0; b < nb; ++b) {
        const int c = hist[(long long)b * nd + d0 + u];
        all[u] += c;
        before[u] += b < (int)blockIdx.x ? c : 0;
      }
      mine += all[u];
    }
  }
  tot[threadIdx.x] = mine;
  __syncthreads();
  for (int o = 1; o < RT; o <<= 1) {  // inclusive scan of the threads' totals
    const int v = threadIdx.x >= o ? tot[threadIdx.x - o] : 0;
    __syncthreads();
    tot[threadIdx.x] += v;
    __syncthreads();
  }
  int base = tot[threadIdx.x] - mine;
#pragma unroll
  for (int u = 0; u < (1 << RB_MAX) / RT; ++u)
    if (u < per && d0 + u < nd) {
      int p = base + before[u];
      for (int v = 0; v < RW; ++v) {
        const int c = at[v][d0 + u];
        at[v][d0 + u] = p;
        p += c;
      }
      base += all[u];
    }
  __syncthreads();
  // items in order: equal digits of one 64-item round by a match over the digit's bits
  for (int i0 = w0; i0 < w1; i0 += 64) {
    const int i = i0 + l;
    const bool ok = i < w1;
    const int k = ok ? radix_key<FIRST>(src, i, V) : 0;
    const int d = (k >> shift) & (nd - 1);
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
      dst[p] = k;
      pdst[p] = FIRST ? i : psrc[i];
    }
  }
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
// first place of `keys` (sorted, n items, from lo) whose key is >= k
__device__ __forceinline__ int lower(const int* keys, int lo, int n, int k) {
  int hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (keys[mid] < k) lo = mid + 1;
    else hi = mid;
  }
  return lo;
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

// lpc lanes share a chunk (8 columns each, `slabs` groups across a row); blocks from `sumb` on zero
// the rows without tokens, 64 rows a block
template <typename T, bool ACC>
__global__ __launch_bounds__(NT) void emb_sum_kernel(const int* __restrict__ keys, const int* __restrict__ perm, int n,
                                                     int V, int W, const T* __restrict__ dy, long long ldy,
                                                     float* __restrict__ dword, float* __restrict__ part, float scale,
                                                     int lpc, int slabs, int sumb) {
  if ((int)blockIdx.x >= sumb) {
    __shared__ unsigned long long has;
    const int r0 = ((int)blockIdx.x - sumb) * 64, nr = min(64, V - r0);
    if (threadIdx.x < 64) {
      const int r = r0 + (int)threadIdx.x;
      bool found = false;
      if (r < V) {
        const int p = lower(keys, 0, n, r);
        found = p < n && keys[p] == r;
      }
      const unsigned long long m = __ballot(found);
      if (threadIdx.x == 0) has = m;
    }
    __syncthreads();
    const unsigned long long m = has;
    const int vpr = W >> 2;
    for (int r = 0; r < nr; ++r) {
      if ((m >> r) & 1) continue;
      float* d = dword + (long long)(r0 + r) * W;
      for (int c = threadIdx.x; c < vpr; c += NT) *(f32x4*)(d + 4 * c) = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    return;
  }
  const long long gid = (long long)blockIdx.x * NT + threadIdx.x, unit = gid / lpc;
  const int chunk = (int)(unit / slabs), col = ((int)(unit % slabs) * lpc + (int)(gid % lpc)) * 8;
  const int c0 = chunk * CHUNK;
  if (c0 >= n || col >= W) return;
  const int c1 = min(n, c0 + CHUNK);
  int cur = keys[c0];
  const bool head = c0 > 0 && keys[c0 - 1] == cur;
  bool first = true;
  float acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
  float* hp = part + ((long long)chunk * 2) * W + col;
  for (int p = c0; p < c1; ++p) {
    const int k = keys[p];
    if (k != cur) {
      if (first && head) store8(hp, acc);
      else put_row<ACC>(dword + (long long)cur * W + col, acc, scale);
      first = false;
      cur = k;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    }
    if (k >= V) return;  // only padding from here on
    float f[8];
    load8<T>(f, dy + (long long)perm[p] * ldy + col);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] += f[e];
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
                                                      float scale, int lpc) {
  __shared__ float red[NT * 8];
  const int chunk = blockIdx.x, c0 = chunk * CHUNK, c1 = c0 + CHUNK;
  if (c1 >= n) return;
  const int k = keys[c1 - 1];
  if (k >= V || keys[c1] != k || (c0 > 0 && keys[c0 - 1] == k)) return;
  const int last = (lower(keys, c1, n, k + 1) - 1) / CHUNK;
  const int groups = NT / lpc, g = threadIdx.x / lpc, li = threadIdx.x % lpc;
  const int col = (blockIdx.y * lpc + li) * 8;
  const int m = last - chunk, per = (m + groups - 1) / groups;
  float acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
  if (col < W) {
    if (g == 0) load8<float>(acc, part + ((long long)chunk * 2 + 1) * W + col);
    const int b = chunk + 1 + g * per, e1 = min(last + 1, b + per);
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
template <typename T>
void emb_sum_launch(const int* keys, const int* perm, int n, int V, int W, const void* dy, long long ldy, float* dword,
                    float* part, float scale, int acc, hipStream_t s) {
  const int lpc = lanes_per_chunk(W), slabs = (W / 8 + lpc - 1) / lpc;
  const long long chunks = ((long long)n + CHUNK - 1) / CHUNK;
  const int sumb = (int)((chunks * slabs * lpc + NT - 1) / NT), zerob = acc ? 0 : (V + 63) / 64;
  if (sumb + zerob == 0) return;
  if (acc) hipLaunchKernelGGL((emb_sum_kernel<T, true>), dim3(sumb), dim3(NT), 0, s, keys, perm, n, V, W, (const T*)dy, ldy, dword, part, scale, lpc, slabs, sumb);
  else hipLaunchKernelGGL((emb_sum_kernel<T, false>), dim3(sumb + zerob), dim3(NT), 0, s, keys, perm, n, V, W, (const T*)dy, ldy, dword, part, scale, lpc, slabs, sumb);
  if (chunks < 2) return;
  const dim3 g((unsigned)(chunks - 1), slabs);
  if (acc) hipLaunchKernelGGL(emb_join_kernel<true>, g, dim3(NT), 0, s, keys, n, V, W, part, dword, scale, lpc);
  else hipLaunchKernelGGL(emb_join_kernel<false>, g, dim3(NT), 0, s, keys, n, V, W, part, dword, scale, lpc);
}
constexpr int COUNT_MAX = 16384;
}  // namespace

extern "C" {
// int32 words of scratch that tfk_token_order needs
long long tfk_token_order_scratch(long long T) {
  if (T <= COUNT_MAX) return 0;
  const long long nb = (T + RTILE - 1) / RTILE;
  return nb * (1 << RB_MAX) + 2 * T;
}
int tfk_token_order(const int* ids, int T, int V, int* perm, int* keys, int* scratch, hipStream_t s) {
  if (T <= 0) return 0;
  if (T <= COUNT_MAX) {
    hipLaunchKernelGGL(order_count_kernel, dim3((T + 63) / 64), dim3(1024), 0, s, ids, T, V, perm, keys);
    return hipGetLastError() == hipSuccess ? 0 : -1;
  }
  int total = 1;
  while (total < 31 && (V >> total)) ++total;  // bits of the largest key, V
  const int passes = (total + RB_MAX - 1) / RB_MAX, bits = (total + passes - 1) / passes;
  const int nb = (T + RTILE - 1) / RTILE;
  int *hist = scratch, *k2 = scratch + (long long)nb * (1 << RB_MAX), *p2 = k2 + T;
  const int *ks = ids, *ps = nullptr;
  for (int p = 0; p < passes; ++p) {
    // the last pass writes keys / perm; the passes before it alternate
    const bool fin = ((passes - 1 - p) & 1) == 0;
    int *kd = fin ? keys : k2, *pd = fin ? perm : p2;
    if (p == 0) {
      hipLaunchKernelGGL(radix_hist_kernel<true>, dim3(nb), dim3(RT), 0, s, ks, T, V, 0, bits, hist);
      hipLaunchKernelGGL(radix_place_kernel<true>, dim3(nb), dim3(RT), 0, s, ks, ps, T, V, 0, bits, hist, kd, pd);
    } else {
      hipLaunchKernelGGL(radix_hist_kernel<false>, dim3(nb), dim3(RT), 0, s, ks, T, V, p * bits, bits, hist);
      hipLaunchKernelGGL(radix_place_kernel<false>, dim3(nb), dim3(RT), 0, s, ks, ps, T, V, p * bits, bits, hist, kd, pd);
    }
    ks = kd;
    ps = pd;
  }
  return hipGetLastError() == hipSuccess ? 0 : -1;
}
// f32 words of workspace that tfk_emb_sorted needs
long long tfk_emb_sorted_part(long long T, int W) { return (T + CHUNK - 1) / CHUNK * 2 * W; }
// dtype: 0 bf16, 1 f16, 2 f32; W % 8 == 0, rows of dy and dword 16-B aligned
int tfk_emb_sorted(const int* keys, const int* perm, int T, int V, int W, const void* dy, int dtype, long long ldy,
                   float* dword, float* part, float scale, int acc, hipStream_t s) {
  if (dtype == 0) emb_sum_launch<bf16>(keys, perm, T, V, W, dy, ldy, dword, part, scale, acc, s);
  else if (dtype == 1) emb_sum_launch<f16>(keys, perm, T, V, W, dy, ldy, dword, part, scale, acc, s);
  else emb_sum_launch<float>(keys, perm, T, V, W, dy, ldy, dword, part, scale, acc, s);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}
}
