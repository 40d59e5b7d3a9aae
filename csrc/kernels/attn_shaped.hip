// hipcc-flags: -Xclang -target-feature -Xclang -packed-fp32-ops
// Shaped attention: document runs and the entry points (kernels: attn_shaped_fwd.h, attn_shaped_bwd.h).
#include "attn_shaped_fwd.h"
#include "attn_shaped_bwd.h"

extern "C" {
int tfk_shaped_fwd_bf16(const void*, float*, hipStream_t, int);
int tfk_shaped_fwd_f16(const void*, float*, hipStream_t, int);
int tfk_shaped_dq_bf16(const void*, hipStream_t, int);
int tfk_shaped_dq_f16(const void*, hipStream_t, int);
int tfk_shaped_dkv_bf16(const void*, float*, hipStream_t, int);
int tfk_shaped_dkv_f16(const void*, float*, hipStream_t, int);
}

namespace {
// out[b][i] = [first, end) of the run of equal ids around position i; (0, 0) where the id is negative.
// One block per row: each thread scans a segment, waves and then the block the segments' borders.
constexpr int DT = 1024;
__global__ __launch_bounds__(DT) void doc_spans_kernel(const int* __restrict__ ids, int S, int2* __restrict__ out) {
  __shared__ int first[DT / 64], next[DT / 64];
  const int* x = ids + (long long)blockIdx.x * S;
  int2* y = out + (long long)blockIdx.x * S;
  const int per = (S + DT - 1) / DT, i0 = min(S, (int)threadIdx.x * per), i1 = min(S, i0 + per);
  int f = -1, n = S;  // last and first border (a position whose predecessor differs) of the segment
  for (int i = i0; i < i1; ++i)
    if (i == 0 || x[i] != x[i - 1]) {
      if (f < 0) n = i;
      f = i;
    }
  // running max of the last borders in front of this segment, running min of the first ones behind it
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int a = __shfl_up(f, o, 64), b = __shfl_down(n, o, 64);
    if (l >= o) f = max(f, a);
    if (l + o < 64) n = min(n, b);
  }
  if (l == 63) first[w] = f;
  if (l == 0) next[w] = n;
  __syncthreads();
  int cur = __shfl_up(f, 1, 64), end = __shfl_down(n, 1, 64);
  if (l == 0) cur = -1;
  if (l == 63) end = S;
  for (int u = 0; u < DT / 64; ++u) {
    if (u < w) cur = max(cur, first[u]);
    if (u > w) end = min(end, next[u]);
  }
  for (int i = i0; i < i1; ++i) {
    if (i == 0 || x[i] != x[i - 1]) cur = i;
    y[i].x = x[i] < 0 ? 0 : cur;
  }
  for (int i = i1 - 1; i >= i0; --i) {
    y[i].y = x[i] < 0 ? 0 : end;
    if (i == 0 || x[i] != x[i - 1]) end = i;
  }
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
  p.p_drop = p_drop; p.scale = scale; p.cap = cap; p.causal = causal; p.seed = seed; p.seed_key = tfk_seed_key();
  // rows of a head: whole tiles where a head has many queries (a tile then walks one head's keys),
  // packed where it has few; dropout hashes quads of queries, so quads stay whole
  const int tile = row_waves(p, (int)shape[5]) * 32;
  p.Sqp = p.Sq >= 64 ? (p.Sq + tile - 1) / tile * tile : (p_drop > 0.f ? (p.Sq + 3) / 4 * 4 : p.Sq);
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
  return f16_ ? tfk_shaped_fwd_f16(&p, ws, s, (int)shape[5]) : tfk_shaped_fwd_bf16(&p, ws, s, (int)shape[5]);
}
long long tfk_shaped_bwd_ws(const long long* shape, float p_drop) {
  const int D = (int)shape[5], kw = dkv_waves(D, p_drop > 0.f) * 32, G = (int)(shape[1] / shape[2]);
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
  const int D = (int)shape[5], rc = f16_ ? tfk_shaped_dq_f16(&p, s, D) : tfk_shaped_dq_bf16(&p, s, D);
  return rc ? rc : f16_ ? tfk_shaped_dkv_f16(&p, ws, s, D) : tfk_shaped_dkv_bf16(&p, ws, s, D);
}
int tfk_doc_spans(const int* ids, long long B, int S, int* out, hipStream_t s) {
  if (B <= 0 || S <= 0) return 0;
  const long long step = 1 << 21;  // rows of a launch: below 2^32 threads (beyond, their count wraps without an error)
  for (long long b = 0; b < B; b += step) {
    hipLaunchKernelGGL(doc_spans_kernel, dim3((unsigned)std::min(step, B - b)), dim3(DT), 0, s, ids + b * S, S, (int2*)out + b * S);
    if (hipGetLastError() != hipSuccess) return -1;
  }
  return 0;
}
}
