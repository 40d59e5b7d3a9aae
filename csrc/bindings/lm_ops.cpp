// Bindings of the language-model operators: attention with shaped scores (attn_shaped.hip), token log
// probabilities (logprobs.hip), token order and the embedding gradient summed in it (embed_sort.hip).
// Every operand is checked (device, type, layout, extents, alignment) before a launch; launches go to
// the current stream of the operands' device, workspaces come from the caching allocator of that stream
// (so a captured graph owns the ones it uses).
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <hip/hip_runtime.h>
#include <algorithm>
#include <numeric>
#include <vector>

#include "bind_util.h"

extern "C" {
int tfk_shaped_fwd(const void*, const void*, const void*, void*, float*, int, const long long*, const long long*,
                   const int*, const int*, const int*, const int*, const float*, float, float, int, float,
                   unsigned long long, float*, hipStream_t);
long long tfk_shaped_fwd_ws(const long long*, float);
int tfk_shaped_bwd(const void*, const void*, const void*, const void*, const void*, const float*, float*, void*, void*,
                   void*, int, const long long*, const long long*, const long long*, const int*, const int*, const int*,
                   const int*, const float*, float, float, int, float, unsigned long long, float*, hipStream_t);
long long tfk_shaped_bwd_ws(const long long*, float);
int tfk_doc_spans(const int*, long long, int, int*, hipStream_t);
int tfk_logprobs_kmax();
long long tfk_logprobs_ws(long long, int, int, int);
int tfk_logprobs_fwd(const void*, int, const int*, int, int, long long, int, int, float*, float*, float*, float*, float*,
                     int*, void*, hipStream_t);
int tfk_logprobs_bwd(const void*, int, const int*, int, int, long long, int, int, const float*, const float*,
                     const int*, const float*, const float*, const float*, void*, long long, int, hipStream_t);
long long tfk_token_order_scratch(long long);
int tfk_token_order(const int*, int, int, int*, int*, int*, hipStream_t);
long long tfk_emb_sorted_part(long long, int);
int tfk_emb_sorted(const int*, const int*, int, int, int, const void*, int, long long, float*, float*, float, int,
                   hipStream_t);
}

namespace {
using Opt = c10::optional<torch::Tensor>;
hipStream_t stream_of(const torch::Tensor& t) { return at::hip::getCurrentHIPStream(t.device().index()).stream(); }
void same_device(const torch::Tensor& t, const torch::Tensor& ref, const char* n) {
  TORCH_CHECK(t.device() == ref.device(), n, " is on ", t.device(), ", expected ", ref.device());
}
void need_opt(const Opt& t, at::ScalarType dt, long long n, const torch::Tensor& ref, const char* name) {
  if (!t.has_value() || !t->defined()) return;
  need(*t, dt, name);
  same_device(*t, ref, name);
  TORCH_CHECK(t->numel() == n, name, " has ", t->numel(), " elements, expected ", n);
}
void need_vec(const torch::Tensor& t, at::ScalarType dt, long long n, const torch::Tensor& ref, const char* name) {
  need(t, dt, name);
  same_device(t, ref, name);
  TORCH_CHECK(t.numel() == n, name, " has ", t.numel(), " elements, expected ", n);
}
// 0 bf16, 1 f16, 2 f32
int type_code(const torch::Tensor& t, bool f32, const char* n) {
  TORCH_CHECK(t.is_cuda(), n, " must be a GPU tensor");
  const auto d = t.scalar_type();
  TORCH_CHECK(d == at::kBFloat16 || d == at::kHalf || (f32 && d == at::kFloat), n, " has dtype ", d,
              f32 ? ", expected bfloat16, float16 or float32" : ", expected bfloat16 or float16");
  return d == at::kBFloat16 ? 0 : d == at::kHalf ? 1 : 2;
}

// A column view of a token-major buffer: W elements at column `off` of tokens `rs` apart, batches `bs` apart.
// `write`: no two tokens may share memory.
void check_cols(const torch::Tensor& t, const torch::Tensor& ref, long long off, long long bs, long long rs, long long B,
                long long S, long long W, bool write, const char* n) {
  TORCH_CHECK(t.is_cuda(), n, " must be a GPU tensor");
  same_device(t, ref, n);
  TORCH_CHECK(t.scalar_type() == ref.scalar_type(), n, " has dtype ", t.scalar_type(), ", expected ", ref.scalar_type());
  TORCH_CHECK(t.dim() >= 2 && (t.size(-1) == 1 || t.stride(-1) == 1), n, " needs unit stride along its last dim");
  TORCH_CHECK(off >= 0 && off + W <= t.size(-1), n, ": columns ", off, "..", off + W, " outside a width of ", t.size(-1));
  TORCH_CHECK(rs % 8 == 0 && bs % 8 == 0 && off % 8 == 0, n, ": strides/offset must be multiples of 8 elements");
  TORCH_CHECK(rs >= W && rs < (1 << 23), n, ": token stride ", rs, " not in ", W, "..2^23");
  const long long have = (long long)(t.storage().nbytes() / t.element_size()) - t.storage_offset();
  TORCH_CHECK(bs >= 0 && off + (B - 1) * bs + (S - 1) * rs + W <= have, n, " too small for its shape");
  TORCH_CHECK((reinterpret_cast<uintptr_t>(t.data_ptr()) + 2 * off) % 16 == 0, n, " must be 16-byte aligned");
  if (write)
    TORCH_CHECK(B == 1 || bs >= (S - 1) * rs + W || (bs >= W && rs >= (B - 1) * bs + W), n, ": tokens overlap");
}
// Two column views share no element.
struct View {
  const char* at;
  long long B, S, bs, rs, w;  // batches of tokens of w bytes, bs and rs bytes apart
  const char* n;
  long long last() const { return (B - 1) * bs + (S - 1) * rs + w; }  // behind the last element
};
View view_of(const torch::Tensor& t, long long off, long long bs, long long rs, long long B, long long S, long long W, const char* n) {
  if (B > 1 && bs == S * rs) return {(const char*)t.data_ptr() + 2 * off, 1, B * S, 0, 2 * rs, 2 * W, n};  // one run of tokens
  return {(const char*)t.data_ptr() + 2 * off, B, S, 2 * bs, 2 * rs, 2 * W, n};
}
long long floor_div(long long a, long long b) { return a / b - (a % b < 0 ? 1 : 0); }
bool share(const View& a, const View& b) {
  const View &lo = a.at <= b.at ? a : b, &hi = a.at <= b.at ? b : a;
  const long long d = hi.at - lo.at;
  if (d >= lo.last()) return false;
  // modulo a divisor of all strides a view is one piece: disjoint pieces (columns of one buffer) share nothing
  long long g = 0;
  for (const View* v : {&lo, &hi}) {
    if (v->B > 1) g = std::gcd(g, v->bs);
    if (v->S > 1) g = std::gcd(g, v->rs);
  }
  if (g > 0 && d % g >= lo.w && d % g + hi.w <= g) return false;
  // equal token strides: for each pair of batches, the tokens i of lo and j of hi with |overlap| > 0 are those
  // whose i - j = m lies in [m0, m1]. (Other strides: taken to share.)
  const long long rs = lo.S > 1 ? lo.rs : hi.S > 1 ? hi.rs : std::max(lo.w, hi.w) + d;
  if ((lo.S > 1 && lo.rs != rs) || (hi.S > 1 && hi.rs != rs) || rs <= 0) return true;
  const auto meet = [&](long long x) {  // x: from a batch of lo to one of hi
    const long long m0 = std::max(floor_div(x - lo.w, rs) + 1, 1 - hi.S), m1 = std::min(floor_div(x + hi.w - 1, rs), lo.S - 1);
    return m0 <= m1;
  };
  if (lo.B * hi.B > 1 << 22 && lo.bs != hi.bs) return true;
  if (lo.bs == hi.bs) {
    for (long long n = 1 - hi.B; n < lo.B; ++n)
      if (meet(d - n * lo.bs)) return true;
    return false;
  }
  for (long long i = 0; i < lo.B; ++i)
    for (long long j = 0; j < hi.B; ++j)
      if (meet(d - i * lo.bs + j * hi.bs)) return true;
  return false;
}
void disjoint(const View& a, const View& b) { TORCH_CHECK(!share(a, b), a.n, " overlaps ", b.n); }
void check_shape(const std::vector<int64_t>& s, double scale, double cap, double p_drop) {
  TORCH_CHECK(s.size() == 6, "attention shape [B,H,Hk,Sq,Sk,D]");
  for (auto v : s) TORCH_CHECK(v >= 1 && v <= 0x7fffffff, "bad attention shape");
  TORCH_CHECK(s[1] % s[2] == 0, "heads must be a multiple of key heads");
  TORCH_CHECK(s[5] == 64 || s[5] == 128, "head dim must be 64 or 128, got ", s[5]);
  // query rows padded to whole tiles (of up to 256); block counts and row indices are 32-bit
  TORCH_CHECK(s[0] * s[1] <= 0x7fffffff && (s[3] + 256) * (s[1] / s[2]) <= 0x3fffffff && s[4] <= 0x7ffffff, "attention shape too large");
  // threads of a launch are below 2^32 (beyond, their count wraps without an error): 2 a padded row of queries or keys
  // and 512 blocks' shares of keys, or 512 a key head of a batch and 1024 blocks' shares where there are few rows
  const long long inst = s[0] * s[2], rows = s[1] / s[2] * (s[3] + 256) + 256, keys = s[4] + 256;
  TORCH_CHECK(2 * inst * std::max(rows, keys) + 512 * 512 <= 0xffffffffll && 512 * (inst + 1024) <= 0xffffffffll, "attention grid too large");
  // (within float32's whole-digit range)
  TORCH_CHECK(scale >= 1.2e-38 && scale <= 2e38, "scale must be positive, got ", scale);
  TORCH_CHECK(cap == 0.0 || (cap >= 1.2e-38 && cap <= 2e38), "softcap must be >= 0, got ", cap);
  TORCH_CHECK(p_drop >= 0.0 && p_drop < 1.0, "p_drop");
}
struct Masks {
  const int *kv_len, *q_start, *prefix, *docs;
  const float* slopes;
};
Masks masks(const Opt& kv_len, const Opt& q_start, const Opt& prefix, const Opt& docs, const Opt& slopes,
            const std::vector<int64_t>& s, const torch::Tensor& ref) {
  need_opt(kv_len, at::kInt, s[0], ref, "kv_len");
  need_opt(q_start, at::kInt, s[0], ref, "q_start");
  need_opt(prefix, at::kInt, s[0], ref, "prefix_len");
  need_opt(docs, at::kInt, 2 * s[0] * s[4], ref, "docs");
  need_opt(slopes, at::kFloat, s[1], ref, "slopes");
  if (docs.has_value() && docs->defined()) need_aligned(*docs, 8, "docs");
  return Masks{opt_ptr<const int>(kv_len), opt_ptr<const int>(q_start), opt_ptr<const int>(prefix),
               opt_ptr<const int>(docs), opt_ptr<const float>(slopes)};
}

// [batch, token] strides of a 2-D [B * S, width] or 3-D [B, S', width] buffer that holds W columns. The stride of a single
// token or batch says nothing (an expanded view's is 0, and a tile is read through a descriptor of rows times stride
// bytes): as in a tight buffer.
void buf_strides(const torch::Tensor& t, long long B, long long S, long long W, long long* st, const char* n) {
  TORCH_CHECK(t.dim() == 2 || t.dim() == 3, n, " must be [B*S, width] or [B, S', width]");
  st[1] = t.stride(-2);
  st[0] = t.dim() == 3 ? t.stride(0) : S * st[1];
  if (S == 1) st[1] = W;
  if (B == 1) st[0] = S * st[1];
}
struct Call {
  int f16;
  long long sh[6], st[8];
};
// shape [B, H, Hk, Sq, Sk, D]; fills everything but the output's strides
Call check_call(const torch::Tensor& q, int64_t qo, const torch::Tensor& k, int64_t ko, const torch::Tensor& v, int64_t vo,
                const std::vector<int64_t>& shape, double scale, double cap, double p_drop) {
  Call c;
  c.f16 = type_code(q, false, "q");
  check_shape(shape, scale, cap, p_drop);
  for (int i = 0; i < 6; ++i) c.sh[i] = shape[i];
  const long long B = shape[0], H = shape[1], Hk = shape[2], Sq = shape[3], Sk = shape[4], D = shape[5];
  buf_strides(q, B, Sq, H * D, c.st, "q");
  buf_strides(k, B, Sk, Hk * D, c.st + 2, "k");
  buf_strides(v, B, Sk, Hk * D, c.st + 4, "v");
  c.st[6] = Sq * H * D;
  c.st[7] = H * D;
  check_cols(q, q, qo, c.st[0], c.st[1], B, Sq, H * D, false, "q");
  check_cols(k, q, ko, c.st[2], c.st[3], B, Sk, Hk * D, false, "k");
  check_cols(v, q, vo, c.st[4], c.st[5], B, Sk, Hk * D, false, "v");
  return c;
}
void* at(const torch::Tensor& t, int64_t o) { return (void*)((char*)t.data_ptr() + 2 * o); }

std::tuple<torch::Tensor, torch::Tensor> shaped_fwd(torch::Tensor q, int64_t qo, torch::Tensor k, int64_t ko, torch::Tensor v,
                                                    int64_t vo, std::vector<int64_t> shape, Opt kv_len, Opt q_start,
                                                    Opt prefix, Opt docs, Opt slopes, double scale, double cap, bool causal,
                                                    double p_drop, int64_t seed) {
  const Call c = check_call(q, qo, k, ko, v, vo, shape, scale, cap, p_drop);
  const c10::DeviceGuard guard(q.device());
  const Masks m = masks(kv_len, q_start, prefix, docs, slopes, shape, q);
  torch::Tensor out = at::empty({c.sh[0] * c.sh[3], c.sh[1] * c.sh[5]}, q.options());
  torch::Tensor lse = at::empty({c.sh[0], c.sh[1], c.sh[3]}, q.options().dtype(at::kFloat)), ws;
  const long long wn = tfk_shaped_fwd_ws(c.sh, (float)p_drop);
  if (wn) ws = at::empty({wn}, lse.options());
  check_rc(tfk_shaped_fwd(at(q, qo), at(k, ko), at(v, vo), out.data_ptr(), lse.data_ptr<float>(), c.f16, c.sh, c.st,
                          m.kv_len, m.q_start, m.prefix, m.docs, m.slopes, (float)scale, (float)cap, causal ? 1 : 0,
                          (float)p_drop, (unsigned long long)seed, wn ? ws.data_ptr<float>() : nullptr, stream_of(q)),
           "shaped_fwd");
  return {out, lse};
}

void shaped_bwd(torch::Tensor q, int64_t qo, torch::Tensor k, int64_t ko, torch::Tensor v, int64_t vo, torch::Tensor out,
                torch::Tensor dout, torch::Tensor lse, torch::Tensor dq, int64_t dqo, torch::Tensor dk, int64_t dko,
                torch::Tensor dv, int64_t dvo, std::vector<int64_t> shape, Opt kv_len, Opt q_start, Opt prefix, Opt docs,
                Opt slopes, double scale, double cap, bool causal, double p_drop, int64_t seed) {
  const Call c = check_call(q, qo, k, ko, v, vo, shape, scale, cap, p_drop);
  const c10::DeviceGuard guard(q.device());
  const long long B = shape[0], H = shape[1], Hk = shape[2], Sq = shape[3], Sk = shape[4], D = shape[5];
  long long gs[6];
  buf_strides(dq, B, Sq, H * D, gs, "dq");
  buf_strides(dk, B, Sk, Hk * D, gs + 2, "dk");
  buf_strides(dv, B, Sk, Hk * D, gs + 4, "dv");
  TORCH_CHECK(out.is_contiguous() && dout.is_contiguous(), "out and dout must be contiguous [B*Sq, H*D]");
  check_cols(out, q, 0, c.st[6], c.st[7], B, Sq, H * D, false, "out");
  check_cols(dout, q, 0, c.st[6], c.st[7], B, Sq, H * D, false, "dout");
  check_cols(dq, q, dqo, gs[0], gs[1], B, Sq, H * D, true, "dq");
  check_cols(dk, q, dko, gs[2], gs[3], B, Sk, Hk * D, true, "dk");
  check_cols(dv, q, dvo, gs[4], gs[5], B, Sk, Hk * D, true, "dv");
  const View in[] = {view_of(q, qo, c.st[0], c.st[1], B, Sq, H * D, "q"), view_of(k, ko, c.st[2], c.st[3], B, Sk, Hk * D, "k"),
                     view_of(v, vo, c.st[4], c.st[5], B, Sk, Hk * D, "v"), view_of(out, 0, c.st[6], c.st[7], B, Sq, H * D, "out"),
                     view_of(dout, 0, c.st[6], c.st[7], B, Sq, H * D, "dout")};
  const View gr[] = {view_of(dq, dqo, gs[0], gs[1], B, Sq, H * D, "dq"), view_of(dk, dko, gs[2], gs[3], B, Sk, Hk * D, "dk"),
                     view_of(dv, dvo, gs[4], gs[5], B, Sk, Hk * D, "dv")};
  for (int i = 0; i < 3; ++i) {
    for (const View& x : in) disjoint(gr[i], x);  // every pass reads what the one before it reads
    for (int j = 0; j < i; ++j) disjoint(gr[i], gr[j]);
  }
  need_vec(lse, at::kFloat, B * H * Sq, q, "lse");
  const Masks m = masks(kv_len, q_start, prefix, docs, slopes, shape, q);
  torch::Tensor delta = at::empty({2 * B * H * Sq}, lse.options()), ws;
  const long long wn = tfk_shaped_bwd_ws(c.sh, (float)p_drop);
  if (wn) ws = at::empty({wn}, lse.options());
  check_rc(tfk_shaped_bwd(at(q, qo), at(k, ko), at(v, vo), out.data_ptr(), dout.data_ptr(), lse.data_ptr<float>(),
                          delta.data_ptr<float>(), at(dq, dqo), at(dk, dko), at(dv, dvo), c.f16, c.sh, c.st, gs, m.kv_len,
                          m.q_start, m.prefix, m.docs, m.slopes, (float)scale, (float)cap, causal ? 1 : 0, (float)p_drop,
                          (unsigned long long)seed, wn ? ws.data_ptr<float>() : nullptr, stream_of(q)),
           "shaped_bwd");
}

torch::Tensor doc_spans(torch::Tensor ids) {
  need(ids, at::kInt, "ids");
  TORCH_CHECK(ids.dim() == 2 && ids.size(1) <= 0x3fffffff, "ids must be [B, S]");
  const c10::DeviceGuard guard(ids.device());
  torch::Tensor out = at::empty({ids.size(0), ids.size(1), 2}, ids.options());
  check_rc(tfk_doc_spans(ids.data_ptr<int>(), ids.size(0), (int)ids.size(1), out.data_ptr<int>(), stream_of(ids)),
           "doc_spans");
  return out;
}

// logits [T, cols] (unit column stride), the first V columns are classes
int check_logits(const torch::Tensor& x, const torch::Tensor& ids, int64_t V, int64_t k) {
  const int dt = type_code(x, true, "logits");
  TORCH_CHECK(x.dim() == 2 && (x.size(1) == 1 || x.stride(1) == 1), "logits must be [T, V] with unit column stride");
  TORCH_CHECK(V >= 1 && V <= x.size(1) && x.size(1) <= 0x3fffffff, "logits: ", V, " classes of ", x.size(1), " columns");
  TORCH_CHECK(k >= 0 && k <= tfk_logprobs_kmax() && k <= V, "top_k must be in 0..min(", tfk_logprobs_kmax(), ", V), got ", k);
  TORCH_CHECK(x.size(0) <= 0x7fffffff, "too many rows");
  need_vec(ids, at::kInt, x.size(0), x, "ids");
  return dt;
}
// -> logp, entropy, lse [T], norm [T, 2], top_logp, top_ids [T, k] (None for k = 0)
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, Opt, Opt> logprobs_fwd(torch::Tensor x,
                                                                                             torch::Tensor ids, int64_t V,
                                                                                             int64_t k, int64_t ignore) {
  const int dt = check_logits(x, ids, V, k);
  const c10::DeviceGuard guard(x.device());
  const long long T = x.size(0);
  const auto f = x.options().dtype(at::kFloat);
  torch::Tensor logp = at::empty({T}, f), ent = at::empty({T}, f), lse = at::empty({T}, f), norm = at::empty({T, 2}, f), w;
  Opt tl, ti;
  if (k) {
    tl = at::empty({T, k}, f);
    ti = at::empty({T, k}, ids.options());
  }
  const long long ws = tfk_logprobs_ws(T, (int)V, dt, (int)k);
  if (ws) w = at::empty({ws}, x.options().dtype(at::kByte));
  check_rc(tfk_logprobs_fwd(x.data_ptr(), dt, ids.data_ptr<int>(), (int)T, (int)V, x.stride(0), (int)k, (int)ignore,
                            logp.data_ptr<float>(), ent.data_ptr<float>(), lse.data_ptr<float>(), norm.data_ptr<float>(),
                            opt_ptr<float>(tl), opt_ptr<int>(ti), ws ? w.data_ptr() : nullptr, stream_of(x)),
           "logprobs_fwd");
  return {logp, ent, lse, norm, tl, ti};
}
torch::Tensor logprobs_bwd(torch::Tensor x, torch::Tensor ids, int64_t V, int64_t ignore, torch::Tensor norm,
                           torch::Tensor ent, Opt top_ids, Opt dlogp, Opt dent, Opt dtop) {
  const bool top = dtop.has_value() && dtop->defined();
  TORCH_CHECK(!top || (top_ids.has_value() && top_ids->defined() && dtop->dim() == 2), "dtop [T, k] needs top_ids");
  const int64_t k = top ? dtop->size(1) : 0;
  const int dt = check_logits(x, ids, V, k);
  const c10::DeviceGuard guard(x.device());
  const long long T = x.size(0);
  need_vec(norm, at::kFloat, 2 * T, x, "norm"); need_vec(ent, at::kFloat, T, x, "entropy");
  need_opt(dlogp, at::kFloat, T, x, "dlogp"); need_opt(dent, at::kFloat, T, x, "dentropy");
  if (top) { need_opt(dtop, at::kFloat, T * k, x, "dtop"); need_opt(top_ids, at::kInt, T * k, x, "top_ids"); }
  torch::Tensor dx = at::empty({T, x.size(1)}, x.options());
  check_rc(tfk_logprobs_bwd(x.data_ptr(), dt, ids.data_ptr<int>(), (int)T, (int)V, x.stride(0), (int)k, (int)ignore,
                            norm.data_ptr<float>(), ent.data_ptr<float>(), top ? opt_ptr<const int>(top_ids) : nullptr,
                            opt_ptr<const float>(dlogp), opt_ptr<const float>(dent), top ? opt_ptr<const float>(dtop) : nullptr,
                            dx.data_ptr(), x.size(1), (int)x.size(1), stream_of(x)),
           "logprobs_bwd");
  return dx;
}

std::tuple<torch::Tensor, torch::Tensor> token_order(torch::Tensor ids, int64_t V) {
  need(ids, at::kInt, "ids");
  const long long T = ids.numel();
  // (a digit's places are counted over the histograms of all tiles: the square of T / 4096)
  TORCH_CHECK(V >= 1 && V < 0x7fffffff && T <= 1 << 24, "token_order: V ", V, ", tokens ", T, " (at most 2^24)");
  const c10::DeviceGuard guard(ids.device());
  torch::Tensor perm = at::empty({T}, ids.options()), keys = at::empty({T}, ids.options()), w;
  const long long ws = tfk_token_order_scratch(T);
  if (ws) w = at::empty({ws}, ids.options());
  check_rc(tfk_token_order(ids.data_ptr<int>(), (int)T, (int)V, perm.data_ptr<int>(), keys.data_ptr<int>(),
                           ws ? w.data_ptr<int>() : nullptr, stream_of(ids)),
           "token_order");
  return {perm, keys};
}
void embedding_bwd_sorted(torch::Tensor perm, torch::Tensor keys, torch::Tensor dy, torch::Tensor dword, double scale,
                          bool accumulate) {
  const int dt = type_code(dy, true, "dy");
  need(dword, at::kFloat, "dword");
  same_device(dword, dy, "dword");
  TORCH_CHECK(dy.dim() == 2 && dword.dim() == 2 && dy.size(1) == dword.size(1), "dy [T, W] and dword [V, W]");
  const long long T = dy.size(0), V = dword.size(0), W = dy.size(1);
  TORCH_CHECK(W >= 8 && W % 8 == 0 && W <= (1 << 20), "embedding width %8, got ", W);
  TORCH_CHECK(V >= 1 && V < 0x7fffffff && T <= 1 << 24, "embedding_bwd_sorted: V ", V, ", tokens ", T, " (at most 2^24)");
  // threads of a launch: W / 8 lanes, in groups of up to 64, for each chunk (2 W words of `part`)
  const long long words = tfk_emb_sorted_part(T, (int)W);
  TORCH_CHECK(words / 16 + words / (2 * W) * 64 <= 0x7fffffff, "embedding_bwd_sorted: ", T, " tokens of width ", W, " are too many");
  TORCH_CHECK((dy.size(1) == 1 || dy.stride(1) == 1) && (T <= 1 || dy.stride(0) % 8 == 0),  // (0: one row for all tokens)
              "dy rows: unit column stride, row stride a multiple of 8");
  need_aligned(dy, 16, "dy"); need_aligned(dword, 16, "dword");
  need_vec(perm, at::kInt, T, dy, "order"); need_vec(keys, at::kInt, T, dy, "order");
  const c10::DeviceGuard guard(dy.device());
  torch::Tensor part = at::empty({words}, dword.options());
  check_rc(tfk_emb_sorted(keys.data_ptr<int>(), perm.data_ptr<int>(), (int)T, (int)V, (int)W, dy.data_ptr(), dt,
                          dy.stride(0), dword.data_ptr<float>(), part.data_ptr<float>(), (float)scale, accumulate ? 1 : 0,
                          stream_of(dy)),
           "embedding_bwd_sorted");
}
}  // namespace

void register_lm_ops(pybind11::module& m) {
  m.def("shaped_fwd", &shaped_fwd);
  m.def("shaped_bwd", &shaped_bwd);
  m.def("doc_spans", &doc_spans);
  m.def("logprobs_fwd", &logprobs_fwd);
  m.def("logprobs_bwd", &logprobs_bwd);
  m.def("token_order", &token_order);
  m.def("embedding_bwd_sorted", &embedding_bwd_sorted);
}
