// Python bindings of softmax attention and of the 8-bit key/value cache.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <cmath>
#include <optional>

#include "kv8.cuh"

namespace {
using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

// Queries of a key/value head from which on a call on the 8-bit cache counts as a portion of a prompt: its codes are laid out once for
// the tensor cores, instead of being read again for every 16 queries.
constexpr int64_t PORTION = 64;
constexpr int64_t MOST_ROWS = 65535ll * 128;  // queries or keys of a sequence: tiles along a grid's second dimension

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }
bool has(const OptTensor& t) { return t.has_value() && t->defined(); }

// [B, rows, heads, D] bf16 as the kernels read it: 16-byte pieces of every row in place. Other layouts are copied (`held` keeps the copy).
tb::AttentionView view_of(const Tensor& x, const Tensor& like, const char* name, Tensor& held) {
  TORCH_CHECK(x.is_cuda() && x.get_device() == like.get_device(), name, " must be on the device of the queries");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 && x.dim() == 4, name, " must be bfloat16 [batch, tokens, heads, head_dim]");
  bool fits = (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15) == 0 && (x.size(3) == 1 || x.stride(3) == 1);
  for (int i = 0; i < 3; ++i) fits = fits && (x.size(i) <= 1 || (x.stride(i) > 0 && x.stride(i) % 8 == 0));  // nothing that is expanded
  held = fits ? x : x.clone(at::MemoryFormat::Contiguous);
  auto step = [&](int i) { return held.size(i) <= 1 ? 0ll : (long long)held.stride(i); };
  return tb::AttentionView{held.data_ptr(), step(1), step(2), step(0)};
}

const long long* numbers(const OptTensor& t, int64_t batch, const Tensor& like, const char* name) {
  if (!has(t)) return nullptr;
  TORCH_CHECK(t->is_cuda() && t->get_device() == like.get_device() && t->scalar_type() == at::kLong && t->is_contiguous() && t->numel() == batch, name,
              " must be int64 [batch] on the device of the queries");
  return reinterpret_cast<const long long*>(t->data_ptr<int64_t>());
}

int* status_of(const Tensor& t) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kInt && t.numel() == 1, "status: one CUDA int32");
  return t.data_ptr<int>();
}

tb::AttentionShape shape_of(const Tensor& q, const Tensor& k, const Tensor& v, double scale, bool causal, int64_t window, const OptTensor& lengths,
                            const OptTensor& starts, int64_t start) {
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.sizes() == k.sizes() && q.size(0) == k.size(0) && q.size(3) == k.size(3),
              "attention: queries [B, T, H, D], keys and values [B, S, G, D]");
  const int64_t T = q.size(1), S = k.size(1), H = q.size(2), G = k.size(2), D = q.size(3);
  TORCH_CHECK(D % 8 == 0 && D >= 8 && D <= 128, "attention: head sizes are multiples of 8 up to 128");
  TORCH_CHECK(G > 0 && H % G == 0, "attention: query heads must be a multiple of the key/value heads");
  TORCH_CHECK(T <= MOST_ROWS && S <= MOST_ROWS && q.size(0) * H < (1ll << 31), "attention: too many rows");
  TORCH_CHECK(std::isfinite(scale) && scale > 0, "attention: the scale must be positive");
  tb::AttentionShape a{(int)q.size(0), (int)T, (int)S, (int)H, (int)G, (int)D, (float)scale, causal, std::min<int64_t>(window, 1ll << 61)};
  a.lengths = numbers(lengths, a.B, q, "key_lengths");
  a.starts = numbers(starts, a.B, q, "query_start");
  a.start = start;
  return a;
}

tb::Kv8Cache cache_of(const Tensor& k8, const Tensor& v8, const Tensor& ks, const Tensor& vs, const Tensor& kt, const Tensor& vt, const Tensor& like) {
  const bool e4m3 = k8.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK(e4m3 || k8.scalar_type() == at::kChar, "kv8: codes are int8 or float8_e4m3fn");
  TORCH_CHECK(k8.dim() == 4 && v8.sizes() == k8.sizes() && v8.scalar_type() == k8.scalar_type(), "kv8: codes [B, G, capacity, pitch]");
  const int64_t B = k8.size(0), G = k8.size(1), C = k8.size(2), P = k8.size(3);
  TORCH_CHECK((P == 64 || P == 128) && C % tb::KV8_BLOCK == 0 && C < (1ll << 30), "kv8: pitch 64 or 128, capacity a multiple of 64");
  for (const Tensor* t : {&ks, &vs})
    TORCH_CHECK(t->scalar_type() == at::kFloat && t->dim() == 3 && t->size(0) == B && t->size(1) == G && t->size(2) == C / tb::KV8_BLOCK,
                "kv8: scales fp32 [B, G, capacity / 64]");
  for (const Tensor* t : {&kt, &vt})
    TORCH_CHECK(t->scalar_type() == at::kBFloat16 && t->dim() == 4 && t->size(0) == B && t->size(1) == G && t->size(2) == tb::KV8_RING && t->size(3) == P,
                "kv8: ring bf16 [B, G, 128, pitch]");
  for (const Tensor* t : {&k8, &v8, &ks, &vs, &kt, &vt})
    TORCH_CHECK(t->is_cuda() && t->get_device() == like.get_device() && t->is_contiguous() && (reinterpret_cast<uintptr_t>(t->data_ptr()) & 15) == 0,
                "kv8: the cache must be contiguous, 16-byte aligned and on the device of the rows");
  return tb::Kv8Cache{(uint8_t*)k8.data_ptr(), (uint8_t*)v8.data_ptr(), ks.data_ptr<float>(), vs.data_ptr<float>(), (__nv_bfloat16*)kt.data_ptr(),
                      (__nv_bfloat16*)vt.data_ptr(), (int)B, (int)G, (int)C, (int)P, e4m3};
}

tb::Kv8Pos pos_of(int64_t host, const OptTensor& dev, int64_t batch, const Tensor& like) {
  if (!has(dev)) return tb::Kv8Pos{host, nullptr, 0};
  TORCH_CHECK(dev->is_cuda() && dev->get_device() == like.get_device() && dev->scalar_type() == at::kLong && dev->is_contiguous() &&
                  (dev->numel() == 1 || dev->numel() == batch),
              "kv8: positions are int64, one or one per sequence, on the device of the rows");
  return tb::Kv8Pos{0, reinterpret_cast<const long long*>(dev->data_ptr<int64_t>()), dev->numel() == 1 ? 0 : 1};
}

void check_rows(const tb::Kv8Cache& c, const Tensor& x, int64_t heads, const char* name) {
  TORCH_CHECK(x.dim() == 4 && x.size(0) == c.B && x.size(2) == heads && x.size(3) % 8 == 0 && x.size(3) >= 8 && x.size(3) <= c.P, "kv8: ", name,
              " [B, T, heads, D] must fit the cache (D a multiple of 8)");
  TORCH_CHECK(x.size(1) < (1ll << 30), "kv8: too many tokens");
}

// New keys and values of a cache. `held`: copies that have to live until all that may run beside the append is launched; their memory
// is handed out again from then on
struct NewRows {
  tb::AttentionView k{}, v{};
  int T, D;
  bool any;
  Tensor held[2];
  NewRows(const tb::Kv8Cache& c, const Tensor& keys, const Tensor& values) {
    check_rows(c, keys, c.G, "keys");
    TORCH_CHECK(values.sizes() == keys.sizes(), "kv8: keys and values differ in shape");
    k = view_of(keys, keys, "keys", held[0]);
    v = view_of(values, keys, "values", held[1]);
    T = (int)keys.size(1), D = (int)keys.size(3), any = keys.numel() > 0;
  }
  void append(const tb::Kv8Cache& c, const tb::Kv8Pos& pos) const {
    if (any) tb::launch_kv8_append(c, k, v, T, D, pos, cur_stream());
  }
};

// Forward pass of f.a; -> out, and what the backward pass wants where it will come
Tensor attend(tb::AttentionFwd& f, const Tensor& q, const Tensor& k, const Tensor& v, bool train, const Tensor& status, Tensor& lse, Tensor& rest) {
  Tensor hq, hk, hv, part;
  f.q = view_of(q, q, "queries", hq);
  f.k = view_of(k, q, "keys", hk);
  f.v = view_of(v, q, "values", hv);
  Tensor out = torch::empty(q.sizes(), q.options());
  const auto f32 = q.options().dtype(at::kFloat);
  if (train) {
    lse = torch::empty({f.a.B, f.a.H, tb::attention_rows(f.a.T)}, f32);
    rest = torch::empty(q.sizes(), q.options());
  }
  if (out.numel() == 0) return out;
  if (f.a.S == 0) {
    if (train) {
      lse.fill_(-INFINITY);
      rest.zero_();
    }
    return out.zero_();
  }
  const long long bytes = tb::attention_fwd_scratch(f.a);
  if (bytes > 0) part = torch::empty({bytes / 4}, f32);
  f.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  f.lse = train ? lse.data_ptr<float>() : nullptr;
  f.rest = train ? reinterpret_cast<__nv_bfloat16*>(rest.data_ptr()) : nullptr;
  f.part = bytes > 0 ? part.data_ptr<float>() : nullptr;
  f.status = status_of(status);
  tb::launch_attention_fwd(f, cur_stream());
  return out;
}

// -> (out, lse, rest); the last two, for the backward pass, are empty without `train`.
std::vector<Tensor> attention_fwd(const Tensor& q, const Tensor& k, const Tensor& v, double scale, bool causal, int64_t window, const OptTensor& lengths,
                                  const OptTensor& starts, int64_t start, bool train, const Tensor& status) {
  tb::AttentionFwd f{};
  f.a = shape_of(q, k, v, scale, causal, window, lengths, starts, start);
  c10::cuda::CUDAGuard guard(q.device());
  Tensor lse, rest, out = attend(f, q, k, v, train, status, lse, rest);
  return {out, lse, rest};
}

// -> (dq, dk, dv)
std::vector<Tensor> attention_bwd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out, const Tensor& rest, const Tensor& dout, const Tensor& lse, double scale,
                                  bool causal, int64_t window, const OptTensor& lengths, const OptTensor& starts, int64_t start, const Tensor& status) {
  tb::AttentionBwd f{};
  f.a = shape_of(q, k, v, scale, causal, window, lengths, starts, start);
  TORCH_CHECK(out.sizes() == q.sizes() && rest.sizes() == q.sizes() && dout.sizes() == q.sizes(), "attention: outputs and their gradients have the queries' shape");
  TORCH_CHECK(lse.is_cuda() && lse.get_device() == q.get_device() && lse.scalar_type() == at::kFloat && lse.is_contiguous() &&
                  lse.numel() == (int64_t)f.a.B * f.a.H * tb::attention_rows(f.a.T) && (reinterpret_cast<uintptr_t>(lse.data_ptr()) & 15) == 0,
              "attention: the forward pass's sums");
  c10::cuda::CUDAGuard guard(q.device());
  Tensor held[6];
  f.q = view_of(q, q, "queries", held[0]);
  f.k = view_of(k, q, "keys", held[1]);
  f.v = view_of(v, q, "values", held[2]);
  f.out = view_of(out, q, "outputs", held[3]);
  f.dout = view_of(dout, q, "gradients", held[4]);
  f.rest = view_of(rest, q, "outputs", held[5]);
  Tensor dq = torch::empty(q.sizes(), q.options()), dk = torch::empty(k.sizes(), k.options()), dv = torch::empty(v.sizes(), v.options());
  if (dq.numel() == 0 || dk.numel() == 0) return {dq.zero_(), dk.zero_(), dv.zero_()};
  Tensor delta = torch::empty(lse.sizes(), lse.options());
  f.lse = lse.data_ptr<float>();
  f.delta = delta.data_ptr<float>();
  f.dq = reinterpret_cast<__nv_bfloat16*>(dq.data_ptr());
  f.dk = reinterpret_cast<__nv_bfloat16*>(dk.data_ptr());
  f.dv = reinterpret_cast<__nv_bfloat16*>(dv.data_ptr());
  f.status = status_of(status);
  tb::launch_attention_bwd(f, cur_stream());
  return {dq, dk, dv};
}

// Attention with its gradient as one node of the graph, without Python in the backward pass: of a small call's time (2 x 37 tokens, forward
// and backward), most was Python.
class AttentionNode : public torch::autograd::Function<AttentionNode> {
 public:
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, double scale, bool causal, int64_t window,
                        const OptTensor& lengths, const OptTensor& starts, int64_t start, const Tensor& status) {
    std::vector<Tensor> r = attention_fwd(q, k, v, scale, causal, window, lengths, starts, start, true, status);
    ctx->save_for_backward({q, k, v, r[0], r[2], r[1], has(lengths) ? *lengths : Tensor(), has(starts) ? *starts : Tensor()});
    ctx->saved_data["status"] = status;  // kept for the process, and written by whoever looks at it: no value that a version is checked of
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["window"] = window;
    ctx->saved_data["start"] = start;
    return r[0];
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto x = ctx->get_saved_variables();
    std::vector<Tensor> r = attention_bwd(x[0], x[1], x[2], x[3], x[4], grads[0].to(x[0].scalar_type()), x[5], ctx->saved_data["scale"].toDouble(),
                                          ctx->saved_data["causal"].toBool(), ctx->saved_data["window"].toInt(), x[6], x[7], ctx->saved_data["start"].toInt(), ctx->saved_data["status"].toTensor());
    if (torch::GradMode::is_enabled()) {  // a graph of the gradients is asked for: they have none, and say so when it is used
      torch::autograd::variable_list leaves;
      for (Tensor& t : r) leaves.push_back(t.detach().requires_grad_(true));
      r = (*std::make_shared<torch::autograd::DelayedError>("attention is differentiable once: its gradients have none", (int64_t)leaves.size()))(std::move(leaves));
    }
    const Tensor none;
    return {r[0], r[1], r[2], none, none, none, none, none, none, none};
  }
};

Tensor attention(const Tensor& q, const Tensor& k, const Tensor& v, double scale, bool causal, int64_t window, const OptTensor& lengths,
                 const OptTensor& starts, int64_t start, const Tensor& status) {
  return AttentionNode::apply(q, k, v, scale, causal, window, lengths, starts, start, status);
}

void kv8_append(const Tensor& k8, const Tensor& v8, const Tensor& ks, const Tensor& vs, const Tensor& kt, const Tensor& vt, const Tensor& k, const Tensor& v,
                int64_t host, const OptTensor& dev) {
  const tb::Kv8Cache c = cache_of(k8, v8, ks, vs, kt, vt, k);
  c10::cuda::CUDAGuard guard(k.device());
  NewRows(c, k, v).append(c, pos_of(host, dev, c.B, k));
}

// -> k, v [B, G, rows, D]
std::vector<Tensor> kv8_expand(const Tensor& k8, const Tensor& v8, const Tensor& ks, const Tensor& vs, const Tensor& kt, const Tensor& vt, int64_t rows,
                               int64_t D, int64_t host, const OptTensor& dev) {
  const tb::Kv8Cache c = cache_of(k8, v8, ks, vs, kt, vt, k8);
  TORCH_CHECK(rows >= 0 && rows <= c.C && D % 8 == 0 && D >= 8 && D <= c.P, "kv8: rows and head size must fit the cache");
  c10::cuda::CUDAGuard guard(k8.device());
  Tensor k = torch::empty({c.B, c.G, rows, D}, kt.options()), v = torch::empty_like(k);
  if (k.numel() > 0)
    tb::launch_kv8_expand(c, reinterpret_cast<__nv_bfloat16*>(k.data_ptr()), reinterpret_cast<__nv_bfloat16*>(v.data_ptr()), (int)rows, (int)D,
                          pos_of(host, dev, c.B, k8), cur_stream());
  return {k, v};
}

// Appends k and v (where given), then attends. `most`: a bound on the tokens a sequence holds then. `as_given`: k and v are read as they are,
// not as the cache holds them.
Tensor kv8_attention(const Tensor& k8, const Tensor& v8, const Tensor& ks, const Tensor& vs, const Tensor& kt, const Tensor& vt, const Tensor& q,
                     const OptTensor& k, const OptTensor& v, int64_t host, const OptTensor& dev, double scale, int64_t most, bool as_given, const Tensor& status) {
  const tb::Kv8Cache c = cache_of(k8, v8, ks, vs, kt, vt, q);
  TORCH_CHECK(q.dim() == 4 && q.size(2) % c.G == 0, "kv8: query heads must be a multiple of the cache's");
  check_rows(c, q, q.size(2), "queries");
  TORCH_CHECK(std::isfinite(scale) && scale > 0, "kv8: the scale must be positive");
  c10::cuda::CUDAGuard guard(q.device());
  tb::Kv8Attention a{};
  a.c = c;
  Tensor hq, part;
  std::optional<NewRows> rows_in;
  a.q = view_of(q, q, "queries", hq);
  a.T = (int)q.size(1);
  a.H = (int)q.size(2);
  a.D = (int)q.size(3);
  a.pos = pos_of(host, dev, c.B, q);
  a.scale = (float)scale;
  a.most = (int)std::max<int64_t>(0, std::min<int64_t>(most, c.C));
  Tensor out;
  if (has(k)) {
    TORCH_CHECK(has(v) && k->dim() == 4 && k->size(1) == q.size(1) && k->size(3) == q.size(3) && k->get_device() == q.get_device(),
                "kv8: new keys and values come with the queries' tokens");
    rows_in.emplace(c, *k, *v);
    if (!as_given) rows_in->append(c, a.pos);  // else once the open block's old tokens are no longer wanted
    a.appended = rows_in->any;
  }
  TORCH_CHECK(has(k) || !as_given, "kv8: new keys and values to read as given");
  if (q.numel() == 0) return torch::empty(q.sizes(), q.options());
  if (a.pos.dev == nullptr && host < 0) return torch::zeros(q.sizes(), q.options());  // idle
  if (!as_given && a.T * (a.H / c.G) < PORTION) {
    out = torch::empty(q.sizes(), q.options());
    a.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
    const long long bytes = tb::kv8_attention_scratch(a);
    if (bytes > 0) part = torch::empty({bytes / 4}, q.options().dtype(at::kFloat));
    a.part = bytes > 0 ? part.data_ptr<float>() : nullptr;
    tb::launch_kv8_attention(a, cur_stream());
    return out;
  }
  tb::AttentionFwd f{};
  if (as_given && a.pos.dev == nullptr && host == 0) {  // nothing comes before them
    rows_in->append(c, a.pos);
    f.a = shape_of(q, *k, *v, scale, true, 0, c10::nullopt, c10::nullopt, 0);
    return attend(f, q, *k, *v, false, status, part, part);
  }
  // a portion of a prompt: codes as bf16 numbers once, then attention on the tensor cores, which applies the blocks' scales
  const int64_t rows = a.most, blocks = (rows + tb::KV8_BLOCK - 1) / tb::KV8_BLOCK;
  if (rows == 0) {  // no room, or none that is to be looked at
    if (as_given) rows_in->append(c, a.pos);
    out = torch::zeros(q.sizes(), q.options());
    if (a.pos.dev != nullptr) tb::launch_kv8_outside(c, reinterpret_cast<__nv_bfloat16*>(out.data_ptr()), a.T, a.H * a.D, a.pos, cur_stream());
    return out;
  }
  Tensor codes = torch::empty({2, c.B, c.G, rows, a.D}, q.options()), scales = torch::empty({2, c.B, c.G, blocks}, q.options().dtype(at::kFloat));
  tb::Kv8Codes to{reinterpret_cast<__nv_bfloat16*>(codes.data_ptr()), nullptr, scales.data_ptr<float>()};
  if (as_given) to.new_k = rows_in->k, to.new_v = rows_in->v;
  to.v = to.k + codes.numel() / 2;
  to.v_scales = to.k_scales + scales.numel() / 2;
  Tensor where;
  if (a.pos.dev != nullptr) {
    where = torch::empty({2, c.B}, q.options().dtype(at::kLong));
    to.starts = reinterpret_cast<long long*>(where.data_ptr<int64_t>());
    to.ends = to.starts + c.B;
  }
  tb::launch_kv8_codes(c, to, (int)rows, a.D, a.pos, a.T, cur_stream());
  if (as_given) rows_in->append(c, a.pos);
  const Tensor kk = codes.select(0, 0).transpose(1, 2), vv = codes.select(0, 1).transpose(1, 2);
  f.a = shape_of(q, kk, vv, scale, true, 0, c10::nullopt, c10::nullopt, a.pos.host);
  if (a.pos.dev != nullptr) f.a.starts = to.starts, f.a.lengths = to.ends;
  f.k_scales = to.k_scales;
  f.v_scales = to.v_scales;
  f.blocks = (int)blocks;
  out = attend(f, q, kk, vv, false, status, part, part);
  if (a.pos.dev != nullptr) tb::launch_kv8_outside(c, reinterpret_cast<__nv_bfloat16*>(out.data_ptr()), a.T, a.H * a.D, a.pos, cur_stream());
  return out;
}

}  // namespace

void register_attention(pybind11::module& m) {
  m.def("attention_fwd", &attention_fwd);
  m.def("attention_bwd", &attention_bwd);
  m.def("attention", &attention);
  m.def("kv8_append", &kv8_append);
  m.def("kv8_expand", &kv8_expand);
  m.def("kv8_attention", &kv8_attention);
}
