// Python bindings of the kernels that check drafted tokens (csrc/kernels/drafts.hip, alternatives.hip): checked wrappers on the current
// stream of the operands' device. Parents, lengths and targets are bounded inside the kernels.
#include <torch/extension.h>
#include <ATen/MemoryOverlap.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cmath>
#include <tuple>
#include <vector>

extern "C" {
int rt_draft_tree(const int*, const int*, const int*, int, int, int64_t*, int*, hipStream_t);
int rt_tree_parts(int, int, int, int, int, int, int);
int rt_tree_attention(int, const void*, long, const void*, const void*, const float*, const float*, int, const int*, const int*, const int64_t*,
                      void*, long, float*, int, int, int, int, int, int, int, int, float, int, hipStream_t);
int rt_tree_accept(const int*, const int64_t*, const int64_t*, const int64_t*, const int*, int*, int*, int64_t*, const void* const*, long, void*,
                   void*, long, float*, float*, long, int, int, int, int, int, int, int, int, int, hipStream_t);
int rt_alternatives(int, const void*, long, const int64_t*, float, long, int, int, float*, float*, float*, int64_t*, float*, hipStream_t);
int rt_alternatives_bwd(int, const void*, long, const int64_t*, float, long, int, int, const int64_t*, const float*, const float*, const float*,
                        const float*, void*, long, hipStream_t);
}

namespace py = pybind11;

namespace {

using at::Tensor;
using c10::optional;

hipStream_t stream() { return c10::hip::getCurrentHIPStream().stream(); }
void rc_ok(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " launch failed (code ", rc, ")"); }
bool has(const optional<Tensor>& t) { return t.has_value() && t->defined(); }
template <typename T> T* ptr(const optional<Tensor>& t) { return has(t) ? t->data_ptr<T>() : nullptr; }

void on(const Tensor& t, const Tensor& like, const char* n) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.device() == like.device(), n, ": expected on ", like.device());
}
void act(const Tensor& t, const char* n) {
  TORCH_CHECK_VALUE(t.is_cuda() && (t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat), n,
                    ": GPU tensor of bf16 or fp32 expected");
}
bool al(const Tensor& t, uintptr_t n) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % n == 0; }
void whole(const Tensor& t, at::ScalarType type, at::IntArrayRef shape, const Tensor& like, const char* n) {
  on(t, like, n);
  TORCH_CHECK_VALUE(t.scalar_type() == type && t.sizes() == shape && t.is_contiguous(), n, ": contiguous ", type, " ", shape, " expected, got ",
                    t.scalar_type(), " ", t.sizes());
}

// memory of `rows` pieces of `width` bytes, `pitch` apart
struct Span { const char* at; int64_t rows, pitch, width; };
Span span(const Tensor& t) {  // contiguous behind its first dimension, or all of it
  const int64_t size = t.element_size();
  if (!t.numel() || t.is_contiguous()) return {(const char*)t.data_ptr(), 1, 0, t.numel() * size};
  return {(const char*)t.data_ptr(), t.size(0), t.stride(0) * size, t.numel() / t.size(0) * size};
}
// a piece that lies in none of the rows of b
bool apart(const char* from, const char* to, const Span& b) {
  if (b.rows == 1 || b.pitch <= 0) return to <= b.at || b.at + b.width <= from;
  const int64_t first = from < b.at + b.width ? 0 : (from - b.at - b.width) / b.pitch + 1;  // the first row that ends behind `from`
  return first >= b.rows || to <= b.at + first * b.pitch;
}
// two that share no byte: other memory, or other columns of the same rows
bool apart(const Span& a, const Span& b) {
  if (!a.width || !b.width) return true;
  if (a.rows == 1) return apart(a.at, a.at + a.width, b);
  if (b.rows == 1) return apart(b.at, b.at + b.width, a);
  if (a.at + (a.rows - 1) * a.pitch + a.width <= b.at || b.at + (b.rows - 1) * b.pitch + b.width <= a.at) return true;
  if (a.pitch != b.pitch || a.pitch <= 0) return false;
  const int64_t col = ((a.at - b.at) % a.pitch + a.pitch) % a.pitch;  // a's first column, of b's
  return col >= b.width && col + a.width <= a.pitch;
}
// layers that are written at once: each has memory of its own
bool layers_apart(const Tensor& t) { return t.size(0) <= 1 || !t.numel() || t.stride(0) >= t.numel() / t.size(0); }

// the slots' scales of an e4m3 cache [.., rows, heads, slots, 128], alike for keys and values
struct Scales { float* k = nullptr; float* v = nullptr; long layer = 0; int slots = 0; };
Scales scales(const Tensor& kc, const optional<Tensor>& k, const optional<Tensor>& v) {
  Scales r;
  TORCH_CHECK_VALUE(has(k) == has(v), "scales of keys and values go together");
  TORCH_CHECK_VALUE(has(k) == (kc.scalar_type() == at::kByte), "scales belong to an e4m3 cache (uint8), and it has them");
  if (!has(k)) return r;
  const int64_t n = kc.dim();
  for (const auto* t : {&*k, &*v}) {
    on(*t, kc, "scales");
    TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat && t->dim() == n - 1 && t->sizes().slice(0, n - 2) == kc.sizes().slice(0, n - 2) &&
                          t->size(n - 2) >= kc.size(n - 2) && (n == 4 ? *t : t->select(0, 0)).is_contiguous() && t->sizes() == k->sizes() &&
                          t->strides() == k->strides(), "scales: fp32 of every row, head and slot expected, got ", t->sizes());
  }
  TORCH_CHECK_VALUE(kc.size(n - 1) == 128, "an e4m3 cache has heads of 128");
  r.k = k->data_ptr<float>();
  r.v = v->data_ptr<float>();
  r.layer = k->stride(0);
  r.slots = (int)k->size(n - 2);
  return r;
}

// whole numbers of a row each, contiguous
Tensor ints(const Tensor& t, at::ScalarType type, at::IntArrayRef shape, const Tensor& like, const char* n) {
  on(t, like, n);
  TORCH_CHECK_VALUE(t.scalar_type() == type && t.sizes() == shape, n, ": ", type, " ", shape, " expected, got ", t.scalar_type(), " ", t.sizes());
  return t.contiguous();
}
optional<Tensor> ints(const optional<Tensor>& t, at::ScalarType type, at::IntArrayRef shape, const Tensor& like, const char* n) {
  if (!has(t)) return c10::nullopt;
  return ints(*t, type, shape, like, n);
}

// What a tree was read with, by key heads, head size and columns of the rows: query heads, or None where not always as many. The
// plain form in Python makes the same keys.
py::int_ rows_of(int64_t Hkv, int64_t D, int64_t cols) { return py::int_(Hkv >> 16 || D >> 17 || cols >> 30 ? -1 : (Hkv << 17 | D) << 30 | cols); }

std::tuple<Tensor, Tensor, Tensor> draft_tree(const Tensor& parent_, const optional<Tensor>& nodes_, const optional<Tensor>& pos0_) {
  TORCH_CHECK_VALUE(parent_.is_cuda() && parent_.dim() == 2 && parent_.size(1) >= 1 && parent_.size(1) <= 64,
                    "parent: [rows, 1 .. 64 nodes] expected, got ", parent_.sizes());
  const int64_t B = parent_.size(0), N = parent_.size(1);
  const Tensor parent = ints(parent_, at::kInt, {B, N}, parent_, "parent");
  const optional<Tensor> nodes = ints(nodes_, at::kInt, {B}, parent, "nodes"), pos0 = ints(pos0_, at::kInt, {B}, parent, "pos0");
  const c10::DeviceGuard guard(parent.device());
  Tensor see = at::empty({B, N}, parent.options().dtype(at::kLong)), pos = at::empty({B, N}, parent.options());
  rc_ok(rt_draft_tree(parent.data_ptr<int>(), ptr<int>(nodes), ptr<int>(pos0), (int)B, (int)N, see.data_ptr<int64_t>(), pos.data_ptr<int>(),
                      stream()), "draft_tree");
  return {parent, see, pos};
}

Tensor tree_attention(const Tensor& qkv, const Tensor& kc, const Tensor& vc, const Tensor& kv_len_, const optional<Tensor>& kv_start_,
                      const Tensor& see, const optional<Tensor>& out_, int64_t Hq, int64_t window, const optional<double>& scale_,
                      const optional<Tensor>& k_scale, const optional<Tensor>& v_scale, bool as_stored, const py::dict& heads) {
  act(qkv, "tree_attention qkv");
  TORCH_CHECK_VALUE(kc.dim() == 4 && see.dim() == 2 && qkv.dim() == 2 && (qkv.stride(1) == 1 || qkv.size(0) == 0),
                    "tree_attention: qkv [rows nodes, columns], caches [rows, heads, slots, dim] expected, got ", qkv.sizes(), ", ", kc.sizes());
  const int64_t B = kc.size(0), Hkv = kc.size(1), Smax = kc.size(2), D = kc.size(3), N = see.size(1);
  TORCH_CHECK_VALUE(N >= 1 && N <= 64, "tree_attention: 1 to 64 nodes a row expected, got a tree ", see.sizes());
  const Scales sc = scales(kc, k_scale, v_scale);
  TORCH_CHECK_VALUE(sc.k || !as_stored, "tree_attention: only an e4m3 cache stores nodes otherwise than they are");
  TORCH_CHECK_VALUE(sc.k ? qkv.scalar_type() == at::kBFloat16 : kc.scalar_type() == qkv.scalar_type(), "caches of ", kc.scalar_type(),
                    " under queries of ", qkv.scalar_type());
  whole(kc, kc.scalar_type(), kc.sizes(), qkv, "tree_attention k_cache");
  whole(vc, kc.scalar_type(), kc.sizes(), qkv, "tree_attention v_cache");
  whole(see, at::kLong, {B, N}, qkv, "tree_attention tree");
  const Tensor kv_len = ints(kv_len_, at::kInt, {B}, qkv, "kv_len");
  const optional<Tensor> kv_start = ints(kv_start_, at::kInt, {B}, qkv, "kv_start");
  TORCH_CHECK_VALUE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && qkv.size(0) == B * N && qkv.size(1) >= (Hq + 2 * Hkv) * D, "tree_attention: ", Hq,
                    " heads over ", Hkv, " of ", D, " and ", B, " rows of ", N, " nodes do not fit qkv ", qkv.sizes());
  const double scale = scale_.has_value() ? *scale_ : 1 / std::sqrt((double)D);
  TORCH_CHECK_VALUE(window >= 0 && scale > 0 && std::isfinite(scale), "tree_attention: window ", window, ", scale ", scale);
  TORCH_CHECK_VALUE(D <= 512 && qkv.size(1) < (1L << 30) && Smax * D < (1L << 30) && window < (1L << 30) && Hq < 65536 && B < 65536, "tree_attention: sizes");
  TORCH_CHECK_VALUE(!at::GradMode::is_enabled() || !(qkv.requires_grad() || kc.requires_grad() || vc.requires_grad()),
                    "tree_attention has no gradient");
  const c10::DeviceGuard guard(qkv.device());
  const Tensor out = has(out_) ? *out_ : at::empty({B * N, Hq * D}, qkv.options());
  on(out, qkv, "tree_attention out");
  TORCH_CHECK_VALUE(out.scalar_type() == qkv.scalar_type() && out.dim() == 2 && out.size(0) == B * N && out.size(1) == Hq * D &&
                        (out.stride(1) == 1 || out.size(0) == 0), "tree_attention: out shape");
  at::assert_no_internal_overlap(out);
  const Span to = span(out);
  TORCH_CHECK_VALUE(apart(to, span(qkv)) && apart(to, span(kc)) && apart(to, span(vc)) && apart(to, span(see)) && apart(to, span(kv_len)) &&
                        (!has(kv_start) || apart(to, span(*kv_start))) && (!sc.k || (apart(to, span(*k_scale)) && apart(to, span(*v_scale)))),
                    "tree_attention: out overlaps what is read");
  const int64_t S = qkv.scalar_type() == at::kBFloat16 && al(kc, 16) && al(vc, 16)
                        ? rt_tree_parts((int)B, (int)N, (int)Hq, (int)Hkv, (int)D, (int)Smax, (int)window) : 0;
  TORCH_CHECK_VALUE(S || !sc.k || !B, "tree_attention: an e4m3 cache of this size");
  // matrix instructions want rows at 16 bytes (the output at 8): others are copied
  Tensor x = qkv, o = out;
  if (S && !(al(x, 16) && x.stride(0) % 8 == 0 && x.stride(0) < (1L << 24))) x = qkv.narrow(1, 0, (Hq + 2 * Hkv) * D).clone(at::MemoryFormat::Contiguous);
  if (S && !(al(o, 8) && o.stride(0) % 4 == 0)) o = at::empty({B * N, Hq * D}, qkv.options());
  Tensor part = S > 1 ? at::empty({S * B * Hkv * ((N * (Hq / Hkv) + 15) / 16) * 16 * (D + 2)}, qkv.options().dtype(at::kFloat)) : Tensor();
  rc_ok(rt_tree_attention(x.scalar_type() == at::kFloat, x.data_ptr(), x.stride(0), kc.data_ptr(), vc.data_ptr(), sc.k, sc.v, sc.slots,
                          kv_len.data_ptr<int>(), ptr<int>(kv_start), see.data_ptr<int64_t>(), o.data_ptr(), o.stride(0), S > 1 ? part.data_ptr<float>() : nullptr,
                          (int)S, (int)B, (int)N, (int)Hq, (int)Hkv, (int)D, (int)Smax, (int)window, (float)scale, as_stored, stream()), "tree_attention");
  if (!o.is_same(out)) out.copy_(o);
  const py::int_ rows = rows_of(Hkv, D, qkv.size(1)), read(Hq);
  PyObject* const before = PyDict_SetDefault(heads.ptr(), rows.ptr(), read.ptr());
  if (!before) throw py::error_already_set();
  if (before != Py_None && PyLong_AsLongLong(before) != Hq) heads[rows] = py::none();
  return out;
}

std::tuple<Tensor, Tensor, Tensor> tree_accept(const Tensor& parent, const Tensor& see, const Tensor& tokens_, const Tensor& choice_,
                                               const std::vector<Tensor>& drafts, Tensor kc, Tensor vc, const Tensor& kv_len_,
                                               const optional<Tensor>& k_scale, const optional<Tensor>& v_scale, int64_t heads, const py::dict& read) {
  if (!has(k_scale)) act(kc, "tree_accept k_cache");
  TORCH_CHECK_VALUE(kc.is_cuda(), "tree_accept k_cache: GPU tensor expected");
  TORCH_CHECK_VALUE(kc.dim() == 5 && see.dim() == 2 && drafts.size() && (int64_t)drafts.size() == kc.size(0) && drafts.size() <= 256,
              "tree_accept: caches [layers, rows, heads, slots, dim] and rows of every layer (256 at most)");
  const int64_t L = kc.size(0), B = kc.size(1), Hkv = kc.size(2), Smax = kc.size(3), D = kc.size(4), N = see.size(1);
  TORCH_CHECK_VALUE(N >= 1 && N <= 64, "tree_accept: 1 to 64 nodes a row expected, got a tree ", see.sizes());
  on(vc, kc, "tree_accept v_cache");
  TORCH_CHECK_VALUE(D > 0 && Hkv > 0, "tree_accept: caches of no heads");
  TORCH_CHECK_VALUE(vc.scalar_type() == kc.scalar_type() && vc.sizes() == kc.sizes() && vc.strides() == kc.strides() && kc[0].is_contiguous(),
              "tree_accept: caches of one type and layout, contiguous in each layer");
  const Scales sc = scales(kc, k_scale, v_scale);
  TORCH_CHECK_VALUE(layers_apart(kc) && (!sc.k || layers_apart(*k_scale)), "tree_accept: layers of one memory");
  const Span keys = span(kc), values = span(vc);
  TORCH_CHECK_VALUE(apart(keys, values) && (!sc.k || apart(span(*k_scale), span(*v_scale))), "tree_accept: keys and values of one memory");
  const Tensor kv_len = ints(kv_len_, at::kInt, {B}, kc, "kv_len");
  whole(parent, at::kInt, {B, N}, kc, "tree_accept tree");
  whole(see, at::kLong, {B, N}, kc, "tree_accept tree");
  const Tensor tokens = ints(tokens_, at::kLong, {B, N}, kc, "tokens"), choice = ints(choice_, at::kLong, {B, N}, kc, "choice");
  bool copy = false;  // e4m3: rows at 16 bytes, others are copied
  const int64_t bytes = drafts[0].dim() == 2 && drafts[0].numel()
                            ? ((drafts[0].size(0) - 1) * drafts[0].stride(0) + drafts[0].size(1)) * drafts[0].element_size() : 0;  // alike, see below
  for (const Tensor& x : drafts) {
    on(x, kc, "tree_accept drafts");
    TORCH_CHECK_VALUE(x.scalar_type() == (sc.k ? at::kBFloat16 : kc.scalar_type()) && x.dim() == 2 && x.stride(1) == 1 && x.sizes() == drafts[0].sizes() &&
                    x.stride(0) == drafts[0].stride(0) && x.size(0) == B * N,
                "tree_accept: drafts [rows nodes, (heads + 2 key heads) dim] of the caches' type, alike in every layer");
    const char* const from = (const char*)x.data_ptr();
    TORCH_CHECK_VALUE(!bytes || (apart(from, from + bytes, keys) && apart(from, from + bytes, values)), "tree_accept: drafts in the caches' memory");
    copy = copy || (sc.k && (!al(x, 16) || x.stride(0) % 8));
  }
  // keys lie behind `heads` queries; where nobody said how many (0), as tree_attention read such rows, or the rows hold nothing behind [q | k | v]
  const int64_t cols = drafts[0].size(1);
  if (!heads) {
    PyObject* const before = PyDict_GetItem(read.ptr(), rows_of(Hkv, D, cols).ptr());
    TORCH_CHECK_VALUE(before != Py_None, "tree_accept: rows of this width were read with different heads: Hq says which these have");
    if (before) heads = PyLong_AsLongLong(before);
  }
  const int64_t Hq = heads ? heads : cols / D - 2 * Hkv;
  TORCH_CHECK_VALUE(Hq > 0 && Hq % Hkv == 0 && Hq < 65536 && cols >= (Hq + 2 * Hkv) * D && (heads || cols % D == 0), "tree_accept: ", Hq,
                    " heads over ", Hkv, " of ", D, " do not fit drafts of ", cols, " columns");
  std::vector<const void*> at;
  std::vector<Tensor> held;
  if (copy)
    for (const Tensor& x : drafts) held.push_back(x.narrow(1, 0, (Hq + 2 * Hkv) * D).clone(at::MemoryFormat::Contiguous));
  const std::vector<Tensor>& rows = copy ? held : drafts;
  for (const Tensor& x : rows) at.push_back(x.data_ptr());
  TORCH_CHECK_VALUE(N * Hkv * D < (1L << 30), "tree_accept: sizes");
  const c10::DeviceGuard guard(kc.device());
  Tensor count = at::empty({B}, parent.options()), path = at::empty({B, N}, parent.options()), next = at::empty({B}, tokens.options());
  rc_ok(rt_tree_accept(parent.data_ptr<int>(), see.data_ptr<int64_t>(), tokens.data_ptr<int64_t>(), choice.data_ptr<int64_t>(),
                       kv_len.data_ptr<int>(), count.data_ptr<int>(), path.data_ptr<int>(), next.data_ptr<int64_t>(), at.data(),
                       rows[0].stride(0), kc.data_ptr(), vc.data_ptr(), kc.stride(0), sc.k, sc.v, sc.layer, sc.slots, (int)B, (int)N, (int)L, (int)Hq, (int)Hkv, (int)Smax, (int)D,
                       (int)kc.element_size(), stream()), "tree_accept");
  return {count, path, next};
}

// -> logp, entropy, alternatives' log-probabilities, their ids, and what the gradient needs of each row
std::vector<Tensor> alternatives(const Tensor& logits, const optional<Tensor>& targets, double c, int64_t top, bool need_stats) {
  const int64_t T = logits.size(0), V = logits.size(1);
  const c10::DeviceGuard guard(logits.device());
  const auto f = logits.options().dtype(at::kFloat);
  Tensor logp = at::empty({T}, f), ent = at::empty({T}, f), lp = at::empty({T, top}, f), stats = at::empty({need_stats ? T : 0, 3}, f);
  Tensor ids = at::empty({T, top}, logits.options().dtype(at::kLong));
  rc_ok(rt_alternatives(logits.scalar_type() == at::kFloat, logits.data_ptr(), logits.stride(0), ptr<int64_t>(targets), (float)c, T, (int)V,
                        (int)top, logp.data_ptr<float>(), ent.data_ptr<float>(), lp.data_ptr<float>(), ids.data_ptr<int64_t>(),
                        need_stats ? stats.data_ptr<float>() : nullptr, stream()), "token_alternatives");
  return {logp, ent, lp, ids, stats};
}

struct AlternativesFn : torch::autograd::Function<AlternativesFn> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& logits, const optional<Tensor>& targets,
                                                double c, int64_t top) {
    auto r = alternatives(logits, targets, c, top, true);
    ctx->save_for_backward({logits, has(targets) ? *targets : Tensor(), r[3], r[4]});
    ctx->saved_data["c"] = c;
    ctx->mark_non_differentiable({r[3]});
    ctx->set_materialize_grads(false);
    r.pop_back();
    return r;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor logits = saved[0], targets = saved[1], ids = saved[2], stats = saved[3];
    const int64_t T = logits.size(0), V = logits.size(1);
    TORCH_CHECK(!at::GradMode::is_enabled(), "token_alternatives has no second derivative");
    for (int i = 0; i < 3; ++i) {
      if (grads[i].defined()) grads[i] = grads[i].to(at::kFloat).contiguous();
    }
    auto g = [&](int i) { return grads[i].defined() ? grads[i].data_ptr<float>() : nullptr; };
    const c10::DeviceGuard guard(logits.device());
    Tensor d = at::empty({T, V}, logits.options());
    rc_ok(rt_alternatives_bwd(logits.scalar_type() == at::kFloat, logits.data_ptr(), logits.stride(0),
                              targets.defined() ? targets.data_ptr<int64_t>() : nullptr, (float)ctx->saved_data["c"].toDouble(), T, (int)V,
                              (int)ids.size(1), ids.data_ptr<int64_t>(), stats.data_ptr<float>(), g(0), g(1), g(2), d.data_ptr(), d.stride(0),
                              stream()), "token_alternatives backward");
    return {d, Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> token_alternatives(const Tensor& logits, const optional<Tensor>& targets, int64_t top, double c) {
  act(logits, "logits");
  TORCH_CHECK_VALUE(logits.dim() == 2 && top >= 1 && top <= 32 && top <= logits.size(1) && logits.size(1) < (1L << 30),
                    "1 to 32 alternatives of logits [tokens, vocabulary] expected: ", top, " of ", logits.sizes());
  TORCH_CHECK_VALUE(logits.size(0) < (1L << 22), "token_alternatives: ", logits.size(0), " rows");  // of up to 1024 threads each in a launch
  TORCH_CHECK_VALUE((float)c > 0 && std::isfinite((float)c), "inverse temperature ", c);
  const Tensor x = logits.stride(1) == 1 || logits.size(1) == 1 ? logits : logits.contiguous();
  optional<Tensor> t;
  if (has(targets)) {
    on(*targets, logits, "targets");
    TORCH_CHECK_VALUE(targets->dim() == 1 && targets->size(0) == logits.size(0) && at::isIntegralType(targets->scalar_type(), false),
                      "targets: ", logits.size(0), " whole numbers expected, got ", targets->scalar_type(), " ", targets->sizes());
    t = targets->to(at::kLong).contiguous();
  }
  auto r = at::GradMode::is_enabled() && x.requires_grad() ? AlternativesFn::apply(x, t, c, top)
                                                            : alternatives(x, t, c, top, false);
  return {r[0], r[1], r[2], r[3]};
}

}  // namespace

void bind_drafts(py::module_& m) {
  m.def("draft_tree", &draft_tree, "ancestors and positions of drafted tokens");
  m.def("tree_attention", &tree_attention, "attention of drafted tokens over the cache and their ancestors");
  m.def("tree_accept", &tree_accept, "the agreed path of a tree, appended to the caches");
  m.def("token_alternatives", &token_alternatives, "log-probabilities of tokens, entropy and the best alternatives (differentiable)");
}
