// Python bindings of the kernels that check drafted tokens (csrc/kernels/drafts.hip, alternatives.hip): checked wrappers on the current
// stream of the operands' device. Parents, lengths and targets are bounded inside the kernels.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>

#include <vector>

extern "C" {
int rt_draft_tree(const int*, const int*, const int*, int, int, int64_t*, int*, hipStream_t);
int rt_tree_parts(int, int, int, int, int, int);
int rt_tree_attention(int, const void*, long, const void*, const void*, const int*, const int*, const int64_t*, void*, long, float*, int, int,
                      int, int, int, int, int, int, float, hipStream_t);
int rt_tree_accept(const int*, const int64_t*, const int64_t*, const int64_t*, const int*, int*, int*, int64_t*, const void* const*, long, void*,
                   void*, long, int, int, int, int, int, int, int, int, hipStream_t);
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
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), n, ": expected on ", like.device());
}
void act(const Tensor& t, const char* n) {
  TORCH_CHECK(t.is_cuda() && (t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat), n,
              ": GPU tensor of bf16 or fp32 expected");
}
bool al(const Tensor& t, uintptr_t n) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % n == 0; }
void whole(const Tensor& t, at::ScalarType type, at::IntArrayRef shape, const Tensor& like, const char* n) {
  on(t, like, n);
  TORCH_CHECK(t.scalar_type() == type && t.sizes() == shape && t.is_contiguous(), n, ": contiguous ", type, " ", shape, " expected, got ",
              t.scalar_type(), " ", t.sizes());
}

std::vector<Tensor> draft_tree(const Tensor& parent, const optional<Tensor>& nodes, const optional<Tensor>& pos0) {
  TORCH_CHECK(parent.is_cuda() && parent.dim() == 2, "draft_tree: parent [rows, nodes]");
  const int64_t B = parent.size(0), N = parent.size(1);
  whole(parent, at::kInt, {B, N}, parent, "draft_tree parent");
  for (const auto* t : {&nodes, &pos0})
    if (has(*t)) whole(**t, at::kInt, {B}, parent, "draft_tree nodes / pos0");
  const c10::DeviceGuard guard(parent.device());
  Tensor see = at::empty({B, N}, parent.options().dtype(at::kLong)), pos = at::empty({B, N}, parent.options());
  rc_ok(rt_draft_tree(parent.data_ptr<int>(), ptr<int>(nodes), ptr<int>(pos0), (int)B, (int)N, see.data_ptr<int64_t>(), pos.data_ptr<int>(),
                      stream()), "draft_tree");
  return {see, pos};
}

void tree_attention(const Tensor& qkv, const Tensor& kc, const Tensor& vc, const Tensor& kv_len, const optional<Tensor>& kv_start,
                    const Tensor& see, Tensor out, int64_t Hq, int64_t window, double scale) {
  act(qkv, "tree_attention qkv");
  TORCH_CHECK(kc.dim() == 4 && see.dim() == 2 && qkv.dim() == 2 && qkv.stride(1) == 1 && out.dim() == 2 && out.stride(1) == 1,
              "tree_attention: qkv [rows nodes, columns], caches [rows, heads, slots, dim], out [rows nodes, columns]");
  const int64_t B = kc.size(0), Hkv = kc.size(1), Smax = kc.size(2), D = kc.size(3), N = see.size(1);
  whole(kc, qkv.scalar_type(), kc.sizes(), qkv, "tree_attention k_cache");
  whole(vc, qkv.scalar_type(), kc.sizes(), qkv, "tree_attention v_cache");
  whole(kv_len, at::kInt, {B}, qkv, "tree_attention kv_len");
  whole(see, at::kLong, {B, N}, qkv, "tree_attention tree");
  if (has(kv_start)) whole(*kv_start, at::kInt, {B}, qkv, "tree_attention kv_start");
  TORCH_CHECK(Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && qkv.size(0) == B * N && qkv.size(1) >= (Hq + 2 * Hkv) * D, "tree_attention: qkv shape");
  on(out, qkv, "tree_attention out");
  TORCH_CHECK(out.scalar_type() == qkv.scalar_type() && out.size(0) == B * N && out.size(1) == Hq * D, "tree_attention: out shape");
  TORCH_CHECK(Smax * D < (1L << 30) && window >= 0 && window < (1L << 30) && scale > 0, "tree_attention: sizes");
  const c10::DeviceGuard guard(qkv.device());
  const int64_t S = qkv.scalar_type() == at::kBFloat16 && al(kc, 16) && al(vc, 16)
                        ? rt_tree_parts((int)B, (int)N, (int)Hq, (int)Hkv, (int)D, (int)Smax) : 0;
  // matrix instructions want rows at 16 bytes (the output at 8): others are copied
  Tensor x = qkv, o = out;
  if (S && !(al(x, 16) && x.stride(0) % 8 == 0 && x.stride(0) < (1L << 24))) x = qkv.narrow(1, 0, (Hq + 2 * Hkv) * D).clone(at::MemoryFormat::Contiguous);
  if (S && !(al(o, 8) && o.stride(0) % 4 == 0)) o = at::empty({B * N, Hq * D}, qkv.options());
  Tensor part = S > 1 ? at::empty({S * B * Hq * N * (D + 2)}, qkv.options().dtype(at::kFloat)) : Tensor();
  rc_ok(rt_tree_attention(x.scalar_type() == at::kFloat, x.data_ptr(), x.stride(0), kc.data_ptr(), vc.data_ptr(), kv_len.data_ptr<int>(),
                          ptr<int>(kv_start), see.data_ptr<int64_t>(), o.data_ptr(), o.stride(0), S > 1 ? part.data_ptr<float>() : nullptr,
                          (int)S, (int)B, (int)N, (int)Hq, (int)Hkv, (int)D, (int)Smax, (int)window, (float)scale, stream()), "tree_attention");
  if (!o.is_same(out)) out.copy_(o);
}

std::vector<Tensor> tree_accept(const Tensor& parent, const Tensor& see, const Tensor& tokens, const Tensor& choice,
                                const std::vector<Tensor>& drafts, Tensor kc, Tensor vc, const Tensor& kv_len) {
  act(kc, "tree_accept k_cache");
  TORCH_CHECK(kc.dim() == 5 && see.dim() == 2 && drafts.size() && (int64_t)drafts.size() == kc.size(0) && drafts.size() <= 256,
              "tree_accept: caches [layers, rows, heads, slots, dim] and rows of every layer (256 at most)");
  const int64_t L = kc.size(0), B = kc.size(1), Hkv = kc.size(2), Smax = kc.size(3), D = kc.size(4), N = see.size(1);
  on(vc, kc, "tree_accept v_cache");
  TORCH_CHECK(vc.scalar_type() == kc.scalar_type() && vc.sizes() == kc.sizes() && vc.strides() == kc.strides() && kc[0].is_contiguous(),
              "tree_accept: caches of one type and layout, contiguous in each layer");
  whole(kv_len, at::kInt, {B}, kc, "tree_accept kv_len");
  whole(parent, at::kInt, {B, N}, kc, "tree_accept tree");
  whole(see, at::kLong, {B, N}, kc, "tree_accept tree");
  whole(tokens, at::kLong, {B, N}, kc, "tree_accept tokens");
  whole(choice, at::kLong, {B, N}, kc, "tree_accept choice");
  std::vector<const void*> at;
  for (const Tensor& x : drafts) {
    on(x, kc, "tree_accept drafts");
    TORCH_CHECK(x.scalar_type() == kc.scalar_type() && x.dim() == 2 && x.stride(1) == 1 && x.sizes() == drafts[0].sizes() &&
                    x.stride(0) == drafts[0].stride(0) && x.size(0) == B * N && x.size(1) % D == 0 && x.size(1) / D > 2 * Hkv,
                "tree_accept: drafts [rows nodes, (heads + 2 key heads) dim] of the caches' type, alike in every layer");
    at.push_back(x.data_ptr());
  }
  const int64_t Hq = drafts[0].size(1) / D - 2 * Hkv;
  TORCH_CHECK(N * Hkv * D < (1L << 30), "tree_accept: sizes");
  const c10::DeviceGuard guard(kc.device());
  Tensor count = at::empty({B}, parent.options()), path = at::empty({B, N}, parent.options()), next = at::empty({B}, tokens.options());
  rc_ok(rt_tree_accept(parent.data_ptr<int>(), see.data_ptr<int64_t>(), tokens.data_ptr<int64_t>(), choice.data_ptr<int64_t>(),
                       kv_len.data_ptr<int>(), count.data_ptr<int>(), path.data_ptr<int>(), next.data_ptr<int64_t>(), at.data(),
                       drafts[0].stride(0), kc.data_ptr(), vc.data_ptr(), kc.stride(0), (int)B, (int)N, (int)L, (int)Hq, (int)Hkv, (int)Smax, (int)D,
                       (int)kc.element_size(), stream()), "tree_accept");
  return {count, path, next};
}

void logit_rows(const Tensor& logits, const optional<Tensor>& targets, int64_t top) {
  act(logits, "alternatives logits");
  TORCH_CHECK(logits.dim() == 2 && (logits.stride(1) == 1 || logits.size(1) == 1) && logits.size(1) < (1L << 30), "alternatives: logits [tokens, vocabulary]");
  TORCH_CHECK(top >= 1 && top <= 32 && top <= logits.size(1), "alternatives: 1 to 32 alternatives of the vocabulary");
  if (has(targets)) whole(*targets, at::kLong, {logits.size(0)}, logits, "alternatives targets");
}

// -> logp, entropy, alternatives' log-probabilities, their ids, and what the gradient needs of each row
std::vector<Tensor> alternatives(const Tensor& logits, const optional<Tensor>& targets, double c, int64_t top, bool need_stats) {
  logit_rows(logits, targets, top);
  const int64_t T = logits.size(0), V = logits.size(1);
  const c10::DeviceGuard guard(logits.device());
  const auto f = logits.options().dtype(at::kFloat);
  Tensor logp = at::empty({T}, f), ent = at::empty({T}, f), lp = at::empty({T, top}, f), stats = at::empty({need_stats ? T : 0, 3}, f);
  Tensor ids = at::empty({T, top}, logits.options().dtype(at::kLong));
  rc_ok(rt_alternatives(logits.scalar_type() == at::kFloat, logits.data_ptr(), logits.stride(0), ptr<int64_t>(targets), (float)c, T, (int)V,
                        (int)top, logp.data_ptr<float>(), ent.data_ptr<float>(), lp.data_ptr<float>(), ids.data_ptr<int64_t>(),
                        need_stats ? stats.data_ptr<float>() : nullptr, stream()), "alternatives");
  return {logp, ent, lp, ids, stats};
}

Tensor alternatives_bwd(const Tensor& logits, const optional<Tensor>& targets, double c, const Tensor& ids, const Tensor& stats,
                        const optional<Tensor>& g_lp, const optional<Tensor>& g_ent, const optional<Tensor>& g_top) {
  TORCH_CHECK(ids.dim() == 2, "alternatives_bwd: ids");
  const int64_t T = logits.size(0), V = logits.size(1), top = ids.size(1);
  logit_rows(logits, targets, top);
  whole(ids, at::kLong, {T, top}, logits, "alternatives_bwd ids");
  whole(stats, at::kFloat, {T, 3}, logits, "alternatives_bwd stats");
  for (const auto* g : {&g_lp, &g_ent})
    if (has(*g)) whole(**g, at::kFloat, {T}, logits, "alternatives_bwd gradients");
  if (has(g_top)) whole(*g_top, at::kFloat, {T, top}, logits, "alternatives_bwd gradients");
  const c10::DeviceGuard guard(logits.device());
  Tensor d = at::empty({T, V}, logits.options());
  rc_ok(rt_alternatives_bwd(logits.scalar_type() == at::kFloat, logits.data_ptr(), logits.stride(0), ptr<int64_t>(targets), (float)c, T, (int)V,
                            (int)top, ids.data_ptr<int64_t>(), stats.data_ptr<float>(), ptr<float>(g_lp), ptr<float>(g_ent),
                            ptr<float>(g_top), d.data_ptr(), d.stride(0), stream()), "alternatives_bwd");
  return d;
}

}  // namespace

void bind_drafts(py::module_& m) {
  m.def("draft_tree", &draft_tree, "ancestors and positions of drafted tokens");
  m.def("tree_attention", &tree_attention, "attention of drafted tokens over the cache and their ancestors");
  m.def("tree_accept", &tree_accept, "the agreed path of a tree, appended to the caches");
  m.def("alternatives", &alternatives, "log-probabilities of tokens, entropy and the best alternatives");
  m.def("alternatives_bwd", &alternatives_bwd, "gradient of alternatives");
}
