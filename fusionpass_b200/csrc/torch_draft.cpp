// Speculative decoding's operators in the torch extension: the 8-bit cache, attention of a tree
// of drafted tokens and the verification of drafted tokens (include/fpkern.h).  They allocate,
// run and raise as the quantised block's operators do (torch_block.cpp).
#include <cmath>
#include <cstring>

#include "torch_ext.h"

namespace fpk_ext {
namespace {

using Optional = c10::optional<at::Tensor>;

// int32 [n] on dev, contiguous
const int32_t* int_vector(const at::Tensor& t, const at::Device& dev, int64_t n, const char* what, const char* name,
                          std::vector<at::Tensor>* keep) {
  check_tensor(t, dev, what, name);
  if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != n)
    value_error(std::string(what) + ": " + name + " must be int32 [" + std::to_string(n) + "]");
  keep->push_back(t.contiguous());
  return keep->back().data_ptr<int32_t>();
}

// [B, T] of one type with a unit last stride, or [T] for all sequences (stride 0)
template <typename E>
const E* table(const at::Tensor& t, at::ScalarType type, const at::Device& dev, int64_t batch, int64_t cols, bool shared,
               const char* what, const char* name, int64_t* stride, std::vector<at::Tensor>* keep) {
  check_tensor(t, dev, what, name);
  const bool one = shared && t.dim() == 1;
  if (t.scalar_type() != type || (!one && (t.dim() != 2 || t.size(0) != batch)) || t.size(-1) != cols)
    value_error(std::string(what) + ": " + name + " must be " + c10::toString(type) + " [" + std::to_string(batch) + ", " +
                std::to_string(cols) + "]" + (shared ? " or [" + std::to_string(cols) + "]" : ""));
  keep->push_back(t.stride(-1) == 1 || cols == 1 ? t : t.contiguous());
  *stride = one ? 0 : keep->back().stride(0);
  return keep->back().data_ptr<E>();
}

bool head_dim_ok(int64_t d) { return d == 16 || d == 32 || d == 64 || d == 128; }

// a tensor that is written in place: no two of its elements share memory
void own_memory(const at::Tensor& t, const char* what, const char* name) {
  if (at::has_internal_overlap(t) == at::MemOverlap::Yes)
    value_error(std::string(what) + ": " + name + " has elements that share memory");
}

// An 8-bit cache [B, Hk, N, D] with its scales [B, Hk, N], read and written where it is
void check_cache(const at::Tensor& c, const at::Tensor& s, const at::Device& dev, const char* what, const char* name,
                 bool written) {
  check_tensor(c, dev, what, name);
  check_tensor(s, dev, what, name);
  if (c.scalar_type() != at::kChar || c.dim() != 4) value_error(std::string(what) + ": " + name + " must be int8 [B, heads, room, D]");
  if (s.scalar_type() != at::kFloat || s.sizes() != c.sizes().slice(0, 3))
    value_error(std::string(what) + ": the scale of " + name + " must be f32 [B, heads, room]");
  if (!head_dim_ok(c.size(3)))
    value_error(std::string(what) + ": head dim " + std::to_string(c.size(3)) + " (16, 32, 64 and 128 only)");
  if (written) {
    own_memory(c, what, name);
    own_memory(s, what, name);
  }
}
// whether the kernels can take the cache where it is
bool cache_strides(const at::Tensor& t, int64_t* st) {
  bool ok = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int i = 0; i < 3; ++i) {
    st[i] = t.size(i) == 1 ? t.size(3) : t.stride(i);  // the stride of a dim of one is never used
    ok = ok && st[i] % 16 == 0;
  }
  return ok || t.numel() == 0;
}
void in_place(const at::Tensor& t, const char* what, const char* name) {
  int64_t st[3];
  if (!cache_strides(t, st))
    value_error(std::string(what) + ": " + name + " must have a unit last stride, and a base and other strides of 16-byte multiples");
}
void scale_strides(const at::Tensor& t, int64_t* st) {
  for (int i = 0; i < 3; ++i) st[i] = t.size(i) == 1 ? 1 : t.stride(i);
}

fpk_cache_desc cache_desc(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks, const at::Tensor& vs,
                          const char* what) {
  if (kc.sizes() != vc.sizes()) value_error(std::string(what) + ": the caches must share one shape");
  fpk_cache_desc d;
  std::memset(&d, 0, sizeof(d));
  d.size = sizeof(d);
  d.version = FPK_ABI_VERSION;
  d.head_dim = static_cast<int32_t>(kc.size(3));
  d.batch = kc.size(0);
  d.heads = kc.size(1);
  d.room = kc.size(2);
  cache_strides(kc, d.k_cache_strides);
  cache_strides(vc, d.v_cache_strides);
  scale_strides(ks, d.k_scale_strides);
  scale_strides(vs, d.v_scale_strides);
  return d;
}

void cache_write(const at::Tensor& k, const at::Tensor& v, const at::Tensor& kc, const at::Tensor& vc,
                 const at::Tensor& ks, const at::Tensor& vs, const at::Tensor& past, const Optional& new_lens) {
  const char* what = "cache_write_q8";
  require_cuda(k, what);
  const at::Device dev = k.device();
  check_tensor(k, dev, what, "k");
  check_tensor(v, dev, what, "v");
  check_cache(kc, ks, dev, what, "k_cache", true);
  check_cache(vc, vs, dev, what, "v_cache", true);
  in_place(kc, what, "k_cache");
  in_place(vc, what, "v_cache");
  if (k.dim() != 4 || k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type())
    value_error("cache_write_q8: k and v must be [B, heads, rows, D] of one shape and dtype");
  fpk_cache_desc d = cache_desc(kc, vc, ks, vs, what);
  if (k.size(0) != d.batch || k.size(1) != d.heads || k.size(3) != d.head_dim)
    value_error("cache_write_q8: k and v must share batch, heads and head dim with the caches");
  d.dtype = type_code(k.scalar_type(), what);
  d.rows = k.size(2);
  std::vector<at::Tensor> keep;
  d.past_lens = int_vector(past, dev, d.batch, what, "past_lens", &keep);
  if (given(new_lens)) d.lens = int_vector(*new_lens, dev, d.batch, what, "new_lens", &keep);
  const at::Tensor* outs[4] = {&kc, &vc, &ks, &vs};
  for (int i = 0; i < 4; ++i) {
    for (int j = 0; j < i; ++j) apart(*outs[i], *outs[j], what);
    for (const at::Tensor* t : {&k, &v}) apart(*outs[i], *t, what);
    for (const at::Tensor& t : keep) apart(*outs[i], t, what);
  }
  const c10::cuda::CUDAGuard guard(dev);
  const int64_t unit = d.dtype == FPK_F32 ? 4 : 8;
  const at::Tensor ka = aligned(k, unit, d.k_strides), va = aligned(v, unit, d.v_strides);
  if (ka.numel() == 0 || kc.numel() == 0) return;
  check_status(fpk_cache_write(&d, ka.data_ptr(), va.data_ptr(), kc.data_ptr(), vc.data_ptr(), ks.data_ptr<float>(),
                               vs.data_ptr<float>(), stream_of(k)),
               "fpk_cache_write");
  for (const at::Tensor* t : outs) written(*t);
}

pybind11::tuple cache_read(const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& ks, const at::Tensor& vs,
                           const pybind11::object& dtype, const Optional& kv_lens) {
  const char* what = "cache_read_q8";
  require_cuda(k_cache, what);
  const at::Device dev = k_cache.device();
  check_cache(k_cache, ks, dev, what, "k_cache", false);
  check_cache(v_cache, vs, dev, what, "v_cache", false);
  const auto there = [](const at::Tensor& t) {  // copied where its layout is not the kernel's
    int64_t st[3];
    return cache_strides(t, st) ? t : t.clone(at::MemoryFormat::Contiguous);
  };
  const at::Tensor kc = there(k_cache), vc = there(v_cache);
  fpk_cache_desc d = cache_desc(kc, vc, ks, vs, what);
  if (!THPDtype_Check(dtype.ptr())) value_error("cache_read_q8: dtype must be a torch.dtype");
  const at::ScalarType dt = reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type;
  d.dtype = type_code(dt, what);
  d.rows = d.room;
  std::vector<at::Tensor> keep;
  if (given(kv_lens)) d.lens = int_vector(*kv_lens, dev, d.batch, what, "kv_lens", &keep);
  const c10::cuda::CUDAGuard guard(dev);
  const at::Tensor k = fresh(kc.sizes(), dt, dev), v = fresh(kc.sizes(), dt, dev);
  if (k.numel() > 0) {
    for (int i = 0; i < 3; ++i) d.k_strides[i] = d.v_strides[i] = k.stride(i);
    check_status(fpk_cache_read(&d, kc.data_ptr(), vc.data_ptr(), ks.data_ptr<float>(), vs.data_ptr<float>(),
                                k.data_ptr(), v.data_ptr(), stream_of(kc)),
                 "fpk_cache_read");
  }
  return pybind11::make_tuple(k, v);
}

void cache_keep(const std::vector<at::Tensor>& caches, const at::Tensor& path, const at::Tensor& counts,
                const at::Tensor& past) {
  const char* what = "cache_keep";
  if (caches.empty() || caches.size() > FPK_KEEP_MAX_CACHES)
    value_error("cache_keep: 1 to " + std::to_string(FPK_KEEP_MAX_CACHES) + " caches");
  require_cuda(caches[0], what);
  const at::Device dev = caches[0].device();
  fpk_keep_desc d;
  std::memset(&d, 0, sizeof(d));
  d.size = sizeof(d);
  d.version = FPK_ABI_VERSION;
  d.batch = caches[0].dim() > 0 ? caches[0].size(0) : 0;
  std::vector<fpk_keep_cache> c(caches.size());
  for (size_t i = 0; i < caches.size(); ++i) {
    const at::Tensor& t = caches[i];
    check_tensor(t, dev, what, "a cache");
    if ((t.dim() != 3 && t.dim() != 4) || t.size(0) != d.batch)
      value_error("cache_keep: a cache is [B, heads, room, D] or [B, heads, room], of one B");
    const int64_t cols = t.dim() == 4 ? t.size(3) : 1, size = t.element_size();
    if (cols > 1 && t.stride(3) != 1) value_error("cache_keep: a cache must have a unit last stride");
    if (cols * size > 1 << 30 || t.size(1) > 1 << 30) value_error("cache_keep: a cache's rows, or heads, are too many");
    own_memory(t, what, "a cache");
    c[i].data = t.data_ptr();
    for (int j = 0; j < 3; ++j) c[i].strides[j] = t.size(j) == 1 ? 0 : t.stride(j) * size;
    c[i].room = t.size(2);
    c[i].heads = cols > 0 ? static_cast<int32_t>(t.size(1)) : 0;
    c[i].row_bytes = static_cast<int32_t>(std::max<int64_t>(cols, 1) * size);
  }
  std::vector<at::Tensor> keep;
  if (path.dim() != 2) value_error("cache_keep: path must be int32 [B, n]");
  if (path.size(1) > FPK_TREE_MAX_NODES)
    value_error("cache_keep: a path has at most " + std::to_string(FPK_TREE_MAX_NODES) + " entries");
  d.n_caches = static_cast<int32_t>(caches.size());
  d.n_path = static_cast<int32_t>(path.size(1));
  d.path = table<int32_t>(path, at::kInt, dev, d.batch, path.size(1), false, what, "path", &d.path_stride, &keep);
  d.counts = int_vector(counts, dev, d.batch, what, "counts", &keep);
  d.past_lens = int_vector(past, dev, d.batch, what, "past_lens", &keep);
  for (size_t i = 0; i < caches.size(); ++i) {
    for (size_t j = 0; j < i; ++j)
      if (caches[i].storage().data() == caches[j].storage().data()) apart(caches[i], caches[j], what);
    for (const at::Tensor& t : keep) apart(caches[i], t, what);
  }
  const c10::cuda::CUDAGuard guard(dev);
  check_status(fpk_cache_keep(&d, c.data(), stream_of(caches[0])), "fpk_cache_keep");
  for (const at::Tensor& t : caches) written(t);
}

at::Tensor tree_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, double scale,
                          const at::Tensor& parents, const at::Tensor& past, const Optional& tree_lens,
                          const Optional& k_scale, const Optional& v_scale, const Optional& out) {
  const char* what = "tree_attention";
  require_cuda(q, what);
  const at::Device dev = q.device();
  check_tensor(q, dev, what, "q");
  check_tensor(k, dev, what, "k");
  check_tensor(v, dev, what, "v");
  if (q.dim() != 4 || k.dim() != 4 || v.dim() != 4)
    value_error("tree_attention: q is [B, heads, nodes, D], k and v are [B, key/value heads, room, D]");
  const bool q8 = given(k_scale);
  if (q8 != given(v_scale)) value_error("tree_attention: give both k_scale and v_scale, or neither");
  const at::ScalarType kv = q8 ? at::kChar : q.scalar_type();
  if (k.scalar_type() != kv || v.scalar_type() != kv)
    value_error(q8 ? "tree_attention: k and v with scales must be int8"
                   : "tree_attention: k and v must have q's dtype, or be int8 with scales");
  if (k.sizes() != v.sizes() || k.size(0) != q.size(0) || k.size(3) != q.size(3))
    value_error("tree_attention: k and v must share one shape, and batch and head dim with q");
  fpk_tree_desc d;
  std::memset(&d, 0, sizeof(d));
  d.size = sizeof(d);
  d.version = FPK_ABI_VERSION;
  d.dtype = type_code(q.scalar_type(), what);
  d.batch = q.size(0);
  d.heads = q.size(1);
  d.nodes = q.size(2);
  d.kv_heads = k.size(1);
  d.room = k.size(2);
  d.flags = q8 ? FPK_TREE_Q8 : 0u;
  if (!head_dim_ok(q.size(3)))
    value_error("tree_attention: head dim " + std::to_string(q.size(3)) + " (16, 32, 64 and 128 only)");
  d.head_dim = static_cast<int32_t>(q.size(3));
  if (d.heads > 0 && (d.kv_heads < 1 || d.heads % d.kv_heads))
    value_error("tree_attention: " + std::to_string(d.heads) + " heads over " + std::to_string(d.kv_heads) +
                " key/value heads");
  if (d.nodes > FPK_TREE_MAX_NODES)
    value_error("tree_attention: a tree has at most " + std::to_string(FPK_TREE_MAX_NODES) + " nodes");
  d.scale = static_cast<float>(scale);
  if (!std::isfinite(d.scale * 1.4426950408889634f)) value_error("tree_attention: scale must be finite, and 1.44 times it");
  std::vector<at::Tensor> keep;
  d.parents = table<int32_t>(parents, at::kInt, dev, d.batch, d.nodes, true, what, "parents", &d.parents_stride, &keep);
  d.past_lens = int_vector(past, dev, d.batch, what, "past_lens", &keep);
  if (given(tree_lens)) d.tree_lens = int_vector(*tree_lens, dev, d.batch, what, "tree_lens", &keep);
  const c10::cuda::CUDAGuard guard(dev);
  if (q8) {
    for (const auto& s : {std::make_pair(&*k_scale, "k_scale"), std::make_pair(&*v_scale, "v_scale")}) {
      check_tensor(*s.first, dev, what, s.second);
      if (s.first->scalar_type() != at::kFloat || s.first->sizes() != k.sizes().slice(0, 3))
        value_error(std::string("tree_attention: ") + s.second + " must be f32 [B, key/value heads, room]");
      bool flat = true;  // an expanded scale is laid out: strides are positive
      for (int i = 0; i < 3; ++i) flat = flat && (s.first->size(i) == 1 || s.first->stride(i) > 0);
      keep.push_back(flat ? *s.first : s.first->contiguous());
      scale_strides(keep.back(), s.first == &*k_scale ? d.k_scale_strides : d.v_scale_strides);
      (s.first == &*k_scale ? d.k_scale : d.v_scale) = keep.back().data_ptr<float>();
    }
  }
  const int64_t unit = d.dtype == FPK_F32 ? 4 : 8, kv_unit = q8 ? 16 : unit;
  const at::Tensor qa = aligned(q, unit, d.q_strides), ka = aligned(k, kv_unit, d.k_strides),
                   va = aligned(v, kv_unit, d.v_strides);
  at::Tensor o;
  if (given(out)) {
    require_cuda(*out, what);
    if (out->sizes() != q.sizes() || out->scalar_type() != q.scalar_type() || out->device() != dev)
      value_error("tree_attention: out must match q's shape, dtype and device");
    no_derivative(*out, what, "out");
    o = *out;
    own_memory(o, what, "out");
    if (o.numel() > 0 && aligned(o, unit, d.o_strides).data_ptr() != o.data_ptr())
      value_error("tree_attention: out must have a unit last stride, and a base and other strides of 16-byte multiples");
  } else {
    o = fresh(q.sizes(), q.scalar_type(), dev);
    aligned(o, unit, d.o_strides);
  }
  if (o.numel() == 0) return o;
  if (given(out)) {
    for (const at::Tensor* t : {&qa, &ka, &va}) apart(o, *t, what);
    for (const at::Tensor& t : keep) apart(o, t, what);
  }
  if (ka.numel() == 0) {  // no rows: nothing to see
    for (int i = 0; i < 3; ++i) d.k_strides[i] = d.v_strides[i] = kv_unit;
    for (int i = 0; i < 3; ++i) d.k_scale_strides[i] = d.v_scale_strides[i] = 1;
  }
  const int64_t bytes = fpk_tree_attention_workspace(&d);
  if (bytes < 0) check_status(static_cast<int>(bytes), "fpk_tree_attention_workspace");
  at::Tensor ws;
  if (bytes > 0) ws = fresh({bytes}, at::kByte, dev);
  check_status(fpk_tree_attention_fwd(&d, qa.data_ptr(), ka.data_ptr(), va.data_ptr(), o.data_ptr(),
                                      bytes > 0 ? ws.data_ptr() : nullptr, bytes, stream_of(q)),
               "fpk_tree_attention_fwd");
  if (given(out)) written(o);
  return o;
}

// probabilities [B, T, V] with a unit last stride
const float* rows_of(const at::Tensor& t, const at::Device& dev, int64_t batch, int64_t nodes, const char* name,
                     int64_t* st, std::vector<at::Tensor>* keep) {
  check_tensor(t, dev, "verify_draft", name);
  if (t.scalar_type() != at::kFloat || t.dim() != 3 || t.size(0) != batch || t.size(1) != nodes)
    value_error(std::string("verify_draft: ") + name + " must be f32 [B, nodes, vocabulary]");
  keep->push_back(t.stride(2) == 1 || t.size(2) == 1 ? t : t.contiguous());
  st[0] = keep->back().stride(0);
  st[1] = keep->back().stride(1);
  return keep->back().data_ptr<float>();
}

pybind11::tuple verify_draft(const at::Tensor& tokens, const at::Tensor& parents, const at::Tensor& target,
                             const Optional& draft, const at::Tensor& uniform, const Optional& tree_lens) {
  const char* what = "verify_draft";
  require_cuda(target, what);
  const at::Device dev = target.device();
  if (tokens.dim() != 2) value_error("verify_draft: tokens must be int32 [B, nodes]");
  fpk_verify_desc d;
  std::memset(&d, 0, sizeof(d));
  d.size = sizeof(d);
  d.version = FPK_ABI_VERSION;
  const int64_t batch = tokens.size(0), nodes = tokens.size(1), vocab = target.dim() == 3 ? target.size(2) : 0;
  if (nodes < 1 || nodes > FPK_TREE_MAX_NODES)
    value_error("verify_draft: a tree has 1 to " + std::to_string(FPK_TREE_MAX_NODES) + " nodes");
  std::vector<at::Tensor> keep;
  const c10::cuda::CUDAGuard guard(dev);
  d.tokens = table<int32_t>(tokens, at::kInt, dev, batch, nodes, false, what, "tokens", &d.tokens_stride, &keep);
  d.parents = table<int32_t>(parents, at::kInt, dev, batch, nodes, true, what, "parents", &d.parents_stride, &keep);
  d.uniform = table<float>(uniform, at::kFloat, dev, batch, nodes, false, what, "uniform", &d.uniform_stride, &keep);
  d.target = rows_of(target, dev, batch, nodes, "target", d.target_strides, &keep);
  if (vocab < 1 || vocab > FPK_VERIFY_MAX_VOCAB)
    value_error("verify_draft: a vocabulary of 1 to " + std::to_string(FPK_VERIFY_MAX_VOCAB) + " tokens");
  if (given(draft)) {
    if (draft->dim() == 3 && draft->size(2) != vocab)
      value_error("verify_draft: target and draft must share one vocabulary");
    d.draft = rows_of(*draft, dev, batch, nodes, "draft", d.draft_strides, &keep);
  }
  if (given(tree_lens)) d.tree_lens = int_vector(*tree_lens, dev, batch, what, "tree_lens", &keep);
  d.batch = batch;
  d.nodes = static_cast<int32_t>(nodes);
  d.vocab = static_cast<int32_t>(vocab);
  const at::Tensor path = fresh({batch, nodes}, at::kInt, dev), counts = fresh({batch}, at::kInt, dev),
                   next = fresh({batch}, at::kInt, dev);
  if (batch > 0) {
    d.path = path.data_ptr<int32_t>();
    d.counts = counts.data_ptr<int32_t>();
    d.next = next.data_ptr<int32_t>();
    check_status(fpk_verify_draft(&d, stream_of(target)), "fpk_verify_draft");
  }
  return pybind11::make_tuple(path, counts, next);
}

}  // namespace

void bind_draft(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("cache_write", &cache_write, "rows of keys and values into an 8-bit cache", py::arg("k"), py::arg("v"),
        py::arg("k_cache"), py::arg("v_cache"), py::arg("k_scale"), py::arg("v_scale"), py::arg("past_lens"),
        py::arg("new_lens"));
  m.def("cache_read", &cache_read, "an 8-bit cache in another type", py::arg("k_cache"), py::arg("v_cache"),
        py::arg("k_scale"), py::arg("v_scale"), py::arg("dtype"), py::arg("kv_lens"));
  m.def("cache_keep", &cache_keep, "rows of an accepted branch moved up", py::arg("caches"), py::arg("path"),
        py::arg("counts"), py::arg("past_lens"));
  m.def("tree_attention", &tree_attention, "attention of a tree of drafted tokens over a cache", py::arg("q"),
        py::arg("k"), py::arg("v"), py::arg("scale"), py::arg("parents"), py::arg("past_lens"), py::arg("tree_lens"),
        py::arg("k_scale"), py::arg("v_scale"), py::arg("out"));
  m.def("verify_draft", &verify_draft, "which drafted tokens stand, and the next one", py::arg("tokens"),
        py::arg("parents"), py::arg("target"), py::arg("draft"), py::arg("uniform"), py::arg("tree_lens"));
}

}  // namespace fpk_ext
