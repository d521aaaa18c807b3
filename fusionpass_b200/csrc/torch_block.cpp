// The quantised block's operators in the torch extension: RMS norm of a sum with its
// output in the input's type or in 8 bits, the 8-bit linear and score attention
// (include/fpkern.h).
//
// They allocate their results (and workspaces) from torch's allocator, run on torch's
// current stream of the tensors' device and raise as the other entry points do:
// ValueError for arguments that cannot describe a call, RuntimeError for a CPU tensor
// or a status of the library.  They have no derivative and refuse an input that asks for one.
#include <cmath>
#include <cstring>

#include "torch_ext.h"

namespace fpk_ext {
namespace {

int64_t pitch16(int64_t cols) { return (cols + 15) / 16 * 16; }

// -> (y | (q, scale)) and, with return_sum, the sum
pybind11::tuple rms_norm(const std::vector<at::Tensor>& addends, const optional<at::Tensor>& weight, double eps,
                         const optional<std::vector<int64_t>>& shape, bool quantize, bool norm, bool return_sum,
                         const optional<at::Tensor>& out) {
  const char* what = norm ? "rms_norm" : "quantize_q8";
  if (addends.empty() || addends.size() > 4) value_error(std::string(what) + ": 1 to 4 addends");
  for (const at::Tensor& t : addends) require_cuda(t, what);
  const at::Device dev = addends[0].device();
  const at::ScalarType dt = addends[0].scalar_type();
  size_t widest = 0;
  for (size_t i = 1; i < addends.size(); ++i)
    if (addends[i].numel() > addends[widest].numel()) widest = i;
  const std::vector<int64_t> dims = shape.has_value() ? *shape : addends[widest].sizes().vec();
  if (dims.empty()) value_error(std::string(what) + ": at least one dim is needed");
  fpk_rms_desc d;
  std::memset(&d, 0, sizeof(d));
  d.size = sizeof(d);
  d.version = FPK_ABI_VERSION;
  d.dtype = type_code(dt, what);
  d.cols = dims.back();
  d.rows = 1;
  for (size_t i = 0; i + 1 < dims.size(); ++i) d.rows *= dims[i];
  d.eps = static_cast<float>(eps);
  d.flags = norm ? 0u : FPK_RMS_QUANT_ONLY;
  if (d.cols < 1) value_error(std::string(what) + ": the last dim must not be empty");
  if (!(eps >= 0.0)) value_error(std::string(what) + ": eps must not be negative");
  const void* ptrs[4];
  int32_t bc[4];
  std::vector<at::Tensor> kept;
  for (size_t i = 0; i < addends.size(); ++i) {
    check_tensor(addends[i], dev, what, "an addend");
    if (addends[i].scalar_type() != dt) value_error(std::string(what) + ": addends must share one dtype");
    if (addends[i].sizes() == at::IntArrayRef(dims)) bc[i] = FPK_BCAST_FULL;
    else if (addends[i].numel() == d.cols && addends[i].dim() > 0 && addends[i].size(-1) == d.cols) bc[i] = FPK_BCAST_COL;
    else value_error(std::string(what) + ": an addend has neither the result's shape nor its last dim's size");
    kept.push_back(addends[i].contiguous());
    ptrs[i] = kept.back().data_ptr();
  }
  at::Tensor w;
  if (given(weight)) {
    check_tensor(*weight, dev, what, "weight");
    if (weight->numel() != d.cols || weight->scalar_type() != dt)
      value_error(std::string(what) + ": weight must be a vector of the last dim's size and the addends' dtype");
    w = weight->contiguous();
  }
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor y, q, scale, sum;
  if (return_sum) sum = fresh(dims, dt, dev);
  if (quantize) {
    std::vector<int64_t> padded = dims;
    padded.back() = pitch16(d.cols);
    q = fresh(padded, at::kChar, dev);
    scale = fresh(at::IntArrayRef(dims.data(), dims.size() - 1), at::kFloat, dev);
    d.q_stride = padded.back();
  } else if (given(out)) {
    y = *out;
    require_cuda(y, what);
    if (y.sizes() != at::IntArrayRef(dims) || y.scalar_type() != dt || y.device() != dev || !y.is_contiguous())
      value_error(std::string(what) + ": out must be a contiguous tensor of the result's shape, dtype and device");
    no_derivative(y, what, "out");
    for (size_t i = 0; i < kept.size(); ++i)  // a row is read before its result is stored
      if (kept[i].data_ptr() != y.data_ptr() || kept[i].numel() != y.numel()) apart(y, kept[i], what);
    if (w.defined()) apart(y, w, what);
  } else {
    y = fresh(dims, dt, dev);
  }
  if (d.rows > 0)
    check_status(fpk_rms_norm_fwd(&d, ptrs, bc, static_cast<int>(addends.size()), w.defined() ? w.data_ptr() : nullptr,
                                  sum.defined() ? sum.data_ptr() : nullptr, y.defined() ? y.data_ptr() : nullptr,
                                  q.defined() ? q.data_ptr() : nullptr,
                                  scale.defined() ? scale.data_ptr<float>() : nullptr, stream_of(addends[0])),
                 "fpk_rms_norm_fwd");
  if (given(out)) written(y);
  if (quantize && d.q_stride != d.cols) q = q.narrow(-1, 0, d.cols);
  if (quantize) return return_sum ? pybind11::make_tuple(q, scale, sum) : pybind11::make_tuple(q, scale);
  return return_sum ? pybind11::make_tuple(y, sum) : pybind11::make_tuple(y);
}

// The row stride of 8-bit rows with unit last stride and leading dims that flatten to one
// stride; any other layout is copied.  (The library lays rows out again that are not on 16
// bytes.)
at::Tensor rows_of(const at::Tensor& t, int64_t k, int64_t* stride_out) {
  int64_t stride = pitch16(k), span = 1;  // of one row: any
  bool ok = t.stride(-1) == 1 || k == 1;
  for (int64_t i = t.dim() - 2; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (span == 1) stride = t.stride(i);
    else ok = ok && t.stride(i) == stride * span;
    span *= t.size(i);
  }
  ok = ok && stride >= k;  // rows that overlap, an expanded one among them, are copied too
  *stride_out = ok ? stride : k;
  return ok ? t : t.contiguous();
}

at::Tensor linear_q8(const at::Tensor& x, const at::Tensor& x_scale, const at::Tensor& w, const at::Tensor& w_scale,
                     const optional<at::Tensor>& bias, const pybind11::object& out_dtype,
                     const optional<at::Tensor>& out) {
  const char* what = "linear_q8";
  require_cuda(x, what);
  const at::Device dev = x.device();
  for (const auto& p : {std::make_pair(&x_scale, "x_scale"), std::make_pair(&w, "w"), std::make_pair(&w_scale, "w_scale")})
    check_tensor(*p.first, dev, what, p.second);
  if (x.scalar_type() != at::kChar || w.scalar_type() != at::kChar) value_error("linear_q8: x and w must be int8");
  if (x.dim() < 1 || w.dim() != 2) value_error("linear_q8: x is [..., K] and w is [N, K]");
  const int64_t k = x.size(-1), n = w.size(0);
  if (w.size(1) != k)
    value_error("linear_q8: x has " + std::to_string(k) + " columns, w has " + std::to_string(w.size(1)));
  if (k < 1 || k > FPK_LINEAR_MAX_K)
    value_error("linear_q8: K must be 1.." + std::to_string(FPK_LINEAR_MAX_K) + " (the sum is kept in 32 bits)");
  if (x_scale.scalar_type() != at::kFloat || x_scale.sizes() != x.sizes().slice(0, x.dim() - 1))
    value_error("linear_q8: x_scale must be f32 of x's shape without its last dim");
  if (w_scale.scalar_type() != at::kFloat || w_scale.dim() != 1 || w_scale.size(0) != n)
    value_error("linear_q8: w_scale must be f32 [N]");
  const at::ScalarType dt = THPDtype_Check(out_dtype.ptr()) ? reinterpret_cast<THPDtype*>(out_dtype.ptr())->scalar_type
                                                             : at::ScalarType::Undefined;
  if (dt == at::ScalarType::Undefined) value_error("linear_q8: out_dtype must be a torch.dtype");
  fpk_linear_desc d;
  std::memset(&d, 0, sizeof(d));
  d.size = sizeof(d);
  d.version = FPK_ABI_VERSION;
  d.out_dtype = type_code(dt, what);
  d.k = k;
  d.n = n;
  d.m = x.numel() / k;
  at::Tensor b;
  if (given(bias)) {
    check_tensor(*bias, dev, what, "bias");
    if (bias->scalar_type() != dt || bias->dim() != 1 || bias->size(0) != n)
      value_error("linear_q8: bias must be a vector of N values of out_dtype");
    b = bias->contiguous();
  }
  std::vector<int64_t> dims = x.sizes().vec();
  dims.back() = n;
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor y;
  if (given(out)) {
    y = *out;
    require_cuda(y, what);
    if (y.sizes() != at::IntArrayRef(dims) || y.scalar_type() != dt || y.device() != dev || !y.is_contiguous())
      value_error("linear_q8: out must be a contiguous tensor of the result's shape, out_dtype and device");
    no_derivative(y, what, "out");
  } else {
    y = fresh(dims, dt, dev);
  }
  if (d.m == 0 || d.n == 0) return y;
  const at::Tensor rx = rows_of(x, k, &d.x_stride), rw = rows_of(w, k, &d.w_stride);
  d.y_stride = n;
  const int64_t bytes = fpk_linear_int_workspace(&d, rx.data_ptr(), rw.data_ptr());
  if (bytes < 0) check_status(static_cast<int>(bytes), "fpk_linear_int_workspace");
  at::Tensor room;
  if (bytes > 0) room = fresh({bytes}, at::kByte, dev);
  const at::Tensor xs = x_scale.contiguous(), ws = w_scale.contiguous();
  if (given(out)) {
    for (const at::Tensor* t : {&rx, &rw, &xs, &ws}) apart(y, *t, what);
    if (b.defined()) apart(y, b, what);
  }
  check_status(fpk_linear_int_fwd(&d, rx.data_ptr(), xs.data_ptr<float>(), rw.data_ptr(), ws.data_ptr<float>(),
                                  b.defined() ? b.data_ptr() : nullptr, y.data_ptr(),
                                  bytes > 0 ? room.data_ptr() : nullptr, bytes, stream_of(x)),
               "fpk_linear_int_fwd");
  if (given(out)) written(y);
  return y;
}

const int32_t* int_vector(const optional<at::Tensor>& t, const at::Device& dev, int64_t n, const char* name,
                          std::vector<at::Tensor>* keep) {
  if (!given(t)) return nullptr;
  check_tensor(*t, dev, "score_attention", name);
  if (t->scalar_type() != at::kInt || t->dim() != 1 || t->size(0) != n)
    value_error(std::string("score_attention: ") + name + " must be int32 [" + std::to_string(n) + "]");
  keep->push_back(t->contiguous());
  return keep->back().data_ptr<int32_t>();
}

at::Tensor score_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, double scale,
                           const optional<double>& softcap, const optional<at::Tensor>& slopes, bool causal,
                           const optional<int64_t>& window, int64_t prefix, const optional<at::Tensor>& prefix_lens,
                           const optional<at::Tensor>& doc_ids, const optional<at::Tensor>& kv_lens,
                           const optional<at::Tensor>& out) {
  const char* what = "score_attention";
  require_cuda(q, what);
  const at::Device dev = q.device();
  check_tensor(q, dev, what, "q");
  check_tensor(k, dev, what, "k");
  check_tensor(v, dev, what, "v");
  if (q.dim() != 4 || k.dim() != 4 || v.dim() != 4) value_error("score_attention: q, k and v are [B, heads, S, D]");
  if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
    value_error("score_attention: q, k and v must share one dtype");
  if (k.sizes() != v.sizes() || k.size(0) != q.size(0) || k.size(3) != q.size(3))
    value_error("score_attention: k and v must share one shape, and batch and head dim with q");
  fpk_score_desc d;
  std::memset(&d, 0, sizeof(d));
  d.size = sizeof(d);
  d.version = FPK_ABI_VERSION;
  d.dtype = type_code(q.scalar_type(), what);
  d.batch = q.size(0);
  d.heads = q.size(1);
  d.q_len = q.size(2);
  d.head_dim = static_cast<int32_t>(q.size(3));
  d.kv_heads = k.size(1);
  d.k_len = k.size(2);
  if (d.head_dim != 16 && d.head_dim != 32 && d.head_dim != 64 && d.head_dim != 128)
    value_error("score_attention: head dim " + std::to_string(q.size(3)) + " (16, 32, 64 and 128 only)");
  if (d.heads > 0 && (d.kv_heads < 1 || d.heads % d.kv_heads))
    value_error("score_attention: " + std::to_string(d.heads) + " heads over " + std::to_string(d.kv_heads) +
                " key/value heads");
  d.scale = static_cast<float>(scale);
  if (!std::isfinite(d.scale * 1.4426950408889634f)) value_error("score_attention: scale must be finite, and 1.44 times it");
  if (softcap.has_value()) {
    d.softcap = static_cast<float>(*softcap);
    if (!(d.softcap > 0.0f) || !std::isfinite(d.softcap)) value_error("score_attention: softcap must be positive");
    if (!std::isfinite(2.8853900817779268f * d.scale / d.softcap))
      value_error("score_attention: softcap is too small for this scale");
    if (d.softcap > FPK_SCORE_MAX_CAP && d.dtype != FPK_F32)
      value_error("score_attention: softcap above " + std::to_string(FPK_SCORE_MAX_CAP) + " is for f32 only");
  }
  if (window.has_value()) {
    d.window = *window;
    if (d.window < 1) value_error("score_attention: window must be at least 1");
  }
  if (prefix < 0) value_error("score_attention: prefix must not be negative");
  d.prefix = prefix;
  d.flags = causal ? FPK_SCORE_CAUSAL : 0u;
  std::vector<at::Tensor> keep;
  if (given(slopes)) {
    check_tensor(*slopes, dev, what, "slopes");
    if (slopes->scalar_type() != at::kFloat || slopes->dim() != 1 || slopes->size(0) != d.heads)
      value_error("score_attention: slopes must be f32 [heads]");
    keep.push_back(slopes->contiguous());
    d.slopes = keep.back().data_ptr<float>();
  }
  d.prefix_lens = int_vector(prefix_lens, dev, d.batch, "prefix", &keep);
  d.kv_lens = int_vector(kv_lens, dev, d.batch, "kv_lens", &keep);
  if (given(doc_ids)) {
    check_tensor(*doc_ids, dev, what, "doc_ids");
    if (doc_ids->scalar_type() != at::kInt || doc_ids->dim() != 2 || doc_ids->size(0) != d.batch ||
        doc_ids->size(1) != d.k_len)
      value_error("score_attention: doc_ids must be int32 [B, keys]");
    keep.push_back(doc_ids->stride(1) == 1 ? *doc_ids : doc_ids->contiguous());
    d.doc_ids = keep.back().data_ptr<int32_t>();
    d.ids_stride = keep.back().stride(0);
  }
  const c10::cuda::CUDAGuard guard(dev);
  const int64_t unit = d.dtype == FPK_F32 ? 4 : 8;
  const at::Tensor qa = aligned(q, unit, d.q_strides), ka = aligned(k, unit, d.k_strides),
                   va = aligned(v, unit, d.v_strides);
  at::Tensor o;
  if (given(out)) {
    require_cuda(*out, what);
    if (out->sizes() != q.sizes() || out->scalar_type() != q.scalar_type() || out->device() != dev)
      value_error("score_attention: out must match q's shape, dtype and device");
    no_derivative(*out, what, "out");
    o = *out;
    if (o.numel() > 0 && aligned(o, unit, d.o_strides).data_ptr() != o.data_ptr())
      value_error("score_attention: out must have a unit last stride, and a base and other strides of 16-byte multiples");
  } else {
    o = fresh(q.sizes(), q.scalar_type(), dev);
    aligned(o, unit, d.o_strides);
  }
  if (o.numel() == 0) return o;
  if (given(out)) {
    for (const at::Tensor* t : {&qa, &ka, &va}) apart(o, *t, what);
    for (const at::Tensor& t : keep) apart(o, t, what);
  }
  if (ka.numel() == 0)  // no keys: every row is empty
    for (int i = 0; i < 3; ++i) d.k_strides[i] = d.v_strides[i] = unit;
  const int64_t bytes = fpk_score_attention_workspace(&d);
  if (bytes < 0) check_status(static_cast<int>(bytes), "fpk_score_attention_workspace");
  at::Tensor ws;
  if (bytes > 0) ws = fresh({bytes}, at::kByte, dev);
  check_status(fpk_score_attention_fwd(&d, qa.data_ptr(), ka.data_ptr(), va.data_ptr(), o.data_ptr(),
                                       bytes > 0 ? ws.data_ptr() : nullptr, bytes, stream_of(q)),
               "fpk_score_attention_fwd");
  if (given(out)) written(o);
  return o;
}

}  // namespace

void bind_block(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("rms_norm", &rms_norm, "RMS norm (or the 8-bit form alone) of the sum of 1..4 addends", py::arg("addends"),
        py::arg("weight"), py::arg("eps"), py::arg("shape") = py::none(), py::arg("quantize") = false,
        py::arg("norm") = true, py::arg("return_sum") = false, py::arg("out") = py::none());
  m.def("linear_q8", &linear_q8, "8-bit product with a scale a token and a scale an output channel", py::arg("x"),
        py::arg("x_scale"), py::arg("w"), py::arg("w_scale"), py::arg("bias"), py::arg("out_dtype"),
        py::arg("out") = py::none());
  m.def("score_attention", &score_attention, "attention with capped, biased and masked scores", py::arg("q"),
        py::arg("k"), py::arg("v"), py::arg("scale"), py::arg("softcap"), py::arg("slopes"), py::arg("causal"),
        py::arg("window"), py::arg("prefix"), py::arg("prefix_lens"), py::arg("doc_ids"), py::arg("kv_lens"),
        py::arg("out"));
}

}  // namespace fpk_ext
