// farq_fast.cpp — C++ launch path of the Python operators.
//
// The Python wrappers (task01.py, task02.py, qk_rope.py, kv_cache.py,
// dsa_attention.py) check tensors and fill the C argument structs in Python,
// which costs 10 to 25 us per call — more than the kernel itself for a few
// rows (the reference's small-M regime,
// reports/task01_fused_add_rmsnorm_group_quant.md:57). This extension does the
// same checks and the struct fill in C++ for the common case (contiguous
// tensors on one CUDA device; strided ones too for the operators of the paged
// cache) and calls the same plain-C entry points (farq_launch,
// dsa_topk_launch, dsa_kv_*_launch) on the current stream. Anything else — an
// unusual layout, a bad argument — returns -1 without launching, and the
// Python path handles the call (and raises its precise error).
#include <torch/extension.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "dsa_kv.h"
#include "dsa_topk.h"
#include "farq.h"

namespace {

constexpr int kNotHandled = -1;

int float_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return FARQ_DTYPE_BF16;
    case at::kHalf: return FARQ_DTYPE_FP16;
    case at::kFloat: return FARQ_DTYPE_FP32;
    default: return -1;
  }
}

bool same_cuda(const at::Tensor& t, const at::Device& dev) {
  return t.defined() && t.device() == dev && t.is_contiguous();
}

bool is_2d(const at::Tensor& t, int64_t rows, int64_t cols) {
  return t.dim() == 2 && t.size(0) == rows && t.size(1) == cols;
}

// fused_add_rmsnorm_group_quant (task01.py); returns farq_launch's status or
// kNotHandled.
int64_t task01(const at::Tensor& x, const at::Tensor& residual, const at::Tensor& gamma,
               const at::Tensor& residual_out, const c10::optional<at::Tensor>& norm_out,
               const at::Tensor& x_q, const at::Tensor& x_scale, double eps, int64_t group_size,
               bool ue8m0) {
  if (!x.defined() || !x.is_cuda() || x.dim() != 2) return kNotHandled;
  const at::Device dev = x.device();
  const int64_t M = x.size(0), D = x.size(1);
  if (!same_cuda(x, dev) || !same_cuda(residual, dev) || !same_cuda(gamma, dev) ||
      !same_cuda(residual_out, dev) || !same_cuda(x_q, dev) || !same_cuda(x_scale, dev))
    return kNotHandled;
  const bool write_norm = norm_out.has_value() && norm_out->defined() && norm_out->numel() > 0;
  if (write_norm && (!same_cuda(*norm_out, dev) || !is_2d(*norm_out, M, D))) return kNotHandled;
  const at::ScalarType xt = x.scalar_type();
  if ((xt != at::kBFloat16 && xt != at::kHalf) || residual.scalar_type() != xt) return kNotHandled;
  const int g_dt = float_code(gamma.scalar_type());
  const int ro_dt = float_code(residual_out.scalar_type());
  const int no_dt = write_norm ? float_code(norm_out->scalar_type()) : 0;
  const at::ScalarType qt = x_q.scalar_type();
  if (g_dt < 0 || ro_dt < 0 || no_dt < 0) return kNotHandled;
  if (qt != at::kChar && qt != at::kFloat8_e4m3fn) return kNotHandled;
  if (x_scale.scalar_type() != at::kFloat) return kNotHandled;
  if (group_size <= 0 || D % group_size != 0) return kNotHandled;
  if (gamma.dim() != 1 || gamma.size(0) != D || !is_2d(residual, M, D) ||
      !is_2d(residual_out, M, D) || !is_2d(x_q, M, D) || !is_2d(x_scale, M, D / group_size))
    return kNotHandled;
  if (M == 0) return FARQ_OK;

  farq_args_t a = {};
  a.struct_size = sizeof(farq_args_t);
  a.x_dtype = xt == at::kBFloat16 ? FARQ_DTYPE_BF16 : FARQ_DTYPE_FP16;
  a.gamma_dtype = g_dt;
  a.residual_out_dtype = ro_dt;
  a.norm_out_dtype = no_dt;
  a.q_dtype = qt == at::kChar ? FARQ_DTYPE_INT8 : FARQ_DTYPE_E4M3;
  a.flags = ue8m0 ? FARQ_FLAG_UE8M0 : 0;
  a.group_size = (int32_t)group_size;
  a.M = M;
  a.D = D;
  a.eps = (float)eps;
  a.x = x.data_ptr();
  a.residual = residual.data_ptr();
  a.gamma = gamma.data_ptr();
  a.residual_out = residual_out.data_ptr();
  a.norm_out = write_norm ? norm_out->data_ptr() : nullptr;
  a.x_q = x_q.data_ptr();
  a.x_scale = x_scale.data_ptr<float>();
  const c10::cuda::CUDAGuard guard(dev);
  return farq_launch(&a, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
}

int index_code(at::ScalarType t) {
  return t == at::kInt ? DSA_DTYPE_INT32 : t == at::kLong ? DSA_DTYPE_INT64 : -1;
}

// dsa_topk_page_table_transform (task02.py); returns dsa_topk_launch's
// status or kNotHandled.
int64_t task02(const at::Tensor& scores, const at::Tensor& page_table, const at::Tensor& q_pos,
               const at::Tensor& kv_lens, const at::Tensor& out_blocks,
               const at::Tensor& out_pages, int64_t block_size, int64_t top_k) {
  if (!scores.defined() || !scores.is_cuda() || scores.dim() != 4) return kNotHandled;
  const at::Device dev = scores.device();
  if (!same_cuda(scores, dev) || !same_cuda(page_table, dev) || !same_cuda(q_pos, dev) ||
      !same_cuda(kv_lens, dev) || !same_cuda(out_blocks, dev) || !same_cuda(out_pages, dev))
    return kNotHandled;
  const int64_t B = scores.size(0), H = scores.size(1), Q = scores.size(2), NB = scores.size(3);
  int s_dt;
  switch (scores.scalar_type()) {
    case at::kFloat: s_dt = DSA_DTYPE_FP32; break;
    case at::kBFloat16: s_dt = DSA_DTYPE_BF16; break;
    case at::kHalf: s_dt = DSA_DTYPE_FP16; break;
    default: return kNotHandled;
  }
  const int i_dt = index_code(q_pos.scalar_type());
  const int p_dt = index_code(page_table.scalar_type());
  const int b_dt = index_code(out_blocks.scalar_type());
  if (i_dt < 0 || p_dt < 0 || b_dt < 0 || kv_lens.scalar_type() != q_pos.scalar_type() ||
      out_pages.scalar_type() != page_table.scalar_type())
    return kNotHandled;
  const std::vector<int64_t> out_shape = {B, H, Q, top_k};
  if (!is_2d(page_table, B, NB) || !is_2d(q_pos, B, Q) || kv_lens.dim() != 1 ||
      kv_lens.size(0) != B || out_blocks.sizes() != at::IntArrayRef(out_shape) ||
      out_pages.sizes() != at::IntArrayRef(out_shape))
    return kNotHandled;
  dsa_topk_args_t a = {};
  a.struct_size = sizeof(dsa_topk_args_t);
  a.scores_dtype = s_dt;
  a.index_dtype = i_dt;
  a.page_dtype = p_dt;
  a.blocks_dtype = b_dt;
  a.block_size = (int32_t)block_size;
  a.top_k = (int32_t)top_k;
  if ((int64_t)a.block_size != block_size || (int64_t)a.top_k != top_k) return kNotHandled;
  a.B = B;
  a.H = H;
  a.Q = Q;
  a.NB = NB;
  a.scores = scores.data_ptr();
  a.page_table = page_table.data_ptr();
  a.q_pos = q_pos.data_ptr();
  a.kv_lens = kv_lens.data_ptr();
  a.out_blocks = out_blocks.data_ptr();
  a.out_pages = out_pages.data_ptr();
  const c10::cuda::CUDAGuard guard(dev);
  return dsa_topk_launch(&a, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
}

// ------------------------------------------------------------ the paged cache
int half_code(at::ScalarType t) {
  return t == at::kBFloat16 ? DSA_KV_BF16 : t == at::kHalf ? DSA_KV_FP16 : -1;
}
int kv_index_code(at::ScalarType t) {
  return t == at::kInt ? DSA_KV_INT32 : t == at::kLong ? DSA_KV_INT64 : -1;
}
bool on(const at::Tensor& t, const at::Device& dev) { return t.defined() && t.device() == dev; }

// A [B, Q, H, D] tensor whose last dimension is contiguous.
bool dense4(const at::Tensor& t, int64_t B, int64_t Q, int64_t H, int64_t D, at::ScalarType type,
            const at::Device& dev, dsa_kv_dense_t* d) {
  if (!on(t, dev) || t.scalar_type() != type || t.dim() != 4 || t.size(0) != B || t.size(1) != Q ||
      t.size(2) != H || t.size(3) != D || (D > 1 && t.stride(3) != 1))
    return false;
  d->ptr = t.data_ptr();
  d->stride_b = t.stride(0);
  d->stride_q = t.stride(1);
  d->stride_h = t.stride(2);
  return true;
}

bool cache_of(const at::Tensor& kc, const at::Tensor& ks, const at::Tensor& vc, const at::Tensor& vs,
              const at::Device& dev, dsa_kv_cache_t* c) {
  if (!on(kc, dev) || !on(ks, dev) || !on(vc, dev) || !on(vs, dev)) return false;
  const at::ScalarType t = kc.scalar_type();
  if ((t != at::kChar && t != at::kFloat8_e4m3fn) || vc.scalar_type() != t || ks.scalar_type() != at::kFloat ||
      vs.scalar_type() != at::kFloat || kc.dim() != 4 || ks.dim() != 3 || vs.dim() != 3 || vc.sizes() != kc.sizes() ||
      ks.sizes() != kc.sizes().slice(0, 3) || vs.sizes() != ks.sizes())
    return false;
  if (kc.size(3) > 1 && (kc.stride(3) != 1 || vc.stride(3) != 1)) return false;
  c->code_dtype = t == at::kChar ? DSA_KV_INT8 : DSA_KV_E4M3;
  c->reserved0 = 0;
  c->P = kc.size(0);
  c->H = kc.size(1);
  c->block_size = kc.size(2);
  c->D = kc.size(3);
  c->k_codes = kc.data_ptr();
  c->v_codes = vc.data_ptr();
  c->k_scale = ks.data_ptr<float>();
  c->v_scale = vs.data_ptr<float>();
  for (int i = 0; i < 3; ++i) {
    c->k_stride[i] = kc.stride(i);
    c->v_stride[i] = vc.stride(i);
    c->k_scale_stride[i] = ks.stride(i);
    c->v_scale_stride[i] = vs.stride(i);
  }
  return true;
}

// qk_rmsnorm_rope (qk_rope.py); returns dsa_kv_rope_launch's status or kNotHandled.
int64_t kv_rope(const at::Tensor& q, const at::Tensor& k, const at::Tensor& q_gamma, const at::Tensor& k_gamma,
                const at::Tensor& cos_sin, const at::Tensor& positions, const at::Tensor& q_out,
                const at::Tensor& k_out, double eps, bool interleaved) {
  if (!q.defined() || !q.is_cuda() || q.dim() != 4 || !k.defined() || k.dim() != 4) return kNotHandled;
  const at::Device dev = q.device();
  dsa_kv_rope_args_t a = {};
  a.struct_size = sizeof(a);
  a.B = q.size(0);
  a.Q = q.size(1);
  a.Hq = q.size(2);
  a.Hk = k.size(2);
  a.D = q.size(3);
  const at::ScalarType t = q.scalar_type();
  a.dtype = half_code(t);
  if (a.dtype < 0 || !dense4(q, a.B, a.Q, a.Hq, a.D, t, dev, &a.q) || !dense4(k, a.B, a.Q, a.Hk, a.D, t, dev, &a.k) ||
      !dense4(q_out, a.B, a.Q, a.Hq, a.D, t, dev, &a.q_out) || !dense4(k_out, a.B, a.Q, a.Hk, a.D, t, dev, &a.k_out))
    return kNotHandled;
  if (!same_cuda(q_gamma, dev) || !same_cuda(k_gamma, dev) || !same_cuda(cos_sin, dev) || !same_cuda(positions, dev))
    return kNotHandled;
  const at::ScalarType gt = q_gamma.scalar_type();
  a.gamma_dtype = gt == at::kFloat ? DSA_KV_FP32 : half_code(gt);
  a.pos_dtype = kv_index_code(positions.scalar_type());
  if (a.gamma_dtype < 0 || a.pos_dtype < 0 || k_gamma.scalar_type() != gt || q_gamma.dim() != 1 ||
      q_gamma.size(0) != a.D || k_gamma.dim() != 1 || k_gamma.size(0) != a.D || cos_sin.dim() != 2 ||
      cos_sin.scalar_type() != at::kFloat || !is_2d(positions, a.B, a.Q))
    return kNotHandled;
  a.max_pos = cos_sin.size(0);
  a.rot = cos_sin.size(1);
  a.interleaved = interleaved ? 1 : 0;
  a.eps = (float)eps;
  a.q_gamma = q_gamma.data_ptr();
  a.k_gamma = k_gamma.data_ptr();
  a.cos_sin = cos_sin.data_ptr<float>();
  a.positions = positions.data_ptr();
  const c10::cuda::CUDAGuard guard(dev);
  return dsa_kv_rope_launch(&a, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
}

// paged_kv_quant_write and paged_kv_dequant_read (kv_cache.py); returns the
// entry point's status or kNotHandled.
int64_t kv_copy(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache, const at::Tensor& k_scale,
                const at::Tensor& v_cache, const at::Tensor& v_scale, const at::Tensor& page_table,
                const at::Tensor& pos, bool write) {
  if (!k.defined() || !k.is_cuda() || k.dim() != 4) return kNotHandled;
  const at::Device dev = k.device();
  dsa_kv_copy_args_t a = {};
  a.struct_size = sizeof(a);
  if (!cache_of(k_cache, k_scale, v_cache, v_scale, dev, &a.cache)) return kNotHandled;
  a.B = k.size(0);
  a.Q = k.size(1);
  const at::ScalarType t = k.scalar_type();
  a.dtype = half_code(t);
  if (a.dtype < 0 || !dense4(k, a.B, a.Q, a.cache.H, a.cache.D, t, dev, &a.k) ||
      !dense4(v, a.B, a.Q, a.cache.H, a.cache.D, t, dev, &a.v) || !same_cuda(page_table, dev) || !same_cuda(pos, dev))
    return kNotHandled;
  a.page_dtype = kv_index_code(page_table.scalar_type());
  a.pos_dtype = kv_index_code(pos.scalar_type());
  if (a.page_dtype < 0 || a.pos_dtype < 0 || page_table.dim() != 2 || page_table.size(0) != a.B) return kNotHandled;
  if (write ? !is_2d(pos, a.B, a.Q) : pos.dim() != 1 || pos.size(0) != a.B) return kNotHandled;
  a.NB = page_table.size(1);
  a.page_table = page_table.data_ptr();
  a.pos = pos.data_ptr();
  const c10::cuda::CUDAGuard guard(dev);
  void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  return write ? dsa_kv_write_launch(&a, stream) : dsa_kv_read_launch(&a, stream);
}

bool selection(const at::Tensor& t, const dsa_kv_attn_args_t& a, const at::Device& dev, int32_t* code, int64_t s[3]) {
  if (!on(t, dev) || t.dim() != 4 || t.size(0) != a.B || t.size(1) != a.cache.H || t.size(2) != a.Q ||
      t.size(3) != a.K || (a.K > 1 && t.stride(3) != 1))
    return false;
  *code = kv_index_code(t.scalar_type());
  for (int i = 0; i < 3; ++i) s[i] = t.stride(i);
  return *code >= 0;
}

// dsa_paged_attention (dsa_attention.py); returns dsa_kv_attn_launch's status or kNotHandled.
int64_t kv_attn(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& k_scale, const at::Tensor& v_cache,
                const at::Tensor& v_scale, const at::Tensor& blocks, const at::Tensor& pages, const at::Tensor& q_pos,
                const at::Tensor& kv_lens, const at::Tensor& out, const at::Tensor* lse,
                double softmax_scale) {
  if (!q.defined() || !q.is_cuda() || q.dim() != 4 || !blocks.defined() || blocks.dim() != 4) return kNotHandled;
  const at::Device dev = q.device();
  dsa_kv_attn_args_t a = {};
  a.struct_size = sizeof(a);
  if (!cache_of(k_cache, k_scale, v_cache, v_scale, dev, &a.cache)) return kNotHandled;
  const int64_t Hq = q.size(2), H = a.cache.H;
  if (H < 1 || Hq < 1 || Hq % H != 0) return kNotHandled;
  a.B = q.size(0);
  a.Q = q.size(1);
  a.G = Hq / H;
  a.K = blocks.size(3);
  const at::ScalarType t = q.scalar_type();
  a.dtype = half_code(t);
  if (a.dtype < 0 || !dense4(q, a.B, a.Q, Hq, a.cache.D, t, dev, &a.q) ||
      !dense4(out, a.B, a.Q, Hq, a.cache.D, t, dev, &a.out) ||
      !selection(blocks, a, dev, &a.block_dtype, a.blocks_stride) ||
      !selection(pages, a, dev, &a.page_dtype, a.pages_stride) || !same_cuda(q_pos, dev) || !same_cuda(kv_lens, dev))
    return kNotHandled;
  a.pos_dtype = kv_index_code(q_pos.scalar_type());
  if (a.pos_dtype < 0 || kv_lens.scalar_type() != q_pos.scalar_type() || !is_2d(q_pos, a.B, a.Q) ||
      kv_lens.dim() != 1 || kv_lens.size(0) != a.B)
    return kNotHandled;
  if (lse) {
    if (!same_cuda(*lse, dev) || lse->scalar_type() != at::kFloat || lse->dim() != 3 || lse->size(0) != a.B ||
        lse->size(1) != a.Q || lse->size(2) != Hq)
      return kNotHandled;
    a.lse = lse->data_ptr<float>();
  }
  a.softmax_scale = (float)softmax_scale;
  a.blocks = blocks.data_ptr();
  a.pages = pages.data_ptr();
  a.q_pos = q_pos.data_ptr();
  a.kv_lens = kv_lens.data_ptr();
  const c10::cuda::CUDAGuard guard(dev);
  return dsa_kv_attn_launch(&a, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
}

// Entry points of the above without pybind11's argument conversion, which takes
// about as long as the checks: positional arguments only, tensors (or
// parameters) and nothing derived from them; anything else is not handled.
bool tensors(PyObject* const* args, int n) {
  for (int i = 0; i < n; ++i)
    if (!THPVariable_CheckExact(args[i])) return false;
  return true;
}
const at::Tensor& tensor(PyObject* o) { return THPVariable_Unpack(o); }
bool number(PyObject* o, double* v) {
  *v = PyFloat_AsDouble(o);
  if (*v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}
template <typename F>
PyObject* answer(const F& f) {
  int64_t st;
  try {
    st = f();
  } catch (const std::exception& e) {  // of torch, for a device that is not there
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
  return PyLong_FromLongLong(st);
}

PyObject* py_kv_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  double eps;
  if (n != 10 || !tensors(a, 8) || !number(a[8], &eps) || !PyBool_Check(a[9])) return PyLong_FromLong(kNotHandled);
  return answer([&] {
    return kv_rope(tensor(a[0]), tensor(a[1]), tensor(a[2]), tensor(a[3]), tensor(a[4]), tensor(a[5]), tensor(a[6]),
                   tensor(a[7]), eps, a[9] == Py_True);
  });
}
PyObject* py_kv_copy(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 9 || !tensors(a, 8) || !PyBool_Check(a[8])) return PyLong_FromLong(kNotHandled);
  return answer([&] {
    return kv_copy(tensor(a[0]), tensor(a[1]), tensor(a[2]), tensor(a[3]), tensor(a[4]), tensor(a[5]), tensor(a[6]),
                   tensor(a[7]), a[8] == Py_True);
  });
}
PyObject* py_kv_attn(PyObject*, PyObject* const* a, Py_ssize_t n) {
  double scale;
  if (n != 12 || !tensors(a, 10) || (a[10] != Py_None && !THPVariable_CheckExact(a[10])) || !number(a[11], &scale))
    return PyLong_FromLong(kNotHandled);
  return answer([&] {
    return kv_attn(tensor(a[0]), tensor(a[1]), tensor(a[2]), tensor(a[3]), tensor(a[4]), tensor(a[5]), tensor(a[6]),
                   tensor(a[7]), tensor(a[8]), tensor(a[9]), a[10] == Py_None ? nullptr : &tensor(a[10]), scale);
  });
}
PyMethodDef kKvMethods[] = {
    {"kv_rope", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&py_kv_rope)), METH_FASTCALL,
     "checks + dsa_kv_rope_launch; status, or -1 when not handled"},
    {"kv_copy", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&py_kv_copy)), METH_FASTCALL,
     "checks + dsa_kv_write_launch / dsa_kv_read_launch; status, or -1 when not handled"},
    {"kv_attn", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&py_kv_attn)), METH_FASTCALL,
     "checks + dsa_kv_attn_launch; status, or -1 when not handled"},
    {nullptr, nullptr, 0, nullptr}};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "C++ launch path of the Python operators";
  m.def("task01", &task01, "checks + farq_launch; status, or -1 when not handled");
  m.def("task02", &task02, "checks + dsa_topk_launch; status, or -1 when not handled");
  // Only for the library that these structs were laid out for: without the entry
  // points every call takes the ctypes path, which refuses another version.
  if (dsa_kv_abi_version() == DSA_KV_ABI_VERSION) {
    m.attr("kv_abi_version") = DSA_KV_ABI_VERSION;
    if (PyModule_AddFunctions(m.ptr(), kKvMethods) != 0) throw py::error_already_set();
  }
}
