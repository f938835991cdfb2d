// The paged-cache operators' Python layer: checks of a call's tensors, its output and scratch, and the call of the C
// ABI.  A decode step makes these calls for every layer, and a call on short sequences is over on the GPU in 2 to 6 us:
// the same checks written in Python took 6.7 to 8 us of a call's 11 to 13.5 us on the host, here they take less than one.
// The C functions come as addresses from the loaded libfqkv_b200.so (bind), so there is one library per process.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <limits>
#include <stdexcept>
#include <string>
#include <utility>

#include "fqkv_b200.h"

namespace {

decltype(&fqkv_last_error) last_error;
decltype(&fqkv_decode_attn_paged) decode_attn_paged;
decltype(&fqkv_paged_workspace_bytes) paged_workspace_bytes;
decltype(&fqkv_rope_append_paged) rope_append_paged;
decltype(&fqkv_evict_paged) evict_paged;
decltype(&fqkv_evict_workspace_bytes) evict_workspace_bytes;

[[noreturn]] void fail(const char* key, const std::string& op, const std::string& what) {
  throw std::runtime_error(std::string(key) + ": " + op + ": " + what);
}
std::string dims(c10::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + ")";
}

// The tensors of one call, all on one GPU.
class Call {
 public:
  std::string op;
  int gpu = -1;

  explicit Call(PyObject* name) {
    const char* s = PyUnicode_AsUTF8(name);
    op = s ? s : "?";
    PyErr_Clear();
  }
  const at::Tensor& need(PyObject* o) {
    if (!THPVariable_Check(o)) fail("cuda", op, "all tensors must be CUDA tensors (there is no CPU path)");
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda()) fail("cuda", op, "all tensors must be CUDA tensors (there is no CPU path)");
    if (gpu < 0) gpu = t.get_device();
    else if (t.get_device() != gpu) fail("cuda", op, "all tensors must be on the same device");
    return t;
  }
  const at::Tensor* maybe(PyObject* o) { return o == Py_None ? nullptr : &need(o); }

  void index_vector(const char* name, const at::Tensor& t, int64_t n) const {
    if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != n || (n > 1 && t.stride(0) != 1))
      fail(name, op, std::string(name) + " must be a contiguous int32 tensor of " + std::to_string(n) + " (got " +
                         c10::toString(t.scalar_type()) + " " + dims(t.sizes()) + ")");
  }
  void slot_weights(const char* name, const at::Tensor& t, const fqkv_paged_kv_t& kv) const {
    const int64_t cap = kv.max_pages * kv.page_size;
    if (t.scalar_type() != at::kFloat || t.dim() != 3 || t.size(0) != kv.B || t.size(1) != kv.Hkv || t.size(2) != cap ||
        !t.is_contiguous())
      fail(name, op, std::string(name) + " must be a contiguous float32 [B, Hkv, max_pages * page_size] = (" +
                         std::to_string(kv.B) + ", " + std::to_string(kv.Hkv) + ", " + std::to_string(cap) + ") tensor (got " +
                         c10::toString(t.scalar_type()) + " " + dims(t.sizes()) + ")");
  }

  // The cache of a call (seq_lens: null where it is not used).
  fqkv_paged_kv_t cache(const at::Tensor& K, const at::Tensor& V, const at::Tensor* Ks, const at::Tensor* Vs,
                        const at::Tensor& table, const at::Tensor* lens) const {
    fqkv_paged_kv_t kv{};
    if (!Ks != !Vs) fail("fp16", op, "Ks and Vs go together");
    if (K.dim() != 4 || V.sizes() != K.sizes()) fail("shape", op, "K and V must both be [num_pages, Hkv, page_size, D]");
    const auto code = Ks ? at::kChar : at::kHalf;
    if (K.scalar_type() != code || V.scalar_type() != code)
      fail(Ks ? "int8" : "fp16", op, std::string("K and V must be ") + c10::toString(code) + " (got " +
                                         c10::toString(K.scalar_type()) + ", " + c10::toString(V.scalar_type()) + ")");
    kv.kv_format = Ks ? FQKV_KV_INT8 : FQKV_KV_F16;
    kv.num_pages = K.size(0);
    kv.Hkv = K.size(1);
    kv.page_size = K.size(2);
    kv.D = K.size(3);
    if (kv.D != 64 && kv.D != 128) fail("D", op, "head_dim must be 64 or 128 (got " + std::to_string(kv.D) + ")");
    if (K.stride(3) != 1 || V.stride(3) != 1) fail("stride", op, "K and V must be contiguous over D");
    for (int i = 0; i < 3; ++i) {
      kv.k_strides[i] = K.stride(i);
      kv.v_strides[i] = V.stride(i);
    }
    if (table.dim() != 2 || table.scalar_type() != at::kInt)
      fail("block_table", op, "block_table must be an int32 [B, max_pages] tensor");
    kv.B = table.size(0);
    kv.max_pages = table.size(1);
    if (table.stride(1) != 1 && kv.max_pages > 1) fail("block_table", op, "block_table must have contiguous rows");
    kv.block_table = static_cast<const int32_t*>(table.data_ptr());
    kv.table_stride = table.stride(0);
    if (lens) {
      index_vector("seq_lens", *lens, kv.B);
      kv.seq_lens = static_cast<const int32_t*>(lens->data_ptr());
    }
    kv.k = K.data_ptr();
    kv.v = V.data_ptr();
    if (Ks) {
      if (Ks->scalar_type() != at::kHalf || Vs->scalar_type() != at::kHalf) fail("fp16", op, "Ks and Vs must be fp16");
      if (Ks->sizes() != K.sizes().slice(0, 3) || Vs->sizes() != Ks->sizes())
        fail("shape", op, "Ks and Vs must be [num_pages, Hkv, page_size] = " + dims(K.sizes().slice(0, 3)));
      if (Ks->stride(2) != 1 || Vs->stride(2) != 1) fail("stride", op, "Ks and Vs must be contiguous over a page's tokens");
      kv.k_scales = Ks->data_ptr();
      kv.v_scales = Vs->data_ptr();
      for (int i = 0; i < 2; ++i) {
        kv.k_scale_strides[i] = Ks->stride(i);
        kv.v_scale_strides[i] = Vs->stride(i);
      }
    }
    return kv;
  }

  // The caller's workspace, or a new one of `bytes` (kept alive in `mine` until the launch is on the stream).
  std::pair<void*, size_t> scratch(const at::Tensor* given, size_t bytes, const at::Tensor& like, at::Tensor& mine) const {
    if (given) {
      if (!given->is_contiguous()) fail("workspace", op, "workspace must be a contiguous tensor on the inputs' device");
      return {given->data_ptr(), size_t(given->numel()) * given->element_size()};
    }
    if (!bytes) return {nullptr, 0};
    mine = at::empty({int64_t(bytes)}, like.options().dtype(at::kByte));
    return {mine.data_ptr(), bytes};
  }
  fqkv_stream_t stream() const {
    return reinterpret_cast<fqkv_stream_t>(c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(gpu)).stream());
  }
  void check(int rc) const {
    if (rc != FQKV_OK)
      throw std::runtime_error("launch: " + op + ": " + last_error() + " [fqkv status " + std::to_string(rc) + "]");
  }
};

// Other Python threads run while memory is sought and the launch is queued.
struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

void arguments(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) throw std::runtime_error("torch_binding: " + std::to_string(want) + " arguments needed");
}

// (op, q, K, V, Ks, Vs, block_table, seq_lens, out, workspace, weights) -> out
PyObject* decode(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 11);
  Call c(v[0]);
  const at::Tensor &q = c.need(v[1]), &K = c.need(v[2]), &V = c.need(v[3]);
  const at::Tensor *Ks = c.maybe(v[4]), *Vs = c.maybe(v[5]);
  const at::Tensor &table = c.need(v[6]), &lens = c.need(v[7]);
  const at::Tensor *given = c.maybe(v[8]), *weights = c.maybe(v[10]);
  if (v[9] != Py_None && !(THPVariable_Check(v[9]) && THPVariable_Unpack(v[9]).is_cuda()))
    fail("workspace", c.op, "workspace must be a contiguous tensor on the inputs' device");
  const at::Tensor* workspace = c.maybe(v[9]);
  const fqkv_paged_kv_t kv = c.cache(K, V, Ks, Vs, table, &lens);
  if (q.dim() != 3 || q.scalar_type() != at::kHalf || !q.is_contiguous())
    fail("fp16", c.op, "q must be a contiguous fp16 [B, Hq, D] tensor");
  if (q.size(0) != kv.B || q.size(2) != kv.D)
    fail("shape", c.op, "q has shape " + dims(q.sizes()) + ", expected (" + std::to_string(kv.B) + ", Hq, " +
                            std::to_string(kv.D) + ")");
  const int64_t Hq = q.size(1);
  float* w = nullptr;
  if (weights) {
    c.slot_weights("weights", *weights, kv);
    w = static_cast<float*>(weights->data_ptr());
  }
  if (given) {
    if (given->scalar_type() != at::kHalf && given->scalar_type() != at::kBFloat16)
      fail("dtype", c.op, std::string("out must be fp16 or bf16 (got ") + c10::toString(given->scalar_type()) + ")");
    if (!given->is_contiguous()) fail("contig", c.op, "out must be contiguous");
    if (given->sizes() != q.sizes())
      fail("shape", c.op, "out has shape " + dims(given->sizes()) + ", expected " + dims(q.sizes()));
  }
  at::Tensor out;
  {
    NoGil no_gil;
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(c.gpu));
    out = given ? *given : at::empty(q.sizes(), q.options());
    at::Tensor mine;
    const size_t need = workspace ? 0 : paged_workspace_bytes(kv.kv_format, kv.B, Hq, kv.Hkv, kv.D, kv.max_pages * kv.page_size,
                                                              w ? 1 : 0);
    const auto ws = c.scratch(workspace, need, q, mine);
    c.check(decode_attn_paged(&kv, out.scalar_type() == at::kBFloat16 ? 1 : 0, q.data_ptr(), out.data_ptr(), Hq, w, ws.first,
                              ws.second, c.stream()));
  }
  if (!given) return THPVariable_Wrap(std::move(out));
  Py_INCREF(v[8]);
  return v[8];
  END_HANDLE_TH_ERRORS
}

// (op, qkv, cos, sin, positions, slots, block_table, q_out, K, V, Ks, Vs, axes, seq_ids)
PyObject* append(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 14);
  Call c(v[0]);
  const at::Tensor &qkv = c.need(v[1]), &cos = c.need(v[2]), &sin = c.need(v[3]), &pos = c.need(v[4]), &slots = c.need(v[5]);
  const at::Tensor &table = c.need(v[6]), &q_out = c.need(v[7]), &K = c.need(v[8]), &V = c.need(v[9]);
  const at::Tensor *Ks = c.maybe(v[10]), *Vs = c.maybe(v[11]), *axes = c.maybe(v[12]), *ids = c.maybe(v[13]);
  const fqkv_paged_kv_t kv = c.cache(K, V, Ks, Vs, table, nullptr);
  const bool bf16 = qkv.scalar_type() == at::kBFloat16;
  if (!bf16 && qkv.scalar_type() != at::kHalf) fail("dtype", c.op, "qkv must be fp16 or bf16");
  if (q_out.dim() != 3 || q_out.scalar_type() != at::kHalf || !q_out.is_contiguous())
    fail("fp16", c.op, "q_out must be a contiguous fp16 [T, Hq, D] tensor");
  const int64_t T = q_out.size(0), Hq = q_out.size(1), width = (Hq + 2 * kv.Hkv) * kv.D;
  if (q_out.size(2) != kv.D || qkv.dim() != 2 || qkv.size(0) != T || qkv.size(1) < width || qkv.stride(1) != 1)
    fail("shape", c.op, "qkv must be [T, >= (Hq + 2 Hkv) D] with contiguous rows and q_out [T, Hq, " + std::to_string(kv.D) +
                            "] (got " + dims(qkv.sizes()) + ", " + dims(q_out.sizes()) + ")");
  if (cos.dim() != 2 || cos.size(1) != kv.D / 2 || sin.sizes() != cos.sizes() || cos.scalar_type() != at::kFloat ||
      sin.scalar_type() != at::kFloat || !cos.is_contiguous() || !sin.is_contiguous())
    fail("tables", c.op, "cos_table and sin_table must be contiguous float32 [rows, D/2 = " + std::to_string(kv.D / 2) + "]");
  c.index_vector("slots", slots, T);
  if (pos.scalar_type() != at::kInt || (pos.dim() != 1 && pos.dim() != 2) || pos.size(-1) != T || (T > 1 && pos.stride(-1) != 1))
    fail("positions", c.op, "positions must be int32 [T = " + std::to_string(T) + "] or [A, T] with contiguous rows");
  const int64_t A = pos.dim() == 2 ? pos.size(0) : 1;
  if (A > 1) {
    if (!axes) fail("axes", c.op, "several position axes need axes [D/2]");
    c.index_vector("axes", *axes, kv.D / 2);
  }
  if (ids) c.index_vector("seq_ids", *ids, T);
  const auto i32 = [](const at::Tensor* t) { return t ? static_cast<const int32_t*>(t->data_ptr()) : nullptr; };
  {
    NoGil no_gil;
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(c.gpu));
    c.check(rope_append_paged(&kv, bf16 ? 1 : 0, qkv.data_ptr(), T > 1 ? qkv.stride(0) : width,
                              static_cast<const float*>(cos.data_ptr()), static_cast<const float*>(sin.data_ptr()), cos.size(0),
                              i32(&pos), A > 1 ? pos.stride(0) : T, int32_t(std::min<int64_t>(A, 1 << 20)),
                              A > 1 ? i32(axes) : nullptr, i32(ids), i32(&slots), q_out.data_ptr(), T, Hq, c.stream()));
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// A Python integer; one that 64 bits cannot hold becomes the nearest.
int64_t integer(PyObject* o) {
  int over = 0;
  const long long x = PyLong_AsLongLongAndOverflow(o, &over);
  if (x == -1 && !over && PyErr_Occurred()) {
    PyErr_Clear();
    throw std::runtime_error("torch_binding: an integer is needed");
  }
  return over ? (over > 0 ? std::numeric_limits<int64_t>::max() : std::numeric_limits<int64_t>::min()) : x;
}

// (op, K, V, Ks, Vs, block_table, seq_lens, weights, budget, recent, weights_out, lens_out, workspace) -> lens_out
PyObject* evict(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 13);
  Call c(v[0]);
  const at::Tensor &K = c.need(v[1]), &V = c.need(v[2]);
  const at::Tensor *Ks = c.maybe(v[3]), *Vs = c.maybe(v[4]);
  const at::Tensor &table = c.need(v[5]), &lens = c.need(v[6]), &weights = c.need(v[7]);
  const int64_t budget = integer(v[8]), recent = integer(v[9]);
  const at::Tensor *w_out = c.maybe(v[10]), *given = c.maybe(v[11]), *workspace = c.maybe(v[12]);
  const fqkv_paged_kv_t kv = c.cache(K, V, Ks, Vs, table, &lens);
  c.slot_weights("weights", weights, kv);
  if (w_out) c.slot_weights("weights_out", *w_out, kv);
  if (given) c.index_vector("lens_out", *given, kv.B);
  at::Tensor out;
  {
    NoGil no_gil;
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(c.gpu));
    out = given ? *given : at::empty(lens.sizes(), lens.options());
    at::Tensor mine;
    const size_t need = workspace ? 0 : evict_workspace_bytes(kv.B, kv.Hkv, kv.max_pages * kv.page_size, budget);
    const auto ws = c.scratch(workspace, need, lens, mine);
    c.check(evict_paged(&kv, static_cast<const float*>(weights.data_ptr()),
                        static_cast<float*>(w_out ? w_out->data_ptr() : weights.data_ptr()),
                        static_cast<int32_t*>(out.data_ptr()), budget, recent, ws.first, ws.second, c.stream()));
  }
  if (!given) return THPVariable_Wrap(std::move(out));
  Py_INCREF(v[11]);
  return v[11];
  END_HANDLE_TH_ERRORS
}

// The C functions' addresses, in the order of the declarations above.
PyObject* bind(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 6);
  void* at[6];
  for (int i = 0; i < 6; ++i) {
    at[i] = PyLong_AsVoidPtr(v[i]);
    if (!at[i]) throw std::runtime_error("torch_binding: a function of libfqkv_b200.so is missing");
  }
  last_error = reinterpret_cast<decltype(last_error)>(at[0]);
  decode_attn_paged = reinterpret_cast<decltype(decode_attn_paged)>(at[1]);
  paged_workspace_bytes = reinterpret_cast<decltype(paged_workspace_bytes)>(at[2]);
  rope_append_paged = reinterpret_cast<decltype(rope_append_paged)>(at[3]);
  evict_paged = reinterpret_cast<decltype(evict_paged)>(at[4]);
  evict_workspace_bytes = reinterpret_cast<decltype(evict_workspace_bytes)>(at[5]);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(F)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<bind>("bind"), method<decode>("decode"), method<append>("append"), method<evict>("evict"),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_binding", "The paged-cache operators' Python layer.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__torch_binding() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_for_torch", BUILT_FOR_TORCH) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
