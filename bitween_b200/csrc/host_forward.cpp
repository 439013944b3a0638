// The host side of the calls that a decode step makes, each in one native call: checks, output allocation and the library's entry
// point on the current stream.  Such a step is launches of a few microseconds each.
//
// First QuantizedLinear's forward where no gradient is recorded: in Python the autograd function (7.5 us), the checks, torch.empty
// and the foreign call took 21 us a layer.
//
// forward(x, qweight, scale, zero_point, bias, bits, group_size[, dtype code]) returns the output (fp16, or bf16 where asked for), or None for every call that
// is not plain: the caller then goes through QuantizedLinearFunction, which converts, records, or raises.  Plain means
// exact torch tensors on the current CUDA device, contiguous and of their final types, no input that gradients are
// recorded for, no forward-mode tangent, and no tracing, dispatch or function mode and no function transform in force.
// The outcome depends on this call's arguments, torch's thread-local modes and the stream's scratch; nothing is kept.
#define PY_SSIZE_T_CLEAN
#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/cuda/EmptyTensor.h>
#include <Python.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <array>
#include <cstring>

#include "bitween_b200.h"

namespace {

// The tensor of a Python argument; null unless it is exactly a torch tensor (or parameter).
const at::Tensor *tensor_of(PyObject *o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

using QMatmul = int (*)(const void *, int, int64_t, int64_t, int64_t, const int32_t *, const void *, const void *, const void *,
                        void *, int, int, int, void *, size_t, void *);
QMatmul g_qmatmul = nullptr;      // of the library that the Python binding has loaded; set once, at import
PyObject *g_workspaces = nullptr; // the binding's dict (device index, stream handle) -> scratch tensor; kept by the binding too

// The stream's scratch, as the Python binding's current_workspace returns it; null inside a capture and before the
// binding has made one.  Called with the GIL held; the tensor stays in the dict, or is replaced by a larger one.
const at::Tensor *workspace_of(int device, cudaStream_t stream) {
    if (stream != nullptr && c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return nullptr;
    PyObject *key = Py_BuildValue("(iK)", device, (unsigned long long)reinterpret_cast<uintptr_t>(stream));
    if (!key) { PyErr_Clear(); return nullptr; }
    PyObject *t = PyDict_GetItemWithError(g_workspaces, key);       // borrowed
    Py_DECREF(key);
    if (!t) { PyErr_Clear(); return nullptr; }
    return tensor_of(t);
}

// A plain tensor: strided, on `device`, contiguous, without tangents or lazy views, and of no interest to autograd.
bool plain(const at::Tensor &t, const c10::Device &device, bool recording) {
    if (!t.defined() || t.layout() != c10::kStrided || !t.is_cuda() || t.device() != device || !t.is_contiguous()) return false;
    if (t.is_neg() || t._is_zerotensor() || t.key_set().has(c10::DispatchKey::Python)) return false;
    if (recording && t.requires_grad()) return false;
    return !t._fw_grad(/*level=*/0).defined();
}

bool modes_active() {
    return c10::impl::TorchDispatchModeTLS::any_modes_set() || at::impl::torch_function_mode_enabled() || torch::jit::tracer::isTracing() ||
           c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
}

PyObject *forward(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 7 && nargs != 8) {
        PyErr_SetString(PyExc_TypeError, "forward(x, qweight, scale, zero_point, bias, bits, group_size[, dtype code])");
        return nullptr;
    }
    const at::Tensor *x = tensor_of(args[0]), *q = tensor_of(args[1]), *s = tensor_of(args[2]), *z = tensor_of(args[3]), *b = nullptr;
    if (!x || !q || !s || !z || !g_qmatmul || !PyLong_CheckExact(args[5]) || !PyLong_CheckExact(args[6])) Py_RETURN_NONE;
    if (args[4] != Py_None && !(b = tensor_of(args[4]))) Py_RETURN_NONE;
    if (nargs == 8 && !PyLong_CheckExact(args[7])) Py_RETURN_NONE;
    const long bits = PyLong_AsLong(args[5]), group = PyLong_AsLong(args[6]), out_code = nargs == 8 ? PyLong_AsLong(args[7]) : BW_F16;
    if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    if (out_code != BW_F16 && out_code != BW_BF16) Py_RETURN_NONE;
    if ((bits != 2 && bits != 4 && bits != 8) || group < 1 || group > 1 << 30 || modes_active()) Py_RETURN_NONE;

    const c10::Device device = x->device();
    if (!device.is_cuda() || device.index() != c10::cuda::current_device()) Py_RETURN_NONE;
    const bool recording = c10::GradMode::is_enabled();
    if (!plain(*x, device, recording) || !plain(*q, device, recording) || !plain(*s, device, recording) || !plain(*z, device, recording) ||
        (b && !plain(*b, device, recording)))
        Py_RETURN_NONE;
    const auto xt = x->scalar_type();
    const int x_code = xt == at::kHalf ? BW_F16 : xt == at::kBFloat16 ? BW_BF16 : xt == at::kFloat ? BW_F32 : -1;
    if (x_code < 0 || q->scalar_type() != at::kInt || s->scalar_type() != at::kHalf || z->scalar_type() != at::kHalf) Py_RETURN_NONE;
    if (x->dim() < 1 || q->dim() != 2 || s->dim() != 2 || z->dim() != 2) Py_RETURN_NONE;
    const int64_t K = x->size(-1), N = q->size(0);
    if (K < 1 || N < 1 || x->numel() < 1 || q->size(1) * (32 / bits) != K || K % group) Py_RETURN_NONE;
    if (s->size(0) != N || s->size(1) != K / group || z->size(0) != N || z->size(1) != K / group) Py_RETURN_NONE;
    if (b && (b->scalar_type() != at::kHalf || b->numel() != N)) Py_RETURN_NONE;

    const int64_t M = x->numel() / K;
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    const at::Tensor *ws = workspace_of(device.index(), stream);
    // (9 to 32 tokens would run without scratch, on a slower kernel)
    if (M > 8 && M <= 32 && (!ws || ws->numel() < 64 * (K + 256))) Py_RETURN_NONE;
    const at::Tensor scratch = ws ? *ws : at::Tensor();              // (held: another thread may replace it in the dict)
    at::Tensor out;
    int rc;
    {
        pybind11::gil_scoped_release no_gil;
        c10::SmallVector<int64_t, 5> sizes(x->sizes().begin(), x->sizes().end());
        sizes.back() = N;
        out = at::empty(sizes, at::TensorOptions().dtype(out_code == BW_F16 ? at::kHalf : at::kBFloat16).device(device));
        rc = g_qmatmul(x->const_data_ptr(), x_code, M, N, K, static_cast<const int32_t *>(q->const_data_ptr()),
                       s->const_data_ptr(), z->const_data_ptr(), b ? b->const_data_ptr() : nullptr, out.mutable_data_ptr(), (int)out_code,
                       (int)bits, (int)group, scratch.defined() ? scratch.mutable_data_ptr() : nullptr,
                       scratch.defined() ? (size_t)scratch.numel() : 0, stream);
    }
    // (a kernel that needs more scratch, or an error: nothing has been launched, the Python path supplies it or raises)
    if (rc != BW_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// set_entry(address of bw_qmatmul, the binding's dict of workspaces)
PyObject *set_entry(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    if (nargs != 2 || !PyDict_CheckExact(args[1])) {
        PyErr_SetString(PyExc_TypeError, "set_entry(address, workspaces)");
        return nullptr;
    }
    void *p = PyLong_AsVoidPtr(args[0]);
    if (!p && PyErr_Occurred()) return nullptr;
    Py_INCREF(args[1]);
    Py_XSETREF(g_workspaces, args[1]);
    g_qmatmul = reinterpret_cast<QMatmul>(p);
    Py_RETURN_NONE;
}

// ---- the quantised key-value cache, rotary positions, the adapters, log probabilities --------------------------------
// None, again, for every call that is not plain (the Python path converts, copies or raises).  Scratch comes from the caching allocator, so
// that calls of other streams, threads and graphs have their own.

using KvAppend = decltype(&bw_kv_append);
using KvRead = decltype(&bw_kv_read);
using KvAttend = decltype(&bw_kv_attend);
using KvAttendBytes = decltype(&bw_kv_attend_workspace_bytes);
using AdapterBytes = decltype(&bw_adapter_hidden_bytes);
using AdapterForward = decltype(&bw_adapter_forward);
using AdapterBackward = decltype(&bw_adapter_backward);
struct Operators {                        // in the order of set_operators
    KvAppend kv_append;
    KvRead kv_read;
    KvAttend kv_attend;
    KvAttendBytes kv_attend_bytes;
    AdapterBytes adapter_bytes;
    AdapterForward adapter_forward;
    AdapterBackward adapter_backward;
    decltype(&bw_kv_attend_window) kv_attend_window;
    decltype(&bw_kv_attend_window_workspace_bytes) kv_attend_window_bytes;
    decltype(&bw_rotate) rotate;
    decltype(&bw_kv_append_rotated) kv_append_rotated;
    decltype(&bw_token_log_probs) token_log_probs;
    decltype(&bw_token_log_probs_grad) token_log_probs_grad;
} g_ops = {};
constexpr int OPERATORS = sizeof(Operators) / sizeof(void *);

int float_code(at::ScalarType t) { return t == at::kHalf ? BW_F16 : t == at::kBFloat16 ? BW_BF16 : t == at::kFloat ? BW_F32 : -1; }

// Like plain(), of any strides, and recorded gradients or not.
bool usable(const at::Tensor *t, const c10::Device &device) {
    return t && t->defined() && t->layout() == c10::kStrided && t->is_cuda() && t->device() == device && !t->is_neg() && !t->_is_zerotensor() &&
           !t->key_set().has(c10::DispatchKey::Python) && !t->_fw_grad(/*level=*/0).defined();
}
bool dense(const at::Tensor *t, const c10::Device &device) { return usable(t, device) && t->is_contiguous(); }
bool on_16_bytes(const at::Tensor &t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0; }
// at::empty without the dispatcher (half a microsecond less): no mode or transform is in force here.
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const c10::Device &device) {
    return at::Tensor(at::detail::empty_cuda(sizes, type, device, std::nullopt));
}
at::Tensor bytes_of(size_t n, const c10::Device &device) { return n ? fresh({(int64_t)n}, at::kByte, device) : at::Tensor(); }

// The cache's tensors, arguments 0 to 3 of each of its calls (k_codes, v_codes, params, bits), on the current device.
struct Cache {
    const at::Tensor *k = nullptr, *v = nullptr, *params = nullptr;
    int bits = 0, heads = 0, page_size = 0, dim = 0;
    int64_t pages = 0;
    c10::Device device = c10::Device(c10::kCPU);
    bool of(PyObject *const *args) {
        k = tensor_of(args[0]);
        v = tensor_of(args[1]);
        params = tensor_of(args[2]);
        if (!k || !v || !params || !PyLong_CheckExact(args[3]) || modes_active()) return false;
        const long b = PyLong_AsLong(args[3]);
        if (b != 2 && b != 4 && b != 8) {
            PyErr_Clear();
            return false;
        }
        bits = (int)b;
        device = k->device();
        if (!device.is_cuda() || device.index() != c10::cuda::current_device() || !dense(k, device) || !dense(v, device) || !dense(params, device)) return false;
        if (k->scalar_type() != at::kInt || v->scalar_type() != at::kInt || params->scalar_type() != at::kHalf) return false;
        if (k->dim() != 4 || v->sizes() != k->sizes() || params->dim() != 4 || params->size(3) != 4) return false;
        for (int i = 0; i < 3; ++i)
            if (params->size(i) != k->size(i) || k->size(i) > INT32_MAX) return false;
        pages = k->size(0);
        heads = (int)k->size(1);
        page_size = (int)k->size(2);
        if (k->size(3) > 64) return false;
        dim = (int)k->size(3) * (32 / bits);
        return true;
    }
    int32_t *k_codes() const { return static_cast<int32_t *>(k->mutable_data_ptr()); }
    int32_t *v_codes() const { return static_cast<int32_t *>(v->mutable_data_ptr()); }
};
bool slots_ok(const at::Tensor *slots, const Cache &c) { return dense(slots, c.device) && slots->scalar_type() == at::kLong && slots->dim() == 1; }

// kv_append(k_codes, v_codes, params, bits, k, v, slots): True
PyObject *kv_append(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    Cache c;
    if (nargs != 7 || !g_ops.kv_append || !c.of(args)) Py_RETURN_NONE;
    const at::Tensor *k = tensor_of(args[4]), *v = tensor_of(args[5]), *slots = tensor_of(args[6]);
    if (!usable(k, c.device) || !usable(v, c.device) || !slots_ok(slots, c)) Py_RETURN_NONE;
    const int code = float_code(k->scalar_type());
    if (code < 0 || v->scalar_type() != k->scalar_type() || k->dim() != 3 || v->sizes() != k->sizes()) Py_RETURN_NONE;
    if (k->size(0) != slots->size(0) || k->size(1) != c.heads || k->size(2) != c.dim || k->stride(2) != 1 || v->stride(2) != 1) Py_RETURN_NONE;
    int rc;
    {
        pybind11::gil_scoped_release no_gil;
        rc = g_ops.kv_append(k->const_data_ptr(), v->const_data_ptr(), code, k->size(0), k->stride(0), k->stride(1), v->stride(0), v->stride(1),
                             static_cast<const int64_t *>(slots->const_data_ptr()), c.heads, c.dim, c.bits, c.pages, c.page_size, c.k_codes(), c.v_codes(),
                             c.params->mutable_data_ptr(), c10::cuda::getCurrentCUDAStream(c.device.index()).stream());
    }
    if (rc != BW_OK) Py_RETURN_NONE;
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// kv_read(k_codes, v_codes, params, bits, slots, dtype code): (k, v)
PyObject *kv_read(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    Cache c;
    if (nargs != 6 || !g_ops.kv_read || !c.of(args)) Py_RETURN_NONE;
    const at::Tensor *slots = tensor_of(args[4]);
    const long code = PyLong_CheckExact(args[5]) ? PyLong_AsLong(args[5]) : -1;
    if (!slots_ok(slots, c) || code < BW_F32 || code > BW_BF16) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    at::Tensor k, v;
    int rc;
    {
        pybind11::gil_scoped_release no_gil;
        const at::ScalarType type = code == BW_F32 ? at::kFloat : code == BW_F16 ? at::kHalf : at::kBFloat16;
        k = fresh({slots->size(0), c.heads, c.dim}, type, c.device);
        v = fresh({slots->size(0), c.heads, c.dim}, type, c.device);
        rc = g_ops.kv_read(c.k_codes(), c.v_codes(), c.params->const_data_ptr(), c.heads, c.dim, c.bits, c.pages, c.page_size,
                           static_cast<const int64_t *>(slots->const_data_ptr()), slots->size(0), k.mutable_data_ptr(), v.mutable_data_ptr(), (int)code,
                           c10::cuda::getCurrentCUDAStream(c.device.index()).stream());
    }
    if (rc != BW_OK) Py_RETURN_NONE;
    PyObject *pk = THPVariable_Wrap(std::move(k)), *pv = THPVariable_Wrap(std::move(v));
    return Py_BuildValue("(NN)", pk, pv);
    END_HANDLE_TH_ERRORS
}

// kv_attend(k_codes, v_codes, params, bits, q, page_table, lengths, softmax_scale[, window, sinks]): the attended values
PyObject *kv_attend(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    Cache c;
    if ((nargs != 8 && nargs != 10) || !g_ops.kv_attend || !PyFloat_CheckExact(args[7]) || !c.of(args)) Py_RETURN_NONE;
    int64_t window = -1, sinks = 0;
    if (nargs == 10) {
        if (!PyLong_CheckExact(args[8]) || !PyLong_CheckExact(args[9])) Py_RETURN_NONE;
        window = PyLong_AsLongLong(args[8]);
        sinks = PyLong_AsLongLong(args[9]);
        if (window < 0 || sinks < 0) {
            PyErr_Clear();
            Py_RETURN_NONE;
        }
    }
    const at::Tensor *q = tensor_of(args[4]), *table = tensor_of(args[5]), *lengths = tensor_of(args[6]);
    if (!usable(q, c.device) || !usable(table, c.device) || !dense(lengths, c.device) || (c10::GradMode::is_enabled() && q->requires_grad())) Py_RETURN_NONE;
    const int code = float_code(q->scalar_type());
    if ((code != BW_F16 && code != BW_BF16) || table->scalar_type() != at::kInt || lengths->scalar_type() != at::kInt) Py_RETURN_NONE;
    if (q->dim() != 3 || q->size(2) != c.dim || q->stride(2) != 1 || q->size(1) < 1 || c.heads < 1 || q->size(1) % c.heads || q->size(1) > INT32_MAX) Py_RETURN_NONE;
    const int64_t batch = q->size(0);
    if (table->dim() != 2 || table->size(0) != batch || table->stride(1) != 1 || lengths->dim() != 1 || lengths->size(0) != batch) Py_RETURN_NONE;
    const float scale = (float)PyFloat_AS_DOUBLE(args[7]);
    at::Tensor out;
    int rc;
    {
        pybind11::gil_scoped_release no_gil;
        const int heads = (int)q->size(1);
        out = fresh({batch, heads, c.dim}, q->scalar_type(), c.device);
        const at::Tensor ws = bytes_of(window < 0 ? g_ops.kv_attend_bytes(batch, heads, c.heads, c.dim, c.page_size, table->size(1))
                                                  : g_ops.kv_attend_window_bytes(batch, heads, c.heads, c.dim, c.page_size, table->size(1), window, sinks), c.device);
        void *scratch = ws.defined() ? ws.mutable_data_ptr() : nullptr;
        const size_t bytes = ws.defined() ? (size_t)ws.numel() : 0;
        const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(c.device.index()).stream();
        const int32_t *pages = static_cast<const int32_t *>(table->const_data_ptr()), *n = static_cast<const int32_t *>(lengths->const_data_ptr());
        if (window < 0)
            rc = g_ops.kv_attend(q->const_data_ptr(), code, batch, heads, q->stride(0), q->stride(1), c.k_codes(), c.v_codes(), c.params->const_data_ptr(), c.bits,
                                 c.pages, c.page_size, c.heads, c.dim, pages, table->stride(0), table->size(1), n, scale, out.mutable_data_ptr(), scratch, bytes, stream);
        else
            rc = g_ops.kv_attend_window(q->const_data_ptr(), code, batch, heads, q->stride(0), q->stride(1), c.k_codes(), c.v_codes(), c.params->const_data_ptr(), c.bits,
                                        c.pages, c.page_size, c.heads, c.dim, pages, table->stride(0), table->size(1), n, window, sinks, scale, out.mutable_data_ptr(),
                                        scratch, bytes, stream);
    }
    if (rc != BW_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// The engine hands each gradient to the stream on which its consumer was recorded.  The default stream cannot take one from a capture, and torch
// does not survive the attempt.
void check_capture(torch::autograd::Node &node, const char *name) {
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
    for (uint32_t i = 0; i < node.num_outputs(); ++i) {
        if (!node.task_should_compute_output(i)) continue;
        const auto stream = node.next_edge(i).function->stream();
        TORCH_CHECK(!stream || c10::cuda::CUDAStream(*stream) != c10::cuda::getDefaultCUDAStream(stream->device_index()), name,
                    ": this backward pass cannot be captured while a graph of the same tensors, recorded on the default stream, is alive; free it, or "
                    "record it on another stream");
    }
}
// Gradients as once_differentiable has them: an error for whoever differentiates these.
void once_only(torch::autograd::variable_list &result) {
    for (auto &t : result)
        if (t.defined()) t = (*std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that was marked with @once_differentiable", 1))(
                             {t.detach().requires_grad_()})[0];
}
// A saved tensor.  Hooks may have made another one of it in the meantime (moved, packed).
at::Tensor saved(const torch::autograd::SavedVariable &v, const char *name, const c10::Device &device, at::IntArrayRef sizes, at::ScalarType type) {
    at::Tensor t = v.unpack();
    TORCH_CHECK(t.defined() && t.layout() == c10::kStrided && t.device() == device && t.scalar_type() == type && t.sizes() == sizes, name,
                ": a tensor saved for the backward pass has come back from its hooks in another shape, type or place");
    return t.resolve_neg();
}

// One call of bw_adapter_forward; `hidden` is what the backward pass needs again.  x [..., K] and the rest are checked.
int adapter_call(const at::Tensor &x, const at::Tensor &down, const at::Tensor &up, const at::Tensor &index, const at::Tensor &scaling, const at::Tensor &base,
                 at::Tensor &out, at::Tensor &hidden) {
    const int64_t K = down.size(2), N = up.size(2), M = x.numel() / K;
    const c10::Device device = x.device();
    if (!out.defined()) {
        c10::SmallVector<int64_t, 5> sizes(x.sizes().begin(), x.sizes().end());
        sizes.back() = N;
        out = fresh(sizes, x.scalar_type(), device);
    }
    hidden = bytes_of(g_ops.adapter_bytes(M, (int)down.size(1)), device);
    return g_ops.adapter_forward(x.const_data_ptr(), float_code(x.scalar_type()), M, N, K, down.const_data_ptr(), up.const_data_ptr(), (int)down.size(0),
                                 (int)down.size(1), static_cast<const int32_t *>(index.const_data_ptr()),
                                 scaling.defined() ? static_cast<const float *>(scaling.const_data_ptr()) : nullptr,
                                 base.defined() ? base.const_data_ptr() : nullptr, out.mutable_data_ptr(), hidden.mutable_data_ptr(), (size_t)hidden.numel(),
                                 c10::cuda::getCurrentCUDAStream(device.index()).stream());
}

// AdapterFunction of the Python package (adapters.py) as a node of the graph, with the same gradients and the same error where they are differentiated
// again.  Edges: x, down, up, base.
struct AdapterNode : torch::autograd::Node {
    torch::autograd::SavedVariable x, down, up, index, scaling, hidden;
    c10::SmallVector<int64_t, 5> x_sizes, index_sizes;
    bool scaled = false, kept = false;        // there are scaling, hidden
    int64_t adapters = 0, rank = 0, K = 0, N = 0, M = 0;
    at::ScalarType type = at::kHalf;
    c10::Device device = c10::Device(c10::kCPU);

    // A saved tensor, as the kernels take it.
    at::Tensor back(const torch::autograd::SavedVariable &v, at::IntArrayRef sizes, at::ScalarType as) const {
        const at::Tensor t = saved(v, "adapter_matmul", device, sizes, as).contiguous();
        return on_16_bytes(t) ? t : t.clone();
    }

    std::string name() const override { return "AdapterNode"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        for (auto *v : {&x, &down, &up, &index, &scaling, &hidden}) v->reset_data();
    }
    torch::autograd::variable_list apply(torch::autograd::variable_list &&grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        torch::autograd::variable_list result(4);
        const at::Tensor g = grads[0];
        if (!g.defined()) return result;
        check_capture(*this, "adapter_matmul");
        const bool again = c10::GradMode::is_enabled();
        if (task_should_compute_output(0) || task_should_compute_output(1) || task_should_compute_output(2)) {
            at::AutoGradMode off(false);
            const at::Tensor xt = back(x, x_sizes, type), dt = back(down, {adapters, rank, K}, type), ut = back(up, {adapters, rank, N}, type), it = back(index, index_sizes, at::kInt),
                             st = scaled ? back(scaling, {adapters}, at::kFloat) : at::Tensor(), ht = kept ? back(hidden, {(int64_t)g_ops.adapter_bytes(M, (int)rank)}, at::kByte) : at::Tensor();
            at::Tensor dense = g.contiguous();
            if (!on_16_bytes(dense)) dense = dense.clone();
            const at::Tensor *like[3] = {&xt, &dt, &ut};
            for (int i = 0; i < 3; ++i)
                if (task_should_compute_output(i)) result[i] = fresh(like[i]->sizes(), like[i]->scalar_type(), like[i]->device());
            const at::Tensor ws = bytes_of(g_ops.adapter_bytes(M, (int)dt.size(1)), xt.device());
            const auto into = [&](int i) { return result[i].defined() ? result[i].mutable_data_ptr() : nullptr; };
            const int rc = g_ops.adapter_backward(dense.const_data_ptr(), float_code(xt.scalar_type()), xt.const_data_ptr(), M, N, K, dt.const_data_ptr(),
                                                  ut.const_data_ptr(), (int)dt.size(0), (int)dt.size(1), static_cast<const int32_t *>(it.const_data_ptr()),
                                                  st.defined() ? static_cast<const float *>(st.const_data_ptr()) : nullptr,
                                                  ht.defined() ? ht.const_data_ptr() : nullptr, ht.defined() ? (size_t)ht.numel() : 0, into(0), into(1), into(2),
                                                  ws.mutable_data_ptr(), (size_t)ws.numel(), c10::cuda::getCurrentCUDAStream(xt.device().index()).stream());
            TORCH_CHECK(rc == BW_OK, "libbitween_b200: bw_adapter_backward returned status ", rc);
        }
        if (again) once_only(result);
        if (task_should_compute_output(3)) result[3] = g;
        return result;
    }
};

// The recorded call: null where it cannot be made (nothing has been launched then).
at::Tensor adapter_recorded(const at::Tensor &x, const at::Tensor &down, const at::Tensor &up, const at::Tensor &index, const at::Tensor &scaling, const at::Tensor &base) {
    at::Tensor out, hidden;
    if (adapter_call(x, down, up, index, scaling, base, out, hidden) != BW_OK) return at::Tensor();
    const std::shared_ptr<AdapterNode> node(new AdapterNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, down, up, base));
    node->x_sizes.assign(x.sizes().begin(), x.sizes().end());
    node->index_sizes.assign(index.sizes().begin(), index.sizes().end());
    node->scaled = scaling.defined();
    node->kept = up.requires_grad();
    node->adapters = down.size(0);
    node->rank = down.size(1);
    node->K = down.size(2);
    node->N = up.size(2);
    node->M = x.numel() / node->K;
    node->type = x.scalar_type();
    node->device = x.device();
    node->x = torch::autograd::SavedVariable(x, false);
    node->down = torch::autograd::SavedVariable(down, false);
    node->up = torch::autograd::SavedVariable(up, false);
    node->index = torch::autograd::SavedVariable(index, false);
    node->scaling = torch::autograd::SavedVariable(scaling, false);
    node->hidden = torch::autograd::SavedVariable(node->kept ? hidden : at::Tensor(), false);
    torch::autograd::set_history(out, node);
    return out;
}

// adapter_matmul(x, down, up, index, scaling, base, out): the result (`out` only where no gradient is recorded)
PyObject *adapter_matmul(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 7 || !g_ops.adapter_forward || modes_active()) Py_RETURN_NONE;
    const at::Tensor *t[7] = {};
    for (int i = 0; i < 7; ++i) {
        if (i >= 4 && args[i] == Py_None) continue;
        if (!(t[i] = tensor_of(args[i]))) Py_RETURN_NONE;
    }
    const at::Tensor *x = t[0], *down = t[1], *up = t[2], *index = t[3], *scaling = t[4], *base = t[5], *given = t[6];
    const c10::Device device = x->device();
    if (!device.is_cuda() || device.index() != c10::cuda::current_device()) Py_RETURN_NONE;
    for (int i = 0; i < 7; ++i)
        if (t[i] && (!dense(t[i], device) || !(i == 3 || i == 4 || (on_16_bytes(*t[i]) && t[i]->scalar_type() == x->scalar_type())))) Py_RETURN_NONE;
    const int code = float_code(x->scalar_type());
    if ((code != BW_F16 && code != BW_BF16) || index->scalar_type() != at::kInt) Py_RETURN_NONE;
    if (x->dim() < 1 || down->dim() != 3 || up->dim() != 3 || down->size(0) != up->size(0) || down->size(1) != up->size(1)) Py_RETURN_NONE;
    const int64_t K = down->size(2), N = up->size(2);
    if (down->size(0) < 1 || down->size(0) > INT32_MAX || down->size(1) < 1 || down->size(1) > 256 || K < 1 || N < 1 || x->size(-1) != K || x->numel() < 1) Py_RETURN_NONE;
    const at::IntArrayRef lead = x->sizes().slice(0, x->dim() - 1);
    if (index->numel() != x->numel() / K || (index->dim() != 1 && index->sizes() != lead)) Py_RETURN_NONE;
    if (scaling && (scaling->scalar_type() != at::kFloat || scaling->dim() != 1 || scaling->size(0) != down->size(0) || scaling->requires_grad())) Py_RETURN_NONE;
    for (const at::Tensor *y : {base, given})
        if (y && (y->dim() != x->dim() || y->sizes().slice(0, x->dim() - 1) != lead || y->size(-1) != N)) Py_RETURN_NONE;
    const bool recording = c10::GradMode::is_enabled() && (x->requires_grad() || down->requires_grad() || up->requires_grad() || (base && base->requires_grad()));
    const at::Tensor none;
    at::Tensor out;
    if (recording) {
        if (given) Py_RETURN_NONE;
        {
            pybind11::gil_scoped_release no_gil;
            out = adapter_recorded(*x, *down, *up, *index, scaling ? *scaling : none, base ? *base : none);
        }
        if (!out.defined()) Py_RETURN_NONE;
    } else {
        if (given) {
            const uintptr_t o = reinterpret_cast<uintptr_t>(given->const_data_ptr());
            for (int i = 0; i < 6; ++i) {                            // (by position: one tensor may be several arguments, and only as base may it be written over)
                const uintptr_t a = t[i] ? reinterpret_cast<uintptr_t>(t[i]->const_data_ptr()) : 0;
                if (t[i] && a < o + given->nbytes() && o < a + t[i]->nbytes() && !(i == 5 && a == o)) Py_RETURN_NONE;
            }
            if (given->requires_grad()) Py_RETURN_NONE;
            out = *given;
        }
        int rc;
        {
            pybind11::gil_scoped_release no_gil;
            at::Tensor hidden;
            rc = adapter_call(*x, *down, *up, *index, scaling ? *scaling : none, base ? *base : none, out, hidden);
        }
        if (rc != BW_OK) Py_RETURN_NONE;
        if (given && !given->is_inference()) given->unsafeGetTensorImpl()->bump_version();      // (written in place, as autograd has to know)
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// ---- rotary positions ----
// Tensors [..., heads, dim] as rows: whether the leading dimensions are one with a stride.
struct HeadRows {
    int64_t tokens = 1, stride = 0;
    bool of(const at::Tensor &x) {
        const int64_t n = x.dim();
        if (n < 2 || x.stride(n - 1) != 1 || x.numel() < 1 || x.size(n - 2) > INT32_MAX || x.size(n - 1) > INT32_MAX) return false;
        for (int64_t i = n - 3; i >= 0; --i) {
            if (x.size(i) == 1) continue;
            if (tokens == 1) stride = x.stride(i);
            else if (x.stride(i) != tokens * stride) return false;
            tokens *= x.size(i);
        }
        return true;
    }
};
// The table and what belongs to it: (table, (rotary_dim, interleaved, number of axes, axes of the pairs as bytes, max_positions)).
struct RotaryCall {
    const at::Tensor *table = nullptr;
    bw_rotary r = {};
    std::array<uint8_t, 128> axes = {};
    bool of(PyObject *t, PyObject *meta, const c10::Device &device) {
        table = tensor_of(t);
        if (!PyTuple_CheckExact(meta) || PyTuple_GET_SIZE(meta) != 5 || !dense(table, device) || table->scalar_type() != at::kFloat || !on_16_bytes(*table)) return false;
        r.rotary_dim = (int)PyLong_AsLong(PyTuple_GET_ITEM(meta, 0));
        r.interleaved = (int)PyLong_AsLong(PyTuple_GET_ITEM(meta, 1));
        r.num_axes = (int)PyLong_AsLong(PyTuple_GET_ITEM(meta, 2));
        r.max_positions = PyLong_AsLongLong(PyTuple_GET_ITEM(meta, 4));
        char *bytes = nullptr;
        Py_ssize_t n = 0;
        if (PyErr_Occurred() || PyBytes_AsStringAndSize(PyTuple_GET_ITEM(meta, 3), &bytes, &n) != 0) {
            PyErr_Clear();
            return false;
        }
        if (r.rotary_dim < 2 || n != r.rotary_dim / 2 || n > 128) return false;
        if (table->dim() != 3 || table->size(0) != r.max_positions || table->size(1) != n || table->size(2) != 2) return false;
        std::memcpy(axes.data(), bytes, (size_t)n);
        r.table = static_cast<const float *>(table->const_data_ptr());
        return true;
    }
    // Positions of the leading shape, or of each axis.
    bool at(const at::Tensor *positions, at::IntArrayRef lead, int64_t tokens, const c10::Device &device) {
        if (!dense(positions, device) || positions->scalar_type() != at::kLong) return false;
        const at::IntArrayRef sizes = positions->sizes();
        if (sizes == lead) r.axis_stride = 0;
        else if (sizes.size() == lead.size() + 1 && sizes[0] == r.num_axes && sizes.slice(1) == lead) r.axis_stride = tokens;
        else return false;
        r.positions = static_cast<const int64_t *>(positions->const_data_ptr());
        return true;
    }
};

// Rows of one or two tensors turned, or turned back, into new tensors; BW_OK or nothing has been launched.
int rotate_call(bw_rotary r, const uint8_t *axes, bool inverse, const at::Tensor *const *x, at::Tensor *out) {
    r.axes = axes;
    const void *from[2] = {};
    void *to[2] = {};
    int heads[2] = {};
    int64_t strides[4] = {}, tokens = 0, dim = 0;
    int n = 0;
    for (int i = 0; i < 2; ++i) {
        if (!x[i]) continue;
        HeadRows rows;
        if (!rows.of(*x[i])) return BW_ERR_UNSUPPORTED;
        out[i] = fresh(x[i]->sizes(), x[i]->scalar_type(), x[i]->device());
        from[n] = x[i]->const_data_ptr();
        to[n] = out[i].mutable_data_ptr();
        heads[n] = (int)x[i]->size(-2);
        strides[2 * n] = rows.stride;
        strides[2 * n + 1] = x[i]->stride(-2);
        tokens = rows.tokens;
        dim = x[i]->size(-1);
        ++n;
    }
    const at::Tensor &any = x[0] ? *x[0] : *x[1];
    return g_ops.rotate(&r, tokens, (int)dim, float_code(any.scalar_type()), inverse, from[0], heads[0], strides[0], strides[1], to[0], from[1], heads[1], strides[2], strides[3],
                        to[1], c10::cuda::getCurrentCUDAStream(any.device().index()).stream());
}

// RotateFunction of the Python package (rotary.py) as a node of the graph.  Edges, and inputs, are the tensors that were rotated.
struct RotateNode : torch::autograd::Node {
    torch::autograd::SavedVariable table, positions;
    c10::SmallVector<int64_t, 5> table_sizes, position_sizes;
    bw_rotary r = {};
    std::array<uint8_t, 128> axes = {};
    c10::Device device = c10::Device(c10::kCPU);

    std::string name() const override { return "RotateNode"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        table.reset_data();
        positions.reset_data();
    }
    torch::autograd::variable_list apply(torch::autograd::variable_list &&grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        torch::autograd::variable_list result(num_outputs());
        at::Tensor held[2], out[2];
        const at::Tensor *x[2] = {};
        for (uint32_t i = 0; i < num_outputs() && i < 2; ++i) {
            if (!grads[i].defined() || !task_should_compute_output(i)) continue;
            held[i] = grads[i].resolve_neg();
            HeadRows rows;
            if (!rows.of(held[i])) held[i] = held[i].contiguous();
            x[i] = &held[i];
        }
        if (!x[0] && !x[1]) return result;
        check_capture(*this, "rotate");
        const bool again = c10::GradMode::is_enabled();
        {
            at::AutoGradMode off(false);
            const at::Tensor t = saved(table, "rotate", device, table_sizes, at::kFloat).contiguous(), p = saved(positions, "rotate", device, position_sizes, at::kLong).contiguous();
            TORCH_CHECK(on_16_bytes(t), "rotate: the table has come back from its hooks off a 16-byte boundary");
            bw_rotary call = r;
            call.table = static_cast<const float *>(t.const_data_ptr());
            call.positions = static_cast<const int64_t *>(p.const_data_ptr());
            const int rc = rotate_call(call, axes.data(), true, x, out);
            TORCH_CHECK(rc == BW_OK, "libbitween_b200: bw_rotate returned status ", rc);
        }
        for (uint32_t i = 0; i < num_outputs() && i < 2; ++i) result[i] = out[i];
        if (again) once_only(result);
        return result;
    }
};

// rotate(table, what belongs to it, positions, x[, y]): the rotated tensor, or both
PyObject *rotate(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if ((nargs != 4 && nargs != 5) || !g_ops.rotate || modes_active()) Py_RETURN_NONE;
    const at::Tensor *positions = tensor_of(args[2]), *x[2] = {tensor_of(args[3]), nargs == 5 ? tensor_of(args[4]) : nullptr};
    if (!x[0] || (nargs == 5 && !x[1])) Py_RETURN_NONE;
    const c10::Device device = x[0]->device();
    if (!device.is_cuda() || device.index() != c10::cuda::current_device()) Py_RETURN_NONE;
    RotaryCall c;
    const int n = nargs == 5 ? 2 : 1;
    bool recording = false;
    for (int i = 0; i < n; ++i) {
        HeadRows rows;
        if (!usable(x[i], device) || float_code(x[i]->scalar_type()) < 0 || x[i]->scalar_type() != x[0]->scalar_type() || !rows.of(*x[i])) Py_RETURN_NONE;
        if (x[i]->dim() != x[0]->dim() || x[i]->size(-1) != x[0]->size(-1) || x[i]->sizes().slice(0, x[i]->dim() - 2) != x[0]->sizes().slice(0, x[0]->dim() - 2)) Py_RETURN_NONE;
        recording = recording || (c10::GradMode::is_enabled() && x[i]->requires_grad());
        if (i == 0 && (!c.of(args[0], args[1], device) || !c.at(positions, x[0]->sizes().slice(0, x[0]->dim() - 2), rows.tokens, device))) Py_RETURN_NONE;
    }
    if (x[0]->size(-1) < c.r.rotary_dim) Py_RETURN_NONE;
    at::Tensor out[2];
    int rc;
    {
        pybind11::gil_scoped_release no_gil;
        rc = rotate_call(c.r, c.axes.data(), false, x, out);
        if (rc == BW_OK && recording) {
            const std::shared_ptr<RotateNode> node(new RotateNode(), torch::autograd::deleteNode);
            node->set_next_edges(n == 2 ? torch::autograd::collect_next_edges(*x[0], *x[1]) : torch::autograd::collect_next_edges(*x[0]));
            node->table_sizes.assign(c.table->sizes().begin(), c.table->sizes().end());
            node->position_sizes.assign(positions->sizes().begin(), positions->sizes().end());
            node->r = c.r;
            node->axes = c.axes;
            node->device = device;
            node->table = torch::autograd::SavedVariable(*c.table, false);
            node->positions = torch::autograd::SavedVariable(*positions, false);
            for (int i = 0; i < n; ++i) torch::autograd::set_history(out[i], node);
        }
    }
    if (rc != BW_OK) Py_RETURN_NONE;
    if (n == 1) return THPVariable_Wrap(std::move(out[0]));
    PyObject *first = THPVariable_Wrap(std::move(out[0])), *second = THPVariable_Wrap(std::move(out[1]));
    return Py_BuildValue("(NN)", first, second);
    END_HANDLE_TH_ERRORS
}

// kv_append_rotated(k_codes, v_codes, params, bits, q or None, k, v, slots, table, what belongs to it, positions): the rotated queries, or True
PyObject *kv_append_rotated(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    Cache c;
    if (nargs != 11 || !g_ops.kv_append_rotated || !c.of(args)) Py_RETURN_NONE;
    const bool queries = args[4] != Py_None;
    const at::Tensor *q = queries ? tensor_of(args[4]) : nullptr, *k = tensor_of(args[5]), *v = tensor_of(args[6]), *slots = tensor_of(args[7]), *positions = tensor_of(args[10]);
    if (!usable(k, c.device) || !usable(v, c.device) || !slots_ok(slots, c) || (queries && !usable(q, c.device))) Py_RETURN_NONE;
    const int code = float_code(k->scalar_type());
    if (code < 0 || v->scalar_type() != k->scalar_type() || k->dim() != 3 || v->sizes() != k->sizes()) Py_RETURN_NONE;
    const int64_t tokens = slots->size(0);
    if (tokens < 1 || k->size(0) != tokens || k->size(1) != c.heads || k->size(2) != c.dim || k->stride(2) != 1 || v->stride(2) != 1) Py_RETURN_NONE;
    if (queries && (q->scalar_type() != k->scalar_type() || q->dim() != 3 || q->size(0) != tokens || q->size(2) != c.dim || q->stride(2) != 1 || q->size(1) < 1 ||
                    q->size(1) > INT32_MAX || (c10::GradMode::is_enabled() && q->requires_grad())))
        Py_RETURN_NONE;
    RotaryCall r;
    if (!r.of(args[8], args[9], c.device) || !r.at(positions, slots->sizes(), tokens, c.device) || r.r.rotary_dim > c.dim) Py_RETURN_NONE;
    r.r.axes = r.axes.data();
    at::Tensor out;
    int rc;
    {
        pybind11::gil_scoped_release no_gil;
        if (queries) out = fresh(q->sizes(), q->scalar_type(), c.device);
        rc = g_ops.kv_append_rotated(&r.r, queries ? q->const_data_ptr() : nullptr, queries ? (int)q->size(1) : 0, queries ? q->stride(0) : 0, queries ? q->stride(1) : 0,
                                     queries ? out.mutable_data_ptr() : nullptr, k->const_data_ptr(), v->const_data_ptr(), code, tokens, k->stride(0), k->stride(1),
                                     v->stride(0), v->stride(1), static_cast<const int64_t *>(slots->const_data_ptr()), c.heads, c.dim, c.bits, c.pages, c.page_size,
                                     c.k_codes(), c.v_codes(), c.params->mutable_data_ptr(), c10::cuda::getCurrentCUDAStream(c.device.index()).stream());
    }
    if (rc != BW_OK) Py_RETURN_NONE;
    if (!queries) Py_RETURN_TRUE;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// ---- log probabilities ----
// Logits [..., vocab] as rows with a stride.
struct LogitRows {
    int64_t rows = 1, stride = 0;
    bool of(const at::Tensor &x) {
        const int64_t n = x.dim();
        if (n < 1 || x.stride(n - 1) != 1 || x.numel() < 1) return false;
        for (int64_t i = n - 2; i >= 0; --i) {
            if (x.size(i) == 1) continue;
            if (rows == 1) stride = x.stride(i);
            else if (x.stride(i) != rows * stride) return false;
            rows *= x.size(i);
        }
        return true;
    }
};

// TokenLogProbsFunction of the Python package (log_probs.py) as a node of the graph.  Inputs: the gradients of what was asked for.
struct LogProbsNode : torch::autograd::Node {
    torch::autograd::SavedVariable logits, tokens, top_tokens, stats;
    c10::SmallVector<int64_t, 5> sizes;
    int at_log_probs = -1, at_entropy = -1, at_top = -1, top = 0;      // which input is which
    bool given = false;                                              // there are tokens
    int64_t rows = 0;
    at::ScalarType type = at::kHalf;
    c10::Device device = c10::Device(c10::kCPU);

    std::string name() const override { return "LogProbsNode"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        for (auto *v : {&logits, &tokens, &top_tokens, &stats}) v->reset_data();
    }
    torch::autograd::variable_list apply(torch::autograd::variable_list &&grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        torch::autograd::variable_list result(1);
        const auto of = [&](int i) { return i >= 0 && grads[i].defined() ? grads[i].resolve_neg().contiguous() : at::Tensor(); };
        const at::Tensor g = of(at_log_probs), e = of(at_entropy), gt = of(at_top);
        if (!(g.defined() || e.defined() || gt.defined()) || !task_should_compute_output(0)) return result;
        check_capture(*this, "token_log_probs");
        const bool again = c10::GradMode::is_enabled();
        {
            at::AutoGradMode off(false);
            const char *me = "token_log_probs";
            const at::IntArrayRef all(sizes), lead = all.slice(0, all.size() - 1);
            c10::SmallVector<int64_t, 5> top_sizes(lead.begin(), lead.end());
            top_sizes.push_back(top);
            at::Tensor x = saved(logits, me, device, all, type);
            LogitRows r;
            if (!r.of(x)) {
                x = x.contiguous();
                r = LogitRows();
                r.of(x);
            }
            const at::Tensor t = given ? saved(tokens, me, device, lead, at::kLong).contiguous() : at::Tensor(),
                             tt = top ? saved(top_tokens, me, device, top_sizes, at::kLong).contiguous() : at::Tensor(), s = saved(stats, me, device, {rows, 4}, at::kFloat).contiguous();
            TORCH_CHECK(on_16_bytes(s), "token_log_probs: a tensor saved for the backward pass has come back from its hooks off a 16-byte boundary");
            result[0] = fresh(all, type, device);
            const auto pointer = [](const at::Tensor &v) { return v.defined() ? v.const_data_ptr() : nullptr; };
            const int rc = g_ops.token_log_probs_grad(x.const_data_ptr(), float_code(type), rows, all.back(), r.stride, static_cast<const int64_t *>(pointer(t)),
                                                      static_cast<const float *>(s.const_data_ptr()), static_cast<const float *>(pointer(g)), static_cast<const float *>(pointer(e)),
                                                      top, static_cast<const int64_t *>(pointer(tt)), static_cast<const float *>(pointer(gt)), result[0].mutable_data_ptr(),
                                                      c10::cuda::getCurrentCUDAStream(device.index()).stream());
            TORCH_CHECK(rc == BW_OK, "libbitween_b200: bw_token_log_probs_grad returned status ", rc);
        }
        if (again) once_only(result);
        return result;
    }
};

// token_log_probs(logits, tokens or None, entropy, top): (log_probs, entropy, top_log_probs, top_tokens), None for what is not asked
PyObject *token_log_probs(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 4 || !g_ops.token_log_probs || modes_active() || !PyBool_Check(args[2]) || !PyLong_CheckExact(args[3])) Py_RETURN_NONE;
    const at::Tensor *x = tensor_of(args[0]), *t = args[1] == Py_None ? nullptr : tensor_of(args[1]);
    if (!x || (args[1] != Py_None && !t)) Py_RETURN_NONE;
    const bool entropy = args[2] == Py_True;
    const long top = PyLong_AsLong(args[3]);
    if (top < 0 || top > 32) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    const c10::Device device = x->device();
    LogitRows r;
    if (!device.is_cuda() || device.index() != c10::cuda::current_device() || !usable(x, device) || float_code(x->scalar_type()) < 0 || !r.of(*x)) Py_RETURN_NONE;
    const int64_t vocab = x->size(-1);
    const at::IntArrayRef lead = x->sizes().slice(0, x->dim() - 1);
    if (top > vocab || (t && (!dense(t, device) || t->scalar_type() != at::kLong || t->sizes() != lead))) Py_RETURN_NONE;
    const bool recording = c10::GradMode::is_enabled() && x->requires_grad() && (t || entropy || top);
    at::Tensor lp, h, top_lp, top_t, stats;
    int rc;
    {
        pybind11::gil_scoped_release no_gil;
        c10::SmallVector<int64_t, 5> top_sizes(lead.begin(), lead.end());
        top_sizes.push_back(top);
        if (t) lp = fresh(lead, at::kFloat, device);
        if (entropy) h = fresh(lead, at::kFloat, device);
        if (top) {
            top_lp = fresh(top_sizes, at::kFloat, device);
            top_t = fresh(top_sizes, at::kLong, device);
        }
        if (recording) stats = fresh({r.rows, 4}, at::kFloat, device);
        const auto into = [](at::Tensor &v) { return v.defined() ? v.mutable_data_ptr() : nullptr; };
        rc = g_ops.token_log_probs(x->const_data_ptr(), float_code(x->scalar_type()), r.rows, vocab, r.stride, t ? static_cast<const int64_t *>(t->const_data_ptr()) : nullptr,
                                   static_cast<float *>(into(lp)), static_cast<float *>(into(h)), (int)top, static_cast<float *>(into(top_lp)),
                                   static_cast<int64_t *>(into(top_t)), static_cast<float *>(into(stats)), c10::cuda::getCurrentCUDAStream(device.index()).stream());
        if (rc == BW_OK && recording) {
            const std::shared_ptr<LogProbsNode> node(new LogProbsNode(), torch::autograd::deleteNode);
            node->set_next_edges(torch::autograd::collect_next_edges(*x));
            node->sizes.assign(x->sizes().begin(), x->sizes().end());
            node->top = (int)top;
            node->given = t != nullptr;
            node->rows = r.rows;
            node->type = x->scalar_type();
            node->device = device;
            node->logits = torch::autograd::SavedVariable(*x, false);
            node->tokens = torch::autograd::SavedVariable(t ? *t : at::Tensor(), false);
            node->top_tokens = torch::autograd::SavedVariable(top_t, false);
            node->stats = torch::autograd::SavedVariable(stats, false);
            int n = 0;
            for (auto [tensor, place] : {std::make_pair(&lp, &node->at_log_probs), std::make_pair(&h, &node->at_entropy), std::make_pair(&top_lp, &node->at_top)})
                if (tensor->defined()) {
                    *place = n++;
                    torch::autograd::set_history(*tensor, node);
                }
        }
    }
    if (rc != BW_OK) Py_RETURN_NONE;
    const auto wrapped = [](at::Tensor &v) -> PyObject * {
        if (v.defined()) return THPVariable_Wrap(std::move(v));
        Py_RETURN_NONE;
    };
    PyObject *a = wrapped(lp), *b = wrapped(h), *c = wrapped(top_lp), *d = wrapped(top_t);
    return Py_BuildValue("(NNNN)", a, b, c, d);
    END_HANDLE_TH_ERRORS
}

// set_operators(addresses of the entry points, in the order of Operators)
PyObject *set_operators(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    if (nargs != OPERATORS) {
        PyErr_Format(PyExc_TypeError, "set_operators(%d addresses)", OPERATORS);
        return nullptr;
    }
    void *p[OPERATORS];
    for (int i = 0; i < OPERATORS; ++i) {
        p[i] = PyLong_AsVoidPtr(args[i]);
        if (!p[i] && PyErr_Occurred()) return nullptr;
    }
    static_assert(sizeof(p) == sizeof(g_ops), "the operators are pointers, one address each");
    std::memcpy(&g_ops, p, sizeof(p));
    Py_RETURN_NONE;
}

#define BW_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    BW_METHOD(kv_append),
    BW_METHOD(kv_read),
    BW_METHOD(kv_attend),
    BW_METHOD(adapter_matmul),
    BW_METHOD(rotate),
    BW_METHOD(kv_append_rotated),
    BW_METHOD(token_log_probs),
    BW_METHOD(set_operators),
    {"forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(forward)), METH_FASTCALL, nullptr},
    {"set_entry", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(set_entry)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host_forward", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host_forward() { return PyModule_Create(&module); }
