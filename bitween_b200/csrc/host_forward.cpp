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

// ---- the quantised key-value cache and the adapters ------------------------------------------------------------------
// None, again, for every call that is not plain (the Python path converts, copies or raises).  Scratch comes from the caching allocator, so
// that calls of other streams, threads and graphs have their own.

using KvAppend = decltype(&bw_kv_append);
using KvRead = decltype(&bw_kv_read);
using KvAttend = decltype(&bw_kv_attend);
using KvAttendBytes = decltype(&bw_kv_attend_workspace_bytes);
using AdapterBytes = decltype(&bw_adapter_hidden_bytes);
using AdapterForward = decltype(&bw_adapter_forward);
using AdapterBackward = decltype(&bw_adapter_backward);
struct Operators {
    KvAppend kv_append;
    KvRead kv_read;
    KvAttend kv_attend;
    KvAttendBytes kv_attend_bytes;
    AdapterBytes adapter_bytes;
    AdapterForward adapter_forward;
    AdapterBackward adapter_backward;
} g_ops = {};

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

// kv_attend(k_codes, v_codes, params, bits, q, page_table, lengths, softmax_scale): the attended values
PyObject *kv_attend(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    Cache c;
    if (nargs != 8 || !g_ops.kv_attend || !PyFloat_CheckExact(args[7]) || !c.of(args)) Py_RETURN_NONE;
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
        const at::Tensor ws = bytes_of(g_ops.kv_attend_bytes(batch, heads, c.heads, c.dim, c.page_size, table->size(1)), c.device);
        rc = g_ops.kv_attend(q->const_data_ptr(), code, batch, heads, q->stride(0), q->stride(1), c.k_codes(), c.v_codes(), c.params->const_data_ptr(), c.bits,
                             c.pages, c.page_size, c.heads, c.dim, static_cast<const int32_t *>(table->const_data_ptr()), table->stride(0), table->size(1),
                             static_cast<const int32_t *>(lengths->const_data_ptr()), scale, out.mutable_data_ptr(), ws.defined() ? ws.mutable_data_ptr() : nullptr,
                             ws.defined() ? (size_t)ws.numel() : 0, c10::cuda::getCurrentCUDAStream(c.device.index()).stream());
    }
    if (rc != BW_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
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

    // A saved tensor, as the kernels take it.  Hooks may have made another tensor of it in the meantime (moved, packed).
    at::Tensor back(const torch::autograd::SavedVariable &saved, at::IntArrayRef sizes, at::ScalarType as) const {
        at::Tensor t = saved.unpack();
        TORCH_CHECK(t.defined() && t.layout() == c10::kStrided && t.device() == device && t.scalar_type() == as && t.sizes() == sizes,
                    "adapter_matmul: a tensor saved for the backward pass has come back from its hooks in another shape, type or place");
        t = t.resolve_neg().contiguous();
        return on_16_bytes(t) ? t : t.clone();
    }

    std::string name() const override { return "AdapterNode"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        for (auto *v : {&x, &down, &up, &index, &scaling, &hidden}) v->reset_data();
    }
    // The engine hands each gradient to the stream on which its consumer was recorded.  The default stream cannot take one from a capture, and torch
    // does not survive the attempt.
    void check_capture() const {
        if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
        for (uint32_t i = 0; i < num_outputs(); ++i) {
            if (!task_should_compute_output(i)) continue;
            const auto stream = next_edge(i).function->stream();
            TORCH_CHECK(!stream || c10::cuda::CUDAStream(*stream) != c10::cuda::getDefaultCUDAStream(stream->device_index()),
                        "adapter_matmul: this backward pass cannot be captured while a graph of the same tensors, recorded on the default stream, is alive; free it, or "
                        "record it on another stream");
        }
    }
    torch::autograd::variable_list apply(torch::autograd::variable_list &&grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        torch::autograd::variable_list result(4);
        const at::Tensor g = grads[0];
        if (!g.defined()) return result;
        check_capture();
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
        if (again) {
            // as once_differentiable has it: an error for whoever differentiates these
            for (auto &t : result)
                if (t.defined()) t = (*std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that was marked with @once_differentiable", 1))(
                                     {t.detach().requires_grad_()})[0];
        }
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

// set_operators(addresses of the entry points, in the order of Operators)
PyObject *set_operators(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    void *p[7];
    if (nargs != 7) {
        PyErr_SetString(PyExc_TypeError, "set_operators(seven addresses)");
        return nullptr;
    }
    for (int i = 0; i < 7; ++i) {
        p[i] = PyLong_AsVoidPtr(args[i]);
        if (!p[i] && PyErr_Occurred()) return nullptr;
    }
    g_ops = {reinterpret_cast<KvAppend>(p[0]),     reinterpret_cast<KvRead>(p[1]),         reinterpret_cast<KvAttend>(p[2]),       reinterpret_cast<KvAttendBytes>(p[3]),
             reinterpret_cast<AdapterBytes>(p[4]), reinterpret_cast<AdapterForward>(p[5]), reinterpret_cast<AdapterBackward>(p[6])};
    Py_RETURN_NONE;
}

#define BW_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    BW_METHOD(kv_append),
    BW_METHOD(kv_read),
    BW_METHOD(kv_attend),
    BW_METHOD(adapter_matmul),
    BW_METHOD(set_operators),
    {"forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(forward)), METH_FASTCALL, nullptr},
    {"set_entry", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(set_entry)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host_forward", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host_forward() { return PyModule_Create(&module); }
