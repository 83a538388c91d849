// calls.cpp -- the Python calls of the hybrid layers' operators: argument checks on
// torch tensors, the device and its current stream, and the call into the C ABI of
// include/genllm_paged.h.  These calls have up to 45 arguments: read and checked in
// Python and passed through ctypes, a single token's calls took 7.5 to 10 us of host
// time; from here they take 4.0 to 4.3, most of it the launch.  The entry points'
// addresses come from the ctypes binding, so that a process has one copy of the
// library.  Every function returns the status code; the interpreter's lock is released
// while the C call runs, as ctypes does.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <sstream>
#include <string>

#include "../../include/genllm_paged.h"

namespace {

decltype(&genllm_gated_delta_workspace_bytes) g_delta_workspace = nullptr;
decltype(&genllm_gated_delta_rule) g_delta = nullptr;
decltype(&genllm_causal_conv) g_conv = nullptr;
decltype(&genllm_qk_norm_rope_axes) g_axes = nullptr;

struct Refused {
    std::string why;
};

// The operator's name in front of every refusal.
struct Checks {
    const char* op;
    c10::Device device = c10::kCPU;
    at::ScalarType dtype = at::kBFloat16;

    [[noreturn]] void refuse(const std::string& why) const { throw Refused{std::string(op) + ": " + why}; }

    const at::Tensor& tensor(PyObject* o, const char* name) const {
        if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
        const at::Tensor& t = THPVariable_Unpack(o);
        if (t.layout() != at::kStrided) refuse(std::string(name) + " must be a strided tensor");
        return t;
    }
    // the first tensor sets device and element type
    const at::Tensor& elements(PyObject* o, const char* name, int64_t dims) {
        const at::Tensor& t = tensor(o, name);
        if (t.scalar_type() != at::kBFloat16 && t.scalar_type() != at::kHalf)
            refuse("bf16 or float16 elements, got " + std::string(c10::toString(t.scalar_type())));
        if (!t.is_cuda()) refuse("expected a GPU tensor");
        if (t.dim() != dims) refuse(std::string(name) + " must have " + std::to_string(dims) + " dims");
        device = t.device(), dtype = t.scalar_type();
        return rows(t, name, t.sizes(), dtype);
    }
    // of that shape, type and the device, the last dim dense
    const at::Tensor& rows(const at::Tensor& t, const char* name, at::IntArrayRef sizes, at::ScalarType type) const {
        if (t.sizes() != sizes || t.scalar_type() != type || t.device() != device ||
            (!sizes.empty() && sizes.back() > 1 && t.strides().back() != 1)) {
            std::ostringstream s;
            s << name << " must be " << type << ' ' << sizes << " on " << device << ", the last dim dense; got "
              << t.scalar_type() << ' ' << t.sizes() << " with strides " << t.strides() << " on " << t.device();
            refuse(s.str());
        }
        return t;
    }
    const at::Tensor& whole(const at::Tensor& t, const char* name, at::IntArrayRef sizes, at::ScalarType type) const {
        if (!rows(t, name, sizes, type).is_contiguous()) refuse(std::string(name) + " must be contiguous");
        return t;
    }
    // null for None
    template <typename T>
    const T* optional(PyObject* o, const char* name, at::IntArrayRef sizes, at::ScalarType type) const {
        if (o == Py_None) return nullptr;
        return static_cast<const T*>(whole(tensor(o, name), name, sizes, type).mutable_data_ptr());
    }
    int32_t code() const { return dtype == at::kHalf ? GENLLM_DTYPE_F16 : GENLLM_DTYPE_BF16; }
    int32_t size(int64_t n) const {
        if (n > INT32_MAX) refuse("a size does not fit in 32 bits");
        return int32_t(n);
    }
};

// None: the device's current stream
void* stream_of(PyObject* o, c10::Device device) {
    if (o == Py_None) return c10::hip::getCurrentHIPStream(device.index()).stream();
    void* p = PyLong_AsVoidPtr(o);
    if (!p && PyErr_Occurred()) throw python_error();
    return p;
}

double number(PyObject* o) {
    const double x = PyFloat_AsDouble(o);
    if (x == -1.0 && PyErr_Occurred()) throw python_error();
    return x;
}

template <typename T = void>
T* data(const at::Tensor& t) {
    return static_cast<T*>(t.mutable_data_ptr());
}

class Unlocked {
    PyThreadState* state_ = PyEval_SaveThread();

  public:
    Unlocked() = default;
    Unlocked(const Unlocked&) = delete;
    ~Unlocked() { PyEval_RestoreThread(state_); }
};

// q, k, v, a, b, state, out, scale, a_log, dt_bias, l2_eps, seq_lens, state_ids, workspace, stream
int gated_delta_rule(PyObject* const* arg) {
    Checks c{"gated_delta_rule"};
    const at::Tensor& q = c.elements(arg[0], "q", 4);
    const at::Tensor& v = c.tensor(arg[2], "v");
    if (v.dim() != 4) c.refuse("v must have 4 dims");
    const int64_t B = q.size(0), S = q.size(1), Hk = q.size(2), Dk = q.size(3), Hv = v.size(2), Dv = v.size(3);
    const int64_t vs[4] = {B, S, Hv, Dv}, gs[3] = {B, S, Hv}, es[1] = {B}, hs[1] = {Hv};
    const at::Tensor& k = c.rows(c.tensor(arg[1], "k"), "k", q.sizes(), c.dtype);
    c.rows(v, "v", vs, c.dtype);
    const at::Tensor& out = c.rows(c.tensor(arg[6], "out"), "out", vs, c.dtype);
    const bool raw = arg[8] != Py_None;
    if (raw != (arg[9] != Py_None)) c.refuse("a_log and dt_bias go together");
    const at::ScalarType gate = raw ? c.dtype : at::kFloat;
    const at::Tensor& a = c.rows(c.tensor(arg[3], "a"), "a", gs, gate);
    const at::Tensor& b = c.rows(c.tensor(arg[4], "b"), "b", gs, gate);
    const at::Tensor& state = c.tensor(arg[5], "state");
    const int64_t ss[4] = {state.dim() ? state.size(0) : 0, Hv, Dk, Dv};
    c.whole(state, "state", ss, at::kFloat);
    const float* a_log = c.optional<float>(arg[8], "a_log", hs, at::kFloat);
    const float* dt_bias = c.optional<float>(arg[9], "dt_bias", hs, at::kFloat);
    const int32_t* lens = c.optional<int32_t>(arg[11], "seq_lens", es, at::kInt);
    const int32_t* ids = c.optional<int32_t>(arg[12], "state_ids", es, at::kInt);
    const c10::DeviceGuard guard(c.device);
    const int32_t n[6] = {c.size(B), c.size(S), c.size(Hk), c.size(Hv), c.size(Dk), c.size(Dv)};
    at::Tensor own;
    void* ws = nullptr;
    size_t ws_bytes = 0;
    if (arg[13] != Py_None) {
        const at::Tensor& w = c.tensor(arg[13], "workspace");
        if (w.device() != c.device || !w.is_contiguous()) c.refuse("the workspace must be contiguous on the tensors' device");
        ws = data(w), ws_bytes = w.nbytes();
    } else if (const size_t need = g_delta_workspace(n[0], n[1], n[2], n[3], n[4], n[5])) {
        // from the current stream's pool, and so for a call on that stream: with another
        // stream the caller brings the workspace
        own = at::empty({int64_t(need)}, at::TensorOptions().dtype(at::kByte).device(c.device));
        ws = data(own), ws_bytes = need;
    }
    const float scale = float(number(arg[7])), eps = arg[10] == Py_None ? -1.0f : float(number(arg[10]));
    void* const stream = stream_of(arg[14], c.device);
    const Unlocked unlocked;
    return g_delta(data(q), q.stride(0), q.stride(1), q.stride(2), data(k), k.stride(0), k.stride(1), k.stride(2), data(v),
                   v.stride(0), v.stride(1), v.stride(2), data(a), a.stride(0), a.stride(1), data(b), b.stride(0),
                   b.stride(1), a_log, dt_bias, data<float>(state), c.size(ss[0]), ids, lens, data(out),
                   out.stride(0), out.stride(1), out.stride(2), n[0], n[1], n[2], n[3], n[4], n[5], c.code(),
                   scale, eps, ws, ws_bytes, stream);
}

// x, weight, out, state, bias, silu, seq_lens, state_ids, stream
int causal_conv(PyObject* const* arg) {
    Checks c{"causal_conv"};
    const at::Tensor& x = c.elements(arg[0], "x", 3);
    const int64_t B = x.size(0), S = x.size(1), C = x.size(2);
    const at::Tensor& out = c.rows(c.tensor(arg[2], "out"), "out", x.sizes(), c.dtype);
    const at::Tensor& weight = c.tensor(arg[1], "weight");
    const int64_t W = weight.dim() ? weight.size(-1) : 0, cs[1] = {C}, wsz[2] = {C, W}, es[1] = {B};
    c.whole(weight, "weight", wsz, c.dtype);
    const void* bias = c.optional<void>(arg[4], "bias", cs, c.dtype);
    void* st = nullptr;
    int64_t n = 0;
    if (arg[3] != Py_None) {
        const at::Tensor& state = c.tensor(arg[3], "state");
        n = state.dim() ? state.size(0) : 0;
        const int64_t ss[3] = {n, W - 1, C};
        st = data(c.whole(state, "state", ss, c.dtype));
    }
    const int silu = PyObject_IsTrue(arg[5]);
    if (silu < 0) throw python_error();
    const int32_t* lens = c.optional<int32_t>(arg[6], "seq_lens", es, at::kInt);
    const int32_t* ids = c.optional<int32_t>(arg[7], "state_ids", es, at::kInt);
    const c10::DeviceGuard guard(c.device);
    void* const stream = stream_of(arg[8], c.device);
    const Unlocked unlocked;
    return g_conv(data(x), x.stride(0), x.stride(1), data(weight), bias, data(out), out.stride(0), out.stride(1), st, c.size(n),
                  ids, lens, c.size(B), c.size(S), c.size(C), c.size(W), c.code(), silu, stream);
}

// q, k, q_out, k_out, gamma_q, gamma_k, eps, cos, sin, positions, sections, interleaved, stream
int qk_norm_rope_axes(PyObject* const* arg) {
    Checks c{"qk_norm_rope_axes"};
    const at::Tensor& q = c.elements(arg[0], "q", 3);
    const int64_t S = q.size(0), D = q.size(2), ds[1] = {D};
    const at::Tensor& q_out = c.rows(c.tensor(arg[2], "q_out"), "q_out", q.sizes(), c.dtype);
    const at::Tensor *k = nullptr, *k_out = nullptr;
    int64_t Hk = 0;
    if (arg[1] != Py_None) {
        k = &c.tensor(arg[1], "k");
        if (k->dim() != 3) c.refuse("k must have 3 dims");
        Hk = k->size(1);
        const int64_t ks[3] = {S, Hk, D};
        c.rows(*k, "k", ks, c.dtype);
        k_out = &c.rows(c.tensor(arg[3], "k_out"), "k_out", ks, c.dtype);
    }
    const float* gamma_q = c.optional<float>(arg[4], "gamma_q", ds, at::kFloat);
    const float* gamma_k = c.optional<float>(arg[5], "gamma_k", ds, at::kFloat);
    const at::Tensor& cos = c.tensor(arg[7], "cos");
    if (cos.dim() != 2) c.refuse("cos must have 2 dims");
    c.whole(cos, "cos", cos.sizes(), at::kFloat);
    const at::Tensor& sin = c.whole(c.tensor(arg[8], "sin"), "sin", cos.sizes(), at::kFloat);
    PyObject* const seq = PySequence_Fast(arg[10], "qk_norm_rope_axes: sections must be a sequence of ints");
    if (!seq) throw python_error();
    const Py_ssize_t axes = PySequence_Fast_GET_SIZE(seq);
    int32_t sections[4] = {};  // the C call refuses more than four
    for (Py_ssize_t i = 0; i < axes && i < 4; ++i) {
        const long x = PyLong_AsLong(PySequence_Fast_GET_ITEM(seq, i));
        if (x == -1 && PyErr_Occurred()) {
            Py_DECREF(seq);
            throw python_error();
        }
        sections[i] = x < INT32_MIN || x > INT32_MAX ? -1 : int32_t(x);
    }
    Py_DECREF(seq);
    const int64_t ps[2] = {axes, S};
    const at::Tensor& pos = c.rows(c.tensor(arg[9], "positions"), "positions", ps, at::kInt);
    const int inter = PyObject_IsTrue(arg[11]);
    if (inter < 0) throw python_error();
    const c10::DeviceGuard guard(c.device);
    const float eps = float(number(arg[6]));
    void* const stream = stream_of(arg[12], c.device);
    const Unlocked unlocked;
    return g_axes(data(q), q.stride(0), q.stride(1), data(q_out), q_out.stride(0), q_out.stride(1), gamma_q, c.size(q.size(1)),
                  k ? data(*k) : nullptr, k ? k->stride(0) : 0, k ? k->stride(1) : 0, k ? data(*k_out) : nullptr,
                  k ? k_out->stride(0) : 0, k ? k_out->stride(1) : 0, gamma_k, c.size(Hk), eps,
                  data<float>(cos), data<float>(sin),
                  c.size(cos.size(0)), c.size(cos.size(1)), data<int32_t>(pos), pos.stride(0),
                  int32_t(axes), sections, inter, c.size(S), c.size(D), c.code(), stream);
}

template <int (*F)(PyObject* const*), Py_ssize_t N>
PyObject* entry(PyObject*, PyObject* const* arg, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", N, n);
        return nullptr;
    }
    if (!g_delta) {
        PyErr_SetString(PyExc_RuntimeError, "bind() comes first");
        return nullptr;
    }
    try {
        return PyLong_FromLong(F(arg));
    } catch (const Refused& r) {
        PyErr_SetString(PyExc_ValueError, r.why.c_str());
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// the addresses of the four C functions
PyObject* bind(PyObject*, PyObject* const* arg, Py_ssize_t n) {
    if (n != 4) {
        PyErr_SetString(PyExc_TypeError, "bind() takes four addresses");
        return nullptr;
    }
    void* p[4];
    for (int i = 0; i < 4; ++i)
        if (!(p[i] = PyLong_AsVoidPtr(arg[i]))) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind(): a null address");
            return nullptr;
        }
    g_delta_workspace = reinterpret_cast<decltype(g_delta_workspace)>(p[0]);
    g_delta = reinterpret_cast<decltype(g_delta)>(p[1]);
    g_conv = reinterpret_cast<decltype(g_conv)>(p[2]);
    g_axes = reinterpret_cast<decltype(g_axes)>(p[3]);
    Py_RETURN_NONE;
}

PyCFunction fast(PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f)); }

PyMethodDef methods[] = {
    {"bind", fast(bind), METH_FASTCALL, "The addresses of the C functions"},
    {"gated_delta_rule", fast(entry<gated_delta_rule, 15>), METH_FASTCALL, "genllm_gated_delta_rule on tensors"},
    {"causal_conv", fast(entry<causal_conv, 9>), METH_FASTCALL, "genllm_causal_conv on tensors"},
    {"qk_norm_rope_axes", fast(entry<qk_norm_rope_axes, 13>), METH_FASTCALL, "genllm_qk_norm_rope_axes on tensors"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", "Calls of the hybrid layers' operators", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&module); }
