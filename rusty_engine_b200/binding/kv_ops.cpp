// kv_ops.cpp -- the per-token calls of rusty_engine_b200.kv on torch tensors: argument checks,
// output allocation and the call of the C ABI (include/rmoe.h), in one native step.
//
// A decode step makes these calls for every layer, on kernels of 3 to 10 us; checking, packing and
// allocating in Python took 11 to 14 us per call and was what bounded them.  Here the same work
// takes about 2 us.  Nothing is computed in this file.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <string>

#include "../../include/rmoe.h"

namespace {

PyObject* g_error = nullptr;  // moe.EngineError
PyObject* g_call = nullptr;   // moe._call: raises for a status that is not OK

struct Raised : std::exception {};  // a Python exception is set

template <typename... A>
[[noreturn]] void refuse(const char* fmt, A... a) {
    PyErr_Format(g_error, fmt, a...);
    throw Raised();
}

void check(rmoe_status s) {
    if (s == RMOE_OK) return;
    PyObject* r = PyObject_CallFunction(g_call, "i", (int)s);
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_SetString(g_error, rmoe_last_error());
    throw Raised();
}

bool none(PyObject* o) { return o == Py_None; }

const at::Tensor& tensor(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) refuse("%s: a tensor, got %R", what, (PyObject*)Py_TYPE(o));
    return THPVariable_Unpack(o);
}

std::string describe(const at::Tensor& t) {
    std::string s = std::string(c10::toString(t.scalar_type())) + " [";
    for (int64_t i = 0; i < t.dim(); i++) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + "] on " + t.device().str();
}

uint32_t type_of(const at::Tensor& t, const char* what) {
    if (t.is_cuda()) {
        if (t.scalar_type() == at::kFloat) return RMOE_GGML_F32;
        if (t.scalar_type() == at::kHalf) return RMOE_GGML_F16;
        if (t.scalar_type() == at::kBFloat16) return RMOE_GGML_BF16;
    }
    refuse("%s: a float32, float16 or bfloat16 CUDA tensor, got %s", what, describe(t).c_str());
}

void on_device(const at::Tensor& t, int64_t device, const char* what) {
    if (t.get_device() != device) refuse("%s is on %s, the handle on device %d", what, t.device().str().c_str(), (int)device);
}

void same(const at::Tensor& t, const at::Tensor& like, const char* what) {
    if (t.scalar_type() != like.scalar_type() || t.device() != like.device())
        refuse("%s: %s beside %s", what, describe(t).c_str(), describe(like).c_str());
}

rmoe_rows rows(const at::Tensor& t, const char* what) {
    if (t.dim() != 3 || (t.stride(2) != 1 && t.size(2) != 1))
        refuse("%s: a [tokens, heads, head_dim] tensor whose heads are contiguous, got %s", what, describe(t).c_str());
    rmoe_rows r;
    r.data = t.data_ptr();
    r.stride_t = t.stride(0);
    r.stride_h = t.stride(1);
    r.heads = (uint32_t)t.size(1);
    r.pad = 0;
    return r;
}

int32_t* ints(const at::Tensor& t, const char* what, int64_t device, int64_t n = -1) {
    if (t.scalar_type() != at::kInt || !t.is_cuda() || t.get_device() != device || !t.is_contiguous())
        refuse("%s: a contiguous int32 tensor on CUDA device %d, got %s", what, (int)device, describe(t).c_str());
    if (n >= 0 && t.numel() != n) refuse("%s: %lld entries, expected %lld", what, (long long)t.numel(), (long long)n);
    return t.data_ptr<int32_t>();
}

at::Tensor like(const at::Tensor& t) { return at::empty(t.sizes(), t.options()); }

int64_t integer(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised();
    return v;
}

double real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised();
    return v;
}

bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Raised();
    return v != 0;
}

// The calls run on the current stream, where their outputs are allocated too.
void* stream_of(int64_t device) { return (void*)c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

PyObject* pair(const at::Tensor& a, const at::Tensor& b) {
    PyObject *x = THPVariable_Wrap(a), *y = THPVariable_Wrap(b), *t = PyTuple_Pack(2, x, y);
    Py_XDECREF(x);
    Py_XDECREF(y);
    return t;
}

// Every entry: no C++ exception leaves it.
template <typename F>
PyObject* entry(F f) {
    try {
        return f();
    } catch (const Raised&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "kv_ops: unknown C++ exception");
    }
    return nullptr;
}

#define ARGS(n)                                                                       \
    if (nargs != (n)) {                                                               \
        PyErr_Format(PyExc_TypeError, "%d arguments expected, got %zd", (n), nargs);  \
        return nullptr;                                                               \
    }

// rope_apply(handle, device, q, positions, k, out, k_out, inverse)
PyObject* rope_apply(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    ARGS(8)
    return entry([&]() -> PyObject* {
        const at::Tensor &q = tensor(a[2], "q"), &pos = tensor(a[3], "positions");
        const int64_t dev = integer(a[1]);
        rmoe_rope_args r{};
        r.type = type_of(q, "q");
        on_device(q, dev, "q");
        r.q = rows(q, "q");
        at::Tensor out = none(a[5]) ? like(q) : tensor(a[5], "out"), ko;
        same(out, q, "out");
        if (out.sizes() != q.sizes()) refuse("out: %s beside q %s", describe(out).c_str(), describe(q).c_str());
        r.q_out = rows(out, "out");
        if (!none(a[4])) {
            const at::Tensor& k = tensor(a[4], "k");
            same(k, q, "k");
            r.k = rows(k, "k");
            ko = none(a[6]) ? like(k) : tensor(a[6], "k_out");
            same(ko, q, "k_out");
            r.k_out = rows(ko, "k_out");
            if (k.size(0) != q.size(0) || k.size(2) != q.size(2) || ko.sizes() != k.sizes())
                refuse("k: %s / %s beside q %s", describe(k).c_str(), describe(ko).c_str(), describe(q).c_str());
        }
        r.T = (uint32_t)q.size(0);
        r.head_dim = (uint32_t)q.size(2);
        r.positions = ints(pos, "positions", dev, q.size(0));
        r.inverse = truth(a[7]);
        check(rmoe_rope_apply((rmoe_rope*)integer(a[0]), &r, stream_of(dev)));
        return ko.defined() ? pair(out, ko) : THPVariable_Wrap(out);
    });
}

// extend(table, lens, new_lens, free, n_free, total, block_size) -> (cu, positions, slots, lens, n_free)
PyObject* extend(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    ARGS(7)
    return entry([&]() -> PyObject* {
        const at::Tensor &table = tensor(a[0], "table"), &lens = tensor(a[1], "lens"), &nl = tensor(a[2], "new_lens"),
                         &fr = tensor(a[3], "free"), &nf = tensor(a[4], "n_free");
        if (table.dim() != 2 || !table.is_cuda())
            refuse("table: a [requests, blocks] CUDA tensor, got %s", describe(table).c_str());
        const int64_t dev = table.get_device(), R = table.size(0), T = integer(a[5]), bs = integer(a[6]);
        if (T < 0 || T > 0x7fffffff || bs < 0 || bs > 0xffff) refuse("total %lld, block size %lld", (long long)T, (long long)bs);
        rmoe_kv_extend_args e{};
        e.table = ints(table, "table", dev);
        e.lens = ints(lens, "lens", dev, R);
        e.new_lens = ints(nl, "new_lens", dev, R);
        e.free_list = ints(fr, "free", dev);
        e.n_free = ints(nf, "n_free", dev, 1);
        const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
        // one allocation, five tensors of it
        const int64_t sizes[5] = {R + 1, T, T, R, 1};
        const at::Tensor buf = at::empty({2 * R + 2 + 2 * T}, table.options());
        at::Tensor out[5];
        int32_t* at_[5];
        for (int64_t i = 0, off = 0; i < 5; off += sizes[i++]) {
            out[i] = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buf.storage()), buf.key_set(), buf.dtype());
            out[i].unsafeGetTensorImpl()->set_sizes_and_strides(c10::IntArrayRef(&sizes[i], 1), c10::IntArrayRef({1}), off);
            at_[i] = buf.data_ptr<int32_t>() + off;
        }
        e.cu = at_[0];
        e.positions = at_[1];
        e.slots = at_[2];
        e.lens_out = at_[3];
        e.n_free_out = at_[4];
        e.R = (uint32_t)R;
        e.max_blocks = (uint32_t)table.size(1);
        e.T = (uint32_t)T;
        e.block_size = (uint32_t)bs;
        e.free_cap = (uint32_t)fr.numel();
        check(rmoe_kv_extend(&e, stream_of(dev)));
        PyObject* t = PyTuple_New(5);
        if (!t) throw Raised();
        for (int i = 0; i < 5; i++) PyTuple_SET_ITEM(t, i, THPVariable_Wrap(out[i]));
        return t;
    });
}

// append(handle, device, n_kv_heads, head_dim, k, v, slots, rope handle, positions, q, q_out) -> q_out
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    ARGS(11)
    return entry([&]() -> PyObject* {
        const int64_t dev = integer(a[1]), H = integer(a[2]), D = integer(a[3]);
        const at::Tensor &k = tensor(a[4], "k"), &v = tensor(a[5], "v");
        rmoe_kv_append_args r{};
        r.type = type_of(k, "k");
        on_device(k, dev, "k");
        same(v, k, "v");
        r.k = rows(k, "k");
        r.v = rows(v, "v");
        const int64_t T = k.size(0);
        if (k.size(1) != H || k.size(2) != D || v.sizes() != k.sizes())
            refuse("k %s / v %s, expected [%lld, %lld, %lld]", describe(k).c_str(), describe(v).c_str(), (long long)T,
                   (long long)H, (long long)D);
        r.T = (uint32_t)T;
        r.slots = ints(tensor(a[6], "slots"), "slots", dev, T);
        r.rope = (rmoe_rope*)integer(a[7]);
        at::Tensor qo;
        if (r.rope) {
            if (none(a[8])) refuse("rope needs positions");
            r.positions = ints(tensor(a[8], "positions"), "positions", dev, T);
        }
        if (!none(a[9])) {
            if (!r.rope) refuse("q is only taken with a rope");
            const at::Tensor& q = tensor(a[9], "q");
            same(q, k, "q");
            r.q = rows(q, "q");
            qo = none(a[10]) ? like(q) : tensor(a[10], "q_out");
            same(qo, k, "q_out");
            r.q_out = rows(qo, "q_out");
            if (q.size(0) != T || q.size(2) != D || qo.sizes() != q.sizes())
                refuse("q %s / %s beside k %s", describe(q).c_str(), describe(qo).c_str(), describe(k).c_str());
        }
        check(rmoe_kv_append((rmoe_kv*)integer(a[0]), &r, stream_of(dev)));
        if (qo.defined()) return THPVariable_Wrap(qo);
        Py_RETURN_NONE;
    });
}

// read(handle, cache codes, slots, like): `like` any tensor of the wanted type -> (k, v)
PyObject* read(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    ARGS(4)
    return entry([&]() -> PyObject* {
        const at::Tensor &codes = tensor(a[1], "codes"), &slots = tensor(a[2], "slots"), &as = tensor(a[3], "like");
        const int64_t dev = codes.get_device(), n = slots.numel();
        const int32_t* p = ints(slots, "slots", dev);
        const uint32_t type = type_of(as, "read");
        if (n > 0x7fffffff) refuse("%lld slots", (long long)n);
        const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
        at::Tensor k = at::empty({n, codes.size(1), codes.size(3)}, as.options()), v = at::empty(k.sizes(), as.options());
        check(rmoe_kv_read((rmoe_kv*)integer(a[0]), p, (uint32_t)n, type, k.data_ptr(), v.data_ptr(), stream_of(dev)));
        return pair(k, v);
    });
}

// attend(handle, device, head_dim, q, table, lens, cu, scale, window, max_new, out, return_lse)
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    ARGS(12)
    return entry([&]() -> PyObject* {
        const int64_t dev = integer(a[1]), D = integer(a[2]);
        const at::Tensor &q = tensor(a[3], "q"), &table = tensor(a[4], "table"), &lens = tensor(a[5], "lens"),
                         &cu = tensor(a[6], "cu");
        rmoe_kv_attend_args r{};
        r.type = type_of(q, "q");
        on_device(q, dev, "q");
        r.q = rows(q, "q");
        at::Tensor out = none(a[10]) ? like(q) : tensor(a[10], "out"), lse;
        same(out, q, "out");
        r.out = rows(out, "out");
        if (q.size(2) != D || out.sizes() != q.sizes())
            refuse("q %s / out %s with head_dim %lld", describe(q).c_str(), describe(out).c_str(), (long long)D);
        if (table.dim() != 2) refuse("table: [requests, blocks], got %s", describe(table).c_str());
        const int64_t T = q.size(0), R = table.size(0), window = integer(a[8]), max_new = integer(a[9]);
        if (window < 0 || window > 0x7fffffff || max_new < 0 || max_new > 0x7fffffff)
            refuse("window %lld, max_new %lld", (long long)window, (long long)max_new);
        r.table = ints(table, "table", dev);
        r.lens = ints(lens, "lens", dev, R);
        r.cu = ints(cu, "cu", dev, R + 1);
        if (truth(a[11])) {
            lse = at::empty({T, q.size(1)}, q.options().dtype(at::kFloat));
            r.lse = lse.data_ptr<float>();
        }
        r.R = (uint32_t)R;
        r.max_blocks = (uint32_t)table.size(1);
        r.T = (uint32_t)T;
        r.scale = (float)real(a[7]);
        r.window = (uint32_t)window;
        r.max_new = (uint32_t)max_new;
        check(rmoe_kv_attend((rmoe_kv*)integer(a[0]), &r, stream_of(dev)));
        return lse.defined() ? pair(out, lse) : THPVariable_Wrap(out);
    });
}

// setup(EngineError, _call)
PyObject* setup(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    ARGS(2)
    Py_INCREF(a[0]);
    Py_INCREF(a[1]);
    g_error = a[0];
    g_call = a[1];
    Py_RETURN_NONE;
}

#define FAST(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(rope_apply), FAST(extend), FAST(append), FAST(read), FAST(attend), FAST(setup), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kv_ops", "torch-tensor entry of rusty_engine_b200.kv", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kv_ops(void) { return PyModule_Create(&module); }
