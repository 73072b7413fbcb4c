// The host path of a call: device pointers of tensors and launches of the C-ABI library without ctypes.
//
// A small kernel takes 2 to 4 us, and with ctypes a call took 6.5 to 10 us of host: about 0.7 us for the checks and the address of each
// tensor in Python, and 2 us to convert the arguments.  Both are done here; bind() makes a function of every entry point that launches
// work, from its own declaration in spiral_mi355.h, and an argument has to be of the declared type.  (us a call with the queue kept full, ctypes
// / here: a four-layer stack on packed weights 7.2 / 5.6, one on row-major weights 11.4 / 7.1, the CEM update 76 / 63, a GEMM of 16 x 16 x 296
// 7.6 / 5.4, a sampled softmax of 32 rows with its outputs allocated 11.7 / 8.7.)  What is left is the runtime's launch, about 4 us.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <dlfcn.h>
#include <string.h>

#include <exception>
#include <memory>
#include <new>
#include <tuple>
#include <type_traits>
#include <utility>
#include <vector>

#include "spiral_mi355.h"

namespace {

PyObject* g_calls = nullptr;      // lists of the tape being recorded: (function, arguments but the stream), tensors
PyObject* g_keep = nullptr;
PyObject* g_void_p = nullptr;     // of ctypes: c_void_p, c_int32, Array, _Pointer, cast, the type of byref(...)
PyObject* g_int32 = nullptr;
PyObject* g_array = nullptr;
PyObject* g_pointer = nullptr;
PyObject* g_cast = nullptr;
PyObject* g_byref = nullptr;

// ---- arguments: what the caller's objects become; false with an exception set if they do not fit ----
constexpr Py_ssize_t MOST = 16;   // elements of a host array given as a list or tuple that need no allocation

bool as_integer(PyObject* o, unsigned long long& v) {      // as ctypes: the low bits of any integer
    if (PyLong_Check(o)) {
        v = PyLong_AsUnsignedLongLongMask(o);
    } else {
        PyObject* i = PyNumber_Index(o);
        if (i == nullptr) return false;
        v = PyLong_AsUnsignedLongLongMask(i);
        Py_DECREF(i);
    }
    return !(v == (unsigned long long)-1 && PyErr_Occurred());
}

bool as_address(PyObject* o, void*& p) {                   // None, an integer or a c_void_p
    if (o == Py_None) {
        p = nullptr;
        return true;
    }
    if (PyLong_Check(o)) {
        p = (void*)PyLong_AsUnsignedLongLongMask(o);      // as ctypes: the low bits
        return true;
    }
    const int is_void_p = PyObject_IsInstance(o, g_void_p);
    if (is_void_p < 0) return false;
    if (is_void_p == 0) {
        PyErr_Format(PyExc_TypeError, "an address is None, an integer or a c_void_p, not %s", Py_TYPE(o)->tp_name);
        return false;
    }
    PyObject* v = PyObject_GetAttrString(o, "value");
    if (v == nullptr) return false;
    const bool ok = as_address(v, p);
    Py_DECREF(v);
    return ok;
}

// The buffer behind an object of ctypes.
struct Buffer {
    Py_buffer view{};
    Buffer() = default;
    Buffer(const Buffer&) = delete;
    ~Buffer() {
        if (view.obj != nullptr) PyBuffer_Release(&view);
    }
    bool take(PyObject* o) { return PyObject_GetBuffer(o, &view, PyBUF_SIMPLE) == 0; }
};

bool refuse(PyObject* o, const char* what) {
    PyErr_Format(PyExc_TypeError, "%s, not %s", what, Py_TYPE(o)->tp_name);
    return false;
}

// Whether `o` is a ctypes array of `element`, or a ctypes pointer to it (`base`: ctypes.Array, ctypes._Pointer); -1 with an exception.
int is_of(PyObject* o, PyObject* base, PyObject* element) {
    const int is_base = PyObject_IsInstance(o, base);
    if (is_base <= 0) return is_base;
    PyObject* type = PyObject_GetAttrString((PyObject*)Py_TYPE(o), "_type_");
    if (type == nullptr) return -1;
    Py_DECREF(type);
    return type == element;
}

// The address that a ctypes pointer object holds.
bool pointed_to(PyObject* o, void*& p) {
    Buffer own;
    if (!own.take(o)) return false;
    p = *(void**)own.view.buf;
    return true;
}

// byref(x): x, if it is an instance of `type` and the reference is to its start; nullptr with an exception if not.
PyObject* referred(PyObject* o, PyObject* type, const char* what) {
    PyObject* target = PyObject_GetAttrString(o, "_obj");
    if (target == nullptr) return nullptr;
    Buffer own;
    PyObject* at = nullptr;
    const bool fits = PyObject_TypeCheck(target, (PyTypeObject*)type) != 0;
    if (fits && own.take(target)) {
        PyObject* address = PyObject_CallFunctionObjArgs(g_cast, o, g_void_p, nullptr);
        at = address != nullptr ? PyObject_GetAttrString(address, "value") : nullptr;
        Py_XDECREF(address);
    }
    const bool start = at != nullptr && at != Py_None && PyLong_AsVoidPtr(at) == own.view.buf;
    Py_XDECREF(at);
    if (!start) {
        if (!PyErr_Occurred()) {
            if (fits) PyErr_Format(PyExc_TypeError, "%s, not a reference with an offset", what);
            else PyErr_Format(PyExc_TypeError, "%s, not a reference to %s", what, Py_TYPE(target)->tp_name);
        }
        Py_DECREF(target);
        return nullptr;
    }
    return target;
}

// Scalars may come as objects of ctypes, of the parameter's own type.
PyObject* g_scalars[5] = {};      // c_int32, c_int64, c_uint32, c_uint64, c_float
const char* const SCALARS[5] = {"c_int32", "c_int64", "c_uint32", "c_uint64", "c_float"};
template <typename T>
PyObject* scalar_type() {
    return g_scalars[std::is_floating_point_v<T> ? 4 : 2 * std::is_unsigned_v<T> + (sizeof(T) == 8)];
}
template <typename Take>
bool unwrapped(PyObject* o, PyObject* type, const Take& take) {
    if (!PyObject_TypeCheck(o, (PyTypeObject*)type)) return take(o);
    PyObject* v = PyObject_GetAttrString(o, "value");
    if (v == nullptr) return false;
    const bool ok = take(v);
    Py_DECREF(v);
    return ok;
}

// What a function is bound to, in a capsule that the function object holds.
struct Bound {
    void* fn;
    PyObject* stream;             // the ctypes structure that stands for sp_philox_t
    const char* name;
    PyObject* function = nullptr; // the function object itself: what the tape records
    void* more = nullptr;         // a second entry point, for the functions that need one
    Bound(void* fn, PyObject* stream, const char* name) : fn(fn), stream(Py_NewRef(stream)), name(name) {}
    Bound(const Bound&) = delete;
    ~Bound() { Py_DECREF(stream); }
};

// HOST_INTS: of an entry point whose const int32_t* are host arrays.  Those that take arrays of addresses take the widths of a stack
// beside them; everywhere else a const int32_t* is device memory.
template <typename T, bool HOST_INTS, typename = void>
struct Arg;

template <typename T, bool HOST_INTS>
struct Arg<T, HOST_INTS, std::enable_if_t<std::is_integral_v<T>>> {
    T value = 0;
    bool load(PyObject* o, const Bound&) {
        unsigned long long v = 0;
        if (PyLong_Check(o) ? !as_integer(o, v) : !unwrapped(o, scalar_type<T>(), [&](PyObject* x) { return as_integer(x, v); })) return false;
        value = (T)v;
        return true;
    }
};

template <typename T, bool HOST_INTS>
struct Arg<T, HOST_INTS, std::enable_if_t<std::is_floating_point_v<T>>> {
    T value = 0;
    bool load(PyObject* o, const Bound&) {
        double v = 0;
        auto number = [&](PyObject* x) {
            v = PyFloat_AsDouble(x);
            return !(v == -1.0 && PyErr_Occurred());
        };
        if (PyFloat_Check(o) ? !number(o) : !unwrapped(o, scalar_type<T>(), number)) return false;
        value = (T)v;
        return true;
    }
};

// Device memory: an address, or a ctypes pointer that holds one.
template <typename T, bool HOST_INTS>
struct Arg<T*, HOST_INTS, std::enable_if_t<!std::is_pointer_v<std::remove_const_t<T>> && !std::is_same_v<T, const sp_philox_t> &&
                                           !(HOST_INTS && std::is_same_v<T, const int32_t>)>> {
    T* value = nullptr;
    bool load(PyObject* o, const Bound&) {
        void* p = nullptr;
        if (o != Py_None && !PyLong_Check(o)) {
            const int is_pointer = PyObject_IsInstance(o, g_pointer);
            if (is_pointer < 0 || (is_pointer > 0 ? !pointed_to(o, p) : !as_address(o, p))) return false;
        } else if (!as_address(o, p)) {
            return false;
        }
        value = (T*)p;
        return true;
    }
};

// A host array of addresses or of 32-bit integers: a list, a tuple, or of ctypes an array of such elements, one of them by reference or a
// pointer to them.  Elements are copied, zeros behind them, so that what reads further than was given -- a stack has eight layers at
// most -- finds zeros; only longer arrays, and what a pointer points to, are read in place.
template <typename T, bool HOST_INTS>
struct Arg<T*, HOST_INTS, std::enable_if_t<std::is_pointer_v<std::remove_const_t<T>> || (HOST_INTS && std::is_same_v<T, const int32_t>)>> {
    typedef std::remove_const_t<T> Element;
    static constexpr bool ADDRESSES = std::is_pointer_v<Element>;
    T* value = nullptr;
    Element few[MOST] = {};
    std::unique_ptr<Element[]> many;
    Buffer buffer;

    bool list(PyObject* o) {
        const Py_ssize_t n = PySequence_Fast_GET_SIZE(o);
        Element* elements = few;
        if (n > MOST) {
            many.reset(new (std::nothrow) Element[n]);
            elements = many.get();
            if (elements == nullptr) {
                PyErr_NoMemory();
                return false;
            }
        }
        for (Py_ssize_t i = 0; i < n; ++i) {
            if (i >= PySequence_Fast_GET_SIZE(o)) {        // (an element's __index__ may shorten the list)
                PyErr_SetString(PyExc_RuntimeError, "a list of arguments changed its size");
                return false;
            }
            PyObject* e = Py_NewRef(PySequence_Fast_GET_ITEM(o, i));
            bool ok;
            if constexpr (ADDRESSES) {
                void* p = nullptr;
                ok = as_address(e, p);
                elements[i] = (Element)p;
            } else {
                unsigned long long v = 0;
                ok = as_integer(e, v);
                elements[i] = (Element)v;
            }
            Py_DECREF(e);
            if (!ok) return false;
        }
        value = elements;
        return true;
    }
    bool memory(PyObject* o) {                             // of an array, or of one element
        if (!buffer.take(o)) return false;
        const size_t n = (size_t)buffer.view.len / sizeof(Element);
        if (n <= (size_t)MOST) memcpy(few, buffer.view.buf, n * sizeof(Element));
        value = n <= (size_t)MOST ? few : (T*)buffer.view.buf;
        return true;
    }
    bool load(PyObject* o, const Bound&) {
        if (PyTuple_Check(o) || PyList_Check(o)) return list(o);
        if (o == Py_None) return true;
        PyObject* const type = ADDRESSES ? g_void_p : g_int32;
        const char* const what = ADDRESSES ? "an array of addresses is None, a list, a tuple or of c_void_p" : "an array of integers is None, a list, a tuple or of c_int32";
        const int is_array = is_of(o, g_array, type);
        if (is_array != 0) return is_array > 0 && memory(o);
        const int is_pointer = is_of(o, g_pointer, type);
        if (is_pointer != 0) {
            void* p = nullptr;
            if (is_pointer < 0 || !pointed_to(o, p)) return false;
            value = (T*)p;
            return true;
        }
        if ((PyObject*)Py_TYPE(o) == g_byref) {
            PyObject* target = referred(o, type, what);
            if (target == nullptr) return false;
            const bool ok = memory(target);
            Py_DECREF(target);
            return ok;
        }
        return refuse(o, what);
    }
};

// The state of a random stream, a host structure: the structure, a reference or a ctypes pointer to it, or an array of them.
template <bool HOST_INTS>
struct Arg<const sp_philox_t*, HOST_INTS> {
    const sp_philox_t* value = nullptr;
    Buffer buffer;
    bool memory(PyObject* o) {
        if (!buffer.take(o)) return false;
        if ((size_t)buffer.view.len < sizeof(sp_philox_t)) return refuse(o, "a random stream needs a whole PhiloxConfig");
        value = (const sp_philox_t*)buffer.view.buf;
        return true;
    }
    bool load(PyObject* o, const Bound& bound) {
        if (o == Py_None) return true;
        if (PyObject_TypeCheck(o, (PyTypeObject*)bound.stream)) return memory(o);
        const char* const what = "a random stream is None or a PhiloxConfig";
        if ((PyObject*)Py_TYPE(o) == g_byref) {
            PyObject* target = referred(o, bound.stream, what);
            if (target == nullptr) return false;
            const bool ok = memory(target);
            Py_DECREF(target);
            return ok;
        }
        const int is_array = is_of(o, g_array, bound.stream);
        if (is_array != 0) return is_array > 0 && memory(o);
        const int is_pointer = is_of(o, g_pointer, bound.stream);
        if (is_pointer == 0) return refuse(o, what);
        void* p = nullptr;
        if (is_pointer < 0 || !pointed_to(o, p)) return false;
        value = (const sp_philox_t*)p;
        return true;
    }
};

// What does not fit is reported as ctypes reports it; as a TypeError, too.
PyObject* g_argument_error = nullptr;
void refuse_argument(int number) {
    if (!PyErr_ExceptionMatches(PyExc_TypeError)) return;
    PyObject *type, *text, *trace;
    PyErr_Fetch(&type, &text, &trace);
    PyErr_Format(g_argument_error, "argument %d: %S", number, text != nullptr ? text : Py_None);
    Py_XDECREF(type);
    Py_XDECREF(text);
    Py_XDECREF(trace);
}

// ---- one function per entry point ----
template <typename F>
struct Entry;
template <typename... A>
struct Entry<int(A...)> {
    static constexpr bool HOST_INTS = ((std::is_pointer_v<A> && std::is_pointer_v<std::remove_const_t<std::remove_pointer_t<A>>>) || ...);

    template <size_t... I>
    static PyObject* run(const Bound& bound, PyObject* const* given, std::index_sequence<I...>) {
        std::tuple<Arg<A, HOST_INTS>...> args;
        if (int at = 0; !((++at, std::get<I>(args).load(given[I], bound)) && ...)) {
            refuse_argument(at);
            return nullptr;
        }
        int (*const fn)(A...) = (int (*)(A...))bound.fn;
        int rc = 0;
        Py_BEGIN_ALLOW_THREADS
        rc = fn(std::get<I>(args).value...);
        Py_END_ALLOW_THREADS
        if (rc == 0 && g_calls != nullptr) {               // the last argument is the stream
            PyObject* kept = PyTuple_New(sizeof...(A) - 1);
            if (kept == nullptr) return nullptr;
            for (size_t i = 0; i + 1 < sizeof...(A); ++i) {
                Py_INCREF(given[i]);
                PyTuple_SET_ITEM(kept, i, given[i]);
            }
            PyObject* call = PyTuple_Pack(2, bound.function, kept);
            Py_DECREF(kept);
            if (call == nullptr) return nullptr;
            const int failed = PyList_Append(g_calls, call);
            Py_DECREF(call);
            if (failed != 0) return nullptr;
        }
        return PyLong_FromLong(rc);
    }
    static PyObject* call(PyObject* capsule, PyObject* const* given, Py_ssize_t n) {
        const Bound* const bound = (const Bound*)PyCapsule_GetPointer(capsule, nullptr);
        if (bound == nullptr) return nullptr;
        if (n != (Py_ssize_t)sizeof...(A)) return PyErr_Format(PyExc_TypeError, "%s takes %zu arguments (%zd given)", bound->name, sizeof...(A), n);
        return run(*bound, given, std::index_sequence_for<A...>{});
    }
};

#define SP_LAUNCHES(X)                                                                                                        \
    X(sp_gemm_abt) X(sp_gemm_abt_batched) X(sp_row_ops) X(sp_row_map_f32) X(sp_row_map_i32) X(sp_row_sample) X(sp_philox_uniforms) \
    X(sp_row_get_prob) X(sp_cem_resample) X(sp_cem_resample_philox) X(sp_row_reduce_f32) X(sp_cem_update_mask) X(sp_row_binarize)   \
    X(sp_map_f32) X(sp_reduce_sum) X(sp_reduce) X(sp_row_l1_normalize) X(sp_reduce_sum_static) X(sp_transpose_inner_b32)            \
    X(sp_mlp_forward) X(sp_mlp_pack_weights) X(sp_mlp_forward_packed) X(sp_mlp_forward_ensemble) X(sp_ensemble_binarize)            \
    X(sp_stack_forward_f32) X(sp_layer_norm) X(sp_layer_norm_backward) X(sp_logits_penalize) X(sp_quantize_blocks) X(sp_gemm_abt_scaled) \
    X(sp_gemm_abt_gated) X(sp_gemm_abt_gated_backward) X(sp_token_log_probs) X(sp_token_log_probs_backward)

// ---- whole calls: checks, outputs and launch of the operators that a decoding step makes of one token at a time ----
//
// As the Python functions of the same names (ml.matmul, ml.primitives) do it, for calls that are right and ordinary: contiguous tensors on the current
// device, nothing recorded.  None for any other call, and where the library refuses: the Python function then goes its own way, and raises what there
// is to raise.  (us a call with the queue kept full, in Python / here: a norm 7.4 / 4.1, a product
// of one row 8.1 / 4.0, a row in 8 bits 9.7 / 5.6, the logits of one row, two launches, 18.7 / 9.7; a launch alone takes 3 to 4.)
PyObject* g_raw_stream = nullptr; // torch's query of the current stream

struct Unusual {};                // thrown to leave a call to Python

struct Whole {
    int device;
    void* stream;
    std::vector<at::Tensor> out;

    static const at::Tensor* given(PyObject* o) {          // nullptr for None
        if (o == Py_None) return nullptr;
        if (!THPVariable_Check(o)) throw Unusual();
        return &THPVariable_Unpack(o);
    }
    // The first tensor of a call, whose device has to be the current one.
    explicit Whole(const at::Tensor* x) {
        if (g_calls != nullptr || g_raw_stream == nullptr || x == nullptr || !x->is_cuda()) throw Unusual();
        device = x->get_device();
        if (c10::impl::VirtualGuardImpl(c10::DeviceType::CUDA).getDevice().index() != device) throw Unusual();
        PyObject* index = PyLong_FromLong(device);
        PyObject* raw = index != nullptr ? PyObject_CallOneArg(g_raw_stream, index) : nullptr;
        Py_XDECREF(index);
        stream = raw != nullptr ? PyLong_AsVoidPtr(raw) : nullptr;
        Py_XDECREF(raw);
        if (PyErr_Occurred()) throw Unusual();
    }
    void* at(const at::Tensor* t, at::ScalarType type) const {     // the address, nullptr for None
        if (t == nullptr) return nullptr;
        if (t->scalar_type() != type || !t->is_cuda() || t->get_device() != device || !t->is_contiguous()) throw Unusual();
        return t->data_ptr();
    }
    void* make(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
        out.push_back(at::empty(sizes, like.options().dtype(type)));
        return out.back().data_ptr();
    }
    // The first `n` outputs as a tuple, or the only one.
    PyObject* result(size_t n) {
        if (n == 1) return THPVariable_Wrap(std::move(out[0]));
        PyObject* all = PyTuple_New((Py_ssize_t)n);
        if (all == nullptr) return nullptr;
        for (size_t i = 0; i < n; ++i) {
            PyObject* one = THPVariable_Wrap(std::move(out[i]));
            if (one == nullptr) {
                Py_DECREF(all);
                return nullptr;
            }
            PyTuple_SET_ITEM(all, (Py_ssize_t)i, one);
        }
        return all;
    }
};

int code_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return SP_F32;
        case at::kHalf: return SP_F16;
        case at::kBFloat16: return SP_BF16;
        default: throw Unusual();
    }
}
int f8_code_of(at::ScalarType t) {
    if (t == at::kFloat8_e4m3fn) return SP_F8_E4M3;
    if (t == at::kFloat8_e5m2) return SP_F8_E5M2;
    throw Unusual();
}
bool yes(PyObject* o) { return o == Py_True ? true : o == Py_False ? false : throw Unusual(); }
double number(PyObject* o) { return PyFloat_Check(o) ? PyFloat_AS_DOUBLE(o) : throw Unusual(); }
at::ScalarType type_of(PyObject* o) { return THPDtype_Check(o) ? ((THPDtype*)o)->scalar_type : throw Unusual(); }
void need(bool ok) {
    if (!ok) throw Unusual();
}
int64_t blocks_of(int64_t n) { return (n + 127) / 128; }

// f(bound, arguments), None for what it throws.
template <typename F>
PyObject* whole(PyObject* capsule, Py_ssize_t n, Py_ssize_t want, const F& f) {
    const Bound* const bound = (const Bound*)PyCapsule_GetPointer(capsule, nullptr);
    if (bound == nullptr) return nullptr;
    if (n != want) return PyErr_Format(PyExc_TypeError, "%zd arguments (%zd given)", want, n);
    try {
        return f(*bound);
    } catch (const Unusual&) {
    } catch (const std::exception&) {
    }
    PyErr_Clear();
    Py_RETURN_NONE;
}
template <typename F, typename... A>
void launch(F* fn, A... args) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fn(args...);
    Py_END_ALLOW_THREADS
    need(rc == 0);
}

// (x, weight, bias, eps, want_stats)
PyObject* whole_layer_norm(PyObject* capsule, PyObject* const* a, Py_ssize_t n) {
    return whole(capsule, n, 5, [&](const Bound& bound) {
        const at::Tensor *x = Whole::given(a[0]), *weight = Whole::given(a[1]), *bias = Whole::given(a[2]);
        Whole call(x);
        need(x->dim() >= 2 && x->numel() > 0);
        const int64_t cols = x->size(-1), rows = x->numel() / cols;
        const at::ScalarType type = x->scalar_type(), weights = weight != nullptr ? weight->scalar_type() : bias != nullptr ? bias->scalar_type() : at::kFloat;
        const int code = code_of(type);
        need(weights == at::kFloat || weights == type);
        for (const at::Tensor* t : {weight, bias}) need(t == nullptr || (t->dim() == 1 && t->size(0) == cols));
        const bool stats = yes(a[4]);
        const double eps = number(a[3]);
        void *from = call.at(x, type), *w = call.at(weight, weights), *b = call.at(bias, weights), *y = call.make(x->sizes(), type, *x), *mean = nullptr, *rstd = nullptr;
        if (stats) {
            const auto lead = x->sizes().slice(0, x->dim() - 1);
            mean = call.make(lead, at::kFloat, *x);
            rstd = call.make(lead, at::kFloat, *x);
        }
        launch((decltype(&sp_layer_norm))bound.fn, code, code_of(weights), from, w, b, y, (float*)mean, (float*)rstd, rows, cols, (float)eps, call.stream);
        return call.result(stats ? 3 : 1);
    });
}

// (dy, x, mean, rstd, weight)
PyObject* whole_layer_norm_backward(PyObject* capsule, PyObject* const* a, Py_ssize_t n) {
    return whole(capsule, n, 5, [&](const Bound& bound) {
        const at::Tensor *dy = Whole::given(a[0]), *x = Whole::given(a[1]), *mean = Whole::given(a[2]), *rstd = Whole::given(a[3]), *weight = Whole::given(a[4]);
        Whole call(x);
        need(bound.more != nullptr && dy != nullptr && mean != nullptr && rstd != nullptr && x->dim() >= 2 && x->numel() > 0 && dy->sizes() == x->sizes());
        const int64_t cols = x->size(-1), rows = x->numel() / cols;
        const auto lead = x->sizes().slice(0, x->dim() - 1);
        need(mean->sizes() == lead && rstd->sizes() == lead);
        const at::ScalarType type = x->scalar_type(), weights = weight != nullptr ? weight->scalar_type() : at::kFloat;
        const int code = code_of(type);
        need((weights == at::kFloat || weights == type) && (weight == nullptr || (weight->dim() == 1 && weight->size(0) == cols)));
        void *g = call.at(dy, type), *from = call.at(x, type), *m = call.at(mean, at::kFloat), *r = call.at(rstd, at::kFloat), *w = call.at(weight, weights);
        void *dx = call.make(x->sizes(), type, *x), *dw = call.make({cols}, at::kFloat, *x), *db = call.make({cols}, at::kFloat, *x);
        const int64_t bytes = ((decltype(&sp_layer_norm_backward_workspace_bytes))bound.more)(rows, cols);
        void* workspace = call.make({bytes > 16 ? bytes : 16}, at::kByte, *x);
        launch((decltype(&sp_layer_norm_backward))bound.fn, code, code_of(weights), g, from, (const float*)m, (const float*)r, w, dx, (float*)dw, (float*)db, rows,
               cols, workspace, bytes, call.stream);
        return call.result(3);
    });
}

// (x, rows of a block, type, plain, transposed)
PyObject* whole_quantize_blocks(PyObject* capsule, PyObject* const* a, Py_ssize_t n) {
    return whole(capsule, n, 5, [&](const Bound& bound) {
        const at::Tensor* x = Whole::given(a[0]);
        Whole call(x);
        need(x->dim() == 2 && x->numel() > 0 && PyLong_Check(a[1]));
        const int64_t size[2] = {x->size(0), x->size(1)};
        const long high = PyLong_AsLong(a[1]);
        const at::ScalarType type = x->scalar_type(), f8 = type_of(a[2]);
        const int code = code_of(type), f8_code = f8_code_of(f8);
        void *from = call.at(x, type), *to[4] = {};
        for (int form = 0; form < 2; ++form) {
            if (!yes(a[3 + form])) continue;
            const int64_t r = size[form], c = size[1 - form];
            to[2 * form] = call.make({r, (c + 15) / 16 * 16}, f8, *x);
            to[2 * form + 1] = call.make({high == 1 ? r : blocks_of(r), blocks_of(c)}, at::kFloat, *x);
        }
        launch((decltype(&sp_quantize_blocks))bound.fn, code, f8_code, (int32_t)high, from, to[0], (float*)to[1], to[2], (float*)to[3], size[0], size[1], call.stream);
        return call.result(call.out.size());
    });
}

// (a, scale_a, b, scale_b, bias, relu, type of C)
PyObject* whole_matmul_abt_scaled(PyObject* capsule, PyObject* const* o, Py_ssize_t n) {
    return whole(capsule, n, 7, [&](const Bound& bound) {
        const at::Tensor *a = Whole::given(o[0]), *sa = Whole::given(o[1]), *b = Whole::given(o[2]), *sb = Whole::given(o[3]), *bias = Whole::given(o[4]);
        Whole call(a);
        for (const at::Tensor* t : {a, sa, b, sb}) need(t != nullptr && t->dim() == 2 && t->numel() > 0);
        const int64_t m = a->size(0), k = a->size(1), rows_b = b->size(0), kb = blocks_of(k), high = sb->size(0) == rows_b ? 1 : 128;
        need(b->size(1) == k && sa->size(0) == m && sa->size(1) == kb && sb->size(1) == kb && (high == 1 || sb->size(0) == blocks_of(rows_b)));
        need(bias == nullptr || (bias->dim() == 1 && bias->size(0) == rows_b));
        const at::ScalarType out = type_of(o[6]);
        const int fa = f8_code_of(a->scalar_type()), fb = f8_code_of(b->scalar_type()), code = code_of(out);
        const bool relu = yes(o[5]);
        void *pa = call.at(a, a->scalar_type()), *psa = call.at(sa, at::kFloat), *pb = call.at(b, b->scalar_type()), *psb = call.at(sb, at::kFloat), *pbias = call.at(bias, at::kFloat);
        void* c = call.make({m, rows_b}, out, *a);
        launch((decltype(&sp_gemm_abt_scaled))bound.fn, fa, fb, code, pa, (const float*)psa, pb, (const float*)psb, (int32_t)high, c, (const float*)pbias, m, rows_b, k, 0.f,
               relu ? SP_GEMM_RELU : 0u, call.stream);
        return call.result(1);
    });
}

// (logits, tokens, lengths, prompt_lengths, repetition, presence, frequency, temperature, bias_ids, bias, mask, want_token)
PyObject* whole_penalize_logits(PyObject* capsule, PyObject* const* a, Py_ssize_t n) {
    return whole(capsule, n, 12, [&](const Bound& bound) {
        const at::Tensor *x = Whole::given(a[0]), *tokens = Whole::given(a[1]), *ids = Whole::given(a[8]), *bias = Whole::given(a[9]), *mask = Whole::given(a[10]);
        Whole call(x);
        need(bound.more != nullptr && x->dim() >= 2 && x->numel() > 0);
        const int64_t cols = x->size(-1), rows = x->numel() / cols, words = (cols + 31) / 32;
        const auto lead = x->sizes().slice(0, x->dim() - 1);
        auto rows_of = [&](const at::Tensor* t) { return t->dim() == x->dim() && t->sizes().slice(0, t->dim() - 1) == lead; };
        const at::Tensor* each[6];                         // one entry per row
        void* at_each[6];
        for (int i = 0; i < 6; ++i) {
            each[i] = Whole::given(a[2 + i]);
            need(each[i] == nullptr || each[i]->sizes() == lead);
            at_each[i] = call.at(each[i], i < 2 ? at::kInt : at::kFloat);
        }
        need(tokens != nullptr ? rows_of(tokens) : each[0] == nullptr && each[1] == nullptr);
        need((ids == nullptr) == (bias == nullptr) && (bias == nullptr || (rows_of(bias) && ids->sizes() == bias->sizes())));
        need(mask == nullptr || (mask->dim() > 0 && mask->size(-1) == words && (mask->numel() == words || mask->sizes().slice(0, mask->dim() - 1) == lead)));
        const int64_t history = tokens != nullptr ? tokens->size(-1) : 0, n_bias = bias != nullptr ? bias->size(-1) : 0;
        const at::ScalarType type = x->scalar_type();
        const int code = code_of(type);
        const bool want_token = yes(a[11]);
        void *from = call.at(x, type), *history_at = call.at(tokens, at::kInt), *ids_at = call.at(ids, at::kInt), *bias_at = call.at(bias, at::kFloat), *mask_at = call.at(mask, at::kInt);
        void *out = call.make(x->sizes(), at::kFloat, *x), *token = nullptr, *workspace = nullptr;
        int64_t bytes = 0;
        if (want_token) {
            token = call.make(lead, at::kInt, *x);
            bytes = ((decltype(&sp_logits_penalize_workspace_bytes))bound.more)(rows, cols);
            workspace = call.make({bytes}, at::kByte, *x);
        }
        launch((decltype(&sp_logits_penalize))bound.fn, code, from, (float*)out, (int32_t*)token, (const int32_t*)(history > 0 ? history_at : nullptr), (const int32_t*)at_each[0],
               (const int32_t*)at_each[1], history, (const float*)at_each[2], (const float*)at_each[3], (const float*)at_each[4], (const float*)at_each[5],
               (const int32_t*)(n_bias > 0 ? ids_at : nullptr), (const float*)(n_bias > 0 ? bias_at : nullptr), n_bias, (const int32_t*)mask_at,
               mask != nullptr ? mask->numel() / words : (int64_t)0, rows, cols, workspace, bytes, call.stream);
        return call.result(want_token ? 2 : 1);
    });
}

// (a, b_gate, b_up, activation, type that is kept)
PyObject* whole_matmul_abt_gated(PyObject* capsule, PyObject* const* o, Py_ssize_t n) {
    return whole(capsule, n, 5, [&](const Bound& bound) {
        const at::Tensor *a = Whole::given(o[0]), *gate = Whole::given(o[1]), *up = Whole::given(o[2]);
        Whole call(a);
        for (const at::Tensor* t : {a, gate, up}) need(t != nullptr && t->dim() == 2 && t->numel() > 0);
        need(gate->sizes() == up->sizes() && gate->size(1) == a->size(1) && PyLong_Check(o[3]));
        const int64_t m = a->size(0), k = a->size(1), cols = gate->size(0);
        const at::ScalarType type = a->scalar_type();
        const int code = code_of(type), activation = (int)PyLong_AsLong(o[3]);
        const bool keeps = o[4] != Py_None, f8 = keeps && type_of(o[4]) == at::kFloat8_e4m3fn;
        need(!keeps || f8 || type_of(o[4]) == type);
        void *pa = call.at(a, type), *pg = call.at(gate, type), *pu = call.at(up, type), *c = call.make({m, cols}, type, *a), *kept[4] = {};
        for (int i = 0; keeps && i < 2; ++i) {
            kept[2 * i] = call.make({m, f8 ? (cols + 15) / 16 * 16 : cols}, f8 ? at::kFloat8_e4m3fn : type, *a);
            if (f8) kept[2 * i + 1] = call.make({m, blocks_of(cols)}, at::kFloat, *a);
        }
        launch((decltype(&sp_gemm_abt_gated))bound.fn, code, activation, pa, pg, pu, c, f8 ? (int)SP_F8_E4M3 : code, kept[0], (float*)kept[1], kept[2], (float*)kept[3], m, cols, k,
               call.stream);
        if (!keeps) return call.result(1);
        PyObject* first = THPVariable_Wrap(std::move(call.out[0]));
        if (first == nullptr) return first;
        call.out.erase(call.out.begin());
        PyObject *rest = call.result(call.out.size()), *both = rest != nullptr ? PyTuple_Pack(2, first, rest) : nullptr;
        Py_DECREF(first);
        Py_XDECREF(rest);
        return both;
    });
}

// (dc, a, b_gate, b_up, gate, its scales, up, its scales, activation)
PyObject* whole_matmul_abt_gated_backward(PyObject* capsule, PyObject* const* o, Py_ssize_t n) {
    return whole(capsule, n, 9, [&](const Bound& bound) {
        const at::Tensor *dc = Whole::given(o[0]), *a = Whole::given(o[1]), *gate = Whole::given(o[2]), *up = Whole::given(o[3]);
        const at::Tensor* kept[4] = {Whole::given(o[4]), Whole::given(o[5]), Whole::given(o[6]), Whole::given(o[7])};
        Whole call(a);
        for (const at::Tensor* t : {dc, a, gate, up, kept[0], kept[2]}) need(t != nullptr && t->dim() == 2 && t->numel() > 0);
        need(bound.more != nullptr && gate->sizes() == up->sizes() && gate->size(1) == a->size(1) && PyLong_Check(o[8]));
        const int64_t m = a->size(0), k = a->size(1), cols = gate->size(0);
        const at::ScalarType type = a->scalar_type(), as = kept[0]->scalar_type();
        const bool f8 = as == at::kFloat8_e4m3fn;
        const int code = code_of(type), activation = (int)PyLong_AsLong(o[8]);
        need(dc->size(0) == m && dc->size(1) == cols && (f8 || as == type) && (kept[1] != nullptr) == f8 && (kept[3] != nullptr) == f8);
        for (int i = 0; i < 4; ++i) {
            const int64_t wide = i % 2 != 0 ? blocks_of(cols) : f8 ? (cols + 15) / 16 * 16 : cols;
            need(kept[i] == nullptr || (kept[i]->dim() == 2 && kept[i]->size(0) == m && kept[i]->size(1) == wide));
        }
        void *pd = call.at(dc, type), *pa = call.at(a, type), *pg = call.at(gate, type), *pu = call.at(up, type);
        void *k0 = call.at(kept[0], as), *k1 = call.at(kept[1], at::kFloat), *k2 = call.at(kept[2], as), *k3 = call.at(kept[3], at::kFloat);
        void *da = call.make({m, k}, type, *a), *dg = call.make({cols, k}, type, *a), *du = call.make({cols, k}, type, *a);
        const int64_t bytes = ((decltype(&sp_gemm_abt_gated_backward_workspace_bytes))bound.more)(code, m, cols, k);
        void* workspace = call.make({bytes}, at::kByte, *a);
        launch((decltype(&sp_gemm_abt_gated_backward))bound.fn, code, activation, pd, pa, pg, pu, f8 ? (int)SP_F8_E4M3 : code, k0, (const float*)k1, k2, (const float*)k3, da, dg, du,
               m, cols, k, workspace, bytes, call.stream);
        return call.result(3);
    });
}

// (logits, tokens, top, want_entropy, want_lse)
PyObject* whole_token_log_probs(PyObject* capsule, PyObject* const* a, Py_ssize_t n) {
    return whole(capsule, n, 5, [&](const Bound& bound) {
        const at::Tensor *x = Whole::given(a[0]), *tokens = Whole::given(a[1]);
        Whole call(x);
        need(bound.more != nullptr && tokens != nullptr && x->dim() >= 2 && x->numel() > 0 && PyLong_Check(a[2]));
        const int64_t cols = x->size(-1), rows = x->numel() / cols;
        const auto lead = x->sizes().slice(0, x->dim() - 1);
        const long top = PyLong_AsLong(a[2]);
        need(tokens->sizes() == lead && top >= 0 && top <= 32);
        const at::ScalarType type = x->scalar_type();
        const int code = code_of(type);
        const bool want_entropy = yes(a[3]), want_lse = yes(a[4]);
        void *from = call.at(x, type), *ids = call.at(tokens, at::kInt), *logp = call.make(lead, at::kFloat, *x), *top_logp = nullptr, *top_ids = nullptr, *workspace = nullptr;
        void* entropy = want_entropy ? call.make(lead, at::kFloat, *x) : nullptr;
        void* lse = want_lse ? call.make(lead, at::kFloat, *x) : nullptr;
        if (top > 0) {
            std::vector<int64_t> each(lead.begin(), lead.end());
            each.push_back(top);
            top_logp = call.make(each, at::kFloat, *x);
            top_ids = call.make(each, at::kInt, *x);
        }
        const size_t results = call.out.size();
        const int64_t bytes = ((decltype(&sp_token_log_probs_workspace_bytes))bound.more)(rows, cols, (int32_t)top);
        if (bytes > 0) workspace = call.make({bytes}, at::kByte, *x);
        launch((decltype(&sp_token_log_probs))bound.fn, code, from, (const int32_t*)ids, (float*)logp, (float*)entropy, (float*)lse, (int32_t)top, (float*)top_logp, (int32_t*)top_ids,
               rows, cols, workspace, bytes, call.stream);
        return call.result(results);
    });
}

// (d_log_probs, logits, tokens, lse, d_entropy, entropy, d_lse)
PyObject* whole_token_log_probs_backward(PyObject* capsule, PyObject* const* a, Py_ssize_t n) {
    return whole(capsule, n, 7, [&](const Bound& bound) {
        const at::Tensor *x = Whole::given(a[1]), *tokens = Whole::given(a[2]);
        Whole call(x);
        need(tokens != nullptr && x->dim() >= 2 && x->numel() > 0);
        const int64_t cols = x->size(-1), rows = x->numel() / cols;
        const auto lead = x->sizes().slice(0, x->dim() - 1);
        need(tokens->sizes() == lead);
        const int at_each[5] = {0, 3, 4, 5, 6};            // d_log_probs, lse, d_entropy, entropy, d_lse
        void* each[5];
        for (int i = 0; i < 5; ++i) {
            const at::Tensor* t = Whole::given(a[at_each[i]]);
            need(t == nullptr || t->sizes() == lead);
            each[i] = call.at(t, at::kFloat);
        }
        need(each[1] != nullptr);
        const at::ScalarType type = x->scalar_type();
        const int code = code_of(type);
        void *from = call.at(x, type), *ids = call.at(tokens, at::kInt), *dx = call.make(x->sizes(), type, *x);
        launch((decltype(&sp_token_log_probs_backward))bound.fn, code, from, (const int32_t*)ids, (const float*)each[1], (const float*)each[3], (const float*)each[0],
               (const float*)each[2], (const float*)each[4], dx, rows, cols, call.stream);
        return call.result(1);
    });
}

// (Python's name, the function, the entry point, another one it asks)
#define SP_WHOLE(X)                                                                                        \
    X(layer_norm, sp_layer_norm, nullptr)                                                                   \
    X(layer_norm_backward, sp_layer_norm_backward, "sp_layer_norm_backward_workspace_bytes")                  \
    X(quantize_blocks, sp_quantize_blocks, nullptr)                                                          \
    X(matmul_abt_scaled, sp_gemm_abt_scaled, nullptr)                                                        \
    X(penalize_logits, sp_logits_penalize, "sp_logits_penalize_workspace_bytes")                              \
    X(matmul_abt_gated, sp_gemm_abt_gated, nullptr)                                                          \
    X(matmul_abt_gated_backward, sp_gemm_abt_gated_backward, "sp_gemm_abt_gated_backward_workspace_bytes")    \
    X(token_log_probs, sp_token_log_probs, "sp_token_log_probs_workspace_bytes")                              \
    X(token_log_probs_backward, sp_token_log_probs_backward, nullptr)

// `as`: the name the function goes by; `other`: a second entry point for it, where the library has it.
bool bind_one(void* library, PyObject* stream, PyObject* functions, const char* name, PyCFunction call, PyMethodDef& def, const char* as, const char* other) {
    void* const fn = dlsym(library, name);
    void* const more = fn != nullptr && other != nullptr ? dlsym(library, other) : nullptr;
    if (fn == nullptr) {
        PyErr_Format(PyExc_RuntimeError, "the library has no %s", name);
        return false;
    }
    def = PyMethodDef{as, call, METH_FASTCALL, nullptr};
    Bound* const bound = new (std::nothrow) Bound(fn, stream, name);
    if (bound != nullptr) bound->more = more;
    if (bound == nullptr) {
        PyErr_NoMemory();
        return false;
    }
    PyObject* capsule = PyCapsule_New(bound, nullptr, [](PyObject* c) { delete (Bound*)PyCapsule_GetPointer(c, nullptr); });
    if (capsule == nullptr) {
        delete bound;
        return false;
    }
    PyObject* function = PyCFunction_New(&def, capsule);
    Py_DECREF(capsule);
    if (function == nullptr) return false;
    bound->function = function;                            // (borrowed: the function holds the capsule)
    const int failed = PyDict_SetItemString(functions, as, function);
    Py_DECREF(function);
    return failed == 0;
}

// bind(path, stream): a dict of the functions behind the library at `path`, which the process keeps; `stream`: the ctypes structure
// that stands for sp_philox_t in their calls.
PyObject* bind(PyObject*, PyObject* const* given, Py_ssize_t n) {
    if (n != 2 || !PyType_Check(given[1])) return PyErr_Format(PyExc_TypeError, "bind takes a path and a structure type");
    const char* p = PyUnicode_AsUTF8(given[0]);
    if (p == nullptr) return nullptr;
    PyObject* ctypes = PyImport_ImportModule("ctypes");
    if (ctypes == nullptr) return nullptr;
    auto get = [&](PyObject*& to, const char* name) { return to != nullptr || (to = PyObject_GetAttrString(ctypes, name)) != nullptr; };
    bool found = get(g_void_p, "c_void_p") && get(g_int32, "c_int32") && get(g_array, "Array") && get(g_pointer, "_Pointer") && get(g_cast, "cast");
    for (int i = 0; i < 5; ++i) found = found && get(g_scalars[i], SCALARS[i]);
    if (found && g_byref == nullptr) {
        PyObject* any = PyObject_CallMethod(ctypes, "c_int", nullptr);
        PyObject* ref = any != nullptr ? PyObject_CallMethod(ctypes, "byref", "O", any) : nullptr;
        if (ref != nullptr) g_byref = Py_NewRef((PyObject*)Py_TYPE(ref));
        Py_XDECREF(ref);
        Py_XDECREF(any);
        found = g_byref != nullptr;
    }
    if (found && g_argument_error == nullptr) {
        PyObject* of_ctypes = PyObject_GetAttrString(ctypes, "ArgumentError");
        PyObject* bases = of_ctypes != nullptr ? PyTuple_Pack(2, of_ctypes, PyExc_TypeError) : nullptr;
        g_argument_error = bases != nullptr ? PyErr_NewException("spiral_host.ArgumentError", bases, nullptr) : nullptr;
        Py_XDECREF(bases);
        Py_XDECREF(of_ctypes);
        found = g_argument_error != nullptr;
    }
    Py_DECREF(ctypes);
    if (!found) return nullptr;
    if (g_raw_stream == nullptr) {                         // (a torch without a GPU has none: no whole calls then)
        PyObject* torch_c = PyImport_ImportModule("torch._C");
        if (torch_c != nullptr) g_raw_stream = PyObject_GetAttrString(torch_c, "_cuda_getCurrentRawStream");
        Py_XDECREF(torch_c);
        PyErr_Clear();
    }
    void* library = dlopen(p, RTLD_NOW | RTLD_LOCAL);
    if (library == nullptr) return PyErr_Format(PyExc_RuntimeError, "%s", dlerror());
    PyObject* functions = PyDict_New();
    if (functions == nullptr) return nullptr;
    bool ok = true;
    enum {
#define SP_ID(name) ID_##name,
        SP_LAUNCHES(SP_ID)
#undef SP_ID
#define SP_ID(as, name, other) ID_whole_##as,
        SP_WHOLE(SP_ID) COUNT
#undef SP_ID
    };
    static PyMethodDef defs[COUNT];
#define SP_BIND(name) ok = ok && bind_one(library, given[1], functions, #name, (PyCFunction)(void (*)(void))&Entry<std::remove_pointer_t<decltype(&::name)>>::call, defs[ID_##name], #name, nullptr);
    SP_LAUNCHES(SP_BIND)
#undef SP_BIND
#define SP_BIND(as, name, other) ok = ok && bind_one(library, given[1], functions, #name, (PyCFunction)(void (*)(void))&whole_##as, defs[ID_whole_##as], "whole_" #as, other);
    SP_WHOLE(SP_BIND)
#undef SP_BIND
    if (!ok) {
        Py_DECREF(functions);
        return nullptr;
    }
    return functions;
}

// ptr(t, dtype=None, name="tensor"): the address of a contiguous ROCm tensor, None for None.
PyObject* ptr(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* keywords) {
    PyObject *t = n > 0 ? args[0] : nullptr, *dtype = n > 1 ? args[1] : Py_None, *name = n > 2 ? args[2] : nullptr;
    if (n > 3) return PyErr_Format(PyExc_TypeError, "ptr takes at most 3 arguments");
    for (Py_ssize_t i = 0; keywords != nullptr && i < PyTuple_GET_SIZE(keywords); ++i) {
        PyObject* key = PyTuple_GET_ITEM(keywords, i);
        if (PyUnicode_CompareWithASCIIString(key, "name") == 0) name = args[n + i];
        else if (PyUnicode_CompareWithASCIIString(key, "dtype") == 0) dtype = args[n + i];
        else if (PyUnicode_CompareWithASCIIString(key, "t") == 0) t = args[n + i];
        else return PyErr_Format(PyExc_TypeError, "ptr has no argument %S", key);
    }
    if (t == nullptr) return PyErr_Format(PyExc_TypeError, "ptr needs a tensor");
    if (t == Py_None) Py_RETURN_NONE;
    PyObject* const named = name;
    auto raise = [&](PyObject* type, const char* text) -> PyObject* {
        if (named != nullptr) return PyErr_Format(type, "%S %s", named, text);
        return PyErr_Format(type, "tensor %s", text);
    };
    try {
        if (!THPVariable_Check(t)) return raise(PyExc_TypeError, "must be a torch.Tensor");
        const at::Tensor& x = THPVariable_Unpack(t);
        if (!x.is_cuda()) return raise(PyExc_ValueError, ("must live on the GPU (got " + x.device().str() + ")").c_str());
        if (!x.is_contiguous()) return raise(PyExc_ValueError, "must be contiguous (row-major, innermost stride 1)");
        if (dtype != Py_None) {
            if (!THPDtype_Check(dtype)) return PyErr_Format(PyExc_TypeError, "dtype must be a torch.dtype");
            if (((THPDtype*)dtype)->scalar_type != x.scalar_type()) {
                PyObject* got = PyObject_GetAttrString(t, "dtype");
                if (got == nullptr) return nullptr;
                if (named != nullptr) PyErr_Format(PyExc_TypeError, "%S must have dtype %S, got %S", named, dtype, got);
                else PyErr_Format(PyExc_TypeError, "tensor must have dtype %S, got %S", dtype, got);
                Py_DECREF(got);
                return nullptr;
            }
        }
        void* const at = x.data_ptr();
        if (g_keep != nullptr && PyList_Append(g_keep, t) != 0) return nullptr;
        return PyLong_FromVoidPtr(at);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// tape(calls, keep): launches and tensors go into these lists from now on; tape(None, None): no longer.
PyObject* tape(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 2 || !((args[0] == Py_None && args[1] == Py_None) || (PyList_Check(args[0]) && PyList_Check(args[1]))))
        return PyErr_Format(PyExc_TypeError, "tape takes two lists, or None twice");
    PyObject *calls = args[0] == Py_None ? nullptr : args[0], *keep = args[1] == Py_None ? nullptr : args[1];
    Py_XINCREF(calls);
    Py_XINCREF(keep);
    std::swap(calls, g_calls);
    std::swap(keep, g_keep);
    Py_XDECREF(calls);
    Py_XDECREF(keep);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, nullptr},
                         {"ptr", (PyCFunction)(void (*)(void))ptr, METH_FASTCALL | METH_KEYWORDS, nullptr},
                         {"tape", (PyCFunction)(void (*)(void))tape, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "spiral_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_spiral_host() { return PyModule_Create(&module); }
