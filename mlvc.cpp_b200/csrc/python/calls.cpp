// Microscaled calls from Python: describes the operands of a call (any objects
// with data_ptr(), and for matrices shape, stride() and dtype) and makes it.
//
// A call on few rows takes a few microseconds on the device, and describing its
// operands attribute by attribute in Python took as long: two streams' rows
// written to a cache and read back 14.6 us a pass (here 11.4), a linear layer on
// one row 8.4 (7.1).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "mlvc_b200.h"

namespace {

struct Library {
    decltype(&mlvc_b200_mx_quantise) quantise;
    decltype(&mlvc_b200_mx_dequantise) dequantise;
    decltype(&mlvc_b200_mx_cache_write) cache_write;
    decltype(&mlvc_b200_mx_cache_read) cache_read;
    decltype(&mlvc_b200_mx_linear) linear;
    decltype(&mlvc_b200_last_error) last_error;
} library;

PyObject *dense_types;  // dtype -> code of mlvc_b200_matrix
PyObject *dense_type;   // called with a dtype that is not there: adds it or raises
PyObject *int32_types;  // set of dtypes
PyObject *is_int32;     // called with a dtype that is not there: adds it and is true, or false
PyObject *name_shape, *name_stride, *name_dtype, *name_data_ptr, *name_get_device, *name_is_contiguous, *name_nbytes;

// A reference that is given up at the end of its scope.
struct Ref {
    PyObject* p;
    explicit Ref(PyObject* q) : p(q) {}
    ~Ref() { Py_XDECREF(p); }
    Ref(const Ref&) = delete;
    Ref& operator=(const Ref&) = delete;
    explicit operator bool() const { return p != nullptr; }
};

template <typename... A>
bool refuse(const char* format, A... a)
{
    PyErr_Format(PyExc_RuntimeError, format, a...);
    return false;
}

bool unsigned_of(PyObject* o, uint64_t& v)
{
    v = PyLong_AsUnsignedLongLong(o);
    return !(v == static_cast<uint64_t>(-1) && PyErr_Occurred());
}

bool address_of(PyObject* t, uint64_t& at)
{
    Ref r(PyObject_CallMethodNoArgs(t, name_data_ptr));
    return r && unsigned_of(r.p, at);
}

// An operand's sizes or strides; `n`: how many there are, `most` of them in `v`.
bool integers(PyObject* sequence, int64_t* v, Py_ssize_t most, Py_ssize_t& n)
{
    Ref fast(PySequence_Fast(sequence, "a shape or strides must be a sequence"));
    if (!fast)
        return false;
    n = PySequence_Fast_GET_SIZE(fast.p);
    for (Py_ssize_t i = 0; i < n && i < most; ++i) {
        v[i] = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(fast.p, i));
        if (v[i] == -1 && PyErr_Occurred())
            return false;
    }
    return true;
}

// A kernel that is given another memory's address faults.  `device`: the
// backend's, None where it only plans; objects that do not tell theirs pass.
bool on_device(PyObject* t, PyObject* device, const char* what)
{
    if (device == Py_None)
        return true;
    Ref r(PyObject_CallMethodNoArgs(t, name_get_device));
    if (!r) {
        if (!PyErr_ExceptionMatches(PyExc_AttributeError))
            return false;
        PyErr_Clear();
        return true;
    }
    const long at = PyLong_AsLong(r.p), own = PyLong_AsLong(device);
    if (PyErr_Occurred())
        return false;
    if (at == own)
        return true;
    return at < 0 ? refuse("mlvc-b200: %s is on the host, the backend on device %ld", what, own)
                  : refuse("mlvc-b200: %s is on device %ld, the backend on device %ld", what, at, own);
}

bool describe(PyObject* t, PyObject* device, mlvc_b200_matrix& m)
{
    int64_t shape[2], stride[2];
    Py_ssize_t n = 0;
    {
        Ref s(PyObject_GetAttr(t, name_shape));
        if (!s || !integers(s.p, shape, 2, n))
            return false;
    }
    if (n != 2)
        return refuse("mlvc-b200: a dense matrix has two dimensions, not %zd", n);
    {
        Ref dtype(PyObject_GetAttr(t, name_dtype));
        if (!dtype)
            return false;
        Ref code(Py_XNewRef(PyDict_GetItemWithError(dense_types, dtype.p)));
        if (!code && !PyErr_Occurred())
            code.p = PyObject_CallOneArg(dense_type, dtype.p);
        if (!code)
            return false;
        m.dtype = static_cast<int32_t>(PyLong_AsLong(code.p));
    }
    if (!on_device(t, device, "a dense matrix"))
        return false;
    {
        Ref s(PyObject_CallMethodNoArgs(t, name_stride));
        if (!s || !integers(s.p, stride, 2, n))
            return false;
    }
    if (n != 2)
        return refuse("mlvc-b200: a dense matrix has two strides, not %zd", n);
    m.reserved = 0;
    m.rows = shape[0];
    m.cols = shape[1];
    m.row_stride = stride[0];
    m.col_stride = stride[1];
    return address_of(t, m.data);
}

// A contiguous int32 device array of `dims` dimensions.
bool describe_ints(PyObject* t, PyObject* device, const char* what, Py_ssize_t dims, int64_t* shape, uint64_t& at)
{
    Py_ssize_t n = 0;
    {
        Ref s(PyObject_GetAttr(t, name_shape));
        if (!s || !integers(s.p, shape, dims, n))
            return false;
    }
    Ref dtype(PyObject_GetAttr(t, name_dtype));
    if (!dtype)
        return false;
    int fits = PySet_Contains(int32_types, dtype.p);
    if (fits == 0) {
        Ref r(PyObject_CallOneArg(is_int32, dtype.p));
        fits = r ? PyObject_IsTrue(r.p) : -1;
    }
    if (fits > 0) {
        Ref r(PyObject_CallMethodNoArgs(t, name_is_contiguous));
        fits = r ? PyObject_IsTrue(r.p) : -1;
    }
    if (fits < 0)
        return false;
    if (!fits || n != dims)
        return refuse("mlvc-b200: %s must be a contiguous int32 array of %zd dimension(s)", what, dims);
    return on_device(t, device, what) && address_of(t, at);
}

bool describe_rows(PyObject* pages, PyObject* offsets, PyObject* starts, PyObject* device, mlvc_b200_mx_rows& r)
{
    int64_t table[2], ends = 0, begins = 0;
    if (!describe_ints(pages, device, "the page table", 2, table, r.pages) ||
        !describe_ints(offsets, device, "offsets", 1, &ends, r.offsets))
        return false;
    r.starts = 0;
    if (starts != Py_None && !describe_ints(starts, device, "starts", 1, &begins, r.starts))
        return false;
    if (ends != table[0] + 1 || (starts != Py_None && begins != table[0]))
        return refuse("mlvc-b200: offsets has one entry more than there are sequences, starts as many");
    r.sequences = table[0];
    r.pages_per_sequence = table[1];
    return true;
}

// Address of a structure that Python holds, or a handle (None: null).
template <typename T>
bool pointer_of(PyObject* o, T*& p)
{
    uint64_t v = 0;
    if (o != Py_None && !unsigned_of(o, v))
        return false;
    p = reinterpret_cast<T*>(static_cast<uintptr_t>(v));
    return true;
}

template <typename F>
PyObject* made(F&& call)
{
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = call();
    Py_END_ALLOW_THREADS
    if (rc) {
        refuse("%s", library.last_error());
        return nullptr;
    }
    Py_RETURN_NONE;
}

bool count_is(Py_ssize_t n, Py_ssize_t want)
{
    if (n != want)
        PyErr_Format(PyExc_TypeError, "%zd arguments where there are %zd", n, want);
    return n == want;
}

// convert(read, backend, dense, address of a mlvc_b200_mx_matrix, stream, device)
PyObject* convert(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    mlvc_b200_backend* backend;
    mlvc_b200_matrix dense;
    mlvc_b200_mx_matrix* held;
    uint64_t stream;
    if (!count_is(n, 6) || !pointer_of(a[1], backend) || !describe(a[2], a[5], dense) || !pointer_of(a[3], held) ||
        !unsigned_of(a[4], stream))
        return nullptr;
    const bool read = a[0] == Py_True;
    return made([&] {
        return read ? library.dequantise(backend, held, &dense, stream) : library.quantise(backend, &dense, held, stream);
    });
}

// cache(read, backend, address of a mlvc_b200_mx_cache, dense, pages, offsets, starts, stream, device)
PyObject* cache(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    mlvc_b200_backend* backend;
    mlvc_b200_mx_cache* held;
    mlvc_b200_matrix dense;
    mlvc_b200_mx_rows rows;
    uint64_t stream;
    if (!count_is(n, 9) || !pointer_of(a[1], backend) || !pointer_of(a[2], held) || !describe(a[3], a[8], dense) ||
        !describe_rows(a[4], a[5], a[6], a[8], rows) || !unsigned_of(a[7], stream))
        return nullptr;
    const auto call = a[0] == Py_True ? library.cache_read : library.cache_write;
    return made([&] { return call(backend, held, &dense, &rows, stream); });
}

// linear(backend, address of the layer's mlvc_b200_mx_linear_args, x, y, residual, workspace, stream, device,
// address of a mlvc_b200_mx_matrix in the place of x, or None)
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    mlvc_b200_backend* backend;
    const mlvc_b200_mx_linear_args* layer;
    uint64_t stream;
    if (!count_is(n, 9) || !pointer_of(a[0], backend) || !pointer_of(a[1], layer) || !unsigned_of(a[6], stream))
        return nullptr;
    mlvc_b200_mx_linear_args l = *layer;
    if (a[8] != Py_None) {
        mlvc_b200_mx_matrix* x;
        if (!pointer_of(a[8], x))
            return nullptr;
        l.a = *x;
    } else if (!describe(a[2], a[7], l.x)) {
        return nullptr;
    }
    if (!describe(a[3], a[7], l.y) || (a[4] != Py_None && !describe(a[4], a[7], l.residual)))
        return nullptr;
    if (a[5] != Py_None) {
        Ref bytes(PyObject_GetAttr(a[5], name_nbytes));
        uint64_t size;
        if (!bytes || !unsigned_of(bytes.p, size) || !on_device(a[5], a[7], "the workspace") || !address_of(a[5], l.workspace))
            return nullptr;
        l.workspace_bytes = size;
    }
    return made([&] { return library.linear(backend, &l, stream); });
}

// connect(addresses of Library's functions, dense_types, dense_type, int32_types, is_int32)
PyObject* connect(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (!count_is(n, 5))
        return nullptr;
    void* address[6];
    if (!PyTuple_Check(a[0]) || PyTuple_GET_SIZE(a[0]) != 6)
        return PyErr_Format(PyExc_TypeError, "six addresses");
    for (int i = 0; i < 6; ++i)
        if (!pointer_of(PyTuple_GET_ITEM(a[0], i), address[i]))
            return nullptr;
    library = {reinterpret_cast<decltype(library.quantise)>(address[0]),
               reinterpret_cast<decltype(library.dequantise)>(address[1]),
               reinterpret_cast<decltype(library.cache_write)>(address[2]),
               reinterpret_cast<decltype(library.cache_read)>(address[3]),
               reinterpret_cast<decltype(library.linear)>(address[4]),
               reinterpret_cast<decltype(library.last_error)>(address[5])};
    if (!PyDict_Check(a[1]) || !PySet_Check(a[3]))
        return PyErr_Format(PyExc_TypeError, "a dict and a set");
    PyObject** const kept[4] = {&dense_types, &dense_type, &int32_types, &is_int32};
    for (int i = 0; i < 4; ++i) {
        Py_XDECREF(*kept[i]);
        *kept[i] = Py_NewRef(a[1 + i]);
    }
    Py_RETURN_NONE;
}

PyCFunction fast(PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t))
{
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef methods[] = {{"convert", fast(convert), METH_FASTCALL, nullptr},
                         {"cache", fast(cache), METH_FASTCALL, nullptr},
                         {"linear", fast(linear), METH_FASTCALL, nullptr},
                         {"connect", fast(connect), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls()
{
    struct {
        PyObject** name;
        const char* text;
    } const names[] = {{&name_shape, "shape"},           {&name_stride, "stride"},
                       {&name_dtype, "dtype"},           {&name_data_ptr, "data_ptr"},
                       {&name_get_device, "get_device"}, {&name_is_contiguous, "is_contiguous"},
                       {&name_nbytes, "nbytes"}};
    for (const auto& n : names)
        if (!(*n.name = PyUnicode_InternFromString(n.text)))
            return nullptr;
    return PyModule_Create(&module);
}
