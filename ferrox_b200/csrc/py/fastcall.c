// Calls of the kernel library's C entry points from Python.  ctypes converts every argument through a converter object and
// describes the call to libffi anew each time: 3 us for the two dozen arguments of a product, which a step that is not a
// replayed graph pays some sixty times.  A `Function` here holds an entry point's address and one code an argument (the kernels'
// signatures), reads plain ints, floats and None straight into the argument registers' images and calls.
//
// The call goes through one function type: all integer arguments as 64-bit words, then eight doubles.  In the System V
// calling convention of x86-64 and in that of AArch64, integer and floating-point arguments are counted apart: the words fill
// the integer registers and then the stack in the order in which the callee has its integers, the doubles the first eight
// floating-point registers (a float in the low half).  What is passed beyond the callee's own arguments is not looked at and is
// the caller's to clean up.  An entry point with more than eight floating-point arguments, or on another machine, is not bound
// (ctypes takes it).
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stddef.h>
#include <stdint.h>
#include <string.h>

#if defined(__x86_64__) && !defined(_WIN32)
#define FX_WORDS_THEN_FLOATS 1
#elif defined(__aarch64__) && defined(__linux__)
#define FX_WORDS_THEN_FLOATS 1
#else
#define FX_WORDS_THEN_FLOATS 0
#endif

#define MAX_WORDS 48
#define MAX_FLOATS 8

typedef int64_t W;
#define W4 W, W, W, W
#define W16 W4, W4, W4, W4
#define D8 double, double, double, double, double, double, double, double
#define A4(i) w[i], w[i + 1], w[i + 2], w[i + 3]
#define A16(i) A4(i), A4(i + 4), A4(i + 8), A4(i + 12)
#define F8 f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7]

static int call_words(void* fn, int n, const W* w, const double* f)
{
    if (n <= 16) return ((int (*)(W16, D8))fn)(A16(0), F8);
    if (n <= 32) return ((int (*)(W16, W16, D8))fn)(A16(0), A16(16), F8);
    return ((int (*)(W16, W16, W16, D8))fn)(A16(0), A16(16), A16(32), F8);
}

typedef struct {
    PyObject_HEAD
    vectorcallfunc vectorcall;
    void* fn;
    int n;
    char codes[MAX_WORDS + MAX_FLOATS + 1];
} Function;

// The entry point's return value; NotImplemented where an argument is none of the kinds that are read here.
static PyObject* function_call(PyObject* self, PyObject* const* args, size_t nargsf, PyObject* kwnames)
{
    Function* f = (Function*)self;
    const Py_ssize_t n = PyVectorcall_NARGS(nargsf);
    if (n != f->n || (kwnames && PyTuple_GET_SIZE(kwnames))) {
        PyErr_Format(PyExc_TypeError, "entry point takes %d arguments (%zd given)", f->n, n);
        return NULL;
    }
    W words[MAX_WORDS];
    double floats[MAX_FLOATS];
    memset(floats, 0, sizeof floats);
    int nw = 0, nf = 0;
    for (int i = 0; i < f->n; ++i) {
        PyObject* a = args[i];
        switch (f->codes[i]) {
            case 'P':
                if (a == Py_None) { words[nw++] = 0; break; }
                if (!PyLong_Check(a)) Py_RETURN_NOTIMPLEMENTED;
                words[nw++] = (W)PyLong_AsUnsignedLongLongMask(a);
                break;
            case 'I': case 'L': case 'U':
                if (!PyLong_Check(a)) Py_RETURN_NOTIMPLEMENTED;
                words[nw] = (W)PyLong_AsUnsignedLongLongMask(a);
                if (f->codes[i] == 'I') words[nw] = (W)(int32_t)words[nw];
                ++nw;
                break;
            default: {
                const double v = PyFloat_AsDouble(a);
                if (v == -1.0 && PyErr_Occurred()) return NULL;
                if (f->codes[i] == 'F') {
                    const float s = (float)v;
                    memcpy(&floats[nf++], &s, sizeof s);
                } else {
                    floats[nf++] = v;
                }
            }
        }
        if (PyErr_Occurred()) return NULL;
    }
    for (int i = nw; i < MAX_WORDS; ++i) words[i] = 0;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = call_words(f->fn, nw, words, floats);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

static void function_free(PyObject* self) { Py_TYPE(self)->tp_free(self); }

static PyTypeObject FunctionType = {
    PyVarObject_HEAD_INIT(NULL, 0)
    .tp_name = "_fx_fastcall.Function",
    .tp_basicsize = sizeof(Function),
    .tp_dealloc = function_free,
    .tp_vectorcall_offset = offsetof(Function, vectorcall),
    .tp_call = PyVectorcall_Call,
    .tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_VECTORCALL,
    .tp_doc = "A C entry point with its arguments' codes.",
};

// bind(address, codes) -> Function, or None where the call cannot be made this way
static PyObject* bind(PyObject* module, PyObject* args)
{
    unsigned long long address;
    const char* codes;
    if (!PyArg_ParseTuple(args, "Ks", &address, &codes)) return NULL;
    int words = 0, floats = 0;
    for (const char* c = codes; *c; ++c) {
        if (strchr("PILU", *c)) ++words;
        else if (strchr("FD", *c)) ++floats;
        else { PyErr_Format(PyExc_ValueError, "unknown argument code %c", *c); return NULL; }
    }
    if (!FX_WORDS_THEN_FLOATS || words > MAX_WORDS || floats > MAX_FLOATS) Py_RETURN_NONE;
    Function* f = PyObject_New(Function, &FunctionType);
    if (!f) return NULL;
    f->vectorcall = function_call;
    f->fn = (void*)(uintptr_t)address;
    f->n = words + floats;
    memset(f->codes, 0, sizeof f->codes);
    memcpy(f->codes, codes, (size_t)f->n);
    return (PyObject*)f;
}

// A tensor's address and row stride as the wrappers ask for them some hundreds of times a step, without a Python frame each;
// what is not as expected (no CUDA tensor, other strides) goes to the Python functions that name the error.
static PyObject *slow_ptr, *slow_rows, *s_is_cuda, *s_data_ptr, *s_dim, *s_stride, *zero, *one;

static PyObject* ptr(PyObject* module, PyObject* t)
{
    if (t == Py_None) Py_RETURN_NONE;
    PyObject* cuda = PyObject_GetAttr(t, s_is_cuda);
    if (!cuda) return NULL;
    const int yes = cuda == Py_True;
    Py_DECREF(cuda);
    return yes ? PyObject_CallMethodNoArgs(t, s_data_ptr) : PyObject_CallOneArg(slow_ptr, t);
}

static PyObject* rows(PyObject* module, PyObject* t)
{
    PyObject* dim = PyObject_CallMethodNoArgs(t, s_dim);
    if (!dim) return NULL;
    const long d = PyLong_AsLong(dim);
    Py_DECREF(dim);
    if (d == 2) {
        PyObject* inner = PyObject_CallMethodOneArg(t, s_stride, one);
        if (!inner) return NULL;
        const long s = PyLong_AsLong(inner);
        Py_DECREF(inner);
        if (s == 1) return PyObject_CallMethodOneArg(t, s_stride, zero);
    }
    if (PyErr_Occurred()) return NULL;
    return PyObject_CallOneArg(slow_rows, t);
}

static PyObject* set_slow(PyObject* module, PyObject* args)
{
    PyObject *p, *r;
    if (!PyArg_ParseTuple(args, "OO", &p, &r)) return NULL;
    Py_INCREF(p); Py_INCREF(r);
    Py_XSETREF(slow_ptr, p);
    Py_XSETREF(slow_rows, r);
    Py_RETURN_NONE;
}

// ---- operands looked at in one go ------------------------------------------------------------------------------------
// An entry point of a dozen tensors costs more in questions about them (50 to 150 ns each) than in its launch.  look(spec,
// tensors...) asks for each tensor once, by DLPack's exchange interface, and compares it with what the call needs; what is not
// so, or what the interface does not give, is left to the caller, who names the error.
//
// spec: a word a tensor: its type (e: e4m3, u: unsigned byte, i: 32-bit integer, f: 32-bit float, x: 32-bit float or bfloat16,
// the same for all of them), then a letter a dimension; the same letter is the same size wherever it stands.  Tensors are
// contiguous, or with ~ at the word's end rows of contiguous elements.  ? at the beginning: the tensor may be None.
// Returns None, or (device, current stream there, x's code, addresses, sizes of the letters in their order of appearance, -1
// for one of an absent tensor, row strides of the words with ~).
typedef struct { int32_t device_type, device_id; } DlDevice;
typedef struct { uint8_t code, bits; uint16_t lanes; } DlType;
typedef struct { void* data; DlDevice device; int32_t ndim; DlType dtype; int64_t *shape, *strides; uint64_t byte_offset; } DlTensor;
typedef struct {
    struct { uint32_t major, minor; } version;
    void *prev, *allocate, *managed_from, *managed_to;
    int (*tensor_from)(void* object, DlTensor* out);
    int (*stream_of)(int32_t device_type, int32_t device_id, void** out);
} DlExchange;
enum { DL_CUDA = 2, DL_INT = 0, DL_UINT = 1, DL_FLOAT = 2, DL_BFLOAT = 4, DL_E4M3 = 10, MAX_LOOKED = 16, MAX_LETTERS = 16 };
static const DlExchange* exchange;

static int type_fits(char want, DlType t, int* x_code)
{
    if (t.lanes != 1) return 0;
    switch (want) {
        case 'e': return t.code == DL_E4M3 && t.bits == 8;
        case 'u': return t.code == DL_UINT && t.bits == 8;
        case 'i': return t.code == DL_INT && t.bits == 32;
        case 'f': return t.code == DL_FLOAT && t.bits == 32;
        default: {
            const int code = t.code == DL_FLOAT && t.bits == 32 ? 0 : t.code == DL_BFLOAT && t.bits == 16 ? 1 : -1;
            if (code < 0 || (*x_code >= 0 && *x_code != code)) return 0;
            *x_code = code;
            return 1;
        }
    }
}

static PyObject* look(PyObject* module, PyObject* const* args, Py_ssize_t n)
{
    if (!exchange || n < 2 || n > MAX_LOOKED + 1) Py_RETURN_NONE;
    const char* c = PyUnicode_AsUTF8(args[0]);
    if (!c) return NULL;
    W address[MAX_LOOKED], size[MAX_LETTERS], row[MAX_LOOKED];
    char letter[MAX_LETTERS];
    int letters = 0, rows = 0, device = -1, x_code = -1;
    for (Py_ssize_t i = 1; i < n; ++i) {
        while (*c == ' ') ++c;
        const int absent = *c == '?' && args[i] == Py_None;
        if (*c == '?') ++c;
        DlTensor t = {0};
        const char type = *c++;
        if (!absent) {
            if (!type || exchange->tensor_from(args[i], &t)) { PyErr_Clear(); Py_RETURN_NONE; }
            if (t.device.device_type != DL_CUDA || (device >= 0 && t.device.device_id != device) || !type_fits(type, t.dtype, &x_code)) Py_RETURN_NONE;
            device = t.device.device_id;
        }
        address[i - 1] = absent ? 0 : (W)(uintptr_t)t.data + (W)t.byte_offset;
        int dims = 0;
        for (; *c && *c != ' ' && *c != '~'; ++c, ++dims) {
            int k = 0;
            while (k < letters && letter[k] != *c) ++k;
            if (k == letters) {
                if (letters == MAX_LETTERS) Py_RETURN_NONE;
                letter[letters] = *c;
                size[letters++] = -1;
            }
            if (absent) continue;
            if (dims >= t.ndim || (size[k] >= 0 && size[k] != t.shape[dims])) Py_RETURN_NONE;
            size[k] = t.shape[dims];
        }
        const int by_rows = *c == '~';
        if (by_rows) ++c;
        if (absent) { if (by_rows) row[rows++] = 0; continue; }
        if (dims != t.ndim || (by_rows && dims != 2)) Py_RETURN_NONE;
        W step = 1;
        int empty = 0;
        for (int d = 0; d < dims; ++d) empty |= t.shape[d] == 0;
        for (int d = dims - 1; d >= by_rows; --d) {
            if (!empty && t.strides && t.shape[d] > 1 && t.strides[d] != step) Py_RETURN_NONE;
            step *= t.shape[d];
        }
        if (by_rows) {                                       // (a single row's stride says nothing)
            row[rows] = t.shape[0] > 1 && t.strides ? t.strides[0] : t.shape[1];
            if (row[rows++] < 0) Py_RETURN_NONE;
        }
    }
    void* stream = NULL;
    if (device < 0 || exchange->stream_of(DL_CUDA, device, &stream)) { PyErr_Clear(); Py_RETURN_NONE; }
    const Py_ssize_t total = 3 + (n - 1) + letters + rows;
    PyObject* out = PyTuple_New(total);
    if (!out) return NULL;
    for (Py_ssize_t i = 0; i < total; ++i) {
        const Py_ssize_t a = i - 3, l = a - (n - 1), r = l - letters;
        PyObject* v = PyLong_FromLongLong(i == 0 ? device : i == 1 ? (W)(uintptr_t)stream : i == 2 ? x_code : a < n - 1 ? address[a] : l < letters ? size[l] : row[r]);
        if (!v) { Py_DECREF(out); return NULL; }
        PyTuple_SET_ITEM(out, i, v);
    }
    return out;
}

// exchange(capsule): DLPack's exchange interface of the tensors' library; whether it is of a kind that is read here
static PyObject* set_exchange(PyObject* module, PyObject* capsule)
{
    const DlExchange* e = PyCapsule_GetPointer(capsule, "dlpack_exchange_api");
    if (!e) return NULL;
    exchange = e->version.major == 1 && e->tensor_from && e->stream_of ? e : NULL;
    return PyBool_FromLong(exchange != NULL);
}

static PyMethodDef methods[] = {
    {"ptr", ptr, METH_O, "A CUDA tensor's address, None for None."},
    {"rows", rows, METH_O, "The row stride of a two-dimensional tensor with contiguous rows."},
    {"set_slow", set_slow, METH_VARARGS, "set_slow(ptr, rows): what takes the arguments that these do not."},
    {"look", (PyCFunction)(void (*)(void))look, METH_FASTCALL, "look(spec, tensors...): what a call needs to know of them, or None."},
    {"set_exchange", set_exchange, METH_O, "set_exchange(capsule): where look finds the tensors' descriptions."},
    {"bind", bind, METH_VARARGS, "bind(address, codes): the C entry point there as a callable, or None."},
    {NULL, NULL, 0, NULL},
};
static struct PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_fx_fastcall", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__fx_fastcall(void)
{
    if (PyType_Ready(&FunctionType) < 0) return NULL;
    s_is_cuda = PyUnicode_InternFromString("is_cuda"); s_data_ptr = PyUnicode_InternFromString("data_ptr");
    s_dim = PyUnicode_InternFromString("dim"); s_stride = PyUnicode_InternFromString("stride");
    zero = PyLong_FromLong(0); one = PyLong_FromLong(1);
    if (!s_is_cuda || !s_data_ptr || !s_dim || !s_stride || !zero || !one) return NULL;
    return PyModule_Create(&module_def);
}
