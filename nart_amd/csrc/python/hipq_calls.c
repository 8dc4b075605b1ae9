/* The per-call functions of nart_amd/hipq.py as a CPython extension: tensors in, one call of the hipq C ABI (include/hipq.h).
 *
 * Why: a small operator is one launch, and the launch is 2.6 - 3.2 us of host time in the HIP runtime; through ctypes the way
 * there cost another 1.3 us (three arguments) to 5 us (lists that became numpy arrays and their addresses), so that the
 * eight operators of an inception block took 44 us of host time for 21 us of GPU time.
 *
 * Each function takes the arguments of its namesake in hipq.py, positionally and complete, launches on torch's current stream
 * and returns the C ABI's status.  Nothing of torch is linked: a tensor is asked for data_ptr() and shape. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <string.h>

#include "hipq.h"

#define MAX_IN HIPQ_MAX_ELTWISE_INPUTS

static PyObject *s_data_ptr, *s_shape, *s_numel, *s_dtype, *s_stride, *s_get_device;
static PyObject *get_device, *get_stream; /* torch's accessors: () -> int, (int) -> address */

static int current_stream(void **out)
{
    if (get_stream == NULL) {
        PyErr_SetString(PyExc_RuntimeError, "hipq_calls: init() has not been called");
        return 0;
    }
    PyObject *dev = PyObject_CallNoArgs(get_device);
    if (dev == NULL)
        return 0;
    PyObject *st = PyObject_CallOneArg(get_stream, dev);
    Py_DECREF(dev);
    if (st == NULL)
        return 0;
    *out = PyLong_AsVoidPtr(st);
    Py_DECREF(st);
    return !(*out == NULL && PyErr_Occurred());
}

/* a tensor's address; None: a null pointer */
static int address(PyObject *t, void **out)
{
    *out = NULL;
    if (t == Py_None)
        return 1;
    PyObject *v = PyObject_CallMethodNoArgs(t, s_data_ptr);
    if (v == NULL)
        return 0;
    *out = PyLong_AsVoidPtr(v);
    Py_DECREF(v);
    return !(*out == NULL && PyErr_Occurred());
}

static int whole(PyObject *o, int *out)
{
    const long v = PyLong_AsLong(o);
    *out = (int)v;
    return !(v == -1 && PyErr_Occurred());
}

static int number(PyObject *o, float *out)
{
    const double v = PyFloat_AsDouble(o);
    *out = (float)v;
    return !(v == -1.0 && PyErr_Occurred());
}

/* the four dimensions of a tensor */
static int shape4(PyObject *t, int d[4])
{
    PyObject *s = PyObject_GetAttr(t, s_shape);
    if (s == NULL)
        return 0;
    int ok = PyTuple_Check(s) && PyTuple_GET_SIZE(s) == 4;
    if (!ok)
        PyErr_SetString(PyExc_ValueError, "a tensor with four dimensions is expected");
    for (int i = 0; ok && i < 4; ++i)
        ok = whole(PyTuple_GET_ITEM(s, i), &d[i]);
    Py_DECREF(s);
    return ok;
}

static int last_dim(PyObject *t, int *out)
{
    PyObject *s = PyObject_GetAttr(t, s_shape);
    if (s == NULL)
        return 0;
    PyObject *v = PySequence_GetItem(s, -1);
    const int ok = v != NULL && whole(v, out);
    Py_XDECREF(v);
    Py_DECREF(s);
    return ok;
}

static int count(PyObject *t, size_t *out)
{
    PyObject *v = PyObject_CallMethodNoArgs(t, s_numel);
    if (v == NULL)
        return 0;
    *out = PyLong_AsSize_t(v);
    Py_DECREF(v);
    return !(*out == (size_t)-1 && PyErr_Occurred());
}

/* the first n entries of a sequence (a list, a tuple, an array) */
static int addresses(PyObject *seq, Py_ssize_t n, const void **out)
{
    for (Py_ssize_t i = 0; i < n; ++i) {
        void *p;
        PyObject *t = PySequence_GetItem(seq, i);
        const int ok = t != NULL && address(t, &p);
        Py_XDECREF(t);
        if (!ok)
            return 0;
        out[i] = p;
    }
    return 1;
}

static int numbers(PyObject *seq, Py_ssize_t n, float *out)
{
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject *v = PySequence_GetItem(seq, i);
        const int ok = v != NULL && number(v, &out[i]);
        Py_XDECREF(v);
        if (!ok)
            return 0;
    }
    return 1;
}

static int wholes(PyObject *seq, Py_ssize_t n, int *out)
{
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject *v = PySequence_GetItem(seq, i);
        const int ok = v != NULL && whole(v, &out[i]);
        Py_XDECREF(v);
        if (!ok)
            return 0;
    }
    return 1;
}

static int bytes_of(PyObject *seq, Py_ssize_t n, uint8_t *out)
{
    int v[MAX_IN];
    if (!wholes(seq, n, v))
        return 0;
    for (Py_ssize_t i = 0; i < n; ++i) {
        if (v[i] < 0 || v[i] > 255) {
            PyErr_SetString(PyExc_OverflowError, "a zero point lies outside 0..255");
            return 0;
        }
        out[i] = (uint8_t)v[i];
    }
    return 1;
}

static int expect(Py_ssize_t got, Py_ssize_t want)
{
    if (got != want)
        PyErr_Format(PyExc_TypeError, "%zd arguments are expected, %zd were given", want, got);
    return got == want;
}

/* a scalar that stands for both directions, or a pair */
static int pair(PyObject *o, int *h, int *w)
{
    if (PyLong_Check(o))
        return whole(o, h) && (*w = *h, 1);
    if (PySequence_Check(o)) {
        const Py_ssize_t n = PySequence_Size(o);
        int v[2];
        if (n != 2) {
            if (n >= 0)
                PyErr_SetString(PyExc_ValueError, "a number or a pair of numbers is expected");
            return 0;
        }
        return wholes(o, 2, v) && (*h = v[0], *w = v[1], 1);
    }
    return whole(o, h) && (*w = *h, 1);
}

#define CALL(EXPR)                         \
    do {                                   \
        int rc_;                           \
        Py_BEGIN_ALLOW_THREADS;            \
        rc_ = (EXPR);                      \
        Py_END_ALLOW_THREADS;              \
        return PyLong_FromLong(rc_);       \
    } while (0)
#define ARGS PyObject *self, PyObject *const *a, Py_ssize_t n

static PyObject *py_init(ARGS)
{
    if (!expect(n, 2))
        return NULL;
    Py_INCREF(a[0]);
    Py_INCREF(a[1]);
    Py_XSETREF(get_device, a[0]);
    Py_XSETREF(get_stream, a[1]);
    Py_RETURN_NONE;
}

/* plan address, x, y, acc */
static PyObject *py_conv2d_run(ARGS)
{
    void *x, *y, *acc, *st;
    if (!expect(n, 4))
        return NULL;
    const void *plan = PyLong_AsVoidPtr(a[0]);
    if ((plan == NULL && PyErr_Occurred()) || !address(a[1], &x) || !address(a[2], &y) || !address(a[3], &acc) || !current_stream(&st))
        return NULL;
    CALL(hipq_conv2d_run((const hipq_conv2d_plan *)plan, x, y, (int32_t *)acc, st));
}

/* a, b, y, ialpha0, izp0, ialpha1, izp1, oalpha, ozp, obits */
static PyObject *py_add_u8(ARGS)
{
    void *p, *q, *y, *st;
    size_t len;
    float a0, a1, ao;
    int z0, z1, zo, bits;
    if (!expect(n, 10) || !address(a[0], &p) || !address(a[1], &q) || !address(a[2], &y) || !count(a[0], &len) || !number(a[3], &a0)
        || !whole(a[4], &z0) || !number(a[5], &a1) || !whole(a[6], &z1) || !number(a[7], &ao) || !whole(a[8], &zo) || !whole(a[9], &bits)
        || !current_stream(&st))
        return NULL;
    CALL(hipq_add_u8(p, q, y, len, a0, z0, a1, z1, ao, zo, bits, st));
}

/* ins, y, ialpha, izp, oalpha, ozp, operation, coeff or None, obits */
static PyObject *py_eltwise_u8(ARGS)
{
    const void *in[MAX_IN];
    float ia[MAX_IN], cf[MAX_IN], ao;
    uint8_t iz[MAX_IN];
    void *y, *st;
    size_t len;
    int zo, op, bits;
    if (!expect(n, 9))
        return NULL;
    const Py_ssize_t m = PySequence_Size(a[0]), k = m < MAX_IN ? m : MAX_IN; /* the C ABI refuses more, by their number */
    if (m < 0 || !addresses(a[0], k, in) || !address(a[1], &y) || !count(a[1], &len) || !numbers(a[2], k, ia) || !bytes_of(a[3], k, iz)
        || !number(a[4], &ao) || !whole(a[5], &zo) || !whole(a[6], &op) || (a[7] != Py_None && !numbers(a[7], k, cf))
        || !whole(a[8], &bits) || !current_stream(&st))
        return NULL;
    CALL(hipq_eltwise_u8(in, (int)m, a[7] == Py_None ? NULL : cf, ia, iz, y, len, op, ao, zo, bits, st));
}

/* x, y, ialpha, izp, oalpha, ozp, obits */
static PyObject *py_relu_u8(ARGS)
{
    void *x, *y, *st;
    size_t len;
    float ai, ao;
    int zi, zo, bits;
    if (!expect(n, 7) || !address(a[0], &x) || !address(a[1], &y) || !count(a[0], &len) || !number(a[2], &ai) || !whole(a[3], &zi)
        || !number(a[4], &ao) || !whole(a[5], &zo) || !whole(a[6], &bits) || !current_stream(&st))
        return NULL;
    CALL(hipq_relu_u8(x, y, len, ai, zi, ao, zo, bits, st));
}

/* ins, channels, y, ialpha, izp, oalpha, ozp, obits */
static PyObject *py_concat_u8(ARGS)
{
    const void *in[MAX_IN];
    float ia[MAX_IN], ao;
    uint8_t iz[MAX_IN];
    int ch[MAX_IN], d[4], zo, bits;
    void *y, *st;
    if (!expect(n, 8))
        return NULL;
    const Py_ssize_t m = PySequence_Size(a[0]), k = m < MAX_IN ? m : MAX_IN; /* the C ABI refuses more, by their number */
    if (m < 0 || !addresses(a[0], k, in) || !wholes(a[1], k, ch) || !address(a[2], &y) || !shape4(a[2], d) || !numbers(a[3], k, ia)
        || !bytes_of(a[4], k, iz) || !number(a[5], &ao) || !whole(a[6], &zo) || !whole(a[7], &bits) || !current_stream(&st))
        return NULL;
    CALL(hipq_concat_u8(in, (int)m, ch, ia, iz, y, (size_t)d[0] * d[1] * d[2], ao, zo, bits, st));
}

/* x, y, C, ialpha, izp, oalpha, ozp, obits */
static PyObject *py_softmax_u8(ARGS)
{
    void *x, *y, *st;
    float ai, ao;
    int d[4], c, zi, zo, bits;
    if (!expect(n, 8) || !address(a[0], &x) || !shape4(a[0], d) || !address(a[1], &y) || !whole(a[2], &c) || !number(a[3], &ai)
        || !whole(a[4], &zi) || !number(a[5], &ao) || !whole(a[6], &zo) || !whole(a[7], &bits) || !current_stream(&st))
        return NULL;
    CALL(hipq_softmax_u8(x, y, (size_t)d[0] * d[1] * d[2], c, d[3], ai, zi, ao, zo, bits, st));
}

/* x, y, C, kernel, pad, stride, method, ialpha, izp, oalpha, ozp, obits */
static PyObject *py_pool_u8(ARGS)
{
    void *x, *y, *st;
    float ai, ao;
    int d[4], o[4], c, kh, kw, ph, pw, sh, sw, method, zi, zo, bits;
    if (!expect(n, 12) || !address(a[0], &x) || !shape4(a[0], d) || !address(a[1], &y) || !shape4(a[1], o) || !whole(a[2], &c)
        || !pair(a[3], &kh, &kw) || !pair(a[4], &ph, &pw) || !pair(a[5], &sh, &sw) || !whole(a[6], &method) || !number(a[7], &ai)
        || !whole(a[8], &zi) || !number(a[9], &ao) || !whole(a[10], &zo) || !whole(a[11], &bits) || !current_stream(&st))
        return NULL;
    CALL(hipq_pool_u8(x, y, d[0], c, d[1], d[2], o[1], o[2], d[3], kh, kw, ph, pw, sh, sw, method, ai, zi, ao, zo, bits, st));
}

/* x (NCHW floats), y (NHWC bytes), oalpha, ozp, obits */
static PyObject *py_quantize_u8(ARGS)
{
    void *x, *y, *st;
    float ao;
    int d[4], cs, zo, bits;
    if (!expect(n, 5) || !address(a[0], &x) || !shape4(a[0], d) || !address(a[1], &y) || !last_dim(a[1], &cs) || !number(a[2], &ao)
        || !whole(a[3], &zo) || !whole(a[4], &bits) || !current_stream(&st))
        return NULL;
    CALL(hipq_quantize_u8(x, y, d[0], d[1], d[2], d[3], cs, ao, zo, bits, st));
}

/* x (NCHW floats), y (NHWC bytes), oalpha, obits */
static PyObject *py_quantize_i8(ARGS)
{
    void *x, *y, *st;
    float ao;
    int d[4], cs, bits;
    if (!expect(n, 4) || !address(a[0], &x) || !shape4(a[0], d) || !address(a[1], &y) || !last_dim(a[1], &cs) || !number(a[2], &ao)
        || !whole(a[3], &bits) || !current_stream(&st))
        return NULL;
    CALL(hipq_quantize_i8(x, y, d[0], d[1], d[2], d[3], cs, ao, bits, st));
}

/* x (NHWC bytes), y (NCHW floats), ialpha, izp */
static PyObject *py_dequantize_u8(ARGS)
{
    void *x, *y, *st;
    float ai;
    int cs, o[4], zi;
    if (!expect(n, 4) || !address(a[0], &x) || !last_dim(a[0], &cs) || !address(a[1], &y) || !shape4(a[1], o) || !number(a[2], &ai)
        || !whole(a[3], &zi) || !current_stream(&st))
        return NULL;
    CALL(hipq_dequantize_u8(x, y, o[0], o[1], o[2], o[3], cs, ai, zi, st));
}

/* x (NHWC bytes), y (NCHW floats), ialpha */
static PyObject *py_dequantize_i8(ARGS)
{
    void *x, *y, *st;
    float ai;
    int cs, o[4];
    if (!expect(n, 3) || !address(a[0], &x) || !last_dim(a[0], &cs) || !address(a[1], &y) || !shape4(a[1], o) || !number(a[2], &ai)
        || !current_stream(&st))
        return NULL;
    CALL(hipq_dequantize_i8(x, y, o[0], o[1], o[2], o[3], cs, ai, st));
}

/* ---- operators of language models: their tensors are checked here, by name ---- */
enum { F32 = HIPQ_REAL_F32, F16 = HIPQ_REAL_F16, BF16 = HIPQ_REAL_BF16, I32, I64, U8, I8, DTYPES };
static const char *const dtype_names[DTYPES] = {"float32", "float16", "bfloat16", "int32", "int64", "uint8", "int8"};
static PyObject *dtypes[DTYPES]; /* torch's objects */
#define MOST_DIMS 4

typedef struct {
    void *p;
    int there, dtype; /* there: 0 for None */
    int64_t shape[MOST_DIMS], stride[MOST_DIMS];
} view_t;

/* the seven dtypes, in the order above */
static PyObject *py_types(ARGS)
{
    (void)self;
    if (!expect(n, DTYPES))
        return NULL;
    for (int i = 0; i < DTYPES; i++) {
        Py_INCREF(a[i]);
        Py_XSETREF(dtypes[i], a[i]);
    }
    Py_RETURN_NONE;
}

static int longs(PyObject *t, const char *name, int dims, int64_t *out)
{
    if (!PyTuple_Check(t) || PyTuple_GET_SIZE(t) != dims) {
        PyErr_Format(PyExc_ValueError, "%s: %d dimensions are expected", name, dims);
        return 0;
    }
    for (int i = 0; i < dims; i++) {
        out[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(t, i));
        if (out[i] == -1 && PyErr_Occurred())
            return 0;
    }
    return 1;
}

static int current_device(int *out)
{
    if (get_device == NULL || dtypes[0] == NULL) {
        PyErr_SetString(PyExc_RuntimeError, "hipq_calls: init() and types() have not been called");
        return 0;
    }
    PyObject *v = PyObject_CallNoArgs(get_device);
    const int ok = v != NULL && whole(v, out);
    Py_XDECREF(v);
    return ok;
}

/* A tensor of the calling thread's device with `dims` dimensions, one of the dtypes in the set `allowed`, its last dimension without gaps. */
static int tensor(PyObject *t, const char *name, int dims, unsigned allowed, int device, view_t *v)
{
    if (t == Py_None) {
        PyErr_Format(PyExc_ValueError, "%s: a tensor is expected", name);
        return 0;
    }
    PyObject *o = PyObject_GetAttr(t, s_dtype);
    if (o == NULL)
        return 0;
    v->there = 1, v->dtype = 0;
    while (v->dtype < DTYPES && dtypes[v->dtype] != o)
        v->dtype++;
    Py_DECREF(o);
    if (v->dtype == DTYPES || !(allowed >> v->dtype & 1)) {
        char list[96] = "";
        for (int i = 0; i < DTYPES; i++)
            if (allowed >> i & 1) {
                if (list[0])
                    strcat(list, " or ");
                strcat(list, dtype_names[i]);
            }
        PyErr_Format(PyExc_ValueError, "%s: %s is expected", name, list);
        return 0;
    }
    o = PyObject_CallMethodNoArgs(t, s_get_device);
    int on, ok = o != NULL && whole(o, &on);
    Py_XDECREF(o);
    if (!ok)
        return 0;
    if (on != device) {
        PyErr_Format(PyExc_ValueError, on < 0 ? "%s is not on the GPU" : "%s is on device %d, the current one is %d", name, on, device);
        return 0;
    }
    o = PyObject_GetAttr(t, s_shape);
    ok = o != NULL && longs(o, name, dims, v->shape);
    Py_XDECREF(o);
    if (!ok)
        return 0;
    o = PyObject_CallMethodNoArgs(t, s_stride);
    ok = o != NULL && longs(o, name, dims, v->stride);
    Py_XDECREF(o);
    if (!ok || !address(t, &v->p))
        return 0;
    if (v->shape[dims - 1] > 1 && v->stride[dims - 1] != 1) {
        PyErr_Format(PyExc_ValueError, "%s: the last dimension has gaps", name);
        return 0;
    }
    for (int i = 0; i < dims; i++) {
        if (v->shape[i] > 0x7fffffff) {
            PyErr_Format(PyExc_ValueError, "%s: too large", name);
            return 0;
        }
        if (v->shape[i] <= 1 && i < dims - 1)
            v->stride[i] = 0; /* says nothing: torch leaves any number there */
    }
    return 1;
}

/* the same, without gaps anywhere; None: a null pointer where that is allowed */
static int whole_tensor(PyObject *t, const char *name, int dims, unsigned allowed, int device, int none, view_t *v)
{
    if (t == Py_None && none) {
        memset(v, 0, sizeof *v);
        return 1;
    }
    if (!tensor(t, name, dims, allowed, device, v))
        return 0;
    int64_t want = 1;
    for (int i = dims - 1; i >= 0; i--) {
        if (v->shape[i] > 1 && v->stride[i] != want) {
            PyErr_Format(PyExc_ValueError, "%s has gaps", name);
            return 0;
        }
        want *= v->shape[i];
    }
    return 1;
}

/* with gaps between rows; None: a null pointer */
static int tensor_or_none(PyObject *t, const char *name, int dims, unsigned allowed, int device, view_t *v)
{
    if (t == Py_None) {
        memset(v, 0, sizeof *v);
        return 1;
    }
    return tensor(t, name, dims, allowed, device, v);
}

static int shaped(const view_t *v, const char *name, int dims, int64_t s0, int64_t s1, int64_t s2)
{
    const int64_t s[3] = {s0, s1, s2};
    for (int i = 0; i < dims; i++)
        if (v->there && v->shape[i] != s[i]) {
            PyErr_Format(PyExc_ValueError, "%s: %lld entries are expected in dimension %d, it has %lld", name, (long long)s[i], i, (long long)v->shape[i]);
            return 0;
        }
    return 1;
}

#define HALVES (1u << F16 | 1u << BF16)

/* plan, M */
static PyObject *py_w4_workspace(ARGS)
{
    (void)self;
    if (!expect(n, 2))
        return NULL;
    void *plan = PyLong_AsVoidPtr(a[0]);
    int m;
    if ((plan == NULL && PyErr_Occurred()) || !whole(a[1], &m))
        return NULL;
    return PyLong_FromSize_t(hipq_w4_workspace((const hipq_w4_plan *)plan, m));
}

/* plan, type, N, K, x, y, workspace or None */
static PyObject *py_w4_run(ARGS)
{
    (void)self;
    view_t x, y, w;
    int device, type, N, K;
    void *st;
    if (!expect(n, 7))
        return NULL;
    void *plan = PyLong_AsVoidPtr(a[0]);
    if ((plan == NULL && PyErr_Occurred()) || !whole(a[1], &type) || !whole(a[2], &N) || !whole(a[3], &K) || !current_device(&device)
        || !tensor(a[4], "x", 2, 1u << type, device, &x) || !tensor(a[5], "y", 2, 1u << type, device, &y)
        || !whole_tensor(a[6], "workspace", 1, 1u << U8, device, 1, &w) || !shaped(&x, "x", 2, x.shape[0], K, 0) || !shaped(&y, "y", 2, x.shape[0], N, 0)
        || !current_stream(&st))
        return NULL;
    CALL(hipq_w4_run((const hipq_w4_plan *)plan, x.p, x.stride[0], y.p, y.stride[0], (int)x.shape[0], w.p, (size_t)w.shape[0], st));
}

/* plan, M */
static PyObject *py_experts_workspace(ARGS)
{
    (void)self;
    if (!expect(n, 2))
        return NULL;
    void *plan = PyLong_AsVoidPtr(a[0]);
    int m;
    if ((plan == NULL && PyErr_Occurred()) || !whole(a[1], &m))
        return NULL;
    return PyLong_FromSize_t(hipq_w4_experts_workspace((const hipq_w4_experts_plan *)plan, m));
}

/* plan, type, N, K, experts, x, logits, y, workspace or None */
static PyObject *py_experts_run(ARGS)
{
    (void)self;
    view_t x, l, y, w;
    int device, type, N, K, experts;
    void *st;
    if (!expect(n, 9))
        return NULL;
    void *plan = PyLong_AsVoidPtr(a[0]);
    if ((plan == NULL && PyErr_Occurred()) || !whole(a[1], &type) || !whole(a[2], &N) || !whole(a[3], &K) || !whole(a[4], &experts) || !current_device(&device)
        || !tensor(a[5], "x", 2, 1u << type, device, &x) || !tensor(a[6], "logits", 2, HALVES | 1u << F32, device, &l) || !tensor(a[7], "y", 2, 1u << type, device, &y)
        || !whole_tensor(a[8], "workspace", 1, 1u << U8, device, 1, &w) || !shaped(&x, "x", 2, x.shape[0], K, 0) || !shaped(&l, "logits", 2, x.shape[0], experts, 0)
        || !shaped(&y, "y", 2, x.shape[0], N, 0) || !current_stream(&st))
        return NULL;
    CALL(hipq_w4_experts_run((const hipq_w4_experts_plan *)plan, x.p, x.stride[0], l.p, l.dtype, l.stride[0], y.p, y.stride[0], (int)x.shape[0], w.p, (size_t)w.shape[0], st));
}

static void free_cache(PyObject *c) { PyMem_Free(PyCapsule_GetPointer(c, "hipq_kv_cache")); }

/* k, v, k_scale or None, v_scale or None: a capsule with the C struct, without its type */
static PyObject *py_kv_cache(ARGS)
{
    (void)self;
    view_t k, v, ks, vs;
    int device;
    if (!expect(n, 4) || !current_device(&device) || !whole_tensor(a[0], "k", 4, HALVES | 1u << I8, device, 0, &k)
        || !whole_tensor(a[1], "v", 4, 1u << k.dtype, device, 0, &v) || !whole_tensor(a[2], "k_scale", 3, 1u << F32, device, k.dtype != I8, &ks)
        || !whole_tensor(a[3], "v_scale", 3, 1u << F32, device, k.dtype != I8, &vs))
        return NULL;
    if (!shaped(&v, "v", 3, k.shape[0], k.shape[1], k.shape[2]))
        return NULL;
    if (v.shape[3] != k.shape[3]) {
        PyErr_SetString(PyExc_ValueError, "v: as wide as k is expected");
        return NULL;
    }
    if ((ks.there || vs.there) && k.dtype != I8) {
        PyErr_SetString(PyExc_ValueError, "scales belong to an int8 cache");
        return NULL;
    }
    if (!shaped(&ks, "k_scale", 3, k.shape[0], k.shape[1], k.shape[2]) || !shaped(&vs, "v_scale", 3, k.shape[0], k.shape[1], k.shape[2]))
        return NULL;
    hipq_kv_cache *c = PyMem_Calloc(1, sizeof *c);
    if (c == NULL)
        return PyErr_NoMemory();
    c->k = k.p, c->v = v.p, c->k_scale = ks.p, c->v_scale = vs.p;
    c->pages = (int)k.shape[0], c->heads = (int)k.shape[1], c->page = (int)k.shape[2], c->dim = (int)k.shape[3];
    c->quantized = k.dtype == I8, c->type = k.dtype;
    PyObject *o = PyCapsule_New(c, "hipq_kv_cache", free_cache);
    if (o == NULL)
        PyMem_Free(c);
    return o;
}

/* the struct of a capsule for queries of `type` on the capsule's device */
static int cache_for(PyObject *o, const view_t *q, hipq_kv_cache *out)
{
    const hipq_kv_cache *c = PyCapsule_GetPointer(o, "hipq_kv_cache");
    if (c == NULL)
        return 0;
    *out = *c;
    if (!c->quantized && c->type != q->dtype) {
        PyErr_Format(PyExc_ValueError, "q: %s is expected, which the cache has", dtype_names[c->type]);
        return 0;
    }
    out->type = q->dtype;
    return 1;
}

static int cache_device(PyObject *o, int device)
{
    int on;
    if (!whole(o, &on))
        return 0;
    if (on != device)
        PyErr_Format(PyExc_ValueError, "the cache is on device %d, the current one is %d", on, device);
    return on == device;
}

/* cache, its device, q, k, v, positions, slots, table or None, out, q_norm or None, k_norm or None, eps, interleaved */
static PyObject *py_kv_append(ARGS)
{
    (void)self;
    hipq_kv_cache c;
    hipq_kv_append_desc d;
    view_t q, k, v, pos, slots, table, out, qn, kn;
    int device;
    void *st;
    memset(&d, 0, sizeof d);
    if (!expect(n, 13) || !current_device(&device) || !cache_device(a[1], device) || !tensor(a[2], "q", 3, HALVES, device, &q) || !cache_for(a[0], &q, &c)
        || !tensor(a[3], "k", 3, 1u << q.dtype, device, &k) || !tensor(a[4], "v", 3, 1u << q.dtype, device, &v)
        || !whole_tensor(a[5], "positions", 1, 1u << I32, device, 0, &pos) || !whole_tensor(a[6], "slots", 1, 1u << I32, device, 0, &slots)
        || !whole_tensor(a[7], "table", 2, 1u << F32, device, 1, &table) || !tensor(a[8], "out", 3, 1u << q.dtype, device, &out)
        || !whole_tensor(a[9], "q_norm", 1, 1u << q.dtype, device, 1, &qn) || !whole_tensor(a[10], "k_norm", 1, 1u << q.dtype, device, 1, &kn)
        || !number(a[11], &d.eps) || !whole(a[12], &d.interleaved))
        return NULL;
    const int64_t t = q.shape[0];
    if (!shaped(&q, "q", 3, t, q.shape[1], c.dim) || !shaped(&k, "k", 3, t, c.heads, c.dim) || !shaped(&v, "v", 3, t, c.heads, c.dim)
        || !shaped(&pos, "positions", 1, t, 0, 0) || !shaped(&slots, "slots", 1, t, 0, 0) || !shaped(&out, "out", 3, t, q.shape[1], c.dim)
        || !shaped(&qn, "q_norm", 1, c.dim, 0, 0) || !shaped(&kn, "k_norm", 1, c.dim, 0, 0) || !current_stream(&st))
        return NULL;
    if ((out.stride[0] <= 0 && t > 1) || (out.stride[1] <= 0 && q.shape[1] > 1)) {
        PyErr_SetString(PyExc_ValueError, "out: rows overlap");
        return NULL;
    }
    d.q = q.p, d.k = k.p, d.v = v.p, d.q_out = out.p;
    d.q_token = q.stride[0], d.q_head = q.stride[1], d.k_token = k.stride[0], d.k_head = k.stride[1], d.v_token = v.stride[0], d.v_head = v.stride[1];
    d.out_token = out.stride[0], d.out_head = out.stride[1];
    d.positions = pos.p, d.slots = slots.p, d.table = table.p, d.q_norm = qn.p, d.k_norm = kn.p;
    d.tokens = (int)t, d.q_heads = (int)q.shape[1], d.table_rows = (int)table.shape[0], d.rot = (int)table.shape[1];
    CALL(hipq_kv_append(&c, &d, st));
}

/* cache, its device, q, out, starts, lens, blocks, mask or None, most_new, longest or None, scale, allocate: (bytes) -> uint8 tensor */
static PyObject *py_kv_attend(ARGS)
{
    (void)self;
    hipq_kv_cache c;
    hipq_kv_attend_desc d;
    view_t q, o, starts, lens, blocks, mask, w;
    int device;
    void *st;
    memset(&d, 0, sizeof d);
    if (!expect(n, 12) || !current_device(&device) || !cache_device(a[1], device) || !tensor(a[2], "q", 3, HALVES, device, &q) || !cache_for(a[0], &q, &c)
        || !tensor(a[3], "out", 3, 1u << q.dtype, device, &o) || !whole_tensor(a[4], "starts", 1, 1u << I32, device, 0, &starts)
        || !whole_tensor(a[5], "lens", 1, 1u << I32, device, 0, &lens) || !tensor(a[6], "blocks", 2, 1u << I32, device, &blocks)
        || !whole_tensor(a[7], "mask", 1, 1u << I64, device, 1, &mask) || !number(a[10], &d.scale))
        return NULL;
    const long most_new = PyLong_AsLong(a[8]);
    if (most_new == -1 && PyErr_Occurred())
        return NULL;
    d.most_new = most_new < -1 ? -1 : most_new > 0x7fffffff ? 0x7fffffff : (int)most_new;
    const int64_t b = lens.shape[0], t = q.shape[0];
    if (!shaped(&q, "q", 3, t, q.shape[1], c.dim) || !shaped(&o, "out", 3, t, q.shape[1], c.dim) || !shaped(&starts, "starts", 1, b + 1, 0, 0)
        || !shaped(&blocks, "blocks", 2, b, blocks.shape[1], 0) || !shaped(&mask, "mask", 1, t, 0, 0))
        return NULL;
    const int64_t capacity = blocks.shape[1] * c.page;
    if (capacity > 0x7fffffff) {
        PyErr_SetString(PyExc_ValueError, "blocks: a sequence has too many");
        return NULL;
    }
    d.longest = (int)capacity;
    if (a[9] != Py_None) {
        const long long longest = PyLong_AsLongLong(a[9]);
        if (longest == -1 && PyErr_Occurred())
            return NULL;
        d.longest = longest < capacity ? (int)(longest < -1 ? -1 : longest) : (int)capacity;
    }
    if (!current_stream(&st))
        return NULL;
    if ((o.stride[0] <= 0 && t > 1) || (o.stride[1] <= 0 && q.shape[1] > 1)) {
        PyErr_SetString(PyExc_ValueError, "out: rows overlap");
        return NULL;
    }
    if (blocks.stride[0] == 0 && b > 1 && blocks.shape[1] > 0) {
        PyErr_SetString(PyExc_ValueError, "blocks: rows overlap");
        return NULL;
    }
    d.q = q.p, d.o = o.p, d.q_token = q.stride[0], d.q_head = q.stride[1], d.o_token = o.stride[0], d.o_head = o.stride[1];
    d.starts = starts.p, d.lens = lens.p, d.blocks = blocks.p, d.mask = mask.p, d.blocks_stride = blocks.stride[0];
    d.sequences = (int)b, d.tokens = (int)t, d.q_heads = (int)q.shape[1], d.blocks_per_sequence = (int)blocks.shape[1];
    const size_t need = hipq_kv_attend_workspace(&c, &d);
    memset(&w, 0, sizeof w);
    PyObject *workspace = NULL;
    if (need > 0) {
        PyObject *size = PyLong_FromSize_t(need);
        workspace = size ? PyObject_CallOneArg(a[11], size) : NULL;
        Py_XDECREF(size);
        if (workspace == NULL)
            return NULL;
        if (!whole_tensor(workspace, "workspace", 1, 1u << U8, device, 0, &w)) {
            Py_DECREF(workspace);
            return NULL;
        }
    }
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = hipq_kv_attend(&c, &d, w.p, (size_t)w.shape[0], st);
    Py_END_ALLOW_THREADS;
    Py_XDECREF(workspace);
    return PyLong_FromLong(rc);
}

/* a number of a longest sequence, or None: `capacity` */
static int bounded(PyObject *o, int64_t capacity, int *out)
{
    *out = (int)capacity;
    if (o != Py_None) {
        const long long v = PyLong_AsLongLong(o);
        if (v == -1 && PyErr_Occurred())
            return 0;
        *out = v < capacity ? (int)(v < -1 ? -1 : v) : (int)capacity;
    }
    return 1;
}

/* a workspace of `need` bytes from the caller's function; NULL where none is needed */
static int allocated(PyObject *allocate, size_t need, int device, PyObject **workspace, view_t *w)
{
    memset(w, 0, sizeof *w);
    *workspace = NULL;
    if (need == 0)
        return 1;
    PyObject *size = PyLong_FromSize_t(need);
    *workspace = size ? PyObject_CallOneArg(allocate, size) : NULL;
    Py_XDECREF(size);
    if (*workspace != NULL && !whole_tensor(*workspace, "workspace", 1, 1u << U8, device, 0, w))
        Py_CLEAR(*workspace);
    return *workspace != NULL;
}

/* [pages][heads][page] of the cache */
static int of_pages(const view_t *w, const char *name, const hipq_kv_cache *c) { return shaped(w, name, 3, c->pages, c->heads, c->page); }

/* cache, its device, q, weights, out, starts, lens, blocks, mask or None, most_new, longest or None, scale, allocate: (bytes) -> uint8 tensor */
static PyObject *py_kv_weigh(ARGS)
{
    (void)self;
    hipq_kv_cache c;
    hipq_kv_weigh_desc d;
    view_t q, weights, out, starts, lens, blocks, mask, w;
    int device;
    void *st;
    memset(&d, 0, sizeof d);
    if (!expect(n, 13) || !current_device(&device) || !cache_device(a[1], device) || !tensor(a[2], "q", 3, HALVES, device, &q) || !cache_for(a[0], &q, &c)
        || !whole_tensor(a[3], "weights", 3, 1u << F32, device, 0, &weights) || !whole_tensor(a[4], "out", 3, 1u << F32, device, 0, &out)
        || !whole_tensor(a[5], "starts", 1, 1u << I32, device, 0, &starts) || !whole_tensor(a[6], "lens", 1, 1u << I32, device, 0, &lens)
        || !tensor(a[7], "blocks", 2, 1u << I32, device, &blocks) || !whole_tensor(a[8], "mask", 1, 1u << I64, device, 1, &mask) || !number(a[11], &d.scale))
        return NULL;
    const long most_new = PyLong_AsLong(a[9]);
    if (most_new == -1 && PyErr_Occurred())
        return NULL;
    d.most_new = most_new < -1 ? -1 : most_new > 0x7fffffff ? 0x7fffffff : (int)most_new;
    const int64_t b = lens.shape[0], t = q.shape[0], capacity = blocks.shape[1] * c.page;
    if (!shaped(&q, "q", 3, t, q.shape[1], c.dim) || !of_pages(&weights, "weights", &c) || !of_pages(&out, "out", &c) || !shaped(&starts, "starts", 1, b + 1, 0, 0)
        || !shaped(&blocks, "blocks", 2, b, blocks.shape[1], 0) || !shaped(&mask, "mask", 1, t, 0, 0))
        return NULL;
    if (capacity > 0x7fffffff) {
        PyErr_SetString(PyExc_ValueError, "blocks: a sequence has too many");
        return NULL;
    }
    if (!bounded(a[10], capacity, &d.longest) || !current_stream(&st))
        return NULL;
    if (blocks.stride[0] == 0 && b > 1 && blocks.shape[1] > 0) {
        PyErr_SetString(PyExc_ValueError, "blocks: rows overlap");
        return NULL;
    }
    d.q = q.p, d.q_token = q.stride[0], d.q_head = q.stride[1], d.weights = weights.p, d.out = out.p;
    d.starts = starts.p, d.lens = lens.p, d.blocks = blocks.p, d.mask = mask.p, d.blocks_stride = blocks.stride[0];
    d.sequences = (int)b, d.tokens = (int)t, d.q_heads = (int)q.shape[1], d.blocks_per_sequence = (int)blocks.shape[1];
    PyObject *workspace;
    if (!allocated(a[12], hipq_kv_weigh_workspace(&c, &d), device, &workspace, &w))
        return NULL;
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = hipq_kv_weigh(&c, &d, w.p, (size_t)w.shape[0], st);
    Py_END_ALLOW_THREADS;
    Py_XDECREF(workspace);
    return PyLong_FromLong(rc);
}

/* `n` entries of a whole tensor have none in common with `rows` rows of another, `entries` each: 4 bytes an entry */
static int apart(const view_t *v, const char *name, int64_t n, const view_t *u, const char *other, int64_t rows, int64_t entries)
{
    const int64_t lo = (int64_t)(uintptr_t)v->p, at = (int64_t)(uintptr_t)u->p, step = 4 * u->stride[0], behind = lo - (at + 4 * entries);
    const int64_t r = behind < 0 ? 0 : step > 0 ? behind / step + 1 : rows; /* the first row that ends behind lo */
    if (n > 0 && entries > 0 && r < rows && at + r * step < lo + 4 * n) {
        PyErr_Format(PyExc_ValueError, "%s lies over %s", name, other);
        return 0;
    }
    return 1;
}

/* cache, its device, weights, lens, blocks, to, left, kept, budget, recent, first, longest or None, allocate: (bytes) -> uint8 tensor */
static PyObject *py_kv_evict(ARGS)
{
    (void)self;
    hipq_kv_evict_desc d;
    view_t weights, lens, blocks, to, left, kept, w;
    int device;
    void *st;
    memset(&d, 0, sizeof d);
    const hipq_kv_cache *c = n == 13 ? PyCapsule_GetPointer(a[0], "hipq_kv_cache") : NULL;
    if (!expect(n, 13) || c == NULL || !current_device(&device) || !cache_device(a[1], device) || !whole_tensor(a[2], "weights", 3, 1u << F32, device, 0, &weights)
        || !whole_tensor(a[3], "lens", 1, 1u << I32, device, 0, &lens) || !tensor(a[4], "blocks", 2, 1u << I32, device, &blocks)
        || !tensor(a[5], "to", 2, 1u << I32, device, &to) || !whole_tensor(a[6], "left", 1, 1u << I32, device, 0, &left)
        || !whole_tensor(a[7], "kept", 3, 1u << I32, device, 0, &kept) || !whole(a[8], &d.budget) || !whole(a[9], &d.recent) || !whole(a[10], &d.first))
        return NULL;
    const int64_t b = lens.shape[0], capacity = blocks.shape[1] * c->page;
    if (!of_pages(&weights, "weights", c) || !shaped(&blocks, "blocks", 2, b, blocks.shape[1], 0) || !shaped(&to, "to", 2, b, to.shape[1], 0) || !shaped(&left, "left", 1, b, 0, 0)
        || !shaped(&kept, "kept", 3, b, c->heads, d.budget))
        return NULL;
    if (capacity > 0x7fffffff) {
        PyErr_SetString(PyExc_ValueError, "blocks: a sequence has too many");
        return NULL;
    }
    if (!bounded(a[11], capacity, &d.longest) || !current_stream(&st))
        return NULL;
    if (b > 1 && ((blocks.stride[0] == 0 && blocks.shape[1] > 0) || (to.stride[0] == 0 && to.shape[1] > 0))) {
        PyErr_SetString(PyExc_ValueError, "blocks: rows overlap");
        return NULL;
    }
    hipq_kv_cache any = *c;
    if (any.quantized)
        any.type = BF16; /* codes are moved as they are */
    d.weights = weights.p, d.lens = lens.p, d.blocks = blocks.p, d.to = to.p, d.left = left.p, d.kept = kept.p;
    d.blocks_stride = blocks.stride[0], d.to_stride = to.stride[0], d.sequences = (int)b, d.blocks_per_sequence = (int)blocks.shape[1], d.to_per_sequence = (int)to.shape[1];
    const size_t need = hipq_kv_evict_workspace(&any, &d);
    /* what is written lies apart from what the launches read, but for left in the place of lens; a call that is refused for something else says that */
    const int64_t many = b * c->heads * d.budget, pool = (int64_t)c->pages * c->heads * c->page;
    const struct {
        const view_t *v;
        const char *name;
        int64_t rows, entries;
    } read[5] = {{&lens, "lens", 1, b}, {&blocks, "blocks", b, blocks.shape[1]}, {&to, "to", b, to.shape[1]}, {&left, "left", 1, b}, {&kept, "kept", 1, many}};
    for (int i = 0; i < 5 && hipq_last_error()[0] == 0; i++)
        if (!apart(&weights, "weights", pool, read[i].v, read[i].name, read[i].rows, read[i].entries)
            || (i < 4 && !apart(&kept, "kept", many, read[i].v, read[i].name, read[i].rows, read[i].entries))
            || (i < 3 && (i > 0 || left.p != lens.p) && !apart(&left, "left", b, read[i].v, read[i].name, read[i].rows, read[i].entries)))
            return NULL;
    PyObject *workspace;
    if (!allocated(a[12], need, device, &workspace, &w))
        return NULL;
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = hipq_kv_evict(&any, &d, w.p, (size_t)w.shape[0], st);
    Py_END_ALLOW_THREADS;
    Py_XDECREF(workspace);
    return PyLong_FromLong(rc);
}

/* logits, uniform, temperature, top_k, top_p, min_p (each or None), out */
static PyObject *py_sample(ARGS)
{
    (void)self;
    view_t x, u, t, k, p, m, out;
    int device;
    void *st;
    if (!expect(n, 7) || !current_device(&device) || !tensor(a[0], "logits", 2, HALVES | 1u << F32, device, &x)
        || !whole_tensor(a[1], "uniform", 1, 1u << F32, device, 0, &u) || !whole_tensor(a[2], "temperature", 1, 1u << F32, device, 1, &t)
        || !whole_tensor(a[3], "top_k", 1, 1u << I32, device, 1, &k) || !whole_tensor(a[4], "top_p", 1, 1u << F32, device, 1, &p)
        || !whole_tensor(a[5], "min_p", 1, 1u << F32, device, 1, &m) || !whole_tensor(a[6], "out", 1, 1u << I64, device, 0, &out))
        return NULL;
    const int64_t r = x.shape[0];
    if (!shaped(&u, "uniform", 1, r, 0, 0) || !shaped(&t, "temperature", 1, r, 0, 0) || !shaped(&k, "top_k", 1, r, 0, 0) || !shaped(&p, "top_p", 1, r, 0, 0)
        || !shaped(&m, "min_p", 1, r, 0, 0) || !shaped(&out, "out", 1, r, 0, 0) || !current_stream(&st))
        return NULL;
    CALL(hipq_sample(x.p, x.dtype, (int)r, (int)x.shape[1], x.stride[0], u.p, t.p, k.p, p.p, m.p, out.p, st));
}

/* logits, out, tokens, lens, prompt_lens, repetition, frequency, presence, bias_tokens, bias, allowed (all but the first two: or None) */
static PyObject *py_penalize(ARGS)
{
    (void)self;
    hipq_penalize_desc d;
    view_t x, out, tokens, lens, prompt, rep, freq, pres, at, bias, bits;
    int device;
    void *st;
    memset(&d, 0, sizeof d);
    if (!expect(n, 11) || !current_device(&device) || !tensor(a[0], "logits", 2, HALVES | 1u << F32, device, &x) || !tensor(a[1], "out", 2, 1u << x.dtype, device, &out)
        || !tensor_or_none(a[2], "tokens", 2, 1u << I32, device, &tokens) || !whole_tensor(a[3], "lens", 1, 1u << I32, device, 1, &lens)
        || !whole_tensor(a[4], "prompt_lens", 1, 1u << I32, device, 1, &prompt) || !whole_tensor(a[5], "repetition", 1, 1u << F32, device, 1, &rep)
        || !whole_tensor(a[6], "frequency", 1, 1u << F32, device, 1, &freq) || !whole_tensor(a[7], "presence", 1, 1u << F32, device, 1, &pres)
        || !tensor_or_none(a[8], "bias_tokens", 2, 1u << I32, device, &at) || !tensor_or_none(a[9], "bias", 2, 1u << F32, device, &bias)
        || !tensor_or_none(a[10], "allowed", 2, 1u << I32, device, &bits))
        return NULL;
    const int64_t r = x.shape[0], v = x.shape[1];
    if (!shaped(&out, "out", 2, r, v, 0) || !shaped(&tokens, "tokens", 1, r, 0, 0) || !shaped(&lens, "lens", 1, r, 0, 0) || !shaped(&prompt, "prompt_lens", 1, r, 0, 0)
        || !shaped(&rep, "repetition", 1, r, 0, 0) || !shaped(&freq, "frequency", 1, r, 0, 0) || !shaped(&pres, "presence", 1, r, 0, 0)
        || !shaped(&at, "bias_tokens", 1, r, 0, 0) || !shaped(&bias, "bias", 2, r, at.shape[1], 0) || !shaped(&bits, "allowed", 2, r, (v + 31) / 32, 0)
        || !current_stream(&st))
        return NULL;
    if (bias.there && r > 1 && bias.stride[0] != at.stride[0]) {
        PyErr_SetString(PyExc_ValueError, "bias: rows as far apart as those of bias_tokens are expected");
        return NULL;
    }
    if (!tokens.there && (lens.there || prompt.there || rep.there || freq.there || pres.there)) {
        PyErr_SetString(PyExc_ValueError, "tokens: a tensor is expected where lengths or penalties are given");
        return NULL;
    }
    if (at.there != bias.there) {
        PyErr_SetString(PyExc_ValueError, "bias and bias_tokens belong together");
        return NULL;
    }
    d.logits = x.p, d.out = out.p, d.stride = x.stride[0], d.out_stride = out.stride[0];
    d.tokens = tokens.p, d.lens = lens.p, d.prompt_lens = prompt.p, d.repetition = rep.p, d.frequency = freq.p, d.presence = pres.p;
    d.bias_tokens = at.p, d.bias = bias.p, d.allowed = bits.p;
    d.tokens_stride = tokens.stride[0], d.bias_stride = at.stride[0], d.allowed_stride = bits.stride[0];
    d.type = x.dtype, d.rows = (int)r, d.vocab = (int)v, d.longest = (int)tokens.shape[1], d.biases = (int)at.shape[1];
    CALL(hipq_penalize(&d, st));
}

#define METHOD(NAME) {#NAME, (PyCFunction)(void (*)(void))py_##NAME, METH_FASTCALL, NULL}
static PyMethodDef methods[] = {
    METHOD(init),        METHOD(conv2d_run),  METHOD(add_u8),      METHOD(eltwise_u8),    METHOD(relu_u8),       METHOD(concat_u8), METHOD(softmax_u8),
    METHOD(pool_u8),     METHOD(quantize_u8), METHOD(quantize_i8), METHOD(dequantize_u8), METHOD(dequantize_i8),
    METHOD(types),       METHOD(w4_workspace), METHOD(w4_run),     METHOD(experts_workspace), METHOD(experts_run), METHOD(kv_cache),      METHOD(kv_append),     METHOD(kv_attend), METHOD(sample),
    METHOD(kv_weigh),    METHOD(kv_evict),    METHOD(penalize),
    {NULL, NULL, 0, NULL},
};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "hipq_calls", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit_hipq_calls(void)
{
    s_data_ptr = PyUnicode_InternFromString("data_ptr");
    s_shape = PyUnicode_InternFromString("shape");
    s_numel = PyUnicode_InternFromString("numel");
    s_dtype = PyUnicode_InternFromString("dtype");
    s_stride = PyUnicode_InternFromString("stride");
    s_get_device = PyUnicode_InternFromString("get_device");
    return s_data_ptr && s_shape && s_numel && s_dtype && s_stride && s_get_device ? PyModule_Create(&module) : NULL;
}
