// The host side of the entry points that a program calls many times a second, as a CPython extension: the checks of
// the operands and the call into libb200dnn in one step.  What bounds a call on a few hundred tokens is not the GPU but
// the interpreter: the same checks and a ctypes call of 17 arguments in Python took 11 us for matmul_ and 13 us for
// sdpa before the library was entered, against 4 to 8 us of device time; here they take 0.7.  A call of 363 tokens
// through a 240 x 1496 projection went from 11.6 to 4.9 us, an attention of 42 x 3 windows of 196 from 13.0 to 7.9.
//
// Each function takes the forms a program ordinarily passes and answers None for every other one, which the Python
// route then takes, declines or refuses exactly as it always has; nothing is decided here that it would decide
// differently.  The library is entered without the interpreter's lock, as ctypes does.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>
#include <string.h>

#include "../../include/b200dnn.h"

typedef struct {
    int64_t ptr, shape[4], stride[4], size;
    int nd, code;
} Arr;

static PyObject *s_ptr, *s_dtype, *s_shape, *s_strides, *s_c, *s_rot, *s_interleaved, *s_gain, *s_freq;
static PyObject *dt_f16, *dt_f32, *dt_i32;   // numpy's own dtype objects; an equal one that is not the same goes the Python route

static int (*p_gemm)(b200_ctx*, int64_t, int64_t, int64_t, const void*, int64_t, const void*, int64_t, const void*, void*,
                     int64_t, int, int, int64_t, int64_t, int64_t, int64_t);
static int (*p_gemv)(b200_ctx*, int64_t, int64_t, const void*, int64_t, const void*, const void*, int, void*, int, int);
static int (*p_attention)(b200_ctx*, int64_t, int64_t, int64_t, int64_t, int64_t, const b200_strided4*, const b200_strided4*,
                          const b200_strided4*, const b200_strided4*, const b200_strided4*, int, float);
static int (*p_layernorm)(b200_ctx*, int64_t, int64_t, const void*, int, void*, int, float*, float*, const void*, const void*,
                          float);
static int (*p_conv)(b200_ctx*, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t,
                     int64_t, int64_t, int64_t, const void*, const void*, const void*, void*, int, int);

static int (*p_rotary)(b200_ctx*, int64_t, int64_t, int64_t, int64_t, const b200_strided4*, const b200_strided4*, const uint64_t*, int64_t, int,
                       float, const int32_t*, int64_t, int64_t, const int32_t*, const int32_t*);
static int (*p_append)(b200_ctx*, const b200_cache8*, int64_t, int64_t, const b200_strided4*, const b200_strided4*, const int32_t*, const int32_t*);
static int (*p_read)(b200_ctx*, const b200_cache8*, int, int64_t, int64_t, const int32_t*, const int32_t*, const b200_strided4*, int);
static int (*p_cachesdpa)(b200_ctx*, const b200_cache8*, int64_t, int64_t, int64_t, const b200_strided4*, const b200_strided4*, int, float, int,
                          const int32_t*, const int32_t*);
static int (*p_matmul4)(b200_ctx*, const b200_q4*, int64_t, const void*, int64_t, const void*, void*, int64_t, int, int);

static int (*p_normrotary)(b200_ctx*, int64_t, int64_t, int64_t, int64_t, const b200_strided4*, const b200_strided4*, const void*, int, int64_t,
                           int64_t, float, const uint64_t*, int64_t, int, float, const int32_t*, int64_t, int64_t, const int32_t*, const int32_t*);
static int (*p_packed)(b200_ctx*, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, const b200_strided4*, const b200_strided4*,
                       const b200_strided4*, const b200_strided4*, int, float, int, const int32_t*, const int32_t*);
static int (*p_beamselect)(b200_ctx*, int64_t, int64_t, int64_t, int64_t, const void*, int, int64_t, int64_t, const float*, const int32_t*, int64_t,
                           float*, int32_t*, int32_t*);
static int (*p_reorder)(b200_ctx*, const b200_cache8*, int64_t, int64_t, int64_t, int32_t*, int64_t, const int32_t*, int64_t, int64_t, const int32_t*,
                        const int32_t*);

static int64_t attr_int(PyObject* o, PyObject* name, int* ok) {
    PyObject* v = PyObject_GetAttr(o, name);
    int64_t r = 0;
    if (v && PyLong_Check(v)) r = PyLong_AsLongLong(v);
    else *ok = 0;
    Py_XDECREF(v);
    return r;
}

static int ints(PyObject* t, int64_t* out, int n) {   // a tuple of n integers
    if (!t || !PyTuple_Check(t) || PyTuple_GET_SIZE(t) != n) return 0;
    for (int i = 0; i < n; ++i) {
        PyObject* v = PyTuple_GET_ITEM(t, i);
        if (!PyLong_Check(v)) return 0;
        out[i] = PyLong_AsLongLong(v);
    }
    return !PyErr_Occurred();
}

enum { CODE_I32 = 100 };   // of an array of counts or page numbers

// A DeviceArray of fp16, fp32 or int32 with one to four axes and a size that is a number here; 0 for anything else.
static int load_any(PyObject* o, Arr* a) {
    int ok;
    PyObject* dt = PyObject_GetAttr(o, s_dtype);
    a->code = dt == dt_f16 ? B200_F16 : dt == dt_f32 ? B200_F32 : dt == dt_i32 ? CODE_I32 : -1;
    Py_XDECREF(dt);   // numpy holds the ones that count
    ok = a->code >= 0;
    a->ptr = ok ? attr_int(o, s_ptr, &ok) : 0;
    if (ok) {
        PyObject *sh = PyObject_GetAttr(o, s_shape), *st = PyObject_GetAttr(o, s_strides);
        a->nd = sh && PyTuple_Check(sh) ? (int)PyTuple_GET_SIZE(sh) : 0;
        ok = a->nd >= 1 && a->nd <= 4 && ints(sh, a->shape, a->nd) && ints(st, a->stride, a->nd);
        a->size = 1;
        for (int i = 0; ok && i < a->nd; ++i) ok = a->shape[i] >= 0 && !__builtin_mul_overflow(a->size, a->shape[i], &a->size);
        Py_XDECREF(sh);
        Py_XDECREF(st);
    }
    if (PyErr_Occurred()) {   // an attribute that is missing or out of range: the Python route meets it again
        PyErr_Clear();
        ok = 0;
    }
    return ok;
}

static int load(PyObject* o, Arr* a) { return load_any(o, a) && a->code != CODE_I32; }   // of fp16 or fp32

static int dense(const Arr* a) {
    int64_t acc = 1;
    for (int i = 0; i < a->nd; ++i) {
        if (a->shape[i] != 1 && a->stride[i] != acc) return 0;
        acc *= a->shape[i];
    }
    return 1;
}
static int64_t colmajor(const Arr* a) {   // leading dimension of a 2-D view with a unit first stride, else -1
    if (a->shape[0] != 1 && a->stride[0] != 1) return -1;
    const int64_t ld = a->shape[1] != 1 ? a->stride[1] : (a->shape[0] > 1 ? a->shape[0] : 1);
    return ld >= a->shape[0] ? ld : -1;
}
// A dense vector of n elements of one type, or None: 1 with *p set, else 0.
static int vector(PyObject* o, int code, int64_t n, const void** p) {
    Arr a;
    *p = NULL;
    if (o == Py_None) return 1;
    if (!load(o, &a) || a.code != code || a.size != n || !dense(&a)) return 0;
    *p = (const void*)a.ptr;
    return 1;
}

#define P(a) ((void*)(a).ptr)
#define ENTER(rc, call)          \
    do {                         \
        Py_BEGIN_ALLOW_THREADS   \
        rc = (call);             \
        Py_END_ALLOW_THREADS     \
    } while (0)

static b200_ctx* handle(PyObject* o) {
    if (!PyLong_Check(o)) return NULL;
    void* p = PyLong_AsVoidPtr(o);
    if (!p && PyErr_Occurred()) PyErr_Clear();
    return (b200_ctx*)p;
}
static int epilogue(PyObject* o) { return PyLong_Check(o) ? (int)PyLong_AsLong(o) : -1; }

// matmul(handle, out, A, B, bias, epilogue)
static PyObject* h_matmul(PyObject* self, PyObject* const* v, Py_ssize_t n) {
    Arr out, A, B;
    const void* bias;
    b200_ctx* c;
    int epi, rc;
    if (n != 6 || !(c = handle(v[0])) || (epi = epilogue(v[5])) < 0) Py_RETURN_NONE;
    if (!load(v[1], &out) || !load(v[2], &A) || !load(v[3], &B) || out.nd != 2 || A.nd != 2 || B.nd != 2) Py_RETURN_NONE;
    const int64_t M = A.shape[0], K = A.shape[1], N = B.shape[1], lim = (int64_t)1 << 31;
    const int64_t lda = colmajor(&A), ldb = colmajor(&B), ldo = colmajor(&out);
    if (A.code != B.code || B.shape[0] != K || out.shape[0] != M || out.shape[1] != N || lda < 0 || ldb < 0 || ldo < 0 ||
        M < 1 || N < 1 || K < 1 || M >= lim || N >= lim || K >= lim || !vector(v[4], A.code, M, &bias))
        Py_RETURN_NONE;
    if (N == 1) {
        if (!dense(&B) || !dense(&out) || (out.code != B200_F32 && out.code != A.code)) Py_RETURN_NONE;
        ENTER(rc, p_gemv(c, M, K, P(A), lda, P(B), bias, A.code, P(out), out.code, epi));
    } else {
        if (A.code != B200_F16) Py_RETURN_NONE;
        ENTER(rc, p_gemm(c, M, N, K, P(A), lda, P(B), ldb, bias, P(out), ldo, out.code, epi, 1, 0, 0, 0));
    }
    return PyLong_FromLong(rc);
}

static void strided(const Arr* a, b200_strided4* s) {
    s->ptr = (const void*)a->ptr;
    for (int i = 0; i < 4; ++i) s->stride[i] = a->stride[i];
}

// sdpa(handle, out, q, k, v, bias, scale)
static PyObject* h_sdpa(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    Arr out, q, k, v, b;
    b200_ctx* c;
    int rc;
    if (n != 7 || !(c = handle(a[0])) || !PyFloat_Check(a[6])) Py_RETURN_NONE;
    if (!load(a[1], &out) || !load(a[2], &q) || !load(a[3], &k) || !load(a[4], &v)) Py_RETURN_NONE;
    if (out.nd != 4 || q.nd != 4 || k.nd != 4 || v.nd != 4 || q.code != B200_F16 || k.code != B200_F16 || v.code != B200_F16)
        Py_RETURN_NONE;
    const int64_t E = q.shape[0], Lq = q.shape[1], H = q.shape[2], B = q.shape[3], Lk = k.shape[1], lim = (int64_t)1 << 31;
    if (E < 8 || E > 128 || E % 8 || Lq < 1 || Lk < 1 || Lq >= lim || Lk >= lim || H < 1 || H > 65535 || B < 1 || B > 65535)
        Py_RETURN_NONE;
    for (int i = 0; i < 4; ++i)
        if (k.shape[i] != (i == 1 ? Lk : q.shape[i]) || v.shape[i] != k.shape[i] || out.shape[i] != q.shape[i]) Py_RETURN_NONE;
    if (q.stride[0] != 1 || k.stride[0] != 1 || v.stride[0] != 1 || out.stride[0] != 1) Py_RETURN_NONE;
    b200_strided4 sq, sk, sv, so, sb;
    strided(&q, &sq);
    strided(&k, &sk);
    strided(&v, &sv);
    strided(&out, &so);
    const int masked = a[5] != Py_None;
    if (masked) {
        const int64_t want[4] = {Lk, Lq, H, B};
        if (!load(a[5], &b) || b.nd != 4 || b.code != B200_F16) Py_RETURN_NONE;
        for (int i = 0; i < 4; ++i) {
            if (b.shape[i] != 1 && b.shape[i] != want[i]) Py_RETURN_NONE;
            if (b.shape[i] == 1) b.stride[i] = 0;   // a size-1 axis broadcasts
        }
        strided(&b, &sb);
    }
    const float scale = (float)PyFloat_AS_DOUBLE(a[6]);
    ENTER(rc, p_attention(c, E, Lq, Lk, H, B, &sq, &sk, &sv, masked ? &sb : NULL, &so, out.code, scale));
    return PyLong_FromLong(rc);
}

// layernorm(handle, out, mean, rstd, a, gamma, beta, C, eps)
static PyObject* h_layernorm(PyObject* self, PyObject* const* v, Py_ssize_t n) {
    Arr out, mean, rstd, a;
    const void *gamma, *beta;
    b200_ctx* c;
    int rc;
    if (n != 9 || !(c = handle(v[0])) || !PyLong_Check(v[7]) || !PyFloat_Check(v[8])) Py_RETURN_NONE;
    if (!load(v[1], &out) || !load(v[2], &mean) || !load(v[3], &rstd) || !load(v[4], &a)) Py_RETURN_NONE;
    int over;
    const int64_t C = PyLong_AsLongLongAndOverflow(v[7], &over), total = a.size;
    if (over || C < 1 || total % C || out.size != total || !dense(&a) || !dense(&out) || !dense(&mean) || !dense(&rstd)) Py_RETURN_NONE;
    const int64_t groups = total / C;
    if (mean.code != B200_F32 || rstd.code != B200_F32 || mean.size < groups || rstd.size < groups) Py_RETURN_NONE;
    if (!vector(v[5], a.code, C, &gamma) || !vector(v[6], a.code, C, &beta)) Py_RETURN_NONE;
    const float eps = (float)PyFloat_AS_DOUBLE(v[8]);
    ENTER(rc, p_layernorm(c, groups, C, P(a), a.code, P(out), out.code, (float*)P(mean), (float*)P(rstd), gamma, beta, eps));
    return PyLong_FromLong(rc);
}

// convolution(handle, out, x, w, bias, stride, padding, dilation, groups, act)
static PyObject* h_convolution(PyObject* self, PyObject* const* v, Py_ssize_t n) {
    Arr out, x, w;
    int64_t s[2], p[2], d[2];
    b200_ctx* c;
    int act, rc, over;
    if (n != 10 || !(c = handle(v[0])) || !PyLong_Check(v[8]) || (act = epilogue(v[9])) < 0) Py_RETURN_NONE;
    const int64_t groups = PyLong_AsLongLongAndOverflow(v[8], &over);
    if (over || !ints(v[5], s, 2) || !ints(v[6], p, 2) || !ints(v[7], d, 2)) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    if (!load(v[1], &out) || !load(v[2], &x) || !load(v[3], &w) || out.nd != 4 || x.nd != 4 || w.nd != 4) Py_RETURN_NONE;
    if (x.code != B200_F16 || w.code != B200_F16 || !dense(&x) || !dense(&w) || !dense(&out)) Py_RETURN_NONE;
    const void* bias;
    if (!vector(v[4], B200_F16, w.shape[3], &bias)) Py_RETURN_NONE;
    if (groups < 1 || w.shape[2] * groups != x.shape[2] || w.shape[3] % groups || out.shape[2] != w.shape[3] || out.shape[3] != x.shape[3])
        Py_RETURN_NONE;
    const int64_t lim = (int64_t)1 << 31;   // past it (no extent of a real convolution) the sums below could wrap
    for (int i = 0; i < 2; ++i) {
        if (x.shape[i] >= lim || w.shape[i] >= lim || s[i] >= lim || p[i] >= lim || d[i] >= lim) Py_RETURN_NONE;
        const int64_t span = x.shape[i] + 2 * p[i] - d[i] * (w.shape[i] - 1) - 1;
        if (s[i] < 1 || d[i] < 1 || p[i] < 0 || span < 0 || out.shape[i] != span / s[i] + 1) Py_RETURN_NONE;
    }
    ENTER(rc, p_conv(c, x.shape[0], x.shape[1], x.shape[2], x.shape[3], w.shape[0], w.shape[1], w.shape[3], s[0], s[1], p[0], p[1],
                     d[0], d[1], groups, P(x), P(w), bias, P(out), out.code, act));
    return PyLong_FromLong(rc);
}

// A dense int32 number for each of B sequences, or None: 1 with *p set, else 0.
static int counts(PyObject* o, int64_t B, const int32_t** p) {
    Arr a;
    *p = NULL;
    if (o == Py_None) return 1;
    if (!load_any(o, &a) || a.code != CODE_I32 || a.size != B || !dense(&a)) return 0;
    *p = (const int32_t*)a.ptr;
    return 1;
}
// The structure that a Python object keeps for the library, copied.
static int kept(PyObject* o, void* to, Py_ssize_t size) {
    Py_buffer b;
    PyObject* c = PyObject_GetAttr(o, s_c);
    int ok = 0;
    if (c && PyObject_GetBuffer(c, &b, PyBUF_SIMPLE) == 0) {
        if ((ok = b.len == size)) memcpy(to, b.buf, (size_t)size);
        PyBuffer_Release(&b);
    }
    Py_XDECREF(c);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        ok = 0;
    }
    return ok;
}
// A cache with a table of page numbers, (pages a sequence, B).
static int cached(PyObject* o, PyObject* table, int64_t B, b200_cache8* c) {
    Arr t;
    if (!kept(o, c, sizeof *c) || !load_any(table, &t) || t.code != CODE_I32 || t.nd != 2 || t.shape[1] != B || (t.shape[0] != 1 && t.stride[0] != 1)) return 0;
    c->table = (const int32_t*)t.ptr;
    c->width = t.shape[0];
    c->table_ld = B > 1 ? t.stride[1] : (t.shape[0] > 1 ? t.shape[0] : 1);
    return 1;
}
// An array of heads, (E, L, H, B) of fp16 or fp32.
static int heads(PyObject* o, Arr* a, int64_t E, int64_t H, b200_strided4* s) {
    if (!load(o, a) || a->nd != 4 || a->shape[0] != E || a->shape[2] != H) return 0;
    strided(a, s);
    return 1;
}

// A plan of positions: 1 with its numbers, else 0.
typedef struct {
    int64_t rot, freq;
    int interleaved;
    float gain;
} Plan;
static int rotation(PyObject* o, Plan* p) {
    int ok = 1;
    p->rot = attr_int(o, s_rot, &ok);
    p->interleaved = attr_int(o, s_interleaved, &ok) != 0;
    PyObject *gain = PyObject_GetAttr(o, s_gain), *freq = PyObject_GetAttr(o, s_freq);
    p->freq = freq ? attr_int(freq, s_ptr, &ok) : 0;
    p->gain = 0.f;
    if (gain && PyFloat_Check(gain)) p->gain = (float)PyFloat_AS_DOUBLE(gain);
    else ok = 0;
    Py_XDECREF(gain);
    Py_XDECREF(freq);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        ok = 0;
    }
    return ok && p->freq;
}
// Heads to turn, x to out, by lengths: 1 where both are what the library takes.
static int turned(PyObject* po, PyObject* px, PyObject* plens, PyObject* pnews, Arr* out, Arr* x, const int32_t** lens, const int32_t** news) {
    if (plens == Py_None || !load(po, out) || !load(px, x)) return 0;
    if (out->nd != 4 || x->nd != 4 || out->code != B200_F16 || x->code != B200_F16) return 0;
    for (int i = 0; i < 4; ++i)
        if (out->shape[i] != x->shape[i]) return 0;
    return counts(plens, x->shape[3], lens) && counts(pnews, x->shape[3], news);
}

// rotary(handle, plan, out, x, lens, news)
static PyObject* h_rotary(PyObject* self, PyObject* const* v, Py_ssize_t n) {
    Arr out, x;
    Plan plan;
    const int32_t *lens, *news;
    b200_ctx* c;
    int rc;
    if (n != 6 || !(c = handle(v[0])) || !turned(v[2], v[3], v[4], v[5], &out, &x, &lens, &news) || !rotation(v[1], &plan)) Py_RETURN_NONE;
    b200_strided4 so, sx;
    strided(&out, &so);
    strided(&x, &sx);
    ENTER(rc, p_rotary(c, x.shape[0], x.shape[1], x.shape[2], x.shape[3], &sx, &so, (const uint64_t*)plan.freq, plan.rot, plan.interleaved, plan.gain,
                       NULL, 0, 0, lens, news));
    return PyLong_FromLong(rc);
}

// normrotary(handle, plan, out, x, weight, eps, split, lens, news)
static PyObject* h_normrotary(PyObject* self, PyObject* const* v, Py_ssize_t n) {
    Arr out, x, w;
    Plan plan;
    const int32_t *lens, *news;
    b200_ctx* c;
    int rc, over = 0;
    if (n != 9 || !(c = handle(v[0])) || !PyFloat_Check(v[5]) || !turned(v[2], v[3], v[7], v[8], &out, &x, &lens, &news) || !rotation(v[1], &plan))
        Py_RETURN_NONE;
    const int64_t E = x.shape[0], H = x.shape[2];
    int64_t split = -1, ld = 0;
    memset(&w, 0, sizeof w);
    if (v[6] != Py_None) {
        if (!PyLong_Check(v[6]) || v[4] == Py_None) Py_RETURN_NONE;
        split = PyLong_AsLongLongAndOverflow(v[6], &over);
        if (over || split < 0 || split > H) Py_RETURN_NONE;
    }
    if (v[4] != Py_None) {
        if (!load(v[4], &w) || w.nd > 2 || w.shape[0] != E || (E > 1 && w.stride[0] != 1)) Py_RETURN_NONE;
        const int64_t columns = w.nd == 1 ? 1 : w.shape[1];
        if (columns != (split >= 0 ? 2 : columns == 1 ? 1 : H)) Py_RETURN_NONE;
        ld = columns == 1 ? 0 : w.stride[1];
    }
    b200_strided4 so, sx;
    strided(&out, &so);
    strided(&x, &sx);
    ENTER(rc, p_normrotary(c, E, x.shape[1], H, x.shape[3], &sx, &so, P(w), w.code, ld, split, (float)PyFloat_AS_DOUBLE(v[5]),
                           (const uint64_t*)plan.freq, plan.rot, plan.interleaved, plan.gain, NULL, 0, 0, lens, news));
    return PyLong_FromLong(rc);
}

// cacheappend(handle, cache, k, v, table, lens, news)
static PyObject* h_cacheappend(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    Arr k, v;
    b200_cache8 cache;
    b200_strided4 sk, sv;
    const int32_t *lens, *news;
    b200_ctx* c;
    int rc;
    if (n != 7 || !(c = handle(a[0])) || !load(a[2], &k) || k.nd != 4 || k.code != B200_F16 || !cached(a[1], a[4], k.shape[3], &cache)) Py_RETURN_NONE;
    if (k.shape[0] != cache.E || k.shape[2] != cache.H || !heads(a[3], &v, cache.E, cache.H, &sv) || v.code != B200_F16) Py_RETURN_NONE;
    if (v.shape[1] != k.shape[1] || v.shape[3] != k.shape[3] || a[5] == Py_None || !counts(a[5], k.shape[3], &lens) || !counts(a[6], k.shape[3], &news))
        Py_RETURN_NONE;
    strided(&k, &sk);
    ENTER(rc, p_append(c, &cache, k.shape[1], k.shape[3], &sk, &sv, lens, news));
    return PyLong_FromLong(rc);
}

// cacheread(handle, out, cache, whether the values, table, lens, starts)
static PyObject* h_cacheread(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    Arr out;
    b200_cache8 cache;
    b200_strided4 so;
    const int32_t *lens, *starts;
    b200_ctx* c;
    int rc;
    if (n != 7 || !(c = handle(a[0])) || !PyBool_Check(a[3]) || !load(a[1], &out) || out.nd != 4 || !cached(a[2], a[4], out.shape[3], &cache)) Py_RETURN_NONE;
    if (out.shape[0] != cache.E || out.shape[2] != cache.H || a[5] == Py_None || !counts(a[5], out.shape[3], &lens) || !counts(a[6], out.shape[3], &starts))
        Py_RETURN_NONE;
    strided(&out, &so);
    ENTER(rc, p_read(c, &cache, a[3] == Py_True, out.shape[1], out.shape[3], starts, lens, &so, out.code));
    return PyLong_FromLong(rc);
}

// cachesdpa(handle, out, q, cache, table, lens, news, scale, causal)
static PyObject* h_cachesdpa(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    Arr out, q;
    b200_cache8 cache;
    b200_strided4 sq, so;
    const int32_t *lens, *news;
    b200_ctx* c;
    int rc;
    if (n != 9 || !(c = handle(a[0])) || !PyFloat_Check(a[7]) || !PyBool_Check(a[8])) Py_RETURN_NONE;
    if (!load(a[2], &q) || q.nd != 4 || q.code != B200_F16 || !cached(a[3], a[4], q.shape[3], &cache)) Py_RETURN_NONE;
    if (q.shape[0] != cache.E || cache.H < 1 || q.shape[2] % cache.H || !heads(a[1], &out, cache.E, q.shape[2], &so)) Py_RETURN_NONE;
    if (out.shape[1] != q.shape[1] || out.shape[3] != q.shape[3] || a[5] == Py_None || !counts(a[5], q.shape[3], &lens) || !counts(a[6], q.shape[3], &news))
        Py_RETURN_NONE;
    strided(&q, &sq);
    const float scale = (float)PyFloat_AS_DOUBLE(a[7]);
    ENTER(rc, p_cachesdpa(c, &cache, q.shape[1], q.shape[2], q.shape[3], &sq, &so, out.code, scale, a[8] == Py_True, lens, news));
    return PyLong_FromLong(rc);
}

// matmul4(handle, out, W, B, bias, epilogue)
static PyObject* h_matmul4(PyObject* self, PyObject* const* v, Py_ssize_t n) {
    Arr out, B;
    const void* bias;
    b200_ctx* c;
    int epi, rc;
    if (n != 6 || !(c = handle(v[0])) || (epi = epilogue(v[5])) < 0 || !load(v[1], &out) || !load(v[3], &B) || out.nd != 2 || B.nd != 2) Py_RETURN_NONE;
    b200_q4 W;
    if (!kept(v[2], &W, sizeof W) || B.code != B200_F16 || B.shape[0] != W.K || out.shape[0] != W.M || out.shape[1] != B.shape[1]) Py_RETURN_NONE;
    const int64_t ldb = colmajor(&B), ldo = colmajor(&out);
    if (ldb < 0 || ldo < 0 || !vector(v[4], B200_F16, W.M, &bias)) Py_RETURN_NONE;
    ENTER(rc, p_matmul4(c, &W, B.shape[1], P(B), ldb, bias, P(out), ldo, out.code, epi));
    return PyLong_FromLong(rc);
}

// binddecode(rotary, append, read, attention, product): a decoder's entry points, as addresses
static PyObject* h_binddecode(PyObject* self, PyObject* args) {
    unsigned long long a, b, c, d, e;
    if (!PyArg_ParseTuple(args, "KKKKK", &a, &b, &c, &d, &e)) return NULL;
    *(void**)&p_rotary = (void*)(uintptr_t)a;
    *(void**)&p_append = (void*)(uintptr_t)b;
    *(void**)&p_read = (void*)(uintptr_t)c;
    *(void**)&p_cachesdpa = (void*)(uintptr_t)d;
    *(void**)&p_matmul4 = (void*)(uintptr_t)e;
    Py_RETURN_NONE;
}

// packedsdpa(handle, out, q, k, v, starts, kstarts, scale, causal)
static PyObject* h_packedsdpa(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    Arr x[4], starts;                  // out, q, k, v
    b200_strided4 s[4];
    const int32_t* kstarts;
    b200_ctx* c;
    int rc;
    if (n != 9 || !(c = handle(a[0])) || !PyFloat_Check(a[7]) || !PyBool_Check(a[8])) Py_RETURN_NONE;
    for (int i = 0; i < 4; ++i) {
        if (!load(a[1 + i], &x[i]) || x[i].nd != 3 || (i > 0 && x[i].code != B200_F16)) Py_RETURN_NONE;
        x[i].stride[3] = 0;
        strided(&x[i], &s[i]);
    }
    for (int i = 0; i < 3; ++i)
        if (x[0].shape[i] != x[1].shape[i] || x[2].shape[i] != x[3].shape[i]) Py_RETURN_NONE;
    const int64_t E = x[1].shape[0], N = x[1].shape[1], Hq = x[1].shape[2], Nk = x[2].shape[1], H = x[2].shape[2];
    if (x[2].shape[0] != E || (H ? Hq % H != 0 : Hq != 0)) Py_RETURN_NONE;
    if (!load_any(a[5], &starts) || starts.code != CODE_I32 || starts.size < 1 || !dense(&starts)) Py_RETURN_NONE;
    if (!counts(a[6], starts.size, &kstarts)) Py_RETURN_NONE;
    if (a[6] == Py_None) {
        if (Nk < N) Py_RETURN_NONE;
        kstarts = (const int32_t*)starts.ptr;
    }
    ENTER(rc, p_packed(c, E, N, Nk, Hq, H, starts.size - 1, &s[1], &s[2], &s[3], &s[0], x[0].code, (float)PyFloat_AS_DOUBLE(a[7]), a[8] == Py_True,
                       (const int32_t*)starts.ptr, kstarts));
    return PyLong_FromLong(rc);
}

// A dense (rows, columns) array of one type, or (where it may be) None: 1 with *p set, else 0.
static int matrix(PyObject* o, int code, int64_t rows, int64_t columns, int may, void* p) {
    Arr a;
    memset(p, 0, sizeof(void*));
    if (o == Py_None) return may;
    if (!load_any(o, &a) || a.code != code || a.nd != 2 || a.shape[0] != rows || a.shape[1] != columns || !dense(&a)) return 0;
    *(void**)p = P(a);
    return 1;
}

// beamselect(handle, best, parents, tokens, logits, scores, ended, pad)
static PyObject* h_beamselect(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    Arr best, x, scores;
    int32_t *parents, *tokens, *ended;
    b200_ctx* c;
    int rc, over;
    if (n != 8 || !(c = handle(a[0])) || !PyLong_Check(a[7]) || !load(a[1], &best) || !load(a[4], &x) || !load(a[5], &scores)) Py_RETURN_NONE;
    const int64_t pad = PyLong_AsLongLongAndOverflow(a[7], &over);
    if (over || best.nd != 2 || best.code != B200_F32 || scores.nd != 2 || scores.code != B200_F32 || !dense(&best) || !dense(&scores)) Py_RETURN_NONE;
    const int64_t K = scores.shape[0], B = scores.shape[1], N = best.shape[0], V = x.shape[0];
    if (best.shape[1] != B || (V > 1 && x.stride[0] != 1)) Py_RETURN_NONE;
    if (x.nd == 3 ? x.shape[1] != K || x.shape[2] != B : x.nd != 2 || x.shape[1] != K * B) Py_RETURN_NONE;
    if (!matrix(a[2], CODE_I32, N, B, 0, &parents) || !matrix(a[3], CODE_I32, N, B, 0, &tokens) || !matrix(a[6], CODE_I32, K, B, 1, &ended)) Py_RETURN_NONE;
    ENTER(rc, p_beamselect(c, V, K, B, N, P(x), x.code, x.stride[1], x.nd == 3 ? x.stride[2] : K * x.stride[1], (const float*)P(scores), ended, pad,
                           (float*)P(best), parents, tokens));
    return PyLong_FromLong(rc);
}

// cachereorder(handle, caches, table, own, parents, lens)
static PyObject* h_cachereorder(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    enum { MOST = 128 };
    b200_cache8 caches[MOST];
    Arr t[2], parents;                 // the table, the beams' own
    const int32_t* lens;
    b200_ctx* c;
    int rc;
    if (n != 6 || !(c = handle(a[0])) || !PyList_Check(a[1]) || PyList_GET_SIZE(a[1]) > MOST) Py_RETURN_NONE;
    const Py_ssize_t count = PyList_GET_SIZE(a[1]);
    if (!load_any(a[4], &parents) || parents.code != CODE_I32 || parents.nd != 2 || !dense(&parents)) Py_RETURN_NONE;
    const int64_t K = parents.shape[0], B = parents.shape[1];
    for (int i = 0; i < 2; ++i)
        if (!load_any(a[2 + i], &t[i]) || t[i].code != CODE_I32 || t[i].nd != 2 || t[i].shape[1] != K * B || (t[i].shape[0] != 1 && t[i].stride[0] != 1))
            Py_RETURN_NONE;
    if (t[0].shape[0] != t[1].shape[0] || a[5] == Py_None || !counts(a[5], K * B, &lens)) Py_RETURN_NONE;
    for (Py_ssize_t i = 0; i < count; ++i)
        if (!kept(PyList_GET_ITEM(a[1], i), &caches[i], sizeof caches[i])) Py_RETURN_NONE;
    int64_t ld[2];
    for (int i = 0; i < 2; ++i) ld[i] = K * B > 1 ? t[i].stride[1] : (t[i].shape[0] > 1 ? t[i].shape[0] : 1);
    ENTER(rc, p_reorder(c, caches, count, K, B, (int32_t*)P(t[0]), ld[0], (const int32_t*)P(t[1]), ld[1], t[0].shape[0], (const int32_t*)P(parents), lens));
    return PyLong_FromLong(rc);
}

// bindaround(norm and rotation, packed attention, beams' choice, reordered caches): the entry points around a decoder's step, as addresses
static PyObject* h_bindaround(PyObject* self, PyObject* args) {
    unsigned long long a, b, c, d;
    if (!PyArg_ParseTuple(args, "KKKK", &a, &b, &c, &d)) return NULL;
    *(void**)&p_normrotary = (void*)(uintptr_t)a;
    *(void**)&p_packed = (void*)(uintptr_t)b;
    *(void**)&p_beamselect = (void*)(uintptr_t)c;
    *(void**)&p_reorder = (void*)(uintptr_t)d;
    Py_RETURN_NONE;
}

// bind(gemm, gemv, attention, layernorm, convolution): the library's entry points, as addresses
static PyObject* h_bind(PyObject* self, PyObject* args) {
    unsigned long long a, b, c, d, e;
    if (!PyArg_ParseTuple(args, "KKKKK", &a, &b, &c, &d, &e)) return NULL;
    *(void**)&p_gemm = (void*)(uintptr_t)a;
    *(void**)&p_gemv = (void*)(uintptr_t)b;
    *(void**)&p_attention = (void*)(uintptr_t)c;
    *(void**)&p_layernorm = (void*)(uintptr_t)d;
    *(void**)&p_conv = (void*)(uintptr_t)e;
    Py_RETURN_NONE;
}

static PyMethodDef methods[] = {{"bind", h_bind, METH_VARARGS, NULL},
                                {"matmul", (PyCFunction)(void (*)(void))h_matmul, METH_FASTCALL, NULL},
                                {"sdpa", (PyCFunction)(void (*)(void))h_sdpa, METH_FASTCALL, NULL},
                                {"layernorm", (PyCFunction)(void (*)(void))h_layernorm, METH_FASTCALL, NULL},
                                {"convolution", (PyCFunction)(void (*)(void))h_convolution, METH_FASTCALL, NULL},
                                {"binddecode", h_binddecode, METH_VARARGS, NULL},
                                {"rotary", (PyCFunction)(void (*)(void))h_rotary, METH_FASTCALL, NULL},
                                {"bindaround", h_bindaround, METH_VARARGS, NULL},
                                {"packedsdpa", (PyCFunction)(void (*)(void))h_packedsdpa, METH_FASTCALL, NULL},
                                {"beamselect", (PyCFunction)(void (*)(void))h_beamselect, METH_FASTCALL, NULL},
                                {"cachereorder", (PyCFunction)(void (*)(void))h_cachereorder, METH_FASTCALL, NULL},
                                {"normrotary", (PyCFunction)(void (*)(void))h_normrotary, METH_FASTCALL, NULL},
                                {"cacheappend", (PyCFunction)(void (*)(void))h_cacheappend, METH_FASTCALL, NULL},
                                {"cacheread", (PyCFunction)(void (*)(void))h_cacheread, METH_FASTCALL, NULL},
                                {"cachesdpa", (PyCFunction)(void (*)(void))h_cachesdpa, METH_FASTCALL, NULL},
                                {"matmul4", (PyCFunction)(void (*)(void))h_matmul4, METH_FASTCALL, NULL},
                                {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "hostcalls", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit_hostcalls(void) {
    s_ptr = PyUnicode_InternFromString("ptr");
    s_dtype = PyUnicode_InternFromString("dtype");
    s_shape = PyUnicode_InternFromString("shape");
    s_strides = PyUnicode_InternFromString("strides");
    s_c = PyUnicode_InternFromString("_c");
    s_rot = PyUnicode_InternFromString("rot");
    s_interleaved = PyUnicode_InternFromString("interleaved");
    s_gain = PyUnicode_InternFromString("gain");
    s_freq = PyUnicode_InternFromString("freq");
    if (!s_ptr || !s_dtype || !s_shape || !s_strides || !s_c || !s_rot || !s_interleaved || !s_gain || !s_freq) return NULL;
    PyObject* np = PyImport_ImportModule("numpy");
    if (!np) return NULL;
    dt_f16 = PyObject_CallMethod(np, "dtype", "s", "float16");
    dt_f32 = PyObject_CallMethod(np, "dtype", "s", "float32");
    dt_i32 = PyObject_CallMethod(np, "dtype", "s", "int32");
    Py_DECREF(np);
    if (!dt_f16 || !dt_f32 || !dt_i32) return NULL;
    return PyModule_Create(&module);
}
