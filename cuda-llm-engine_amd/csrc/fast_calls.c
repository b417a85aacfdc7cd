/* The Python face's calls of the operators a decode step issues most, as one native function each:
 * tensor checks, the current stream and the C-ABI call without the interpreter between them. A
 * small operator takes 2 to 3 us on the GPU; its checks in Python and its ctypes call took longer.
 *
 * Every function answers the C-ABI's status, or None where an argument is not plainly right (not a
 * torch.Tensor itself, another device or dtype, not contiguous, too small, a stream that is neither
 * None nor a number, a number out of range): the caller then takes the checks in __init__.py, which
 * accept or name what is wrong. Nothing is kept between calls. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <limits.h>
#include <stdint.h>

#include "llmk.h"

static PyObject *tensor_type, *half_dtype, *int_dtype, *float_dtype, *get_device, *get_stream,
    *e4m3_dtype;
static PyObject *s_is_cuda, *s_dtype, *s_is_contiguous, *s_numel, *s_data_ptr, *s_get_device;

/* The device address of t when it is a contiguous CUDA torch.Tensor of this dtype with at least
 * `least` elements; 0 otherwise, with no exception set. (A tensor of no elements has no address
 * to give: 0 as well.) */
static void* address(PyObject* t, PyObject* dtype, long long least) {
  if ((PyObject*)Py_TYPE(t) != tensor_type) return NULL;
  long long n = -1;
  void* p = NULL;
  PyObject* v = PyObject_GetAttr(t, s_is_cuda);
  int ok = v == Py_True;
  Py_XDECREF(v);
  if (ok) {
    v = PyObject_GetAttr(t, s_dtype);
    ok = v == dtype;
    Py_XDECREF(v);
  }
  if (ok) {
    v = PyObject_CallMethodNoArgs(t, s_is_contiguous);
    ok = v == Py_True;
    Py_XDECREF(v);
  }
  if (ok && (v = PyObject_CallMethodNoArgs(t, s_numel))) {
    n = PyLong_AsLongLong(v);
    Py_DECREF(v);
  }
  if (ok && n >= least && n > 0 && (v = PyObject_CallMethodNoArgs(t, s_data_ptr))) {
    p = PyLong_AsVoidPtr(v);
    Py_DECREF(v);
  }
  if (PyErr_Occurred()) {
    PyErr_Clear();
    p = NULL;
  }
  return p;
}

/* address() of a tensor of this device, and how many elements it has. The device number of a tensor that
 * is not on a GPU is -1. */
static void* address_on(PyObject* t, PyObject* dtype, long long least, long long device,
                        long long* numel) {
  if ((PyObject*)Py_TYPE(t) != tensor_type) return NULL;
  long long n = -1, at = -1;
  void* p = NULL;
  PyObject* v = PyObject_CallMethodNoArgs(t, s_get_device);
  if (v) {
    at = PyLong_AsLongLong(v);
    Py_DECREF(v);
  }
  int ok = at == device && at >= 0;
  if (ok) {
    v = PyObject_GetAttr(t, s_dtype);
    ok = v == dtype;
    Py_XDECREF(v);
  }
  if (ok) {
    v = PyObject_CallMethodNoArgs(t, s_is_contiguous);
    ok = v == Py_True;
    Py_XDECREF(v);
  }
  if (ok && (v = PyObject_CallMethodNoArgs(t, s_numel))) {
    n = PyLong_AsLongLong(v);
    Py_DECREF(v);
  }
  if (ok && n >= least && n > 0 && (v = PyObject_CallMethodNoArgs(t, s_data_ptr))) {
    p = PyLong_AsVoidPtr(v);
    Py_DECREF(v);
  }
  if (PyErr_Occurred()) {
    PyErr_Clear();
    p = NULL;
  }
  if (numel) *numel = n;
  return p;
}

/* torch's current stream for None, the number itself for a number. */
static int stream_of(PyObject* o, void** stream) {
  PyObject* v = NULL;
  if (o == Py_None) {
    PyObject* dev = PyObject_CallNoArgs(get_device);
    if (dev) v = PyObject_CallOneArg(get_stream, dev);
    Py_XDECREF(dev);
  } else if (PyLong_CheckExact(o)) {
    v = Py_NewRef(o);
  }
  if (v) {
    *stream = PyLong_AsVoidPtr(v);
    Py_DECREF(v);
  }
  const int ok = v && !PyErr_Occurred();
  if (!ok) PyErr_Clear();
  return ok;
}

/* The current device, -1 if it cannot be told, and the stream as stream_of() gives it. */
static long long device_and_stream(PyObject* o, void** stream) {
  long long at = -1;
  PyObject *dev = PyObject_CallNoArgs(get_device), *v = NULL;
  if (dev) {
    at = PyLong_AsLongLong(dev);
    v = o == Py_None ? PyObject_CallOneArg(get_stream, dev)
                     : PyLong_CheckExact(o) ? Py_NewRef(o) : NULL;
    Py_DECREF(dev);
  }
  if (v) {
    *stream = PyLong_AsVoidPtr(v);
    Py_DECREF(v);
  }
  const int ok = v && !PyErr_Occurred();
  if (!ok) PyErr_Clear();
  return ok ? at : -1;
}

/* A Python int from 0 to INT_MAX, the products of two of which fit a long long. */
static int count_of(PyObject* o, int* out) {
  if (!PyLong_CheckExact(o)) return 0;
  const long v = PyLong_AsLong(o);
  if (PyErr_Occurred()) PyErr_Clear();
  else if (v >= 0 && v <= INT_MAX) {
    *out = (int)v;
    return 1;
  }
  return 0;
}

static int float_of(PyObject* o, float* out) {
  if (!PyFloat_CheckExact(o)) return 0;
  *out = (float)PyFloat_AS_DOUBLE(o);
  return 1;
}

#define COUNT(name, at) \
  int name;             \
  if (!count_of(args[at], &name)) Py_RETURN_NONE
#define FLOAT(name, at) \
  float name;           \
  if (!float_of(args[at], &name)) Py_RETURN_NONE
#define TENSOR(type, name, at, dtype, least)          \
  type* name = (type*)address(args[at], dtype, least); \
  if (!name) Py_RETURN_NONE
#define HALF(name, at, least) TENSOR(uint16_t, name, at, half_dtype, least)
#define STREAM(at)    \
  void* stream;       \
  if (!stream_of(args[at], &stream)) Py_RETURN_NONE
#define ANSWER(call)                   \
  int status;                          \
  Py_BEGIN_ALLOW_THREADS status = call; \
  Py_END_ALLOW_THREADS return PyLong_FromLong(status)
#define FUNCTION(name, n)                                                            \
  static PyObject* name(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {   \
    (void)self;                                                                      \
    if (nargs != n) Py_RETURN_NONE;

FUNCTION(rmsnorm, 7)
  COUNT(rows, 3);
  COUNT(hidden, 4);
  FLOAT(eps, 5);
  HALF(x, 0, (long long)rows * hidden);
  HALF(w, 1, hidden);
  HALF(out, 2, (long long)rows * hidden);
  STREAM(6);
  ANSWER(llmk_rmsnorm(x, w, out, rows, hidden, eps, stream));
}

FUNCTION(add_rmsnorm, 8)
  COUNT(rows, 4);
  COUNT(hidden, 5);
  FLOAT(eps, 6);
  const long long n = (long long)rows * hidden;
  HALF(residual, 0, n);
  HALF(x, 1, n);
  HALF(w, 2, hidden);
  HALF(out, 3, n);
  STREAM(7);
  ANSWER(llmk_add_rmsnorm(residual, x, w, out, rows, hidden, eps, stream));
}

FUNCTION(residual_add, 5)
  COUNT(n, 3);
  HALF(a, 0, n);
  HALF(b, 1, n);
  HALF(out, 2, n);
  STREAM(4);
  ANSWER(llmk_residual_add(a, b, out, (size_t)n, stream));
}

FUNCTION(swiglu, 5)
  COUNT(n, 3);
  HALF(gate, 0, n);
  HALF(up, 1, n);
  HALF(out, 2, n);
  STREAM(4);
  ANSWER(llmk_swiglu(gate, up, out, (size_t)n, stream));
}

FUNCTION(swiglu_rows, 5)
  COUNT(rows, 2);
  COUNT(inter, 3);
  if (inter == 0) Py_RETURN_NONE;
  HALF(gate_up, 0, 2LL * rows * inter);
  HALF(out, 1, (long long)rows * inter);
  STREAM(4);
  ANSWER(llmk_swiglu_rows(gate_up, out, rows, inter, stream));
}

FUNCTION(linear, 8)
  COUNT(T, 4);
  COUNT(in, 5);
  COUNT(out, 6);
  if (in == 0 || out == 0) Py_RETURN_NONE;
  if (!PyLong_CheckExact(args[0])) Py_RETURN_NONE;
  llmk_blas* h = (llmk_blas*)PyLong_AsVoidPtr(args[0]);
  if (!h) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  HALF(x, 1, (long long)T * in);
  HALF(w, 2, (long long)out * in);
  HALF(y, 3, (long long)T * out);
  STREAM(7);
  ANSWER(llmk_linear(h, x, w, y, T, in, out, stream));
}

FUNCTION(linear_rows_residual, 7)
  COUNT(T, 3);
  COUNT(in, 4);
  COUNT(out, 5);
  HALF(x, 0, (long long)T * in);
  HALF(w, 1, (long long)out * in);
  HALF(residual, 2, (long long)T * out);
  STREAM(6);
  ANSWER(llmk_linear_rows_residual(x, w, residual, T, in, out, stream));
}

FUNCTION(linear_rows_swiglu, 9)
  COUNT(T, 5);
  COUNT(in, 6);
  COUNT(inter, 7);
  FLOAT(eps, 2);
  if (inter > INT_MAX / 2) Py_RETURN_NONE;
  HALF(x, 0, (long long)T * in);
  HALF(norm_w, 1, in);
  HALF(w, 3, 2LL * inter * in);
  HALF(act, 4, (long long)T * inter);
  STREAM(8);
  ANSWER(llmk_linear_rows_swiglu(x, norm_w, eps, w, act, T, in, inter, stream));
}

FUNCTION(attention_decode_fast, 15)
  COUNT(n, 7);
  COUNT(max_pages, 8);
  COUNT(page_size, 9);
  COUNT(heads, 10);
  COUNT(kv_heads, 11);
  COUNT(head_dim, 12);
  COUNT(splits, 13);
  if (n > 65535 || heads > 65535 || head_dim > 65535) Py_RETURN_NONE;
  const long long rows = (long long)n * heads * head_dim;
  const size_t floats = llmk_attention_decode_fast_workspace_floats(n, heads, splits);
  if (floats > (size_t)LLONG_MAX) Py_RETURN_NONE;
  HALF(q, 0, rows);
  HALF(k_pool, 1, 0);
  HALF(v_pool, 2, 0);
  TENSOR(int32_t, tables, 3, int_dtype, (long long)n * max_pages);
  TENSOR(int32_t, lens, 4, int_dtype, n);
  HALF(out, 5, rows);
  TENSOR(float, workspace, 6, float_dtype, splits > 1 ? (long long)floats : 0);
  STREAM(14);
  ANSWER(llmk_attention_decode_fast(q, k_pool, v_pool, tables, lens, out, workspace, n, max_pages,
                                    page_size, heads, kv_heads, head_dim, splits, stream));
}

/* Tensors of the calls below: on the current device, `here`. OPT: or None. The stream is argument `at`. */
#define HERE(at)                                               \
  void* stream;                                                \
  const long long here = device_and_stream(args[at], &stream); \
  if (here < 0) Py_RETURN_NONE
#define TENSOR_ON(type, name, at, dtype, least)                           \
  type* name = (type*)address_on(args[at], dtype, least, here, NULL);      \
  if (!name) Py_RETURN_NONE
#define OPT_ON(type, name, at, dtype, least)                                                 \
  type* name = args[at] == Py_None ? NULL                                                    \
                                   : (type*)address_on(args[at], dtype, least, here, NULL);  \
  if (!name && args[at] != Py_None) Py_RETURN_NONE
/* A cache's pool and scales, which have to fit each other, at `at` and at + 1. */
#define POOL(name, at, kv_heads, page_size, head_dim)                                           \
  long long name##_n = 0, name##_scales = 0;                                                    \
  uint8_t* name##_pool = (uint8_t*)address_on(args[at], e4m3_dtype, 0, here, &name##_n);        \
  float* name##_scale = (float*)address_on(args[at + 1], float_dtype, 0, here, &name##_scales); \
  if (!name##_pool || !name##_scale || name##_scales % kv_heads ||                              \
      name##_n / ((long long)page_size * head_dim) != name##_scales ||                          \
      name##_n % ((long long)page_size * head_dim))                                             \
  Py_RETURN_NONE
/* The tensors of a batch, at `at` and the two behind. */
#define BATCH(at)                                                                 \
  TENSOR_ON(int32_t, tables, at, int_dtype, (long long)n_seqs * max_pages);       \
  OPT_ON(int32_t, starts, (at) + 1, int_dtype, (long long)n_seqs + 1);            \
  TENSOR_ON(int32_t, lens, (at) + 2, int_dtype, n_seqs)

FUNCTION(kv8_append, 19)
  COUNT(ld, 1);
  COUNT(n_rows, 11);
  COUNT(n_seqs, 12);
  COUNT(max_pages, 13);
  COUNT(page_size, 14);
  COUNT(heads, 15);
  COUNT(kv_heads, 16);
  COUNT(head_dim, 17);
  if (!n_rows || !page_size || !heads || !kv_heads || !head_dim || heads > 65535 ||
      kv_heads > 65535 || head_dim > 65535 || page_size > 65535)
    Py_RETURN_NONE;
  const long long width = (heads + 2LL * kv_heads) * head_dim;
  if (ld < width) Py_RETURN_NONE;
  HERE(18);
  TENSOR_ON(uint16_t, qkv, 0, half_dtype, (n_rows - 1LL) * ld + width);
  TENSOR_ON(uint16_t, q_out, 2, half_dtype, (long long)n_rows * heads * head_dim);
  POOL(k, 3, kv_heads, page_size, head_dim);
  POOL(v, 5, kv_heads, page_size, head_dim);
  BATCH(7);
  TENSOR_ON(float, inv_freq, 10, float_dtype, head_dim / 2);
  ANSWER(llmk_kv8_append(qkv, ld, q_out, k_pool, k_scale, v_pool, v_scale, tables, starts, lens,
                         inv_freq, n_rows, n_seqs, max_pages, page_size, heads, kv_heads, head_dim,
                         stream));
}

FUNCTION(kv8_gather, 16)
  COUNT(n_rows, 9);
  COUNT(n_seqs, 10);
  COUNT(max_pages, 11);
  COUNT(page_size, 12);
  COUNT(kv_heads, 13);
  COUNT(head_dim, 14);
  if (!n_rows || !page_size || !kv_heads || !head_dim || kv_heads > 65535 || head_dim > 65535 ||
      page_size > 65535)
    Py_RETURN_NONE;
  HERE(15);
  POOL(k, 0, kv_heads, page_size, head_dim);
  POOL(v, 2, kv_heads, page_size, head_dim);
  BATCH(4);
  TENSOR_ON(uint16_t, k_out, 7, half_dtype, (long long)n_rows * kv_heads * head_dim);
  TENSOR_ON(uint16_t, v_out, 8, half_dtype, (long long)n_rows * kv_heads * head_dim);
  ANSWER(llmk_kv8_gather(k_pool, k_scale, v_pool, v_scale, tables, starts, lens, k_out, v_out,
                         n_rows, n_seqs, max_pages, page_size, kv_heads, head_dim, stream));
}

FUNCTION(kv8_attention, 19)
  COUNT(n_rows, 10);
  COUNT(n_seqs, 11);
  COUNT(max_rows, 12);
  COUNT(max_pages, 13);
  COUNT(page_size, 14);
  COUNT(heads, 15);
  COUNT(kv_heads, 16);
  COUNT(head_dim, 17);
  if (!n_rows || !page_size || !heads || !kv_heads || !head_dim || heads > 65535 ||
      kv_heads > 65535 || head_dim > 65535 || page_size > 65535)
    Py_RETURN_NONE;
  HERE(18);
  TENSOR_ON(uint16_t, q, 0, half_dtype, (long long)n_rows * heads * head_dim);
  POOL(k, 1, kv_heads, page_size, head_dim);
  POOL(v, 3, kv_heads, page_size, head_dim);
  BATCH(5);
  TENSOR_ON(uint16_t, out, 8, half_dtype, (long long)n_rows * heads * head_dim);
  OPT_ON(float, workspace, 9, float_dtype,
         (long long)llmk_kv8_attention_workspace_floats(head_dim));
  ANSWER(llmk_kv8_attention(q, k_pool, k_scale, v_pool, v_scale, tables, starts, lens, out,
                            workspace, n_rows, n_seqs, max_rows, max_pages, page_size, heads,
                            kv_heads, head_dim, stream));
}

FUNCTION(verify_drafts, 14)
  COUNT(n_rows, 10);
  COUNT(n_seqs, 11);
  COUNT(vocab, 12);
  if (!n_rows || !vocab) Py_RETURN_NONE;
  const long long given = args[3] != Py_None ? n_rows : 0;
  const size_t floats = llmk_verify_drafts_workspace_floats(n_rows, n_seqs, vocab);
  if (floats > (size_t)LLONG_MAX) Py_RETURN_NONE;
  HERE(13);
  TENSOR_ON(uint16_t, logits, 0, half_dtype, (long long)n_rows * vocab);
  OPT_ON(uint16_t, draft_logits, 1, half_dtype, given * vocab);
  OPT_ON(int32_t, drafts, 2, int_dtype, given);
  OPT_ON(int32_t, starts, 3, int_dtype, (long long)n_seqs + 1);
  OPT_ON(float, temperature, 4, float_dtype, n_seqs);
  OPT_ON(float, accept_u, 5, float_dtype, given);
  TENSOR_ON(float, sample_u, 6, float_dtype, n_seqs);
  TENSOR_ON(int32_t, n_accepted, 7, int_dtype, n_seqs);
  TENSOR_ON(int32_t, tokens, 8, int_dtype, n_rows);
  TENSOR_ON(float, workspace, 9, float_dtype, (long long)floats);
  ANSWER(llmk_verify_drafts(logits, draft_logits, drafts, starts, temperature, accept_u, sample_u,
                            n_accepted, tokens, workspace, n_rows, n_seqs, vocab, stream));
}

/* setup(torch.Tensor, torch.float16, torch.int32, torch.float32, current device, current stream
 * of a device, torch.float8_e4m3fn) */
static PyObject* setup(PyObject* self, PyObject* args) {
  (void)self;
  PyObject** to[] = {&tensor_type, &half_dtype, &int_dtype, &float_dtype,
                     &get_device,  &get_stream, &e4m3_dtype};
  PyObject* from[7];
  if (!PyArg_ParseTuple(args, "OOOOOOO", &from[0], &from[1], &from[2], &from[3], &from[4], &from[5],
                        &from[6]))
    return NULL;
  for (int i = 0; i < 7; ++i) {
    PyObject* old = *to[i];
    *to[i] = Py_NewRef(from[i]);
    Py_XDECREF(old);
  }
  Py_RETURN_NONE;
}

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, NULL}
static PyMethodDef methods[] = {METHOD(rmsnorm),
                                METHOD(add_rmsnorm),
                                METHOD(residual_add),
                                METHOD(swiglu),
                                METHOD(swiglu_rows),
                                METHOD(linear),
                                METHOD(linear_rows_residual),
                                METHOD(linear_rows_swiglu),
                                METHOD(attention_decode_fast),
                                METHOD(kv8_append),
                                METHOD(kv8_gather),
                                METHOD(kv8_attention),
                                METHOD(verify_drafts),
                                {"setup", setup, METH_VARARGS, NULL},
                                {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast_calls", NULL, -1, methods,
                                    NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__fast_calls(void) {
  if (!(s_is_cuda = PyUnicode_InternFromString("is_cuda")) ||
      !(s_dtype = PyUnicode_InternFromString("dtype")) ||
      !(s_is_contiguous = PyUnicode_InternFromString("is_contiguous")) ||
      !(s_numel = PyUnicode_InternFromString("numel")) ||
      !(s_data_ptr = PyUnicode_InternFromString("data_ptr")) ||
      !(s_get_device = PyUnicode_InternFromString("get_device")))
    return NULL;
  return PyModule_Create(&module);
}
