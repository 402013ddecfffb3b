/* Host-side packing of one step's request list into the int32 upload buffer of
 * lms_build_step_indices, as a CPython extension module (lmserve_b200._packer).
 *
 * LMServe's model worker walks the request list in Python and builds one list per index array
 * (runtime/worker/llm_worker/model_worker.py:330-407); converting those lists element by element
 * is what its per-step preparation costs.  This module walks the same request objects in C and
 * writes
 *     [input_len | filled_token_len | context_len | len(block_ids)]   (batch entries each)
 *     block_ids of every request, concatenated
 *     input_ids of every request, concatenated
 * straight into a caller-provided buffer (the pinned staging memory).  The requests are any
 * objects with the InferInput attributes of proto/worker.proto:40-47; block_ids and input_ids are
 * any sequences of integers.  Sorting stays with the caller (list.sort, as the reference does).
 *
 * The other small helpers of the Python layer live here too: flattening of block maps, calls of
 * write plans, and the argument checks of the attention-layer calls.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "../../include/lmserve_kv.h"

/* Attribute names, interned once at module start-up (a lookup by C string builds a new str
 * object per call). */
static PyObject *s_input_len, *s_filled_token_len, *s_context_len, *s_block_ids, *s_input_ids;

/* Value of a Python int: the one-digit ("compact") form that every id, length and position here
 * has is read in place; anything else takes the general conversion. */
static inline int as_i32(PyObject* v, int32_t* out, const char* what) {
  long long x;
#if PY_VERSION_HEX >= 0x030C0000
  if (PyLong_CheckExact(v) && PyUnstable_Long_IsCompact((const PyLongObject*)v)) {
    x = (long long)PyUnstable_Long_CompactValue((const PyLongObject*)v);
  } else
#endif
  {
    x = PyLong_AsLongLong(v);
    if (x == -1 && PyErr_Occurred()) return -1;
  }
  if (x < INT32_MIN || x > INT32_MAX) {
    PyErr_Format(PyExc_OverflowError, "%s does not fit 32 bits", what);
    return -1;
  }
  *out = (int32_t)x;
  return 0;
}

static int get_i32(PyObject* obj, PyObject* name, const char* what, int32_t* out) {
  PyObject* v = PyObject_GetAttr(obj, name);
  if (!v) return -1;
  const int rc = as_i32(v, out, what);
  Py_DECREF(v);
  return rc;
}

/* Copies the integers of `seq` (already a list or tuple) to dst[0..n). */
static int copy_ints(PyObject* fast, Py_ssize_t n, int32_t* dst, const char* what) {
  PyObject** items = PySequence_Fast_ITEMS(fast);
  for (Py_ssize_t i = 0; i < n; ++i)
    if (as_i32(items[i], dst + i, what)) return -1;
  return 0;
}

/* pack(inputs, out) -> (batch, total_tokens, total_blocks, prefill_input_len, num_prefill, num_decode,
 *                       prefill_blocks, decode_blocks)
 * `out` is a writable, C-contiguous buffer of int32 (a numpy array); ValueError when it is too
 * small or when a request is inconsistent, with the messages of the pure-Python packer. */
static PyObject* pack(PyObject* self, PyObject* args) {
  PyObject* inputs;
  Py_buffer out;
  if (!PyArg_ParseTuple(args, "Ow*", &inputs, &out)) return NULL;
  PyObject* result = NULL;
  PyObject* reqs = PySequence_Fast(inputs, "inputs must be a sequence of requests");
  PyObject** blocks = NULL;
  PyObject** ids = NULL;
  Py_ssize_t batch = 0;
  if (!reqs) goto done;
  if (out.itemsize != 4 && out.itemsize != 1) {
    PyErr_SetString(PyExc_TypeError, "out must be an int32 (or byte) buffer");
    goto done;
  }
  batch = PySequence_Fast_GET_SIZE(reqs);
  {
    const Py_ssize_t cap = out.len / 4;
    int32_t* buf = (int32_t*)out.buf;
    if (4 * batch > cap) {
      PyErr_Format(PyExc_ValueError, "step needs at least %zd int32 words of staging, the buffer has %zd",
                   4 * batch, cap);
      goto done;
    }
    blocks = (PyObject**)PyMem_Calloc(batch ? batch : 1, sizeof(PyObject*));
    ids = (PyObject**)PyMem_Calloc(batch ? batch : 1, sizeof(PyObject*));
    if (!blocks || !ids) {
      PyErr_NoMemory();
      goto done;
    }
    long long total_tokens = 0, total_blocks = 0, prefill_len = 0, n_pre = 0, n_dec = 0;
    long long prefill_blocks = 0, decode_blocks = 0;
    for (Py_ssize_t b = 0; b < batch; ++b) {
      PyObject* r = PySequence_Fast_GET_ITEM(reqs, b);
      int32_t q, filled, ctx;
      if (get_i32(r, s_input_len, "input_len", &q) ||
          get_i32(r, s_filled_token_len, "filled_token_len", &filled) ||
          get_i32(r, s_context_len, "context_len", &ctx))
        goto done;
      PyObject* a = PyObject_GetAttr(r, s_block_ids);
      if (!a) goto done;
      blocks[b] = PySequence_Fast(a, "block_ids must be a sequence");
      Py_DECREF(a);
      if (!blocks[b]) goto done;
      a = PyObject_GetAttr(r, s_input_ids);
      if (!a) goto done;
      ids[b] = PySequence_Fast(a, "input_ids must be a sequence");
      Py_DECREF(a);
      if (!ids[b]) goto done;
      const Py_ssize_t n_ids = PySequence_Fast_GET_SIZE(ids[b]);
      if (n_ids != q) {
        PyErr_Format(PyExc_ValueError, "request %zd: input_len %d but %zd input ids", b, (int)q, n_ids);
        goto done;
      }
      if ((long long)ctx - filled != q) {
        PyErr_Format(PyExc_ValueError,
                     "request %zd: context_len - filled_token_len = %lld but input_len = %d", b,
                     (long long)ctx - filled, (int)q);
        goto done;
      }
      const Py_ssize_t nb = PySequence_Fast_GET_SIZE(blocks[b]);
      if (q > 1) {
        prefill_len += q;
        ++n_pre;
        prefill_blocks += nb;
      } else if (q == 1) {
        ++n_dec;
        decode_blocks += nb;
      }
      buf[b] = q;
      buf[batch + b] = filled;
      buf[2 * batch + b] = ctx;
      buf[3 * batch + b] = (int32_t)nb;
      total_tokens += q > 0 ? q : 0;
      total_blocks += nb;
    }
    const long long need = 4 * (long long)batch + total_blocks + total_tokens;
    if (need > cap || total_blocks > INT32_MAX || total_tokens > INT32_MAX) {
      PyErr_Format(PyExc_ValueError, "step needs %lld int32 words of staging, the buffer has %zd", need, cap);
      goto done;
    }
    int32_t* dst = buf + 4 * batch;
    for (Py_ssize_t b = 0; b < batch; ++b) {
      const Py_ssize_t nb = PySequence_Fast_GET_SIZE(blocks[b]);
      if (copy_ints(blocks[b], nb, dst, "block_ids")) goto done;
      dst += nb;
    }
    for (Py_ssize_t b = 0; b < batch; ++b) {
      const Py_ssize_t n = PySequence_Fast_GET_SIZE(ids[b]);
      if (copy_ints(ids[b], n, dst, "input_ids")) goto done;
      dst += n;
    }
    result = Py_BuildValue("(nLLLLLLL)", batch, total_tokens, total_blocks, prefill_len, n_pre, n_dec,
                           prefill_blocks, decode_blocks);
  }
done:
  if (blocks)
    for (Py_ssize_t b = 0; b < batch; ++b) Py_XDECREF(blocks[b]);
  if (ids)
    for (Py_ssize_t b = 0; b < batch; ++b) Py_XDECREF(ids[b]);
  PyMem_Free(blocks);
  PyMem_Free(ids);
  Py_XDECREF(reqs);
  PyBuffer_Release(&out);
  return result;
}

/* flatten_dict(src_to_dst, out) -> n: writes the (src, dst) pairs of {src: [dst, ...]} - the
 * argument of LMServe's copy_blocks (ops/cache_ops.py:8-15) - into the int64 buffer `out`
 * ([n, 2], row-major) in the dict's iteration order.  ValueError if `out` is too small. */
static PyObject* flatten_dict(PyObject* self, PyObject* args) {
  PyObject* d;
  Py_buffer out;
  if (!PyArg_ParseTuple(args, "O!w*", &PyDict_Type, &d, &out)) return NULL;
  int64_t* dst = (int64_t*)out.buf;
  const Py_ssize_t cap = out.len / 16;
  Py_ssize_t n = 0, pos = 0;
  PyObject *key, *value;
  PyObject* result = NULL;
  while (PyDict_Next(d, &pos, &key, &value)) {
    const long long src = PyLong_AsLongLong(key);
    if (src == -1 && PyErr_Occurred()) goto done;
    PyObject* fast = PySequence_Fast(value, "destinations must be a sequence of block ids");
    if (!fast) goto done;
    const Py_ssize_t m = PySequence_Fast_GET_SIZE(fast);
    if (n + m > cap) {
      Py_DECREF(fast);
      PyErr_SetString(PyExc_ValueError, "pair buffer too small for the block map");
      goto done;
    }
    PyObject** items = PySequence_Fast_ITEMS(fast);
    for (Py_ssize_t i = 0; i < m; ++i) {
      const long long dd = PyLong_AsLongLong(items[i]);
      if (dd == -1 && PyErr_Occurred()) {
        Py_DECREF(fast);
        goto done;
      }
      dst[2 * (n + i)] = src;
      dst[2 * (n + i) + 1] = dd;
    }
    n += m;
    Py_DECREF(fast);
  }
  result = PyLong_FromSsize_t(n);
done:
  PyBuffer_Release(&out);
  return result;
}

static int get_i64(PyObject* obj, PyObject* name, int64_t* out) {
  PyObject* v = PyObject_GetAttr(obj, name);
  if (!v) return -1;
  const long long x = PyLong_AsLongLong(v);
  Py_DECREF(v);
  if (x == -1 && PyErr_Occurred()) return -1;
  *out = x;
  return 0;
}

/* flatten_entries(entries, out) -> n: (e.src_block_id, e.dst_block_id) of every entry of a
 * BlockMapping (proto/worker.proto:78-86) into the int64 buffer `out` ([n, 2]). */
static PyObject* flatten_entries(PyObject* self, PyObject* args) {
  PyObject* entries;
  Py_buffer out;
  if (!PyArg_ParseTuple(args, "Ow*", &entries, &out)) return NULL;
  PyObject* result = NULL;
  PyObject* src_name = PyUnicode_InternFromString("src_block_id");
  PyObject* dst_name = PyUnicode_InternFromString("dst_block_id");
  PyObject* fast = PySequence_Fast(entries, "entries must be a sequence");
  if (!fast || !src_name || !dst_name) goto done;
  {
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(fast);
    if (n > out.len / 16) {
      PyErr_SetString(PyExc_ValueError, "pair buffer too small for the entries");
      goto done;
    }
    int64_t* dst = (int64_t*)out.buf;
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* e = PySequence_Fast_GET_ITEM(fast, i);
      if (get_i64(e, src_name, dst + 2 * i) || get_i64(e, dst_name, dst + 2 * i + 1)) goto done;
    }
    result = PyLong_FromSsize_t(n);
  }
done:
  Py_XDECREF(fast);
  Py_XDECREF(src_name);
  Py_XDECREF(dst_name);
  PyBuffer_Release(&out);
  return result;
}

/* call_plan(fn_address, plan_handle, stream) -> status
 *
 * Calls an `int fn(const void* plan, void* stream)` entry point of the C ABI (lms_write_plan_run)
 * through its address.  The decode loop issues one such call per layer per step; going through
 * ctypes costs about a microsecond per call in argument conversion, a third of what the launch
 * itself takes.  The three arguments are plain integers (addresses), nothing is dereferenced
 * here. */
typedef int (*plan_run_fn)(const void*, void*);

static PyObject* call_plan(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 3) {
    PyErr_SetString(PyExc_TypeError, "call_plan(fn_address, plan_handle, stream)");
    return NULL;
  }
  void* fn = PyLong_AsVoidPtr(args[0]);
  void* plan = PyLong_AsVoidPtr(args[1]);
  void* stream = PyLong_AsVoidPtr(args[2]);
  if (PyErr_Occurred()) return NULL;
  if (fn == NULL) {
    PyErr_SetString(PyExc_ValueError, "call_plan: NULL function address");
    return NULL;
  }
  plan_run_fn run;
  memcpy(&run, &fn, sizeof(run)); /* object pointer -> function pointer without a cast warning */
  return PyLong_FromLong((long)run(plan, stream));
}

/* ---- calls of the attention layer ---------------------------------------------------------
 *
 * A layer of a decode step makes one head-norm call and one attention call, each with five to
 * twelve tensors, and reading what has to be checked of them is most of what a small call costs on
 * the host.  The two functions below read every attribute once, through the tensors' own Python
 * attributes, check it, fill the argument structure of the C entry point and call it.  They return
 * the entry point's status, or None where an argument is not one they take: the Python caller then
 * says what is wrong with it (or brings it into shape and calls again). */
#define FACTS_MAX_DIM 6
typedef struct {
  PyObject* dtype; /* borrowed: compared by identity, torch's dtypes live for ever */
  int64_t device;  /* -1 on the host */
  int64_t ptr;
  int dim;
  int64_t size[FACTS_MAX_DIM], stride[FACTS_MAX_DIM]; /* in elements */
} facts;

static PyObject *s_dtype, *s_get_device, *s_data_ptr, *s_shape, *s_stride, *s_new_empty;

static int int_of(PyObject* v, int64_t* out) { /* takes the reference */
  if (!v) return -1;
  *out = PyLong_AsLongLong(v);
  Py_DECREF(v);
  return *out == -1 && PyErr_Occurred() ? -1 : 0;
}

static int ints_of(PyObject* v, int64_t* out, int* n) { /* takes the reference */
  if (!v) return -1;
  int rc = -1;
  if (PyTuple_Check(v) && PyTuple_GET_SIZE(v) <= FACTS_MAX_DIM) {
    *n = (int)PyTuple_GET_SIZE(v);
    rc = 0;
    for (int i = 0; i < *n && rc == 0; ++i) {
      out[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(v, i));
      if (out[i] == -1 && PyErr_Occurred()) rc = -1;
    }
  }
  Py_DECREF(v);
  return rc;
}

/* 0, or -1 for anything that is not a tensor of at most FACTS_MAX_DIM dimensions */
static int facts_of(PyObject* t, facts* f) {
  int n = 0;
  PyObject* d = PyObject_GetAttr(t, s_dtype);
  if (!d) return -1;
  f->dtype = d;
  Py_DECREF(d);
  if (int_of(PyObject_CallMethodNoArgs(t, s_get_device), &f->device)) return -1;
  if (f->device < 0) { /* nothing on the host is taken */
    f->dim = -1;
    return 0;
  }
  if (int_of(PyObject_CallMethodNoArgs(t, s_data_ptr), &f->ptr)) return -1;
  if (ints_of(PyObject_GetAttr(t, s_shape), f->size, &f->dim)) return -1;
  if (ints_of(PyObject_CallMethodNoArgs(t, s_stride), f->stride, &n) || n != f->dim) return -1;
  return 0;
}

static int is_vector(const facts* f, PyObject* dtype, int64_t device, int64_t n) { /* n < 0: any length */
  return f->dim == 1 && f->dtype == dtype && f->device == device && (n < 0 || f->size[0] == n) &&
         (f->size[0] <= 1 || f->stride[0] == 1);
}

#define AS_PTR(x) ((void*)(uintptr_t)(x))

/* The dtype objects, given once by the Python side. */
static PyObject *dt_f16, *dt_bf16, *dt_i32, *dt_i64, *dt_f32;

static PyObject* set_dtypes(PyObject* self, PyObject* args) {
  (void)self;
  PyObject *a, *b, *c, *d, *e;
  if (!PyArg_ParseTuple(args, "OOOOO", &a, &b, &c, &d, &e)) return NULL;
  dt_f16 = Py_NewRef(a);
  dt_bf16 = Py_NewRef(b);
  dt_i32 = Py_NewRef(c);
  dt_i64 = Py_NewRef(d);
  dt_f32 = Py_NewRef(e);
  Py_RETURN_NONE;
}

static PyObject* not_taken(void) {
  PyErr_Clear();
  Py_RETURN_NONE;
}

/* attention(size_fn, run_fn, stream, device, query, k_cache, v_cache | None, kv_indptr, kv_indices,
 *           kv_last, qo_indptr | None, prefix_indptr | None, prefix_indices, prefix_last,
 *           group_indptr | None, scale | None, causal, out, lse | None) -> status | None
 *
 * v_cache None: k_cache is the interleaved [num_pages, 2, page_size, H, D]. */
typedef int64_t (*attention_size_fn)(const lms_attention_args*);
typedef int (*attention_run_fn)(const lms_attention_args*, void*);

static PyObject* attention(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 19 || dt_i32 == NULL) {
    PyErr_SetString(PyExc_TypeError, "attention() takes 19 arguments, after set_dtypes()");
    return NULL;
  }
  void* size_ptr = PyLong_AsVoidPtr(args[0]);
  void* run_ptr = PyLong_AsVoidPtr(args[1]);
  void* stream = PyLong_AsVoidPtr(args[2]);
  const int64_t device = PyLong_AsLongLong(args[3]);
  if (PyErr_Occurred()) return NULL;
  if (!size_ptr || !run_ptr) {
    PyErr_SetString(PyExc_ValueError, "attention: NULL function address");
    return NULL;
  }
  facts q, k, v, out, x;
  lms_attention_args a;
  memset(&a, 0, sizeof(a));
  if (device < 0 || facts_of(args[4], &q) || facts_of(args[5], &k)) return not_taken();
  const int half = k.dtype == dt_f16;
  if ((!half && k.dtype != dt_bf16) || q.dtype != k.dtype || q.device != device || k.device != device) return not_taken();
  const int pair = args[6] != Py_None;
  if (k.dim != (pair ? 4 : 5)) return not_taken();
  const int at = k.dim - 3;
  const int64_t BS = k.size[at], H = k.size[at + 1], D = k.size[at + 2];
  if (k.stride[at] != H * D || k.stride[at + 1] != D || k.stride[at + 2] != 1 || H <= 0 || D <= 0) return not_taken();
  a.key_cache = AS_PTR(k.ptr);
  if (pair) {
    if (facts_of(args[6], &v) || v.dtype != k.dtype || v.device != device || v.dim != 4 ||
        memcmp(v.size, k.size, 4 * sizeof(int64_t)) || memcmp(v.stride, k.stride, 4 * sizeof(int64_t)))
      return not_taken();
    a.value_cache = AS_PTR(v.ptr);
  } else {
    if (k.size[1] != 2) return not_taken();
    a.value_cache = AS_PTR(k.ptr + k.stride[1] * 2);
  }
  int64_t HQ;
  const int64_t T = q.dim > 0 ? q.size[0] : 0;
  if (q.dim == 3) {
    HQ = q.size[1];
    if (q.size[2] != D || (T && (q.stride[2] != 1 || (HQ != 1 && q.stride[1] != D)))) return not_taken();
  } else if (q.dim == 2) {
    HQ = q.size[1] / D;
    if (HQ * D != q.size[1] || (T && q.stride[1] != 1)) return not_taken();
  } else {
    return not_taken();
  }
  if (HQ <= 0 || HQ % H) return not_taken();
  if (facts_of(args[17], &out) || out.dtype != q.dtype || out.device != device || out.dim != q.dim ||
      memcmp(out.size, q.size, (size_t)q.dim * sizeof(int64_t)) ||
      (T && (out.stride[q.dim - 1] != 1 || (q.dim == 3 && HQ != 1 && out.stride[1] != D))))
    return not_taken();
  if (facts_of(args[7], &x) || !is_vector(&x, dt_i32, device, -1) || x.size[0] < 1) return not_taken();
  const int64_t B = x.size[0] - 1;
  a.kv_indptr = AS_PTR(x.ptr);
  if (facts_of(args[8], &x) || !is_vector(&x, dt_i32, device, -1)) return not_taken();
  a.kv_indices = AS_PTR(x.ptr);
  a.num_kv_indices = x.size[0];
  if (facts_of(args[9], &x) || !is_vector(&x, dt_i32, device, B)) return not_taken();
  a.kv_last_page_len = AS_PTR(x.ptr);
  if (args[10] != Py_None) {
    if (facts_of(args[10], &x) || !is_vector(&x, dt_i32, device, B + 1)) return not_taken();
    a.qo_indptr = AS_PTR(x.ptr);
  } else if (T != B) {
    return not_taken();
  }
  if (args[11] != Py_None) {
    if (facts_of(args[11], &x) || !is_vector(&x, dt_i32, device, -1) || x.size[0] < 1) return not_taken();
    a.num_groups = x.size[0] - 1;
    a.prefix_indptr = AS_PTR(x.ptr);
    if (facts_of(args[12], &x) || !is_vector(&x, dt_i32, device, -1)) return not_taken();
    a.prefix_indices = AS_PTR(x.ptr);
    a.num_prefix_indices = x.size[0];
    if (facts_of(args[13], &x) || !is_vector(&x, dt_i32, device, a.num_groups)) return not_taken();
    a.prefix_last_page_len = AS_PTR(x.ptr);
    if (args[14] != Py_None) {
      if (facts_of(args[14], &x) || !is_vector(&x, dt_i32, device, a.num_groups + 1)) return not_taken();
      a.group_indptr = AS_PTR(x.ptr);
    } else if (a.num_groups != 1) {
      return not_taken();
    }
  }
  if (args[18] != Py_None) {
    if (facts_of(args[18], &x) || x.dtype != dt_f32 || x.device != device || x.dim != 2 || x.size[0] != T ||
        x.size[1] != HQ || (T > 1 && x.stride[0] != HQ) || (T && HQ > 1 && x.stride[1] != 1))
      return not_taken();
    a.lse = AS_PTR(x.ptr);
  }
  if (args[15] == Py_None) {
    a.scale = 1.0 / sqrt((double)D);
  } else {
    a.scale = PyFloat_AsDouble(args[15]);
    if (PyErr_Occurred()) return NULL;
  }
  a.causal = PyObject_IsTrue(args[16]);
  if (a.causal < 0) return NULL;
  if (T == 0 || B == 0) return PyLong_FromLong(0);
  a.query = AS_PTR(q.ptr);
  a.out = AS_PTR(out.ptr);
  a.query_token_stride = T > 1 ? q.stride[0] * 2 : 0; /* the distance to a next token, if there is one */
  a.out_token_stride = T > 1 ? out.stride[0] * 2 : 0;
  a.block_stride = k.stride[0] * 2;
  a.slot_stride = H * D * 2;
  a.num_tokens = T;
  a.num_requests = B;
  a.num_blocks = k.size[0];
  a.num_heads = HQ;
  a.num_kv_heads = H;
  a.head_dim = D;
  a.block_size = BS;
  a.dtype = half ? 0 : 1;

  attention_size_fn size;
  attention_run_fn run;
  memcpy(&size, &size_ptr, sizeof(size));
  memcpy(&run, &run_ptr, sizeof(run));
  const int64_t need = size(&a);
  if (need < 0) return PyLong_FromLongLong(need);
  PyObject* workspace = NULL;
  if (need > 0) {
    /* taken per call from torch's allocator: ordered by the stream it is used on, and a captured call
     * keeps its own; `need` is a multiple of 256, the tensor is int32 as kv_indptr is */
    PyObject* n = PyLong_FromLongLong(need / 4);
    if (!n) return NULL;
    workspace = PyObject_CallMethodOneArg(args[7], s_new_empty, n);
    Py_DECREF(n);
    int64_t ptr = 0;
    if (!workspace) return NULL;
    if (int_of(PyObject_CallMethodNoArgs(workspace, s_data_ptr), &ptr)) {
      Py_DECREF(workspace);
      return NULL;
    }
    a.workspace = AS_PTR(ptr);
    a.workspace_bytes = need;
  }
  const int rc = run(&a, stream);
  Py_XDECREF(workspace);
  return PyLong_FromLong((long)rc);
}

/* qk_norm(run_fn, stream, device, query, key, value | None, query_weight, key_weight, positions,
 *         cos_sin_cache, head_dim, kv_cache | None, slots | None, eps, q_out, k_out | None)
 *         -> status | None
 *
 * q_out and k_out are fresh, contiguous and shaped as query and key. */
typedef int (*qk_norm_run_fn)(const lms_qk_norm_args*, void*);

static PyObject* qk_norm(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 16 || dt_i32 == NULL) {
    PyErr_SetString(PyExc_TypeError, "qk_norm() takes 16 arguments, after set_dtypes()");
    return NULL;
  }
  void* run_ptr = PyLong_AsVoidPtr(args[0]);
  void* stream = PyLong_AsVoidPtr(args[1]);
  const int64_t device = PyLong_AsLongLong(args[2]);
  const int64_t D = PyLong_AsLongLong(args[10]);
  const double eps = PyFloat_AsDouble(args[13]);
  if (PyErr_Occurred()) return NULL;
  if (!run_ptr) {
    PyErr_SetString(PyExc_ValueError, "qk_norm: NULL function address");
    return NULL;
  }
  facts q, k, x;
  lms_qk_norm_args a;
  memset(&a, 0, sizeof(a));
  if (device < 0 || D <= 0 || facts_of(args[3], &q) || facts_of(args[4], &k)) return not_taken();
  PyObject* const dtype = q.dtype;
  if ((dtype != dt_f16 && dtype != dt_bf16) || k.dtype != dtype || q.device != device || k.device != device ||
      q.dim != 2 || k.dim != 2 || k.size[0] != q.size[0])
    return not_taken();
  const int64_t T = q.size[0], heads = q.size[1] / D, kv_heads = k.size[1] / D;
  if (heads <= 0 || kv_heads <= 0 || heads * D != q.size[1] || kv_heads * D != k.size[1] || q.stride[1] != 1 ||
      k.stride[1] != 1)
    return not_taken();
  if (facts_of(args[6], &x) || !is_vector(&x, dtype, device, D)) return not_taken();
  a.query_weight = AS_PTR(x.ptr);
  if (facts_of(args[7], &x) || !is_vector(&x, dtype, device, D)) return not_taken();
  a.key_weight = AS_PTR(x.ptr);
  if (facts_of(args[8], &x)) return not_taken();
  a.positions_are_int64 = x.dtype == dt_i64;
  if (!is_vector(&x, a.positions_are_int64 ? dt_i64 : dt_i32, device, T)) return not_taken();
  a.positions = AS_PTR(x.ptr);
  if (facts_of(args[9], &x) || x.dtype != dtype || x.device != device || x.dim != 2 || x.size[1] != 2 * D ||
      x.stride[1] != 1)
    return not_taken();
  a.cos_sin_cache = AS_PTR(x.ptr);
  a.cos_sin_row_stride = x.size[0] > 1 ? x.stride[0] * 2 : 0;
  a.max_position = x.size[0];
  const int one = T == 1; /* the distance to a next token means nothing */
  if (args[11] != Py_None) {
    const int64_t row = kv_heads * D;
    if (facts_of(args[11], &x) || x.dtype != dtype || x.device != device || x.dim != 5 || x.size[1] != 2 ||
        x.size[3] != kv_heads || x.size[4] != D)
      return not_taken();
    const int64_t NB = x.size[0], BS = x.size[2];
    if (NB && (x.stride[1] != BS * row || x.stride[2] != row || x.stride[3] != D || x.stride[4] != 1)) return not_taken();
    a.key_cache = AS_PTR(x.ptr);
    a.value_cache = AS_PTR(x.ptr + BS * row * 2);
    a.block_stride = x.stride[0] * 2;
    a.slot_stride = row * 2;
    a.block_size = BS;
    a.num_slots = NB * BS;
    if (facts_of(args[5], &x) || x.dtype != dtype || x.device != device || x.dim != 2 || x.size[0] != T ||
        x.size[1] != k.size[1] || x.stride[1] != 1)
      return not_taken();
    a.value = AS_PTR(x.ptr);
    a.value_token_stride = one ? 0 : x.stride[0] * 2;
    if (facts_of(args[12], &x) || !is_vector(&x, dt_i64, device, T)) return not_taken();
    a.slot_mapping = AS_PTR(x.ptr);
  }
  if (T == 0) return PyLong_FromLong(0);
  int64_t ptr;
  if (int_of(PyObject_CallMethodNoArgs(args[14], s_data_ptr), &ptr)) return NULL;
  a.q_out = AS_PTR(ptr);
  a.q_out_token_stride = q.size[1] * 2;
  if (args[15] != Py_None) {
    if (int_of(PyObject_CallMethodNoArgs(args[15], s_data_ptr), &ptr)) return NULL;
    a.k_out = AS_PTR(ptr);
    a.k_out_token_stride = k.size[1] * 2;
  }
  a.query = AS_PTR(q.ptr);
  a.key = AS_PTR(k.ptr);
  a.query_token_stride = one ? 0 : q.stride[0] * 2;
  a.key_token_stride = one ? 0 : k.stride[0] * 2;
  a.eps = eps;
  a.num_tokens = T;
  a.num_heads = heads;
  a.num_kv_heads = kv_heads;
  a.head_dim = D;
  a.dtype = dtype == dt_f16 ? 0 : 1;
  qk_norm_run_fn run;
  memcpy(&run, &run_ptr, sizeof(run));
  return PyLong_FromLong((long)run(&a, stream));
}

static PyMethodDef methods[] = {
    {"flatten_dict", flatten_dict, METH_VARARGS, "flatten_dict(src_to_dst, out) -> number of pairs"},
    {"flatten_entries", flatten_entries, METH_VARARGS, "flatten_entries(entries, out) -> number of pairs"},
    {"pack", pack, METH_VARARGS,
     "pack(inputs, out) -> (batch, total_tokens, total_blocks, prefill_input_len, num_prefill, num_decode, "
     "prefill_blocks, decode_blocks)"},
    {"call_plan", (PyCFunction)(void (*)(void))call_plan, METH_FASTCALL,
     "call_plan(fn_address, plan_handle, stream) -> status of int fn(plan, stream)"},
    {"set_dtypes", set_dtypes, METH_VARARGS, "set_dtypes(float16, bfloat16, int32, int64, float32)"},
    {"attention", (PyCFunction)(void (*)(void))attention, METH_FASTCALL,
     "attention(...) -> status of lms_paged_attention, or None for arguments it does not take"},
    {"qk_norm", (PyCFunction)(void (*)(void))qk_norm, METH_FASTCALL,
     "qk_norm(...) -> status of lms_qk_norm_rope_and_cache, or None for arguments it does not take"},
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_packer",
                                    "Packs a step's request list into the index-preparation upload buffer.",
                                    -1, methods};

PyMODINIT_FUNC PyInit__packer(void) {
  s_input_len = PyUnicode_InternFromString("input_len");
  s_filled_token_len = PyUnicode_InternFromString("filled_token_len");
  s_context_len = PyUnicode_InternFromString("context_len");
  s_block_ids = PyUnicode_InternFromString("block_ids");
  s_input_ids = PyUnicode_InternFromString("input_ids");
  s_dtype = PyUnicode_InternFromString("dtype");
  s_get_device = PyUnicode_InternFromString("get_device");
  s_data_ptr = PyUnicode_InternFromString("data_ptr");
  s_shape = PyUnicode_InternFromString("shape");
  s_stride = PyUnicode_InternFromString("stride");
  s_new_empty = PyUnicode_InternFromString("new_empty");
  if (!s_dtype || !s_get_device || !s_data_ptr || !s_shape || !s_stride || !s_new_empty) return NULL;
  if (!s_input_len || !s_filled_token_len || !s_context_len || !s_block_ids || !s_input_ids) return NULL;
  return PyModule_Create(&module);
}
