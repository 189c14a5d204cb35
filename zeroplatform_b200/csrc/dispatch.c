// dispatch.c -- the short way from zeroplatform_b200.ops to the mixed-serving-batch entries of libzero_tensor.so.
//
// A call of one of these operators runs for a few microseconds on the GPU; checking its tensors attribute by attribute
// and marshalling its arguments through ctypes takes about as long.  This CPython module does both in one call: it reads
// tensors through PyTorch's DLPack exchange table (shapes, strides, type, device and address without Python calls),
// checks what ops.py checks, and calls the C entry on the current stream.  Every function returns True when the call
// was enqueued and False when anything is not as expected (types, shapes, devices, a status other than 0); nothing has
// happened then, and ops.py takes its own way, which says what is wrong or handles the rarer forms.

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/dlpack.h>
#include <math.h>
#include <stdint.h>

#include "../../include/zero_tensor_cuda.h"

static const DLPackExchangeAPI* g_api;
static PyTypeObject* g_tensor;   // torch.Tensor itself: subclasses may redefine what an address means
static PyObject *g_torch_c, *g_get_device;
static __typeof__(&zcu_pages_reserve) p_reserve;
static __typeof__(&zcu_pages_trim) p_trim;
static __typeof__(&zcu_append_kv) p_append;
static __typeof__(&zcu_sparse_paged_attention) p_sparse;
static __typeof__(&zcu_lora_add) p_lora;
static __typeof__(&zcu_process_logits) p_logits;

enum { I8, I32, I64, F32, F16, BF16, OTHER };

typedef struct {
  void* p;
  const int64_t* shape;
  const int64_t* strides;  // NULL: contiguous
  int ndim, type, device;
} Ten;

// 1: a CUDA tensor, 0: not one that this module takes.  None gives p = NULL where `optional`.
static int take(PyObject* o, Ten* t, int optional) {
  t->p = NULL;
  t->ndim = -1;
  if (o == Py_None) return optional;
  if (Py_TYPE(o) != g_tensor) return 0;
  DLTensor d;
  if (g_api->dltensor_from_py_object_no_sync(o, &d) != 0) {
    PyErr_Clear();
    return 0;
  }
  if (d.device.device_type != kDLCUDA || d.dtype.lanes != 1) return 0;
  const int bits = d.dtype.bits;
  switch (d.dtype.code) {
    case kDLInt: t->type = bits == 8 ? I8 : bits == 32 ? I32 : bits == 64 ? I64 : OTHER; break;
    case kDLFloat: t->type = bits == 32 ? F32 : bits == 16 ? F16 : OTHER; break;
    case kDLBfloat: t->type = bits == 16 ? BF16 : OTHER; break;
    default: t->type = OTHER;
  }
  t->p = (char*)d.data + d.byte_offset;
  t->shape = d.shape;
  t->strides = d.strides;
  t->ndim = d.ndim;
  t->device = d.device.device_id;
  return 1;
}

static int64_t stride(const Ten* t, int dim) {
  if (t->strides) return t->strides[dim];
  int64_t s = 1;
  for (int i = t->ndim - 1; i > dim; --i) s *= t->shape[i];
  return s;
}

static int contiguous(const Ten* t) {
  int64_t s = 1;
  for (int i = 0; i < t->ndim; ++i)
    if (t->shape[i] == 0) return 1;
  for (int i = t->ndim - 1; i >= 0; --i) {
    if (t->shape[i] != 1 && stride(t, i) != s) return 0;
    s *= t->shape[i];
  }
  return 1;
}

// Takes a contiguous tensor of that type and device whose shape is the n given sizes (-1: any).
static int plain(PyObject* o, Ten* t, int optional, int type, int device, int n, const int64_t* shape) {
  if (!take(o, t, optional)) return 0;
  if (t->ndim < 0) return 1;  // None
  if (t->type != type || t->device != device || t->ndim != n || !contiguous(t)) return 0;
  for (int i = 0; i < n; ++i)
    if (shape[i] >= 0 && t->shape[i] != shape[i]) return 0;
  return 1;
}
#define PLAIN(o, t, opt, type, n, ...) plain(o, t, opt, type, dev, n, (const int64_t[]){__VA_ARGS__})

static int fits32(int64_t v) { return v >= 0 && v <= 0x7fffffff; }

static int whole(PyObject* o, int64_t* v) {
  if (!PyLong_CheckExact(o)) return 0;
  *v = PyLong_AsLongLong(o);
  if (*v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return 0;
  }
  return *v >= -0x7fffffff - 1LL && *v <= 0x7fffffff;
}

// The device is the current one, and its current stream.
static int on_stream(int device, void** stream) {
  PyObject* r = PyObject_CallMethodNoArgs(g_torch_c, g_get_device);
  if (!r) {
    PyErr_Clear();
    return 0;
  }
  const long cur = PyLong_AsLong(r);
  Py_DECREF(r);
  if (cur != device) {
    PyErr_Clear();
    return 0;
  }
  if (g_api->current_work_stream(kDLCUDA, device, stream) != 0) {
    PyErr_Clear();
    return 0;
  }
  return 1;
}

#define CALL(rc, expr)        \
  int32_t rc;                 \
  Py_BEGIN_ALLOW_THREADS      \
  rc = (expr);                \
  Py_END_ALLOW_THREADS

// page_table, seq_len, free_pages, free_count, page_size
typedef struct {
  Ten table, len, list, count;
  int64_t page;
} Pool;
static int take_pool(PyObject* const* a, Pool* p, int* dev_out) {
  if (!take(a[0], &p->table, 0)) return 0;
  const int dev = *dev_out = p->table.device;
  const Ten* t = &p->table;
  return t->type == I32 && t->ndim == 2 && contiguous(t) && fits32(t->shape[0]) && fits32(t->shape[1]) &&
         PLAIN(a[1], &p->len, 0, I32, 1, t->shape[0]) && PLAIN(a[2], &p->list, 0, I32, 1, -1) &&
         fits32(p->list.shape[0]) && PLAIN(a[3], &p->count, 0, I32, 1, 1) && whole(a[4], &p->page);
}

// reserve_pages(page_table, seq_len, free_pages, free_count, page_size, n_new, rows, start, slots, positions,
//               token_rows, ctx_len, granted)
static PyObject* reserve_pages(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  Pool p;
  int dev;
  Ten add, rows, start, slots, pos, trow, ctx, granted;
  void* s;
  if (n != 13 || !take_pool(a, &p, &dev) || !PLAIN(a[5], &add, 0, I32, 1, -1)) Py_RETURN_FALSE;
  const int64_t b = add.shape[0];
  if (!PLAIN(a[6], &rows, 1, I32, 1, b) || !PLAIN(a[7], &start, 0, I32, 1, b + 1) ||
      !PLAIN(a[8], &slots, 0, I64, 1, -1))
    Py_RETURN_FALSE;
  const int64_t tokens = slots.shape[0];
  if (!PLAIN(a[9], &pos, 0, I32, 1, tokens) || !PLAIN(a[10], &trow, 0, I32, 1, tokens) ||
      !PLAIN(a[11], &ctx, 0, I32, 1, tokens) || !PLAIN(a[12], &granted, 0, I32, 1, b) || !fits32(b) ||
      !fits32(tokens) || !on_stream(dev, &s))
    Py_RETURN_FALSE;
  CALL(rc, p_reserve(p.table.p, p.len.p, p.list.p, p.count.p, (int)p.table.shape[0], (int)p.table.shape[1],
                     (int)p.list.shape[0], (int)p.page, rows.p, add.p, (int)b, (int)tokens, start.p, slots.p, pos.p,
                     trow.p, ctx.p, granted.p, s));
  return PyBool_FromLong(rc == 0);
}

// trim_pages(page_table, seq_len, free_pages, free_count, page_size, new_len, rows)
static PyObject* trim_pages(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  Pool p;
  int dev;
  Ten len, rows;
  void* s;
  if (n != 7 || !take_pool(a, &p, &dev) || !PLAIN(a[5], &len, 0, I32, 1, -1) || !fits32(len.shape[0]) ||
      !PLAIN(a[6], &rows, 1, I32, 1, len.shape[0]) || !on_stream(dev, &s))
    Py_RETURN_FALSE;
  CALL(rc, p_trim(p.table.p, p.len.p, p.list.p, p.count.p, (int)p.table.shape[0], (int)p.table.shape[1],
                  (int)p.list.shape[0], (int)p.page, rows.p, len.p, (int)len.shape[0], s));
  return PyBool_FromLong(rc == 0);
}

// Both pools [pages, hkv, page size, hd], fp32 or fp16, the same strides, contiguous heads.
static int take_pools(PyObject* ko, PyObject* vo, Ten* k, Ten* v) {
  if (!take(ko, k, 0) || !take(vo, v, 0) || k->ndim != 4 || v->ndim != 4 || k->type != v->type ||
      k->device != v->device || (k->type != F32 && k->type != F16))
    return 0;
  for (int i = 0; i < 4; ++i)
    if (!fits32(k->shape[i]) || k->shape[i] != v->shape[i] || stride(k, i) != stride(v, i)) return 0;
  return stride(k, 3) == 1;
}

// append_kv(k, v, slots, k_pool, v_pool, bounds, scales)
static PyObject* append_kv(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  Ten k, v, slots, kp, vp, bounds, scales;
  void* s;
  if (n != 7 || !take_pools(a[3], a[4], &kp, &vp) || !take(a[0], &k, 0) || !take(a[1], &v, 0)) Py_RETURN_FALSE;
  const int dev = kp.device;
  const int64_t pages = kp.shape[0], hkv = kp.shape[1], page = kp.shape[2], hd = kp.shape[3];
  if (k.ndim != 3 || v.ndim != 3 || k.type != v.type || (k.type != F32 && k.type != F16) || k.device != dev ||
      v.device != dev || !fits32(k.shape[0]))
    Py_RETURN_FALSE;
  for (int i = 0; i < 3; ++i)
    if (k.shape[i] != v.shape[i]) Py_RETURN_FALSE;
  if (k.shape[1] != hkv || k.shape[2] != hd || stride(&k, 2) != 1 || stride(&v, 2) != 1 ||
      (hkv > 1 && (stride(&k, 1) != hd || stride(&v, 1) != hd)))
    Py_RETURN_FALSE;
  const int64_t tokens = k.shape[0];
  if (!PLAIN(a[2], &slots, 0, I64, 1, tokens) || !PLAIN(a[5], &bounds, 1, I8, 4, pages, hkv, 2, hd) ||
      !PLAIN(a[6], &scales, 1, F32, 2, pages, hkv) || !on_stream(dev, &s))
    Py_RETURN_FALSE;
  CALL(rc, p_append(k.p, v.p, k.type == F16, stride(&k, 0), stride(&v, 0), slots.p, (int)tokens, kp.p, vp.p,
                    kp.type == F16, (int)hkv, (int)hd, (int)page, (int)pages, stride(&kp, 0), stride(&kp, 2),
                    stride(&kp, 1), bounds.p, scales.p, s));
  return PyBool_FromLong(rc == 0);
}

// sparse_paged_attention(q, k_pool, v_pool, bounds, scales, page_table, ctx_len, budget, rows, sink, recent, scale,
//                        max_ctx, out, sel); scale and max_ctx may be None
static PyObject* sparse_paged_attention(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  Ten q, kp, vp, bounds, scales, table, ctx, rows, out, sel;
  int64_t budget, sink, recent, max_ctx;
  void* s;
  if (n != 15 || !take_pools(a[1], a[2], &kp, &vp) || !take(a[0], &q, 0)) Py_RETURN_FALSE;
  const int dev = kp.device;
  const int64_t pages = kp.shape[0], hkv = kp.shape[1], page = kp.shape[2], hd = kp.shape[3];
  if (q.ndim != 3 || q.type != F32 || q.device != dev || q.shape[2] != hd || !fits32(q.shape[0]) ||
      !fits32(q.shape[1]) || stride(&q, 2) != 1 || (q.shape[1] > 1 && stride(&q, 1) != hd))
    Py_RETURN_FALSE;
  const int64_t batch = q.shape[0], hq = q.shape[1];
  if (!whole(a[7], &budget) || !whole(a[9], &sink) || !whole(a[10], &recent) ||
      !PLAIN(a[3], &bounds, 0, I8, 4, pages, hkv, 2, hd) || !PLAIN(a[4], &scales, 0, F32, 2, pages, hkv) ||
      !PLAIN(a[5], &table, 0, I32, 2, -1, -1) || !PLAIN(a[6], &ctx, 0, I32, 1, batch) ||
      !PLAIN(a[8], &rows, 1, I32, 1, batch) || !PLAIN(a[13], &out, 0, F32, 3, batch, hq, hd) ||
      !PLAIN(a[14], &sel, 0, I32, 3, batch, hkv, budget) || !fits32(table.shape[0]) || !fits32(table.shape[1]))
    Py_RETURN_FALSE;
  double scale = 1.0 / sqrt((double)hd);
  if (a[11] != Py_None) {
    if (!PyFloat_CheckExact(a[11])) Py_RETURN_FALSE;
    scale = PyFloat_AS_DOUBLE(a[11]);
  }
  if (a[12] == Py_None) {
    const int64_t most = (1 << 30) - page;
    max_ctx = table.shape[1] * page < most ? table.shape[1] * page : most;
  } else if (!whole(a[12], &max_ctx)) {
    Py_RETURN_FALSE;
  }
  if (!on_stream(dev, &s)) Py_RETURN_FALSE;
  CALL(rc, p_sparse(q.p, stride(&q, 0), kp.p, vp.p, kp.type == F16, bounds.p, scales.p, table.p, (int)table.shape[0],
                    rows.p, ctx.p, out.p, sel.p, (int)batch, (int)hq, (int)hkv, (int)hd, (int)page,
                    (int)table.shape[1], (int)pages, stride(&kp, 0), stride(&kp, 2), stride(&kp, 1), (float)scale,
                    (int)max_ctx, (int)budget, (int)sink, (int)recent, s));
  return PyBool_FromLong(rc == 0);
}

// A matrix with contiguous rows, of that type and those sizes (-1: any).
static int matrix(PyObject* o, Ten* t, int type, int device, int64_t rows, int64_t cols) {
  return take(o, t, 0) && t->ndim == 2 && (type < 0 || t->type == type) && t->device == device &&
         (rows < 0 || t->shape[0] == rows) && (cols < 0 || t->shape[1] == cols) && fits32(t->shape[0]) &&
         fits32(t->shape[1]) && stride(t, 1) == 1;
}

static int float_code(int type) { return type == F32 ? 0 : type == F16 ? 1 : type == BF16 ? 2 : -1; }

// lora_add(y, x, a, b, adapter, ranks, scales, out)
static PyObject* lora_add(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  Ten y, x, wa, wb, adapter, ranks, scales, out;
  void* s;
  if (n != 8 || !take(a[2], &wa, 0) || wa.ndim != 3 || float_code(wa.type) < 0 || !contiguous(&wa)) Py_RETURN_FALSE;
  const int dev = wa.device;
  const int64_t na = wa.shape[0], rank = wa.shape[1], k = wa.shape[2];
  if (!fits32(na) || !fits32(rank) || !fits32(k) || !matrix(a[0], &y, F32, dev, -1, -1)) Py_RETURN_FALSE;
  const int64_t rows = y.shape[0], cols = y.shape[1];
  if (!matrix(a[1], &x, F32, dev, rows, k) || !matrix(a[7], &out, F32, dev, rows, cols) ||
      !PLAIN(a[3], &wb, 0, wa.type, 3, na, cols, rank) || !PLAIN(a[4], &adapter, 0, I32, 1, rows) ||
      !PLAIN(a[5], &ranks, 1, I32, 1, na) || !PLAIN(a[6], &scales, 1, F32, 1, na) || !on_stream(dev, &s))
    Py_RETURN_FALSE;
  CALL(rc, p_lora(x.p, stride(&x, 0), y.p, stride(&y, 0), out.p, stride(&out, 0), wa.p, wb.p, float_code(wa.type),
                  adapter.p, ranks.p, scales.p, (int)rows, (int)k, (int)cols, (int)na, (int)rank, s));
  return PyBool_FromLong(rc == 0);
}

// process_logits(logits, out, past, past_len, prompt_len, past_rows, repetition, frequency, presence, bias_start,
//                bias_ids, bias, mask, mask_rows)
static PyObject* process_logits(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  Ten x, out, past, plen, prompt, prows, rep, freq, pres, bstart, bids, bias, mask, mrows;
  void* s;
  if (n != 14 || !take(a[0], &x, 0)) Py_RETURN_FALSE;
  const int dev = x.device;
  if (!matrix(a[0], &x, -1, dev, -1, -1) || float_code(x.type) < 0) Py_RETURN_FALSE;
  const int64_t rows = x.shape[0], vocab = x.shape[1];
  if (!matrix(a[1], &out, F32, dev, rows, vocab) || !PLAIN(a[2], &past, 1, I32, 2, -1, -1)) Py_RETURN_FALSE;
  const int64_t np = past.ndim < 0 ? 0 : past.shape[0], cap = past.ndim < 0 ? 0 : past.shape[1];
  if (!PLAIN(a[3], &plen, 1, I32, 1, np) || !PLAIN(a[4], &prompt, 1, I32, 1, np) ||
      !PLAIN(a[5], &prows, 1, I32, 1, rows) || !PLAIN(a[6], &rep, 1, F32, 1, rows) ||
      !PLAIN(a[7], &freq, 1, F32, 1, rows) || !PLAIN(a[8], &pres, 1, F32, 1, rows) ||
      !PLAIN(a[9], &bstart, 1, I32, 1, rows + 1) || !PLAIN(a[11], &bias, 1, F32, 1, -1))
    Py_RETURN_FALSE;
  const int64_t nb = bias.ndim < 0 ? 0 : bias.shape[0];
  if (!PLAIN(a[10], &bids, 1, I32, 1, nb) || (bstart.ndim < 0) != (bias.ndim < 0) || (bids.ndim < 0) != (bias.ndim < 0) ||
      !PLAIN(a[12], &mask, 1, I32, 2, -1, -1) || !PLAIN(a[13], &mrows, 1, I32, 1, rows))
    Py_RETURN_FALSE;
  if (past.ndim >= 0 && prows.ndim < 0 && np < rows) Py_RETURN_FALSE;
  if (!fits32(np) || !fits32(cap) || !fits32(nb) || (mask.ndim >= 0 && !fits32(mask.shape[0])) || !on_stream(dev, &s))
    Py_RETURN_FALSE;
  const zcu_logits_rules r = {past.p, plen.p, prompt.p, prows.p, (int)cap, (int)np, rep.p, freq.p, pres.p, bstart.p,
                              bids.p, bias.p, (int)nb, mask.ndim < 0 ? 0 : (int)mask.shape[0], mask.p, mrows.p,
                              mask.ndim < 0 ? 0 : mask.shape[1]};
  CALL(rc, p_logits(x.p, float_code(x.type), stride(&x, 0), out.p, stride(&out, 0), (int)rows, (int)vocab, &r, s));
  return PyBool_FromLong(rc == 0);
}

// init(torch.Tensor, torch._C, addresses of zcu_pages_reserve, zcu_pages_trim, zcu_append_kv,
//      zcu_sparse_paged_attention, zcu_lora_add, zcu_process_logits): False where this PyTorch has no exchange table.
static PyObject* init(PyObject* self, PyObject* args) {
  PyObject *tensor, *torch_c;
  unsigned long long f[6];
  if (!PyArg_ParseTuple(args, "OOKKKKKK", &tensor, &torch_c, &f[0], &f[1], &f[2], &f[3], &f[4], &f[5])) return NULL;
  PyObject* capsule = PyObject_GetAttrString(tensor, "__dlpack_c_exchange_api__");
  const DLPackExchangeAPI* api =
      capsule ? (const DLPackExchangeAPI*)PyCapsule_GetPointer(capsule, "dlpack_exchange_api") : NULL;
  Py_XDECREF(capsule);  // the table lives as long as the process
  if (!api || api->header.version.major != DLPACK_MAJOR_VERSION || !api->dltensor_from_py_object_no_sync ||
      !api->current_work_stream) {
    PyErr_Clear();
    Py_RETURN_FALSE;
  }
  g_get_device = PyUnicode_InternFromString("_cuda_getDevice");
  Py_INCREF(tensor);
  Py_INCREF(torch_c);
  g_tensor = (PyTypeObject*)tensor;
  g_torch_c = torch_c;
  g_api = api;
  p_reserve = (__typeof__(p_reserve))(uintptr_t)f[0];
  p_trim = (__typeof__(p_trim))(uintptr_t)f[1];
  p_append = (__typeof__(p_append))(uintptr_t)f[2];
  p_sparse = (__typeof__(p_sparse))(uintptr_t)f[3];
  p_lora = (__typeof__(p_lora))(uintptr_t)f[4];
  p_logits = (__typeof__(p_logits))(uintptr_t)f[5];
  Py_RETURN_TRUE;
}

#define FAST(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, NULL}
static PyMethodDef methods[] = {FAST(reserve_pages),  FAST(trim_pages),
                                FAST(append_kv),      FAST(sparse_paged_attention),
                                FAST(lora_add),       FAST(process_logits),
                                {"init", init, METH_VARARGS, NULL}, {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_dispatch", NULL, -1, methods};

PyMODINIT_FUNC PyInit__dispatch(void) { return PyModule_Create(&module); }
