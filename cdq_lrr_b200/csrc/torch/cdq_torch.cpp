// Direct Python entry of the calls whose host time counts (a decode step's
// cache and sampling calls): one C++ function a call instead of a dozen
// interpreted checks and a ctypes call (about 9 us instead of 18 on the test
// machine's host cores for an attention call, two launches included).
//
// Every function looks its arguments over completely and returns None for
// anything out of the ordinary (a wrong type or shape, rows that have to be
// copied, a device that is not current); the Python method behind it then
// takes the general path, which copies what it must and raises what it has to.
// The module sees the library through its C ABI only.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>

#include "cdq.h"

namespace {

struct Rows {
    const uint16_t* p;
    int64_t seq, tok;
};

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }
bool none(PyObject* o) { return o == Py_None; }
bool on(const at::Tensor& t, int dev) { return t.is_cuda() && t.get_device() == dev; }
template <class T>
T* ptr(const at::Tensor& t) {
    return static_cast<T*>(t.data_ptr());
}

// bf16 [batch, n, heads, head_dim] with contiguous heads and 16-byte rows
bool rows(const at::Tensor& t, int dev, int64_t batch, int64_t heads, int64_t hd, Rows* r) {
    if (!on(t, dev) || t.scalar_type() != at::kBFloat16 || t.dim() != 4) return false;
    const auto size = t.sizes(), stride = t.strides();
    if (size[0] != batch || size[3] != hd || (heads && size[2] != heads) || stride[3] != 1 || stride[2] != hd ||
        stride[0] < 0 || stride[1] < 0 || stride[0] % 8 || stride[1] % 8)
        return false;
    r->p = ptr<uint16_t>(t), r->seq = stride[0], r->tok = stride[1];
    return (uintptr_t)r->p % 16 == 0;
}
const int32_t* index(PyObject* o, int dev, int64_t n) {
    const at::Tensor* t = tensor(o);
    return t && on(*t, dev) && t->scalar_type() == at::kInt && t->numel() == n && t->is_contiguous() ? ptr<int32_t>(*t) : nullptr;
}
struct Rope {
    const uint16_t *c = nullptr, *s = nullptr;
    int32_t rows = 0;
    const int32_t* pos = nullptr;
};
// (cos, sin) or None, and rope_pos or None
bool rope(PyObject* tables, PyObject* pos, const cdq_kv_cache* c, int dev, Rope* r) {
    if (none(tables)) return none(pos);
    if (!PyTuple_Check(tables) || PyTuple_GET_SIZE(tables) != 2) return false;
    const at::Tensor* t[2] = {tensor(PyTuple_GET_ITEM(tables, 0)), tensor(PyTuple_GET_ITEM(tables, 1))};
    for (const at::Tensor* x : t)
        if (!x || !on(*x, dev) || x->scalar_type() != at::kBFloat16 || x->dim() != 2 || x->size(1) != c->head_dim ||
            x->size(0) < 1 || x->size(0) > INT_MAX || !x->is_contiguous() || (uintptr_t)x->data_ptr() % 16)
            return false;
    if (t[0]->size(0) != t[1]->size(0)) return false;
    r->c = ptr<uint16_t>(*t[0]), r->s = ptr<uint16_t>(*t[1]), r->rows = (int32_t)t[0]->size(0);
    return none(pos) || (r->pos = index(pos, dev, c->batch));
}

const cdq_kv_cache* cache_of(PyObject* address) {
    return static_cast<const cdq_kv_cache*>(PyLong_AsVoidPtr(address));
}
// (a cache on the CPU has device -1: no CUDA call, which could fail, before the general path refuses it)
bool current(int dev) { return dev >= 0 && c10::cuda::current_device() == dev; }
void* stream(int dev) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }
at::Tensor empty(at::IntArrayRef size, at::ScalarType type, int dev) {
    return at::empty(size, at::TensorOptions().dtype(type).device(at::kCUDA, (c10::DeviceIndex)dev));
}
// A call's scratch, ordered by the current stream like a tensor's memory.
c10::DataPtr scratch(int64_t bytes) {
    return bytes ? c10::cuda::CUDACachingAllocator::get()->allocate((size_t)bytes) : c10::DataPtr();
}

// a status that is not CDQ_OK goes back as a number: the caller raises it
PyObject* status(cdq_status st) { return PyLong_FromLong(st); }

#define CDQ_ENTRY(name, count)                                             \
    PyObject* name(PyObject*, PyObject* const* a, Py_ssize_t n_args) {     \
        if (n_args != count) {                                             \
            PyErr_SetString(PyExc_TypeError, #name ": argument count");    \
            return nullptr;                                                \
        }                                                                  \
        try {
#define CDQ_EXIT                                            \
    }                                                       \
    catch (const c10::OutOfMemoryError&) {                  \
        Py_RETURN_NONE; /* the general path raises torch's */ \
    }                                                       \
    catch (const std::exception& e) {                       \
        PyErr_SetString(PyExc_RuntimeError, e.what());      \
        return nullptr;                                     \
    }                                                       \
    }

// (cache, device, k, v, pos, rope, rope_pos) -> status
CDQ_ENTRY(kv_append, 7)
const cdq_kv_cache* c = cache_of(a[0]);
const int dev = (int)PyLong_AsLong(a[1]);
const at::Tensor *k = tensor(a[2]), *v = tensor(a[3]);
Rows kr, vr;
Rope r;
if (!k || !v || !current(dev) || !rows(*k, dev, c->batch, c->kv_heads, c->head_dim, &kr) ||
    !rows(*v, dev, c->batch, c->kv_heads, c->head_dim, &vr) || v->size(1) != k->size(1) || k->size(1) < 1 ||
    k->size(1) > INT_MAX || !rope(a[5], a[6], c, dev, &r))
    Py_RETURN_NONE;
const int32_t* pos = index(a[4], dev, c->batch);
if (!pos) Py_RETURN_NONE;
return status(cdq_kv_append(c, kr.p, kr.seq, kr.tok, vr.p, vr.seq, vr.tok, pos, (int32_t)k->size(1), r.c, r.s, r.rows,
                            r.pos, stream(dev)));
CDQ_EXIT

// (cache, device, pos, n) -> status or (k, v)
CDQ_ENTRY(kv_read, 4)
const cdq_kv_cache* c = cache_of(a[0]);
const int dev = (int)PyLong_AsLong(a[1]);
const int32_t* pos = none(a[2]) ? nullptr : index(a[2], dev, c->batch);
int beyond = 0;
const int64_t n = PyLong_Check(a[3]) ? PyLong_AsLongLongAndOverflow(a[3], &beyond) : 0;  // (beyond 64 bits: -1)
if ((!none(a[2]) && !pos) || n < 1 || n > INT_MAX || !current(dev)) Py_RETURN_NONE;
const at::Tensor k = empty({c->batch, n, c->kv_heads, c->head_dim}, at::kBFloat16, dev);
const at::Tensor v = empty({c->batch, n, c->kv_heads, c->head_dim}, at::kBFloat16, dev);
const cdq_status st = cdq_kv_read(c, pos, (int32_t)n, ptr<uint16_t>(k), ptr<uint16_t>(v), stream(dev));
if (st) return status(st);
PyObject *pk = THPVariable_Wrap(k), *pv = THPVariable_Wrap(v);
return Py_BuildValue("(NN)", pk, pv);
CDQ_EXIT

// (cache, device, q, pos, rope, rope_pos, scale or None, prefix or None, prefix_len or None, out or None)
// -> status or out; `prefix` is checked by the caller
CDQ_ENTRY(kv_attend, 10)
const cdq_kv_cache* c = cache_of(a[0]);
const int dev = (int)PyLong_AsLong(a[1]);
const at::Tensor* q = tensor(a[2]);
Rows qr;
Rope r;
if (!q || !current(dev) || !rows(*q, dev, c->batch, 0, c->head_dim, &qr) || !rope(a[4], a[5], c, dev, &r)) Py_RETURN_NONE;
const int64_t n = q->size(1), heads = q->size(2);
if (n < 1 || n > CDQ_KV_MAX_NEW || heads < c->kv_heads || heads > 65535 || heads % c->kv_heads) Py_RETURN_NONE;
const int32_t* pos = index(a[3], dev, c->batch);
const cdq_kv_cache* prefix = none(a[7]) ? nullptr : cache_of(a[7]);
const int32_t* prefix_len = prefix ? index(a[8], dev, 1) : nullptr;
if (!pos || (prefix && !prefix_len) || (!prefix && !none(a[8]))) Py_RETURN_NONE;
double scale = 1.0 / std::sqrt((double)c->head_dim);
if (!none(a[6])) {
    if (!PyFloat_Check(a[6])) Py_RETURN_NONE;
    scale = PyFloat_AS_DOUBLE(a[6]);
}
at::Tensor made;
const at::Tensor* out = &made;
if (none(a[9])) {
    made = empty(q->sizes(), at::kBFloat16, dev);
} else {
    out = tensor(a[9]);
    if (!out || !on(*out, dev) || out->scalar_type() != at::kBFloat16 || out->sizes() != q->sizes() || !out->is_contiguous() ||
        (uintptr_t)out->data_ptr() % 16)
        Py_RETURN_NONE;
    const auto *o = ptr<uint16_t>(*out), *q_end = qr.p + (c->batch - 1) * qr.seq + (n - 1) * qr.tok + heads * c->head_dim;
    if (o < q_end && qr.p < o + out->numel()) Py_RETURN_NONE;
}
int64_t need = 0;
cdq_status st = cdq_kv_attend_workspace(c, (int32_t)heads, (int32_t)n, prefix, &need);
if (st) return status(st);
const c10::DataPtr ws = scratch(need);
st = cdq_kv_attend(c, qr.p, qr.seq, qr.tok, (int32_t)heads, (int32_t)n, pos, r.c, r.s, r.rows, r.pos, (float)scale, prefix,
                   prefix_len, ptr<uint16_t>(*out), ws.get(), need, stream(dev));
if (st) return status(st);
return THPVariable_Wrap(*out);
CDQ_EXIT

// logits [.., vocab] with contiguous rows: 0 bf16, 1 float32, -1 neither
int logits(const at::Tensor& t, int dim) {
    const int type = t.scalar_type() == at::kBFloat16 ? 0 : t.scalar_type() == at::kFloat ? 1 : -1;
    if (type < 0 || !t.is_cuda() || t.dim() != dim || t.numel() < 1 || t.stride(dim - 1) != 1) return -1;
    for (int i = 0; i < dim; ++i)
        if (t.stride(i) < 0 || t.size(i) > INT_MAX) return -1;
    return type;
}
const float* uniforms(PyObject* o, int dev, int64_t n0, int64_t n1) {
    const at::Tensor* t = tensor(o);
    if (!t || !on(*t, dev) || t->scalar_type() != at::kFloat || !t->is_contiguous()) return nullptr;
    return (n1 < 0 ? t->dim() == 1 && t->size(0) == n0 : t->dim() == 2 && t->size(0) == n0 && t->size(1) == n1) ? ptr<float>(*t)
                                                                                                               : nullptr;
}

// (target logits, drafts, draft logits or None, u_accept, u_sample, temperature) -> status or (tokens, n_accepted)
CDQ_ENTRY(verify_drafts, 6)
const at::Tensor *t = tensor(a[0]), *x = tensor(a[1]), *d = none(a[2]) ? nullptr : tensor(a[2]);
const int type = t ? logits(*t, 3) : -1;
if (type < 0 || !x || (!none(a[2]) && !d) || !PyFloat_Check(a[5])) Py_RETURN_NONE;
const int dev = t->get_device();
const int64_t batch = t->size(0), k = t->size(1) - 1, vocab = t->size(2);
const double temperature = PyFloat_AS_DOUBLE(a[5]);
if (k < 1 || k > CDQ_VERIFY_MAX_DRAFTS || !current(dev) || !on(*x, dev) || x->scalar_type() != at::kLong || x->dim() != 2 ||
    x->size(0) != batch || x->size(1) != k || !x->is_contiguous() || !(temperature >= 1e-30 && temperature <= 1e30))
    Py_RETURN_NONE;
if (d && (logits(*d, 3) != type || d->get_device() != dev || d->size(0) != batch || d->size(1) != k || d->size(2) != vocab))
    Py_RETURN_NONE;
const float *ua = uniforms(a[3], dev, batch, k), *us = uniforms(a[4], dev, batch, -1);
if (!ua || !us) Py_RETURN_NONE;
const at::Tensor tokens = empty({batch, k + 1}, at::kLong, dev), kept = empty({batch}, at::kInt, dev);
const int64_t need = batch * (d ? 2 * k + 1 : k + 1) * CDQ_VERIFY_ROW_BYTES;
const c10::DataPtr ws = scratch(need);
const cdq_status st = cdq_verify_drafts(
    t->data_ptr(), t->stride(0), t->stride(1), d ? d->data_ptr() : nullptr, d ? d->stride(0) : 0, d ? d->stride(1) : 0, type,
    ptr<int64_t>(*x), ua, us, (int32_t)batch, (int32_t)k, (int32_t)vocab, temperature, ptr<int64_t>(tokens),
    ptr<int32_t>(kept), ws.get(), need, stream(dev));
if (st) return status(st);
PyObject *pt = THPVariable_Wrap(tokens), *pk = THPVariable_Wrap(kept);
return Py_BuildValue("(NN)", pt, pk);
CDQ_EXIT

// (logits, u, temperature, out or None) -> status or out
CDQ_ENTRY(sample_tokens, 4)
const at::Tensor* t = tensor(a[0]);
const int type = t ? logits(*t, 2) : -1;
if (type < 0 || !PyFloat_Check(a[2])) Py_RETURN_NONE;
const int dev = t->get_device();
const double temperature = PyFloat_AS_DOUBLE(a[2]);
const float* us = uniforms(a[1], dev, t->size(0), -1);
if (!us || !current(dev) || !(temperature >= 1e-30 && temperature <= 1e30)) Py_RETURN_NONE;
at::Tensor made;
const at::Tensor* out = &made;
if (none(a[3])) {
    made = empty({t->size(0)}, at::kLong, dev);
} else {
    out = tensor(a[3]);
    if (!out || !on(*out, dev) || out->scalar_type() != at::kLong || out->dim() != 1 || out->size(0) != t->size(0) ||
        !out->is_contiguous())
        Py_RETURN_NONE;
}
const cdq_status st = cdq_verify_drafts(t->data_ptr(), t->stride(0), 0, nullptr, 0, 0, type, nullptr, nullptr, us,
                                        (int32_t)t->size(0), 0, (int32_t)t->size(1), temperature, ptr<int64_t>(*out), nullptr,
                                        nullptr, 0, stream(dev));
if (st) return status(st);
return THPVariable_Wrap(*out);
CDQ_EXIT

#define CDQ_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {CDQ_METHOD(kv_append),     CDQ_METHOD(kv_read),       CDQ_METHOD(kv_attend),
                         CDQ_METHOD(verify_drafts), CDQ_METHOD(sample_tokens), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_cdq_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__cdq_torch() { return PyModule_Create(&module); }
