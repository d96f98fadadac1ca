// Operator calls from Python without the interpreter in between: argument checks, result allocation and the launch through
// the C ABI in one native call (a call spent ~14 us in Python around a launch of 2 us; here the whole call is ~4 us).
//
// Every function returns None when the arguments are anything but the plain case it knows (device, type, shape, layout) or something
// in it throws (a tensor without storage, no memory for the result); the Python operator then takes its own path, which handles or
// refuses them.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <climits>
#include <cmath>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "b200_eagle.h"

namespace {

// A CUDA tensor of `type` without gaps, or NULL.
const at::Tensor* plain(PyObject* o, at::ScalarType type) {
    if (!THPVariable_Check(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.is_cuda() && t.scalar_type() == type && t.is_contiguous() ? &t : nullptr;
}

// The tensor's device index when it is the current one, else -1.
int on_current(const at::Tensor& t) {
    const int dev = t.get_device();
    return dev == c10::cuda::current_device() ? dev : -1;
}

bool same_device(int dev, const at::Tensor* t) { return t == nullptr || t->get_device() == dev; }

at::Tensor result(at::IntArrayRef sizes, const at::Tensor& like) {
    return at::detail::empty_cuda(sizes, at::kHalf, like.device(), c10::nullopt);
}

void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream(dev).stream(); }

bool int_arg(PyObject* o, long* v) {
    *v = PyLong_AsLong(o);
    if (*v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}

// qmm(x, w, s, b, group_size, bias, workspace) -> y
PyObject* qmm(PyObject* const* a, Py_ssize_t n) {
    long group;
    if (n != 7 || !int_arg(a[4], &group) || group != 64) Py_RETURN_NONE;
    const at::Tensor *x = plain(a[0], at::kHalf), *s = plain(a[2], at::kHalf), *b = plain(a[3], at::kHalf);
    const at::Tensor *bias = a[5] == Py_None ? nullptr : plain(a[5], at::kHalf), *ws = plain(a[6], at::kByte);
    if (!x || !s || !b || !ws || (a[5] != Py_None && !bias) || !THPVariable_Check(a[1])) Py_RETURN_NONE;
    const at::Tensor& w = THPVariable_Unpack(a[1]);
    if (!w.is_cuda() || (w.scalar_type() != at::kInt && w.scalar_type() != at::kUInt32) || !w.is_contiguous()) Py_RETURN_NONE;
    const int dev = on_current(*x);
    if (dev < 0 || !same_device(dev, s) || !same_device(dev, b) || !same_device(dev, &w) || !same_device(dev, bias) || !same_device(dev, ws) ||
        x->dim() < 1 || w.dim() != 2 || s->dim() != 2 || b->dim() != 2)
        Py_RETURN_NONE;
    const int64_t K = x->size(-1), N = w.size(0);
    if (K < 128 || K % 128 || w.size(1) * 8 != K || s->size(0) != N || s->size(1) * 64 != K || b->size(0) != N || b->size(1) * 64 != K) Py_RETURN_NONE;
    const int64_t M = x->numel() / K;
    if (M < 1 || M > INT_MAX || N > INT_MAX || (bias && bias->numel() != N)) Py_RETURN_NONE;
    c10::SmallVector<int64_t, 5> sizes(x->sizes().begin(), x->sizes().end());
    sizes.back() = N;
    at::Tensor y = result(sizes, *x);
    const int rc = b200_qmm(x->data_ptr(), static_cast<const uint32_t*>(w.data_ptr()), s->data_ptr(), b->data_ptr(), bias ? bias->data_ptr() : nullptr,
                            y.data_ptr(), (int)M, (int)N, (int)K, 64, 0, ws->data_ptr(), (size_t)ws->numel(), stream_of(dev));
    if (rc != B200_OK) Py_RETURN_NONE;                   // (nothing was launched: the Python operator reports it)
    return THPVariable_Wrap(std::move(y));
}

// qmm_tiled(x, wt, n, bias, workspace) -> y
PyObject* qmm_tiled(PyObject* const* a, Py_ssize_t n) {
    long N;
    if (n != 5 || !int_arg(a[2], &N)) Py_RETURN_NONE;
    const at::Tensor *x = plain(a[0], at::kHalf), *wt = plain(a[1], at::kByte), *ws = plain(a[4], at::kByte);
    const at::Tensor* bias = a[3] == Py_None ? nullptr : plain(a[3], at::kHalf);
    if (!x || !wt || !ws || (a[3] != Py_None && !bias) || x->dim() != 2) Py_RETURN_NONE;
    const int dev = on_current(*x);
    if (dev < 0 || !same_device(dev, wt) || !same_device(dev, bias) || !same_device(dev, ws)) Py_RETURN_NONE;
    const int64_t M = x->size(0), K = x->size(1);
    if (M < 1 || M > 32 || N < 8 || N > INT_MAX || K > INT_MAX || (bias && bias->numel() != N)) Py_RETURN_NONE;
    const size_t need = b200_qmm_tiled_bytes((int)N, (int)K);
    if (need == 0 || (size_t)wt->numel() < need) Py_RETURN_NONE;
    at::Tensor y = result({M, (int64_t)N}, *x);
    const int rc = b200_qmm_tiled(x->data_ptr(), wt->data_ptr(), nullptr, bias ? bias->data_ptr() : nullptr, nullptr, y.data_ptr(), (int)M, (int)N,
                                  (int)K, B200_EPI_NONE, ws->data_ptr(), (size_t)ws->numel(), stream_of(dev));
    if (rc != B200_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(y));
}

// rope_positions(inp, offsets, inv_freqs, scaling_factor) -> out
PyObject* rope_positions(PyObject* const* a, Py_ssize_t n) {
    if (n != 4) Py_RETURN_NONE;
    const at::Tensor *x = plain(a[0], at::kHalf), *pos = plain(a[1], at::kInt), *inv = plain(a[2], at::kFloat);
    const double scaling = PyFloat_AsDouble(a[3]);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    if (!x || !pos || !inv || x->dim() != 4) Py_RETURN_NONE;
    const int dev = on_current(*x);
    const int64_t B = x->size(0), H = x->size(1), L = x->size(2), D = x->size(3);
    if (dev < 0 || !same_device(dev, pos) || !same_device(dev, inv) || pos->numel() != B * L || inv->numel() != D / 2) Py_RETURN_NONE;
    at::Tensor y = result(x->sizes(), *x);
    const int rc = b200_rope_positions(x->data_ptr(), static_cast<const int*>(pos->data_ptr()), static_cast<const float*>(inv->data_ptr()),
                                       (float)scaling, y.data_ptr(), (int)B, (int)H, (int)L, (int)D, stream_of(dev));
    if (rc != B200_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(y));
}

// A CUDA tensor of `dims` dimensions on device `dev` whose last dimension is contiguous, or NULL.
const at::Tensor* strided(PyObject* o, int64_t dims, int dev) {
    if (!THPVariable_Check(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.is_cuda() && t.get_device() == dev && t.dim() == dims && (t.size(-1) <= 1 || t.stride(-1) == 1) ? &t : nullptr;
}

// B200_DTYPE_* of a tensor, or -1.
int dtype_of(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kHalf: return B200_DTYPE_F16;
        case at::kBFloat16: return B200_DTYPE_BF16;
        case at::kFloat: return B200_DTYPE_F32;
        default: return -1;
    }
}

// A CUDA tensor of this type and number of values on device `dev`, without gaps and of one dimension, or NULL.
const at::Tensor* list_of(PyObject* o, at::ScalarType type, int64_t n, int dev) {
    const at::Tensor* t = plain(o, type);
    return t != nullptr && t->dim() == 1 && t->get_device() == dev && (n < 0 || t->numel() == n) ? t : nullptr;
}

int current_device() { return c10::cuda::current_device(); }

bool double_arg(PyObject* o, double* v) {
    *v = PyFloat_AsDouble(o);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}

// The rotation from Python's arguments: positions (or None), inv_freqs, scaling_factor, magnitude, interleaved, inverse.
bool rotary_args(PyObject* const* a, int64_t tokens, int64_t dim, int dev, b200_rotary* r) {
    double magnitude;
    if (a[0] != Py_None) {
        const at::Tensor* pos = list_of(a[0], at::kInt, tokens, dev);
        r->positions_64 = pos == nullptr;
        if (pos == nullptr) pos = list_of(a[0], at::kLong, tokens, dev);
        if (pos == nullptr) return false;
        r->positions = pos->data_ptr();
    }
    const at::Tensor* inv = list_of(a[1], at::kFloat, -1, dev);
    const int interleaved = PyObject_IsTrue(a[4]), inverse = PyObject_IsTrue(a[5]);
    if (inv == nullptr || inv->numel() < 1 || 2 * inv->numel() > dim || !double_arg(a[2], &r->scaling) || !double_arg(a[3], &magnitude) ||
        interleaved < 0 || inverse < 0) {
        PyErr_Clear();
        return false;
    }
    r->inv_freqs = static_cast<const float*>(inv->data_ptr());
    r->magnitude = (float)magnitude;
    r->rotary_dim = 2 * (int)inv->numel();
    r->interleaved = interleaved;
    r->inverse = inverse;
    return true;
}

// rotate(x, positions, inv_freqs, scaling_factor, magnitude, interleaved, inverse) -> out
PyObject* rotate(PyObject* const* a, Py_ssize_t n) {
    if (n != 7 || a[1] == Py_None) Py_RETURN_NONE;
    const int dev = current_device();
    const at::Tensor* x = strided(a[0], 3, dev);
    if (!x || dtype_of(*x) < 0 || x->numel() == 0 || x->size(0) > INT_MAX || x->size(1) > 65535 || x->size(2) > 2048) Py_RETURN_NONE;
    b200_rotary r{};
    if (!rotary_args(a + 1, x->size(0), x->size(2), dev, &r)) Py_RETURN_NONE;
    at::Tensor y = at::detail::empty_cuda(x->sizes(), x->scalar_type(), x->device(), c10::nullopt);
    const int rc = b200_rotate(&r, x->data_ptr(), x->stride(0), x->stride(1), y.data_ptr(), y.stride(0), y.stride(1), dtype_of(*x), (int)x->size(0),
                               (int)x->size(1), (int)x->size(2), stream_of(dev));
    if (rc != B200_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(y));
}

// The pass from Python's arguments q, k_pages, v_pages, page_table, lengths, row_starts.
const at::Tensor* paged_args(PyObject* oq, PyObject* const* a, int dev, b200_paged* c) {
    const at::Tensor *q = strided(oq, 3, dev), *k = strided(a[0], 4, dev), *v = strided(a[1], 4, dev), *table = strided(a[2], 2, dev);
    const at::Tensor *lengths = list_of(a[3], at::kInt, -1, dev), *starts = list_of(a[4], at::kInt, -1, dev);
    if (!q || !k || !v || !table || !lengths || !starts || q->numel() == 0 || k->numel() == 0) return nullptr;
    c->dtype = dtype_of(*q);
    if ((c->dtype != B200_DTYPE_F16 && c->dtype != B200_DTYPE_BF16) || k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type() ||
        table->scalar_type() != at::kInt || k->sizes() != v->sizes() || k->strides() != v->strides() || k->size(3) != q->size(2) ||
        starts->numel() != lengths->numel() + 1 || table->size(0) != lengths->numel() || lengths->numel() == 0)
        return nullptr;
    for (int i = 0; i < 3; i++)
        if (k->size(i) > INT_MAX || (k->size(i) > 1 && k->stride(i) == 0)) return nullptr;
    if (q->size(0) > INT_MAX || q->size(1) > 4096 || q->size(1) % k->size(1) || q->size(2) > 2048 || table->size(1) > INT_MAX) return nullptr;
    const int64_t page = k->size(2);
    if (!(page == 8 || page == 16 || page == 32 || page == 64 || (page >= 128 && page % 128 == 0))) return nullptr;
    c->requests = (int)lengths->numel(); c->tokens = (int)q->size(0); c->heads = (int)q->size(1); c->kv_heads = (int)k->size(1);
    c->head_dim = (int)q->size(2); c->pages = (int)k->size(0); c->page_size = (int)page; c->table_width = (int)table->size(1);
    c->page_table = static_cast<const int*>(table->data_ptr()); c->table_stride = table->stride(0);
    c->lengths = static_cast<const int*>(lengths->data_ptr()); c->row_starts = static_cast<const int*>(starts->data_ptr());
    c->k_pages = k->data_ptr(); c->v_pages = v->data_ptr();
    c->page_stride = k->stride(0); c->head_stride = k->stride(1); c->row_stride = k->stride(2);
    return q;
}

// paged_append(q, k, v, k_pages, v_pages, page_table, lengths, row_starts, prefix_length, positions, inv_freqs, scaling_factor, magnitude, interleaved,
//              inverse) -> q_out
PyObject* paged_append(PyObject* const* a, Py_ssize_t n) {
    long prefix;
    if (n != 15 || !int_arg(a[8], &prefix) || prefix < 0 || prefix > INT_MAX) Py_RETURN_NONE;
    const int dev = current_device();
    b200_paged c{};
    const at::Tensor *q = paged_args(a[0], a + 3, dev, &c), *k = strided(a[1], 3, dev), *v = strided(a[2], 3, dev);
    if (!q || !k || !v || k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type() || k->sizes() != v->sizes() ||
        k->strides() != v->strides() || k->size(0) != c.tokens || k->size(1) != c.kv_heads || k->size(2) != c.head_dim)
        Py_RETURN_NONE;
    b200_rotary r{};
    if (!rotary_args(a + 9, c.tokens, c.head_dim, dev, &r)) Py_RETURN_NONE;
    at::Tensor y = at::detail::empty_cuda(q->sizes(), q->scalar_type(), q->device(), c10::nullopt);
    const int rc = b200_paged_append(&c, &r, q->data_ptr(), q->stride(0), q->stride(1), k->data_ptr(), v->data_ptr(), k->stride(0), k->stride(1),
                                     y.data_ptr(), y.stride(0), y.stride(1), (int)prefix, stream_of(dev));
    if (rc != B200_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(y));
}

// paged_attention(q, k_pages, v_pages, page_table, lengths, row_starts, prefix_pages, prefix_length, mask, scale, error) -> out
PyObject* paged_attention(PyObject* const* a, Py_ssize_t n) {
    long prefix;
    if (n != 11 || !int_arg(a[7], &prefix) || prefix < 0 || prefix > INT_MAX) Py_RETURN_NONE;
    const int dev = current_device();
    b200_paged c{};
    const at::Tensor *q = paged_args(a[0], a + 1, dev, &c), *error = list_of(a[10], at::kInt, 1, dev);
    if (!q || !error) Py_RETURN_NONE;
    const at::Tensor* pages = a[6] == Py_None ? nullptr : list_of(a[6], at::kInt, -1, dev);
    const at::Tensor* mask = a[8] == Py_None ? nullptr : list_of(a[8], at::kLong, c.tokens, dev);
    double scale = std::pow((double)c.head_dim, -0.5);
    if ((a[6] != Py_None && !pages) || (a[8] != Py_None && !mask) || (prefix > 0 && (!pages || pages->numel() * c.page_size < prefix)) ||
        (a[9] != Py_None && !double_arg(a[9], &scale)))
        Py_RETURN_NONE;
    const size_t room = b200_paged_attention_workspace_bytes(&c);
    at::Tensor y = at::detail::empty_cuda(q->sizes(), q->scalar_type(), q->device(), c10::nullopt);
    at::Tensor ws = at::detail::empty_cuda({(int64_t)room}, at::kByte, q->device(), c10::nullopt);
    const int rc = b200_paged_attention(&c, q->data_ptr(), q->stride(0), q->stride(1), y.data_ptr(), y.stride(0), y.stride(1),
                                        pages ? static_cast<const int*>(pages->data_ptr()) : nullptr, (int)prefix,
                                        mask ? static_cast<const unsigned long long*>(mask->data_ptr()) : nullptr, (float)scale, ws.data_ptr(), room,
                                        static_cast<int*>(error->data_ptr()), stream_of(dev));
    if (rc != B200_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(y));
}

// verify_tokens(draft_tokens, target_probs, uniforms, draft_probs, draft_lengths) -> (tokens, accepted)
PyObject* verify_tokens(PyObject* const* a, Py_ssize_t n) {
    if (n != 5) Py_RETURN_NONE;
    const int dev = current_device();
    const at::Tensor *tokens = strided(a[0], 2, dev), *p = strided(a[1], 3, dev), *u = strided(a[2], 2, dev);
    if (!tokens || !p || !u || dtype_of(*p) < 0 || tokens->scalar_type() != at::kInt || u->scalar_type() != at::kFloat) Py_RETURN_NONE;
    const int64_t B = p->size(0), K = p->size(1) - 1, V = p->size(2);
    if (B < 1 || B > 65535 || K < 0 || K > 1024 || V < 1 || V > (1 << 30) || tokens->size(0) != B || tokens->size(1) != K || u->size(0) != B ||
        u->size(1) != K + 1)
        Py_RETURN_NONE;
    const at::Tensor* q = a[3] == Py_None ? nullptr : strided(a[3], 3, dev);
    const at::Tensor* lengths = a[4] == Py_None ? nullptr : list_of(a[4], at::kInt, B, dev);
    if ((a[3] != Py_None && (!q || q->scalar_type() != p->scalar_type() || q->size(0) != B || q->size(1) != K || q->size(2) != V)) ||
        (a[4] != Py_None && !lengths))
        Py_RETURN_NONE;
    at::Tensor out = at::detail::empty_cuda({B, K + 1}, at::kInt, p->device(), c10::nullopt);
    at::Tensor accepted = at::detail::empty_cuda({B}, at::kInt, p->device(), c10::nullopt);
    const int rc = b200_verify_tokens(static_cast<const int*>(tokens->data_ptr()), tokens->stride(0), p->data_ptr(), p->stride(0), p->stride(1),
                                      q ? q->data_ptr() : nullptr, q ? q->stride(0) : 0, q ? q->stride(1) : 0, static_cast<const float*>(u->data_ptr()),
                                      u->stride(0), lengths ? static_cast<const int*>(lengths->data_ptr()) : nullptr, dtype_of(*p), (int)B, (int)K, (int)V,
                                      static_cast<int*>(out.data_ptr()), static_cast<int*>(accepted.data_ptr()), stream_of(dev));
    if (rc != B200_OK) Py_RETURN_NONE;
    PyObject* first = THPVariable_Wrap(std::move(out));
    PyObject* second = THPVariable_Wrap(std::move(accepted));
    PyObject* both = first != nullptr && second != nullptr ? PyTuple_Pack(2, first, second) : nullptr;
    Py_XDECREF(first);
    Py_XDECREF(second);
    return both;
}

// layer_pointers(layers, table[, fast]) -> 0: `table` (address of [layers][8] pointers in the order of b200_forward_desc.layer_table) holds
// the device pointers of the layers already, 1: it does now, -1: a layer is not as it should be (no re-laid-out weights, say).
// Runs ahead of every pass, so that a pass never sees the address of a tensor that has been replaced: ~0.35 us a layer.  `fast` (address of 32
// bits) becomes 1 if every re-laid-out matrix is known to allow the short expansion as it is now, as QLinear.scales_fast, 0 if not.  (Asked
// for every pass like the addresses: a matrix that has taken the place of one that was freed can have its address and its count of changes.)
PyObject* layer_pointers(PyObject*, PyObject* const* a, Py_ssize_t n) {
    static PyObject* const linears[] = {PyUnicode_InternFromString("qkv"), PyUnicode_InternFromString("o"), PyUnicode_InternFromString("gate"),
                                        PyUnicode_InternFromString("up"), PyUnicode_InternFromString("down")};
    static PyObject* const norms[] = {PyUnicode_InternFromString("input_norm"), PyUnicode_InternFromString("post_norm")};
    static PyObject* const tiled = PyUnicode_InternFromString("tiled");
    static PyObject* const bias = PyUnicode_InternFromString("bias");
    static PyObject* const fast_of = PyUnicode_InternFromString("_fast_of");
    void** table = (n == 2 || n == 3) && (PyList_Check(a[0]) || PyTuple_Check(a[0])) ? static_cast<void**>(PyLong_AsVoidPtr(a[1])) : nullptr;
    uint32_t* fast = table != nullptr && n == 3 ? static_cast<uint32_t*>(PyLong_AsVoidPtr(a[2])) : nullptr;
    if (PyErr_Occurred()) return nullptr;
    if (table == nullptr) return PyLong_FromLong(-1);
    if (fast != nullptr) *fast = 0;
    bool plain = true, same = true, all_fast = fast != nullptr;
    auto put = [&](PyObject* t, bool optional) {              // (borrowed, may be NULL)
        void* q = nullptr;
        if (t == nullptr || !THPVariable_Check(t)) plain = plain && optional && t == Py_None;
        else q = THPVariable_Unpack(t).data_ptr();
        same = same && *table == q;
        *table++ = q;
    };
    auto put_attr = [&](PyObject* o, PyObject* name, bool optional) {
        PyObject* t = o == nullptr ? nullptr : PyObject_GetAttr(o, name);
        if (t == nullptr) PyErr_Clear();
        put(t, optional);
        if (name == tiled && all_fast) {                         // (the tensor looked at, its count of changes then)
            PyObject* of = t == nullptr ? nullptr : PyObject_GetAttr(o, fast_of);
            if (of == nullptr) PyErr_Clear();
            all_fast = of != nullptr && PyTuple_Check(of) && PyTuple_GET_SIZE(of) == 2 && PyTuple_GET_ITEM(of, 0) == t && THPVariable_Check(t) &&
                       !THPVariable_Unpack(t).is_inference() && PyLong_AsLongLong(PyTuple_GET_ITEM(of, 1)) == (long long)THPVariable_Unpack(t)._version();
            if (PyErr_Occurred()) PyErr_Clear();                 // (no number there)
            Py_XDECREF(of);
        }
        Py_XDECREF(t);                                           // (the layer still holds it)
    };
    try {
        const Py_ssize_t layers = PySequence_Fast_GET_SIZE(a[0]);
        for (Py_ssize_t l = 0; l < layers; l++) {
            PyObject* layer = PySequence_Fast_GET_ITEM(a[0], l);
            if (!PyDict_Check(layer)) return PyLong_FromLong(-1);
            for (int i = 0; i < 5; i++) {
                PyObject* lin = PyDict_GetItem(layer, linears[i]);
                put_attr(lin, tiled, false);
                if (i == 0) put_attr(lin, bias, true);
            }
            for (PyObject* name : norms) put(PyDict_GetItem(layer, name), false);
        }
    } catch (const std::exception&) {                            // (a tensor without storage)
        plain = false;
    }
    if (fast != nullptr) *fast = plain && all_fast;
    return PyLong_FromLong(!plain ? -1 : (same ? 0 : 1));
}

// No C++ exception passes through the interpreter's frames: it would end the process.
template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyObject* caught(PyObject*, PyObject* const* a, Py_ssize_t n) {
    try {
        return F(a, n);
    } catch (const std::exception&) {
        Py_RETURN_NONE;
    }
}

#define FAST(name, f) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST("qmm", caught<qmm>), FAST("qmm_tiled", caught<qmm_tiled>), FAST("rope_positions", caught<rope_positions>),
                         FAST("rotate", caught<rotate>), FAST("paged_append", caught<paged_append>), FAST("paged_attention", caught<paged_attention>),
                         FAST("verify_tokens", caught<verify_tokens>),
                         FAST("layer_pointers", layer_pointers), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_b200ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__b200ops(void) { return PyModule_Create(&module); }
