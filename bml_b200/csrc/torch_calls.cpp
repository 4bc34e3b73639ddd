// torch_calls.cpp -- the usual calls of bml_b200/paged.py without Python's
// share of the time: argument checks, output allocation and the C call of its
// functions for plain CUDA tensors on the current device and stream.
//
// Every function returns None when anything is not the usual case (an argument
// that is not a plain contiguous tensor of the right type and shape, another
// device, a C call that refused); paged.py then takes its own way, which checks
// again, says what is wrong, or makes the call.  It takes every call where this
// module is missing or was built for another torch.  A refused C call has launched
// nothing.  The entry points of libbmlattn.so are handed over by set_calls().
//
// Host time of a call beside a B200, against the way through ctypes: page_plan 5.3
// and 20 us, paged_append 3.3 and 10, tree_attention (two launches) 7.1 and 16.5,
// paged_commit 4.2 and 12.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <Python.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/bml_attn.h"

namespace {

using PlanFn = decltype(&bml_paged_plan);
using AppendFn = decltype(&bml_paged_append);
using TreeFn = decltype(&bml_attn_tree_sized);
using CommitFn = decltype(&bml_paged_commit);
PlanFn g_plan = nullptr;
AppendFn g_append = nullptr;
TreeFn g_tree = nullptr;
CommitFn g_commit = nullptr;
decltype(&bml_attn_tree_workspace_size) g_tree_bytes = nullptr;
decltype(&bml_attn_chunk) g_chunk = nullptr;
decltype(&bml_attn_chunk_workspace_size) g_chunk_bytes = nullptr;
decltype(&bml_verify_drafts) g_verify = nullptr;
decltype(&bml_page_fork) g_fork = nullptr;
decltype(&bml_page_free) g_free = nullptr;
decltype(&bml_page_compact) g_compact = nullptr;

// Scratch bytes of tree_attention, asked for once a device and head size; -1: refused.
int64_t tree_bytes(int device, int64_t d) {
    static int64_t known[64][2];  // under the interpreter's lock
    const int k = d == 64 ? 0 : d == 128 ? 1 : -1;
    if (k < 0 || device < 0 || device >= 64) return -1;
    if (known[device][k] == 0) {
        size_t bytes = 0;
        if (g_tree_bytes((uint32_t)d, device, &bytes) != BML_OK) return -1;
        known[device][k] = (int64_t)bytes;
    }
    return known[device][k];
}

// A plain contiguous CUDA tensor argument, or null.
const at::Tensor *plain(PyObject *o, int64_t dim) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.dim() != dim || !t.is_contiguous() || t.is_conj() || t.is_neg()) return nullptr;
    return &t;
}

const at::Tensor *typed(PyObject *o, int64_t dim, at::ScalarType type, c10::Device dev) {
    const at::Tensor *t = plain(o, dim);
    return t && t->scalar_type() == type && t->device() == dev ? t : nullptr;
}

bool here(c10::Device dev) { return dev.index() == c10::cuda::current_device(); }
void *stream_of(c10::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

// bml_dtype of a torch type, or -1
int code(at::ScalarType t) {
    return t == at::kFloat ? BML_F32 : t == at::kHalf ? BML_F16 : t == at::kBFloat16 ? BML_BF16 : -1;
}

at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, c10::Device dev) {
    return at::detail::empty_cuda(sizes, type, dev, std::nullopt);
}

// Elements of `type` from element `at` of a buffer on, as a tensor of its own.
PyObject *piece(const at::Tensor &buf, const caffe2::TypeMeta &type, int64_t at, at::IntArrayRef sizes) {
    auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(buf.storage()), buf.key_set(), type);
    impl->set_storage_offset(at);
    impl->set_sizes_contiguous(sizes);
    return THPVariable_Wrap(at::Tensor(std::move(impl)));
}

#define USUAL(cond) \
    do {            \
        if (!(cond)) Py_RETURN_NONE; \
    } while (0)

bool integer(PyObject *o, int64_t *v) {
    if (!PyLong_CheckExact(o)) return false;
    int over = 0;
    *v = PyLong_AsLongLongAndOverflow(o, &over);
    return over == 0 && *v >= 0 && *v < (1ll << 31);
}

// lens, n_new, owned, block_table, free_pages, free_used, page_size, n_tokens, parents, n_words
PyObject *plan_impl(PyObject *const *a) {
    const at::Tensor *lens = plain(a[0], 1);
    USUAL(lens && lens->scalar_type() == at::kInt);
    const c10::Device dev = lens->device();
    const int64_t n = lens->size(0);
    const at::Tensor *n_new = typed(a[1], 1, at::kInt, dev), *owned = typed(a[2], 1, at::kInt, dev);
    const at::Tensor *table = typed(a[3], 2, at::kInt, dev), *free = typed(a[4], 1, at::kInt, dev);
    const at::Tensor *used = typed(a[5], 1, at::kInt, dev);
    int64_t page, n_tokens, words = 0;
    USUAL(here(dev) && n > 0 && n_new && owned && table && free && used && integer(a[6], &page) && integer(a[7], &n_tokens) &&
          integer(a[9], &words));
    USUAL(n_new->size(0) == n && owned->size(0) == n && table->size(0) == n && used->size(0) == 1);
    USUAL(free->size(0) < (1ll << 31) && table->size(1) < (1ll << 31) && n < (1ll << 31));
    const at::Tensor *parents = nullptr;
    if (a[8] != Py_None) {
        parents = typed(a[8], 1, at::kInt, dev);
        USUAL(parents && parents->size(0) == n_tokens && words >= 1 && words <= 4);
    }
    // all results in one buffer: slots and mask, then the int32 arrays
    const int64_t wide = n_tokens * (parents ? 1 + words : 1);
    at::Tensor all = fresh({wide + (n_tokens + 4 * n + 3) / 2}, at::kLong, dev);
    int64_t *slots = all.mutable_data_ptr<int64_t>();
    int32_t *pos = reinterpret_cast<int32_t *>(slots + wide), *b = pos + n_tokens;
    const bml_status st =
        g_plan(lens->const_data_ptr<int32_t>(), n_new->const_data_ptr<int32_t>(), owned->const_data_ptr<int32_t>(), (uint32_t)n,
               free->const_data_ptr<int32_t>(), (uint32_t)free->size(0), used->const_data_ptr<int32_t>(), (uint32_t)page,
               (uint32_t)table->size(1), table->mutable_data_ptr<int32_t>(),
               parents ? parents->const_data_ptr<int32_t>() : nullptr, (uint32_t)n_tokens, (uint32_t)words, b, b + n + 1,
               b + 2 * n + 1, b + 4 * n + 1, slots, pos, parents ? reinterpret_cast<uint64_t *>(slots + n_tokens) : nullptr,
               b + 3 * n + 1, stream_of(dev));
    USUAL(st == BML_OK);
    PyObject *out = PyTuple_New(8);
    if (!out) return nullptr;
    static const caffe2::TypeMeta i32 = caffe2::TypeMeta::Make<int32_t>(), i64 = caffe2::TypeMeta::Make<int64_t>();
    const int64_t p0 = 2 * wide, o = p0 + n_tokens;
    PyTuple_SET_ITEM(out, 0, piece(all, i32, o, {n + 1}));              // node_start
    PyTuple_SET_ITEM(out, 1, piece(all, i32, o + n + 1, {n}));          // kv_lens
    PyTuple_SET_ITEM(out, 2, piece(all, i32, o + 2 * n + 1, {n}));      // owned
    PyTuple_SET_ITEM(out, 3, piece(all, i32, o + 4 * n + 1, {1}));      // free_used
    PyTuple_SET_ITEM(out, 4, piece(all, i32, o + 3 * n + 1, {n}));      // status
    PyTuple_SET_ITEM(out, 5, piece(all, i32, p0, {n_tokens}));          // positions
    PyTuple_SET_ITEM(out, 6, piece(all, i64, 0, {n_tokens}));           // slots
    if (parents) {
        PyTuple_SET_ITEM(out, 7, piece(all, i64, n_tokens, {n_tokens, words}));
    } else {
        Py_INCREF(Py_None);
        PyTuple_SET_ITEM(out, 7, Py_None);
    }
    return out;
}

// q, k, v, slots, positions, k_pool, v_pool, q_out, theta -> q_out
PyObject *append_impl(PyObject *const *a) {
    const at::Tensor *k = plain(a[1], 3);
    USUAL(k);
    const c10::Device dev = k->device();
    const at::ScalarType type = k->scalar_type();
    const int64_t n = k->size(0), n_kv = k->size(1), d = k->size(2);
    const at::Tensor *v = typed(a[2], 3, type, dev), *slots = typed(a[3], 1, at::kLong, dev), *kp = plain(a[5], 4);
    USUAL(here(dev) && v && slots && kp && kp->device() == dev && code(type) >= 0 && code(kp->scalar_type()) >= 0);
    const at::Tensor *vp = typed(a[6], 4, kp->scalar_type(), dev);
    USUAL(vp && v->sizes() == k->sizes() && slots->size(0) == n && vp->sizes() == kp->sizes() && kp->size(2) == n_kv &&
          kp->size(3) == d && n < (1ll << 31));
    const at::Tensor *pos = nullptr, *q = nullptr, *q_out = nullptr;
    if (a[4] != Py_None) {
        pos = typed(a[4], 1, at::kInt, dev);
        USUAL(pos && pos->size(0) == n);
    }
    PyObject *ret = Py_None;
    int64_t heads = 0;
    if (a[0] != Py_None) {
        q = q_out = typed(a[0], 3, type, dev);
        USUAL(q && q->size(0) == n && q->size(2) == d);
        heads = q->size(1);
        ret = a[0];
        if (a[7] != Py_None) {
            q_out = typed(a[7], 3, type, dev);
            USUAL(q_out && q_out->sizes() == q->sizes());
            ret = a[7];
        }
    } else {
        USUAL(a[7] == Py_None);
    }
    const double theta = PyFloat_CheckExact(a[8]) ? PyFloat_AS_DOUBLE(a[8]) : -1.0;
    const bml_status st = g_append(
        q ? q->const_data_ptr() : nullptr, k->const_data_ptr(), v->const_data_ptr(), (bml_dtype)code(type),
        slots->const_data_ptr<int64_t>(), pos ? pos->const_data_ptr<int32_t>() : nullptr, (uint32_t)n, (uint32_t)heads,
        (uint32_t)n_kv, (uint32_t)d, theta, q_out ? q_out->mutable_data_ptr() : nullptr, kp->mutable_data_ptr(),
        vp->mutable_data_ptr(), (bml_dtype)code(kp->scalar_type()), (uint64_t)(kp->size(0) * kp->size(1)), stream_of(dev));
    USUAL(st == BML_OK);
    // q None: something that is not None says that the call was made
    if (ret == Py_None) Py_RETURN_TRUE;
    Py_INCREF(ret);
    return ret;
}

// q, k_pool, v_pool, block_table, kv_lens, node_start, mask, scale, n_live, max_new -> out
PyObject *tree_impl(PyObject *const *a) {
    const at::Tensor *q = plain(a[0], 3), *k = plain(a[1], 4), *lens = plain(a[4], 1);
    USUAL(q && k && lens);
    const c10::Device dev = q->device();
    const at::Tensor *v = typed(a[2], 4, k->scalar_type(), dev), *table = typed(a[3], 2, at::kInt, dev);
    const at::Tensor *start = typed(a[5], 1, at::kInt, dev);
    USUAL(here(dev) && k->device() == dev && lens->device() == dev && lens->scalar_type() == at::kInt && v && table && start &&
          code(q->scalar_type()) >= 0 && code(k->scalar_type()) >= 0);
    const int64_t n = lens->size(0), n_tokens = q->size(0), d = q->size(2);
    USUAL(v->sizes() == k->sizes() && k->size(3) == d && start->size(0) == n + 1 && table->size(0) == n && n > 0 && n_tokens > 0 &&
          n_tokens < (1ll << 31) && k->size(0) < (1ll << 31) && k->size(1) < (1ll << 31) && table->size(1) < (1ll << 31));
    const at::Tensor *mask = nullptr;
    if (a[6] != Py_None) {
        mask = typed(a[6], 2, at::kLong, dev);
        USUAL(mask && mask->size(0) == n_tokens && mask->size(1) >= 1 && mask->size(1) <= 4);
    }
    const int64_t ws_bytes = tree_bytes(dev.index(), d);
    int64_t live, most;
    USUAL(PyFloat_CheckExact(a[7]) && ws_bytes > 0 && integer(a[8], &live) && integer(a[9], &most));
    at::Tensor out = fresh(q->sizes(), q->scalar_type(), dev), ws = fresh({ws_bytes}, at::kByte, dev);
    const bml_status st =
        g_tree(q->const_data_ptr(), (bml_dtype)code(q->scalar_type()), (uint32_t)n_tokens, (uint32_t)q->size(1),
               (uint32_t)k->size(2), (uint32_t)d, k->const_data_ptr(), v->const_data_ptr(), (bml_dtype)code(k->scalar_type()),
               (uint32_t)k->size(0), (uint32_t)k->size(1), table->const_data_ptr<int32_t>(), (uint32_t)table->size(1),
               lens->const_data_ptr<int32_t>(), start->const_data_ptr<int32_t>(), (uint32_t)n,
               mask ? reinterpret_cast<const uint64_t *>(mask->const_data_ptr<int64_t>()) : nullptr,
               mask ? (uint32_t)mask->size(1) : 0u, (float)PyFloat_AS_DOUBLE(a[7]), out.mutable_data_ptr(), ws.mutable_data_ptr(),
               (size_t)ws_bytes, (uint32_t)live, (uint32_t)most, stream_of(dev));
    USUAL(st == BML_OK);
    return THPVariable_Wrap(std::move(out));
}

// k_pools, v_pools, block_table, lens, kv_lens, node_start, path, n_accept -> new lens
PyObject *commit_impl(PyObject *const *a) {
    const at::Tensor *k = plain(a[0], 5);
    USUAL(k);
    const c10::Device dev = k->device();
    const at::Tensor *v = typed(a[1], 5, k->scalar_type(), dev), *table = typed(a[2], 2, at::kInt, dev);
    const at::Tensor *lens = typed(a[3], 1, at::kInt, dev), *kv = typed(a[4], 1, at::kInt, dev);
    const at::Tensor *start = typed(a[5], 1, at::kInt, dev), *path = typed(a[6], 2, at::kInt, dev);
    const at::Tensor *accept = typed(a[7], 1, at::kInt, dev);
    USUAL(here(dev) && v && table && lens && kv && start && path && accept && code(k->scalar_type()) >= 0);
    const int64_t n = lens->size(0);
    USUAL(v->sizes() == k->sizes() && n > 0 && kv->size(0) == n && start->size(0) == n + 1 && accept->size(0) == n &&
          table->size(0) == n && path->size(0) == n && n < (1ll << 31) && path->size(1) < (1ll << 31) &&
          table->size(1) < (1ll << 31) && k->size(0) < (1ll << 31) && k->size(1) < (1ll << 31) && k->size(2) < (1ll << 31));
    at::Tensor out = fresh({n}, at::kInt, dev);
    const bml_status st =
        g_commit(k->mutable_data_ptr(), v->mutable_data_ptr(), (uint32_t)k->size(0), (uint32_t)k->size(1), (uint32_t)k->size(2),
                 (uint32_t)k->size(3), (uint32_t)k->size(4), (bml_dtype)code(k->scalar_type()), table->const_data_ptr<int32_t>(),
                 (uint32_t)table->size(1), lens->const_data_ptr<int32_t>(), kv->const_data_ptr<int32_t>(),
                 start->const_data_ptr<int32_t>(), (uint32_t)n, path->const_data_ptr<int32_t>(), (uint32_t)path->size(1),
                 accept->const_data_ptr<int32_t>(), out.mutable_data_ptr<int32_t>(), stream_of(dev));
    USUAL(st == BML_OK);
    return THPVariable_Wrap(std::move(out));
}

// q, k_pool, v_pool, block_table, kv_lens, node_start, scale -> out
PyObject *chunk_impl(PyObject *const *a) {
    const at::Tensor *q = plain(a[0], 3), *k = plain(a[1], 4), *lens = plain(a[4], 1);
    USUAL(q && k && lens);
    const c10::Device dev = q->device();
    const at::Tensor *v = typed(a[2], 4, k->scalar_type(), dev), *table = typed(a[3], 2, at::kInt, dev);
    const at::Tensor *start = typed(a[5], 1, at::kInt, dev);
    USUAL(here(dev) && k->device() == dev && lens->device() == dev && lens->scalar_type() == at::kInt && v && table && start &&
          code(q->scalar_type()) >= 0 && code(k->scalar_type()) >= 0 && PyFloat_CheckExact(a[6]));
    const int64_t n = lens->size(0), n_tokens = q->size(0), d = q->size(2);
    USUAL(v->sizes() == k->sizes() && k->size(3) == d && start->size(0) == n + 1 && table->size(0) == n && n > 0 && n_tokens > 0 &&
          n < (1ll << 31) && n_tokens < (1ll << 31) && k->size(0) < (1ll << 31) && k->size(1) < (1ll << 31) && table->size(1) < (1ll << 31));
    size_t ws_bytes = 0;
    int64_t live, most;
    USUAL(integer(a[7], &live) && integer(a[8], &most));
    USUAL(g_chunk_bytes((uint32_t)d, (uint32_t)n_tokens, (uint32_t)n, dev.index(), &ws_bytes) == BML_OK);
    at::Tensor out = fresh(q->sizes(), q->scalar_type(), dev), ws = fresh({(int64_t)ws_bytes}, at::kByte, dev);
    const bml_status st =
        g_chunk(q->const_data_ptr(), (bml_dtype)code(q->scalar_type()), (uint32_t)n_tokens, (uint32_t)q->size(1), (uint32_t)k->size(2),
                (uint32_t)d, k->const_data_ptr(), v->const_data_ptr(), (bml_dtype)code(k->scalar_type()), (uint32_t)k->size(0),
                (uint32_t)k->size(1), table->const_data_ptr<int32_t>(), (uint32_t)table->size(1), lens->const_data_ptr<int32_t>(),
                start->const_data_ptr<int32_t>(), (uint32_t)n, (float)PyFloat_AS_DOUBLE(a[6]), out.mutable_data_ptr(),
                ws.mutable_data_ptr(), ws_bytes, (uint32_t)live, (uint32_t)most, stream_of(dev));
    USUAL(st == BML_OK);
    return THPVariable_Wrap(std::move(out));
}

// Consecutive pieces of an int32 buffer, as a tuple of vectors.
PyObject *pieces(const at::Tensor &buf, std::initializer_list<int64_t> sizes) {
    static const caffe2::TypeMeta i32 = caffe2::TypeMeta::Make<int32_t>();
    PyObject *out = PyTuple_New((Py_ssize_t)sizes.size());
    if (!out) return nullptr;
    int64_t at = 0;
    Py_ssize_t i = 0;
    for (int64_t n : sizes) {
        PyTuple_SET_ITEM(out, i++, piece(buf, i32, at, {n}));
        at += n;
    }
    return out;
}

// target, draft, tokens, parents, node_start, u, u_next, max_path -> path, n_accept, next
PyObject *verify_impl(PyObject *const *a) {
    const at::Tensor *p = plain(a[0], 2);
    USUAL(p && code(p->scalar_type()) >= 0);
    const c10::Device dev = p->device();
    const at::Tensor *q = nullptr, *tok = typed(a[2], 1, at::kInt, dev), *par = typed(a[3], 1, at::kInt, dev);
    const at::Tensor *start = typed(a[4], 1, at::kInt, dev), *u = typed(a[5], 1, at::kFloat, dev), *un = typed(a[6], 1, at::kFloat, dev);
    int64_t most;
    USUAL(here(dev) && tok && par && start && u && un && integer(a[7], &most) && most > 0);
    if (a[1] != Py_None) {
        q = typed(a[1], 2, p->scalar_type(), dev);
        USUAL(q && q->sizes() == p->sizes());
    }
    const int64_t rows = p->size(0), n = start->size(0) - 1;
    USUAL(n > 0 && n < (1ll << 31) && rows < (1ll << 31) && p->size(1) < (1ll << 31) && tok->size(0) == rows && par->size(0) == rows &&
          u->size(0) == rows && un->size(0) == n);
    at::Tensor all = fresh({n * (most + 2)}, at::kInt, dev);
    int32_t *path = all.mutable_data_ptr<int32_t>();
    const bml_status st =
        g_verify(p->const_data_ptr(), q ? q->const_data_ptr() : nullptr, (bml_dtype)code(p->scalar_type()), (uint32_t)p->size(1),
                 tok->const_data_ptr<int32_t>(), par->const_data_ptr<int32_t>(), (uint32_t)rows, start->const_data_ptr<int32_t>(),
                 (uint32_t)n, u->const_data_ptr<float>(), un->const_data_ptr<float>(), (uint32_t)most, path, path + n * most,
                 path + n * most + n, stream_of(dev));
    USUAL(st == BML_OK);
    static const caffe2::TypeMeta i32 = caffe2::TypeMeta::Make<int32_t>();
    PyObject *out = PyTuple_New(3);
    if (!out) return nullptr;
    PyTuple_SET_ITEM(out, 0, piece(all, i32, 0, {n, most}));
    PyTuple_SET_ITEM(out, 1, piece(all, i32, n * most, {n}));
    PyTuple_SET_ITEM(out, 2, piece(all, i32, n * most + n, {n}));
    return out;
}

// Whether a layered pool's sizes fit the C calls'.
bool sizes32(const at::Tensor *k) {
    for (int64_t s : k->sizes())
        if (s >= (1ll << 31)) return false;
    return true;
}

// k_pools, v_pools, src, dst, lens, owned, block_table, shared, free_pages, free_used
//   -> lens, owned, shared, free_used, status
PyObject *fork_impl(PyObject *const *a) {
    const at::Tensor *k = plain(a[0], 5);
    USUAL(k && code(k->scalar_type()) >= 0 && sizes32(k));
    const c10::Device dev = k->device();
    const at::Tensor *v = typed(a[1], 5, k->scalar_type(), dev), *src = typed(a[2], 1, at::kInt, dev), *dst = typed(a[3], 1, at::kInt, dev);
    const at::Tensor *lens = typed(a[4], 1, at::kInt, dev), *owned = typed(a[5], 1, at::kInt, dev), *table = typed(a[6], 2, at::kInt, dev);
    const at::Tensor *shared = typed(a[7], 1, at::kInt, dev), *free = typed(a[8], 1, at::kInt, dev), *used = typed(a[9], 1, at::kInt, dev);
    USUAL(here(dev) && v && src && dst && lens && owned && table && shared && free && used);
    const int64_t n = lens->size(0), m = src->size(0), pages = k->size(1);
    USUAL(v->sizes() == k->sizes() && n > 0 && n < (1ll << 31) && m < (1ll << 31) && dst->size(0) == m && owned->size(0) == n &&
          table->size(0) == n && table->size(1) < (1ll << 31) && shared->size(0) == pages && free->size(0) < (1ll << 31) &&
          used->size(0) == 1);
    at::Tensor all = fresh({2 * n + pages + 1 + m}, at::kInt, dev);
    int32_t *o = all.mutable_data_ptr<int32_t>();
    const bml_status st =
        g_fork(k->mutable_data_ptr(), v->mutable_data_ptr(), (uint32_t)k->size(0), (uint32_t)pages, (uint32_t)k->size(2),
               (uint32_t)k->size(3), (uint32_t)k->size(4), (bml_dtype)code(k->scalar_type()), src->const_data_ptr<int32_t>(),
               dst->const_data_ptr<int32_t>(), (uint32_t)m, lens->const_data_ptr<int32_t>(), owned->const_data_ptr<int32_t>(), (uint32_t)n,
               table->mutable_data_ptr<int32_t>(), (uint32_t)table->size(1), shared->const_data_ptr<int32_t>(),
               free->const_data_ptr<int32_t>(), (uint32_t)free->size(0), used->const_data_ptr<int32_t>(), o, o + n, o + 2 * n,
               o + 2 * n + pages, o + 2 * n + pages + 1, stream_of(dev));
    USUAL(st == BML_OK);
    return pieces(all, {n, n, pages, 1, m});
}

// keep, lens, owned, block_table, page_size, shared, free_pages, free_used
//   -> lens, owned, shared, free_pages, free_used, status
PyObject *free_impl(PyObject *const *a) {
    const at::Tensor *lens = plain(a[1], 1);
    USUAL(lens && lens->scalar_type() == at::kInt);
    const c10::Device dev = lens->device();
    const int64_t n = lens->size(0);
    const at::Tensor *keep = typed(a[0], 1, at::kInt, dev), *owned = typed(a[2], 1, at::kInt, dev), *table = typed(a[3], 2, at::kInt, dev);
    const at::Tensor *shared = typed(a[5], 1, at::kInt, dev), *free = typed(a[6], 1, at::kInt, dev), *used = typed(a[7], 1, at::kInt, dev);
    int64_t page;
    USUAL(here(dev) && n > 0 && n < (1ll << 31) && keep && owned && table && shared && free && used && integer(a[4], &page));
    const int64_t pages = shared->size(0), n_free = free->size(0);
    USUAL(keep->size(0) == n && owned->size(0) == n && table->size(0) == n && table->size(1) < (1ll << 31) && pages < (1ll << 31) &&
          n_free < (1ll << 31) && used->size(0) == 1);
    const int64_t work = 1024 + (n_free + 31) / 32;
    at::Tensor all = fresh({3 * n + pages + n_free + 1 + work}, at::kInt, dev);
    int32_t *o = all.mutable_data_ptr<int32_t>();
    const bml_status st =
        g_free(keep->const_data_ptr<int32_t>(), lens->const_data_ptr<int32_t>(), owned->const_data_ptr<int32_t>(), (uint32_t)n,
               table->const_data_ptr<int32_t>(), (uint32_t)table->size(1), (uint32_t)page, shared->const_data_ptr<int32_t>(),
               (uint32_t)pages, free->const_data_ptr<int32_t>(), (uint32_t)n_free, used->const_data_ptr<int32_t>(), o, o + n, o + 2 * n,
               o + 2 * n + pages, o + 2 * n + pages + n_free, o + 2 * n + pages + n_free + 1, o + 3 * n + pages + n_free + 1, 4 * (size_t)work,
               stream_of(dev));
    USUAL(st == BML_OK);
    return pieces(all, {n, n, pages, n_free, 1, n});
}

// k_pools, v_pools, owned, block_table, shared -> block_table, shared, free_pages, free_used
PyObject *compact_impl(PyObject *const *a) {
    const at::Tensor *k = plain(a[0], 5);
    USUAL(k && code(k->scalar_type()) >= 0 && sizes32(k));
    const c10::Device dev = k->device();
    const at::Tensor *v = typed(a[1], 5, k->scalar_type(), dev), *owned = typed(a[2], 1, at::kInt, dev);
    const at::Tensor *table = typed(a[3], 2, at::kInt, dev), *shared = typed(a[4], 1, at::kInt, dev);
    USUAL(here(dev) && v && owned && table && shared && v->sizes() == k->sizes());
    const int64_t n = owned->size(0), wide = table->size(1), pages = k->size(1);
    USUAL(n > 0 && n < (1ll << 31) && table->size(0) == n && wide < (1ll << 31) && shared->size(0) == pages);
    at::Tensor all = fresh({n * wide + 2 * pages + 1}, at::kInt, dev), work = fresh({3 * pages + 1}, at::kInt, dev);
    int32_t *o = all.mutable_data_ptr<int32_t>(), *s = o + n * wide;
    const bml_status st =
        g_compact(k->mutable_data_ptr(), v->mutable_data_ptr(), (uint32_t)k->size(0), (uint32_t)pages, (uint32_t)k->size(2),
                  (uint32_t)k->size(3), (uint32_t)k->size(4), (bml_dtype)code(k->scalar_type()), owned->const_data_ptr<int32_t>(),
                  (uint32_t)n, table->const_data_ptr<int32_t>(), (uint32_t)wide, shared->const_data_ptr<int32_t>(), o, s, s + pages,
                  s + 2 * pages, work.mutable_data_ptr(), (size_t)(4 * (3 * pages + 1)), stream_of(dev));
    USUAL(st == BML_OK);
    static const caffe2::TypeMeta i32 = caffe2::TypeMeta::Make<int32_t>();
    PyObject *out = PyTuple_New(4);
    if (!out) return nullptr;
    PyTuple_SET_ITEM(out, 0, piece(all, i32, 0, {n, wide}));
    PyTuple_SET_ITEM(out, 1, piece(all, i32, n * wide, {pages}));
    PyTuple_SET_ITEM(out, 2, piece(all, i32, n * wide + pages, {pages}));
    PyTuple_SET_ITEM(out, 3, piece(all, i32, n * wide + 2 * pages, {1}));
    return out;
}

// No C++ exception leaves: an allocation that fails is left to paged.py, which
// meets it again and raises it.
template <PyObject *(*F)(PyObject *const *), Py_ssize_t kArgs>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (n != kArgs) {
        PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", kArgs, n);
        return nullptr;
    }
    try {
        return F(args);
    } catch (...) {
        Py_RETURN_NONE;
    }
}

PyObject *set_calls(PyObject *, PyObject *const *args, Py_ssize_t n) {
    constexpr Py_ssize_t kCalls = 11;
    if (n != kCalls) {
        PyErr_Format(PyExc_TypeError, "%zd addresses expected", kCalls);
        return nullptr;
    }
    void *p[kCalls];
    for (Py_ssize_t i = 0; i < kCalls; ++i) {
        p[i] = PyLong_AsVoidPtr(args[i]);
        if (!p[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
            return nullptr;
        }
    }
    g_plan = reinterpret_cast<PlanFn>(p[0]);
    g_append = reinterpret_cast<AppendFn>(p[1]);
    g_tree = reinterpret_cast<TreeFn>(p[2]);
    g_commit = reinterpret_cast<CommitFn>(p[3]);
    g_tree_bytes = reinterpret_cast<decltype(g_tree_bytes)>(p[4]);
    g_chunk = reinterpret_cast<decltype(g_chunk)>(p[5]);
    g_chunk_bytes = reinterpret_cast<decltype(g_chunk_bytes)>(p[6]);
    g_verify = reinterpret_cast<decltype(g_verify)>(p[7]);
    g_fork = reinterpret_cast<decltype(g_fork)>(p[8]);
    g_free = reinterpret_cast<decltype(g_free)>(p[9]);
    g_compact = reinterpret_cast<decltype(g_compact)>(p[10]);
    Py_RETURN_NONE;
}

#define ENTRY(name, n) \
    {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<name##_impl, n>)), METH_FASTCALL, nullptr}

PyMethodDef methods[] = {
    ENTRY(plan, 10),
    ENTRY(append, 9),
    ENTRY(tree, 10),
    ENTRY(commit, 8),
    ENTRY(chunk, 9),
    ENTRY(verify, 8),
    ENTRY(fork, 10),
    ENTRY(free, 8),
    ENTRY(compact, 5),
    {"set_calls", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&set_calls)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// built_for: the torch version, which paged.py compares: the classes above are
// that version's.
PyMODINIT_FUNC PyInit__torch_calls(void) {
    PyObject *m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "built_for", BML_TORCH_VERSION) < 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
