// cscr._fast: the ordinary calls of the 8-bit cache, norm, scored-attention and 8-bit
// projection ops without their Python argument handling.
//
// Each function takes the op's tensors, looks them over, allocates the results
// and calls the C ABI's entry point: about 5 us of host time less than the same
// steps in Python, which is most of a small call. It answers None for every call
// that is not plainly in order (a check that fails, an error of the entry point,
// a stream being captured, a device other than the current one, scratch not yet
// there); the op's Python code then takes the call from the start and raises
// its messages. So nothing here reports an error, and nothing depends on this
// module being there.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <ATen/record_function.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <vector>

#include "tinyllama_b200.h"

namespace {

using at::ScalarType;
using at::Tensor;

// Entry points of the loaded library (bind()).
int (*g_attention)(const tlb_scored_attention_args*, void*) = nullptr;
int (*g_write)(const tlb_quantized_write_args*, void*) = nullptr;
int (*g_read)(const tlb_dequantize_args*, void*) = nullptr;
int (*g_norm)(const tlb_qk_norm_rope_args*, void*) = nullptr;
int (*g_rows)(const tlb_quantize_rows_args*, void*) = nullptr;
int (*g_product)(const tlb_matmul_quantized_args*, void*) = nullptr;

// Scratch of the attention op: owned by the Python side, one for each stream.
struct Scratch {
    int device;
    void* stream;
    void* ptr;
    int64_t bytes;
};
std::vector<Scratch> g_scratch;  // under the GIL

int code_of(ScalarType t) {
    switch (t) {
        case ScalarType::Float: return TLB_FLOAT32;
        case ScalarType::Half: return TLB_FLOAT16;
        case ScalarType::BFloat16: return TLB_BFLOAT16;
        case ScalarType::Int: return TLB_INT32;
        case ScalarType::Long: return TLB_INT64;
        case ScalarType::Float8_e4m3fn: return TLB_FLOAT8_E4M3;
        case ScalarType::Char: return TLB_INT8;
        default: return -1;
    }
}
bool is_float(ScalarType t) {
    return t == ScalarType::Float || t == ScalarType::Half || t == ScalarType::BFloat16;
}
bool is_index(ScalarType t) { return t == ScalarType::Int || t == ScalarType::Long; }
bool is_8bit(ScalarType t) { return t == ScalarType::Float8_e4m3fn || t == ScalarType::Char; }

// The tensor of an argument; null when it is something else.
const Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// Device and stream of a call, and its tensors' agreement with them.
struct Place {
    int device;
    void* stream;
    explicit Place(const Tensor& t) : device(-1), stream(nullptr) {
        if (!t.is_cuda() || t.get_device() != c10::cuda::current_device()) return;
        device = (int)t.get_device();
        stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
    }
    bool ok() const { return device >= 0; }
    // a contiguous tensor on this device
    bool has(const Tensor* t) const {
        return t != nullptr && t->is_cuda() && t->get_device() == device && t->is_contiguous();
    }
};

// 8-bit caches [NB, KVH, bs, D] and their scales [NB, KVH, bs].
bool quantized_caches(const Place& at, const Tensor* kc, const Tensor* vc, const Tensor* ks,
                      const Tensor* vs) {
    return at.has(kc) && at.has(vc) && at.has(ks) && at.has(vs) && kc->dim() == 4 &&
           vc->sizes() == kc->sizes() && is_8bit(kc->scalar_type()) &&
           vc->scalar_type() == kc->scalar_type() &&
           ks->scalar_type() == ScalarType::Float8_e8m0fnu &&
           vs->scalar_type() == ScalarType::Float8_e8m0fnu &&
           ks->sizes() == kc->sizes().slice(0, 3) && vs->sizes() == ks->sizes() && kc->numel() > 0;
}

// [T, KVH, D] or [T, KVH * D] with each token's heads contiguous.
bool token_rows(const Place& at, const Tensor* x, int64_t tokens, int64_t kvh, int64_t d) {
    if (x == nullptr || !x->is_cuda() || x->get_device() != at.device) return false;
    if (x->dim() == 3)
        return x->size(0) == tokens && x->size(1) == kvh && x->size(2) == d && x->stride(2) == 1 &&
               (kvh == 1 || x->stride(1) == d);
    return x->dim() == 2 && x->size(0) == tokens && x->size(1) == kvh * d && x->stride(1) == 1;
}

bool number(PyObject* o, double* x) {
    *x = PyFloat_AsDouble(o);
    if (*x == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}
bool whole(PyObject* o, int64_t* x) {
    if (!PyLong_Check(o)) return false;
    *x = PyLong_AsLongLong(o);
    if (*x == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}

bool truth(PyObject* o, bool* x) {
    const int t = PyObject_IsTrue(o);
    *x = t > 0;
    if (t < 0) PyErr_Clear();
    return t >= 0;
}

PyObject* later() { Py_RETURN_NONE; }

// Whether nothing but the allocator takes part in an allocation: no dispatch mode or other
// key of this thread, no fill of new memory under deterministic algorithms, no profiler.
bool only_allocates() {
    const auto keys = c10::impl::tls_local_dispatch_key_set().included_;
    const at::Context& context = at::globalContext();
    return (keys - c10::default_included_set).empty() && !at::hasCallbacks() &&
           !(context.deterministicAlgorithms() && context.deterministicFillUninitializedMemory());
}

// A new dense tensor; through the dispatcher it takes 0.3 us longer.
Tensor dense(const Tensor& like, at::IntArrayRef sizes, ScalarType type) {
    if (!only_allocates())
        return at::empty(sizes, like.options().dtype(type), at::MemoryFormat::Contiguous);
    return Tensor(at::detail::empty_cuda(sizes, type, like.device(), at::MemoryFormat::Contiguous));
}

// attention(query, key_cache, value_cache, key_scales, value_scales, block_tables,
//           seq_lens, scale, softcap, alibi_slopes, window, overlap)
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 12 || g_attention == nullptr) return later();
    const Tensor *q = tensor(a[0]), *kc = tensor(a[1]), *vc = tensor(a[2]), *ks = tensor(a[3]),
                 *vs = tensor(a[4]), *bt = tensor(a[5]), *sl = tensor(a[6]), *slopes = tensor(a[9]);
    double scale, softcap;
    int64_t window;
    bool overlap;
    if (q == nullptr || !number(a[7], &scale) || !number(a[8], &softcap) ||
        !whole(a[10], &window) || !truth(a[11], &overlap))
        return later();
    const Place at(*q);
    if (!at.ok() || !at.has(kc) || !at.has(vc) || !at.has(bt) || !at.has(sl)) return later();
    if (q->dim() != 3 || kc->dim() != 4 || bt->dim() != 2 || sl->dim() != 1 ||
        vc->sizes() != kc->sizes() || vc->scalar_type() != kc->scalar_type() ||
        !is_float(q->scalar_type()))
        return later();
    const int64_t S = q->size(0), H = q->size(1), D = q->size(2), kvh = kc->size(1);
    if (S == 0 || H == 0 || D == 0 || kc->numel() == 0 || bt->size(1) == 0 || H % kvh != 0 ||
        kc->size(3) != D || q->stride(2) != 1 || q->stride(1) != D || bt->size(0) != S ||
        sl->size(0) != S || bt->scalar_type() != ScalarType::Int ||
        sl->scalar_type() != ScalarType::Int)
        return later();
    if (ks != nullptr ? !quantized_caches(at, kc, vc, ks, vs)
                      : a[3] != Py_None || a[4] != Py_None || kc->scalar_type() != q->scalar_type())
        return later();
    if (slopes != nullptr ? !at.has(slopes) || slopes->scalar_type() != ScalarType::Float ||
                                slopes->dim() != 1 || slopes->size(0) != H
                          : a[9] != Py_None)
        return later();
    const Scratch* scratch = nullptr;
    for (const Scratch& s : g_scratch)
        if (s.device == at.device && s.stream == at.stream) scratch = &s;
    if (scratch == nullptr || at::cuda::currentStreamCaptureStatusMayInitCtx() !=
                                  at::cuda::CaptureStatus::None)
        return later();
    Tensor out = dense(*q, q->sizes(), q->scalar_type());
    tlb_scored_attention_args p{};
    p.out = out.data_ptr();
    p.query = q->data_ptr();
    p.key_cache = kc->data_ptr();
    p.value_cache = vc->data_ptr();
    p.key_scales = ks ? ks->data_ptr() : nullptr;
    p.value_scales = ks ? vs->data_ptr() : nullptr;
    p.block_tables = static_cast<const int32_t*>(bt->data_ptr());
    p.seq_lens = static_cast<const int32_t*>(sl->data_ptr());
    p.alibi_slopes = slopes ? static_cast<const float*>(slopes->data_ptr()) : nullptr;
    p.workspace = scratch->ptr;
    p.workspace_bytes = scratch->bytes;
    p.num_seqs = S;
    p.num_heads = H;
    p.num_kv_heads = kvh;
    p.head_dim = D;
    p.num_blocks = kc->size(0);
    p.block_size = kc->size(2);
    p.max_blocks_per_seq = bt->size(1);
    p.query_stride = q->stride(0);
    p.window = window;
    p.dtype = code_of(q->scalar_type());
    p.cache_dtype = code_of(kc->scalar_type());
    p.flags = overlap ? TLB_ATTN_OVERLAP_PROLOGUE : 0;
    p.scale = scale;
    p.softcap = softcap;
    if (g_attention(&p, at.stream) != TLB_OK) return later();
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// write(key, value, key_cache, value_cache, key_scales, value_scales, slots)
PyObject* write(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 7 || g_write == nullptr) return later();
    const Tensor *k = tensor(a[0]), *v = tensor(a[1]), *kc = tensor(a[2]), *vc = tensor(a[3]),
                 *ks = tensor(a[4]), *vs = tensor(a[5]), *slots = tensor(a[6]);
    if (kc == nullptr) return later();
    const Place at(*kc);
    if (!at.ok() || !quantized_caches(at, kc, vc, ks, vs) || !at.has(slots) || slots->dim() != 1 ||
        !is_index(slots->scalar_type()))
        return later();
    const int64_t T = slots->size(0), kvh = kc->size(1), D = kc->size(3);
    if (T == 0 || !token_rows(at, k, T, kvh, D) || !token_rows(at, v, T, kvh, D) ||
        !is_float(k->scalar_type()) || v->scalar_type() != k->scalar_type())
        return later();
    tlb_quantized_write_args p{};
    p.key = k->data_ptr();
    p.value = v->data_ptr();
    p.key_cache = kc->data_ptr();
    p.value_cache = vc->data_ptr();
    p.key_scales = ks->data_ptr();
    p.value_scales = vs->data_ptr();
    p.slots = slots->data_ptr();
    p.slot_dtype = code_of(slots->scalar_type());
    p.num_tokens = T;
    p.num_kv_heads = kvh;
    p.head_size = D;
    p.num_blocks = kc->size(0);
    p.block_size = kc->size(2);
    p.key_stride = k->stride(0);
    p.value_stride = v->stride(0);
    p.dtype = code_of(k->scalar_type());
    p.cache_dtype = code_of(kc->scalar_type());
    if (g_write(&p, at.stream) != TLB_OK) return later();
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// read(key_cache, value_cache, key_scales, value_scales, block_ids, dtype)
PyObject* read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6 || g_read == nullptr) return later();
    const Tensor *kc = tensor(a[0]), *vc = tensor(a[1]), *ks = tensor(a[2]), *vs = tensor(a[3]),
                 *ids = tensor(a[4]);
    if (kc == nullptr || !THPDtype_Check(a[5])) return later();
    const ScalarType type = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
    const Place at(*kc);
    if (!at.ok() || !quantized_caches(at, kc, vc, ks, vs) || !at.has(ids) || ids->dim() != 1 ||
        ids->size(0) == 0 || !is_index(ids->scalar_type()) || !is_float(type))
        return later();
    const int64_t shape[4] = {ids->size(0), kc->size(1), kc->size(2), kc->size(3)};
    Tensor k = dense(*kc, shape, type), v = dense(*kc, shape, type);
    tlb_dequantize_args p{};
    p.key_out = k.data_ptr();
    p.value_out = v.data_ptr();
    p.key_cache = kc->data_ptr();
    p.value_cache = vc->data_ptr();
    p.key_scales = ks->data_ptr();
    p.value_scales = vs->data_ptr();
    p.block_ids = ids->data_ptr();
    p.id_dtype = code_of(ids->scalar_type());
    p.num_ids = shape[0];
    p.num_kv_heads = shape[1];
    p.head_size = shape[3];
    p.num_blocks = kc->size(0);
    p.block_size = shape[2];
    p.dtype = code_of(type);
    p.cache_dtype = code_of(kc->scalar_type());
    if (g_read(&p, at.stream) != TLB_OK) return later();
    PyObject *pk = THPVariable_Wrap(std::move(k)), *pv = THPVariable_Wrap(std::move(v));
    PyObject* both = pk && pv ? PyTuple_Pack(2, pk, pv) : nullptr;
    Py_XDECREF(pk);
    Py_XDECREF(pv);
    return both;
    END_HANDLE_TH_ERRORS
}

// norm(positions, query, key, value, query_weight, key_weight, eps, key_cache,
//      value_cache, slots, head_size, cos_sin_cache, block_tables, key_scales,
//      value_scales, overlap); value and caches None: (query, key), else query
PyObject* norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 16 || g_norm == nullptr) return later();
    const Tensor *pos = tensor(a[0]), *q = tensor(a[1]), *k = tensor(a[2]), *v = tensor(a[3]),
                 *wq = tensor(a[4]), *wk = tensor(a[5]), *kc = tensor(a[7]), *vc = tensor(a[8]),
                 *slots = tensor(a[9]), *table = tensor(a[11]), *bt = tensor(a[12]),
                 *ks = tensor(a[13]), *vs = tensor(a[14]);
    double eps;
    int64_t D;
    bool overlap;
    if (q == nullptr || k == nullptr || !number(a[6], &eps) || !whole(a[10], &D) || D <= 0 ||
        !truth(a[15], &overlap))
        return later();
    const Place at(*q);
    if (!at.ok() || !at.has(pos) || !at.has(wq) || !at.has(wk) || !at.has(table) || !k->is_cuda() ||
        k->get_device() != at.device)
        return later();
    const ScalarType type = q->scalar_type();
    if (!is_float(type) || k->scalar_type() != type || wq->scalar_type() != type ||
        wk->scalar_type() != type || table->scalar_type() != type || pos->dim() != 1 ||
        !is_index(pos->scalar_type()) || q->dim() != 2 || k->dim() != 2 || table->dim() != 2 ||
        wq->dim() != 1 || wk->dim() != 1 || wq->size(0) != D || wk->size(0) != D)
        return later();
    const int64_t T = pos->size(0);
    if (T == 0 || q->size(0) != T || k->size(0) != T || q->stride(1) != 1 || k->stride(1) != 1 ||
        q->size(1) == 0 || k->size(1) == 0 || q->size(1) % D != 0 || k->size(1) % D != 0)
        return later();
    const int64_t kvh = k->size(1) / D;
    tlb_qk_norm_rope_args p{};
    Tensor k_out;
    if (kc == nullptr) {
        if (a[7] != Py_None) return later();
        k_out = dense(*k, k->sizes(), type);
        p.key_out = k_out.data_ptr();
        p.slot_dtype = TLB_INT64;
        p.cache_dtype = code_of(type);
    } else {
        if (ks != nullptr) {
            if (!quantized_caches(at, kc, vc, ks, vs)) return later();
            p.key_scales = ks->data_ptr();
            p.value_scales = vs->data_ptr();
        } else if (a[13] != Py_None || a[14] != Py_None || !at.has(kc) || !at.has(vc) ||
                   kc->dim() != 4 || vc->sizes() != kc->sizes() || kc->scalar_type() != type ||
                   vc->scalar_type() != type || kc->numel() == 0) {
            return later();
        }
        if (kc->size(1) != kvh || kc->size(3) != D || !token_rows(at, v, T, kvh, D) ||
            v->scalar_type() != type)
            return later();
        if (slots != nullptr) {
            if (!at.has(slots) || slots->dim() != 1 || slots->size(0) != T ||
                !is_index(slots->scalar_type()))
                return later();
            p.slots = slots->data_ptr();
            p.slot_dtype = code_of(slots->scalar_type());
        } else {
            if (a[9] != Py_None || !at.has(bt) || bt->dim() != 2 || bt->size(0) < T ||
                bt->size(1) == 0 || bt->scalar_type() != ScalarType::Int)
                return later();
            p.block_tables = static_cast<const int32_t*>(bt->data_ptr());
            p.max_blocks_per_seq = bt->size(1);
            p.slot_dtype = TLB_INT64;
        }
        p.value = v->data_ptr();
        p.value_stride = v->stride(0);
        p.key_cache = kc->data_ptr();
        p.value_cache = vc->data_ptr();
        p.num_blocks = kc->size(0);
        p.block_size = kc->size(2);
        p.cache_dtype = code_of(kc->scalar_type());
    }
    Tensor q_out = dense(*q, q->sizes(), type);
    p.query_out = q_out.data_ptr();
    p.positions = pos->data_ptr();
    p.query = q->data_ptr();
    p.key = k->data_ptr();
    p.query_weight = wq->data_ptr();
    p.key_weight = wk->data_ptr();
    p.cos_sin_cache = table->data_ptr();
    p.pos_dtype = code_of(pos->scalar_type());
    p.num_tokens = T;
    p.num_heads = q->size(1) / D;
    p.num_kv_heads = kvh;
    p.head_size = D;
    p.cache_rows = table->size(0);
    p.rot_dim = table->size(1);
    p.query_stride = q->stride(0);
    p.key_stride = k->stride(0);
    p.dtype = code_of(type);
    p.flags = overlap ? TLB_ROPE_OVERLAP_PREVIOUS : 0;
    p.eps = eps;
    if (g_norm(&p, at.stream) != TLB_OK) return later();
    PyObject* po = THPVariable_Wrap(std::move(q_out));
    if (kc != nullptr || po == nullptr) return po;
    PyObject* pk = THPVariable_Wrap(std::move(k_out));
    PyObject* both = pk ? PyTuple_Pack(2, po, pk) : nullptr;
    Py_DECREF(po);
    Py_XDECREF(pk);
    return both;
    END_HANDLE_TH_ERRORS
}

// [T, K] on this device, each row contiguous.
bool rows_of(const Place& at, const Tensor* x) {
    return x != nullptr && x->is_cuda() && x->get_device() == at.device && x->dim() == 2 &&
           x->size(1) > 0 && (x->stride(1) == 1 || x->size(1) == 1);
}
int64_t groups_of(int64_t width) { return (width + 127) / 128; }

// rows(x, op, weight, eps, residual, residual_out): (values, scales), and what the norm
// returns as its third: residual_out, a new one, or None
PyObject* rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6 || g_rows == nullptr) return later();
    const Tensor *x = tensor(a[0]), *w = tensor(a[2]), *res = tensor(a[4]), *out = tensor(a[5]);
    int64_t op;
    double eps;
    if (x == nullptr || !whole(a[1], &op) || !number(a[3], &eps)) return later();
    const Place at(*x);
    const ScalarType type = x->scalar_type();
    if (!at.ok() || !rows_of(at, x) || !is_float(type) || x->size(0) == 0) return later();
    const int64_t T = x->size(0), K = op == TLB_ROWS_SILU_AND_MUL ? x->size(1) / 2 : x->size(1);
    tlb_quantize_rows_args p{};
    Tensor h;
    if (op == TLB_ROWS_RMS_NORM) {
        if (!at.has(w) || w->dim() != 1 || w->size(0) != K || w->scalar_type() != type ||
            !(eps >= 0))
            return later();
        p.weight = w->data_ptr();
        if (res != nullptr) {
            if (!rows_of(at, res) || res->sizes() != x->sizes() || res->scalar_type() != type)
                return later();
            if (out != nullptr) {
                if (!rows_of(at, out) || out->sizes() != x->sizes() ||
                    out->scalar_type() != type || (T > 1 && out->stride(0) < K))
                    return later();
                h = *out;
            } else {
                if (a[5] != Py_None) return later();
                h = dense(*x, x->sizes(), type);
            }
            p.residual = res->data_ptr();
            p.residual_stride = res->stride(0);
            p.residual_out = h.data_ptr();
            p.residual_out_stride = h.stride(0);
        } else if (a[4] != Py_None || a[5] != Py_None) {
            return later();
        }
    } else if (op == TLB_ROWS_SILU_AND_MUL && x->size(1) != 2 * K) {
        return later();
    }
    Tensor q = dense(*x, {T, K}, ScalarType::Float8_e4m3fn),
           s = dense(*x, {T, groups_of(K)}, ScalarType::Float8_e8m0fnu);
    p.out = q.data_ptr();
    p.scales = s.data_ptr();
    p.x = x->data_ptr();
    p.op = op;
    p.num_rows = T;
    p.width = K;
    p.x_stride = x->stride(0);
    p.dtype = code_of(type);
    p.eps = eps;
    if (g_rows(&p, at.stream) != TLB_OK) return later();
    PyObject *pq = THPVariable_Wrap(std::move(q)), *ps = THPVariable_Wrap(std::move(s));
    PyObject* all = nullptr;
    if (op != TLB_ROWS_RMS_NORM) {
        if (pq && ps) all = PyTuple_Pack(2, pq, ps);
    } else if (res == nullptr || out != nullptr) {
        if (pq && ps) all = PyTuple_Pack(3, pq, ps, res == nullptr ? Py_None : a[5]);
    } else {
        PyObject* ph = THPVariable_Wrap(std::move(h));
        if (pq && ps && ph) all = PyTuple_Pack(3, pq, ps, ph);
        Py_XDECREF(ph);
    }
    Py_XDECREF(pq);
    Py_XDECREF(ps);
    return all;
    END_HANDLE_TH_ERRORS
}

// product(x, x_scales, weight, weight_scales, out_dtype, bias)
PyObject* product(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6 || g_product == nullptr) return later();
    const Tensor *x = tensor(a[0]), *xs = tensor(a[1]), *w = tensor(a[2]), *ws = tensor(a[3]),
                 *bias = tensor(a[5]);
    if (x == nullptr || !THPDtype_Check(a[4])) return later();
    const ScalarType type = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
    const Place at(*x);
    if (!at.ok() || !is_float(type) || !rows_of(at, x) || !rows_of(at, w) || !rows_of(at, xs) ||
        !rows_of(at, ws) || x->scalar_type() != ScalarType::Float8_e4m3fn ||
        w->scalar_type() != ScalarType::Float8_e4m3fn ||
        xs->scalar_type() != ScalarType::Float8_e8m0fnu ||
        ws->scalar_type() != ScalarType::Float8_e8m0fnu)
        return later();
    const int64_t T = x->size(0), K = x->size(1), N = w->size(0), G = groups_of(K);
    if (T == 0 || N == 0 || w->size(1) != K || xs->size(0) != T || xs->size(1) != G ||
        ws->size(0) != groups_of(N) || ws->size(1) != G)
        return later();
    if (bias != nullptr ? !at.has(bias) || bias->dim() != 1 || bias->size(0) != N ||
                              bias->scalar_type() != type
                        : a[5] != Py_None)
        return later();
    Tensor out = dense(*x, {T, N}, type);
    tlb_matmul_quantized_args p{};
    p.out = out.data_ptr();
    p.x = x->data_ptr();
    p.x_scales = xs->data_ptr();
    p.weight = w->data_ptr();
    p.weight_scales = ws->data_ptr();
    p.bias = bias ? bias->data_ptr() : nullptr;
    p.num_tokens = T;
    p.width = K;
    p.features = N;
    p.x_stride = x->stride(0);
    p.x_scales_stride = xs->stride(0);
    p.weight_stride = w->stride(0);
    p.weight_scales_stride = ws->stride(0);
    p.out_stride = N;
    p.out_dtype = code_of(type);
    if (g_product(&p, at.stream) != TLB_OK) return later();
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// bind(attention, write, read, norm, rows, product): addresses of the library's entry
// points
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    void* p[6] = {};
    for (Py_ssize_t i = 0; i < 6 && i < n; ++i) p[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) return nullptr;
    g_attention = reinterpret_cast<decltype(g_attention)>(p[0]);
    g_write = reinterpret_cast<decltype(g_write)>(p[1]);
    g_read = reinterpret_cast<decltype(g_read)>(p[2]);
    g_norm = reinterpret_cast<decltype(g_norm)>(p[3]);
    g_rows = reinterpret_cast<decltype(g_rows)>(p[4]);
    g_product = reinterpret_cast<decltype(g_product)>(p[5]);
    Py_RETURN_NONE;
}

// scratch(device, stream, address, bytes): the attention scratch of a stream from
// now on; address 0 forgets every stream's of the device
PyObject* scratch(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 4) {
        PyErr_SetString(PyExc_TypeError, "scratch takes four arguments");
        return nullptr;
    }
    const int device = (int)PyLong_AsLong(a[0]);
    void *stream = PyLong_AsVoidPtr(a[1]), *ptr = PyLong_AsVoidPtr(a[2]);
    const int64_t bytes = PyLong_AsLongLong(a[3]);
    if (PyErr_Occurred()) return nullptr;
    std::vector<Scratch> kept;
    for (const Scratch& s : g_scratch)
        if (s.device != device || (ptr != nullptr && s.stream != stream)) kept.push_back(s);
    if (ptr != nullptr) kept.push_back({device, stream, ptr, bytes});
    g_scratch.swap(kept);
    Py_RETURN_NONE;
}

#define TLB_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), \
                       METH_FASTCALL, nullptr}
PyMethodDef methods[] = {TLB_METHOD(attention), TLB_METHOD(write), TLB_METHOD(read),
                         TLB_METHOD(norm),      TLB_METHOD(rows),  TLB_METHOD(product),
                         TLB_METHOD(bind),      TLB_METHOD(scratch),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

// torch_version: the torch whose headers (and so tensor layout) this was built with
PyMODINIT_FUNC PyInit__fast(void) {
    PyObject* m = PyModule_Create(&module);
    if (m != nullptr && PyModule_AddStringConstant(m, "torch_version", TLB_TORCH_VERSION) != 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
