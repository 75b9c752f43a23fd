// paged_host.cpp -- the host side of the paged cache's operators (transformers/paged_kv.py): checks, outputs, scratch, stream and launch of the
// plain call in one native call (in Python 25 to 35 us around kernels of 3 to 20).  Each function returns None when a call is not the plain
// case: the Python statements then serve or refuse it.
#include <cmath>
#include "host_common.h"
#include "paged_host.h"

namespace {

using StepFn = int (*)(const int32_t*, const int32_t*, int, int32_t*, int64_t, int, const int32_t*, int, const int32_t*, int32_t*, int, int64_t, int32_t*, int32_t*, int64_t*,
                       int64_t*, int32_t*, void*);
using AppendFn = int (*)(void*, int, int64_t, int64_t, int, int, int, int, const void*, const void*, int, int64_t, int64_t, const int64_t*, const int64_t*, void*, const int64_t*,
                         void*, const int64_t*, int, int, int, void*);
using SizeFn = size_t (*)(int64_t, int, int, int, int, int64_t);
using PagedFn = int (*)(const void*, int, const int64_t*, int64_t, const void*, const int64_t*, const void*, const int64_t*, int, int, int, const int32_t*, int64_t, int,
                        const int32_t*, const int32_t*, int, int, int, int, float, int64_t, void*, const int64_t*, void*, size_t, void*);
using PackedFn = int (*)(const void*, int, const int64_t*, int64_t, const void*, const int64_t*, const void*, const int64_t*, const int32_t*, int, int, int, int, float, int,
                         int64_t, void*, const int64_t*, void*, size_t, void*);
StepFn g_step = nullptr;
AppendFn g_append = nullptr;
SizeFn g_paged_size = nullptr, g_packed_size = nullptr;
PagedFn g_paged = nullptr;
PackedFn g_packed = nullptr;

}  // namespace

PyObject* attach_paged(PyObject*, PyObject* args) {
    unsigned long long s, a, ps, p, ks, k;
    if (!PyArg_ParseTuple(args, "KKKKKK", &s, &a, &ps, &p, &ks, &k)) return nullptr;
    g_step = reinterpret_cast<StepFn>(s);
    g_append = reinterpret_cast<AppendFn>(a);
    g_paged_size = reinterpret_cast<SizeFn>(ps);
    g_paged = reinterpret_cast<PagedFn>(p);
    g_packed_size = reinterpret_cast<SizeFn>(ks);
    g_packed = reinterpret_cast<PackedFn>(k);
    Py_RETURN_NONE;
}

// paged_step(query_lens, context_lens, block_table, free_pages, free_count, page_size, n_tokens, free_left | None) -> the six tensors of a PagedStep
PyObject* paged_step(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 8 || !g_step) Py_RETURN_NONE;
    const at::Tensor *fresh = plain(a[0]), *held = plain(a[1]), *table = plain(a[2]), *pages = plain(a[3]), *count = plain(a[4]), *left = a[7] == Py_None ? nullptr : plain(a[7]);
    int64_t page, tokens;
    if (!fresh || fresh->dim() != 1 || !integer(a[5], &page) || !integer(a[6], &tokens) || page <= 0 || page > 0x7fffffff || tokens < 0) Py_RETURN_NONE;
    const int64_t R = fresh->size(0);
    if (R <= 0 || !ints(fresh, R, at::kInt, *fresh) || !ints(held, R, at::kInt, *fresh) || !table_ok(table, *fresh) || table->size(0) != R || !pages || pages->dim() != 1 ||
        !ints(pages, pages->size(0), at::kInt, *fresh) || pages->size(0) <= 0 || pages->size(0) > 0x7fffffff || !ints(count, 1, at::kInt, *fresh) ||
        (a[7] != Py_None && !ints(left, 1, at::kInt, *fresh)))
        Py_RETURN_NONE;
    at::Tensor out[6];
    int rc;
    {
        const WithoutGil released;
        const c10::cuda::CUDAGuard guard(fresh->device());
        const auto options = fresh->options();
        const at::Tensor small = at::empty({2 * R + 3}, options), wide = at::empty({2 * tokens}, options.dtype(at::kLong));
        out[0] = piece(small, 0, R + 1);
        out[1] = piece(small, R + 1, R);
        out[2] = piece(wide, 0, tokens);
        out[3] = piece(wide, tokens, tokens);
        out[4] = left ? *left : piece(small, 2 * R + 1, 1);
        out[5] = piece(small, 2 * R + 2, 1);
        int32_t* const s = small.mutable_data_ptr<int32_t>();
        int64_t* const w = tokens ? wide.mutable_data_ptr<int64_t>() : nullptr;
        rc = g_step(fresh->const_data_ptr<int32_t>(), held->const_data_ptr<int32_t>(), (int)R, table->mutable_data_ptr<int32_t>(), table->stride(0), (int)table->size(1),
                    pages->const_data_ptr<int32_t>(), (int)pages->size(0), count->const_data_ptr<int32_t>(), out[4].mutable_data_ptr<int32_t>(), (int)page, tokens, s, s + R + 1, w,
                    w ? w + tokens : nullptr, s + 2 * R + 2, stream_of(*fresh));
    }
    if (rc) return PyLong_FromLong(rc);
    PyObject* const r = PyTuple_New(6);
    if (!r) return nullptr;
    for (int i = 0; i < 6; i++) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(std::move(out[i])));
    return r;
    END_HANDLE_TH_ERRORS
}

// paged_append(qkv, heads, kv heads, head_dim, cos | None, sin, positions, slots, k_cache, v_cache) -> True
PyObject* paged_append(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 10 || !g_append) Py_RETURN_NONE;
    const at::Tensor *x = plain(a[0]), *slots = plain(a[7]), *k = plain(a[8]), *v = plain(a[9]);
    int64_t Hq, Hkv, D;
    if (!x || !integer(a[1], &Hq) || !integer(a[2], &Hkv) || !integer(a[3], &D) || x->dim() != 2 || half_code(*x) < 0 || wants_grad(*x) || Hq < 0 || Hkv <= 0 || D <= 0 ||
        Hq > 65536 || Hkv > 65536 || D > 65536)
        Py_RETURN_NONE;
    const int64_t T = x->size(0);
    if (T <= 0 || x->size(1) != (Hq + 2 * Hkv) * D || x->stride(1) != 1 || (T > 1 && x->stride(0) < x->size(1)) || !ints(slots, T, at::kLong, *x) || !caches_ok(k, v, *x, D) ||
        k->size(2) != Hkv || wants_grad(*k) || wants_grad(*v))
        Py_RETURN_NONE;
    const at::Tensor *cos = nullptr, *sin = nullptr, *pos = nullptr;
    int64_t R = 0;
    int table = 0;
    if (a[4] != Py_None) {
        cos = plain(a[4]), sin = plain(a[5]), pos = plain(a[6]);
        if (!cos || !sin || !ints(pos, T, at::kLong, *x) || cos->dim() != 2 || sin->sizes() != cos->sizes() || sin->strides() != cos->strides() || cos->stride(1) != 1 ||
            cos->size(0) <= 0 || cos->scalar_type() != sin->scalar_type() || cos->device() != x->device() || sin->device() != x->device() || wants_grad(*cos) ||
            wants_grad(*sin))
            Py_RETURN_NONE;
        table = cos->scalar_type() == at::kFloat ? 0 : half_code(*cos);
        R = cos->size(1);
        if (table < 0 || R <= 0 || R > D || R % 2) Py_RETURN_NONE;
    } else if (a[5] != Py_None) Py_RETURN_NONE;
    int rc;
    {
        const WithoutGil released;
        const c10::cuda::CUDAGuard guard(x->device());
        const int64_t ks[3] = {k->stride(0), k->stride(1), k->stride(2)}, vs[3] = {v->stride(0), v->stride(1), v->stride(2)};
        const int dt = half_code(*x);
        rc = g_append(x->mutable_data_ptr(), dt, T > 1 ? x->stride(0) : x->size(1), T, (int)Hq, (int)Hkv, (int)D, (int)R, cos ? cos->const_data_ptr() : nullptr,
                      sin ? sin->const_data_ptr() : nullptr, table, cos ? cos->stride(0) : 0, cos ? cos->size(0) : 0, pos ? pos->const_data_ptr<int64_t>() : nullptr,
                      slots->const_data_ptr<int64_t>(), k->mutable_data_ptr(), ks, v->mutable_data_ptr(), vs, k->scalar_type() == at::kByte ? kE5m2 : dt, (int)k->size(0),
                      (int)k->size(1), stream_of(*x));
    }
    if (rc) return PyLong_FromLong(rc);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

namespace {
// what both attentions ask of their queries; *scale: 1 / sqrt(D) for None
bool queries_ok(const at::Tensor* q, int64_t Hkv, PyObject* scale_in, PyObject* most_in, float* scale, int64_t* most) {
    if (!q || q->dim() != 3 || half_code(*q) < 0 || wants_grad(*q) || q->numel() == 0 || !aligned(*q)) return false;
    const int64_t D = q->size(2);
    if (Hkv <= 0 || q->size(1) % Hkv || D % 16 || D > 256) return false;
    if (scale_in == Py_None) *scale = (float)(1.0 / std::sqrt((double)D));
    else if (PyFloat_CheckExact(scale_in)) *scale = (float)PyFloat_AS_DOUBLE(scale_in);
    else return false;
    if (most_in == Py_None) *most = q->size(0);
    else if (!integer(most_in, most)) return false;
    return *scale > 0.0f && *most >= 0;
}
}  // namespace

// sdp_paged(query, k_cache, v_cache, block_table, seq_lens, cu_seqlens, scale | None, max_query_len | None) -> the result
PyObject* sdp_paged(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 8 || !g_paged) Py_RETURN_NONE;
    const at::Tensor *q = plain(a[0]), *k = plain(a[1]), *v = plain(a[2]), *table = plain(a[3]), *lens = plain(a[4]), *cu = plain(a[5]);
    float scale;
    int64_t most;
    if (!q || q->dim() != 3 || !caches_ok(k, v, *q, q->size(2)) || wants_grad(*k) || wants_grad(*v) || !aligned(*k) || !aligned(*v) || !queries_ok(q, k->size(2), a[6], a[7], &scale, &most) || !table_ok(table, *q))
        Py_RETURN_NONE;
    const int64_t R = table->size(0), T = q->size(0), H = q->size(1), D = q->size(2);
    if (!ints(lens, R, at::kInt, *q) || !ints(cu, R + 1, at::kInt, *q) || table->size(1) * k->size(1) >= (int64_t)1 << 31) Py_RETURN_NONE;
    at::Tensor out;
    int rc;
    {
        const WithoutGil released;
        const c10::cuda::CUDAGuard guard(q->device());
        const auto options = q->options().requires_grad(false);
        out = at::empty({T, H, D}, options);
        const size_t need = g_paged_size(T, (int)R, (int)H, (int)k->size(2), (int)D, most);
        const at::Tensor scratch = at::empty({(int64_t)need}, options.dtype(at::kByte));
        const int64_t qs[2] = {q->stride(0), q->stride(1)}, os[2] = {H * D, D}, ks[3] = {k->stride(0), k->stride(1), k->stride(2)},
                      vs[3] = {v->stride(0), v->stride(1), v->stride(2)};
        const int dt = half_code(*q);
        rc = g_paged(q->const_data_ptr(), dt, qs, T, k->const_data_ptr(), ks, v->const_data_ptr(), vs, k->scalar_type() == at::kByte ? kE5m2 : dt, (int)k->size(0), (int)k->size(1),
                     table->const_data_ptr<int32_t>(), table->stride(0), (int)table->size(1), lens->const_data_ptr<int32_t>(), cu->const_data_ptr<int32_t>(), (int)R, (int)H,
                     (int)k->size(2), (int)D, scale, most, out.mutable_data_ptr(), os, scratch.mutable_data_ptr(), need, stream_of(*q));
    }
    if (rc) return PyLong_FromLong(rc);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// sdp_packed(query, key, value, cu_seqlens, scale | None, is_causal, max_seqlen | None) -> the result
PyObject* sdp_packed(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 7 || !g_packed || !PyBool_Check(a[5])) Py_RETURN_NONE;
    const at::Tensor *q = plain(a[0]), *k = plain(a[1]), *v = plain(a[2]), *cu = plain(a[3]);
    float scale;
    int64_t most;
    if (!q || !k || !v || q->dim() != 3 || k->dim() != 3 || v->sizes() != k->sizes() || k->size(0) != q->size(0) || k->size(2) != q->size(2) ||
        k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type() || k->device() != q->device() || v->device() != q->device() || k->numel() == 0 ||
        wants_grad(*k) || wants_grad(*v) || !aligned(*k) || !aligned(*v) || !queries_ok(q, k->size(1), a[4], a[6], &scale, &most) || !cu || cu->dim() != 1 || cu->size(0) < 2 ||
        cu->size(0) > 0x7fffffff || !ints(cu, cu->size(0), at::kInt, *q))
        Py_RETURN_NONE;
    const int64_t R = cu->size(0) - 1, T = q->size(0), H = q->size(1), D = q->size(2);
    at::Tensor out;
    int rc;
    {
        const WithoutGil released;
        const c10::cuda::CUDAGuard guard(q->device());
        const auto options = q->options().requires_grad(false);
        out = at::empty({T, H, D}, options);
        const size_t need = g_packed_size(T, (int)R, (int)H, (int)k->size(1), (int)D, most);
        const at::Tensor scratch = at::empty({(int64_t)need}, options.dtype(at::kByte));
        const int64_t qs[2] = {q->stride(0), q->stride(1)}, ks[2] = {k->stride(0), k->stride(1)}, vs[2] = {v->stride(0), v->stride(1)}, os[2] = {H * D, D};
        rc = g_packed(q->const_data_ptr(), half_code(*q), qs, T, k->const_data_ptr(), ks, v->const_data_ptr(), vs, cu->const_data_ptr<int32_t>(), (int)R, (int)H, (int)k->size(1),
                      (int)D, scale, a[5] == Py_True, most, out.mutable_data_ptr(), os, scratch.mutable_data_ptr(), need, stream_of(*q));
    }
    if (rc) return PyLong_FromLong(rc);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}
