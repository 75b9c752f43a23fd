// step_host.cpp -- the host side of what a server's step has beside its attention (transformers/paged_kv.py, lora.py, logprobs.py): checks, outputs,
// scratch, stream and launch of the plain call in one native call (in Python 25 to 35 us around kernels of 3 to 20, 110 for the copies of 16 caches).  Each
// function returns None when a call is not the plain case: the Python statements then serve or refuse it; an int: the native error code.
#include <cmath>
#include <vector>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include "host_common.h"
#include "paged_host.h"

namespace {

using NormFn = int (*)(void*, int, int64_t, int64_t, int, int, int, int, const void*, const void*, int, float, const void*, const void*, int, int64_t, int64_t, const int64_t*,
                       const int64_t*, void*, const int64_t*, void*, const int64_t*, int, int, int, void*);
using ForkFn = int (*)(const int32_t*, const int32_t*, int, int32_t*, int32_t*, int64_t, int, int, const int32_t*, int, const int32_t*, int32_t*, int32_t*, int, int32_t*, int32_t*,
                       int32_t*, void*);
using ReleaseSizeFn = size_t (*)(int, int, int);
using ReleaseFn = int (*)(const uint8_t*, const int32_t*, int, int, int32_t*, int64_t, int, int32_t*, int, int32_t*, int32_t*, void*, size_t, void*);
using CompactSizeFn = size_t (*)(int);
using CompactFn = int (*)(const int32_t*, int64_t, int, int, const int32_t*, int, const int32_t*, const int32_t*, int32_t*, int32_t*, int32_t*, int32_t*, int32_t*, int32_t*, void*,
                          size_t, void*);
using CopyFn = int (*)(const int32_t*, const int32_t*, int, void* const*, int, int, int64_t, int64_t, void*);
using LoraSizeFn = size_t (*)(int64_t, int, int64_t, int, int, int, int);
using LoraFn = int (*)(const void*, int64_t, int, int64_t, int, const void*, int64_t, const void*, int64_t, int, const float*, int, const int32_t*, const int32_t*, int, const int*, int,
                       void*, int64_t, void*, size_t, void*);
using LogprobsFn = int (*)(const void*, int, int64_t, int64_t, int64_t, const int64_t*, float, int, float*, float*, int64_t*, float*, float*, void*);
using LogprobsGradFn = int (*)(const void*, int, int64_t, int64_t, int64_t, const int64_t*, float, int, const int64_t*, const float*, const float*, const float*, const float*, void*, int64_t,
                               void*);
NormFn g_norm = nullptr;
ForkFn g_fork = nullptr;
ReleaseSizeFn g_release_size = nullptr;
ReleaseFn g_release = nullptr;
CompactSizeFn g_compact_size = nullptr;
CompactFn g_compact = nullptr;
CopyFn g_copy = nullptr;
LoraSizeFn g_lora_size = nullptr;
LoraFn g_lora = nullptr;
LogprobsFn g_logprobs = nullptr;
LogprobsGradFn g_logprobs_grad = nullptr;

int float_code(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? 0 : half_code(t); }
bool number(PyObject* o, double* out) {
    if (!PyFloat_CheckExact(o)) return false;
    *out = PyFloat_AS_DOUBLE(o);
    return true;
}
// the stack and its count
bool stack_ok(const at::Tensor* pages, const at::Tensor* count, const at::Tensor& like) {
    return pages && pages->dim() == 1 && pages->size(0) > 0 && pages->size(0) <= 0x7fffffff && ints(pages, pages->size(0), at::kInt, like) && ints(count, 1, at::kInt, like);
}
// rows of a matrix contiguous, apart and on 16 bytes
bool rows_ok(const at::Tensor& t) { return aligned(t) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)); }
// whether matrices of as many rows share memory: columns of one buffer side by side do not
bool overlap(const at::Tensor& a, const at::Tensor& b) {
    const int64_t rows = a.size(0), size = (int64_t)a.element_size(), wide_a = a.size(1) * size, wide_b = b.size(1) * size, step = rows > 1 ? a.stride(0) * size : 0;
    const int64_t pa = (int64_t)reinterpret_cast<uintptr_t>(a.const_data_ptr()), pb = (int64_t)reinterpret_cast<uintptr_t>(b.const_data_ptr());
    if (pa + (rows - 1) * step + wide_a <= pb || pb + (rows > 1 ? (rows - 1) * b.stride(0) * size : 0) + wide_b <= pa) return false;
    if (rows <= 1 || a.stride(0) != b.stride(0)) return true;
    const int64_t behind = ((pb - pa) % step + step) % step;
    return behind < wide_a || behind + wide_b > step;
}
// autograd hears of what a kernel writes over (a tensor of inference mode keeps no count)
void written(const at::Tensor& t) { if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version(); }
// a stack of adapters, each in one run on 16 bytes
bool adapters_ok(const at::Tensor& t, int64_t each) {
    int64_t run = 1;
    for (int64_t d = t.dim() - 1; d > 0; run *= t.size(d), d--)
        if (t.size(d) != 1 && t.stride(d) != run) return false;
    return !(reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) && (t.size(0) == 1 || (t.stride(0) >= each && t.stride(0) % 8 == 0));
}

}  // namespace

PyObject* attach_step(PyObject*, PyObject* args) {
    unsigned long long f[11];
    if (!PyArg_ParseTuple(args, "KKKKKKKKKKK", f, f + 1, f + 2, f + 3, f + 4, f + 5, f + 6, f + 7, f + 8, f + 9, f + 10)) return nullptr;
    g_norm = reinterpret_cast<NormFn>(f[0]);
    g_fork = reinterpret_cast<ForkFn>(f[1]);
    g_release_size = reinterpret_cast<ReleaseSizeFn>(f[2]);
    g_release = reinterpret_cast<ReleaseFn>(f[3]);
    g_compact_size = reinterpret_cast<CompactSizeFn>(f[4]);
    g_compact = reinterpret_cast<CompactFn>(f[5]);
    g_copy = reinterpret_cast<CopyFn>(f[6]);
    g_lora_size = reinterpret_cast<LoraSizeFn>(f[7]);
    g_lora = reinterpret_cast<LoraFn>(f[8]);
    g_logprobs = reinterpret_cast<LogprobsFn>(f[9]);
    g_logprobs_grad = reinterpret_cast<LogprobsGradFn>(f[10]);
    Py_RETURN_NONE;
}

// paged_norm_append(qkv, heads, kv heads, head_dim, q_weight, k_weight, eps, cos | None, sin, positions, slots, k_cache | None, v_cache) -> True
PyObject* paged_norm_append(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 13 || !g_norm) Py_RETURN_NONE;
    const at::Tensor *x = plain(a[0]), *qw = plain(a[4]), *kw = plain(a[5]);
    int64_t Hq, Hkv, D;
    double eps;
    if (!x || !integer(a[1], &Hq) || !integer(a[2], &Hkv) || !integer(a[3], &D) || !number(a[6], &eps) || x->dim() != 2 || half_code(*x) < 0 || wants_grad(*x) || Hq < 0 || Hkv <= 0 ||
        D <= 0 || Hq > 65536 || Hkv > 65536 || D > 65536 || !(eps >= 0.0) || !(eps < INFINITY) || !qw || !kw)
        Py_RETURN_NONE;
    for (const at::Tensor* w : {qw, kw})
        if (w->dim() != 1 || w->size(0) != D || !w->is_contiguous() || w->device() != x->device() || float_code(*w) < 0 || w->scalar_type() != qw->scalar_type() || wants_grad(*w))
            Py_RETURN_NONE;
    const int64_t T = x->size(0);
    if (T <= 0 || x->size(1) != (Hq + 2 * Hkv) * D || x->stride(1) != 1 || (T > 1 && x->stride(0) < x->size(1))) Py_RETURN_NONE;
    const at::Tensor *slots = nullptr, *k = nullptr, *v = nullptr;
    if (a[11] != Py_None) {
        slots = plain(a[10]), k = plain(a[11]), v = plain(a[12]);
        if (!ints(slots, T, at::kLong, *x) || !caches_ok(k, v, *x, D) || k->size(2) != Hkv || wants_grad(*k) || wants_grad(*v)) Py_RETURN_NONE;
    } else if (a[12] != Py_None) Py_RETURN_NONE;
    const at::Tensor *cos = nullptr, *sin = nullptr, *pos = nullptr;
    int64_t R = 0;
    int table = 0;
    if (a[7] != Py_None) {
        cos = plain(a[7]), sin = plain(a[8]), pos = plain(a[9]);
        if (!cos || !sin || !ints(pos, T, at::kLong, *x) || cos->dim() != 2 || sin->sizes() != cos->sizes() || sin->strides() != cos->strides() || cos->stride(1) != 1 ||
            cos->size(0) <= 0 || cos->scalar_type() != sin->scalar_type() || cos->device() != x->device() || sin->device() != x->device() || wants_grad(*cos) || wants_grad(*sin))
            Py_RETURN_NONE;
        table = float_code(*cos);
        R = cos->size(1);
        if (table < 0 || R <= 0 || R > D || R % 2) Py_RETURN_NONE;
    } else if (a[8] != Py_None) Py_RETURN_NONE;
    int rc;
    {
        const WithoutGil released;
        const c10::cuda::CUDAGuard guard(x->device());
        int64_t ks[3] = {}, vs[3] = {};
        for (int d = 0; k && d < 3; d++) ks[d] = k->stride(d), vs[d] = v->stride(d);
        const int dt = half_code(*x);
        rc = g_norm(x->mutable_data_ptr(), dt, T > 1 ? x->stride(0) : x->size(1), T, (int)Hq, (int)Hkv, (int)D, (int)R, qw->const_data_ptr(), kw->const_data_ptr(), float_code(*qw),
                    (float)eps, cos ? cos->const_data_ptr() : nullptr, sin ? sin->const_data_ptr() : nullptr, table, cos ? cos->stride(0) : 0, cos ? cos->size(0) : 0,
                    pos ? pos->const_data_ptr<int64_t>() : nullptr, slots ? slots->const_data_ptr<int64_t>() : nullptr, k ? k->mutable_data_ptr() : nullptr, ks,
                    v ? v->mutable_data_ptr() : nullptr, vs, k && k->scalar_type() == at::kByte ? kE5m2 : dt, k ? (int)k->size(0) : 0, k ? (int)k->size(1) : 0, stream_of(*x));
    }
    if (rc) return PyLong_FromLong(rc);
    written(*x);
    if (k) {
        written(*k);
        written(*v);
    }
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// paged_fork(parents, children, context_lens, block_table, free_pages, free_count, shared, page_size, free_left | None) -> the four tensors of a PagedFork
PyObject* paged_fork(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 9 || !g_fork) Py_RETURN_NONE;
    const at::Tensor *par = plain(a[0]), *ch = plain(a[1]), *lens = plain(a[2]), *table = plain(a[3]), *pages = plain(a[4]), *count = plain(a[5]), *shared = plain(a[6]),
                     *left = a[8] == Py_None ? nullptr : plain(a[8]);
    int64_t page;
    if (!par || par->dim() != 1 || !integer(a[7], &page) || page <= 0 || page > 0x7fffffff) Py_RETURN_NONE;
    const int64_t F = par->size(0);
    if (F <= 0 || F > 0x7fffffff || !ints(par, F, at::kInt, *par) || !ints(ch, F, at::kInt, *par) || !table_ok(table, *par) || !ints(lens, table->size(0), at::kInt, *par) ||
        !stack_ok(pages, count, *par) || !ints(shared, pages->size(0), at::kInt, *par) || (a[8] != Py_None && !ints(left, 1, at::kInt, *par)))
        Py_RETURN_NONE;
    at::Tensor out[4];
    int rc;
    {
        const WithoutGil released;
        const c10::cuda::CUDAGuard guard(par->device());
        const at::Tensor all = at::empty({2 * F + 2}, par->options());
        out[0] = piece(all, 0, F);
        out[1] = piece(all, F, F);
        out[2] = left ? *left : piece(all, 2 * F, 1);
        out[3] = piece(all, 2 * F + 1, 1);
        int32_t* const o = all.mutable_data_ptr<int32_t>();
        rc = g_fork(par->const_data_ptr<int32_t>(), ch->const_data_ptr<int32_t>(), (int)F, lens->mutable_data_ptr<int32_t>(), table->mutable_data_ptr<int32_t>(), table->stride(0),
                    (int)table->size(0), (int)table->size(1), pages->const_data_ptr<int32_t>(), (int)pages->size(0), count->const_data_ptr<int32_t>(),
                    out[2].mutable_data_ptr<int32_t>(), shared->mutable_data_ptr<int32_t>(), (int)page, o, o + F, o + 2 * F + 1, stream_of(*par));
    }
    if (rc) return PyLong_FromLong(rc);
    for (const at::Tensor* t : {lens, table, shared, left})
        if (t) written(*t);
    PyObject* const r = PyTuple_New(4);
    if (!r) return nullptr;
    for (int i = 0; i < 4; i++) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(std::move(out[i])));
    return r;
    END_HANDLE_TH_ERRORS
}

// paged_share_release(done, block_table, free_pages, free_count, held | None, page_size | None, shared) -> True
PyObject* paged_share_release(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 7 || !g_release) Py_RETURN_NONE;
    const at::Tensor *done = plain(a[0]), *table = plain(a[1]), *pages = plain(a[2]), *count = plain(a[3]), *held = a[4] == Py_None ? nullptr : plain(a[4]), *shared = plain(a[6]);
    int64_t page = 1;
    if (!done || done->dim() != 1 || (done->scalar_type() != at::kBool && done->scalar_type() != at::kByte) || !done->is_contiguous() || done->size(0) <= 0 || !table_ok(table, *done) ||
        table->size(0) != done->size(0) || !stack_ok(pages, count, *done) || !ints(shared, pages->size(0), at::kInt, *done) || (a[4] == Py_None) != (a[5] == Py_None) ||
        (a[4] != Py_None && (!ints(held, done->size(0), at::kInt, *done) || !integer(a[5], &page) || page <= 0 || page > 0x7fffffff)))
        Py_RETURN_NONE;
    int rc;
    {
        const WithoutGil released;
        const c10::cuda::CUDAGuard guard(done->device());
        const size_t need = g_release_size((int)pages->size(0), (int)done->size(0), (int)table->size(1));
        const at::Tensor scratch = at::empty({(int64_t)need}, done->options().dtype(at::kByte));
        rc = g_release(static_cast<const uint8_t*>(done->const_data_ptr()), held ? held->const_data_ptr<int32_t>() : nullptr, (int)page, (int)done->size(0),
                       table->mutable_data_ptr<int32_t>(), table->stride(0), (int)table->size(1), pages->mutable_data_ptr<int32_t>(), (int)pages->size(0),
                       count->mutable_data_ptr<int32_t>(), shared->mutable_data_ptr<int32_t>(), scratch.mutable_data_ptr(), need, stream_of(*done));
    }
    if (rc) return PyLong_FromLong(rc);
    for (const at::Tensor* t : {table, pages, count, shared}) written(*t);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// paged_compact(block_table, free_pages, free_count, shared | None) -> the six of a PagedCompact
PyObject* paged_compact(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 4 || !g_compact) Py_RETURN_NONE;
    const at::Tensor *table = plain(a[0]), *pages = plain(a[1]), *count = plain(a[2]), *shared = a[3] == Py_None ? nullptr : plain(a[3]);
    if (!table || !table_ok(table, *table) || !stack_ok(pages, count, *table) || (a[3] != Py_None && !ints(shared, pages->size(0), at::kInt, *table))) Py_RETURN_NONE;
    const int64_t n = pages->size(0);
    at::Tensor out[6];
    int rc;
    {
        const WithoutGil released;
        const c10::cuda::CUDAGuard guard(table->device());
        const at::Tensor all = at::empty({4 * n + 1}, table->options());
        out[0] = at::empty({table->size(0), table->size(1)}, table->options());
        out[1] = piece(all, 0, n);
        out[2] = piece(all, 4 * n, 1);
        if (shared) out[3] = piece(all, n, n);
        out[4] = piece(all, 2 * n, n);
        out[5] = piece(all, 3 * n, n);
        const size_t need = g_compact_size((int)n);
        const at::Tensor scratch = at::empty({(int64_t)need}, table->options().dtype(at::kByte));
        int32_t* const o = all.mutable_data_ptr<int32_t>();
        rc = g_compact(table->const_data_ptr<int32_t>(), table->stride(0), (int)table->size(0), (int)table->size(1), pages->const_data_ptr<int32_t>(), (int)n,
                       count->const_data_ptr<int32_t>(), shared ? shared->const_data_ptr<int32_t>() : nullptr, out[0].mutable_data_ptr<int32_t>(), o, o + 4 * n,
                       shared ? o + n : nullptr, o + 2 * n, o + 3 * n, scratch.mutable_data_ptr(), need, stream_of(*table));
    }
    if (rc) return PyLong_FromLong(rc);
    PyObject* const r = PyTuple_New(6);
    if (!r) return nullptr;
    for (int i = 0; i < 6; i++) {
        if (i == 3 && !shared) { Py_INCREF(Py_None); PyTuple_SET_ITEM(r, i, Py_None); }
        else PyTuple_SET_ITEM(r, i, THPVariable_Wrap(std::move(out[i])));
    }
    return r;
    END_HANDLE_TH_ERRORS
}

// paged_copy(src, dst, [caches]) -> True
PyObject* paged_copy(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 3 || !g_copy || !PyList_CheckExact(a[2])) Py_RETURN_NONE;
    const at::Tensor *src = plain(a[0]), *dst = plain(a[1]);
    if (!src || src->dim() != 1 || src->size(0) <= 0 || src->size(0) > 0x7fffffff || !ints(src, src->size(0), at::kInt, *src) || !ints(dst, src->size(0), at::kInt, *src)) Py_RETURN_NONE;
    struct Group { int64_t pages, stride, bytes; std::vector<void*> at; };
    std::vector<Group> groups;
    const Py_ssize_t n = PyList_GET_SIZE(a[2]);
    for (Py_ssize_t i = 0; i < n; i++) {
        const at::Tensor* c = plain(PyList_GET_ITEM(a[2], i));
        if (!c || c->dim() < 2 || c->dim() > 6 || c->numel() == 0 || c->device() != src->device() || wants_grad(*c) || c->size(0) > 0x7fffffff) Py_RETURN_NONE;
        const int64_t page = c->numel() / c->size(0), size = (int64_t)c->element_size();
        // whether a page is one run: its dimensions in the order of their strides
        int64_t run = 1;
        for (int64_t left = page; left > 1;) {
            int64_t step = 0;
            for (int64_t d = 1; d < c->dim() && !step; d++)
                if (c->size(d) > 1 && c->stride(d) == run) step = c->size(d);
            if (!step) Py_RETURN_NONE;
            run *= step;
            left /= step;
        }
        if (run != page || (c->size(0) > 1 && c->stride(0) < page)) Py_RETURN_NONE;
        const int64_t stride = (c->stride(0) > page ? c->stride(0) : page) * size;
        Group* g = nullptr;
        for (Group& x : groups)
            if (x.pages == c->size(0) && x.stride == stride && x.bytes == page * size) { g = &x; break; }
        if (!g) {
            groups.push_back({c->size(0), stride, page * size, {}});
            g = &groups.back();
        }
        g->at.push_back(c->mutable_data_ptr());
    }
    int rc = 0;
    {
        const WithoutGil released;
        const c10::cuda::CUDAGuard guard(src->device());
        for (const Group& g : groups) {
            rc = g_copy(src->const_data_ptr<int32_t>(), dst->const_data_ptr<int32_t>(), (int)src->size(0), g.at.data(), (int)g.at.size(), (int)g.pages, g.stride, g.bytes, stream_of(*src));
            if (rc) break;
        }
    }
    for (Py_ssize_t i = 0; i < n; i++) written(*plain(PyList_GET_ITEM(a[2], i)));
    if (rc) return PyLong_FromLong(rc);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// lora_add(out, x, a, b, scales, adapter_ids, cu_seqlens, [splits] | None) -> True
PyObject* lora_add(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 8 || !g_lora) Py_RETURN_NONE;
    const at::Tensor *out = plain(a[0]), *x = plain(a[1]), *wa = plain(a[2]), *wb = plain(a[3]), *scales = plain(a[4]), *ids = plain(a[5]), *cu = plain(a[6]);
    if (!out || !x || !wa || !wb || !scales || !ids || x->dim() != 2 || out->dim() != 2 || (wa->dim() != 3 && wa->dim() != 4) || wb->dim() != 3 || half_code(*x) < 0) Py_RETURN_NONE;
    for (const at::Tensor* t : {out, wa, wb})
        if (t->scalar_type() != x->scalar_type() || t->device() != x->device()) Py_RETURN_NONE;
    for (const at::Tensor* t : {out, x, wa, wb, scales})
        if (wants_grad(*t)) Py_RETURN_NONE;
    const int64_t T = x->size(0), K = x->size(1), N = out->size(1), L = wb->size(0), R = wb->size(2), S = wa->dim() == 4 ? wa->size(1) : 1;
    constexpr int64_t most = 0x7fffff00;
    if (T <= 0 || out->size(0) != T || K <= 0 || K % 8 || K > most || N <= 0 || N > most || L <= 0 || L > most || R <= 0 || R % 8 || R > 256 || S <= 0 || S > 8 || wa->size(0) != L ||
        wa->size(wa->dim() - 2) != R || wa->size(wa->dim() - 1) != K || wb->size(1) != N || scales->scalar_type() != at::kFloat || scales->dim() != 1 || scales->size(0) != L ||
        !scales->is_contiguous() || scales->device() != x->device() || ids->dim() != 1 || ids->size(0) <= 0 || ids->size(0) > most || !ints(ids, ids->size(0), at::kInt, *x) ||
        !ints(cu, ids->size(0) + 1, at::kInt, *x) || !rows_ok(*out) || !rows_ok(*x) || !adapters_ok(*wa, S * R * K) || !adapters_ok(*wb, N * R) || overlap(*out, *x))
        Py_RETURN_NONE;
    int splits[8] = {(int)N};
    if (a[7] != Py_None) {
        if (!PyList_CheckExact(a[7]) || PyList_GET_SIZE(a[7]) != S) Py_RETURN_NONE;
        int64_t sum = 0;
        for (int64_t i = 0; i < S; i++) {
            int64_t n;
            if (!integer(PyList_GET_ITEM(a[7], i), &n) || n <= 0 || n > N || n % 8) Py_RETURN_NONE;
            splits[i] = (int)n;
            sum += n;
        }
        if (sum != N) Py_RETURN_NONE;
    } else if (S != 1 || N % 8) Py_RETURN_NONE;
    int rc;
    {
        const WithoutGil released;
        const c10::cuda::CUDAGuard guard(x->device());
        const size_t need = g_lora_size(T, (int)K, N, (int)R, (int)S, (int)L, (int)ids->size(0));
        at::Tensor scratch;
        if (need) scratch = at::empty({(int64_t)need}, x->options().dtype(at::kByte).requires_grad(false));
        rc = g_lora(x->const_data_ptr(), T > 1 ? x->stride(0) : K, half_code(*x), T, (int)K, wa->const_data_ptr(), L > 1 ? wa->stride(0) : S * R * K, wb->const_data_ptr(),
                    L > 1 ? wb->stride(0) : N * R, (int)R, scales->const_data_ptr<float>(), (int)L, ids->const_data_ptr<int32_t>(), cu->const_data_ptr<int32_t>(), (int)ids->size(0), splits,
                    (int)S, out->mutable_data_ptr(), T > 1 ? out->stride(0) : N, need ? scratch.mutable_data_ptr() : nullptr, need, stream_of(*x));
    }
    if (rc) return PyLong_FromLong(rc);
    written(*out);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

namespace {

// the gradient of token_logprobs (in Python, the engine's thread and two statements of 20 us beside kernels of 5)
struct TokenLogprobsBackward : public torch::autograd::Node {
    torch::autograd::SavedVariable logits, tokens, ids, stats;
    float temperature = 1.0f;
    int64_t k = 0;
    std::string name() const override { return "TokenLogprobsBackward"; }
    void release_variables() override { logits.reset_data(); tokens.reset_data(); ids.reset_data(); stats.reset_data(); }
    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
        at::Tensor x = logits.unpack(), t = tokens.unpack(), s = stats.unpack(), i = k ? ids.unpack() : at::Tensor();
        // a hook for saved tensors may have brought them back in another layout
        if (x.stride(1) != 1 || (x.size(0) > 1 && x.stride(0) < x.size(1))) x = x.contiguous();
        t = t.contiguous();
        s = s.contiguous();
        if (k) i = i.contiguous();
        TORCH_CHECK(x.is_cuda() && t.device() == x.device() && s.device() == x.device() && float_code(x) >= 0 && s.scalar_type() == at::kFloat && t.scalar_type() == at::kLong &&
                        (!k || (i.device() == x.device() && i.scalar_type() == at::kLong)), "what token_logprobs saved came back as something else");
        at::Tensor given[3], grad;
        const float* at[3] = {};
        for (size_t n = 0; n < grads.size() && n < 3; n++)
            if (grads[n].defined()) {
                given[n] = grads[n].to(at::kFloat).contiguous();
                at[n] = given[n].const_data_ptr<float>();
            }
        {
            const at::NoGradGuard none;
            const c10::cuda::CUDAGuard guard(x.device());
            const int64_t rows = x.size(0), V = x.size(1);
            grad = at::empty({rows, V}, x.options().requires_grad(false));
            const int rc = g_logprobs_grad(x.const_data_ptr(), float_code(x), rows > 1 ? x.stride(0) : V, rows, V, t.const_data_ptr<int64_t>(), temperature, (int)k,
                                           k ? i.const_data_ptr<int64_t>() : nullptr, at[0], at[1], at[2], s.const_data_ptr<float>(), grad.mutable_data_ptr(), V, stream_of(x));
            TORCH_CHECK(rc == 0, "lowbit_token_logprobs_grad_cuda: native error ", rc);
        }
        if (at::GradMode::is_enabled()) {                      // create_graph: there is no derivative of this
            auto error = std::make_shared<torch::autograd::DelayedError>("the gradient of token_logprobs has no derivative", 1);
            return (*error)({grad.requires_grad_()});
        }
        return {grad};
    }
};

}  // namespace

// token_logprobs(logits [rows, vocabulary], tokens, top_k, temperature) -> the four of a TokenLogprobs, with a gradient where the logits want one
PyObject* token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 4 || !g_logprobs) Py_RETURN_NONE;
    const at::Tensor *x = plain(a[0]), *tokens = plain(a[1]);
    int64_t k;
    double temperature;
    if (x && x->requires_grad() && at::GradMode::is_enabled() && c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) {
        // the engine would make a leaf's node's stream wait for the recorded one, which the default stream cannot: that ends the recording, and the process with it
        const at::TensorBase& leaf = x->is_view() ? x->_base() : *x;
        const auto node = leaf.is_leaf() && leaf.requires_grad() ? torch::autograd::impl::try_get_grad_accumulator(leaf) : nullptr;
        TORCH_CHECK(!node || node->stream() != c10::cuda::getDefaultCUDAStream(x->device().index()).unwrap(),
                    "these logits have a gradient's node of the default stream from outside the recording: let go of what was computed from them before");
    }
    if (!x || x->dim() != 2 || float_code(*x) < 0 || x->_fw_grad(0).defined() || !integer(a[2], &k) || !number(a[3], &temperature) || !(temperature >= 1e-7) || !(temperature <= 1e7))
        Py_RETURN_NONE;
    const int64_t rows = x->size(0), V = x->size(1);
    if (rows <= 0 || V <= 0 || k < 0 || k > 32 || k > V || (V > 1 && x->stride(1) != 1) || (rows > 1 && x->stride(0) < V) || !ints(tokens, rows, at::kLong, *x)) Py_RETURN_NONE;
    const bool grad = x->requires_grad() && at::GradMode::is_enabled();
    at::Tensor out[4];
    int rc;
    {
        const WithoutGil released;
        const c10::cuda::CUDAGuard guard(x->device());
        const auto options = x->options().dtype(at::kFloat).requires_grad(false);
        at::Tensor stats;
        if (k) out[2] = at::empty({rows, k}, options.dtype(at::kLong));
        if (grad) {
            // tensors of their own: each may be written to without the others noticing
            out[0] = at::empty({rows}, options);
            out[1] = at::empty({rows}, options);
            if (k) out[3] = at::empty({rows, k}, options);
            stats = at::empty({rows, 4}, options);
        } else {
            const at::Tensor all = at::empty({rows * (2 + k)}, options);
            out[0] = piece(all, 0, rows);
            out[1] = piece(all, rows, rows);
            if (k) out[3] = piece(all, 2 * rows, rows * k).view({rows, k});
        }
        rc = g_logprobs(x->const_data_ptr(), float_code(*x), rows > 1 ? x->stride(0) : V, rows, V, tokens->const_data_ptr<int64_t>(), (float)temperature, (int)k,
                        out[0].mutable_data_ptr<float>(), out[1].mutable_data_ptr<float>(), k ? out[2].mutable_data_ptr<int64_t>() : nullptr,
                        k ? out[3].mutable_data_ptr<float>() : nullptr, grad ? stats.mutable_data_ptr<float>() : nullptr, stream_of(*x));
        if (grad && rc == 0) {
            const std::shared_ptr<TokenLogprobsBackward> node(new TokenLogprobsBackward(), torch::autograd::deleteNode);
            node->set_next_edges(torch::autograd::collect_next_edges(*x));
            node->logits = torch::autograd::SavedVariable(*x, false);
            node->tokens = torch::autograd::SavedVariable(*tokens, false);
            node->stats = torch::autograd::SavedVariable(stats, false);
            if (k) node->ids = torch::autograd::SavedVariable(out[2], false);
            node->temperature = (float)temperature;
            node->k = k;
            torch::autograd::set_history(out[0], node);
            torch::autograd::set_history(out[1], node);
            if (k) torch::autograd::set_history(out[3], node);
        }
    }
    if (rc) return PyLong_FromLong(rc);
    PyObject* const r = PyTuple_New(4);
    if (!r) return nullptr;
    for (int i = 0; i < 4; i++) {
        if (i >= 2 && !k) { Py_INCREF(Py_None); PyTuple_SET_ITEM(r, i, Py_None); }
        else PyTuple_SET_ITEM(r, i, THPVariable_Wrap(std::move(out[i])));
    }
    return r;
    END_HANDLE_TH_ERRORS
}
