// what the host sides of a server's operators share (paged_host.cpp, step_host.cpp): looks at their arguments
#pragma once
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

namespace {

struct WithoutGil {
    PyThreadState* const state = PyEval_SaveThread();
    ~WithoutGil() { PyEval_RestoreThread(state); }
};
[[maybe_unused]] int half_code(const at::Tensor& t) { return t.scalar_type() == at::kHalf ? 1 : t.scalar_type() == at::kBFloat16 ? 2 : -1; }
[[maybe_unused]] constexpr int kE5m2 = 19;

// an exact tensor with storage on a CUDA device
[[maybe_unused]] const at::Tensor* plain(PyObject* o) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.is_cuda() && t.has_storage() ? &t : nullptr;
}
[[maybe_unused]] bool ints(const at::Tensor* t, int64_t n, at::ScalarType type, const at::Tensor& like) {
    return t && t->scalar_type() == type && t->dim() == 1 && t->size(0) == n && t->is_contiguous() && t->device() == like.device();
}
[[maybe_unused]] bool table_ok(const at::Tensor* t, const at::Tensor& like) {
    return t && t->scalar_type() == at::kInt && t->dim() == 2 && t->numel() > 0 && t->stride(1) == 1 && t->stride(0) >= t->size(1) && t->device() == like.device() &&
           t->size(0) <= 0x7fffffff && t->size(1) <= 0x7fffffff;
}
// rows of the last dimension contiguous and on 16 bytes
[[maybe_unused]] bool aligned(const at::Tensor& t) {
    const int64_t unit = 16 / t.element_size();
    if (t.stride(-1) != 1 || (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15)) return false;
    for (int64_t d = 0; d + 1 < t.dim(); d++)
        if (t.stride(d) % unit) return false;
    return true;
}
// a gradient, or a tangent of forward mode (which no_grad does not end)
[[maybe_unused]] bool wants_grad(const at::Tensor& t) { return (t.requires_grad() && at::GradMode::is_enabled()) || t._fw_grad(0).defined(); }
[[maybe_unused]] bool caches_ok(const at::Tensor* k, const at::Tensor* v, const at::Tensor& like, int64_t dim) {
    return k && v && k->dim() == 4 && v->sizes() == k->sizes() && k->numel() > 0 && k->scalar_type() == v->scalar_type() && k->stride(3) == 1 && v->stride(3) == 1 &&
           k->size(3) == dim && k->device() == like.device() && v->device() == like.device() && (k->scalar_type() == at::kByte || k->scalar_type() == like.scalar_type()) &&
           k->size(0) <= 0x7fffffff && k->size(1) <= 0x7fffffff;
}
// a piece of a buffer as a tensor of its own (a view, without the dispatcher's share)
[[maybe_unused]] at::Tensor piece(const at::Tensor& base, int64_t offset, int64_t n) {
    auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(base.storage()), base.key_set(), base.dtype());
    impl->set_storage_offset(offset);
    impl->set_sizes_contiguous({n});
    return at::Tensor(std::move(impl));
}
[[maybe_unused]] bool integer(PyObject* o, int64_t* out) {
    if (!PyLong_CheckExact(o)) return false;
    int over = 0;
    *out = PyLong_AsLongLongAndOverflow(o, &over);
    return !over;
}
[[maybe_unused]] void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

}  // namespace
