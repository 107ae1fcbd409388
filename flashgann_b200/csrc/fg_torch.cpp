// fg_torch.cpp -- the torch binding of the cache and attention calls
// (flashgann_b200/_torch_ops.so, used by flashgann_b200/attention.py).
//
// The other calls of the library are bound by ctypes.  These are made once for
// each layer of a decode step, where filling the argument structs and making
// the outputs in Python took 12 of 16 us and the kernel's launch 3; here it is
// the same checks and allocations in C++ (a call of one kernel: 6.9 us on the
// host).  No work beside that: every call ends in
// the C ABI (include/flashgann.h).
#include <cmath>
#include <cstdint>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/flashgann.h"

namespace {

[[noreturn]] void raise(int status, const std::string& message) {
    const py::object cls = py::module_::import("flashgann_b200._capi").attr("FlashGANNError");
    const py::object error = cls(status, message);
    PyErr_SetObject(cls.ptr(), error.ptr());
    throw py::error_already_set();
}

void check(int rc, const char* call) {
    if (rc != FG_OK) raise(rc, std::string(call) + ": " + fg_status_string(rc) + " (" + fg_last_error() + ")");
}

// a macro: the message is put together only where it is raised
#define FG_NEED(ok, message)                      \
    do {                                          \
        if (!(ok)) raise(FG_ERR_ARG, (message));  \
    } while (0)

int32_t i32(int64_t x, const char* name) {
    FG_NEED(x >= INT32_MIN && x <= INT32_MAX, std::string(name) + " " + std::to_string(x) + " is out of range");
    return static_cast<int32_t>(x);
}

std::string shape(const at::Tensor& t) {
    std::string s = std::string(at::toString(t.scalar_type())) + " [";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + "]";
}

// The device and stream of one call.  Tensors made while it lives belong to
// that stream; inputs that live on another one are marked as in use there, so
// that the caller may drop them right after the call.
class On {
public:
    // stream: a handle, or -1 for the current one
    On(const at::Tensor& like, int64_t stream) {
        FG_NEED(like.is_cuda(), "expected a CUDA tensor");
        index_ = like.device().index();
        device_.emplace(index_);
        stream_ = c10::cuda::getCurrentCUDAStream(index_);
        if (stream != -1 && reinterpret_cast<cudaStream_t>(stream) != stream_->stream()) {
            stream_ = stream ? c10::cuda::getStreamFromExternal(reinterpret_cast<cudaStream_t>(stream), index_)
                             : c10::cuda::getDefaultCUDAStream(index_);
            other_.emplace(*stream_);
        }
    }
    template <typename... Tensors>
    void uses(const at::Tensor& t, const Tensors&... more) {
        FG_NEED(t.is_cuda() && t.device().index() == index_, "a tensor is on " + t.device().str() + ", not on device " + std::to_string(index_));
        if (other_) t.record_stream(stream_->unwrap());
        if constexpr (sizeof...(more) > 0) uses(more...);
    }
    void* stream() const { return stream_->stream(); }

private:
    c10::DeviceIndex index_ = 0;
    std::optional<c10::cuda::CUDAGuard> device_;
    std::optional<c10::cuda::CUDAStream> stream_;
    std::optional<c10::cuda::CUDAStreamGuard> other_;
};

// The calls have no backward pass: a gradient that would be lost is refused.
template <typename... Tensors>
void no_gradient(const char* names, const Tensors&... t) {
    FG_NEED(!c10::GradMode::is_enabled() || !(... || t.requires_grad()),
            std::string("one of ") + names + " requires a gradient, and this call computes none: call it under torch.no_grad()");
}
// What a call writes in place, for autograd's count of a tensor's versions.
void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

at::Tensor ints(const at::Tensor& t, int64_t dims, const char* name, at::ScalarType type = at::kInt) {
    FG_NEED(t.scalar_type() == type && t.dim() == dims,
            std::string(name) + " must be " + at::toString(type) + " with " + std::to_string(dims) + " dimension(s), not " + shape(t));
    return t.stride(-1) == 1 || t.size(-1) <= 1 ? t : t.contiguous();
}

// [tokens, heads, dim] with a contiguous last axis and 16-byte aligned rows (a copy where it is not)
at::Tensor rows(const at::Tensor& t, const char* name) {
    FG_NEED(t.dim() == 3, std::string(name) + " must be [tokens, heads, dim], not " + shape(t));
    const int64_t strides = (t.size(0) > 1 ? t.stride(0) : 0) | (t.size(1) > 1 ? t.stride(1) : 0);
    if ((t.stride(2) != 1 && t.size(2) > 1) || strides % 8 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16)
        return t.clone(at::MemoryFormat::Contiguous);
    return t;
}

fg_kv_cache cache(const at::Tensor& k, const at::Tensor& v) {
    FG_NEED(k.dim() == 4 && v.sizes() == k.sizes(), "caches must be [pages, page_size, heads, dim] alike, not " + shape(k) + " and " + shape(v));
    FG_NEED((k.scalar_type() == at::kHalf || k.scalar_type() == at::kBFloat16) && v.scalar_type() == k.scalar_type(),
            "caches must both be float16 or bfloat16, not " + shape(k) + " and " + shape(v));
    for (int64_t i = 0; i < 3; ++i)  // torch leaves the stride of an axis of one entry open
        FG_NEED(k.stride(i) == v.stride(i) || k.size(i) == 1, "caches must have the same strides");
    FG_NEED(k.stride(3) == 1 && v.stride(3) == 1, "caches must have a contiguous last axis");
    fg_kv_cache c{};
    c.k = k.data_ptr();
    c.v = v.data_ptr();
    c.page_stride = k.stride(0);
    c.token_stride = k.stride(1);
    c.head_stride = k.stride(2);
    c.pages = i32(k.size(0), "pages");
    c.page_size = i32(k.size(1), "page size");
    c.heads = i32(k.size(2), "heads");
    c.dim = i32(k.size(3), "dim");
    c.dtype = k.scalar_type() == at::kHalf ? FG_DTYPE_F16 : FG_DTYPE_BF16;
    return c;
}

using Six = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>;

Six kv_plan(at::Tensor ctx_len, at::Tensor new_len, const at::Tensor& table, at::Tensor free_pages, int64_t tokens, int64_t page_size,
            const std::optional<at::Tensor>& free_head, int64_t stream) {
    On on(ctx_len, stream);
    on.uses(ctx_len, new_len, table, free_pages);
    if (free_head) on.uses(*free_head);
    ctx_len = ints(ctx_len, 1, "ctx_len");
    new_len = ints(new_len, 1, "new_len");
    free_pages = ints(free_pages, 1, "free_pages");
    const int64_t R = ctx_len.size(0), T = i32(tokens, "tokens") > 0 ? tokens : 0;
    FG_NEED(new_len.size(0) == R, "ctx_len and new_len differ in length");
    FG_NEED(table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) == R && (table.size(1) <= 1 || table.stride(1) == 1),
            "block_table must be int32 [" + std::to_string(R) + ", width] with contiguous rows");
    FG_NEED(!free_head || (free_head->scalar_type() == at::kInt && free_head->numel() == 1), "free_head must be int32 [1]");
    const at::Tensor slot = at::empty({T}, ctx_len.options().dtype(at::kLong));
    const at::Tensor all = at::empty({3 * R + 2 + T}, ctx_len.options());
    int32_t* p = all.data_ptr<int32_t>();
    check(fg_kv_plan_device(ctx_len.data_ptr<int32_t>(), new_len.data_ptr<int32_t>(), i32(R, "requests"), free_pages.data_ptr<int32_t>(),
                            i32(free_pages.size(0), "free pages"), free_head ? free_head->data_ptr<int32_t>() : nullptr,
                            i32(page_size, "page size"), table.data_ptr<int32_t>(), i32(table.size(1), "table width"), table.stride(0),
                            i32(tokens, "tokens"), p, p + R + 1, p + 3 * R + 2, slot.data_ptr<int64_t>(), p + 2 * R + 1, p + 2 * R + 2,
                            on.stream()),
          "fg_kv_plan_device");
    written(table);
    const std::vector<at::Tensor> v = all.split_with_sizes({R + 1, R, 1, R, T});
    return {v[0], v[1], v[4], slot, v[2], v[3]};
}

void kv_append(const at::Tensor& k_cache, const at::Tensor& v_cache, at::Tensor k, at::Tensor v, at::Tensor slot, int64_t stream) {
    On on(k_cache, stream);
    on.uses(k_cache, v_cache, k, v, slot);
    no_gradient("k_cache, v_cache, k and v", k_cache, v_cache, k, v);
    const fg_kv_cache c = cache(k_cache, v_cache);
    slot = ints(slot, 1, "slot", at::kLong);
    const int64_t T = slot.size(0);
    for (const at::Tensor* t : {&k, &v})
        FG_NEED(t->scalar_type() == k_cache.scalar_type() && t->dim() == 3 && t->size(0) == T && t->size(1) == c.heads && t->size(2) == c.dim,
                "k and v must be " + std::string(at::toString(k_cache.scalar_type())) + " [" + std::to_string(T) + ", " + std::to_string(c.heads) +
                    ", " + std::to_string(c.dim) + "], not " + shape(*t));
    k = rows(k, "k");
    v = rows(v, "v");
    check(fg_kv_append_device(&c, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), slot.data_ptr<int64_t>(),
                              i32(T, "tokens"), on.stream()),
          "fg_kv_append_device");
    written(k_cache);
    written(v_cache);
}

std::tuple<at::Tensor, std::optional<at::Tensor>> attention(at::Tensor q, const at::Tensor& k_cache, const at::Tensor& v_cache, at::Tensor table,
                                                            at::Tensor query_start, at::Tensor kv_len, int64_t max_new,
                                                            std::optional<at::Tensor> ids, int64_t window, int64_t sinks,
                                                            std::optional<double> scale, const std::optional<at::Tensor>& out_or_none,
                                                            bool return_lse, int64_t stream) {
    On on(q, stream);
    on.uses(q, k_cache, v_cache, table, query_start, kv_len);
    if (ids) on.uses(*ids);
    if (out_or_none) on.uses(*out_or_none);
    no_gradient("q, k_cache, v_cache and out", q, k_cache, v_cache, out_or_none ? *out_or_none : q);
    const fg_kv_cache c = cache(k_cache, v_cache);
    q = rows(q, "q");
    const int64_t T = q.size(0), heads = q.size(1), dim = q.size(2);
    FG_NEED(q.scalar_type() == k_cache.scalar_type() && dim == c.dim,
            "q must be " + std::string(at::toString(k_cache.scalar_type())) + " [tokens, heads, " + std::to_string(c.dim) + "], not " + shape(q));
    table = ints(table, 2, "block_table");
    query_start = ints(query_start, 1, "query_start");
    kv_len = ints(kv_len, 1, "kv_len");
    const int64_t R = kv_len.size(0);
    FG_NEED(query_start.size(0) == R + 1 && table.size(0) == R,
            std::to_string(R) + " lengths need " + std::to_string(R + 1) + " query_start entries and " + std::to_string(R) + " table rows, not " +
                std::to_string(query_start.size(0)) + " and " + std::to_string(table.size(0)));
    at::Tensor out;
    if (out_or_none) {
        out = *out_or_none;
        FG_NEED(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.stride(2) == 1,
                "out must be like q, " + shape(q) + ", with a contiguous last axis");
    } else {
        out = at::empty({T, heads, dim}, q.options());
    }
    std::optional<at::Tensor> lse;
    if (return_lse) lse = at::empty({T, heads}, q.options().dtype(at::kFloat));
    fg_attention x{};
    if (ids) {
        FG_NEED(ids->scalar_type() == at::kInt && ids->dim() == 3 && ids->size(0) == T && ids->size(1) == heads,
                "ids must be int32 [" + std::to_string(T) + ", " + std::to_string(heads) + ", count], not " + shape(*ids));
        if (ids->stride(2) != 1 && ids->size(2) > 1) ids = ids->contiguous();
        x.ids = ids->data_ptr<int32_t>();
        x.ids_token_stride = ids->stride(0);
        x.ids_head_stride = ids->stride(1);
        x.ids_count = i32(ids->size(2), "ids");
    }
    x.q = q.data_ptr();
    x.q_token_stride = q.stride(0);
    x.q_head_stride = q.stride(1);
    x.out = out.data_ptr();
    x.out_token_stride = out.stride(0);
    x.out_head_stride = out.stride(1);
    x.lse = lse ? lse->data_ptr<float>() : nullptr;
    x.block_table = table.data_ptr<int32_t>();
    x.table_stride = table.stride(0);
    x.query_start = query_start.data_ptr<int32_t>();
    x.kv_len = kv_len.data_ptr<int32_t>();
    x.tokens = i32(T, "tokens");
    x.heads = i32(heads, "heads");
    x.requests = i32(R, "requests");
    x.table_width = i32(table.size(1), "table width");
    x.max_new = i32(max_new, "max_new");
    x.window = i32(window, "window");
    x.sinks = i32(sinks, "sinks");
    x.scale = static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(dim)));
    uint64_t bytes = 0;
    check(fg_attention_workspace_bytes(&c, &x, ids.has_value(), &bytes), "fg_attention_workspace_bytes");
    at::Tensor work;
    if (bytes) {
        work = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
        x.workspace = work.data_ptr();
        x.workspace_bytes = bytes;
    }
    if (ids) check(fg_retrieved_attention_device(&c, &x, on.stream()), "fg_retrieved_attention_device");
    else check(fg_paged_attention_device(&c, &x, on.stream()), "fg_paged_attention_device");
    if (out_or_none) written(out);
    return {out, lse};
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
    m.def("kv_plan", &kv_plan);
    m.def("kv_append", &kv_append);
    m.def("attention", &attention);
}
