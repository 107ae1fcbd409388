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

fg_kv_cache cache(const at::Tensor& k, const at::Tensor& v) {  // (k, k) where only the keys are read
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

// The lengths that say where a batch's requests are, checked against one another.
void requests(at::Tensor& table, at::Tensor& query_start, at::Tensor& kv_len) {
    table = ints(table, 2, "block_table");
    query_start = ints(query_start, 1, "query_start");
    kv_len = ints(kv_len, 1, "kv_len");
    const int64_t R = kv_len.size(0);
    FG_NEED(query_start.size(0) == R + 1 && table.size(0) == R,
            std::to_string(R) + " lengths need " + std::to_string(R + 1) + " query_start entries and " + std::to_string(R) + " table rows, not " +
                std::to_string(query_start.size(0)) + " and " + std::to_string(table.size(0)));
}

std::tuple<at::Tensor, std::optional<at::Tensor>> attention(at::Tensor q, const at::Tensor& k_cache, const at::Tensor& v_cache, at::Tensor table,
                                                            at::Tensor query_start, at::Tensor kv_len, int64_t max_new,
                                                            std::optional<at::Tensor> ids, bool blocks, int64_t window, int64_t sinks,
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
    requests(table, query_start, kv_len);
    const int64_t R = kv_len.size(0);
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
        const int64_t lists = blocks ? c.heads : heads;
        FG_NEED(ids->scalar_type() == at::kInt && ids->dim() == 3 && ids->size(0) == T && ids->size(1) == lists,
                std::string(blocks ? "blocks" : "ids") + " must be int32 [" + std::to_string(T) + ", " + std::to_string(lists) + ", count], not " +
                    shape(*ids));
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
    check(fg_attention_workspace_bytes(&c, &x, !ids ? 0 : blocks ? 2 : 1, &bytes), "fg_attention_workspace_bytes");
    at::Tensor work;
    if (bytes) {
        work = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
        x.workspace = work.data_ptr();
        x.workspace_bytes = bytes;
    }
    if (ids && blocks) check(fg_block_attention_device(&c, &x, on.stream()), "fg_block_attention_device");
    else if (ids) check(fg_retrieved_attention_device(&c, &x, on.stream()), "fg_retrieved_attention_device");
    else check(fg_paged_attention_device(&c, &x, on.stream()), "fg_paged_attention_device");
    if (out_or_none) written(out);
    return {out, lse};
}

fg_kv_summary summary(const at::Tensor& bounds, const at::Tensor& scale, int64_t page_size) {
    FG_NEED(bounds.scalar_type() == at::kChar && bounds.dim() == 4 && bounds.size(2) == 2,
            "bounds must be int8 [pages, heads, 2, dim], not " + shape(bounds));
    FG_NEED(bounds.stride(3) == 1 && bounds.stride(2) == bounds.size(3), "bounds must have contiguous last two axes");
    FG_NEED(scale.scalar_type() == at::kFloat && scale.dim() == 2 && scale.size(0) == bounds.size(0) && scale.size(1) == bounds.size(1),
            "scale must be float32 [" + std::to_string(bounds.size(0)) + ", " + std::to_string(bounds.size(1)) + "], not " + shape(scale));
    fg_kv_summary s{};
    s.bounds = bounds.data_ptr<int8_t>();
    s.scale = scale.data_ptr<float>();
    s.bounds_page_stride = bounds.stride(0);
    s.bounds_head_stride = bounds.stride(1);
    s.scale_page_stride = scale.stride(0);
    s.scale_head_stride = scale.stride(1);
    s.pages = i32(bounds.size(0), "pages");
    s.page_size = i32(page_size, "page size");
    s.heads = i32(bounds.size(1), "heads");
    s.dim = i32(bounds.size(3), "dim");
    return s;
}

void kv_summarize(const at::Tensor& k_cache, const at::Tensor& bounds, const at::Tensor& scale, at::Tensor table, at::Tensor query_start,
                  at::Tensor kv_len, int64_t tokens, int64_t stream) {
    On on(k_cache, stream);
    on.uses(k_cache, bounds, scale, table, query_start, kv_len);
    no_gradient("k_cache and scale", k_cache, scale);
    const fg_kv_cache c = cache(k_cache, k_cache);
    const fg_kv_summary s = summary(bounds, scale, c.page_size);
    requests(table, query_start, kv_len);
    check(fg_kv_summarize_device(&c, &s, table.data_ptr<int32_t>(), i32(table.size(1), "table width"), table.stride(0),
                                 query_start.data_ptr<int32_t>(), kv_len.data_ptr<int32_t>(), i32(kv_len.size(0), "requests"),
                                 i32(tokens, "tokens"), on.stream()),
          "fg_kv_summarize_device");
    written(bounds);
    written(scale);
}

at::Tensor select_blocks(at::Tensor q, const at::Tensor& bounds, const at::Tensor& scale, at::Tensor table, at::Tensor query_start,
                         at::Tensor kv_len, int64_t count, int64_t page_size, int64_t window, int64_t sinks,
                         const std::optional<at::Tensor>& out_or_none, int64_t stream) {
    On on(q, stream);
    on.uses(q, bounds, scale, table, query_start, kv_len);
    if (out_or_none) on.uses(*out_or_none);
    no_gradient("q and scale", q, scale);
    const fg_kv_summary s = summary(bounds, scale, page_size);
    q = rows(q, "q");
    FG_NEED((q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16) && q.size(2) == s.dim,
            "q must be float16 or bfloat16 [tokens, heads, " + std::to_string(s.dim) + "], not " + shape(q));
    requests(table, query_start, kv_len);
    const int64_t T = q.size(0);
    FG_NEED(count >= 0, "count " + std::to_string(count) + " is negative");
    i32(count, "count");
    at::Tensor out;
    if (out_or_none) {
        out = *out_or_none;
        FG_NEED(out.scalar_type() == at::kInt && out.dim() == 3 && out.size(0) == T && out.size(1) == s.heads && out.size(2) == count &&
                    (out.stride(2) == 1 || count <= 1),
                "out must be int32 [" + std::to_string(T) + ", " + std::to_string(s.heads) + ", " + std::to_string(count) +
                    "] with a contiguous last axis, not " + shape(out));
    } else {
        out = at::empty({T, s.heads, count}, q.options().dtype(at::kInt));
    }
    fg_block_selection x{};
    x.q = q.data_ptr();
    x.q_token_stride = q.stride(0);
    x.q_head_stride = q.stride(1);
    x.block_table = table.data_ptr<int32_t>();
    x.table_stride = table.stride(0);
    x.query_start = query_start.data_ptr<int32_t>();
    x.kv_len = kv_len.data_ptr<int32_t>();
    x.blocks = out.data_ptr<int32_t>();
    x.blocks_token_stride = out.stride(0);
    x.blocks_head_stride = out.stride(1);
    x.tokens = i32(T, "tokens");
    x.heads = i32(q.size(1), "heads");
    x.requests = i32(kv_len.size(0), "requests");
    x.table_width = i32(table.size(1), "table width");
    x.window = i32(window, "window");
    x.sinks = i32(sinks, "sinks");
    x.count = i32(count, "count");
    x.dtype = q.scalar_type() == at::kHalf ? FG_DTYPE_F16 : FG_DTYPE_BF16;
    uint64_t bytes = 0;
    check(fg_select_blocks_workspace_bytes(&s, &x, &bytes), "fg_select_blocks_workspace_bytes");
    at::Tensor work;
    if (bytes) {
        work = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
        x.workspace = work.data_ptr();
        x.workspace_bytes = bytes;
    }
    check(fg_select_blocks_device(&s, &x, on.stream()), "fg_select_blocks_device");
    if (out_or_none) written(out);
    return out;
}

// float32 [pages, heads, page_size] beside a cache
void check_weights(const at::Tensor& weights, const fg_kv_cache& c) {
    FG_NEED(weights.scalar_type() == at::kFloat && weights.dim() == 3 && weights.size(0) == c.pages && weights.size(1) == c.heads &&
                weights.size(2) == c.page_size && (weights.stride(2) == 1 || c.page_size == 1),
            "weights must be float32 [" + std::to_string(c.pages) + ", " + std::to_string(c.heads) + ", " + std::to_string(c.page_size) +
                "] with a contiguous last axis, not " + shape(weights));
}

void attention_weights(at::Tensor q, const at::Tensor& k_cache, const at::Tensor& weights, at::Tensor table, at::Tensor query_start,
                       at::Tensor kv_len, at::Tensor lse, std::optional<at::Tensor> held, int64_t window, int64_t sinks,
                       std::optional<double> scale, int64_t stream) {
    On on(q, stream);
    on.uses(q, k_cache, weights, table, query_start, kv_len, lse);
    if (held) on.uses(*held);
    no_gradient("q, k_cache, weights and lse", q, k_cache, weights, lse);
    const fg_kv_cache c = cache(k_cache, k_cache);
    check_weights(weights, c);
    q = rows(q, "q");
    const int64_t T = q.size(0), heads = q.size(1), dim = q.size(2);
    FG_NEED(q.scalar_type() == k_cache.scalar_type() && dim == c.dim,
            "q must be " + std::string(at::toString(k_cache.scalar_type())) + " [tokens, heads, " + std::to_string(c.dim) + "], not " + shape(q));
    FG_NEED(lse.scalar_type() == at::kFloat && lse.dim() == 2 && lse.size(0) == T && lse.size(1) == heads,
            "lse must be float32 [" + std::to_string(T) + ", " + std::to_string(heads) + "], not " + shape(lse));
    lse = lse.contiguous();
    requests(table, query_start, kv_len);
    if (held) {
        held = ints(*held, 1, "held");
        FG_NEED(held->size(0) == kv_len.size(0), "held and kv_len differ in length");
    }
    fg_attention x{};
    x.q = q.data_ptr();
    x.q_token_stride = q.stride(0);
    x.q_head_stride = q.stride(1);
    x.lse = lse.data_ptr<float>();
    x.block_table = table.data_ptr<int32_t>();
    x.table_stride = table.stride(0);
    x.query_start = query_start.data_ptr<int32_t>();
    x.kv_len = kv_len.data_ptr<int32_t>();
    x.tokens = i32(T, "tokens");
    x.heads = i32(heads, "heads");
    x.requests = i32(kv_len.size(0), "requests");
    x.table_width = i32(table.size(1), "table width");
    x.window = i32(window, "window");
    x.sinks = i32(sinks, "sinks");
    x.scale = static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(dim)));
    check(fg_attention_weights_device(&c, &x, weights.data_ptr<float>(), weights.stride(0), weights.stride(1),
                                      held ? held->data_ptr<int32_t>() : nullptr, on.stream()),
          "fg_attention_weights_device");
    written(weights);
}

std::tuple<at::Tensor, at::Tensor> kv_evict(const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& weights, at::Tensor table,
                                            at::Tensor kv_len, int64_t budget, int64_t recent, int64_t sinks, int64_t stream) {
    On on(k_cache, stream);
    on.uses(k_cache, v_cache, weights, table, kv_len);
    no_gradient("k_cache, v_cache and weights", k_cache, v_cache, weights);
    const fg_kv_cache c = cache(k_cache, v_cache);
    check_weights(weights, c);
    table = ints(table, 2, "block_table");
    kv_len = ints(kv_len, 1, "kv_len");
    const int64_t R = kv_len.size(0);
    FG_NEED(table.size(0) == R, std::to_string(R) + " lengths need as many table rows, not " + std::to_string(table.size(0)));
    FG_NEED(budget >= 1, "budget " + std::to_string(budget) + " is not positive");
    const at::Tensor len = at::empty({R}, kv_len.options());
    const at::Tensor kept = at::empty({R, c.heads, i32(budget, "budget")}, kv_len.options());
    check(fg_kv_evict_device(&c, weights.data_ptr<float>(), weights.stride(0), weights.stride(1), table.data_ptr<int32_t>(),
                             i32(table.size(1), "table width"), table.stride(0), kv_len.data_ptr<int32_t>(), i32(R, "requests"),
                             i32(budget, "budget"), i32(recent, "recent"), i32(sinks, "sinks"), len.data_ptr<int32_t>(),
                             kept.data_ptr<int32_t>(), on.stream()),
          "fg_kv_evict_device");
    written(k_cache);
    written(v_cache);
    written(weights);
    return {len, kept};
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
    m.def("kv_plan", &kv_plan);
    m.def("kv_append", &kv_append);
    m.def("attention", &attention);
    m.def("kv_summarize", &kv_summarize);
    m.def("select_blocks", &select_blocks);
    m.def("attention_weights", &attention_weights);
    m.def("kv_evict", &kv_evict);
}
