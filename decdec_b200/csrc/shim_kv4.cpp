// decdec_b200._kv4: the tensor-level functions behind decdec_b200.kv4, a thin torch/pybind11 shim over the C ABI of
// libdecdec_b200.so.  It checks tensors, allocates outputs and the workspace of attention on the current stream, and turns status
// codes into RuntimeError.  (Through ctypes the same calls cost 26 to 41 us of host time, more than most of the kernels.)
#include <torch/extension.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <pybind11/stl.h>

#include <limits>
#include <optional>

#include "decdec_b200.h"

namespace {

using at::Tensor;
using Maybe = std::optional<Tensor>;

constexpr int64_t kMost = 0x7fffffff;

int dt_of(at::ScalarType t) { return t == at::kFloat ? DECDEC_FP32 : t == at::kHalf ? DECDEC_FP16 : DECDEC_BF16; }
bool is16(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }

void ok(int code) { TORCH_CHECK(code == 0, decdec_last_error()); }
void* stream_of(const Tensor& t) { return static_cast<void*>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()); }

// memory of the caching allocator without the way through the dispatcher, which costs as much again
Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Device& device) { return at::detail::empty_cuda(sizes, type, device, std::nullopt); }
// n elements of a contiguous tensor from element `at` on: a view that only these functions hand out
Tensor part(const Tensor& base, int64_t at, int64_t n) {
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(base.storage()), base.key_set(), base.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(base.storage_offset() + at);
    t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
    return t;
}

void rows(const Tensor& t, const char* name) {
    TORCH_CHECK(t.dim() == 3, name, " must be of shape (tokens, heads, head_dim).");
    TORCH_CHECK(t.stride(2) == 1 || t.size(2) <= 1, "elements of a head of ", name, " must be neighbours.");
    TORCH_CHECK(t.size(0) <= kMost && t.size(1) <= kMost && t.size(2) <= kMost, name, " is too large.");
}

void on_gpu(const Tensor& first, std::initializer_list<const Tensor*> others) {
    TORCH_CHECK(first.is_cuda(), "tensors must be on GPU.");
    for (const Tensor* t : others) TORCH_CHECK(!t || t->device() == first.device(), "all tensors must be on the same GPU.");
}

constexpr const char* kOverlap = "an output must not share memory with itself, another output or an input.";

// rows [tokens][heads][d]: elements from the first to the last of a token, of a head, of all
int64_t token_extent(const Tensor& t) { return (t.size(1) - 1) * t.stride(1) + t.size(2); }
int64_t head_extent(const Tensor& t) { return (t.size(0) - 1) * t.stride(0) + t.size(2); }
int64_t extent(const Tensor& t) { return (t.size(0) - 1) * t.stride(0) + token_extent(t); }
bool same(const Tensor& a, const Tensor& b) { return a.data_ptr() == b.data_ptr() && a.strides() == b.strides(); }
// whether no two elements of t share a place: tokens one after another, or heads (views whose heads and tokens are wound into one another count as
// sharing)
bool spread(const Tensor& t) {
    if (t.numel() == 0) return true;
    const bool one_token = t.size(0) == 1, one_head = t.size(1) == 1;
    return ((one_head || t.stride(1) >= t.size(2)) && (one_token || t.stride(0) >= token_extent(t))) ||
           ((one_token || t.stride(0) >= t.size(2)) && (one_head || t.stride(1) >= head_extent(t)));
}
// whether a and b share no place: ranges apart, or the same token stride and different parts of it (parts of a fused projection), or the
// same head stride and different parts of that; and the other way about for heads that hold all tokens.  What it cannot tell counts as sharing.
bool apart(const Tensor& a, const Tensor& b) {
    if (!a.numel() || !b.numel()) return true;
    const int64_t size = a.element_size(), pa = (int64_t)a.data_ptr() / size, pb = (int64_t)b.data_ptr() / size;
    if (pa + extent(a) <= pb || pb + extent(b) <= pa) return true;
    auto within = [&](int64_t period, int64_t na, int64_t nb) {
        if (period <= 0) return false;
        const int64_t d = ((pb - pa) % period + period) % period;
        return d >= na && d + nb <= period;
    };
    const bool token = a.stride(0) == b.stride(0), head = a.stride(1) == b.stride(1);
    if (token && within(a.stride(0), token_extent(a), token_extent(b))) return true;
    if (head && within(a.stride(1), head_extent(a), head_extent(b))) return true;
    if (!token || !head) return false;
    const int64_t inner = std::min(a.stride(0), a.stride(1)), outer = std::max(a.stride(0), a.stride(1));
    return inner > 0 && outer % inner == 0 && within(inner, a.size(2), b.size(2));
}

// What a call writes and what else it reads, by their ranges in memory: tables, lengths and the cache are tensors of their own.
void separate(const Tensor& written, std::initializer_list<const Tensor*> read) {
    if (!written.numel()) return;
    auto bytes = [](const Tensor& t) {
        int64_t n = 1;
        for (int64_t i = 0; i < t.dim(); ++i) n += (t.size(i) - 1) * t.stride(i);
        return n * (int64_t)t.element_size();
    };
    const char* w = static_cast<const char*>(written.data_ptr());
    const int64_t size = bytes(written);
    for (const Tensor* t : read) {
        if (!t || !t->numel()) continue;
        const char* r = static_cast<const char*>(t->data_ptr());
        TORCH_CHECK(w + size <= r || r + bytes(*t) <= w, kOverlap);
    }
}

const Tensor* at_or_null(const Maybe& t) { return t ? &*t : nullptr; }

int index(const Tensor& t, int64_t n, const char* name) {
    TORCH_CHECK((t.scalar_type() == at::kInt || t.scalar_type() == at::kLong) && t.dim() == 1 && t.is_contiguous() && t.numel() == n, name,
                " must be a contiguous int32 or int64 tensor of ", n, " entries.");
    return t.scalar_type() == at::kLong;
}

const int32_t* int32s(const Tensor& t, int64_t n, const char* name) {      // n < 0: any number
    TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous() && t.numel() <= kMost, name, " must be a contiguous int32 tensor.");
    TORCH_CHECK(n < 0 || t.numel() == n, name, " must have ", n, " entries, got ", t.numel(), ".");
    return t.data_ptr<int32_t>();
}

void table(const Tensor& t, int64_t requests) {
    TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 2 && t.size(0) == requests && (t.size(1) <= 1 || t.stride(1) == 1) && t.size(1) <= kMost,
                "block_table must be an int32 tensor of shape (requests, pages) with neighbouring entries.");
}

int64_t cell_bytes(int64_t head_dim, int64_t group_size) {
    TORCH_CHECK(head_dim == 64 || head_dim == 128 || head_dim == 256, "head_dim must be 64, 128 or 256, got ", head_dim, ".");
    TORCH_CHECK((group_size == 32 || group_size == 64 || group_size == 128) && group_size <= head_dim,
                "group_size must be 32, 64 or 128 and not above head_dim, got ", group_size, ".");
    return 16 * (head_dim + 8 * head_dim / group_size);
}

struct Cache {
    void* p;
    uint32_t pages, page_size, kv_heads;
};

Cache cache_of(const Tensor& cache, int64_t head_dim, int64_t group_size) {
    TORCH_CHECK(cache.scalar_type() == at::kByte && cache.dim() == 3 && cache.is_contiguous(), "cache must be a contiguous uint8 tensor [pages, kv_heads, bytes].");
    const int64_t cell = cell_bytes(head_dim, group_size), size = cache.size(2);
    TORCH_CHECK(size > 0 && size % cell == 0 && cache.size(0) <= kMost && cache.size(1) <= kMost && size / cell * 16 <= kMost, "a page of ", size,
                " bytes is no whole number of cells of ", cell, " bytes (head_dim ", head_dim, ", group_size ", group_size, ").");
    return Cache{cache.data_ptr(), (uint32_t)cache.size(0), (uint32_t)(size / cell * 16), (uint32_t)cache.size(1)};
}

std::tuple<Tensor, Maybe> rotary(const Tensor& q, const Maybe& k, const Tensor& positions, const Tensor& frequencies, bool interleaved, double factor,
                                 const Maybe& q_out, const Maybe& k_out) {
    TORCH_CHECK(is16(q.scalar_type()) || q.scalar_type() == at::kFloat, "Unsupported data type.");
    rows(q, "q");
    if (k) {
        rows(*k, "k");
        TORCH_CHECK(k->scalar_type() == q.scalar_type() && k->size(0) == q.size(0) && k->size(2) == q.size(2), "q and k must share data type, tokens and head_dim.");
    }
    on_gpu(q, {at_or_null(k), &positions, &frequencies, at_or_null(q_out), at_or_null(k_out)});
    const int64_t tokens = q.size(0), d = q.size(2);
    TORCH_CHECK(frequencies.scalar_type() == at::kDouble && frequencies.dim() == 1 && frequencies.is_contiguous(), "frequencies must be a contiguous float64 vector.");
    TORCH_CHECK(frequencies.numel() > 0 && 2 * frequencies.numel() <= d, "there are more frequencies than pairs in a head, or none.");
    const int wide = index(positions, tokens, "positions");
    c10::cuda::CUDAGuard guard(q.device());
    Tensor qo;
    Maybe ko;
    if (q_out) {
        TORCH_CHECK(k_out.has_value() == k.has_value(), "out must have the shapes and types of q and k.");
        TORCH_CHECK(q_out->sizes() == q.sizes() && q_out->scalar_type() == q.scalar_type(), "out must have the shapes and types of q and k.");
        TORCH_CHECK(!k || (k_out->sizes() == k->sizes() && k_out->scalar_type() == k->scalar_type()), "out must have the shapes and types of q and k.");
        rows(*q_out, "out");
        if (k_out) rows(*k_out, "out");
        // an output may be its own input, and shares memory with nothing else that is read or written
        TORCH_CHECK(spread(*q_out) && (same(*q_out, q) || apart(*q_out, q)), kOverlap);
        separate(*q_out, {&positions, &frequencies});
        if (k) {
            TORCH_CHECK(spread(*k_out) && (same(*k_out, *k) || apart(*k_out, *k)), kOverlap);
            TORCH_CHECK(apart(*q_out, *k) && apart(*k_out, q) && apart(*k_out, *q_out), kOverlap);
            separate(*k_out, {&positions, &frequencies});
        }
        qo = *q_out;
        ko = k_out;
    } else {
        qo = empty({tokens, q.size(1), d}, q.scalar_type(), q.device());
        if (k) ko = empty({tokens, k->size(1), d}, q.scalar_type(), q.device());
    }
    ok(decdec_rotary(q.data_ptr(), q.stride(0), q.stride(1), (uint32_t)q.size(1), k ? k->data_ptr() : nullptr, k ? k->stride(0) : 0, k ? k->stride(1) : 0,
                     k ? (uint32_t)k->size(1) : 0, qo.data_ptr(), qo.stride(0), qo.stride(1), ko ? ko->data_ptr() : nullptr, ko ? ko->stride(0) : 0,
                     ko ? ko->stride(1) : 0, positions.data_ptr(), wide, frequencies.data_ptr<double>(), (uint32_t)tokens, (uint32_t)d,
                     (uint32_t)(2 * frequencies.numel()), interleaved, (float)factor, dt_of(q.scalar_type()), stream_of(q)));
    return {qo, ko};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> plan(const Tensor& lengths, const Tensor& fresh, const Tensor& block_table, const Tensor& free_pages,
                                                                const Tensor& free_count, int64_t page_size, int64_t tokens) {
    const int64_t requests = lengths.numel();
    on_gpu(lengths, {&fresh, &block_table, &free_pages, &free_count});
    const int32_t* len = int32s(lengths, -1, "lengths");
    const int32_t* add = int32s(fresh, requests, "new_lengths");
    table(block_table, requests);
    TORCH_CHECK(requests <= 1 || block_table.stride(0) >= block_table.size(1), "rows of block_table must not overlap, it is written.");
    separate(block_table, {&lengths, &fresh, &free_pages, &free_count});
    const int32_t* pages = int32s(free_pages, -1, "free_pages");
    const int32_t* count = int32s(free_count, 1, "free_count");
    TORCH_CHECK(tokens >= 0 && tokens <= kMost, "tokens must be from 0 to 2^31 - 1.");
    TORCH_CHECK(page_size > 0 && page_size <= kMost, "page_size must be a multiple of 16 up to 65536, got ", page_size);
    c10::cuda::CUDAGuard guard(lengths.device());
    const Tensor wide = empty({2 * tokens}, at::kLong, lengths.device()), narrow = empty({2 * requests + 3}, at::kInt, lengths.device());
    const Tensor positions = part(wide, 0, tokens), slots = part(wide, tokens, tokens), starts = part(narrow, 0, requests + 1),
                 after = part(narrow, requests + 1, requests), left = part(narrow, 2 * requests + 1, 1), status = part(narrow, 2 * requests + 2, 1);
    int64_t* w = wide.data_ptr<int64_t>();
    int32_t* n = narrow.data_ptr<int32_t>();
    ok(decdec_kv4_plan(len, add, (uint32_t)requests, block_table.data_ptr<int32_t>(), block_table.stride(0), (uint32_t)block_table.size(1), pages,
                       (uint32_t)free_pages.numel(), count, (uint32_t)page_size, (uint32_t)tokens, w, w + tokens, n,
                       n + requests + 1, n + 2 * requests + 1, n + 2 * requests + 2, stream_of(lengths)));
    return {positions, slots, starts, after, left, status};
}

void append(const Tensor& cache, const Tensor& k, const Tensor& v, const Tensor& slots, int64_t group_size) {
    TORCH_CHECK(is16(k.scalar_type()) && v.scalar_type() == k.scalar_type(), "k and v must both be half or both bfloat16.");
    rows(k, "k");
    rows(v, "v");
    TORCH_CHECK(k.sizes() == v.sizes(), "k and v must have the same shape.");
    on_gpu(k, {&v, &slots, &cache});
    const Cache c = cache_of(cache, k.size(2), group_size);
    TORCH_CHECK(k.size(1) == c.kv_heads, "the cache has ", c.kv_heads, " heads, k and v have ", k.size(1), ".");
    const int wide = index(slots, k.size(0), "slots");
    separate(cache, {&k, &v, &slots});
    c10::cuda::CUDAGuard guard(k.device());
    ok(decdec_kv4_append(k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), slots.data_ptr(), wide, (uint32_t)k.size(0), c.p, c.pages,
                         c.page_size, c.kv_heads, (uint32_t)k.size(2), (uint32_t)group_size, dt_of(k.scalar_type()), stream_of(k)));
}

std::tuple<Tensor, Tensor> gather(const Tensor& cache, const Tensor& slots, int64_t head_dim, int64_t group_size, at::ScalarType dtype) {
    TORCH_CHECK(is16(dtype), "dtype must be half or bfloat16.");
    on_gpu(cache, {&slots});
    const Cache c = cache_of(cache, head_dim, group_size);
    const int64_t n = slots.numel();
    const int wide = index(slots, n, "slots");
    TORCH_CHECK(n <= kMost, "too many slots.");
    c10::cuda::CUDAGuard guard(cache.device());
    const Tensor k = empty({n, c.kv_heads, head_dim}, dtype, cache.device()), v = empty({n, c.kv_heads, head_dim}, dtype, cache.device());
    ok(decdec_kv4_gather(c.p, c.pages, c.page_size, c.kv_heads, (uint32_t)head_dim, (uint32_t)group_size, slots.data_ptr(), wide, (uint32_t)n, k.data_ptr(),
                         v.data_ptr(), dt_of(dtype), stream_of(cache)));
    return {k, v};
}

std::tuple<Tensor, Maybe> attention(const Tensor& q, const Tensor& cache, const Tensor& block_table, const Tensor& lengths, const Tensor& query_starts,
                                    int64_t group_size, std::optional<int64_t> max_queries, std::optional<double> scale, int64_t window, const Maybe& out_given,
                                    bool return_lse) {
    TORCH_CHECK(is16(q.scalar_type()), "q must be half or bfloat16.");
    rows(q, "q");
    on_gpu(q, {&cache, &block_table, &lengths, &query_starts, at_or_null(out_given)});
    const int64_t tokens = q.size(0), heads = q.size(1), d = q.size(2), requests = lengths.numel();
    const Cache c = cache_of(cache, d, group_size);
    TORCH_CHECK(c.kv_heads > 0 && heads > 0 && heads % c.kv_heads == 0, "heads of q must be a multiple of the cache's ", c.kv_heads, ", got ", heads, ".");
    table(block_table, requests);
    const int32_t* len = int32s(lengths, -1, "lengths");
    const int32_t* starts = int32s(query_starts, requests + 1, "query_starts");
    TORCH_CHECK(window >= 0, "window must not be negative.");
    TORCH_CHECK(!max_queries || *max_queries >= 1, "max_queries must be at least 1.");
    const uint32_t most = (uint32_t)std::max<int64_t>(1, max_queries ? std::min(*max_queries, tokens) : tokens);
    c10::cuda::CUDAGuard guard(q.device());
    Tensor out;
    if (out_given) {
        TORCH_CHECK(out_given->sizes() == q.sizes() && out_given->scalar_type() == q.scalar_type(), "out must have the shape and type of q.");
        rows(*out_given, "out");
        TORCH_CHECK(spread(*out_given) && apart(*out_given, q), kOverlap);
        separate(*out_given, {&cache, &block_table, &lengths, &query_starts});
        out = *out_given;
    } else {
        out = empty({tokens, heads, d}, q.scalar_type(), q.device());
    }
    Maybe lse;
    if (return_lse) lse = at::full({tokens, heads}, -std::numeric_limits<double>::infinity(), q.options().dtype(at::kFloat));
    const int dt = dt_of(q.scalar_type());
    size_t bytes = 0;
    ok(decdec_kv4_attention_workspace((uint32_t)requests, (uint32_t)tokens, (uint32_t)heads, c.kv_heads, (uint32_t)d, (uint32_t)group_size, most, dt, &bytes));
    const Tensor workspace = empty({(int64_t)bytes}, at::kByte, q.device());
    ok(decdec_kv4_attention(q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(), out.stride(0), out.stride(1), lse ? lse->data_ptr<float>() : nullptr, c.p,
                            c.pages, c.page_size, block_table.data_ptr<int32_t>(), block_table.stride(0), (uint32_t)block_table.size(1), len, starts,
                            (uint32_t)requests, (uint32_t)tokens, (uint32_t)heads, c.kv_heads, (uint32_t)d, (uint32_t)group_size, most,
                            scale ? (float)*scale : 1.0f / std::sqrt((float)d), (uint32_t)std::min(window, kMost), !out_given, workspace.data_ptr(), bytes, dt,
                            stream_of(q)));
    return {out, lse};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("cell_bytes", &cell_bytes);
    m.def("rotary", &rotary);
    m.def("plan", &plan);
    m.def("append", &append);
    m.def("gather", [](const Tensor& cache, const Tensor& slots, int64_t head_dim, int64_t group_size, const py::object& dtype) {
        return gather(cache, slots, head_dim, group_size, torch::python::detail::py_object_to_dtype(dtype));
    });
    m.def("attention", &attention);
}
