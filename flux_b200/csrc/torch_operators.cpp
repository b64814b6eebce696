// torch.ops.flux.* over the C ABI for the operators that a serving loop calls
// many times per token: the paged key/value cache and the logits' processing.
// They are registered here rather than from Python because their smallest calls
// take the GPU 4-6 us: a call, checks and launch included, takes the host 5-10
// us (an in-place add of torch's own 4.7), and several times that from Python.
//
// One function serves the CUDA, CPU and Meta keys.  It checks its arguments
// first, on any device; then a CUDA call launches, a Meta call (FakeTensor)
// returns the shapes, and a CPU call is refused: there is no CPU compute path.
// A Meta call whose sizes are symbols goes to a function of its own, which checks
// ranks, types and sizes and keeps the symbols.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <cmath>
#include <initializer_list>
#include <string>

#include "flux_b200.h"

namespace {

using at::Tensor;
using Optional = std::optional<Tensor>;

void check(fx_status status) { TORCH_CHECK(status == FX_OK, fx_last_error()); }

void* stream_of(const Tensor& t) {
    return static_cast<void*>(at::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

// A workspace for this call, from torch's allocator on the current stream: like
// a tensor's memory, without the tensor (0.3 us of host time).
template <typename T>
struct Workspace {
    int64_t size;
    c10::DataPtr memory;
    explicit Workspace(int64_t elements)
        : size(elements), memory(c10::cuda::CUDACachingAllocator::get()->allocate(elements * sizeof(T))) {}
    T* data() const { return static_cast<T*>(memory.get()); }
};

// Whether to launch: true for CUDA tensors, false for Meta ones; a CPU call
// has passed the checks by now and is refused.
bool launches(const char* op, const Tensor& t) {
    if (t.is_meta()) return false;
    TORCH_CHECK(t.is_cuda(), op, ": CUDA tensors are required; flux_b200 has no CPU implementation");
    return true;
}

void same_device(const char* op, const Tensor& first, std::initializer_list<const Tensor*> others) {
    for (const Tensor* t : others)
        TORCH_CHECK(t->device() == first.device(), op, ": all tensors must be on the same device");
}

void no_grad(const char* op, std::initializer_list<const Tensor*> tensors) {
    const bool backward = at::GradMode::is_enabled();
    const bool forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
    if (!backward && !forward) return;
    for (const Tensor* t : tensors) {
        TORCH_CHECK(!backward || !t->requires_grad(), op,
                    " is inference-only; use torch.no_grad() or torch.inference_mode() for tensors that require "
                    "gradients");
        TORCH_CHECK(!forward || !t->_fw_grad(0).defined(), op,
                    " is inference-only; it has no forward-mode derivative");
    }
}

int32_t dtype_of(const char* op, const Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case at::kFloat: return FX_F32;
        case at::kBFloat16: return FX_BF16;
        case at::kHalf: return FX_F16;
        default: TORCH_CHECK(false, op, ": ", name, " must be float32, bfloat16 or float16");
    }
}

// Byte range [first, last) a tensor's elements lie in.
std::pair<const char*, const char*> extent(const Tensor& t) {
    const char* first = static_cast<const char*>(t.data_ptr());
    int64_t last = 0;
    for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
    return {first, first + (last + 1) * t.element_size()};
}

bool overlaps(const Tensor& a, const Tensor& b) {
    if (a.numel() == 0 || b.numel() == 0) return false;
    const auto x = extent(a), y = extent(b);
    return x.first < y.second && y.first < x.second;
}

// A one-dimensional contiguous int64 tensor; `size` < 0: any size.
void index_vector(const char* op, const Tensor& t, const char* name, int64_t size) {
    TORCH_CHECK(t.dim() == 1 && t.scalar_type() == at::kLong && t.is_contiguous(), op, ": ", name,
                " must be a contiguous one-dimensional int64 tensor");
    TORCH_CHECK(size < 0 || t.size(0) == size, op, ": ", name, " has ", std::to_string(t.size(0)),
                " entries, expected ", std::to_string(size));
}

int64_t stride_of(const Tensor& t, int64_t d) { return t.size(d) == 1 ? 0 : t.stride(d); }

// The pools: [pages, kv_heads, page_size, head_dim] of one layer, or with
// `layers` a dimension of layers before it.
fx_pages pages_of(const char* op, const Tensor& keys, const Tensor& values, bool layers, bool written) {
    const int64_t rank = layers ? 5 : 4;
    TORCH_CHECK(keys.dim() == rank && values.dim() == rank, op, ": key_pages and value_pages must be ",
                layers ? "[layers, pages, kv_heads, page_size, head_dim]" : "[pages, kv_heads, page_size, head_dim]");
    TORCH_CHECK(keys.sizes() == values.sizes(), op, ": key_pages and value_pages must have the same shape");
    TORCH_CHECK(keys.scalar_type() == values.scalar_type(), op, ": key_pages and value_pages must have the same type");
    TORCH_CHECK(keys.numel() > 0, op, ": key_pages must be non-empty");
    same_device(op, keys, {&values});
    no_grad(op, {&keys, &values});
    fx_pages p{};
    p.dtype = dtype_of(op, keys, "key_pages");
    const int64_t d = layers ? 1 : 0;
    p.layers = layers ? keys.size(0) : 1;
    p.pages = keys.size(d);
    p.kv_heads = keys.size(d + 1);
    p.page_size = keys.size(d + 2);
    p.head_dim = keys.size(d + 3);
    TORCH_CHECK(p.head_dim % 8 == 0 && p.head_dim <= 256, op, ": head_dim must be a multiple of 8 up to 256");
    TORCH_CHECK(keys.stride(d + 3) == 1 && values.stride(d + 3) == 1, op,
                ": the elements of a key or value row must be contiguous");
    for (int64_t i = 0; i < 4; ++i) {
        p.key_strides[i] = d + i - 1 < 0 ? 0 : stride_of(keys, d + i - 1);
        p.value_strides[i] = d + i - 1 < 0 ? 0 : stride_of(values, d + i - 1);
    }
    if (written)
        for (int64_t i = 0; i < rank; ++i)
            TORCH_CHECK((keys.size(i) == 1 || keys.stride(i) > 0) && (values.size(i) == 1 || values.stride(i) > 0), op,
                        ": pages that are written must not be expanded");
    if (!keys.is_meta()) {
        TORCH_CHECK(keys.data_ptr() != values.data_ptr(), op, ": key_pages and value_pages must not be the same memory");
        p.keys = keys.data_ptr();
        p.values = values.data_ptr();
    }
    return p;
}

struct Table {
    int32_t* data;
    int64_t sequences, columns, stride;
};

Table table_of(const char* op, const Tensor& t) {
    TORCH_CHECK(t.dim() == 2 && t.scalar_type() == at::kInt, op, ": page_table must be a two-dimensional int32 tensor");
    TORCH_CHECK(t.numel() > 0, op, ": page_table must be non-empty");
    TORCH_CHECK(t.size(1) == 1 || t.stride(1) == 1, op, ": the entries of a page_table row must be contiguous");
    TORCH_CHECK(t.size(0) == 1 || t.stride(0) >= t.size(1), op, ": page_table rows must not overlap");
    return {t.is_meta() ? nullptr : static_cast<int32_t*>(t.data_ptr()), t.size(0), t.size(1),
            t.size(0) == 1 ? t.size(1) : t.stride(0)};
}

void counts_of(const char* op, const Tensor& t, int64_t pages) {
    TORCH_CHECK(t.dim() == 1 && t.scalar_type() == at::kInt && t.is_contiguous(), op,
                ": page_counts must be a contiguous one-dimensional int32 tensor");
    TORCH_CHECK(pages < 0 || t.size(0) == pages, op, ": page_counts must have one entry per page");
    TORCH_CHECK(t.size(0) > 0, op, ": page_counts must be non-empty");
}

// ---------------------------------------------------- packed QKV into pages

Tensor paged_qkv_rope_cache(const Tensor& packed, const Tensor& cos, const Tensor& sin, const Tensor& key_pages,
                            const Tensor& value_pages, const Tensor& page_table, const Tensor& positions,
                            const Optional& sequences) {
    const char* op = "flux::paged_qkv_rope_cache";
    const fx_pages p = pages_of(op, key_pages, value_pages, false, true);
    TORCH_CHECK(packed.dim() == 2 && packed.size(1) % p.head_dim == 0 &&
                    packed.size(1) / p.head_dim > 2 * p.kv_heads,
                op, ": packed_qkv must be [tokens, (query_heads + 2 kv_heads) * head_dim]");
    TORCH_CHECK(packed.stride(1) == 1, op, ": the elements of a packed_qkv row must be contiguous");
    TORCH_CHECK(packed.scalar_type() == at::kFloat || packed.scalar_type() == key_pages.scalar_type(), op,
                ": packed_qkv must be float32 or have the pages' type");
    const int32_t dtype = dtype_of(op, packed, "packed_qkv");
    TORCH_CHECK(cos.dim() == 2 && cos.sizes() == sin.sizes() && cos.size(0) > 0 && cos.size(1) == p.head_dim, op,
                ": cos and sin must be tables [positions, head_dim]");
    TORCH_CHECK(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat && cos.stride(1) == 1 &&
                    sin.stride(1) == 1,
                op, ": cos and sin must be float32 with contiguous rows");
    const Table table = table_of(op, page_table);
    const int64_t tokens = packed.size(0), heads = packed.size(1) / p.head_dim - 2 * p.kv_heads;
    index_vector(op, positions, "positions", tokens);
    if (sequences.has_value())
        index_vector(op, *sequences, "sequences", tokens);
    else
        TORCH_CHECK(tokens == table.sequences, op, ": without sequences there is one token per page_table row");
    same_device(op, key_pages, {&packed, &cos, &sin, &page_table, &positions});
    if (sequences.has_value()) same_device(op, key_pages, {&*sequences});
    no_grad(op, {&packed, &cos, &sin});
    if (!packed.is_meta())
        TORCH_CHECK(!overlaps(packed, key_pages) && !overlaps(packed, value_pages), op,
                    ": packed_qkv must not alias the pages");
    const c10::OptionalDeviceGuard guard(at::device_of(packed));
    Tensor query = at::empty({tokens, heads, 1, p.head_dim}, packed.options());
    if (!launches(op, packed) || tokens == 0) return query;
    check(fx_paged_qkv_rope_cache(packed.data_ptr(), dtype, packed.stride(0), tokens, heads, cos.data_ptr<float>(),
                                  cos.stride(0), sin.data_ptr<float>(), sin.stride(0), cos.size(0), &p, table.data,
                                  table.sequences, table.columns, table.stride, positions.data_ptr<int64_t>(),
                                  sequences.has_value() ? sequences->data_ptr<int64_t>() : nullptr, query.data_ptr(),
                                  stream_of(packed)));
    return query;
}

// ----------------------------------------------------------- paged attention

struct Attend {
    fx_pages pages;
    Table table;
    int32_t dtype;
};

Attend attend_arguments(const char* op, const Tensor& query, const Tensor& key_pages, const Tensor& value_pages,
                        const Tensor& page_table, const Tensor& lengths, double scale) {
    Attend a{pages_of(op, key_pages, value_pages, false, false), {}, 0};
    TORCH_CHECK(query.dim() == 4 && query.size(2) == 1, op, ": query must be [batch, query_heads, 1, head_dim]");
    if (query.size(0) > 0) a.table = table_of(op, page_table);
    TORCH_CHECK(query.size(3) == a.pages.head_dim, op, ": cache head dimension must match query");
    TORCH_CHECK(query.stride(3) == 1, op, ": the elements of a query row must be contiguous");
    TORCH_CHECK(query.size(1) > 0 && query.size(1) % a.pages.kv_heads == 0, op,
                ": query heads must be divisible by KV heads");
    TORCH_CHECK(query.scalar_type() == at::kFloat || query.scalar_type() == key_pages.scalar_type(), op,
                ": query must be float32 or have the pages' type");
    a.dtype = dtype_of(op, query, "query");
    TORCH_CHECK(query.size(0) == 0 || query.size(0) == a.table.sequences, op,
                ": page_table must have one row per sequence of the query");
    index_vector(op, lengths, "lengths", query.size(0));
    TORCH_CHECK(std::isfinite(scale) && std::isfinite(static_cast<float>(scale)), op,
                ": scale must be a finite FP32 value");
    same_device(op, query, {&key_pages, &page_table, &lengths});
    no_grad(op, {&query});
    return a;
}

void attend_launch(const Attend& a, const Tensor& query, const Tensor& lengths, double scale, const Tensor& output,
                   float* workspace, int64_t floats) {
    const int64_t strides[2] = {query.stride(0), query.stride(1)};
    check(fx_paged_gqa_decode_attention(query.data_ptr(), a.dtype, strides, query.size(0), query.size(1), &a.pages,
                                        a.table.data, a.table.columns, a.table.stride, lengths.data_ptr<int64_t>(),
                                        static_cast<float>(scale), output.data_ptr(), workspace, floats,
                                        stream_of(query)));
}

Tensor paged_gqa_decode_attention(const Tensor& query, const Tensor& key_pages, const Tensor& value_pages,
                                  const Tensor& page_table, const Tensor& lengths, double scale) {
    const char* op = "flux::paged_gqa_decode_attention";
    const Attend a = attend_arguments(op, query, key_pages, value_pages, page_table, lengths, scale);
    const c10::OptionalDeviceGuard guard(at::device_of(query));
    Tensor output = at::empty(query.sizes(), query.options());
    if (!launches(op, query) || query.size(0) == 0) return output;
    const Workspace<float> workspace(
        fx_paged_gqa_decode_attention_workspace_floats(query.size(1), a.pages.kv_heads, a.pages.head_dim));
    attend_launch(a, query, lengths, scale, output, workspace.data(), workspace.size);
    return output;
}

Tensor paged_gqa_decode_attention_out(const Tensor& query, const Tensor& key_pages, const Tensor& value_pages,
                                      const Tensor& page_table, const Tensor& lengths, double scale,
                                      const Tensor& output, const Tensor& workspace) {
    const char* op = "flux::paged_gqa_decode_attention_out";
    const Attend a = attend_arguments(op, query, key_pages, value_pages, page_table, lengths, scale);
    TORCH_CHECK(output.sizes() == query.sizes(), op, ": output shape must match query");
    TORCH_CHECK(output.scalar_type() == query.scalar_type() && output.is_contiguous(), op,
                ": output must be contiguous and have the query's type");
    const int64_t floats =
        fx_paged_gqa_decode_attention_workspace_floats(query.size(1), a.pages.kv_heads, a.pages.head_dim);
    TORCH_CHECK(workspace.scalar_type() == at::kFloat && workspace.is_contiguous() && workspace.numel() >= floats, op,
                ": workspace must be contiguous float32 with at least ", std::to_string(floats), " elements");
    same_device(op, query, {&output, &workspace});
    no_grad(op, {&output, &workspace});
    if (!launches(op, query) || query.size(0) == 0) return output;
    TORCH_CHECK(!overlaps(output, workspace), op, ": output and workspace must not alias");
    for (const Tensor* t : {&query, &key_pages, &value_pages, &page_table, &lengths})
        TORCH_CHECK(!overlaps(output, *t) && !overlaps(workspace, *t), op, ": outputs must not alias inputs");
    const c10::OptionalDeviceGuard guard(at::device_of(query));
    attend_launch(a, query, lengths, scale, output, workspace.data_ptr<float>(), workspace.numel());
    return output;
}

// ------------------------------------------------------------ page operations

void cache_pages_copy(const Tensor& key_pages, const Tensor& value_pages, const Tensor& source,
                      const Tensor& destination) {
    const char* op = "flux::cache_pages_copy";
    const fx_pages p = pages_of(op, key_pages, value_pages, true, true);
    index_vector(op, source, "source", -1);
    index_vector(op, destination, "destination", source.size(0));
    same_device(op, key_pages, {&source, &destination});
    if (!launches(op, key_pages) || source.size(0) == 0) return;
    const c10::OptionalDeviceGuard guard(at::device_of(key_pages));
    check(fx_cache_pages_copy(&p, source.data_ptr<int64_t>(), destination.data_ptr<int64_t>(), source.size(0),
                              stream_of(key_pages)));
}

Tensor cache_sequences_reserve(const Tensor& page_table, const Tensor& lengths, const Tensor& page_counts,
                               const Tensor& sequences, const Tensor& rows, int64_t page_size) {
    const char* op = "flux::cache_sequences_reserve";
    const Table table = table_of(op, page_table);
    counts_of(op, page_counts, -1);
    index_vector(op, lengths, "lengths", table.sequences);
    index_vector(op, sequences, "sequences", -1);
    index_vector(op, rows, "rows", sequences.size(0));
    TORCH_CHECK(page_size > 0, op, ": page_size must be positive");
    same_device(op, page_table, {&lengths, &page_counts, &sequences, &rows});
    const c10::OptionalDeviceGuard guard(at::device_of(page_table));
    const int64_t count = sequences.size(0), pages = page_counts.size(0);
    Tensor status = at::empty({count}, page_counts.options());
    if (!launches(op, page_table) || count == 0) return status;
    const Workspace<int32_t> workspace(count + pages);
    check(fx_cache_sequences_reserve(table.data, table.sequences, table.columns, table.stride,
                                     lengths.data_ptr<int64_t>(), page_counts.data_ptr<int32_t>(), pages, page_size,
                                     sequences.data_ptr<int64_t>(), rows.data_ptr<int64_t>(), count,
                                     status.data_ptr<int32_t>(), workspace.data(),
                                     stream_of(page_table)));
    return status;
}

Tensor cache_sequences_fork(const Tensor& key_pages, const Tensor& value_pages, const Tensor& page_table,
                            const Tensor& lengths, const Tensor& page_counts, const Tensor& parents,
                            const Tensor& children) {
    const char* op = "flux::cache_sequences_fork";
    const fx_pages p = pages_of(op, key_pages, value_pages, true, true);
    const Table table = table_of(op, page_table);
    counts_of(op, page_counts, p.pages);
    index_vector(op, lengths, "lengths", table.sequences);
    index_vector(op, parents, "parents", -1);
    index_vector(op, children, "children", parents.size(0));
    same_device(op, key_pages, {&page_table, &lengths, &page_counts, &parents, &children});
    const c10::OptionalDeviceGuard guard(at::device_of(key_pages));
    const int64_t count = parents.size(0);
    Tensor status = at::empty({count}, page_counts.options());
    if (!launches(op, key_pages) || count == 0) return status;
    const Workspace<int32_t> workspace(3 * count);
    check(fx_cache_sequences_fork(&p, table.data, table.sequences, table.columns, table.stride,
                                  lengths.data_ptr<int64_t>(), page_counts.data_ptr<int32_t>(),
                                  parents.data_ptr<int64_t>(), children.data_ptr<int64_t>(), count,
                                  status.data_ptr<int32_t>(), workspace.data(), stream_of(key_pages)));
    return status;
}

void cache_sequences_free(const Tensor& page_table, const Tensor& lengths, const Tensor& page_counts,
                          const Tensor& sequences) {
    const char* op = "flux::cache_sequences_free";
    const Table table = table_of(op, page_table);
    counts_of(op, page_counts, -1);
    index_vector(op, lengths, "lengths", table.sequences);
    index_vector(op, sequences, "sequences", -1);
    same_device(op, page_table, {&lengths, &page_counts, &sequences});
    if (!launches(op, page_table) || sequences.size(0) == 0) return;
    const c10::OptionalDeviceGuard guard(at::device_of(page_table));
    check(fx_cache_sequences_free(table.data, table.sequences, table.columns, table.stride,
                                  lengths.data_ptr<int64_t>(), page_counts.data_ptr<int32_t>(), page_counts.size(0),
                                  sequences.data_ptr<int64_t>(), sequences.size(0), stream_of(page_table)));
}

Tensor cache_pages_compact(const Tensor& key_pages, const Tensor& value_pages, const Tensor& page_table,
                           const Tensor& page_counts) {
    const char* op = "flux::cache_pages_compact";
    const fx_pages p = pages_of(op, key_pages, value_pages, true, true);
    const Table table = table_of(op, page_table);
    counts_of(op, page_counts, p.pages);
    same_device(op, key_pages, {&page_table, &page_counts});
    const c10::OptionalDeviceGuard guard(at::device_of(key_pages));
    Tensor used = at::empty({}, page_counts.options());
    if (!launches(op, key_pages)) return used;
    const Workspace<int32_t> workspace(2 * p.pages + 1);
    check(fx_cache_pages_compact(&p, table.data, table.sequences, table.columns, table.stride,
                                 page_counts.data_ptr<int32_t>(), used.data_ptr<int32_t>(),
                                 workspace.data(), stream_of(key_pages)));
    return used;
}

// ------------------------------------------------------------------- logits

// A [width], [1, width] or [rows, width] tensor; its row stride (0 broadcasts).
int64_t row_stride(const char* op, const Tensor& t, const char* name, int64_t rows, int64_t width) {
    const int64_t d = t.dim();
    TORCH_CHECK((d == 1 || (d == 2 && (t.size(0) == 1 || t.size(0) == rows))) && t.size(d - 1) == width, op, ": ", name,
                " must be [", std::to_string(width), "] or [", std::to_string(rows), ", ", std::to_string(width), "]");
    TORCH_CHECK(width == 1 || t.stride(d - 1) == 1, op, ": ", name, " rows must be contiguous");
    return d == 1 || t.size(0) == 1 ? 0 : t.stride(0);
}

void logits_launch(const char* op, const Tensor& logits, const Optional& tokens, const Optional& prompt_lengths,
                   const Optional& lengths, const Optional& penalties, const Optional& bias, const Optional& allowed,
                   Tensor& output, bool checked_output) {
    TORCH_CHECK(logits.dim() == 2 && logits.size(1) > 0, op, ": logits must be [rows, vocabulary]");
    const int32_t dtype = dtype_of(op, logits, "logits");
    const int64_t rows = logits.size(0), vocab = logits.size(1);
    TORCH_CHECK(vocab == 1 || logits.stride(1) == 1, op, ": the elements of a logits row must be contiguous");
    TORCH_CHECK(rows <= 1 || logits.stride(0) >= vocab, op, ": logits rows must not overlap");
    no_grad(op, {&logits});
    const bool history = tokens.has_value();
    TORCH_CHECK(history == prompt_lengths.has_value() && history == lengths.has_value() &&
                    history == penalties.has_value(),
                op, ": tokens, prompt_lengths, lengths and penalties go together");
    if (history) {
        TORCH_CHECK(tokens->dim() == 2 && tokens->size(0) == rows && tokens->scalar_type() == at::kLong, op,
                    ": tokens must be int64 [rows, history]");
        TORCH_CHECK(tokens->size(1) <= 1 || tokens->stride(1) == 1, op, ": the tokens of a row must be contiguous");
        index_vector(op, *prompt_lengths, "prompt_lengths", rows);
        index_vector(op, *lengths, "lengths", rows);
        TORCH_CHECK(penalties->dim() == 2 && penalties->size(0) == rows && penalties->size(1) == 3 &&
                        penalties->scalar_type() == at::kFloat && penalties->is_contiguous(),
                    op, ": penalties must be contiguous float32 [rows, 3]");
        same_device(op, logits, {&*tokens, &*prompt_lengths, &*lengths, &*penalties});
        no_grad(op, {&*penalties});
    }
    int64_t bias_stride = 0, allowed_stride = 0;
    if (bias.has_value()) {
        TORCH_CHECK(bias->scalar_type() == at::kFloat, op, ": bias must be float32");
        bias_stride = row_stride(op, *bias, "bias", rows, vocab);
        same_device(op, logits, {&*bias});
        no_grad(op, {&*bias});
    }
    if (allowed.has_value()) {
        TORCH_CHECK(allowed->scalar_type() == at::kInt, op, ": allowed must be int32 words of 32 token bits");
        allowed_stride = row_stride(op, *allowed, "allowed", rows, (vocab + 31) / 32);
        same_device(op, logits, {&*allowed});
    }
    if (checked_output) {
        TORCH_CHECK(output.sizes() == logits.sizes() && output.scalar_type() == logits.scalar_type(), op,
                    ": output must have the shape and type of logits");
        TORCH_CHECK((vocab == 1 || output.stride(1) == 1) && (rows <= 1 || output.stride(0) >= vocab), op,
                    ": output rows must be contiguous and must not overlap");
        same_device(op, logits, {&output});
        no_grad(op, {&output});
        if (!output.is_meta()) {
            const bool in_place = output.data_ptr() == logits.data_ptr() && output.strides() == logits.strides();
            TORCH_CHECK(in_place || !overlaps(output, logits), op,
                        ": output must be logits itself or must not alias it");
            for (const Optional* t : {&tokens, &prompt_lengths, &lengths, &penalties, &bias, &allowed})
                TORCH_CHECK(!t->has_value() || !overlaps(output, **t), op, ": output must not alias the other inputs");
        }
    }
    const c10::OptionalDeviceGuard guard(at::device_of(logits));
    if (!checked_output) output = at::empty(logits.sizes(), logits.options());
    if (!launches(op, logits) || rows == 0) return;
    const bool counted = history && tokens->size(1) > 0;
    check(fx_logits_process(logits.data_ptr(), dtype, rows, vocab, logits.stride(0),
                            counted ? tokens->data_ptr<int64_t>() : nullptr, counted ? tokens->size(1) : 0,
                            counted ? tokens->stride(0) : 0, counted ? prompt_lengths->data_ptr<int64_t>() : nullptr,
                            counted ? lengths->data_ptr<int64_t>() : nullptr,
                            counted ? penalties->data_ptr<float>() : nullptr,
                            bias.has_value() ? bias->data_ptr<float>() : nullptr, bias_stride,
                            allowed.has_value() ? allowed->data_ptr<int32_t>() : nullptr, allowed_stride,
                            output.data_ptr(), output.stride(0), stream_of(logits)));
}

Tensor logits_process(const Tensor& logits, const Optional& tokens, const Optional& prompt_lengths,
                      const Optional& lengths, const Optional& penalties, const Optional& bias,
                      const Optional& allowed) {
    Tensor output;
    logits_launch("flux::logits_process", logits, tokens, prompt_lengths, lengths, penalties, bias, allowed, output,
                  false);
    return output;
}

Tensor logits_process_out(const Tensor& logits, const Optional& tokens, const Optional& prompt_lengths,
                          const Optional& lengths, const Optional& penalties, const Optional& bias,
                          const Optional& allowed, const Tensor& output) {
    Tensor out = output;
    logits_launch("flux::logits_process_out", logits, tokens, prompt_lengths, lengths, penalties, bias, allowed, out,
                  true);
    return out;
}

// --------------------------------------------------- sizes that are symbols

bool symbolic(std::initializer_list<const Tensor*> tensors) {
    for (const Tensor* t : tensors)
        if (t->unsafeGetTensorImpl()->has_symbolic_sizes_strides()) return true;
    return false;
}

const Tensor* given(const Optional& t, const Tensor& otherwise) { return t.has_value() ? &*t : &otherwise; }

void symbolic_pages(const char* op, const Tensor& keys, const Tensor& values, int64_t rank) {
    TORCH_CHECK(keys.dim() == rank && values.dim() == rank, op, ": key_pages and value_pages must be ",
                rank == 5 ? "[layers, pages, kv_heads, page_size, head_dim]" : "[pages, kv_heads, page_size, head_dim]");
    for (int64_t d = 0; d < rank; ++d)
        TORCH_SYM_CHECK(keys.sym_size(d).sym_eq(values.sym_size(d)), op,
                        ": key_pages and value_pages must have the same shape");
    TORCH_CHECK(keys.scalar_type() == values.scalar_type(), op, ": key_pages and value_pages must have the same type");
    dtype_of(op, keys, "key_pages");
    const c10::SymInt dim = keys.sym_size(rank - 1);
    TORCH_SYM_CHECK((dim % 8).sym_eq(0).sym_and(dim.sym_le(256)), op, ": head_dim must be a multiple of 8 up to 256");
    no_grad(op, {&keys, &values});
}

void symbolic_table(const char* op, const Tensor& t) {
    TORCH_CHECK(t.dim() == 2 && t.scalar_type() == at::kInt, op, ": page_table must be a two-dimensional int32 tensor");
}

void symbolic_vector(const char* op, const Tensor& t, const char* name, const c10::SymInt& size) {
    TORCH_CHECK(t.dim() == 1 && t.scalar_type() == at::kLong, op, ": ", name,
                " must be a contiguous one-dimensional int64 tensor");
    TORCH_SYM_CHECK(t.sym_size(0).sym_eq(size), op, ": ", name, " has another number of entries than expected");
}

void symbolic_state(const char* op, const Tensor& table, const Tensor& counts) {
    symbolic_table(op, table);
    TORCH_CHECK(counts.dim() == 1 && counts.scalar_type() == at::kInt, op,
                ": page_counts must be a contiguous one-dimensional int32 tensor");
}

Tensor paged_qkv_rope_cache_meta(const Tensor& packed, const Tensor& cos, const Tensor& sin, const Tensor& keys,
                                 const Tensor& values, const Tensor& table, const Tensor& positions,
                                 const Optional& sequences) {
    const char* op = "flux::paged_qkv_rope_cache";
    if (!symbolic({&packed, &cos, &sin, &keys, &values, &table, &positions, given(sequences, positions)}))
        return paged_qkv_rope_cache(packed, cos, sin, keys, values, table, positions, sequences);
    symbolic_pages(op, keys, values, 4);
    symbolic_table(op, table);
    const char* shape = ": packed_qkv must be [tokens, (query_heads + 2 kv_heads) * head_dim]";
    TORCH_CHECK(packed.dim() == 2, op, shape);
    const c10::SymInt tokens = packed.sym_size(0), width = packed.sym_size(1), dim = keys.sym_size(3);
    TORCH_SYM_CHECK((width % dim).sym_eq(0), op, shape);
    const c10::SymInt heads = width / dim - keys.sym_size(1) * 2;
    TORCH_SYM_CHECK(heads.sym_gt(0), op, shape);
    TORCH_CHECK(packed.scalar_type() == at::kFloat || packed.scalar_type() == keys.scalar_type(), op,
                ": packed_qkv must be float32 or have the pages' type");
    TORCH_CHECK(cos.dim() == 2 && sin.dim() == 2, op, ": cos and sin must be tables [positions, head_dim]");
    TORCH_SYM_CHECK(cos.sym_size(0).sym_eq(sin.sym_size(0)).sym_and(cos.sym_size(1).sym_eq(dim))
                        .sym_and(sin.sym_size(1).sym_eq(dim)),
                    op, ": cos and sin must be tables [positions, head_dim]");
    TORCH_CHECK(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat, op,
                ": cos and sin must be float32 with contiguous rows");
    symbolic_vector(op, positions, "positions", tokens);
    if (sequences.has_value())
        symbolic_vector(op, *sequences, "sequences", tokens);
    else
        TORCH_SYM_CHECK(tokens.sym_eq(table.sym_size(0)), op, ": without sequences there is one token per page_table row");
    same_device(op, keys, {&values, &packed, &cos, &sin, &table, &positions, given(sequences, positions)});
    no_grad(op, {&packed, &cos, &sin});
    return at::empty_symint({tokens, heads, 1, dim}, packed.options());
}

void symbolic_attend(const char* op, const Tensor& query, const Tensor& keys, const Tensor& values, const Tensor& table,
                     const Tensor& lengths, double scale) {
    symbolic_pages(op, keys, values, 4);
    TORCH_CHECK(query.dim() == 4, op, ": query must be [batch, query_heads, 1, head_dim]");
    TORCH_SYM_CHECK(query.sym_size(2).sym_eq(1), op, ": query must be [batch, query_heads, 1, head_dim]");
    symbolic_table(op, table);
    TORCH_SYM_CHECK(query.sym_size(3).sym_eq(keys.sym_size(3)), op, ": cache head dimension must match query");
    TORCH_SYM_CHECK((query.sym_size(1) % keys.sym_size(1)).sym_eq(0), op, ": query heads must be divisible by KV heads");
    TORCH_CHECK(query.scalar_type() == at::kFloat || query.scalar_type() == keys.scalar_type(), op,
                ": query must be float32 or have the pages' type");
    TORCH_SYM_CHECK(query.sym_size(0).sym_eq(table.sym_size(0)), op,
                    ": page_table must have one row per sequence of the query");
    symbolic_vector(op, lengths, "lengths", query.sym_size(0));
    TORCH_CHECK(std::isfinite(scale) && std::isfinite(static_cast<float>(scale)), op,
                ": scale must be a finite FP32 value");
    same_device(op, query, {&keys, &values, &table, &lengths});
    no_grad(op, {&query});
}

Tensor paged_gqa_decode_attention_meta(const Tensor& query, const Tensor& keys, const Tensor& values,
                                       const Tensor& table, const Tensor& lengths, double scale) {
    if (!symbolic({&query, &keys, &values, &table, &lengths}))
        return paged_gqa_decode_attention(query, keys, values, table, lengths, scale);
    symbolic_attend("flux::paged_gqa_decode_attention", query, keys, values, table, lengths, scale);
    return at::empty_symint(query.sym_sizes(), query.options());
}

void symbolic_output(const char* op, const Tensor& output, const Tensor& like, const char* message) {
    TORCH_CHECK(output.dim() == like.dim() && output.scalar_type() == like.scalar_type(), op, message);
    for (int64_t d = 0; d < like.dim(); ++d)
        TORCH_SYM_CHECK(output.sym_size(d).sym_eq(like.sym_size(d)), op, message);
    same_device(op, like, {&output});
    no_grad(op, {&output});
}

Tensor paged_gqa_decode_attention_out_meta(const Tensor& query, const Tensor& keys, const Tensor& values,
                                           const Tensor& table, const Tensor& lengths, double scale,
                                           const Tensor& output, const Tensor& workspace) {
    const char* op = "flux::paged_gqa_decode_attention_out";
    if (!symbolic({&query, &keys, &values, &table, &lengths, &output, &workspace}))
        return paged_gqa_decode_attention_out(query, keys, values, table, lengths, scale, output, workspace);
    symbolic_attend(op, query, keys, values, table, lengths, scale);
    symbolic_output(op, output, query, ": output must have the shape and type of query");
    TORCH_CHECK(workspace.scalar_type() == at::kFloat, op, ": workspace must be contiguous float32");
    return output;
}

void cache_pages_copy_meta(const Tensor& keys, const Tensor& values, const Tensor& source, const Tensor& destination) {
    const char* op = "flux::cache_pages_copy";
    if (!symbolic({&keys, &values, &source, &destination})) return cache_pages_copy(keys, values, source, destination);
    symbolic_pages(op, keys, values, 5);
    TORCH_CHECK(source.dim() == 1, op, ": source must be a contiguous one-dimensional int64 tensor");
    symbolic_vector(op, source, "source", source.sym_size(0));
    symbolic_vector(op, destination, "destination", source.sym_size(0));
    same_device(op, keys, {&values, &source, &destination});
}

Tensor cache_sequences_reserve_meta(const Tensor& table, const Tensor& lengths, const Tensor& counts,
                                    const Tensor& sequences, const Tensor& rows, int64_t page_size) {
    const char* op = "flux::cache_sequences_reserve";
    if (!symbolic({&table, &lengths, &counts, &sequences, &rows}))
        return cache_sequences_reserve(table, lengths, counts, sequences, rows, page_size);
    symbolic_state(op, table, counts);
    symbolic_vector(op, lengths, "lengths", table.sym_size(0));
    TORCH_CHECK(sequences.dim() == 1, op, ": sequences must be a contiguous one-dimensional int64 tensor");
    symbolic_vector(op, sequences, "sequences", sequences.sym_size(0));
    symbolic_vector(op, rows, "rows", sequences.sym_size(0));
    TORCH_CHECK(page_size > 0, op, ": page_size must be positive");
    same_device(op, table, {&lengths, &counts, &sequences, &rows});
    return at::empty_symint({sequences.sym_size(0)}, counts.options());
}

Tensor cache_sequences_fork_meta(const Tensor& keys, const Tensor& values, const Tensor& table, const Tensor& lengths,
                                 const Tensor& counts, const Tensor& parents, const Tensor& children) {
    const char* op = "flux::cache_sequences_fork";
    if (!symbolic({&keys, &values, &table, &lengths, &counts, &parents, &children}))
        return cache_sequences_fork(keys, values, table, lengths, counts, parents, children);
    symbolic_pages(op, keys, values, 5);
    symbolic_state(op, table, counts);
    TORCH_SYM_CHECK(counts.sym_size(0).sym_eq(keys.sym_size(1)), op, ": page_counts must have one entry per page");
    symbolic_vector(op, lengths, "lengths", table.sym_size(0));
    TORCH_CHECK(parents.dim() == 1, op, ": parents must be a contiguous one-dimensional int64 tensor");
    symbolic_vector(op, parents, "parents", parents.sym_size(0));
    symbolic_vector(op, children, "children", parents.sym_size(0));
    same_device(op, keys, {&values, &table, &lengths, &counts, &parents, &children});
    return at::empty_symint({parents.sym_size(0)}, counts.options());
}

void cache_sequences_free_meta(const Tensor& table, const Tensor& lengths, const Tensor& counts,
                               const Tensor& sequences) {
    const char* op = "flux::cache_sequences_free";
    if (!symbolic({&table, &lengths, &counts, &sequences}))
        return cache_sequences_free(table, lengths, counts, sequences);
    symbolic_state(op, table, counts);
    symbolic_vector(op, lengths, "lengths", table.sym_size(0));
    TORCH_CHECK(sequences.dim() == 1, op, ": sequences must be a contiguous one-dimensional int64 tensor");
    symbolic_vector(op, sequences, "sequences", sequences.sym_size(0));
    same_device(op, table, {&lengths, &counts, &sequences});
}

Tensor cache_pages_compact_meta(const Tensor& keys, const Tensor& values, const Tensor& table, const Tensor& counts) {
    const char* op = "flux::cache_pages_compact";
    if (!symbolic({&keys, &values, &table, &counts})) return cache_pages_compact(keys, values, table, counts);
    symbolic_pages(op, keys, values, 5);
    symbolic_state(op, table, counts);
    TORCH_SYM_CHECK(counts.sym_size(0).sym_eq(keys.sym_size(1)), op, ": page_counts must have one entry per page");
    same_device(op, keys, {&values, &table, &counts});
    return at::empty({}, counts.options());
}

// [width], [1, width] or [rows, width]
void symbolic_row(const char* op, const Tensor& t, const char* name, const c10::SymInt& rows, const c10::SymInt& width) {
    TORCH_CHECK(t.dim() == 1 || t.dim() == 2, op, ": ", name, " must be one row or one row per row of logits");
    c10::SymBool fits = t.sym_size(t.dim() - 1).sym_eq(width);
    if (t.dim() == 2) fits = fits.sym_and(t.sym_size(0).sym_eq(1).sym_or(t.sym_size(0).sym_eq(rows)));
    TORCH_SYM_CHECK(fits, op, ": ", name, " must be one row or one row per row of logits, as wide as they are");
}

bool symbolic_logits(const char* op, const Tensor& logits, const Optional& tokens, const Optional& prompt_lengths,
                     const Optional& lengths, const Optional& penalties, const Optional& bias, const Optional& allowed,
                     const Tensor& output) {
    if (!symbolic({&logits, &output, given(tokens, logits), given(prompt_lengths, logits), given(lengths, logits),
                   given(penalties, logits), given(bias, logits), given(allowed, logits)}))
        return false;
    TORCH_CHECK(logits.dim() == 2, op, ": logits must be [rows, vocabulary]");
    dtype_of(op, logits, "logits");
    const c10::SymInt rows = logits.sym_size(0), vocab = logits.sym_size(1);
    const bool history = tokens.has_value();
    TORCH_CHECK(history == prompt_lengths.has_value() && history == lengths.has_value() &&
                    history == penalties.has_value(),
                op, ": tokens, prompt_lengths, lengths and penalties go together");
    if (history) {
        TORCH_CHECK(tokens->dim() == 2 && tokens->scalar_type() == at::kLong, op, ": tokens must be int64 [rows, history]");
        TORCH_SYM_CHECK(tokens->sym_size(0).sym_eq(rows), op, ": tokens must be int64 [rows, history]");
        symbolic_vector(op, *prompt_lengths, "prompt_lengths", rows);
        symbolic_vector(op, *lengths, "lengths", rows);
        TORCH_CHECK(penalties->dim() == 2 && penalties->scalar_type() == at::kFloat, op,
                    ": penalties must be contiguous float32 [rows, 3]");
        TORCH_SYM_CHECK(penalties->sym_size(0).sym_eq(rows).sym_and(penalties->sym_size(1).sym_eq(3)), op,
                        ": penalties must be contiguous float32 [rows, 3]");
        no_grad(op, {&*penalties});
    }
    if (bias.has_value()) {
        TORCH_CHECK(bias->scalar_type() == at::kFloat, op, ": bias must be float32");
        symbolic_row(op, *bias, "bias", rows, vocab);
        no_grad(op, {&*bias});
    }
    if (allowed.has_value()) {
        TORCH_CHECK(allowed->scalar_type() == at::kInt, op, ": allowed must be int32 words of 32 token bits");
        symbolic_row(op, *allowed, "allowed", rows, (vocab + 31) / 32);
    }
    same_device(op, logits, {given(tokens, logits), given(prompt_lengths, logits), given(lengths, logits),
                             given(penalties, logits), given(bias, logits), given(allowed, logits)});
    no_grad(op, {&logits});
    return true;
}

Tensor logits_process_meta(const Tensor& logits, const Optional& tokens, const Optional& prompt_lengths,
                           const Optional& lengths, const Optional& penalties, const Optional& bias,
                           const Optional& allowed) {
    if (!symbolic_logits("flux::logits_process", logits, tokens, prompt_lengths, lengths, penalties, bias, allowed,
                         logits))
        return logits_process(logits, tokens, prompt_lengths, lengths, penalties, bias, allowed);
    return at::empty_symint(logits.sym_sizes(), logits.options());
}

Tensor logits_process_out_meta(const Tensor& logits, const Optional& tokens, const Optional& prompt_lengths,
                               const Optional& lengths, const Optional& penalties, const Optional& bias,
                               const Optional& allowed, const Tensor& output) {
    const char* op = "flux::logits_process_out";
    if (!symbolic_logits(op, logits, tokens, prompt_lengths, lengths, penalties, bias, allowed, output))
        return logits_process_out(logits, tokens, prompt_lengths, lengths, penalties, bias, allowed, output);
    symbolic_output(op, output, logits, ": output must have the shape and type of logits");
    return output;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(flux, m) {
    m.def("paged_qkv_rope_cache(Tensor packed_qkv, Tensor cos, Tensor sin, Tensor(a!) key_pages, "
          "Tensor(b!) value_pages, Tensor page_table, Tensor positions, Tensor? sequences=None) -> Tensor");
    m.def("paged_gqa_decode_attention(Tensor query, Tensor key_pages, Tensor value_pages, Tensor page_table, "
          "Tensor lengths, float scale) -> Tensor");
    m.def("paged_gqa_decode_attention_out(Tensor query, Tensor key_pages, Tensor value_pages, Tensor page_table, "
          "Tensor lengths, float scale, Tensor(a!) output, Tensor(b!) workspace) -> Tensor(a!)");
    m.def("cache_pages_copy(Tensor(a!) key_pages, Tensor(b!) value_pages, Tensor source, Tensor destination) -> ()");
    m.def("cache_sequences_reserve(Tensor(a!) page_table, Tensor lengths, Tensor(b!) page_counts, Tensor sequences, "
          "Tensor rows, int page_size) -> Tensor");
    m.def("cache_sequences_fork(Tensor(a!) key_pages, Tensor(b!) value_pages, Tensor(c!) page_table, "
          "Tensor(d!) lengths, Tensor(e!) page_counts, Tensor parents, Tensor children) -> Tensor");
    m.def("cache_sequences_free(Tensor(a!) page_table, Tensor(b!) lengths, Tensor(c!) page_counts, "
          "Tensor sequences) -> ()");
    m.def("cache_pages_compact(Tensor(a!) key_pages, Tensor(b!) value_pages, Tensor(c!) page_table, "
          "Tensor(d!) page_counts) -> Tensor");
    m.def("logits_process(Tensor logits, Tensor? tokens=None, Tensor? prompt_lengths=None, Tensor? lengths=None, "
          "Tensor? penalties=None, Tensor? bias=None, Tensor? allowed=None) -> Tensor");
    m.def("logits_process_out(Tensor logits, Tensor? tokens, Tensor? prompt_lengths, Tensor? lengths, "
          "Tensor? penalties, Tensor? bias, Tensor? allowed, Tensor(a!) output) -> Tensor(a!)");
}

#define FLUX_SERVING_OPERATORS(m, form) \
    m.impl("paged_qkv_rope_cache", TORCH_FN(paged_qkv_rope_cache##form)); \
    m.impl("paged_gqa_decode_attention", TORCH_FN(paged_gqa_decode_attention##form)); \
    m.impl("paged_gqa_decode_attention_out", TORCH_FN(paged_gqa_decode_attention_out##form)); \
    m.impl("cache_pages_copy", TORCH_FN(cache_pages_copy##form)); \
    m.impl("cache_sequences_reserve", TORCH_FN(cache_sequences_reserve##form)); \
    m.impl("cache_sequences_fork", TORCH_FN(cache_sequences_fork##form)); \
    m.impl("cache_sequences_free", TORCH_FN(cache_sequences_free##form)); \
    m.impl("cache_pages_compact", TORCH_FN(cache_pages_compact##form)); \
    m.impl("logits_process", TORCH_FN(logits_process##form)); \
    m.impl("logits_process_out", TORCH_FN(logits_process_out##form))

TORCH_LIBRARY_IMPL(flux, CUDA, m) { FLUX_SERVING_OPERATORS(m, ); }
TORCH_LIBRARY_IMPL(flux, CPU, m) { FLUX_SERVING_OPERATORS(m, ); }
TORCH_LIBRARY_IMPL(flux, Meta, m) { FLUX_SERVING_OPERATORS(m, _meta); }
