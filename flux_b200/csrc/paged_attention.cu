// One-token attention over a paged cache: the entry point, and the merge of
// units that span CTAs.
//
//   out[b, h] = sum_r p_r V[r] / sum_r p_r,   p_r = exp(s_r - max s),   s_r = scale q[b, h] . K[r]
//
// over the visible rows r of sequence b (r < length, page not a hole).  The
// sums are taken in one pass: a state (m, l, o) holds the maximum of the
// scores seen, the sum of exp(s - m) and the sum of exp(s - m) V; a new
// maximum m' rescales l and o by exp(m - m'), and two states join the same way.
#include "paged_attention.cuh"

#include <cmath>
#include <cstdint>

namespace fx {
namespace {

// A running softmax state: maximum, sum, N output dims.
template <int N>
struct State {
    float m = -INFINITY, l = 0.0f, o[N] = {};

    // Joins K pieces that have been loaded.
    template <int K>
    __device__ __forceinline__ void join(const float (&pm)[K], const float (&pl)[K], const float (&po)[K][N]) {
        float top = m;
#pragma unroll
        for (int u = 0; u < K; ++u) top = fmaxf(top, pm[u]);
        const float base = top == -INFINITY ? 0.0f : top, keep = exp2f(m - base);
        l *= keep;
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] *= keep;
        m = top;
#pragma unroll
        for (int u = 0; u < K; ++u) {
            const float f = exp2f(pm[u] - base);
            l = fmaf(pl[u], f, l);
#pragma unroll
            for (int e = 0; e < N; ++e) o[e] = fmaf(po[u][e], f, o[e]);
        }
    }
};

// Piece j of the unit that starts in attention CTA i, head h of the group.
__device__ __forceinline__ const float* piece_of(const PagedAttend& a, int i, int j, int h) {
    const int64_t slot = j == 0 ? 2 * static_cast<int64_t>(i) + 1 : 2 * (static_cast<int64_t>(i) + j);
    return paged_pieces(a) + (slot * a.group + h) * (a.dim + 2);
}

// Many units, a few pieces each: one warp per (attention CTA, head of the
// group) joins the unit that starts in that CTA and ends in a later one: piece
// 1 of the first, then piece 0 of each up to the last.  Waiting for memory is
// the whole cost, so four pieces are loaded at a time.
template <typename T, int N>
__global__ void __launch_bounds__(256) paged_merge_kernel(const __grid_constant__ PagedAttend a, int ctas) {
    grid_dependency_wait();
    constexpr int K = 4;
    const int task = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int h = task / ctas, i = task - h * ctas;
    if (h >= a.group) return;
    State<N> s;
    float pm[K], pl[K], po[K][N];
    const auto load = [&](int j0, int end) {
#pragma unroll
        for (int u = 0; u < K; ++u) {
            const bool any = j0 + u < end;
            const float* p = piece_of(a, i, j0 + u, h);
            pm[u] = any ? p[0] : -INFINITY;
            pl[u] = any ? p[1] : 0.0f;
#pragma unroll
            for (int e = 0; e < N; ++e) po[u][e] = any && lane + 32 * e < a.dim ? p[2 + lane + 32 * e] : 0.0f;
        }
    };
    load(0, ctas - i);  // before it is known how many there are; what lies in the others does not count
    const int* d = reinterpret_cast<const int*>(a.workspace) + i * kPagedDescriptor;
    const int b = d[0], head = d[1], count = d[2] - i + 1;
    if (d[3] == 0) return;
#pragma unroll
    for (int u = 0; u < K; ++u)
        if (u >= count) {
            pm[u] = -INFINITY;
            pl[u] = 0.0f;
#pragma unroll
            for (int e = 0; e < N; ++e) po[u][e] = 0.0f;
        }
    s.join(pm, pl, po);
    for (int j0 = K; j0 < count; j0 += K) {
        load(j0, count);
        s.join(pm, pl, po);
    }
    T* out = static_cast<T*>(a.out) + (static_cast<int64_t>(b) * a.heads + head * a.group + h) * a.dim;
#pragma unroll
    for (int e = 0; e < N; ++e)
        if (lane + 32 * e < a.dim) out[lane + 32 * e] = from_float<T>(s.l == 0.0f ? 0.0f : s.o[e] / s.l);
}

// Few units, many pieces each: one CTA per (unit, head of the group).  A thread
// takes one output dim of every 1024 / span-th piece, eight at a time.
template <typename T>
__global__ void __launch_bounds__(1024) paged_merge_long_kernel(const __grid_constant__ PagedAttend a) {
    grid_dependency_wait();
    constexpr int K = 8;
    __shared__ float part_m[32], part_l[32], part_o[1024];
    const int tid = threadIdx.x, unit = blockIdx.x, h = blockIdx.y;
    const int* place = reinterpret_cast<const int*>(a.workspace) + kPagedMaxGrid * kPagedDescriptor + 2 * unit;
    const int i = place[0], count = place[1] - i + 1;
    if (place[1] < 0) return;  // one CTA had the whole unit
    const int span = (a.dim + 31) / 32 * 32, parts = 1024 / span;
    const int part = tid / span, e = tid % span;
    State<1> s;
    if (part < parts)
        for (int j0 = part; j0 < count; j0 += K * parts) {
            float pm[K], pl[K], po[K][1];
#pragma unroll
            for (int u = 0; u < K; ++u) {
                const bool any = j0 + u * parts < count;
                const float* p = piece_of(a, i, j0 + u * parts, h);
                pm[u] = any ? p[0] : -INFINITY;
                pl[u] = any ? p[1] : 0.0f;
                po[u][0] = any && e < a.dim ? p[2 + e] : 0.0f;
            }
            s.join(pm, pl, po);
        }
    part_o[tid] = s.o[0];
    if (e == 0 && part < parts) {
        part_m[part] = s.m;
        part_l[part] = s.l;
    }
    __syncthreads();
    if (tid >= a.dim) return;
    State<1> all;
    for (int p = 0; p < parts; p += 4) {
        float pm[4], pl[4], po[4][1];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            pm[u] = p + u < parts ? part_m[p + u] : -INFINITY;
            pl[u] = p + u < parts ? part_l[p + u] : 0.0f;
            po[u][0] = p + u < parts ? part_o[(p + u) * span + tid] : 0.0f;
        }
        all.join(pm, pl, po);
    }
    static_cast<T*>(a.out)[(static_cast<int64_t>(unit) * a.group + h) * a.dim + tid] =
        from_float<T>(all.l == 0.0f ? 0.0f : all.o[0] / all.l);
}

}  // namespace

template <typename T>
fx_status launch_paged_merge(const PagedAttend& a, int ctas, cudaStream_t stream) {
    const char* what = "launching the paged attention merge";
    const int64_t units = static_cast<int64_t>(a.batch) * a.kv_heads;
    if (units <= kPagedUnits && units * 8 <= ctas)  // eight pieces each, or more
        return launch_dependent(paged_merge_long_kernel<T>, dim3(static_cast<unsigned>(units), a.group), dim3(1024), 0,
                                stream, what, a);
    const dim3 grid((ctas * a.group + 7) / 8), block(256);
    if (a.dim <= 64) return launch_dependent(paged_merge_kernel<T, 2>, grid, block, 0, stream, what, a, ctas);
    if (a.dim <= 128) return launch_dependent(paged_merge_kernel<T, 4>, grid, block, 0, stream, what, a, ctas);
    return launch_dependent(paged_merge_kernel<T, 8>, grid, block, 0, stream, what, a, ctas);
}
template fx_status launch_paged_merge<float>(const PagedAttend&, int, cudaStream_t);
template fx_status launch_paged_merge<__nv_bfloat16>(const PagedAttend&, int, cudaStream_t);
template fx_status launch_paged_merge<__half>(const PagedAttend&, int, cudaStream_t);

}  // namespace fx

using namespace fx;

// Query heads of a unit: all that read a KV head, up to 16; of more the largest
// part that divides them, and each part reads the rows again.  64 x 4096 rows of
// one KV head of 64 BF16 dims take 26 us with 16 query heads, 35 with 32 (two
// parts) and 45 with 48, but 146 with 17 (17 parts of one head) and 545 with 71.
static int64_t heads_together(int64_t group) {
    int64_t heads = group < kPagedMaxGroup ? group : kPagedMaxGroup;
    while (group % heads != 0) --heads;
    return heads;
}

extern "C" int64_t fx_paged_gqa_decode_attention_workspace_floats(int64_t query_heads, int64_t kv_heads,
                                                                  int64_t head_dim) {
    if (query_heads <= 0 || kv_heads <= 0 || head_dim <= 0) return 0;
    const int64_t group = heads_together((query_heads - 1) / kv_heads + 1);
    // Two pieces of (max, sum, output) per CTA; the limits of the call keep the product small.
    if (head_dim > kPagedMaxDim) return INT64_MAX;
    return kPagedMaxGrid * (kPagedDescriptor + 2 * group * (head_dim + 2)) + 2 * kPagedUnits;
}

extern "C" fx_status fx_paged_gqa_decode_attention(const void* query, int32_t dtype, const int64_t* query_strides2,
                                                   int64_t batch, int64_t query_heads, const fx_pages* pages,
                                                   const int32_t* page_table, int64_t table_columns,
                                                   int64_t table_stride, const int64_t* lengths, float scale,
                                                   void* output, float* workspace, int64_t workspace_floats,
                                                   void* stream) {
    const char* op = "fx_paged_gqa_decode_attention";
    fx_status st = check_pages(op, pages, false);
    if (st != FX_OK) return st;
    FX_REQUIRE(batch >= 0, "fx_paged_gqa_decode_attention: batch must not be negative");
    if (batch == 0) return FX_OK;
    st = check_table(op, page_table, batch, table_columns, table_stride, pages->page_size);
    if (st != FX_OK) return st;
    FX_REQUIRE(query && query_strides2 && lengths && output && workspace,
               "fx_paged_gqa_decode_attention: null pointer");
    FX_REQUIRE(dtype == pages->dtype || dtype == FX_F32,
               "fx_paged_gqa_decode_attention: query must be float32 or have the pages' type");
    FX_REQUIRE(query_heads > 0 && query_heads % pages->kv_heads == 0,
               "fx_paged_gqa_decode_attention: query heads must be divisible by KV heads");
    FX_REQUIRE(query_heads <= 65535, "fx_paged_gqa_decode_attention: at most 65535 query heads");
    FX_REQUIRE(std::isfinite(scale * kLog2e), "fx_paged_gqa_decode_attention: scale must be finite");
    FX_REQUIRE(workspace_floats >=
                   fx_paged_gqa_decode_attention_workspace_floats(query_heads, pages->kv_heads, pages->head_dim),
               "fx_paged_gqa_decode_attention: workspace is too small");
    // Tiles of at least 32 rows are numbered in 31 bits.
    const int64_t group = query_heads / pages->kv_heads, share = group / heads_together(group);
    FX_REQUIRE(batch * pages->kv_heads * share <= INT_MAX / ((table_columns * pages->page_size + 31) / 32),
               "fx_paged_gqa_decode_attention: batch * kv_heads * table rows is too large");
    PagedAttend a{};
    a.q = query;
    a.q_batch = query_strides2[0];
    a.q_head = query_strides2[1];
    a.keys = pages->keys;
    a.values = pages->values;
    for (int i = 0; i < 3; ++i) {
        a.ks[i] = pages->key_strides[i + 1];
        a.vs[i] = pages->value_strides[i + 1];
    }
    a.table = page_table;
    a.table_stride = table_stride;
    a.lengths = lengths;
    a.out = output;
    a.workspace = workspace;
    a.scale = scale * kLog2e;
    a.pages = static_cast<int>(pages->pages);
    a.batch = static_cast<int>(batch);
    a.heads = static_cast<int>(query_heads);
    a.kv_heads = static_cast<int>(pages->kv_heads * share);
    a.group = static_cast<int>(group / share);
    a.dim = static_cast<int>(pages->head_dim);
    a.capacity = static_cast<int>(table_columns * pages->page_size);
    a.page_size = FastDivide::by(pages->page_size);
    a.per_head = FastDivide::by(a.dim);
    a.share = FastDivide::by(share);
    a.alike = true;
    for (int i = 0; i < 3; ++i) a.alike = a.alike && a.ks[i] == a.vs[i];
    int device = 0, sms = 0;
    FX_CUDA_TRY(cudaGetDevice(&device), "looking up the device");
    FX_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device), "counting the SMs");
    a.whole = paged_whole(a, sms);
    cudaStream_t s = as_stream(stream);
    if (dtype == FX_BF16) return launch_paged_bf16(a, sms, s);
    if (dtype == FX_F16) return launch_paged_f16(a, sms, s);
    if (pages->dtype == FX_F32) return a.group <= 4 ? launch_paged_f32(a, sms, s) : launch_paged_f32_wide(a, sms, s);
    return pages->dtype == FX_BF16 ? launch_paged_f32_on_bf16(a, sms, s) : launch_paged_f32_on_f16(a, sms, s);
}
