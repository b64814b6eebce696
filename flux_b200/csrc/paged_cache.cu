// The paged key/value cache: packed QKV rows into pages, and the management
// of pages (copy, reserve, fork, free, compact).  Nothing here waits for the
// GPU: what the host cannot know (lengths, free pages, how much is to be
// moved) is decided by a one-CTA planning kernel, and the kernel that moves
// the data reads the plan.
#include "paged.cuh"

#include <algorithm>
#include <cstdint>
#include <string>

namespace fx {

namespace {

fx_status refuse(const char* op, const char* what) {
    set_error(std::string(op) + ": " + what);
    return FX_ERR_INVALID;
}

}  // namespace

fx_status check_pages(const char* op, const fx_pages* p, bool blocks) {
    if (p == nullptr || p->keys == nullptr || p->values == nullptr) return refuse(op, "null pointer");
    if (p->dtype != FX_F32 && p->dtype != FX_BF16 && p->dtype != FX_F16) return refuse(op, "unknown page type");
    if (p->layers < 1 || p->pages < 1 || p->kv_heads < 1 || p->page_size < 1 || p->head_dim < 1)
        return refuse(op, "page sizes must be positive");
    if (p->head_dim % 8 != 0 || p->head_dim > kPagedMaxDim)
        return refuse(op, "head_dim must be a multiple of 8 up to 256");
    if (p->page_size > kPagedMaxPageSize || p->pages > INT_MAX || p->kv_heads > 65535)
        return refuse(op, "too many pages, heads or rows of a page");
    const int64_t size = dtype_size(p->dtype);
    if (reinterpret_cast<uintptr_t>(p->keys) % 16 != 0 || reinterpret_cast<uintptr_t>(p->values) % 16 != 0)
        return refuse(op, "pages must start on 16-byte boundaries");
    for (int i = 0; i < 4; ++i)
        if (p->key_strides[i] * size % 16 != 0 || p->value_strides[i] * size % 16 != 0)
            return refuse(op, "page strides must be multiples of 16 bytes");
    if (blocks && (!pages_are_blocks(*p, p->key_strides) || !pages_are_blocks(*p, p->value_strides)))
        return refuse(op, "each page must be one contiguous block");
    return FX_OK;
}

fx_status check_table(const char* op, const int32_t* table, int64_t sequences, int64_t columns, int64_t stride,
                      int64_t page_size) {
    if (table == nullptr) return refuse(op, "null pointer");
    if (sequences < 1 || columns < 1 || stride < columns) return refuse(op, "page table sizes must be positive");
    if (sequences > INT_MAX || columns > INT_MAX / page_size)
        return refuse(op, "a sequence can have at most 2^31 - 1 rows");
    return FX_OK;
}

namespace {

// ------------------------------------------------ packed QKV -> RoPE -> pages

struct WriteArgs {
    const void* packed;
    int64_t packed_stride, tokens, query_heads, kv_heads, dim;
    const float* cos;
    const float* sin;
    int64_t cos_stride, sin_stride, rope_rows;
    void* keys;
    void* values;
    int64_t ks[3], vs[3];  // page, head, row
    int64_t pages;
    FastDivide page_size;
    const int32_t* table;
    int64_t sequences, columns, table_stride;
    const int64_t* positions;
    const int64_t* owners;
    void* query;
    FastDivide per_token, pieces;  // threads per token, pieces of half a row
    int span;                      // heads of a thread
};

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack { T v[N]; };

__device__ __forceinline__ float2 pair_of(const float* x) { return make_float2(x[0], x[1]); }
__device__ __forceinline__ float2 pair_of(const __nv_bfloat16* x) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(x));
}
__device__ __forceinline__ float2 pair_of(const __half* x) {
    return __half22float2(*reinterpret_cast<const __half2*>(x));
}
__device__ __forceinline__ void store_pair(float* to, float2 x) { to[0] = x.x; to[1] = x.y; }
__device__ __forceinline__ void store_pair(__nv_bfloat16* to, float2 x) {
    *reinterpret_cast<__nv_bfloat162*>(to) = __float22bfloat162_rn(x);
}
__device__ __forceinline__ void store_pair(__half* to, float2 x) {
    *reinterpret_cast<__half2*>(to) = __float22half2_rn(x);
}

// Products and sum rounded apart.  (The two-element instructions would halve
// their number, but the compiler joins a product and a sum of them.)
__device__ __forceinline__ float rotate(float x, float partner, float c, float s) {
    return __fadd_rn(__fmul_rn(x, c), __fmul_rn(partner, s));
}

// Memory bounds it: every packed element is read once and stored once, as
// pieces of N elements (16 bytes of the packed type where addresses allow).  A
// thread owns the same piece of both halves of a row, which rotate into one
// another, for `span` heads of one token, H of them at a time, so that it finds
// the token's page and loads its cos and sin once.  CTAs of 128 threads (four
// per SM at their 128 registers) come and go in smaller steps than those of 256
// (8191 tokens of 48 heads of 128 in BF16, 16 heads a thread: 39.8 us, 41.0).
constexpr int kWriteThreads = 128;

template <typename T, typename P, int N, int H>
__global__ void __launch_bounds__(kWriteThreads, 4) paged_write_kernel(const __grid_constant__ WriteArgs a) {
    grid_dependency_wait();
    const uint32_t i = blockIdx.x * static_cast<uint32_t>(kWriteThreads) + threadIdx.x;
    uint32_t rest, piece;
    const int64_t t = a.per_token.quotient(i, &rest);
    if (t >= a.tokens) return;
    const int begin = static_cast<int>(a.pieces.quotient(rest, &piece)) * a.span, d = piece * N;
    const int half = static_cast<int>(a.dim) / 2, rotated = static_cast<int>(a.query_heads + a.kv_heads);
    const int heads = rotated + static_cast<int>(a.kv_heads), end = min(begin + a.span, heads);
    const int64_t p = a.positions[t];
    const int64_t s = a.owners == nullptr ? t : a.owners[t];
    const T* x = static_cast<const T*>(a.packed) + t * a.packed_stride + d;
    Pack<T, N> lower[H], upper[H];
    const auto load = [&](int h0) {
#pragma unroll
        for (int j = 0; j < H; ++j)
            if (h0 + j < end) {
                lower[j] = *reinterpret_cast<const Pack<T, N>*>(x + (h0 + j) * a.dim);
                upper[j] = *reinterpret_cast<const Pack<T, N>*>(x + (h0 + j) * a.dim + half);
            }
    };
    load(begin);
    const bool turned = p >= 0 && p < a.rope_rows;
    Pack<float, N> c[2], n[2];
    if (begin < rotated && turned) {
        constexpr int M = N < 4 ? N : 4;
        const float* cos = a.cos + p * a.cos_stride + d;
        const float* sin = a.sin + p * a.sin_stride + d;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < N; e += M) {
                reinterpret_cast<Pack<float, M>*>(&c[u])[e / M] = *reinterpret_cast<const Pack<float, M>*>(cos + u * half + e);
                reinterpret_cast<Pack<float, M>*>(&n[u])[e / M] = *reinterpret_cast<const Pack<float, M>*>(sin + u * half + e);
            }
#pragma unroll
        for (int e = 0; e < N; ++e) n[0].v[e] = -n[0].v[e];  // the partner of the first half enters negated
    }
    int64_t page = -1;
    uint32_t slot = 0;
    if (turned && s >= 0 && s < a.sequences && p < a.columns * a.page_size.divisor) {
        page = a.table[s * a.table_stride + a.page_size.quotient(static_cast<uint32_t>(p), &slot)];
        if (page >= a.pages) page = -1;
    }
    const int64_t krow = page * a.ks[0] + slot * a.ks[2] + d, vrow = page * a.vs[0] + slot * a.vs[2] + d;
    T* query = static_cast<T*>(a.query) + t * a.query_heads * a.dim + d;
    for (int h0 = begin; h0 < end; h0 += H) {
        if (h0 > begin) load(h0);
#pragma unroll
        for (int j = 0; j < H; ++j) {
            const int h = h0 + j;
            if (h >= end) break;
            if constexpr (N == 1) {
                float y0 = to_float(lower[j].v[0]), y1 = to_float(upper[j].v[0]);
                if (h < rotated && turned) {
                    const float z = rotate(y0, y1, c[0].v[0], n[0].v[0]);
                    y1 = rotate(y1, y0, c[1].v[0], n[1].v[0]);
                    y0 = z;
                }
                if (h < a.query_heads) {
                    query[h * a.dim] = from_float<T>(turned ? y0 : 0.0f);
                    query[h * a.dim + half] = from_float<T>(turned ? y1 : 0.0f);
                } else if (page >= 0) {
                    P* row = h < rotated ? static_cast<P*>(a.keys) + krow + (h - a.query_heads) * a.ks[1]
                                         : static_cast<P*>(a.values) + vrow + (h - rotated) * a.vs[1];
                    row[0] = from_float<P>(y0);
                    row[half] = from_float<P>(y1);
                }
            } else {
                if (h < rotated) {
                    if (!turned) {  // no angle: a zero query, no key
                        if (h >= a.query_heads) continue;
                        Pack<T, N> zero;
#pragma unroll
                        for (int e = 0; e < N; ++e) zero.v[e] = from_float<T>(0.0f);
                        *reinterpret_cast<Pack<T, N>*>(query + h * a.dim) = zero;
                        *reinterpret_cast<Pack<T, N>*>(query + h * a.dim + half) = zero;
                        continue;
                    }
                    float2 z[2][N / 2];
#pragma unroll
                    for (int e = 0; e < N; e += 2) {
                        const float2 y0 = pair_of(&lower[j].v[e]), y1 = pair_of(&upper[j].v[e]);
                        z[0][e / 2] = make_float2(rotate(y0.x, y1.x, c[0].v[e], n[0].v[e]),
                                                  rotate(y0.y, y1.y, c[0].v[e + 1], n[0].v[e + 1]));
                        z[1][e / 2] = make_float2(rotate(y1.x, y0.x, c[1].v[e], n[1].v[e]),
                                                  rotate(y1.y, y0.y, c[1].v[e + 1], n[1].v[e + 1]));
                    }
                    if (h < a.query_heads) {
                        Pack<T, N> out[2];
#pragma unroll
                        for (int e = 0; e < N; e += 2) {
                            store_pair(&out[0].v[e], z[0][e / 2]);
                            store_pair(&out[1].v[e], z[1][e / 2]);
                        }
                        *reinterpret_cast<Pack<T, N>*>(query + h * a.dim) = out[0];
                        *reinterpret_cast<Pack<T, N>*>(query + h * a.dim + half) = out[1];
                    } else if (page >= 0) {
                        Pack<P, N> out[2];
#pragma unroll
                        for (int e = 0; e < N; e += 2) {
                            store_pair(&out[0].v[e], z[0][e / 2]);
                            store_pair(&out[1].v[e], z[1][e / 2]);
                        }
                        P* row = static_cast<P*>(a.keys) + krow + (h - a.query_heads) * a.ks[1];
                        *reinterpret_cast<Pack<P, N>*>(row) = out[0];
                        *reinterpret_cast<Pack<P, N>*>(row + half) = out[1];
                    }
                } else if (page >= 0) {
                    Pack<P, N> out[2];
#pragma unroll
                    for (int e = 0; e < N; e += 2) {
                        store_pair(&out[0].v[e], pair_of(&lower[j].v[e]));
                        store_pair(&out[1].v[e], pair_of(&upper[j].v[e]));
                    }
                    P* row = static_cast<P*>(a.values) + vrow + (h - rotated) * a.vs[1];
                    *reinterpret_cast<Pack<P, N>*>(row) = out[0];
                    *reinterpret_cast<Pack<P, N>*>(row + half) = out[1];
                }
            }
        }
    }
}

template <typename T, typename P, int N, int H>
fx_status launch_write_pieces(WriteArgs a, int span, cudaStream_t stream) {
    const int64_t heads = a.query_heads + 2 * a.kv_heads;
    a.span = span;
    a.pieces = FastDivide::by(a.dim / 2 / N);
    a.per_token = FastDivide::by((heads + span - 1) / span * (a.dim / 2 / N));
    const int64_t threads = a.tokens * a.per_token.divisor;
    const unsigned blocks = static_cast<unsigned>((threads + kWriteThreads - 1) / kWriteThreads);
    return launch_dependent(paged_write_kernel<T, P, N, H>, dim3(blocks), dim3(kWriteThreads), 0, stream,
                            "launching paged QKV/RoPE/cache update", a);
}

template <typename T, typename P>
fx_status launch_write(const WriteArgs& a, cudaStream_t stream) {
    constexpr int N = 16 / sizeof(T);
    const auto aligned = [](const void* p, int64_t stride_bytes) {
        return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride_bytes % 16 == 0;
    };
    const bool pieces = a.dim / 2 % N == 0 && a.dim / 2 >= N && aligned(a.packed, a.packed_stride * sizeof(T)) &&
                        aligned(a.cos, a.cos_stride * sizeof(float)) && aligned(a.sin, a.sin_stride * sizeof(float)) &&
                        aligned(a.query, 0);
    if (!pieces) return launch_write_pieces<T, P, 1, 1>(a, 1, stream);
    const int64_t heads = a.query_heads + 2 * a.kv_heads;
    // Heads of a thread: as few groups of them as still give every SM its four CTAs,
    // so that all threads are there at once; one head each where that leaves fewer
    // than four (8191 tokens of 48 heads of 128 in BF16: 37.0 us with all 48, 40.1
    // with 16, 63 with one; 1024 tokens 8.3, 10.3 with one).
    const int64_t groups = std::max<int64_t>(1, 148 * 4 * kWriteThreads / (a.tokens * (a.dim / 2 / N)));
    const int64_t span = (heads + groups - 1) / groups;
    if (span >= 4) return launch_write_pieces<T, P, N, 4>(a, static_cast<int>((span + 3) / 4 * 4), stream);
    return launch_write_pieces<T, P, N, 1>(a, 1, stream);
}

// ------------------------------------------------------------------- copies

// The pools as 16-byte words: word w of page p in layer l of pool i (0 keys,
// 1 values) is base[i] + l * layer[i] + p * page[i] + w.  A page of one layer
// and pool is moved in strips of 32 words, one per lane.
struct PoolWords {
    uint4* base[2];
    int64_t layer[2], page[2];
    int64_t layers, words, pages;
    FastDivide strips, per_pair;  // of a page in one layer and pool; of a pair in all of them
};

PoolWords pool_words(const fx_pages& p) {
    const int64_t size = dtype_size(p.dtype);
    PoolWords w{};
    w.base[0] = static_cast<uint4*>(p.keys);
    w.base[1] = static_cast<uint4*>(p.values);
    w.layer[0] = p.key_strides[0] * size / 16;
    w.layer[1] = p.value_strides[0] * size / 16;
    w.page[0] = p.key_strides[1] * size / 16;
    w.page[1] = p.value_strides[1] * size / 16;
    w.layers = p.layers;
    w.words = p.kv_heads * p.page_size * p.head_dim * size / 16;
    w.pages = p.pages;
    const int64_t strips = (w.words + 31) / 32;
    if (2 * strips * p.layers <= INT_MAX) {
        w.strips = FastDivide::by(strips);
        w.per_pair = FastDivide::by(2 * strips * p.layers);
    }
    return w;
}

constexpr int kCopyThreads = 256;
constexpr int kCopyBlocks = 1 << 20;  // with more work, CTAs stride
constexpr int kInFlight = 8;  // strips of a warp

// Copies pages that no pair both reads and writes.  Reading and writing HBM
// bounds it: each warp has 8 loads of 512 bytes in flight.  Many short CTAs that
// start one after another keep the whole GPU in one part of the list: 333 pages
// of 64 KB in 24 layers take 316 us (the measured copy rate), and 362 us with
// CTAs that stay and stride through it.  Where a page has a multiple of 8 strips a
// warp finds its place once for all 8 (a fork that copies one page of 30 layers
// 17.8 -> 16.5 us, 8000 pages of 32 KB in 4 layers 706 -> 653).
template <typename Index>
__device__ void move_pages(const PoolWords& pool, const Index* source, const Index* destination, uint32_t count,
                           uint32_t block, uint32_t blocks) {
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t total = static_cast<uint64_t>(count) * pool.per_pair.divisor;  // below 2^31 (checked by the host)
    const uint64_t step = static_cast<uint64_t>(blocks) * (kCopyThreads / 32) * kInFlight;
    for (uint64_t first = (static_cast<uint64_t>(block) * (kCopyThreads / 32) + threadIdx.x / 32) * kInFlight;
         first < total; first += step) {
        uint4 data[kInFlight];
        if (pool.strips.divisor % kInFlight == 0u) {  // all of one page in one place: `total` is a multiple too
            uint32_t rest, part;
            const uint32_t pair = pool.per_pair.quotient(static_cast<uint32_t>(first), &rest);
            const uint32_t place = pool.strips.quotient(rest, &part);
            const uint32_t k = place & 1u, w = part * 32 + lane;
            const int64_t s = source[pair], d = destination[pair];
            if (s < 0 || s >= pool.pages || d < 0 || d >= pool.pages || s == d) continue;
            uint4* base = pool.base[k] + (place >> 1) * pool.layer[k] + w;
            const uint4* from = base + s * pool.page[k];
            uint4* to = base + d * pool.page[k];
#pragma unroll
            for (int i = 0; i < kInFlight; ++i)
                if (w + 32 * i < pool.words) data[i] = __ldcs(from + 32 * i);
#pragma unroll
            for (int i = 0; i < kInFlight; ++i)
                if (w + 32 * i < pool.words) __stcs(to + 32 * i, data[i]);
            continue;
        }
        uint4* to[kInFlight];
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) {
            to[i] = nullptr;
            const uint32_t strip = static_cast<uint32_t>(first) + i;
            if (strip >= total) continue;
            uint32_t rest, part;
            const uint32_t pair = pool.per_pair.quotient(strip, &rest);
            const uint32_t place = pool.strips.quotient(rest, &part);
            const uint32_t k = place & 1u, w = part * 32 + lane;
            const int64_t s = source[pair], d = destination[pair];
            if (w >= pool.words || s < 0 || s >= pool.pages || d < 0 || d >= pool.pages || s == d) continue;
            uint4* base = pool.base[k] + (place >> 1) * pool.layer[k] + w;
            data[i] = __ldcs(base + s * pool.page[k]);
            to[i] = base + d * pool.page[k];
        }
#pragma unroll
        for (int i = 0; i < kInFlight; ++i)
            if (to[i] != nullptr) __stcs(to[i], data[i]);
    }
}

// One thread owns word w of every page of one layer and pool and walks the
// pairs in order: the result is that of copying pair after pair, whatever
// pages the list repeats.
__device__ void copy_in_order(const PoolWords& pool, const int64_t* source, const int64_t* destination,
                              int64_t count) {
    const int64_t columns = 2 * pool.layers * pool.words;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < columns;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int64_t w = i % pool.words, l = i / pool.words % pool.layers, k = i / (pool.words * pool.layers);
        uint4* base = pool.base[k] + l * pool.layer[k] + w;
        for (int64_t n = 0; n < count; ++n) {
            const int64_t from = source[n], to = destination[n];
            if (from < 0 || from >= pool.pages || to < 0 || to >= pool.pages) continue;
            base[to * pool.page[k]] = base[from * pool.page[k]];
        }
    }
}

// Every CTA looks for a page that is written twice, or written by one pair and
// read by another, with one bit per page; all come to the same answer.  Without
// one, the order of the pairs does not matter.
__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const __grid_constant__ PoolWords pool,
                                                            const int64_t* source, const int64_t* destination,
                                                            int64_t count, bool look) {
    grid_dependency_wait();
    extern __shared__ uint32_t written[];
    bool conflict = !look;
    if (look) {
        for (int64_t i = threadIdx.x; i < (pool.pages + 31) / 32; i += kCopyThreads) written[i] = 0u;
        __syncthreads();
        const auto moved = [&](int64_t s, int64_t d) {
            return s >= 0 && s < pool.pages && d >= 0 && d < pool.pages && s != d;
        };
#pragma unroll 4
        for (int64_t i = threadIdx.x; i < count; i += kCopyThreads) {
            const int64_t s = source[i], d = destination[i];
            if (moved(s, d)) conflict |= (atomicOr(&written[d >> 5], 1u << (d & 31)) >> (d & 31)) & 1u;
        }
        __syncthreads();
#pragma unroll 4
        for (int64_t i = threadIdx.x; i < count; i += kCopyThreads) {
            const int64_t s = source[i], d = destination[i];
            if (moved(s, d)) conflict |= (written[s >> 5] >> (s & 31)) & 1u;
        }
        conflict = __syncthreads_or(conflict);
    }
    if (conflict)
        copy_in_order(pool, source, destination, count);
    else
        move_pages(pool, source, destination, static_cast<uint32_t>(count), blockIdx.x, gridDim.x);
}

constexpr size_t kPlainShared = 40 * 1024;  // beside its static shared memory a kernel may use that much without being allowed more
constexpr int64_t kMaxLookPages = 1 << 20;  // a bit for each in the shared memory of copy_kernel (128 KB)

// `looked`: the bytes that a CTA goes through before it copies.  It then copies
// at least as many, in several rounds if need be, unless that would leave SMs
// idle: with one round each, 8000 pairs of 32 KB in 4 layers took 1633 us instead
// of 706, and 64000 in one layer 22.4 ms instead of 1.54.
unsigned copy_blocks(const PoolWords& pool, int64_t pairs, int64_t looked = 0) {
    const int64_t strips = pairs * 2 * pool.layers * ((pool.words + 31) / 32);
    const int64_t per_round = kCopyThreads / 32 * kInFlight;
    const int64_t all = (strips + per_round - 1) / per_round, rounds = looked / (2 * 512 * per_round) + 1;
    const int64_t blocks = std::max<int64_t>((all + rounds - 1) / rounds, std::min<int64_t>(all, 148 * 8));
    return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(blocks, kCopyBlocks)));
}

// Whether `pairs` pairs can be cut into strips that 31 bits number.
bool strips_fit(const PoolWords& pool, int64_t pairs) {
    return pool.strips.divisor != 0 && pairs <= INT_MAX / static_cast<int64_t>(pool.per_pair.divisor);
}

// ----------------------------------------------------------------- planning

constexpr int kPlanThreads = 1024;
constexpr int64_t kMaxSequences = 262144;  // three bits per sequence in the planner's shared memory (96 KB)
constexpr int64_t kMaxPages = 1 << 20;     // a scan over 1024 threads' needs stays below 2^31

// Exclusive prefix sum over the CTA's threads; *total gets the sum.
__device__ __forceinline__ int block_scan(int v, int* scratch, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int sum = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
    }
    __syncthreads();
    if (lane == 31) scratch[warp] = sum;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < kPlanThreads / 32; ++w) {
        const int n = scratch[w];
        before += w < warp ? n : 0;
        all += n;
    }
    *total = all;
    return before + sum - v;
}

// The counts of four pages from p on; pages behind the last are in use.
__device__ __forceinline__ int4 four_counts(const int32_t* counts, int64_t pages, int64_t p) {
    if (p + 4 <= pages && reinterpret_cast<uintptr_t>(counts) % 16 == 0)
        return *reinterpret_cast<const int4*>(counts + p);
    return make_int4(p < pages ? counts[p] : 1, p + 1 < pages ? counts[p + 1] : 1, p + 2 < pages ? counts[p + 2] : 1,
                     p + 3 < pages ? counts[p + 3] : 1);
}

// Writes the `wanted` lowest pages with count 0 to list, in order; returns how
// many there were.  Every thread of the CTA calls it, with the counts of its
// first four pages, which the caller loads as early as it can.
__device__ int lowest_free(const int32_t* counts, int64_t pages, int wanted, int32_t* list, int* scratch, int4 four) {
    int found = 0;
    for (int64_t base = 0; base < pages && found < wanted; base += 4 * kPlanThreads) {
        const int64_t p = base + 4 * threadIdx.x;
        if (base > 0) four = four_counts(counts, pages, p);
        const int free[4] = {four.x <= 0, four.y <= 0, four.z <= 0, four.w <= 0};
        int total = 0;
        int rank = found + block_scan(free[0] + free[1] + free[2] + free[3], scratch, &total);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (free[i]) {
                if (rank < wanted) list[rank] = static_cast<int32_t>(p + i);
                ++rank;
            }
        found += total;
    }
    __syncthreads();
    return min(found, wanted);
}

constexpr int kNearPages = 1024;  // free lists up to this long stay in shared memory

struct TableArgs {
    int32_t* table;
    int64_t sequences, columns, stride;
    int64_t* lengths;
    int32_t* counts;
    int64_t pages, page_size;
    FastDivide by_columns, by_page;  // a table has at most 2^31 - 1 rows
};

TableArgs table_args(int32_t* table, int64_t sequences, int64_t columns, int64_t stride, int64_t* lengths,
                     int32_t* counts, int64_t pages, int64_t page_size) {
    return {table, sequences, columns, stride, lengths, counts, pages, page_size,
            FastDivide::by(columns), FastDivide::by(page_size)};
}

// Entry k of the rows of a list of sequences: entry *e of the returned one.
__device__ __forceinline__ int64_t listed_entry(const TableArgs& t, int64_t k, int64_t* e) {
    if (k > INT_MAX) {
        *e = k % t.columns;
        return k / t.columns;
    }
    uint32_t rest;
    const uint32_t i = t.by_columns.quotient(static_cast<uint32_t>(k), &rest);
    *e = rest;
    return i;
}

// Pages that n rows take up.
__device__ __forceinline__ int64_t pages_of(const TableArgs& t, int64_t n) {
    uint32_t rest;
    const uint32_t full = t.by_page.quotient(static_cast<uint32_t>(n), &rest);
    return full + (rest != 0u ? 1 : 0);
}

__device__ __forceinline__ bool test_bit(const uint32_t* bits, int64_t i) { return (bits[i >> 5] >> (i & 31)) & 1u; }
__device__ __forceinline__ bool set_bit(uint32_t* bits, int64_t i) {
    return (atomicOr(&bits[i >> 5], 1u << (i & 31)) >> (i & 31)) & 1u;
}

// Rows of a sequence, clamped to its table.
__device__ __forceinline__ int64_t rows_of(const TableArgs& t, int64_t s) {
    const int64_t n = t.lengths[s];
    return n < 0 ? 0 : (n > t.columns * t.page_size ? t.columns * t.page_size : n);
}

// The plans are chains of dependent loads by one CTA, most of a microsecond a
// link: what does not depend on the chain (the counts, the tables of sequences
// that will be refused) is loaded beside it, many threads walk it side by side,
// and short free lists stay in shared memory.
constexpr int kTeam = 8;  // lanes that look at one sequence's entries together

__global__ void __launch_bounds__(kPlanThreads) reserve_kernel(TableArgs t, const int64_t* ids, const int64_t* rows,
                                                               int64_t count, int32_t* status, int32_t* workspace) {
    grid_dependency_wait();
    extern __shared__ uint32_t bits[];
    __shared__ int scratch[32];
    __shared__ int32_t near[kNearPages];
    const int64_t words = (t.sequences + 31) / 32;
    uint32_t* listed = bits;
    uint32_t* twice = bits + words;
    const int4 four = four_counts(t.counts, t.pages, 4 * threadIdx.x);
    for (int64_t i = threadIdx.x; i < 2 * words; i += kPlanThreads) bits[i] = 0u;
    __syncthreads();
    // The entries each sequence lacks; -1: refused.
    int32_t* need = workspace;
    const int lane = threadIdx.x % kTeam, team = threadIdx.x / kTeam, first = (threadIdx.x & 31) / kTeam * kTeam;
    const unsigned all = ((1u << kTeam) - 1u) << first;
    for (int64_t i = team; i < count; i += kPlanThreads / kTeam) {
        const int64_t s = ids[i];
        int n = -1;
        if (s >= 0 && s < t.sequences) {
            if (lane == 0 && set_bit(listed, s)) set_bit(twice, s);
            const int64_t have = rows_of(t, s), more = rows[i];
            if (more >= 0 && more <= t.columns * t.page_size - have) {
                n = 0;
                const int64_t last = pages_of(t, have + more);
                for (int64_t e = pages_of(t, have) + lane; e < last; e += kTeam) {
                    const int32_t p = t.table[s * t.stride + e];
                    n += p < 0 || p >= t.pages ? 1 : 0;
                }
#pragma unroll
                for (int o = kTeam / 2; o > 0; o >>= 1) n += __shfl_xor_sync(all, n, o);
            }
        }
        if (lane == 0) need[i] = n;
    }
    __syncthreads();
    // need[i] becomes the inclusive sum, capped at pages + 1 (enough to fail).
    int wanted = 0;
    for (int64_t base = 0; base < count; base += kPlanThreads) {
        const int64_t i = base + threadIdx.x;
        int n = i < count ? need[i] : -1;
        if (n >= 0 && test_bit(twice, ids[i])) n = -1;
        int total = 0;
        const int capped = n < 0 ? 0 : static_cast<int>(min(static_cast<int64_t>(n), t.pages + 1));
        const int before = block_scan(capped, scratch, &total);
        if (i < count) {
            const int64_t end = static_cast<int64_t>(wanted) + before + capped;
            status[i] = n < 0 ? FX_PAGES_REFUSED : (n == 0 ? FX_PAGES_OK : FX_PAGES_EXHAUSTED);
            need[i] = static_cast<int32_t>(end > t.pages ? t.pages + 1 : end);
        }
        const int64_t sum = static_cast<int64_t>(wanted) + total;
        wanted = static_cast<int>(sum > t.pages ? t.pages + 1 : sum);
    }
    if (wanted == 0) return;
    int32_t* list = wanted <= kNearPages ? near : workspace + count;
    const int found =
        lowest_free(t.counts, t.pages, min(wanted, static_cast<int>(t.pages)), list, scratch, four);
    for (int64_t i = team; i < count; i += kPlanThreads / kTeam) {
        if (status[i] != FX_PAGES_EXHAUSTED || need[i] > found) continue;
        const int64_t s = ids[i], have = rows_of(t, s);
        const int64_t last = pages_of(t, have + rows[i]);
        int next = i > 0 ? need[i - 1] : 0;
        for (int64_t e0 = pages_of(t, have); e0 < last; e0 += kTeam) {
            const int64_t e = e0 + lane;
            const int32_t p = e < last ? t.table[s * t.stride + e] : 0;
            const bool hole = e < last && (p < 0 || p >= t.pages);
            const unsigned holes = (__ballot_sync(all, hole) & all) >> first;
            if (hole) {
                const int32_t page = list[next + __popc(holes & ((1u << lane) - 1u))];
                t.table[s * t.stride + e] = page;
                t.counts[page] = 1;
            }
            next += __popc(holes);
        }
        __syncwarp(all);
        if (lane == 0) status[i] = FX_PAGES_OK;
    }
}

// copies: the partial pages' sources, then their destinations (-1: none), then
// a long free list.
__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(TableArgs t, const int64_t* parents,
                                                                 const int64_t* children, int64_t count,
                                                                 int32_t* status, int32_t* copies) {
    grid_dependency_wait();
    extern __shared__ uint32_t bits[];
    __shared__ int scratch[32];
    __shared__ int32_t near[kNearPages];
    const int64_t words = (t.sequences + 31) / 32;
    uint32_t* listed = bits;
    uint32_t* barred = bits + words;  // children listed twice or not empty
    uint32_t* parent = bits + 2 * words;
    const int4 four = four_counts(t.counts, t.pages, 4 * threadIdx.x);
    for (int64_t i = threadIdx.x; i < 3 * words; i += kPlanThreads) bits[i] = 0u;
    __syncthreads();
    for (int64_t i = threadIdx.x; i < count; i += kPlanThreads) {
        const int64_t p = parents[i], c = children[i];
        int32_t source = -1;
        if (c >= 0 && c < t.sequences && (set_bit(listed, c) || t.lengths[c] != 0)) set_bit(barred, c);
        if (p >= 0 && p < t.sequences) {
            set_bit(parent, p);
            uint32_t rest;
            const uint32_t full = t.by_page.quotient(static_cast<uint32_t>(rows_of(t, p)), &rest);
            if (rest != 0u) source = t.table[p * t.stride + full];
        }
        copies[i] = source >= 0 && source < t.pages ? source : -1;
    }
    // A child has to be empty: as many threads as there are for each look
    // through its row of the table.
    int shift = 10;  // 1024 threads
    while (shift > 3 && (count << shift) > kPlanThreads) --shift;
    for (int64_t i = threadIdx.x >> shift; i < count; i += kPlanThreads >> shift) {
        const int64_t c = children[i];
        if (c < 0 || c >= t.sequences) continue;
        const int32_t* row = t.table + c * t.stride;
        bool busy = false;
#pragma unroll 8
        for (int64_t e = threadIdx.x & ((1 << shift) - 1); e < t.columns; e += 1 << shift) {
            const int32_t page = row[e];
            busy |= page >= 0 && page < t.pages;
        }
        if (busy) set_bit(barred, c);
    }
    __syncthreads();
    int wanted = 0;
    for (int64_t base = 0; base < count; base += kPlanThreads) {
        const int64_t i = base + threadIdx.x;
        int need = 0;
        if (i < count) {
            const int64_t p = parents[i], c = children[i];
            const bool ok = p >= 0 && p < t.sequences && c >= 0 && c < t.sequences && !test_bit(barred, c) &&
                            !test_bit(parent, c);
            need = ok && copies[i] >= 0 ? 1 : 0;
            status[i] = ok ? FX_PAGES_OK : FX_PAGES_REFUSED;
            if (!ok) copies[i] = -1;
        }
        int total = 0;
        const int rank = wanted + block_scan(need, scratch, &total);
        if (i < count) copies[count + i] = need ? rank : -1;
        wanted += total;
    }
    if (wanted == 0) return;
    int32_t* list = wanted <= kNearPages ? near : copies + 2 * count;
    const int found = lowest_free(t.counts, t.pages, wanted, list, scratch, four);
    for (int64_t i = threadIdx.x; i < count; i += kPlanThreads) {
        const int32_t rank = copies[count + i];
        if (rank < 0) continue;
        if (rank < found) {
            copies[count + i] = list[rank];
        } else {  // no page left for this pair
            status[i] = FX_PAGES_EXHAUSTED;
            copies[i] = copies[count + i] = -1;
        }
    }
}

// The first `table_blocks` CTAs: table rows, counts and lengths of the children.
// The others: the partial pages.
__global__ void __launch_bounds__(kCopyThreads) fork_apply_kernel(const __grid_constant__ PoolWords pool, TableArgs t,
                                                                  const int64_t* parents, const int64_t* children,
                                                                  int64_t count, const int32_t* status,
                                                                  const int32_t* copies, uint32_t table_blocks) {
    grid_dependency_wait();
    if (blockIdx.x >= table_blocks) {
        move_pages(pool, copies, copies + count, static_cast<uint32_t>(count), blockIdx.x - table_blocks,
                   gridDim.x - table_blocks);
        return;
    }
    const int64_t total = count * t.columns;
    for (int64_t k = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; k < total;
         k += static_cast<int64_t>(table_blocks) * blockDim.x) {
        int64_t e;
        const int64_t i = listed_entry(t, k, &e);
        if (status[i] != FX_PAGES_OK) continue;
        const int64_t p = parents[i], c = children[i], n = rows_of(t, p);
        const int64_t full = t.by_page.quotient(static_cast<uint32_t>(n));
        int32_t page = -1;
        if (e < full) {
            page = t.table[p * t.stride + e];
            if (page >= 0 && page < t.pages) atomicAdd(&t.counts[page], 1);
        } else if (e == full) {
            page = copies[count + i];
            if (page >= 0) t.counts[page] = 1;
        }
        t.table[c * t.stride + e] = page;
        if (e == 0) t.lengths[c] = n;
    }
}

__global__ void free_kernel(TableArgs t, const int64_t* ids, int64_t count) {
    grid_dependency_wait();
    const int64_t total = count * t.columns;
    for (int64_t k = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; k < total;
         k += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        int64_t e;
        const int64_t s = ids[listed_entry(t, k, &e)];
        if (s < 0 || s >= t.sequences) continue;
        // The exchange hands each entry to one thread, so a sequence listed
        // twice is not counted down twice.
        const int32_t page = atomicExch(&t.table[s * t.stride + e], -1);
        if (page >= 0 && page < t.pages) atomicSub(&t.counts[page], 1);
        if (e == 0) t.lengths[s] = 0;
    }
}

// workspace[0] gets the number of moves, the next `pages` words their sources
// in order; place, behind them, the free pages below `used` in order (the
// moves' destinations), and from `used` on where each page went.
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(int32_t* counts, int64_t pages, int32_t* used_out,
                                                                    int32_t* workspace) {
    grid_dependency_wait();
    __shared__ int scratch[32];
    int mine = 0, used = 0;
    for (int64_t p = 4 * threadIdx.x; p < pages; p += 4 * kPlanThreads) {
        const int4 four = four_counts(counts, pages, p);
        const int64_t left = pages - p;  // what four_counts adds behind the last page does not count
        mine += (four.x > 0) + (four.y > 0 && left > 1) + (four.z > 0 && left > 2) + (four.w > 0 && left > 3);
    }
    block_scan(mine, scratch, &used);
    int32_t* source = workspace + 1;
    int32_t* place = workspace + 1 + pages;
    int holes = 0, moves = 0;
    for (int64_t base = 0; base < pages; base += 4 * kPlanThreads) {
        const int64_t p = base + 4 * threadIdx.x;
        const int4 four = p < pages ? four_counts(counts, pages, p) : make_int4(1, 1, 1, 1);
        const int n[4] = {four.x, four.y, four.z, four.w};
        bool hole[4], move[4];
        int packed = 0;  // holes below, moves above 16 bits: at most 4096 of each
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            hole[i] = p + i < used && n[i] <= 0;
            move[i] = p + i < pages && p + i >= used && n[i] > 0;
            packed += (hole[i] ? 1 : 0) + (move[i] ? 1 << 16 : 0);
        }
        int total = 0;
        const int before = block_scan(packed, scratch, &total);
        int to = holes + (before & 0xffff), from = moves + (before >> 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (hole[i]) place[to++] = static_cast<int32_t>(p + i);
            if (move[i]) source[from++] = static_cast<int32_t>(p + i);
            if (p + i >= used && p + i < pages) place[p + i] = static_cast<int32_t>(p + i);
        }
        holes += total & 0xffff;
        moves += total >> 16;
    }
    __syncthreads();
    for (int64_t k = threadIdx.x; k < moves; k += kPlanThreads) {
        const int32_t from = source[k], to = place[k];
        place[from] = to;
        counts[to] = counts[from];
        counts[from] = 0;
    }
    if (threadIdx.x == 0) {
        workspace[0] = moves;
        *used_out = used;
    }
}

// The first `table_blocks` CTAs rewrite the table entries that name moved pages,
// the others move them (no page is both read and written).
__global__ void __launch_bounds__(kCopyThreads) compact_apply_kernel(const __grid_constant__ PoolWords pool,
                                                                     TableArgs t, const int32_t* used,
                                                                     const int32_t* workspace, uint32_t table_blocks) {
    grid_dependency_wait();
    const int32_t* source = workspace + 1;
    const int32_t* place = workspace + 1 + pool.pages;
    if (blockIdx.x >= table_blocks) {
        // The k-th source goes to the k-th hole, which place lists from the start.
        move_pages(pool, source, place, static_cast<uint32_t>(workspace[0]), blockIdx.x - table_blocks,
                   gridDim.x - table_blocks);
        return;
    }
    const int64_t first = *used;
    const int64_t threads = static_cast<int64_t>(table_blocks) * blockDim.x;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < t.sequences * t.columns;
         i += threads) {
        int64_t e;
        int32_t* entry = t.table + listed_entry(t, i, &e) * t.stride;
        entry += e;
        if (*entry >= first && *entry < t.pages) *entry = place[*entry];
    }
}

size_t plan_bits(int64_t sequences, int kinds) { return static_cast<size_t>(kinds) * ((sequences + 31) / 32) * 4; }

unsigned table_blocks(int64_t entries) {
    return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>((entries + 255) / 256, 148 * 8)));
}

}  // namespace
}  // namespace fx

using namespace fx;

extern "C" fx_status fx_paged_qkv_rope_cache(const void* packed_qkv, int32_t dtype, int64_t packed_stride,
                                             int64_t tokens, int64_t query_heads, const float* cos,
                                             int64_t cos_stride, const float* sin, int64_t sin_stride,
                                             int64_t rope_rows, const fx_pages* pages, const int32_t* page_table,
                                             int64_t sequences, int64_t table_columns, int64_t table_stride,
                                             const int64_t* positions, const int64_t* token_sequences,
                                             void* query_out, void* stream) {
    const char* op = "fx_paged_qkv_rope_cache";
    fx_status st = check_pages(op, pages, false);
    if (st != FX_OK) return st;
    st = check_table(op, page_table, sequences, table_columns, table_stride, pages->page_size);
    if (st != FX_OK) return st;
    FX_REQUIRE(packed_qkv && cos && sin && positions && query_out, "fx_paged_qkv_rope_cache: null pointer");
    FX_REQUIRE(dtype == pages->dtype || dtype == FX_F32,
               "fx_paged_qkv_rope_cache: packed_qkv must be float32 or have the pages' type");
    FX_REQUIRE(tokens >= 0 && query_heads > 0 && query_heads <= 65535 && rope_rows > 0,
               "fx_paged_qkv_rope_cache: sizes must be positive");
    FX_REQUIRE(token_sequences != nullptr || tokens == sequences,
               "fx_paged_qkv_rope_cache: without token_sequences there is one token per sequence");
    FX_REQUIRE(tokens <= INT_MAX / ((query_heads + 2 * pages->kv_heads) * pages->head_dim),
               "fx_paged_qkv_rope_cache: too many tokens");
    if (tokens == 0) return FX_OK;
    WriteArgs a{};
    a.packed = packed_qkv; a.packed_stride = packed_stride; a.tokens = tokens; a.query_heads = query_heads;
    a.kv_heads = pages->kv_heads; a.dim = pages->head_dim;
    a.cos = cos; a.sin = sin; a.cos_stride = cos_stride; a.sin_stride = sin_stride; a.rope_rows = rope_rows;
    a.keys = pages->keys; a.values = pages->values;
    for (int i = 0; i < 3; ++i) { a.ks[i] = pages->key_strides[i + 1]; a.vs[i] = pages->value_strides[i + 1]; }
    a.pages = pages->pages;
    a.page_size = FastDivide::by(pages->page_size);
    a.table = page_table; a.sequences = sequences; a.columns = table_columns; a.table_stride = table_stride;
    a.positions = positions; a.owners = token_sequences; a.query = query_out;
    cudaStream_t s = as_stream(stream);
    if (dtype == FX_BF16) return launch_write<__nv_bfloat16, __nv_bfloat16>(a, s);
    if (dtype == FX_F16) return launch_write<__half, __half>(a, s);
    if (pages->dtype == FX_F32) return launch_write<float, float>(a, s);
    return pages->dtype == FX_BF16 ? launch_write<float, __nv_bfloat16>(a, s) : launch_write<float, __half>(a, s);
}

extern "C" fx_status fx_cache_pages_copy(const fx_pages* pages, const int64_t* source, const int64_t* destination,
                                         int64_t count, void* stream) {
    const fx_status st = check_pages("fx_cache_pages_copy", pages, true);
    if (st != FX_OK) return st;
    FX_REQUIRE(count >= 0, "fx_cache_pages_copy: count must not be negative");
    if (count == 0) return FX_OK;
    FX_REQUIRE(source && destination, "fx_cache_pages_copy: null pointer");
    const PoolWords pool = pool_words(*pages);
    // Longer lists, larger pools: straight to the walk in order.
    const bool look = strips_fit(pool, count) && pool.pages <= kMaxLookPages;
    const size_t bits = look ? static_cast<size_t>((pool.pages + 31) / 32) * 4 : 0;
    if (bits > kPlainShared) {
        const fx_status raised = raise_smem_limit(reinterpret_cast<const void*>(copy_kernel), kMaxLookPages / 8,
                                                  "raising the page copy's shared memory");
        if (raised != FX_OK) return raised;
    }
    const int64_t looked = look ? 32 * count + static_cast<int64_t>(bits) : 0;
    return launch_dependent(copy_kernel, dim3(copy_blocks(pool, count, looked)), dim3(kCopyThreads), bits,
                            as_stream(stream), "launching page copies", pool, source, destination, count, look);
}

extern "C" fx_status fx_cache_sequences_reserve(int32_t* page_table, int64_t sequences_total, int64_t table_columns,
                                                int64_t table_stride, const int64_t* lengths, int32_t* page_counts,
                                                int64_t pages, int64_t page_size, const int64_t* sequences,
                                                const int64_t* rows, int64_t count, int32_t* status,
                                                int32_t* workspace, void* stream) {
    const char* op = "fx_cache_sequences_reserve";
    FX_REQUIRE(pages > 0 && page_size > 0 && page_size <= kPagedMaxPageSize && count >= 0 && count <= INT_MAX,
               "fx_cache_sequences_reserve: sizes must be positive");
    FX_REQUIRE(pages <= kMaxPages, "fx_cache_sequences_reserve: at most 1048576 pages");
    const fx_status st = check_table(op, page_table, sequences_total, table_columns, table_stride, page_size);
    if (st != FX_OK) return st;
    FX_REQUIRE(sequences_total <= kMaxSequences, "fx_cache_sequences_reserve: at most 262144 sequences");
    if (count == 0) return FX_OK;
    FX_REQUIRE(lengths && page_counts && sequences && rows && status && workspace,
               "fx_cache_sequences_reserve: null pointer");
    const TableArgs t = table_args(page_table, sequences_total, table_columns, table_stride, const_cast<int64_t*>(lengths),
                      page_counts, pages, page_size);
    const size_t smem = plan_bits(sequences_total, 2);
    if (smem > kPlainShared) {
        const fx_status raised = raise_smem_limit(reinterpret_cast<const void*>(reserve_kernel),
                                                  plan_bits(kMaxSequences, 2), "raising the page planner's shared memory");
        if (raised != FX_OK) return raised;
    }
    return launch_dependent(reserve_kernel, dim3(1), dim3(kPlanThreads), smem, as_stream(stream),
                            "launching the page reservation", t, sequences, rows, count, status, workspace);
}

extern "C" fx_status fx_cache_sequences_fork(const fx_pages* pages, int32_t* page_table, int64_t sequences_total,
                                             int64_t table_columns, int64_t table_stride, int64_t* lengths,
                                             int32_t* page_counts, const int64_t* parents, const int64_t* children,
                                             int64_t count, int32_t* status, int32_t* workspace, void* stream) {
    const char* op = "fx_cache_sequences_fork";
    fx_status st = check_pages(op, pages, true);
    if (st != FX_OK) return st;
    st = check_table(op, page_table, sequences_total, table_columns, table_stride, pages->page_size);
    if (st != FX_OK) return st;
    FX_REQUIRE(sequences_total <= kMaxSequences, "fx_cache_sequences_fork: at most 262144 sequences");
    FX_REQUIRE(pages->pages <= kMaxPages, "fx_cache_sequences_fork: at most 1048576 pages");
    FX_REQUIRE(count >= 0 && count <= INT_MAX, "fx_cache_sequences_fork: count must not be negative");
    const PoolWords pool = pool_words(*pages);
    FX_REQUIRE(strips_fit(pool, count), "fx_cache_sequences_fork: too many pairs for pages of this size");
    if (count == 0) return FX_OK;
    FX_REQUIRE(lengths && page_counts && parents && children && status && workspace,
               "fx_cache_sequences_fork: null pointer");
    const TableArgs t = table_args(page_table, sequences_total, table_columns, table_stride, lengths, page_counts, pages->pages,
                      pages->page_size);
    const size_t smem = plan_bits(sequences_total, 3);
    if (smem > kPlainShared) {
        st = raise_smem_limit(reinterpret_cast<const void*>(fork_plan_kernel), plan_bits(kMaxSequences, 3),
                              "raising the page planner's shared memory");
        if (st != FX_OK) return st;
    }
    cudaStream_t s = as_stream(stream);
    st = launch_dependent(fork_plan_kernel, dim3(1), dim3(kPlanThreads), smem, s,
                          "launching the fork plan", t, parents, children, count, status, workspace);
    if (st != FX_OK) return st;
    const uint32_t tables = table_blocks(count * table_columns);
    return launch_dependent(fork_apply_kernel, dim3(tables + copy_blocks(pool, count)), dim3(kCopyThreads), 0, s,
                            "launching the fork", pool, t, parents, children, count,
                            static_cast<const int32_t*>(status), static_cast<const int32_t*>(workspace), tables);
}

extern "C" fx_status fx_cache_sequences_free(int32_t* page_table, int64_t sequences_total, int64_t table_columns,
                                             int64_t table_stride, int64_t* lengths, int32_t* page_counts,
                                             int64_t pages, const int64_t* sequences, int64_t count, void* stream) {
    FX_REQUIRE(pages > 0 && pages <= INT_MAX && count >= 0, "fx_cache_sequences_free: sizes must be positive");
    const fx_status st = check_table("fx_cache_sequences_free", page_table, sequences_total, table_columns,
                                     table_stride, 1);
    if (st != FX_OK) return st;
    if (count == 0) return FX_OK;
    FX_REQUIRE(lengths && page_counts && sequences, "fx_cache_sequences_free: null pointer");
    const TableArgs t = table_args(page_table, sequences_total, table_columns, table_stride, lengths, page_counts, pages, 1);
    return launch_dependent(free_kernel, dim3(table_blocks(count * table_columns)), dim3(256), 0, as_stream(stream),
                            "launching the release of sequences", t, sequences, count);
}

extern "C" fx_status fx_cache_pages_compact(const fx_pages* pages, int32_t* page_table, int64_t sequences_total,
                                            int64_t table_columns, int64_t table_stride, int32_t* page_counts,
                                            int32_t* used, int32_t* workspace, void* stream) {
    const char* op = "fx_cache_pages_compact";
    fx_status st = check_pages(op, pages, true);
    if (st != FX_OK) return st;
    st = check_table(op, page_table, sequences_total, table_columns, table_stride, pages->page_size);
    if (st != FX_OK) return st;
    FX_REQUIRE(page_counts && used && workspace, "fx_cache_pages_compact: null pointer");
    FX_REQUIRE(pages->pages <= kMaxPages, "fx_cache_pages_compact: at most 1048576 pages");
    const TableArgs t = table_args(page_table, sequences_total, table_columns, table_stride, nullptr, page_counts, pages->pages,
                      pages->page_size);
    const PoolWords pool = pool_words(*pages);
    FX_REQUIRE(strips_fit(pool, pages->pages / 2), "fx_cache_pages_compact: the pools are too large");  // moves at most
    cudaStream_t s = as_stream(stream);
    st = launch_dependent(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, "launching the compaction plan",
                          page_counts, pages->pages, used, workspace);
    if (st != FX_OK) return st;
    const uint32_t tables = table_blocks(sequences_total * table_columns);
    return launch_dependent(compact_apply_kernel, dim3(tables + copy_blocks(pool, (pages->pages + 1) / 2)),
                            dim3(kCopyThreads), 0, s, "launching the compaction", pool, t,
                            static_cast<const int32_t*>(used), static_cast<const int32_t*>(workspace), tables);
}
