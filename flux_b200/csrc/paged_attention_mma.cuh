// Paged decode attention on 16-bit pages, on the warp-level tensor instructions
// (m16n8k16, FP32 accumulators): for queries of the pages' type and for FP32
// queries.
//
// The heads of a group are rows of the products' first operand, which has 16.
// One warp takes 16 keys at a time from its ring:
//   S [heads x 16 keys] = Q K^T, D / 16 steps;
//   running maximum, p = exp2(S - max), on the accumulators' layout;
//   O [heads x D] = O keep + P V.
// Keys and values are exact in 16 bits; what is not is carried as a sum of
// 16-bit terms, each the nearest to what the ones before leave:
//   P, two terms for 16-bit queries: one would lose 2^-9 of each weight
//     (bfloat16), two leave 2^-17, below the output's own rounding;
//   Q and P, three terms each for FP32 queries: 24 bits, as many as FP32 has.
// Groups leave rows free, and the terms go there: with up to 4 heads (8 for
// 16-bit queries) one product does the work of three (two), with up to 8 heads
// two do that of three; the terms' rows of S are added before the maximum, those
// of O once at the end of a unit.  64 x 8192 rows of 3 KV heads with 3 FP32 query
// heads of 64 dims on BF16 pages take 69 us (89 % of the measured copy rate)
// against 88 with a product for each term; 64 x 4096 of 4 KV heads with 8 of 128
// 92 against 111.
//
// float16's narrow range is met by scaling: a query row so that its largest
// element lies in [2^13, 2^14), the weights by 2^14 (their sum too, so that it
// cancels).  The tensor cores truncate when they accumulate, by 2^-25 a product on
// average and always towards zero.  For FP32 queries P V is therefore added to O
// with an FP32 instruction.  For 16-bit queries O is the accumulator, which stays
// below a 16-bit output's rounding for tables of up to 65536 rows; in longer ones
// it is summed in runs of 256 tiles, which are joined in FP32 (one run of 4 M rows
// would be off by 0.8 %).
//
// A decode step has one row per head, so the larger tcgen05 tiles (64 or 128
// rows) would be 4-8 times emptier still and would add a trip through TMEM
// between the two products.
//
// Shared memory: rows of DP elements whose 16-byte pieces are exchanged by
// piece ^ (row & 7), so that the 8 rows a matrix load reads lie in different
// banks.
#pragma once

#include "paged_attention.cuh"

namespace fx {

template <typename T>
struct Mma;
template <>
struct Mma<__nv_bfloat16> {
    static __device__ __forceinline__ void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    // The nearest 16-bit values of x and y, and what they leave in x and y.
    static __device__ __forceinline__ uint32_t term(float& x, float& y) { return term(x, y, x, y); }
    // The first of several: bfloat16 ends half a place before FP32 does, and
    // there the largest one is taken.
    static __device__ __forceinline__ uint32_t first_term(float& x, float& y) {
        const float most = __uint_as_float(0x7f7f0000u);
        return term(x, y, fminf(fmaxf(x, -most), most), fminf(fmaxf(y, -most), most));
    }
    static __device__ __forceinline__ uint32_t term(float& x, float& y, float near_x, float near_y) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(near_x, near_y);
        const float2 f = __bfloat1622float2(h);
        x -= f.x;
        y -= f.y;
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static constexpr float kWeightBits = 0.0f;  // log2 of the weights' scale
};
template <>
struct Mma<__half> {
    static __device__ __forceinline__ void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ uint32_t term(float& x, float& y) {
        const __half2 h = __floats2half2_rn(x, y);
        const float2 f = __half22float2(h);
        x -= f.x;
        y -= f.y;
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ uint32_t first_term(float& x, float& y) { return term(x, y); }  // scaled queries
    static constexpr float kWeightBits = 14.0f;
};

__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t address) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(address)
                 : "memory");
}
__device__ __forceinline__ void load_matrices_transposed(uint32_t (&r)[4], uint32_t address) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(address)
                 : "memory");
}

// T: the pages' type, Q: the queries', Heads: 4, 8 or 16, room for a unit's heads.
template <typename T, typename Q, int DP, int Heads>
struct MmaShape {
    static constexpr bool kExact = !std::is_same<T, Q>::value;  // FP32 queries
    static constexpr bool kPacked = Heads < 16;                 // terms lie in rows without a head
    static constexpr int kTerms = kExact ? 3 : 2;               // of the weights
    static constexpr int kTermsPerOperand = 16 / Heads < kTerms ? 16 / Heads : kTerms;
    static constexpr int kWeightOperands = (kTerms + kTermsPerOperand - 1) / kTermsPerOperand;
    static constexpr int kQueryOperands = kExact ? kWeightOperands : 1;
    static constexpr int kHalves = kPacked ? 1 : 2;             // of the 16 rows that hold heads
    static_assert(Heads != 4 || kExact, "four heads leave room for three terms");
    static constexpr int kRows = 16;
    static constexpr int kWarps = 4;
    static constexpr int kThreads = 32 * kWarps;
    static constexpr int kTile = kRows * kWarps;
    static constexpr int kRowBytes = 2 * DP;
    using Ring = PagedRing<T, kRows, DP, ByRow, ByRow>;
    static constexpr int kLevel = kWarps * Ring::kBytes;
    // The query operand lies in shared memory in its own layout (16 bytes a
    // lane and step), and in registers where one term of it fits.
    static constexpr bool kHoldQueries = kQueryOperands == 1 && DP <= 128;
    static constexpr int kQueryBytes = kQueryOperands * (DP / 16) * 512;
    static constexpr int kFixed = kQueryBytes + kWarps * Heads * (DP + 2) * static_cast<int>(sizeof(float)) + 512;
    static constexpr int kPerSm = DP <= 64 ? 3 : DP <= 128 ? 2 : 1;
    static constexpr int kFit = ((kPerSm == 3 ? 74 : kPerSm == 2 ? 112 : 226) * 1024 - kFixed) / kLevel;
    static constexpr int kStages = kFit > 6 ? 6 : kFit;
    static constexpr int kShared = kFixed + kStages * kLevel;
    static_assert(kStages >= 2, "two stages at least");
};

// Runs: O is summed in runs of kRun tiles.
template <typename T, typename Q, int DP, int Heads, bool Runs>
__global__ void __launch_bounds__(MmaShape<T, Q, DP, Heads>::kThreads, MmaShape<T, Q, DP, Heads>::kPerSm)
    paged_mma_kernel(const __grid_constant__ PagedAttend a) {
    using S = MmaShape<T, Q, DP, Heads>;
    using Ring = typename S::Ring;
    constexpr int kSteps = DP / 16;
    constexpr int kRun = 256;
    constexpr bool kQuarters = Heads == 4;  // terms in rows 0-3, 4-7 and 8-11
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ PagedStart start;
    __shared__ int scratch[S::kWarps];
    __shared__ uint32_t masks[S::kWarps][S::kStages];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    T* ring = reinterpret_cast<T*>(smem + warp * S::kStages * Ring::kBytes);
    uint4* queries = reinterpret_cast<uint4*>(smem + S::kStages * S::kLevel);  // [term][step][lane]
    float* states = reinterpret_cast<float*>(smem + S::kStages * S::kLevel + S::kQueryBytes);

    grid_dependency_wait();
    if (!a.whole) paged_launch_merge();
    paged_start<S::kTile, S::kThreads>(a, &start, scratch);
    if (start.left == 0) {
        paged_describe_none(a);
        return;
    }
    if (a.dim < DP) {  // dims that the copies never write
        for (int i = lane; i < S::kStages * Ring::kBytes / 16; i += 32)
            reinterpret_cast<uint4*>(ring)[i] = make_uint4(0u, 0u, 0u, 0u);
        __syncwarp();
    }
    PagedStream<Ring, T, S::kTile, S::kStages> stream(a, start, ring, masks[warp]);

    // Rows and 16-byte pieces this lane points the matrix loads at.
    const int k_row = (lane & 7) + ((lane >> 4) << 3), k_piece = (lane >> 3) & 1;
    const int v_row = (lane & 7) + (lane & 8), v_piece = lane >> 4;
    // Accumulator rows lane / 4 and lane / 4 + 8; columns pair, pair + 1.
    //   16 heads: heads top_head and top_head + 8.
    //   8 heads: head top_head, its first term and (if it has one) its second; an
    //     operand of its own for a third.
    //   4 heads: head top_head, its first term in rows 0-3 (`leads`), its second in
    //     rows 4-7, its third in rows 8-11.
    const int top_head = kQuarters ? (lane >> 2) & 3 : lane >> 2, pair = 2 * (lane & 3);
    const bool leads = lane < 16;

    while (stream.now.left > 0) {
        const int count = stream.now.piece(), first = stream.now.tile, tiles = stream.now.tiles;
        const int b = stream.now.b, head = stream.now.head;
        // The unit's queries (unused heads and dims are zeros).
        const Q* unit = static_cast<const Q*>(a.q) + b * a.q_batch + head * a.group * a.q_head;
        const auto element = [&](int i, int half, int across, int e) {
            const int h = top_head + 8 * half, d = 16 * i + 8 * across + pair + e;
            return h < a.group && d < a.dim ? to_float(unit[h * a.q_head + d]) : 0.0f;
        };
        float scale[S::kHalves], factor[S::kHalves];  // of this lane's heads
#pragma unroll
        for (int r = 0; r < S::kHalves; ++r) {
            scale[r] = a.scale;
            factor[r] = 1.0f;
            if constexpr (S::kExact && std::is_same<T, __half>::value) {
                float top = 0.0f;
#pragma unroll 4
                for (int i = 0; i < kSteps; ++i)
#pragma unroll
                    for (int across = 0; across < 2; ++across)
                        top = fmaxf(top, fmaxf(fabsf(element(i, r, across, 0)), fabsf(element(i, r, across, 1))));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // 2^(13 - floor(log2 top)), or the largest power of two
                const int bits = 13 + 127 - static_cast<int>((__float_as_uint(top) >> 23) & 255u) + 127;
                factor[r] = __uint_as_float(static_cast<uint32_t>(min(bits, 254)) << 23);
                scale[r] = a.scale / factor[r];
            }
        }
        // In the operand's layout: entry r of a step holds two dims of row lane / 4
        // (r even) or lane / 4 + 8, 8 dims further on for r >= 2.
        for (int i = warp; i < kSteps; i += S::kWarps) {
            if constexpr (S::kPacked) {
                uint32_t w[S::kQueryOperands][4] = {};
#pragma unroll
                for (int across = 0; across < 2; ++across) {
                    float x = element(i, 0, across, 0) * factor[0], y = element(i, 0, across, 1) * factor[0];
                    w[0][2 * across] = S::kExact ? Mma<T>::first_term(x, y) : Mma<T>::term(x, y);
                    if constexpr (S::kExact) {
                        const uint32_t two = Mma<T>::term(x, y), three = Mma<T>::term(x, y);
                        if constexpr (kQuarters) {
                            w[0][2 * across] = leads ? w[0][2 * across] : two;
                            w[0][2 * across + 1] = leads ? three : 0u;
                        } else {
                            w[0][2 * across + 1] = two;
                            w[S::kQueryOperands - 1][2 * across] = three;
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < S::kQueryOperands; ++n)
                    queries[(n * kSteps + i) * 32 + lane] = make_uint4(w[n][0], w[n][1], w[n][2], w[n][3]);
            } else {
                float x[4][2];
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int e = 0; e < 2; ++e) x[r][e] = element(i, r & 1, r >> 1, e) * factor[r & 1];
#pragma unroll
                for (int term = 0; term < S::kQueryOperands; ++term) {
                    uint32_t w[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        w[r] = S::kExact && term == 0 ? Mma<T>::first_term(x[r][0], x[r][1])
                                                      : Mma<T>::term(x[r][0], x[r][1]);
                    queries[(term * kSteps + i) * 32 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
        __syncthreads();
        const auto operand = [&](uint32_t(&f)[4], int term, int i) {
            const uint4 x = queries[(term * kSteps + i) * 32 + lane];
            f[0] = x.x;
            f[1] = x.y;
            f[2] = x.z;
            f[3] = x.w;
        };
        uint32_t q[S::kHoldQueries ? kSteps : 1][4];
        if constexpr (S::kHoldQueries) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) operand(q[i], 0, i);
        }
        float m[S::kHalves], l[S::kHalves], o[DP / 8][4];
        const auto clear = [&] {
#pragma unroll
            for (int r = 0; r < S::kHalves; ++r) {
                m[r] = -INFINITY;
                l[r] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < DP / 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;
        };
        const int width = a.dim + 2;
        float* mine = states + warp * a.group * width;
        // Joins the state that the warp left in shared memory to the one it holds.
        const auto take_back = [&] {
#pragma unroll
            for (int r = 0; r < S::kHalves; ++r) {
                const int h = top_head + 8 * r;
                const bool any = h < a.group;
                const float before = any ? mine[h * width] : -INFINITY, sum = any ? mine[h * width + 1] : 0.0f;
                const float top = fmaxf(m[r], before), base = top == -INFINITY ? 0.0f : top;
                const float now = exp2f(m[r] - base), then = exp2f(before - base);
                m[r] = top;
                l[r] = fmaf(l[r], now, (lane & 3) == 0 ? sum * then : 0.0f);
#pragma unroll
                for (int j = 0; j < DP / 8; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float x = any && 8 * j < a.dim ? mine[h * width + 2 + 8 * j + pair + e] : 0.0f;
                        o[j][2 * r + e] = fmaf(o[j][2 * r + e], now, x * then);
                        if constexpr (S::kPacked) o[j][2 + e] *= now;
                    }
            }
            __syncwarp();  // all of it is read
        };
        int done = 0;
        do {
            const int until = Runs ? min(count - done, kRun) : count;
            clear();
            for (int t = 0; t < until; ++t) {
                // Kernels that HBM bounds keep their warps to one tile: apart, they read a
                // page's rows at different times (64 x 8192 rows of 3 KV heads of 64 16-bit
                // dims: FP32 queries 72 us, 69 together; 16-bit ones 72 and 68).  With more
                // products the wait costs more than it gives (92 us, 96).
                if (S::kWeightOperands == 1) __syncthreads();
                stream.advance();
                const uint32_t keys = static_cast<uint32_t>(__cvta_generic_to_shared(stream.keys()));
                const uint32_t values = keys + Ring::kHalf * 2;
                float s[2][4] = {}, rest[2][4] = {};
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    uint32_t k[4];
                    load_matrices(k, keys + k_row * S::kRowBytes + (((2 * i + k_piece) ^ (k_row & 7)) << 4));
                    if constexpr (!S::kHoldQueries) operand(q[0], 0, i);
                    Mma<T>::run(s[0], q[S::kHoldQueries ? i : 0], k[0], k[1]);
                    Mma<T>::run(s[1], q[S::kHoldQueries ? i : 0], k[2], k[3]);
#pragma unroll
                    for (int term = 1; term < S::kQueryOperands; ++term) {
                        operand(q[0], term, i);
                        Mma<T>::run(rest[0], q[0], k[0], k[1]);
                        Mma<T>::run(rest[1], q[0], k[2], k[3]);
                    }
                }
                if constexpr (S::kExact) {
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 2 * S::kHalves; ++e) {
                            if constexpr (S::kPacked) s[n][e] += s[n][2 + e] + rest[n][e];
                            else s[n][e] += rest[n][e];
                            // Both lanes of a head come to the same sum.
                            if constexpr (kQuarters) s[n][e] += __shfl_xor_sync(0xffffffffu, s[n][e], 16);
                        }
                }
                const uint32_t mask = stream.mask() >> pair;
                float keep[S::kHalves];
#pragma unroll
                for (int r = 0; r < S::kHalves; ++r) {
                    float top = m[r];
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float& x = s[n][2 * r + e];
                            x = (mask >> (8 * n + e)) & 1u ? x * scale[r] : -INFINITY;
                            top = fmaxf(top, x);
                        }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const float base = top == -INFINITY ? 0.0f : top;
                    keep[r] = exp2f(m[r] - base);
                    m[r] = top;
                    l[r] *= keep[r];
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float& x = s[n][2 * r + e];
                            x = exp2f(x - base + Mma<T>::kWeightBits);
                            l[r] += x;
                        }
                }
                uint32_t p[S::kWeightOperands][4] = {};
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    if constexpr (S::kPacked) {
                        const uint32_t one = Mma<T>::term(s[n][0], s[n][1]), two = Mma<T>::term(s[n][0], s[n][1]);
                        p[0][2 * n] = one;
                        p[0][2 * n + 1] = two;
                        if constexpr (S::kExact) {
                            const uint32_t three = Mma<T>::term(s[n][0], s[n][1]);
                            if constexpr (kQuarters) {
                                p[0][2 * n] = leads ? one : two;
                                p[0][2 * n + 1] = leads ? three : 0u;
                            } else {
                                p[S::kWeightOperands - 1][2 * n] = three;
                            }
                        }
                    } else {
#pragma unroll
                        for (int term = 0; term < S::kWeightOperands; ++term)
#pragma unroll
                            for (int r = 0; r < 2; ++r)
                                p[term][2 * n + r] = Mma<T>::term(s[n][2 * r], s[n][2 * r + 1]);
                    }
                }
                const auto kept = [&](int e) { return keep[S::kHalves == 2 ? e >> 1 : 0]; };
                if constexpr (!S::kExact) {
                    if (__any_sync(0xffffffffu, kept(0) != 1.0f || kept(2) != 1.0f)) {
#pragma unroll
                        for (int j = 0; j < DP / 8; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[j][e] *= kept(e);
                    }
                }
#pragma unroll
                for (int j = 0; j < DP / 8; j += 2) {
                    uint32_t v[4];
                    load_matrices_transposed(v, values + v_row * S::kRowBytes + (((j + v_piece) ^ (v_row & 7)) << 4));
                    if constexpr (!S::kExact) {
#pragma unroll
                        for (int term = S::kWeightOperands - 1; term >= 0; --term) {
                            Mma<T>::run(o[j], p[term], v[0], v[1]);
                            Mma<T>::run(o[j + 1], p[term], v[2], v[3]);
                        }
                        continue;
                    }
                    float x[2][4] = {};
#pragma unroll
                    for (int term = S::kWeightOperands - 1; term >= 0; --term) {
                        Mma<T>::run(x[0], p[term], v[0], v[1]);
                        Mma<T>::run(x[1], p[term], v[2], v[3]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        o[j][e] = fmaf(o[j][e], kept(e), x[0][e]);
                        o[j + 1][e] = fmaf(o[j + 1][e], kept(e), x[1][e]);
                    }
                }
                stream.release();
            }
            if constexpr (Runs)
                if (done > 0) take_back();
#pragma unroll
            for (int r = 0; r < S::kHalves; ++r) {
                l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
                l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
                const int h = top_head + 8 * r;
                const bool any = h < a.group && (!kQuarters || leads);
                if (any && (lane & 3) == 0) {
                    mine[h * width] = m[r];
                    mine[h * width + 1] = l[r];
                }
#pragma unroll
                for (int j = 0; j < DP / 8; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float x = o[j][2 * r + e];
                        if constexpr (S::kPacked) x += o[j][2 + e];
                        if constexpr (kQuarters) x += __shfl_xor_sync(0xffffffffu, x, 16);
                        if (any && 8 * j < a.dim) mine[h * width + 2 + 8 * j + pair + e] = x;
                    }
            }
            if constexpr (Runs) __syncwarp();
            done += until;
        } while (Runs && done < count);
        paged_join<Q, S::kTile, S::kWarps>(a, start, states, b, head, first, count, tiles, stream.now.left == 0);
    }
}

template <typename T, typename Q, int DP, int Heads, bool Runs>
fx_status launch_mma(const PagedAttend& a, int sms, cudaStream_t stream) {
    using S = MmaShape<T, Q, DP, Heads>;
    const auto kernel = paged_mma_kernel<T, Q, DP, Heads, Runs>;
    const fx_status st = raise_smem_limit(reinterpret_cast<const void*>(kernel), S::kShared,
                                          "raising paged attention shared memory");
    if (st != FX_OK) return st;
    const int grid = paged_grid<S::kTile>(a, sms, S::kPerSm);
    const fx_status launched =
        launch_dependent(kernel, dim3(grid), dim3(S::kThreads), S::kShared, stream, "launching paged attention", a);
    if (launched != FX_OK) return launched;
    return a.whole ? FX_OK : launch_paged_merge<Q>(a, grid, stream);
}

template <typename T, typename Q, int DP, bool Runs>
fx_status launch_mma_heads(const PagedAttend& a, int sms, cudaStream_t stream) {
    if constexpr (!std::is_same<T, Q>::value)
        if (a.group <= 4) return launch_mma<T, Q, DP, 4, false>(a, sms, stream);
    return a.group <= 8 ? launch_mma<T, Q, DP, 8, Runs>(a, sms, stream)
                        : launch_mma<T, Q, DP, 16, Runs>(a, sms, stream);
}

template <typename T, typename Q, bool Runs>
fx_status launch_mma_dims(const PagedAttend& a, int sms, cudaStream_t stream) {
    if (a.dim <= 64) return launch_mma_heads<T, Q, 64, Runs>(a, sms, stream);
    if (a.dim <= 128) return launch_mma_heads<T, Q, 128, Runs>(a, sms, stream);
    return launch_mma_heads<T, Q, 256, Runs>(a, sms, stream);
}

// A CTA may get all rows of a sequence.  1024 tiles in one sum lose 2^-14 on
// average and 2^-12 at most, less than half a step of float16.  Kernels with runs
// are larger, which short calls pay for (16 sequences of 200 rows: 10.3 us, 9.7
// without), and otherwise 0-1 % slower.
constexpr int kSumRows = 65536;

template <typename T, typename Q>
fx_status launch_mma_pages(const PagedAttend& a, int sms, cudaStream_t stream) {
    if constexpr (std::is_same<T, Q>::value)
        if (a.capacity > kSumRows) return launch_mma_dims<T, Q, true>(a, sms, stream);
    return launch_mma_dims<T, Q, false>(a, sms, stream);
}

}  // namespace fx
