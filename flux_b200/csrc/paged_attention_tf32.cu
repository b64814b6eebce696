// Paged decode attention for FP32 queries on FP32 pages with 5 to 16 query heads
// per KV head, on the warp-level tensor instructions (m16n8k8, TF32 operands,
// FP32 accumulators).  The FP32 units would be the bound there: here 8 heads take
// 55 us and 16 heads 69 for 64 x 4096 rows of 2 KV heads of 64 dims (268 MB, 74 %
// and 60 % of the measured copy rate; one CTA per SM instead of two took 57 and 77
// when two took 53 and 67).  No one unit is full with 16 heads: tensor pipe 37 %,
// issue slots 58 %, HBM 46 %; warps wait for the products and the splitting before
// them (math pipe and fixed latency are the first stalls).  With 3 heads it is
// slower than the FP32 units (61 us for 64 x 512-4096 rows when those took 46).
//
// Every operand x is carried as hi = tf32(x) and lo = tf32(x - hi), and a
// product is hi hi + lo hi + hi lo: what is dropped is below 2^-20 of it.  The
// tensor cores truncate when they accumulate, so hi hi products of at most 64
// dims share an accumulator and P V is added to the output with an FP32
// instruction; the cross terms, 2^-11 of the result, have one of their own.  Up to
// 8 heads leave half of the first operand's rows free: lo lies there, and two
// products do the work of three (32 x 2048 rows of 4 KV heads with 8 query heads of
// 128 dims: 65 us -> 52 when that came, 53 now).
//
// One warp takes 8 keys at a time:
//   S [16 heads x 8 keys] = Q K^T, D / 8 steps;
//   O [16 heads x D] = O keep + P V, one step of 8 keys for every 8 dims.
// Which dims make up a step, and which key a row of the second operand is, is
// free as long as both operands agree.  So a lane (g, c) = (lane / 4, lane % 4)
// reads 16 bytes of one key row, dims 4 c.. of a block of 16, and takes them
// for two steps; the weights stay in the accumulators' layout, whose columns 2
// c and 2 c + 1 become rows c and c + 4 of the second product; and of a value
// row a lane reads dims 4 g.. of a block of 32, for four columns of products.
// The 16-byte pieces of key rows are exchanged by 4 (row & 1), those of value
// rows by 2 ((row / 2) & 3): the 8 lanes served together then hit 8 different
// pieces of the banks.
#include "paged_attention.cuh"

namespace fx {
namespace {

struct KeyPieces { static __device__ __forceinline__ int at(int piece, int row) { return piece ^ ((row & 1) << 2); } };
struct ValuePieces { static __device__ __forceinline__ int at(int piece, int row) { return piece ^ (((row >> 1) & 3) << 1); } };

// hi: x to the nearest TF32 value, ties away from zero (half of its last place
// is added, the rest cut off); lo: what that leaves, cut off to TF32.  Half a
// place below the end of FP32's range the nearest value would be infinite: hi
// is then the largest one, and lo holds more (of an infinity, all).
__device__ __forceinline__ void split(float x, uint32_t& hi, uint32_t& lo) {
    float near;  // the smaller magnitude, with x's sign
    asm("min.xorsign.abs.f32 %0, %1, %2;" : "=f"(near) : "f"(x), "f"(__uint_as_float(0x7f7fefffu)));
    hi = (__float_as_uint(near) + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}
// The same of a weight, which is at most 1.
__device__ __forceinline__ void split_weight(float x, uint32_t& hi, uint32_t& lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Heads: 8 or 16, room for a unit's heads.  With 8, rows 8-15 of the first
// operands hold the lo terms of rows 0-7.
template <int DP, int Heads>
struct Tf32Shape {
    static constexpr bool kPacked = Heads == 8;
    static constexpr int kOperands = kPacked ? 1 : 2;  // of a query or weight
    static constexpr int kHalves = kPacked ? 1 : 2;    // of the 16 rows that hold heads
    static constexpr int kRows = 8;
    static constexpr int kWarps = DP == 256 ? 4 : 8;
    static constexpr int kThreads = 32 * kWarps;
    static constexpr int kTile = kRows * kWarps;
    using Ring = PagedRing<float, kRows, DP, KeyPieces, ValuePieces>;
    static constexpr int kLevel = kWarps * Ring::kBytes;
    // The query operand, hi and lo, in its own layout (16 bytes a lane and
    // step) for the whole CTA; states of joining warps.
    static constexpr int kQueryBytes = kOperands * (DP / 8) * 512;
    static constexpr int kFixed = kQueryBytes + kWarps * Heads * (DP + 2) * static_cast<int>(sizeof(float)) + 512;
    static constexpr int kPerSm = DP == 64 ? 2 : 1;
    static constexpr int kFit = ((kPerSm == 2 ? 112 : 226) * 1024 - kFixed) / kLevel;
    static constexpr int kStages = kFit > 6 ? 6 : kFit;
    static constexpr int kShared = kFixed + kStages * kLevel;
    static_assert(kStages >= 2, "two stages at least");
};

template <int DP, int Heads>
__global__ void __launch_bounds__(Tf32Shape<DP, Heads>::kThreads, (Tf32Shape<DP, Heads>::kPerSm))
    paged_tf32_kernel(const __grid_constant__ PagedAttend a) {
    using S = Tf32Shape<DP, Heads>;
    using Ring = typename S::Ring;
    constexpr int kSteps = DP / 8;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ PagedStart start;
    __shared__ int scratch[S::kWarps];
    __shared__ uint32_t masks[S::kWarps][S::kStages];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    float* ring = reinterpret_cast<float*>(smem) + warp * S::kStages * 2 * Ring::kHalf;
    uint4* queries = reinterpret_cast<uint4*>(smem + S::kStages * S::kLevel);  // [hi, lo][step][lane]
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
    PagedStream<Ring, float, S::kTile, S::kStages> stream(a, start, ring, masks[warp]);

    while (stream.now.left > 0) {
        const int count = stream.now.piece(), first = stream.now.tile, tiles = stream.now.tiles;
        const int b = stream.now.b, head = stream.now.head;
        // Step i's rows k = c and c + 4 are dims 16 (i / 2) + 4 c + 2 (i & 1) and the next.
        const float* unit = static_cast<const float*>(a.q) + b * a.q_batch + head * a.group * a.q_head;
        for (int i = warp; i < kSteps; i += S::kWarps) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int h = S::kPacked ? g : g + 8 * (r & 1), d = 16 * (i >> 1) + 4 * c + 2 * (i & 1) + (r >> 1);
                split(h < a.group && d < a.dim ? unit[h * a.q_head + d] : 0.0f, hi[r], lo[r]);
            }
            if constexpr (S::kPacked) {
                queries[i * 32 + lane] = make_uint4(hi[0], lo[0], hi[2], lo[2]);
            } else {
                queries[i * 32 + lane] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                queries[(kSteps + i) * 32 + lane] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
        }
        __syncthreads();
        float m[S::kHalves], l[S::kHalves];
#pragma unroll
        for (int r = 0; r < S::kHalves; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.0f;
        }
        float o[DP / 8][4];
#pragma unroll
        for (int j = 0; j < DP / 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;

        for (int t = 0; t < count; ++t) {
            stream.advance();
            const float* keys = stream.keys();
            const float* values = keys + Ring::kHalf;
            float s[4] = {}, part[4] = {}, cross[4] = {};
#pragma unroll
            for (int i = 0; i < kSteps; i += 2) {
                const float4 k = *reinterpret_cast<const float4*>(keys + g * DP + 4 * KeyPieces::at(2 * i + c, g));
                uint32_t hi[4], lo[4];
                split(k.x, hi[0], lo[0]);
                split(k.y, hi[1], lo[1]);
                split(k.z, hi[2], lo[2]);
                split(k.w, hi[3], lo[3]);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint4 x = queries[(i + u) * 32 + lane];
                    const uint32_t qh[4] = {x.x, x.y, x.z, x.w};  // packed: hi and lo
                    mma(part, qh, hi[2 * u], hi[2 * u + 1]);
                    if constexpr (!S::kPacked) {
                        const uint4 y = queries[(kSteps + i + u) * 32 + lane];
                        const uint32_t ql[4] = {y.x, y.y, y.z, y.w};
                        mma(cross, ql, hi[2 * u], hi[2 * u + 1]);
                    }
                    mma(cross, qh, lo[2 * u], lo[2 * u + 1]);
                }
                if (i % 8 == 6) {  // 64 dims
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[e] += part[e];
                        part[e] = 0.0f;
                    }
                }
            }
            if constexpr (S::kPacked) {
#pragma unroll
                for (int e = 0; e < 2; ++e) cross[e] += s[2 + e];  // lo hi
            }
            const uint32_t mask = stream.mask() >> (2 * c);
            float keep[S::kHalves];
#pragma unroll
            for (int r = 0; r < S::kHalves; ++r) {
                float top = m[r];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float& x = s[2 * r + e];
                    x = (mask >> e) & 1u ? (x + cross[2 * r + e]) * a.scale : -INFINITY;
                    top = fmaxf(top, x);
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float base = top == -INFINITY ? 0.0f : top;
                keep[r] = exp2f(m[r] - base);
                m[r] = top;
                l[r] *= keep[r];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float& x = s[2 * r + e];
                    x = exp2f(x - base);
                    l[r] += x;
                }
            }
            // Rows k = c and c + 4 of the second product are keys 2 c and 2 c + 1.
            uint32_t ph[4], pl[4];
            if constexpr (S::kPacked) {
                split_weight(s[0], ph[0], ph[1]);
                split_weight(s[1], ph[2], ph[3]);
            } else {
                split_weight(s[0], ph[0], pl[0]);
                split_weight(s[2], ph[1], pl[1]);
                split_weight(s[1], ph[2], pl[2]);
                split_weight(s[3], ph[3], pl[3]);
            }
#pragma unroll
            for (int j = 0; j < DP / 8; j += 4) {  // 32 dims: columns g of four products are dims 4 g, 4 g + 1, ...
                const float4 v0 = *reinterpret_cast<const float4*>(values + 2 * c * DP + 4 * ValuePieces::at(2 * j + g, 2 * c));
                const float4 v1 =
                    *reinterpret_cast<const float4*>(values + (2 * c + 1) * DP + 4 * ValuePieces::at(2 * j + g, 2 * c + 1));
                const float x[2][4] = {{v0.x, v0.y, v0.z, v0.w}, {v1.x, v1.y, v1.z, v1.w}};
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    uint32_t h0, l0, h1, l1;
                    split(x[0][u], h0, l0);
                    split(x[1][u], h1, l1);
                    float y[4] = {};
                    if constexpr (!S::kPacked) mma(y, pl, h0, h1);
                    mma(y, ph, l0, l1);
                    mma(y, ph, h0, h1);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[j + u][e] = fmaf(o[j + u][e], keep[S::kPacked ? 0 : e >> 1], y[e]);
                }
            }
            stream.release();
        }

        const int width = a.dim + 2;
        float* mine = states + warp * a.group * width;
#pragma unroll
        for (int r = 0; r < S::kHalves; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            const int h = g + 8 * r;
            if (h >= a.group) continue;
            if (c == 0) {
                mine[h * width] = m[r];
                mine[h * width + 1] = l[r];
            }
#pragma unroll
            for (int j = 0; j < DP / 8; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int d = 8 * (j & ~3) + 4 * (2 * c + e) + (j & 3);  // column 2 c + e of product j
                    if (d < a.dim) mine[h * width + 2 + d] = S::kPacked ? o[j][e] + o[j][2 + e] : o[j][2 * r + e];
                }
        }
        paged_join<float, S::kTile, S::kWarps>(a, start, states, b, head, first, count, tiles, stream.now.left == 0);
    }
}

template <int DP, int Heads>
fx_status launch(const PagedAttend& a, int sms, cudaStream_t stream) {
    using S = Tf32Shape<DP, Heads>;
    const fx_status st = raise_smem_limit(reinterpret_cast<const void*>(paged_tf32_kernel<DP, Heads>), S::kShared,
                                          "raising paged attention shared memory");
    if (st != FX_OK) return st;
    const int grid = paged_grid<S::kTile>(a, sms, S::kPerSm);
    const fx_status launched = launch_dependent(paged_tf32_kernel<DP, Heads>, dim3(grid), dim3(S::kThreads), S::kShared, stream,
                                                "launching paged attention", a);
    if (launched != FX_OK) return launched;
    return a.whole ? FX_OK : launch_paged_merge<float>(a, grid, stream);
}

}  // namespace

fx_status launch_paged_f32_wide(const PagedAttend& a, int sms, cudaStream_t stream) {
    const bool packed = a.group <= 8;
    if (a.dim <= 64) return packed ? launch<64, 8>(a, sms, stream) : launch<64, 16>(a, sms, stream);
    if (a.dim <= 128) return packed ? launch<128, 8>(a, sms, stream) : launch<128, 16>(a, sms, stream);
    return packed ? launch<256, 8>(a, sms, stream) : launch<256, 16>(a, sms, stream);
}

}  // namespace fx
