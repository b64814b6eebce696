// The split of paged decode attention over the GPU, shared by its kernels:
// paged_attention_simt.cu (FP32 pages, up to 4 query heads per KV head),
// paged_attention_tf32.cu (FP32 pages, 5-16 heads) and paged_attention_mma.cuh
// (16-bit pages, with queries of their type or FP32 ones).
//
// A unit is one (sequence, KV head) with its group of query heads, or one of
// the equal parts of a group of more than 16; its rows are cut into tiles of kTile rows
// (a sequence without rows still has one tile, so that its zeros get written).
// The tiles of all units form one line, which the CTAs divide evenly: CTA i of
// n owns tiles [i N / n, (i + 1) N / n).  Every CTA finds its own part from the
// lengths alone, so the host knows nothing of them, a long sequence is split
// as far as it takes to fill the GPU and short ones are hardly split at all.
// Within a CTA warp w takes rows [w R, (w + 1) R) of each tile, with its own
// softmax state and its own ring of copies in flight, which runs on across
// units.  (Warps with tiles of their own, 8 times as many streams of rows, lost
// 6-10 % of the bandwidth on long sequences.)
//
// Where a unit ends, the warps leave their states in shared memory and all
// threads join them.  (Going on at once, with one warp that joins for all, was
// no faster in an earlier form of these kernels, and 2 us slower for a single
// short sequence.)  A unit that lies in one CTA is finished
// there.  One that spans CTAs leaves (max, sum, unnormalised output) of each
// piece in the workspace for the merge kernel.  All in an order fixed by the
// lengths: results repeat bit for bit.
//
// Where no sequence can have many rows (paged_whole), CTAs take whole units
// instead, which saves the merge launch.
#pragma once

#include <cstdint>
#include <type_traits>

#include "paged.cuh"

namespace fx {

// CTAs of one launch at most; the workspace holds two pieces for each.
constexpr int kPagedMaxGrid = 512;
constexpr int kPagedDescriptor = 4;  // ints per CTA before the pieces: sequence, KV head, last CTA, valid
constexpr int kPagedUnits = 64;      // units whose first and last CTA are noted too (two ints each)
constexpr float kLog2e = 1.4426950408889634f;

struct PagedAttend {
    const void* q;
    int64_t q_batch, q_head;
    const void* keys;
    const void* values;
    int64_t ks[3], vs[3];  // page, head, row (elements)
    const int32_t* table;
    int64_t table_stride;
    const int64_t* lengths;
    void* out;
    float* workspace;
    float scale;            // of the scores, times log2(e): the softmax is taken in base 2
    int pages, batch, heads, dim;
    int kv_heads, group;    // units of a sequence, query heads of a unit
    int capacity;           // rows a table row can hold
    bool whole;             // CTAs take whole units
    bool alike;             // keys and values have the same strides
    FastDivide page_size, per_head, share;  // rows of a page; dims of a head; units of a KV head
};

__device__ __forceinline__ float* paged_pieces(const PagedAttend& a) {
    return a.workspace + kPagedMaxGrid * kPagedDescriptor + 2 * kPagedUnits;
}

__host__ __device__ __forceinline__ int paged_rows(const PagedAttend& a, int b) {
    const int64_t n = a.lengths[b];
    return n < 0 ? 0 : (n > a.capacity ? a.capacity : static_cast<int>(n));
}

template <int kTile>
__host__ __device__ __forceinline__ int paged_tiles(int rows) {
    return rows <= kTile ? 1 : static_cast<int>((static_cast<uint32_t>(rows) + (kTile - 1)) / kTile);
}

// The first of `total` tiles that CTA i of `ctas` takes.
__host__ __device__ __forceinline__ int paged_first(int64_t i, int total, int ctas) {
    return static_cast<int>(i * total / ctas);
}
// The CTA that takes tile t.
__host__ __device__ __forceinline__ int paged_owner(int64_t t, int total, int ctas) {
    return static_cast<int>(((t + 1) * ctas - 1) / total);
}

// Where a CTA starts: tile `tile` of KV head `head` of sequence `b`, and how
// many tiles it takes from there.
struct PagedStart {
    int b, head, tile, left;
    int rows;         // of sequence b
    int total, ctas;  // tiles of all units, CTAs that have any
};

// Sequence, KV head and tile of the tile `rest` from the start of sequence b on.
template <int kTile>
__host__ __device__ __forceinline__ PagedStart paged_locate(const PagedAttend& a, int b, int rest) {
    for (; b < a.batch; ++b) {
        const int rows = paged_rows(a, b), tiles = paged_tiles<kTile>(rows);
        if (rest < tiles * a.kv_heads) return {b, rest / tiles, rest % tiles, 0, rows, 0, 0};
        rest -= tiles * a.kv_heads;
    }
    return {};
}

// Each thread sums the tiles of a run of sequences, the CTA scans the sums, and
// the thread whose run holds the CTA's first tile looks it up.
template <int kTile, int kThreads>
__device__ __forceinline__ void paged_start(const PagedAttend& a, PagedStart* start, int* scratch) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (a.whole) {  // units [first, last); there are as many CTAs as units, or fewer
        const int64_t units = static_cast<int64_t>(a.batch) * a.kv_heads;
        const int64_t first = blockIdx.x * units / gridDim.x, last = (blockIdx.x + int64_t{1}) * units / gridDim.x;
        const int b0 = static_cast<int>(first / a.kv_heads), b1 = static_cast<int>((last - 1) / a.kv_heads);
        int sum = 0;
        for (int b = b0 + tid; b <= b1; b += kThreads) {
            const int64_t from = max(first, static_cast<int64_t>(b) * a.kv_heads);
            const int64_t to = min(last, (b + int64_t{1}) * a.kv_heads);
            sum += static_cast<int>(to - from) * paged_tiles<kTile>(paged_rows(a, b));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) scratch[warp] = sum;
        __syncthreads();
        if (tid == 0) {
            sum = 0;
            for (int w = 0; w < kThreads / 32; ++w) sum += scratch[w];
            *start = {b0, static_cast<int>(first - static_cast<int64_t>(b0) * a.kv_heads), 0, sum, paged_rows(a, b0), 1, 1};
        }
        __syncthreads();
        return;
    }
    const int run = (a.batch + kThreads - 1) / kThreads;
    const int b0 = min(a.batch, tid * run), b1 = min(a.batch, b0 + run);
    int sum = 0;
    for (int b = b0; b < b1; ++b) sum += paged_tiles<kTile>(paged_rows(a, b));
    int upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += up;
    }
    if (lane == 31) scratch[warp] = upto;
    __syncthreads();
    int before = upto - sum, total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        before += w < warp ? scratch[w] : 0;
        total += scratch[w];
    }
    total *= a.kv_heads;
    const int ctas = min(static_cast<int>(gridDim.x), total);
    const int first = paged_first(blockIdx.x, total, ctas), last = paged_first(blockIdx.x + int64_t{1}, total, ctas);
    if (tid == 0 && static_cast<int>(blockIdx.x) >= ctas) *start = {0, 0, 0, 0, 0, total, ctas};
    if (static_cast<int>(blockIdx.x) < ctas && before * a.kv_heads <= first && first < (before + sum) * a.kv_heads) {
        PagedStart found = paged_locate<kTile>(a, b0, first - before * a.kv_heads);
        found.left = last - first;
        found.total = total;
        found.ctas = ctas;
        *start = found;
    }
    __syncthreads();
}

// Walks the CTA's tiles.
template <int kTile>
struct PagedCursor {
    int b, head, tile, left, rows, tiles;

    __host__ __device__ __forceinline__ void begin(const PagedStart& s) {
        b = s.b;
        head = s.head;
        tile = s.tile;
        left = s.left;
        rows = s.rows;
        tiles = paged_tiles<kTile>(rows);
    }
    // Tiles of the current unit that belong to this CTA, from the current one on.
    __host__ __device__ __forceinline__ int piece() const { return min(tiles - tile, left); }
    __host__ __device__ __forceinline__ void next(const PagedAttend& a) {
        --left;
        if (++tile < tiles || left == 0) return;
        tile = 0;
        if (++head == a.kv_heads) {
            head = 0;
            b = min(b + 1, a.batch - 1);
            rows = paged_rows(a, b);
            tiles = paged_tiles<kTile>(rows);
        }
    }
};

struct PagedRow {
    int page, head;
    uint32_t row;  // of the last tile of 2^31 - 1 rows, some are numbered beyond them
    int rows;      // of the sequence from `row` on
    bool any;      // a tile is left (the same for all lanes)

    __host__ __device__ __forceinline__ static PagedRow at(int head, int tile_row, int offset, int rows, bool any) {
        const uint32_t row = static_cast<uint32_t>(tile_row) + static_cast<uint32_t>(offset);
        return {-1, head, row, static_cast<int>(static_cast<uint32_t>(rows) - row), any};
    }
};

// How the 16-byte pieces of a row are exchanged in shared memory, so that the
// rows a load touches together lie in different banks.
struct Straight { static __device__ __forceinline__ int at(int piece, int) { return piece; } };
struct ByRow { static __device__ __forceinline__ int at(int piece, int row) { return piece ^ (row & 7); } };

// One warp's ring of row copies.  A stage holds R key rows and R value rows of
// DP elements.  Rows that are not visible are filled with zeros and have a 0 in
// the stage's mask.
//
// Where pages are multiples of R rows (`runs`), the R rows lie in one page: all
// lanes look up the first and step from row to row by the row stride.
// Otherwise lane r looks up row r and hands its place to the lanes that copy it,
// which costs the tensor-core kernels up to a tenth of their time (64 x 4096 rows
// of 4 KV heads of 256 BF16 dims: 184 us that way, 168 by runs).
template <typename P, int R, int DP, typename KeyPieces, typename ValuePieces>
struct PagedRing {
    static constexpr int kChunks = DP * static_cast<int>(sizeof(P)) / 16;  // 16-byte pieces of a row
    static constexpr int kHalf = R * DP;                                   // elements of the keys, and of the values
    static constexpr int kBytes = 2 * kHalf * static_cast<int>(sizeof(P));

    static __device__ __forceinline__ bool runs(const PagedAttend& a) { return a.page_size.divisor % R == 0u; }

    // This lane's row of a tile (the first one of a run), its page looked up one
    // tile before the copies start.  The cursor moves on.
    template <int kTile>
    static __device__ __forceinline__ PagedRow look(const PagedAttend& a, PagedCursor<kTile>& at) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        const int mine = runs(a) ? 0 : lane;
        PagedRow r = PagedRow::at(at.head, at.tile * kTile, warp * R + mine, at.rows, at.left > 0);
        if (!r.any) return r;
        if (mine < R && r.rows > 0) r.page = a.table[at.b * a.table_stride + a.page_size.quotient(r.row)];
        at.next(a);
        return r;
    }

    static __device__ __forceinline__ void fetch(const PagedAttend& a, P* stage, uint32_t* mask, const PagedRow& at) {
        constexpr int kSteps = (R * kChunks + 31) / 32, kElements = 16 / static_cast<int>(sizeof(P));
        const int lane = threadIdx.x & 31;
        if (!at.any) return;
        uint32_t slot;
        a.page_size.quotient(at.row & 0x7fffffffu, &slot);  // a row with a page is below 2^31
        const uint32_t head = a.share.quotient(static_cast<uint32_t>(at.head));
        const P* keys = static_cast<const P*>(a.keys);
        const P* values = static_cast<const P*>(a.values);
        const int width = a.dim / kElements;
        const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(stage));
        if (runs(a)) {
            const int page = at.page >= 0 && at.page < a.pages ? at.page : 0;
            const int count = page != at.page ? 0 : min(at.rows, R);  // visible rows
            if (lane == 0) *mask = (1u << count) - 1u;
            const int r0 = lane / kChunks, col0 = lane % kChunks;
            keys += page * a.ks[0] + head * a.ks[1] + (slot + r0) * a.ks[2] + col0 * kElements;
            values += page * a.vs[0] + head * a.vs[1] + (slot + r0) * a.vs[2] + col0 * kElements;
            constexpr int kAcross = kChunks > 32 ? kChunks / 32 : 1, kDown = kChunks > 32 ? 1 : 32 / kChunks;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const int r = r0 + i / kAcross * kDown, col = col0 + i % kAcross * 32;
                if (r < R && col < width) {
                    const uint32_t bytes = r < count ? 16u : 0u;
                    copy16(to + (r * kChunks + KeyPieces::at(col, r)) * 16, keys + i % kAcross * 32 * kElements, bytes);
                    copy16(to + (R * kChunks + r * kChunks + ValuePieces::at(col, r)) * 16,
                           values + i % kAcross * 32 * kElements, bytes);
                }
                if (i % kAcross == kAcross - 1) {
                    keys += kDown * a.ks[2];
                    values += kDown * a.vs[2];
                }
            }
            return;
        }
        const bool visible = lane < R && at.page >= 0 && at.page < a.pages;
        const unsigned seen = __ballot_sync(0xffffffffu, visible);
        if (lane == 0) *mask = seen;
        const int64_t koff = visible ? at.page * a.ks[0] + head * a.ks[1] + slot * a.ks[2] : 0;
        const int64_t voff = visible ? at.page * a.vs[0] + head * a.vs[1] + slot * a.vs[2] : 0;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int c = lane + 32 * i, r = c / kChunks, col = c % kChunks;
            const int64_t ko = __shfl_sync(0xffffffffu, koff, r);
            const int64_t vo = a.alike ? ko : __shfl_sync(0xffffffffu, voff, r);
            if (r < R && col < width) {
                const uint32_t bytes = (seen >> r) & 1u ? 16u : 0u;
                copy16(to + (r * kChunks + KeyPieces::at(col, r)) * 16, keys + ko + col * kElements, bytes);
                copy16(to + (R * kChunks + r * kChunks + ValuePieces::at(col, r)) * 16, values + vo + col * kElements,
                       bytes);
            }
        }
    }

    // The first to leave L2, since as a rule nobody reads a row again soon (64
    // sequences of 512-4096 FP32 rows, twelve caches in turn: 46.4 us without the
    // hint, 44.9 with it).  Parts of a group of more than 16 heads and sequences that
    // share pages do; what the hint costs them has not been measured.
    static __device__ __forceinline__ void copy16(uint32_t dst, const P* src, uint32_t bytes) {
        uint64_t streamed;
        asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(streamed));
        asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(bytes),
                     "l"(streamed)
                     : "memory");
    }
};

__device__ __forceinline__ void paged_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Lets the merge launch start as soon as CTAs of this one make room.
__device__ __forceinline__ void paged_launch_merge() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void paged_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A warp's copies: the ring, the look-ahead, the place of the present stage.
template <typename Ring, typename P, int kTile, int kStages>
struct PagedStream {
    const PagedAttend& a;
    P* ring;
    uint32_t* masks;
    PagedCursor<kTile> ahead, now;
    PagedRow upcoming;
    int slot_in, slot;

    __device__ __forceinline__ PagedStream(const PagedAttend& args, const PagedStart& start, P* ring_, uint32_t* masks_)
        : a(args), ring(ring_), masks(masks_), slot_in(kStages - 1), slot(0) {
        ahead.begin(start);
        now = ahead;
        PagedRow rows[kStages];  // all the first look-ups at once
#pragma unroll
        for (int i = 0; i < kStages; ++i) rows[i] = Ring::look(a, ahead);
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) {
            Ring::fetch(a, ring + i * 2 * Ring::kHalf, &masks[i], rows[i]);
            paged_commit();
        }
        upcoming = rows[kStages - 1];
    }
    // Starts the copies of the stage that is kStages - 1 further on and waits
    // for the present one.
    __device__ __forceinline__ void advance() {
        const PagedRow at = upcoming;
        upcoming = Ring::look(a, ahead);
        Ring::fetch(a, ring + slot_in * 2 * Ring::kHalf, &masks[slot_in], at);
        paged_commit();
        slot_in = slot_in + 1 == kStages ? 0 : slot_in + 1;
        paged_wait<kStages - 1>();
        __syncwarp();
    }
    __device__ __forceinline__ const P* keys() const { return ring + slot * 2 * Ring::kHalf; }
    __device__ __forceinline__ uint32_t mask() const { return masks[slot]; }
    // The present stage may be overwritten.
    __device__ __forceinline__ void release() {
        __syncwarp();
        slot = slot + 1 == kStages ? 0 : slot + 1;
        now.next(a);
    }
};

// Joins the states that the warps of a CTA have at the end of a piece: `count`
// tiles of the unit's `tiles` from `first` on; `last`: the CTA has no more.
// states[w][h] is warp w's (max, sum, output) of head h, dim + 2 floats.
template <typename T, int kTile, int kWarps>
__device__ __forceinline__ void paged_join(const PagedAttend& a, const PagedStart& start, float* states, int b,
                                           int head, int first, int count, int tiles, bool last) {
    __syncthreads();
    const int width = a.dim + 2, stride = a.group * width;
    const bool whole = first == 0 && count == tiles;
    float* piece = paged_pieces(a) + static_cast<int64_t>(2 * blockIdx.x + (first == 0 ? 1 : 0)) * stride;
    T* out = static_cast<T*>(a.out) + (static_cast<int64_t>(b) * a.heads + head * a.group) * a.dim;
    for (int i = threadIdx.x; i < a.group * a.dim; i += 32 * kWarps) {
        uint32_t d;
        const int h = static_cast<int>(a.per_head.quotient(static_cast<uint32_t>(i), &d));
        const float* s = states + h * width;
        float m = s[0];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) m = fmaxf(m, s[w * stride]);
        const float base = m == -INFINITY ? 0.0f : m;
        float l = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = exp2f(s[w * stride] - base);
            l = fmaf(s[w * stride + 1], f, l);
            o = fmaf(s[w * stride + 2 + d], f, o);
        }
        if (whole) {
            out[i] = from_float<T>(l == 0.0f ? 0.0f : o / l);
        } else {
            piece[h * width + 2 + d] = o;
            if (d == 0) {
                piece[h * width] = m;
                piece[h * width + 1] = l;
            }
        }
    }
    if (threadIdx.x == 0 && (last || first == 0)) {
        // For the merge kernel: the unit that starts in this CTA and ends in another.
        const bool open = first == 0 && !whole;
        const int64_t end = int64_t{paged_first(blockIdx.x + int64_t{1}, start.total, start.ctas)} + (tiles - count) - 1;
        const int to = open ? paged_owner(end, start.total, start.ctas) : -1;
        int* note = reinterpret_cast<int*>(a.workspace) + blockIdx.x * kPagedDescriptor;
        if (last) {
            note[0] = b;
            note[1] = head;
            note[2] = to;
            note[3] = open ? 1 : 0;
        }
        const int64_t unit = static_cast<int64_t>(b) * a.kv_heads + head;
        if (first == 0 && unit < kPagedUnits) {
            int* place = reinterpret_cast<int*>(a.workspace) + kPagedMaxGrid * kPagedDescriptor + 2 * unit;
            place[0] = blockIdx.x;
            place[1] = to;
        }
    }
    __syncthreads();  // the states may be overwritten
}

// A CTA without tiles.
__device__ __forceinline__ void paged_describe_none(const PagedAttend& a) {
    if (threadIdx.x == 0) reinterpret_cast<int*>(a.workspace)[blockIdx.x * kPagedDescriptor + 3] = 0;
}

// Joins the units that span CTAs of a launch of `ctas` (paged_attention.cu).
template <typename T>
fx_status launch_paged_merge(const PagedAttend& a, int ctas, cudaStream_t stream);

// Each in a file of its own.
fx_status launch_paged_f32(const PagedAttend& a, int sms, cudaStream_t stream);       // FP32 pages, group <= 4
fx_status launch_paged_f32_wide(const PagedAttend& a, int sms, cudaStream_t stream);  // FP32 pages, any group
fx_status launch_paged_bf16(const PagedAttend& a, int sms, cudaStream_t stream);
fx_status launch_paged_f16(const PagedAttend& a, int sms, cudaStream_t stream);
fx_status launch_paged_f32_on_bf16(const PagedAttend& a, int sms, cudaStream_t stream);
fx_status launch_paged_f32_on_f16(const PagedAttend& a, int sms, cudaStream_t stream);

// Whether units stay whole, which saves the merge launch: always up to 256 rows,
// four tiles of 64, which take a CTA about as long as that launch (64 sequences of
// 256 rows of 3 KV heads: 10.4 us whole, 14.4 in pieces); and up to 512 rows where
// the units about fill the GPU (64 sequences of 500: 16.5 and 18.4; 8: 12.4 and
// 10.3; 128: 28.3 and 26.0).
constexpr int64_t kWholeRows = 256;
inline bool paged_whole(const PagedAttend& a, int sms) {
    const int64_t units = static_cast<int64_t>(a.batch) * a.kv_heads;
    return a.capacity <= kWholeRows || (a.capacity <= 2 * kWholeRows && 2 * units >= sms && units <= 2 * sms);
}

// CTAs of a launch: `per_sm` on every SM, but no more than there can be tiles
// (or units).
template <int kTile>
inline int paged_grid(const PagedAttend& a, int sms, int per_sm) {
    const int64_t most =
        static_cast<int64_t>(a.batch) * a.kv_heads * (a.whole ? 1 : paged_tiles<kTile>(a.capacity));
    int64_t grid = static_cast<int64_t>(sms) * per_sm;
    if (grid > kPagedMaxGrid) grid = kPagedMaxGrid;
    return static_cast<int>(grid < most ? grid : most);
}

}  // namespace fx
