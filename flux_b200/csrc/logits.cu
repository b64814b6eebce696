// Penalties, bias and token mask on a step's logits.
//
// Reading and writing HBM bounds it (a few operations per logit), if the
// history does not get in the way: which tokens a row has seen, and how often,
// has to be known before the first logit is stored.  A CTA takes a part of a
// row's vocabulary at a time, with a 16-bit counter per token in shared
// memory, and reads the row's whole history for it (from L2: the row's other
// parts read it too).  Counters are integers: their order does not matter.
//
// Counting is a chain of waits that would leave HBM idle, so a CTA counts for
// its next part while it handles the present one: the next tokens are loaded
// and the next logits sent for (into L2) first, then the present logits are
// processed, then the tokens are counted into the second set of counters.
// Logits go in pieces of 16 bytes from wherever a row's first 16-byte boundary
// lies, since a vocabulary need not be a multiple of anything; the few logits
// before and after are handled one by one.
#include "paged.cuh"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace fx {
namespace {

constexpr int64_t kMostCounters = 98304;  // bytes of the counters of an SM's CTAs, one set each

struct LogitsArgs {
    const void* logits;
    void* output;
    int64_t vocab, in_stride, out_stride;
    const int64_t* tokens;
    int64_t history, tokens_stride;
    const int64_t* prompts;
    const int64_t* lengths;
    const float* penalties;
    const float* bias;
    int64_t bias_stride;
    const int32_t* allowed;
    int64_t allowed_stride;
    int64_t part;  // tokens of a part, a multiple of 32
    FastDivide parts;  // of a row
    int items;         // parts of all rows
    int counter_bytes;
};

// A counter: the top bit says that the prompt has the token, the rest how
// often it was emitted.
template <typename C>
constexpr uint32_t kPrompt = 1u << (8 * sizeof(C) - 1);

struct Penalties { float repetition, inverse, presence, frequency; };

__device__ __forceinline__ Penalties penalties_of(const LogitsArgs& a, int row) {
    const float* p = a.penalties + 3 * static_cast<int64_t>(row);
    return {p[0], __frcp_rn(p[0]), p[1], p[2]};
}

// FP32 in the order of the definition: a division or a product, then the product
// that the frequency adds and two differences, each rounded on its own.
//
// The quotient: with the divisor's reciprocal y rounded to nearest, q = x y and
// its remainder r = x - q d, which a fused product gives exactly, q + r y is the
// quotient rounded to nearest (Markstein, 1990), except for divisors whose
// mantissa is all ones or whose reciprocal is no normal number: off by one step of
// FP32 at most there.  A division per seen logit would be slower (1 x 49152 FP32
// logits 5.5 us, 4.8 in this way).  16-bit logits take q as it is: one step of FP32
// is far below their own rounding (256 x 100277 BF16 logits 55.5 us, 57.2 with the
// remainder).
template <typename T>
__device__ __forceinline__ float divided(float x, const Penalties& p) {
    const float q = x * p.inverse;
    if constexpr (sizeof(T) == 2) return q;
    const float near = fmaf(fmaf(-q, p.repetition, x), p.inverse, q);
    return q < INFINITY ? near : q;  // an infinite q has no remainder
}
template <typename T, typename C>
__device__ __forceinline__ float penalised(float x, uint32_t count, const Penalties& p) {
    x = x > 0.0f ? divided<T>(x, p) : x * p.repetition;
    const uint32_t n = count & (kPrompt<C> - 1u);
    if (n != 0u) x = __fsub_rn(__fsub_rn(x, __fmul_rn(p.frequency, static_cast<float>(n))), p.presence);
    return x;
}

// Asks for `bytes` (a multiple of 16) from a 16-byte boundary on to be brought into L2.
__device__ __forceinline__ void prefetch_l2(const void* from, int bytes) {
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(from), "r"(bytes) : "memory");
}

// Where one part of one row lies.  Logits [lead, lead + N * pieces) of the part
// go in pieces; parts start at multiples of 32 tokens.
template <typename T>
struct Part {
    static constexpr int N = 16 / sizeof(T);
    const T* in;
    T* out;
    const float* bias;
    const uint32_t* allowed;
    int64_t first;
    int row, n, lead, pieces, bias_pieces;

    __device__ __forceinline__ void find(const LogitsArgs& a, int item) {
        row = static_cast<int>(a.parts.quotient(static_cast<uint32_t>(item)));
        first = (item - row * static_cast<int>(a.parts.divisor)) * a.part;
        const int64_t rest = a.vocab - first;
        n = static_cast<int>(rest < 0 ? 0 : (rest < a.part ? rest : a.part));
        in = static_cast<const T*>(a.logits) + row * a.in_stride + first;
        out = static_cast<T*>(a.output) + row * a.out_stride + first;
        bias = a.bias == nullptr ? nullptr : a.bias + row * a.bias_stride + first;
        allowed = a.allowed == nullptr
                      ? nullptr
                      : reinterpret_cast<const uint32_t*>(a.allowed) + row * a.allowed_stride + first / 32;
        const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(in) / sizeof(T) % N);
        const bool alike = static_cast<int>(reinterpret_cast<uintptr_t>(out) / sizeof(T) % N) == skew;
        lead = alike ? (N - skew) % N : 0;
        pieces = alike && n > lead ? (n - lead) / N : 0;
        bias_pieces = reinterpret_cast<uintptr_t>(bias + lead) % 16 == 0;
    }
    // Counters of a piece lie on a 16-byte boundary.
    __device__ __forceinline__ int pad() const { return (N - lead) % N; }
    __device__ __forceinline__ void prefetch() const {
        if (pieces == 0) return;
        prefetch_l2(in + lead, pieces * 16);
        if (bias != nullptr && bias_pieces) prefetch_l2(bias + lead, pieces * N * 4);
    }
};

template <typename T>
__device__ __forceinline__ float finished(float v, const Part<T>& part, uint32_t at) {
    if (part.bias != nullptr) v += part.bias[at];
    if (part.allowed != nullptr && !((part.allowed[at / 32] >> (at % 32)) & 1u)) v = -INFINITY;
    return v;
}

// Word i of four that lie in registers.
__device__ __forceinline__ uint32_t pick(const uint4& w, uint32_t i) {
    const uint32_t low = i & 1u ? w.y : w.x, high = i & 1u ? w.w : w.z;
    return i & 2u ? high : low;
}

// Stores logit e of the piece at `at` once more, with its penalties.
template <typename T, typename C>
__device__ __forceinline__ void replace(const Part<T>& part, const uint4& raw, uint32_t at, uint32_t e,
                                        uint32_t count, uint32_t mask, const Penalties& p) {
    float x;
    if constexpr (sizeof(T) == 4) {
        x = __uint_as_float(pick(raw, e));
    } else {
        const uint32_t half = pick(raw, e >> 1) >> (16u * (e & 1u));
        const uint16_t bits = static_cast<uint16_t>(half);
        x = to_float(*reinterpret_cast<const T*>(&bits));
    }
    x = penalised<T, C>(x, count, p);
    if (part.bias != nullptr) x += part.bias[at + e];
    part.out[at + e] = from_float<T>((mask >> e) & 1u ? x : -INFINITY);
}

// Replaces the logits of the piece at `at` that have a counter, and clears it.
// Few have, so the lanes of a warp take theirs one by one, side by side.
template <typename T, typename C>
__device__ __forceinline__ void replace_seen(const Part<T>& part, const uint4& raw, uint32_t at, C* counts,
                                             uint32_t mask, const Penalties& p) {
    constexpr int N = Part<T>::N;
    if constexpr (sizeof(C) == 2) {
        using Words = std::conditional_t<N == 8, uint4, uint2>;
        Words& stored = *reinterpret_cast<Words*>(counts + at);
        const Words words = stored;
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&words);
        uint32_t seen = 0u;  // bit e: logit e has a counter
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            // The top bit of each half that is not 0.
            const uint32_t top = (((w[i] & 0x7fff7fffu) + 0x7fff7fffu) | w[i]) & 0x80008000u;
            seen |= (top >> (15 - 2 * i) | top >> (30 - 2 * i)) & (3u << (2 * i));
        }
        if (seen != 0u) stored = Words{};
        while (seen != 0u) {
            const uint32_t e = __ffs(static_cast<int>(seen)) - 1;
            seen &= seen - 1u;
            uint4 four;
            if constexpr (N == 8) four = words;
            else four = make_uint4(words.x, words.y, 0u, 0u);
            const uint32_t count = (pick(four, e >> 1) >> (16u * (e & 1u))) & 0xffffu;
            replace<T, C>(part, raw, at, e, count, mask, p);
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const uint32_t count = counts[at + e];
            if (count != 0u) {
                counts[at + e] = 0u;
                replace<T, C>(part, raw, at, e, count, mask, p);
            }
        }
    }
}

// The logits of a part.  counts[i] counts token i; what was counted is cleared
// again, since only the thread that handles a logit reads its counter.  C: the
// counters' type, void without a history.
template <typename T, typename C, int kThreads>
__device__ __forceinline__ void process(const Part<T>& part, void* counters, const Penalties& p) {
    constexpr bool kHistory = !std::is_void<C>::value;
    using Counter = std::conditional_t<kHistory, C, uint32_t>;
    constexpr int N = Part<T>::N;
    constexpr int kPieces = 8 / N;  // loaded together: 8 logits of a thread
    Counter* counts = static_cast<Counter*>(counters) + part.pad();
    const T* in = part.in;
    T* out = part.out;
    const float* bias = part.bias;
    const uint32_t* allowed = part.allowed;
    const int lead = part.lead, pieces = part.pieces, tail = lead + pieces * N;
    // The logits outside the pieces (all of them if input and output rows lie
    // differently to 16-byte boundaries).
    const int singles = min(lead, part.n) + max(part.n - tail, 0);
    for (int i = threadIdx.x; i < singles; i += kThreads) {
        const int at = i < lead ? i : tail + i - lead;
        float v = to_float(in[at]);
        if constexpr (kHistory) {
            const uint32_t c = counts[at];
            if (c != 0u) {
                v = penalised<T, C>(v, c, p);
                counts[at] = 0;
            }
        }
        out[at] = from_float<T>(finished<T>(v, part, at));
    }
    for (int k0 = threadIdx.x; k0 < pieces; k0 += kPieces * kThreads) {
        uint4 raw[kPieces];
        float add[kPieces][N];
        uint32_t low[kPieces], high[kPieces];
#pragma unroll
        for (int u = 0; u < kPieces; ++u) {
            const int k = k0 + u * kThreads;
            if (k >= pieces) continue;
            const uint32_t at = static_cast<uint32_t>(lead + k * N);
            raw[u] = *reinterpret_cast<const uint4*>(in + at);
            if (bias != nullptr) {
                if (part.bias_pieces) {
#pragma unroll
                    for (int e = 0; e < N; e += 4) {
                        const float4 four = *reinterpret_cast<const float4*>(bias + at + e);
                        add[u][e] = four.x;
                        add[u][e + 1] = four.y;
                        add[u][e + 2] = four.z;
                        add[u][e + 3] = four.w;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < N; ++e) add[u][e] = bias[at + e];
                }
            }
            low[u] = high[u] = 0xffffffffu;
            if (allowed != nullptr) {
                low[u] = allowed[at / 32];
                high[u] = allowed[(at + N - 1) / 32];
            }
        }
#pragma unroll
        for (int u = 0; u < kPieces; ++u) {
            const int k = k0 + u * kThreads;
            if (k >= pieces) break;
            const uint32_t at = static_cast<uint32_t>(lead + k * N);
            const uint32_t mask = __funnelshift_r(low[u], high[u], at % 32);
            const T* x = reinterpret_cast<const T*>(&raw[u]);
            uint4 packed;
            T* z = reinterpret_cast<T*>(&packed);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                float y = to_float(x[e]);
                if (bias != nullptr) y += add[u][e];
                z[e] = from_float<T>((mask >> e) & 1u ? y : -INFINITY);
            }
            *reinterpret_cast<uint4*>(out + at) = packed;
            if constexpr (kHistory) replace_seen<T, C>(part, raw[u], at, counts, mask, p);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) logits_plain_kernel(const __grid_constant__ LogitsArgs a) {
    grid_dependency_wait();
    Part<T> part;
    part.find(a, blockIdx.x);
    process<T, void, 256>(part, nullptr, Penalties{});
}

constexpr int kTogether = 8;  // tokens a thread loads at once

template <int kThreads>
__device__ __forceinline__ void load_tokens(int64_t (&token)[kTogether], const LogitsArgs& a, int row, int i0) {
    const int64_t* tokens = a.tokens + row * a.tokens_stride + i0 + threadIdx.x;
    const int left = static_cast<int>(a.history) - i0 - static_cast<int>(threadIdx.x);
#pragma unroll
    for (int j = 0; j < kTogether; ++j) token[j] = j * kThreads < left ? tokens[j * kThreads] : -1;  // length not known yet
}

// Counts the history of a part; `token` holds its first tokens.
template <typename T, typename C, int kThreads>
__device__ __forceinline__ void count_history(int64_t (&token)[kTogether], const LogitsArgs& a, const Part<T>& part,
                                              void* counters) {
    const int length = static_cast<int>(max(int64_t{0}, min(a.lengths[part.row], a.history)));
    const int prompt = static_cast<int>(max(int64_t{0}, min(a.prompts[part.row], static_cast<int64_t>(length))));
    uint32_t* words = static_cast<uint32_t*>(counters);
    const uint32_t pad = part.pad();
    for (int64_t i0 = 0;;) {
        const int left = length - static_cast<int>(i0) - static_cast<int>(threadIdx.x);
        const int in_prompt = prompt - static_cast<int>(i0) - static_cast<int>(threadIdx.x);
#pragma unroll
        for (int j = 0; j < kTogether; ++j) {
            const uint64_t v = static_cast<uint64_t>(token[j] - part.first);
            if (j * kThreads >= left || v >= static_cast<uint64_t>(part.n)) continue;
            const uint32_t at = static_cast<uint32_t>(v) + pad;
            const uint32_t bit = sizeof(C) == 4 ? 0u : 16u * (at & 1u);
            uint32_t* word = words + (sizeof(C) == 4 ? at : at >> 1);
            if (j * kThreads < in_prompt)
                atomicOr(word, kPrompt<C> << bit);
            else
                atomicAdd(word, 1u << bit);
        }
        i0 += kTogether * kThreads;
        if (i0 >= length) break;
        load_tokens<kThreads>(token, a, part.row, static_cast<int>(i0));
    }
}

template <typename T, typename C, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) logits_history_kernel(const __grid_constant__ LogitsArgs a) {
    grid_dependency_wait();
    extern __shared__ __align__(16) unsigned char smem[];
    // The present part, the next one and the one after, found by one thread.
    __shared__ Part<T> parts[3];
    const int bytes = a.counter_bytes;  // of one set of counters, a multiple of 16
    const int step = static_cast<int>(gridDim.x);
    int64_t token[kTogether];
    int item = blockIdx.x, set = 0, now = 0;
    load_tokens<kThreads>(token, a, static_cast<int>(a.parts.quotient(static_cast<uint32_t>(item))), 0);
    if (threadIdx.x < 2 && item + static_cast<int>(threadIdx.x) * step < a.items) {
        parts[threadIdx.x].find(a, item + threadIdx.x * step);
        if (threadIdx.x == 0) parts[0].prefetch();
    }
    for (int i = threadIdx.x; i < bytes / 16 * (item + step < a.items ? 2 : 1); i += kThreads)
        reinterpret_cast<uint4*>(smem)[i] = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
    count_history<T, C, kThreads>(token, a, parts[0], smem);
    __syncthreads();
    for (;;) {
        const int next = now == 2 ? 0 : now + 1;
        const bool more = item + step < a.items;
        if (more) {
            if (threadIdx.x == 0) {
                parts[next].prefetch();
                if (item + 2 * static_cast<int64_t>(step) < a.items) parts[next == 2 ? 0 : next + 1].find(a, item + 2 * step);
            }
            load_tokens<kThreads>(token, a, parts[next].row, 0);
        }
        const Part<T> part = parts[now];
        process<T, C, kThreads>(part, smem + set * bytes, penalties_of(a, part.row));
        if (!more) break;
        set ^= 1;
        count_history<T, C, kThreads>(token, a, parts[next], smem + set * bytes);
        __syncthreads();  // the next set is counted, the present one cleared
        item += step;
        now = next;
    }
}

constexpr int64_t kSms = 148;
constexpr int64_t kLongHistory = 8192;

void set_parts(LogitsArgs& a, int64_t rows, int64_t parts) {
    a.part = ((a.vocab + parts - 1) / parts + 31) / 32 * 32;
    parts = (a.vocab + a.part - 1) / a.part;
    a.parts = FastDivide::by(parts);
    a.items = static_cast<int>(rows * parts);
}

template <typename T, typename C, int kThreads>
fx_status launch_history(LogitsArgs a, int64_t rows, cudaStream_t stream) {
    const auto up = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
    // Few logits: as many parts of 2048 tokens or more as there is room for CTAs.
    // Many: parts as large as two sets of counters allow, since each reads the
    // history again, or smaller down to half of that where that leaves the CTAs'
    // last round fuller.
    constexpr int64_t kPerSm = 1024 / kThreads, kCtas = kPerSm * kSms, kMost = kMostCounters / kPerSm;
    const int64_t low = up(a.vocab, kMost / static_cast<int64_t>(sizeof(C)));
    int64_t parts = std::min(up(a.vocab, 2048), kCtas / rows);
    if (parts < low) {
        int64_t work = INT64_MAX;
        for (int64_t n = low; n <= 2 * low; ++n) {
            const int64_t rounds = up(rows * n, kCtas) * up(a.vocab, n);
            if (rounds < work) {
                work = rounds;
                parts = n;
            }
        }
    }
    set_parts(a, rows, parts);
    a.counter_bytes = static_cast<int>(a.part * sizeof(C)) + 32;  // and the padding of a piece
    const int64_t grid = std::min<int64_t>(a.items, kCtas);
    const size_t smem = static_cast<size_t>(a.counter_bytes) * (a.items > grid ? 2 : 1);
    const fx_status st = raise_smem_limit(reinterpret_cast<const void*>(logits_history_kernel<T, C, kThreads>),
                                          2 * (kMost + 32), "raising the logits' shared memory");
    if (st != FX_OK) return st;
    return launch_dependent(logits_history_kernel<T, C, kThreads>, dim3(static_cast<unsigned>(grid)), dim3(kThreads), smem, stream,
                            "launching logits processing", a);
}

template <typename T>
fx_status launch_rows(LogitsArgs a, int64_t rows, cudaStream_t stream) {
    FX_REQUIRE(rows <= INT_MAX / ((a.vocab + 1023) / 1024 + 1), "fx_logits_process: rows * vocabulary is too large");
    // Two CTAs per SM, so that one handles logits while the other waits; for a
    // long history, which is read once for each part, one with parts twice as
    // large (256 rows of 100277 BF16 logits with 4096 tokens each: 56 us
    // in two, 57 in one; with 8192: 72 and 66; with 30000: 136 and 107).
    // 15 bits count any history below 32768; longer ones take 32-bit counters.
    if (a.tokens != nullptr) {
        if (a.history < kLongHistory) return launch_history<T, uint16_t, 512>(a, rows, stream);
        return a.history < (1 << 15) ? launch_history<T, uint16_t, 1024>(a, rows, stream)
                                     : launch_history<T, uint32_t, 1024>(a, rows, stream);
    }
    set_parts(a, rows, (a.vocab * static_cast<int64_t>(sizeof(T)) + 8191) / 8192);  // 8 KB of logits per CTA
    return launch_dependent(logits_plain_kernel<T>, dim3(a.items), dim3(256), 0, stream, "launching logits processing", a);
}

}  // namespace
}  // namespace fx

using namespace fx;

extern "C" fx_status fx_logits_process(const void* logits, int32_t dtype, int64_t rows, int64_t vocab,
                                       int64_t logits_stride, const int64_t* tokens, int64_t history,
                                       int64_t tokens_stride, const int64_t* prompt_lengths, const int64_t* lengths,
                                       const float* penalties, const float* bias, int64_t bias_stride,
                                       const int32_t* allowed, int64_t allowed_stride, void* output,
                                       int64_t output_stride, void* stream) {
    FX_REQUIRE(dtype == FX_F32 || dtype == FX_BF16 || dtype == FX_F16, "fx_logits_process: unknown type");
    FX_REQUIRE(rows >= 0 && vocab > 0, "fx_logits_process: the vocabulary must be non-empty");
    FX_REQUIRE(rows <= 65535 && vocab <= INT_MAX, "fx_logits_process: at most 65535 rows and 2^31 - 1 tokens");
    const bool history_given = tokens != nullptr;
    FX_REQUIRE(history_given == (prompt_lengths != nullptr) && history_given == (lengths != nullptr) &&
                   history_given == (penalties != nullptr),
               "fx_logits_process: tokens, prompt_lengths, lengths and penalties go together");
    FX_REQUIRE(!history_given || (history >= 0 && history <= INT_MAX), "fx_logits_process: history out of range");
    if (rows == 0) return FX_OK;
    FX_REQUIRE(logits && output, "fx_logits_process: null pointer");
    const LogitsArgs a{logits, output, vocab, logits_stride, output_stride, tokens, history, tokens_stride,
                       prompt_lengths, lengths, penalties, bias, bias_stride, allowed, allowed_stride, 0, {}, 0, 0};
    cudaStream_t s = as_stream(stream);
    if (dtype == FX_F32) return launch_rows<float>(a, rows, s);
    return dtype == FX_BF16 ? launch_rows<__nv_bfloat16>(a, rows, s) : launch_rows<__half>(a, rows, s);
}
