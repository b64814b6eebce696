// Shared pieces of the paged-cache operators: element types, the pools' checks
// and the lookup of a row in the pages.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>

#include "common.cuh"

namespace fx {

constexpr int64_t kPagedMaxDim = 256;
constexpr int64_t kPagedMaxGroup = 16;
constexpr int64_t kPagedMaxPageSize = 65536;

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }

// Round to nearest, ties to even: the one rounding of each stored result.
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

inline int64_t dtype_size(int32_t dtype) { return dtype == FX_F32 ? 4 : 2; }

// n / d for n < 2^31 and a divisor the host knows: with s = ceil(log2 d) and
// M = ceil(2^(31+s) / d), M d - 2^(31+s) < d <= 2^s, so n M / 2^(31+s) exceeds
// n / d by less than 1 / d.
struct FastDivide {
    uint32_t divisor, magic, shift;

    __host__ static FastDivide by(int64_t d) {
        uint32_t s = 0;
        while ((int64_t{1} << s) < d) ++s;
        return {static_cast<uint32_t>(d), static_cast<uint32_t>(((uint64_t{1} << (31 + s)) + d - 1) / d), 31 + s};
    }
    __host__ __device__ __forceinline__ uint32_t quotient(uint32_t n) const {
        return static_cast<uint32_t>((static_cast<uint64_t>(n) * magic) >> shift);
    }
    __host__ __device__ __forceinline__ uint32_t quotient(uint32_t n, uint32_t* remainder) const {
        const uint32_t q = quotient(n);
        *remainder = n - q * divisor;
        return q;
    }
};

// The page operations move whole pages: kv_heads and page_size are the outer
// dimensions of one contiguous block, in either order.
inline bool pages_are_blocks(const fx_pages& p, const int64_t* strides) {
    const int64_t head = strides[2], row = strides[3];
    if (p.kv_heads == 1 && p.page_size == 1) return true;
    if (p.kv_heads == 1) return row == p.head_dim;
    if (p.page_size == 1) return head == p.head_dim;
    return (row == p.head_dim && head == p.page_size * p.head_dim) ||
           (head == p.head_dim && row == p.kv_heads * p.head_dim);
}

// Checks what every paged operator asks of the pools; `op` prefixes messages.
fx_status check_pages(const char* op, const fx_pages* p, bool blocks);
// Checks a page table against the pools (or against `pages`, `page_size`).
fx_status check_table(const char* op, const int32_t* table, int64_t sequences, int64_t columns, int64_t stride,
                      int64_t page_size);

}  // namespace fx
