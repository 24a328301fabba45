// bfft_cache.cuh -- what the position and cache kernels share: element types,
// packed loads, the 8-bit codes, the views of a paged cache and of ragged
// sequences, and the search for the sequence of a row.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "../../include/bfft.h"
#include "bfft_async.cuh"

namespace bfft {

// ---------------------------------------------------------------- element types
template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// P values moved by one load or store of P * sizeof(T) <= 16 bytes.
template <typename T, int P>
struct alignas(sizeof(T) * P) Pack {
    T v[P];
};

// ---------------------------------------------------------------- 8-bit codes
// A block (one page of one kv head) of codes c with the scale s stands for
// c * s.  Int8 codes are symmetric (+-127); e4m3 codes use +-448.
enum : int { kCodeInt8 = 0, kCodeE4m3 = 1 };

__device__ __forceinline__ float finite(float v) { return fmaxf(v, -3.0e38f); }  // NaN becomes a number

template <int CODE>
struct CodeRange {
    static constexpr float most = CODE == kCodeInt8 ? 127.f : 448.f;
};

// Codes of P values within the block's range (|v| <= most but for the last bit of
// a product; ties to even).  Int8: v + 1.5 * 2^23 leaves the integer in the low
// byte.  NaN gives any code but e4m3's NaN: its block reads as NaN through the scale,
// and a NaN code would reach rows that do not see its token.
template <int CODE, int P>
__device__ __forceinline__ Pack<uint8_t, P> to_codes(const float* v) {
    Pack<uint8_t, P> c;
    if constexpr (CODE == kCodeInt8) {
        uint32_t w[P];
#pragma unroll
        for (int i = 0; i < P; ++i) w[i] = __float_as_uint(__fadd_rn(v[i], 12582912.f));
        if constexpr (P % 4 == 0) {
            uint32_t* q = reinterpret_cast<uint32_t*>(&c);
#pragma unroll
            for (int i = 0; i < P; i += 4)
                q[i / 4] = __byte_perm(__byte_perm(w[i], w[i + 1], 0x0040), __byte_perm(w[i + 2], w[i + 3], 0x0040), 0x5410);
        } else {
#pragma unroll
            for (int i = 0; i < P; ++i) c.v[i] = static_cast<uint8_t>(w[i]);
        }
    } else if constexpr (P % 4 == 0) {
        uint32_t* q = reinterpret_cast<uint32_t*>(&c);
#pragma unroll
        for (int i = 0; i < P; i += 4) {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(finite(v[i]), finite(v[i + 1])), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(finite(v[i + 2]), finite(v[i + 3])), __NV_SATFINITE, __NV_E4M3);
            q[i / 4] = lo | (hi << 16);
        }
    } else {
#pragma unroll
        for (int i = 0; i < P; ++i)
            c.v[i] = static_cast<uint8_t>(__nv_cvt_float_to_fp8(finite(v[i]), __NV_SATFINITE, __NV_E4M3));
    }
    return c;
}

// Nearest code of v (ties to even), saturating.
template <int CODE>
__device__ __forceinline__ uint8_t to_code(double v) {
    if constexpr (CODE == kCodeInt8) {
        const int q = __double2int_rn(v);  // NaN gives some code: its block reads as NaN through the scale
        return static_cast<uint8_t>(static_cast<int8_t>(q < -127 ? -127 : (q > 127 ? 127 : q)));
    } else {
        return static_cast<uint8_t>(__nv_cvt_double_to_fp8(v == v ? v : 0.0, __NV_SATFINITE, __NV_E4M3));
    }
}
template <int CODE>
__device__ __forceinline__ float code_value(uint8_t c) {
    if constexpr (CODE == kCodeInt8) {
        return static_cast<float>(static_cast<int8_t>(c));
    } else {
        return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
    }
}

// ---------------------------------------------------------------- views
struct CacheView {
    uint8_t* k;       // codes [pages][kv_heads][page][dim]
    uint8_t* v;
    float* k_scale;   // [pages][kv_heads]
    float* v_scale;
    int64_t pages;
    int kv_heads;
    int page_log2;
    int dim;
};

struct SequenceView {
    const int32_t* block_table;  // [seqs][max_pages]: the page of each run of `page` tokens
    int64_t table_stride;
    const int32_t* lens;         // [seqs]
    const int32_t* starts;       // [seqs + 1]: first ragged row of each sequence
    int seqs;
    int max_pages;
    int64_t tokens;              // ragged rows
};

// The sequence of ragged row t: the largest s with starts[s] <= t (the one that
// owns the row, also next to sequences without rows).  All 32 lanes call it with
// the same t and get the same answer; each round looks at 32 evenly spaced
// starts, so 1024 sequences take two rounds of one load instead of ten.
__device__ __forceinline__ int find_sequence(const int32_t* __restrict__ starts, int seqs, int64_t t) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = seqs;
    while (n > 1) {
        const int step = (n + 31) >> 5;
        const int i = lane * step;
        const bool le = i < n && starts[lo + i] <= t;
        const int c = __popc(__ballot_sync(0xffffffffu, le));
        const int skip = (c > 0 ? c - 1 : 0) * step;
        lo += skip;
        n = n - skip < step ? n - skip : step;
    }
    return lo;
}

// Page that holds token `pos` of sequence s, or -1 where the table has no valid
// entry for it (such a token is neither written nor read).
__device__ __forceinline__ int64_t page_of(const SequenceView& q, const CacheView& c, int s, int64_t pos) {
    const int64_t i = pos >> c.page_log2;
    if (pos < 0 || i >= q.max_pages) return -1;
    const int64_t p = q.block_table[s * q.table_stride + i];
    return p >= 0 && p < c.pages ? p : -1;
}

// Launch as a programmatic dependent of the kernel before on the stream: this one's
// CTAs may take their places while that one drains (append and read of 8 tokens
// 12.3 -> 10.0 us, a decode over 700 tokens 10.2 -> 8.5).  Every kernel launched so
// begins with griddep_wait(), so nothing of it is read or written earlier.
template <typename... P, typename... A>
inline cudaError_t launch_dependent(void (*kernel)(P...), unsigned grid, dim3 block, size_t smem, cudaStream_t s,
                                    const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3(grid);
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Host side (bfft_rotary.cu).  An error's text goes to bfft_last_error(); the runtime's
// own record of it is cleared, so that the next call on this thread does not report it.
bfft_status fail(bfft_status st, const char* fmt, ...);
bfft_status launched(cudaError_t e, const char* call);  // the status of a call's launches
inline bool aligned(const void* p, int64_t bytes) {
    return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0;
}

// The call's device, and the caller's again when the call returns.
struct Device {
    int prev = -1;
    bool ok = true, changed = false;
    explicit Device(int64_t dev);
    ~Device();
};

// The checks that every call on a cache makes.
bfft_status check_cache(const bfft_cache_desc* c);
bfft_status check_sequences(const bfft_sequence_desc* q);
CacheView cache_view(const bfft_cache_desc* c);
SequenceView sequence_view(const bfft_sequence_desc* q);

}  // namespace bfft
