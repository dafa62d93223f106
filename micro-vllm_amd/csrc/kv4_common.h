// kv4_common.h -- device helpers of the 4-bit key/value cache's kernels.
#pragma once

#include "kv4.h"
#include "mfma_common.h"

namespace mvllm_hip {

// t / page for pages of a multiple of 16 tokens up to 1024: with u = t / 16 < 2^26 and
// p = page / 16 <= 64, floor(u / p) = floor(u * M / 2^32) for M = floor(2^32 / p) + 1, since
// M * p exceeds 2^32 by at most p and u * p < 2^32.  p = 1 would need M = 2^32 + 1: rcp is 0.
inline uint32_t kv4_page_rcp(int page) {
    const uint32_t p = (uint32_t)page / 16;
    return p == 1 ? 0u : (uint32_t)((uint64_t(1) << 32) / p) + 1u;
}
__device__ __forceinline__ int kv4_page_of(const Kv4View &c, int t) {
    const uint32_t u = (uint32_t)t >> 4, q = __umulhi(u, c.rcp);
    return (int)(c.rcp ? q : u);
}

// The pool page of a sequence's page pg, or -1 where there is none.
__device__ __forceinline__ int kv4_phys(const Kv4View &c, const int *row, int max_pages, int pg) {
    if ((unsigned)pg >= (unsigned)max_pages)
        return -1;
    const int p = row[pg];
    return (unsigned)p < (unsigned)c.n_pages ? p : -1;
}

// Row (page, head, slot) of the cache.
__device__ __forceinline__ size_t kv4_row(const Kv4View &c, int phys, int head, int slot) {
    return ((size_t)phys * c.n_kv + head) * c.page + slot;
}

// A sequence's tokens that have a place: its length, within its table.
__device__ __forceinline__ int kv4_len(const Kv4View &c, int len, int max_pages) {
    return max(0, min(len, max_pages * c.page));
}

template <typename T> struct Vec8;  // 8 consecutive elements as f32
template <> struct Vec8<float> {
    static __device__ __forceinline__ void load(const float *p, float (&x)[8]) {
        const float4 a = reinterpret_cast<const float4 *>(p)[0];
        const float4 b = reinterpret_cast<const float4 *>(p)[1];
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
    static __device__ __forceinline__ void store(float *p, const float (&x)[8]) {
        reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
};
template <> struct Vec8<__bf16> {
    static __device__ __forceinline__ void load(const __bf16 *p, float (&x)[8]) {
        const bf16x8 a = *reinterpret_cast<const bf16x8 *>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] = (float)a[i];
    }
    static __device__ __forceinline__ void store(__bf16 *p, const float (&x)[8]) {
        bf16x8 a;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            a[i] = (__bf16)x[i];
        *reinterpret_cast<bf16x8 *>(p) = a;
    }
};

}  // namespace mvllm_hip
