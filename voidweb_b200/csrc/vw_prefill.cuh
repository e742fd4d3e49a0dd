// vw_prefill.cuh -- small helpers that the prefill kernels share.
#pragma once
#include <cstdint>

#include "vw_internal.h"
#include "vw_ptx.cuh"

namespace vw {

namespace {

constexpr int pf_align(int x, int a) { return (x + a - 1) / a * a; }

template <int IO>
__device__ __forceinline__ float pf_io_to_f32(uint32_t h) {
    return IO == kBF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
}
template <int IO>
__device__ __forceinline__ uint16_t pf_f32_to_io(float f) {
    return IO == kBF16 ? f32_to_bf16_bits(f) : f32_to_f16_bits(f);
}

// Largest b with pfx[b] <= x over b in [0, B).
__device__ __forceinline__ int pf_find(const int* pfx, int B, int x) {
    int lo = 0, hi = B - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (pfx[mid] <= x) lo = mid; else hi = mid - 1;
    }
    return lo;
}

}  // namespace

}  // namespace vw
