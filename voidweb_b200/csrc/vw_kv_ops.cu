// vw_kv_ops.cu -- byte-moving kernels of the paged KV pool: reshape-and-cache
// append, copy-on-write / compaction block copies, and the block-table gather.
//
// All three are HBM-bound copies: a warp moves whole token rows of one KV head
// (D elements) with 8-B or 16-B vector accesses, so it touches whole 32-B
// sectors, and keeps several rows' loads in flight before it stores them.  Pool layout:
//   data  [L][NB][Hkv][2][16][D]   (2 = K, V; element f16/bf16 or an E4M3 code)
//   scale [L][NB][Hkv][2][16]      (FP8 pools only)
// or, 4-bit pools, [L][NB][Hkv] records of codes and scales (vw_fp4.cuh).
// Bounds: every block id and slot is checked against the pool before it is
// used; a bad one sets a bit in the pool's device error word and the row is
// skipped, so no kernel here can write outside the pool.
#include <cuda_runtime.h>
#include <cstdint>

#include "vw_fp8.cuh"
#include "vw_internal.h"
#include "vw_ptx.cuh"
#include "vw_fp4.cuh"

namespace vw {

namespace {

__device__ __forceinline__ float io_f32(uint32_t h, uint32_t io) {
    return io == kBF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
}

// Row w of a launch over n tokens -> (token i, K or V, KV head h), with w in
// the order [token][K, V][head].  Index math is 32-bit (the host keeps the row
// count below 2^31): a 64-bit division costs ~100 instructions per warp, which
// bounded these short copies by issue rather than by memory.
struct RowIdx {
    uint32_t i, kv, h;
};
__device__ __forceinline__ RowIdx row_index(uint32_t w, uint32_t Hkv) {
    const uint32_t q = w / Hkv;
    return RowIdx{q >> 1, q & 1u, w - q * Hkv};
}

// Pool row (token slot t of block blk, head h, K or V) of a layer.
__device__ __forceinline__ uint64_t pool_row(const PoolGeom& g, uint32_t layer, uint32_t blk, uint32_t h,
                                             uint32_t kv, uint32_t t) {
    return ((((uint64_t)layer * g.num_blocks + blk) * g.num_kv_heads + h) * 2 + kv) * kBlockSize + t;
}

constexpr uint32_t kRowsPerWarp = 4;     // a warp's loads of 4 rows are in flight together

// The same with the division by Hkv as a product: floor(w / d) = (w * m) >> (31 + s) for
// w < 2^31, s = ceil(log2 d), m = ceil(2^(31 + s) / d) (Granlund and Montgomery).
struct HeadDiv {
    uint32_t d, m, s;
};
HeadDiv head_div(uint32_t d) {
    uint32_t s = 0;
    while ((1ull << s) < d) ++s;
    return HeadDiv{d, (uint32_t)(((1ull << (31 + s)) + d - 1) / d), s};
}
__device__ __forceinline__ RowIdx row_index(uint32_t w, const HeadDiv& h) {
    const uint32_t q = (uint32_t)(((uint64_t)w * h.m) >> (31 + h.s));
    return RowIdx{q >> 1, q & 1u, w - q * h.d};
}

// 4-bit record of (layer, block, head).
template <int D>
__device__ __forceinline__ uint64_t fp4_record(const PoolGeom& g, uint32_t layer, uint32_t blk, uint32_t h) {
    return (((uint64_t)layer * g.num_blocks + blk) * g.num_kv_heads + h) * Fp4Rec<D>::BYTES;
}

// Append to a 4-bit pool.  A warp takes kFp4Rows rows; a lane quantises a chunk of
// eight elements (16 B in, a word of codes out), D/8 lanes a row, with all its
// chunks' loads in flight first.  Two neighbouring lanes share a group's scale.
// Instructions bound it, not bytes: 8191 tokens of 8 KV heads of 128 elements
// take 11.7 us, 3.7 TB/s (12.7 with one element at a time).
constexpr uint32_t kFp4Rows = 8;

template <int D>
__global__ void __launch_bounds__(256) fp4_append_kernel(PoolGeom g, uint8_t* __restrict__ data, uint32_t layer,
                                                         const uint16_t* __restrict__ k_new,
                                                         const uint16_t* __restrict__ v_new,
                                                         const int64_t* __restrict__ slots, uint32_t n, HeadDiv hd,
                                                         uint32_t* err) {
    using R = Fp4Rec<D>;
    constexpr int WORDS = D / 8, N = kFp4Rows * WORDS / 32;      // chunks of a row, of a lane
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t w0 = (blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * kFp4Rows;
    const uint32_t rows = n * 2u * g.num_kv_heads;
    uint4 raw[N];
    uint8_t *code[N], *scale[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        raw[j] = make_uint4(0, 0, 0, 0);
        code[j] = nullptr;
        const uint32_t unit = j * 32 + lane, w = w0 + unit / WORDS, word = unit % WORDS;
        if (w >= rows) continue;
        const RowIdx x = row_index(w, hd);
        const int64_t slot = __ldg(slots + x.i);
        if (slot < 0) continue;
        if (slot >= (int64_t)g.num_blocks * kBlockSize) {
            if (word == 0) atomicOr(err, kDevErrSlot);
            continue;
        }
        const uint16_t* src = (x.kv == 0 ? k_new : v_new) + ((size_t)x.i * g.num_kv_heads + x.h) * D;
        raw[j] = __ldg(reinterpret_cast<const uint4*>(src) + word);
        uint8_t* rec = data + fp4_record<D>(g, layer, (uint32_t)(slot / kBlockSize), x.h);
        const uint32_t t = (uint32_t)(slot % kBlockSize), grp = word / 2;
        code[j] = rec + x.kv * R::V + t * R::CODE_ROW + word * 4;
        scale[j] = rec + (x.kv == 0 ? R::KS + t * R::GROUPS + grp : R::VS + grp * 16 + t);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const uint32_t two[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
        float v[8], amax = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k += 2) {
            v[k] = io_f32(two[k / 2] & 0xFFFFu, g.io_kind);
            v[k + 1] = io_f32(two[k / 2] >> 16, g.io_kind);
            amax = fmax3(amax, fabsf(v[k]), fabsf(v[k + 1]));
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        const uint32_t sc = fp4_scale_code(amax);
        const float inv = fp4_inverse(sc);
        const uint32_t codes = fp4_encode4(v, inv) | (fp4_encode4(v + 4, inv) << 16);
        if (code[j]) {
            *reinterpret_cast<uint32_t*>(code[j]) = codes;
            if ((lane & 1) == 0) *scale[j] = (uint8_t)sc;
        }
    }
}

// Reshape-and-cache.  The reference has no append kernel; its paging rule
// (kernels/attention/flash_attention.bm:132-140: token p lives in logical block
// p/16 at slot p%16) defines slot = block_table[p/16]*16 + p%16.  Warp w of the
// grid handles rows 4w .. 4w+3 (token i, kv, head h); negative slots are
// padding and skipped.  16-bit pools: every lane loads its piece of the four
// rows before it stores any; FP8 pools quantise row by row.
__global__ void __launch_bounds__(256) kv_append_kernel(PoolGeom g, uint8_t* __restrict__ data,
                                                        float* __restrict__ scales, uint32_t layer,
                                                        const uint16_t* __restrict__ k_new,
                                                        const uint16_t* __restrict__ v_new,
                                                        const int64_t* __restrict__ slots,
                                                        uint32_t n, uint32_t* err) {
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t w0 = (blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * kRowsPerWarp;
    const uint32_t rows = n * 2u * g.num_kv_heads;
    const uint32_t D = g.head_dim;
    if (g.kv_kind != kFP8) {
        // D 16-bit elements = D/4 u64 words per row: one word per lane (D 128) or
        // one per lane of the first half-warp (D 64)
        const bool active = lane < D / 4;
        uint64_t v[kRowsPerWarp];
        uint64_t* dst[kRowsPerWarp];
#pragma unroll
        for (uint32_t r = 0; r < kRowsPerWarp; ++r) {
            dst[r] = nullptr;
            const uint32_t w = w0 + r;
            if (w >= rows) continue;
            const RowIdx x = row_index(w, g.num_kv_heads);
            const int64_t slot = __ldg(slots + x.i);
            if (slot < 0) continue;
            if (slot >= (int64_t)g.num_blocks * kBlockSize) {
                if (lane == 0) atomicOr(err, kDevErrSlot);
                continue;
            }
            const uint16_t* src = (x.kv == 0 ? k_new : v_new) + ((size_t)x.i * g.num_kv_heads + x.h) * D;
            if (active) v[r] = __ldg(reinterpret_cast<const uint64_t*>(src) + lane);
            dst[r] = reinterpret_cast<uint64_t*>(
                data + pool_row(g, layer, (uint32_t)(slot / kBlockSize), x.h, x.kv,
                                (uint32_t)(slot % kBlockSize)) * D * 2);
        }
#pragma unroll
        for (uint32_t r = 0; r < kRowsPerWarp; ++r)
            if (dst[r] && active) dst[r][lane] = v[r];
        return;
    }
    // FP8: 4 elements per lane (head_dim 128), one row at a time (the row's
    // scale needs the whole row's maximum)
    for (uint32_t r = 0; r < kRowsPerWarp; ++r) {
        const uint32_t w = w0 + r;
        if (w >= rows) return;
        const RowIdx x = row_index(w, g.num_kv_heads);
        const int64_t slot = __ldg(slots + x.i);
        if (slot < 0) continue;
        if (slot >= (int64_t)g.num_blocks * kBlockSize) {
            if (lane == 0) atomicOr(err, kDevErrSlot);
            continue;
        }
        const uint16_t* src = (x.kv == 0 ? k_new : v_new) + ((size_t)x.i * g.num_kv_heads + x.h) * D;
        const uint64_t row = pool_row(g, layer, (uint32_t)(slot / kBlockSize), x.h, x.kv,
                                      (uint32_t)(slot % kBlockSize));
        const uint2 raw = __ldg(reinterpret_cast<const uint2*>(src) + lane);
        float v[4] = {io_f32(raw.x & 0xFFFFu, g.io_kind), io_f32(raw.x >> 16, g.io_kind),
                      io_f32(raw.y & 0xFFFFu, g.io_kind), io_f32(raw.y >> 16, g.io_kind)};
        float amax = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
        const float scale = fp8_row_scale(amax);
        *reinterpret_cast<uint32_t*>(data + row * D + lane * 4) = fp8_encode4(v, scale, g.fp8_ocp != 0);
        if (lane == 0) scales[row] = scale;
    }
}

// Block copy for copy-on-write and compaction moves (no reference counterpart;
// the decision point is the ref-count in engine/kv_cache.bm:94-113).  CTA
// (pair, layer) copies that layer's K and V rows of every head, plus the FP8
// scales, from block src to block dst with 16-B accesses, eight loads in
// flight per thread before their stores.  Pairs must have distinct
// destinations that are not sources in the same call.
constexpr uint32_t kCopyUnroll = 8;

__global__ void __launch_bounds__(256) block_copy_kernel(PoolGeom g, uint8_t* __restrict__ data,
                                                         float* __restrict__ scales,
                                                         const uint32_t* __restrict__ pairs,
                                                         uint32_t n, uint32_t* err) {
    const uint32_t pi = blockIdx.x, layer = blockIdx.y;
    if (pi >= n) return;
    const uint32_t src = __ldg(pairs + 2 * pi), dst = __ldg(pairs + 2 * pi + 1);
    if (src >= g.num_blocks || dst >= g.num_blocks) {
        if (threadIdx.x == 0) atomicOr(err, kDevErrBlockId);
        return;
    }
    const uint32_t bytes = g.num_kv_heads * page_head_bytes(g.kv_kind, g.head_dim);
    const uint4* s = reinterpret_cast<const uint4*>(data + ((uint64_t)layer * g.num_blocks + src) * bytes);
    uint4* d = reinterpret_cast<uint4*>(data + ((uint64_t)layer * g.num_blocks + dst) * bytes);
    const uint32_t n16 = bytes / 16;
    for (uint32_t k0 = threadIdx.x; k0 < n16; k0 += blockDim.x * kCopyUnroll) {
        uint4 v[kCopyUnroll];
#pragma unroll
        for (uint32_t j = 0; j < kCopyUnroll; ++j) {
            const uint32_t k = k0 + j * blockDim.x;
            if (k < n16) v[j] = __ldg(s + k);
        }
#pragma unroll
        for (uint32_t j = 0; j < kCopyUnroll; ++j) {
            const uint32_t k = k0 + j * blockDim.x;
            if (k < n16) d[k] = v[j];
        }
    }
    if (g.kv_kind == kFP8) {
        const uint32_t ns = 2u * g.num_kv_heads * kBlockSize;
        const float* ss = scales + ((uint64_t)layer * g.num_blocks + src) * ns;
        float* ds = scales + ((uint64_t)layer * g.num_blocks + dst) * ns;
        for (uint32_t k = threadIdx.x; k < ns; k += blockDim.x) ds[k] = __ldg(ss + k);
    }
}

// Block-table gather of a 4-bit pool: the rows' values (exact) in the io type,
// into [Hkv][seq_len][D].  A warp takes kFp4Rows rows; a lane expands a word
// of eight codes, half a group, into 16 B, so D/8 lanes write a row.  8191 tokens of
// 8 KV heads of 128 elements take 9.6 us, 4.5 TB/s (instructions, as in the append).
template <int D>
__global__ void __launch_bounds__(256) fp4_gather_kernel(PoolGeom g, const uint8_t* __restrict__ data, uint32_t layer,
                                                         const uint32_t* __restrict__ block_table, uint32_t seq_len,
                                                         uint16_t* __restrict__ out_k, uint16_t* __restrict__ out_v,
                                                         HeadDiv hd, uint32_t* err) {
    using R = Fp4Rec<D>;
    constexpr int WORDS = D / 8, N = kFp4Rows * WORDS / 32;      // words of a row, words of a lane
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t w0 = (blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * kFp4Rows;
    const uint32_t rows = seq_len * 2u * g.num_kv_heads;
    uint32_t code[N], sc[N];
    uint16_t* dst[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        dst[j] = nullptr;
        const uint32_t unit = j * 32 + lane, w = w0 + unit / WORDS, word = unit % WORDS;
        if (w >= rows) continue;
        const RowIdx x = row_index(w, hd);      // x.i = the position p
        const uint32_t blk = __ldg(block_table + x.i / kBlockSize);
        if (blk >= g.num_blocks) {
            if (word == 0) atomicOr(err, kDevErrBlockId);
            continue;
        }
        const uint8_t* rec = data + fp4_record<D>(g, layer, blk, x.h);
        const uint32_t t = x.i % kBlockSize, grp = word / 2;
        code[j] = __ldg(reinterpret_cast<const uint32_t*>(rec + x.kv * R::V + t * R::CODE_ROW) + word);
        sc[j] = __ldg(rec + (x.kv == 0 ? R::KS + t * R::GROUPS + grp : R::VS + grp * 16 + t));
        dst[j] = (x.kv == 0 ? out_k : out_v) + ((size_t)x.h * seq_len + x.i) * D + word * 8;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        if (!dst[j]) continue;
        uint32_t h[4];
        fp4x8_to_f16(code[j], h);
        const uint32_t s2 = e4m3x2_to_f16x2(sc[j] | (sc[j] << 8));
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            h[k] = f16x2_mul(h[k], s2);
            if (g.io_kind == kBF16) h[k] = fp4_f16x2_to_bf16x2(h[k]);
        }
        *reinterpret_cast<uint4*>(dst[j]) = make_uint4(h[0], h[1], h[2], h[3]);
    }
}

// Block-table gather of one sequence: raw rows into out_k/out_v
// [Hkv][seq_len][D] and, for FP8, their scales [Hkv][seq_len].  Follows the
// paging walk of kernels/attention/flash_attention.bm:132-140.  Warp w moves
// rows 4w .. 4w+3 ([position][K, V][head] order), all four loads in flight
// before the stores.
__global__ void __launch_bounds__(256) kv_gather_kernel(PoolGeom g, const uint8_t* __restrict__ data,
                                                        const float* __restrict__ scales,
                                                        uint32_t layer,
                                                        const uint32_t* __restrict__ block_table,
                                                        uint32_t seq_len, uint8_t* __restrict__ out_k,
                                                        uint8_t* __restrict__ out_v,
                                                        float* __restrict__ out_ks,
                                                        float* __restrict__ out_vs, uint32_t* err) {
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t w0 = (blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * kRowsPerWarp;
    const uint32_t rows = seq_len * 2u * g.num_kv_heads;
    const uint32_t rb = g.head_dim * (uint32_t)elem_bytes(g.kv_kind);   // 64, 128 or 256 B
    const uint32_t words = rb / 8;                                       // u64 words per row
    const bool active = lane < words;
    uint64_t v[kRowsPerWarp];
    uint64_t* dst[kRowsPerWarp];
#pragma unroll
    for (uint32_t r = 0; r < kRowsPerWarp; ++r) {
        dst[r] = nullptr;
        const uint32_t w = w0 + r;
        if (w >= rows) continue;
        const RowIdx x = row_index(w, g.num_kv_heads);      // x.i = the position p
        const uint32_t blk = __ldg(block_table + x.i / kBlockSize);
        if (blk >= g.num_blocks) {
            if (lane == 0) atomicOr(err, kDevErrBlockId);
            continue;
        }
        const uint64_t row = pool_row(g, layer, blk, x.h, x.kv, x.i % kBlockSize);
        const uint64_t o = (uint64_t)x.h * seq_len + x.i;
        if (active) v[r] = __ldg(reinterpret_cast<const uint64_t*>(data + row * rb) + lane);
        dst[r] = reinterpret_cast<uint64_t*>((x.kv == 0 ? out_k : out_v) + o * rb);
        if (g.kv_kind == kFP8 && lane == 0) (x.kv == 0 ? out_ks : out_vs)[o] = __ldg(scales + row);
    }
#pragma unroll
    for (uint32_t r = 0; r < kRowsPerWarp; ++r)
        if (dst[r] && active) dst[r][lane] = v[r];
}

}  // namespace

cudaError_t launch_kv_append(const PoolGeom& g, uint8_t* data, float* scales, uint32_t layer,
                             const void* k_new, const void* v_new, const int64_t* slots,
                             uint32_t n, uint32_t* err, cudaStream_t s) {
    if (n == 0) return cudaSuccess;
    const uint64_t rows = (uint64_t)n * 2 * g.num_kv_heads;
    const unsigned grid = (unsigned)((rows + 8 * kRowsPerWarp - 1) / (8 * kRowsPerWarp));
    if (g.kv_kind == kFP4) {
        const unsigned grid = (unsigned)((rows + 8 * kFp4Rows - 1) / (8 * kFp4Rows));
        const HeadDiv hd = head_div(g.num_kv_heads);
        const uint16_t *k = static_cast<const uint16_t*>(k_new), *v = static_cast<const uint16_t*>(v_new);
        if (g.head_dim == 128) fp4_append_kernel<128><<<grid, 256, 0, s>>>(g, data, layer, k, v, slots, n, hd, err);
        else fp4_append_kernel<64><<<grid, 256, 0, s>>>(g, data, layer, k, v, slots, n, hd, err);
        return cudaGetLastError();
    }
    kv_append_kernel<<<grid, 256, 0, s>>>(g, data, scales, layer,
                                          static_cast<const uint16_t*>(k_new),
                                          static_cast<const uint16_t*>(v_new), slots, n, err);
    return cudaGetLastError();
}

cudaError_t launch_block_copy(const PoolGeom& g, uint8_t* data, float* scales,
                              const uint32_t* pairs, uint32_t n, uint32_t* err, cudaStream_t s) {
    if (n == 0) return cudaSuccess;
    block_copy_kernel<<<dim3(n, g.num_layers), 256, 0, s>>>(g, data, scales, pairs, n, err);
    return cudaGetLastError();
}

cudaError_t launch_kv_gather(const PoolGeom& g, const uint8_t* data, const float* scales,
                             uint32_t layer, const uint32_t* block_table, uint32_t seq_len,
                             void* out_k, void* out_v, float* out_ks, float* out_vs,
                             uint32_t* err, cudaStream_t s) {
    if (seq_len == 0) return cudaSuccess;
    const uint64_t rows = (uint64_t)seq_len * 2 * g.num_kv_heads;
    const unsigned grid = (unsigned)((rows + 8 * kRowsPerWarp - 1) / (8 * kRowsPerWarp));
    if (g.kv_kind == kFP4) {
        const unsigned grid = (unsigned)((rows + 8 * kFp4Rows - 1) / (8 * kFp4Rows));
        const HeadDiv hd = head_div(g.num_kv_heads);
        uint16_t *k = static_cast<uint16_t*>(out_k), *v = static_cast<uint16_t*>(out_v);
        if (g.head_dim == 128) fp4_gather_kernel<128><<<grid, 256, 0, s>>>(g, data, layer, block_table, seq_len, k, v, hd, err);
        else fp4_gather_kernel<64><<<grid, 256, 0, s>>>(g, data, layer, block_table, seq_len, k, v, hd, err);
        return cudaGetLastError();
    }
    kv_gather_kernel<<<grid, 256, 0, s>>>(g, data, scales, layer, block_table, seq_len,
                                          static_cast<uint8_t*>(out_k), static_cast<uint8_t*>(out_v),
                                          out_ks, out_vs, err);
    return cudaGetLastError();
}

}  // namespace vw
