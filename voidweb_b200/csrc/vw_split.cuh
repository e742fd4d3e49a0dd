// vw_split.cuh -- what the decode kernels share: the split of a batch's pages over
// the decode CTAs, the prefixes it is computed from, and the combine grid that
// merges the split-K partials.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

#include "vw_internal.h"
#include "vw_ptx.cuh"
#include "vw_window.cuh"

// (vw_decode.cu's phase timeline; nothing elsewhere)
#ifndef VW_TRACE
#define VW_TRACE(slot, val) ((void)0)
#endif

namespace vw {

namespace {

constexpr float kRescaleThreshold = 8.0f;             // log2 units: p <= 2^8 vs a stale max

__host__ __device__ constexpr int align_up_c(int x, int a) { return (x + a - 1) / a * a; }
__host__ __device__ constexpr int gcd_c(int a, int b) { return b == 0 ? a : gcd_c(b, a % b); }

// Largest b with Hkv * pfx[b] <= x (x < Hkv * pfx[B]).
__device__ __forceinline__ int find_seq(const int* pfx, int B, int Hkv, long long x) {
    int lo = 0, hi = B - 1;
    while (lo < hi) {
        int mid = (lo + hi + 1) >> 1;
        if ((long long)Hkv * pfx[mid] <= x) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// Page ranges of the decode CTAs.  The (sequence b, KV head h) segments,
// ordered by (b, h), lie end to end.  A CTA that crosses a segment boundary
// pays for a second query tile, a merge of its warps' states and a partial
// write, and it is the one that finishes last; so each segment is followed by
// a gap of `cost` virtual pages (DecodeParams::seg_cost) and the virtual line
// is cut into equal lengths vper.  Page x of the segment with ordinal k (among
// segments with pages) sits at v(x) = x + cost * k; CTA c takes the pages
// whose v falls in [c * vper, (c + 1) * vper), so the CTA holding page x is
// v(x) / vper.  With cost 0 this is the plain equal split.  The decode, its
// combine grid and the plan all cut with the launch's cost.

// Virtual positions stay far below 2^31: a launch covers fewer than 2^26 pages
// (the pool's rows are checked against 2^31 at creation) plus at most
// kMaxSegmentCost per segment.
__host__ __device__ __forceinline__ int virtual_total(int total_pages, int segments, int cost) {
    return total_pages + cost * segments;
}
__host__ __device__ __forceinline__ int virtual_per_cta(int vtotal, int grid) {
    const int v = (vtotal + grid - 1) / grid;
    return v < kMinPagesPerCta ? kMinPagesPerCta : v;
}

// First page x with v(x) >= t (total when there is none), from the exclusive
// prefixes of pages (pfx) and of sequences with pages (nzp) over B sequences.
__device__ __forceinline__ int range_start(const int* pfx, const int* nzp, int B, int Hkv, int cost, int t) {
    const int total = Hkv * pfx[B];
    if (t >= virtual_total(total, Hkv * nzp[B], cost)) return total;
    // largest b whose first virtual position is <= t (always a sequence with pages)
    int lo = 0, hi = B - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (virtual_total(Hkv * pfx[mid], Hkv * nzp[mid], cost) <= t) lo = mid; else hi = mid - 1;
    }
    const int np = pfx[lo + 1] - pfx[lo];
    const int r = t - virtual_total(Hkv * pfx[lo], Hkv * nzp[lo], cost);
    const int h = r / (np + cost);
    const int off = r - h * (np + cost);
    // inside the gap after segment h: the range starts at the next segment
    return Hkv * pfx[lo] + h * np + (off < np ? off : np);
}

__device__ __forceinline__ void set_err(uint32_t* err, uint32_t bit) { atomicOr(err, bit); }

// Pages per sequence -> exclusive prefixes of pages (pfx) and of sequences with
// pages (nzp), by one warp, 32 sequences at a time, keeping each seq_len in
// slen when given.  A seq_len of 0 gives no pages and one longer than its
// block-table row is clamped to the row; both are flagged when `report`.  With
// WIN only the pages that the window and the sinks leave visible count.
template <bool WIN>
__device__ __forceinline__ void warp_prefixes(const uint32_t* seq_lens, int B, int bt_stride,
                                              uint32_t* err, bool report, int* pfx, int* nzp,
                                              int* slen, int lane, uint32_t window, uint32_t sinks) {
    int run = 0, run_nz = 0;
    if (lane == 0) { pfx[0] = 0; nzp[0] = 0; }
    for (int base_b = 0; base_b < B; base_b += 32) {
        const int b = base_b + lane;
        int np = 0;
        if (b < B) {
            const int sl = (int)__ldg(seq_lens + b);
            if (slen) slen[b] = sl;
            np = pages_of(sl);
            if (sl <= 0 || np > bt_stride) {
                if (report) set_err(err, kDevErrSeqLen);
                np = sl <= 0 ? 0 : bt_stride;
            }
            if (WIN && np > 0) np = decode_span(sl, bt_stride, window, sinks).n;
        }
        int incl = np, incl_nz = np > 0 ? 1 : 0;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, off);
            const int vz = __shfl_up_sync(0xffffffffu, incl_nz, off);
            if (lane >= off) { incl += v; incl_nz += vz; }
        }
        if (b < B) { pfx[b + 1] = run + incl; nzp[b + 1] = run_nz + incl_nz; }
        run += __shfl_sync(0xffffffffu, incl, 31);
        run_nz += __shfl_sync(0xffffffffu, incl_nz, 31);
    }
}

template <int IO>
__device__ __forceinline__ float io_to_f32(uint32_t h) {
    return IO == kBF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
}
template <int IO>
__device__ __forceinline__ uint16_t f32_to_io(float f) {
    return IO == kBF16 ? f32_to_bf16_bits(f) : f32_to_f16_bits(f);
}

// Merge of the split-K pieces of one segment (b, h) for query head j and
// output elements d..d+3: the pieces (o, max, sum) left by decode CTAs
// c0..c0+n-1 (CTA c0 in slot slot0, the others in slot 0) are weighted by
// 2^(max_c - max), the online-softmax rule of flash_attention.bm:149-157
// applied across pieces; up to kCombineBatch pieces per memory round trip.
constexpr int kCombineBatch = 8;

template <int D, int G, int IO>
__device__ __forceinline__ void merge_unit(const DecodeParams& p, int b, int h, int j, int d, int c0,
                                           int n, int slot0, float vfold) {
    uint16_t* out = reinterpret_cast<uint16_t*>(p.out);
    const int g = (int)p.group;
    float M = -INFINITY, Ls = 0.0f, a0 = 0.0f, a1 = 0.0f, a2 = 0.0f, a3 = 0.0f;
    for (int k0 = 0; k0 < n; k0 += kCombineBatch) {
        float2 ml[kCombineBatch];
        float4 o[kCombineBatch];
#pragma unroll
        for (int k = 0; k < kCombineBatch; ++k) {
            ml[k] = make_float2(-INFINITY, 0.0f);
            o[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (k0 + k < n) {
                const int c = c0 + k0 + k;
                const size_t piece = (size_t)c * 2 + (c == c0 ? slot0 : 0);
                ml[k] = __ldcg(reinterpret_cast<const float2*>(p.part_ml + (piece * G + j) * 2));
                o[k] = __ldcg(reinterpret_cast<const float4*>(p.part_o + (piece * G + j) * D + d));
            }
        }
        float Mn = M;
#pragma unroll
        for (int k = 0; k < kCombineBatch; ++k) Mn = fmaxf(Mn, ml[k].x);
        const float r = M > -INFINITY ? ex2(M - Mn) : 0.0f;
        Ls *= r; a0 *= r; a1 *= r; a2 *= r; a3 *= r;
#pragma unroll
        for (int k = 0; k < kCombineBatch; ++k) {
            const float w = ml[k].x > -INFINITY ? ex2(ml[k].x - Mn) : 0.0f;
            Ls += ml[k].y * w;
            a0 += o[k].x * w; a1 += o[k].y * w; a2 += o[k].z * w; a3 += o[k].w * w;
        }
        M = Mn;
    }
    const float r = vfold / Ls;
    const uint32_t lo = (uint32_t)f32_to_io<IO>(a0 * r) | ((uint32_t)f32_to_io<IO>(a1 * r) << 16);
    const uint32_t hi = (uint32_t)f32_to_io<IO>(a2 * r) | ((uint32_t)f32_to_io<IO>(a3 * r) << 16);
    *reinterpret_cast<uint2*>(out + ((size_t)b * p.Hq + (size_t)h * g + j) * D + d) = make_uint2(lo, hi);
}

// ------------------------------------------------------------------ combine

// The combine grid is resident next to the decode grids of this layer and the
// next one (it launches before the decode grid ends and waits in
// griddepcontrol.wait), so its CTAs must fit beside two decode CTAs.  The
// register file is split over the SM's four sub-partitions (16,384 each); ten
// 128-register decode warps leave 4,096 in a sub-partition holding three of
// them, so a combine CTA is a single warp of at most 80 registers (2,560),
// and it runs with the decode's shared-memory carveout.  (The decode of 4-bit pools leaves no
// such room: its two CTAs take the whole register file, and its combine starts as
// they leave.)  CTA (segment, j) merges query head j of the segment, four output
// elements per lane.
constexpr int kCombineWarps = 1;
constexpr int kCombineThreads = kCombineWarps * 32;
constexpr int kCombineMinBlocks = 25;  // 65,536 / (32 x 25) -> a cap of 80 registers

// Merge of the split-K partials, one CTA per (sequence, KV head) segment.  The
// CTA recomputes the decode grid's page ranges from seq_lens (same clamping,
// same per-CTA quantum), returns at once for a segment that one decode CTA
// finished (CTA 0 waits all the same), and otherwise merges the pieces (o, max, sum) left by decode CTAs
// c0..c1 with weights 2^(max_c - max) -- the merge rule of the online softmax
// in flash_attention.bm:149-157, applied across pieces instead of tokens.
// Launched as a programmatic dependent of its decode grid: the geometry is
// computed while the decode still runs, the partials are read after
// griddepcontrol.wait.  Each thread produces four consecutive output elements.
template <int D, int G, int IO, bool WIN>
__global__ void __launch_bounds__(kCombineThreads, kCombineMinBlocks) combine_kernel(const DecodeParams p, int dec_grid,
                                                                  float vfold) {
    __shared__ int red[kCombineThreads / 32][4];
    if (threadIdx.x == 0) VW_TRACE(12, globaltimer());
    // the next grid (the following layer's decode) may start its prologue now;
    // it waits for this whole grid before it writes anything this grid reads
    griddep_launch_dependents();
    const int Hkv = (int)p.Hkv;
    const int b = (int)blockIdx.x / Hkv, h = (int)blockIdx.x - b * Hkv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto pages = [&](int i) {
        const int sl = (int)__ldcg(p.seq_lens + i);
        const int np = pages_of(sl);
        if (WIN && sl > 0) return decode_span(sl, (int)p.bt_stride, p.window, p.sinks).n;
        return sl <= 0 ? 0 : min(np, (int)p.bt_stride);
    };
    // pages and sequences with pages, before b and in all (the decode's prefixes)
    int before = 0, all = 0, nz_before = 0, nz_all = 0;
    for (int i = threadIdx.x; i < (int)p.B; i += kCombineThreads) {
        const int np = pages(i);
        all += np;
        nz_all += np > 0;
        if (i < b) { before += np; nz_before += np > 0; }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, off);
        all += __shfl_xor_sync(0xffffffffu, all, off);
        nz_before += __shfl_xor_sync(0xffffffffu, nz_before, off);
        nz_all += __shfl_xor_sync(0xffffffffu, nz_all, off);
    }
    if (lane == 0) { red[warp][0] = before; red[warp][1] = all; red[warp][2] = nz_before; red[warp][3] = nz_all; }
    __syncthreads();
    before = all = nz_before = nz_all = 0;
#pragma unroll
    for (int w = 0; w < kCombineThreads / 32; ++w) {
        before += red[w][0]; all += red[w][1]; nz_before += red[w][2]; nz_all += red[w][3];
    }
    const int np = pages(b);
    // A grid that launches on this one waits for it alone, so this one must not complete
    // before the decode: its first CTA always waits (the others may return early, and
    // make room for those with something to merge).
    const bool first = blockIdx.x == 0 && blockIdx.y == 0;
    if (np == 0) {
        griddep_wait_if(first);
        return;
    }
    const int cost = (int)p.seg_cost;
    const int vper = virtual_per_cta(virtual_total(Hkv * all, Hkv * nz_all, cost), dec_grid);
    const int s_begin = Hkv * before + h * np;
    const int k = Hkv * nz_before + h;        // segment ordinal
    const int v0 = s_begin + cost * k;
    const int c0 = v0 / vper, c1 = (v0 + np - 1) / vper;
    if (c0 == c1) {                            // written out by the decode CTA itself
        griddep_wait_if(first);
        return;
    }
    // CTA c0 holds this segment in slot 0 when the segment starts its range
    // (the page before it, of segment k-1, lies in an earlier CTA), else in
    // slot 1 (its last segment); every later CTA starts inside it
    const int slot0 = (k == 0 || (s_begin - 1) + cost * (k - 1) < c0 * vper) ? 0 : 1;
    griddep_wait();
    if (threadIdx.x == 0) VW_TRACE(13, globaltimer());
    const int g = (int)p.group;
    const int n = c1 - c0 + 1;
    const int j = (int)blockIdx.y * kCombineWarps + warp, d = lane * 4;
    if (j < g && d < D) merge_unit<D, G, IO>(p, b, h, j, d, c0, n, slot0, vfold);
    if (threadIdx.x == 0) VW_TRACE(14, globaltimer());
}


// The combine behind a decode of the same launch; vfold multiplies the outputs.
template <int D, int G, int IO, bool WIN>
cudaError_t launch_combine(const DecodeLaunch& L, float vfold) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(L.p.B * L.p.Hkv, (L.p.group + kCombineWarps - 1) / kCombineWarps);
    cfg.blockDim = dim3(kCombineThreads);
    cfg.stream = L.stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, combine_kernel<D, G, IO, WIN>, L.p, L.grid, vfold);
}

}  // namespace

}  // namespace vw
