// vw_prefill_group.cu -- the prefill attention of 4-bit pools, and of f16 / bf16 pools under a
// window.
//
//  * Work split.  The query heads of a KV head are taken together: row r of a
//    (sequence, KV head) is query head r % group of chunk token r / group, and a CTA takes
//    128 consecutive rows, the M of the matrix instructions.  A CTA so spans few
//    tokens (19 with 7 query heads), which visit hardly more keys than one of them
//    does, and a short chunk still fills its tile.
//  * Rounds of 64 keys, as in vw_prefill.cu: S = Q K^T into one of two S buffers in
//    tensor memory while the softmax works on the other, P over S, O += P V; two
//    CTAs per SM.  (Rounds of 128 keys leave tensor memory for one S per tile: S,
//    softmax and P V then follow one another, and measured slower with one tile
//    per CTA and two CTAs, 5757 cycles per 128 keys and SM against 4033, and with two tiles
//    per CTA, 4593.)
//  * Warps 0-3: softmax, one row per thread.  Warp 4 issues the matrix instructions.
//    f16 / bf16 pages: warp 5 streams K tiles, warp 6 V tiles (TMA).  4-bit pages:
//    warp 5 expands the records' K halves into f16 tiles, warp 6 the V halves.
//  * bf16 probabilities are a pair hi + lo (two P V products, as in vw_prefill.cu),
//    those of f16 and 4-bit pages one f16.
//  * Few tiles (a short question over a long document) leave most SMs idle while a CTA
//    walks all its keys, some 1.1 us per round: the rounds of a tile are then split over
//    up to kMaxSplit CTAs, which leave unnormalised outputs with their maxima and sums
//    in f32, and a small grid merges them.
//  * Measured, Qwen2.5-7B heads, 4 chunks of 2048 tokens: under a window of 1024 tokens 176 to
//    187 us (570 to 606 TFLOP/s of visible work; of some 2300 cycles of a pair of rounds the matrix
//    instructions take 2032), over 4-bit pages 227 us (581 TFLOP/s; the softmax and the
//    decoders set the pace).
//  * Every wait is bounded; on timeout the kernel records kDevErrTimeout, waits
//    for its copies and matrix instructions in flight and returns.
#define VW_MBAR_SUSPEND_HINT_NS 0
#include <cuda.h>
#include <cuda_runtime.h>
#include <algorithm>
#include <atomic>
#include <cstdint>

#include "vw_prefill.cuh"
#include "vw_fp4.cuh"
#include "vw_rope.cuh"
#include "vw_tc.cuh"
#include "vw_window.cuh"

namespace vw {

namespace {

constexpr int kGRows = kPrefillTileRows;          // query rows per CTA
constexpr int kGKeys = 64;                        // keys per round
constexpr int kGPages = kGKeys / kBlockSize;
constexpr int kMaxSplit = 8;
constexpr int kMinRounds = 2;                     // rounds of a split, at least
constexpr float kGRescale = 8.0f;                 // log2 units: p <= 2^8 against a stale max

template <int D_, int IO_, int KV_>
struct Grp {
    static constexpr int D = D_, IO = IO_;
    static constexpr bool FP4 = KV_ == kFP4;
    static constexpr bool MBF = IO == kBF16 && !FP4;          // the matrix instructions' type is bf16
    static constexpr bool PSPLIT = MBF;
    static constexpr int CH = D * 2 / 128;                    // 128-B columns of a row
    static constexpr int QTILE = CH * 128 * 128;              // [CH][128 rows][128 B]
    static constexpr int TILE = CH * kGKeys * 128;            // one K or V tile
    // K tiles and V tiles: a K tile frees when S of its round completes, rounds before the V
    // tile of that round, so where shared memory allows the K ring is one deeper
    static constexpr int NSTK = D == 64 ? 4 : 3;
    static constexpr int NSTV = D == 64 ? 4 : 2;
    static constexpr int KSTEPS = D / 16;
    static constexpr int COL_S = D;                           // O in columns [0, D), two S buffers after it
    // full, empty of K and V tiles; s_full, p_full, p_free of both buffers; q_full, landed, done
    static constexpr int NBAR = 2 * NSTK + 2 * NSTV + 9;
    static constexpr int TPFX = pf_align((kMaxBatchPerLaunch + 1) * 4, 128);
    static constexpr int SMEM = QTILE + (NSTK + NSTV) * TILE + NBAR * 8 + 16;
    static constexpr int THREADS = 7 * 32;
    static constexpr uint32_t IDESC_S = idesc_f16(MBF, false, 128, kGKeys);
    static constexpr uint32_t IDESC_PV = idesc_f16(MBF, true, 128, D);
    static_assert(COL_S + 2 * kGKeys <= 256, "tensor-memory columns");
    static_assert(2 * (SMEM + 1024) <= 233472, "two CTAs per SM");
    static_assert(3 * (SMEM + 1024) > 233472, "at most two CTAs per SM (tensor memory)");
    static_assert(TPFX <= TILE, "the tile prefix fits in a V tile");
};

// Rounds of a tile (or of a part of them) as its CTA and the merge compute them.
struct Rounds {
    int all, per, parts;        // rounds of the tile, of a part, parts
};
__device__ __forceinline__ Rounds split_rounds(int npages, int splits) {
    Rounds r;
    r.all = (npages + kGPages - 1) / kGPages;
    r.per = max((r.all + splits - 1) / splits, kMinRounds);
    r.parts = (r.all + r.per - 1) / r.per;
    return r;
}

// Prefix of the tiles of every sequence over the batch, by one warp.
__device__ __forceinline__ void tile_prefix(const int32_t* cu_q, int B, int T, int g, int* tpfx, int lane) {
    int run = 0;
    if (lane == 0) tpfx[0] = 0;
    for (int b0 = 0; b0 < B; b0 += 32) {
        const int b = b0 + lane;
        int nt = 0;
        if (b < B) {
            const int n = __ldg(cu_q + b + 1) - __ldg(cu_q + b);
            // (a chunk past q's T rows is refused later)
            nt = n > 0 ? (int)(((long long)min(n, T) * g + kGRows - 1) / kGRows) : 0;
        }
        int incl = nt;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, off);
            if (lane >= off) incl += v;
        }
        if (b < B) tpfx[b + 1] = run + incl;
        run += __shfl_sync(0xffffffffu, incl, 31);
    }
}

// The tile of CTA column `col` (the last tiles, which visit the most keys of a causal chunk,
// come first): its sequence, rows and keys.  False: none, or a chunk outside q's
// T rows or past its block-table row (bad).
struct TileGeom {
    int b, row0, q_off, n, cs, total, rows, npages;
    PageSpan span;
    bool bad;
};
template <bool WIN>
__device__ __forceinline__ bool tile_geom(const PrefillParams& p, const int* tpfx, int col, TileGeom& t) {
    const int x = tpfx[p.B] - 1 - col, g = (int)p.group;
    t.bad = false;
    if (x < 0) return false;
    t.b = pf_find(tpfx, (int)p.B, x);
    t.row0 = (x - tpfx[t.b]) * kGRows;                 // first row in its (sequence, KV head)
    t.q_off = __ldg(p.cu_q + t.b);
    t.n = __ldg(p.cu_q + t.b + 1) - t.q_off;
    t.cs = __ldg(p.ctx_start + t.b);
    t.total = t.cs + t.n;
    t.rows = (int)((unsigned)t.n * (unsigned)g);
    t.bad = t.q_off < 0 || t.n > (int)p.T || t.q_off > (int)p.T - t.n || t.cs < 0 || t.row0 < 0 || t.row0 >= t.rows ||
            (long long)t.cs + t.n > (long long)p.bt_stride * kBlockSize;
    if (t.bad) return false;
    const int tok0 = t.row0 / g, tok1 = (min(t.row0 + kGRows, t.rows) - 1) / g;
    const int kend = p.causal ? t.cs + tok1 + 1 : t.total;         // keys [0, kend)
    t.npages = (kend + kBlockSize - 1) / kBlockSize;   // pages visited (ordinals, mapped by span.page)
    t.span = PageSpan{};
    if constexpr (WIN) {
        t.span = page_span(t.npages, t.cs + tok0, p.window, p.sinks);
        t.npages = t.span.n;
    }
    return true;
}

// One lane's units a, b of a bf16 query row -> f16, times the row's factor; HALF neighbouring
// lanes hold the row and get the factor.
template <int HALF>
__device__ __forceinline__ float query_to_f16(uint4& a, uint4& b) {
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}, top = bf16_top<8>(w);
#pragma unroll
    for (int off = 1; off < HALF; off <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
    const float f = fp4_query_factor(top);
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = fp4_query_pair(w[k], f);
    a = make_uint4(w[0], w[1], w[2], w[3]), b = make_uint4(w[4], w[5], w[6], w[7]);
    return f;
}

__device__ __forceinline__ uint4 bf16_to_f16x8(uint4 v) {
    return make_uint4(fp4_query_pair(v.x, 1.0f), fp4_query_pair(v.y, 1.0f), fp4_query_pair(v.z, 1.0f), fp4_query_pair(v.w, 1.0f));
}

template <class T, bool WIN>
__global__ void __launch_bounds__(T::THREADS, 2)
prefill_group_kernel(const __grid_constant__ CUtensorMap tmap, const PrefillParams p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    // the 128-B-swizzled tiles need 1024-B alignment; the layout has no slack
    if (smem_u32(smem_raw) & 1023u) {
        if (threadIdx.x == 0) atomicOr(p.err, kDevErrLaunch);
        return;
    }
    uint8_t* qs = smem_raw;
    uint8_t* ktiles = qs + T::QTILE;
    uint8_t* vtiles = ktiles + T::NSTK * T::TILE;
    int* tpfx = reinterpret_cast<int*>(vtiles + (T::NSTV - 1) * T::TILE);   // prologue only
    uint64_t* full_k = reinterpret_cast<uint64_t*>(vtiles + T::NSTV * T::TILE);
    uint64_t* empty_k = full_k + T::NSTK;
    uint64_t* full_v = empty_k + T::NSTK;
    uint64_t* empty_v = full_v + T::NSTV;
    uint64_t* s_full = empty_v + T::NSTV;
    uint64_t* p_full = s_full + 2;
    uint64_t* p_free = p_full + 2;
    uint64_t* q_full = p_free + 2;
    uint64_t* landed = q_full + 1;
    uint64_t* done = landed + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint64_t deadline = cycles() + (p.wait_cycles ? p.wait_cycles : kWaitDeadlineCycles);
    // test hook (vw_debug_set_wait_limit): no K/V tile is filled
    const bool withhold = p.wait_cycles != 0;

    if (threadIdx.x == 0) {
        // (full: the decoder, or the TMA transaction)
        for (int s = 0; s < T::NSTK; ++s) { mbar_init(&full_k[s], 1); mbar_init(&empty_k[s], 1); }
        for (int s = 0; s < T::NSTV; ++s) { mbar_init(&full_v[s], 1); mbar_init(&empty_v[s], 1); }
        for (int c = 0; c < 2; ++c) { mbar_init(&s_full[c], 1); mbar_init(&p_full[c], 4); mbar_init(&p_free[c], 1); }
        mbar_init(q_full, 4);
        mbar_init(landed, 1);
        mbar_init(done, 1);
        fence_mbar_init();
    }
    if (p.flags & kDecodePdl) griddep_wait();          // q, chunk rows and pages from the predecessor
    // the merge of a split launch may come up now: it waits for this whole grid
    if (gridDim.z > 1) griddep_launch_dependents();
    const int g = (int)p.group;
    if (warp == 0) tile_prefix(p.cu_q, (int)p.B, (int)p.T, g, tpfx, lane);
    __syncthreads();
    // (more CTAs than the grid: chunk offsets that are not those of T rows)
    if (tpfx[p.B] > (int)gridDim.x && blockIdx.x == 0 && threadIdx.x == 0) atomicOr(p.err, kDevErrSeqLen);
    TileGeom geo;
    if (!tile_geom<WIN>(p, tpfx, (int)blockIdx.x, geo)) {
        // the offsets come from device memory: such a chunk is flagged and skipped
        if (geo.bad && threadIdx.x == 0) atomicOr(p.err, kDevErrSeqLen);
        return;
    }
    const PageSpan span = geo.span;
    const int row0 = geo.row0, q_off = geo.q_off, cs = geo.cs, total = geo.total, rows = geo.rows;
    const int h = blockIdx.y;
    // this CTA's part of the rounds: page ordinals from page0 on
    const Rounds rounds = split_rounds(geo.npages, (int)gridDim.z);
    const int round0 = (int)blockIdx.z * rounds.per;
    if (round0 >= rounds.all) return;
    const int nrounds = min(rounds.per, rounds.all - round0), page0 = round0 * kGPages;
    const int npages = min(geo.npages - page0, nrounds * kGPages);
    const bool partial = rounds.parts > 1;
    const uint32_t* bt = p.block_tables + (size_t)geo.b * p.bt_stride;
    auto page_of = [&](int o) { return WIN ? span.page(page0 + o) : page0 + o; };
    auto id_of = [&](int o) { return o < npages ? __ldg(bt + page_of(o)) : 0xFFFFFFFFu; };

    if (warp == 4) {
        tmem_alloc(tmem_slot, 256);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();                                   // tensor memory, and the prefix is read by all
    tc_fence_after();
    const uint32_t tbase = *tmem_slot;

    if (warp < 4) {
        // ---- softmax: thread r owns query row row0 + r
        const int r = threadIdx.x, row = row0 + r;
        const bool live = row < rows;
        const int tq = live ? row / g : 0;
        float scale_log2 = p.scale_log2;               // of this thread's row
        {
            // The warp's query rows into the swizzled K-major tile: 16-B unit u goes to column
            // u / 8, unit (u % 8) ^ (r % 8); rotated first with rope_theta > 0.  A lane takes
            // units u and u + D/16 (the pairs of the rotation) of a row in 512/D rows, all its loads
            // in flight together.  (A row per lane, unit after unit, took 8700 cycles of some
            // 57,000 that a tile of 17 rounds takes, these 4500.)
            constexpr int HALF = T::D / 16, STEP = 32 / HALF, N = 32 / STEP;
            constexpr bool CONV = T::FP4 && T::IO == kBF16;            // 4-bit pages compute in f16
            constexpr uint32_t FIRST = HALF == 8 ? 0x01010101u : 0x11111111u;      // the first lane of each row
            const int u = lane % HALF, u2 = u + HALF;
            uint4 lo[N], hi[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int rr = i * STEP + lane / HALF, qr = row0 + warp * 32 + rr;      // the row, in the warp and overall
                const int tok = __shfl_sync(0xffffffffu, tq, rr);
                lo[i] = hi[i] = make_uint4(0, 0, 0, 0);
                if (qr < rows) {
                    const uint4* src = reinterpret_cast<const uint4*>(
                        reinterpret_cast<const uint8_t*>(p.q) +
                        ((size_t)(q_off + tok) * p.Hq + (size_t)h * g + (qr - tok * g)) * T::D * 2);
                    lo[i] = __ldg(src + u);
                    hi[i] = __ldg(src + u2);
                }
            }
            bool again = p.rope_theta > 0.0f;          // rows to rotate, or bf16 rows outside f16's range
            if constexpr (CONV) {
                bool high = false, low = false;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const uint32_t w[8] = {lo[i].x, lo[i].y, lo[i].z, lo[i].w, hi[i].x, hi[i].y, hi[i].z, hi[i].w};
                    const uint32_t own = bf16_top<8>(w);
                    high |= own >= kQueryHigh;
                    uint32_t big = __ballot_sync(0xffffffffu, own >= kQueryLow || row0 + warp * 32 + i * STEP + lane / HALF >= rows);
#pragma unroll
                    for (int off = 1; off < HALF; off <<= 1) big |= big >> off;
                    low |= (big & FIRST) != FIRST;
                }
                again |= low || __any_sync(0xffffffffu, high);
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int rr = warp * 32 + i * STEP + lane / HALF;
                uint4 a = lo[i], b = hi[i];
                if (CONV && !again) a = bf16_to_f16x8(a), b = bf16_to_f16x8(b);
                *reinterpret_cast<uint4*>(qs + (u >> 3) * 16384 + rr * 128 + (((u & 7) ^ (rr & 7)) << 4)) = a;
                *reinterpret_cast<uint4*>(qs + (u2 >> 3) * 16384 + rr * 128 + (((u2 & 7) ^ (rr & 7)) << 4)) = b;
            }
            if (again) {
                // in place, by the lane that wrote the units: out of the way of calls without it
#pragma unroll 1
                for (int i = 0; i < N; ++i) {
                    const int rr = warp * 32 + i * STEP + lane / HALF;
                    const float pos = (float)(cs + __shfl_sync(0xffffffffu, tq, i * STEP + lane / HALF));
                    uint4* pa = reinterpret_cast<uint4*>(qs + (u >> 3) * 16384 + rr * 128 + (((u & 7) ^ (rr & 7)) << 4));
                    uint4* pb = reinterpret_cast<uint4*>(qs + (u2 >> 3) * 16384 + rr * 128 + (((u2 & 7) ^ (rr & 7)) << 4));
                    uint4 a = *pa, b = *pb;
                    uint32_t e[4] = {a.x, a.y, a.z, a.w}, f[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                    for (int w = 0; w < 4 && p.rope_theta > 0.0f; ++w) {
                        // pairs (d, d + D/2)
                        float ar = pf_io_to_f32<T::IO>(e[w] & 0xFFFFu), ai = pf_io_to_f32<T::IO>(f[w] & 0xFFFFu);
                        float br = pf_io_to_f32<T::IO>(e[w] >> 16), bi = pf_io_to_f32<T::IO>(f[w] >> 16);
                        const int d = u * 8 + 2 * w;
                        rope_pair(ar, ai, d, T::D, p.rope_theta, pos);
                        rope_pair(br, bi, d + 1, T::D, p.rope_theta, pos);
                        e[w] = (uint32_t)pf_f32_to_io<T::IO>(ar) | ((uint32_t)pf_f32_to_io<T::IO>(br) << 16);
                        f[w] = (uint32_t)pf_f32_to_io<T::IO>(ai) | ((uint32_t)pf_f32_to_io<T::IO>(bi) << 16);
                    }
                    a = make_uint4(e[0], e[1], e[2], e[3]), b = make_uint4(f[0], f[1], f[2], f[3]);
                    if (CONV) {
                        const float f = __shfl_sync(0xffffffffu, query_to_f16<HALF>(a, b), lane % STEP * HALF);
                        if (lane / STEP == i) scale_log2 *= fp4_query_unfactor(f);
                    }
                    *pa = a, *pb = b;
                }
            }
            // generic-proxy writes, read next by the tensor cores (async proxy)
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        {
            const int kend_r = live ? (p.causal ? cs + tq + 1 : total) : 0;
            const int lo_r = WIN ? max(0, kend_r - (int)p.window) : 0;      // first key of the row's window
            const uint32_t lanes = (uint32_t)(warp * 32) << 16;
            const uint32_t ocol = tbase + lanes;
            float m_ref = -INFINITY, l = 0.0f;
            bool ok = true;
            for (int t = 0; t < nrounds; ++t) {
                const int bb = t & 1;
                const uint32_t scol = tbase + lanes + T::COL_S + bb * kGKeys;
                if (!__all_sync(0xffffffffu, mbar_wait(&s_full[bb], (t >> 1) & 1, deadline))) { ok = false; break; }
                tc_fence_after();
                float xs[kGKeys];
                tmem_ld32f(scol, xs);
                tmem_ld32f(scol + 32, xs + 32);
                tmem_wait_ld();
                // does the row see every key of the round?  (a round of sink pages and
                // window pages is taken key by key)
                const int f = page_of(t * kGPages) * kBlockSize, e = page_of(t * kGPages + kGPages - 1) * kBlockSize;
                bool whole = e + kBlockSize <= kend_r;
                if constexpr (WIN)
                    whole = whole && e - f == (kGPages - 1) * kBlockSize && (f >= lo_r || e + kBlockSize <= span.sinks);
                if (!__all_sync(0xffffffffu, whole)) {
                    // keys of page-heads past npages are stale rows; they lie past kend_r
#pragma unroll
                    for (int k = 0; k < kGKeys; ++k) {
                        const int pos = page_of(t * kGPages + k / kBlockSize) * kBlockSize + k % kBlockSize;
                        xs[k] = pos < kend_r && (!WIN || pos >= lo_r || pos < span.sinks) ? xs[k] : -INFINITY;
                    }
                }
                // Scores stay unscaled (scale > 0 keeps the order); the scale is folded into
                // the exponent below.  Four chains of maxima, not one of 64 steps.
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int k = 0; k < kGKeys; k += 8)
#pragma unroll
                    for (int c = 0; c < 4; ++c) m4[c] = fmax3(m4[c], xs[k + 2 * c], xs[k + 2 * c + 1]);
                const float tmax = fmaxf(fmax3(m4[0], m4[1], m4[2]), m4[3]) * scale_log2;
                const bool need = tmax > m_ref + kGRescale;
                float alpha = 1.0f;
                if (need) {
                    alpha = ex2(m_ref - tmax);      // 0 while the row had no key
                    m_ref = tmax;
                }
                if (__any_sync(0xffffffffu, need && t > 0)) {
                    // rescale O: after P V of the round before (whose phase is the next of its
                    // buffer: S of this round was issued after P V two rounds before completed)
                    if (!__all_sync(0xffffffffu, mbar_wait(&p_free[bb ^ 1], ((t - 1) >> 1) & 1, deadline))) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
#pragma unroll 1
                    for (int c0 = 0; c0 < T::D; c0 += 16) {
                        uint32_t o16[16];
                        tmem_ld16(ocol + c0, o16);
                        tmem_wait_ld();
#pragma unroll
                        for (int k = 0; k < 16; ++k) o16[k] = __float_as_uint(__uint_as_float(o16[k]) * alpha);
                        tmem_st16(ocol + c0, o16);
                    }
                }
                l *= alpha;
                const float mu = m_ref == -INFINITY ? 0.0f : m_ref;
                const float2 sc2 = make_float2(scale_log2, scale_log2), mu2 = make_float2(-mu, -mu);
                float2 ls[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
                // P over S: 32 keys take 16 columns of hi (or of the one f16) and, with a pair,
                // 16 of lo
#pragma unroll
                for (int c = 0; c < kGKeys / 32; ++c) {
                    uint32_t ph[16], pl[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const float2 ev = fma2(make_float2(xs[32 * c + 2 * k], xs[32 * c + 2 * k + 1]), sc2, mu2);
                        const float2 pr = make_float2(ex2(ev.x), ex2(ev.y));
                        ls[k & 1] = add2(ls[k & 1], pr);
                        ph[k] = pack2<T::MBF>(pr.x, pr.y);
                        if constexpr (T::PSPLIT) {
                            // hi as a negative pair, then lo = p - hi
                            const float2 hi = make_float2(__uint_as_float((ph[k] << 16) ^ 0x80000000u),
                                                          __uint_as_float((ph[k] & 0xFFFF0000u) ^ 0x80000000u));
                            const float2 lo = add2(pr, hi);
                            pl[k] = pack2<true>(lo.x, lo.y);
                        }
                    }
                    tmem_st16(scol + 32 * c, ph);
                    if constexpr (T::PSPLIT) tmem_st16(scol + 32 * c + 16, pl);
                }
                l += (ls[0].x + ls[0].y) + (ls[1].x + ls[1].y);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[bb]);
            }
            // epilogue: O / l, after the last P V
            if (ok && __all_sync(0xffffffffu, mbar_wait(done, 0, deadline))) {
                tc_fence_after();
                const float inv = l > 0.0f ? 1.0f / l : 0.0f;
                const size_t qrow = (size_t)(q_off + tq) * p.Hq + (size_t)h * g + (live ? row - tq * g : 0);
                uint8_t* dst = reinterpret_cast<uint8_t*>(p.out) + qrow * T::D * 2;
                const size_t part = ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * gridDim.z + blockIdx.z;
                float* po = p.part_o + (part * kGRows + r) * T::D;
                if (partial) *reinterpret_cast<float2*>(p.part_ml + (part * kGRows + r) * 2) = make_float2(m_ref, l);
#pragma unroll 1
                for (int c0 = 0; c0 < T::D; c0 += 32) {
                    float o[32];
                    tmem_ld32f(ocol + c0, o);
                    tmem_wait_ld();
                    if (partial) {
#pragma unroll
                        for (int u = 0; u < 8; ++u)
                            *reinterpret_cast<float4*>(po + c0 + 4 * u) =
                                make_float4(o[4 * u], o[4 * u + 1], o[4 * u + 2], o[4 * u + 3]);
                        continue;
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        uint32_t w[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            w[k] = (uint32_t)pf_f32_to_io<T::IO>(o[8 * u + 2 * k] * inv) |
                                   ((uint32_t)pf_f32_to_io<T::IO>(o[8 * u + 2 * k + 1] * inv) << 16);
                        if (live) *reinterpret_cast<uint4*>(dst + c0 * 2 + 16 * u) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            } else if (lane == 0) {
                atomicOr(p.err, kDevErrTimeout);
            }
        }
    } else if (warp == 4) {
        // ---- MMA issuer: the warp runs as one, lane 0 issues
        const uint32_t on = lane == 0;
        // descriptors: bases to which a k-step adds (kk / 4) * column + (kk % 4) * 32 bytes
        // (>> 4 in the address field, which never carries: shared memory ends below
        // 256 KB).  K tile: K-major, 8-key groups 1024 B apart; V tile: MN-major, 64-element
        // columns 8 KB apart, 8-key groups 1024 B apart.
        const uint64_t qdesc = smem_desc_sw128(smem_u32(qs), 16, 1024);
        const uint64_t kdesc = smem_desc_sw128(smem_u32(ktiles), 16, 1024);
        const uint64_t vdesc = smem_desc_sw128(smem_u32(vtiles), kGKeys * 128, 1024);
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            return __all_sync(0xffffffffu, mbar_wait(bar, parity, deadline)) != 0;
        };
        auto issue_pv = [&](int t) -> bool {
            const int bb = t & 1, st = t % T::NSTV, pages = min(kGPages, npages - t * kGPages);
            if (!wait(&full_v[st], (t / T::NSTV) & 1) || !wait(&p_full[bb], (t >> 1) & 1)) return false;
            tc_fence_after();
            const uint64_t vst = vdesc + (uint64_t)((st * T::TILE) >> 4);
            const uint32_t pcol = tbase + T::COL_S + bb * kGKeys;
#pragma unroll
            for (int pg = 0; pg < kGPages; ++pg) {              // 16 keys each
                if (pg >= pages) break;
                const uint64_t vd = vst + (uint64_t)((pg * 2048) >> 4);
                const uint32_t pc = pcol + 32 * (pg >> 1) + 8 * (pg & 1);
                tc_mma_ts_if(on, tbase, pc, vd, T::IDESC_PV, (t > 0 || pg > 0) ? 1u : 0u);
                if constexpr (T::PSPLIT) tc_mma_ts_if(on, tbase, pc + 16, vd, T::IDESC_PV, 1u);
            }
            tc_commit_if(on, &empty_v[st]);
            tc_commit_if(on, &p_free[bb]);
            return true;
        };
        bool ok = wait(q_full, 0);
        for (int t = 0; t < nrounds && ok; ++t) {
            const int bb = t & 1, st = t % T::NSTK;
            // buffer bb holds P of round t - 2 until its products complete
            ok = wait(&full_k[st], (t / T::NSTK) & 1) && (t < 2 || wait(&p_free[bb], ((t - 2) >> 1) & 1));
            if (!ok) break;
            tc_fence_after();
            const uint64_t kst = kdesc + (uint64_t)((st * T::TILE) >> 4);
            const uint32_t dcol = tbase + T::COL_S + bb * kGKeys;
#pragma unroll
            for (int kk = 0; kk < T::KSTEPS; ++kk)
                tc_mma_ss_if(on, dcol, qdesc + (uint64_t)(((kk >> 2) * 16384 + (kk & 3) * 32) >> 4),
                             kst + (uint64_t)(((kk >> 2) * (kGKeys * 128) + (kk & 3) * 32) >> 4), T::IDESC_S, kk > 0 ? 1u : 0u);
            tc_commit_if(on, &empty_k[st]);
            tc_commit_if(on, &s_full[bb]);
            if (t >= 1) ok = issue_pv(t - 1);
        }
        if (ok) ok = issue_pv(nrounds - 1);
        if (!ok && lane == 0) atomicOr(p.err, kDevErrTimeout);
        // everything issued here, the arrivals above among it, completes before tensor
        // memory is freed and the CTA leaves: in bounded time, so this wait has a
        // deadline of its own (after a timeout the kernel's may have run out)
        tc_commit_if(on, done);
        if (!__all_sync(0xffffffffu, mbar_wait(done, 0, cycles() + kWaitDeadlineCycles)) && lane == 0)
            atomicOr(p.err, kDevErrTimeout);
    } else if constexpr (!T::FP4) {
        // ---- producers: warp 5 streams the rounds' K tiles, warp 6 their V tiles.  The block
        // ids come in windows of 32 pages, one per lane, the next window loaded when the
        // current one starts.
        const int kv = warp - 5;
        const int ns = kv ? T::NSTV : T::NSTK;
        uint64_t* fbar = kv ? full_v : full_k;
        uint64_t* ebar = kv ? empty_v : empty_k;
        uint8_t* tiles = kv ? vtiles : ktiles;
        if (lane == 0) prefetch_tensormap(&tmap);
        constexpr int IDW = 32 / kGPages;
        uint32_t win = id_of(lane), nwin = id_of(32 + lane);
        bool ok = true;
        int issued = 0, nland = 0;
        for (int t = 0; t < nrounds && !withhold; ++t) {
            const int st = t % ns;
            if (t > 0 && t % IDW == 0) {
                win = nwin;
                nwin = id_of((t / IDW + 1) * 32 + lane);
            }
            if (t >= ns && !__all_sync(0xffffffffu, mbar_wait(&ebar[st], ((t / ns) - 1) & 1, deadline))) {
                ok = false;
                break;
            }
            const int pg0 = t * kGPages, m = min(kGPages, npages - pg0);
            // V rows that no query of the CTA sees (past the sequence's end, outside the
            // window) may hold anything; the few page-heads with such rows are zeroed
            // there before the round is handed on, so that P = 0 meets no NaN or Inf
            bool dirty = false;
            if (kv) {
                for (int k = 0; k < m; ++k) {
                    const int lp = page_of(pg0 + k);
                    int z0 = 0, z1 = 0;
                    if constexpr (WIN) span.hidden(lp, z0, z1);
                    dirty |= z0 < z1 || total - lp * kBlockSize < kBlockSize;
                }
            }
            uint64_t* fb = dirty ? landed : &fbar[st];
            if (lane == 0) mbar_arrive_expect_tx(fb, (uint32_t)(m * T::CH * 2048));
            __syncwarp();
            // one box per lane: lane l copies column l % CH of page-head l / CH (from one lane, one
            // after another: 197 us against 191 in the Qwen2.5-7B case)
            const int pg = lane / T::CH, c = lane % T::CH;
            const uint32_t bj = __shfl_sync(0xffffffffu, win, (t % IDW) * kGPages + (pg < kGPages ? pg : 0));
            if (pg < m) {
                int prow = -32;                          // negative rows: TMA zero-fills
                if (bj < p.num_blocks)
                    prow = (int)(((p.layer * p.num_blocks + bj) * p.Hkv + (uint32_t)h) * 32u) + 16 * kv;
                else if (kv == 0 && c == 0)
                    atomicOr(p.err, kDevErrBlockId);
                tma_load_2d(tiles + st * T::TILE + c * (kGKeys * 128) + pg * 2048, &tmap, fb, c * 64, prow);
            }
            if (dirty) {
                // (its copies are waited for under a deadline of their own, below and here)
                if (!__all_sync(0xffffffffu, mbar_wait(landed, nland & 1, cycles() + kWaitDeadlineCycles))) {
                    ok = false;
                    break;
                }
                ++nland;
                for (int k = 0; k < m; ++k) {
                    const int lp = page_of(pg0 + k);
                    int z0 = 0, z1 = 0;
                    if constexpr (WIN) span.hidden(lp, z0, z1);
                    const int endr = total - lp * kBlockSize;
                    for (int u = lane; u < kBlockSize * T::CH * 8; u += 32) {
                        const int row = u & 15, cu = u >> 4;           // 16-B unit cu of the row
                        if ((row >= z0 && row < z1) || row >= endr)
                            *reinterpret_cast<uint4*>(tiles + st * T::TILE + (cu >> 3) * (kGKeys * 128) +
                                                      (k * kBlockSize + row) * 128 + (cu & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&fbar[st]);
            }
            issued = t + 1;
        }
        if (lane == 0) {
            if (!ok) atomicOr(p.err, kDevErrTimeout);
            // drain: no TMA write may land after the CTA has exited.  The copies still in
            // flight are this warp's last rounds in the ring; they land in bounded time, so the
            // drain has a deadline of its own (the kernel's may have run out already)
            const uint64_t drain_deadline = cycles() + kWaitDeadlineCycles;
            for (int t = issued > ns ? issued - ns : 0; t < issued; ++t)
                if (!mbar_wait(&fbar[t % ns], (t / ns) & 1, drain_deadline)) {
                    atomicOr(p.err, kDevErrTimeout);
                    break;
                }
        }
    } else {
        // ---- decoders: warp 5 the K halves, warp 6 the V halves of the records.  A chunk is 16
        // B, 32 codes of one row, with the scales of its two groups; codes times scales are
        // exact in f16 and go to the tiles that TMA gives f16 pools: unit u of key row
        // k at (u ^ (k % 8)) * 16 of its column.  The chunks of a whole round are in registers,
        // loaded while the round before is expanded: once a page-head's are used, those
        // of the same place in the next round are on their way (one bulk copy per half
        // instead cost its warp some 300 cycles to issue).  Lanes resolve 32 pages at a
        // time, one batch ahead.
        using Rec = Fp4Rec<T::D>;
        constexpr int U = T::D / 32, PER = U / 2;          // chunks of a row, of a lane and page-head
        const int kv = warp - 5;
        // the lane's chunk of its rows: the 8 lanes of a store phase take two units of four
        // rows, whose eight slots of a 128-B line differ (a lane order of 4 units by 2 rows met
        // each slot twice; the tensor cores' operand reads leave no bandwidth for that)
        const int chunk_u = U == 4 ? (lane & 1) | (lane >> 2 & 2) : lane & 1;
        const int chunk_row = U == 4 ? (lane >> 1 & 3) | (lane >> 2 & 4) : lane >> 1;
        const int ns = kv ? T::NSTV : T::NSTK;
        uint64_t* fbar = kv ? full_v : full_k;
        uint64_t* ebar = kv ? empty_v : empty_k;
        uint8_t* tiles = kv ? vtiles : ktiles;
        const uint8_t* data = p.kv_data + kv * Rec::HALF;
        auto resolve = [&](int o) {
            const uint32_t blk = id_of(o);
            if (blk < p.num_blocks) return (int)((p.layer * p.num_blocks + blk) * p.Hkv + (uint32_t)h);
            if (o < npages) atomicOr(p.err, kDevErrBlockId);
            return -1;
        };
        int next = 0;                                      // the page that fetch loads
        // (through a shuffle: a value that is itself a load's result would be waited for, with
        // the loads around it, wherever it is used)
        int cur = __shfl_sync(0xffffffffu, resolve(lane), lane), nxt = resolve(32 + lane);
        uint4 w[kGPages][PER];
        uint32_t sc[kGPages][PER][2];                      // K: both scales in the first, V: one each
        uint32_t shown = 0;                                // bit e * PER + i: the chunk holds keys
        auto fetch = [&](int e) {
            const int rec = __shfl_sync(0xffffffffu, cur, next & 31);
            // (a page without a record reads record 0; nothing of it is used)
            const uint8_t* half = data + (size_t)max(rec, 0) * Rec::BYTES;
            const int pos0 = page_of(next) * kBlockSize;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int u = chunk_u, rr = chunk_row + 8 * i, pos = pos0 + rr;
                w[e][i] = __ldg(reinterpret_cast<const uint4*>(half + rr * Rec::CODE_ROW + u * 16));
                const uint8_t* scales = half + Rec::KS;
                if (kv == 0) {
                    sc[e][i][0] = __ldg(reinterpret_cast<const uint16_t*>(scales + rr * Rec::GROUPS + 2 * u));
                } else {
                    sc[e][i][0] = __ldg(scales + 32 * u + rr);
                    sc[e][i][1] = __ldg(scales + 32 * u + 16 + rr);
                }
                // rows past the sequence's end, that no query of the CTA sees, or of a block id
                // outside the pool (flagged) become zeros
                const uint32_t bit = 1u << (e * PER + i);
                const bool in = next < npages && rec >= 0 && pos < total && (!WIN || pos < span.sinks || pos >= span.lo);
                shown = in ? shown | bit : shown & ~bit;
            }
            if ((++next & 31) == 0) {
                cur = __shfl_sync(0xffffffffu, nxt, lane);
                nxt = resolve(next + 32 + lane);
            }
        };
#pragma unroll
        for (int e = 0; e < kGPages; ++e) fetch(e);
        bool ok = true;
        for (int t = 0; t < nrounds && !withhold; ++t) {
            const int st = t % ns;
            if (t >= ns && !__all_sync(0xffffffffu, mbar_wait(&ebar[st], ((t / ns) - 1) & 1, deadline))) {
                ok = false;
                break;
            }
            uint8_t* tile = tiles + st * T::TILE;
#pragma unroll
            for (int e = 0; e < kGPages; ++e) {
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    const int u = chunk_u, rr = chunk_row + 8 * i, key = e * 16 + rr;
                    uint8_t* row = tile + (u >> 1) * (kGKeys * 128) + key * 128;
                    const uint32_t both = kv == 0 ? sc[e][i][0] : sc[e][i][0] | (sc[e][i][1] << 8);
                    const uint32_t s = e4m3x2_to_f16x2((shown >> (e * PER + i)) & 1u ? both : 0u);
                    const uint32_t s0 = __byte_perm(s, s, 0x1010u), s1 = __byte_perm(s, s, 0x3232u);
                    const uint32_t word[4] = {w[e][i].x, w[e][i].y, w[e][i].z, w[e][i].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t f[4];
                        fp4x8_to_f16(word[k], f);
                        const uint32_t mm = k < 2 ? s0 : s1;
                        *reinterpret_cast<uint4*>(row + ((((u & 1) * 4 + k) ^ (key & 7)) << 4)) =
                            make_uint4(f16x2_mul(f[0], mm), f16x2_mul(f[1], mm), f16x2_mul(f[2], mm), f16x2_mul(f[3], mm));
                    }
                }
                fetch(e);
            }
            // generic-proxy writes, read next by the tensor cores (async proxy)
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&fbar[st]);
        }
        if (!ok && lane == 0) atomicOr(p.err, kDevErrTimeout);
    }
    // tensor memory is freed by the warp that allocated it, after every use
    tc_fence_before();
    __syncthreads();
    if (warp == 4) {
        tc_fence_after();
        tmem_dealloc(tbase, 256);
    }
}

// Merge of a split tile: weights 2^(max_i - max) over its parts, as the decode's combine.  CTA
// (tile, KV head, 4 rows): a row per warp, D/32 elements per lane, every part's loads in
// flight together.  The geometry is computed while the parts still run.
constexpr int kMergeRows = 4;

template <class T, bool WIN>
__global__ void __launch_bounds__(128) prefill_merge_kernel(const PrefillParams p, int splits) {
    __shared__ int tpfx[kMaxBatchPerLaunch + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = (int)p.group;
    if (warp == 0) tile_prefix(p.cu_q, (int)p.B, (int)p.T, g, tpfx, lane);
    __syncthreads();
    TileGeom geo;
    const bool has = tile_geom<WIN>(p, tpfx, (int)blockIdx.x, geo);
    griddep_wait();
    if (!has) return;
    const Rounds rounds = split_rounds(geo.npages, splits);
    if (rounds.parts == 1) return;                     // written by its CTA
    constexpr int PER = T::D / 32;
    const size_t part0 = ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * splits;
    const int r = (int)blockIdx.z * kMergeRows + warp, row = geo.row0 + r;
    if (row >= geo.rows) return;
    float2 ml[kMaxSplit], v[kMaxSplit][PER / 2];
    float M = -INFINITY;
#pragma unroll
    for (int i = 0; i < kMaxSplit; ++i) {
        ml[i] = make_float2(-INFINITY, 0.0f);
        if (i >= rounds.parts) continue;
        ml[i] = __ldcg(reinterpret_cast<const float2*>(p.part_ml + ((part0 + i) * kGRows + r) * 2));
        const float* po = p.part_o + ((part0 + i) * kGRows + r) * T::D + lane * PER;
#pragma unroll
        for (int e = 0; e < PER / 2; ++e) v[i][e] = __ldcg(reinterpret_cast<const float2*>(po) + e);
    }
#pragma unroll
    for (int i = 0; i < kMaxSplit; ++i) M = fmaxf(M, ml[i].x);
    float l = 0.0f, o[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) o[e] = 0.0f;
#pragma unroll
    for (int i = 0; i < kMaxSplit; ++i) {
        if (ml[i].x == -INFINITY) continue;            // no such part, or one without a key the row sees
        const float w = ex2(ml[i].x - M);
        l += w * ml[i].y;
#pragma unroll
        for (int e = 0; e < PER / 2; ++e) {
            o[2 * e] += w * v[i][e].x;
            o[2 * e + 1] += w * v[i][e].y;
        }
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    const int tq = row / g;
    uint8_t* dst = reinterpret_cast<uint8_t*>(p.out) +
                   (((size_t)(geo.q_off + tq) * p.Hq + (size_t)blockIdx.y * g + (row - tq * g)) * T::D + lane * PER) * 2;
#pragma unroll
    for (int e = 0; e < PER; e += 2)
        reinterpret_cast<uint32_t*>(dst)[e / 2] =
            (uint32_t)pf_f32_to_io<T::IO>(o[e] * inv) | ((uint32_t)pf_f32_to_io<T::IO>(o[e + 1] * inv) << 16);
}

template <class T, bool WIN>
cudaError_t launch_grp(const PrefillLaunch& L) {
    // the dynamic-smem opt-in is per device; remember it per device ordinal
    static std::atomic<uint64_t> configured{0};
    int dev = 0;
    cudaGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (!(configured.load() & bit)) {
        cudaError_t e = cudaFuncSetAttribute(prefill_group_kernel<T, WIN>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM);
        if (e != cudaSuccess) return e;
        configured.fetch_or(bit);
    }
    const PrefillParams& p = L.p;
    // an upper bound on the CTAs: sum over b of ceil(n_b * group / 128) <= T * group / 128 + B
    const uint64_t ctas = ((uint64_t)p.T * p.group + kGRows - 1) / kGRows + p.B;
    // Parts of a tile: while there is an SM (and a tile of scratch) for each, and a block-table
    // row holds kMinRounds rounds for each.  (Llama-3-8B heads, 32 tokens behind 8192:
    // 130.6 us whole, 32.8 in eight parts.  Two CTAs on an SM slow one another, so
    // with two parts of 112 tiles, 40 tokens behind 1500 of 7 sequences, 40.2 us against
    // 33.8 whole.)
    const uint64_t tiles = ctas * p.Hkv, row_rounds = (p.bt_stride + kGPages - 1) / kGPages;
    uint64_t splits = (uint64_t)L.sms / tiles;
    splits = std::min<uint64_t>({splits, kMaxSplit, row_rounds / kMinRounds});
    if (splits < 1) splits = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas, p.Hkv, (unsigned)splits);
    cfg.blockDim = dim3(T::THREADS);
    cfg.dynamicSmemBytes = T::SMEM;
    cfg.stream = L.stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    if (p.flags & kDecodePdl) {
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    }
    cudaError_t e = cudaLaunchKernelEx(&cfg, prefill_group_kernel<T, WIN>, *L.tmap, p);
    if (e != cudaSuccess || splits == 1) return e;
    cfg.gridDim = dim3((unsigned)ctas, p.Hkv, kGRows / kMergeRows);
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, prefill_merge_kernel<T, WIN>, p, (int)splits);
}

template <int D, int IO>
cudaError_t launch_gd(const PrefillLaunch& L) {
    if (L.kv_kind == kFP4)
        return L.p.window > 0 ? launch_grp<Grp<D, IO, kFP4>, true>(L) : launch_grp<Grp<D, IO, kFP4>, false>(L);
    return launch_grp<Grp<D, IO, IO>, true>(L);      // f16 / bf16 pools: windowed calls only
}

}  // namespace

cudaError_t launch_group_prefill(const PrefillLaunch& L) {
    if (L.head_dim == 64) return L.io_kind == kBF16 ? launch_gd<64, kBF16>(L) : launch_gd<64, kF16>(L);
    return L.io_kind == kBF16 ? launch_gd<128, kBF16>(L) : launch_gd<128, kF16>(L);
}

}  // namespace vw
