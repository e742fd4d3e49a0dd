// vw_decode_fp4.cu -- paged decode attention over 4-bit pools (vw_fp4.cuh has the codec
// and the record): o = softmax(q K^T * scale) V over each sequence's pages, the same
// split over the grid, partials and combine as the decode of the other pools
// (vw_split.cuh), optionally fused with the append and under a window.
//
//  * A page-head is 2304 B (head_dim 128), so at the memory's rate an SM has some 100
//    cycles for each: what bounds this kernel is instructions and their
//    latencies, not bytes.  The split of work among warps follows from that:
//    every warp has a ring of its own and copies the pages that it will read,
//    16 B per lane (cp.async, whose groups complete in order), as soon as the codes
//    of an earlier page are in registers.  There are no producer warps, no
//    barriers while pages stream, and no shared query ring; nothing here waits for
//    anything but its own copies.  (One bulk copy per page-head instead cost its
//    warp some 300 cycles to issue.)
//  * Warp w takes every W-th page-head of its CTA's range; the lanes resolve 32
//    of its pages at a time, one batch ahead.
//  * S^T = K Q^T and O^T = V^T P^T are m16n8k16 micro-tiles with the tokens as M (as K)
//    and the query heads of the KV head as N.  Codes become f16 with one byte
//    conversion per pair, times their scale with one packed multiply, both
//    exact.  Interior pages are taken kPair at a time, with no mask; the last
//    page and those a window cuts go one at a time.
//  * Online softmax in the log2 domain with a lazily raised maximum (a score must
//    exceed it by 8 before it is raised); sums and outputs in f32.
//    Probabilities enter P V as one f16, off by at most 2^-11 of themselves, 2^-25 below
//    2^-14: the results' relative error, in the root mean square, becomes 2.4e-4 to
//    2.8e-4 in f16, whose own rounding is 2.1e-4, and stays at 1.7e-3 in bf16; it saves
//    a quarter of the matrix instructions.
//  * bf16 queries go into f16 by rows (fp4_query_factor), so that no value of theirs is lost.
//  * Two CTAs of eight warps and 128 registers fill the register file (with two query-head
//    tiles, 64,512 of it), so the combine's CTAs come up as decode CTAs leave, not beside
//    them; the D 128 instances spill 32 to 44 B besides.
//  * Measured: Llama-3-8B heads, 64 sequences of 1024 to 16,384 tokens, 96.1 us a layer (4.2
//    TB/s; 325 instructions per page-head, ALU 51 %, and some 17 us of 512 segments'
//    starts and merges); Qwen2.5-7B heads, 16 sequences of 512 to 4096, 14.1 us.
#include <cuda_runtime.h>
#include <atomic>
#include <cstdint>

#include "vw_ptx.cuh"
#include "vw_fp4.cuh"
#include "vw_internal.h"
#include "vw_rope.cuh"
#include "vw_split.cuh"

#ifndef VW_FP4_WARPS
#define VW_FP4_WARPS 8
#endif
#ifndef VW_FP4_STAGES
#define VW_FP4_STAGES 3
#endif
#ifndef VW_FP4_PAIR
#define VW_FP4_PAIR 2
#endif

namespace vw {

namespace {

template <int D_, int NT_, int IO_>
struct F4 {
    static constexpr int D = D_, NT = NT_, IO = IO_;
    using Rec = Fp4Rec<D>;
    // Eight warps (128 registers) with one query-head tile: 64 sequences of 16,384 tokens, 8 KV
    // heads, 244 us against 257 with six; two tiles need the 168 registers of six
    static constexpr int W = NT == 1 ? VW_FP4_WARPS : 6, THREADS = W * 32;
    // interior page-heads per step (one: 257 us in the same case)
    static constexpr int PAIR = NT == 1 ? VW_FP4_PAIR : 1;
    static constexpr int SW = VW_FP4_STAGES * (128 / D);     // ring slots of a warp
    static constexpr int G = 8 * NT;
    static constexpr int KT = D / 16, MT = D / 16;
    // merge rows of D + 4 floats: a warp's stores of its O^T fragments then fall on
    // 32 different banks (with merge_col)
    static constexpr int MROW = D + 4;
    static constexpr int MERGE = W * 8 * (MROW + 2) * 4 + (W + 2) * 8 * 4;
    static constexpr int PFX = align_up_c((3 * kMaxBatchPerLaunch + 2) * 4, 128);
    static constexpr int RING = W * SW * Rec::BYTES;
    static constexpr int SMEM = 128 + RING + align_up_c(MERGE, 128) + PFX;
    static_assert(SW >= PAIR && SW < 32, "a step's pages are in the ring together");
    static_assert(RING % 128 == 0 && SMEM <= 233472 / 2 - 1024, "two CTAs per SM");
};

template <class T>
struct F4Smem {
    uint8_t* ring;      // [W][SW][BYTES]
    float *mo, *mm, *ml, *mf;   // one 8-head tile of the warp states, as in vw_decode.cu
    int *pfx, *nzp, *slen;
};

template <class T>
__device__ __forceinline__ F4Smem<T> f4_carve(uint8_t* p) {
    F4Smem<T> s;
    s.ring = p; p += T::RING;
    s.mo = reinterpret_cast<float*>(p);
    s.mm = s.mo + T::W * 8 * T::MROW;
    s.ml = s.mm + T::W * 8;
    s.mf = s.ml + T::W * 8;
    p += align_up_c(T::MERGE, 128);
    s.pfx = reinterpret_cast<int*>(p);
    s.nzp = s.pfx + (kMaxBatchPerLaunch + 1);
    s.slen = s.nzp + (kMaxBatchPerLaunch + 1);
    return s;
}

// The A rows of S^T = K Q^T and the columns of V^T are the page's tokens in the order
// fp4_token(r): rows that the lanes of one load phase read then lie an odd number
// of rows apart, which halves the bank conflicts of the V loads.
//  * K: lane (g, c) takes the D/4 codes c*D/4 .. of token rows g and g+8; k-step kt uses
//    its codes 4kt .. 4kt+3 (the reduction order inside a k-step is free; the
//    query fragments follow it), so a lane needs the scales of D/64 groups only.
//  * V: lane (g, c) takes the D/8 codes g*D/8 .. of token rows 2c, 2c+1, 2c+8, 2c+9; the
//    codes of two rows interleave into bytes that convert to a pair (two tokens,
//    one element) at once; row r of d-tile mt is fp4_out_d(r, mt).
__device__ __forceinline__ int fp4_token(int r) { return r ^ ((r >> 1) & 1); }

template <int D>
__device__ __forceinline__ int fp4_out_d(int r, int mt) {
    return (D / 8) * (r & 7) + (D / 16) * (r >> 3) + mt;
}

// Column of output element d in a merge row: a store's lanes g = 0..7 hold d values
// D/8 apart; flipping the low bits of d by them spreads the lanes over the banks.
template <int D>
__device__ __forceinline__ int merge_col(int d) {
    return d ^ ((d / (D / 8)) & 7);
}

template <int D>
struct Fp4Codes {
    uint32_t k[2][D / 32];     // codes of token rows g, g+8
    uint32_t v[4][D / 64];     // of token rows 2c, 2c+1, 2c+8, 2c+9
    uint32_t ks[2];            // E4M3 K scales of the lane's groups (rows g, g+8)
    uint32_t vs[2];            // E4M3 V scales of tokens 2c, 2c+1 and 2c+8, 2c+9, in the page's order
};

template <int D>
__device__ __forceinline__ void load_codes(const uint8_t* st, int lane, Fp4Codes<D>& f) {
    using R = Fp4Rec<D>;
    const int g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int rr = 0; rr < 2; ++rr) {
        const int tok = fp4_token(g) + 8 * rr;
        const uint8_t* kp = st + tok * R::CODE_ROW + c * (D / 8);
        if constexpr (D == 128) {
            const uint4 w = *reinterpret_cast<const uint4*>(kp);
            f.k[rr][0] = w.x; f.k[rr][1] = w.y; f.k[rr][2] = w.z; f.k[rr][3] = w.w;
            f.ks[rr] = *reinterpret_cast<const uint16_t*>(st + R::KS + tok * R::GROUPS + 2 * c);
        } else {
            const uint2 w = *reinterpret_cast<const uint2*>(kp);
            f.k[rr][0] = w.x; f.k[rr][1] = w.y;
            f.ks[rr] = st[R::KS + tok * R::GROUPS + c];
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int tok = fp4_token(2 * c + (r & 1)) + 8 * (r >> 1);
        const uint8_t* vp = st + R::V + tok * R::CODE_ROW + g * (D / 16);
        if constexpr (D == 128) {
            const uint2 w = *reinterpret_cast<const uint2*>(vp);
            f.v[r][0] = w.x; f.v[r][1] = w.y;
        } else {
            f.v[r][0] = *reinterpret_cast<const uint32_t*>(vp);
        }
    }
#pragma unroll
    for (int q = 0; q < 2; ++q)
        f.vs[q] = *reinterpret_cast<const uint16_t*>(st + R::VS + (D == 128 ? g : g >> 1) * 16 + 8 * q + 2 * c);
}

// Query fragments (B operand of S^T = K Q^T) of the segment's query rows: lane (g, c)
// holds elements c*D/4 .. +D/4-1 of query head g (and g + 8), in f16; rotated at
// position pos first with rope_theta > 0 (the partner d +- D/2 is in lane c ^ 2) and
// rounded to the io type, as a separate RoPE pass would.  Returns (to the whole warp) whether
// bf16 rows are multiplied to fit f16 (fp4_query_factor); the inverses are then in
// unscale[nt * W * 8 + head of the tile].
template <class T>
__device__ __forceinline__ bool load_q(const DecodeParams& p, const uint8_t* rows, int lane, float pos,
                                       uint32_t (&qf)[T::NT][T::KT][2], float* unscale) {
    constexpr int NW = T::D / 8;
    const int c = lane & 3;
    bool any = false;
#pragma unroll
    for (int nt = 0; nt < T::NT; ++nt) {
        const int j = nt * 8 + (lane >> 2);
        const bool live = j < (int)p.group;
        const uint8_t* row = rows + (live ? j : 0) * T::D * 2 + c * (T::D / 2);
        uint32_t w[NW];
#pragma unroll
        for (int u = 0; u < NW / 4; ++u) {
            const uint4 v = live ? *reinterpret_cast<const uint4*>(row + u * 16) : make_uint4(0, 0, 0, 0);
            w[4 * u] = v.x; w[4 * u + 1] = v.y; w[4 * u + 2] = v.z; w[4 * u + 3] = v.w;
        }
        if (p.rope_theta > 0.0f) {
            const bool lo = c < 2;                  // elements below D/2
#pragma unroll
            for (int m = 0; m < NW; ++m) {
                const uint32_t other = __shfl_xor_sync(0xffffffffu, w[m], 2);
                const uint32_t rw = lo ? w[m] : other, iw = lo ? other : w[m];
                float r0 = io_to_f32<T::IO>(rw & 0xFFFFu), i0 = io_to_f32<T::IO>(iw & 0xFFFFu);
                float r1 = io_to_f32<T::IO>(rw >> 16), i1 = io_to_f32<T::IO>(iw >> 16);
                const int d = (c & 1) * (T::D / 4) + 2 * m;   // index of the lower element
                rope_pair(r0, i0, d, T::D, p.rope_theta, pos);
                rope_pair(r1, i1, d + 1, T::D, p.rope_theta, pos);
                w[m] = lo ? ((uint32_t)f32_to_io<T::IO>(r0) | ((uint32_t)f32_to_io<T::IO>(r1) << 16))
                          : ((uint32_t)f32_to_io<T::IO>(i0) | ((uint32_t)f32_to_io<T::IO>(i1) << 16));
            }
        }
        if constexpr (T::IO == kBF16) {
            // (Every warp does this for every segment, so the ordinary case has no more than two
            // votes: 16 sequences of Qwen2.5-7B heads, 512 to 4096 tokens, with fused append 14.66 us a
            // layer, 14.8 with the row's maximum reduced over its lanes, 14.4 with no check.)
            const uint32_t own = bf16_top<NW>(w);
            uint32_t big = __ballot_sync(0xffffffffu, !live || own >= kQueryLow);
            big |= big >> 1;
            big |= big >> 2;                        // bit 4 g: row g has an element of 2^-1 or more
            if (__any_sync(0xffffffffu, own >= kQueryHigh) || (big & 0x11111111u) != 0x11111111u) {
                uint32_t top = max(own, __shfl_xor_sync(0xffffffffu, own, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float factor = fp4_query_factor(top);
                if (c == 0) unscale[nt * T::W * 8 + (lane >> 2)] = fp4_query_unfactor(factor);
                any = true;
#pragma unroll
                for (int m = 0; m < NW; ++m) w[m] = fp4_query_pair(w[m], factor);
            } else {
#pragma unroll
                for (int m = 0; m < NW; ++m) w[m] = fp4_query_pair(w[m], 1.0f);
                if (T::NT > 1 && c == 0) unscale[nt * T::W * 8 + (lane >> 2)] = 1.0f;
            }
        }
#pragma unroll
        for (int m = 0; m < NW; ++m) qf[nt][m >> 1][m & 1] = w[m];
    }
    __syncwarp();
    return any;
}

// This lane's D/32 elements of the step's new K and V rows of one (sequence, KV head), the K
// row rotated at position pos (partners d +- D/2 in lane ^ 16).
template <class T>
__device__ __forceinline__ void load_new_rows(const DecodeParams& p, size_t row, int lane, float pos,
                                              uint32_t (&nkv)[2][2]) {
    constexpr int PER = T::D / 32;
    const size_t off = (row * T::D + lane * PER) * 2;
#pragma unroll
    for (int k = 0; k < PER / 2; ++k) {
        nkv[0][k] = reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint8_t*>(p.k_new) + off)[k];
        nkv[1][k] = reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint8_t*>(p.v_new) + off)[k];
    }
    if (p.rope_theta > 0.0f) {
        const bool lo = lane < 16;
#pragma unroll
        for (int k = 0; k < PER / 2; ++k) {
            const uint32_t own = nkv[0][k];
            const uint32_t other = __shfl_xor_sync(0xffffffffu, own, 16);
            const uint32_t rw = lo ? own : other, iw = lo ? other : own;
            float r0 = io_to_f32<T::IO>(rw & 0xFFFFu), i0 = io_to_f32<T::IO>(iw & 0xFFFFu);
            float r1 = io_to_f32<T::IO>(rw >> 16), i1 = io_to_f32<T::IO>(iw >> 16);
            const int d = (lane & 15) * PER + 2 * k;
            rope_pair(r0, i0, d, T::D, p.rope_theta, pos);
            rope_pair(r1, i1, d + 1, T::D, p.rope_theta, pos);
            nkv[0][k] = lo ? ((uint32_t)f32_to_io<T::IO>(r0) | ((uint32_t)f32_to_io<T::IO>(r1) << 16))
                           : ((uint32_t)f32_to_io<T::IO>(i0) | ((uint32_t)f32_to_io<T::IO>(i1) << 16));
        }
    }
}

// V rows [from, to) of a staged record become zeros, codes and scales (a code of 0 times a
// NaN scale is NaN), so that masked tokens inject nothing through 0 * garbage.
template <int D>
__device__ __forceinline__ void zero_rows(uint8_t* st, int from, int to, int lane) {
    using R = Fp4Rec<D>;
    for (int k = lane; k < (to - from) * (R::CODE_ROW / 16); k += 32)
        reinterpret_cast<uint4*>(st + R::V + from * R::CODE_ROW)[k] = make_uint4(0, 0, 0, 0);
    for (int k = lane; k < (to - from) * R::GROUPS; k += 32)
        st[R::VS + k % R::GROUPS * 16 + from + k / R::GROUPS] = 0;
}

// A warp's pages of its CTA's range: page k of the warp is page warp + k * W of the
// range.  Lanes resolve 32 of them at once into record numbers (-1: a block id outside
// the pool).
template <class T, bool WIN>
struct Feed {
    const DecodeParams& p;
    const F4Smem<T>& sm;
    uint8_t* ring;
    int begin, n, warp, lane;
    int left;                    // pages not issued yet
    int issued = 0;              // pages issued; those of batch issued/32 are in cur
    int cur, nxt;
    uint32_t in = 0, out = 0;    // byte offsets of the slot to fill and of the oldest page (the ring is no power of two)

    static __device__ __forceinline__ uint32_t after(uint32_t s) {
        return s + T::Rec::BYTES == T::SW * T::Rec::BYTES ? 0u : s + T::Rec::BYTES;
    }

    __device__ __forceinline__ int resolve(int k) const {
        const int i = warp + k * T::W;
        if (i >= n) return -1;
        const int x = begin + i;
        const int b = find_seq(sm.pfx, (int)p.B, (int)p.Hkv, x);
        const int np = sm.pfx[b + 1] - sm.pfx[b];
        const int r = x - (int)p.Hkv * sm.pfx[b];
        const int h = r / np, o = r - h * np;
        const int pg = WIN ? decode_span(sm.slen[b], (int)p.bt_stride, p.window, p.sinks).page(o) : o;
        const uint32_t blk = __ldg(p.block_tables + (size_t)b * p.bt_stride + pg);
        if (blk >= p.num_blocks) {
            set_err(p.err, kDevErrBlockId);
            return -1;
        }
        return (int)((p.layer * p.num_blocks + blk) * p.Hkv + (uint32_t)h);
    }

    // (the whole warp) copy the next page into its slot, which is free.  Every call ends a
    // group, so that page k is in group k whether it exists or not.
    __device__ __forceinline__ void issue() {
        if (left > 0) {
            --left;
            const int rec = __shfl_sync(0xffffffffu, cur, issued & 31);
            uint8_t* st = ring + in;
            in = after(in);
            if (rec >= 0) {
                const uint8_t* src = p.kv_data + (size_t)rec * T::Rec::BYTES + lane * 16;
                uint8_t* dst = st + lane * 16;
#pragma unroll
                for (int k = 0; k < T::Rec::BYTES / 16; k += 32)
                    if (k + 32 <= T::Rec::BYTES / 16 || k + lane < T::Rec::BYTES / 16) cp_async16(dst + k * 16, src + k * 16);
            } else {
                // a block id outside the pool (flagged): a record of zeros
                for (int k = lane; k < T::Rec::BYTES / 16; k += 32) reinterpret_cast<uint4*>(st)[k] = make_uint4(0, 0, 0, 0);
            }
            if ((++issued & 31) == 0) {
                cur = __shfl_sync(0xffffffffu, nxt, lane);
                nxt = resolve(issued + 32 + lane);
            }
        }
        cp_async_commit();
    }
};

template <class T>
struct State {
    float o[T::NT][T::MT][4];
    float m[T::NT][2], l[T::NT][2];      // running maximum (log2 units) and sum
    float thr[T::NT][2];                 // raw score above which the maximum is raised
};

// P page-heads into the state.  MASK: token t counts when its bit in `seen` is set.
template <class T, bool WIN, int P, bool MASK>
__device__ __forceinline__ void step(const DecodeParams& p, Feed<T, WIN>& feed, uint8_t* const (&st)[P], uint32_t seen,
                                     const uint32_t (&qf)[T::NT][T::KT][2], bool scaled, const float* unscale, State<T>& s,
                                     int lane) {
    Fp4Codes<T::D> f[P];
#pragma unroll
    for (int a = 0; a < P; ++a) load_codes<T::D>(st[a], lane, f[a]);
    // all the record's bytes that this warp needs are in registers: refill the slots
    __syncwarp();
#pragma unroll
    for (int a = 0; a < P; ++a) feed.issue();

    // ---- S^T = K Q^T
    float sc[P][T::NT][4];
#pragma unroll
    for (int a = 0; a < P; ++a)
#pragma unroll
        for (int nt = 0; nt < T::NT; ++nt) sc[a][nt][0] = sc[a][nt][1] = sc[a][nt][2] = sc[a][nt][3] = 0.0f;
#pragma unroll
    for (int a = 0; a < P; ++a) {
        const uint32_t s0 = e4m3x2_to_f16x2(f[a].ks[0]), s1 = e4m3x2_to_f16x2(f[a].ks[1]);
#pragma unroll
        for (int kw = 0; kw < T::KT / 2; ++kw) {               // a word of codes: two k-steps
            const uint32_t sel = (T::D == 128 && kw >= T::KT / 4) ? 0x3232u : 0x1010u;
            const uint32_t m0 = __byte_perm(s0, s0, sel), m1 = __byte_perm(s1, s1, sel);
            uint32_t r0[4], r1[4];
            fp4x8_to_f16(f[a].k[0][kw], r0);
            fp4x8_to_f16(f[a].k[1][kw], r1);
#pragma unroll
            for (int j = 0; j < 4; ++j) { r0[j] = f16x2_mul(r0[j], m0); r1[j] = f16x2_mul(r1[j], m1); }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int nt = 0; nt < T::NT; ++nt)
                    mma_16816<false>(sc[a][nt], r0[2 * h], r1[2 * h], r0[2 * h + 1], r1[2 * h + 1],
                                     qf[nt][2 * kw + h][0], qf[nt][2 * kw + h][1]);
        }
    }
    if (scaled) {                                              // (seldom: fp4_query_factor)
#pragma unroll
        for (int nt = 0; nt < T::NT; ++nt) {
            const float f0 = unscale[nt * T::W * 8 + 2 * (lane & 3)], f1 = unscale[nt * T::W * 8 + 2 * (lane & 3) + 1];
#pragma unroll
            for (int a = 0; a < P; ++a) {
                sc[a][nt][0] *= f0; sc[a][nt][1] *= f1;
                sc[a][nt][2] *= f0; sc[a][nt][3] *= f1;
            }
        }
    }

    // ---- online softmax
    if constexpr (MASK) {
        const int t0 = fp4_token(lane >> 2);
        const bool v0 = (seen >> t0) & 1u, v1 = (seen >> (t0 + 8)) & 1u;
#pragma unroll
        for (int a = 0; a < P; ++a)
#pragma unroll
            for (int nt = 0; nt < T::NT; ++nt) {
                sc[a][nt][0] = v0 ? sc[a][nt][0] : -INFINITY;
                sc[a][nt][1] = v0 ? sc[a][nt][1] : -INFINITY;
                sc[a][nt][2] = v1 ? sc[a][nt][2] : -INFINITY;
                sc[a][nt][3] = v1 ? sc[a][nt][3] : -INFINITY;
            }
    }
    float mx[T::NT][2];
    bool need = false;
#pragma unroll
    for (int nt = 0; nt < T::NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            mx[nt][k] = fmaxf(sc[0][nt][k], sc[0][nt][2 + k]);
#pragma unroll
            for (int a = 1; a < P; ++a) mx[nt][k] = fmaxf(mx[nt][k], fmaxf(sc[a][nt][k], sc[a][nt][2 + k]));
            need |= mx[nt][k] > s.thr[nt][k];
        }
    if (__any_sync(0xffffffffu, need)) {
#pragma unroll
        for (int nt = 0; nt < T::NT; ++nt) {
            float al[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float x = mx[nt][k];
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
                const float mn = fmaxf(s.m[nt][k], x * p.scale_log2);
                al[k] = ex2(s.m[nt][k] - mn);
                s.m[nt][k] = mn;
                s.thr[nt][k] = (mn + kRescaleThreshold) / p.scale_log2;
                s.l[nt][k] *= al[k];
            }
#pragma unroll
            for (int mt = 0; mt < T::MT; ++mt) {
                s.o[nt][mt][0] *= al[0]; s.o[nt][mt][1] *= al[1];
                s.o[nt][mt][2] *= al[0]; s.o[nt][mt][3] *= al[1];
            }
        }
    }
    uint32_t pb[P][T::NT][2];
#pragma unroll
    for (int a = 0; a < P; ++a)
#pragma unroll
        for (int nt = 0; nt < T::NT; ++nt) {
            const float p00 = ex2(fmaf(sc[a][nt][0], p.scale_log2, -s.m[nt][0]));
            const float p01 = ex2(fmaf(sc[a][nt][1], p.scale_log2, -s.m[nt][1]));
            const float p10 = ex2(fmaf(sc[a][nt][2], p.scale_log2, -s.m[nt][0]));
            const float p11 = ex2(fmaf(sc[a][nt][3], p.scale_log2, -s.m[nt][1]));
            s.l[nt][0] += p00 + p10;
            s.l[nt][1] += p01 + p11;
            pb[a][nt][0] = movmatrix_t(pack2<false>(p00, p01));
            pb[a][nt][1] = movmatrix_t(pack2<false>(p10, p11));
        }

    // ---- O^T += V^T P^T
    const uint32_t order = (lane & 1) ? 0x1032u : 0x3210u;      // fp4_token swaps the pair of odd c
#pragma unroll
    for (int a = 0; a < P; ++a) {
        // even and odd elements of the lane's run, tokens 2c, 2c+1 (q 0) and 2c+8, 2c+9
        uint32_t ve[2][2][T::D / 64];
        uint32_t vs[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const uint32_t x = e4m3x2_to_f16x2(f[a].vs[q]);
            vs[q] = __byte_perm(x, x, order);
#pragma unroll
            for (int k = 0; k < T::D / 64; ++k)
                fp4_interleave(f[a].v[2 * q][k], f[a].v[2 * q + 1][k], ve[0][q][k], ve[1][q][k]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            // element x of the run: row g of d-tile x for x < MT, row g + 8 of d-tile x - MT after
            uint32_t w[2][T::D / 64][4];
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int k = 0; k < T::D / 64; ++k) {
                    fp4x8_to_f16(ve[e][q][k], w[q][k]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[q][k][j] = f16x2_mul(w[q][k][j], vs[q]);
                }
#pragma unroll
            for (int mt = e; mt < T::MT; mt += 2) {
                const int x1 = T::MT + mt;
#pragma unroll
                for (int nt = 0; nt < T::NT; ++nt)
                    mma_16816<false>(s.o[nt][mt], w[0][0][mt >> 1], w[0][x1 >> 3][(x1 & 7) >> 1], w[1][0][mt >> 1],
                                     w[1][x1 >> 3][(x1 & 7) >> 1], pb[a][nt][0], pb[a][nt][1]);
            }
        }
    }
}

template <class T, bool WIN>
__global__ void __launch_bounds__(T::THREADS, 2) fp4_decode_kernel(const DecodeParams p) {
    extern __shared__ __align__(128) uint8_t smem_raw[];
    const F4Smem<T> sm = f4_carve<T>(smem_raw + ((128u - (smem_u32(smem_raw) & 127u)) & 127u));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
    constexpr int W = T::W, NTH = T::THREADS;
    // Programmatic dependent launch, as in vw_decode.cu: without early pages
    // everything waits for the predecessor; the combine may launch as soon as it finds room.
    const bool pdl = (p.flags & kDecodePdl) != 0, early = pdl && (p.flags & kDecodeEarlyPages) != 0;
    if (pdl && !early) griddep_wait();
    griddep_launch_dependents();
    int begin, end;
    if (p.plan != nullptr) {
        const int* entry = p.plan + kPlanCta + (size_t)blockIdx.x * kPlanCtaInts;
        for (int i = tid; i <= (int)p.B; i += NTH) {
            sm.pfx[i] = __ldcg(p.plan + kPlanPfx + i);
            sm.nzp[i] = __ldcg(p.plan + kPlanNzp + i);
            if (i < (int)p.B) sm.slen[i] = (int)__ldg(p.seq_lens + i);
        }
        begin = __ldcg(entry);
        end = __ldcg(entry + 1);
        __syncthreads();
    } else {
        if (warp == 0)
            warp_prefixes<WIN>(p.seq_lens, (int)p.B, (int)p.bt_stride, p.err, blockIdx.x == 0, sm.pfx, sm.nzp, sm.slen,
                               lane, p.window, p.sinks);
        __syncthreads();
        const int total = (int)p.Hkv * sm.pfx[p.B], cost = (int)p.seg_cost;
        const int vper = virtual_per_cta(virtual_total(total, (int)p.Hkv * sm.nzp[p.B], cost), (int)gridDim.x);
        begin = range_start(sm.pfx, sm.nzp, (int)p.B, (int)p.Hkv, cost, (int)blockIdx.x * vper);
        end = range_start(sm.pfx, sm.nzp, (int)p.B, (int)p.Hkv, cost, ((int)blockIdx.x + 1) * vper);
    }
    // (a batch of no pages: the grids behind this one still come after those before it)
    griddep_wait_if(early && blockIdx.x == 0 && begin >= end);
    if (begin >= end) return;

    Feed<T, WIN> feed{p, sm, sm.ring + warp * T::SW * T::Rec::BYTES, begin, end - begin, warp, lane,
                      (end - begin - warp + W - 1) / W};
    // (through a shuffle: a value that is itself a load's result would be waited for, with the
    // loads around it, wherever it is used)
    feed.cur = __shfl_sync(0xffffffffu, feed.resolve(lane), lane);
    for (int k = 0; k < T::SW; ++k) feed.issue();
    feed.nxt = feed.resolve(32 + lane);
    if (early) griddep_wait();            // q, k_new, v_new may come from the predecessor

    const int Hkv = (int)p.Hkv, g = (int)p.group;
    const bool append = p.k_new != nullptr;
    int i = warp;                         // the warp's next page of the range
    for (int x = begin; x < end;) {
        const int b = find_seq(sm.pfx, (int)p.B, Hkv, x);
        const int np = sm.pfx[b + 1] - sm.pfx[b];
        const int r = x - Hkv * sm.pfx[b];
        const int h = r / np, pg0 = r - h * np;
        const int cnt = min(np - pg0, end - x);
        const bool complete = cnt == np;
        const int i_base = x - begin, i_end = i_base + cnt;
        const int seq_len = sm.slen[b];
        PageSpan span{};
        if constexpr (WIN) span = decode_span(seq_len, (int)p.bt_stride, p.window, p.sinks);

        uint32_t nkv[2][2] = {{0u, 0u}, {0u, 0u}};
        if (append && pg0 + cnt == np) load_new_rows<T>(p, (size_t)(b * Hkv + h), lane, (float)(seq_len - 1), nkv);
        uint32_t qf[T::NT][T::KT][2];
        // (this warp's maxima of the merge below: nothing is there while pages stream)
        float* const unscale = sm.mm + warp * 8;
        const bool scaled = load_q<T>(p, reinterpret_cast<const uint8_t*>(p.q) + (size_t)(b * p.Hq + h * p.group) * T::D * 2,
                                      lane, (float)(seq_len - 1), qf, unscale);

        State<T> s;
#pragma unroll
        for (int nt = 0; nt < T::NT; ++nt) {
            s.m[nt][0] = s.m[nt][1] = s.thr[nt][0] = s.thr[nt][1] = -INFINITY;
            s.l[nt][0] = s.l[nt][1] = 0.0f;
#pragma unroll
            for (int mt = 0; mt < T::MT; ++mt) s.o[nt][mt][0] = s.o[nt][mt][1] = s.o[nt][mt][2] = s.o[nt][mt][3] = 0.0f;
        }
        // pages that are not wholly visible: the last one, and (rows [sinks, lo)) those a window cuts
        auto whole = [&](int pg) {
            if (pg == np - 1) return false;
            if constexpr (WIN) {
                int a, z;
                span.hidden(span.page(pg), a, z);
                return a >= z;
            }
            return true;
        };
        auto slot = [&]() {
            uint8_t* st = feed.ring + feed.out;
            feed.out = Feed<T, WIN>::after(feed.out);
            return st;
        };
        while (i < i_end) {
            const int pg = pg0 + (i - i_base);
            // SW groups follow the last page consumed: the oldest one or two have to be there,
            // for this lane, then (__syncwarp) for all
            if (whole(pg)) {
                if (T::PAIR == 2 && i + W < i_end && whole(pg + W)) {
                    cp_async_wait<T::SW - 2>();
                    __syncwarp();
                    uint8_t* const st[2] = {slot(), slot()};
                    step<T, WIN, 2, false>(p, feed, st, 0, qf, scaled, unscale, s, lane);
                    i += 2 * W;
                } else {
                    cp_async_wait<T::SW - 1>();
                    __syncwarp();
                    uint8_t* const st[1] = {slot()};
                    step<T, WIN, 1, false>(p, feed, st, 0, qf, scaled, unscale, s, lane);
                    i += W;
                }
                continue;
            }
            cp_async_wait<T::SW - 1>();
            __syncwarp();
            uint8_t* const st[1] = {slot()};
            const int lp = WIN ? span.page(pg) : pg;
            uint32_t seen = 0xFFFFu;
            if (pg == np - 1) {
                // a seq_len beyond the table (flagged in the prologue) reads its
                // pages as full and appends nothing
                int valid = seq_len - lp * 16;
                if (append && valid <= 16) {
                    const uint32_t blk = __ldg(p.block_tables + (size_t)b * p.bt_stride + lp);
                    const bool ok = blk < p.num_blocks;
                    uint8_t* rec = p.kv_data + (((size_t)p.layer * p.num_blocks + (ok ? blk : 0)) * p.Hkv + h) * T::Rec::BYTES;
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int k = 0; k < T::D / 64; ++k) {
                            v[2 * k] = io_to_f32<T::IO>(nkv[kv][k] & 0xFFFFu);
                            v[2 * k + 1] = io_to_f32<T::IO>(nkv[kv][k] >> 16);
                        }
                        fp4_store_row<T::D>(st[0], ok ? rec : nullptr, kv, valid - 1, lane, v);
                    }
                }
                valid = min(valid, 16);
                if (valid < 16) zero_rows<T::D>(st[0], valid, 16, lane);
                seen = 0xFFFFu >> (16 - valid);
            }
            if constexpr (WIN) {
                int a, z;
                span.hidden(lp, a, z);
                if (a < z) {
                    zero_rows<T::D>(st[0], a, z, lane);
                    seen &= ~((0xFFFFu >> (16 - (z - a))) << a);
                }
            }
            __syncwarp();
            step<T, WIN, 1, true>(p, feed, st, seen, qf, scaled, unscale, s, lane);
            i += W;
        }

        // ---- merge the W warps' states for this segment, one 8-head tile at a time
        // (three barriers per tile), as in vw_decode.cu
        float* mo = sm.mo + warp * 8 * T::MROW;
        uint16_t* out = reinterpret_cast<uint16_t*>(p.out);
        const int piece = (x == begin) ? 0 : 1;
        float* po = p.part_o + ((size_t)blockIdx.x * 2 + piece) * T::G * T::D;
        float* pml = p.part_ml + ((size_t)blockIdx.x * 2 + piece) * T::G * 2;
#pragma unroll
        for (int nt = 0; nt < T::NT; ++nt) {
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
                s.l[nt][0] += __shfl_xor_sync(0xffffffffu, s.l[nt][0], off);
                s.l[nt][1] += __shfl_xor_sync(0xffffffffu, s.l[nt][1], off);
            }
            const int jl = 2 * (lane & 3), r0 = lane >> 2;      // this lane's heads in the tile: jl, jl + 1
#pragma unroll
            for (int mt = 0; mt < T::MT; ++mt) {
                const int dA = merge_col<T::D>(fp4_out_d<T::D>(r0, mt)), dB = merge_col<T::D>(fp4_out_d<T::D>(r0 + 8, mt));
                mo[jl * T::MROW + dA] = s.o[nt][mt][0];
                mo[(jl + 1) * T::MROW + dA] = s.o[nt][mt][1];
                mo[jl * T::MROW + dB] = s.o[nt][mt][2];
                mo[(jl + 1) * T::MROW + dB] = s.o[nt][mt][3];
            }
            if (lane < 4) {
                sm.mm[warp * 8 + jl] = s.m[nt][0];
                sm.mm[warp * 8 + jl + 1] = s.m[nt][1];
                sm.ml[warp * 8 + jl] = s.l[nt][0];
                sm.ml[warp * 8 + jl + 1] = s.l[nt][1];
            }
            __syncthreads();
            const int jn = min(8, g - nt * 8);    // live query heads of the tile
            if (tid < jn) {
                float M = -INFINITY;
#pragma unroll
                for (int w = 0; w < W; ++w) M = fmaxf(M, sm.mm[w * 8 + tid]);
                float Ls = 0.0f;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const float mw = sm.mm[w * 8 + tid];
                    const float f = mw > -INFINITY ? ex2(mw - M) : 0.0f;
                    Ls += sm.ml[w * 8 + tid] * f;
                    sm.mf[w * 8 + tid] = f;
                }
                sm.mf[W * 8 + tid] = M;
                sm.mf[(W + 1) * 8 + tid] = Ls;
            }
            __syncthreads();
            for (int idx = tid; idx < jn * T::D; idx += NTH) {
                const int jt = idx / T::D, d = idx - jt * T::D, j = nt * 8 + jt;
                float Os = 0.0f;
#pragma unroll
                for (int w = 0; w < W; ++w)
                    Os += sm.mo[(w * 8 + jt) * T::MROW + merge_col<T::D>(d)] * sm.mf[w * 8 + jt];
                if (complete) {
                    out[((size_t)b * p.Hq + (size_t)h * g + j) * T::D + d] =
                        f32_to_io<T::IO>(Os / sm.mf[(W + 1) * 8 + jt]);
                } else {
                    po[j * T::D + d] = Os;
                    if (d == 0) { pml[j * 2] = sm.mf[W * 8 + jt]; pml[j * 2 + 1] = sm.mf[(W + 1) * 8 + jt]; }
                }
            }
            __syncthreads();
        }
        x += cnt;
    }
    // (each warp has consumed every page that it copied: none is in flight)
}

template <class T, bool WIN>
cudaError_t launch_f4(const DecodeLaunch& L) {
    // the dynamic-smem opt-in is per device; remember it per device ordinal
    static std::atomic<uint64_t> configured{0};
    int dev = 0;
    cudaGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (!(configured.load() & bit)) {
        cudaError_t e = cudaFuncSetAttribute(fp4_decode_kernel<T, WIN>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(fp4_decode_kernel<T, WIN>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                     (int)cudaSharedmemCarveoutMaxShared);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(combine_kernel<T::D, T::G, T::IO, WIN>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                     (int)cudaSharedmemCarveoutMaxShared);
        if (e != cudaSuccess) return e;
        configured.fetch_or(bit);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(L.grid);
    cfg.blockDim = dim3(T::THREADS);
    cfg.dynamicSmemBytes = T::SMEM;
    cfg.stream = L.stream;
    cudaLaunchAttribute attr[1];
    if (L.p.flags & kDecodePdl) {
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    }
    cudaError_t e = cudaLaunchKernelEx(&cfg, fp4_decode_kernel<T, WIN>, L.p);
    if (e != cudaSuccess) return e;
    return launch_combine<T::D, T::G, T::IO, WIN>(L, 1.0f);
}

template <int D, int IO>
cudaError_t launch_fd(const DecodeLaunch& L) {
    if (L.p.window > 0) return L.p.group <= 8 ? launch_f4<F4<D, 1, IO>, true>(L) : launch_f4<F4<D, 2, IO>, true>(L);
    return L.p.group <= 8 ? launch_f4<F4<D, 1, IO>, false>(L) : launch_f4<F4<D, 2, IO>, false>(L);
}

}  // namespace

cudaError_t launch_fp4_decode(const DecodeLaunch& L) {
    if (L.head_dim == 64) return L.io_kind == kBF16 ? launch_fd<64, kBF16>(L) : launch_fd<64, kF16>(L);
    return L.io_kind == kBF16 ? launch_fd<128, kBF16>(L) : launch_fd<128, kF16>(L);
}

}  // namespace vw
