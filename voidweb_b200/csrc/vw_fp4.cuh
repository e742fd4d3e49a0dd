// vw_fp4.cuh -- 4-bit KV codec on the device and the record it is stored in.
//
// Every 16 consecutive elements of a row share the scale s = E4M3(amax / 6) (to
// nearest even, saturating at 448) and each is held as the E2M1 code of x / s
// (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives; to nearest even, saturating); a
// group whose scale rounds to 0 holds zeros.  A code stands for code * s: two
// times four significant bits between 2^-10 and 2688, exact in f16 and in bf16,
// so the attention multiplies codes by scales in f16 and rounds nothing.  Neither
// quotient needs a division to fall on the right side of a border between codes
// (fp4_scale_code, fp4_quotient).  NaN elements encode as 6 (the conversion's
// rule) and do not count in amax.
//
// One page-head (16 tokens of one KV head) is one record of 18 D bytes, a K half
// and a V half:
//   K codes [16][D/2]      element 2i in the low half of byte i
//   K scales [16][D/16]    a token's groups together
//   V codes [16][D/2]
//   V scales [D/16][16]    a group's tokens together: the P V product pairs two tokens
//                          of one element
#pragma once
#include <cstdint>

namespace vw {

template <int D>
struct Fp4Rec {
    static constexpr int CODE_ROW = D / 2;      // bytes of one token's codes
    static constexpr int GROUPS = D / 16;
    static constexpr int KS = 16 * CODE_ROW;    // first K scale
    static constexpr int HALF = KS + 16 * GROUPS;
    static constexpr int V = HALF;              // first V code
    static constexpr int VS = HALF + KS;        // first V scale
    static constexpr int BYTES = 2 * HALF;
};
static_assert(Fp4Rec<128>::BYTES == 2304 && Fp4Rec<64>::BYTES == 1152, "18 D bytes");

// E4M3 scale code of a group with the given largest magnitude: amax / 6 as a product,
// within 2^-23 (relative), rounded to 15 bits (x - (x * 2^k - ..), the splitting of a
// product by a constant of Dekker's), which decides the code as the real quotient
// does: a border b between codes times 6 has at most 7 significant bits and amax at
// most 11, so amax / 6 is either b, and rounds to it, or off it by at least 2^-11 b.
// (Past 2^20 every group saturates.)
__device__ __forceinline__ uint32_t fp4_scale_code(float amax) {
    const float t = __fmul_rn(fminf(amax, 1048576.0f), 1.0f / 6.0f), c = __fmul_rn(t, 513.0f);
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(__fsub_rn(c, __fsub_rn(c, t))));
    return r & 0xFFu;
}

// f16 pair of codes times scales -> bf16 pair, exact: five or fewer mantissa bits, magnitudes
// 0 or normal.  The f16 bits shifted into bf16's fields are the value times 2^-112.
__device__ __forceinline__ uint32_t fp4_f16x2_to_bf16x2(uint32_t h) {
    uint32_t r;
    const uint32_t small = ((h >> 3) & 0x0FFF0FFFu) | (h & 0x80008000u);
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(small), "r"(0x77807780u));   // 2^112
    return r;
}

// Two E4M3 codes (low byte first) -> f16 pair.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t codes) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)codes));
    return r;
}

__device__ __forceinline__ float e4m3_to_f32(uint32_t code) {
    return f16_bits_to_f32(e4m3x2_to_f16x2(code) & 0xFFFFu);
}

// 1 / s of a scale code, 0 for a scale of 0 (all its elements then encode as 0).
__device__ __forceinline__ float fp4_inverse(uint32_t scale_code) {
    const float s = e4m3_to_f32(scale_code);
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
    return s == 0.0f ? 0.0f : r;
}

// x / s to a multiple of 2^-13, which decides the code as the real quotient does: x * inverse is within 2^-21 of
// x / s (relative).  A border b between codes (.25, .75, .. 5) times s has at most 7 significant bits and x at most
// 11, so x / s is either b, and the sum rounds to b exactly (b is a multiple of .25), or off it by at least
// 2^-11 b >= 2^-13, a whole step.  Two additions instead of a division, for two elements at once.
__device__ __forceinline__ float2 fp4_quotient(float x, float y, float inverse) {
    const float2 q = fma2(make_float2(x, y), make_float2(inverse, inverse), make_float2(-0.0f, -0.0f));
    return add2(add2(q, make_float2(1536.0f, 1536.0f)), make_float2(-1536.0f, -1536.0f));
}

// Four elements -> four E2M1 codes, the first in the low half of the low byte.
__device__ __forceinline__ uint32_t fp4_encode4(const float* v, float inverse) {
    const float2 a = fp4_quotient(v[0], v[1], inverse), b = fp4_quotient(v[2], v[3], inverse);
    uint16_t r;
    asm("{\n\t.reg .b8 lo, hi;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 lo, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 hi, %4, %3;\n\t"
        "mov.b16 %0, {lo, hi};\n\t}"
        : "=h"(r) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}

// Eight codes of a word -> four f16 pairs (exact).  The word is one that its lane
// loaded whole, or a bitwise mix of such words.  Under ptxas 12.9 a kernel that
// converted the bytes of its own parameter (perhaps from a uniform register) raised
// "misaligned address", and the bytes of a zero-extended 16-bit value became zeros;
// why is not known.
__device__ __forceinline__ void fp4x8_to_f16(uint32_t w, uint32_t (&r)[4]) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(w));
}

// The codes of two words interleaved: even elements into e, odd ones into o, each
// byte holding a's code in its low half and b's in its high half.
__device__ __forceinline__ void fp4_interleave(uint32_t a, uint32_t b, uint32_t& e, uint32_t& o) {
    e = (a & 0x0F0F0F0Fu) | ((b << 4) & 0xF0F0F0F0u);
    o = ((a >> 4) & 0x0F0F0F0Fu) | (b & 0xF0F0F0F0u);
}

__device__ __forceinline__ uint32_t f16x2_mul(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// bf16 queries meet 4-bit pages in f16.  A row whose largest magnitude lies in [2^-1, 2^16) goes
// as it is: its elements are multiples of 2^-24 or rounded to one, off by at most 2^-24 of
// the largest.  Any other row (its large elements would be infinite, its small ones lost) is
// multiplied by the power of two that brings its largest element to [2^14, 2^15), and the
// row's scores by the inverse.  `top`: the row's largest magnitude, bf16 bits; a row of zeros
// and one with an infinity or a NaN stay (1).
constexpr uint32_t kQueryLow = 0x3F00u, kQueryHigh = 0x4780u;      // 2^-1, 2^16

__device__ __forceinline__ float fp4_query_factor(uint32_t top) {
    if (top == 0u || top >= 0x7F80u || (top >= kQueryLow && top < kQueryHigh)) return 1.0f;
    return __uint_as_float((uint32_t)min(14 + 127 - (int)(top >> 7) + 127, 253) << 23);
}
__device__ __forceinline__ float fp4_query_unfactor(float factor) {      // 1 / factor, exactly
    return __uint_as_float((254u << 23) - __float_as_uint(factor));
}

// bf16 pair times a power of two -> f16 pair.
__device__ __forceinline__ uint32_t fp4_query_pair(uint32_t w, float factor) {
    return pack2<false>(bf16_bits_to_f32(w & 0xFFFFu) * factor, bf16_bits_to_f32(w >> 16) * factor);
}

// The largest magnitude of N bf16 pairs (bits; NaN if one is).
template <int N>
__device__ __forceinline__ uint32_t bf16_top(const uint32_t (&w)[N]) {
    uint32_t t[N];
#pragma unroll
    for (int k = 0; k < N; ++k) asm("abs.bf16x2 %0, %1;" : "=r"(t[k]) : "r"(w[k]));
#pragma unroll
    for (int n = N / 2; n > 0; n /= 2)
#pragma unroll
        for (int k = 0; k < n; ++k) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(t[k]) : "r"(t[k]), "r"(t[k + n]));
    return max(t[0] & 0xFFFFu, t[0] >> 16);
}

// One row of a record by one warp: lane l holds elements l*D/32 .. +D/32-1 (the
// first D/32 of v).  Writes codes and scales of token t into the records at rec
// and, when rec2 is given, the same at rec2.
template <int D>
__device__ __forceinline__ void fp4_store_row(uint8_t* rec, uint8_t* rec2, int kv, int t, int lane, const float (&v)[4]) {
    using R = Fp4Rec<D>;
    constexpr int PER = D / 32, LANES = 16 / PER;      // lanes of a group: 4 (D 128) or 8 (D 64)
    float amax = fmaxf(fabsf(v[0]), fabsf(v[1]));
    if constexpr (PER == 4) amax = fmaxf(amax, fmaxf(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
    for (int off = 1; off < LANES; off <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    const uint32_t sc = fp4_scale_code(amax);
    const uint32_t codes = fp4_encode4(v, fp4_inverse(sc));
    const int co = kv * R::V + t * R::CODE_ROW + lane * (PER / 2);
    const int g = lane / LANES;
    const int so = kv == 0 ? R::KS + t * R::GROUPS + g : R::VS + g * 16 + t;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        uint8_t* r = k == 0 ? rec : rec2;
        if (!r) continue;
        if constexpr (PER == 4) *reinterpret_cast<uint16_t*>(r + co) = (uint16_t)codes;
        else r[co] = (uint8_t)codes;
        if (lane % LANES == 0) r[so] = (uint8_t)sc;
    }
}

}  // namespace vw
