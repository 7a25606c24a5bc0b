// How K and V vectors are held in pages of 8 and 4 bits: shared by what writes, reads and
// attends to them (kv_cache.hip, kv_step.hip, attention_paged.hip).
//
// 8 bits: s = f32(max|x| / 127), c = clamp(rint(f32(x / s)), -127, 127), value = c * s
// (kv_cache.hip).
// 4 bits: every 32 neighbouring dims have a base z and a scale s in f16,
//   z = f16(min x), s = f16(f32(f32(max x - z) / 15)), c = clamp(rint(f32(f32(x - z) / s)), 0, 15),
//   value = f16(c * s + z), rounded once,
// so a value is off by at most s / 2, by the rounding of the codes' ends (15 s 2^-11 and z 2^-11)
// and by its own (2^-11 of it).  An f16 value, because both products of the attention take f16
// operands: what they multiply is then what the codes stand for, exactly.  Elements beyond f16's
// range are held to its ends; a group with an infinity or a NaN gets s = z = NaN and reads as NaN.
// Dim i of a vector is nibble i % 8 of word i / 8 (its codes, head_dim / 2 bytes), and group i / 32
// is word i / 32 of its scales, s below z.
#pragma once
#include "common.hpp"
#include "kernels.hpp"

namespace cellm {

// vector number of token `slot` of row table `table` for head 0, or -1: no position, or its page is missing
__device__ __forceinline__ long long vector_of(const KvGeom& g, int table, int slot)
{
    if (slot < 0) return -1;
    const int b = slot / g.tpb;
    if (b >= g.max_blocks) return -1;
    const uint32_t blk = g.bt[(size_t)table * g.max_blocks + b];
    if (blk >= (uint32_t)g.total_blocks) return -1;
    return ((long long)blk * g.n_layers + g.layer) * g.n_kv * (long long)g.tpb + (slot - b * g.tpb);
}

__device__ __forceinline__ uint16_t bf16_rne(float v)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0x7FC0;
    return (uint16_t)((u + 0x7FFFu + (u >> 16 & 1u)) >> 16);
}

// rint(f32(x / s)) of the N values for which that is an integer from lo to hi; what lies outside may be any value beyond
// the end that it is nearest to.  x times the approximate 1 / s is off by 1.5 2^-23 of it (2.3e-5 at 127, with the quotient's own
// rounding 2.7e-5): where that stays clear of half way between two integers, both have the same; the few lanes that
// come nearer divide.
template <int N>
__device__ __forceinline__ void rounded_quotients(const float (&x)[N], float s, float (&c)[N])
{
    constexpr float kClear = 0.5f - 0x1p-14f;
    const float r = __builtin_amdgcn_rcpf(s);
    float far = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float q = x[i] * r;
        c[i] = rintf(q);
        far = fmaxf(far, fabsf(q - c[i]));
    }
    if (far > kClear) {
#pragma unroll
        for (int i = 0; i < N; ++i) c[i] = rintf(x[i] / s);
    }
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu; }

// The 8-bit codes of a vector of which each of T lanes has x[0..3] and x[4..7] (a word each), and its scale.
template <int T>
__device__ __forceinline__ float quantise8(const float (&x)[8], uint32_t (&w)[2])
{
    uint32_t m = 0;  // |x| in the order of its bits: NaN above infinity above the finite
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, abs_bits(x[i]));
    m = team_max_u32<T>(m);
    float s = __builtin_bit_cast(float, m) / 127.0f;
    if (!(s >= 1.1754943508222875e-38f)) s = 0.0f;
    s = fminf(s, 0x1.0204060000000p+121f);  // 127 of it are finite: the quotient of the largest f32 is rounded up
    const bool finite = m < 0x7F800000u;
    w[0] = w[1] = 0;
    if (finite && s > 0.0f) {
        float c[8];
        rounded_quotients(x, s, c);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i >> 2] |= (uint32_t)((int)fminf(fmaxf(c[i], -127.0f), 127.0f) & 0xFF) << (8 * (i & 3));
    }
    return finite ? s : __builtin_nanf("");
}

// The 4-bit codes (16 bits) of the four dims that each of 8 lanes has of a group, and its scale word.
__device__ __forceinline__ uint32_t quantise4(const float (&in)[4], uint32_t& scale)
{
#pragma clang fp contract(off)
    constexpr float kEnd = 65504.0f;
    float x[4], lo, hi;
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m = max(m, abs_bits(in[i]));
        x[i] = fminf(fmaxf(in[i], -kEnd), kEnd);
    }
    lo = fminf(fminf(x[0], x[1]), fminf(x[2], x[3]));
    hi = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    m = team_max_u32<8>(m);
    lo = -group_max<8>(-lo);
    hi = group_max<8>(hi);
    if (m >= 0x7F800000u) {
        scale = 0x7E007E00u;
        return 0;
    }
    const _Float16 z16 = (_Float16)lo;
    const float z = (float)z16, r = hi - z;
    _Float16 s16 = (_Float16)fmaxf(r / 15.0f, 0.0f);
    uint16_t sb = __builtin_bit_cast(uint16_t, s16);
    // the last code would stand for an infinity: ends near f16's, scale rounded up
    if (15.0f * (float)s16 + z >= 65520.0f) s16 = __builtin_bit_cast(_Float16, --sb);
    scale = (uint32_t)sb | (uint32_t)__builtin_bit_cast(uint16_t, z16) << 16;
    const float s = (float)s16;
    uint32_t w = 0;
    if (s > 0.0f) {
        float d[4], c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = x[i] - z;
        rounded_quotients(d, s, c);
#pragma unroll
        for (int i = 0; i < 4; ++i) w |= (uint32_t)(int)fminf(fmaxf(c[i], 0.0f), 15.0f) << (4 * i);
    }
    return w;
}

// Two f16 values from two 4-bit codes, each half of `codes` below 16: c * s + z in one rounding.
__device__ __forceinline__ h2_t values4(uint32_t codes, h2_t s, h2_t z)
{
    const h2_t c = as_h2(codes | 0x64006400u) - h2_t{(_Float16)1024.0f, (_Float16)1024.0f};  // the f16 1024 + c, exactly
    return __builtin_elementwise_fma(c, s, z);
}
// Eight f16 values from the nibbles 0 .. 7 of w, 11 instructions: pairs (0, 2), (4, 6), (1, 3), (5, 7), with the scales of
// the first and of the second of each pair.  A byte below 16 is the 8-bit float (1 sign, 4 exponent, 3 fraction bits)
// that is 2^-9 of it: numbers below 8 are the subnormal ones, and the first exponent goes on where those end.
__device__ __forceinline__ void values4x8(uint32_t w, h2_t s, h2_t z, uint32_t (&y)[4])
{
    const uint32_t even = w & 0x0F0F0F0Fu, odd = w >> 4 & 0x0F0F0F0Fu;
    const h2_t c[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(even, 512.0f, false), __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(even, 512.0f, true),
                       __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(odd, 512.0f, false), __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(odd, 512.0f, true)};
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = as_u32(__builtin_elementwise_fma(c[i], s, z));
}
// The lower or upper half of a word in both of them: as an operand of packed f16 arithmetic it takes no instruction
__device__ __forceinline__ uint32_t both_low(uint32_t m) { return as_u32(__builtin_shufflevector(as_h2(m), as_h2(m), 0, 0)); }
__device__ __forceinline__ uint32_t both_high(uint32_t m) { return as_u32(__builtin_shufflevector(as_h2(m), as_h2(m), 1, 1)); }

}  // namespace cellm
