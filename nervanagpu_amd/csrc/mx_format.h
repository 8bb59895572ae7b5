// Block-scaled ("MX") matrices: blocks of 32 consecutive values along one axis,
// a code per value and one power of two per block (the OCP microscaling formats
// MXFP4 and MXINT8).
//
//   value = element(code) * 2^(scale - 127)      scale byte 255: the block is NaN
//   fp4   element(code) = +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}, sign in bit 3 (E2M1)
//   int8  element(code) = code / 64, codes -127 .. 127 are written
//
// A line is one run of the blocked axis (`depth` values, nb = ceil(depth / 32)
// blocks).  Lines follow each other:
//   codes   16 (fp4) or 32 (int8) bytes a block, no padding between lines beyond
//           the last block's; element 2i of a line is the low half of byte i
//   scales  one byte a block, lines padded to a multiple of 8 bytes
// What stands in the padding bytes of the scales never reaches a result.
#pragma once

#include "ng_internal.h"
#include "ng_device_common.h"

namespace ng {

constexpr int MX_BLOCK = 32;

inline int mx_blocks(int depth) { return (depth + MX_BLOCK - 1) / MX_BLOCK; }
inline long mx_code_pitch(int fmt, int depth) { return (long)mx_blocks(depth) * (fmt == NG_MX_FP4 ? 16 : 32); }
inline long mx_scale_pitch(int depth) { return (long)((mx_blocks(depth) + 7) / 8) * 8; }

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float float2_t __attribute__((ext_vector_type(2)));

// maximum over the four lanes of a quad (two lane permutes on the vector unit)
NG_DEV unsigned mx_quad_max(unsigned v)
{
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));   // lanes 1 0 3 2
    return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));   // lanes 2 3 0 1
}

// Exponent e of a block (value = grid(code) * 2^e) from the largest magnitude's
// fp32 bit pattern.  Nearest: the largest element keeps its binade (4..6 in fp4,
// 64..127 in int8) and what rounds beyond the grid saturates, as the formats'
// conversion rule has it.  Stochastic fp4: one more where the largest element lies
// above 6, so that nothing saturates and every element is right on average (two blocks in
// five would saturate, by up to a quarter of the value).  Stochastic int8 saturates above
// 127 like the nearest: 1 % of all blocks, by less than a unit; one power more there would
// cost their other 31 elements a bit.
template <int FMT, bool SR>
NG_DEV int mx_exponent(unsigned amax_bits)
{
    const int top = (int)(amax_bits >> 23) - 127 - (FMT == NG_MX_FP4 ? 2 : 6);
    const int bump = (FMT == NG_MX_FP4 && SR && (amax_bits & 0x7FFFFFu) > 0x400000u) ? 1 : 0;
    return (top < -126) ? -126 : top + bump;
}

NG_DEV bool mx_not_finite(unsigned amax_bits) { return amax_bits >= 0x7F800000u; }
template <int FMT> NG_DEV unsigned mx_scale_byte(int e) { return (unsigned)(e + 127 + (FMT == NG_MX_FP4 ? 0 : 6)); }
// 2^e for -126 <= e <= 127
NG_DEV float mx_pow2(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

// fp32 value of a scale byte (NaN for 255)
NG_DEV float mx_scale_value(unsigned byte)
{
    const unsigned bits = byte ? byte << 23 : 0x00400000u;
    return __uint_as_float(byte == 255u ? 0x7FC00000u : bits);
}

// 16 random bits for element idx of a stream: neighbours 2i and 2i+1 take the
// high and the low half of word i (as the fp16 stores' stochastic rounding does)
NG_DEV unsigned mx_random16(unsigned word, bool odd) { return odd ? (word & 0xFFFFu) : (word >> 16); }

// |x| * 2^-e (at most 6) -> code by adding a uniform fraction of the local unit and
// truncating: T = floor(|x| 2^-e 2^15); the unit is 2^14 below 2, 2^15 below 4 and 2^16
// above, the random number the top 14, 15 or 16 of the 16 bits.  In the fp32 pattern of T
// all three units are the same place, bit 22, so one addition serves them: what the
// pattern of T leaves free below its last bit takes the random bits that do not count.
// Below 1, where the unit stays 2^14, T + 2^15 takes its place: [1, 2) two codes up.
NG_DEV unsigned mx_fp4_stochastic(float a, unsigned r16)
{
    const unsigned T = (unsigned)(a * 32768.0f);
    const bool low = T < 32768u;
    const unsigned bits = __float_as_uint((float)(low ? T + 32768u : T));
    return ((bits + (r16 << 6)) >> 22) - (low ? 284u : 282u);
}

NG_DEV unsigned mx_int8_magnitude_stochastic(float a, unsigned r16)
{
    return min(((unsigned)(a * 65536.0f) + r16) >> 16, 127u);
}

// codes of 8 neighbouring values of one block -> 4 (fp4) or 8 (int8) bytes.
// idx0: stream index of the first value (SR only); EVEN: it is even
template <int FMT, bool SR, bool EVEN>
NG_DEV void mx_encode8_words(const float (&v)[8], int e, unsigned seed, unsigned stream, unsigned long long idx0, unsigned (&out)[2])
{
    unsigned words[5];
    bool odd = false;
    if constexpr (SR) {
        odd = !EVEN && (idx0 & 1) != 0;
        const unsigned w0 = (unsigned)(idx0 >> 1);
#pragma unroll
        for (int i = 0; i < 4; i++) words[i] = ng_rand32(seed, stream, w0 + i);
        words[4] = odd ? ng_rand32(seed, stream, w0 + 4) : 0u;
    }
    auto random = [&](int i) {
        return odd ? mx_random16(words[(i + 1) / 2], (i & 1) == 0) : mx_random16(words[i / 2], (i & 1) != 0);
    };
    out[0] = out[1] = 0;
    if constexpr (FMT == NG_MX_FP4 && !SR) {
        // the hardware's conversion divides by the scale, rounds to nearest even and saturates at 6
        const float s = mx_pow2(e);
        unsigned w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], s, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], s, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], s, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], s, 3);
        out[0] = w;
    } else if constexpr (FMT == NG_MX_FP4) {
        const float inv = mx_pow2(-e);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const unsigned code = mx_fp4_stochastic(__builtin_fabsf(v[i]) * inv, random(i));
            out[0] |= (code | ((__float_as_uint(v[i]) >> 28) & 8u)) << (4 * i);
        }
    } else {
        const float inv = mx_pow2(-e);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            int q;
            if constexpr (SR) {
                const int mag = (int)mx_int8_magnitude_stochastic(__builtin_fabsf(v[i]) * inv, random(i));
                q = v[i] < 0.0f ? -mag : mag;
            } else {
                q = (int)rintf(fminf(fmaxf(v[i] * inv, -127.0f), 127.0f));
            }
            out[i / 4] |= ((unsigned)q & 255u) << (8 * (i & 3));
        }
    }
}

// idx0 = line * depth + i with i a multiple of 8: with an even depth it is even for
// every line, the pairs that share a word are fixed and nothing has to be selected
template <int FMT, bool SR>
NG_DEV void mx_encode8(const float (&v)[8], int e, unsigned seed, unsigned stream, int line, int depth, int i, unsigned (&out)[2])
{
    const unsigned long long idx0 = (unsigned long long)(unsigned)line * (unsigned)depth + (unsigned)i;
    if (!SR || (depth & 1) == 0) mx_encode8_words<FMT, SR, true>(v, e, seed, stream, idx0, out);
    else                         mx_encode8_words<FMT, SR, false>(v, e, seed, stream, idx0, out);
}

// 8 neighbouring values (4 or 8 bytes of codes) in fp32
template <int FMT>
NG_DEV void mx_decode8(const unsigned (&in)[2], unsigned scale_byte, float (&v)[8])
{
    const float s = mx_scale_value(scale_byte);
    if constexpr (FMT == NG_MX_FP4) {
        const float2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(in[0], 1.0f, 0);
        const float2_t b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(in[0], 1.0f, 1);
        const float2_t c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(in[0], 1.0f, 2);
        const float2_t d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(in[0], 1.0f, 3);
        const float grid[8] = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = grid[i] * s;
    } else {
        const float unit = s * 0.015625f;      // exact, subnormal units too, and so is a product with a code
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int q = (int)(in[i / 4] << (24 - 8 * (i & 3))) >> 24;
            v[i] = (float)q * unit;
        }
    }
}

}  // namespace ng
