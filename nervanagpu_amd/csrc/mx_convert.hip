// Conversions between dense and block-scaled matrices, and the activation
// functions that keep an 8-bit checkpoint of their input.  All of them read each value once
// and write it once.  fp16 of 16384x8192, calls back to back, against 4.9 TB/s of a large copy:
//   backward gelu from the checkpoint   116 us, 675 MB, 5.8 TB/s: memory, and the vector unit close behind
//   forward silu with checkpoint        110 us, 675 MB, 6.1 TB/s: memory (gelu 122, tanh 133: the library's)
//   fp16 to fp4, nearest                 58 us, 340 MB, 5.9 TB/s: memory
//   ... stochastic                       91 us, 340 MB, 3.7 TB/s: the vector unit (two 32-bit
//                                        products of the random word a pair of values, 10 operations a value)
//   fp4 to fp16                          67 us, 340 MB, 5.0 TB/s: memory
//   fp16 to int8 and back                70 (stochastic 80) and 69 us, 407 MB: memory
//   across the rows                      fp4 171 (186) and 109 us, int8 187 (192) and 120 us (pieces of 128 bytes
//                                        of a row, 64 to 128 of a line's codes)
// and at 4096x128 the launch: 2.3 to 3.9 us a kernel.
#include "mx_format.h"

#include <algorithm>
#include <climits>

namespace ng {

typedef unsigned mx_uint2_t __attribute__((ext_vector_type(2)));
typedef unsigned mx_uint4_t __attribute__((ext_vector_type(4)));

// 8 values at p, the first `count` of them inside the row; VEC: p is 16-byte
// aligned and whole groups of 8 may be read
template <typename T, bool VEC>
NG_DEV void load8(const T* p, int count, float (&v)[8])
{
    if (VEC && count >= 8) {
        if constexpr (sizeof(T) == 2) {
            const mx_uint4_t w = *reinterpret_cast<const mx_uint4_t*>(p);
            const T* h = reinterpret_cast<const T*>(&w);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = (float)h[i];
        } else {
            const mx_uint4_t lo = reinterpret_cast<const mx_uint4_t*>(p)[0], hi = reinterpret_cast<const mx_uint4_t*>(p)[1];
#pragma unroll
            for (int i = 0; i < 4; i++) { v[i] = __uint_as_float(lo[i]); v[i + 4] = __uint_as_float(hi[i]); }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = i < count ? (float)p[i] : 0.0f;
    }
}

template <typename T, bool VEC>
NG_DEV void store8(T* p, int count, const float (&v)[8])
{
    if (VEC && count >= 8) {
        if constexpr (sizeof(T) == 2) {
            T h[8];
#pragma unroll
            for (int i = 0; i < 8; i++) h[i] = (T)v[i];
            mx_uint4_t w;
            __builtin_memcpy(&w, h, 16);
            *reinterpret_cast<mx_uint4_t*>(p) = w;
        } else {
            mx_uint4_t lo, hi;
#pragma unroll
            for (int i = 0; i < 4; i++) { lo[i] = __float_as_uint(v[i]); hi[i] = __float_as_uint(v[i + 4]); }
            reinterpret_cast<mx_uint4_t*>(p)[0] = lo;
            reinterpret_cast<mx_uint4_t*>(p)[1] = hi;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < count) p[i] = (T)v[i];
    }
}

NG_DEV unsigned abs_max_bits(const float (&v)[8])
{
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return m;
}

// where unit u (8 values, a quarter of a block) of a line-contiguous matrix lies;
// units are numbered line by line, 4 nb to a line
struct UnitMap {
    FastDiv per_line;   // by 4 nb
    int units_per_line;
    int depth;
    unsigned total;
    NG_DEV void locate(unsigned u, int& line, int& unit) const
    {
        line = (int)per_line.div(u);
        unit = (int)(u - (unsigned)line * (unsigned)units_per_line);
    }
};

// codes of one unit and, from the first of a block's four lanes, its scale
template <int FMT, bool SR>
NG_DEV void write_unit(const float (&v)[8], int line, int unit, const UnitMap& map, unsigned char* codes, unsigned char* scales,
                       long scale_pitch, unsigned seed, unsigned stream)
{
    const unsigned amax = mx_quad_max(abs_max_bits(v));
    const int e = mx_not_finite(amax) ? 0 : mx_exponent<FMT, SR>(amax);
    unsigned w[2];
    mx_encode8<FMT, SR>(v, e, seed, stream, line, map.depth, unit * 8, w);
    if (mx_not_finite(amax)) w[0] = w[1] = 0;
    const size_t u = (size_t)line * map.units_per_line + unit;
    if constexpr (FMT == NG_MX_FP4) reinterpret_cast<unsigned*>(codes)[u] = w[0];
    else                            reinterpret_cast<mx_uint2_t*>(codes)[u] = mx_uint2_t{w[0], w[1]};
    if ((unit & 3) == 0)
        scales[(long)line * scale_pitch + (unit >> 2)] = (unsigned char)(mx_not_finite(amax) ? 255u : mx_scale_byte<FMT>(e));
}

// Blocks along the contiguous axis.  A thread takes 8 values (one 16-byte load in
// fp16), four lanes a block: loads and stores of a wavefront are contiguous and the
// block's maximum is two lane permutes away.
template <typename T, int FMT, bool SR, bool VEC>
__global__ __launch_bounds__(256)
void mx_quantize_along_kernel(const T* __restrict__ A, long lda, UnitMap map, unsigned char* __restrict__ codes,
                              unsigned char* __restrict__ scales, long scale_pitch, unsigned seed, unsigned stream)
{
    const unsigned u = blockIdx.x * 256u + threadIdx.x;
    if (u >= map.total) return;     // whole quads leave: the total is a multiple of 4
    int line, unit;
    map.locate(u, line, unit);
    float v[8];
    load8<T, VEC>(A + (long)line * lda + (long)unit * 8, map.depth - unit * 8, v);
    write_unit<FMT, SR>(v, line, unit, map, codes, scales, scale_pitch, seed, stream);
}

// Blocks across the contiguous axis: element (line, i) at A[i * lda + line].  A
// wavefront takes 64 neighbouring lines and one block of 32 rows, a line per lane, so
// each row is one coalesced load, the maximum of a block needs no exchange and the
// codes of a block are one lane's 16 (32) bytes.  The four wavefronts of a workgroup take four
// neighbouring blocks and put the codes together in LDS, for stores of 64 (128)
// contiguous bytes per line.
template <typename T, int FMT, bool SR>
__global__ __launch_bounds__(256)
void mx_quantize_across_kernel(const T* __restrict__ A, long lda, int lines, int depth, unsigned char* __restrict__ codes,
                               unsigned char* __restrict__ scales, long code_pitch, long scale_pitch, unsigned seed,
                               unsigned stream)
{
    constexpr int CB = FMT == NG_MX_FP4 ? 16 : 32;    // code bytes of a block
    constexpr int PITCH = 4 * CB + 16;                // of a line in LDS
    __shared__ __attribute__((aligned(16))) unsigned char tile[64 * PITCH];
    __shared__ unsigned char tile_scales[64 * 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int line0 = (int)blockIdx.x * 64, line = line0 + lane;
    const int block0 = (int)blockIdx.y * 4, block = block0 + wave;
    const int nb = (depth + MX_BLOCK - 1) / MX_BLOCK;
    const int i0 = block * MX_BLOCK;
    float v[4][8];
    const T* p = A + (long)i0 * lda + line;
#pragma unroll
    for (int i = 0; i < 32; i++) v[i / 8][i % 8] = (line < lines && i0 + i < depth) ? (float)p[(long)i * lda] : 0.0f;
    unsigned amax = 0;
#pragma unroll
    for (int q = 0; q < 4; q++) amax = max(amax, abs_max_bits(v[q]));
    const bool bad = mx_not_finite(amax);
    const int e = bad ? 0 : mx_exponent<FMT, SR>(amax);
    unsigned char* mine = tile + lane * PITCH + wave * CB;
#pragma unroll
    for (int q = 0; q < 4; q++) {
        unsigned w[2];
        mx_encode8<FMT, SR>(v[q], e, seed, stream, line, depth, i0 + q * 8, w);
        if (bad) w[0] = w[1] = 0;
        if constexpr (FMT == NG_MX_FP4) reinterpret_cast<unsigned*>(mine)[q] = w[0];
        else                            reinterpret_cast<mx_uint2_t*>(mine)[q] = mx_uint2_t{w[0], w[1]};
    }
    tile_scales[lane * 4 + wave] = (unsigned char)(block >= nb ? 0u : bad ? 255u : mx_scale_byte<FMT>(e));
    __syncthreads();
    constexpr int CHUNKS = 4 * CB / 16;               // 16-byte pieces of a line in this tile
#pragma unroll
    for (int c = 0; c < 64 * CHUNKS / 256; c++) {
        const int id = tid + c * 256, l = id / CHUNKS, piece = id % CHUNKS;
        if (line0 + l < lines && block0 + piece * 16 / CB < nb)
            *reinterpret_cast<mx_uint4_t*>(codes + (long)(line0 + l) * code_pitch + (long)block0 * CB + piece * 16) =
                *reinterpret_cast<const mx_uint4_t*>(tile + l * PITCH + piece * 16);
    }
    // four scale bytes at once: lines are padded to a multiple of 8, so they are there
    if (tid < 64 && line < lines)
        *reinterpret_cast<unsigned*>(scales + (long)line * scale_pitch + block0) = *reinterpret_cast<const unsigned*>(tile_scales + lane * 4);
}

// The same for matrices of few blocks, where that kernel leaves most of the chip idle: a
// wavefront takes 16 lines, four lanes a block of 8 rows each, whose maxima meet in two
// exchanges (4096 rows x 128 lines: 64 workgroups and 6.3 us there, 256 here)
template <typename T, int FMT, bool SR>
__global__ __launch_bounds__(256)
void mx_quantize_across_small_kernel(const T* __restrict__ A, long lda, int lines, int depth, unsigned char* __restrict__ codes,
                                     unsigned char* __restrict__ scales, long code_pitch, long scale_pitch, unsigned seed,
                                     unsigned stream)
{
    constexpr int CB = FMT == NG_MX_FP4 ? 16 : 32;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int line = ((int)blockIdx.x * 4 + wave) * 16 + (lane & 15), quarter = lane >> 4;
    const int block = (int)blockIdx.y, i0 = block * MX_BLOCK + quarter * 8;
    float v[8];
    const T* p = A + (long)i0 * lda + line;
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = (line < lines && i0 + i < depth) ? (float)p[(long)i * lda] : 0.0f;
    unsigned amax = abs_max_bits(v);
    amax = max(amax, (unsigned)__shfl_xor((int)amax, 16, 64));
    amax = max(amax, (unsigned)__shfl_xor((int)amax, 32, 64));
    const bool bad = mx_not_finite(amax);
    const int e = bad ? 0 : mx_exponent<FMT, SR>(amax);
    unsigned w[2];
    mx_encode8<FMT, SR>(v, e, seed, stream, line, depth, i0, w);
    if (bad) w[0] = w[1] = 0;
    if (line >= lines) return;
    unsigned char* out = codes + (long)line * code_pitch + (long)block * CB + quarter * (CB / 4);
    if constexpr (FMT == NG_MX_FP4) *reinterpret_cast<unsigned*>(out) = w[0];
    else                            *reinterpret_cast<mx_uint2_t*>(out) = mx_uint2_t{w[0], w[1]};
    if (quarter == 0) scales[(long)line * scale_pitch + block] = (unsigned char)(bad ? 255u : mx_scale_byte<FMT>(e));
}

template <int FMT>
NG_DEV void read_unit(const unsigned char* codes, const unsigned char* scales, long scale_pitch, int line, int unit,
                      int units_per_line, float (&v)[8])
{
    const size_t u = (size_t)line * units_per_line + unit;
    unsigned w[2];
    if constexpr (FMT == NG_MX_FP4) {
        w[0] = reinterpret_cast<const unsigned*>(codes)[u];
        w[1] = 0;
    } else {
        const mx_uint2_t both = reinterpret_cast<const mx_uint2_t*>(codes)[u];
        w[0] = both[0];
        w[1] = both[1];
    }
    mx_decode8<FMT>(w, scales[(long)line * scale_pitch + (unit >> 2)], v);
}

template <typename T, int FMT, bool VEC>
__global__ __launch_bounds__(256)
void mx_dequantize_along_kernel(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales,
                                long scale_pitch, UnitMap map, T* __restrict__ out, long ldo)
{
    const unsigned u = blockIdx.x * 256u + threadIdx.x;
    if (u >= map.total) return;
    int line, unit;
    map.locate(u, line, unit);
    const int count = map.depth - unit * 8;
    if (count <= 0) return;
    float v[8];
    read_unit<FMT>(codes, scales, scale_pitch, line, unit, map.units_per_line, v);
    store8<T, VEC>(out + (long)line * ldo + (long)unit * 8, count, v);
}

// element (line, i) to out[i * ldo + line]: 64 lines x 64 values turned in LDS
template <typename T, int FMT>
__global__ __launch_bounds__(256)
void mx_dequantize_across_kernel(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales,
                                 long scale_pitch, int lines, int depth, int units_per_line, T* __restrict__ out, long ldo)
{
    __shared__ float tile[64][65];
    const int tid = threadIdx.x;
    const int line0 = (int)blockIdx.x * 64, i0 = (int)blockIdx.y * 64;
#pragma unroll
    for (int c = 0; c < 2; c++) {
        const int id = tid + c * 256, l = id >> 3, unit = (i0 >> 3) + (id & 7);
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (line0 + l < lines && unit < units_per_line)
            read_unit<FMT>(codes, scales, scale_pitch, line0 + l, unit, units_per_line, v);
#pragma unroll
        for (int i = 0; i < 8; i++) tile[(id & 7) * 8 + i][l] = v[i];
    }
    __syncthreads();
    const int l = tid & 63;
    if (line0 + l < lines)
#pragma unroll 4
        for (int i = tid >> 6; i < 64; i += 4)
            if (i0 + i < depth) out[(long)(i0 + i) * ldo + line0 + l] = (T)tile[i][l];
}

// ---- activation functions ----------------------------------------------------------

// For fp16 all but the value of tanh are evaluated from the hardware's exponential and reciprocal
// (one unit in the last place each), the normal distribution from a polynomial: over all fp16
// arguments the values are within 0.006 units of fp16 before they are rounded to it.  The
// library's erfc alone kept the kernel from the memory's rate (backward gelu of 134M values: 275 us
// with it).  fp32 takes the library's functions.
//
// 1 / (1 + e^-z); where e^-z is infinite, below -88, the value is zero in fp16.  fp32 takes
// e^z / (1 + e^z) on the left, whose tail goes on to -103.
template <bool FAST> NG_DEV float act_logistic(float z)
{
    if (FAST) return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f));
    const float t = expf(-__builtin_fabsf(z)), r = 1.0f / (1.0f + t);
    return z < 0.0f ? t * r : r;
}
// logistic(z) logistic(-z) as t / (1 + t)^2 with t = e^-|z|: one less the other factor would
// keep none of its digits where the function saturates
template <bool FAST> NG_DEV float act_logistic_slope(float z)
{
    const float x = __builtin_fabsf(z);
    const float t = FAST ? __builtin_amdgcn_exp2f(x * -1.44269504088896341f) : expf(-x);
    const float r = FAST ? __builtin_amdgcn_rcpf(1.0f + t) : 1.0f / (1.0f + t);
    return t * r * r;
}
// e^(-z^2 / 2)
template <bool FAST> NG_DEV float act_bell(float z)
{
    if (FAST) return __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
    return expf(-0.5f * z * z);
}
// P(X > x) / e^(-x^2 / 2) - c x of a standard normal X, x >= 0.  The quotient (Mills ratio over
// sqrt(2 pi)) is t P(t), t = 1 / (1 + 0.3 x), so that the left tail of gelu has the bell's digits
// however small it is.  P is a fit made for this file that minimises the largest relative error over
// 0 <= x <= 8, counted 16-fold around x = 0.75 where the slope crosses zero and half as much again below
// 0.3: 2.4e-6, 1.5e-7 and 1.6e-6.  Behind 8, where an fp16 result is zero, it stays bounded.
NG_DEV float act_tail(float x, float c)
{
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3f, x, 1.0f));
    float p = __builtin_fmaf(-0.0821394026f, t, 0.231396079f);
    p = __builtin_fmaf(p, t, -0.0348565318f);
    p = __builtin_fmaf(p, t, 0.154140592f);
    p = __builtin_fmaf(p, t, 0.111123458f);
    p = __builtin_fmaf(p, t, 0.12033502f);
    return c == 0.0f ? p * t : __builtin_fmaf(p, t, -c * x);
}
// z P(X < z); P is 0.5 erfc(-z / sqrt 2) in fp32
template <bool FAST> NG_DEV float act_gelu(float z)
{
    if (FAST) {
        const float tail = act_bell<true>(z) * act_tail(__builtin_fabsf(z), 0.0f);
        return z * (z > 0.0f ? 1.0f - tail : tail);
    }
    return z * (0.5f * erfcf(z * -0.70710678118654752f));
}
// P(X < z) + z density(z): the tail of |z| less |z| times the density there, or 1 less that
template <bool FAST> NG_DEV float act_gelu_slope(float z)
{
    constexpr float C = 0.39894228040143268f;      // 1 / sqrt(2 pi)
    const float bell = act_bell<FAST>(z);
    if (FAST) {
        const float left = bell * act_tail(__builtin_fabsf(z), C);
        return z > 0.0f ? 1.0f - left : left;
    }
    return 0.5f * erfcf(z * -0.70710678118654752f) + z * (C * bell);
}

template <int ACT, bool FAST>
NG_DEV float act_value(float z)
{
    if constexpr (ACT == NG_ACT_RELU) return z <= 0.0f ? 0.0f : z;     // NaN stays NaN
    if constexpr (ACT == NG_ACT_SIG)  return act_logistic<FAST>(z);
    if constexpr (ACT == NG_ACT_TANH) return tanhf(z);
    if constexpr (ACT == NG_ACT_SILU) return z * act_logistic<FAST>(z);
    return act_gelu<FAST>(z);
}

template <int ACT, bool FAST>
NG_DEV float act_slope(float z)
{
    // a block that is marked NaN has no derivative, under relu as under the others
    if constexpr (ACT == NG_ACT_RELU) return z > 0.0f ? 1.0f : z <= 0.0f ? 0.0f : z;
    if constexpr (ACT == NG_ACT_SIG) return act_logistic_slope<FAST>(z);
    if constexpr (ACT == NG_ACT_TANH) return 4.0f * act_logistic_slope<FAST>(z + z);      // tanh(z) = 2 logistic(2z) - 1
    if constexpr (ACT == NG_ACT_SILU) { const float s = act_logistic<FAST>(z); return s * (1.0f + z * (1.0f - s)); }
    return act_gelu_slope<FAST>(z);
}

template <typename T, int ACT, bool SAVE, bool VEC>
__global__ __launch_bounds__(256)
void act_fprop_kernel(const T* I, long ldi, T* O, long ldo, UnitMap map,
                      unsigned char* __restrict__ codes, unsigned char* __restrict__ scales, long scale_pitch)
{
    const unsigned u = blockIdx.x * 256u + threadIdx.x;
    if (u >= map.total) return;
    int line, unit;
    map.locate(u, line, unit);
    const int count = map.depth - unit * 8;
    float v[8], y[8];
    load8<T, VEC>(I + (long)line * ldi + (long)unit * 8, count, v);
    if constexpr (SAVE) write_unit<NG_MX_INT8, false>(v, line, unit, map, codes, scales, scale_pitch, 0, 0);
#pragma unroll
    for (int i = 0; i < 8; i++) y[i] = act_value<ACT, sizeof(T) == 2>(v[i]);
    store8<T, VEC>(O + (long)line * ldo + (long)unit * 8, count, y);
}

template <typename T, int ACT, bool VEC>
__global__ __launch_bounds__(256)
void act_bprop_kernel(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales, long scale_pitch,
                      UnitMap map, const T* E, long lde, T* G, long ldg)
{
    const unsigned u = blockIdx.x * 256u + threadIdx.x;
    if (u >= map.total) return;
    int line, unit;
    map.locate(u, line, unit);
    const int count = map.depth - unit * 8;
    if (count <= 0) return;
    float z[8], g[8];
    read_unit<NG_MX_INT8>(codes, scales, scale_pitch, line, unit, map.units_per_line, z);
    load8<T, VEC>(E + (long)line * lde + (long)unit * 8, count, g);
#pragma unroll
    for (int i = 0; i < 8; i++) g[i] *= act_slope<ACT, sizeof(T) == 2>(z[i]);
    store8<T, VEC>(G + (long)line * ldg + (long)unit * 8, count, g);
}

// ---- host side -----------------------------------------------------------------------

static bool unit_map(int lines, int depth, UnitMap& map)
{
    const long per = (long)mx_blocks(depth) * 4;
    if (per * lines >= (1L << 31)) return false;
    map.units_per_line = (int)per;
    map.per_line = FastDiv::make((unsigned)per);
    map.depth = depth;
    map.total = (unsigned)(per * lines);
    return true;
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
static bool row_vec(const void* p, long ld, size_t elem) { return aligned16(p) && (ld * (long)elem) % 16 == 0; }

// the checks that every conversion shares; 1: nothing to do
static int check_matrix(const char* what, int dtype, const void* p, long ld, int along, int lines, int depth)
{
    if (dtype != NG_F16 && dtype != NG_F32) return fail(-80, "%s: the dense matrix must be fp16 or fp32", what);
    if (lines < 0 || depth < 0) return fail(-81, "%s: negative extent", what);
    // grids and blocks are counted in int, rounded up
    if (lines > INT_MAX - 256 || depth > INT_MAX - 256) return fail(-87, "%s: extent of 2^31 - 256 or more", what);
    if (!lines || !depth) return 1;
    if (!p) return fail(-82, "%s: null matrix", what);
    if (ld < (along ? depth : lines) && (along ? lines : depth) > 1) return fail(-83, "%s: rows overlap (pitch %ld)", what, ld);
    return 0;
}

static int check_codes(const char* what, int format, const void* codes, const void* scales)
{
    if (format != NG_MX_FP4 && format != NG_MX_INT8) return fail(-84, "%s: unknown block-scaled format %d", what, format);
    if (!codes || !scales) return fail(-85, "%s: null codes or scales", what);
    if (!aligned16(codes) || !aligned16(scales)) return fail(-86, "%s: codes and scales must be 16-byte aligned", what);
    return 0;
}

static int too_large(const char* what) { return fail(-87, "%s: matrix of 2^34 or more values", what); }

struct QuantArgs {
    const void* A; long lda; int along, lines, depth;
    void *codes, *scales;
    unsigned seed, rng_stream;
    hipStream_t stream;
};

template <typename T, int FMT, bool SR>
static int quantize(const QuantArgs& q)
{
    const long cp = mx_code_pitch(FMT, q.depth), sp = mx_scale_pitch(q.depth);
    if (q.along) {
        UnitMap map;
        if (!unit_map(q.lines, q.depth, map)) return too_large("ng_mx_quantize");
        const dim3 grid((map.total + 255u) / 256u);
        if (row_vec(q.A, q.lda, sizeof(T)))
            hipLaunchKernelGGL((mx_quantize_along_kernel<T, FMT, SR, true>), grid, dim3(256), 0, q.stream, (const T*)q.A, q.lda,
                               map, (unsigned char*)q.codes, (unsigned char*)q.scales, sp, q.seed, q.rng_stream);
        else
            hipLaunchKernelGGL((mx_quantize_along_kernel<T, FMT, SR, false>), grid, dim3(256), 0, q.stream, (const T*)q.A, q.lda,
                               map, (unsigned char*)q.codes, (unsigned char*)q.scales, sp, q.seed, q.rng_stream);
    } else {
        const int groups = (mx_blocks(q.depth) + 3) / 4;
        if (groups > 65535) return fail(-88, "ng_mx_quantize: depth beyond 2^23 across the rows");
        const dim3 grid((unsigned)((q.lines + 63) / 64), (unsigned)groups);
        if ((long)grid.x * grid.y < 2l * device_cu_count() && mx_blocks(q.depth) <= 65535)
            hipLaunchKernelGGL((mx_quantize_across_small_kernel<T, FMT, SR>), dim3(grid.x, (unsigned)mx_blocks(q.depth)), dim3(256), 0,
                               q.stream, (const T*)q.A, q.lda, q.lines, q.depth, (unsigned char*)q.codes, (unsigned char*)q.scales, cp, sp,
                               q.seed, q.rng_stream);
        else
            hipLaunchKernelGGL((mx_quantize_across_kernel<T, FMT, SR>), grid, dim3(256), 0, q.stream, (const T*)q.A, q.lda, q.lines,
                               q.depth, (unsigned char*)q.codes, (unsigned char*)q.scales, cp, sp, q.seed, q.rng_stream);
    }
    NG_CHECK_LAUNCH("mx quantize");
    return 0;
}

template <typename T, int FMT>
static int dequantize(const void* codes, const void* scales, int lines, int depth, void* out, long ldo, int along,
                      hipStream_t stream)
{
    const long sp = mx_scale_pitch(depth);
    const unsigned char *c = (const unsigned char*)codes, *s = (const unsigned char*)scales;
    if (along) {
        UnitMap map;
        if (!unit_map(lines, depth, map)) return too_large("ng_mx_dequantize");
        const dim3 grid((map.total + 255u) / 256u);
        if (row_vec(out, ldo, sizeof(T)))
            hipLaunchKernelGGL((mx_dequantize_along_kernel<T, FMT, true>), grid, dim3(256), 0, stream, c, s, sp, map, (T*)out, ldo);
        else
            hipLaunchKernelGGL((mx_dequantize_along_kernel<T, FMT, false>), grid, dim3(256), 0, stream, c, s, sp, map, (T*)out, ldo);
    } else {
        const int groups = (depth + 63) / 64;
        if (groups > 65535) return fail(-88, "ng_mx_dequantize: depth beyond 2^22 across the rows");
        hipLaunchKernelGGL((mx_dequantize_across_kernel<T, FMT>), dim3((unsigned)((lines + 63) / 64), (unsigned)groups), dim3(256),
                           0, stream, c, s, sp, lines, depth, mx_blocks(depth) * 4, (T*)out, ldo);
    }
    NG_CHECK_LAUNCH("mx dequantize");
    return 0;
}

struct ActArgs {
    int rows, cols;
    const void* in; long ld_in;      // I, or E
    void* out; long ld_out;          // O, or gradI
    void *codes, *scales;
    hipStream_t stream;
};

template <typename T, int ACT>
static int act_fprop(const ActArgs& a)
{
    UnitMap map;
    if (!unit_map(a.rows, a.cols, map)) return too_large("ng_act_fprop");
    const long sp = mx_scale_pitch(a.cols);
    const dim3 grid((map.total + 255u) / 256u);
    const bool vec = row_vec(a.in, a.ld_in, sizeof(T)) && row_vec(a.out, a.ld_out, sizeof(T));
    unsigned char *c = (unsigned char*)a.codes, *s = (unsigned char*)a.scales;
#define NG_ACT_LAUNCH(SAVE, VEC)                                                                                            \
    hipLaunchKernelGGL((act_fprop_kernel<T, ACT, SAVE, VEC>), grid, dim3(256), 0, a.stream, (const T*)a.in, a.ld_in, (T*)a.out, \
                       a.ld_out, map, c, s, sp)
    if (c) { if (vec) NG_ACT_LAUNCH(true, true); else NG_ACT_LAUNCH(true, false); }
    else   { if (vec) NG_ACT_LAUNCH(false, true); else NG_ACT_LAUNCH(false, false); }
#undef NG_ACT_LAUNCH
    NG_CHECK_LAUNCH("activation");
    return 0;
}

template <typename T, int ACT>
static int act_bprop(const ActArgs& a)
{
    UnitMap map;
    if (!unit_map(a.rows, a.cols, map)) return too_large("ng_act_bprop");
    const long sp = mx_scale_pitch(a.cols);
    const dim3 grid((map.total + 255u) / 256u);
    const unsigned char *c = (const unsigned char*)a.codes, *s = (const unsigned char*)a.scales;
    if (row_vec(a.in, a.ld_in, sizeof(T)) && row_vec(a.out, a.ld_out, sizeof(T)))
        hipLaunchKernelGGL((act_bprop_kernel<T, ACT, true>), grid, dim3(256), 0, a.stream, c, s, sp, map, (const T*)a.in, a.ld_in,
                           (T*)a.out, a.ld_out);
    else
        hipLaunchKernelGGL((act_bprop_kernel<T, ACT, false>), grid, dim3(256), 0, a.stream, c, s, sp, map, (const T*)a.in, a.ld_in,
                           (T*)a.out, a.ld_out);
    NG_CHECK_LAUNCH("activation gradient");
    return 0;
}

template <typename T>
static int act_dispatch(int act, bool back, const ActArgs& a)
{
    switch (act) {
    case NG_ACT_RELU: return back ? act_bprop<T, NG_ACT_RELU>(a) : act_fprop<T, NG_ACT_RELU>(a);
    case NG_ACT_SIG:  return back ? act_bprop<T, NG_ACT_SIG>(a)  : act_fprop<T, NG_ACT_SIG>(a);
    case NG_ACT_TANH: return back ? act_bprop<T, NG_ACT_TANH>(a) : act_fprop<T, NG_ACT_TANH>(a);
    case NG_ACT_SILU: return back ? act_bprop<T, NG_ACT_SILU>(a) : act_fprop<T, NG_ACT_SILU>(a);
    case NG_ACT_GELU: return back ? act_bprop<T, NG_ACT_GELU>(a) : act_fprop<T, NG_ACT_GELU>(a);
    default: return fail(-89, "unknown activation function %d", act);
    }
}

}  // namespace ng

using namespace ng;

extern "C" {

int ng_mx_quantize(int format, int dtype, const void* A, long lda, int along, int lines, int depth,
                   void* codes, void* scales, unsigned flags, unsigned seed, unsigned rng_stream, void* stream)
{
    int rc = check_matrix("ng_mx_quantize", dtype, A, lda, along, lines, depth);
    if (rc) return rc < 0 ? rc : 0;
    rc = check_codes("ng_mx_quantize", format, codes, scales);
    if (rc) return rc;
    const QuantArgs q{A, lda, along, lines, depth, codes, scales, seed, rng_stream, (hipStream_t)stream};
    const bool sr = (flags & NG_FLAG_SR) != 0;
    if (dtype == NG_F16) {
        if (format == NG_MX_FP4) return sr ? quantize<_Float16, NG_MX_FP4, true>(q) : quantize<_Float16, NG_MX_FP4, false>(q);
        return sr ? quantize<_Float16, NG_MX_INT8, true>(q) : quantize<_Float16, NG_MX_INT8, false>(q);
    }
    if (format == NG_MX_FP4) return sr ? quantize<float, NG_MX_FP4, true>(q) : quantize<float, NG_MX_FP4, false>(q);
    return sr ? quantize<float, NG_MX_INT8, true>(q) : quantize<float, NG_MX_INT8, false>(q);
}

int ng_mx_dequantize(int format, const void* codes, const void* scales, int lines, int depth,
                     int dtype, void* out, long ldo, int along, void* stream)
{
    int rc = check_matrix("ng_mx_dequantize", dtype, out, ldo, along, lines, depth);
    if (rc) return rc < 0 ? rc : 0;
    rc = check_codes("ng_mx_dequantize", format, codes, scales);
    if (rc) return rc;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == NG_F16)
        return format == NG_MX_FP4 ? dequantize<_Float16, NG_MX_FP4>(codes, scales, lines, depth, out, ldo, along, st)
                                   : dequantize<_Float16, NG_MX_INT8>(codes, scales, lines, depth, out, ldo, along, st);
    return format == NG_MX_FP4 ? dequantize<float, NG_MX_FP4>(codes, scales, lines, depth, out, ldo, along, st)
                               : dequantize<float, NG_MX_INT8>(codes, scales, lines, depth, out, ldo, along, st);
}

int ng_act_fprop(int act, int dtype, int rows, int cols, const void* I, long ldi, void* O, long ldo,
                 void* codes, void* scales, void* stream)
{
    int rc = check_matrix("ng_act_fprop", dtype, I, ldi, 1, rows, cols);
    if (rc) return rc < 0 ? rc : 0;
    rc = check_matrix("ng_act_fprop", dtype, O, ldo, 1, rows, cols);
    if (rc) return rc;
    if (codes || scales) {
        rc = check_codes("ng_act_fprop", NG_MX_INT8, codes, scales);
        if (rc) return rc;
    }
    const ActArgs a{rows, cols, I, ldi, O, ldo, codes, scales, (hipStream_t)stream};
    return dtype == NG_F16 ? act_dispatch<_Float16>(act, false, a) : act_dispatch<float>(act, false, a);
}

int ng_act_bprop(int act, int dtype, int rows, int cols, const void* codes, const void* scales,
                 const void* E, long lde, void* gradI, long ldg, void* stream)
{
    int rc = check_matrix("ng_act_bprop", dtype, E, lde, 1, rows, cols);
    if (rc) return rc < 0 ? rc : 0;
    rc = check_matrix("ng_act_bprop", dtype, gradI, ldg, 1, rows, cols);
    if (rc) return rc;
    rc = check_codes("ng_act_bprop", NG_MX_INT8, codes, scales);
    if (rc) return rc;
    const ActArgs a{rows, cols, E, lde, gradI, ldg, const_cast<void*>(codes), const_cast<void*>(scales), (hipStream_t)stream};
    return dtype == NG_F16 ? act_dispatch<_Float16>(act, true, a) : act_dispatch<float>(act, true, a);
}

}  // extern "C"
