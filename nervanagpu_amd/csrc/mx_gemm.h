// LDS-tiled products of block-scaled operands for gfx950.
//
//   mx44_kernel   fp4 . fp4 on the scaled matrix instruction (v_mfma_scale 32x32x64):
//                 a lane's 32 contraction values are exactly one block, so an operand
//                 register quad is one 16-byte chunk as it lies in memory and the block's
//                 scale byte goes into the instruction.
//   mxmix_kernel  fp4 or int8 . fp16 on v_mfma 32x32x16 f16: codes travel through LDS as
//                 they are and become fp16 in registers, in the shadow of the matrix pipe.
//
// Both operands lie with the contraction contiguous (a line per row of A / column of
// B).  Tiles are staged with loads that write LDS directly; a tile's scales (4 blocks,
// a dword, per line) are staged beside its codes.  The order of fetching is that of
// gemm_core.h: NSTAGE tiles resident or in flight, one barrier per tile, the first
// fragments of the next tile read behind the last products of the current one.
#pragma once

#include "gemm_core.h"
#include "mx_format.h"

namespace ng {

typedef int int8v_t __attribute__((ext_vector_type(8)));
typedef unsigned uint2v_t __attribute__((ext_vector_type(2)));

// one operand: lines of `pitch` bytes of which `chunks` 16-byte chunks exist
struct MxSide {
    const char* data;
    const char* scales;
    long pitch, scale_pitch;
    int lines;
    int chunks;
    int blocks;     // of a line; 0 for a dense operand
};

#ifndef NG_HOST_EMULATION
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 4 bytes per lane from a buffer straight into LDS: lane l writes lds_base + 4 l
// (see buffer_load_chunk_to_lds)
__device__ __forceinline__ void buffer_load_dword_to_lds(BufferRsrc rsrc, char* lds_base, unsigned byte_offset)
{
    const unsigned lds_addr = (unsigned)(unsigned long)(NG_LDS char*)lds_base;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
                 :: "s"(lds_addr), "v"(byte_offset), "s"(rsrc) : "memory", "m0");
}
#pragma clang diagnostic pop
#endif

// ROWS lines of LINE_BYTES each, 16-byte chunks permuted inside a line so that 16
// neighbouring lines read at one chunk index touch all 16 chunk slots of a bank period
template <int ROWS, int LINE_BYTES>
struct MxTile {
    static constexpr int CPR = LINE_BYTES / 16;
    static constexpr int CHUNKS = ROWS * CPR;
    static constexpr int BYTES = ROWS * LINE_BYTES;
    static constexpr int LP = CPR >= 16 ? 1 : 16 / CPR;
    static __device__ __forceinline__ int swizzle(int line) { return (line / LP) % CPR; }
    // LDS chunk position -> line and chunk of the line it holds
    static __device__ __forceinline__ void chunk_pos(int id, int& line, int& c)
    {
        line = id / CPR;
        c = (id % CPR) ^ swizzle(line);
    }
    static __device__ __forceinline__ int offset(int line, int c) { return line * LINE_BYTES + ((c ^ swizzle(line)) * 16); }
};

// Fetches one operand's tiles.  Addresses: a 64-bit base that steps along the
// contraction plus 32-bit offsets inside the rows of the tile.
template <class Tile, int ROWS, int NT, bool SCALES>
struct MxFetch {
    static constexpr int DATA = Tile::CHUNKS / NT;
    static_assert(Tile::CHUNKS % NT == 0, "tile chunks must divide evenly over threads");
    unsigned off[DATA];
    int col[DATA];
    const char* base;
    int left;                // chunks of a line not yet fetched
    __device__ __forceinline__ void init(const MxSide& s, int row0, int kt, int tid)
    {
        base = s.data + (long)row0 * s.pitch + (long)kt * (Tile::CPR * 16);
        left = s.chunks - kt * Tile::CPR;
#pragma unroll
        for (int i = 0; i < DATA; i++) {
            int line;
            Tile::chunk_pos(tid + i * NT, line, col[i]);
            off[i] = row0 + line < s.lines ? (unsigned)line * (unsigned)s.pitch + (unsigned)col[i] * 16u : NG_OOB_OFFSET;
        }
    }
    __device__ __forceinline__ void issue(int i, char* lds, int wave) const
    {
        buffer_load_chunk_to_lds(make_rsrc(base), lds + (i * NT + wave * 64) * 16, col[i] < left ? off[i] : NG_OOB_OFFSET);
    }
    __device__ __forceinline__ void advance()
    {
        base += Tile::CPR * 16;
        left -= Tile::CPR;
    }
};

// fp16 values 8 s .. 8 s + 7 of a lane's 32-value fp4 block
__device__ __forceinline__ half8_t mx_expand_fp4(unsigned w, float scale)
{
    const half2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0);
    const half2_t b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1);
    const half2_t c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2);
    const half2_t d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3);
    return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Scale of an int8 block as fp16 factors.  code * 2^e is formed as
// ((1024 + code + 128) * s1 - 1152 * s1) * s2 with s1 s2 = 2^e: the bytes become
// fp16 1024 + u by placing them under the exponent of 1024, s1 = 2^(-14 .. 5) keeps
// the fused product exact, and s2 rounds once (not at all for codes of fp16 values)
// and overflows to infinity like any fp16 rounding.
struct MxInt8Scale { half2_t s1, off, s2; };
__device__ __forceinline__ MxInt8Scale mx_int8_scale(unsigned byte)
{
    const int e = (int)byte - 127 - 6;
    const int e1 = min(max(e, -14), 5);
    const int e2 = min(max(e - e1, -24), 15);
    float f1 = mx_pow2(e1);
    if (byte == 255u) f1 = __uint_as_float(0x7FC00000u);
    const _Float16 a = (_Float16)f1, o = (_Float16)(f1 * -1152.0f), b = (_Float16)mx_pow2(e2);
    MxInt8Scale r;
    r.s1 = half2_t{a, a};
    r.off = half2_t{o, o};
    r.s2 = half2_t{b, b};
    return r;
}
// four codes -> two fp16 pairs
__device__ __forceinline__ void mx_expand_int8(unsigned w, const MxInt8Scale& s, half2_t& lo, half2_t& hi)
{
    const unsigned u = w ^ 0x80808080u;
    const half2_t p = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u));
    const half2_t q = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u));
    lo = __builtin_elementwise_fma(p, s.s1, s.off) * s.s2;
    hi = __builtin_elementwise_fma(q, s.s1, s.off) * s.s2;
}

// mask of the scale bytes of contraction tile dword `first` (a multiple of 4) that exist
__device__ __forceinline__ unsigned mx_scale_mask(int blocks, int first)
{
    const int valid = blocks - first;
    return valid >= 4 ? 0xFFFFFFFFu : valid <= 0 ? 0u : (1u << (8 * valid)) - 1u;
}

// Scale dwords of a tile: 64 lines per wavefront request, the requests of both
// operands dealt to the wavefronts in turn; every wavefront issues the same number.
template <int ROWS_A, int ROWS_B, int WAVES>
struct MxScaleFetch {
    static constexpr int REQ_A = (ROWS_A + 63) / 64, REQ_B = (ROWS_B + 63) / 64;
    static constexpr int PER = (REQ_A + REQ_B + WAVES - 1) / WAVES;
    static constexpr int BYTES = PER * WAVES * 256;
    static constexpr int B_OFFSET = REQ_A * 256;
    unsigned off[PER];
    bool is_b[PER];
    __device__ __forceinline__ void init(const MxSide& a, const MxSide& b, int m0, int n0, int wave, int lane)
    {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int req = wave + i * WAVES;
            is_b[i] = req >= REQ_A;
            const int row = (is_b[i] ? req - REQ_A : req) * 64 + lane;
            const MxSide& s = is_b[i] ? b : a;
            const int rows = is_b[i] ? ROWS_B : ROWS_A, first = is_b[i] ? n0 : m0;
            off[i] = (row < rows && first + row < s.lines && s.blocks > 0) ? (unsigned)row * (unsigned)s.scale_pitch : NG_OOB_OFFSET;
        }
    }
    // `first`: first block of the dword
    __device__ __forceinline__ void issue(int i, const char* a_base, const char* b_base, int first, char* lds, int wave) const
    {
        buffer_load_dword_to_lds(make_rsrc((is_b[i] ? b_base : a_base) + first), lds + (wave + i * WAVES) * 256, off[i]);
    }
};

// ---- fp4 . fp4 --------------------------------------------------------------------
template <int BM, int BN, int WM, int WN, int NSTAGE, class Epi>
__global__ __launch_bounds__(WM * WN * 64)
void mx44_kernel(MxSide a, MxSide b, Epi epi, CoreShape s)
{
    constexpr int BK = 128, LINE = BK / 2, NT = WM * WN * 64, WAVES = WM * WN;
    constexpr int TM = BM / WM / 32, TN = BN / WN / 32, WTN = BN / WN;
    using TA = MxTile<BM, LINE>;
    using TB = MxTile<BN, LINE>;
    using FA = MxFetch<TA, BM, NT, true>;
    using FB = MxFetch<TB, BN, NT, true>;
    using SF = MxScaleFetch<BM, BN, WAVES>;
    constexpr int STAGE = TA::BYTES + TB::BYTES + SF::BYTES;
    constexpr int SCALES = TA::BYTES + TB::BYTES;
    constexpr int LOADS = FA::DATA + FB::DATA + SF::PER;     // requests of a wavefront per tile
    constexpr int EPITCH = WTN * 4 + 16, EPI_BYTES = 32 * EPITCH;
    constexpr int SMEM = NSTAGE * STAGE > EPI_BYTES * WAVES ? NSTAGE * STAGE : EPI_BYTES * WAVES;
    static_assert(SMEM <= 160 * 1024, "tile stages exceed the LDS of a compute unit");
    static_assert((NSTAGE - 1) * LOADS < 64, "the wait counter holds 6 bits");
    __shared__ __attribute__((aligned(16))) char smem[SMEM];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WM, wn = wave / WM;
    const int half = lane >> 5, row = lane & 31;

    int tm, tn, split;
    if (!block_work(s, tm, tn, split)) return;
    const int m0 = tm * BM, n0 = tn * BN;
    const int per = (s.k_tiles + s.splits - 1) / s.splits;
    const int t_begin = split * per, t_end = min(t_begin + per, s.k_tiles);
    const int ntiles = t_end - t_begin;

    FA fa;
    FB fb;
    SF sf;
    fa.init(a, m0, t_begin, tid);
    fb.init(b, n0, t_begin, tid);
    sf.init(a, b, m0, n0, wave, lane);
    const char* a_scales = a.scales + (long)m0 * a.scale_pitch;
    const char* b_scales = b.scales + (long)n0 * b.scale_pitch;
    int g_block = t_begin * 4;
    auto gissue = [&](int stage_off) {
        char* st = smem + stage_off;
#pragma unroll
        for (int i = 0; i < SF::PER; i++) sf.issue(i, a_scales, b_scales, g_block, st + SCALES, wave);
#pragma unroll
        for (int i = 0; i < FA::DATA; i++) fa.issue(i, st, wave);
#pragma unroll
        for (int i = 0; i < FB::DATA; i++) fb.issue(i, st + TA::BYTES, wave);
        fa.advance();
        fb.advance();
        g_block += 4;
    };

    float16_t acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int v = 0; v < 16; v++) acc[i][j][v] = 0.0f;

    // lane-constant addresses: block 2 st + half of the lane's line; the swizzle only
    // depends on the line inside a block of 32
    int a_off[TM], b_off[TN];
#pragma unroll
    for (int i = 0; i < TM; i++) a_off[i] = TA::offset((wm * TM + i) * 32 + row, half);
#pragma unroll
    for (int j = 0; j < TN; j++) b_off[j] = TA::BYTES + TB::offset((wn * TN + j) * 32 + row, half);
    const int as_off = SCALES + (wm * TM * 32 + row) * 4, bs_off = SCALES + SF::B_OFFSET + (wn * TN * 32 + row) * 4;

    uint4_t qa[2][TM], qb[2][TN];
    int xa[2][TM], xb[2][TN];     // scales of a tile, this half's block of step 0 in byte 0, of step 1 in byte 2
    auto load_step = [&](int stage_off, int st, uint4_t (&na)[TM], uint4_t (&nb)[TN]) {
        const char* p = smem + stage_off;
#pragma unroll
        for (int i = 0; i < TM; i++) na[i] = *reinterpret_cast<const uint4_t*>(p + (a_off[i] ^ (st * 32)));
#pragma unroll
        for (int j = 0; j < TN; j++) nb[j] = *reinterpret_cast<const uint4_t*>(p + (b_off[j] ^ (st * 32)));
    };
    auto load_scales = [&](int stage_off, int first, int (&na)[TM], int (&nb)[TN]) {
        const char* p = smem + stage_off;
        const unsigned ma = mx_scale_mask(a.blocks, first);
        const int shift = 8 * half;
#pragma unroll
        for (int i = 0; i < TM; i++) na[i] = (int)((*reinterpret_cast<const unsigned*>(p + as_off + i * 128) & ma) >> shift);
#pragma unroll
        for (int j = 0; j < TN; j++) nb[j] = (int)((*reinterpret_cast<const unsigned*>(p + bs_off + j * 128) & ma) >> shift);
    };
    auto operand = [](const uint4_t& q) { return int8v_t{(int)q[0], (int)q[1], (int)q[2], (int)q[3], 0, 0, 0, 0}; };
    auto multiply0 = [&](const uint4_t (&ca)[TM], const uint4_t (&cb)[TN], const int (&ea)[TM], const int (&eb)[TN]) {
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int j = 0; j < TN; j++)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(ca[i]), operand(cb[j]), acc[i][j], 4, 4, 0, ea[i], 0, eb[j]);
    };
    auto multiply1 = [&](const uint4_t (&ca)[TM], const uint4_t (&cb)[TN], const int (&ea)[TM], const int (&eb)[TN]) {
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int j = 0; j < TN; j++)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(ca[i]), operand(cb[j]), acc[i][j], 4, 4, 2, ea[i], 2, eb[j]);
    };

#pragma unroll
    for (int p = 0; p < NSTAGE; p++)
        if (p < ntiles) gissue(p * STAGE);
    if (ntiles >= NSTAGE) __builtin_amdgcn_s_waitcnt(WaitVmLgkm0<(NSTAGE - 1) * LOADS>::IMM);
    else                  __builtin_amdgcn_s_waitcnt(WaitVmLgkm0<0>::IMM);
    __syncthreads();
    auto next_stage = [&](int off) { return (off + STAGE == NSTAGE * STAGE) ? 0 : off + STAGE; };
    int rd = 0;
    if (ntiles > 0) {
        load_scales(0, t_begin * 4, xa[0], xb[0]);
        load_step(0, 0, qa[0], qb[0]);
    }
    // one tile: step 0 with the reads of step 1 behind it, then the tile's barrier,
    // then step 1 with the reads of the next tile behind it
    auto tile = [&](int t, bool more, auto& cxa, auto& cxb, auto& nxa, auto& nxb, bool request, int vm_wait) {
        load_step(rd, 1, qa[1], qb[1]);
        multiply0(qa[0], qb[0], cxa, cxb);
        if (!more) {
            multiply1(qa[1], qb[1], cxa, cxb);
            return;
        }
        if (vm_wait) __builtin_amdgcn_s_waitcnt(WaitVmLgkm0<(NSTAGE - 2) * LOADS>::IMM);
        else         __builtin_amdgcn_s_waitcnt(WaitVmLgkm0<0>::IMM);
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
        const int freed = rd;
        rd = next_stage(rd);
        if (request) gissue(freed);
        load_scales(rd, (t_begin + t + 1) * 4, nxa, nxb);
        load_step(rd, 0, qa[0], qb[0]);
        multiply1(qa[1], qb[1], cxa, cxb);
    };
    int t = 0;
    for (; t + NSTAGE + 1 < ntiles; t += 2) {
        tile(t, true, xa[0], xb[0], xa[1], xb[1], true, 1);
        tile(t + 1, true, xa[1], xb[1], xa[0], xb[0], true, 1);
    }
    // the rest: at most NSTAGE + 1 tiles
    for (; t < ntiles; t += 2) {
        tile(t, t + 1 < ntiles, xa[0], xb[0], xa[1], xb[1], t + NSTAGE < ntiles, 0);
        if (t + 1 < ntiles) tile(t + 1, t + 2 < ntiles, xa[1], xb[1], xa[0], xb[0], t + 1 + NSTAGE < ntiles, 0);
    }

    __syncthreads();
    char* stage = smem + wave * EPI_BYTES;
    EpilogueBands<TM, TN, WTN, EPITCH, 0>::run(acc, stage, lane, m0 + wm * (BM / WM), n0 + wn * WTN, 0, split, epi);
}

// ---- block scaled . fp16 -----------------------------------------------------------
// One side's fragments.  A contraction tile is 64 values (two blocks); lanes 0..31
// take the first block, lanes 32..63 the second, 8 values a step: the contraction
// order inside a tile is a permutation both sides share.
template <int FMT, int T> struct MxFrags;

template <int T>
struct MxFrags<NG_MX_NONE, T> {
    static constexpr int LINE = 128;
    half8_t v[2][T];
    int off[T];
    template <class Tile> __device__ __forceinline__ void init(int row0, int lane, int base)
    {
#pragma unroll
        for (int i = 0; i < T; i++) off[i] = base + Tile::offset(row0 + i * 32 + (lane & 31), (lane >> 5) * 4);
    }
    __device__ __forceinline__ void load_tile(const char*, int, int, int, unsigned) {}
    // chunk 4 half + step of the line: the xor with the swizzle distributes
    __device__ __forceinline__ void load_step(const char* stage, int step, int to)
    {
#pragma unroll
        for (int i = 0; i < T; i++) v[to][i] = *reinterpret_cast<const half8_t*>(stage + (off[i] ^ (step * 16)));
    }
    __device__ __forceinline__ half8_t get(int i, int step, int /*tile*/) const { return v[step & 1][i]; }
};

template <int T>
struct MxFrags<NG_MX_FP4, T> {
    static constexpr int LINE = 32;
    uint4_t raw[2][T];
    float scale[2][T];
    int off[T], soff;
    template <class Tile> __device__ __forceinline__ void init(int row0, int lane, int base)
    {
#pragma unroll
        for (int i = 0; i < T; i++) off[i] = base + Tile::offset(row0 + i * 32 + (lane & 31), lane >> 5);
    }
    __device__ __forceinline__ void load_tile(const char* stage, int scales, int shift, int to, unsigned mask)
    {
#pragma unroll
        for (int i = 0; i < T; i++) {
            raw[to][i] = *reinterpret_cast<const uint4_t*>(stage + off[i]);
            scale[to][i] = mx_scale_value(((*reinterpret_cast<const unsigned*>(stage + scales + i * 128) & mask) >> shift) & 255u);
        }
    }
    __device__ __forceinline__ void load_step(const char*, int, int) {}
    __device__ __forceinline__ half8_t get(int i, int step, int tile) const { return mx_expand_fp4(raw[tile][i][step], scale[tile][i]); }
};

template <int T>
struct MxFrags<NG_MX_INT8, T> {
    static constexpr int LINE = 64;
    uint4_t raw[2][T][2];
    unsigned scale[2][T];
    int off[T];
    template <class Tile> __device__ __forceinline__ void init(int row0, int lane, int base)
    {
#pragma unroll
        for (int i = 0; i < T; i++) off[i] = base + Tile::offset(row0 + i * 32 + (lane & 31), (lane >> 5) * 2);
    }
    __device__ __forceinline__ void load_tile(const char* stage, int scales, int shift, int to, unsigned mask)
    {
#pragma unroll
        for (int i = 0; i < T; i++) {
            raw[to][i][0] = *reinterpret_cast<const uint4_t*>(stage + off[i]);
            raw[to][i][1] = *reinterpret_cast<const uint4_t*>(stage + (off[i] ^ 16));
            scale[to][i] = ((*reinterpret_cast<const unsigned*>(stage + scales + i * 128) & mask) >> shift) & 255u;
        }
    }
    __device__ __forceinline__ void load_step(const char*, int, int) {}
    __device__ __forceinline__ half8_t get(int i, int step, int tile) const
    {
        const MxInt8Scale s = mx_int8_scale(scale[tile][i]);
        const uint4_t& q = raw[tile][i][step >> 1];
        half2_t a, b, c, d;
        mx_expand_int8(q[(step & 1) * 2], s, a, b);
        mx_expand_int8(q[(step & 1) * 2 + 1], s, c, d);
        return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
};

template <int FA_, int FB_, int BM, int BN, int WM, int WN, int NSTAGE, class Epi>
__global__ __launch_bounds__(WM * WN * 64)
void mxmix_kernel(MxSide a, MxSide b, Epi epi, CoreShape s)
{
    constexpr int NT = WM * WN * 64, WAVES = WM * WN;
    constexpr int TM = BM / WM / 32, TN = BN / WN / 32, WTN = BN / WN;
    using GA = MxFrags<FA_, TM>;
    using GB = MxFrags<FB_, TN>;
    using TA = MxTile<BM, GA::LINE>;
    using TB = MxTile<BN, GB::LINE>;
    using FA = MxFetch<TA, BM, NT, FA_ != NG_MX_NONE>;
    using FB = MxFetch<TB, BN, NT, FB_ != NG_MX_NONE>;
    // only the block-scaled side has scales
    constexpr int SROWS_A = FA_ != NG_MX_NONE ? BM : 0, SROWS_B = FB_ != NG_MX_NONE ? BN : 0;
    using SF = MxScaleFetch<SROWS_A, SROWS_B, WAVES>;
    constexpr int SCALES = TA::BYTES + TB::BYTES;
    constexpr int STAGE = SCALES + SF::BYTES;
    constexpr int LOADS = FA::DATA + FB::DATA + SF::PER;
    constexpr int EPITCH = WTN * 4 + 16, EPI_BYTES = 32 * EPITCH;
    constexpr int SMEM = NSTAGE * STAGE > EPI_BYTES * WAVES ? NSTAGE * STAGE : EPI_BYTES * WAVES;
    static_assert(SMEM <= 160 * 1024, "tile stages exceed the LDS of a compute unit");
    static_assert((NSTAGE - 1) * LOADS < 64, "the wait counter holds 6 bits");
    static_assert((FA_ == NG_MX_NONE) != (FB_ == NG_MX_NONE), "one side is block scaled");
    __shared__ __attribute__((aligned(16))) char smem[SMEM];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WM, wn = wave / WM;

    int tm, tn, split;
    if (!block_work(s, tm, tn, split)) return;
    const int m0 = tm * BM, n0 = tn * BN;
    const int per = (s.k_tiles + s.splits - 1) / s.splits;
    const int t_begin = split * per, t_end = min(t_begin + per, s.k_tiles);
    const int ntiles = t_end - t_begin;

    FA fa;
    FB fb;
    SF sf;
    fa.init(a, m0, t_begin, tid);
    fb.init(b, n0, t_begin, tid);
    sf.init(a, b, m0, n0, wave, lane);
    const char* a_scales = FA_ != NG_MX_NONE ? a.scales + (long)m0 * a.scale_pitch : nullptr;
    const char* b_scales = FB_ != NG_MX_NONE ? b.scales + (long)n0 * b.scale_pitch : nullptr;
    const int blocks = FA_ != NG_MX_NONE ? a.blocks : b.blocks;
    int g_tile = t_begin;
    auto gissue = [&](int stage_off) {
        char* st = smem + stage_off;
        // two tiles share a dword of scales
#pragma unroll
        for (int i = 0; i < SF::PER; i++) sf.issue(i, a_scales, b_scales, (2 * g_tile) & ~3, st + SCALES, wave);
#pragma unroll
        for (int i = 0; i < FA::DATA; i++) fa.issue(i, st, wave);
#pragma unroll
        for (int i = 0; i < FB::DATA; i++) fb.issue(i, st + TA::BYTES, wave);
        fa.advance();
        fb.advance();
        g_tile++;
    };

    float16_t acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int v = 0; v < 16; v++) acc[i][j][v] = 0.0f;

    GA ga;
    GB gb;
    ga.template init<TA>(wm * TM * 32, lane, 0);
    gb.template init<TB>(wn * TN * 32, lane, TA::BYTES);
    const int as_off = SCALES + (wm * TM * 32 + (lane & 31)) * 4;
    const int bs_off = SCALES + SF::B_OFFSET + (wn * TN * 32 + (lane & 31)) * 4;
    auto load_tile = [&](int stage_off, int kt, int to) {
        const char* p = smem + stage_off;
        const unsigned mask = mx_scale_mask(blocks, (2 * kt) & ~3);
        const int shift = 8 * (((2 * kt) & 2) + (lane >> 5));
        ga.load_tile(p, as_off, shift, to, mask);
        gb.load_tile(p, bs_off, shift, to, mask);
    };
    auto load_step = [&](int stage_off, int step) {
        const char* p = smem + stage_off;
        ga.load_step(p, step, step & 1);
        gb.load_step(p, step, step & 1);
    };
    auto multiply = [&](int step, int tile) {
        half8_t fb_[TN];
#pragma unroll
        for (int j = 0; j < TN; j++) fb_[j] = gb.get(j, step, tile);
#pragma unroll
        for (int i = 0; i < TM; i++) {
            const half8_t fa_ = ga.get(i, step, tile);
#pragma unroll
            for (int j = 0; j < TN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa_, fb_[j], acc[i][j], 0, 0, 0);
        }
    };

#pragma unroll
    for (int p = 0; p < NSTAGE; p++)
        if (p < ntiles) gissue(p * STAGE);
    if (ntiles >= NSTAGE) __builtin_amdgcn_s_waitcnt(WaitVmLgkm0<(NSTAGE - 1) * LOADS>::IMM);
    else                  __builtin_amdgcn_s_waitcnt(WaitVmLgkm0<0>::IMM);
    __syncthreads();
    auto next_stage = [&](int off) { return (off + STAGE == NSTAGE * STAGE) ? 0 : off + STAGE; };
    int rd = 0;
    if (ntiles > 0) {
        load_tile(0, t_begin, 0);
        load_step(0, 0);
    }
    auto tile = [&](int t, bool more, int cur, bool request, int vm_wait) {
#pragma unroll
        for (int st = 0; st < 3; st++) {
            load_step(rd, st + 1);
            multiply(st, cur);
        }
        if (!more) {
            multiply(3, cur);
            return;
        }
        if (vm_wait) __builtin_amdgcn_s_waitcnt(WaitVmLgkm0<(NSTAGE - 2) * LOADS>::IMM);
        else         __builtin_amdgcn_s_waitcnt(WaitVmLgkm0<0>::IMM);
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
        const int freed = rd;
        rd = next_stage(rd);
        if (request) gissue(freed);
        load_tile(rd, t_begin + t + 1, cur ^ 1);
        load_step(rd, 0);
        multiply(3, cur);
    };
    int t = 0;
    for (; t + NSTAGE + 1 < ntiles; t += 2) {
        tile(t, true, 0, true, 1);
        tile(t + 1, true, 1, true, 1);
    }
    for (; t < ntiles; t += 2) {
        tile(t, t + 1 < ntiles, 0, t + NSTAGE < ntiles, 0);
        if (t + 1 < ntiles) tile(t + 1, t + 2 < ntiles, 1, t + 1 + NSTAGE < ntiles, 0);
    }

    __syncthreads();
    char* stage = smem + wave * EPI_BYTES;
    EpilogueBands<TM, TN, WTN, EPITCH, 0>::run(acc, stage, lane, m0 + wm * (BM / WM), n0 + wn * WTN, 0, split, epi);
}

}  // namespace ng
