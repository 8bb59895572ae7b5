// LDS-tiled products of block-scaled operands for gfx950.
//
//   mx44_kernel   fp4 . fp4 on the scaled matrix instruction (v_mfma_scale 32x32x64):
//                 a lane's 32 contraction values are exactly one block, so an operand
//                 register quad is one 16-byte chunk as it lies in memory and the block's
//                 scale byte goes into the instruction.
//   mxmix_kernel  fp4 or int8 . fp16 on v_mfma 32x32x16 f16: codes travel through LDS as
//                 they are and become fp16 in registers, in the shadow of the matrix pipe.
//
// What bounds them.  fp4 . fp4 at 8192^3: 280..300 us, 3700..3900 TFLOP/s, where a loop of
// nothing but the instruction on random operands reaches 6400 (power; 8850 on zeros) and
// the library's product 3175.  What it took: 256 x 256 tiles of 256 values (128-byte lines: half the
// memory requests of 128 values, 310 -> 298 us), scales fetched for four lanes' dwords of a line
// at once (340 -> 310 us: a dword a line made as many requests as the codes), and every tile on one
// path without a drain loop (454 -> 345 us).  fp16 . int8 at 4096x8192x8000: 460 us, 1140
// TFLOP/s (a plain fp16 product of the library: 415 us); fp16 . fp4 there 430 us.
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

// Fetches one operand's tiles: request i of a tile brings lines i * STEP .. of it.  The
// swizzle repeats after STEP lines, so the requests differ by a scalar base alone and a
// lane keeps one offset.  What does not exist reads as zero: lines behind the last one
// lie behind the descriptor's end, chunks behind a line's last take an offset that does.
template <class Tile, int NT>
struct MxFetch {
    // PART: the tile has fewer chunks than the workgroup threads; its first WAVES_WITH wavefronts bring it
    static constexpr bool PART = Tile::CHUNKS < NT;
    static constexpr int WAVES_WITH = PART ? Tile::CHUNKS / 64 : NT / 64;
    static constexpr int DATA = PART ? 1 : Tile::CHUNKS / NT, STEP = NT / Tile::CPR;
    static_assert((PART ? Tile::CHUNKS % 64 : Tile::CHUNKS % NT) == 0 && NT % Tile::CPR == 0, "tile chunks must divide evenly over threads");
    static_assert(DATA == 1 || (STEP / Tile::LP) % Tile::CPR == 0, "requests must be whole periods of the swizzle");
    const char* base;        // of the next tile
    int bytes;               // from there to the end of the operand, 2^31 - 1 if that is further
    int pitch;
    unsigned off;
    int col, left;           // the lane's chunk of a line, chunks of a line not yet fetched
    __device__ __forceinline__ void init(const MxSide& s, int row0, int kt, int tid)
    {
        pitch = (int)s.pitch;
        base = s.data + (long)row0 * s.pitch + (long)kt * (Tile::CPR * 16);
        // a tile's lines span less than 2^30 bytes and so does a line, so a clamped end stays out of reach
        bytes = (int)min((long)(s.lines - 1 - row0) * s.pitch + (long)s.chunks * 16 - (long)kt * (Tile::CPR * 16), 0x7FFFFFFFl);
        left = s.chunks - kt * Tile::CPR;
        int line;
        Tile::chunk_pos(tid, line, col);
        off = (unsigned)line * (unsigned)s.pitch + (unsigned)col * 16u;
    }
    __device__ __forceinline__ unsigned lane_offset() const { return col < left ? off : NG_OOB_OFFSET; }
    __device__ __forceinline__ void issue(int i, unsigned lane_off, char* lds, int wave) const
    {
        const int skip = i * STEP * pitch;
        const BufferRsrc r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base + skip), 0, max(bytes - skip, 0), 0x00020000);
        buffer_load_chunk_to_lds(r, lds + (i * NT + wave * 64) * 16, lane_off);
    }
    __device__ __forceinline__ void advance()
    {
        base += Tile::CPR * 16;
        bytes -= Tile::CPR * 16;
        left -= Tile::CPR;
    }
};

// A dense operand whose lines lie across the contiguous axis (value i of line r at
// [i * ld + r]): 64 rows of LINES neighbouring values, read with the transposing LDS
// read, which takes 64 bytes from each of 4 rows, so rows differ in their 64-byte group.
template <int LINES>
struct MxAcrossTile {
    static constexpr int CPR = LINES / 8;
    static constexpr int PITCH = LINES * 2;
    static constexpr int CHUNKS = 64 * CPR;
    static constexpr int BYTES = 64 * PITCH;
    static_assert(CPR == 8 || CPR % 16 == 0, "rows of 128 bytes or whole periods of 256");
    // rows of 128 bytes take turns in a period by themselves
    static __device__ __forceinline__ int swizzle(int i) { return CPR == 8 ? ((i >> 1) & 1) * 4 : (i & 3) * 4; }
};

template <class Tile, int NT>
struct MxAcrossFetch {
    static constexpr int DATA = Tile::CHUNKS / NT, STEP = NT / Tile::CPR;
    static_assert(Tile::CHUNKS % NT == 0 && NT % Tile::CPR == 0 && STEP % 4 == 0, "requests must be whole periods of the swizzle");
    const char* base;        // of the next tile
    int pitch, row_bytes;    // of a row of the matrix; from this tile's first line to the last one
    int left;                // rows not yet fetched
    unsigned off;
    // s.lines: lines (values of a row), s.chunks: rows
    __device__ __forceinline__ void init(const MxSide& s, int line0, int kt, int tid)
    {
        pitch = (int)s.pitch;
        row_bytes = min(s.lines - line0, Tile::CPR * 8) * 2;
        base = s.data + (long)kt * 64 * s.pitch + (long)line0 * 2;
        left = s.chunks - kt * 64;
        const int i = tid / Tile::CPR, c = (tid % Tile::CPR) ^ Tile::swizzle(i);
        off = c * 16 < row_bytes ? (unsigned)i * (unsigned)pitch + (unsigned)c * 16u : NG_OOB_OFFSET;
    }
    __device__ __forceinline__ unsigned lane_offset() const { return off; }
    __device__ __forceinline__ void issue(int i, unsigned lane_off, char* lds, int wave) const
    {
        const int rows = min(left - i * STEP, STEP);
        const BufferRsrc r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base + (long)(i * STEP) * pitch), 0,
                                                               rows > 0 ? (rows - 1) * pitch + row_bytes : 0, 0x00020000);
        buffer_load_chunk_to_lds(r, lds + (i * NT + wave * 64) * 16, lane_off);
    }
    __device__ __forceinline__ void advance()
    {
        base += 64l * pitch;
        left -= 64;
    }
};

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

// Scales of the fp4 . fp4 kernel.  Fetched a dword (a tile of 128 values) per line they
// would be as many memory requests as the codes, since every line is a request of its own.
// So four lanes take the four dwords of one line (four tiles, a group) and a request
// serves 16 lines of them.  A tile's turn fetches a quarter of the group after next
// into a ring of three, so every tile issues the same number of requests.
template <int ROWS_A, int ROWS_B, int WAVES>
struct MxScaleRing {
    static constexpr int ROWS = ROWS_A + ROWS_B;
    static constexpr int PER = (ROWS + 64 * WAVES - 1) / (64 * WAVES);   // requests of a wavefront per quarter
    static constexpr int SLOT = 4 * PER * WAVES * 256, BYTES = 3 * SLOT;
    static_assert(ROWS_A % 16 == 0, "a request serves lines of one operand");
    const char *a_base, *b_base;    // scales of the tile's first lines from the slice's first block on
    int a_lines, b_lines, row;
    long pitch;                     // both operands have the same depth
    unsigned off;
    int dword;
    __device__ __forceinline__ void init(const MxSide& a, const MxSide& b, int m0, int n0, int first, int lane)
    {
        a_base = a.scales + (long)m0 * a.scale_pitch + first;
        b_base = b.scales + (long)n0 * b.scale_pitch + first;
        a_lines = a.lines - m0;
        b_lines = b.lines - n0;
        pitch = a.scale_pitch;
        row = lane >> 2;
        dword = (lane & 3) * 4;
        off = (unsigned)row * (unsigned)pitch + (unsigned)dword;
    }
    // request i of quarter p of group `group`, `left` blocks of the lines from the group's
    // first one on; dwords behind the last block are not read (they may lie behind the
    // scales' memory)
    __device__ __forceinline__ void issue(int p, int i, int group, int left, char* slot, int wave) const
    {
        const int id = (p * PER + i) * WAVES + wave;
        const bool is_b = id * 16 >= ROWS_A;
        const int row0 = id * 16 - (is_b ? ROWS_A : 0);
        const char* base = (is_b ? b_base : a_base) + row0 * pitch + group * 16;
        int lines = (is_b ? b_lines : a_lines) - row0;
        if (4 * PER * WAVES * 16 != ROWS) lines = id * 16 < ROWS ? lines : 0;
        const bool there = (row < lines) & (dword < left);     // no branch: it would split the products' schedule
        buffer_load_dword_to_lds(make_rsrc(base), slot + id * 256, there ? off : NG_OOB_OFFSET);
    }
};

// ---- fp4 . fp4 --------------------------------------------------------------------
template <int BM, int BN, int BK, int WM, int WN, int NSTAGE, class Epi>
__global__ __launch_bounds__(WM * WN * 64)
void mx44_kernel(MxSide a, MxSide b, Epi epi, CoreShape s)
{
    constexpr int LINE = BK / 2, NT = WM * WN * 64, WAVES = WM * WN;
    constexpr int STEPS = BK / 64, DW = BK / 128;            // matrix steps and scale dwords of a tile
    constexpr int TM = BM / WM / 32, TN = BN / WN / 32, WTN = BN / WN;
    using TA = MxTile<BM, LINE>;
    using TB = MxTile<BN, LINE>;
    using FA = MxFetch<TA, NT>;
    using FB = MxFetch<TB, NT>;
    using SF = MxScaleRing<BM, BN, WAVES>;
    constexpr int STAGE = TA::BYTES + TB::BYTES;
    constexpr int SCALES = NSTAGE * STAGE;
    constexpr int SREQ = SF::PER * DW;                       // scale requests of a wavefront per tile
    constexpr int LOADS = FA::DATA + FB::DATA + SREQ;        // all its requests
    constexpr int EPITCH = WTN * 4 + 16, EPI_BYTES = 32 * EPITCH;
    constexpr int SMEM = SCALES + SF::BYTES > EPI_BYTES * WAVES ? SCALES + SF::BYTES : EPI_BYTES * WAVES;
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
    sf.init(a, b, m0, n0, t_begin * (BK / 32), lane);
    const int blocks = a.blocks - t_begin * (BK / 32);      // from this slice's first one on
    // request q of a tile into the stage at st: its codes, and quarters p .. p + DW - 1 of a
    // group of scales 8 dwords ahead
    auto request = [&](int q, char* st, int p, int group, char* slot) {
        if (q < FA::DATA) fa.issue(q, fa.lane_offset(), st, wave);
        else if (q < FA::DATA + FB::DATA) fb.issue(q - FA::DATA, fb.lane_offset(), st + TA::BYTES, wave);
        else if (q < LOADS) sf.issue(p + (q - FA::DATA - FB::DATA) / SF::PER, (q - FA::DATA - FB::DATA) % SF::PER, group, blocks - group * 16, slot, wave);
    };
    auto advance = [&]() {
        fa.advance();
        fb.advance();
    };

    float16_t acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int v = 0; v < 16; v++) acc[i][j][v] = 0.0f;

    // lane-constant addresses of block `half` of the lane's line; blocks of 32 lines lie a
    // constant apart, and the step's chunk is an xor away (the swizzle distributes)
    const int a_off = TA::offset(wm * TM * 32 + row, half), b_off = TA::BYTES + TB::offset(wn * TN * 32 + row, half);
    const int as_off = SCALES + (wm * TM * 32 + row) * 16, bs_off = SCALES + (BM + wn * TN * 32 + row) * 16;

    uint4_t qa[2][TM], qb[2][TN];
    // scales of this and the next tile: of a dword's four blocks this half's of the even
    // step in byte 0, of the odd step in byte 2
    int xa[DW][TM], xb[DW][TN];
    unsigned ya[DW][TM], yb[DW][TN];
    auto read_a = [&](const char* st, int step, int i) { return *reinterpret_cast<const uint4_t*>(st + (a_off ^ (step * 32)) + i * 32 * LINE); };
    auto read_b = [&](const char* st, int step, int j) { return *reinterpret_cast<const uint4_t*>(st + (b_off ^ (step * 32)) + j * 32 * LINE); };
    // scale dwords of the tile whose first dword is number d, from ring slot `slot` (a byte offset)
    auto load_scales = [&](int slot, int d, unsigned (&na)[DW][TM], unsigned (&nb)[DW][TN]) {
#pragma unroll
        for (int w = 0; w < DW; w++) {
            const char* p = smem + slot + ((d + w) & 3) * 4;
#pragma unroll
            for (int i = 0; i < TM; i++) na[w][i] = *reinterpret_cast<const unsigned*>(p + as_off + i * 512);
#pragma unroll
            for (int j = 0; j < TN; j++) nb[w][j] = *reinterpret_cast<const unsigned*>(p + bs_off + j * 512);
        }
    };
    auto take_scales = [&](int d) {
        const int shift = 8 * half;
#pragma unroll
        for (int w = 0; w < DW; w++) {
            const unsigned mask = mx_scale_mask(blocks, (d + w) * 4);
#pragma unroll
            for (int i = 0; i < TM; i++) xa[w][i] = (int)((ya[w][i] & mask) >> shift);
#pragma unroll
            for (int j = 0; j < TN; j++) xb[w][j] = (int)((yb[w][j] & mask) >> shift);
        }
    };
    auto product = [&](int step, int i, int j) {
        const int8v_t va{(int)qa[step & 1][i][0], (int)qa[step & 1][i][1], (int)qa[step & 1][i][2], (int)qa[step & 1][i][3], 0, 0, 0, 0};
        const int8v_t vb{(int)qb[step & 1][j][0], (int)qb[step & 1][j][1], (int)qb[step & 1][j][2], (int)qb[step & 1][j][3], 0, 0, 0, 0};
        const int ea = xa[step / 2][i], eb = xb[step / 2][j];
        if ((step & 1) == 0) acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(va, vb, acc[i][j], 4, 4, 0, ea, 0, eb);
        else                 acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(va, vb, acc[i][j], 4, 4, 2, ea, 2, eb);
    };

    // Requests run NSTAGE tiles ahead, past the last tile too: those fetch zeros (every
    // chunk is out of range), so all tiles take the same path and the wait counts are
    // constants.  Scales: all of group 0 and what of group 1 does not come with the first tiles.
    static_assert(NSTAGE * DW <= 4, "the first tiles bring at most the four quarters of group 1");
    auto next_slot = [&](int slot) { return slot == 2 * SF::SLOT ? 0 : slot + SF::SLOT; };
#pragma unroll
    for (int p = 0; p < 8 - NSTAGE * DW; p++)
#pragma unroll
        for (int i = 0; i < SF::PER; i++) {
            const int q = p < 4 ? p : p - 4 + NSTAGE * DW, group = p < 4 ? 0 : 1;
            sf.issue(q, i, group, blocks - group * 16, smem + SCALES + group * SF::SLOT, wave);
        }
#pragma unroll
    for (int p = 0; p < NSTAGE; p++) {
#pragma unroll
        for (int q = 0; q < LOADS; q++) request(q, smem + p * STAGE, p * DW, 1, smem + SCALES + SF::SLOT);
        advance();
    }
    __builtin_amdgcn_s_waitcnt(WaitVmLgkm0<(NSTAGE - 1) * LOADS>::IMM);
    __syncthreads();
    int rd = 0;
    int read_slot = 0, write_slot = 2 * SF::SLOT;       // ring slots of the group read next and of the one requested now
    load_scales(0, 0, ya, yb);
    take_scales(0);
#pragma unroll
    for (int i = 0; i < TM; i++) qa[0][i] = read_a(smem, 0, i);
#pragma unroll
    for (int j = 0; j < TN; j++) qb[0][j] = read_b(smem, 0, j);

    constexpr int N = TM * TN;
    constexpr int REQ = (LOADS + N - 1) / N, READ = (TM + TN + N - 1) / N;
    // A tile: all steps but the last with the fragment reads of the following step between
    // the products; the barrier (behind it no wavefront reads this stage any more: the last
    // step's fragments are in registers); the last step with the requests into the freed
    // stage and the reads of the next tile between its products, so neither comes in a burst.
    for (int t = 0; t < ntiles; t++) {
#pragma unroll
        for (int step = 0; step < STEPS - 1; step++)
#pragma unroll
            for (int p = 0; p < N; p++) {
#pragma unroll
                for (int q = p * READ; q < (p + 1) * READ; q++) {
                    if (q < TM) qa[(step + 1) & 1][q < TM ? q : 0] = read_a(smem + rd, step + 1, q < TM ? q : 0);
                    else if (q < TM + TN) qb[(step + 1) & 1][q >= TM && q < TM + TN ? q - TM : 0] = read_b(smem + rd, step + 1, q >= TM && q < TM + TN ? q - TM : 0);
                }
                product(step, p / TN, p % TN);
                __builtin_amdgcn_sched_barrier(0);
            }
        __builtin_amdgcn_s_waitcnt(WaitVmLgkm0<(NSTAGE - 2) * LOADS>::IMM);
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
        const int freed = rd, d = t * DW;
        rd = (rd + STAGE == NSTAGE * STAGE) ? 0 : rd + STAGE;
        if (((d + DW) & 3) == 0) read_slot = next_slot(read_slot);
#pragma unroll
        for (int p = 0; p < N; p++) {
            product(STEPS - 1, p / TN, p % TN);
            if (p == 0) load_scales(read_slot, d + DW, ya, yb);
#pragma unroll
            for (int q = p * READ; q < (p + 1) * READ; q++) {
                if (q < TM) qa[0][q < TM ? q : 0] = read_a(smem + rd, 0, q < TM ? q : 0);
                else if (q < TM + TN) qb[0][q >= TM && q < TM + TN ? q - TM : 0] = read_b(smem + rd, 0, q >= TM && q < TM + TN ? q - TM : 0);
            }
#pragma unroll
            for (int q = p * REQ; q < (p + 1) * REQ; q++) request(q, smem + freed, d & 3, (d >> 2) + 2, smem + SCALES + write_slot);
            __builtin_amdgcn_sched_barrier(0);
        }
        advance();
        if (((d + DW) & 3) == 0) write_slot = next_slot(write_slot);
        take_scales(d + DW);
    }
    __builtin_amdgcn_s_waitcnt(WaitVmLgkm0<0>::IMM);    // nothing may land in LDS behind the next barrier

    __syncthreads();
    char* stage = smem + wave * EPI_BYTES;
    EpilogueBands<TM, TN, WTN, EPITCH, 0>::run(acc, stage, lane, m0 + wm * (BM / WM), n0 + wn * WTN, 0, split, epi);
}

// ---- block scaled . fp16 -----------------------------------------------------------
// A contraction tile is 64 values (two blocks): lanes 0..31 of a fragment take the
// first block, lanes 32..63 the second, 8 values a step.  The contraction order inside
// a tile is a permutation that both sides share.
//
// codes of one lane's block for the four steps of a tile, and their way to fp16 in two
// halves of four values
template <int FMT> struct MxBlock;
template <> struct MxBlock<NG_MX_FP4> {
    static constexpr int BYTES = 16;          // of a block
    uint4_t raw;
    float scale;
    __device__ __forceinline__ void load(const char* p, int, unsigned byte)
    {
        raw = *reinterpret_cast<const uint4_t*>(p);
        scale = mx_scale_value(byte);
    }
    template <int STEP, int HALF> __device__ __forceinline__ void expand(half8_t& v) const
    {
        const half2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(raw[STEP], scale, 2 * HALF);
        const half2_t b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(raw[STEP], scale, 2 * HALF + 1);
        v[4 * HALF] = a[0]; v[4 * HALF + 1] = a[1]; v[4 * HALF + 2] = b[0]; v[4 * HALF + 3] = b[1];
    }
};
template <> struct MxBlock<NG_MX_INT8> {
    static constexpr int BYTES = 32;
    uint4_t raw[2];
    MxInt8Scale scale;
    // the second chunk of the block lies at p2 (the tile's swizzle has moved it)
    __device__ __forceinline__ void load(const char* p, int to_second, unsigned byte)
    {
        raw[0] = *reinterpret_cast<const uint4_t*>(p);
        raw[1] = *reinterpret_cast<const uint4_t*>(p + to_second);
        scale = mx_int8_scale(byte);
    }
    template <int STEP, int HALF> __device__ __forceinline__ void expand(half8_t& v) const
    {
        half2_t a, b;
        mx_expand_int8(raw[STEP / 2][(STEP & 1) * 2 + HALF], scale, a, b);
        v[4 * HALF] = a[0]; v[4 * HALF + 1] = a[1]; v[4 * HALF + 2] = b[0]; v[4 * HALF + 3] = b[1];
    }
};

// X: the block-scaled operand (rows of C if X_IS_A, else its columns), D: the dense one.
// WX x WD wavefronts; a wavefront expands BX / WX lines of codes and multiplies them
// with BD / WD dense lines, so few X lines a wavefront mean little expansion.  ACROSS: the
// dense lines lie across the contiguous axis.
template <int FMT, bool X_IS_A, bool ACROSS, int BX, int BD, int WX, int WD, int NSTAGE, class Epi>
__global__ __launch_bounds__(WX * WD * 64)
void mxmix_kernel(MxSide x, MxSide d, Epi epi, CoreShape s)
{
    constexpr int NT = WX * WD * 64, WAVES = WX * WD;
    constexpr int TX = BX / WX / 32, TD = BD / WD / 32;
    constexpr int BM = X_IS_A ? BX : BD, BN = X_IS_A ? BD : BX;
    constexpr int TM = X_IS_A ? TX : TD, TN = X_IS_A ? TD : TX, WTN = TN * 32;
    using Block = MxBlock<FMT>;
    using TileX = MxTile<BX, 2 * Block::BYTES>;
    using TileD = std::conditional_t<ACROSS, MxAcrossTile<BD>, MxTile<BD, 128>>;
    using FX = MxFetch<TileX, NT>;
    using FD = std::conditional_t<ACROSS, MxAcrossFetch<MxAcrossTile<BD>, NT>, MxFetch<MxTile<BD, 128>, NT>>;
    // scales: groups of 16 blocks (8 tiles), four lanes a line, in a ring of two slots
    constexpr int SPER = BX / 16 / WAVES, SLOT = BX * 16;
    static_assert(BX % (16 * WAVES) == 0 && SPER <= 4, "scale requests must divide evenly over wavefronts");
    constexpr int STAGE = TileX::BYTES + TileD::BYTES, SCALES = NSTAGE * STAGE;
    constexpr int LOADS = FX::DATA + FD::DATA;          // one less for wavefronts without codes to bring (PART)
    constexpr int EPITCH = WTN * 4 + 16, EPI_BYTES = 32 * EPITCH;
    constexpr int SMEM = SCALES + 2 * SLOT > EPI_BYTES * WAVES ? SCALES + 2 * SLOT : EPI_BYTES * WAVES;
    static_assert(SMEM <= 160 * 1024, "tile stages exceed the LDS of a compute unit");
    static_assert((NSTAGE - 1) * LOADS < 64, "the wait counter holds 6 bits");
    __shared__ __attribute__((aligned(16))) char smem[SMEM];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wx = wave % WX, wd = wave / WX;
    const int half = lane >> 5, row = lane & 31;

    int tm, tn, split;
    if (!block_work(s, tm, tn, split)) return;
    const int m0 = tm * BM, n0 = tn * BN;
    const int x0 = X_IS_A ? m0 : n0, d0 = X_IS_A ? n0 : m0;
    const int per = (s.k_tiles + s.splits - 1) / s.splits;
    const int t_begin = split * per, t_end = min(t_begin + per, s.k_tiles);
    const int ntiles = t_end - t_begin;

    FX fx;
    FD fd;
    fx.init(x, x0, t_begin, tid);
    fd.init(d, d0, t_begin, tid);
    auto request = [&](int q, char* st) {
        if (q < FX::DATA) { if constexpr (!FX::PART) fx.issue(q, fx.lane_offset(), st, wave); }
        else if (q < LOADS) fd.issue(q - FX::DATA, fd.lane_offset(), st + TileX::BYTES, wave);
    };
    // codes that part of the wavefronts bring are requested before the tile's dense chunks
    auto request_part = [&](char* st) {
        if constexpr (FX::PART) {
            if (wave < FX::WAVES_WITH) fx.issue(0, fx.lane_offset(), st, wave);
        }
    };
    // at most `tiles` tiles' requests outstanding
    auto wait_tiles = [&](auto tiles) {
        constexpr int T = decltype(tiles)::value;
        if (!FX::PART || wave < FX::WAVES_WITH) __builtin_amdgcn_s_waitcnt(WaitVmLgkm0<T * LOADS>::IMM);
        else                                    __builtin_amdgcn_s_waitcnt(WaitVmLgkm0<T * (LOADS - 1)>::IMM);
    };
    auto advance = [&]() {
        fx.advance();
        fd.advance();
    };
    const int first = (2 * t_begin) & ~3;             // a dword of scales holds two tiles
    const int s_skip = 2 * t_begin - first;           // 0, or 2 where the slice starts inside a dword
    const int blocks = x.blocks - first;
    const char* s_base = x.scales + (long)x0 * x.scale_pitch + first;
    const unsigned s_off = (unsigned)(lane >> 2) * (unsigned)x.scale_pitch + (unsigned)(lane & 3) * 4u;
    // 16 lines of group `group`; dwords behind the last block are not read (they may lie
    // behind the scales' memory)
    auto request_scales = [&](int i, int group) {
        const int line = (i * WAVES + wave) * 16;
        const bool there = ((lane >> 2) < x.lines - x0 - line) & ((lane & 3) * 4 < blocks - group * 16);
        buffer_load_dword_to_lds(make_rsrc(s_base + line * x.scale_pitch + group * 16), smem + SCALES + (group & 1) * SLOT + line * 16,
                                 there ? s_off : NG_OOB_OFFSET);
    };

    float16_t acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int v = 0; v < 16; v++) acc[i][j][v] = 0.0f;

    constexpr int XC = Block::BYTES / 16;             // chunks of a block
    const int x_off = TileX::offset(wx * TX * 32 + row, half * XC);
    const int x_second = XC == 2 ? TileX::offset(row, half * XC + 1) - TileX::offset(row, half * XC) : 0;
    // dense fragments: contiguous lines have one address (the swizzle only depends on the
    // line inside a block of 32); lines across have one per block of 32, of row 32 half + (l / 4)
    // and the lane's 8-byte piece (l: lane inside 16)
    constexpr int DOFF = ACROSS ? TD : 1;
    int d_off[DOFF];
    if constexpr (ACROSS) {
        const int l = lane & 15, i = half * 32 + (l >> 2);
#pragma unroll
        for (int t = 0; t < TD; t++) {
            const int c = (wd * TD + t) * 4 + ((lane >> 4) & 1) * 2 + ((l >> 1) & 1);
            d_off[t] = TileX::BYTES + i * TileD::PITCH + ((c ^ TileD::swizzle(i)) * 16) + (l & 1) * 8;
        }
    } else {
        d_off[0] = TileX::BYTES + TileD::offset(wd * TD * 32 + row, half * 4);
    }
    const int s_read = SCALES + (wx * TX * 32 + row) * 16 + half;

    Block blk[TX];
    // few products a step cover the latency of LDS only two steps ahead: then all four steps'
    // dense fragments have registers of their own
    constexpr bool DEEP = TM * TN <= 4;
    constexpr int DBUF = DEEP ? 4 : 2;
    half8_t fx_[2][TX], fd_[DBUF][TD];
    // codes and scales of tile t (counted from the slice's first)
    auto load_blocks = [&](int stage_off, int t, int i, Block (&to)[TX]) {
        const int b = s_skip + 2 * t;                  // of the tile's first block
        const unsigned byte = *reinterpret_cast<const unsigned char*>(smem + s_read + ((b >> 4) & 1) * SLOT + i * 512 + (b & 15));
        to[i].load(smem + stage_off + x_off + i * 64 * Block::BYTES, x_second, b + half < blocks ? byte : 0u);
    };
    // dense chunk 4 half + step of the line: the xor with the swizzle distributes
    auto load_dense = [&](int stage_off, int step, int to, int i) {
        if constexpr (ACROSS) {
            const char* p = smem + stage_off + d_off[ACROSS ? i : 0] + step * 8 * TileD::PITCH;
            const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((NG_LDS short4_t*)(p));
            const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((NG_LDS short4_t*)(p + 4 * TileD::PITCH));
            const short8_t both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            fd_[to][i] = __builtin_bit_cast(half8_t, both);
        } else {
            fd_[to][i] = *reinterpret_cast<const half8_t*>(smem + stage_off + (d_off[0] ^ (step * 16)) + i * 32 * 128);
        }
    };
    auto product = [&](int step, int p) {
        const int i = p / TN, j = p % TN;
        if constexpr (X_IS_A) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fx_[step & 1][i], fd_[step % DBUF][j], acc[i][j], 0, 0, 0);
        else                  acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fd_[step % DBUF][i], fx_[step & 1][j], acc[i][j], 0, 0, 0);
    };
    // piece c (half of a line's 8 values) of a step's expansion
    auto expand0 = [&](int c, const Block (&from)[TX]) { if (c & 1) from[c / 2].template expand<0, 1>(fx_[0][c / 2]); else from[c / 2].template expand<0, 0>(fx_[0][c / 2]); };
    auto expand1 = [&](int c, const Block (&from)[TX]) { if (c & 1) from[c / 2].template expand<1, 1>(fx_[1][c / 2]); else from[c / 2].template expand<1, 0>(fx_[1][c / 2]); };
    auto expand2 = [&](int c, const Block (&from)[TX]) { if (c & 1) from[c / 2].template expand<2, 1>(fx_[0][c / 2]); else from[c / 2].template expand<2, 0>(fx_[0][c / 2]); };
    auto expand3 = [&](int c, const Block (&from)[TX]) { if (c & 1) from[c / 2].template expand<3, 1>(fx_[1][c / 2]); else from[c / 2].template expand<3, 0>(fx_[1][c / 2]); };

    // Requests run NSTAGE tiles ahead, past the last tile too: those fetch zeros (every
    // chunk is out of range), so all tiles take the same path.  The waits count the codes'
    // and the dense requests only; where scale requests lie between them, they wait for a little more.
#pragma unroll
    for (int i = 0; i < SPER; i++) request_scales(i, 0);
#pragma unroll
    for (int p = 0; p < NSTAGE; p++) {
        request_part(smem + p * STAGE);
#pragma unroll
        for (int q = 0; q < LOADS; q++) request(q, smem + p * STAGE);
        advance();
    }
    wait_tiles(std::integral_constant<int, NSTAGE - 1>{});
    __syncthreads();
    int rd = 0;
#pragma unroll
    for (int i = 0; i < TX; i++) load_blocks(0, 0, i, blk);
#pragma unroll
    for (int i = 0; i < TD; i++) load_dense(0, 0, 0, i);
    if constexpr (DEEP) {
#pragma unroll
        for (int i = 0; i < TD; i++) load_dense(0, 1, 1, i);
    }
#pragma unroll
    for (int c = 0; c < 2 * TX; c++) expand0(c, blk);

    constexpr int N = TM * TN;
    constexpr int REQ = (LOADS + N - 1) / N, READ = (TD + N - 1) / N, PIECES = (2 * TX + N - 1) / N;
    constexpr int TAIL = N / 2, TAIL_PIECES = (2 * TX + (N - TAIL) - 1) / (N - TAIL);
    // the group of scales after tile t's, one request at each of the group's first tiles (the
    // slot's last group has been read: the tile before this group took its scales two barriers ago)
    auto next_scales = [&](int t) {
        const int b = s_skip + 2 * t, i = (b & 15) / 2 - (s_skip && b < 16 ? 1 : 0);
        if (i < SPER) request_scales(i, (b >> 4) + 1);
    };
    if constexpr (DEEP) {
        Block nblk[TX];
        for (int t = 0; t < ntiles; t++) {
            // steps 0 and 1 with the dense reads of 2 and 3
#pragma unroll
            for (int step = 0; step < 2; step++)
#pragma unroll
                for (int p = 0; p < N; p++) {
#pragma unroll
                    for (int q = p * READ; q < (p + 1) * READ; q++)
                        if (q < TD) load_dense(rd, step + 2, step + 2, q < TD ? q : 0);
                    product(step, p);
#pragma unroll
                    for (int c = p * PIECES; c < (p + 1) * PIECES; c++)
                        if (c < 2 * TX) {
                            if (step == 0) expand1(c < 2 * TX ? c : 0, blk);
                            else           expand2(c < 2 * TX ? c : 0, blk);
                        }
                    __builtin_amdgcn_sched_barrier(0);
                }
            wait_tiles(std::integral_constant<int, NSTAGE - 2>{});
            __syncthreads();
            __builtin_amdgcn_sched_barrier(0);
            // steps 2 and 3 with the requests into the freed stage and the reads of the next tile
            const int freed = rd;
            rd = (rd + STAGE == NSTAGE * STAGE) ? 0 : rd + STAGE;
            next_scales(t);
            request_part(smem + freed);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int step = 2; step < 4; step++)
#pragma unroll
                for (int p = 0; p < N; p++) {
                    product(step, p);
                    if (step == 2) {
#pragma unroll
                        for (int q = p; q < TX; q += N) load_blocks(rd, t + 1, q, nblk);
                    }
#pragma unroll
                    for (int q = p * READ; q < (p + 1) * READ; q++)
                        if (q < TD) load_dense(rd, step - 2, step - 2, q < TD ? q : 0);
                    if (step == 2) {
#pragma unroll
                        for (int q = p * REQ; q < (p + 1) * REQ; q++) request(q, smem + freed);
                    }
#pragma unroll
                    for (int c = p * PIECES; c < (p + 1) * PIECES; c++)
                        if (c < 2 * TX) {
                            if (step == 2) expand3(c < 2 * TX ? c : 0, blk);
                            else           expand0(c < 2 * TX ? c : 0, nblk);
                        }
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
            for (int i = 0; i < TX; i++) blk[i] = nblk[i];
            advance();
        }
    } else {
        for (int t = 0; t < ntiles; t++) {
            // steps 0 .. 2, each with the dense reads and the expansion of the next between its products
#pragma unroll
            for (int step = 0; step < 3; step++)
#pragma unroll
                for (int p = 0; p < N; p++) {
#pragma unroll
                    for (int q = p * READ; q < (p + 1) * READ; q++)
                        if (q < TD) load_dense(rd, step + 1, (step + 1) & 1, q < TD ? q : 0);
                    product(step, p);
#pragma unroll
                    for (int c = p * PIECES; c < (p + 1) * PIECES; c++)
                        if (c < 2 * TX) {
                            if (step == 0) expand1(c < 2 * TX ? c : 0, blk);
                            else if (step == 1) expand2(c < 2 * TX ? c : 0, blk);
                            else expand3(c < 2 * TX ? c : 0, blk);
                        }
                    __builtin_amdgcn_sched_barrier(0);
                }
            wait_tiles(std::integral_constant<int, NSTAGE - 2>{});
            __syncthreads();
            __builtin_amdgcn_sched_barrier(0);
            const int freed = rd;
            rd = (rd + STAGE == NSTAGE * STAGE) ? 0 : rd + STAGE;
            next_scales(t);
            request_part(smem + freed);
            __builtin_amdgcn_sched_barrier(0);
            // last step: the next tile's codes first, the requests into the freed stage, the
            // next tile's dense reads, and in the second half its first expansion
#pragma unroll
            for (int i = 0; i < TX; i++) load_blocks(rd, t + 1, i, blk);
#pragma unroll
            for (int p = 0; p < N; p++) {
                product(3, p);
#pragma unroll
                for (int q = p * READ; q < (p + 1) * READ; q++)
                    if (q < TD) load_dense(rd, 0, 0, q < TD ? q : 0);
#pragma unroll
                for (int q = p * REQ; q < (p + 1) * REQ; q++) request(q, smem + freed);
                if (p >= TAIL) {
#pragma unroll
                    for (int c = (p - TAIL) * TAIL_PIECES; c < (p - TAIL + 1) * TAIL_PIECES; c++)
                        if (c < 2 * TX) expand0(c < 2 * TX ? c : 0, blk);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            advance();
        }
    }
    __builtin_amdgcn_s_waitcnt(WaitVmLgkm0<0>::IMM);    // nothing may land in LDS behind the next barrier

    __syncthreads();
    char* stage = smem + wave * EPI_BYTES;
    const int wm = X_IS_A ? wx : wd, wn = X_IS_A ? wd : wx;
    EpilogueBands<TM, TN, WTN, EPITCH, 0>::run(acc, stage, lane, m0 + wm * TM * 32, n0 + wn * WTN, 0, split, epi);
}

// The stores of a product: those of ScaleStoreEpilogue, whose relu keeps NaN here (the mark of a
// block with an infinity or a NaN shows in a rectified product), and PartialEpilogue, except that 8
// neighbouring values of a row that is not 16-byte aligned (an odd row length) still go out
// in wide stores, which the hardware takes at any alignment, instead of one by one
// (4001x5003 fp32 outputs of fp16 by int8, k = 64: 64 us one by one, 28 us so).
template <typename T>
struct MxStoreEpilogue : ScaleStoreEpilogue<T, true> {
    typedef ScaleStoreEpilogue<T, true> Base;
    typedef typename Base::bits_t bits_t;
    __device__ __forceinline__ void store8(int i, int j0, int z, int split, const float (&acc)[8]) const
    {
        if (this->vec || i >= this->m || j0 + 8 > this->n) {
            Base::store8(i, j0, z, split, acc);
            return;
        }
        bits_t* p = reinterpret_cast<bits_t*>(this->C + (long)i * this->ldc + j0);
        bits_t out[8];
        if (this->beta != 0.0f) __builtin_memcpy(out, p, sizeof(out));
#pragma unroll
        for (int e = 0; e < 8; e++) {
            float v = this->scale(acc[e]);
            if (this->beta != 0.0f) v += this->beta * StoreBits<T>::widen(out[e]);
            out[e] = StoreBits<T>::round(v, this->sr_bits, this->seed, this->stream, this->rng_index(i, j0 + e, z));
        }
        __builtin_memcpy(p, out, sizeof(out));
    }
};
struct MxPartialEpilogue : PartialEpilogue {
    __device__ __forceinline__ void store8(int i, int j0, int z, int split, const float (&acc)[8]) const
    {
        if (vec || i >= m || j0 + 8 > n) PartialEpilogue::store8(i, j0, z, split, acc);
        else                             __builtin_memcpy(ws + ((long)split * m + i) * (long)n + j0, acc, sizeof(acc));
    }
};

// tile: 256, 128 or 64 lines of either side; defined in mx_mix.hip for the epilogues of products
template <int FMT, class Epi>
void launch_mix(bool x_is_a, bool across, int tile, const MxSide& x, const MxSide& d, const Epi& epi, const CoreShape& s, dim3 grid,
                hipStream_t stream);

}  // namespace ng
