// fp4 by a few fp16 lines (one token, some streams): bound by reading the codes once, and for
// small matrices by the launch (4096x4096 by one line: 5.1 us, of which the 9 MB of codes are
// 1.8 at the rate of a copy; 4096x25088 by 16 lines: 19 us, codes 11, the rest mostly the 16 dense
// lines that each workgroup reads from L2).  On 128x128 tiles these took 17 and 43 us.
//
// A workgroup owns 16 lines of codes and the whole contraction, which its WAVES
// wavefronts cut into equal shares; their sums meet in LDS, so there is one launch and no
// partial result in memory however few lines there are.  Matrix steps are 16 x 16 x 32 f16
// with the dense lines as the other operand.  Lane l takes line l & 15 and, of every
// 128 values, block l >> 4: one 16-byte load is the block, whose 8-value quarters feed
// four steps (both operands use that order of the contraction).
#pragma once

#include "mx_gemm.h"

namespace ng {

// Dense lines in fragment order: of every 256 values, 8 requests of a wavefront (16 bytes
// a lane, contiguous), request p holding for lane l values 128 (p / 4) + 32 (l / 16) + 8 (p % 4) .. + 7
// of line 16 c + l % 16; zeros where the matrix ends.  Read where they lie, 64 lanes' pieces
// would be 64 requests: 25088 x 16 values took 24 us of a 33 us product.
constexpr int MX_SKINNY_UNIT = 256;
inline size_t mx_fragment_bytes(int lines, int k)
{
    return (size_t)((k + MX_SKINNY_UNIT - 1) / MX_SKINNY_UNIT) * ((lines + 15) / 16) * 8192;
}

static __global__ __launch_bounds__(256)
void mx_pack_fragments_kernel(const unsigned short* __restrict__ X, long ld, int along, int lines, int depth, int groups,
                              unsigned total, unsigned short* __restrict__ out)
{
    const unsigned id = blockIdx.x * 256u + threadIdx.x;      // ((unit * groups + c) * 8 + p) * 64 + lane
    if (id >= total) return;
    const int lane = (int)(id & 63u), p = (int)((id >> 6) & 7u);
    const int uc = (int)(id >> 9), u = uc / groups, c = uc - u * groups;
    const int line = c * 16 + (lane & 15), k0 = u * MX_SKINNY_UNIT + (p >> 2) * 128 + (lane >> 4) * 32 + (p & 3) * 8;
    unsigned short v[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
        v[i] = (line < lines && k0 + i < depth) ? X[along ? (long)line * ld + k0 + i : (long)(k0 + i) * ld + line] : (unsigned short)0;
    uint4_t w;
    __builtin_memcpy(&w, v, 16);
    *reinterpret_cast<uint4_t*>(out + (size_t)id * 8) = w;
}

// NC: groups of 16 dense lines; PACKED: they are in fragment order, else one line lies
// contiguous (and the lanes of the others read nothing)
template <bool X_IS_A, int NC, int WAVES, bool PACKED, class Epi>
__global__ __launch_bounds__(WAVES * 64)
void mx_skinny_kernel(MxSide x, MxSide d, Epi epi, int xl, int dl, int depth8)
{
    constexpr int UNIT = MX_SKINNY_UNIT;    // values an iteration takes: two blocks a lane, 8 bytes of scales a line
    static_assert(PACKED || NC == 1, "only a single line is read where it lies");
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row = lane & 15, quarter = lane >> 4;
    const int x0 = (int)blockIdx.x * 16;
    const int units = (x.blocks + 7) / 8;   // of the contraction
    const int per = (units + WAVES - 1) / WAVES;
    const int u_begin = wave * per, u_end = min(u_begin + per, units);

    // lines past the end read line 0 and are not stored
    const char* codes = x.data + (long)(x0 + row < xl ? x0 + row : x0) * x.pitch + quarter * 16;
    const char* scales = x.scales + (long)(x0 + row < xl ? x0 + row : x0) * x.scale_pitch;
    const char* dense = PACKED ? d.data + lane * 16 : d.data + quarter * 64;

    struct Stage { uint4_t q[2]; uint2v_t s; half8_t v[NC][8]; };
    auto fetch = [&](int u, Stage& st) {
        st.s = *reinterpret_cast<const uint2v_t*>(scales + (long)u * 8);
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const int block = u * 8 + b * 4 + quarter;
            st.q[b] = uint4_t{0, 0, 0, 0};
            if (block < x.blocks) st.q[b] = *reinterpret_cast<const uint4_t*>(codes + (long)u * 128 + b * 64);
        }
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int p = 0; p < 8; p++) {
                if constexpr (PACKED) {
                    st.v[c][p] = *reinterpret_cast<const half8_t*>(dense + ((long)u * NC + c) * 8192 + p * 1024);
                } else {
                    const int k8 = u * (UNIT / 8) + (p >> 2) * 16 + quarter * 4 + (p & 3);     // which 8 values
                    st.v[c][p] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
                    if (k8 < depth8 && row == 0) st.v[c][p] = *reinterpret_cast<const half8_t*>(dense + (long)u * (UNIT * 2) + (p >> 2) * 256 + (p & 3) * 16);
                }
            }
    };
    float4_t acc[NC];
#pragma unroll
    for (int c = 0; c < NC; c++) acc[c] = float4_t{0, 0, 0, 0};
    auto multiply = [&](int u, const Stage& st) {
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const bool there = u * 8 + b * 4 + quarter < x.blocks;
            const float scale = mx_scale_value(there ? (st.s[b] >> (8 * quarter)) & 255u : 127u);
#pragma unroll
            for (int step = 0; step < 4; step++) {
                const half2_t e0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(st.q[b][step], scale, 0);
                const half2_t e1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(st.q[b][step], scale, 1);
                const half2_t e2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(st.q[b][step], scale, 2);
                const half2_t e3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(st.q[b][step], scale, 3);
                const half8_t w{e0[0], e0[1], e1[0], e1[1], e2[0], e2[1], e3[0], e3[1]};
#pragma unroll
                for (int c = 0; c < NC; c++) acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, st.v[c][b * 4 + step], acc[c], 0, 0, 0);
            }
        }
    };
    // the next unit is in flight while one is multiplied
    Stage cur, next;
    if (u_begin < u_end) fetch(u_begin, cur);
    for (int u = u_begin; u < u_end; u++) {
        if (u + 1 < u_end) fetch(u + 1, next);
        multiply(u, cur);
        cur = next;
    }

    // lane: dense line l & 15, code lines 4 (l >> 4) .. + 3
    __shared__ float sums[WAVES][NC][16][17];
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
        for (int v = 0; v < 4; v++) sums[wave][c][4 * quarter + v][row] = acc[c][v];
    __syncthreads();
    for (int id = tid; id < NC * 256; id += WAVES * 64) {
        // neighbouring threads take neighbouring elements of C
        const int c = id >> 8, r = X_IS_A ? (id >> 4) & 15 : id & 15, l = X_IS_A ? id & 15 : (id >> 4) & 15;
        if (x0 + r >= xl || c * 16 + l >= dl) continue;
        float sum = 0.0f;
#pragma unroll 4
        for (int w = 0; w < WAVES; w++) sum += sums[w][c][r][l];
        if (X_IS_A) epi.apply(x0 + r, c * 16 + l, 0, sum);
        else        epi.apply(c * 16 + l, x0 + r, 0, sum);
    }
}

}  // namespace ng
