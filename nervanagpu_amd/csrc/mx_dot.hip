// Products of block-scaled matrices: C = round(beta*C + relu(alpha * A.B)).
#include "mx_skinny.h"

#include <algorithm>

namespace ng {

// A dense operand as the kernels want it: lines of 16-byte chunks with the contraction
// contiguous and zeros beyond it.
//
// Lines that are contiguous but not in whole, aligned chunks: a thread a chunk.
__global__ __launch_bounds__(256)
void mx_pack_along_kernel(const unsigned short* __restrict__ X, long ld, FastDiv per_line, int chunks, int depth, unsigned total,
                          unsigned short* __restrict__ out)
{
    const unsigned id = blockIdx.x * 256u + threadIdx.x;
    if (id >= total) return;
    const int line = (int)per_line.div(id), i0 = (int)(id - (unsigned)line * (unsigned)chunks) * 8;
    unsigned short v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = i0 + i < depth ? X[(long)line * ld + i0 + i] : (unsigned short)0;
    uint4_t w;
    __builtin_memcpy(&w, v, 16);
    *reinterpret_cast<uint4_t*>(out + (size_t)id * 8) = w;
}

// Lines across the contiguous axis: 64 lines x 64 values turned in LDS, all of a
// thread's loads in flight at once
__global__ __launch_bounds__(256)
void mx_pack_across_kernel(const unsigned short* __restrict__ X, long ld, int lines, int depth, int padded,
                           unsigned short* __restrict__ out)
{
    __shared__ unsigned short tile[64][66];
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    const int line0 = (int)blockIdx.x * 64, i0 = (int)blockIdx.y * 64;
    unsigned short v[16];
#pragma unroll
    for (int j = 0; j < 16; j++) {
        const int i = i0 + j * 4 + ty;
        v[j] = (line0 + tx < lines && i < depth) ? X[(long)i * ld + line0 + tx] : (unsigned short)0;
    }
#pragma unroll
    for (int j = 0; j < 16; j++) tile[tx][j * 4 + ty] = v[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 16; j++) {
        const int line = line0 + j * 4 + ty;
        if (line < lines && i0 + tx < padded) out[(long)line * padded + i0 + tx] = tile[j * 4 + ty][tx];
    }
}

struct MxArgs {
    int c_dtype, m, n, k;
    ng_mx_operand A, B;
    void* C; int ldc;
    float alpha, beta;
    unsigned flags, seed, rng_stream;
    char* ws; size_t ws_bytes;
    hipStream_t stream;
};

static int ceil_div(int a, int b) { return (a + b - 1) / b; }

static int padded_depth(int k) { return ceil_div(k, 8) * 8; }

// a dense operand that the kernels can read where it lies: whole 16-byte chunks, along
// the contraction, or (right operand of a fp4 one) across it
static bool dense_in_place(const ng_mx_operand& o, const ng_mx_operand* left, int lines, int k)
{
    if (((uintptr_t)o.codes & 15) != 0) return false;
    if (o.along) return k % 8 == 0 && (lines <= 1 || (o.ld % 8 == 0 && o.ld < (1L << 21)));
    return left && left->format == NG_MX_FP4 && lines % 8 == 0 && o.ld % 8 == 0 && o.ld < (1L << 21);
}

// whether this product takes the kernel for few dense lines
static bool is_skinny(const ng_mx_operand& A, const ng_mx_operand& B, int m, int n)
{
    return (A.format == NG_MX_FP4 && B.format == NG_MX_NONE && n <= 32) || (A.format == NG_MX_NONE && B.format == NG_MX_FP4 && m <= 32);
}

// room for a copy of a dense operand that is not laid out for its kernel
static size_t pack_bytes(const ng_mx_operand& o, const ng_mx_operand* left, bool skinny, int lines, int k)
{
    if (o.format != NG_MX_NONE) return 0;
    if (skinny && lines > 1) return mx_fragment_bytes(lines, k);
    if (dense_in_place(o, skinny ? nullptr : left, lines, k)) return 0;
    return align_up((size_t)lines * padded_depth(k) * 2, 256);
}

// skinny: groups of 16 dense lines of the kernel for few of them, 0 for tiles
struct MxPlan { int bm, bn, bk, splits, skinny; };

// as many slices of the contraction as give about one workgroup per CU, each at least
// `least` tiles deep
static int choose_slices(int out_tiles, int k_tiles, int least, size_t slice_bytes, size_t ws_bytes)
{
    const int cus = device_cu_count();
    int splits = std::max(1, cus / std::max(out_tiles, 1));
    splits = std::min(splits, std::max(1, k_tiles / least));
    if (ws_bytes != SIZE_MAX && slice_bytes) splits = (int)std::min<size_t>((size_t)splits, std::max<size_t>(1, ws_bytes / slice_bytes));
    while (splits > 1 && (splits - 1) * ceil_div(k_tiles, splits) >= k_tiles) splits--;
    return std::max(splits, 1);
}

static bool is_44(const ng_mx_operand& A, const ng_mx_operand& B) { return A.format == NG_MX_FP4 && B.format == NG_MX_FP4; }

static MxPlan choose_plan(int m, int n, int k, const ng_mx_operand& A, const ng_mx_operand& B, size_t ws_bytes)
{
    const int cus = device_cu_count();
    auto tiles = [&](int bm, int bn) { return (long)ceil_div(m, bm) * ceil_div(n, bn); };
    MxPlan p{128, 128, 64, 1, 0};
    // a slice of less than 512 values costs more in the sum of the slices than it saves
    // (300x500 outputs of k = 600: two slices 16 us)
    int least = 8;
    if (is_skinny(A, B, m, n)) {
        p.skinny = ((A.format == NG_MX_NONE ? m : n) + 15) / 16;
        return p;
    }
    if (is_44(A, B)) {
        p.bk = 256;
        least = 2;
        // 256 x 256 where they cover half the chip and more than two of their tiles follow each other; 64 x 64 where
        // 128 x 128 would leave half of it idle (1111x777 outputs of k = 2500: 20 us and a sum of slices, 12 us without)
        if (m >= 256 && n >= 256 && tiles(256, 256) > cus / 2 && k > 512) p.bm = p.bn = 256;
        else if (tiles(128, 128) <= cus / 2) p.bm = p.bn = 64;
    } else if (m >= 256 && n >= 256 && tiles(256, 256) > cus / 2 && k > 256) {
        // a contraction of few tiles is all prologue and store: more, smaller workgroups overlap
        // those (9216x4096 outputs of k = 128: 48 us on 256x256 tiles, 35 us on 128x128 with two stages)
        p.bm = p.bn = 256;
    } else if (tiles(128, 128) <= cus / 2 && tiles(128, 128) * std::max(1, ceil_div(k, 64) / least) < cus) {
        // a few workgroups wait out each tile's latency: four times as many where slices of the contraction do not
        // make up for them (512^3 7.5 us, 11.0 on 128x128 tiles; 600x900 outputs of k = 8000 66 us, 32 on 128x128 in slices;
        // 4096x48 of k = 4096 14.9 and 14.8)
        p.bm = p.bn = 64;
    }
    const int out_tiles = (int)std::min<long>(tiles(p.bm, p.bn), 1 << 30);
    p.splits = choose_slices(out_tiles, ceil_div(k, p.bk), least, (size_t)m * n * 4, ws_bytes);
    return p;
}

static MxSide make_side(const ng_mx_operand& o, int lines, int k)
{
    MxSide s;
    s.data = (const char*)o.codes;
    s.scales = (const char*)o.scales;
    s.lines = lines;
    if (o.format == NG_MX_NONE) {
        s.pitch = o.ld * 2;
        s.scale_pitch = 0;
        s.chunks = o.along ? k / 8 : k;     // rows, where the lines lie across them
        s.blocks = 0;
    } else {
        s.pitch = mx_code_pitch(o.format, k);
        s.scale_pitch = mx_scale_pitch(k);
        s.chunks = (int)(s.pitch / 16);
        s.blocks = mx_blocks(k);
    }
    return s;
}

static unsigned mx_sr_bits(unsigned flags, int dtype)
{
    if (!(flags & NG_FLAG_SR)) return 0;
    unsigned bits = flags >> 16;
    if (bits == 0) bits = 10;
    return std::max(1u, std::min(bits, dtype == NG_F16 ? 10u : 15u));
}

template <typename T, int FA, int FB, class Epi>
static void launch_tiles(const MxArgs& g, const MxPlan& p, const MxSide& a, const MxSide& b, const Epi& epi, const CoreShape& s,
                         dim3 grid)
{
    if constexpr (FA == NG_MX_FP4 && FB == NG_MX_FP4) {
        if (p.bm == 256)      hipLaunchKernelGGL((mx44_kernel<256, 256, 256, 2, 4, 2, Epi>), grid, dim3(512), 0, g.stream, a, b, epi, s);
        else if (p.bm == 128) hipLaunchKernelGGL((mx44_kernel<128, 128, 256, 2, 2, 2, Epi>), grid, dim3(256), 0, g.stream, a, b, epi, s);
        else                  hipLaunchKernelGGL((mx44_kernel<64, 64, 256, 2, 2, 2, Epi>), grid, dim3(256), 0, g.stream, a, b, epi, s);
    } else {
        constexpr bool X_IS_A = FA != NG_MX_NONE;
        const MxSide &x = X_IS_A ? a : b, &d = X_IS_A ? b : a;
        const bool across = !(X_IS_A ? g.B : g.A).along;
        launch_mix<X_IS_A ? FA : FB, Epi>(X_IS_A, across, p.bm, x, d, epi, s, grid, g.stream);
    }
}

template <bool X_IS_A, class Epi>
static int launch_skinny(const MxArgs& g, int groups, const MxSide& x, const MxSide& d, const Epi& epi)
{
    const dim3 grid((unsigned)ceil_div(x.lines, 16));
    // as many wavefronts as the contraction has units of 256, up to what a workgroup (and
    // with two groups of dense lines, the registers) holds: all loads of a short one are in flight at once
    const int units = ceil_div(x.blocks, 8);
#define NG_SKINNY(NC, WAVES, PACKED)                                                                                             \
    hipLaunchKernelGGL((mx_skinny_kernel<X_IS_A, NC, WAVES, PACKED, Epi>), grid, dim3(WAVES * 64), 0, g.stream, x, d, epi, x.lines, \
                       d.lines, d.chunks)
    if (d.lines == 1)     { if (units >= 16) NG_SKINNY(1, 16, false); else NG_SKINNY(1, 4, false); }
    else if (groups == 1) { if (units >= 16) NG_SKINNY(1, 16, true); else NG_SKINNY(1, 4, true); }
    else                  { if (units >= 16) NG_SKINNY(2, 8, true); else NG_SKINNY(2, 4, true); }
#undef NG_SKINNY
    NG_CHECK_LAUNCH("mx product of few lines");
    return 0;
}

template <typename T, int FA, int FB>
static int launch_product(const MxArgs& g, const MxSide& a, const MxSide& b)
{
    const MxPlan p = choose_plan(g.m, g.n, g.k, g.A, g.B, g.ws_bytes);
    CoreShape s;
    s.m = g.m;
    s.n = g.n;
    s.k_tiles = ceil_div(g.k, p.bk);
    s.passes = 1;
    s.splits = p.splits;
    s.tiles_m = ceil_div(g.m, p.bm);
    s.tiles_n = ceil_div(g.n, p.bn);
    const int tiles = s.tiles_m * s.tiles_n;
    const dim3 grid(grid_tiles(tiles, s.splits), grid_slices(tiles, s.splits), 1);
    const MxStoreEpilogue<T> epi{{(T*)g.C, 0, g.ldc, g.m, g.n, g.alpha, g.beta, (g.flags & NG_FLAG_RELU) ? 1u : 0u,
                                  mx_sr_bits(g.flags, g.c_dtype), g.seed, g.rng_stream,
                                  (((uintptr_t)g.C & 15) == 0 && g.ldc % 8 == 0 && g.n % 8 == 0) ? 1u : 0u}};
    if constexpr ((FA == NG_MX_FP4) != (FB == NG_MX_FP4)) {
        if (p.skinny) return launch_skinny<FA == NG_MX_FP4>(g, p.skinny, FA == NG_MX_FP4 ? a : b, FA == NG_MX_FP4 ? b : a, epi);
    }
    if (s.splits == 1) {
        launch_tiles<T, FA, FB>(g, p, a, b, epi, s, grid);
        NG_CHECK_LAUNCH("mx product");
    } else {
        const MxPartialEpilogue pe{{(float*)g.ws, g.m, g.n, 1, (g.n % 8 == 0) ? 1u : 0u}};
        launch_tiles<T, FA, FB>(g, p, a, b, pe, s, grid);
        NG_CHECK_LAUNCH("mx product slices");
        launch_splitk_reduce<T, MxStoreEpilogue<T>>((const float*)g.ws, s.splits, 1, g.m, g.n, epi, g.stream);
        NG_CHECK_LAUNCH("mx product sum");
    }
    return 0;
}

template <typename T>
static int dispatch(const MxArgs& g, const MxSide& a, const MxSide& b)
{
    const int fa = g.A.format, fb = g.B.format;
    if (fa == NG_MX_FP4 && fb == NG_MX_FP4)   return launch_product<T, NG_MX_FP4, NG_MX_FP4>(g, a, b);
    if (fa == NG_MX_FP4 && fb == NG_MX_NONE)  return launch_product<T, NG_MX_FP4, NG_MX_NONE>(g, a, b);
    if (fa == NG_MX_NONE && fb == NG_MX_FP4)  return launch_product<T, NG_MX_NONE, NG_MX_FP4>(g, a, b);
    if (fa == NG_MX_INT8 && fb == NG_MX_NONE) return launch_product<T, NG_MX_INT8, NG_MX_NONE>(g, a, b);
    return launch_product<T, NG_MX_NONE, NG_MX_INT8>(g, a, b);
}

static int check_operand(const char* name, const ng_mx_operand* o, int lines, int k)
{
    if (!o) return fail(-90, "ng_mx_gemm: null operand %s", name);
    if (o->format < NG_MX_NONE || o->format > NG_MX_INT8) return fail(-91, "ng_mx_gemm: unknown format %d of %s", o->format, name);
    if (!lines || !k) return 0;
    if (!o->codes || (o->format != NG_MX_NONE && !o->scales)) return fail(-92, "ng_mx_gemm: null operand %s", name);
    if (o->format != NG_MX_NONE && ((((uintptr_t)o->codes) | ((uintptr_t)o->scales)) & 15))
        return fail(-93, "ng_mx_gemm: codes and scales of %s must be 16-byte aligned", name);
    if (o->format == NG_MX_NONE && o->ld < (o->along ? k : lines) && (o->along ? lines : k) > 1)
        return fail(-94, "ng_mx_gemm: leading dimension of %s smaller than row length", name);
    return 0;
}

// formats, extents and what the kernels' 32-bit offsets hold; 0 or a status
static int check_product(int c_dtype, int m, int n, int k, const ng_mx_operand* A, const ng_mx_operand* B)
{
    if (c_dtype != NG_F16 && c_dtype != NG_F32) return fail(-95, "ng_mx_gemm: C must be fp16 or fp32");
    if (m < 0 || n < 0 || k < 0) return fail(-96, "ng_mx_gemm: negative extent");
    int rc = check_operand("A", A, m, k);
    if (!rc) rc = check_operand("B", B, n, k);
    if (rc) return rc;
    const bool ok = (A->format == NG_MX_FP4 && B->format == NG_MX_FP4) || ((A->format == NG_MX_NONE) != (B->format == NG_MX_NONE));
    if (!ok) return fail(-97, "ng_mx_gemm: formats %d and %d do not multiply (fp4 by fp4, or one dense fp16 operand)", A->format, B->format);
    if (k >= (1 << 21)) return fail(-98, "ng_mx_gemm: contraction of 2^21 or more");
    if ((long)m * n >= (1L << 32)) return fail(-99, "ng_mx_gemm: output of 2^32 or more elements");
    if (m >= (1 << 26) || n >= (1 << 26)) return fail(-99, "ng_mx_gemm: output of 2^26 or more rows or columns");
    return 0;
}

}  // namespace ng

using namespace ng;

extern "C" {

size_t ng_mx_gemm_workspace_bytes(int c_dtype, int m, int n, int k, const ng_mx_operand* A, const ng_mx_operand* B)
{
    if (!A || !B || m <= 0 || n <= 0 || k <= 0) return 0;
    (void)c_dtype;
    const MxPlan p = choose_plan(m, n, k, *A, *B, SIZE_MAX);
    const size_t slices = p.splits > 1 ? align_up((size_t)p.splits * m * n * 4, 256) : 0;
    const bool skinny = p.skinny != 0;
    return slices + pack_bytes(*A, nullptr, skinny, m, k) + pack_bytes(*B, A, skinny, n, k);
}

int ng_mx_gemm(int c_dtype, int m, int n, int k, const ng_mx_operand* A, const ng_mx_operand* B, void* C, int ldc,
               float alpha, float beta, unsigned flags, unsigned seed, unsigned rng_stream,
               void* workspace, size_t workspace_bytes, void* stream)
{
    int rc = check_product(c_dtype, m, n, k, A, B);
    if (rc) return rc;
    if (!m || !n) return 0;
    if (!C) return fail(-100, "ng_mx_gemm: null C");
    if (ldc < n && m > 1) return fail(-101, "ng_mx_gemm: leading dimension of C smaller than row length");
    const size_t need = ng_mx_gemm_workspace_bytes(c_dtype, m, n, k, A, B);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
        return fail(NG_MX_WORKSPACE, "ng_mx_gemm: this product needs %zu bytes of 16-byte aligned workspace, got %zu", need,
                    workspace ? workspace_bytes : (size_t)0);
    MxArgs g{c_dtype, m, n, k, *A, *B, C, ldc, alpha, beta, flags, seed, rng_stream,
             (char*)workspace, workspace_bytes, (hipStream_t)stream};
    // the pitch of a single line has no meaning and may be anything
    if (m == 1 && g.A.along) g.A.ld = k;
    if (n == 1 && g.B.along) g.B.ld = k;
    // dense operands that are not laid out for the kernels are copied behind the slices
    char* end = g.ws + need;
    int lines = m;
    const bool skinny = is_skinny(*A, *B, m, n);
    for (ng_mx_operand* o : {&g.A, &g.B}) {
        const size_t bytes = k ? pack_bytes(*o, o == &g.B ? A : nullptr, skinny, lines, k) : 0;
        if (bytes) {
            end -= bytes;
            const int padded = padded_depth(k);
            const unsigned short* from = (const unsigned short*)o->codes;
            unsigned short* to = (unsigned short*)end;
            if (skinny && lines > 1) {
                const unsigned total = (unsigned)(bytes / 16);
                hipLaunchKernelGGL(mx_pack_fragments_kernel, dim3((total + 255u) / 256u), dim3(256), 0, g.stream, from, o->ld, o->along,
                                   lines, k, (lines + 15) / 16, total, to);
            } else if (o->along && (long)lines * (padded / 8) < (1L << 31)) {
                const unsigned total = (unsigned)lines * (unsigned)(padded / 8);
                hipLaunchKernelGGL(mx_pack_along_kernel, dim3((total + 255u) / 256u), dim3(256), 0, g.stream, from, o->ld,
                                   FastDiv::make((unsigned)padded / 8u), padded / 8, k, total, to);
            } else if (!o->along) {
                hipLaunchKernelGGL(mx_pack_across_kernel, dim3((unsigned)ceil_div(lines, 64), (unsigned)ceil_div(padded, 64)), dim3(256), 0,
                                   g.stream, from, o->ld, lines, k, padded, to);
            } else {
                return fail(-98, "ng_mx_gemm: dense operand of 2^34 or more values that is not laid out in whole chunks");
            }
            NG_CHECK_LAUNCH("mx pack");
            o->codes = end;
            o->along = 1;
            o->ld = padded;
        }
        lines = n;
    }
    g.ws_bytes = (size_t)(end - g.ws);
    const int kd = (g.A.format == NG_MX_NONE || g.B.format == NG_MX_NONE) ? padded_depth(k) : k;
    const MxSide a = make_side(g.A, m, g.A.format == NG_MX_NONE && g.A.along ? kd : k);
    const MxSide b = make_side(g.B, n, g.B.format == NG_MX_NONE && g.B.along ? kd : k);
    return c_dtype == NG_F16 ? dispatch<_Float16>(g, a, b) : dispatch<float>(g, a, b);
}

}  // extern "C"
