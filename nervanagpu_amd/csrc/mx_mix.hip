// Tiles of block scaled . fp16 products: the instantiations of mxmix_kernel.
#include "mx_gemm.h"

namespace ng {

// A contraction of two tiles gains nothing from a third stage, and without it two
// workgroups more fit a CU (9216x4096 outputs of k = 128: 40 us with three, 35 us with two).
// Longer ones take eight wavefronts, two on a SIMD: expanding the codes keeps one wavefront from
// issuing products (4096x1000 outputs of k = 9216 in fp4 93 -> 88 us, across the rows 99 -> 95; 1024x4096
// of k = 4096 in int8 60 -> 55; with two stages four are better, 35 and 42 us).
template <int FMT, bool X_IS_A, bool ACROSS, class Epi>
static void launch(int tile, const MxSide& x, const MxSide& d, const Epi& epi, const CoreShape& s, dim3 grid, hipStream_t stream)
{
    if (tile == 256)         hipLaunchKernelGGL((mxmix_kernel<FMT, X_IS_A, ACROSS, 256, 256, 4, 2, 3, Epi>), grid, dim3(512), 0, stream, x, d, epi, s);
    else if (tile == 64)     hipLaunchKernelGGL((mxmix_kernel<FMT, X_IS_A, ACROSS, 64, 64, 2, 1, 4, Epi>), grid, dim3(128), 0, stream, x, d, epi, s);
    else if (s.k_tiles <= 2) hipLaunchKernelGGL((mxmix_kernel<FMT, X_IS_A, ACROSS, 128, 128, 2, 2, 2, Epi>), grid, dim3(256), 0, stream, x, d, epi, s);
    else                     hipLaunchKernelGGL((mxmix_kernel<FMT, X_IS_A, ACROSS, 128, 128, 4, 2, 3, Epi>), grid, dim3(512), 0, stream, x, d, epi, s);
}

template <int FMT, class Epi>
void launch_mix(bool x_is_a, bool across, int tile, const MxSide& x, const MxSide& d, const Epi& epi, const CoreShape& s, dim3 grid,
                hipStream_t stream)
{
    if constexpr (FMT == NG_MX_FP4) {
        if (x_is_a && across) return launch<FMT, true, true>(tile, x, d, epi, s, grid, stream);
    }
    if (x_is_a) launch<FMT, true, false>(tile, x, d, epi, s, grid, stream);
    else        launch<FMT, false, false>(tile, x, d, epi, s, grid, stream);
}

#define NG_MIX(FMT, EPI)                                                                                                   \
    template void launch_mix<FMT, EPI>(bool, bool, int, const MxSide&, const MxSide&, const EPI&, const CoreShape&, dim3, hipStream_t)
#ifndef NG_MX_MIX_FORMAT
#define NG_MX_MIX_FORMAT NG_MX_FP4
#endif
NG_MIX(NG_MX_MIX_FORMAT, MxStoreEpilogue<_Float16>);
NG_MIX(NG_MX_MIX_FORMAT, MxStoreEpilogue<float>);
NG_MIX(NG_MX_MIX_FORMAT, MxPartialEpilogue);
#undef NG_MIX

}  // namespace ng
