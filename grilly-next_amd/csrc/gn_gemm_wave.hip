// gn_gemm_wave.hip — bf16 products whose large tiles would leave most of the GPU idle: few
// tokens, or a few hundred over a narrow output.
//
// A block owns a BM x BN tile (32 or 64 each way) of C and splits K over its four waves: wave w
// takes the 64-deep k-tiles w, w + 4, ...  Each wave streams its own k-tiles by LDS DMA through
// a private ring of S stages and multiplies the whole tile, so the main loop has no barrier and
// the block keeps up to 144 KB of reads in flight; the four partial tiles are added in wave
// order through LDS at the end (fp32, deterministic).  What bounds it: the DMA of a few k-tiles and the
// latency ahead of them, the matrix cores being 1-4 % busy (37 x 5632 x 2048, 16 x 768 x 32000).
#include <algorithm>

#include "gn_gemm_wave_core.h"

namespace gn {
namespace {

template <bool TA, bool TB, typename CT, int BM, int BN, int EPI, int S>
int launch_wave(const GemmDesc& g, hipStream_t s) {
    using T = WaveTile<BM, BN, S>;
    static const bool ok = allow_lds(gemm_wave<TA, TB, CT, BM, BN, EPI, S>, T::SMEM);
    if (!ok) {
        set_error("gemm: cannot reserve %zu B of LDS", T::SMEM);
        return GN_E_HIP;
    }
    const int tiles = ((g.M + BM - 1) / BM) * ((g.N + BN - 1) / BN);
    hipLaunchKernelGGL((gemm_wave<TA, TB, CT, BM, BN, EPI, S>), dim3(tiles), dim3(256), T::SMEM, s, g);
    GN_LAUNCH_CHECK("gemm (wave-split)");
    return GN_OK;
}

template <bool TA, bool TB, typename CT, int EPI>
int launch_tile(const GemmDesc& g, int shape, hipStream_t s) {
    switch (shape) {
        case 0: return launch_wave<TA, TB, CT, 64, 64, EPI, 2>(g, s);
        case 1: return launch_wave<TA, TB, CT, 64, 32, EPI, 3>(g, s);
        case 2: return launch_wave<TA, TB, CT, 32, 64, EPI, 3>(g, s);
        default: return launch_wave<TA, TB, CT, 32, 32, EPI, 4>(g, s);
    }
}

template <typename CT>
int launch_plain(const GemmDesc& g, int ta, int tb, int shape, hipStream_t s) {
    if (!ta && !tb) return launch_tile<false, false, CT, 0>(g, shape, s);
    if (!ta && tb) return launch_tile<false, true, CT, 0>(g, shape, s);
    if (ta && !tb) return launch_tile<true, false, CT, 0>(g, shape, s);
    return launch_tile<true, true, CT, 0>(g, shape, s);
}

}  // namespace

// The tile that runs g fastest here, or -1 where the large tiles do.  Time model, fitted to
// MI355X sweeps of both over M from 1 to 4096 on the FFN and decoder products: a round of
// blocks (one per CU) takes a fixed time and one step per four k-tiles; the steps are bound by
// the LDS DMA (64 x 64: 64 KB in 0.7 us = 92 GB/s per CU), so a small tile pays where
// the large ones leave CUs idle: they move half the bytes per FLOP but take 0.3-0.55 us per k-tile
// on however few CUs.  The other side is the kernel that would run instead: bf16 C the streamed
// tiles (gemm_stream_us), fp32 C and the GLU epilogue the core's.
// Measured (us, replayed; streamed tiles -> here): 64 x 5632 x 2048 13.2 -> 7.8, 64 x 2048 x 5632
// 28.9 -> 10.3, 384 x 2048 x 5632 33.4 -> 20.0, 1003 x 768 x 6144 40.9 -> 24.6, an LM head's dX 16 x 768 x
// 32000 142 -> 61, 1003 rows 175 -> 98; the streamed tiles lead at 200 x 5632 x 2048 (13.7 against 17.1),
// 768 x 2048 x 5632 (34.4 / 36.5), 1536 x 768 x 6144 (38.5 / 39.3) and 2001 x 768 x 32000 (level alone, 279
// against 342 beside its weight gradient).  fp32 C, core -> here: dW 768 x 768 over 512 rows 8.6 -> 5.8,
// over 4096 23.7 -> 17.6.  Of 240 bf16 products in that sweep the lines drawn (0.95 of the streamed
// time, 0.85 of the core's) give each the faster kernel.
int gemm_wave_shape(const GemmDesc& g, int transA, int transB, int c_dtype) {
    const bool ta = transA != 0;
    const size_t c_bytes = g.epi == 1 || c_dtype != GN_F32 ? 2 : 4;
    double best;
    if (g.epi == 0 && c_bytes == 2) {
        best = 0.95 * gemm_stream_us(g);
    } else {
        const TileChoice tc = choose_tile(g, ta, c_bytes, g.epi);
        if (tc.m_first > 0) return -1;
        best = 0.85 * tile_cost(g, ta, c_bytes, g.epi, tc.shape, tc.ksplit, tc.ksplit > 2);
    }
    static constexpr int bm[4] = {64, 64, 32, 32}, bn[4] = {64, 32, 64, 32};
    static constexpr double fixed[4] = {3.2, 1.8, 1.8, 1.6}, step[4] = {0.70, 0.52, 0.52, 0.34};
    const int steps = (k_tiles(g) + 3) / 4;
    int shape = -1;
    for (int i = 0; i < 4; ++i) {
        const long blocks = (long)((g.M + bm[i] - 1) / bm[i]) * ((g.N + bn[i] - 1) / bn[i]);
        const double f = (double)(blocks % 256) / 256.0;
        const double rounds = (double)(blocks / 256) + (f > 0 ? 0.6 + 0.4 * f : 0.0);
        // transposed operands read their fragments in two halves, fp32 tiles store twice the bytes
        const double t = rounds * (fixed[i] * (c_bytes == 4 ? 1.4 : 1.0) + steps * step[i] * (ta ? 1.4 : 1.0));
        if (t < best) { best = t; shape = i; }
    }
    return shape;
}

int gemm_wave_launch(const GemmDesc& g, int shape, int transA, int transB, int c_dtype, hipStream_t s) {
    if (g.epi == 1) return launch_tile<false, false, bf16_t, 1>(g, shape, s);
    if (c_dtype == GN_F32) return launch_plain<float>(g, transA, transB, shape, s);
    return launch_plain<bf16_t>(g, transA, transB, shape, s);
}

}  // namespace gn
