// gn_gemm_stream.hip — bf16-output products (every operand orientation) and the fp32 weight gradients
// of several rounds on blocks that stay: one per CU, each walking its share of the tiles with the
// k-tiles of all of them as one stream.
//
// A block per tile (gn_gemm_dma_core.h) spends ~11 us on its DMA prologue, pipeline fill and
// fp32-staged epilogue around the 10 us that 12 k-tiles of a 256 x 128 tile need.  Here the four
// producer waves run on into the next tile's k-tiles while the four compute waves store the
// finished one, and the store goes out through 4 KB of LDS per wave, so that a tile costs
// its k-tiles and ~3 us.  What bounds it: at 12 k-tiles the store bursts and the k-tiles about
// equally, from ~32 k-tiles on the matrix cores (63-68 % busy over 4096 x 2048 x 11264 and dW 11264 x
// 2048 x 4096) and the LDS reads that feed them.
//   us, a block per tile -> here (A k-contiguous, B row-major [N][K]; in brackets B [K][N]):
//   8192 x 32000 x 768  689 -> 447 (668 -> 464)    8192 x 3072 x 768   63 -> 42
//   2001 x 32000 x 768  152 -> 99                  8192 x  768 x 768   19 -> 15 (16 -> 14)
//   4096 x 5632 x 2048  112 -> 89  (100 -> 87)     8192 x  768 x 6144  78 -> 68 (67 -> 66)
//   8192 x 8192 x 4096  515 -> 454                 4096 x  768 x 768   10 -> 9.5
// The main loop, the order of every output's sum and its roundings are those of the core: the
// results are the same bits.
#include <algorithm>

#include "gn_gemm_stream_core.h"

namespace gn {
namespace {

template <bool TA, bool TB, int BM, typename CT = bf16_t>
int launch(const GemmDesc& g, int blocks, hipStream_t s) {
    constexpr int BN = 128, STAGES = 3;
    constexpr size_t smem = (size_t)STAGES * (BM + BN) * BK * sizeof(bf16_t) + 4 * 4096;  // 160 KB at 256 rows
    static_assert(smem <= 160 * 1024, "LDS per CU");
    static const bool ok = allow_lds(gemm_stream<TA, TB, CT, BM, BN, STAGES>, smem);
    if (!ok) {
        set_error("gemm: cannot reserve %zu B of LDS", smem);
        return GN_E_HIP;
    }
    const long tiles = (long)((g.M + BM - 1) / BM) * ((g.N + BN - 1) / BN);
    // beside another product a block per tile: blocks that stay would keep the other's waiting
    // (dX 4096 x 5632 x 2048 beside dW 2048 x 5632 x 4096: 190 -> 180 us, 188 -> 173 replayed)
    const unsigned grid = (unsigned)(g.beside ? tiles : std::min<long>(tiles, blocks));
    hipLaunchKernelGGL((gemm_stream<TA, TB, CT, BM, BN, STAGES>), dim3(grid), dim3(512), smem, s, g);
    GN_LAUNCH_CHECK("gemm (streamed tiles)");
    return GN_OK;
}

// Tile rows for g, and the time the product then takes (us, bf16 C): rounds of 256 x 128 or
// 128 x 128 tiles, whichever need less.  A round of the small ones takes 0.6 of a round of the
// large: 4.2 us + 0.29 per k-tile against 6.5 + 0.52 (up to 0.4 and 0.6 where a round fills the
// chip).  Measured, 256 -> 128 rows: 4096 x 768 x 3072 (one round either way) 33 -> 24 us, 2048^3
// 24.5 -> 20.2; 8192 x 768 x 3072 (one round against two) 39 -> 48, 2816 x 2304 x 768 14 -> 16.
int choose_rows(const GemmDesc& g, int blocks, double* us) {
    const long tn = (g.N + 127) / 128;
    const long r256 = ((g.M + 255) / 256 * tn + blocks - 1) / blocks;
    const long r128 = ((g.M + 127) / 128 * tn + blocks - 1) / blocks;
    const bool small = 0.62 * (double)r128 < (double)r256;
    *us = small ? (double)r128 * (4.2 + 0.29 * k_tiles(g)) : (double)r256 * (6.5 + 0.52 * k_tiles(g));
    return small ? 128 : 256;
}

template <int BM>
int launch_tile(const GemmDesc& g, int transA, int transB, int blocks, hipStream_t s) {
    if (!transA && !transB) return launch<false, false, BM>(g, blocks, s);
    if (!transA && transB) return launch<false, true, BM>(g, blocks, s);
    if (transA && !transB) return launch<true, false, BM>(g, blocks, s);
    return launch<true, true, BM>(g, blocks, s);
}

}  // namespace

double gemm_stream_us(const GemmDesc& g) {
    double us;
    choose_rows(g, stream_blocks(), &us);
    return us;
}

int gemm_dma_bf16(const GemmDesc& g, int transA, int transB, hipStream_t s) {
    if (g.Msplit < g.M) {
        set_error("gemm: a bf16 product has one destination");
        return GN_E_INVALID;
    }
    const int blocks = stream_blocks();
    double us;
    return choose_rows(g, blocks, &us) == 128 ? launch_tile<128>(g, transA, transB, blocks, s)
                                              : launch_tile<256>(g, transA, transB, blocks, s);
}

// Up to 1024 rows of dY and X, where a dW tile is mostly its store: this one leaves as whole row
// segments, the core's, staged per wave, in half the speed (us, register-staged 128 x 128 tiles -> core
// -> here, M x N x K of dW): 2048 x 2048 x 8 8.1 -> 14.9 -> 8.2, x 200 11.0 -> 14.4 -> 9.2, x 1003
// 25 -> 20.0 -> 14.6; 5632 x 2048 x 200 21.2 -> 31.0 -> 16.7; 4096 x 4096 x 8 16.4 -> 33.2 -> 17.2.
constexpr int kShortK = 16;  // k-tiles

// Or more than two rounds of 256 x 128 tiles, alone on the GPU.  Measured (us, a block per tile -> here,
// M x N x K of dW): 11264 x 2048 x 4096 180 -> 172, x 2048 112 -> 91; 32000 x 768 x 2001 120 -> 95;
// 8192 x 8192 x 4096 555 -> 472; the least gain just above the line (10240 x 1792 x 4096, 560 tiles,
// 153 -> 149).  Beside another product (an LM head's dX, 48 tiles over K = 32000) the core's blocks go
// on sharing the GPU: with blocks that stay the pair's pass was 522 -> 532.
bool gemm_stream_f32_wins(const GemmDesc& g, int transA, int transB) {
    if (!transA || transB || g.bias || g.cbias) return false;
    const long tiles = (long)((g.M + 255) / 256) * ((g.N + 127) / 128);
    return k_tiles(g) <= kShortK || (!g.beside && tiles > 2L * stream_blocks());
}

// Over a round of such tiles the column sums' own launch (one, ~5 us, up to these 1024 rows) costs less
// than the core's store: backward with db of 200 x 5632 x 2048 (replayed) 42.7 with the register-staged
// tiles -> 53.4 on the core -> 41 here; of 200 x 2048 x 2048, 128 tiles, 23.0 with the core's fused sums,
// which stays.
bool gemm_stream_sums_apart(const GemmDesc& g) {
    const long tiles = (long)((g.M + 255) / 256) * ((g.N + 127) / 128);
    return k_tiles(g) <= kShortK && tiles > stream_blocks() && gemm_stream_f32_wins(g, 1, 0);
}

int gemm_stream_f32(const GemmDesc& g, hipStream_t s) {
    const int blocks = stream_blocks();
    double us;
    if (k_tiles(g) <= kShortK && choose_rows(g, blocks, &us) == 128) return launch<true, false, 128, float>(g, blocks, s);
    return launch<true, false, 256, float>(g, blocks, s);
}

}  // namespace gn
