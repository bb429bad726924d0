// gn_gemm_wave_core.h — the kernel of products on small tiles with K split over a block's waves
// (gn_gemm_wave.hip says what for and how it works).  Kernel template with internal linkage; the finished
// tile is stored as C or handed, eight columns of a row at a time, to an epilogue object (gn_linear_act.hip).
#pragma once

#include "gn_gemm_dma_core.h"

namespace gn {
namespace {

template <int N>
__device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

template <int BM, int BN, int S>
struct WaveTile {
    static constexpr int A_E = BM * BK, STAGE = (BM + BN) * BK * 2, RING = S * STAGE;
    static constexpr int NA = BM / 8, NB = BN / 8, ND = NA + NB;  // DMA instructions of a k-tile
    static constexpr int PITCH = BN + 4;
    static constexpr size_t SMEM = (size_t)4 * RING;
    static_assert(SMEM <= 160 * 1024 && (size_t)BM * (PITCH + 1) * 4 <= RING, "LDS per CU");
    static_assert((S - 1) * ND < 64, "vmcnt range");
};

// BIAS: row sums of op(A) (a weight gradient's db), from an MFMA of A against ones in the blocks
// of the first column tile.  EPIL: none, or one object whose store8() takes the sums of columns n .. n + 7 of
// row m (n below g.N).
template <bool TA, bool TB, typename CT, int BM, int BN, int EPI, int S, typename... EPIL>
__global__ __launch_bounds__(256, 1) void gemm_wave(GemmDesc g, EPIL... epil) {
    using T = WaveTile<BM, BN, S>;
    constexpr int FM = BM / 32, FN = BN / 32;
    constexpr bool BIAS = EPI == 0 && TA && !TB && sizeof(CT) == 4 && sizeof...(EPIL) == 0;
    extern __shared__ __align__(16) unsigned char smem_raw[];

    const int tilesM = (g.M + BM - 1) / BM, tilesN = (g.N + BN - 1) / BN;
    const int nblk = tilesM * tilesN;
    // one contiguous range of tiles per XCD (its L2 then holds the ranges' operands), walked
    // eight tile rows at a time
    const int xcd = blockIdx.x & 7, per = nblk >> 3, extra = nblk & 7;
    const int pid = xcd * per + min(xcd, extra) + ((int)blockIdx.x >> 3);
    constexpr int GROUP = 8;
    const int group_id = pid / (GROUP * tilesN);
    const int first_m = group_id * GROUP;
    const int gsize = min(tilesM - first_m, GROUP);
    const int in_group = pid % (GROUP * tilesN);
    const int m0 = (first_m + in_group % gsize) * BM, n0 = (in_group / gsize) * BN;

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // wave-uniform
    unsigned char* ring = smem_raw + wave * T::RING;
    const uint32_t ring_a = lds_addr(ring);

    const int kt0 = (g.Ks[0] + BK - 1) / BK;
    const int KT = kt0 + (g.nseg > 1 ? (g.Ks[1] + BK - 1) / BK : 0);
    const int nt = (KT - wave + 3) >> 2;  // this wave's k-tiles: wave + 4 i, i < nt

    uint32_t voa[T::NA], vob[T::NB];
    int oseg = -1;
    auto dma = [&](int i) {
        const int t = wave + 4 * i;
        const int sg = t >= kt0 ? 1 : 0;
        const int k0 = (sg ? t - kt0 : t) * BK, klim = g.Ks[sg];
        const bf16_t* A = g.A[sg];
        const bf16_t* B = g.B[sg];
        const int lda = g.lda[sg], ldb = g.ldb[sg];
        const uint32_t base = ring_a + (uint32_t)(i % S) * T::STAGE;
        if (k0 + BK > klim) {
            stage_tail<BM, !TA, 1>(A, lda, m0, g.M, k0, klim, 0, base);
            stage_tail<BN, TB, 1>(B, ldb, n0, g.N, k0, klim, 0, base + T::A_E * 2);
            return;
        }
        if (oseg != sg) {
            oseg = sg;
            stage_offsets<BM, !TA, 1>(lda, m0, g.M, 0, voa);
            stage_offsets<BN, TB, 1>(ldb, n0, g.N, 0, vob);
        }
        const bf16_t* sa = stage_base<!TA>(A, lda, m0, k0);
        const bf16_t* sb = stage_base<TB>(B, ldb, n0, k0);
#pragma unroll
        for (int q = 0; q < T::NA; ++q) dma16s(sa, voa[q], base + 1024u * q);
#pragma unroll
        for (int q = 0; q < T::NB; ++q) dma16s(sb, vob[q], base + T::A_E * 2 + 1024u * q);
    };

    f32x16_t acc[FM][FN], rows[BIAS ? FM : 1];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) zero16(acc[i][j]);
#pragma unroll
    for (int i = 0; i < (BIAS ? FM : 1); ++i) zero16(rows[i]);
    const bool sums = BIAS && g.bias && n0 == 0;

    for (int i = 0; i < min(S, nt); ++i) dma(i);
    for (int i = 0; i < nt; ++i) {
        // tile i has landed; the younger tiles of the ring may still be in flight
        const int younger = min(nt - 1 - i, S - 1);
        if (younger >= 3 && S > 3) wait_vm<(S > 3 ? 3 : 0) * T::ND>();
        else if (younger == 2 && S > 2) wait_vm<(S > 2 ? 2 : 0) * T::ND>();
        else if (younger == 1) wait_vm<T::ND>();
        else wait_vm<0>();
        const bf16_t* sa = reinterpret_cast<const bf16_t*>(ring + (i % S) * T::STAGE);
        const bf16_t* sb = sa + T::A_E;
        bf16x8_t fa[4][FM], fb[4][FN];
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
#pragma unroll
            for (int a = 0; a < FM; ++a) fa[ks][a] = frag<BM, !TA>(sa, a * 32, ks);
#pragma unroll
            for (int b = 0; b < FN; ++b) fb[ks][b] = frag<BN, TB>(sb, b * 32, ks);
        }
        // every read of the stage has returned before its refill is issued
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        if (i + S < nt) dma(i + S);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int a = 0; a < FM; ++a)
#pragma unroll
                for (int b = 0; b < FN; ++b) acc[a][b] = mfma32(fa[ks][a], fb[ks][b], acc[a][b]);
        if constexpr (BIAS) {
            if (sums) {
                bf16x8_t one;
#pragma unroll
                for (int e = 0; e < 8; ++e) one[e] = (__bf16)1.0f;
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                    for (int a = 0; a < FM; ++a) rows[a] = mfma32(fa[ks][a], one, rows[a]);
            }
        }
    }

    // partial tiles into the waves' own rings (every DMA has landed), then summed by the block
    float* st = reinterpret_cast<float*>(ring);
    const int rq = (lane >> 5) * 4;
#pragma unroll
    for (int a = 0; a < FM; ++a)
#pragma unroll
        for (int b = 0; b < FN; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                st[(a * 32 + 8 * (r >> 2) + rq + (r & 3)) * T::PITCH + b * 32 + (lane & 31)] = acc[a][b][r];
    if constexpr (BIAS) {
        if (sums && (lane & 31) == 0) {
#pragma unroll
            for (int a = 0; a < FM; ++a)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    st[BM * T::PITCH + a * 32 + 8 * (r >> 2) + rq + (r & 3)] = rows[a][r];
        }
    }
    __syncthreads();
    const float* p0 = reinterpret_cast<const float*>(smem_raw);
    constexpr int CPR = BN / 8, WS = T::RING / 4;
#pragma unroll
    for (int c = threadIdx.x; c < BM * CPR; c += 256) {
        const int r = c / CPR, col = (c % CPR) * 8;
        const int m = m0 + r, n = n0 + col;
        const float* p = p0 + r * T::PITCH + col;
        float v[8];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float4 lo = *reinterpret_cast<const float4*>(p + w * WS);
            const float4 hi = *reinterpret_cast<const float4*>(p + w * WS + 4);
            const float u[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = w == 0 ? u[e] : v[e] + u[e];
        }
        if (m < g.M && n < g.N) {
            if constexpr (sizeof...(EPIL) > 0) (epil.store8(m, n, v), ...);
            else store8<CT, EPI>(g, m, n, v);
        }
    }
    if constexpr (BIAS) {
        const int m = m0 + threadIdx.x;
        if (sums && threadIdx.x < BM && m < g.M) {
            const float* p = p0 + BM * T::PITCH + threadIdx.x;
            const float v = ((p[0] + p[WS]) + p[2 * WS]) + p[3 * WS];
            float* dst = m < g.Msplit ? g.bias + m : g.bias2 + (m - g.Msplit);
            *dst = g.accumulate ? *dst + v : v;
        }
    }
}

}  // namespace
}  // namespace gn
