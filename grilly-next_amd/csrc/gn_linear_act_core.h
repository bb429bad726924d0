// gn_linear_act_core.h — the epilogues of gn_linear_act.hip's products and their launches, instantiated in compilation units
// of their own: gn_linear_act_{bf16,f32,bwd}.hip.
#pragma once

#include <algorithm>
#include <type_traits>

#include "gn_act.h"
#include "gn_gemm_stream_core.h"
#include "gn_gemm_wave_core.h"

namespace gn {
namespace {

// ---- epilogues ---------------------------------------------------------------------------------
// Four elements of a row from its column n on (p: the first of them), of `cols` columns: in one access (VEC: the rows are multiples of four and the
// tensor 16-byte aligned), or singly, short of the last column.
template <typename T> struct Four;
template <> struct Four<float> {
    uint4 w;
    __device__ __forceinline__ void get(float (&v)[4]) const {
        v[0] = __uint_as_float(w.x); v[1] = __uint_as_float(w.y); v[2] = __uint_as_float(w.z); v[3] = __uint_as_float(w.w);
    }
};
template <> struct Four<bf16_t> {
    uint2 w;
    __device__ __forceinline__ void get(float (&v)[4]) const {
        v[0] = __uint_as_float(w.x << 16); v[1] = __uint_as_float(w.x & 0xffff0000u);
        v[2] = __uint_as_float(w.y << 16); v[3] = __uint_as_float(w.y & 0xffff0000u);
    }
};
template <bool VEC>
__device__ __forceinline__ Four<float> fetch4(const float* p, int n, int cols) {
    Four<float> r;
    if constexpr (VEC) {
        r.w = *reinterpret_cast<const uint4*>(p);
    } else {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = n + e < cols ? p[e] : 0.f;
        r.w = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
    return r;
}
template <bool VEC>
__device__ __forceinline__ Four<bf16_t> fetch4(const bf16_t* p, int n, int cols) {
    Four<bf16_t> r;
    if constexpr (VEC) {
        r.w = *reinterpret_cast<const uint2*>(p);
    } else {
        uint32_t v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = n + e < cols ? p[e] : 0;
        r.w = make_uint2(v[0] | (v[1] << 16), v[2] | (v[3] << 16));
    }
    return r;
}
template <bool VEC>
__device__ __forceinline__ void put4(float* p, int n, int cols, const float (&v)[4]) {
    if constexpr (VEC) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < cols) p[e] = v[e];
    }
}
template <bool VEC>
__device__ __forceinline__ void put4(bf16_t* p, int n, int cols, const float (&v)[4]) {
    const uint2 w = make_uint2(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]));
    if constexpr (VEC) {
        *reinterpret_cast<uint2*>(p) = w;
    } else {
        const uint32_t q[4] = {w.x & 0xffffu, w.x >> 16, w.y & 0xffffu, w.y >> 16};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < cols) p[e] = (bf16_t)q[e];
    }
}
// l elements behind p; where p is the wave's, the address needs no vector instruction.
template <typename T>
__device__ __forceinline__ T* at(T* p, uint32_t l) {
    using C = std::conditional_t<std::is_const_v<T>, const char, char>;
    return reinterpret_cast<T*>(reinterpret_cast<C*>(p) + l * (uint32_t)sizeof(T));
}

// A tile of a streamed product, 32 FM x 64 of a wave, through its 4 KB of LDS in blocks of 32 x 32: E::fetch() starts an
// epilogue's loads of four columns of a row, E::work() finishes them.  The loads are started some blocks ahead, into the
// registers of the next tile's fragments (kAgain): memory operations end in order, so a load behind the stores of
// the block before waits for those too.  A block's sums go into LDS before the block in front is worked on.  The activation is chosen
// once around the whole tile: chosen at every piece, the code is 200 KB and the tile waits 8 us for its
// instructions, against ~2 here.
template <typename E>
struct Tiles {
    static constexpr bool kAgain = true;
    E e;
    template <int FM>
    __device__ __forceinline__ void begin(const GemmDesc&, int, unsigned char*, int) const {}
    template <int FM, int FN>
    __device__ __forceinline__ void tile(const GemmDesc& g, const f32x16_t (&acc)[FM][FN], int m0, int n0, unsigned char* st,
                                         int lane) const {
        if (n0 >= e.N) return;
        asm volatile("" : "+v"(lane));  // opaque: addresses are formed here, not kept across the k loop
        const int mr = lane & 31, c8 = lane & 7, r8 = lane >> 3;
        constexpr int NB = FM * FN;
        by_act<E::kAct, E::kNone>(e.act, [&](auto ACT_) __attribute__((always_inline)) {
            constexpr int ACT = decltype(ACT_)::value;
            typename E::Col col[FN];
#pragma unroll
            for (int j = 0; j < FN; ++j) col[j] = e.column(min(n0 + 32 * j + 4 * c8, e.N - 1));
            constexpr int AHEAD = E::ahead(NB);  // blocks whose loads are under way
            typename E::Ext ext[AHEAD][4];
            const uint32_t lo = (uint32_t)(r8 * e.N + 4 * c8);
            const int last = E::kVec ? e.N - 4 : e.N - 1;
            // a block's first row, formed when it is needed: its addresses held over the others would not fit the registers
            auto row = [&](int b) __attribute__((always_inline)) {
                int m = m0 + 32 * (b / FN);
                asm volatile("" : "+s"(m));
                return m;
            };
            auto inside = [&](int b, int q, int mu) __attribute__((always_inline)) {
                return n0 + 32 * (b % FN) + 4 * c8 < e.N && mu + 8 * q + r8 < g.M;
            };
            // lanes past the edge read an element that is there: no branch between the rows
            auto load = [&](int b, typename E::Ext (&x)[4]) __attribute__((always_inline)) {
                const int n = min(n0 + 32 * (b % FN), last), mu = row(b);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const bool in = inside(b, q, mu);
                    x[q] = e.fetch((size_t)min(mu + 8 * q, g.M - 1) * e.N + n, in ? lo : 0u, in ? n + 4 * c8 : n);
                }
            };
            auto spread = [&](auto B_) __attribute__((always_inline)) {
                constexpr int i = decltype(B_)::value / FN, j = decltype(B_)::value % FN;
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<float4*>(st + mr * 128 + (((2 * q + (lane >> 5)) ^ (mr & 7)) * 16)) =
                        make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
            };
#pragma unroll
            for (int b = 0; b < AHEAD; ++b) load(b, ext[b]);
            wave_lds_sync();
            spread(std::integral_constant<int, 0>{});
            static_for<NB>([&](auto B_) __attribute__((always_inline)) {
                constexpr int b = decltype(B_)::value;
                wave_lds_sync();
                float v[4][4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float4 x = *reinterpret_cast<const float4*>(st + (8 * q + r8) * 128 + ((c8 ^ r8) * 16));
                    v[q][0] = x.x; v[q][1] = x.y; v[q][2] = x.z; v[q][3] = x.w;
                }
                wave_lds_sync();
                if constexpr (b + 1 < NB) spread(std::integral_constant<int, b + 1>{});
                const int n = n0 + 32 * (b % FN) + 4 * c8, mu = row(b);
                auto first = [&](int q) __attribute__((always_inline)) { return (size_t)(mu + 8 * q) * e.N + (n0 + 32 * (b % FN)); };
                // all rows are worked on, then stored: their chains run side by side
                if (e.keeps()) {
                    float pre[4][4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) e.template work<ACT>(v[q], ext[b % AHEAD][q], col[b % FN], pre[q]);
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (inside(b, q, mu)) e.keep(first(q), lo, n, pre[q]), e.store(first(q), lo, n, v[q]);
                } else {
                    float pre[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) e.template work<ACT>(v[q], ext[b % AHEAD][q], col[b % FN], pre);
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (inside(b, q, mu)) e.store(first(q), lo, n, v[q]);
                }
                if constexpr (b + AHEAD < NB) load(b + AHEAD, ext[b % AHEAD]);
            });
        });
    }
    // (gemm_wave's tiles)
    __device__ __forceinline__ void store8(int m, int n, float (&v)[8]) const {
        by_act<E::kAct, E::kNone>(e.act, [&](auto ACT_) __attribute__((always_inline)) {
            constexpr int ACT = decltype(ACT_)::value;
            const size_t u = (size_t)m * e.N;
            typename E::Ext x[2];
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (n + 4 * k < e.N) x[k] = e.fetch(u + n + 4 * k, 0u, n + 4 * k);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float w[4] = {v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]}, pre[4];
                if (n + 4 * k >= e.N) continue;
                e.template work<ACT>(w, x[k], e.column(n + 4 * k), pre);
                if (e.keeps()) e.keep(u + n + 4 * k, 0u, n + 4 * k, pre);
                e.store(u + n + 4 * k, 0u, n + 4 * k, w);
            }
        });
    }
};

// Y = R + act(v + b), P.  TY: of R and Y.
template <typename TY, bool VEC, int ACT_>
struct Forward {
    static constexpr bool kNone = true, kVec = VEC;
    static constexpr int kAct = ACT_;
    static constexpr int ahead(int) { return sizeof(TY) == 4 ? 2 : 4; }
    const bf16_t* b;
    const TY* R;
    TY* Y;
    bf16_t* P;
    int N, act;
    using Ext = Four<TY>;
    struct Col {
        float b[4];
    };
    __device__ __forceinline__ Col column(int n) const {
        Col c{};
        if (VEC) n &= ~3;
        if (b) fetch4<VEC>(b + n, n, N).get(c.b);
        return c;
    }
    __device__ __forceinline__ Ext fetch(size_t u, uint32_t l, int n) const { return R ? fetch4<VEC>(at(R + u, l), n, N) : Ext{}; }
    // v to Y, pre: what P holds
    template <int ACT>
    __device__ __forceinline__ void work(float (&v)[4], const Ext& x, const Col& c, float (&pre)[4]) const {
        float r[4] = {0.f, 0.f, 0.f, 0.f};
        if (R) x.get(r);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] += c.b[e];
            pre[e] = v[e];
            if constexpr (ACT != GN_ACT_NONE) v[e] = act_of<ACT>(v[e]);
            if constexpr (ACT == GN_ACT_TANH || ACT == GN_ACT_SIGMOID) pre[e] = v[e];
            v[e] += r[e];
        }
    }
    __device__ __forceinline__ bool keeps() const { return P != nullptr; }
    __device__ __forceinline__ void keep(size_t u, uint32_t l, int n, const float (&v)[4]) const { put4<VEC>(at(P + u, l), n, N, v); }
    __device__ __forceinline__ void store(size_t u, uint32_t l, int n, const float (&v)[4]) const { put4<VEC>(at(Y + u, l), n, N, v); }
};

// dP = v act'(P)
template <bool VEC, int ACT_>
struct Backward {
    static constexpr bool kNone = false, kVec = VEC;
    static constexpr int kAct = ACT_;
    static constexpr int ahead(int) { return 4; }
    const bf16_t* P;
    bf16_t* dP;
    int N, act;
    using Ext = Four<bf16_t>;
    struct Col {};
    __device__ __forceinline__ Col column(int) const { return Col{}; }
    __device__ __forceinline__ Ext fetch(size_t u, uint32_t l, int n) const { return fetch4<VEC>(at(P + u, l), n, N); }
    template <int ACT>
    __device__ __forceinline__ void work(float (&v)[4], const Ext& x, const Col&, float (&)[4]) const {
        float p[4];
        x.get(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= slope_of<ACT>(p[e]);
    }
    __device__ __forceinline__ bool keeps() const { return false; }
    __device__ __forceinline__ void keep(size_t, uint32_t, int, const float (&)[4]) const {}
    __device__ __forceinline__ void store(size_t u, uint32_t l, int n, const float (&v)[4]) const { put4<VEC>(at(dP + u, l), n, N, v); }
};

template <bool TB, int BM, typename E>
int launch_stream(const GemmDesc& g, const E& e, int blocks, hipStream_t s) {
    constexpr int BN = 128, STAGES = 3;
    constexpr size_t smem = (size_t)STAGES * (BM + BN) * BK * sizeof(bf16_t) + 4 * 4096;
    static_assert(smem <= 160 * 1024, "LDS per CU");
    static const bool ok = allow_lds(gemm_stream<false, TB, bf16_t, BM, BN, STAGES, Tiles<E>>, smem);
    if (!ok) {
        set_error("linear: cannot reserve %zu B of LDS", smem);
        return GN_E_HIP;
    }
    const long tiles = (long)((g.M + BM - 1) / BM) * ((g.N + BN - 1) / BN);
    const unsigned grid = (unsigned)(g.beside ? tiles : std::min<long>(tiles, blocks));
    hipLaunchKernelGGL((gemm_stream<false, TB, bf16_t, BM, BN, STAGES, Tiles<E>>), dim3(grid), dim3(512), smem, s, g, Tiles<E>{e});
    GN_LAUNCH_CHECK("linear (streamed tiles)");
    return GN_OK;
}

template <bool TB, int BM, int BN, int S, typename E>
int launch_wave(const GemmDesc& g, const E& e, hipStream_t s) {
    using T = WaveTile<BM, BN, S>;
    static const bool ok = allow_lds(gemm_wave<false, TB, bf16_t, BM, BN, 0, S, Tiles<E>>, T::SMEM);
    if (!ok) {
        set_error("linear: cannot reserve %zu B of LDS", T::SMEM);
        return GN_E_HIP;
    }
    const int tiles = ((g.M + BM - 1) / BM) * ((g.N + BN - 1) / BN);
    hipLaunchKernelGGL((gemm_wave<false, TB, bf16_t, BM, BN, 0, S, Tiles<E>>), dim3(tiles), dim3(256), T::SMEM, s, g, Tiles<E>{e});
    GN_LAUNCH_CHECK("linear (wave-split)");
    return GN_OK;
}

// The tiles are the plain product's (gemm_wave_shape, gemm_stream_rows): the choice leaves out the epilogue's own time, 16 to 18 us of
// a hundred at 4096 x 5632 x 2048, and other tiles were not timed with one.  The streamed tiles' kernels are an activation's each.
template <bool TB, typename E, typename F>
int launch(const GemmDesc& g, const E& any, F&& of_act, hipStream_t s) {
    switch (gemm_wave_shape(g, 0, TB, GN_BF16)) {
        case 0: return launch_wave<TB, 64, 64, 2>(g, any, s);
        case 1: return launch_wave<TB, 64, 32, 3>(g, any, s);
        case 2: return launch_wave<TB, 32, 64, 3>(g, any, s);
        case 3: return launch_wave<TB, 32, 32, 4>(g, any, s);
        default: break;
    }
    const int blocks = stream_blocks();
    auto go = [&](const auto& e) {
        return gemm_stream_rows(g) == 128 ? launch_stream<TB, 128>(g, e, blocks, s) : launch_stream<TB, 256>(g, e, blocks, s);
    };
    return of_act(go);
}

template <typename TY, bool VEC>
int forward(const GemmDesc& d, int act, const void* b, const void* R, void* Y, void* P, hipStream_t s) {
    auto make = [&](auto A) {
        return Forward<TY, VEC, decltype(A)::value>{(const bf16_t*)b, (const TY*)R, (TY*)Y, (bf16_t*)P, d.N, act};
    };
    using std::integral_constant;
    return launch<true>(d, make(integral_constant<int, kAny>{}), [&](auto&& go) {
        switch (act) {
            case GN_ACT_RELU: return go(make(integral_constant<int, GN_ACT_RELU>{}));
            case GN_ACT_GELU_TANH: return go(make(integral_constant<int, GN_ACT_GELU_TANH>{}));
            case GN_ACT_GELU_ERF: return go(make(integral_constant<int, GN_ACT_GELU_ERF>{}));
            case GN_ACT_SILU: return go(make(integral_constant<int, GN_ACT_SILU>{}));
            case GN_ACT_TANH: return go(make(integral_constant<int, GN_ACT_TANH>{}));
            case GN_ACT_SIGMOID: return go(make(integral_constant<int, GN_ACT_SIGMOID>{}));
            default: return go(make(integral_constant<int, GN_ACT_NONE>{}));
        }
    }, s);
}

}  // namespace
}  // namespace gn
