// gn_linear_act.hip — a Linear's forward with bias, activation and residual in the product's epilogue, and
// the backward of a Linear behind an activation, whose input-gradient product leaves the gradient in front of it.
//
//   forward    v = X W^T + b,  Y = R + act(v),  P = v (tanh, sigmoid: act(v))
//   backward   dP = (dY W) act'(P),  dW = dY^T A,  db = column sums of dY
//
// bf16 products run on the streamed tiles (gn_gemm_stream_core.h) or, where those would leave compute units
// idle, on the small ones (gn_gemm_wave_core.h), with the epilogues below: the sums stay in fp32 until Y, P or dP
// is rounded once.  A streamed tile goes through 4 KB of LDS a wave, 16 rows of 64 columns at a time, so that P, R
// and Y move as whole 128-byte row segments; the residual's and P's loads of the next 16 rows are under way
// meanwhile.  Sizes and addresses that the products' 16-byte pieces do not take are laid out first in the
// workspace.  fp32 products are gn_linear_fwd's and gn_gemm's, with a pass behind them where there is an
// activation or a residual.
#include <algorithm>

#include "gn_gemm_stream_core.h"
#include "gn_gemm_wave_core.h"

namespace gn {
namespace {

inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// ---- activations of eight values ---------------------------------------------------------------
// With the hardware's reciprocal (1 ulp), not the correctly rounded division of six more instructions.
__device__ __forceinline__ float rcp(float x) { return __builtin_amdgcn_rcpf(x); }
__device__ __forceinline__ float exp_neg(float x) { return __builtin_amdgcn_exp2f(x * -1.4426950408889634f); }
// 1 + tanh(z) = 2 sigmoid(2 z)
__device__ __forceinline__ float gelu_gate(float x) {
    return rcp(1.0f + exp_neg(x * (2.0f * kSqrt2OverPi) * (1.0f + kGeluC * x * x)));
}

template <int KIND>
__device__ __forceinline__ float act_of(float x) {
    if constexpr (KIND == GN_ACT_RELU) return x > 0.f ? x : 0.f;
    else if constexpr (KIND == GN_ACT_GELU_TANH) return x * gelu_gate(x);
    else if constexpr (KIND == GN_ACT_GELU_ERF) return 0.5f * x * (1.0f + erff(x * 0.70710678118654752f));
    else if constexpr (KIND == GN_ACT_SILU) return x * rcp(1.0f + exp_neg(x));
    else if constexpr (KIND == GN_ACT_TANH) return 1.0f - 2.0f * rcp(1.0f + exp_neg(-2.0f * x));
    else return rcp(1.0f + exp_neg(x));
}
// tanh and sigmoid at their output
template <int KIND>
__device__ __forceinline__ float slope_of(float x) {
    if constexpr (KIND == GN_ACT_GELU_TANH) {
        const float s = gelu_gate(x);
        return s + x * s * (1.0f - s) * (2.0f * kSqrt2OverPi) * (1.0f + 3.0f * kGeluC * x * x);
    } else if constexpr (KIND == GN_ACT_SILU) {
        const float s = rcp(1.0f + exp_neg(x));
        return s + x * s * (1.0f - s);
    } else {
        return act_grad<KIND>(x);
    }
}

template <int KIND>
__device__ __forceinline__ void act8(float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = act_of<KIND>(v[e]);
}
__device__ __forceinline__ void act8(int kind, float (&v)[8]) {
    switch (kind) {
        case GN_ACT_RELU: act8<GN_ACT_RELU>(v); break;
        case GN_ACT_GELU_TANH: act8<GN_ACT_GELU_TANH>(v); break;
        case GN_ACT_GELU_ERF: act8<GN_ACT_GELU_ERF>(v); break;
        case GN_ACT_SILU: act8<GN_ACT_SILU>(v); break;
        case GN_ACT_TANH: act8<GN_ACT_TANH>(v); break;
        case GN_ACT_SIGMOID: act8<GN_ACT_SIGMOID>(v); break;
        default: break;
    }
}
template <int KIND>
__device__ __forceinline__ void slope8(float (&v)[8], const float (&p)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= slope_of<KIND>(p[e]);
}
__device__ __forceinline__ void slope8(int kind, float (&v)[8], const float (&p)[8]) {
    switch (kind) {
        case GN_ACT_RELU: slope8<GN_ACT_RELU>(v, p); break;
        case GN_ACT_GELU_TANH: slope8<GN_ACT_GELU_TANH>(v, p); break;
        case GN_ACT_GELU_ERF: slope8<GN_ACT_GELU_ERF>(v, p); break;
        case GN_ACT_SILU: slope8<GN_ACT_SILU>(v, p); break;
        case GN_ACT_TANH: slope8<GN_ACT_TANH>(v, p); break;
        default: slope8<GN_ACT_SIGMOID>(v, p); break;
    }
}

// ---- epilogues ---------------------------------------------------------------------------------
// Eight elements of a row from column n on, of a matrix of `cols` columns in T: in 16-byte pieces, or (odd
// widths and addresses) singly, short of the last column.
struct Piece {
    uint4 a, b;  // b: of fp32
};
__device__ __forceinline__ void unpack(const Piece& p, bool f32, float (&v)[8]) {
    const uint32_t w[4] = {p.a.x, p.a.y, p.a.z, p.a.w}, u[4] = {p.b.x, p.b.y, p.b.z, p.b.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (f32) {
            v[e] = __uint_as_float(w[e]);
            v[4 + e] = __uint_as_float(u[e]);
        } else {
            v[2 * e] = __uint_as_float(w[e] << 16);
            v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        }
    }
}
__device__ __forceinline__ Piece fetch(const void* p, bool f32, size_t row, int n, int cols, bool vec) {
    Piece r{};
    if (vec) {
        const char* at = (const char*)p + (row + n) * (f32 ? 4 : 2);
        r.a = *reinterpret_cast<const uint4*>(at);
        if (f32) r.b = *reinterpret_cast<const uint4*>(at + 16);
    } else {
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            w[e] = 0;
            if (n + e < cols) w[e] = f32 ? ((const uint32_t*)p)[row + n + e] : ((const uint16_t*)p)[row + n + e];
        }
        if (f32) {
            r.a = make_uint4(w[0], w[1], w[2], w[3]);
            r.b = make_uint4(w[4], w[5], w[6], w[7]);
        } else {
            r.a = make_uint4(w[0] | (w[1] << 16), w[2] | (w[3] << 16), w[4] | (w[5] << 16), w[6] | (w[7] << 16));
        }
    }
    return r;
}
__device__ __forceinline__ void put(void* p, bool f32, size_t row, int n, int cols, bool vec, const float (&v)[8]) {
    if (vec) {
        if (f32) chunk8<float>::st((float*)p + row + n, v);
        else chunk8<bf16_t>::st((bf16_t*)p + row + n, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (n + e < cols) {
                if (f32) ((float*)p)[row + n + e] = v[e];
                else ((bf16_t*)p)[row + n + e] = f2bf(v[e]);
            }
    }
}

// A tile of a streamed product, 32 FM x 64 of a wave, through its 4 KB of LDS: E::fetch() starts an epilogue's
// loads of eight columns of a row, E::done() finishes them.
template <typename E>
struct Tiles {
    static constexpr bool kAgain = true;
    E e;
    template <int FM>
    __device__ __forceinline__ void begin(const GemmDesc&, int, unsigned char*, int) const {}
    template <int FM, int FN>
    __device__ __forceinline__ void tile(const GemmDesc& g, const f32x16_t (&acc)[FM][FN], int m0, int n0, unsigned char* st,
                                         int lane) const {
        static_assert(FN == 2, "64 columns a wave");
        if (n0 >= g.N) return;
        asm volatile("" : "+v"(lane));  // opaque: addresses are formed here, not kept across the k loop
        const int mr = lane & 31, c = lane & 7, r8 = lane >> 3, n = n0 + 8 * c;
        const bool nok = n < g.N;
        typename E::Col col = e.column(n, nok);
        typename E::Ext ext[2][2];
        auto load = [&](int h, typename E::Ext (&x)[2]) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int m = m0 + 16 * h + 8 * q + r8;
                if (nok && m < g.M) x[q] = e.fetch(m, n);
            }
        };
        load(0, ext[0]);
        static_for<2 * FM>([&](auto H_) {
            constexpr int h = decltype(H_)::value, i = h / 2;
            if constexpr (h + 1 < 2 * FM) load(h + 1, ext[(h + 1) & 1]);
            wave_lds_sync();
            if ((mr >> 4) == (h & 1))
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int at = 8 * j + 2 * q + (lane >> 5);  // 16-byte chunk of the row's 16
                        *reinterpret_cast<float4*>(st + (mr & 15) * 256 + ((at ^ (mr & 15)) * 16)) =
                            make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
                    }
            wave_lds_sync();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int r = 8 * q + r8, m = m0 + 16 * h + r;
                const float4 lo = *reinterpret_cast<const float4*>(st + r * 256 + (((2 * c) ^ r) * 16));
                const float4 hi = *reinterpret_cast<const float4*>(st + r * 256 + (((2 * c + 1) ^ r) * 16));
                float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
                if (nok && m < g.M) e.done(m, n, v, ext[h & 1][q], col);
            }
        });
    }
    __device__ __forceinline__ void store8(int m, int n, float (&v)[8]) const { e.done(m, n, v, e.fetch(m, n), e.column(n, true)); }
};

// Y = R + act(v + b), P
struct Forward {
    const bf16_t* b;
    const void* R;
    void* Y;
    bf16_t* P;
    int N, act;
    bool y32, vec, out_is_pre;  // out_is_pre: P holds the activation's output (tanh, sigmoid)
    using Ext = Piece;
    struct Col {
        float b[8];
    };
    __device__ __forceinline__ Col column(int n, bool ok) const {
        Col c{};
        if (b && ok) unpack(gn::fetch(b, false, 0, n, N, vec), false, c.b);
        return c;
    }
    __device__ __forceinline__ Ext fetch(int m, int n) const { return R ? gn::fetch(R, y32, (size_t)m * N, n, N, vec) : Ext{}; }
    __device__ __forceinline__ void done(int m, int n, float (&v)[8], const Ext& x, const Col& c) const {
        const size_t row = (size_t)m * N;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += c.b[e];
        if (P && !out_is_pre) put(P, false, row, n, N, vec, v);
        act8(act, v);
        if (P && out_is_pre) put(P, false, row, n, N, vec, v);
        if (R) {
            float r[8];
            unpack(x, y32, r);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += r[e];
        }
        put(Y, y32, row, n, N, vec, v);
    }
};

// dP = v act'(P)
struct Backward {
    const bf16_t* P;
    bf16_t* dP;
    int N, act;
    bool vec;
    using Ext = Piece;
    struct Col {};
    __device__ __forceinline__ Col column(int, bool) const { return Col{}; }
    __device__ __forceinline__ Ext fetch(int m, int n) const { return gn::fetch(P, false, (size_t)m * N, n, N, vec); }
    __device__ __forceinline__ void done(int m, int n, float (&v)[8], const Ext& x, const Col&) const {
        float p[8];
        unpack(x, false, p);
        slope8(act, v, p);
        put(dP, false, (size_t)m * N, n, N, vec, v);
    }
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

// The tiles are the plain product's (gemm_wave_shape, gemm_stream_rows), whose time the epilogues change little.
template <bool TB, typename E>
int launch(const GemmDesc& g, const E& e, hipStream_t s) {
    switch (gemm_wave_shape(g, 0, TB, GN_BF16)) {
        case 0: return launch_wave<TB, 64, 64, 2>(g, e, s);
        case 1: return launch_wave<TB, 64, 32, 3>(g, e, s);
        case 2: return launch_wave<TB, 32, 64, 3>(g, e, s);
        case 3: return launch_wave<TB, 32, 32, 4>(g, e, s);
        default: break;
    }
    const int blocks = stream_blocks();
    return gemm_stream_rows(g) == 128 ? launch_stream<TB, 128>(g, e, blocks, s) : launch_stream<TB, 256>(g, e, blocks, s);
}

// ---- passes ------------------------------------------------------------------------------------
// The epilogue of fp32 products, in place: v (fp32, or nullptr: a product of no terms, v = b) -> P, Y.  TR: R and Y.
template <typename TR, typename TB>
__global__ __launch_bounds__(256) void finish_forward(const float* v, const TB* b, const TR* R, TR* Y, TB* P, int64_t n, int N,
                                                      int act, bool out_is_pre) {
    for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float x = (v ? v[i] : 0.f) + (b ? io<TB>::ld(b, i % N) : 0.f);
        if (P && !out_is_pre) io<TB>::st(P, i, x);
        float t[8] = {x, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        act8(act, t);
        x = t[0];
        if (P && out_is_pre) io<TB>::st(P, i, x);
        io<TR>::st(Y, i, R ? x + io<TR>::ld(R, i) : x);
    }
}
// dP *= act'(P), fp32
__global__ __launch_bounds__(256) void finish_backward(float* dP, const float* P, int64_t n, int act) {
    for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float t[8] = {dP[i], 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, p[8] = {P[i], 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        slope8(act, t, p);
        dP[i] = t[0];
    }
}

// dst [Rp x dp] = src [R x d], zeros around it
__global__ __launch_bounds__(256) void lay_out(const bf16_t* __restrict__ src, bf16_t* __restrict__ dst, int R, int d, int Rp, int dp) {
    const int64_t n = (int64_t)Rp * dp;
    for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int r = (int)(i / dp), c = (int)(i - (int64_t)r * dp);
        dst[i] = r < R && c < d ? src[(size_t)r * d + c] : (bf16_t)0;
    }
}
int copy(const void* src, void* dst, int R, int d, int Rp, int dp, hipStream_t s) {
    lay_out<<<grid_for((int64_t)Rp * dp, 1024, 16384), 256, 0, s>>>((const bf16_t*)src, (bf16_t*)dst, R, d, Rp, dp);
    GN_LAUNCH_CHECK("linear (layout)");
    return GN_OK;
}

inline int up8(int n) { return (n + 7) / 8 * 8; }
inline size_t up16(size_t n) { return (n + 15) / 16 * 16; }

// The operands of a bf16 product laid out: of the forward X [M x K'], W [N x K'], of the backward dY [M x N'],
// W [N' x K'].
size_t layout_bytes(int M, int N, int K, bool backward) {
    if (backward) return up16((size_t)M * up8(N) * 2) + up16((size_t)up8(N) * up8(K) * 2);
    return up16((size_t)M * up8(K) * 2) + up16((size_t)N * up8(K) * 2);
}

// ---- checks ------------------------------------------------------------------------------------
struct Span {
    const void* p;
    size_t bytes;
    const char* name;
    bool written;
};
bool share(const Span& a, const Span& b) {
    return a.p && b.p && (const char*)a.p < (const char*)b.p + b.bytes && (const char*)b.p < (const char*)a.p + a.bytes;
}
// What is written shares no memory with anything else of the call; but the first tensor may be the second, as
// a whole.
template <int N>
int check_spans(const char* who, const Span (&t)[N]) {
    for (int i = 0; i < N; ++i)
        for (int j = 0; j < N && t[i].written; ++j)
            GN_REQUIRE(i == j || !share(t[i], t[j]) || (i == 0 && j == 1 && t[0].p == t[1].p), "%s: %s and %s may not share memory",
                       who, t[i].name, t[j].name);
    return GN_OK;
}

bool sizes_fit(int M, int N, int K) {
    return M < (1 << 28) && N < (1 << 28) && K < (1 << 28) && (int64_t)M * std::max(N, K) < (1ll << 36) && (int64_t)N * K < (1ll << 36);
}
int check_sizes(const char* who, int M, int N, int K, int dtype) {
    GN_REQUIRE(M >= 0 && N >= 0 && K >= 0, "%s: negative size", who);
    GN_REQUIRE(dtype == GN_F32 || dtype == GN_BF16, "%s: dtype %d not supported (f32, bf16)", who, dtype);
    GN_REQUIRE(sizes_fit(M, N, K), "%s: M, N and K below 2^28, M * N, M * K and N * K below 2^36", who);
    return GN_OK;
}
int check_ws(const char* who, const void* ws, size_t ws_bytes, size_t need) {
    if (!ws || ws_bytes < need || !al16(ws)) {
        set_error("%s: workspace of %zu bytes (16-byte aligned) required", who, need);
        return GN_E_WORKSPACE;
    }
    return GN_OK;
}

}  // namespace
}  // namespace gn

using namespace gn;

extern "C" size_t gn_linear_act_workspace_bytes(int M, int N, int K, int dtype) {
    if (M <= 0 || N <= 0 || K <= 0 || dtype != GN_BF16 || !sizes_fit(M, N, K)) return 0;
    return std::max(layout_bytes(M, N, K, false), layout_bytes(M, N, K, true));
}

extern "C" int gn_linear_act_fwd(int act, const void* X, const void* W, const void* b, const void* R, void* P, void* Y, int M,
                                 int N, int K, int dtype, int y_dtype, void* ws, size_t ws_bytes, void* stream) {
    clear_error();
    const char* const who = "gn_linear_act_fwd";
    if (const int rc = check_sizes(who, M, N, K, dtype)) return rc;
    GN_REQUIRE(act >= GN_ACT_NONE && act <= GN_ACT_SIGMOID, "%s: activation %d", who, act);
    GN_REQUIRE(y_dtype == dtype || (dtype == GN_BF16 && y_dtype == GN_F32), "%s: y dtype %d under dtype %d", who, y_dtype, dtype);
    if (M == 0 || N == 0) return GN_OK;
    GN_REQUIRE(Y && (K == 0 || (X && W)), "%s: null pointer", who);
    const size_t es = dtype == GN_F32 ? 4 : 2, ys = y_dtype == GN_F32 ? 4 : 2, n = (size_t)M * N;
    GN_REQUIRE((((uintptr_t)X | (uintptr_t)W | (uintptr_t)b | (uintptr_t)P) & (es - 1)) == 0 &&
                   (((uintptr_t)R | (uintptr_t)Y) & (ys - 1)) == 0, "%s: a tensor is not aligned to its elements", who);
    const bool lay = dtype == GN_BF16 && K > 0 && (K % 8 || !al16(X) || !al16(W));
    const size_t need = lay ? layout_bytes(M, N, K, false) : 0;
    const Span spans[] = {{Y, n * ys, "Y", true}, {R, n * ys, "R", false}, {P, n * es, "P", true},
                          {X, (size_t)M * K * es, "X", false}, {W, (size_t)N * K * es, "W", false},
                          {b, (size_t)N * es, "b", false}, {need ? ws : nullptr, need, "ws", true}};
    if (const int rc = check_spans(who, spans)) return rc;
    hipStream_t s = as_stream(stream);
    const bool out_is_pre = act == GN_ACT_TANH || act == GN_ACT_SIGMOID;
    const unsigned grid = grid_for((int64_t)n, 1024, 16384);
    if (K == 0) {  // no terms
        if (dtype == GN_F32)
            finish_forward<float, float><<<grid, 256, 0, s>>>(nullptr, (const float*)b, (const float*)R, (float*)Y, (float*)P, n, N, act, out_is_pre);
        else if (y_dtype == GN_F32)
            finish_forward<float, bf16_t><<<grid, 256, 0, s>>>(nullptr, (const bf16_t*)b, (const float*)R, (float*)Y, (bf16_t*)P, n, N, act, out_is_pre);
        else
            finish_forward<bf16_t, bf16_t><<<grid, 256, 0, s>>>(nullptr, (const bf16_t*)b, (const bf16_t*)R, (bf16_t*)Y, (bf16_t*)P, n, N, act, out_is_pre);
        GN_LAUNCH_CHECK(who);
        return GN_OK;
    }
    if (dtype == GN_F32) {
        // the product goes where it disturbs nothing: P, or Y unless that is the residual
        GN_REQUIRE(P || !R || Y != R, "%s: an fp32 Y may be the residual only with P", who);
        float* const v = (float*)(P ? P : Y);
        if (const int rc = gn_linear_fwd(X, W, b, v, M, N, K, dtype, stream)) return rc;
        if (P || R || act != GN_ACT_NONE) {
            finish_forward<float, float><<<grid, 256, 0, s>>>(v, nullptr, (const float*)R, (float*)Y, (float*)P, n, N, act, out_is_pre);
            GN_LAUNCH_CHECK(who);
        }
        return GN_OK;
    }
    if (lay) {
        if (const int rc = check_ws(who, ws, ws_bytes, need)) return rc;
        const int Kp = up8(K);
        char* const w = (char*)ws + up16((size_t)M * Kp * 2);
        if (const int rc = copy(X, ws, M, K, M, Kp, s)) return rc;
        if (const int rc = copy(W, w, N, K, N, Kp, s)) return rc;
        X = ws;
        W = w;
        K = Kp;
    }
    GemmDesc d{};
    d.nseg = 1;
    d.A[0] = (const bf16_t*)X; d.lda[0] = K; d.Ks[0] = K;
    d.B[0] = (const bf16_t*)W; d.ldb[0] = K;
    d.M = M; d.N = N; d.Msplit = M; d.ldc = N;
    Forward f{};
    f.b = (const bf16_t*)b;
    f.R = R;
    f.Y = Y;
    f.P = (bf16_t*)P;
    f.N = N;
    f.act = act;
    f.y32 = y_dtype == GN_F32;
    f.vec = N % 8 == 0 && al16(b) && al16(R) && al16(Y) && al16(P);
    f.out_is_pre = out_is_pre;
    return launch<true>(d, f, s);
}

extern "C" int gn_act_linear_bwd(int act, const void* dY, const void* P, const void* A, const void* W, void* dP, void* dW,
                                 void* db, int M, int N, int K, int dtype, unsigned flags, void* ws, size_t ws_bytes,
                                 void* stream) {
    clear_error();
    const char* const who = "gn_act_linear_bwd";
    if (const int rc = check_sizes(who, M, N, K, dtype)) return rc;
    GN_REQUIRE(act >= GN_ACT_RELU && act <= GN_ACT_SIGMOID, "%s: activation %d", who, act);
    GN_REQUIRE(dW || !db, "%s: db without dW", who);
    const size_t es = dtype == GN_F32 ? 4 : 2, m = (size_t)M, n = (size_t)N, k = (size_t)K;
    if (M > 0 && N > 0 && K > 0) GN_REQUIRE(dY && W && (!dP || P) && (!dW || A), "%s: null pointer", who);
    GN_REQUIRE((((uintptr_t)dY | (uintptr_t)P | (uintptr_t)A | (uintptr_t)W | (uintptr_t)dP) & (es - 1)) == 0 &&
                   (((uintptr_t)dW | (uintptr_t)db) & 3) == 0, "%s: a tensor is not aligned to its elements", who);
    const bool lay = dtype == GN_BF16 && dP && (N % 8 || K % 8 || !al16(dY) || !al16(W));
    const size_t need = lay ? layout_bytes(M, N, K, true) : 0;
    const Span spans[] = {{dP, m * k * es, "dP", true}, {P, m * k * es, "P", false}, {dW, n * k * 4, "dW", true}, {db, n * 4, "db", true},
                          {dY, m * n * es, "dY", false}, {A, m * k * es, "A", false}, {W, n * k * es, "W", false},
                          {ws, ws_bytes, "ws", true}};
    if (const int rc = check_spans(who, spans)) return rc;
    GN_REQUIRE(dtype == GN_BF16 || !dP || dP != P, "%s: an fp32 dP may not be P, which is read behind its product", who);
    hipStream_t s = as_stream(stream);
    if (M == 0 || N == 0 || K == 0) {  // dP of no terms is 0, and so are dW and db of no rows
        const bool clear = !(flags & GN_ACCUMULATE) && M == 0;
        hipError_t e = dP && m * k ? launch_zero(dP, m * k * es, s) : hipSuccess;
        if (e == hipSuccess && clear && dW && n * k) e = launch_zero(dW, n * k * 4, s);
        if (e == hipSuccess && clear && db && n) e = launch_zero(db, n * 4, s);
        if (e != hipSuccess) {
            set_error("%s: clear failed", who);
            return GN_E_HIP;
        }
        if (K == 0 && M > 0 && db && n) return gn_colsum(dY, (float*)db, M, N, dtype, flags, stream);
        return GN_OK;
    }
    if (need)
        if (const int rc = check_ws(who, ws, ws_bytes, need)) return rc;
    char* const rest = ws ? (char*)ws + need : nullptr;  // the weight gradient's partial sums
    const size_t rest_bytes = ws && ws_bytes > need ? ws_bytes - need : 0;
    const int64_t nk = (int64_t)m * K;
    const unsigned grid = grid_for(nk, 1024, 16384);
    if (dtype == GN_F32) {
        if (dP)
            if (const int rc = gn_gemm(dY, W, N, nullptr, nullptr, 0, dP, M, K, 0, 0, dtype, dtype, 0, stream)) return rc;
        if (dP) {
            finish_backward<<<grid, 256, 0, s>>>((float*)dP, (const float*)P, nk, act);
            GN_LAUNCH_CHECK(who);
        }
        return dW ? gn_linear_bwd_ws(dY, A, W, nullptr, dW, db, M, N, K, dtype, flags, rest, rest_bytes, stream) : GN_OK;
    }
    const double flop = 2.0 * M * N * (double)K;
    SideBySide sb(s, dP && dW ? side_by_side(dtype, flop, flop, M, K, N, K) : Fork::kNever);
    int rc = GN_OK;
    if (dW) rc = weight_grad(dY, N, A, K, M, N, K, dW, dW, N, (float*)db, nullptr, dtype, flags, s, rest, rest_bytes, sb.side() != s);
    if (rc == GN_OK && dP) {
        hipStream_t side = sb.side();
        int Kp = K, Np = N;
        if (lay) {
            Kp = up8(K);
            Np = up8(N);
            char* const w = (char*)ws + up16(m * Np * 2);
            rc = copy(dY, ws, M, N, M, Np, side);
            if (rc == GN_OK) rc = copy(W, w, N, K, Np, Kp, side);
            dY = ws;
            W = w;
        }
        if (rc == GN_OK) {
            GemmDesc d{};
            d.nseg = 1;
            d.A[0] = (const bf16_t*)dY; d.lda[0] = Np; d.Ks[0] = Np;
            d.B[0] = (const bf16_t*)W; d.ldb[0] = Kp;
            d.M = M; d.N = Kp; d.Msplit = M; d.ldc = Kp;
            d.beside = side != s;
            Backward f{};
            f.P = (const bf16_t*)P;
            f.dP = (bf16_t*)dP;
            f.N = K;
            f.act = act;
            f.vec = K % 8 == 0 && al16(P) && al16(dP);
            rc = launch<false>(d, f, side);
        }
    }
    const int jr = sb.join();
    return rc ? rc : jr;
}
