// gn_linear_act.hip — a Linear's forward with bias, activation and residual in the product's epilogue, and
// the backward of a Linear behind an activation, whose input-gradient product leaves the gradient in front of it.
//
//   forward    v = X W^T + b,  Y = R + act(v),  P = v (tanh, sigmoid: act(v))
//   backward   dP = (dY W) act'(P),  dW = dY^T A,  db = column sums of dY
//
// bf16 products run on the streamed tiles (gn_gemm_stream_core.h) or, where those would leave compute units
// idle, on the small ones (gn_gemm_wave_core.h), with the epilogues of gn_linear_act_core.h: the sums stay in fp32 until Y, P or dP
// is rounded once.  Sizes and addresses that the products' 16-byte pieces do not take are laid out first in the
// workspace.  fp32 products are gn_linear_fwd's and gn_linear_bwd_ws's, with a pass behind them where there is an
// activation or a residual.
//
// Measured (us, bf16; in brackets the library's products alone, without bias, activation, residual or stored P):
//   4096 x 5632 x 2048 with bias, gelu and P   107 (89)   0.88 PFLOP/s
//   4001 x 2048 x 5632, bias, fp32 residual     95 (81)   0.97
//   backward of 4096 x 2048 x 5632, gelu, db   209 (99 + 110)   0.90 over both products
//   8 x 5632 x 2048 with bias and silu         8.3, 7.3 of it the kernel: 3.2 TB/s of W
// The matrix cores bound the large ones; beside them stand the epilogue's reads of R or P and its stores, which a tile's compute waves do
// themselves with the matrix pipe idle, and dW's 176 tiles of 256 x 256 on 256 CUs.  A few rows are bound by the latency of
// the k loop's loads on 176 blocks.
#include <algorithm>

#include "gn_act.h"
#include "gn_gemm_dma.h"
#include "gn_lane.h"

namespace gn {

// Their bf16 products with the epilogues (gn_linear_act_{bf16,f32,bwd}.hip: Y in bf16, in fp32; the backward, of N columns).
// vec: four elements of a row at a time.
int linear_act_bf16(const GemmDesc& d, int act, const void* b, const void* R, void* Y, void* P, bool vec, hipStream_t s);
int linear_act_f32(const GemmDesc& d, int act, const void* b, const void* R, void* Y, void* P, bool vec, hipStream_t s);
int act_linear_dp(const GemmDesc& d, int act, const void* P, void* dP, int N, bool vec, hipStream_t s);

namespace {

inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// ---- passes ------------------------------------------------------------------------------------
// Memory bounds the passes behind fp32 products, so that their activations are not gn_act.h's few instructions, whose 2^-22 of 1 under
// tanh or erf is several steps of a smaller value, but the math library's e^x, tanh and erfc (erfc(-u) = 1 + erf(u)) with
// true quotients: a few steps of the value itself.  4096 x 5632 x 2048, forward: silu 553 -> 556 us, erf gelu 558 -> 561; backward 502 -> 504.
__device__ __forceinline__ float gelu_2z(float x) { return x * fmaf(x * x, kG3, kG1); }
template <int KIND>
__device__ __forceinline__ float act_f32(float x) {
    if constexpr (KIND == GN_ACT_GELU_TANH) return x / (1.0f + expf(-gelu_2z(x)));
    else if constexpr (KIND == GN_ACT_GELU_ERF) return 0.5f * x * erfcf(x * -0.70710678118654752f);
    else if constexpr (KIND == GN_ACT_SILU) return x / (1.0f + expf(-x));
    else if constexpr (KIND == GN_ACT_TANH) return tanhf(x);
    else if constexpr (KIND == GN_ACT_SIGMOID) return 1.0f / (1.0f + expf(-x));
    else return act_of<KIND>(x);
}
// of x sigmoid(u): s + x s (1 - s) u' with s and 1 - s of e^-|u|, neither as a difference from 1
__device__ __forceinline__ float gated_slope(float x, float u, float du) {
    const float e = expf(-fabsf(u)), r = 1.0f / (1.0f + e), s = u < 0.f ? e * r : r;
    return fmaf(x * du, e * r * r, s);
}
template <int KIND>
__device__ __forceinline__ float slope_f32(float x) {
    if constexpr (KIND == GN_ACT_GELU_TANH) {
        const float c = fabsf(x) > 20.f ? copysignf(20.f, x) : x;  // (as in slope_of; a NaN stays)
        return gated_slope(c, gelu_2z(c), fmaf(c * c, 3.0f * kG3, kG1));
    } else if constexpr (KIND == GN_ACT_GELU_ERF) {
        return fmaf(x * 0.3989422804014327f, expf(-0.5f * x * x), 0.5f * erfcf(x * -0.70710678118654752f));
    } else if constexpr (KIND == GN_ACT_SILU) {
        return gated_slope(x, x, 1.0f);
    } else if constexpr (KIND == GN_ACT_TANH) {
        return fmaf(-x, x, 1.0f);
    } else {
        return slope_of<KIND>(x);
    }
}
// The epilogue of fp32 products, in place: v (fp32, or nullptr: a product of no terms, v = b) -> P, Y.  TR: R and Y.
template <typename TR, typename TB>
__global__ __launch_bounds__(256) void finish_forward(const float* v, const TB* b, const TR* R, TR* Y, TB* P, int64_t n, int N,
                                                      int act, bool out_is_pre) {
    for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float x = (v ? v[i] : 0.f) + (b ? io<TB>::ld(b, i % N) : 0.f);
        if (P && !out_is_pre) io<TB>::st(P, i, x);
        by_act<kAny, true>(act, [&](auto A) {
            if constexpr (decltype(A)::value != GN_ACT_NONE) x = act_f32<decltype(A)::value>(x);
        });
        if (P && out_is_pre) io<TB>::st(P, i, x);
        io<TR>::st(Y, i, R ? x + io<TR>::ld(R, i) : x);
    }
}
// dP *= act'(P), fp32: n4 pieces of four elements, or (V 1) n4 elements
template <int V>
__global__ __launch_bounds__(256) void finish_backward(float* dP, const float* P, int64_t n4, int act) {
    by_act<kAny, false>(act, [&](auto A) {
        for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n4; i += (int64_t)gridDim.x * 256) {
            float p[V], d[V];
            if constexpr (V == 4) {
                const float4 x = reinterpret_cast<const float4*>(P)[i], y = reinterpret_cast<const float4*>(dP)[i];
                p[0] = x.x; p[1] = x.y; p[2] = x.z; p[3] = x.w;
                d[0] = y.x; d[1] = y.y; d[2] = y.z; d[3] = y.w;
            } else {
                p[0] = P[i];
                d[0] = dP[i];
            }
#pragma unroll
            for (int e = 0; e < V; ++e) d[e] *= slope_f32<decltype(A)::value>(p[e]);
            if constexpr (V == 4) reinterpret_cast<float4*>(dP)[i] = make_float4(d[0], d[1], d[2], d[3]);
            else dP[i] = d[0];
        }
    });
}

// dst [Rp x dp] = src [R x d], zeros around it; dp a multiple of 8, dst 16-byte aligned: eight elements a thread
__global__ __launch_bounds__(256) void lay_out(const bf16_t* __restrict__ src, bf16_t* __restrict__ dst, int R, int d, int Rp, int dp) {
    const int per = dp >> 3;
    const int64_t n = (int64_t)Rp * per;
    for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int r = (int)(i / per), c = 8 * (int)(i - (int64_t)r * per);
        const bf16_t* const from = src + (size_t)r * d + c;
        uint32_t v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = r < R && c + e < d ? from[e] : 0;
        *reinterpret_cast<uint4*>(dst + 8 * i) = make_uint4(v[0] | (v[1] << 16), v[2] | (v[3] << 16), v[4] | (v[5] << 16), v[6] | (v[7] << 16));
    }
}
int copy(const void* src, void* dst, int R, int d, int Rp, int dp, hipStream_t s) {
    lay_out<<<grid_for((int64_t)Rp * (dp / 8), 256, 16384), 256, 0, s>>>((const bf16_t*)src, (bf16_t*)dst, R, d, Rp, dp);
    GN_LAUNCH_CHECK("linear (layout)");
    return GN_OK;
}

inline int up8(int n) { return (n + 7) / 8 * 8; }
inline size_t up16(size_t n) { return (n + 15) / 16 * 16; }

// dst [R x d] (+)= src [R x dp]
__global__ __launch_bounds__(256) void take_rows(const float* __restrict__ src, float* __restrict__ dst, int R, int d, int dp, int accumulate) {
    const int64_t n = (int64_t)R * d;
    for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int r = (int)(i / d), c = (int)(i - (int64_t)r * d);
        const float v = src[(size_t)r * dp + c];
        dst[i] = accumulate ? dst[i] + v : v;
    }
}
int take(const float* src, void* dst, int R, int d, int dp, bool accumulate, hipStream_t s) {
    take_rows<<<grid_for((int64_t)R * d, 1024, 16384), 256, 0, s>>>(src, (float*)dst, R, d, dp, accumulate);
    GN_LAUNCH_CHECK("linear (layout)");
    return GN_OK;
}

// The operands of the forward's bf16 product laid out: X [M x K'], W [N x K'].
size_t layout_bytes(int M, int N, int K) { return up16((size_t)M * up8(K) * 2) + up16((size_t)N * up8(K) * 2); }

// Those of the backward's: dY [M x N'] for either product; W [N' x K'] for dP; A [M x K'], and the padded dW [N' x K'] and
// db [N'] in fp32, for dW.
struct BackwardLayout {
    size_t dY, W, A, dW, db, bytes;
    BackwardLayout(int M, int N, int K, bool dp, bool dw) {
        const size_t Np = up8(N), Kp = up8(K);
        bytes = 0;
        auto place = [&](size_t n) {
            const size_t at = bytes;
            bytes += up16(n);
            return at;
        };
        dY = place(dp || dw ? M * Np * 2 : 0);
        W = place(dp ? Np * Kp * 2 : 0);
        A = place(dw ? M * Kp * 2 : 0);
        dW = place(dw ? Np * Kp * 4 : 0);
        db = place(dw ? Np * 4 : 0);
    }
};

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

// (a tile's loads are 32 bits of bytes from its first row: 255 rows of 2^23 bf16 elements at most)
bool sizes_fit(int M, int N, int K) {
    return M < (1 << 28) && N < (1 << 23) && K < (1 << 23) && (int64_t)M * std::max(N, K) < (1ll << 36) && (int64_t)N * K < (1ll << 36);
}
int check_sizes(const char* who, int M, int N, int K, int dtype) {
    GN_REQUIRE(M >= 0 && N >= 0 && K >= 0, "%s: negative size", who);
    GN_REQUIRE(dtype == GN_F32 || dtype == GN_BF16, "%s: dtype %d not supported (f32, bf16)", who, dtype);
    GN_REQUIRE(sizes_fit(M, N, K), "%s: M below 2^28, N and K below 2^23, M * N, M * K and N * K below 2^36", who);
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
    // beyond the layout, the partial planes of the padded weight gradient: gn_linear_workspace_bytes has none for such sizes
    // (8192 x 1027 x 1031 73 -> 67 us, 8192 x 513 x 519 56 -> 48 with them)
    const size_t planes = N % 8 || K % 8 ? weight_grad_ws_bytes(M, up8(N), up8(K), dtype) : 0;
    return std::max(layout_bytes(M, N, K), BackwardLayout(M, N, K, true, true).bytes + planes);
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
    const size_t need = lay ? layout_bytes(M, N, K) : 0;
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
            // (a P of the sums themselves is the product's, and complete)
            finish_forward<float, float><<<grid, 256, 0, s>>>(v, nullptr, (const float*)R, (float*)Y, out_is_pre ? (float*)P : nullptr, n, N, act, out_is_pre);
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
    const bool vec = N % 4 == 0 && al16(b) && al16(R) && al16(Y) && al16(P);
    return y_dtype == GN_F32 ? linear_act_f32(d, act, b, R, Y, P, vec, s) : linear_act_bf16(d, act, b, R, Y, P, vec, s);
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
    const bool odd = N % 8 || K % 8 || !al16(dY), bf = dtype == GN_BF16;
    const bool lay_p = bf && dP && (odd || !al16(W)), lay_w = bf && dW && (odd || !al16(A) || !al16(dW));
    const BackwardLayout at(M, N, K, lay_p, lay_w);
    const size_t need = at.bytes;
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
    char* const rest = ws ? (char*)ws + need : nullptr;  // the products' partial sums
    const size_t rest_bytes = ws && ws_bytes > need ? ws_bytes - need : 0;
    const int64_t nk = (int64_t)m * K;
    if (dtype == GN_F32) {
        // dP's product and dW's as the plain layer's backward has them: one pass over W for up to 8 rows, one launch for small
        // layers, ranges of the terms in the workspace (us, silu, with two products of their own and no ranges -> so; the plain
        // layer and gn_act_bwd: 8 x 5632 x 2048 148 -> 41, 41; 128 x 4096 x 1024 110 -> 38, 39; 64 x 10 x 256 7.4 -> 4.8, 4.9;
        // 64 x 256 x 784 17.3 -> 18.7, 18.6).  Without the workspace the few rows' sums would be atomics, and where dW is
        // added onto, dP would be too: then dP's product by itself.
        const bool both = dP && dW && !(flags & GN_ACCUMULATE) &&
                          (skinny_bwd_ws_bytes(M, N, K) == 0 || (al16(rest) && rest_bytes >= skinny_bwd_ws_bytes(M, N, K)));
        int rc = GN_OK;
        if (dW) rc = gn_linear_bwd_ws(dY, A, W, both ? dP : nullptr, dW, db, M, N, K, dtype, flags, rest, rest_bytes, stream);
        if (rc == GN_OK && dP && !both) rc = gemm_dispatch(dY, W, N, nullptr, nullptr, 0, dP, M, K, 0, 0, dtype, dtype, 0, s, rest, rest_bytes, false);
        if (rc == GN_OK && dP) {
            if (nk % 4 == 0 && al16(dP) && al16(P))
                finish_backward<4><<<grid_for(nk / 4, 256, 8192), 256, 0, s>>>((float*)dP, (const float*)P, nk / 4, act);
            else
                finish_backward<1><<<grid_for(nk, 256, 8192), 256, 0, s>>>((float*)dP, (const float*)P, nk, act);
            GN_LAUNCH_CHECK(who);
        }
        return rc;
    }
    char* const base = (char*)ws;
    const bool accumulate = flags & GN_ACCUMULATE;
    const int Np = up8(N), Kp = up8(K);
    int rc = GN_OK;
    const void* dYp = dY;
    if (lay_p || lay_w) {
        rc = copy(dY, base + at.dY, M, N, M, Np, s);
        dYp = base + at.dY;
    }
    if (rc == GN_OK && lay_w) {
        // the weight gradient of the padded operands; the framework's own for such sizes, element by element, takes
        // 1226 us for 4096 x 5633 x 2048 against 166 here
        rc = copy(A, base + at.A, M, K, M, Kp, s);
        float *const dWp = (float*)(base + at.dW), *const dbp = (float*)(base + at.db);
        if (rc == GN_OK)
            rc = weight_grad(dYp, Np, base + at.A, Kp, M, Np, Kp, dWp, dWp, Np, db ? dbp : nullptr, nullptr, dtype, 0, s, rest, rest_bytes, false);
        if (rc == GN_OK) rc = take(dWp, dW, N, K, Kp, accumulate, s);
        if (rc == GN_OK && db) rc = take(dbp, db, 1, N, Np, accumulate, s);
    }
    if (rc != GN_OK) return rc;
    const double flop = 2.0 * M * N * (double)K;
    SideBySide sb(s, dP && dW && !lay_p && !lay_w ? side_by_side(dtype, flop, flop, M, K, N, K) : Fork::kNever);
    if (dW && !lay_w) rc = weight_grad(dY, N, A, K, M, N, K, dW, dW, N, (float*)db, nullptr, dtype, flags, s, rest, rest_bytes, sb.side() != s);
    if (rc == GN_OK && dP) {
        hipStream_t side = sb.side();
        const int ldw = lay_p ? Kp : K, terms = lay_p ? Np : N;
        if (lay_p) rc = copy(W, base + at.W, N, K, Np, Kp, side);
        if (rc == GN_OK) {
            GemmDesc d{};
            d.nseg = 1;
            d.A[0] = (const bf16_t*)(lay_p ? dYp : dY); d.lda[0] = terms; d.Ks[0] = terms;
            d.B[0] = (const bf16_t*)(lay_p ? base + at.W : W); d.ldb[0] = ldw;
            d.M = M; d.N = ldw; d.Msplit = M; d.ldc = ldw;
            d.beside = side != s;
            rc = act_linear_dp(d, act, P, dP, K, K % 4 == 0 && al16(P) && al16(dP), side);
        }
    }
    const int jr = sb.join();
    return rc ? rc : jr;
}
