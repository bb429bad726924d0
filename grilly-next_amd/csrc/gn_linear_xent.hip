// gn_linear_xent.hip — softmax cross entropy of a linear head (l = h E^T) without its logits, forward
// and backward, a piece of the vocabulary at a time.
//
//   forward    per piece: l = h E_c^T (fp32, in the workspace); each row's running maximum and sum of
//              exp take the piece in; the target's logit is picked up in passing
//   backward   per piece: l again, G = u (exp(l - lse) - [target]) + z exp(l - lse),
//              dE_c (+)= G^T h,  dh += G E_c
//
// The products are the library's own (gemm_run).  On the bf16 path G is stored as bf16, and for an
// fp32 dE as two bf16 pieces, hi + lo, whose products with h are summed as two k-segments of one
// product: |G - hi - lo| <= 2^-17 |G|, where bf16 alone (2^-9) would be the gradient's largest error.
#include <algorithm>
#include <cmath>

#include "gn_common.h"
#include "gn_gemm_dma.h"

namespace gn {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// A part of a row: its maximum m and the sum s of exp2 about it, (-inf, 0) when it is empty.  A NaN
// among the logits is in s only (m skips it) and stays there.
// s about another maximum n >= m
__device__ __forceinline__ float about(float s, float m, float n) {
    return s * __builtin_amdgcn_exp2f(m - (n == -INFINITY ? 0.f : n));
}
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
    const float n = fmaxf(m, m2);
    s = about(s, m, n) + about(s2, m2, n);
    m = n;
}

// A row's statistics over one piece, joined with those of the pieces before; the last piece
// turns them into lse and loss.  Statistics in units of log2.
__global__ __launch_bounds__(256) void piece_stats(const float* __restrict__ L, int ld, int v0, int nv,
                                                   const int32_t* __restrict__ tgt, float2* __restrict__ st,
                                                   float* __restrict__ lt, float* __restrict__ loss,
                                                   float* __restrict__ lse, int V, int first, int last) {
    __shared__ float sm[4], ss[4];
    const int t = blockIdx.x;
    const float* row = L + (size_t)t * ld;
    float m = -INFINITY, s = 0.f;
    for (int v = threadIdx.x; v < nv; v += 256) {
        const float x = row[v] * kLog2e;
        if (x > m) {
            s = s * __builtin_amdgcn_exp2f(m - x) + 1.f;
            m = x;
        } else if (x != -INFINITY) {
            s += __builtin_amdgcn_exp2f(x - m);
        }
    }
    const float mw = wave_max(m);
    s = wave_sum(about(s, m, mw));
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
        sm[w] = mw;
        ss[w] = s;
    }
    __syncthreads();
    if (threadIdx.x) return;
    m = first ? -INFINITY : st[t].x;
    s = first ? 0.f : st[t].y;
#pragma unroll
    for (int i = 0; i < 4; ++i) join(m, s, sm[i], ss[i]);
    const int g = tgt[t];
    if (g >= v0 && g < v0 + nv) lt[t] = row[g - v0];
    if (!last) {
        st[t] = make_float2(m, s);
        return;
    }
    const float z = (m + __builtin_amdgcn_logf(s)) / kLog2e;
    if (lse) lse[t] = z;
    if (loss) loss[t] = g >= 0 && g < V ? z - lt[t] : 0.f;
}

// u and z of a row
__device__ __forceinline__ float2 row_scale(int t, const int32_t* tgt, const float* dloss, const float* dlse, float scale,
                                            int V) {
    const int g = tgt[t];
    const float u = g >= 0 && g < V ? (dloss ? scale * dloss[t] : scale) : 0.f;
    return make_float2(u, dlse ? scale * dlse[t] : 0.f);
}

// G of one piece: fp32 in place (hi == nullptr), or as bf16 hi and (lo != nullptr) lo
__global__ __launch_bounds__(256) void piece_grad(float* __restrict__ L, bf16_t* __restrict__ hi, bf16_t* __restrict__ lo,
                                                  int ld, int v0, int nv, const int32_t* __restrict__ tgt,
                                                  const float* __restrict__ lse, const float* __restrict__ dloss,
                                                  const float* __restrict__ dlse, float scale, int V) {
    const int t = blockIdx.x, g = tgt[t] - v0;
    const float2 uz = row_scale(t, tgt, dloss, dlse, scale, V);
    const float a = uz.x + uz.y, b = lse[t] * kLog2e;
    for (int v = blockIdx.y * 256 + threadIdx.x; v < nv; v += 256 * gridDim.y) {
        const size_t i = (size_t)t * ld + v;
        float x = a * __builtin_amdgcn_exp2f(L[i] * kLog2e - b);
        if (v == g) x -= uz.x;
        if (!hi) {
            L[i] = x;
        } else {
            const bf16_t p = f2bf(x);
            hi[i] = p;
            if (lo) lo[i] = f2bf(x - bf2f(p));
        }
    }
}

__global__ __launch_bounds__(256) void round_rows(const float* __restrict__ a, bf16_t* __restrict__ o, int64_t n) {
    for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) o[i] = f2bf(a[i]);
}

// The vocabulary's pieces: as many columns as keep a piece's fp32 logits at 256 MB, multiples of 64.
int piece_columns(int T, int V) {
    const int64_t c = std::max<int64_t>(256, ((int64_t)64 << 20) / std::max(T, 1) / 64 * 64);
    return (int)std::min<int64_t>(c, ((int64_t)V + 63) / 64 * 64);
}

size_t up(size_t b) { return (b + 255) / 256 * 256; }

// The workspace of both directions
struct Layout {
    int vc, pieces;
    size_t logits, stats, target, hi, lo, acc, bytes;
    Layout(int T, int d, int V, int dtype) {
        vc = piece_columns(T, V);
        pieces = (V + vc - 1) / vc;
        size_t at = 0;
        auto take = [&](size_t n) {
            const size_t p = at;
            at += up(n);
            return p;
        };
        const bool bf = dtype == GN_BF16;
        logits = take((size_t)T * vc * 4);
        stats = take((size_t)T * 8);
        target = take((size_t)T * 4);
        hi = take(bf ? (size_t)T * vc * 2 : 0);
        lo = take(bf ? (size_t)T * vc * 2 : 0);
        acc = take(bf ? (size_t)T * d * 4 : 0);
        bytes = at;
    }
};

GemmDesc product(const void* A, int lda, const void* B, int ldb, int K, void* C, int ldc, int M, int N) {
    GemmDesc g{};
    g.A[0] = (const bf16_t*)A;
    g.B[0] = (const bf16_t*)B;
    g.lda[0] = lda;
    g.ldb[0] = ldb;
    g.Ks[0] = K;
    g.nseg = 1;
    g.M = M;
    g.N = N;
    g.C = g.C2 = C;
    g.Msplit = M;
    g.ldc = ldc;
    g.ksplit = 1;
    return g;
}

inline bool al16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

int check(const char* who, const void* h, const void* E, const int32_t* tgt, int T, int d, int V, int dtype) {
    GN_REQUIRE(dtype == GN_F32 || dtype == GN_BF16, "%s: dtype %d not supported (f32, bf16)", who, dtype);
    GN_REQUIRE(T >= 0 && d >= 1 && V >= 1, "%s: bad shape", who);
    GN_REQUIRE(T == 0 || (h && E && tgt), "%s: null pointer", who);
    const int es = dtype == GN_F32 ? 4 : 2;
    GN_REQUIRE((((uintptr_t)h | (uintptr_t)E) & (es - 1)) == 0 && ((uintptr_t)tgt & 3u) == 0,
               "%s: a tensor is not aligned to its elements", who);
    return GN_OK;
}

int check_ws(const char* who, const Layout& w, const void* ws, size_t ws_bytes) {
    if (!ws || ws_bytes < w.bytes || !al16(ws)) {
        set_error("%s: workspace of %zu bytes (16-byte aligned) required", who, w.bytes);
        return GN_E_WORKSPACE;
    }
    return GN_OK;
}

}  // namespace
}  // namespace gn

using namespace gn;

extern "C" size_t gn_linear_xent_workspace_bytes(int T, int d, int V, int dtype) {
    if (T <= 0 || d <= 0 || V <= 0 || (dtype != GN_F32 && dtype != GN_BF16)) return 0;
    return Layout(T, d, V, dtype).bytes;
}

extern "C" int gn_linear_xent_fwd(const void* h, const void* E, const int32_t* targets, float* loss, float* lse, int T,
                                  int d, int V, int dtype, void* ws, size_t ws_bytes, void* stream) {
    const char* who = "gn_linear_xent_fwd";
    clear_error();
    if (const int rc = check(who, h, E, targets, T, d, V, dtype)) return rc;
    GN_REQUIRE((((uintptr_t)loss | (uintptr_t)lse) & 3u) == 0, "%s: loss, lse must be aligned to 4 bytes", who);
    if (T == 0 || (!loss && !lse)) return GN_OK;
    const Layout w(T, d, V, dtype);
    if (const int rc = check_ws(who, w, ws, ws_bytes)) return rc;
    hipStream_t s = as_stream(stream);
    char* const base = (char*)ws;
    const int es = dtype == GN_F32 ? 4 : 2;
    for (int p = 0; p < w.pieces; ++p) {
        const int v0 = p * w.vc, nv = std::min(w.vc, V - v0);
        const GemmDesc g = product(h, d, (const char*)E + (size_t)v0 * d * es, d, d, base + w.logits, w.vc, T, nv);
        if (const int rc = gemm_run(g, 0, 1, dtype, GN_F32, s)) return rc;
        piece_stats<<<T, 256, 0, s>>>((const float*)(base + w.logits), w.vc, v0, nv, targets, (float2*)(base + w.stats),
                                      (float*)(base + w.target), loss, lse, V, p == 0, p == w.pieces - 1);
        GN_LAUNCH_CHECK(who);
    }
    return GN_OK;
}

extern "C" int gn_linear_xent_bwd(const void* h, const void* E, const int32_t* targets, const float* lse,
                                  const float* dloss, const float* dlse, float scale, void* dh, void* dE, int dE_dtype,
                                  int T, int d, int V, int dtype, unsigned flags, void* ws, size_t ws_bytes,
                                  void* stream) {
    const char* who = "gn_linear_xent_bwd";
    clear_error();
    if (const int rc = check(who, h, E, targets, T, d, V, dtype)) return rc;
    GN_REQUIRE(dE_dtype == GN_F32 || (dE_dtype == GN_BF16 && dtype == GN_BF16), "%s: dE must be f32, or bf16 on the bf16 path", who);
    GN_REQUIRE((flags & ~GN_ACCUMULATE) == 0, "%s: unknown flags", who);
    const bool acc = flags & GN_ACCUMULATE;
    GN_REQUIRE(!acc || dE_dtype == GN_F32, "%s: only an fp32 dE accumulates", who);
    GN_REQUIRE(((uintptr_t)dE & (dE_dtype == GN_F32 ? 3u : 1u)) == 0 && ((uintptr_t)dh & (dtype == GN_F32 ? 3u : 1u)) == 0 &&
                   (((uintptr_t)lse | (uintptr_t)dloss | (uintptr_t)dlse) & 3u) == 0,
               "%s: a tensor is not aligned to its elements", who);
    hipStream_t s = as_stream(stream);
    if (T == 0) {  // no rows: dE is zero
        if (dE && !acc && launch_zero(dE, (size_t)V * d * (dE_dtype == GN_F32 ? 4 : 2), s) != hipSuccess) {
            set_error("%s: clear failed", who);
            return GN_E_HIP;
        }
        return GN_OK;
    }
    GN_REQUIRE(lse, "%s: null pointer", who);
    if (!dh && !dE) return GN_OK;
    const Layout w(T, d, V, dtype);
    if (const int rc = check_ws(who, w, ws, ws_bytes)) return rc;
    char* const base = (char*)ws;
    const bool bf = dtype == GN_BF16;
    const int es = bf ? 2 : 4;
    float* const L = (float*)(base + w.logits);
    bf16_t* const hi = bf ? (bf16_t*)(base + w.hi) : nullptr;
    bf16_t* const lo = bf && dE && dE_dtype == GN_F32 ? (bf16_t*)(base + w.lo) : nullptr;
    // dh of one piece is rounded by its product; of several it is summed in fp32 first
    const bool direct = !bf || w.pieces == 1;
    void* const sum = direct ? dh : base + w.acc;
    for (int p = 0; p < w.pieces; ++p) {
        const int v0 = p * w.vc, nv = std::min(w.vc, V - v0);
        const char* Ec = (const char*)E + (size_t)v0 * d * es;
        if (const int rc = gemm_run(product(h, d, Ec, d, d, L, w.vc, T, nv), 0, 1, dtype, GN_F32, s)) return rc;
        piece_grad<<<dim3(T, std::min(64, (nv + 1023) / 1024)), 256, 0, s>>>(L, hi, lo, w.vc, v0, nv, targets, lse, dloss,
                                                                            dlse, scale, V);
        GN_LAUNCH_CHECK(who);
        const void* G = bf ? (const void*)hi : L;
        if (dE) {
            GemmDesc g = product(G, w.vc, h, d, T, (char*)dE + (size_t)v0 * d * (dE_dtype == GN_F32 ? 4 : 2), d, nv, d);
            if (lo) {
                g.nseg = 2;
                g.A[1] = lo;
                g.lda[1] = w.vc;
                g.B[1] = g.B[0];
                g.ldb[1] = d;
                g.Ks[1] = T;
            }
            g.accumulate = acc;
            if (const int rc = gemm_run(g, 1, 0, dtype, dE_dtype, s)) return rc;
        }
        if (dh) {
            GemmDesc g = product(G, w.vc, Ec, d, nv, sum, d, T, d);
            g.accumulate = p > 0;
            if (const int rc = gemm_run(g, 0, 0, dtype, bf && direct ? GN_BF16 : GN_F32, s)) return rc;
        }
    }
    if (dh && !direct) {
        const int64_t n = (int64_t)T * d;
        round_rows<<<grid_for(n, 1024, 8192), 256, 0, s>>>((const float*)sum, (bf16_t*)dh, n);
        GN_LAUNCH_CHECK(who);
    }
    return GN_OK;
}
