// gn_rope.hip — rotary positions and per-head RMS norms of queries and keys (forward and
// backward), one kernel template for all of them.
//
//   rotation   a = position * freq,  (u, w) -> m (u cos a - w sin a, w cos a + u sin a)
//   norm       r = rsqrt(mean x^2 + eps),  y = rotation(x r w)
//   backward   g = rotation^T(dy),  dx = r (w g - x r^2 mean(w g x)),  dw = sum g x r
//
// Every element is read once and written once, so the passes are bound by HBM (and, at a token
// a sequence, by the launch).  A block takes a tile of tokens: its threads first put the tile's
// cos and sin into LDS, each pair of a token computed once for all of its heads (an fp64 product
// and sincospi a pair, which per head would cost more than the pass's memory time), then walk the
// tile's rows (token, head).  A row of D elements belongs to LPR lanes; a lane holds both
// members of each of its pairs, 2 x 8 elements as two 16-byte pieces (rows of 16-byte aligned
// heads with D and rot multiples of 16), or single elements otherwise, a wave per row.  The row
// sums of the norm are DPP moves within the LPR lanes.  The head split or merge of the layouts
// is nothing but strides.
//
// Measured (a large copy reaches 5.0 TB/s, an update in place 6.0): rotation of 307 MB in and out
// 61.8 us (4.97 TB/s), fp32 of 49 MB 10.3 us (4.8); norms, rotation and head split of 403 MB 78.0 us
// (5.2); their backward, which reads x again, 570 MB 126 us (4.5: two dependent row sums between a row's
// loads and its stores, and three waves a SIMD, no more, hold two rows each); both 206 us.  Stores past the
// caches take 17 us off the two and add 10 to them with a reader behind, so they are ordinary ones.  fp32: norms,
// rotation and head split of 805 MB 171 us (4.7), their backward 244.  A token a sequence: 3.4 us of kernel,
// 5.3 with the norms, under the calls' host time of 8.7 and 21.7.  Few tokens: the backward of 3 x 777 tokens
// (8 + 2 heads of 96, fp32, 30 MB) 20 us of kernel, a tile being two tokens there (tile()): 16 rows of q and 4 of k
// for a block's 32 lane groups.  dw is summed in fp32 (a lane's rows, the lane groups, the blocks, in that
// order): 2e-7 of its norm off there, where sums in fp64 leave 7e-8.  16-byte pieces against elements: bf16 rotation of 4 x 4096 x 32
// heads, 128 wide 42.7 and 92.4 us, 64 wide 22.0 and 75.8; fp32 102 and 106, 48 and 84.  (A pair's second half
// starts at rot / 2, and what is behind the rotation splits in two: pieces of eight elements need multiples of
// 16.  Pieces of 8 bytes for multiples of 8 are not built.)
#include <algorithm>
#include <cmath>

#include "gn_common.h"

namespace gn {
namespace {

constexpr int kThreads = 256;
// Forward tiles along x, the others along y: a launch's threads in one dimension are counted in 32 bits, which
// one token a tile and 256 threads would pass at 2^24 tokens.
constexpr int kTilesX = 1 << 22;

enum Kind { kRotate, kNorm };

struct Group {
    const void *x, *dy, *w;  // input of the norm (or of the rotation); upstream gradient; weights
    void* y;
    int64_t xs[3], ds[3], ys[3];  // batch, token and head strides of x, dy, y
    int H;
    uint32_t magic;  // ceil(2^32 / H), 0 for one head: r / H for rows r of a tile
};

struct Args {
    Group g[2];     // the rotated tensors
    Group copy;     // values: copied (H = 0: none)
    int ng;
    const double* freqs;
    const int32_t* pos;
    int64_t pos_sb, pos0;
    float mscale, sgn, eps;  // sgn: -1 turns back
    int rot, S, D, tokens;
    int TB[2], tiles[2];  // tokens of a tile and tiles: of all groups, or (backward) of q and of k, v
    int nq, with_copy;    // backward: the blocks of q; whose blocks copy the values
    float* part;          // [gridDim.x][D] partial dw, nullptr: not wanted
    float* dw[2];         // where one block has all of a dw, it goes straight here
    int accumulate;
};

// A lane's part of a row of D elements
template <typename T, int LPR, bool VEC, bool HALF>
struct Row {
    static constexpr int NP = VEC ? 8 : 4;          // pairs of a lane
    static constexpr int NG = kThreads / LPR;       // rows at a time
    int c0, c1;  // VEC: its two pieces
    bool on, turn;
    int l, D, rot;

    __device__ __forceinline__ Row(int D_, int rot_) : l(threadIdx.x & (LPR - 1)), D(D_), rot(rot_) {
        if constexpr (VEC) {
            const int half = rot >> 4;  // pieces of the rotated part's first half
            turn = l < half;
            const int j = l - half, pass = (D - rot) >> 1;
            on = l < (D >> 4);
            c0 = turn ? 8 * l : rot + 8 * j;
            c1 = turn ? (rot >> 1) + 8 * l : rot + pass + 8 * j;
        } else {
            on = turn = true;
            c0 = c1 = 0;
        }
    }
    // the elements of pair i
    __device__ __forceinline__ int first(int i) const {
        if constexpr (VEC) {
            if constexpr (HALF) return c0 + i;
            return i < 4 ? c0 + 2 * i : c1 + 2 * (i - 4);
        }
        const int p = l + 64 * i;
        if (2 * p >= rot) return 2 * p;
        return HALF ? p : 2 * p;
    }
    __device__ __forceinline__ int second(int i) const {
        if constexpr (VEC) {
            if constexpr (HALF) return c1 + i;
            return first(i) + 1;
        }
        const int p = l + 64 * i;
        if (2 * p >= rot) return 2 * p + 1;
        return HALF ? p + (rot >> 1) : 2 * p + 1;
    }
    __device__ __forceinline__ bool has(int i) const { return VEC ? on : 2 * (l + 64 * i) < D; }
    // whether pair i is rotated; the others are taken as they are (0 times an infinite partner is NaN)
    __device__ __forceinline__ bool turns(int i) const { return VEC ? turn : 2 * (l + 64 * i) < rot; }

    // a lane's elements as they lie in memory
    struct Raw {
        static constexpr int Q = VEC ? 8 * (int)sizeof(T) / 16 : 1;
        uint4 a[Q], b[Q];
        T s[VEC ? 1 : 2 * NP];
    };
    __device__ __forceinline__ void raw(const T* p, bool live, Raw& r) const {
        if constexpr (VEC) {
#pragma unroll
            for (int q = 0; q < Raw::Q; ++q) r.a[q] = r.b[q] = make_uint4(0, 0, 0, 0);
            if (live && on) {
#pragma unroll
                for (int q = 0; q < Raw::Q; ++q) {
                    r.a[q] = reinterpret_cast<const uint4*>(p + c0)[q];
                    r.b[q] = reinterpret_cast<const uint4*>(p + c1)[q];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const bool ok = live && has(i);
                r.s[2 * i] = ok ? p[first(i)] : (T)0;
                r.s[2 * i + 1] = ok ? p[second(i)] : (T)0;
            }
        }
    }
    static __device__ __forceinline__ void widen8(const uint4* p, float (&v)[8]) {
        if constexpr (sizeof(T) == 2) {
            const uint32_t w[4] = {p->x, p->y, p->z, p->w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                v[4 * q] = __uint_as_float(p[q].x);
                v[4 * q + 1] = __uint_as_float(p[q].y);
                v[4 * q + 2] = __uint_as_float(p[q].z);
                v[4 * q + 3] = __uint_as_float(p[q].w);
            }
        }
    }
    __device__ __forceinline__ void widen(const Raw& r, float (&u)[NP], float (&w)[NP]) const {
        if constexpr (VEC) {
            float a[8], b[8];
            widen8(r.a, a);
            widen8(r.b, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                u[i] = HALF ? a[i] : (i < 4 ? a[(2 * i) & 7] : b[(2 * i) & 7]);
                w[i] = HALF ? b[i] : (i < 4 ? a[(2 * i + 1) & 7] : b[(2 * i + 1) & 7]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                u[i] = io<T>::ld(r.s, 2 * i);
                w[i] = io<T>::ld(r.s, 2 * i + 1);
            }
        }
    }
    __device__ __forceinline__ void ld(const T* p, bool live, float (&u)[NP], float (&w)[NP]) const {
        Raw r;
        raw(p, live, r);
        widen(r, u, w);
    }
    __device__ __forceinline__ void st(T* p, bool live, const float (&u)[NP], const float (&w)[NP]) const {
        if constexpr (VEC) {
            float a[8], b[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                a[i] = HALF ? u[i] : (i & 1 ? w[i >> 1] : u[i >> 1]);
                b[i] = HALF ? w[i] : (i & 1 ? w[4 + (i >> 1)] : u[4 + (i >> 1)]);
            }
            if (live && on) {
                chunk8<T>::st(p + c0, a);
                chunk8<T>::st(p + c1, b);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NP; ++i)
                if (live && has(i)) {
                    io<T>::st(p, first(i), u[i]);
                    io<T>::st(p, second(i), w[i]);
                }
        }
    }
    // cos and sin of the lane's pairs of tile token tt
    __device__ __forceinline__ void angles(const float* cosv, const float* sinv, int tt, float (&c)[NP],
                                           float (&s)[NP]) const {
        const int hr = rot >> 1;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            c[i] = 1.f;
            s[i] = 0.f;
        }
        if constexpr (VEC) {
            if (!turn) return;
            const int p0 = tt * hr + (HALF ? 8 * l : 4 * l), p1 = tt * hr + (HALF ? 8 * l + 4 : (hr >> 1) + 4 * l);
            const float4 ca = *reinterpret_cast<const float4*>(cosv + p0), cb = *reinterpret_cast<const float4*>(cosv + p1);
            const float4 sa = *reinterpret_cast<const float4*>(sinv + p0), sb = *reinterpret_cast<const float4*>(sinv + p1);
            c[0] = ca.x; c[1] = ca.y; c[2] = ca.z; c[3] = ca.w; c[4] = cb.x; c[5] = cb.y; c[6] = cb.z; c[7] = cb.w;
            s[0] = sa.x; s[1] = sa.y; s[2] = sa.z; s[3] = sa.w; s[4] = sb.x; s[5] = sb.y; s[6] = sb.z; s[7] = sb.w;
        } else {
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int p = l + 64 * i;
                if (2 * p < rot) {
                    c[i] = cosv[tt * hr + p];
                    s[i] = sinv[tt * hr + p];
                }
            }
        }
    }
    // the sum over the row's lanes, in each of them
    static __device__ __forceinline__ float sum(float v) {
        if constexpr (LPR == 64) return wave_sum(v);
        if constexpr (LPR >= 2) v += dpp_mov<0xB1>(v);
        if constexpr (LPR >= 4) v += dpp_mov<0x4E>(v);
        if constexpr (LPR >= 8) v += dpp_mov<0x141>(v);
        if constexpr (LPR >= 16) v += dpp_mov<0x140>(v);
        if constexpr (LPR >= 32) v += __shfl_xor(v, 16);
        return v;
    }
};

__device__ __forceinline__ int64_t at(const int64_t (&st)[3], int2 bs, int h) {
    return bs.x * st[0] + bs.y * st[1] + h * st[2];
}

// token and head of row r of a tile
__device__ __forceinline__ void token_head(const Group& g, int r, int& tt, int& h) {
    tt = g.magic ? (int)__umulhi((uint32_t)r, g.magic) : r;
    h = r - tt * g.H;
}

// Forward: rows in flight, U a lane (two: rotation of 307 MB 53.3 us, one: 55.0)
template <typename T, int LPR, bool VEC, bool HALF, int KIND>
__device__ __forceinline__ void group(const Args& a, const Group& g, int n, const float* cosv, const float* sinv,
                                      const int2* bs, const Row<T, LPR, VEC, HALF>& row) {
    using R = Row<T, LPR, VEC, HALF>;
    constexpr int NP = R::NP, NG = R::NG, U = 2;
    const int rows = n * g.H, mine = threadIdx.x / LPR;
    float wu[NP], ww[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) wu[i] = ww[i] = 1.f;
    if (KIND != kRotate && g.w) row.ld((const T*)g.w, true, wu, ww);
    const float inv_d = 1.0f / (float)a.D;
    for (int base = 0; base < rows; base += NG * U) {
        float u[U][NP], w[U][NP];
        int tt[U], h[U];
        bool live[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int r = base + k * NG + mine;
            live[k] = r < rows;
            token_head(g, min(r, rows - 1), tt[k], h[k]);
            row.ld((const T*)g.x + at(g.xs, bs[tt[k]], h[k]), live[k], u[k], w[k]);
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            float c[NP], s[NP], yu[NP], yw[NP];
            row.angles(cosv, sinv, tt[k], c, s);
            if constexpr (KIND == kNorm) {
                float s2 = 0.f;
#pragma unroll
                for (int i = 0; i < NP; ++i) s2 += u[k][i] * u[k][i] + w[k][i] * w[k][i];
                const float r = rsqrtf(R::sum(s2) * inv_d + a.eps);
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    u[k][i] *= r * wu[i];
                    w[k][i] *= r * ww[i];
                }
            }
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                yu[i] = row.turns(i) ? u[k][i] * c[i] - w[k][i] * s[i] : u[k][i];
                yw[i] = row.turns(i) ? w[k][i] * c[i] + u[k][i] * s[i] : w[k][i];
            }
            row.st((T*)g.y + at(g.ys, bs[tt[k]], h[k]), live[k], yu, yw);
        }
    }
}

// Backward: the next row's x and dy are loaded, as they lie in memory, before a row is worked on.
template <typename T, int LPR, bool VEC, bool HALF>
__device__ __forceinline__ void group_bwd(const Args& a, const Group& g, int n, const float* cosv, const float* sinv,
                                          const int2* bs, const Row<T, LPR, VEC, HALF>& row,
                                          float (&du)[Row<T, LPR, VEC, HALF>::NP],
                                          float (&dv)[Row<T, LPR, VEC, HALF>::NP]) {
    using R = Row<T, LPR, VEC, HALF>;
    constexpr int NP = R::NP, NG = R::NG;
    const int rows = n * g.H, mine = threadIdx.x / LPR;
    const float inv_d = 1.0f / (float)a.D;
    typename R::Raw x, dy, wr;
    int tt, h;
    row.raw((const T*)g.w, g.w != nullptr, wr);
    token_head(g, min(mine, rows - 1), tt, h);
    row.raw((const T*)g.x + at(g.xs, bs[tt], h), mine < rows, x);
    row.raw((const T*)g.dy + at(g.ds, bs[tt], h), mine < rows, dy);
    for (int base = 0; base < rows; base += NG) {
        const int r0 = base + mine, t0 = tt, h0 = h;
        float u[NP], w[NP], yu[NP], yw[NP];
        row.widen(x, u, w);
        {
            float gu[NP], gw[NP], c[NP], s[NP];
            row.widen(dy, gu, gw);
            if (base + NG < rows) {
                token_head(g, min(r0 + NG, rows - 1), tt, h);
                row.raw((const T*)g.x + at(g.xs, bs[tt], h), r0 + NG < rows, x);
                row.raw((const T*)g.dy + at(g.ds, bs[tt], h), r0 + NG < rows, dy);
            }
            row.angles(cosv, sinv, t0, c, s);
#pragma unroll
            for (int i = 0; i < NP; ++i) {  // dy turned back (sin carries the sign)
                yu[i] = row.turns(i) ? gu[i] * c[i] - gw[i] * s[i] : gu[i];
                yw[i] = row.turns(i) ? gw[i] * c[i] + gu[i] * s[i] : gw[i];
            }
        }
        float wu[NP], ww[NP], s2 = 0.f, sx = 0.f;
        row.widen(wr, wu, ww);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            if (!g.w) wu[i] = ww[i] = 1.f;
            s2 += u[i] * u[i] + w[i] * w[i];
            sx += wu[i] * yu[i] * u[i] + ww[i] * yw[i] * w[i];
        }
        s2 = R::sum(s2);
        sx = R::sum(sx);
        // lanes past the tile's rows hold zeros, and with eps 0 their r would be inf: nothing into dw
        const float r = r0 < rows ? rsqrtf(s2 * inv_d + a.eps) : 0.f, q = r * r * sx * inv_d;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            du[i] += yu[i] * u[i] * r;
            dv[i] += yw[i] * w[i] * r;
            yu[i] = r * (wu[i] * yu[i] - u[i] * q);
            yw[i] = r * (ww[i] * yw[i] - w[i] * q);
        }
        row.st((T*)g.y + at(g.ys, bs[t0], h0), r0 < rows, yu, yw);
    }
}

template <typename T, int LPR, bool VEC, bool HALF>
__device__ __forceinline__ void copy_group(const Group& g, int n, const int2* bs, const Row<T, LPR, VEC, HALF>& row) {
    using R = Row<T, LPR, VEC, HALF>;
    const int rows = n * g.H;
    for (int r = threadIdx.x / LPR; r < rows; r += R::NG) {
        int tt, h;
        token_head(g, r, tt, h);
        const T* src = (const T*)g.x + at(g.xs, bs[tt], h);
        T* dst = (T*)g.y + at(g.ys, bs[tt], h);
        if constexpr (VEC) {
            if (!row.on) continue;
            constexpr int Q = 8 * sizeof(T) / 16;
            uint4 v[2 * Q];
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                v[q] = reinterpret_cast<const uint4*>(src + row.c0)[q];
                v[Q + q] = reinterpret_cast<const uint4*>(src + row.c1)[q];
            }
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                reinterpret_cast<uint4*>(dst + row.c0)[q] = v[q];
                reinterpret_cast<uint4*>(dst + row.c1)[q] = v[Q + q];
            }
        } else {
#pragma unroll
            for (int i = 0; i < R::NP; ++i)
                if (row.has(i)) {
                    const T p = src[row.first(i)], q = src[row.second(i)];
                    dst[row.first(i)] = p;
                    dst[row.second(i)] = q;
                }
        }
    }
}

// A tile's places and angles
__device__ __forceinline__ void tile_angles(const Args& a, int t0, int n, float* cosv, float* sinv, int2* bs) {
    const int hr = a.rot >> 1;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const int b = (t0 + i) / a.S;
        bs[i] = make_int2(b, t0 + i - b * a.S);
    }
    for (int i = threadIdx.x; i < n * hr; i += kThreads) {
        const int tt = i / hr, p = i - tt * hr, b = (t0 + tt) / a.S, s = t0 + tt - b * a.S;
        const double pos = a.pos ? (double)a.pos[b * a.pos_sb + s] : (double)a.pos0 + s;
        const double turns = pos * (a.freqs[p] * 0.15915494309189533577);
        float sn, cs;
        sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
        cosv[i] = a.mscale * cs;
        sinv[i] = a.mscale * a.sgn * sn;
    }
    __syncthreads();
}

template <typename T, int LPR, bool VEC, bool HALF, int KIND>
__global__ __launch_bounds__(kThreads) void rope_kernel(Args a) {
    extern __shared__ __align__(16) unsigned char smem[];
    float* const cosv = reinterpret_cast<float*>(smem);
    float* const sinv = cosv + a.TB[0] * (a.rot >> 1);
    int2* const bs = reinterpret_cast<int2*>(sinv + a.TB[0] * (a.rot >> 1));
    const Row<T, LPR, VEC, HALF> row(a.D, a.rot);
    // a block past the last tile has no tokens (n below 1; it runs through without a test of its own, whose wait
    // for the arguments took 0.3 us of a token's 3.3)
    const unsigned first = (blockIdx.y * kTilesX + blockIdx.x) * (unsigned)a.TB[0];
    const int t0 = (int)first, n = min(a.TB[0], (int)((unsigned)a.tokens - first));
    tile_angles(a, t0, n, cosv, sinv, bs);
    group<T, LPR, VEC, HALF, KIND>(a, a.g[0], n, cosv, sinv, bs, row);
    if (KIND != kRotate && a.ng > 1) group<T, LPR, VEC, HALF, KIND>(a, a.g[1], n, cosv, sinv, bs, row);
    if (KIND != kRotate && a.copy.H) copy_group<T, LPR, VEC, HALF>(a.copy, n, bs, row);
}

// Backward: the first nq blocks take the queries, the others the keys and values (a block's dw is one
// weight's: half the registers of both), each walking over its tiles.  Three waves a SIMD: forward and
// backward of the 570 MB took 208 us, with the registers of four 212, of five (spilling) 416.
template <typename T, int LPR, bool VEC, bool HALF>
__global__ __launch_bounds__(kThreads, 3) void norm_bwd_kernel(Args a) {
    using R = Row<T, LPR, VEC, HALF>;
    constexpr int NP = R::NP, NG = R::NG;
    extern __shared__ __align__(16) unsigned char smem[];
    const int k = (int)blockIdx.x >= a.nq;
    const int TB = a.TB[k], first = k ? blockIdx.x - a.nq : blockIdx.x, step = k ? gridDim.x - a.nq : a.nq;
    float* const cosv = reinterpret_cast<float*>(smem);
    float* const sinv = cosv + TB * (a.rot >> 1);
    int2* const bs = reinterpret_cast<int2*>(sinv + TB * (a.rot >> 1));
    const R row(a.D, a.rot);
    float du[NP], dv[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) du[i] = dv[i] = 0.f;
    // unsigned: near 2^31 tiles the step past the last one is no int
    for (unsigned tile = first; tile < (unsigned)a.tiles[k]; tile += step) {
        const int t0 = (int)tile * TB, n = min(TB, a.tokens - t0);
        __syncthreads();  // the tile before has been read
        tile_angles(a, t0, n, cosv, sinv, bs);
        if (a.g[k].H) group_bwd<T, LPR, VEC, HALF>(a, a.g[k], n, cosv, sinv, bs, row, du, dv);
        if (k == a.with_copy && a.copy.H) copy_group<T, LPR, VEC, HALF>(a.copy, n, bs, row);
    }
    if (!a.part && !a.dw[k]) return;
    // the block's dw: its NG lane groups added in order
    float* const red = reinterpret_cast<float*>(smem);
    __syncthreads();
    float* mine = red + (threadIdx.x / LPR) * a.D;
#pragma unroll
    for (int i = 0; i < NP; ++i)
        if (row.has(i)) {
            mine[row.first(i)] = du[i];
            mine[row.second(i)] = dv[i];
        }
    __syncthreads();
    for (int j = threadIdx.x; j < a.D; j += kThreads) {
        float v = 0.f;
        for (int q = 0; q < NG; ++q) v += red[q * a.D + j];
        if (a.part) a.part[(size_t)blockIdx.x * a.D + j] = v;
        else a.dw[k][j] = a.accumulate ? a.dw[k][j] + v : v;
    }
}

// dw (+)= the sum of the partial rows, of the first nq blocks for q and of the others for k: 16 columns x
// 64 slices of the rows a block, the slices added in order (1536 rows: 4.5 us, a launch's time)
__global__ __launch_bounds__(1024) void dw_finish(const float* __restrict__ part, int nq, int nb, int D, float* dwq,
                                                  float* dwk, int accumulate) {
    __shared__ float sh[64][17];
    float* const dw = blockIdx.y ? dwk : dwq;
    if (!dw) return;
    const int c = threadIdx.x & 15, sl = threadIdx.x >> 4, j = blockIdx.x * 16 + c;
    const int end = blockIdx.y ? nb : nq;
    float v = 0.f;
    if (j < D) {
#pragma unroll 8
        for (int b = (blockIdx.y ? nq : 0) + sl; b < end; b += 64) v += part[(size_t)b * D + j];
    }
    sh[sl][c] = v;
    __syncthreads();
    if (threadIdx.x < 16 && j < D) {
        v = 0.f;
#pragma unroll
        for (int q = 0; q < 64; ++q) v += sh[q][c];
        dw[j] = accumulate ? dw[j] + v : v;
    }
}

// ---- host -------------------------------------------------------------------------------
constexpr int kMaxD = 512, kMaxH = 1024;
constexpr int kBwdBlocks = 1536;  // partial dw rows at most: two rounds of three blocks a compute unit
                                // (768, 1024, 2048: 209, 211, 208 us for 205)

int lanes_for(int D) {  // of a row in 16-byte pieces
    int l = 2;
    while (16 * l < D) l *= 2;
    return l;
}

constexpr int kBwd = 2;  // launch_kind: the backward

template <typename T, int LPR, bool VEC, bool HALF, int KIND>
int launch(const Args& a, int grid, size_t smem, hipStream_t s) {
    if constexpr (KIND == kBwd)
        hipLaunchKernelGGL((norm_bwd_kernel<T, LPR, VEC, HALF>), dim3(grid), dim3(kThreads), smem, s, a);
    else
        hipLaunchKernelGGL((rope_kernel<T, LPR, VEC, HALF, KIND>),
                           dim3(std::min(grid, kTilesX), (grid - 1) / kTilesX + 1), dim3(kThreads), smem, s, a);
    GN_LAUNCH_CHECK("rope / qk norm");
    return GN_OK;
}

template <typename T, bool HALF, int KIND>
int launch_lanes(const Args& a, bool vec, int grid, size_t smem, hipStream_t s) {
    if (!vec) return launch<T, 64, false, HALF, KIND>(a, grid, smem, s);
    switch (lanes_for(a.D)) {
        case 2: return launch<T, 2, true, HALF, KIND>(a, grid, smem, s);
        case 4: return launch<T, 4, true, HALF, KIND>(a, grid, smem, s);
        case 8: return launch<T, 8, true, HALF, KIND>(a, grid, smem, s);
        case 16: return launch<T, 16, true, HALF, KIND>(a, grid, smem, s);
        default: return launch<T, 32, true, HALF, KIND>(a, grid, smem, s);
    }
}

template <int KIND>
int launch_kind(const Args& a, int dtype, int mode, bool vec, int grid, size_t smem, hipStream_t s) {
    const bool half = mode == GN_ROPE_HALF;
    if (dtype == GN_F32)
        return half ? launch_lanes<float, true, KIND>(a, vec, grid, smem, s)
                    : launch_lanes<float, false, KIND>(a, vec, grid, smem, s);
    return half ? launch_lanes<bf16_t, true, KIND>(a, vec, grid, smem, s)
                : launch_lanes<bf16_t, false, KIND>(a, vec, grid, smem, s);
}

// the last element's offset + 1
int64_t span(const gn_heads& t, int B, int S, int D) {
    return (B - 1) * t.sb + (S - 1) * t.ss + (int64_t)(t.H - 1) * t.sh + D;
}

// Whether a and b may share an element.  Disjoint ranges do not; neither do parts of one buffer's
// rows (equal head, token or batch strides, the two blocks apart within the period).
bool overlap(const gn_heads& a, const gn_heads& b, int B, int S, int D, int es) {
    const char *pa = (const char*)a.p, *pb = (const char*)b.p;
    if (pa + span(a, B, S, D) * es <= pb || pb + span(b, B, S, D) * es <= pa) return false;
    const int64_t bytes = pb - pa;
    if (bytes % es) return true;
    auto apart = [&](int64_t period, int64_t ea, int64_t eb) {
        if (period <= 0 || ea > period || eb > period) return false;
        const int64_t d = ((bytes / es) % period + period) % period;
        return d >= ea && d + eb <= period;
    };
    const int64_t ha = (int64_t)(a.H - 1) * a.sh + D, hb = (int64_t)(b.H - 1) * b.sh + D;
    const bool same_b = B == 1 || a.sb == b.sb, same_s = S == 1 || a.ss == b.ss;
    const int64_t ps = S > 1 ? a.ss : B > 1 ? a.sb : 0;
    if (same_b && same_s && (S == 1 || B == 1 || a.sb % a.ss == 0) && apart(ps, ha, hb)) return false;
    const bool same_h = a.H == b.H && (a.H == 1 || a.sh == b.sh);
    if (same_b && same_s && same_h && a.H > 1 && a.sh > 0 && (S == 1 || a.ss % a.sh == 0) &&
        (B == 1 || a.sb % a.sh == 0) && apart(a.sh, D, D))
        return false;
    if (same_b && B > 1 && apart(a.sb, ha + (S - 1) * a.ss, hb + (S - 1) * b.ss)) return false;
    return true;
}

// Whether one of t's elements lies in [lo, hi): the heads' rows are searched by their strides, the largest
// first; of views that overlap themselves it may say so without one.
bool holds(const gn_heads& t, int B, int S, int D, int es, const void* lo, const void* hi) {
    if (!lo || t.H == 0 || B == 0 || S == 0) return false;
    const int64_t n[3] = {B, S, t.H}, st[3] = {t.sb * es, t.ss * es, t.sh * es};
    int order[3] = {0, 1, 2};
    std::sort(order, order + 3, [&](int i, int j) { return st[i] > st[j]; });
    int64_t inner[4];  // bytes that the dimensions from the k-th on span
    inner[3] = (int64_t)D * es;
    for (int k = 2; k >= 0; --k) inner[k] = inner[k + 1] + (n[order[k]] - 1) * st[order[k]];
    auto search = [&](auto& self, int k, const char* at) -> bool {
        if (at + inner[k] <= (const char*)lo || (const char*)hi <= at) return false;
        if (k == 3) return true;
        const int64_t s = st[order[k]], most = n[order[k]] - 1;
        if (s == 0 || most == 0) return self(self, k + 1, at);
        const int64_t before = (const char*)lo - at - inner[k + 1];  // i s > before, at + i s < hi
        const int64_t i0 = before < 0 ? 0 : before / s + 1, i1 = std::min(most, ((const char*)hi - at - 1) / s);
        if (i1 - i0 > 1024) return true;
        for (int64_t i = i0; i <= i1; ++i)
            if (self(self, k + 1, at + i * s)) return true;
        return false;
    };
    return search(search, 0, (const char*)t.p);
}

// whether an output's elements are all different ones
bool writable(const gn_heads& t, int B, int S, int D) {
    int64_t n[3] = {B, S, t.H}, st[3] = {t.sb, t.ss, t.sh};
    int order[3] = {0, 1, 2};
    std::sort(order, order + 3, [&](int i, int j) { return st[i] < st[j]; });
    int64_t ext = D;
    for (int i : order) {
        if (n[i] <= 1) continue;
        if (st[i] < ext) return false;
        ext += st[i] * (n[i] - 1);
    }
    return true;
}

bool same(const gn_heads& a, const gn_heads& b, int B, int S) {
    return a.p == b.p && (B == 1 || a.sb == b.sb) && (S == 1 || a.ss == b.ss) && (a.H == 1 || a.sh == b.sh);
}

bool pieces16(const gn_heads& t, int es) {  // every row starts at a multiple of 16 bytes
    return ((uintptr_t)t.p & 15u) == 0 && (t.sb * es) % 16 == 0 && (t.ss * es) % 16 == 0 && (t.sh * es) % 16 == 0;
}

int check_heads(const char* who, const char* name, const gn_heads* t, int es, bool any) {
    GN_REQUIRE(t->H >= 0 && t->H <= kMaxH, "%s: %s must have 0..%d heads", who, name, kMaxH);
    GN_REQUIRE(!any || t->H == 0 || t->p, "%s: %s is a null pointer", who, name);
    GN_REQUIRE(t->sb >= 0 && t->ss >= 0 && t->sh >= 0, "%s: %s has a negative stride", who, name);
    GN_REQUIRE(((uintptr_t)t->p & (es - 1)) == 0, "%s: %s is not aligned to its elements", who, name);
    return GN_OK;
}

struct Named {
    const gn_heads* t;
    const char* name;
};

// Memory of a call beside its heads: weights, frequencies, positions, weight gradients, the workspace
struct Flat {
    const void* p;
    int64_t bytes;
    const char* name;
    bool written;
};

// What is written may share no memory with anything else of the call.
int check_flat(const char* who, const Named* in, int ni, const Named* out, int no, const Flat* f, int nf, int B, int S,
               int D, int dtype) {
    const int es = dtype == GN_F32 ? 4 : 2;
    auto end = [](const Flat& x) { return (const char*)x.p + x.bytes; };
    for (int i = 0; i < nf; ++i) {
        if (!f[i].p || f[i].bytes <= 0) continue;
        for (int j = 0; j < no; ++j)
            GN_REQUIRE(!holds(*out[j].t, B, S, D, es, f[i].p, end(f[i])), "%s: %s shares memory with %s", who, out[j].name,
                       f[i].name);
        if (!f[i].written) continue;
        for (int j = 0; j < ni; ++j)
            GN_REQUIRE(!holds(*in[j].t, B, S, D, es, f[i].p, end(f[i])), "%s: %s shares memory with %s", who, f[i].name,
                       in[j].name);
        for (int j = 0; j < nf; ++j)
            GN_REQUIRE(j == i || !f[j].p || (const char*)f[j].p >= end(f[i]) || (const char*)f[i].p >= end(f[j]),
                       "%s: %s and %s may not share memory", who, f[i].name, f[j].name);
    }
    return GN_OK;
}

// the rotation's frequencies and positions
int add_rope(Flat* f, int n, const gn_rope* r, int B, int S) {
    if (!r || r->rot == 0) return n;
    f[n++] = {r->freqs, (int64_t)r->rot / 2 * 8, "freqs", false};
    f[n++] = {r->positions, ((int64_t)(B - 1) * r->pos_sb + S) * 4, "positions", false};
    return n;
}

// The shapes, the rotation and the tensors' places; fills a's common part.
int check(const char* who, const gn_rope* r, int B, int S, int D, int dtype, const Named* in, int ni, const Named* out,
          int no, const int* own, Args& a, bool& vec, int& mode) {
    GN_REQUIRE(dtype == GN_F32 || dtype == GN_BF16, "%s: dtype %d not supported (f32, bf16)", who, dtype);
    GN_REQUIRE(B >= 0 && S >= 0 && (int64_t)B * S < (1ll << 31), "%s: B * S must be below 2^31", who);
    GN_REQUIRE(D >= 2 && D <= kMaxD && D % 2 == 0, "%s: D must be even, 2..%d", who, kMaxD);
    const int rot = r ? r->rot : 0;
    mode = r && rot ? r->mode : GN_ROPE_HALF;
    if (rot) {
        GN_REQUIRE(rot > 0 && rot <= D && rot % 2 == 0, "%s: rot must be even, 0..D", who);
        GN_REQUIRE(mode == GN_ROPE_HALF || mode == GN_ROPE_INTERLEAVED, "%s: unknown rope mode %d", who, mode);
        GN_REQUIRE(r->freqs, "%s: freqs is a null pointer", who);
        GN_REQUIRE(r->pos_sb >= 0, "%s: positions have a negative stride", who);
        GN_REQUIRE(((uintptr_t)r->freqs & 7u) == 0 && ((uintptr_t)r->positions & 3u) == 0,
                   "%s: freqs or positions are not aligned to their elements", who);
    }
    const int es = dtype == GN_F32 ? 4 : 2;
    vec = D % 16 == 0 && rot % 16 == 0;
    for (int i = 0; i < ni; ++i) {
        if (const int rc = check_heads(who, in[i].name, in[i].t, es, B * S > 0)) return rc;
        vec = vec && pieces16(*in[i].t, es);
    }
    for (int i = 0; i < no; ++i) {
        if (const int rc = check_heads(who, out[i].name, out[i].t, es, B * S > 0)) return rc;
        vec = vec && pieces16(*out[i].t, es);
    }
    if (B * S > 0) {
        for (int i = 0; i < no; ++i) {
            if (out[i].t->H == 0) continue;
            GN_REQUIRE(writable(*out[i].t, B, S, D), "%s: %s overlaps itself", who, out[i].name);
            for (int j = 0; j < i; ++j)
                GN_REQUIRE(out[j].t->H == 0 || !overlap(*out[i].t, *out[j].t, B, S, D, es), "%s: %s overlaps %s", who,
                           out[i].name, out[j].name);
            for (int j = 0; j < ni; ++j)
                GN_REQUIRE(in[j].t->H == 0 || !overlap(*out[i].t, *in[j].t, B, S, D, es) ||
                               (own[j] == i && same(*out[i].t, *in[j].t, B, S)),
                           "%s: %s overlaps %s", who, out[i].name, in[j].name);
        }
    }
    a.freqs = rot ? r->freqs : nullptr;
    a.pos = rot ? r->positions : nullptr;
    a.pos_sb = rot ? r->pos_sb : 0;
    a.pos0 = rot ? r->pos0 : 0;
    a.mscale = rot ? r->mscale : 1.f;
    a.rot = rot;
    a.S = S;
    a.D = D;
    a.tokens = B * S;
    return GN_OK;
}

void fill(Group& g, const gn_heads* x, const gn_heads* dy, const void* w, const gn_heads* y) {
    auto strides = [](int64_t (&d)[3], const gn_heads* t) { d[0] = t->sb; d[1] = t->ss; d[2] = t->sh; };
    g.x = x->p;
    strides(g.xs, x);
    if (dy) {
        g.dy = dy->p;
        strides(g.ds, dy);
    }
    g.w = w;
    g.y = y->p;
    strides(g.ys, y);
    g.H = x->H;
    g.magic = g.H > 1 ? (uint32_t)(((1ull << 32) + g.H - 1) / g.H) : 0;
}

// Tokens of tile k: enough rows for `rounds` rounds of the block's lane groups (norms of 403 MB: two 78 us,
// four 83), cos and sin in 16 KB, and at least a thousand tiles (four blocks a compute unit) before a
// tile gets a second token.
void tile(Args& a, int k, int heads, int rows_at_once, int rounds) {
    int tb = std::max(1, rows_at_once * rounds / std::max(heads, 1));
    tb = std::min(tb, 64);
    if (a.rot) tb = std::min(tb, std::max(1, 4096 / a.rot));
    tb = std::min(tb, std::max(1, a.tokens / 1024));
    a.TB[k] = tb;
    a.tiles[k] = (int)(((int64_t)a.tokens + tb - 1) / tb);
}

size_t tile_smem(const Args& a) {
    const int tb = std::max(a.TB[0], a.TB[1]);
    return (size_t)tb * a.rot * 4 + (size_t)tb * 8;
}

int rope_call(const char* who, const gn_heads* x, const gn_heads* y, const gn_rope* r, int B, int S, int D, int dtype,
              float sgn, void* stream) {
    clear_error();
    GN_REQUIRE(x && y && r, "%s: null pointer", who);
    GN_REQUIRE(x->H == y->H, "%s: input and output differ in their heads", who);
    Args a{};
    bool vec;
    int mode;
    const Named in{x, "the input"}, out{y, "the output"};
    const int own = 0;
    if (const int rc = check(who, r, B, S, D, dtype, &in, 1, &out, 1, &own, a, vec, mode)) return rc;
    if (a.tokens == 0 || x->H == 0) return GN_OK;
    Flat flat[2];
    if (const int rc = check_flat(who, &in, 1, &out, 1, flat, add_rope(flat, 0, r, B, S), B, S, D, dtype)) return rc;
    fill(a.g[0], x, nullptr, nullptr, y);
    a.ng = 1;
    a.sgn = sgn;
    tile(a, 0, x->H, 2 * kThreads / (vec ? lanes_for(D) : 64), 2);
    return launch_kind<kRotate>(a, dtype, mode, vec, a.tiles[0], tile_smem(a), as_stream(stream));
}

}  // namespace
}  // namespace gn

using namespace gn;

extern "C" int gn_rope_freqs(int rot, double theta, int scaling, double factor, double trained, double fast, double slow,
                             double* freqs, float* mscale) {
    clear_error();
    GN_REQUIRE(rot >= 0 && rot % 2 == 0 && rot <= kMaxD, "gn_rope_freqs: rot must be even, 0..%d", kMaxD);
    GN_REQUIRE(theta > 0 && std::isfinite(theta), "gn_rope_freqs: theta must be positive");
    GN_REQUIRE((freqs || rot == 0) && mscale, "gn_rope_freqs: null pointer");
    GN_REQUIRE(scaling >= GN_ROPE_SCALE_NONE && scaling <= GN_ROPE_SCALE_YARN, "gn_rope_freqs: unknown scaling %d", scaling);
    if (scaling != GN_ROPE_SCALE_NONE)
        GN_REQUIRE(factor >= 1 && std::isfinite(factor), "gn_rope_freqs: factor must be at least 1");
    if (scaling == GN_ROPE_SCALE_YARN)
        GN_REQUIRE(trained > 0 && fast > slow && std::isfinite(trained) && std::isfinite(fast) && std::isfinite(slow),
                   "gn_rope_freqs: YARN needs trained > 0 and fast > slow");
    *mscale = scaling == GN_ROPE_SCALE_YARN ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    // rot = 2 has the one pair of frequency 1: no base slows it
    const double base = scaling == GN_ROPE_SCALE_NTK && rot > 2 ? theta * std::pow(factor, rot / (rot - 2.0)) : theta;
    for (int i = 0; i < rot / 2; ++i) {
        double f = std::pow(base, -2.0 * i / rot);
        if (scaling == GN_ROPE_SCALE_LINEAR) f /= factor;
        if (scaling == GN_ROPE_SCALE_YARN) {
            const double turns = trained * f * 0.15915494309189533577;
            const double keep = std::min(1.0, std::max(0.0, (turns - slow) / (fast - slow)));
            f = f * keep + f / factor * (1.0 - keep);
        }
        freqs[i] = f;
    }
    return GN_OK;
}

extern "C" int gn_rope_fwd(const gn_heads* x, const gn_heads* y, const gn_rope* rope, int B, int S, int D, int dtype,
                           void* stream) {
    return rope_call("gn_rope_fwd", x, y, rope, B, S, D, dtype, 1.f, stream);
}

extern "C" int gn_rope_bwd(const gn_heads* dy, const gn_heads* dx, const gn_rope* rope, int B, int S, int D, int dtype,
                           void* stream) {
    return rope_call("gn_rope_bwd", dy, dx, rope, B, S, D, dtype, -1.f, stream);
}

extern "C" int gn_qk_norm_rope_fwd(const gn_heads* q, const gn_heads* k, const gn_heads* v, const void* wq,
                                   const void* wk, const gn_heads* yq, const gn_heads* yk, const gn_heads* yv,
                                   const gn_rope* rope, int B, int S, int D, float eps, int dtype, void* stream) {
    const char* who = "gn_qk_norm_rope_fwd";
    clear_error();
    GN_REQUIRE(q && yq && !k == !yk && !v == !yv, "%s: null pointer", who);
    GN_REQUIRE(q->H == yq->H && (!k || k->H == yk->H) && (!v || v->H == yv->H), "%s: input and output differ in their heads", who);
    GN_REQUIRE(!k || !v || k->H == v->H, "%s: k and v differ in their heads", who);
    GN_REQUIRE(eps >= 0 && std::isfinite(eps), "%s: eps must not be negative", who);
    Named in[3], out[3];
    int own[3], n = 0;
    auto add = [&](const gn_heads* x, const char* xn, const gn_heads* y, const char* yn) {
        in[n] = {x, xn};
        out[n] = {y, yn};
        own[n] = n;
        ++n;
    };
    add(q, "q", yq, "yq");
    if (k) add(k, "k", yk, "yk");
    if (v) add(v, "v", yv, "yv");
    Args a{};
    bool vec;
    int mode;
    if (const int rc = check(who, rope, B, S, D, dtype, in, n, out, n, own, a, vec, mode)) return rc;
    const int es = dtype == GN_F32 ? 4 : 2;
    GN_REQUIRE((((uintptr_t)wq | (uintptr_t)wk) & (es - 1)) == 0, "%s: the weights are not aligned to their elements", who);
    vec = vec && (((uintptr_t)wq | (uintptr_t)wk) & 15u) == 0;
    const int heads = q->H + (k ? k->H : 0) + (v ? v->H : 0);
    if (a.tokens == 0 || heads == 0) return GN_OK;
    Flat flat[4] = {{wq, (int64_t)D * es, "wq", false}, {wk, (int64_t)D * es, "wk", false}};
    if (const int rc = check_flat(who, in, n, out, n, flat, add_rope(flat, 2, rope, B, S), B, S, D, dtype)) return rc;
    fill(a.g[0], q, nullptr, wq, yq);
    if (k) fill(a.g[1], k, nullptr, wk, yk);
    if (v) fill(a.copy, v, nullptr, nullptr, yv);
    a.ng = k ? 2 : 1;
    a.sgn = 1.f;
    a.eps = eps;
    tile(a, 0, heads, 2 * kThreads / (vec ? lanes_for(D) : 64), 2);
    return launch_kind<kNorm>(a, dtype, mode, vec, a.tiles[0], tile_smem(a), as_stream(stream));
}

extern "C" size_t gn_qk_norm_rope_workspace_bytes(int B, int S, int D) {
    if (B <= 0 || S <= 0 || D <= 0) return 0;
    return (size_t)std::min<int64_t>(kBwdBlocks, 2 * (int64_t)B * S) * D * sizeof(float);
}

extern "C" int gn_qk_norm_rope_bwd(const gn_heads* dyq, const gn_heads* dyk, const gn_heads* dyv, const gn_heads* q,
                                   const gn_heads* k, const void* wq, const void* wk, const gn_heads* dq,
                                   const gn_heads* dk, const gn_heads* dv, float* dwq, float* dwk, const gn_rope* rope,
                                   int B, int S, int D, float eps, int dtype, unsigned flags, void* ws, size_t ws_bytes,
                                   void* stream) {
    const char* who = "gn_qk_norm_rope_bwd";
    clear_error();
    GN_REQUIRE(q && dyq && dq && !k == !dyk && !k == !dk && !dyv == !dv, "%s: null pointer", who);
    GN_REQUIRE(!dwk || k, "%s: dwk without k", who);
    GN_REQUIRE(q->H == dyq->H && q->H == dq->H && (!k || (k->H == dyk->H && k->H == dk->H)) && (!dv || dv->H == dyv->H),
               "%s: inputs and outputs differ in their heads", who);
    GN_REQUIRE(!k || !dv || k->H == dv->H, "%s: k and v differ in their heads", who);
    GN_REQUIRE(eps >= 0 && std::isfinite(eps), "%s: eps must not be negative", who);
    GN_REQUIRE((flags & ~GN_ACCUMULATE) == 0, "%s: unknown flags", who);
    Named in[5], out[3];
    int own[5], ni = 0, no = 0;
    auto add = [&](const gn_heads* dy, const char* dyn, const gn_heads* x, const char* xn, const gn_heads* dx, const char* dxn) {
        in[ni] = {dy, dyn};
        own[ni++] = no;
        if (x) {
            in[ni] = {x, xn};
            own[ni++] = no;
        }
        out[no++] = {dx, dxn};
    };
    add(dyq, "dyq", q, "q", dq, "dq");
    if (k) add(dyk, "dyk", k, "k", dk, "dk");
    if (dv) add(dyv, "dyv", nullptr, "", dv, "dv");
    Args a{};
    bool vec;
    int mode;
    if (const int rc = check(who, rope, B, S, D, dtype, in, ni, out, no, own, a, vec, mode)) return rc;
    const int es = dtype == GN_F32 ? 4 : 2;
    GN_REQUIRE((((uintptr_t)wq | (uintptr_t)wk) & (es - 1)) == 0, "%s: the weights are not aligned to their elements", who);
    GN_REQUIRE((((uintptr_t)dwq | (uintptr_t)dwk) & 3u) == 0, "%s: dwq, dwk must be aligned to 4 bytes", who);
    GN_REQUIRE(!dwq || !dwk || dwq + D <= dwk || dwk + D <= dwq, "%s: dwq and dwk may not share memory", who);
    vec = vec && (((uintptr_t)wq | (uintptr_t)wk) & 15u) == 0;
    hipStream_t s = as_stream(stream);
    const bool acc = flags & GN_ACCUMULATE;
    const int heads = q->H + (k ? k->H : 0) + (dv ? dv->H : 0);
    if (a.tokens == 0 || heads == 0) {
        if (!acc && ((dwq && launch_zero(dwq, (size_t)D * 4, s) != hipSuccess) ||
                     (dwk && launch_zero(dwk, (size_t)D * 4, s) != hipSuccess))) {
            set_error("%s: clear failed", who);
            return GN_E_HIP;
        }
        return GN_OK;
    }
    fill(a.g[0], q, dyq, wq, dq);
    if (k) fill(a.g[1], k, dyk, wk, dk);
    if (dv) fill(a.copy, dyv, nullptr, nullptr, dv);
    a.ng = k ? 2 : 1;
    a.sgn = -1.f;
    a.eps = eps;
    a.accumulate = acc;
    const int at_once = kThreads / (vec ? lanes_for(D) : 64);
    // the blocks by the bytes of each side: two reads and a write a row of q and k, one each of v; as
    // with values also without them, so that dw has the same bits either way
    const int hk = k ? k->H : 0, hv = dv ? dv->H : 0;
    const bool second = hk > 0;  // values without keys go with the queries
    a.with_copy = second;
    tile(a, 0, q->H + (second ? 0 : hv), at_once, 4);
    if (second) tile(a, 1, 2 * hk, at_once, 4);
    int grid = std::min(a.tiles[0] + a.tiles[1], kBwdBlocks);
    a.nq = grid;
    if (second) {
        const double share = 3.0 * q->H / (3.0 * q->H + 5.0 * hk);
        a.nq = std::min(a.tiles[0], std::max(1, std::min(grid - 1, (int)(share * grid + 0.5))));
        grid = a.nq + std::min(a.tiles[1], grid - a.nq);
    }
    if ((dwq && a.nq > 1) || (dwk && grid - a.nq > 1)) {
        const size_t need = (size_t)grid * D * sizeof(float);
        if (!ws || ws_bytes < need || ((uintptr_t)ws & 15u)) {
            set_error("%s: workspace of %zu bytes (16-byte aligned) required", who, need);
            return GN_E_WORKSPACE;
        }
        a.part = (float*)ws;
    }
    Flat flat[7] = {{wq, (int64_t)D * es, "wq", false},
                    {wk, (int64_t)D * es, "wk", false},
                    {dwq, (int64_t)D * 4, "dwq", true},
                    {dwk, (int64_t)D * 4, "dwk", true},
                    {a.part, (int64_t)grid * D * 4, "the workspace", true}};
    if (const int rc = check_flat(who, in, ni, out, no, flat, add_rope(flat, 5, rope, B, S), B, S, D, dtype)) return rc;
    a.dw[0] = dwq;
    a.dw[1] = dwk;
    if (dwk && !second && !acc && launch_zero(dwk, (size_t)D * 4, s) != hipSuccess) {  // keys without heads
        set_error("%s: clear failed", who);
        return GN_E_HIP;
    }
    const size_t smem = std::max(tile_smem(a), (size_t)at_once * D * sizeof(float));
    if (const int rc = launch_kind<kBwd>(a, dtype, mode, vec, grid, smem, s)) return rc;
    if (a.part) {
        dw_finish<<<dim3((D + 15) / 16, 2), 1024, 0, s>>>(a.part, a.nq, grid, D, dwq, second ? dwk : nullptr, acc);
        GN_LAUNCH_CHECK("qk norm weight gradients");
    }
    return GN_OK;
}
