// gn_residual.hip — a block's residual branch: dropout from a counter-based generator, and the norm after
// a block, its dropout, gate and scale, the residual sum and the norm before the next block in one pass,
// forward and backward.
//
//   forward    n = post(h),  y = res_scale x + scale gate drop(n),  z = pre(y)
//   backward   dY = dy + pre'(dz; y),  dx = res_scale dY,  e = scale drop(dY)  (the same mask),
//              dgate = sum e n,  dn = gate e,  dh = post'(dn; h)
//   a norm     v^ = (v - mu) r,  r = rsqrt(mean (v - mu)^2 + eps)  (mu = 0: RMS),  out = v^ w + b
//   its gradient at d with g = w d:  r (g - mean g - v^ mean(g v^))  (RMS: without mean g),
//              dw = sum d v^,  db = sum d
//
// Everything is read once and written once, so HBM bounds the passes.  A row of up to 8192 elements belongs
// to 1 to 8 waves whose lanes hold it in registers, 8 or 16 elements each, between its loads and its stores;
// the next row's loads are under way meanwhile.  Row sums are DPP moves within a wave and one
// exchange through LDS, with one barrier, between waves.  Weights stay in registers over a block's rows.
// The backward's sums over rows stay in registers too (fp32), are added over a block's rows of waves in
// LDS, and leave as one partial row a block, which a second launch adds in a fixed order: no atomics.
// Wider rows are read three times or more (kernels at the end).
//
// Measured (us; a large copy reaches 5.1 to 5.2 TB/s on the card, reads alone 6.0): dropout of 8192 x 5632 bf16 34.9, 5.3 TB/s; forward
// 8192 x 768, dropout, LayerNorm before the next block, fp32 stream 14.0, 5.4 TB/s, and 16001 x 4096 bf16, two RMS norms and a gate 96, 5.5;
// backward of the first, which without a norm after the block or a gate does not read h, 25.2, 4.0 TB/s, of the second 178, 4.4: 4 us of
// either are the second launch, and what the loads ahead do not cover of two or three dependent sums a row is the rest (with an
// RMS norm after the block the first takes 15.9 and 35.6).  Rows that vectors do not divide hold an element's mask word each, not
// eight elements' four: 2107 x 1027 fp32 backward 33, 1.6 TB/s; its waves, two a SIMD, compute 28 % of their time and wait for loads
// and the sums' barriers 44 %.  A token's row costs its launch: 3.7 of 9.4 with the call.  Past 8192 elements the passes are far from HBM's
// rate: 4096 x 12288 bf16 with two RMS norms 342 forward, 908 backward (4096 x 8192: 51, 99).
#include <algorithm>
#include <type_traits>

#include "gn_common.h"
#include "gn_rng.h"

namespace gn {
namespace {

inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// ---- dropout ---------------------------------------------------------------------------------
// A lane takes two pieces of eight elements, 256 pieces apart, so that both loads are under way before the
// first mask is formed; ACC adds onto Y.
template <typename T, bool ACC>
__global__ __launch_bounds__(256) void dropout_vec(const T* X, T* Y, int64_t n, Mask m) {
    const int64_t nvec = n >> 3, c0 = (int64_t)blockIdx.x * 512 + threadIdx.x;
    const uint64_t key = m.key();
    float v[2][8];
#pragma unroll
    for (int k = 0; k < 2; ++k)
        if (c0 + 256 * k < nvec) chunk8<T>::ld(X + 8 * (c0 + 256 * k), v[k]);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int64_t c = c0 + 256 * k;
        if (c >= nvec) continue;
        drop8(v[k], key, 8 * (uint64_t)c, m.t, m.keep);
        if constexpr (ACC) {
            float o[8];
            chunk8<T>::ld(Y + 8 * c, o);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[k][e] += o[e];
        }
        chunk8<T>::st(Y + 8 * c, v[k]);
    }
    // the last n % 8 elements
    if (blockIdx.x == 0 && (int64_t)threadIdx.x < n - 8 * nvec) {
        const int64_t i = 8 * nvec + threadIdx.x;
        const float d = drop1(io<T>::ld(X, i), key, (uint64_t)i, m.t, m.keep);
        io<T>::st(Y, i, ACC ? d + io<T>::ld(Y, i) : d);
    }
}

template <typename T, bool ACC>
__global__ __launch_bounds__(256) void dropout_one(const T* X, T* Y, int64_t n, Mask m) {
    const uint64_t key = m.key();
    for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const float d = drop1(io<T>::ld(X, i), key, (uint64_t)i, m.t, m.keep);
        io<T>::st(Y, i, ACC ? d + io<T>::ld(Y, i) : d);
    }
}

template <typename T, bool ACC>
int dropout_launch(const void* X, void* Y, int64_t n, const Mask& m, hipStream_t s) {
    const int64_t blocks = ((n >> 3) + 511) / 512;
    if (al16(X) && al16(Y) && grid_fits(blocks, 256))
        dropout_vec<T, ACC><<<(unsigned)std::max<int64_t>(blocks, 1), 256, 0, s>>>((const T*)X, (T*)Y, n, m);
    else
        dropout_one<T, ACC><<<grid_for(n, 256, 16384), 256, 0, s>>>((const T*)X, (T*)Y, n, m);
    GN_LAUNCH_CHECK("gn_dropout");
    return GN_OK;
}

// [p, p + np) and [q, q + nq) have bytes in common
bool share(const void* p, size_t np, const void* q, size_t nq) {
    return p && q && (const char*)p < (const char*)q + nq && (const char*)q < (const char*)p + np;
}

int dropout(const char* who, const void* X, void* Y, int64_t n, double p, const gn_rng* rng, int dtype, bool acc,
            hipStream_t s) {
    clear_error();
    GN_REQUIRE(n >= 0 && n < (1ll << 56), "%s: %lld elements", who, (long long)n);
    GN_REQUIRE(dtype == GN_F32 || dtype == GN_BF16, "%s: dtype %d not supported (f32, bf16)", who, dtype);
    Mask m;
    GN_REQUIRE(make_mask(rng, p, &m), "%s: p must be at least 0 and below 1", who);
    GN_REQUIRE(rng || p == 0.0, "%s: no generator", who);
    GN_REQUIRE(((uintptr_t)m.step_dev & 7u) == 0, "%s: step_dev is not aligned to 8 bytes", who);
    if (n == 0) return GN_OK;
    GN_REQUIRE(X && Y, "%s: null pointer", who);
    const size_t es = dtype == GN_F32 ? 4 : 2;
    GN_REQUIRE((((uintptr_t)X | (uintptr_t)Y) & (es - 1)) == 0, "%s: a tensor is not aligned to its elements", who);
    GN_REQUIRE((X == Y && !acc) || !share(X, n * es, Y, n * es), "%s: input and output may not share memory%s", who,
               acc ? "" : " but as a whole");
    GN_REQUIRE(!share(m.step_dev, 8, Y, n * es), "%s: step_dev and the output may not share memory", who);
    if (dtype == GN_BF16)
        return acc ? dropout_launch<bf16_t, true>(X, Y, n, m, s) : dropout_launch<bf16_t, false>(X, Y, n, m, s);
    return acc ? dropout_launch<float, true>(X, Y, n, m, s) : dropout_launch<float, false>(X, Y, n, m, s);
}

// ---- rows in registers -----------------------------------------------------------------------
constexpr int kMaxF = 8192;  // elements of a row that a block's lanes hold

// Which of a row's F elements a lane has: VEC in pieces of eight (16-byte accesses), else singly, a whole
// wave side by side.
template <int T, int NC, bool VEC>
struct Cols {
    int t, F;
    __device__ __forceinline__ int at(int j, int e) const { return VEC ? 8 * (t + T * j) + e : t + T * (8 * j + e); }
    __device__ __forceinline__ bool has(int j, int e) const { return at(j, VEC ? 0 : e) < F; }
    // the place of element e in a row p: the wave's address and 32 bits of the lane's, without a vector instruction
    template <typename E>
    __device__ __forceinline__ E* in(E* p, int j, int e) const {
        using B = std::conditional_t<std::is_const_v<E>, const char, char>;
        return reinterpret_cast<E*>(reinterpret_cast<B*>(p) + (uint32_t)at(j, e) * (uint32_t)sizeof(E));
    }
};

// Eight elements of a lane as they lie in memory (bf16 stays packed until it is used).
template <typename T, bool VEC> struct Raw;
template <bool VEC> struct Raw<float, VEC> {
    float v[8];
    template <typename C>
    __device__ __forceinline__ void load(const float* p, const C& c, int j) {
        if constexpr (VEC) {
            if (c.has(j, 0)) { chunk8<float>::ld(c.in(p, j, 0), v); return; }
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.f;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = c.has(j, e) ? *c.in(p, j, e) : 0.f;
        }
    }
    template <typename C>
    __device__ __forceinline__ void fill(float x, const C& c, int j) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c.has(j, e) ? x : 0.f;
    }
    __device__ __forceinline__ float operator[](int e) const { return v[e]; }
};
template <bool VEC> struct Raw<bf16_t, VEC> {
    uint32_t w[4];
    template <typename C>
    __device__ __forceinline__ void load(const bf16_t* p, const C& c, int j) {
        if constexpr (VEC) {
            uint4 x = make_uint4(0u, 0u, 0u, 0u);
            if (c.has(j, 0)) x = *reinterpret_cast<const uint4*>(c.in(p, j, 0));
            w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
        } else {
            uint32_t q[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) q[e] = c.has(j, e) ? (uint32_t)*c.in(p, j, e) : 0u;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = q[2 * e] | (q[2 * e + 1] << 16);
        }
    }
    template <typename C>
    __device__ __forceinline__ void fill(float x, const C& c, int j) {
        const uint32_t b = __float_as_uint(x) >> 16;  // (0 and 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (c.has(j, 2 * e) ? b : 0u) | (c.has(j, 2 * e + 1) ? b << 16 : 0u);
    }
    __device__ __forceinline__ float operator[](int e) const {
        return __uint_as_float((e & 1) ? (w[e >> 1] & 0xffff0000u) : (w[e >> 1] << 16));
    }
};

template <typename T, bool VEC, typename C>
__device__ __forceinline__ void store8(T* p, const C& c, int j, const float (&v)[8]) {
    if constexpr (VEC) {
        if (c.has(j, 0)) chunk8<T>::st(c.in(p, j, 0), v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c.has(j, e)) io<T>::st(c.in(p, j, e), 0, v[e]);
    }
}

template <bool VEC, typename C, typename F = NoMore>
__device__ __forceinline__ void drop_piece(float (&v)[8], const C& c, int j, uint64_t key, uint64_t row0, const Mask& m, F&& f = F{}) {
    if constexpr (VEC) {
        drop8(v, key, row0 + (uint64_t)c.at(j, 0), m.t, m.keep, f);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            v[e] = drop1(v[e], key, row0 + (uint64_t)c.at(j, e), m.t, m.keep, [&](int, bool kept) { f(e, kept); });
    }
}

// The sum of a wave's lanes, in lane 63: within rows of 16 lanes as wave_sum (gn_common.h), then row 0 onto row 1 and
// row 2 onto row 3 (row_bcast15), then the lower half onto the upper (row_bcast31).
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ float wave_total(float v) {
    v = dpp_add<0xB1, 0xF>(v);
    v = dpp_add<0x4E, 0xF>(v);
    v = dpp_add<0x141, 0xF>(v);
    v = dpp_add<0x140, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);
    return dpp_add<0x143, 0xC>(v);
}

// Sums of N values over the lanes of a row.  Rows of several waves exchange theirs through one of two
// LDS buffers in turn: a wave that writes a buffer again has passed the barrier of the sum in between,
// which every wave reached after its reads of it.  Lane l reads the sums of wave l % WPR, and DPP moves among WPR
// lanes add them up: one LDS read, whatever the number of waves.
template <int WPR>
struct RowSum {
    float4 (*buf)[WPR][2];  // [2]
    int wave, lane, turn;
    template <int N>
    __device__ __forceinline__ void operator()(float (&v)[N]) {
        static_assert(N <= 8, "buffer");
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = wave_total(v[k]);
        if constexpr (WPR == 1) {
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] = lane_f(v[k], 63);
        } else {
            auto value = [&](int k) { return k < N ? v[k < N ? k : 0] : 0.f; };
            if (lane == 63) {
                buf[turn][wave][0] = make_float4(value(0), value(1), value(2), value(3));
                if constexpr (N > 4) buf[turn][wave][1] = make_float4(value(4), value(5), value(6), value(7));
            }
            __syncthreads();
            const float4 w = buf[turn][lane & (WPR - 1)][0], x = N > 4 ? buf[turn][lane & (WPR - 1)][1] : w;
            const float u[8] = {w.x, w.y, w.z, w.w, x.x, x.y, x.z, x.w};
#pragma unroll
            for (int k = 0; k < N; ++k) {
                v[k] = dpp_add<0xB1, 0xF>(u[k]);
                if constexpr (WPR > 2) v[k] = dpp_add<0x4E, 0xF>(v[k]);
                if constexpr (WPR > 4) v[k] = dpp_add<0x141, 0xF>(v[k]);
            }
            turn ^= 1;
        }
    }
};

template <typename TX, typename TH>
struct FwdArgs {
    const TH *h, *post_w, *post_b, *pre_w, *pre_b, *gate;
    const TX* x;
    TX* y;
    TH* z;
    int rows, F, gates, gate_rows, post, pre;
    float scale, res_scale, post_eps, pre_eps;
    Mask mask;
};

// The statistics of a row v (0 in the places that it does not have): mu and r.
template <int NC, typename C, typename SUM>
__device__ __forceinline__ void row_stats(const float (&v)[NC][8], int kind, float eps, const C& c, SUM& sum, float& mu,
                                          float& r) {
    mu = 0.f;
    r = 1.f;
    if (kind == GN_NORM_NONE) return;
    const float inv = 1.0f / (float)c.F;
    if (kind == GN_NORM_LAYER) {
        float s[1] = {0.f};
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) s[0] += v[j][e];
        sum(s);
        mu = s[0] * inv;
    }
    float q[1] = {0.f};
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float d = c.has(j, e) ? v[j][e] - mu : 0.f;
            q[0] += d * d;
        }
    sum(q);
    r = rsqrtf(q[0] * inv + eps);
}

template <typename TX, typename TH, int WPR, int NC, bool VEC>
__global__ __launch_bounds__(WPR == 1 ? 256 : 64 * WPR) void residual_fwd(FwdArgs<TX, TH> a) {
    constexpr int T = 64 * WPR, RPB = WPR == 1 ? 4 : 1;  // rows of a block at a time
    __shared__ float4 buf[2][WPR][2];
    const Cols<T, NC, VEC> c{(int)threadIdx.x & (T - 1), a.F};
    RowSum<WPR> sum{buf, (int)(threadIdx.x >> 6) & (WPR - 1), (int)threadIdx.x & 63, 0};
    const uint64_t key = a.mask.t ? a.mask.key() : 0;

    Raw<TH, VEC> wp[NC], bp[NC], wn[NC], bn[NC], gate[NC];
#pragma unroll
    for (int j = 0; j < NC; ++j) {
        auto weights = [&](Raw<TH, VEC>& to, const TH* p, float absent) {
            if (p) to.load(p, c, j);
            else to.fill(absent, c, j);
        };
        weights(wp[j], a.post_w, 1.f);
        weights(bp[j], a.post_b, 0.f);
        weights(wn[j], a.pre_w, 1.f);
        weights(bn[j], a.pre_b, 0.f);
        weights(gate[j], a.gate, 1.f);
    }
    int at_gate = 0;

    const int64_t stride = (int64_t)gridDim.x * RPB;
    int64_t r = (int64_t)blockIdx.x * RPB + (WPR == 1 ? __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) : 0);
    Raw<TH, VEC> h[NC];
    Raw<TX, VEC> x[NC];
    auto load = [&](int64_t row, Raw<TH, VEC> (&hh)[NC], Raw<TX, VEC> (&xx)[NC]) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            hh[j].load(a.h + row * a.F, c, j);
            xx[j].load(a.x + row * a.F, c, j);
        }
    };
    if (r < a.rows) load(r, h, x);
    while (r < a.rows) {  // the same number of rows for all waves of one
        const int64_t next = r + stride;
        Raw<TH, VEC> hn[NC];
        Raw<TX, VEC> xn[NC];
        if (next < a.rows) load(next, hn, xn);
        if (a.gates > 1) {
            const int g = (int)r / a.gate_rows;
            if (g != at_gate) {
                at_gate = g;
#pragma unroll
                for (int j = 0; j < NC; ++j) gate[j].load(a.gate + (size_t)g * a.F, c, j);
            }
        }
        float v[NC][8], mu, rs;
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[j][e] = h[j][e];
        row_stats<NC>(v, a.post, a.post_eps, c, sum, mu, rs);
#pragma unroll
        for (int j = 0; j < NC; ++j) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[j][e] = (v[j][e] - mu) * rs * wp[j][e] + bp[j][e];
            if (a.mask.t) drop_piece<VEC>(v[j], c, j, key, (uint64_t)r * a.F, a.mask);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[j][e] = a.res_scale * x[j][e] + a.scale * gate[j][e] * v[j][e];
            store8<TX, VEC>(a.y + r * a.F, c, j, v[j]);
        }
        if (a.pre != GN_NORM_NONE) {
            row_stats<NC>(v, a.pre, a.pre_eps, c, sum, mu, rs);
#pragma unroll
            for (int j = 0; j < NC; ++j) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[j][e] = (v[j][e] - mu) * rs * wn[j][e] + bn[j][e];
                store8<TH, VEC>(a.z + r * a.F, c, j, v[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < NC; ++j) { h[j] = hn[j]; x[j] = xn[j]; }
        r = next;
    }
}

// ---- backward ------------------------------------------------------------------------------
// Planes of partial sums: the parameters' gradients, each [blocks][F].
enum Plane { kGate, kPostW, kPostB, kPreW, kPreB, kPlanes };

// How the rows go to blocks: each of `groups` (the gate's, where its gradient is wanted and has rows to add
// up) to `per` blocks, or, with more groups than blocks (per 0), whole groups to a block.
struct Split {
    int groups, group_rows, per, blocks;
    // the groups of block b, and its rows of one of them
    __host__ __device__ __forceinline__ void of(int b, int& g0, int& g1) const {
        g0 = per ? b / per : (int)((int64_t)groups * b / blocks);
        g1 = per ? g0 + 1 : (int)((int64_t)groups * (b + 1) / blocks);
    }
    __host__ __device__ __forceinline__ void rows(int b, int g, int& r0, int& r1) const {
        const int k = per ? b % per : 0, n = per ? per : 1;
        r0 = g * group_rows + (int)((int64_t)group_rows * k / n);
        r1 = g * group_rows + (int)((int64_t)group_rows * (k + 1) / n);
    }
};

template <typename TX, typename TH>
struct BwdArgs {
    const TX *dy, *y;
    const TH *dz, *h, *post_w, *post_b, *pre_w, *gate;
    TH* dh;
    TX* dx;
    float* grad[kPlanes];  // nullptr: not wanted
    float* part;           // [plane][blocks][F]; unused planes too
    float* stats;          // wide rows: [rows][8]
    int rows, F, gates, gate_rows, post, pre, accumulate;
    float scale, res_scale, post_eps, pre_eps;
    Mask mask;
    Split split;
};

// The backward of one norm at its statistics: u = mean g, w = mean g v^ (u = 0: RMS), in the row's sums
// a = sum g, b = sum g (v - mu).
__device__ __forceinline__ float norm_grad(float g, float vc, float r, float u, float w) {
    return r * (g - u - vc * (r * w));
}

// Eight weights of a lane: as they lie in memory, or as floats times a factor.
template <typename T, bool VEC, bool FLOATS>
struct Weights : Raw<std::conditional_t<FLOATS, float, T>, VEC> {
    template <typename C>
    __device__ __forceinline__ void set(const T* p, float absent, float factor, const C& c, int j) {
        if constexpr (FLOATS) {
            Raw<T, VEC> r;
            if (p) r.load(p, c, j);
            else r.fill(absent, c, j);
#pragma unroll
            for (int e = 0; e < 8; ++e) this->v[e] = r[e] * factor;
        } else {
            if (p) this->load(p, c, j);
            else this->fill(absent, c, j);
        }
    }
};

// POST: there is a norm after the block; LAYER: a LayerNorm among the norms (biases and means); GATE: the
// gate's gradient is wanted.  Between a row's loads and its stores are two or three sums with barriers, which
// something has to hide.  Where the registers of a wave leave room for four a SIMD, that is a second block a
// CU (two_blocks); where there are three sums over rows or fewer, a wave works on two rows side by side (RP), whose sums
// share their barriers, with weights as floats; otherwise the next row's loads alone.  Measured (us, one row and one
// block a CU -> two blocks, two rows): 8192 x 768 LayerNorm, fp32 stream 29.4 -> 25.8, 28.2; 16001 x 4096 with both norms and a
// gate 185 -> 226 (spills), 178.
__host__ __device__ constexpr bool two_blocks(bool vec, bool post, bool layer, bool gate, size_t x_size) {
    return vec && !gate && (!post || (!layer && x_size == 2));
}
constexpr bool lds_sums(int nc, bool post, bool layer, bool gate) {
    return nc > 1 && gate + (post ? 1 + layer : 0) + 1 + layer >= 3;
}
template <typename TX, typename TH, int WPR, int NC, bool VEC, bool POST, bool LAYER, bool GATE>
__global__ __launch_bounds__(512, NC == 1 && two_blocks(VEC, POST, LAYER, GATE, sizeof(TX)) ? 4 : 2) void residual_bwd(BwdArgs<TX, TH> a) {
    constexpr int T = 64 * WPR, RG = 512 / T;  // rows of a block side by side, times RP
    constexpr int SUMS = GATE + (POST ? 1 + LAYER : 0) + 1 + LAYER;
    constexpr int RP = NC == 1 && SUMS <= 3 && !two_blocks(VEC, POST, LAYER, GATE, sizeof(TX)) ? 2 : 1;
    constexpr bool AHEAD = NC == 1, FW = RP == 2;  // AHEAD: the next rows' loads before these rows' work
    constexpr int NS = POST ? 3 : 2;
    // Sixteen elements a lane and three sums or more do not fit the registers beside the row: all sums but pre_w's are
    // then in LDS, where every lane has columns of its own (one row a block).  4096 x 6144, both LayerNorms and a
    // gate: 331 us with what the registers spilled, 191 so.
    constexpr bool IN_LDS = lds_sums(NC, POST, LAYER, GATE);
    constexpr int L_GATE = 0, L_PW = GATE, L_PB = GATE + POST, L_NB = GATE + POST + (POST && LAYER);
    extern __shared__ __align__(16) float lds_sum[];  // [SUMS - 1][F up to a multiple of 8]
    const int pitch = (a.F + 7) & ~7;
    __shared__ float4 rbuf[RG][2][WPR][2];
    __shared__ __align__(16) float acc_lds[RG > 1 ? RG * T * NC * 8 : 4];
    const int rg = __builtin_amdgcn_readfirstlane((int)threadIdx.x / T);  // the wave's
    const Cols<T, NC, VEC> c{(int)threadIdx.x & (T - 1), a.F};
    RowSum<WPR> sum{rbuf[rg], (int)(threadIdx.x >> 6) & (WPR - 1), (int)threadIdx.x & 63, 0};
    const uint64_t key = a.mask.t ? a.mask.key() : 0;
    const float inv = 1.0f / (float)a.F, gate_scale = FW ? 1.f : a.scale;  // of the gate's weights as they are held

    Weights<TH, VEC, FW> wp[POST ? NC : 1], bp[POST && LAYER && GATE ? NC : 1], wn[NC], gate[NC];
#pragma unroll
    for (int j = 0; j < NC; ++j) {
        if constexpr (POST) wp[j].set(a.post_w, 1.f, 1.f, c, j);
        if constexpr (POST && LAYER && GATE) bp[j].set(a.post_b, 0.f, 1.f, c, j);
        wn[j].set(a.pre_w, 1.f, 1.f, c, j);
        gate[j].set(a.gate, 1.f, a.scale, c, j);
    }
    int at_gate = 0;

    constexpr int NR = IN_LDS ? 1 : NC;
    float dg[GATE ? NR : 1][8], dwp[POST ? NR : 1][8], dbp[POST && LAYER ? NR : 1][8], dwn[NC][8], dbn[LAYER ? NR : 1][8];
    // a lane's eight sums of plane p in LDS, f(place, e) each
    auto lds_each = [&](int p, int j, auto f) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c.has(j, e)) f(lds_sum + p * pitch + c.at(j, e), e);
    };
    auto clear = [&](auto& v, int p) {
        if constexpr (IN_LDS) {
#pragma unroll
            for (int j = 0; j < NC; ++j) lds_each(p, j, [](float* to, int) { *to = 0.f; });
        } else {
            for (auto& r : v)
#pragma unroll
                for (int e = 0; e < 8; ++e) r[e] = 0.f;
        }
    };
    auto add = [&](auto& v, int p, int j, const float (&x)[8]) __attribute__((always_inline)) {
        if constexpr (IN_LDS) {
            if constexpr (VEC) {
                if (c.has(j, 0)) {
                    float4* to = reinterpret_cast<float4*>(lds_sum + p * pitch + c.at(j, 0));
                    const float4 u = to[0], w = to[1];
                    to[0] = make_float4(u.x + x[0], u.y + x[1], u.z + x[2], u.w + x[3]);
                    to[1] = make_float4(w.x + x[4], w.y + x[5], w.z + x[6], w.w + x[7]);
                }
            } else {
                lds_each(p, j, [&](float* to, int e) { *to += x[e]; });
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[j][e] += x[e];
        }
    };
    // what add() added up, for emit()
    auto summed = [&](auto& v, int p, float (&out)[NC][8]) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            if constexpr (IN_LDS) {
                lds_each(p, j, [&](float* from, int e) { out[j][e] = *from; });
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) out[j][e] = v[j][e];
            }
        }
    };
    if constexpr (GATE) clear(dg, L_GATE);
    if constexpr (POST) clear(dwp, L_PW);
    if constexpr (POST && LAYER) clear(dbp, L_PB);
    if constexpr (LAYER) clear(dbn, L_NB);
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) dwn[j][e] = 0.f;

    struct Row {
        Raw<TH, VEC> h[NC], dz[NC];
        Raw<TX, VEC> y[NC], dy[NC];
    };
    auto load = [&](int64_t r, Row& w) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            if (a.dz) w.dz[j].load(a.dz + r * a.F, c, j), w.y[j].load(a.y + r * a.F, c, j);
            else w.dz[j].fill(0.f, c, j), w.y[j].fill(0.f, c, j);
            if (a.dy) w.dy[j].load(a.dy + r * a.F, c, j);
            else w.dy[j].fill(0.f, c, j);
            if (POST || GATE) w.h[j].load(a.h + r * a.F, c, j);
        }
    };
    // a wave's rows of a turn, from r on, of those below r1; past them zeros, which add nothing to any sum
    auto load_turn = [&](int r, int r1, Row (&w)[RP]) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < RP; ++k) {
            if (r + k * RG < r1) {
                load(r + k * RG, w[k]);
            } else {
#pragma unroll
                for (int j = 0; j < NC; ++j) {
                    w[k].h[j].fill(0.f, c, j);
                    w[k].dz[j].fill(0.f, c, j);
                    w[k].y[j].fill(0.f, c, j);
                    w[k].dy[j].fill(0.f, c, j);
                }
            }
        }
    };

    // a sum over the block's rows: dst[f] (+)= its value
    auto emit = [&](float (&v)[NC][8], float* dst, bool add) {
        if constexpr (RG == 1) {
#pragma unroll
            for (int j = 0; j < NC; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c.has(j, e)) dst[c.at(j, e)] = add ? dst[c.at(j, e)] + v[j][e] : v[j][e];
        } else {
            constexpr int P = T * NC * 8;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                float* to = acc_lds + rg * P;
                if constexpr (VEC) {
                    *reinterpret_cast<float4*>(to + c.at(j, 0)) = make_float4(v[j][0], v[j][1], v[j][2], v[j][3]);
                    *reinterpret_cast<float4*>(to + c.at(j, 4)) = make_float4(v[j][4], v[j][5], v[j][6], v[j][7]);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) to[c.at(j, e)] = v[j][e];
                }
            }
            __syncthreads();
            for (int f = threadIdx.x; f < a.F; f += 512) {
                float s = acc_lds[f];
#pragma unroll
                for (int k = 1; k < RG; ++k) s += acc_lds[k * P + f];
                dst[f] = add ? dst[f] + s : s;
            }
        }
    };

    int g0, g1;
    a.split.of(blockIdx.x, g0, g1);
    for (int g = g0; g < g1; ++g) {
        int r0, r1;
        a.split.rows(blockIdx.x, g, r0, r1);
        const int turns = (r1 - r0 + RP * RG - 1) / (RP * RG);  // the same for all waves: they meet at barriers
        Row cur[RP];
        load_turn(r0 + rg, r1, cur);
        for (int i = 0; i < turns; ++i) {
            const int r = r0 + i * RP * RG + rg;
            Row nxt[RP];
            if (AHEAD && i + 1 < turns) load_turn(r + RP * RG, r1, nxt);
            // statistics: h's, y's and the sums of the pre norm's gradient, together
            float mp[RP] = {}, rp[RP], mn[RP] = {}, rn[RP], u[RP] = {}, w[RP], q[RP * NS] = {};
            if constexpr (LAYER) {
                float s[RP * NS] = {};
#pragma unroll
                for (int k = 0; k < RP; ++k)
#pragma unroll
                    for (int j = 0; j < NC; ++j)
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            s[NS * k] += cur[k].y[j][e];
                            s[NS * k + 1] += wn[j][e] * cur[k].dz[j][e];
                            if constexpr (POST) s[NS * k + 2] += cur[k].h[j][e];
                        }
                sum(s);
#pragma unroll
                for (int k = 0; k < RP; ++k) {
                    if (a.pre == GN_NORM_LAYER) mn[k] = s[NS * k] * inv, u[k] = s[NS * k + 1] * inv;
                    if constexpr (POST)
                        if (a.post == GN_NORM_LAYER) mp[k] = s[NS * k + 2] * inv;
                }
            }
            // v - mu, 0 in the places that the row does not have
            auto centred = [&](float v, float mu, int j, int e) __attribute__((always_inline)) {
                if constexpr (LAYER) return c.has(j, e) ? v - mu : 0.f;
                return v;
            };
#pragma unroll
            for (int k = 0; k < RP; ++k)
#pragma unroll
                for (int j = 0; j < NC; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float yc = centred(cur[k].y[j][e], mn[k], j, e);
                        q[NS * k] += yc * yc;
                        q[NS * k + 1] += wn[j][e] * cur[k].dz[j][e] * yc;
                        if constexpr (POST) {
                            const float hc = centred(cur[k].h[j][e], mp[k], j, e);
                            q[NS * k + 2] += hc * hc;
                        }
                    }
            sum(q);
            float d[RP][NC][8], s[RP * (1 + LAYER)] = {};
#pragma unroll
            for (int k = 0; k < RP; ++k) {
                const int row = r + k * RG;
                const bool on = row < r1;
                // (of no row: 1, not the 1 / sqrt(eps) that may be inf and make its zeros NaN)
                rn[k] = on && a.dz ? rsqrtf(q[NS * k] * inv + a.pre_eps) : 1.f;
                rp[k] = 1.f;
                if constexpr (POST) rp[k] = on ? rsqrtf(q[NS * k + 2] * inv + a.post_eps) : 1.f;
                w[k] = q[NS * k + 1] * inv * rn[k];
                if (a.gates > 1 && on) {
                    const int at = row / a.gate_rows;
                    if (at != at_gate) {
                        at_gate = at;
#pragma unroll
                        for (int j = 0; j < NC; ++j) gate[j].set(a.gate + (size_t)at * a.F, 1.f, a.scale, c, j);
                    }
                }
#pragma unroll
                for (int j = 0; j < NC; ++j) {
                    float (&dk)[8] = d[k][j];
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float yh = centred(cur[k].y[j][e], mn[k], j, e) * rn[k], dz = cur[k].dz[j][e];
                        float gr = wn[j][e] * dz;
                        if constexpr (LAYER) gr -= u[k];
                        dk[e] = cur[k].dy[j][e] + rn[k] * (gr - yh * w[k]);
                        dwn[j][e] += dz * yh;
                        x[e] = dz;
                    }
                    if constexpr (LAYER) add(dbn, L_NB, j, x);
                    if (on && a.dx) {
                        float o[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) o[e] = a.res_scale * dk[e];
                        store8<TX, VEC>(a.dx + (int64_t)row * a.F, c, j, o);
                    }
                    float o[8];  // n, then dgate / scale: drop(n)'s terms, so that a dropped inf or NaN adds 0
                    if constexpr (GATE) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            o[e] = cur[k].h[j][e];
                            if constexpr (POST) {
                                o[e] = centred(o[e], mp[k], j, e) * rp[k] * wp[j][e];
                                if constexpr (LAYER) o[e] += bp[j][e];
                            }
                        }
                    }
                    if (a.mask.t)
                        drop_piece<VEC>(dk, c, j, key, (uint64_t)row * a.F, a.mask, [&](int e, bool kept) __attribute__((always_inline)) {
                            if constexpr (GATE) o[e] = kept ? o[e] : 0.f;
                        });
                    if constexpr (GATE) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) o[e] *= dk[e];
                        add(dg, L_GATE, j, o);
                        if (a.gate_rows == 1 && a.gates > 1 && on) {  // a gate a row: its gradient has no sum
                            float* const to = a.grad[kGate] + (int64_t)row * a.F;
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                if (c.has(j, e)) to[c.at(j, e)] = a.accumulate ? to[c.at(j, e)] + a.scale * o[e] : a.scale * o[e];
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        dk[e] *= FW ? gate[j][e] : gate_scale * gate[j][e];
                        if constexpr (POST) {
                            const float hh = centred(cur[k].h[j][e], mp[k], j, e) * rp[k];
                            x[e] = dk[e] * hh;
                            s[k * (1 + LAYER)] += x[e] * wp[j][e];
                            if constexpr (LAYER) s[k * (1 + LAYER) + 1] += dk[e] * wp[j][e];
                        }
                    }
                    if constexpr (POST) {
                        add(dwp, L_PW, j, x);
                        if constexpr (LAYER) add(dbp, L_PB, j, dk);
#pragma unroll
                        for (int e = 0; e < 8; ++e) dk[e] *= wp[j][e];
                    }
                }
            }
            if constexpr (POST) sum(s);
#pragma unroll
            for (int k = 0; k < RP; ++k) {
                if constexpr (POST) {
                    const float pw = s[k * (1 + LAYER)] * inv;
                    float pu = 0.f;
                    if constexpr (LAYER)
                        if (a.post == GN_NORM_LAYER) pu = s[k * (1 + LAYER) + 1] * inv;
#pragma unroll
                    for (int j = 0; j < NC; ++j)
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float hh = (LAYER ? cur[k].h[j][e] - mp[k] : cur[k].h[j][e]) * rp[k];
                            if constexpr (LAYER) d[k][j][e] -= pu;
                            d[k][j][e] = rp[k] * (d[k][j][e] - hh * pw);
                        }
                }
                const int row = r + k * RG;
                if (row < r1 && a.dh)
#pragma unroll
                    for (int j = 0; j < NC; ++j) store8<TH, VEC>(a.dh + (int64_t)row * a.F, c, j, d[k][j]);
            }
#pragma unroll
            for (int k = 0; k < RP; ++k)
                if constexpr (AHEAD) cur[k] = nxt[k];
            if (!AHEAD && i + 1 < turns) load_turn(r + RP * RG, r1, cur);
        }
        if constexpr (GATE)
            if (a.gate_rows > 1 || a.gates <= 1) {
                const bool whole = a.split.per <= 1;  // the group's rows are all this block's
                float all[NC][8];
                summed(dg, L_GATE, all);
#pragma unroll
                for (int j = 0; j < NC; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e) all[j][e] *= a.scale;
                emit(all, whole ? a.grad[kGate] + (size_t)g * a.F : a.part + ((size_t)kGate * a.split.blocks + blockIdx.x) * a.F,
                     whole && a.accumulate);
                clear(dg, L_GATE);
            }
    }
    auto plane = [&](auto& v, int l, int p) {
        if (!a.grad[p]) return;
        const bool one = a.split.blocks == 1;
        float all[NC][8];
        summed(v, l, all);
        emit(all, one ? a.grad[p] : a.part + ((size_t)p * a.split.blocks + blockIdx.x) * a.F, one && a.accumulate);
    };
    if constexpr (POST) plane(dwp, L_PW, kPostW);
    if constexpr (POST && LAYER) plane(dbp, L_PB, kPostB);
    if constexpr (LAYER) plane(dbn, L_NB, kPreB);
    if (a.grad[kPreW]) {
        const bool one = a.split.blocks == 1;
        emit(dwn, one ? a.grad[kPreW] : a.part + ((size_t)kPreW * a.split.blocks + blockIdx.x) * a.F, one && a.accumulate);
    }
}

// out[f] (+)= the sum of `count` partial rows.  16 waves of 64 columns, each a share of the rows, added in
// a fixed order; blockIdx.y: the item (a parameter, or one group of the gate).
struct FinishArgs {
    const float* part;
    float* grad[kPlanes];
    int F, blocks, per, groups;  // groups: of the gate, 0: its gradient is complete
    int plane[kPlanes], planes;  // the wanted ones
    int accumulate;
};
__global__ __launch_bounds__(1024) void residual_finish(FinishArgs a) {
    __shared__ float sh[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, f = blockIdx.x * 64 + lane;
    for (int item = blockIdx.y; item < a.planes + a.groups; item += gridDim.y) {
        const bool is_gate = item >= a.planes;
        const int p = is_gate ? (int)kGate : a.plane[item], g = item - a.planes;
        const float* part = a.part + ((size_t)p * a.blocks + (is_gate ? (size_t)g * a.per : 0)) * a.F;
        float* out = a.grad[p] + (is_gate ? (size_t)g * a.F : 0);
        const int n = is_gate ? a.per : a.blocks;
        float s = 0.f;
        if (f < a.F) {
#pragma unroll 16
            for (int k = wave; k < n; k += 16) s += part[(size_t)k * a.F + f];
        }
        sh[wave][lane] = s;
        __syncthreads();
        if (wave == 0 && f < a.F) {
            float t = sh[0][lane];
#pragma unroll
            for (int w = 1; w < 16; ++w) t += sh[w][lane];
            out[f] = a.accumulate ? out[f] + t : t;
        }
        __syncthreads();
    }
}

// ---- wider rows ------------------------------------------------------------------------------
constexpr int kWide = 512;  // threads of a row

template <typename T> __device__ __forceinline__ float weight(const T* w, int64_t i, float absent) {
    return w ? io<T>::ld(w, i) : absent;
}

template <typename TX, typename TH>
__global__ __launch_bounds__(kWide) void residual_fwd_wide(FwdArgs<TX, TH> a) {
    __shared__ float sh[kWide / 64];
    const uint64_t key = a.mask.t ? a.mask.key() : 0;
    const float inv = 1.0f / (float)a.F;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const TH* h = a.h + r * a.F;
        const TX* x = a.x + r * a.F;
        const TH* gate = a.gate ? a.gate + (a.gates > 1 ? r / a.gate_rows : 0) * a.F : nullptr;
        float mu = 0.f, rs = 1.f;
        auto stats = [&](int kind, float eps, auto value) {
            mu = 0.f;
            rs = 1.f;
            float m = 0.f, q = 0.f;
            if (kind == GN_NORM_LAYER) {
                for (int f = threadIdx.x; f < a.F; f += kWide) m += value(f);
                m = block_sum<kWide / 64>(m, sh) * inv;
            }
            if (kind != GN_NORM_NONE) {
                for (int f = threadIdx.x; f < a.F; f += kWide) {
                    const float d = value(f) - m;
                    q += d * d;
                }
                q = block_sum<kWide / 64>(q, sh) * inv;
                rs = rsqrtf(q + eps);
            }
            mu = m;
        };
        stats(a.post, a.post_eps, [&](int f) { return io<TH>::ld(h, f); });
        const float pm = mu, pr = rs;
        auto stream = [&](int f) {
            float n = (io<TH>::ld(h, f) - pm) * pr * weight(a.post_w, f, 1.f) + weight(a.post_b, f, 0.f);
            if (a.mask.t) n = drop1(n, key, (uint64_t)(r * a.F + f), a.mask.t, a.mask.keep);
            return a.res_scale * io<TX>::ld(x, f) + a.scale * weight(gate, f, 1.f) * n;
        };
        stats(a.pre, a.pre_eps, stream);
        for (int f = threadIdx.x; f < a.F; f += kWide) {
            const float y = stream(f);
            io<TX>::st(a.y, r * a.F + f, y);
            if (a.pre != GN_NORM_NONE)
                io<TH>::st(a.z, r * a.F + f, (y - mu) * rs * weight(a.pre_w, f, 1.f) + weight(a.pre_b, f, 0.f));
        }
    }
}

// A wide row's numbers: both norms' mu and r, and the means u and w of their gradients.
struct WideRow {
    float mp, rp, mn, rn, u, w, pu, pw;
};
template <typename TX, typename TH>
__device__ __forceinline__ float wide_dY(const BwdArgs<TX, TH>& a, const WideRow& s, int64_t i, int f) {
    float d = a.dy ? io<TX>::ld(a.dy, i) : 0.f;
    if (a.dz)
        d += norm_grad(weight(a.pre_w, f, 1.f) * io<TH>::ld(a.dz, i), io<TX>::ld(a.y, i) - s.mn, s.rn, s.u, s.w);
    return d;
}

// The rows' numbers, a block a row.
template <typename TX, typename TH>
__global__ __launch_bounds__(kWide) void residual_bwd_stats(BwdArgs<TX, TH> a) {
    __shared__ float sh[kWide / 64];
    const uint64_t key = a.mask.t ? a.mask.key() : 0;
    const float inv = 1.0f / (float)a.F;
    auto mean = [&](auto value) {
        float v = 0.f;
        for (int f = threadIdx.x; f < a.F; f += kWide) v += value(f);
        return block_sum<kWide / 64>(v, sh) * inv;
    };
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const int64_t at = r * a.F;
        const TH* gate = a.gate ? a.gate + (a.gates > 1 ? r / a.gate_rows : 0) * a.F : nullptr;
        WideRow s{0.f, 1.f, 0.f, 1.f, 0.f, 0.f, 0.f, 0.f};
        if (a.dz) {
            if (a.pre == GN_NORM_LAYER) {
                s.mn = mean([&](int f) { return io<TX>::ld(a.y, at + f); });
                s.u = mean([&](int f) { return weight(a.pre_w, f, 1.f) * io<TH>::ld(a.dz, at + f); });
            }
            s.rn = rsqrtf(mean([&](int f) { const float d = io<TX>::ld(a.y, at + f) - s.mn; return d * d; }) + a.pre_eps);
            s.w = s.rn * mean([&](int f) {
                return weight(a.pre_w, f, 1.f) * io<TH>::ld(a.dz, at + f) * (io<TX>::ld(a.y, at + f) - s.mn);
            });
        }
        if (a.post != GN_NORM_NONE) {
            if (a.post == GN_NORM_LAYER) s.mp = mean([&](int f) { return io<TH>::ld(a.h, at + f); });
            s.rp = rsqrtf(mean([&](int f) { const float d = io<TH>::ld(a.h, at + f) - s.mp; return d * d; }) + a.post_eps);
            auto g = [&](int f) {
                float d = wide_dY(a, s, at + f, f);
                if (a.mask.t) d = drop1(d, key, (uint64_t)(at + f), a.mask.t, a.mask.keep);
                return a.scale * weight(gate, f, 1.f) * d * weight(a.post_w, f, 1.f);
            };
            if (a.post == GN_NORM_LAYER) s.pu = mean(g);
            s.pw = s.rp * mean([&](int f) { return g(f) * (io<TH>::ld(a.h, at + f) - s.mp); });
        }
        if (threadIdx.x == 0) *reinterpret_cast<WideRow*>(a.stats + 8 * r) = s;
    }
}

// A column of a block's rows: dx, dh and the sums.
template <typename TX, typename TH>
__global__ __launch_bounds__(256) void residual_bwd_cols(BwdArgs<TX, TH> a) {
    const int f = blockIdx.x * 256 + threadIdx.x, b = blockIdx.y;
    if (f >= a.F) return;
    const uint64_t key = a.mask.t ? a.mask.key() : 0;
    const float wp = weight(a.post_w, f, 1.f), bp = weight(a.post_b, f, 0.f);
    float dwp = 0.f, dbp = 0.f, dwn = 0.f, dbn = 0.f;
    int g0, g1;
    a.split.of(b, g0, g1);
    for (int g = g0; g < g1; ++g) {
        int r0, r1;
        a.split.rows(b, g, r0, r1);
        float dg = 0.f;
        for (int r = r0; r < r1; ++r) {
            const WideRow s = *reinterpret_cast<const WideRow*>(a.stats + 8 * (int64_t)r);
            const int64_t i = (int64_t)r * a.F + f;
            float d = wide_dY(a, s, i, f);
            if (a.dz) {
                const float dz = io<TH>::ld(a.dz, i);
                dwn += dz * (io<TX>::ld(a.y, i) - s.mn) * s.rn;
                dbn += dz;
            }
            if (a.dx) io<TX>::st(a.dx, i, a.res_scale * d);
            const float hc = io<TH>::ld(a.h, i) - s.mp;
            float n = hc * s.rp * wp + bp;
            if (a.mask.t)  // (dgate takes drop(n): a dropped inf or NaN adds 0)
                d = drop1(d, key, (uint64_t)i, a.mask.t, a.mask.keep, [&](int, bool kept) { n = kept ? n : 0.f; });
            d *= a.scale;
            dg += d * n;
            if (a.grad[kGate] && a.gate_rows == 1 && a.gates > 1) {
                float* to = a.grad[kGate] + i;
                *to = a.accumulate ? *to + d * n : d * n;
            }
            if (a.gate) d *= io<TH>::ld(a.gate, (a.gates > 1 ? (int64_t)(r / a.gate_rows) : 0) * a.F + f);
            dwp += d * hc * s.rp;
            dbp += d;
            if (a.post != GN_NORM_NONE) d = norm_grad(d * wp, hc, s.rp, s.pu, s.pw);
            if (a.dh) io<TH>::st(a.dh, i, d);
        }
        if (a.grad[kGate] && (a.gate_rows > 1 || a.gates <= 1)) {
            if (a.split.per <= 1) {
                float* to = a.grad[kGate] + (size_t)g * a.F + f;
                *to = a.accumulate ? *to + dg : dg;
            } else {
                a.part[((size_t)kGate * a.split.blocks + b) * a.F + f] = dg;
            }
        }
    }
    const float v[kPlanes] = {0.f, dwp, dbp, dwn, dbn};
#pragma unroll
    for (int p = kPostW; p < kPlanes; ++p) {
        if (!a.grad[p]) continue;
        if (a.split.blocks == 1) a.grad[p][f] = a.accumulate ? a.grad[p][f] + v[p] : v[p];
        else a.part[((size_t)p * a.split.blocks + b) * a.F + f] = v[p];
    }
}

// ---- launches --------------------------------------------------------------------------------
// Waves of a row of F elements: one piece of eight elements a lane up to 4096, two above.
inline int waves_of(int F) { return F <= 512 ? 1 : F <= 1024 ? 2 : F <= 2048 ? 4 : 8; }

int device_cus() {
    int dev = 0, cus = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
        cus = 256;
    return cus;
}

template <typename TX, typename TH, bool VEC>
int launch_fwd(const FwdArgs<TX, TH>& a, hipStream_t s) {
    if (a.F > kMaxF) {
        residual_fwd_wide<TX, TH><<<std::min(a.rows, 1 << 20), kWide, 0, s>>>(a);
    } else {
        const int w = waves_of(a.F);
        // 16 waves a CU
        const int64_t blocks = std::min<int64_t>(((int64_t)a.rows + (w == 1 ? 3 : 0)) / (w == 1 ? 4 : 1), device_cus() * (w == 1 ? 4 : 16 / w));
        const dim3 grid((unsigned)blocks);
        switch (w) {
            case 1: residual_fwd<TX, TH, 1, 1, VEC><<<grid, 256, 0, s>>>(a); break;
            case 2: residual_fwd<TX, TH, 2, 1, VEC><<<grid, 128, 0, s>>>(a); break;
            case 4: residual_fwd<TX, TH, 4, 1, VEC><<<grid, 256, 0, s>>>(a); break;
            default:
                if (a.F <= 4096) residual_fwd<TX, TH, 8, 1, VEC><<<grid, 512, 0, s>>>(a);
                else residual_fwd<TX, TH, 8, 2, VEC><<<grid, 512, 0, s>>>(a);
        }
    }
    GN_LAUNCH_CHECK("gn_residual_norm_fwd");
    return GN_OK;
}

template <typename TX, typename TH, bool VEC, bool POST, bool LAYER, bool GATE>
int launch_rows(const BwdArgs<TX, TH>& a, hipStream_t s) {
    const dim3 grid((unsigned)a.split.blocks);
    switch (waves_of(a.F)) {
        case 1: residual_bwd<TX, TH, 1, 1, VEC, POST, LAYER, GATE><<<grid, 512, 0, s>>>(a); break;
        case 2: residual_bwd<TX, TH, 2, 1, VEC, POST, LAYER, GATE><<<grid, 512, 0, s>>>(a); break;
        case 4: residual_bwd<TX, TH, 4, 1, VEC, POST, LAYER, GATE><<<grid, 512, 0, s>>>(a); break;
        default:
            if (a.F <= 4096) {
                residual_bwd<TX, TH, 8, 1, VEC, POST, LAYER, GATE><<<grid, 512, 0, s>>>(a);
            } else {
                constexpr int planes = lds_sums(2, POST, LAYER, GATE) ? GATE + (POST ? 1 + LAYER : 0) + LAYER : 0;
                if constexpr (planes > 0) {
                    static const bool ok = hipFuncSetAttribute(reinterpret_cast<const void*>(&residual_bwd<TX, TH, 8, 2, VEC, POST, LAYER, GATE>),
                                                               hipFuncAttributeMaxDynamicSharedMemorySize, planes * kMaxF * 4) == hipSuccess;
                    if (!ok) {
                        (void)hipGetLastError();
                        set_error("gn_residual_norm_bwd: cannot reserve %d B of LDS", planes * kMaxF * 4);
                        return GN_E_HIP;
                    }
                }
                residual_bwd<TX, TH, 8, 2, VEC, POST, LAYER, GATE><<<grid, 512, (size_t)planes * ((a.F + 7) & ~7) * 4, s>>>(a);
            }
    }
    return GN_OK;
}

template <typename TX, typename TH, bool VEC>
int launch_kinds(const BwdArgs<TX, TH>& a, hipStream_t s) {
    const bool post = a.post != GN_NORM_NONE, layer = a.post == GN_NORM_LAYER || a.pre == GN_NORM_LAYER;
    const bool gate = a.grad[kGate] != nullptr;
    if (post && layer) return gate ? launch_rows<TX, TH, VEC, true, true, true>(a, s) : launch_rows<TX, TH, VEC, true, true, false>(a, s);
    if (post) return gate ? launch_rows<TX, TH, VEC, true, false, true>(a, s) : launch_rows<TX, TH, VEC, true, false, false>(a, s);
    if (layer) return gate ? launch_rows<TX, TH, VEC, false, true, true>(a, s) : launch_rows<TX, TH, VEC, false, true, false>(a, s);
    return gate ? launch_rows<TX, TH, VEC, false, false, true>(a, s) : launch_rows<TX, TH, VEC, false, false, false>(a, s);
}

// Blocks of the backward for rows of F elements in `groups`: a block a CU, or two, with two turns of rows each
// or more.
Split make_split(int rows, int F, int groups, bool two) {
    const int turn = F > kMaxF ? 16 : 8 / waves_of(F);
    const int most = F > kMaxF ? 64 : two && F <= kMaxF / 2 ? 512 : 256;
    const int blocks = std::max(1, std::min(most, rows / (2 * turn)));
    Split s;
    s.groups = std::max(groups, 1);
    s.group_rows = rows / s.groups;
    s.per = blocks / s.groups;
    s.blocks = s.per ? s.groups * s.per : blocks;
    return s;
}

size_t stats_bytes(int rows, int F) { return F > kMaxF ? (size_t)rows * sizeof(WideRow) : 0; }

// Partial rows for any of the groupings that a call of these sizes may take.
size_t workspace_bytes(int rows, int F, int gates) {
    // (the gate's groups with its gradient, and then one block a CU)
    const int b = std::max(make_split(rows, F, gates, false).blocks, make_split(rows, F, 1, true).blocks);
    return stats_bytes(rows, F) + (size_t)kPlanes * b * F * 4;
}

template <typename TX, typename TH>
int launch_bwd(BwdArgs<TX, TH>& a, bool vec, hipStream_t s) {
    if (a.F > kMaxF) {
        residual_bwd_stats<TX, TH><<<std::min(a.rows, 1 << 20), kWide, 0, s>>>(a);
        GN_LAUNCH_CHECK("gn_residual_norm_bwd");
        residual_bwd_cols<TX, TH><<<dim3((a.F + 255) / 256, a.split.blocks), 256, 0, s>>>(a);
    } else if (const int rc = vec ? launch_kinds<TX, TH, true>(a, s) : launch_kinds<TX, TH, false>(a, s)) {
        return rc;
    }
    GN_LAUNCH_CHECK("gn_residual_norm_bwd");
    FinishArgs f{};
    f.part = a.part;
    f.F = a.F;
    f.blocks = a.split.blocks;
    f.per = a.split.per;
    f.accumulate = a.accumulate;
    for (int p = 0; p < kPlanes; ++p) {
        f.grad[p] = a.grad[p];
        if (p != kGate && a.grad[p] && a.split.blocks > 1) f.plane[f.planes++] = p;
    }
    if (a.grad[kGate] && a.split.per > 1 && !(a.gates > 1 && a.gate_rows == 1)) f.groups = a.split.groups;
    const int items = f.planes + f.groups;
    if (items) {
        residual_finish<<<dim3((a.F + 63) / 64, std::min(items, 4096)), 1024, 0, s>>>(f);
        GN_LAUNCH_CHECK("gn_residual_norm_bwd (parameters)");
    }
    return GN_OK;
}

// ---- checks ----------------------------------------------------------------------------------
struct Span {
    const void* p;
    size_t bytes;
    const char* name;
    bool written;
};

int check_branch(const char* who, const gn_branch* b, int h_dtype, int x_dtype, int rows, int F, Mask* m) {
    GN_REQUIRE(b, "%s: null pointer", who);
    GN_REQUIRE(rows >= 0 && F >= 1, "%s: %d rows of %d elements", who, rows, F);
    GN_REQUIRE(F <= (1 << 24), "%s: rows of more than 2^24 elements", who);
    // (row numbers are 32 bits, also of the rows past the last that a turn looks for)
    GN_REQUIRE(rows < (1 << 30), "%s: %d rows (2^30 or more)", who, rows);
    const bool f32 = h_dtype == GN_F32 && x_dtype == GN_F32, bf = h_dtype == GN_BF16 && (x_dtype == GN_BF16 || x_dtype == GN_F32);
    GN_REQUIRE(f32 || bf, "%s: h dtype %d with x dtype %d not supported (f32/f32, bf16/bf16, bf16/f32)", who, h_dtype, x_dtype);
    for (int k : {b->post, b->pre}) GN_REQUIRE(k >= GN_NORM_NONE && k <= GN_NORM_LAYER, "%s: norm kind %d", who, k);
    GN_REQUIRE((b->post != GN_NORM_NONE || !b->post_w) && (b->post == GN_NORM_LAYER || !b->post_b) &&
                   (b->pre != GN_NORM_NONE || !b->pre_w) && (b->pre == GN_NORM_LAYER || !b->pre_b),
               "%s: weights without their norm (a bias goes with GN_NORM_LAYER)", who);
    GN_REQUIRE(b->gate ? b->gates >= 1 : b->gates == 0, "%s: gate and gates go together", who);
    GN_REQUIRE(!b->gate || rows % b->gates == 0, "%s: %d rows are no multiple of %d gates", who, rows, b->gates);
    GN_REQUIRE(make_mask(&b->rng, b->p, m), "%s: p must be at least 0 and below 1", who);
    if (!m->t) m->step_dev = nullptr;  // not read
    GN_REQUIRE(((uintptr_t)m->step_dev & 7u) == 0, "%s: step_dev is not aligned to 8 bytes", who);
    return GN_OK;
}

// What is written shares no memory with anything else of the call; but the first tensor may be the second,
// as a whole.
template <int N>
int check_spans(const char* who, const Span (&t)[N]) {
    for (int i = 0; i < N; ++i)
        for (int j = 0; j < N && t[i].written; ++j)
            GN_REQUIRE(i == j || !share(t[i].p, t[i].bytes, t[j].p, t[j].bytes) || (i == 0 && j == 1 && t[0].p == t[1].p),
                       "%s: %s and %s may not share memory", who, t[i].name, t[j].name);
    return GN_OK;
}

template <typename TX, typename TH>
int fwd(const gn_branch* b, const Mask& m, const void* h, const void* x, void* y, void* z, int rows, int F, hipStream_t s) {
    FwdArgs<TX, TH> a{};
    a.h = (const TH*)h;
    a.x = (const TX*)x;
    a.y = (TX*)y;
    a.z = (TH*)z;
    a.post_w = (const TH*)b->post_w;
    a.post_b = (const TH*)b->post_b;
    a.pre_w = (const TH*)b->pre_w;
    a.pre_b = (const TH*)b->pre_b;
    a.gate = (const TH*)b->gate;
    a.rows = rows;
    a.F = F;
    a.gates = b->gates;
    a.gate_rows = b->gates ? rows / b->gates : rows;
    a.post = b->post;
    a.pre = b->pre;
    a.scale = b->scale;
    a.res_scale = b->res_scale;
    a.post_eps = b->post_eps;
    a.pre_eps = b->pre_eps;
    a.mask = m;
    const bool vec = F % 8 == 0 && al16(h) && al16(x) && al16(y) && al16(z) && al16(b->post_w) && al16(b->post_b) &&
                     al16(b->pre_w) && al16(b->pre_b) && al16(b->gate);
    return vec ? launch_fwd<TX, TH, true>(a, s) : launch_fwd<TX, TH, false>(a, s);
}

template <typename TX, typename TH>
int bwd(const gn_branch* b, const Mask& m, const void* dy, const void* dz, const void* h, const void* y, void* dh, void* dx,
        float* const (&grad)[kPlanes], int rows, int F, unsigned flags, void* ws, hipStream_t s) {
    BwdArgs<TX, TH> a{};
    a.dy = (const TX*)dy;
    a.dz = (const TH*)dz;
    a.h = (const TH*)h;
    a.y = (const TX*)y;
    a.dh = (TH*)dh;
    a.dx = (TX*)dx;
    a.post_w = (const TH*)b->post_w;
    a.post_b = (const TH*)b->post_b;
    a.pre_w = (const TH*)b->pre_w;
    a.gate = (const TH*)b->gate;
    for (int p = 0; p < kPlanes; ++p) a.grad[p] = grad[p];
    a.rows = rows;
    a.F = F;
    a.gates = b->gates;
    a.gate_rows = b->gates ? rows / b->gates : rows;
    a.post = b->post;
    a.pre = b->pre;
    a.accumulate = (flags & GN_ACCUMULATE) ? 1 : 0;
    a.scale = b->scale;
    a.res_scale = b->res_scale;
    a.post_eps = b->post_eps;
    a.pre_eps = b->pre_eps;
    a.mask = m;
    a.stats = (float*)ws;
    a.part = (float*)((char*)ws + stats_bytes(rows, F));
    const bool vec = F % 8 == 0 && al16(dy) && al16(dz) && al16(h) && al16(y) && al16(dh) && al16(dx) && al16(b->post_w) &&
                     al16(b->post_b) && al16(b->pre_w) && al16(b->gate);
    const bool layer = a.post == GN_NORM_LAYER || a.pre == GN_NORM_LAYER;
    a.split = make_split(rows, F, grad[kGate] && a.gate_rows > 1 ? b->gates : 1,
                         two_blocks(vec, a.post != GN_NORM_NONE, layer, grad[kGate] != nullptr, sizeof(TX)));
    return launch_bwd<TX, TH>(a, vec, s);
}

}  // namespace
}  // namespace gn

using namespace gn;

extern "C" int gn_dropout_fwd(const void* X, void* Y, int64_t n, double p, const gn_rng* rng, int dtype, void* stream) {
    return dropout("gn_dropout_fwd", X, Y, n, p, rng, dtype, false, as_stream(stream));
}

extern "C" int gn_dropout_bwd(const void* dY, void* dX, int64_t n, double p, const gn_rng* rng, int dtype,
                              unsigned flags, void* stream) {
    return dropout("gn_dropout_bwd", dY, dX, n, p, rng, dtype, flags & GN_ACCUMULATE, as_stream(stream));
}

extern "C" int gn_residual_norm_fwd(const gn_branch* b, const void* h, int h_dtype, const void* x, int x_dtype, void* y,
                                    void* z, int rows, int F, void* stream) {
    clear_error();
    const char* const who = "gn_residual_norm_fwd";
    Mask m;
    if (const int rc = check_branch(who, b, h_dtype, x_dtype, rows, F, &m)) return rc;
    GN_REQUIRE((z != nullptr) == (b->pre != GN_NORM_NONE) || rows == 0, "%s: z goes with the norm before the next block", who);
    if (rows == 0) return GN_OK;
    GN_REQUIRE(h && x && y, "%s: null pointer", who);
    const size_t hs = h_dtype == GN_F32 ? 4 : 2, xs = x_dtype == GN_F32 ? 4 : 2, n = (size_t)rows * F, w = F * hs;
    const uintptr_t hp = (uintptr_t)h | (uintptr_t)z | (uintptr_t)b->gate | (uintptr_t)b->post_w | (uintptr_t)b->post_b |
                         (uintptr_t)b->pre_w | (uintptr_t)b->pre_b;
    GN_REQUIRE((hp & (hs - 1)) == 0 && (((uintptr_t)x | (uintptr_t)y) & (xs - 1)) == 0,
               "%s: a tensor is not aligned to its elements", who);
    const Span spans[] = {{y, n * xs, "y", true}, {x, n * xs, "x", false}, {z, n * hs, "z", true}, {h, n * hs, "h", false},
                          {b->gate, (size_t)b->gates * w, "gate", false}, {b->post_w, w, "post_w", false},
                          {b->post_b, w, "post_b", false}, {b->pre_w, w, "pre_w", false}, {b->pre_b, w, "pre_b", false},
                          {m.step_dev, 8, "step_dev", false}};
    if (const int rc = check_spans(who, spans)) return rc;
    hipStream_t s = as_stream(stream);
    if (h_dtype == GN_F32) return fwd<float, float>(b, m, h, x, y, z, rows, F, s);
    if (x_dtype == GN_F32) return fwd<float, bf16_t>(b, m, h, x, y, z, rows, F, s);
    return fwd<bf16_t, bf16_t>(b, m, h, x, y, z, rows, F, s);
}

extern "C" size_t gn_residual_norm_workspace_bytes(int rows, int F, int gates) {
    if (rows <= 0 || rows >= (1 << 30) || F < 1 || F > (1 << 24) || gates < 0 || (gates && rows % gates)) return 0;
    return workspace_bytes(rows, F, gates);
}

extern "C" int gn_residual_norm_bwd(const gn_branch* b, const void* dy, const void* dz, const void* h, int h_dtype,
                                    const void* y, int x_dtype, void* dh, void* dx, const gn_branch_grads* grads, int rows,
                                    int F, unsigned flags, void* ws, size_t ws_bytes, void* stream) {
    clear_error();
    const char* const who = "gn_residual_norm_bwd";
    Mask m;
    if (const int rc = check_branch(who, b, h_dtype, x_dtype, rows, F, &m)) return rc;
    const gn_branch_grads none{};
    const gn_branch_grads& g = grads ? *grads : none;
    GN_REQUIRE((!g.dgate || b->gate) && (!g.dpost_w || b->post != GN_NORM_NONE) && (!g.dpost_b || b->post == GN_NORM_LAYER) &&
                   (!g.dpre_w || b->pre != GN_NORM_NONE) && (!g.dpre_b || b->pre == GN_NORM_LAYER),
               "%s: a gradient without its parameter", who);
    GN_REQUIRE(!dz || b->pre != GN_NORM_NONE, "%s: dz goes with the norm before the next block", who);
    GN_REQUIRE(rows == 0 || dy || dz, "%s: neither dy nor dz", who);
    const size_t hs = h_dtype == GN_F32 ? 4 : 2, xs = x_dtype == GN_F32 ? 4 : 2, n = (size_t)rows * F, w = F * hs;
    float* const grad[kPlanes] = {g.dgate, g.dpost_w, g.dpost_b, g.dpre_w, g.dpre_b};
    const size_t gb = (size_t)F * 4, gate_bytes = (size_t)b->gates * gb;
    const bool any = g.dgate || g.dpost_w || g.dpost_b || g.dpre_w || g.dpre_b;
    uintptr_t gp = 0;
    for (float* p : grad) gp |= (uintptr_t)p;
    const uintptr_t hp = (uintptr_t)h | (uintptr_t)dz | (uintptr_t)dh | (uintptr_t)b->gate | (uintptr_t)b->post_w |
                         (uintptr_t)b->post_b | (uintptr_t)b->pre_w;
    GN_REQUIRE((hp & (hs - 1)) == 0 && (((uintptr_t)dy | (uintptr_t)y | (uintptr_t)dx) & (xs - 1)) == 0 && (gp & 3) == 0,
               "%s: a tensor is not aligned to its elements", who);
    hipStream_t s = as_stream(stream);
    if (rows == 0) {  // sums over no rows
        for (int p = 0; p < kPlanes && !(flags & GN_ACCUMULATE); ++p)
            if (grad[p] && launch_zero(grad[p], p == kGate ? gate_bytes : gb, s) != hipSuccess) {
                set_error("%s: clear failed", who);
                return GN_E_HIP;
            }
        return GN_OK;
    }
    GN_REQUIRE(h && y, "%s: null pointer", who);
    const size_t need = any || F > kMaxF ? workspace_bytes(rows, F, b->gates) : 0;
    if (need && (!ws || ws_bytes < need || !al16(ws))) {
        set_error("%s: workspace of %zu bytes (16-byte aligned) required", who, need);
        return GN_E_WORKSPACE;
    }
    const Span spans[] = {{dx, n * xs, "dx", true}, {dy, n * xs, "dy", false}, {dh, n * hs, "dh", true},
                          {dz, n * hs, "dz", false}, {h, n * hs, "h", false}, {y, n * xs, "y", false},
                          {b->gate, (size_t)b->gates * w, "gate", false}, {b->post_w, w, "post_w", false},
                          {b->post_b, w, "post_b", false}, {b->pre_w, w, "pre_w", false},
                          {g.dgate, gate_bytes, "dgate", true}, {g.dpost_w, gb, "dpost_w", true},
                          {g.dpost_b, gb, "dpost_b", true}, {g.dpre_w, gb, "dpre_w", true}, {g.dpre_b, gb, "dpre_b", true},
                          {need ? ws : nullptr, need, "ws", true}, {m.step_dev, 8, "step_dev", false}};
    if (const int rc = check_spans(who, spans)) return rc;
    if (h_dtype == GN_F32) return bwd<float, float>(b, m, dy, dz, h, y, dh, dx, grad, rows, F, flags, ws, s);
    if (x_dtype == GN_F32) return bwd<float, bf16_t>(b, m, dy, dz, h, y, dh, dx, grad, rows, F, flags, ws, s);
    return bwd<bf16_t, bf16_t>(b, m, dy, dz, h, y, dh, dx, grad, rows, F, flags, ws, s);
}
