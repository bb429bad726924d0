// gn_linear_xent.hip — softmax cross entropy of a linear head (l = h E^T) without its logits, forward
// and backward.
//
// bf16.  The logits exist in the accumulators of the product's tiles only (gemm_stream, 256 x 128 or
// 128 x 128 tiles, blocks that stay):
//   forward    a finished tile leaves each row's maximum and sum of exp over 64 columns, 8 bytes for
//              64 logits, and the target's logit where it comes by; row_stats joins them
//   backward   a piece of the vocabulary at a time: a finished tile of the same product leaves
//              G = u (exp(l - lse) - [target]) + z exp(l - lse) in bf16, then dE_c (+)= G^T h and
//              dh += G E_c (fp32) from it
// A lane holds 16 columns of one row of each 32 x 32 accumulator, so the row statistics take one
// exchange between lanes.  For an fp32 dE, G is stored as two or three bf16 pieces, whose products with h
// are one product's longer k: two leave 2^-17 of an element (and up to 16384 rows target_rest takes the
// targets' rest), three nothing that fp32 holds, where bf16 alone (2^-8) would be the gradient's largest
// error.  For dh the first piece is enough but at the target: there the rounding of a row's largest
// element, which shows in all of dh's row, is kept in fp32 and its product with E[target] added when dh is
// rounded (dh_finish); dh is then off from fp64 by 1.7e-3 of its norm, what its own rounding leaves.  A
// bf16 dE takes two pieces up to 512 rows and the first alone above, where a second would be half a product
// more for G's rounding beside dE's own (kWholeBf16).
//
// fp32.  The pieces' logits are stored (fp32, in the workspace) between the library's fp32 products
// and row kernels, G in their place.
//
// Measured (rows x d x vocabulary): forward and both gradients of 8192 x 2048 x 128000 18.9-19.1 ms, of 8190 x
// 768 x 32000 2.26-2.30 ms: five products where the formulas have three (the logits again, dE's second
// piece), 21.5 and 2.0 TFLOP at 1.13 and 0.88 PFLOP/s.  At d = 2048 the matrix cores bound them, and on them
// the clock: the logits with their statistics take 3.5-3.8 ms, 74 % of the matrix pipe at 1.5 GHz, the
// library's product alone 3.5-4.1, 77 % at 1.4.  At d = 768 the epilogues do: the four compute waves run
// them between tiles of twelve k-tiles, the pipe is busy for 54 % of the forward and 26 % of G's pieces.
// 256 x 256 tiles of four waves that issue their own loads took 2 % off the larger and put 6 % onto smaller
// ones; staggered starts of the blocks gave nothing.  Few rows are a read of E: 16 x 2048 x 32000 forward
// 26 us + 4 for 131 MB (5.0 TB/s).  fp32 of 1003 x 768 x 32000: 1.14-1.17 ms, four products, 0.197 TFLOP at
// six bf16 ones each, 1.0 PFLOP/s of those.
//
// Widths, row counts and vocabularies that the products' vectors do not divide: h and E's piece are
// laid out to multiples of q = 8 (bf16) or 4 (fp32) elements first; the last V % q columns go
// through products of q rows and through dh_finish.
#include <algorithm>
#include <cmath>

#include "gn_gemm_stream_core.h"

namespace gn {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;

// exp(x - m) as exp2(x kLog2e - b) takes b = m kLog2e, whose rounding (2^-20 at 17) would go into every term
// of a row alike: what it was off by, without log2e's own rounding, which x kLog2e has too (it cancels
// where x is near m: x = m gives exactly 1)
__device__ __forceinline__ float off(float m, float b) { return fmaf(m, kLog2e, -b); }

// A part of a row: its maximum m and the sum s of exp about it, (-inf, 0) when it is empty.  A NaN among
// the logits is in s only (m skips it) and stays there.
// s about another maximum n >= m
__device__ __forceinline__ float about(float s, float m, float n) {
    return s * __builtin_amdgcn_exp2f((m - (n == -INFINITY ? 0.f : n)) * kLog2e);
}
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
    const float n = fmaxf(m, m2);
    s = about(s, m, n) + about(s2, m2, n);
    m = n;
}

// ---- bf16: epilogues of the logits' product -------------------------------------------------
// Element r of a 32 x 32 accumulator: row lane % 32, column 8 (r / 4) + 4 (lane / 32) + r % 4.

// What the epilogue takes of each of the wave's rows is brought into the wave's LDS by DMA while the tile's
// k-tiles run (loads at the tile's end would stand in its way, and registers over the k loop are
// not to be had).  BYTES 4 or 16 a row, 32 FM rows; begin() starts it, wait() ends it.
template <int FM, int BYTES>
__device__ __forceinline__ void rows_begin(const void* src, int m0, int M, unsigned char* st, int lane) {
    // the previous tile's reads of this LDS have returned
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(63) & 0xF0FFu);
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds_addr(st));
#pragma unroll
    for (int k = 0; k < (FM + 1) / 2; ++k) {  // 64 rows an instruction (32 FM of them are used)
        const char* from = (const char*)src + (size_t)min(m0 + 64 * k + lane, M - 1) * BYTES;
        if constexpr (BYTES == 16) {
            dma16(from, to + 1024u * k);
        } else {
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
                         : : "s"(to + 256u * k), "v"(from) : "memory", "m0");
        }
    }
}
__device__ __forceinline__ void rows_wait() {
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    wave_lds_sync();
}

// Each row's statistics over the wave's 64 columns, and its target's logit.
struct StatsTile {
    static constexpr bool kAgain = false;
    const int32_t* tgt;
    float* lt;      // [T] the target's logit
    float2* part;   // [strips][T]
    int v0;         // the vocabulary's column of column 0 here
    template <int FM>
    __device__ __forceinline__ void begin(const GemmDesc& g, int m0, unsigned char* st, int lane) const {
        rows_begin<FM, 4>(tgt, m0, g.M, st, lane);
    }
    template <int FM, int FN>
    __device__ __forceinline__ void tile(const GemmDesc& g, const f32x16_t (&acc)[FM][FN], int m0, int n0,
                                         unsigned char* st, int lane) const {
        static_assert(FN == 2, "64 columns a wave");
        rows_wait();
        if (n0 >= g.N) return;
        asm volatile("" : "+v"(lane));  // opaque: addresses are formed here, not kept across the k loop
        const int nh = 4 * (lane >> 5);
        float2* const out = part + (size_t)((v0 + n0) >> 6) * g.M;
        const bool edge = n0 + 64 > g.N;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const int row = m0 + i * 32 + (lane & 31);
            const int c = reinterpret_cast<const int*>(st)[i * 32 + (lane & 31)] - v0 - n0;  // the target's column among the wave's
            // column of element e, and the element with -inf past the vocabulary's end
            auto col = [&](int e) { return (e >> 4) * 32 + ((e >> 2) & 3) * 8 + nh + (e & 3); };
            auto at = [&](int e) { return edge && n0 + col(e) >= g.N ? -INFINITY : acc[i][e >> 4][e & 15]; };
            float m = -INFINITY;
#pragma unroll
            for (int e = 0; e < 32; ++e) m = fmaxf(m, at(e));
            m = fmaxf(m, __shfl_xor(m, 32));
            const float b = m == -INFINITY ? 0.f : m * kLog2e;
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < 32; ++e) s += __builtin_amdgcn_exp2f(fmaf(at(e), kLog2e, -b));
            s += __shfl_xor(s, 32);
            if (lane < 32 && row < g.M)
                out[row] = make_float2(m, m == -INFINITY ? s : s * __builtin_amdgcn_exp2f(-off(m, b)));
            if (__any((unsigned)c < 64u)) {
                float x = 0.f;
#pragma unroll
                for (int e = 0; e < 32; ++e) x = c == col(e) ? acc[i][e >> 4][e & 15] : x;
                if ((unsigned)c < 64u && (c & 4) == nh && row < g.M) lt[row] = x;
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// What a row's G takes: {b = lse log2e, (u + z) corrected for b's rounding, u, the target's column (as bits;
// -1: none)}
typedef float4 RowScale;

// G of the tile, as P bf16 pieces; columns from N up to ld are zeros.  G and then what a piece left of it
// stay in the accumulators, and the next tile's fragments are read again after the epilogue of several
// pieces: held through it they make the compiler spill 22 registers for 2 (dE of 8190 x 768 x 32000, two pieces,
// 1428 -> 1406 us; of 2001 x 1024 x 50001, three, 941 -> 902).
template <int P>
struct GradTile {
    static constexpr bool kAgain = P > 1;
    const RowScale* rows;
    bf16_t* G;      // P planes [T x ld]
    size_t plane;
    float* resid;   // [T] what rounding the target's element to the first piece left
    int ld, v0;
    template <int FM>
    __device__ __forceinline__ void begin(const GemmDesc& g, int m0, unsigned char* st, int lane) const {
        rows_begin<FM, 16>(rows, m0, g.M, st, lane);
    }
    template <int FM, int FN>
    __device__ __forceinline__ void tile(const GemmDesc& g, f32x16_t (&acc)[FM][FN], int m0, int n0, unsigned char* st,
                                         int lane) const {
        static_assert(FN == 2, "64 columns a wave");
        rows_wait();
        if (n0 >= ld) return;
        asm volatile("" : "+v"(lane));  // as above
        const int mr = lane & 31, nh = 4 * (lane >> 5);
        RowScale scales[FM];  // out of the LDS that G then goes through
#pragma unroll
        for (int i = 0; i < FM; ++i) scales[i] = reinterpret_cast<const RowScale*>(st)[i * 32 + mr];
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const RowScale rs = scales[i];
            const int mw = m0 + i * 32, row = mw + mr;
            const int c = __float_as_int(rs.w) - v0 - n0;
            const bool hit = __any((unsigned)c < 64u), edge = n0 + 64 > g.N;
            float left = 0.f;
#pragma unroll
            for (int p = 0; p < P; ++p) {
                wave_lds_sync();
#pragma unroll
                for (int k = 0; k < 8; ++k) {  // four columns: 8 k + nh
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = acc[i][k >> 2][4 * (k & 3) + e];
                    if (p == 0) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = rs.y * __builtin_amdgcn_exp2f(fmaf(x[e], kLog2e, -rs.x));
                        if (hit) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const bool at = c == 8 * k + nh + e;
                                x[e] -= at ? rs.z : 0.f;
                                left = at ? x[e] - bf2f(f2bf(x[e])) : left;
                            }
                        }
                        if (edge) {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (n0 + 8 * k + nh + e >= g.N) x[e] = 0.f;
                        }
                    }
                    const uint2 h = make_uint2(pack_bf2(x[0], x[1]), pack_bf2(x[2], x[3]));
                    *reinterpret_cast<uint2*>(st + mr * 128 + ((k ^ (mr & 7)) * 16) + nh * 2) = h;
                    if (p + 1 < P) {
                        acc[i][k >> 2][4 * (k & 3)] = x[0] - __uint_as_float(h.x << 16);
                        acc[i][k >> 2][4 * (k & 3) + 1] = x[1] - __uint_as_float(h.x & 0xffff0000u);
                        acc[i][k >> 2][4 * (k & 3) + 2] = x[2] - __uint_as_float(h.y << 16);
                        acc[i][k >> 2][4 * (k & 3) + 3] = x[3] - __uint_as_float(h.y & 0xffff0000u);
                    }
                    if (k & 1) __builtin_amdgcn_sched_barrier(0);
                }
                if (p == 0 && hit && (unsigned)c < 64u && (c & 4) == nh && row < g.M) resid[row] = left;
                wave_lds_sync();
                flush(G + p * plane, g.M, mw, n0, st, lane);
            }
        }
    }
    // 32 rows x 64 columns from the wave's LDS, as 128-byte row segments
    __device__ __forceinline__ void flush(bf16_t* to, int M, int mw, int n0, const unsigned char* st, int lane) const {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int r = q * 8 + (lane >> 3), n = n0 + (lane & 7) * 8;
            const uint4 v = *reinterpret_cast<const uint4*>(st + r * 128 + (((lane & 7) ^ (lane >> 3)) * 16));
            if (mw + r < M && n < ld) *reinterpret_cast<uint4*>(to + (size_t)(mw + r) * ld + n) = v;
        }
    }
};

// ---- bf16, up to 32 rows --------------------------------------------------------------------
// The product is then a read of E, and the tiles above read it 128 bytes of a row at a time (4.0 TB/s
// where a whole-row reader reaches 6.0: 16 x 2048 x 32000, 33 us).  Here a stage is 32 rows of E, 512
// bytes of each; eight stages (128 KB of LDS) run through, 112 KB of E on their way to each compute
// unit.  The four waves share a stage's k, 64 each, and keep their part of h in registers for all of the
// block's tiles (32 rows x NS 256 k: 16 NS registers); a tile's four partial 32 x 32 products are summed
// in LDS in the waves' order.  Lane l then has row l % 32, and of the tile's columns wave w's
// 8 w + 4 (l / 32) + 0..3.
constexpr int kFewRows = 32, kFewStages = 8, kFewStage = 32 * 512;
constexpr size_t kFewSmem = (size_t)kFewStages * kFewStage + 4 * 4096;

template <int NS, typename EPI>
__global__ __launch_bounds__(256, 1) void logits_few(const bf16_t* __restrict__ h, int T, const bf16_t* __restrict__ E,
                                                     int V, EPI epi) {
    constexpr int d = 256 * NS;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const uint32_t lds0 = lds_addr(smem_raw);
    float* const red = reinterpret_cast<float*>(smem_raw + kFewStages * kFewStage);
    const int lane = threadIdx.x & 63, row = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles = (V + 31) / 32;
    const int ntile = (tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;

    // the stream of stages: tile fi of the block, its s-th 256 k
    int fi = 0, fs = 0;
    uint32_t vo[4];
    const bf16_t* src;
    auto place = [&]() __attribute__((always_inline)) {
        const int r0 = ((int)blockIdx.x + fi * (int)gridDim.x) * 32;
        src = E + (size_t)r0 * d;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int r = 2 * (4 * wave + q) + (lane >> 5);
            vo[q] = (uint32_t)(min(r0 + r, V - 1) - r0) * (d * 2) + (uint32_t)((row ^ (r & 15)) * 16);
        }
    };
    auto issue = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            dma16s(src + fs * 256, vo[q], lds0 + (uint32_t)(slot * kFewStage + (4 * wave + q) * 1024));
        if (fs + 1 < NS) {
            ++fs;
        } else if (fi + 1 < ntile) {  // past the end: the last stage again
            ++fi;
            fs = 0;
            place();
        }
    };
    place();
#pragma unroll
    for (int k = 0; k < kFewStages - 1; ++k) issue(k);
    bf16x8_t hf[NS][4];
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
            hf[s][ks] = ld_frag16(h + (size_t)min(row, T - 1) * d + 256 * s + 64 * wave + 16 * ks + 8 * (lane >> 5));
    epi.start(T, row);
    int fo[4];  // a fragment's place in a stage
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) fo[ks] = row * 512 + (((8 * wave + 2 * ks + (lane >> 5)) ^ (row & 15)) * 16);

    int slot = 0;
    for (int i = 0; i < ntile; ++i) {
        f32x16_t acc;
        zero16(acc);
        static_for<NS>([&](auto S_) {
            constexpr int s = decltype(S_)::value;
            // this stage has landed (six may be on their way), and every wave has left the one before
            __builtin_amdgcn_s_waitcnt(vmcnt_imm(4 * (kFewStages - 2)) & 0xF0FFu);
            __syncthreads();
            issue((slot + kFewStages - 1) & (kFewStages - 1));
            const unsigned char* at = smem_raw + slot * kFewStage;
            bf16x8_t e[4];
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) e[ks] = __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const uint4*>(at + fo[ks]));
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) acc = mfma32(e[ks], hf[s][ks], acc);
            slot = (slot + 1) & (kFewStages - 1);
        });
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<float4*>(red + ((wave * 4 + q) * 64 + lane) * 4) =
                make_float4(acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]);
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(63) & 0xF0FFu);
        __syncthreads();
        float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float4 p = *reinterpret_cast<const float4*>(red + ((w * 4 + wave) * 64 + lane) * 4);
            x[0] += p.x; x[1] += p.y; x[2] += p.z; x[3] += p.w;
        }
        epi.tile(((int)blockIdx.x + i * (int)gridDim.x) * 32 + 8 * wave + 4 * (lane >> 5), V, x);
    }
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    __syncthreads();
    epi.finish(red, wave, lane);
}

// A block's statistics of each row, one strip a block; c: the target's column
struct StatsFew {
    const int32_t* tgt;
    float* lt;
    float2* part;  // [gridDim.x][T]
    int v0, strip0;
    int T, t, c;
    float m, s;
    __device__ __forceinline__ void start(int T_, int row) {
        T = T_;
        t = row;
        c = row < T ? tgt[row] - v0 : -1;
        m = -INFINITY;
        s = 0.f;
    }
    __device__ __forceinline__ void tile(int v, int V, const float (&x)[4]) {
        float y[4], n = m;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            y[e] = v + e < V ? x[e] : -INFINITY;
            n = fmaxf(n, y[e]);
        }
        const float b = n == -INFINITY ? 0.f : n;
        s = about(s, m, n);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            s += __builtin_amdgcn_exp2f((y[e] - b) * kLog2e);
            if (v + e == c && v + e < V) lt[t] = x[e];
        }
        m = n;
    }
    __device__ __forceinline__ void finish(float* red, int wave, int lane) {
        float2* const sh = reinterpret_cast<float2*>(red);
        sh[(2 * wave + (lane >> 5)) * 32 + t] = make_float2(m, s);
        __syncthreads();
        if (wave || lane >= 32 || t >= T) return;
#pragma unroll
        for (int k = 1; k < 8; ++k) join(m, s, sh[k * 32 + t].x, sh[k * 32 + t].y);
        part[(size_t)(strip0 + blockIdx.x) * T + t] = make_float2(m, s);
    }
};

// G of the tile's columns (below ld), as P bf16 pieces
template <int P>
struct GradFew {
    const RowScale* rows;
    bf16_t* G;
    size_t plane;
    float* resid;
    int ld, v0;
    int T, t, c;
    RowScale rs;
    __device__ __forceinline__ void start(int T_, int row) {
        T = T_;
        t = row;
        rs = rows[min(row, T - 1)];
        c = row < T ? __float_as_int(rs.w) - v0 : -1;
    }
    __device__ __forceinline__ void tile(int v, int V, const float (&x)[4]) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            y[e] = rs.y * __builtin_amdgcn_exp2f(fmaf(x[e], kLog2e, -rs.x));
            if (v + e == c) {
                y[e] -= rs.z;
                resid[t] = y[e] - bf2f(f2bf(y[e]));
            }
            if (v + e >= V) y[e] = 0.f;
        }
        if (t >= T || v >= ld) return;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const uint2 g = make_uint2(pack_bf2(y[0], y[1]), pack_bf2(y[2], y[3]));
            *reinterpret_cast<uint2*>(G + p * plane + (size_t)t * ld + v) = g;
            y[0] -= __uint_as_float(g.x << 16);
            y[1] -= __uint_as_float(g.x & 0xffff0000u);
            y[2] -= __uint_as_float(g.y << 16);
            y[3] -= __uint_as_float(g.y & 0xffff0000u);
        }
    }
    __device__ __forceinline__ void finish(float*, int, int) {}
};

// whether logits_few takes a product (h in registers: 32 rows of up to 2048; forward here and on the tiles: 16 x 2048 x
// 32000 31 and 36 us, 1 x 2048 x 128000 94 and 110), and its blocks (and strips of statistics) over N columns: no more than
// the tiles' strips of 64, which the workspace has room for
bool few_takes(const GemmDesc& g) { return g.M <= kFewRows && g.Ks[0] % 256 == 0 && g.Ks[0] <= 2048; }
int few_blocks(int N) { return std::min((N + 63) / 64, stream_blocks()); }

template <int NS, typename EPI>
int launch_few(const GemmDesc& g, const EPI& epi, hipStream_t s) {
    static const bool ok = allow_lds(logits_few<NS, EPI>, kFewSmem);
    if (!ok) {
        set_error("linear xent: cannot reserve %zu B of LDS", kFewSmem);
        return GN_E_HIP;
    }
    hipLaunchKernelGGL((logits_few<NS, EPI>), dim3(few_blocks(g.N)), dim3(256), kFewSmem, s, g.A[0], g.M, g.B[0], g.N, epi);
    GN_LAUNCH_CHECK("linear xent (logits of few rows)");
    return GN_OK;
}

template <typename EPI>
int launch_few(const GemmDesc& g, const EPI& epi, hipStream_t s) {
    switch (g.Ks[0] / 256) {
        case 1: return launch_few<1>(g, epi, s);
        case 2: return launch_few<2>(g, epi, s);
        case 3: return launch_few<3>(g, epi, s);
        case 4: return launch_few<4>(g, epi, s);
        case 5: return launch_few<5>(g, epi, s);
        case 6: return launch_few<6>(g, epi, s);
        case 7: return launch_few<7>(g, epi, s);
        default: return launch_few<8>(g, epi, s);
    }
}

template <int BM, int STAGES, typename EPI>
int launch_logits_tile(const GemmDesc& g, const EPI& epi, hipStream_t s) {
    constexpr int BN = 128;
    constexpr size_t smem = (size_t)STAGES * (BM + BN) * BK * sizeof(bf16_t) + 4 * 4096;
    static_assert(smem <= 160 * 1024, "LDS per CU");
    static const bool ok = allow_lds(gemm_stream<false, true, float, BM, BN, STAGES, EPI>, smem);
    if (!ok) {
        set_error("linear xent: cannot reserve %zu B of LDS", smem);
        return GN_E_HIP;
    }
    const long tiles = (long)((g.M + BM - 1) / BM) * ((g.N + BN - 1) / BN);
    const unsigned grid = (unsigned)std::min<long>(tiles, stream_blocks());
    hipLaunchKernelGGL((gemm_stream<false, true, float, BM, BN, STAGES, EPI>), dim3(grid), dim3(512), smem, s, g, epi);
    GN_LAUNCH_CHECK("linear xent (logits)");
    return GN_OK;
}

// 256-row tiles, or 128-row ones where they need less (the streamed products' rule: a round of them
// takes 0.6 of a round of the large).  Up to 64 rows 64-row tiles, which leave the LDS to six stages: a
// read of E again (64 x 1024 x 50000 forward 28.6 us).
template <typename EPI>
int launch_logits(const GemmDesc& g, const EPI& epi, hipStream_t s) {
    const long blocks = stream_blocks(), tn = (g.N + 127) / 128;
    const long r256 = ((g.M + 255) / 256 * tn + blocks - 1) / blocks, r128 = ((g.M + 127) / 128 * tn + blocks - 1) / blocks;
    if (g.M <= 64) return launch_logits_tile<64, 6>(g, epi, s);
    return 0.62 * (double)r128 < (double)r256 ? launch_logits_tile<128, 3>(g, epi, s) : launch_logits_tile<256, 3>(g, epi, s);
}

// The loss is (m - target's logit) + ln s, not lse less the logit: of far logits lse has lost a confident row's
// loss to its rounding (2^-16 at 300).
__device__ __forceinline__ void finish_row(int t, float m, float s, const int32_t* tgt, const float* lt, float* loss,
                                           float* lse, int V) {
    const float ln = __builtin_amdgcn_logf(s) * kLn2;
    if (lse) lse[t] = m + ln;
    const int g = tgt[t];
    if (loss) loss[t] = g >= 0 && g < V ? (m - lt[t]) + ln : 0.f;
}

// lse and loss from the strips' statistics: R rows x 256 / R slices of the strips a block.  2 below 256 rows
// (whole forwards of 16 rows: the 256 strips that logits_few leaves at d = 2048 29.8 us, with 16 30.1; the 500 of
// the tiles at d = 4096 43.6 and 44.7), 16 from there on (782 strips of 2001 rows: 9.5 us, with 2 16).
template <int R>
__global__ __launch_bounds__(256) void row_stats(const float2* __restrict__ part, int strips, int T,
                                                 const int32_t* __restrict__ tgt, const float* __restrict__ lt,
                                                 float* __restrict__ loss, float* __restrict__ lse, int V) {
    constexpr int SL = 256 / R;
    __shared__ float2 sh[SL][R + 1];
    const int r = threadIdx.x % R, sl = threadIdx.x / R, t = blockIdx.x * R + r;
    float m = -INFINITY, s = 0.f;
    if (t < T) {
        for (int k = sl; k < strips; k += 8 * SL) {
            float2 p[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                p[j] = k + SL * j < strips ? part[(size_t)(k + SL * j) * T + t] : make_float2(-INFINITY, 0.f);
            float n = m;
#pragma unroll
            for (int j = 0; j < 8; ++j) n = fmaxf(n, p[j].x);
            s = about(s, m, n);
#pragma unroll
            for (int j = 0; j < 8; ++j) s += about(p[j].y, p[j].x, n);
            m = n;
        }
    }
    sh[sl][r] = make_float2(m, s);
    for (int k = SL / 2; k > 0; k /= 2) {
        __syncthreads();
        if (sl < k) {
            const float2 o = sh[sl + k][r];
            join(m, s, o.x, o.y);
            sh[sl][r] = make_float2(m, s);
        }
    }
    if (sl == 0 && t < T) finish_row(t, m, s, tgt, lt, loss, lse, V);
}

// Every row's scales, and no residual yet; rows from T up to Tp (the fp32 products' padding) have none.
__global__ __launch_bounds__(256) void row_scales(RowScale* __restrict__ rows, float* __restrict__ resid, int T, int Tp,
                                                  const int32_t* __restrict__ tgt, const float* __restrict__ lse,
                                                  const float* __restrict__ dloss, const float* __restrict__ dlse,
                                                  float scale, int V) {
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t >= Tp) return;
    RowScale r = make_float4(0.f, 0.f, 0.f, __int_as_float(-1));
    if (t < T) {
        const int g = tgt[t];
        const bool has = g >= 0 && g < V;
        const float u = has ? (dloss ? scale * dloss[t] : scale) : 0.f;
        const float b = lse[t] * kLog2e, a = u + (dlse ? scale * dlse[t] : 0.f);
        r = make_float4(b, a * __builtin_amdgcn_exp2f(-off(lse[t], b)), u, __int_as_float(has ? g : -1));
    }
    rows[t] = r;
    resid[t] = 0.f;
}

// ---- fp32: row kernels over a piece's stored logits -------------------------------------------
// A launch's threads in one dimension are counted in 32 bits, which a row a block of 256 would pass at
// 2^24 rows: blocks go on in another dimension from 2^22 on.
constexpr int kRowsX = 1 << 22;
inline dim3 blocks_of(int n, int y = 1) { return dim3(std::min(n, kRowsX), y, (n - 1) / kRowsX + 1); }
__device__ __forceinline__ int block_of() { return blockIdx.z * gridDim.x + blockIdx.x; }

// A row's statistics over one piece, joined with those of the pieces before (st); the last
// piece's are turned into lse and loss.  ld and L are multiples of 4 elements and 16 bytes.
__global__ __launch_bounds__(256) void piece_stats(const float* __restrict__ L, int ld, int T, int v0, int nv,
                                                   const int32_t* __restrict__ tgt, float2* __restrict__ st,
                                                   float* __restrict__ lt, float* __restrict__ loss,
                                                   float* __restrict__ lse, int V, int first, int last) {
    __shared__ float sm[4], ss[4];
    const int t = block_of();
    if (t >= T) return;
    const float* row = L + (size_t)t * ld;
    float m = -INFINITY, s = 0.f;
    for (int v = 4 * threadIdx.x; v < nv; v += 4096) {
        float x[16];
        float n = m;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = v + 1024 * j;
            const float4 q = c < nv ? *reinterpret_cast<const float4*>(row + c)
                                    : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            x[4 * j] = q.x;
            x[4 * j + 1] = c + 1 < nv ? q.y : -INFINITY;
            x[4 * j + 2] = c + 2 < nv ? q.z : -INFINITY;
            x[4 * j + 3] = c + 3 < nv ? q.w : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) n = fmaxf(n, x[e]);
        const float b = n == -INFINITY ? 0.f : n;
        s = about(s, m, n);
#pragma unroll
        for (int e = 0; e < 16; ++e) s += __builtin_amdgcn_exp2f((x[e] - b) * kLog2e);
        m = n;
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
    if (last) finish_row(t, m, s, tgt, lt, loss, lse, V);
    else st[t] = make_float2(m, s);
}

// G of one piece in its logits' place, zeros from nv up to the next multiple of 4
__global__ __launch_bounds__(256) void piece_grad(float* __restrict__ L, int ld, int Tp, int v0, int nv,
                                                  const RowScale* __restrict__ rows) {
    const int t = block_of();
    if (t >= Tp) return;
    const RowScale r = rows[t];
    float* const row = L + (size_t)t * ld;
    const int g = __float_as_int(r.w) - v0;
    for (int v = 4 * (blockIdx.y * 256 + threadIdx.x); v < nv; v += 1024 * gridDim.y) {
        float4* p = reinterpret_cast<float4*>(row + v);
        const float4 q = *p;
        float x[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] = r.y * __builtin_amdgcn_exp2f(fmaf(x[e], kLog2e, -r.x));
            if (v + e == g) x[e] -= r.z;
            if (v + e >= nv) x[e] = 0.f;
        }
        *p = make_float4(x[0], x[1], x[2], x[3]);
    }
}

// The last nv % 4 logits of a piece's rows: a wave's dot product each, L[t][nq + j] = h[t] . E[j];
// zeros in the padding's rows
__global__ __launch_bounds__(256) void tail_logits(const float* __restrict__ h, const float* __restrict__ E,
                                                   float* __restrict__ L, int ld, int T, int Tp, int d, int tail) {
    const int64_t w = block_of() * (int64_t)4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, t = (int)(w / tail), j = (int)(w - (int64_t)t * tail);
    if (t >= Tp) return;
    float s = 0.f;
    for (int k = lane; t < T && k < d; k += 64) s = fmaf(h[(size_t)t * d + k], E[(size_t)j * d + k], s);
    s = wave_sum(s);
    if (lane == 0) L[(size_t)t * ld + j] = s;
}

// ---- both ---------------------------------------------------------------------------------
// dst [Rp x dp] = src [R x d], zeros around it, `times` over
template <typename T>
__global__ __launch_bounds__(256) void lay_out(const T* __restrict__ src, T* __restrict__ dst, int R, int d, int Rp, int dp,
                                               int times) {
    const int64_t n = (int64_t)Rp * dp;
    for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int r = (int)(i / dp), c = (int)(i - (int64_t)r * dp);
        const T v = r < R && c < d ? src[(size_t)r * d + c] : (T)0;
        for (int k = 0; k < times; ++k) dst[k * n + i] = v;
    }
}

// dst [R x d] (+)= src [R x dp]
template <typename T>
__global__ __launch_bounds__(256) void take_rows(const float* __restrict__ src, T* __restrict__ dst, int R, int d, int dp,
                                                 int accumulate) {
    const int64_t n = (int64_t)R * d;
    for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int r = (int)(i / d), c = (int)(i - (int64_t)r * d);
        const float v = src[(size_t)r * dp + c];
        io<T>::st(dst, i, accumulate ? v + io<T>::ld(dst, i) : v);
    }
}

// dh's rows from their fp32 sums (acc [T x dp], nullptr: nothing), the target's residual and the
// last `tail` columns of the vocabulary (G [T x ld] from that column on, Et its rows of E)
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void dh_finish(const float* __restrict__ acc, int dp, const RowScale* __restrict__ rows,
                                                 const float* __restrict__ resid, const T* __restrict__ E,
                                                 const T* __restrict__ G, int ld, const T* __restrict__ Et, int tail,
                                                 T* __restrict__ dh, int n, int d) {
    constexpr int W = VEC ? 8 : 1;
    const int per = d / W;
    const int64_t all = (int64_t)n * per;
    for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int t = (int)(i / per), c = (int)(i - (int64_t)t * per) * W;
        float v[8], e[8];
        auto add = [&](float f, const T* p) {
            if constexpr (VEC) chunk8<T>::ld(p + c, e);
            else e[0] = io<T>::ld(p, c);
#pragma unroll
            for (int j = 0; j < W; ++j) v[j] += f * e[j];
        };
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = 0.f;
        if (acc) {
            if constexpr (VEC) chunk8<float>::ld(acc + (size_t)t * dp + c, v);
            else v[0] = acc[(size_t)t * dp + c];
        }
        const float f = resid[t];
        if (f != 0.f) add(f, E + (size_t)__float_as_int(rows[t].w) * d);
        for (int j = 0; j < tail; ++j) add(io<T>::ld(G, (size_t)t * ld + j), Et + (size_t)j * d);
        if constexpr (VEC) chunk8<T>::st(dh + (size_t)t * d + c, v);
        else io<T>::st(dh, (size_t)t * d + c, v[0]);
    }
}

// ---- bf16, an fp32 dE of two pieces -------------------------------------------------------------
// What the pieces left of the target elements (resid less its rounding) times h, onto dE: the largest
// elements of G by far while p is small, alike in every row of a mean, and so what the 2^-17 showed in (dE of
// 8192 x 2048 x 128000 off by 3.5e-6 of its norm before and by 0.9e-6 now; fp32 torch products are by
// 1.6e-6).  Block t has the tokens of t's target in their order, if t is the first of them; it finds them
// by reading the targets through, 1024 at a time: latency, eight blocks a compute unit against it (63 us of
// the 18.8 ms there, 5 blocks 80).
template <bool VEC>
__global__ __launch_bounds__(256, 8) void target_rest(const int32_t* __restrict__ tgt, const float* __restrict__ resid,
                                                   const bf16_t* __restrict__ h, float* __restrict__ dE, int T, int d,
                                                   int V) {
    constexpr int W = VEC ? 8 : 1;
    __shared__ int who[1024];
    __shared__ float rest[1024];
    __shared__ int count[16];
    const int t = blockIdx.x, c = tgt[t];
    if (c < 0 || c >= V) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i0 = 0; i0 < t; i0 += 1024) {
        bool before = false;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = i0 + 256 * k + threadIdx.x;
            before |= i < t && tgt[i] == c;
        }
        if (__syncthreads_or(before)) return;
    }
    for (int i0 = t; i0 < T; i0 += 1024) {
        unsigned long long m[4], any = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = i0 + 256 * k + threadIdx.x;
            m[k] = __ballot(i < T && tgt[i] == c);
            any |= m[k];
            if (lane == 0) count[4 * k + wave] = __popcll(m[k]);
        }
        if (!__syncthreads_or(any != 0)) continue;
        int n = 0;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            if ((k & 3) == wave && (m[k >> 2] >> lane & 1)) {
                const int j = n + __popcll(m[k >> 2] & ((1ull << lane) - 1)), i = i0 + 256 * (k >> 2) + threadIdx.x;
                const float r = resid[i];
                who[j] = i;
                rest[j] = r - bf2f(f2bf(r));
            }
            n += count[k];
        }
        __syncthreads();
        for (int j = threadIdx.x * W; j < d; j += 256 * W) {
            float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, e[8];
#pragma unroll 4
            for (int k = 0; k < n; ++k) {
                const bf16_t* p = h + (size_t)who[k] * d + j;
                if constexpr (VEC) chunk8<bf16_t>::ld(p, e);
                else e[0] = bf2f(*p);
#pragma unroll
                for (int q = 0; q < W; ++q) v[q] = fmaf(rest[k], e[q], v[q]);
            }
            float* const to = dE + (size_t)c * d + j;
            if constexpr (VEC) chunk8<float>::ld(to, e);
            else e[0] = *to;
#pragma unroll
            for (int q = 0; q < W; ++q) e[q] += v[q];
            if constexpr (VEC) chunk8<float>::st(to, e);
            else *to = e[0];
        }
        __syncthreads();
    }
}

// ---- bf16, few rows: dh -----------------------------------------------------------------------
// dh = G E over the whole vocabulary is a read of E too, with a long k and few outputs, which the products'
// splits in eight left on 64 blocks (16 rows, 32000 x 2048: 70 us of dh alone).  Here a block takes 256
// columns, 32 RT rows and one of S ranges of the vocabulary, 64 rows of E (512 bytes of each) and of G a
// stage, four stages in LDS; its partial sums go to plane blockIdx.y, added in order afterwards.
constexpr int kFewDhStages = 4;
template <int RT>
constexpr size_t few_dh_smem = (size_t)kFewDhStages * (256 + 32 * RT) * BK * 2;

template <int RT>
__global__ __launch_bounds__(256, 1) void dh_few(const bf16_t* __restrict__ G, int ldg, const bf16_t* __restrict__ E, int nv,
                                                 int T, int N, int per, float* __restrict__ part) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const uint32_t lds0 = lds_addr(smem_raw);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr int kStage = (256 + 32 * RT) * BK * 2;
    const int t0 = blockIdx.z * 32 * RT, n0 = blockIdx.x * 256;
    const int k0 = blockIdx.y * per, k1 = min(nv, k0 + per), KT = (k1 - k0 + BK - 1) / BK;
    constexpr int ND = 256 / 32 + RT;  // DMA instructions of a wave a stage
    // E's rows past the range's end are read as zeros, and G's past its columns (zeros up to a multiple of 8)
    auto issue = [&](int t) __attribute__((always_inline)) {
        const int k = k0 + min(t, KT - 1) * BK;
        const uint32_t base = lds0 + (uint32_t)((t & (kFewDhStages - 1)) * kStage);
        stage_tail<256, false, 4>(E, N, n0, N, k, k1, wave, base);
        stage_tail<32 * RT, true, 4>(G, ldg, t0, T, k, (k1 + 7) & ~7, wave, base + 256 * BK * 2);
    };
    f32x16_t acc[RT][2];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        zero16(acc[i][0]);
        zero16(acc[i][1]);
    }
#pragma unroll
    for (int t = 0; t < kFewDhStages - 1; ++t) issue(t);
    for (int t = 0; t < KT; ++t) {
        __builtin_amdgcn_s_waitcnt(vmcnt_imm((kFewDhStages - 2) * ND) & 0xF0FFu);
        __syncthreads();  // stage t has landed, and every wave has left the one before
        issue(t + kFewDhStages - 1);
        const bf16_t* e = reinterpret_cast<const bf16_t*>(smem_raw + (t & (kFewDhStages - 1)) * kStage);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            const bf16x8_t b0 = frag<256, false>(e, wave * 64, ks), b1 = frag<256, false>(e, wave * 64 + 32, ks);
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const bf16x8_t a = frag<32 * RT, true>(e + 256 * BK, 32 * i, ks);
                acc[i][0] = mfma32(a, b0, acc[i][0]);
                acc[i][1] = mfma32(a, b1, acc[i][1]);
            }
        }
    }
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    float* const out = part + (size_t)blockIdx.y * T * N;
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int n = n0 + wave * 64 + j * 32 + (lane & 31);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int t = t0 + 32 * i + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
                if (t < T && n < N) out[(size_t)t * N + n] = acc[i][j][r];
            }
        }
}

// Taken up to 128 rows from three million elements of E on.  dh alone, microseconds here and through the
// library's products: 64 x 1024 x 50000 79 and 135, 128 x 1024 x 50000 96 and 130, 128 x 768 x 8000 32.5 and
// 33.4, 64 x 512 x 8000 28 and 32; at 256 rows 111 and 103.  Below, the second launch costs more than the
// ranges give: 64 x 512 x 4000 25 and 24, 16 x 256 x 2000 21 and 18.
constexpr int kFewDhRows = 128;
inline bool dh_few_takes(int T, int V, int N) { return T <= kFewDhRows && (size_t)V * N >= 3u << 20; }

// ranges of the vocabulary at most (two blocks a compute unit), the rows of one for nv in all (whole stages,
// four at least), and their number, which is no more than few_dh_most or nv / 256 rounded up
int few_dh_most(int T, int N) { return std::max(1, 2 * stream_blocks() / ((N + 255) / 256 * ((T + 63) / 64))); }
int few_dh_rows(int nv, int T, int N) {
    const int most = few_dh_most(T, N);
    return std::max(4 * BK, ((nv + most - 1) / most + BK - 1) / BK * BK);
}
int few_dh_ranges(int nv, int T, int N) { return (nv + few_dh_rows(nv, T, N) - 1) / few_dh_rows(nv, T, N); }

template <int RT>
int launch_dh_few(const GemmDesc& g, hipStream_t s) {
    static const bool ok = allow_lds(dh_few<RT>, few_dh_smem<RT>);
    if (!ok) {
        set_error("linear xent: cannot reserve %zu B of LDS", few_dh_smem<RT>);
        return GN_E_HIP;
    }
    dh_few<RT><<<dim3((g.N + 255) / 256, g.ksplit, (g.M + 32 * RT - 1) / (32 * RT)), 256, few_dh_smem<RT>, s>>>(
        g.A[0], g.lda[0], g.B[0], g.Ks[0], g.M, g.N, few_dh_rows(g.Ks[0], g.M, g.N), g.part);
    GN_LAUNCH_CHECK("linear xent (dh of few rows)");
    launch_split_reduce(g, s);
    GN_LAUNCH_CHECK("linear xent (dh of few rows, sums)");
    return GN_OK;
}

// ---- host -----------------------------------------------------------------------------------
inline bool al16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
inline int round_up(int n, int q) { return (n + q - 1) / q * q; }

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

// A call's shapes and its workspace.  lay: h, E's pieces and dE go through copies in the products'
// layout (widths that are no multiple of q, or tensors off the 16-byte grid).
struct Plan {
    bool bf, lay;
    int T, d, V, q, es, dp, Tp;
    int planes;      // bf16: pieces of G that an fp32 dE takes
    int vc, pieces;  // columns of a piece, a multiple of 128 (or all of a smaller vocabulary)
    size_t h, hs, E, lt, rows, resid, stats, logits, G, acc, de, det, part, part_bytes, bytes;

    Plan(int T_, int d_, int V_, int dtype, bool lay_, bool bwd) : bf(dtype == GN_BF16), lay(lay_), T(T_), d(d_), V(V_) {
        q = bf ? 8 : 4;
        es = bf ? 2 : 4;
        lay = lay || d % q;
        dp = round_up(d, q);
        Tp = bf ? T : round_up(T, 4);
        planes = T > kTwoPieces ? 2 : 3;
        // a piece's G, or the fp32 logits it replaces
        int64_t most = kPieceBytes / (lay ? 4 : 1) / (bf ? 2 * planes : 4) / std::max(Tp, 1);
        if (lay) most = std::min(most, kPieceBytes / ((int64_t)dp * (es + 4)));  // the copies of E's and dE's piece
        // whole rounds of 256 x 128 tiles of dE's product on the compute units, or what there is room for
        const int64_t round = (int64_t)std::max(1, stream_blocks() / ((dp + 127) / 128)) * 256;
        int64_t cols = most >= round ? most / round * round : 2 * most >= round ? round : most / 128 * 128;
        vc = (int)std::min<int64_t>(round_up(V, 128), std::max<int64_t>(512, cols));
        pieces = (V + vc - 1) / vc;
        // the products' own split workspaces: of a whole piece and of the last one
        part_bytes = 0;
        const int last = (V - (pieces - 1) * vc) / q * q;
        for (int nv : {pieces > 1 ? vc : 0, last, V % q ? q : 0}) {
            if (nv <= 0 || (bf && !bwd)) continue;
            GemmDesc a = product(nullptr, vc, nullptr, dp, Tp, nullptr, dp, nv, dp);
            GemmDesc b = product(nullptr, vc, nullptr, dp, nv, nullptr, dp, Tp, dp);
            if (bf) {
                if (planes == 2) {
                    a.nseg = 2;
                    a.lda[1] = vc;
                    a.ldb[1] = dp;
                    a.Ks[1] = T;
                } else {
                    a.Ks[0] = 3 * T;
                }
                part_bytes = std::max({part_bytes, gemm_dma_part_bytes(a, 1, GN_F32), gemm_dma_part_bytes(b, 0, GN_F32)});
                a.accumulate = b.accumulate = 1;
                part_bytes = std::max({part_bytes, gemm_dma_part_bytes(a, 1, GN_F32), gemm_dma_part_bytes(b, 0, GN_F32)});
            } else {
                const GemmDesc l = product(nullptr, dp, nullptr, dp, dp, nullptr, vc, Tp, nv);
                part_bytes = std::max({part_bytes, gemm_f32_part_bytes(a), gemm_f32_part_bytes(b), gemm_f32_part_bytes(l)});
            }
        }
        if (bf && bwd && dh_few_takes(T, V, dp))
            part_bytes = std::max(part_bytes, (size_t)std::min(few_dh_most(T, dp), (vc + 255) / 256) * T * dp * sizeof(float));
        size_t at = 0;
        auto take = [&](size_t n) {
            const size_t p = at;
            at += (n + 255) / 256 * 256;
            return p;
        };
        h = take(lay || Tp != T ? (size_t)Tp * dp * es : 0);
        E = take(lay ? (size_t)vc * dp * es : 0);
        lt = take((size_t)T * 4);
        logits = take(bf ? 0 : (size_t)Tp * vc * 4);
        part = take(part_bytes);
        if (!bwd) {
            stats = take(bf ? (size_t)((V + 127) / 128 * 2) * T * 8 : (size_t)T * 8);
            bytes = at;
            return;
        }
        rows = take((size_t)Tp * sizeof(RowScale));
        resid = take((size_t)Tp * 4);
        hs = take(bf && planes == 3 ? (size_t)3 * T * dp * 2 : 0);
        G = take(bf ? (size_t)planes * T * vc * 2 : 0);
        acc = take((size_t)Tp * dp * 4);
        de = take(lay ? (size_t)vc * dp * 4 : 0);
        det = take((size_t)q * dp * 4);
        bytes = at;
    }
    // Measured (us, pieces of 128, 256, 512, 1024 MB in plain multiples of 128 columns): 8190 x 768 x
    // 32000 2479, 2376, 2412, 2238; 2001 x 1024 x 50001 971, 931, 920, 918; 8192 x 2048 x 128000 19.7,
    // 19.1, 20.1, 20.0 ms.  Whole rounds at 256 MB took the backward of the first 1821 -> 1793, of the
    // second (bf16 dE) 709 -> 678.
    // Rows from which an fp32 dE takes two pieces of G (2^-17 of an element): the fp32 sum over that many
    // rows is itself no better (sqrt(4096) 2^-24 = 2^-18).  Below it takes three, as good as fp32 (of 8192 x
    // 2048 x 128000 23.5 ms in place of 18.9, of 8190 x 768 x 32000 2.56 in place of 2.13).  Up to kTargets
    // rows target_rest makes the target elements whole; its reading grows with the square of the rows, and
    // beyond sqrt(16384) 2^-24 = 2^-17.
    static constexpr int kTwoPieces = 4096, kTargets = 16384;
    // Rows up to which a bf16 dE takes two pieces.  Its norm lies in the targets' rows, each of them G's element
    // at the target, with its rounding, times a row of h: of few rows the error is up to twice what dE's own
    // rounding leaves (16 x 768 x 32000 3.4e-3 for 1.66e-3, 256 x 768 2.9e-3, 512 x 2048 2.6e-3), of many it
    // is about sqrt 2 times that (2001 x 1024 x 50001 2.25e-3).  Both gradients, one piece and two, us: 16 x 2048 x 32000
    // 98 and 102, 64 107 and 118, 128 126 and 146, 512 224 and 287; 2001 x 1024 x 50001 688 and 905, 8190 x 768 x
    // 32000 1210 and 1812.
    static constexpr int kWholeBf16 = 512;
    static constexpr int64_t kPieceBytes = (int64_t)256 << 20;
};

// of either direction, whatever the tensors' alignment
size_t workspace_bytes(int T, int d, int V, int dtype) {
    size_t most = 0;
    for (const bool lay : {false, true})
        for (const bool bwd : {false, true}) most = std::max(most, Plan(T, d, V, dtype, lay, bwd).bytes);
    return most;
}

// the sizes taken: the products count their tiles, and a block its k-tiles, in 31 bits
bool within(int T, int d, int V) {
    return T < (1 << 28) && d <= (1 << 20) && V < (1 << 30) && (int64_t)T * V < (1ll << 43) && (double)T * V * d < 0x1p58;
}

int check(const char* who, const void* h, const void* E, const int32_t* tgt, int T, int d, int V, int dtype) {
    GN_REQUIRE(dtype == GN_F32 || dtype == GN_BF16, "%s: dtype %d not supported (f32, bf16)", who, dtype);
    GN_REQUIRE(T >= 0 && d >= 1 && V >= 1, "%s: bad shape", who);
    GN_REQUIRE(within(T, d, V), "%s: T below 2^28, d up to 2^20, V below 2^30, T * V below 2^43, T * V * d below 2^58", who);
    GN_REQUIRE(T == 0 || (h && E && tgt), "%s: null pointer", who);
    const int es = dtype == GN_F32 ? 4 : 2;
    GN_REQUIRE((((uintptr_t)h | (uintptr_t)E) & (es - 1)) == 0 && ((uintptr_t)tgt & 3u) == 0,
               "%s: a tensor is not aligned to its elements", who);
    return GN_OK;
}

// A tensor of a call, or its workspace
struct Span {
    const void* p;
    size_t bytes;
    const char* name;
    bool written;
};

// What is written may share no memory with anything else of the call.
template <int N>
int check_spans(const char* who, const Span (&t)[N]) {
    for (int i = 0; i < N; ++i)
        for (int j = 0; j < N && t[i].written; ++j)
            GN_REQUIRE(i == j || !t[i].p || !t[j].p || (const char*)t[i].p >= (const char*)t[j].p + t[j].bytes ||
                           (const char*)t[j].p >= (const char*)t[i].p + t[i].bytes,
                       "%s: %s and %s may not share memory", who, t[i].name, t[j].name);
    return GN_OK;
}

int check_ws(const char* who, const Plan& w, int dtype, const void* ws, size_t ws_bytes) {
    // the query's answer for the shape at hand (four plans, some microseconds)
    thread_local int of[4] = {0, 0, 0, 0};
    thread_local size_t need = 0;
    if (of[0] != w.T || of[1] != w.d || of[2] != w.V || of[3] != dtype) {
        need = workspace_bytes(w.T, w.d, w.V, dtype);
        of[0] = w.T, of[1] = w.d, of[2] = w.V, of[3] = dtype;
    }
    if (!ws || ws_bytes < need || !al16(ws)) {
        set_error("%s: workspace of %zu bytes (16-byte aligned) required", who, need);
        return GN_E_WORKSPACE;
    }
    return GN_OK;
}

// One call's tensors in the products' layout.
struct Call {
    const char* who;
    const Plan& w;
    char* base;
    const void *h, *E;
    hipStream_t s;
    int dtype;
    const void* hp = nullptr;  // [Tp x dp]

    int copy(const void* src, size_t to, int R, int Rp, int times = 1) {
        const unsigned grid = grid_for((int64_t)Rp * w.dp, 1024, 16384);
        if (w.bf) lay_out<bf16_t><<<grid, 256, 0, s>>>((const bf16_t*)src, (bf16_t*)(base + to), R, w.d, Rp, w.dp, times);
        else lay_out<float><<<grid, 256, 0, s>>>((const float*)src, (float*)(base + to), R, w.d, Rp, w.dp, times);
        GN_LAUNCH_CHECK(who);
        return GN_OK;
    }
    int start() {
        hp = h;
        if (!w.lay && w.Tp == w.T) return GN_OK;
        hp = base + w.h;
        return copy(h, w.h, w.T, w.Tp);
    }
    // rows v0 .. v0 + nv of E as the products take them
    int piece(int v0, int nv, const void** Ec) {
        *Ec = (const char*)E + (size_t)v0 * w.d * w.es;
        if (!w.lay) return GN_OK;
        const int rc = copy(*Ec, w.E, nv, std::min(round_up(nv, w.q), w.vc));
        *Ec = base + w.E;
        return rc;
    }
    void scratch(GemmDesc& g) {
        g.part = (float*)(base + w.part);
        g.part_cap = w.part_bytes;
    }
    // fp32: a piece's logits
    int logits32(const void* Ec, int nv) {
        float* const L = (float*)(base + w.logits);
        const int nq = nv / w.q * w.q, cols = w.lay ? round_up(nv, w.q) : nq;
        if (cols) {
            GemmDesc g = product(hp, w.dp, Ec, w.dp, w.dp, L, w.vc, w.Tp, cols);
            scratch(g);
            if (const int rc = gemm_run(g, 0, 1, dtype, GN_F32, s)) return rc;
        }
        if (cols >= nv) return GN_OK;
        tail_logits<<<blocks_of((w.Tp * (nv - nq) + 3) / 4), 256, 0, s>>>((const float*)h, (const float*)Ec + (size_t)nq * w.d, L + nq,
                                                             w.vc, w.T, w.Tp, w.d, nv - nq);
        GN_LAUNCH_CHECK(who);
        return GN_OK;
    }
};

}  // namespace
}  // namespace gn

using namespace gn;

extern "C" size_t gn_linear_xent_workspace_bytes(int T, int d, int V, int dtype) {
    if (T <= 0 || d <= 0 || V <= 0 || !within(T, d, V) || (dtype != GN_F32 && dtype != GN_BF16)) return 0;
    return workspace_bytes(T, d, V, dtype);
}

extern "C" int gn_linear_xent_fwd(const void* h, const void* E, const int32_t* targets, float* loss, float* lse, int T,
                                  int d, int V, int dtype, void* ws, size_t ws_bytes, void* stream) {
    const char* who = "gn_linear_xent_fwd";
    clear_error();
    if (const int rc = check(who, h, E, targets, T, d, V, dtype)) return rc;
    GN_REQUIRE((((uintptr_t)loss | (uintptr_t)lse) & 3u) == 0, "%s: loss, lse must be aligned to 4 bytes", who);
    if (T == 0 || (!loss && !lse)) return GN_OK;
    const Plan w(T, d, V, dtype, !al16(h) || !al16(E), false);
    const size_t es = dtype == GN_F32 ? 4 : 2, row = (size_t)T * 4;
    const Span spans[] = {{h, (size_t)T * d * es, "h", false}, {E, (size_t)V * d * es, "E", false}, {targets, row, "targets", false},
                          {loss, row, "loss", true}, {lse, row, "lse", true}, {ws, w.bytes, "the workspace", true}};
    if (const int rc = check_spans(who, spans)) return rc;
    if (const int rc = check_ws(who, w, dtype, ws, ws_bytes)) return rc;
    char* const base = (char*)ws;
    Call c{who, w, base, h, E, as_stream(stream), dtype};
    if (const int rc = c.start()) return rc;
    float* const lt = (float*)(base + w.lt);
    int strips = 0;
    const int step = w.bf && !w.lay ? V : w.vc;  // all at once where E is read as it lies
    for (int v0 = 0; v0 < V; v0 += step) {
        const int nv = std::min(step, V - v0);
        const void* Ec;
        if (const int rc = c.piece(v0, nv, &Ec)) return rc;
        if (w.bf) {
            const GemmDesc g = product(c.hp, w.dp, Ec, w.dp, w.dp, nullptr, 0, T, nv);
            float2* const part = (float2*)(base + w.stats);
            const int rc = few_takes(g) ? launch_few(g, StatsFew{targets, lt, part, v0, strips}, c.s)
                                        : launch_logits(g, StatsTile{targets, lt, part, v0}, c.s);
            if (rc) return rc;
            strips += few_takes(g) ? few_blocks(nv) : (nv + 63) / 64;
        } else {
            if (const int rc = c.logits32(Ec, nv)) return rc;
            piece_stats<<<blocks_of(T), 256, 0, c.s>>>((const float*)(base + w.logits), w.vc, T, v0, nv, targets,
                                                       (float2*)(base + w.stats), lt, loss, lse, V, v0 == 0, v0 + nv == V);
            GN_LAUNCH_CHECK(who);
        }
    }
    if (w.bf) {
        const float2* part = (const float2*)(base + w.stats);
        if (T < 256) row_stats<2><<<(T + 1) / 2, 256, 0, c.s>>>(part, strips, T, targets, lt, loss, lse, V);
        else row_stats<16><<<(T + 15) / 16, 256, 0, c.s>>>(part, strips, T, targets, lt, loss, lse, V);
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
    const int des = dE_dtype == GN_F32 ? 4 : 2;
    GN_REQUIRE(!acc || dE_dtype == GN_F32, "%s: only an fp32 dE accumulates", who);
    GN_REQUIRE(((uintptr_t)dE & (des - 1)) == 0 && ((uintptr_t)dh & (dtype == GN_F32 ? 3u : 1u)) == 0 &&
                   (((uintptr_t)lse | (uintptr_t)dloss | (uintptr_t)dlse) & 3u) == 0,
               "%s: a tensor is not aligned to its elements", who);
    hipStream_t s = as_stream(stream);
    if (T == 0) {  // no rows: dE is zero
        if (dE && !acc && launch_zero(dE, (size_t)V * d * des, s) != hipSuccess) {
            set_error("%s: clear failed", who);
            return GN_E_HIP;
        }
        return GN_OK;
    }
    GN_REQUIRE(lse, "%s: null pointer", who);
    if (!dh && !dE) return GN_OK;
    const Plan w(T, d, V, dtype, !al16(h) || !al16(E) || !al16(dE), true);
    const size_t es = dtype == GN_F32 ? 4 : 2, nh = (size_t)T * d * es, nE = (size_t)V * d, row = (size_t)T * 4;
    const Span spans[] = {{h, nh, "h", false}, {E, nE * es, "E", false}, {targets, row, "targets", false}, {lse, row, "lse", false},
                          {dloss, row, "dloss", false}, {dlse, row, "dlse", false}, {dh, nh, "dh", true},
                          {dE, nE * des, "dE", true}, {ws, w.bytes, "the workspace", true}};
    if (const int rc = check_spans(who, spans)) return rc;
    if (const int rc = check_ws(who, w, dtype, ws, ws_bytes)) return rc;
    char* const base = (char*)ws;
    Call c{who, w, base, h, E, s, dtype};
    if (const int rc = c.start()) return rc;
    const int planes = !w.bf || !dE ? 1 : dE_dtype == GN_F32 ? w.planes : T <= Plan::kWholeBf16 ? 2 : 1;
    const bool stacked = planes > 1 && T <= Plan::kTwoPieces;  // pieces under each other beside h as often
    const size_t plane = (size_t)T * w.vc;
    RowScale* const rows = (RowScale*)(base + w.rows);
    float* const resid = (float*)(base + w.resid);
    char* const G = base + (w.bf ? w.G : w.logits);
    if (stacked) {  // one k-segment of planes T rows
        if (const int rc = c.copy(h, w.hs, T, T, planes)) return rc;
    }
    row_scales<<<(w.Tp + 255) / 256, 256, 0, s>>>(rows, resid, T, w.Tp, targets, lse, dloss, dlse, scale, V);
    GN_LAUNCH_CHECK(who);
    // dst (+)= G's columns c0 .. c0 + M, transposed, times h: fp32 or in dE's own type
    auto weight = [&](int c0, int M, void* dst, int c_dtype, bool add) {
        GemmDesc g = product(G + (size_t)c0 * w.es, w.vc, c.hp, w.dp, w.Tp, dst, w.dp, M, w.dp);
        if (stacked) {
            g.B[0] = (const bf16_t*)(base + w.hs);
            g.Ks[0] = planes * T;
        } else if (planes == 2) {
            g.nseg = 2;
            g.A[1] = (const bf16_t*)G + plane + c0;
            g.lda[1] = w.vc;
            g.B[1] = g.B[0];
            g.ldb[1] = w.dp;
            g.Ks[1] = T;
        }
        g.accumulate = add;
        if (c_dtype == GN_F32) c.scratch(g);
        return gemm_run(g, 1, 0, dtype, c_dtype, s);
    };
    // rows v .. v + R of dE from an fp32 [R x dp]
    auto rows_out = [&](size_t from, int v, int R) {
        const unsigned grid = grid_for((int64_t)R * d, 1024, 16384);
        char* dst = (char*)dE + (size_t)v * d * des;
        if (des == 2) take_rows<bf16_t><<<grid, 256, 0, s>>>((const float*)(base + from), (bf16_t*)dst, R, d, w.dp, 0);
        else take_rows<float><<<grid, 256, 0, s>>>((const float*)(base + from), (float*)dst, R, d, w.dp, acc);
        GN_LAUNCH_CHECK(who);
        return (int)GN_OK;
    };
    const bool few = w.bf && dh_few_takes(T, V, w.dp);  // dh takes every column as it is
    const int tail = few ? 0 : V % w.q;
    for (int v0 = 0; v0 < V; v0 += w.vc) {
        const int nv = std::min(w.vc, V - v0), nq = nv / w.q * w.q;
        const void* Ec;
        if (const int rc = c.piece(v0, nv, &Ec)) return rc;
        if (w.bf) {
            const GemmDesc g = product(c.hp, w.dp, Ec, w.dp, w.dp, nullptr, 0, T, nv);
            auto logits = [&](auto P_) {
                constexpr int P = decltype(P_)::value;
                bf16_t* const Gp = (bf16_t*)G;
                if (few_takes(g)) return launch_few(g, GradFew<P>{rows, Gp, plane, resid, w.vc, v0}, s);
                return launch_logits(g, GradTile<P>{rows, Gp, plane, resid, w.vc, v0}, s);
            };
            const int rc = planes == 3   ? logits(std::integral_constant<int, 3>{})
                           : planes == 2 ? logits(std::integral_constant<int, 2>{})
                                         : logits(std::integral_constant<int, 1>{});
            if (rc) return rc;
        } else {
            if (const int rc = c.logits32(Ec, nv)) return rc;
            piece_grad<<<blocks_of(w.Tp, std::min(16, (nv + 4095) / 4096)), 256, 0, s>>>((float*)G, w.vc, w.Tp, v0, nv, rows);
            GN_LAUNCH_CHECK(who);
        }
        if (dE && w.lay) {
            const int M = round_up(nv, w.q);
            if (const int rc = weight(0, M, base + w.de, GN_F32, false)) return rc;
            if (const int rc = rows_out(w.de, v0, nv)) return rc;
        } else if (dE) {
            if (nq) {
                if (const int rc = weight(0, nq, (char*)dE + (size_t)v0 * d * des, dE_dtype, acc)) return rc;
            }
            if (nv > nq) {
                if (const int rc = weight(nq, w.q, base + w.det, GN_F32, false)) return rc;
                if (const int rc = rows_out(w.det, v0 + nq, nv - nq)) return rc;
            }
        }
        if (dh && few) {
            GemmDesc g = product(G, w.vc, Ec, w.dp, nv, base + w.acc, w.dp, T, w.dp);
            g.accumulate = v0 > 0;
            g.ksplit = few_dh_ranges(nv, T, w.dp);
            c.scratch(g);
            if (const int rc = T <= 32 ? launch_dh_few<1>(g, s) : launch_dh_few<2>(g, s)) return rc;
        } else if (dh && nq) {
            GemmDesc g = product(G, w.vc, Ec, w.dp, nq, base + w.acc, w.dp, w.Tp, w.dp);
            g.accumulate = v0 > 0;
            c.scratch(g);
            if (const int rc = gemm_run(g, 0, 0, dtype, GN_F32, s)) return rc;
        }
    }
    if (planes == 2 && !stacked && T <= Plan::kTargets) {
        const auto rest = d % 8 == 0 && al16(h) && al16(dE) ? target_rest<true> : target_rest<false>;
        rest<<<T, 256, 0, s>>>(targets, resid, (const bf16_t*)h, (float*)dE, T, d, V);
        GN_LAUNCH_CHECK(who);
    }
    if (dh) {
        const float* sum = few || V >= w.q ? (const float*)(base + w.acc) : nullptr;
        const size_t col = (size_t)((V - 1) % w.vc + 1 - tail) * w.es;  // the tail's first column in the last piece
        const char* Et = (const char*)E + (size_t)(V - tail) * d * w.es;
        const bool vec = d % 8 == 0 && al16(dh) && al16(E);
        const unsigned grid = grid_for((int64_t)T * (vec ? d / 8 : d), 256, 16384);
        auto go = [&](auto VEC_) {
            constexpr bool VEC = decltype(VEC_)::value;
            if (w.bf)
                dh_finish<bf16_t, VEC><<<grid, 256, 0, s>>>(sum, w.dp, rows, resid, (const bf16_t*)E, (const bf16_t*)(G + col),
                                                            w.vc, (const bf16_t*)Et, tail, (bf16_t*)dh, T, d);
            else
                dh_finish<float, VEC><<<grid, 256, 0, s>>>(sum, w.dp, rows, resid, (const float*)E, (const float*)(G + col),
                                                           w.vc, (const float*)Et, tail, (float*)dh, T, d);
        };
        if (vec) go(std::true_type{});
        else go(std::false_type{});
        GN_LAUNCH_CHECK(who);
    }
    return GN_OK;
}
