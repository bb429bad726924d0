// gn_rng.h — the counter-based generator of the dropout masks (gn_residual.hip).
//
// Its output function is splitmix64's (Steele, Lea and Flood 2014), as in the surrogate loss's noise:
//   key = mix(mix(seed + phi (stream + 1)) + phi (step + 1)),   word w = mix(key + phi (w + 1))
// Element i of a call takes the low (i even) or high half of word i / 2 and is dropped where that is
// below t = round(p 2^32); a kept one is multiplied by 1 / (1 - t / 2^32), the factor of the probability
// that the mask has.  Two levels of key: seed and step mixed together in one would make (seed, step + 1)
// and another seed's (seed + phi, step) the same mask.
#pragma once

#include <cmath>

#include "gn_common.h"

namespace gn {

constexpr uint64_t kPhi = 0x9E3779B97F4A7C15ull;

__host__ __device__ __forceinline__ uint64_t mix64(uint64_t z) {
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}

// A call's mask as a kernel takes it.
struct Mask {
    uint64_t site;            // mix(seed + phi (stream + 1))
    uint64_t step;
    const int64_t* step_dev;  // added to step, nullptr: 0
    uint32_t t;               // 0: nothing is dropped
    float keep;               // the factor on what is kept

    __device__ __forceinline__ uint64_t key() const {
        const uint64_t at = step + (step_dev ? (uint64_t)*step_dev : 0ull);
        return mix64(site + kPhi * (at + 1));
    }
};

// Eight elements from i0 (a multiple of 8) on, or one: kept times the factor, or 0.  A dropped inf or NaN is 0.  f(e, kept) follows
// what becomes of element e.
struct NoMore {
    __device__ __forceinline__ void operator()(int, bool) const {}
};
template <typename F = NoMore>
__device__ __forceinline__ void drop8(float (&v)[8], uint64_t key, uint64_t i0, uint32_t t, float keep, F&& f = F{}) {
    uint64_t z = key + kPhi * ((i0 >> 1) + 1);
#pragma unroll
    for (int k = 0; k < 4; ++k, z += kPhi) {
        const uint64_t w = mix64(z);
        const bool k0 = (uint32_t)w >= t, k1 = (uint32_t)(w >> 32) >= t;
        v[2 * k] = k0 ? v[2 * k] * keep : 0.f;
        v[2 * k + 1] = k1 ? v[2 * k + 1] * keep : 0.f;
        f(2 * k, k0);
        f(2 * k + 1, k1);
    }
}
template <typename F = NoMore>
__device__ __forceinline__ float drop1(float v, uint64_t key, uint64_t i, uint32_t t, float keep, F&& f = F{}) {
    const uint64_t w = mix64(key + kPhi * ((i >> 1) + 1));
    const bool kept = ((i & 1) ? (uint32_t)(w >> 32) : (uint32_t)w) >= t;
    f(0, kept);
    return kept ? v * keep : 0.f;
}

// A probability below 1 as the mask takes it; false: not one.
inline bool make_mask(const gn_rng* r, double p, Mask* m) {
    if (!(p >= 0.0 && p < 1.0)) return false;
    const double t = std::nearbyint(p * 4294967296.0);
    if (t > 4294967295.0) return false;
    m->t = (uint32_t)t;
    m->keep = (float)(4294967296.0 / (4294967296.0 - t));
    m->site = r ? mix64(r->seed + kPhi * (r->stream + 1)) : 0;
    m->step = r ? r->step : 0;
    m->step_dev = r ? r->step_dev : nullptr;
    return true;
}

}  // namespace gn
