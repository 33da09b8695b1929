// k1_sample_math.cuh -- arithmetic of the sampling kernel that also runs on the host, where the
// tests reach it with any values.
#pragma once

#include <cmath>
#include <cstdint>
#include <cstring>

#define K1_HD __host__ __device__ __forceinline__

namespace k1 {
namespace sample {

// A list's weights as whole numbers, so that their sums do not depend on their order: the weight
// in units of the list's own above 12 bits of count, in one word.
//
// The unit is a power of two that puts the list's mass between 2^50 and 2^51 units.  Sums over a
// list (2048 entries at most, each rounded by half a unit) then fit 52 bits, are within 2^-40 of
// the mass, and the heaviest entry has 2^39 units or more however small the weights are.  (A unit
// of the row's heaviest weight, 2^-40 of it, would leave nothing of a list that lies e^-28 below.)
constexpr int kCountBits = 12;
constexpr int kMassBits = 51;

// Units per weight of 1; `mass` is finite and >= 0, and a list without mass gets any unit.
K1_HD double list_unit(double mass) {
    uint64_t bits;
    memcpy(&bits, &mass, sizeof bits);
    int e = (int)(bits >> 52) - 1022;  // mass < 2^e
    e = e < -900 ? -900 : e;
    bits = (uint64_t)(kMassBits - e + 1023) << 52;
    double unit;
    memcpy(&unit, &bits, sizeof unit);
    return unit;
}
K1_HD uint64_t weight_word(float w, double unit) {
    return ((uint64_t)((double)w * unit + 0.5) << kCountBits) | 1u;
}
K1_HD uint64_t count_word() { return ((uint64_t)1 << kCountBits) | 1u; }
K1_HD uint64_t word_weight(uint64_t v) { return v >> kCountBits; }

// `mass` units, rounded up, as a target that a list of `all` units reaches: 1 to `all` (0 where the
// list has no mass).
K1_HD uint64_t list_target(double mass, uint64_t all) {
    const double t = ceil(mass);
    if (!(t > 1.0)) return all < 1 ? all : 1;
    return t < (double)all ? (uint64_t)t : all;
}

// The element of a lane's vector at which the mass, `cum` in front of the vector, first exceeds
// `target`, or the last one with a weight; -1 if none has any.  The first one with a weight is taken
// even where `cum` is above the target already: `cum` is the lane's prefix sum less its own mass,
// which in floating point may come out above the prefix of the lane before, the one that was compared.
template <int E>
K1_HD int pick_element(const float (&w)[E], double cum, double target) {
    int at = -1;
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (w[e] > 0.f && (at < 0 || !(cum > target))) {
            cum += (double)w[e];
            at = e;
        }
    return at;
}

}  // namespace sample
}  // namespace k1
