// Buckets of the learned relative position bias.
#pragma once

#include "common.cuh"

namespace rgd {
namespace relbias {

constexpr int MAX_SIDE = RGD_RELBIAS_MAX_SIDE;

// Buckets of one direction: borders[k] is the least distance of bucket k + 1.  Travels with the kernel's
// parameters, so a call keeps nothing on the device.
struct Borders {
    int side, both;
    int32_t at[MAX_SIDE - 1];
};

// Number of borders at or below n, by bisection.
__device__ __forceinline__ int bucket_of_distance(const int32_t *at, int side, int n) {
    int lo = 0, hi = side - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (at[mid] <= n) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}
// difference: key position - query position
__device__ __forceinline__ int bucket_of(const int32_t *at, int side, int both, int difference) {
    const int n = difference > 0 ? (both ? difference : 0) : -difference;
    return bucket_of_distance(at, side, n) + (both && difference > 0 ? side : 0);
}

inline int check(const rgd_relbias *b) {
    if (!b) return RGD_E_NULL;
    if (!dtype_ok(b->dtype)) return RGD_E_DTYPE;
    const int side = b->bidirectional ? b->num_buckets / 2 : b->num_buckets;
    if (b->num_buckets < 1 || (b->bidirectional && b->num_buckets % 2 != 0)) return RGD_E_INVALID;
    if (side > MAX_SIDE) return RGD_E_SIZE;
    if (side > 1 && !b->borders) return RGD_E_NULL;
    for (int k = 0; k + 1 < side; ++k)
        if (b->borders[k] < 1 || (k > 0 && b->borders[k] < b->borders[k - 1])) return RGD_E_INVALID;
    return RGD_OK;
}
inline Borders make_borders(const rgd_relbias &b) {
    Borders o{};
    o.both = b.bidirectional ? 1 : 0;
    o.side = o.both ? b.num_buckets / 2 : b.num_buckets;
    for (int k = 0; k + 1 < o.side; ++k) o.at[k] = b.borders[k];
    return o;
}

}  // namespace relbias
}  // namespace rgd
