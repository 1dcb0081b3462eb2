// What the log probabilities of a row are joined from (logprobs.hip), for kernels that leave it themselves.
#pragma once

#include "common.h"

namespace aegist {

typedef unsigned long long u64;

// Order of the alternatives as one number: the larger value first (NaN before all, -0 as +0), then the lower
// token. Larger keys come first; 0 is below every element's.
__device__ __forceinline__ u64 lp_key(float v, uint32_t id) {
    const uint32_t b = v != v ? 0x7fc00000u : __float_as_uint(v + 0.f);
    return (u64)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (uint32_t)~id;
}
// What a split of a row leaves: maximum, sums relative to it, the token's logit if it lies in the split; NaN or
// +inf seen. Its alternatives follow apart.
struct Part {
    float m, z, s, tok;
    int bad, pad[3];
};

// Where a product's epilogue leaves the statistics of its rows: parts [M][splits], keys [M][splits] (NULL: none are
// asked for). Splits are halves of 256-column tiles.
struct RowStats {
    const int* tokens;
    Part* parts;
    u64* keys;
    int splits;
};
__host__ __device__ inline int row_stats_splits(int N) { return (N + 255) / 256 * 2; }

}  // namespace aegist
