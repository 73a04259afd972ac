// Trees of drafted tokens: a sequence's up to 64 nodes, node i hanging on the earlier node parents[i], or on the cached tokens
// (-1).  Shared by the kernels that attend over such a tree, check it and keep a path of it.
#pragma once

#include "common.h"

namespace t2h {

constexpr int TREE_MAX = T2H_TREE_MAX_NODES;
static_assert(TREE_MAX == T2H_WAVE, "a node a lane, and a bit of a 64-bit set");

// How many of a sequence's n rows are nodes.
__device__ __forceinline__ int tree_count(const int32_t* counts, uint32_t seq, uint32_t n) {
    if (!counts) return (int)n;
    const int c = counts[seq];
    return c < 0 ? 0 : (c < (int)n ? c : (int)n);
}

// The same, with the nodes that have no slot behind a sequence's `len` cached tokens dropped.  A length outside the cache
// drops all of them.
__device__ __forceinline__ int tree_count_at(const int32_t* counts, uint32_t seq, uint32_t n, int len, uint32_t s_cap) {
    if (len < 0 || (uint32_t)len > s_cap) return 0;
    const int c = tree_count(counts, seq, n), room = (int)(s_cap - (uint32_t)len);
    return c < room ? c : room;
}

// Lane i's set of nodes: node i and its ancestors, or none where that is no node (i past the count, or a parent on the way up
// that is not an earlier node).  Each of the six steps doubles how far up a lane has looked; -1 and -2 end the way.
__device__ __forceinline__ uint64_t tree_lineage(const int32_t* parents, uint32_t seq, uint32_t n, int count) {
    const int lane = threadIdx.x & 63;
    int up = lane - 1;
    if (parents && lane < (int)n) up = parents[(size_t)seq * n + lane];
    if (lane >= count || up < -1 || up >= lane) up = -2;
    uint32_t lo = lane < 32 ? 1u << lane : 0u, hi = lane < 32 ? 0u : 1u << (lane - 32);
#pragma unroll
    for (int i = 0; i < 6; ++i) {
        const int from = up < 0 ? lane : up;
        const uint32_t olo = (uint32_t)__shfl((int)lo, from), ohi = (uint32_t)__shfl((int)hi, from);
        const int oup = __shfl(up, from);
        lo |= olo;
        hi |= ohi;
        up = oup;  // a lane whose way has ended asked itself
    }
    return up == -2 ? 0u : (uint64_t)hi << 32 | lo;
}

}  // namespace t2h
