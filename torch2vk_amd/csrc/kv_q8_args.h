// Host side of the 8-bit KV cache's entry points: the cache's pointers, checked.
#pragma once

#include "kv_q8.h"

namespace t2h {

constexpr uint32_t Q8_MAX_GROUP = 16;  // q heads of a KV head

// cache: k, v, k_scale, v_scale, k_tail, v_tail
static inline int q8_cache(void* const* cache, uint32_t s_cap, uint32_t n_seq, uint32_t nh, uint32_t nk, uint32_t d, KvQ8& c) {
    if (!cache) return T2H_ERR_NULL;
    for (int i = 0; i < 6; ++i)
        if (!cache[i]) return T2H_ERR_NULL;
    if (d != (uint32_t)Q8_D) return T2H_ERR_UNSUPPORTED;
    if (n_seq == 0 || nk == 0 || nh == 0 || nh % nk != 0) return T2H_ERR_SHAPE;
    if (nh / nk > Q8_MAX_GROUP) return T2H_ERR_UNSUPPORTED;
    if (s_cap == 0 || s_cap % Q8_BLOCK != 0 || s_cap > 0x40000000u) return T2H_ERR_SHAPE;
    if ((uint64_t)n_seq * nk > 0x7fffffu) return T2H_ERR_SHAPE;
    for (int i = 0; i < 6; ++i)
        if (reinterpret_cast<uintptr_t>(cache[i]) & (i == 2 || i == 3 ? 3 : 15)) return T2H_ERR_ALIGN;
    c.k = reinterpret_cast<int8_t*>(cache[0]);
    c.v = reinterpret_cast<int8_t*>(cache[1]);
    c.ks = reinterpret_cast<float*>(cache[2]);
    c.vs = reinterpret_cast<float*>(cache[3]);
    c.kt = reinterpret_cast<uint16_t*>(cache[4]);
    c.vt = reinterpret_cast<uint16_t*>(cache[5]);
    c.nb = s_cap / Q8_BLOCK;
    c.nk = nk;
    return T2H_OK;
}

}  // namespace t2h
