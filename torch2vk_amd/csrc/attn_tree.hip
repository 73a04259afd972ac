// Attention of a tree of drafted tokens over a bf16 KV cache: q/k norm and RoPE of the nodes, their rows into the cache, and
// softmax(q . k / sqrt(d)) . v over the cached tokens, a node's ancestors and itself.
#include <math.h>

#include "kv_q8.h"
#include "tree.h"

namespace t2h {

constexpr int TA_D = 128;
constexpr int TA_MAX_GROUP = 16;

struct TreeAttnArgs {
    const float* q;
    const float* k_new;
    const float* v_new;
    size_t q_row, k_row, v_row;
    const float* q_norm_w;
    const float* k_norm_w;
    float eps, scale_log2;
    int rope;
    double log2_theta;
    const int32_t* lengths;
    const int32_t* parents;
    const int32_t* counts;
    uint16_t* k_cache;
    uint16_t* v_cache;
    size_t k_seq, v_seq;
    uint32_t s_cap, n, n_seq, nh, nk, group;
    uint16_t* out;
    float* qs;       // [n_seq][n][nh][128] rotated queries
    uint64_t* line;  // [n_seq][n] sets of seen nodes
};

constexpr int TP_HEADS = 4;  // heads a wave

// One wave: heads TP_HEADS * part .. of a node's row, q's, then k's, then v's.
__global__ __launch_bounds__(256) void tree_rows_kernel(const TreeAttnArgs a) {
    const int lane = threadIdx.x & 63;
    const uint32_t heads = a.nh + 2 * a.nk, parts = (heads + TP_HEADS - 1) / TP_HEADS;
    const uint64_t unit = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (unit >= (uint64_t)a.n_seq * a.n * parts) return;
    const uint32_t row = (uint32_t)(unit / parts), h0 = (uint32_t)(unit % parts) * TP_HEADS;
    const uint32_t seq = row / a.n, i = row % a.n;
    const int len = a.lengths[seq];
    const int count = tree_count_at(a.counts, seq, a.n, len, a.s_cap);
    const uint64_t lines = tree_lineage(a.parents, seq, a.n, count);
    const uint64_t line = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(lines >> 32), (int)i) << 32 |
                          (uint32_t)__builtin_amdgcn_readlane((int)lines, (int)i);
    if (h0 == 0 && lane == 0) a.line[row] = line;
    if (line == 0) return;
    float cs = 1.0f, sn = 0.0f;
    if (a.rope) rope_at(rope_turns(lane, a.log2_theta), len + __popcll(line) - 1, cs, sn);
    const bool has_w = a.q_norm_w != nullptr;
    for (uint32_t h = h0; h < h0 + TP_HEADS && h < heads; ++h) {
        const size_t slot = (size_t)len + i;
        if (h < a.nh) {
            const float* x = a.q + row * a.q_row + (size_t)h * TA_D;
            float r0, r1;
            q8_norm_rope(x[lane], x[lane + 64], has_w, has_w ? a.q_norm_w[lane] : 1.0f, has_w ? a.q_norm_w[lane + 64] : 1.0f,
                         a.eps, cs, sn, r0, r1);
            float* y = a.qs + ((size_t)row * a.nh + h) * TA_D;
            y[lane] = r0;
            y[lane + 64] = r1;
        } else if (h < a.nh + a.nk) {
            const uint32_t kh = h - a.nh;
            const float* x = a.k_new + row * a.k_row + (size_t)kh * TA_D;
            float r0, r1;
            q8_norm_rope(x[lane], x[lane + 64], has_w, has_w ? a.k_norm_w[lane] : 1.0f, has_w ? a.k_norm_w[lane + 64] : 1.0f,
                         a.eps, cs, sn, r0, r1);
            uint16_t* y = a.k_cache + seq * a.k_seq + (slot * a.nk + kh) * TA_D;
            y[lane] = (uint16_t)f32_to_bf16_bits(r0);
            y[lane + 64] = (uint16_t)f32_to_bf16_bits(r1);
        } else {
            const uint32_t vh = h - a.nh - a.nk;
            const float* x = a.v_new + row * a.v_row + (size_t)vh * TA_D;
            uint16_t* y = a.v_cache + seq * a.v_seq + (slot * a.nk + vh) * TA_D;
            y[lane] = (uint16_t)f32_to_bf16_bits(x[lane]);
            y[lane + 64] = (uint16_t)f32_to_bf16_bits(x[lane + 64]);
        }
    }
}

// One wave a (node, head): 64 keys at a time, a lane a key for the scores and two dims for the sum.
__global__ __launch_bounds__(64) void tree_attn_kernel(const TreeAttnArgs a) {
    __shared__ float qs[TA_D];
    const int lane = threadIdx.x;
    const uint32_t h = blockIdx.x % a.nh, row = blockIdx.x / a.nh, seq = row / a.n;
    uint32_t* const out = reinterpret_cast<uint32_t*>(a.out + ((size_t)row * a.nh + h) * TA_D);
    const uint64_t line = a.line[row];
    if (line == 0) {
        out[lane] = 0u;
        return;
    }
    const float* q = a.qs + ((size_t)row * a.nh + h) * TA_D;
    qs[lane] = q[lane];
    qs[lane + 64] = q[lane + 64];
    __syncthreads();
    const int len = a.lengths[seq], end = len + 64 - __builtin_clzll(line);
    const uint16_t* const kb = a.k_cache + seq * a.k_seq + (size_t)(h / a.group) * TA_D;
    const uint16_t* const vb = a.v_cache + seq * a.v_seq + (size_t)(h / a.group) * TA_D;
    float m = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int t0 = 0; t0 < end; t0 += 64) {
        const int t = t0 + lane;
        const bool seen = t < len || (t < end && (line >> (t - len) & 1));
        float s = -INFINITY;
        if (seen) {
            const uint4* k = reinterpret_cast<const uint4*>(kb + (size_t)t * a.nk * TA_D);
            s = 0.0f;
            for (int c = 0; c < TA_D / 8; ++c) {
                const uint4 w = k[c];
                const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s = fmaf(qs[8 * c + 2 * j], __uint_as_float(x[j] << 16), s);
                    s = fmaf(qs[8 * c + 2 * j + 1], __uint_as_float(x[j] & 0xffff0000u), s);
                }
            }
            s *= a.scale_log2;
        }
        const float now = fmaxf(m, wave_max(s)), base = now == -INFINITY ? 0.0f : now;
        const float keep = __builtin_amdgcn_exp2f(m - base);
        const float p = seen ? __builtin_amdgcn_exp2f(s - base) : 0.0f;
        m = now;
        l = fmaf(l, keep, wave_sum(p));
        o0 *= keep;
        o1 *= keep;
        uint64_t todo = __ballot(seen);
        while (todo) {
            const int j = __builtin_ctzll(todo);
            todo &= todo - 1;
            const float pj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(p), j));
            const uint32_t v = reinterpret_cast<const uint32_t*>(vb + (size_t)(t0 + j) * a.nk * TA_D)[lane];
            o0 = fmaf(pj, __uint_as_float(v << 16), o0);
            o1 = fmaf(pj, __uint_as_float(v & 0xffff0000u), o1);
        }
    }
    out[lane] = pack_bf16x2(o0 / l, o1 / l);
}

}  // namespace t2h

using namespace t2h;

static bool ta_shape(uint32_t n_seq, uint32_t n, uint32_t nh, uint32_t nk, uint32_t s_cap) {
    return n_seq != 0 && n <= (uint32_t)TREE_MAX && nk != 0 && nh != 0 && nh % nk == 0 && s_cap != 0 && s_cap <= 0x7fffff00u;
}

extern "C" size_t t2h_attn_tree_workspace_bytes(uint32_t n_seq, uint32_t n, uint32_t nh, uint32_t nk, uint32_t d,
                                                uint32_t s_cap) {
    if (!ta_shape(n_seq, n, nh, nk, s_cap) || n == 0 || nh / nk > TA_MAX_GROUP || d != TA_D) return 0;
    return (size_t)n_seq * n * (8 + (size_t)nh * TA_D * 4);
}

extern "C" int t2h_attn_tree(const float* q, uint64_t q_row, const float* k_new, uint64_t k_row, const float* v_new,
                             uint64_t v_row, const float* q_norm_w, const float* k_norm_w, float eps, float theta,
                             const int32_t* lengths, const int32_t* parents, const int32_t* counts, void* k_cache,
                             uint64_t k_seq, void* v_cache, uint64_t v_seq, uint32_t s_cap, void* out, uint32_t n,
                             uint32_t n_seq, uint32_t nh, uint32_t nk, uint32_t d, void* workspace, size_t workspace_bytes,
                             void* stream) {
    if (!q || !k_new || !v_new || !lengths || !k_cache || !v_cache || !out || !workspace) return T2H_ERR_NULL;
    if ((q_norm_w == nullptr) != (k_norm_w == nullptr)) return T2H_ERR_NULL;
    if (d != TA_D) return T2H_ERR_UNSUPPORTED;
    if (!ta_shape(n_seq, n, nh, nk, s_cap)) return T2H_ERR_SHAPE;
    if (nh / nk > TA_MAX_GROUP) return T2H_ERR_UNSUPPORTED;
    if (q_row < (uint64_t)nh * d || k_row < (uint64_t)nk * d || v_row < (uint64_t)nk * d) return T2H_ERR_SHAPE;
    const uint64_t seq = (uint64_t)s_cap * nk * d;
    if (n_seq > 1 && (k_seq < seq || v_seq < seq)) return T2H_ERR_SHAPE;
    if ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) | reinterpret_cast<uintptr_t>(out) |
         reinterpret_cast<uintptr_t>(workspace) | (n_seq > 1 ? (k_seq | v_seq) * 2 : 0)) & 15)
        return T2H_ERR_ALIGN;
    if (n == 0) return T2H_OK;
    if (workspace_bytes < t2h_attn_tree_workspace_bytes(n_seq, n, nh, nk, d, s_cap)) return T2H_ERR_WORKSPACE;
    TreeAttnArgs a;
    a.q = q;
    a.k_new = k_new;
    a.v_new = v_new;
    a.q_row = (size_t)q_row;
    a.k_row = (size_t)k_row;
    a.v_row = (size_t)v_row;
    a.q_norm_w = q_norm_w;
    a.k_norm_w = k_norm_w;
    a.eps = eps;
    a.scale_log2 = 1.4426950408889634f / sqrtf((float)TA_D);
    a.rope = theta > 0.0f;
    a.log2_theta = a.rope ? log2((double)theta) : 0.0;
    a.lengths = lengths;
    a.parents = parents;
    a.counts = counts;
    a.k_cache = reinterpret_cast<uint16_t*>(k_cache);
    a.v_cache = reinterpret_cast<uint16_t*>(v_cache);
    a.k_seq = (size_t)k_seq;
    a.v_seq = (size_t)v_seq;
    a.s_cap = s_cap;
    a.n = n;
    a.n_seq = n_seq;
    a.nh = nh;
    a.nk = nk;
    a.group = nh / nk;
    a.out = reinterpret_cast<uint16_t*>(out);
    const uint64_t rows = (uint64_t)n_seq * n;
    a.qs = reinterpret_cast<float*>(workspace);
    a.line = reinterpret_cast<uint64_t*>(a.qs + rows * nh * TA_D);
    const uint64_t waves = rows * ((nh + 2 * nk + TP_HEADS - 1) / TP_HEADS);
    if (waves > 0x7fffffffu || rows * nh > 0x7fffffffu) return T2H_ERR_SHAPE;
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(tree_rows_kernel, dim3((uint32_t)((waves + 3) / 4)), dim3(256), 0, st, a);
    T2H_LAUNCH_CHECK();
    hipLaunchKernelGGL(tree_attn_kernel, dim3((uint32_t)(rows * nh)), dim3(64), 0, st, a);
    T2H_LAUNCH_CHECK();
    return T2H_OK;
}
