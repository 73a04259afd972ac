// Attention over the 8-bit KV cache (layout: kv_q8.h): out = softmax(q . k / sqrt(d)) . v for one token of each sequence
// or a chunk of tokens, and the attention weight that each cached token got.
//
// One wave a query row: a lane is a token of the block for the scores and two dimensions for the output; one pass over
// the keys with the running maximum and sum of the softmax, in fp32.
#include <math.h>

#include "kv_q8.h"
#include "kv_q8_args.h"
#include "rope.h"

namespace t2h {

struct AttnQ8Args {
    KvQ8 c;
    const void* q;  // bf16 or fp32 [n_seq][n][nh][128]
    uint16_t* out;
    float* lse;  // [n_seq][n][nh] natural log of the softmax's denominator, or null
    const int32_t* lengths;
    const int32_t* counts;
    const float* w_in;
    float* w_out;
    uint32_t n, n_seq, nh;
    float scale;
};

// token p's key . q, and its value's dimension
__device__ __forceinline__ float q8_key_dot(const AttnQ8Args& a, uint32_t seq, uint32_t h, int p, bool in_tail, const float* q) {
    float s = 0.0f;
    if (in_tail) {
        const uint16_t* k = a.c.kt + a.c.tail_at(seq, h) + (p % Q8_BLOCK) * Q8_D;
        for (int i = 0; i < Q8_D; ++i) s = fmaf(bf16_bits_to_f32(k[i]), q[i], s);
        return s;
    }
    const uint32_t* k = reinterpret_cast<const uint32_t*>(a.c.k + a.c.block_at(seq, p / Q8_BLOCK, h) + (p % Q8_BLOCK) * Q8_D);
    for (int i = 0; i < Q8_D; ++i) s = fmaf(q8_value(k[i / 4], i % 4), q[i], s);
    return s * a.c.ks[a.c.scale_at(seq, p / Q8_BLOCK, h)];
}

__device__ __forceinline__ float q8_v(const AttnQ8Args& a, uint32_t seq, uint32_t h, int p, bool in_tail, int d) {
    if (in_tail) return bf16_bits_to_f32(a.c.vt[a.c.tail_at(seq, h) + d * Q8_BLOCK + p % Q8_BLOCK]);
    return (float)a.c.v[a.c.block_at(seq, p / Q8_BLOCK, h) + d * Q8_BLOCK + p % Q8_BLOCK] * a.c.vs[a.c.scale_at(seq, p / Q8_BLOCK, h)];
}

__device__ __forceinline__ float q8_q(const AttnQ8Args& a, size_t i, bool f32) {
    return f32 ? reinterpret_cast<const float*>(a.q)[i] : bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(a.q)[i]);
}

template <bool F32>
__global__ __launch_bounds__(64) void attn_q8_kernel(const AttnQ8Args a) {
    __shared__ float qs[Q8_D];
    const int lane = threadIdx.x;
    const uint32_t h = blockIdx.x % a.nh, row = blockIdx.x / a.nh;
    const uint32_t seq = row / a.n, t = row % a.n;
    const uint32_t kvh = h / (a.nh / a.c.nk);
    const Q8Span s = q8_span(a.lengths, a.counts, seq, a.n, a.c.nb);
    const size_t at = (size_t)blockIdx.x * Q8_D;
    const int count = a.counts ? a.counts[seq] : (int)a.n;
    const int len = a.lengths[seq];
    int last = len < 0 || (int)t >= count ? 0 : len + (int)t + 1;
    last = last < 0 || last > s.end ? s.end : last;
    qs[lane] = q8_q(a, at + lane, F32);
    qs[lane + 64] = q8_q(a, at + lane + 64, F32);
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int p0 = 0; p0 < last; p0 += Q8_BLOCK) {
        const bool in_tail = p0 == s.end / Q8_BLOCK * Q8_BLOCK;
        const int p = p0 + lane;
        const float x = p < last ? q8_key_dot(a, seq, kvh, p, in_tail, qs) * a.scale : -INFINITY;
        const float top = fmaxf(m, wave_max(x));
        const float base = top == -INFINITY ? 0.0f : top;
        const float e = p < last ? expf(x - base) : 0.0f;
        const float f = expf(m - base);
        l = l * f + wave_sum(e);
        o0 *= f;
        o1 *= f;
        m = top;
        for (int i = 0; i < Q8_BLOCK && p0 + i < last; ++i) {
            const float w = __shfl(e, i, T2H_WAVE);
            o0 = fmaf(w, q8_v(a, seq, kvh, p0 + i, in_tail, 2 * lane), o0);
            o1 = fmaf(w, q8_v(a, seq, kvh, p0 + i, in_tail, 2 * lane + 1), o1);
        }
    }
    const float inv = last > 0 ? 1.0f / l : 0.0f;
    reinterpret_cast<uint32_t*>(a.out + at)[lane] = pack_bf16x2(o0 * inv, o1 * inv);
    if (a.lse && lane == 0) a.lse[blockIdx.x] = m + logf(l);
}

// weights_out[token] = weights_in (0 for a new token) + sum of p over the queries and the heads of the KV head
template <bool F32>
__global__ __launch_bounds__(64) void attn_q8_weights_kernel(const AttnQ8Args a) {
    __shared__ float qs[Q8_D];
    const int lane = threadIdx.x;
    const uint32_t kvh = blockIdx.x % a.c.nk;
    const uint32_t rest = blockIdx.x / a.c.nk;
    const uint32_t b = rest % a.c.nb, seq = rest / a.c.nb;
    const Q8Span s = q8_span(a.lengths, a.counts, seq, a.n, a.c.nb);
    const int p0 = (int)b * Q8_BLOCK, p = p0 + lane;
    if (p0 >= s.end) return;
    const bool in_tail = p0 == s.end / Q8_BLOCK * Q8_BLOCK;
    const int group = a.nh / a.c.nk;
    const int count = a.counts ? min(a.counts[seq], (int)a.n) : (int)a.n;
    const size_t wi = ((size_t)seq * a.c.nk + kvh) * a.c.nb * Q8_BLOCK + p;
    float sum = 0.0f;
    for (int t = 0; t < count; ++t) {
        for (int g = 0; g < group; ++g) {
            const size_t row = ((size_t)seq * a.n + t) * a.nh + kvh * group + g;
            __syncthreads();
            qs[lane] = q8_q(a, row * Q8_D + lane, F32);
            qs[lane + 64] = q8_q(a, row * Q8_D + lane + 64, F32);
            __syncthreads();
            if (p < s.end && p <= a.lengths[seq] + t) sum += expf(q8_key_dot(a, seq, kvh, p, in_tail, qs) * a.scale - a.lse[row]);
        }
    }
    if (p < s.end) a.w_out[wi] = (p < s.len ? a.w_in[wi] : 0.0f) + sum;
}

template <bool F32>
static int attn_q8_launch(const AttnQ8Args& a, void* stream) {
    const uint64_t rows = (uint64_t)a.n_seq * a.n * a.nh, blocks = (uint64_t)a.n_seq * a.c.nb * a.c.nk;
    if (rows > 0x7fffffffu || blocks > 0x7fffffffu) return T2H_ERR_SHAPE;
    hipLaunchKernelGGL(attn_q8_kernel<F32>, dim3((uint32_t)rows), dim3(64), 0, reinterpret_cast<hipStream_t>(stream), a);
    T2H_LAUNCH_CHECK();
    if (a.w_out) {
        hipLaunchKernelGGL(attn_q8_weights_kernel<F32>, dim3((uint32_t)blocks), dim3(64), 0, reinterpret_cast<hipStream_t>(stream), a);
        T2H_LAUNCH_CHECK();
    }
    return T2H_OK;
}

}  // namespace t2h

using namespace t2h;

extern "C" size_t t2h_attn_decode_q8_workspace_bytes(uint32_t n_seq, uint32_t nh, uint32_t nk, uint32_t d, uint32_t s_cap,
                                                     int weights) {
    if (n_seq == 0 || nk == 0 || nh == 0 || nh % nk != 0 || nh / nk > Q8_MAX_GROUP || d != (uint32_t)Q8_D || s_cap == 0 ||
        s_cap % Q8_BLOCK != 0)
        return 0;
    return (size_t)n_seq * nh * (4 * Q8_D + 4) + 256;
}

extern "C" int t2h_attn_decode_q8(const float* q, uint64_t q_row, const float* k_new, uint64_t k_row, const float* v_new,
                                  uint64_t v_row, const float* q_norm_w, const float* k_norm_w, float eps, float theta,
                                  const int32_t* lengths, const int32_t* rope_offsets, void* const* cache, uint32_t s_cap,
                                  const float* weights, float* weights_out, void* out, uint32_t n_seq, uint32_t nh,
                                  uint32_t nk, uint32_t d, void* workspace, size_t workspace_bytes, void* stream) {
    AttnQ8Args a;
    if (!lengths || !out || !workspace) return T2H_ERR_NULL;
    if ((weights == nullptr) != (weights_out == nullptr)) return T2H_ERR_NULL;
    if (const int e = q8_cache(cache, s_cap, n_seq, nh, nk, d, a.c)) return e;
    if (reinterpret_cast<uintptr_t>(out) & 3) return T2H_ERR_ALIGN;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return T2H_ERR_ALIGN;
    if (workspace_bytes < t2h_attn_decode_q8_workspace_bytes(n_seq, nh, nk, d, s_cap, weights != nullptr)) return T2H_ERR_WORKSPACE;
    if (!q || !k_new || !v_new) return T2H_ERR_NULL;
    const int e = q8_write_launch(q, q_row, k_new, k_row, v_new, v_row, q_norm_w, k_norm_w, eps, theta, lengths, nullptr,
                                            rope_offsets, 1, n_seq, nh, nk, d, workspace, true, cache, s_cap, stream);
    if (e) return e;
    a.q = workspace;
    a.out = reinterpret_cast<uint16_t*>(out);
    a.lse = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(workspace) + (size_t)n_seq * nh * 4 * Q8_D);
    a.lengths = lengths;
    a.counts = nullptr;
    a.w_in = weights;
    a.w_out = weights_out;
    a.n = 1;
    a.n_seq = n_seq;
    a.nh = nh;
    a.scale = 1.0f / sqrtf((float)Q8_D);
    return attn_q8_launch<true>(a, stream);
}

extern "C" size_t t2h_flash_attn_prefill_q8_workspace_bytes(uint32_t n, uint32_t n_seq, uint32_t nh, uint32_t nk,
                                                            uint32_t s_cap, int weights) {
    return (size_t)n_seq * n * nh * 4 + 256;
}

extern "C" int t2h_flash_attn_prefill_q8(const void* q, void* const* cache, uint32_t s_cap, const int32_t* lengths,
                                         const int32_t* counts, const float* weights, float* weights_out, void* out,
                                         uint32_t n, uint32_t n_seq, uint32_t nh, uint32_t nk, uint32_t d, float scale,
                                         void* workspace, size_t workspace_bytes, void* stream) {
    AttnQ8Args a;
    if (!q || !lengths || !out || !workspace) return T2H_ERR_NULL;
    if ((weights == nullptr) != (weights_out == nullptr)) return T2H_ERR_NULL;
    if (const int e = q8_cache(cache, s_cap, n_seq, nh, nk, d, a.c)) return e;
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15)
        return T2H_ERR_ALIGN;
    if (workspace_bytes < t2h_flash_attn_prefill_q8_workspace_bytes(n, n_seq, nh, nk, s_cap, weights != nullptr))
        return T2H_ERR_WORKSPACE;
    if (n == 0) return T2H_OK;
    a.q = q;
    a.out = reinterpret_cast<uint16_t*>(out);
    a.lse = reinterpret_cast<float*>(workspace);
    a.lengths = lengths;
    a.counts = counts;
    a.w_in = weights;
    a.w_out = weights_out;
    a.n = n;
    a.n_seq = n_seq;
    a.nh = nh;
    a.scale = scale > 0.0f ? scale : 1.0f / sqrtf((float)Q8_D);
    return attn_q8_launch<false>(a, stream);
}
