// The 8-bit KV cache: layout, rounding and positions, shared by the kernels that write, read and evict it.
//
// A sequence's tokens are held in blocks of 64 per KV head.  A whole block is 8-bit codes under one fp32 scale for its
// keys and one for its values: x ~ code * s with s = max|x| / 127, code = round(x / s), ties to even.  The tokens of the
// last, unfinished block are bf16 rows (the tail); a block is rounded once, from its bf16 values, when its last token
// arrives, so what the cache holds depends on the tokens and not on the chunks that they came in.
//   k  int8 [n_seq][n_blocks][nk][64][128]    k_tail bf16 [n_seq][nk][64][128]     k_scale fp32 [n_seq][n_blocks][nk]
//   v  int8 [n_seq][n_blocks][nk][128][64]    v_tail bf16 [n_seq][nk][128][64]     v_scale fp32 [n_seq][n_blocks][nk]
// Values are transposed within a block: P.V contracts over tokens, so a matrix-core operand is 16 consecutive tokens of
// one dimension, one 16-byte load; that costs nothing here because a block is only ever written whole.
#pragma once

#include "common.h"

namespace t2h {

constexpr int Q8_BLOCK = T2H_KV_Q8_BLOCK;  // tokens a block
constexpr int Q8_D = 128;                  // head dimension
constexpr int Q8_BYTES = Q8_BLOCK * Q8_D;  // bytes of a block's keys, and of its values

struct KvQ8 {
    int8_t* k;
    int8_t* v;
    float* ks;
    float* vs;
    uint16_t* kt;
    uint16_t* vt;
    uint32_t nb;  // blocks of a sequence
    uint32_t nk;  // KV heads

    __device__ __forceinline__ size_t scale_at(uint32_t seq, uint32_t b, uint32_t h) const {
        return ((size_t)seq * nb + b) * nk + h;
    }
    __device__ __forceinline__ size_t block_at(uint32_t seq, uint32_t b, uint32_t h) const {
        return scale_at(seq, b, h) * Q8_BYTES;
    }
    __device__ __forceinline__ size_t tail_at(uint32_t seq, uint32_t h) const {
        return ((size_t)seq * nk + h) * Q8_BYTES;
    }
};

// One sequence's tokens in a call that brings up to n new ones: rows [0, len) are cached, [len, end) are new.
// A negative length is a sequence that takes no part (end 0); rows past the capacity are dropped.
struct Q8Span {
    int len, end;
};

__device__ __forceinline__ Q8Span q8_span(const int32_t* lengths, const int32_t* counts, uint32_t seq, uint32_t n,
                                          uint32_t nb) {
    const int cap = (int)(nb * Q8_BLOCK);
    const int len = lengths[seq];
    if (len < 0) return {0, 0};
    int c = (int)n;
    if (counts) {
        const int given = counts[seq];
        c = given < 0 ? 0 : (given < c ? given : c);
    }
    if (len >= cap) return {cap, cap};
    return {len, c < cap - len ? len + c : cap};
}

// Bits of |x|, which order as the values do and put infinities and NaN on top.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The larger |x| of two bf16 values, as fp32 bits.
__device__ __forceinline__ uint32_t bf16_abs_max(uint32_t w) { return max(w << 16 & 0x7fffffffu, w & 0x7fff0000u); }

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)v, off, T2H_WAVE);
        v = v > o ? v : o;
    }
    return v;
}

// Sums over the lanes up to each: within rows of 16, then over the rows.
__device__ __forceinline__ uint32_t wave_scan_u32(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false);  // 1 lane up
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);  // a row's last lane to the odd rows
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);  // lane 31 to the upper half
    return v;
}

// A block's scale and the factor that its values are multiplied by before rounding, from the bits of its max|x|.
// Values under 1.3e-28 are held as zeros; a block with a NaN or an infinity has a NaN scale, so that whoever reads it
// sees NaN and not numbers.
__device__ __forceinline__ void q8_scale(uint32_t amax_bits, float& s, float& inv) {
    s = __uint_as_float(amax_bits) * (1.0f / 127.0f);
    inv = 0.0f;
    if (amax_bits >= 0x7f800000u)
        s = __uint_as_float(0x7fc00000u);
    else if (s < 1e-30f)
        s = 0.0f;
    else
        inv = 1.0f / s;
}

// code of x; 0 where inv is 0 (x may be NaN or infinite there)
__device__ __forceinline__ int q8_code(float x, float inv) { return inv == 0.0f ? 0 : (int)rintf(x * inv); }

__device__ __forceinline__ uint32_t q8_pack4(float a, float b, float c, float d, float inv) {
    return (uint32_t)(q8_code(a, inv) & 255) | (uint32_t)(q8_code(b, inv) & 255) << 8 |
           (uint32_t)(q8_code(c, inv) & 255) << 16 | (uint32_t)q8_code(d, inv) << 24;
}

__device__ __forceinline__ float q8_value(uint32_t word, int byte) { return (float)(int8_t)(word >> (8 * byte)); }

// Rotations a token of frequency theta^(-lane / 64) in 64 bits: at position 10^5 a 32-bit product has lost the angle's
// third decimal.  The fraction of a turn then needs 32 bits only.  log2_theta comes from the host.
__device__ __forceinline__ double rope_turns(int lane, double log2_theta) {
    return exp2(-(double)lane * log2_theta * (1.0 / 64.0)) * 0.15915494309189535;
}

// One wave's head: RMSNorm (with has_w) of lane's dims lane and lane + 64, then the rotation by (cs, sn), (1, 0) for none.
__device__ __forceinline__ void q8_norm_rope(float x0, float x1, bool has_w, float w0, float w1, float eps, float cs, float sn,
                                             float& r0, float& r1) {
    if (has_w) {
        const float inv = __builtin_amdgcn_rsqf(wave_sum(x0 * x0 + x1 * x1) * (1.0f / Q8_D) + eps);
        x0 *= inv * w0;
        x1 *= inv * w1;
    }
    r0 = x0 * cs - x1 * sn;
    r1 = x1 * cs + x0 * sn;
}

__device__ __forceinline__ void rope_at(double turns, int pos, float& cs, float& sn) {
    const double t = (double)pos * turns;
    sincospif(2.0f * (float)(t - floor(t)), &sn, &cs);
}

}  // namespace t2h
