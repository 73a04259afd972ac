// Attention over the 8-bit KV cache (layout: kv_q8.h): out = softmax(q . k / sqrt(d)) . v for one token of each sequence
// or a chunk of tokens, and the attention weight that each cached token got.  One pass over the keys with the running
// maximum and sum of the softmax, both in fp32, scores in log2 units.
#include <math.h>
#include <type_traits>

#include "kv_q8.h"
#include "kv_q8_args.h"

namespace t2h {

// ------------------------------------------------------------------------------------------- one token a sequence --
//
// Bound by memory: every cached byte is read once, for all q heads of its KV head.  The work is cut into units of up to
// `chunk` consecutive cache blocks of one (sequence, KV head), equal for all sequences of a ragged batch and worked out
// from the lengths on the device, so that a captured launch follows them; thread block (unit, head) walks one.  A wave
// takes whole blocks of 64 tokens (its thread block's b0 + wave, + 4, ...) with no barrier in its loop:
//   * scores S^T = K . Q^T and output O^T = V^T . P^T on the matrix cores (16 x 16 x 32, fp16 in, fp32 out), the q heads
//     of the KV head as columns.  A lane's 16-byte loads are the operands: 16 dims of a key row, 16 tokens of a value
//     dim.  The rows of a key tile are taken in the order that leaves a lane with the 16 tokens whose values it loads, so
//     the softmax's weights go from one product into the other in registers, and a softmax over tokens needs two
//     exchanges between lanes a block;
//   * codes become fp16 exactly (bytes beside 0x64 are 1024 + code + 128), scales multiply scores and weights in fp32;
//   * q is split into two fp16 terms (22 bits of elements down to 2^-16 of the largest, 18 at 2^-20), so that scores are about as
//     good as fp32's; weights are rounded once, to 11 bits,
//     relative to the wave's largest value scale times 2^12 (they stay normal over scales 2^26 apart);
//   * the unfinished block's bf16 rows go through the bf16 products, a quarter a wave, q and weights in two bf16 terms, their
//     values as they are.
// The wave that holds the new token writes it; the four round its block if that is now whole, and then read it as codes.
// Measured (32 / 8 heads): 32 sequences of 15000 to 16200 tokens 181 us, 5.6 TB/s of the cache's bytes, each read once; one of
// 4096 tokens 11.2 us, of 200 8.0 us, where the chain of lengths, q, codes, products and join is what is left (an empty launch
// takes 1.7).  Two waves a SIMD (184 registers hold a block's codes while the next one's are on their way): at three, with the
// loads later, the long case took 10 % more.

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int DQ_WAVES = 4;
constexpr int DQ_ROW = Q8_D + 4;          // fp32 row in LDS, padded
constexpr int DQ_QROW = Q8_D + 8;         // fp16 row
constexpr uint32_t DQ_SLOTS = 512;        // thread blocks that the chip holds at once
constexpr uint32_t DQ_CHUNK_MAX = 32;     // blocks a unit, at most
constexpr float DQ_P_SCALE = 4096.0f;

struct DecodeQ8Args {
    KvQ8 c;
    const float* q;
    const float* k_new;
    const float* v_new;
    size_t q_row, k_row, v_row;
    const float* q_norm_w;
    const float* k_norm_w;
    const int32_t* lengths;
    const int32_t* offsets;
    const float* w_in;
    float* w_out;
    uint16_t* out;
    float* part_ml;  // [units][nk][group][2]: log2 maximum, sum
    float* part_o;   // [units][nk][group][128]
    uint32_t* done;  // [n_seq][nk] units that have left their parts; zero between calls
    float* scores;   // [n_seq][nh][s_cap] log2 scores, or null
    uint32_t n_seq, nh, group, units;
    float eps, scale_log2;
    double log2_theta;
    int rope;
};

// What units are found from: the lengths before a call of up to n new tokens a sequence.
struct UnitsOf {
    const int32_t* lengths;
    const int32_t* counts;
    uint32_t n, n_seq, nb, nk;

    __device__ __forceinline__ int blocks(uint32_t seq) const {
        if (counts && counts[seq] <= 0) return 0;
        return (q8_span(lengths, counts, seq, n, nb).end + Q8_BLOCK - 1) / Q8_BLOCK;
    }
};

struct DecodeUnit {
    uint32_t seq, first, count;  // the sequence, where its parts begin and how many units it has
    int part;                    // the unit among them
    int chunk, blocks, len;      // blocks a unit, the sequence's blocks and its length before the call
};

// Blocks a unit, for the blocks of all sequences: 4 (one a wave) where that makes a sequence one unit, which needs no join, or
// its units many; 1 or 2 between, as a CU takes a block in no less than 0.5 us and the chip is far from full.  Then one thread
// block a CU until units have 8, then two a CU, which the registers allow, or one where the sequences' heads alone are that many,
// until units have 32, where what a unit costs besides its blocks (3 to 4 us: lengths, q, joining) no longer matters and ragged
// lengths want the chip refilled.  Measured (us, 32 / 8 heads but for the sixth): 200 tokens 8.4 in units of 4, 9.0 of 1; 500 11.4
// and 9.1; 2000 11.5 of 4, 10.4 of 2, 11.8 of 1; 16000 15.1 of 8, 18.3 of 4; 16 sequences of 100 to 8000 39 of 20, 44 of 12, 46 of
// 32; 128 of 300 to 1200, 4 KV heads, 32 at one a CU, 38 at two; 64 of 100 to 16000 209 of up to 32, 219 of 64.
__device__ __forceinline__ uint32_t dq_chunk(uint64_t total, uint32_t n_seq, uint32_t nk) {
    const uint64_t blocks = total * nk, one = (blocks + 255) / 256;
    const uint64_t two = (blocks * (n_seq * nk >= DQ_SLOTS / 2 ? 2 : 1) + DQ_SLOTS - 1) / DQ_SLOTS;
    const uint64_t c = one <= 8 ? one : (two > 8 ? two : 8);
    if (c <= 2 && total > (uint64_t)n_seq * DQ_WAVES) {
        if (c < 2 && total <= (uint64_t)n_seq * 16) return 1;
        if (total <= (uint64_t)n_seq * 32) return 2;
    }
    return c <= DQ_WAVES ? DQ_WAVES : c >= DQ_CHUNK_MAX ? DQ_CHUNK_MAX : (uint32_t)((c + DQ_WAVES - 1) / DQ_WAVES * DQ_WAVES);
}

// The unit `unit` (by_seq false), or sequence `unit`; false where there is none.  Units of a whole chunk come first, the
// sequences' last, shorter ones behind them, so that what the chip ends with is short (64 sequences of 100 to 16000
// tokens: 219 us, 240 sequence by sequence).  A sequence without blocks has one unit, which writes its zeros.
__device__ bool dq_find(const UnitsOf& a, uint32_t unit, bool by_seq, DecodeUnit& u) {
    const uint32_t lane = threadIdx.x & 63;
    if (a.n_seq == 1) {
        u.blocks = a.blocks(0);
        u.chunk = (int)dq_chunk((uint64_t)u.blocks, 1, a.nk);
        u.seq = u.first = 0;
        u.part = (int)unit;
        u.count = u.blocks ? (uint32_t)((u.blocks + u.chunk - 1) / u.chunk) : 1u;
        u.len = a.lengths[0];
        return by_seq || unit < u.count;
    }
    uint32_t total = 0;
    for (uint32_t i = lane; i < a.n_seq; i += 64) total += (uint32_t)a.blocks(i);
    total = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan_u32(total), 63);
    u.chunk = (int)dq_chunk(total, a.n_seq, a.nk);
    uint32_t fulls = 0;  // units of a whole chunk
    if (!by_seq) {
        for (uint32_t i = lane; i < a.n_seq; i += 64) fulls += (uint32_t)a.blocks(i) / (uint32_t)u.chunk;
        fulls = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan_u32(fulls), 63);
    }
    uint32_t before = 0, fulls_before = 0;
    for (uint32_t base = 0; base < a.n_seq; base += 64) {
        const uint32_t i = base + lane;
        const uint32_t n = i < a.n_seq ? (uint32_t)a.blocks(i) : 0u, full = n / (uint32_t)u.chunk;
        const uint32_t mine = i < a.n_seq ? (n ? (n + u.chunk - 1) / u.chunk : 1u) : 0u;
        const uint32_t upto = before + wave_scan_u32(mine), fulls_upto = fulls_before + wave_scan_u32(full);
        const uint32_t rest_upto = upto - fulls_upto;  // units of less than a chunk, up to one a sequence
        const bool is_full = unit < fulls;
        const uint64_t hit = by_seq    ? __ballot(i == unit)
                             : is_full ? __ballot(unit >= fulls_upto - full && unit < fulls_upto)
                                       : __ballot(mine > full && unit - fulls == rest_upto - 1);
        if (hit) {
            const int at = __builtin_ctzll(hit);
            u.seq = base + at;
            u.count = (uint32_t)__builtin_amdgcn_readlane((int)mine, at);
            u.first = (uint32_t)__builtin_amdgcn_readlane((int)(upto - mine), at);
            u.part = is_full ? (int)(unit - (uint32_t)__builtin_amdgcn_readlane((int)(fulls_upto - full), at)) : (int)u.count - 1;
            u.blocks = a.blocks(u.seq);
            u.len = a.lengths[u.seq];
            return true;
        }
        before = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
        fulls_before = (uint32_t)__builtin_amdgcn_readlane((int)fulls_upto, 63);
    }
    return false;
}

// Four codes as fp16: 0x6400 + byte is 1024 + byte.
__device__ __forceinline__ void codes_f16(uint32_t w, f16x2_t& lo, f16x2_t& hi) {
    const uint32_t x = w ^ 0x80808080u;
    const f16x2_t off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    lo = __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) + off;
    hi = __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) + off;
}

__device__ __forceinline__ f16x8 codes_f16x8(uint32_t w0, uint32_t w1) {
    f16x2_t r[4];
    codes_f16(w0, r[0], r[1]);
    codes_f16(w1, r[2], r[3]);
    return __builtin_bit_cast(f16x8, r);
}

__device__ __forceinline__ bf16x8 as_bf16x8(uint4 v) { return __builtin_bit_cast(bf16x8, v); }

// The codes of four bf16 values.
__device__ __forceinline__ uint32_t bf16_codes(uint32_t w0, uint32_t w1, float inv) {
    return q8_pack4(__uint_as_float(w0 << 16), __uint_as_float(w0 & 0xffff0000u), __uint_as_float(w1 << 16),
                    __uint_as_float(w1 & 0xffff0000u), inv);
}

// Whether the low or the high one of two bf16 values is a NaN or an infinity, which becomes 0.
__device__ __forceinline__ bool bf16_drop_broken(uint32_t& w, int high) {
    const uint32_t mask = high ? 0xffff0000u : 0xffffu;
    if ((w & mask & 0x7f807f80u) != (mask & 0x7f807f80u)) return false;
    w &= ~mask;
    return true;
}

// Two floats past the caches that the chip's parts do not share.
__device__ __forceinline__ void put_pair(float* p, float x, float y) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), (uint64_t)__float_as_uint(x) | (uint64_t)__float_as_uint(y) << 32,
                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get_pair(const float* p) {
    const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// A query in fp16: its largest value is brought to [2^13, 2^14) by a power of two.  Its products with codes stay in fp32's range
// and what fp16 holds least, 2^-24, is 2^-37 of that value or less: near 1 it would be 2^-24 of it, and an element 2^-18 of the
// largest, whose keys may be the larger by as much, would have lost all but 7 bits.
__device__ __forceinline__ uint32_t q_exponent(float largest) {
    const uint32_t e = __float_as_uint(largest) >> 23;
    return e < 14 ? 14 : (e > 253 ? 253 : e);
}
__device__ __forceinline__ float q_to_fp16(uint32_t e) { return __uint_as_float((267u - e) << 23); }
__device__ __forceinline__ float q_from_fp16(uint32_t e) { return __uint_as_float((e - 13u) << 23); }

template <bool WEIGHTS>
__global__ __launch_bounds__(DQ_WAVES * 64, 2) void attn_decode_q8_kernel(const DecodeQ8Args a) {
    __shared__ __align__(16) _Float16 qs[2][16][DQ_QROW];      // q's two terms (q_to_fp16)
    __shared__ float qf[16];                                  // what that took off, with the softmax's scale and log2 e
    __shared__ __align__(16) uint16_t fresh[2][Q8_D];         // the new token's key and value
    __shared__ float wml[DQ_WAVES][16][2];
    __shared__ __align__(16) float wo[DQ_WAVES][16][DQ_ROW];
    __shared__ uint32_t arrived, top[2][DQ_WAVES];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t h = blockIdx.x % a.c.nk;
    const uint32_t unit = blockIdx.x / a.c.nk;
    DecodeUnit u;
    // (every wave of a thread block finds the same)
    if (!dq_find({a.lengths, nullptr, 1, a.n_seq, a.c.nb, a.c.nk}, unit, false, u)) return;
    const int group = (int)a.group;
    uint32_t* const out = reinterpret_cast<uint32_t*>(a.out + ((size_t)u.seq * a.nh + h * group) * Q8_D);
    if (u.blocks == 0) {
        for (int i = tid; i < group * (Q8_D / 2); i += DQ_WAVES * 64) out[i] = 0u;
        return;
    }
    const int b0 = u.part * u.chunk;
    const int b1 = b0 + u.chunk < u.blocks ? b0 + u.chunk : u.blocks;
    const int c = lane & 15, g4 = lane >> 4;
    const bool has_new = u.len < (int)(a.c.nb * Q8_BLOCK);
    const int new_b = has_new ? u.len / Q8_BLOCK : -1;  // the block of the new token, in bf16 unless the token finishes it
    const int r = u.len % Q8_BLOCK;
    const int tail_b = r == Q8_BLOCK - 1 ? -1 : new_b;
    const bool new_here = new_b >= b0 && new_b < b1;
    const bool has_tail = tail_b >= b0 && tail_b < b1;
    const bool writes = new_here && (new_b - b0) % DQ_WAVES == wave;

    // 1. the small operands (loads return in order: what is asked for after the codes would wait for them), then the first
    // block's codes
    const bool has_w = a.q_norm_w != nullptr;
    float w0 = 1.0f, w1 = 1.0f, kw0 = 1.0f, kw1 = 1.0f;
    if (has_w) {
        w0 = a.q_norm_w[lane];
        w1 = a.q_norm_w[lane + 64];
    }
    float x0[4], x1[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int g = wave + DQ_WAVES * i < group ? wave + DQ_WAVES * i : 0;
        const float* x = a.q + u.seq * a.q_row + (size_t)(h * group + g) * Q8_D;
        if (DQ_WAVES * i < group) {
            x0[i] = x[lane];
            x1[i] = x[lane + 64];
        }
    }
    float kx0 = 0.0f, kx1 = 0.0f, vx0 = 0.0f, vx1 = 0.0f;
    if (writes) {
        const float* kx = a.k_new + u.seq * a.k_row + (size_t)h * Q8_D;
        const float* vx = a.v_new + u.seq * a.v_row + (size_t)h * Q8_D;
        kx0 = kx[lane];
        kx1 = kx[lane + 64];
        vx0 = vx[lane];
        vx1 = vx[lane + 64];
        if (has_w) {
            kw0 = a.k_norm_w[lane];
            kw1 = a.k_norm_w[lane + 64];
        }
    }
    const int pos = u.len + (a.offsets ? a.offsets[u.seq] : 0);
    // the largest value scale of the wave's blocks; a block that is only now rounded comes later
    float smax = 0.0f;
    for (int i = b0 + wave + DQ_WAVES * lane; i < b1; i += DQ_WAVES * 64)
        if (i != new_b) smax = fmaxf(smax, a.c.vs[a.c.scale_at(u.seq, (uint32_t)i, h)]);
    const int krow = ((c >> 2) * 16 + (c & 3)) * Q8_D + g4 * 16;  // + t * 4 rows + j * 64
    const int vrow = c * Q8_BLOCK + g4 * 16;                      // + dt * 16 rows
    uint4 kr[8], vr[8];  // key tile t, dims 64 j ..: 2 t + j
    float ks = 0.0f, vs = 0.0f;
    auto load_k = [&](int b) {
        const int8_t* p = a.c.k + a.c.block_at(u.seq, (uint32_t)b, h) + krow;
#pragma unroll
        for (int n = 0; n < 8; ++n) kr[n] = load_nt_u4(p + (n >> 1) * 4 * Q8_D + (n & 1) * 64);
        ks = a.c.ks[a.c.scale_at(u.seq, (uint32_t)b, h)];
    };
    auto load_v = [&](int b) {
        const int8_t* p = a.c.v + a.c.block_at(u.seq, (uint32_t)b, h) + vrow;
#pragma unroll
        for (int n = 0; n < 8; ++n) vr[n] = load_nt_u4(p + n * 16 * Q8_BLOCK);
        vs = a.c.vs[a.c.scale_at(u.seq, (uint32_t)b, h)];
    };
    // the tail's rows, a quarter a wave: token 16 (c / 4) + 4 wave + c % 4, dims 64 j + 16 g4 + 8 i; and the values of
    // tokens 16 g4 + 4 wave .. of dim 16 n + c
    const size_t tail = a.c.tail_at(u.seq, h);
    auto load_tail = [&](uint4 (&tk)[4], uint2 (&tv)[8]) {
#pragma unroll
        for (int n = 0; n < 4; ++n) tk[n] = load_u4(a.c.kt + tail + krow + wave * 4 * Q8_D + 64 * (n >> 1) + 8 * (n & 1));
#pragma unroll
        for (int n = 0; n < 8; ++n) tv[n] = *reinterpret_cast<const uint2*>(a.c.vt + tail + vrow + n * 16 * Q8_BLOCK + 4 * wave);
    };
    // the new token among them: its key a row, its value one of a word's two tokens (behind it: zeros)
    auto put_new = [&](uint4 (&tk)[4], uint2 (&tv)[8]) {
        if ((c >> 2) * 16 + wave * 4 + (c & 3) == r) {
#pragma unroll
            for (int n = 0; n < 4; ++n) tk[n] = *reinterpret_cast<const uint4*>(&fresh[0][64 * (n >> 1) + 16 * g4 + 8 * (n & 1)]);
        }
        const int ahead = r - 16 * g4 - 4 * wave;
        const uint32_t old0 = ahead <= 0 ? 0u : ahead == 1 ? 0xffffu : 0xffffffffu;
        const uint32_t old1 = ahead <= 2 ? 0u : ahead == 3 ? 0xffffu : 0xffffffffu;
        const uint32_t new0 = ahead == 0 ? 0xffffu : ahead == 1 ? 0xffff0000u : 0u;
        const uint32_t new1 = ahead == 2 ? 0xffffu : ahead == 3 ? 0xffff0000u : 0u;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const uint32_t vnew = fresh[1][16 * n + c] * 0x10001u;
            tv[n] = make_uint2((tv[n].x & old0) | (vnew & new0), (tv[n].y & old1) | (vnew & new1));
        }
    };
    int b = b0 + wave;
    if (b < b1 && b != new_b) {
        load_k(b);
        load_v(b);
    }

    // 2. q and the new token
    float cs = 1.0f, sn = 0.0f;
    if (a.rope && (wave < group || writes)) rope_at(rope_turns(lane, a.log2_theta), pos, cs, sn);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int g = wave + DQ_WAVES * i;
        if (g >= group) break;
        float y[2];
        q8_norm_rope(x0[i], x1[i], has_w, w0, w1, a.eps, cs, sn, y[0], y[1]);
        const uint32_t e = q_exponent(wave_max(fmaxf(fabsf(y[0]), fabsf(y[1]))));  // (a NaN stays one whatever e is)
        const float down = q_to_fp16(e);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const _Float16 hi = (_Float16)(y[n] * down);
            qs[0][g][lane + 64 * n] = hi;
            qs[1][g][lane + 64 * n] = (_Float16)(y[n] * down - (float)hi);
        }
        if (lane == 0) qf[g] = q_from_fp16(e) * a.scale_log2;
    }
    if (writes) {
        float y[2];
        q8_norm_rope(kx0, kx1, has_w, kw0, kw1, a.eps, cs, sn, y[0], y[1]);
        const float v[2] = {vx0, vx1};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint16_t kb = (uint16_t)f32_to_bf16_bits(y[i]), vb = (uint16_t)f32_to_bf16_bits(v[i]);
            fresh[0][lane + 64 * i] = kb;
            fresh[1][lane + 64 * i] = vb;
            a.c.kt[tail + r * Q8_D + lane + 64 * i] = kb;
            a.c.vt[tail + (lane + 64 * i) * Q8_BLOCK + r] = vb;
        }
    }
    __syncthreads();
    if (new_here) {
        if (!has_tail) {  // the new token finishes its block: rounded here, then read as codes
            uint4 tk[4];
            uint2 tv[8];
            load_tail(tk, tv);
            put_new(tk, tv);
            uint32_t kmax = 0, vmax = 0;
#pragma unroll
            for (int n = 0; n < 4; ++n) kmax = max(max(kmax, max(bf16_abs_max(tk[n].x), bf16_abs_max(tk[n].y))),
                                                   max(bf16_abs_max(tk[n].z), bf16_abs_max(tk[n].w)));
#pragma unroll
            for (int n = 0; n < 8; ++n) vmax = max(vmax, max(bf16_abs_max(tv[n].x), bf16_abs_max(tv[n].y)));
            kmax = wave_max_u32(kmax);
            vmax = wave_max_u32(vmax);
            if (lane == 0) {
                top[0][wave] = kmax;
                top[1][wave] = vmax;
            }
            __syncthreads();
            float k_scale, v_scale, k_inv, v_inv;
            q8_scale(max(max(top[0][0], top[0][1]), max(top[0][2], top[0][3])), k_scale, k_inv);
            q8_scale(max(max(top[1][0], top[1][1]), max(top[1][2], top[1][3])), v_scale, v_inv);
            const size_t at = a.c.block_at(u.seq, (uint32_t)new_b, h), scale_at = a.c.scale_at(u.seq, (uint32_t)new_b, h);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint4 x = tk[2 * j], y = tk[2 * j + 1];
                *reinterpret_cast<uint4*>(a.c.k + at + krow + wave * 4 * Q8_D + 64 * j) =
                    make_uint4(bf16_codes(x.x, x.y, k_inv), bf16_codes(x.z, x.w, k_inv), bf16_codes(y.x, y.y, k_inv),
                               bf16_codes(y.z, y.w, k_inv));
            }
#pragma unroll
            for (int n = 0; n < 8; ++n)
                *reinterpret_cast<uint32_t*>(a.c.v + at + vrow + n * 16 * Q8_BLOCK + 4 * wave) = bf16_codes(tv[n].x, tv[n].y, v_inv);
            if (tid == 0) {
                a.c.ks[scale_at] = k_scale;
                a.c.vs[scale_at] = v_scale;
            }
            __threadfence_block();
            __syncthreads();
            if (writes) smax = fmaxf(smax, v_scale);
            if (b == new_b) {
                load_k(b);
                load_v(b);
            }
        }
    }
    const float qfac = qf[c];  // lanes past the group hold what no one reads: a head is a column of the products
    smax = wave_max(smax);
    auto query = [&](int term, int j, int i) {  // dims 64 j + 16 g4 + 8 i
        return *reinterpret_cast<const f16x8*>(&qs[term][c][64 * j + 16 * g4 + 8 * i]);
    };

    // 3. the wave's blocks
    float m = -INFINITY, l = 0.0f;
    f32x4 o[8];
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) o[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    // scores of key tiles t0, t0 + 1, .. of a block (x: dot products, to be multiplied by f) -> weights; a lane's tokens are
    // 16 g4 + 4 t + i
    auto soften = [&](auto& x, int t0, float f, int b, int live) {
        constexpr int N = sizeof(x) / sizeof(x[0]);
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[t][i] *= f;
                if (live < Q8_BLOCK && 16 * g4 + 4 * (t0 + t) + i >= live) x[t][i] = -INFINITY;
                top = fmaxf(top, x[t][i]);
            }
        if (WEIGHTS && c < group) {
            float* to = a.scores + ((size_t)u.seq * a.nh + h * group + c) * a.c.nb * Q8_BLOCK + b * Q8_BLOCK + 16 * g4 + 4 * t0;
#pragma unroll
            for (int t = 0; t < N; ++t) *reinterpret_cast<f32x4*>(to + 4 * t) = x[t];
        }
        top = fmaxf(m, xor_max<32>(xor_max<16>(top)));
        const float base = top == -INFINITY ? 0.0f : top;
        const float keep = __builtin_amdgcn_exp2f(m - base);
        float sum = 0.0f;
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[t][i] = __builtin_amdgcn_exp2f(x[t][i] - base);
                sum += x[t][i];
            }
        l = fmaf(l, keep, sum);
        m = top;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) o[dt] *= keep;
    };

    for (; b < b1 && b != tail_b; b += DQ_WAVES) {
        f32x4 x[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const f16x8 h0 = query(0, j, 0), l0 = query(1, j, 0), h1 = query(0, j, 1), l1 = query(1, j, 1);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                __builtin_amdgcn_sched_barrier(0);
                const uint4 kk = kr[2 * t + j];
                const f16x8 k0 = codes_f16x8(kk.x, kk.y), k1 = codes_f16x8(kk.z, kk.w);
                x[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, h0, x[t], 0, 0, 0);
                x[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, l0, x[t], 0, 0, 0);
                x[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, h1, x[t], 0, 0, 0);
                x[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, l1, x[t], 0, 0, 0);
            }
        }
        const float fk = ks * qfac;
        const int next = b + DQ_WAVES;
        const bool more = next < b1 && next != tail_b;
        if (more) load_k(next);
        soften(x, 0, fk, b, Q8_BLOCK);
        const float fv = vs * (DQ_P_SCALE / (smax > 0.0f ? smax : 1.0f));
        f16x8 p[2];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) p[s][e] = (_Float16)(x[2 * s + e / 4][e % 4] * fv);
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
            __builtin_amdgcn_sched_barrier(0);
            o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_f16x8(vr[dt].x, vr[dt].y), p[0], o[dt], 0, 0, 0);
            o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_f16x8(vr[dt].z, vr[dt].w), p[1], o[dt], 0, 0, 0);
        }
        if (more) load_v(next);
    }

    float unscale = (smax > 0.0f ? smax : 1.0f) * (1.0f / DQ_P_SCALE);  // the unit that the accumulators are in
    if (has_tail) {  // tile `wave` of the unfinished block
        uint4 tk[4];
        uint2 tv[8];
        load_tail(tk, tv);
        put_new(tk, tv);
        f32x4 x[1] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int j = n >> 1, i = n & 1;
            const f16x8 hi = query(0, j, i), lo = query(1, j, i);
            bf16x8 q2[2];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = (float)hi[e] + (float)lo[e];
                q2[0][e] = (__bf16)y;
                q2[1][e] = (__bf16)(y - (float)q2[0][e]);
            }
            const bf16x8 kk = as_bf16x8(tk[n]);
            x[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kk, q2[0], x[0], 0, 0, 0);
            x[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kk, q2[1], x[0], 0, 0, 0);
        }
        soften(x, wave, qfac, tail_b, r + 1);
        // the values as they are: in the blocks' unit, which they may be any number of times, products could leave fp32's range
        bf16x4 ph, pl;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            ph[e] = (__bf16)x[0][e];
            pl[e] = (__bf16)(x[0][e] - (float)ph[e]);
        }
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) o[dt] *= unscale;
        unscale = 1.0f;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
            o[dt] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(t2h_v4i16, tv[dt]), __builtin_bit_cast(t2h_v4i16, ph),
                                                              o[dt], 0, 0, 0);
            o[dt] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(t2h_v4i16, tv[dt]), __builtin_bit_cast(t2h_v4i16, pl),
                                                              o[dt], 0, 0, 0);
        }
    }

    // 4. the waves' states joined; one unit: the output itself, more: the unit's part of it
    l = xor_sum<32>(xor_sum<16>(l));
    if (c < group) {
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) *reinterpret_cast<f32x4*>(&wo[wave][c][16 * dt + 4 * g4]) = o[dt] * unscale;
        if (g4 == 0) {
            wml[wave][c][0] = m;
            wml[wave][c][1] = l;
        }
    }
    __syncthreads();
    const int waves = !has_tail && b1 - b0 < DQ_WAVES ? b1 - b0 : DQ_WAVES;
    for (int i = tid; i < group * (Q8_D / 4); i += DQ_WAVES * 64) {
        const int g = i / (Q8_D / 4), d = i % (Q8_D / 4) * 4;
        float M = -INFINITY, L = 0.0f;
        for (int w = 0; w < waves; ++w) M = fmaxf(M, wml[w][g][0]);
        const float base = M == -INFINITY ? 0.0f : M;
        f32x4 sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int w = 0; w < waves; ++w) {
            const float f = __builtin_amdgcn_exp2f(wml[w][g][0] - base);
            L = fmaf(f, wml[w][g][1], L);
            sum += *reinterpret_cast<const f32x4*>(&wo[w][g][d]) * f;
        }
        const size_t part = ((size_t)(u.first + (uint32_t)u.part) * a.c.nk + h) * a.group + g;
        if (u.count == 1) {
            const float inv = 1.0f / L;
            out[(g * Q8_D + d) / 2] = pack_bf16x2(sum[0] * inv, sum[1] * inv);
            out[(g * Q8_D + d) / 2 + 1] = pack_bf16x2(sum[2] * inv, sum[3] * inv);
        } else {
            put_pair(a.part_o + part * Q8_D + d, sum[0], sum[1]);
            put_pair(a.part_o + part * Q8_D + d + 2, sum[2], sum[3]);
        }
        if (d == 0 && (WEIGHTS || u.count > 1)) put_pair(a.part_ml + 2 * part, M, L);
    }
    if (u.count == 1) return;

    // 5. the last unit of a (sequence, head) to get here joins them.  Parts are written and read past the caches that the
    // chip's parts do not share (agent scope), and are there before the count is raised.
    __builtin_amdgcn_s_waitcnt(0);
    asm volatile("" ::: "memory");
    __syncthreads();
    if (tid == 0) {
        uint32_t* const done = a.done + (size_t)u.seq * a.c.nk + h;
        arrived = __hip_atomic_fetch_add(done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u;
        if (arrived == u.count) __hip_atomic_store(done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (arrived != u.count) return;
    // slices of the units, each a sum of its own in LDS
    const int pieces = group * (Q8_D / 4);
    const int slices = DQ_WAVES * 64 / pieces > 0 ? DQ_WAVES * 64 / pieces : 1;
    constexpr int BATCH = 16;  // parts of a slice in flight
    for (int i = tid; i < pieces * slices; i += DQ_WAVES * 64) {
        const int slice = i / pieces, g = i % pieces / (Q8_D / 4), d = i % (Q8_D / 4) * 4;
        float M = -INFINITY, L = 0.0f;
        f32x4 sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t n0 = (uint32_t)slice; n0 < u.count; n0 += (uint32_t)slices * BATCH) {
            float2 ml[BATCH], lo[BATCH], hi[BATCH];
#pragma unroll
            for (int e = 0; e < BATCH; ++e) {
                const uint32_t n = n0 + (uint32_t)(slices * e);
                const size_t part = ((size_t)(u.first + (n < u.count ? n : n0)) * a.c.nk + h) * a.group + g;
                ml[e] = get_pair(a.part_ml + 2 * part);
                lo[e] = get_pair(a.part_o + part * Q8_D + d);
                hi[e] = get_pair(a.part_o + part * Q8_D + d + 2);
            }
#pragma unroll
            for (int e = 0; e < BATCH; ++e) {
                if (n0 + (uint32_t)(slices * e) >= u.count) break;
                const float now = fmaxf(M, ml[e].x), base = now == -INFINITY ? 0.0f : now;
                const float keep = __builtin_amdgcn_exp2f(M - base), f = __builtin_amdgcn_exp2f(ml[e].x - base);
                L = fmaf(L, keep, f * ml[e].y);
                sum = sum * keep + f32x4{lo[e].x, lo[e].y, hi[e].x, hi[e].y} * f;
                M = now;
            }
        }
        const int at = slice * group + g;  // less than 16: 8 slices are of one head
        *reinterpret_cast<f32x4*>(&wo[0][at][d]) = sum;
        if (d == 0) {
            wml[0][at][0] = M;
            wml[0][at][1] = L;
        }
    }
    __syncthreads();
    for (int i = tid; i < pieces; i += DQ_WAVES * 64) {
        const int g = i / (Q8_D / 4), d = i % (Q8_D / 4) * 4;
        float M = -INFINITY, L = 0.0f;
        for (int n = 0; n < slices; ++n) M = fmaxf(M, wml[0][n * group + g][0]);
        const float base = M == -INFINITY ? 0.0f : M;
        f32x4 sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int n = 0; n < slices; ++n) {
            const float f = __builtin_amdgcn_exp2f(wml[0][n * group + g][0] - base);
            L = fmaf(f, wml[0][n * group + g][1], L);
            sum += *reinterpret_cast<const f32x4*>(&wo[0][n * group + g][d]) * f;
        }
        const float inv = 1.0f / L;
        out[(g * Q8_D + d) / 2] = pack_bf16x2(sum[0] * inv, sum[1] * inv);
        out[(g * Q8_D + d) / 2 + 1] = pack_bf16x2(sum[2] * inv, sum[3] * inv);
    }
}

// log2 maximum and sum of a head over the units of its sequence; every lane gets them
__device__ __forceinline__ void dq_total(const DecodeQ8Args& a, const DecodeUnit& u, uint32_t h, uint32_t g, float& M, float& L) {
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml);
    M = -INFINITY;
    L = 0.0f;
    for (uint32_t i = threadIdx.x & 63; i < u.count; i += 64) M = fmaxf(M, ml[((size_t)(u.first + i) * a.c.nk + h) * a.group + g].x);
    M = wave_max(M);
    const float base = M == -INFINITY ? 0.0f : M;
    for (uint32_t i = threadIdx.x & 63; i < u.count; i += 64) {
        const float2 x = ml[((size_t)(u.first + i) * a.c.nk + h) * a.group + g];
        L = fmaf(__builtin_amdgcn_exp2f(x.x - base), x.y, L);
    }
    L = wave_sum(L);
}

constexpr int DQ_SEGMENT = 1024;  // tokens of a thread block that adds up weights

// weights_out[token] = weights_in (0 for the new token) + sum of exp2(score - log2 sum) over the heads of the KV head:
// 1024 tokens of a (sequence, KV head) a thread block.  A second kernel, because a token's weight needs the sum over all units:
// the scores pass through memory (4 bytes a head and token beside the cache's 256 a KV head and token).  6.3 us for 16
// sequences of 100 to 8000 tokens, beside the attention's 35.
__global__ __launch_bounds__(256) void attn_decode_q8_weights_kernel(const DecodeQ8Args a) {
    __shared__ float lse[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t h = blockIdx.x % a.c.nk, rest = blockIdx.x / a.c.nk;
    const uint32_t segments = (a.c.nb * Q8_BLOCK + DQ_SEGMENT - 1) / DQ_SEGMENT;
    const uint32_t seq = rest / segments;
    const int first = (int)(rest % segments) * DQ_SEGMENT, t0 = first + 4 * tid;
    const int len = a.lengths[seq], cap = (int)(a.c.nb * Q8_BLOCK);
    const int end = len < 0 ? 0 : (len < cap ? len + 1 : cap);
    if (first >= end) return;
    // what does not wait for the sums is asked for before them
    const float* const scores = a.scores + ((size_t)seq * a.nh + h * a.group) * cap + t0;
    const size_t at = ((size_t)seq * a.c.nk + h) * cap + t0;
    constexpr uint32_t AHEAD = 4;
    f32x4 early[AHEAD];
    float before[4];
    if (t0 < end) {
#pragma unroll
        for (uint32_t g = 0; g < AHEAD; ++g)
            if (g < a.group) early[g] = *reinterpret_cast<const f32x4*>(scores + (size_t)g * cap);
#pragma unroll
        for (int j = 0; j < 4; ++j) before[j] = t0 + j < len ? a.w_in[at + j] : 0.0f;
    }
    DecodeUnit u;
    dq_find({a.lengths, nullptr, 1, a.n_seq, a.c.nb, a.c.nk}, seq, true, u);
    for (uint32_t g = wave; g < a.group; g += 4) {
        float M, L;
        dq_total(a, u, h, g, M, L);
        if (lane == 0) lse[g] = M + log2f(L);
    }
    __syncthreads();
    if (t0 >= end) return;
    f32x4 sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    auto add = [&](f32x4 s, uint32_t g) {
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] += __builtin_amdgcn_exp2f(s[j] - lse[g]);
    };
#pragma unroll
    for (uint32_t g = 0; g < AHEAD; ++g)
        if (g < a.group) add(early[g], g);
    for (uint32_t g = AHEAD; g < a.group; ++g) add(*reinterpret_cast<const f32x4*>(scores + (size_t)g * cap), g);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (t0 + j < end) a.w_out[at + j] = before[j] + sum[j];
}

// Counters at the start of the workspace, as many for every shape (of up to 16384 sequences times KV heads), so that calls of
// several shapes may share one: another shape's parts never lie where counters are.
static size_t dq_counters(uint32_t n_seq, uint32_t nk) {
    const size_t heads = (size_t)n_seq * nk;
    return heads <= 16384 ? 16384 : (heads + 3) / 4 * 4;
}

// Units that sequences of any lengths can have: sum of ceil(blocks / chunk) <= total / chunk + n_seq, and total / chunk is at
// most that of the largest total or the slots' share, as the chunk grows with the total in between.
static uint32_t dq_units(uint32_t n_seq, uint32_t nk, uint32_t nb) {
    const uint64_t most = (uint64_t)n_seq * nb, slots = DQ_SLOTS / nk, full = most / DQ_CHUNK_MAX;
    const uint64_t units = (slots > full ? slots : full) + n_seq;
    return (uint32_t)(units < most ? units : most);
}

// ------------------------------------------------------------------------------------------------------ chunks --
//
// Bound by the matrix cores and, as much, by the softmax's and the conversion's vector instructions.  The queries of a KV
// head's q heads are rows of one matrix (row = t * group + g), so a key tile serves them all; a wave takes
// 32 rows, a thread block 4 or 8 waves, and walks the cache a block of 64 tokens at a time:
//   * a block's codes go to registers one step ahead, become bf16 keys and fp16 values (both exact) and go to the other of
//     two LDS buffers: one barrier a step;
//   * S^T = K . Q^T and O^T = V^T . P^T (32 x 32 x 16), so that a lane has 32 of a row's 64 scores in registers: one
//     exchange a step for the row's maximum, none between the products (the key rows are taken in the order that makes a
//     lane's scores the tokens of its operand of the second one);
//   * scales go into the exponent: p of a block is exp2(s * ks + log2(vs / largest vs so far) - max), rounded once to fp16's 11
//     bits; the accumulators follow a maximum only when it has grown by more than 2^2, and a scale when it has more than
//     doubled, and then only in the rows that see its block.
// Where there are few rows the keys are split over thread blocks, and a second kernel joins the parts.
//
// Measured (32 / 8 heads): 8 x 2048 tokens 318 us, 865 TFLOP/s of the pairs that are seen; a prompt of 16000 1958 us, 1071, where
// a bf16 product of 8192^3 reaches 1197; 1901 tokens 47 us; 4 x 512 of 16 / 8 heads at 7000 144 us, 845, with the join.  At 8 x
// 2048 the matrix cores are busy for 38 % of the time and the vector units for 50 %: about 208 vector instructions and 32 products
// a step, half of the former the softmax's, a fifth the conversion's.  What took vector instructions out of the step paid (318 us;
// 337 with LDS addresses that depend on the buffer and a division a step); what let the two units overlap otherwise did not: a
// third buffer with half of the waves a phase behind, raised priority around the products, fewer LDS conflicts (22 -> 9 million
// cycles).

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr uint32_t CQ_WIDE_GRID = 512;
constexpr float CQ_SHIFT_LEAST = -60.0f;
constexpr float CQ_SLACK = 2.0f;        // log2 that a row's weights may pass 1 by: 2^12 * 2^2 * 2 is in fp16's range

struct ChunkQ8Args {
    KvQ8 c;
    const uint16_t* q;  // bf16 [n_seq][n][nh][128]
    uint16_t* out;
    float* lse;         // log2 of the softmax's denominator [n_seq][nk][n * group], or null
    float* part_ml;     // [splits][n_seq][nk][n * group][2]
    float* part_o;      // the same rows of 128
    const int32_t* lengths;
    const int32_t* counts;
    const float* w_in;
    float* w_out;
    float* w_part;      // [w_splits][n_seq][nk][s_cap] sums, or null
    uint32_t n, n_seq, nh, group, tiles, splits, w_splits;
    float scale_log2;
};

__device__ __forceinline__ f32x16 mfma_bf16(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma_f16(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Eight codes as bf16 (8 bits of significand hold them).
__device__ __forceinline__ uint4 codes_bf16x8(uint32_t w0, uint32_t w1) {
    return make_uint4(pack_bf16x2(q8_value(w0, 0), q8_value(w0, 1)), pack_bf16x2(q8_value(w0, 2), q8_value(w0, 3)),
                      pack_bf16x2(q8_value(w1, 0), q8_value(w1, 1)), pack_bf16x2(q8_value(w1, 2), q8_value(w1, 3)));
}

// LDS places of 16 bytes: keys and queries [64][128] and values [128][64], 2 bytes each, chunks of a row permuted by the row
// (two rows of values fill the banks once) so that the lanes of an operand's read, which are rows, meet different banks.
__device__ __forceinline__ int cq_key_at(int token, int chunk) { return token * 16 + (chunk ^ (token & 15)); }
__device__ __forceinline__ int cq_value_at(int d, int chunk) { return d * 8 + (chunk ^ (d >> 1 & 7)); }

template <int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void attn_chunk_q8_kernel(const ChunkQ8Args a) {
    constexpr int ROWS = 32 * WAVES, THREADS = 64 * WAVES, PIECES = Q8_BYTES / 16 / THREADS;
    __shared__ __align__(16) uint4 keys[2][Q8_BLOCK * 16];
    __shared__ __align__(16) uint4 values[2][Q8_D * 8];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, half = lane >> 5;
    // The longest tiles first; in every other round of 256 thread blocks, one a CU, from the shortest up, so that the CUs of
    // a grid of two or three rounds get long and short ones alike.  An XCD (of 8, in turn) keeps its share of the heads.
    uint32_t rest = blockIdx.x;
    if (rest / 256 & 1) {
        const uint32_t left = gridDim.x - rest / 256 * 256, size = left < 256 ? left / 8 * 8 : 256;
        if (rest % 256 < size) rest = rest / 256 * 256 + (size - 8 - rest % 256 / 8 * 8) + rest % 8;
    }
    const uint32_t h = rest % a.c.nk;  // neighbours work on different heads: with 8 of them an XCD's L2 holds one head's keys
    rest /= a.c.nk;
    const uint32_t split = rest % a.splits;
    rest /= a.splits;
    const uint32_t seq = rest % a.n_seq;
    const int tile = (int)(a.tiles - 1 - rest / a.n_seq);
    const Q8Span s = q8_span(a.lengths, a.counts, seq, a.n, a.c.nb);
    const int len = min(a.lengths[seq], (int)(a.c.nb * Q8_BLOCK));
    int count = a.counts ? a.counts[seq] : (int)a.n;
    count = len < 0 || count < 0 ? 0 : (count < (int)a.n ? count : (int)a.n);
    const int group = (int)a.group, rows = count * group;
    const size_t head_row = ((size_t)seq * a.c.nk + h) * a.n * group;  // of row 0 in lse and the parts

    // rows of this wave: row0 + lane % 32; `last` is the last token that the lane's row sees
    const int row0 = tile * ROWS + wave * 32;
    const int row = row0 + col;
    const int t = row / group, g = row - t * group;
    const int last = row < rows ? (len + t < s.end ? len + t : s.end - 1) : -1;
    const int wave_top = row0 + 31 < rows ? row0 + 31 : rows - 1;  // its last live row, below row0 if it has none
    const int wave_last = wave_top >= row0 ? (len + wave_top / group < s.end ? len + wave_top / group : s.end - 1) : -1;
    // (a wave without rows takes all of every block for seen, and what it computes for nothing)
    const int wave_first = row0 < rows ? (len + row0 / group < s.end ? len + row0 / group : s.end - 1) : 0x7fffffff;
    const int top_row = (tile + 1) * ROWS < rows ? (tile + 1) * ROWS - 1 : rows - 1;
    const int tile_last = tile * ROWS < rows ? (len + top_row / group < s.end ? len + top_row / group : s.end - 1) : -1;
    const int blocks = tile_last >= 0 ? tile_last / Q8_BLOCK + 1 : 0;
    const int b0 = (int)((int64_t)blocks * split / a.splits), b1 = (int)((int64_t)blocks * (split + 1) / a.splits);
    const int tail_b = s.end % Q8_BLOCK ? s.end / Q8_BLOCK : -1;  // held in bf16
    const bool has_tail = tail_b >= b0 && tail_b < b1;
    const int whole = has_tail ? b1 - 1 : b1;

    // a block's codes: 16-byte pieces tid, tid + THREADS .., of a token (8 pieces) and of a value's dim (4)
    uint4 kc[PIECES], vc[PIECES];
    float ks = 0.0f, vs = 0.0f, ks_next = 0.0f, vs_next = 0.0f;
    auto load = [&](int b) {
        const size_t at = a.c.block_at(seq, (uint32_t)b, h);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            kc[i] = load_u4(a.c.k + at + (tid + THREADS * i) * 16);
            vc[i] = load_u4(a.c.v + at + (tid + THREADS * i) * 16);
        }
        ks_next = a.c.ks[a.c.scale_at(seq, (uint32_t)b, h)];
        vs_next = a.c.vs[a.c.scale_at(seq, (uint32_t)b, h)];
    };
    // 16 bytes of LDS at a time: 0, 1: keys of piece 0, then its values, then those of piece 1
    auto store = [&](int buf, int e) {
        const int i = e >> 2, n = tid + THREADS * i;
        const uint32_t lo = e & 1 ? (e & 2 ? vc[i].z : kc[i].z) : (e & 2 ? vc[i].x : kc[i].x);
        const uint32_t hi = e & 1 ? (e & 2 ? vc[i].w : kc[i].w) : (e & 2 ? vc[i].y : kc[i].y);
        if (e & 2)
            values[buf][cq_value_at(n >> 2, 2 * (n & 3) + (e & 1))] = __builtin_bit_cast(uint4, codes_f16x8(lo, hi));
        else
            keys[buf][cq_key_at(n >> 3, 2 * (n & 7) + (e & 1))] = codes_bf16x8(lo, hi);
    };
    if (b0 < whole) load(b0);
    // the row's query
    uint4 q[8];
    const size_t q_at = ((size_t)seq * a.n + (row < rows ? t : 0)) * a.nh + h * group + (row < rows ? g : 0);
    const uint16_t* qp = a.q + q_at * Q8_D + 8 * half;
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = load_u4(qp + 16 * i);
    float m = -INFINITY, l = 0.0f;
    float smax = 0.0f;  // the largest value scale so far, or half of it: the accumulators are in units of smax / 2^12
    float own = 0.0f;   // the same of the blocks that the row sees, which its accumulators stay in
    float to_unit = DQ_P_SCALE;
    f32x16 o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[i][j] = 0.0f;
    const int key_row = (col & 19) | (col & 8) >> 1 | (col & 4) << 1;  // of operand row `col`: bits 2 and 3 change places

    // one block from LDS; f: the scores' factor, shift: log2 of the weights' (both of the whole block)
    auto scores = [&](int buf, f32x16 (&x)[2]) {
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
            for (int j = 0; j < 16; ++j) x[tt][j] = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                x[tt] = mfma_bf16(as_bf16x8(keys[buf][cq_key_at(32 * tt + key_row, 2 * i + half)]), as_bf16x8(q[i]), x[tt]);
        }
    };
    // What comes before the weights: rows that do not see all of the block, and the row's maximum, which the accumulators
    // follow.  A lane's scores j of tile tt are the tokens 32 tt + 16 (j / 8) + 8 half + j % 8; f is their factor, unit what the
    // accumulators' unit is to be multiplied by (1: as it is).
    auto ready = [&](f32x16 (&x)[2], int b, float& f, float unit) {
        if (b * Q8_BLOCK + Q8_BLOCK - 1 > wave_first) {
            const int mine = last - b * Q8_BLOCK - 8 * half;
            const bool broken = f != f;  // a scale that is NaN reaches the rows that see its block only
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    if (broken) x[tt][j] = __uint_as_float(0x7fc00000u);
                    if (32 * tt + 16 * (j >> 3) + (j & 7) > mine) x[tt][j] = -INFINITY;
                }
            if (broken) f = 1.0f;
        }
        // the maximum before the factor: ks and the scale are not negative
        float top = -INFINITY;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int j = 0; j < 16; ++j) top = fmaxf(top, x[tt][j]);
        top = xor_max<32>(top);
        top = top == -INFINITY ? top : top * f;
        if (unit != 1.0f || __any(top > m + CQ_SLACK)) {
            const float now = fmaxf(m, top);
            const float keep = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - now);
            l *= keep;
            m = now;
            const bool sees = last >= b * Q8_BLOCK;
            const float turn = sees ? keep * unit : keep;
            if (sees) own = smax;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) o[i][j] *= turn;
        }
    };
    // weights j0 .. j1 - 1 of the 8 that a lane has of 16 tokens, and their sum
    auto weigh = [&](f32x16 (&x)[2], int i, int j0, int j1, float f, float base, float& sum, float (&w)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (j < j0 || j >= j1) continue;
            w[j] = __builtin_amdgcn_exp2f(fmaf(x[i >> 1][8 * (i & 1) + j], f, -base));
            sum += w[j];
        }
    };

    // A step, in the order that it is issued in: block b's scores, a product for each of two tiles at a time and 8 codes of
    // block b + 1 between them (they came during the step before and go to the other buffer); then 8 weights of a lane's at a
    // time, two of them between two products of the 8 before.  Left to itself the compiler puts the products of a step in a
    // row, which leaves the vector unit idle, or all operands in flight, for which there are no registers.
    if (b0 < whole) {
#pragma unroll
        for (int e = 0; e < 4 * PIECES; ++e) store(0, e);
        ks = ks_next;
        vs = vs_next;
        if (b0 + 1 < whole) load(b0 + 1);
    }
    __syncthreads();
    auto step = [&](int b, auto which) {
        constexpr int buf = decltype(which)::value;
        f32x16 x[2];
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int j = 0; j < 16; ++j) x[tt][j] = 0.0f;
        uint4 kf[3][2];  // operands two steps ahead
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) kf[i][tt] = keys[buf][cq_key_at(32 * tt + key_row, 2 * i + half)];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            if (i < 6) {
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) kf[(i + 2) % 3][tt] = keys[buf][cq_key_at(32 * tt + key_row, 2 * (i + 2) + half)];
            }
            x[0] = mfma_bf16(as_bf16x8(kf[i % 3][0]), as_bf16x8(q[i]), x[0]);
            x[1] = mfma_bf16(as_bf16x8(kf[i % 3][1]), as_bf16x8(q[i]), x[1]);
            if (PIECES == 2 || i % 2 == 0) store(buf ^ 1, PIECES == 2 ? i : i / 2);  // (behind the last block: what no one reads)
        }
        __builtin_amdgcn_sched_barrier(0);
        const float kf_scale = ks, vf_scale = vs;
        ks = ks_next;
        vs = vs_next;
        if (b + 2 < whole) load(b + 2);
        float unit = 1.0f;
        if (!(vf_scale <= 2.0f * smax)) {  // up to twice the unit's scale is in fp16's range too
            unit = smax / vf_scale;        // NaN: so become the outputs of the rows that see the block, but not their sums
            if (vf_scale == vf_scale) {
                smax = vf_scale;
                to_unit = DQ_P_SCALE / smax;
            }
        }
        // a block of zeros may have any scale: its scores or its values are zeros all the same
        float shift = vf_scale > 0.0f ? __builtin_amdgcn_logf(vf_scale * to_unit) : 0.0f;
        // Weights under 2^-25 of a unit are 0 in fp16 already; further down their fp32 sum would go the same way.
        if (shift < CQ_SHIFT_LEAST) shift = CQ_SHIFT_LEAST;
        float f = (kf_scale == 0.0f ? 1.0f : kf_scale) * a.scale_log2;
        ready(x, b, f, unit);
        const float base = (m == -INFINITY ? 0.0f : m) - shift;
        float sum = 0.0f;
        uint4 vf[3];
#pragma unroll
        for (int i = 0; i < 2; ++i) vf[i] = values[buf][cq_value_at(32 * i + col, half)];
        float w[8];
        weigh(x, 0, 0, 8, f, base, sum, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f16x8 p;
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = (_Float16)w[j];
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) {
                const int n = 4 * i + dt;
                __builtin_amdgcn_sched_barrier(0);
                if (n < 14) vf[(n + 2) % 3] = values[buf][cq_value_at(32 * ((n + 2) & 3) + col, 2 * ((n + 2) >> 2) + half)];
                o[dt] = mfma_f16(__builtin_bit_cast(f16x8, vf[n % 3]), p, o[dt]);
                if (i < 3) weigh(x, i + 1, 2 * dt, 2 * dt + 2, f, base, sum, w);
            }
        }
        l = fmaf(sum, __builtin_amdgcn_exp2f(-shift), l);
        __syncthreads();
    };
    for (int b = b0; b < whole; b += 2) {
        step(b, std::integral_constant<int, 0>{});
        if (b + 1 < whole) step(b + 1, std::integral_constant<int, 1>{});
    }
    if (has_tail) {
        // bf16 rows as they are; weights in two bf16 terms
        const size_t at = a.c.tail_at(seq, h);
        const int live = s.end % Q8_BLOCK;
        int* const broken_from = reinterpret_cast<int*>(values[1]);  // [128]; no one reads that buffer any more
        uint4 vt[2 * PIECES];
#pragma unroll
        for (int i = 0; i < 2 * PIECES; ++i) {
            const int n = tid + THREADS * i;
            keys[0][cq_key_at(n >> 4, n & 15)] = load_u4(a.c.kt + at + n * 8);
            vt[i] = load_u4(a.c.vt + at + n * 8);
        }
#pragma unroll
        for (int i = 0; i < 2 * PIECES; ++i) {
            const int n = tid + THREADS * i;
            uint4 v = vt[i];
            uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // nothing that lies behind the last token
                if ((n & 7) * 8 + 2 * e >= live) w[e] = 0u;
                else if ((n & 7) * 8 + 2 * e + 1 >= live) w[e] &= 0xffffu;
            }
            // A NaN or an infinity would make the products of rows that do not see its token NaN too (0 times it): they take it
            // for 0, and the first such token of a dim is noted.
            int first = Q8_BLOCK;
            if (__any(max(max(bf16_abs_max(v.x), bf16_abs_max(v.y)), max(bf16_abs_max(v.z), bf16_abs_max(v.w))) >= 0x7f800000u)) {
#pragma unroll
                for (int e = 7; e >= 0; --e)
                    if (bf16_drop_broken(w[e >> 1], e & 1)) first = (n & 7) * 8 + e;
#pragma unroll
                for (int off = 1; off < 8; off <<= 1) first = min(first, __shfl_xor(first, off));  // the dim's 8 lanes
            }
            if ((n & 7) == 0) broken_from[n >> 3] = first;
            values[0][cq_value_at(n >> 3, n & 7)] = v;
        }
        __syncthreads();
        if (tail_b * Q8_BLOCK <= wave_last) {
            // the values as they are: in the blocks' unit, which they may be any number of times, products could leave fp32's range
#pragma unroll
            for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                for (int j = 0; j < 16; ++j) o[dt][j] *= own * (1.0f / DQ_P_SCALE);
            own = smax = DQ_P_SCALE;
            f32x16 x[2];
            scores(0, x);
            float f = a.scale_log2;
            ready(x, tail_b, f, 1.0f);
            if (__any(min(broken_from[lane], broken_from[lane + 64]) < Q8_BLOCK)) {
                const int mine = last - tail_b * Q8_BLOCK;
#pragma unroll
                for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (broken_from[32 * dt + 8 * (j >> 2) + 4 * half + (j & 3)] <= mine) o[dt][j] = __uint_as_float(0x7fc00000u);
            }
            const float base = m == -INFINITY ? 0.0f : m;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float w[8];
                weigh(x, i, 0, 8, f, base, sum, w);
                bf16x8 ph, pl;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    ph[j] = (__bf16)w[j];
                    pl[j] = (__bf16)(w[j] - (float)ph[j]);
                }
#pragma unroll
                for (int dt = 0; dt < 4; ++dt) {
                    const bf16x8 v = as_bf16x8(values[0][cq_value_at(32 * dt + col, 2 * i + half)]);
                    o[dt] = mfma_bf16(v, ph, o[dt]);
                    o[dt] = mfma_bf16(v, pl, o[dt]);
                }
            }
            l += sum;
        }
    }
    l = xor_sum<32>(l);
    // a lane's outputs: dims 32 dt + 8 (j / 4) + 4 half + j % 4 of its row; rows past the count are zeros
    if (row >= (int)a.n * group) return;
    if (row >= rows) {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) o[i][j] = 0.0f;
    }
    const float unit = own * (1.0f / DQ_P_SCALE);
    if (a.splits == 1) {
        const float inv = l == 0.0f ? 0.0f : unit / l;
        uint16_t* to = a.out + (((size_t)seq * a.n + t) * a.nh + h * group + g) * Q8_D + 4 * half;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<uint2*>(to + 32 * dt + 8 * j) =
                    make_uint2(pack_bf16x2(o[dt][4 * j] * inv, o[dt][4 * j + 1] * inv),
                               pack_bf16x2(o[dt][4 * j + 2] * inv, o[dt][4 * j + 3] * inv));
        if (a.lse && half == 0) a.lse[head_row + row] = m + log2f(l);
        return;
    }
    const size_t part = (size_t)split * a.n_seq * a.c.nk * a.n * group + head_row + row;
    float* to = a.part_o + part * Q8_D + 4 * half;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *reinterpret_cast<f32x4*>(to + 32 * dt + 8 * j) = f32x4{o[dt][4 * j] * unit, o[dt][4 * j + 1] * unit,
                                                                    o[dt][4 * j + 2] * unit, o[dt][4 * j + 3] * unit};
    if (half == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * part) = make_float2(m, l);
}

// A row's parts joined: 8 rows a thread block, 32 lanes a row.  Bound by memory: 12 us for the 2 parts of 4 x 512 x 16 rows.
__global__ __launch_bounds__(256) void attn_chunk_q8_merge_kernel(const ChunkQ8Args a) {
    const uint64_t all = (uint64_t)a.n_seq * a.c.nk * a.n * a.group;
    const uint64_t at = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (at >= all) return;
    const int d = (threadIdx.x & 31) * 4;
    const uint32_t row = (uint32_t)(at % ((uint64_t)a.n * a.group));
    const uint64_t head = at / ((uint64_t)a.n * a.group);
    const uint32_t h = (uint32_t)(head % a.c.nk), seq = (uint32_t)(head / a.c.nk);
    const uint32_t t = row / a.group, g = row % a.group;
    constexpr uint32_t BATCH = 8;  // parts in flight
    float M = -INFINITY, L = 0.0f;
    f32x4 sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t i0 = 0; i0 < a.splits; i0 += BATCH) {
        float2 ml[BATCH];
        f32x4 part[BATCH];
#pragma unroll
        for (uint32_t e = 0; e < BATCH; ++e) {
            const uint64_t i = (i0 + e < a.splits ? i0 + e : i0) * all + at;
            ml[e] = *reinterpret_cast<const float2*>(a.part_ml + 2 * i);
            part[e] = *reinterpret_cast<const f32x4*>(a.part_o + i * Q8_D + d);
        }
#pragma unroll
        for (uint32_t e = 0; e < BATCH; ++e) {
            if (i0 + e >= a.splits) ml[e].x = -INFINITY;
            const float now = fmaxf(M, ml[e].x), base = now == -INFINITY ? 0.0f : now;
            const float keep = __builtin_amdgcn_exp2f(M - base), f = __builtin_amdgcn_exp2f(ml[e].x - base);
            L = fmaf(L, keep, f * ml[e].y);
            sum = sum * keep + part[e] * f;
            M = now;
        }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    *reinterpret_cast<uint2*>(a.out + (((size_t)seq * a.n + t) * a.nh + h * a.group + g) * Q8_D + d) =
        make_uint2(pack_bf16x2(sum[0] * inv, sum[1] * inv), pack_bf16x2(sum[2] * inv, sum[3] * inv));
    if (a.lse && d == 0) a.lse[at] = M + log2f(L);
}

// weights_out[token] = weights_in (0 for a new token) + sum of exp2(score - lse) over the rows of the KV head.  A wave takes
// 64 tokens, one cache block, as the operand that stays in registers; the rows' queries pass through LDS, 64 at a time and
// the next 64 on their way, the same for the thread block's four waves.  Sums are in a fixed order.  Bound by the products and
// the three vector instructions a pair (scale, exponential, sum), which overlap little: 80 to 87 us for 4 x 512 tokens of 16 / 8
// heads at 7000 (61 GFLOP, 238 million pairs).  Products of one half with the other half's exponentials between them took 5 %
// more: with both halves' scores the registers do not hold the keys.
__global__ __launch_bounds__(256, 2) void attn_chunk_q8_weights_kernel(const ChunkQ8Args a) {
    constexpr int STEP = 64;  // rows
    __shared__ __align__(16) uint4 queries[2][STEP * 16];
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t h = blockIdx.x % a.c.nk;
    uint32_t rest = blockIdx.x / a.c.nk;
    const uint32_t split = rest % a.w_splits;
    rest /= a.w_splits;
    const uint32_t per = (a.c.nb + 3) / 4;
    const uint32_t seq = rest / per;
    const int first_b = (int)(rest % per) * 4, b = first_b + wave;
    const Q8Span s = q8_span(a.lengths, a.counts, seq, a.n, a.c.nb);
    if (first_b * Q8_BLOCK >= s.end) return;
    const int len = min(a.lengths[seq], (int)(a.c.nb * Q8_BLOCK));
    int count = a.counts ? a.counts[seq] : (int)a.n;
    count = len < 0 || count < 0 ? 0 : (count < (int)a.n ? count : (int)a.n);
    const int group = (int)a.group, rows = count * group;
    const bool mine = b * Q8_BLOCK < s.end;
    const bool in_tail = s.end % Q8_BLOCK && b == s.end / Q8_BLOCK;
    // from the first row that sees the thread block's first token, a share of the steps
    const int t_first = first_b * Q8_BLOCK - len;
    const int step0 = t_first > 0 ? (int)((int64_t)t_first * group / STEP) : 0, steps = (rows + STEP - 1) / STEP - step0;
    const int row_first = (step0 + (int)((int64_t)steps * split / a.w_splits)) * STEP;
    const int row_end = min(rows, (step0 + (int)((int64_t)steps * (split + 1) / a.w_splits)) * STEP);
    uint4 next[4];
    float sub[2], sub_next[2];  // rows lane % 32 and 32 + lane % 32; one that is not there weighs nothing
    const float* lse = a.lse + ((size_t)seq * a.c.nk + h) * a.n * group;
    // 16 bytes of a row: piece tid % 16 of rows tid / 16, + 16 ..; their heads and places in q, from STEP rows to the next
    // without a division
    int g_at[4];
    uint32_t q_at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = row_first + (tid >> 4) + 16 * i, t = row / group;
        g_at[i] = row - t * group;
        q_at[i] = (uint32_t)t * a.nh + (uint32_t)g_at[i];
    }
    // (in the place of a row that is not there the last one, which sees every token: a NaN of it is in every sum already)
    const uint32_t q_last = rows > 0 ? (uint32_t)((rows - 1) / group) * a.nh + (uint32_t)((rows - 1) % group) : 0u;
    const int g_step = STEP % group;
    const uint32_t q_step = (uint32_t)(STEP / group) * a.nh + (uint32_t)g_step, q_wrap = a.nh - a.group;
    const uint16_t* const q_from = a.q + ((size_t)seq * a.n * a.nh + h * group) * Q8_D + 8 * (tid & 15);
    auto load = [&](int row0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            next[i] = load_u4(q_from + (size_t)(row0 + (tid >> 4) + 16 * i < rows ? q_at[i] : q_last) * Q8_D);
            g_at[i] += g_step;
            q_at[i] += q_step + (g_at[i] >= group ? q_wrap : 0u);
            g_at[i] -= g_at[i] >= group ? group : 0;
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = row0 + 32 * r + col;
            sub_next[r] = row < rows ? lse[row] : INFINITY;
        }
    };
    auto store = [&](int buf) {
#pragma unroll
        for (int i = 0; i < 4; ++i) queries[buf][cq_key_at((tid >> 4) + 16 * i, tid & 15)] = next[i];
    };
    load(row_first);
    bf16x8 k[2][8];
    float f = a.scale_log2;
    if (in_tail) {
        const uint16_t* p = a.c.kt + a.c.tail_at(seq, h) + 8 * half;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int i = 0; i < 8; ++i) k[tt][i] = as_bf16x8(load_u4(p + (32 * tt + col) * Q8_D + 16 * i));
    } else {
        const int from = mine ? b : first_b;  // (a wave without a block helps with the queries)
        const int8_t* p = a.c.k + a.c.block_at(seq, (uint32_t)from, h) + 8 * half;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint2 w = *reinterpret_cast<const uint2*>(p + (32 * tt + col) * Q8_D + 16 * i);
                k[tt][i] = as_bf16x8(codes_bf16x8(w.x, w.y));
            }
        f *= a.c.ks[a.c.scale_at(seq, (uint32_t)from, h)];
    }
    float sum[2][16];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int j = 0; j < 16; ++j) sum[tt][j] = 0.0f;
    store(0);
    __syncthreads();
    for (int row0 = row_first; row0 < row_end; row0 += STEP) {
        const int buf = (row0 - row_first) / STEP & 1;
        sub[0] = sub_next[0];
        sub[1] = sub_next[1];
        if (row0 + STEP < row_end) load(row0 + STEP);
        if (mine) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = row0 + 32 * r + col;
                f32x16 x[2];
#pragma unroll
                for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                    for (int j = 0; j < 16; ++j) x[tt][j] = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const bf16x8 q = as_bf16x8(queries[buf][cq_key_at(32 * r + col, 2 * i + half)]);
                    x[0] = mfma_bf16(k[0][i], q, x[0]);
                    x[1] = mfma_bf16(k[1][i], q, x[1]);
                }
                if (b * Q8_BLOCK + Q8_BLOCK - 1 > len + (row0 + 32 * r) / group) {
                    const int seen = len + row / group - b * Q8_BLOCK - 4 * half;  // tokens 32 tt + 8 (j / 4) + 4 half + j % 4
#pragma unroll
                    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const float p = __builtin_amdgcn_exp2f(fmaf(x[tt][j], f, -sub[r]));
                            sum[tt][j] += row >= rows || 32 * tt + 8 * (j >> 2) + (j & 3) > seen ? 0.0f : p;
                        }
                } else {
#pragma unroll
                    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                        for (int j = 0; j < 16; ++j) sum[tt][j] += __builtin_amdgcn_exp2f(fmaf(x[tt][j], f, -sub[r]));
                }
            }
        }
        if (row0 + STEP < row_end) store(buf ^ 1);
        __syncthreads();
    }
    if (!mine) return;
    // over the 32 rows that the lanes of a half hold; a lane writes one token
    const int p = b * Q8_BLOCK + 32 * (col >> 4) + 8 * (col >> 2 & 3) + 4 * half + (col & 3);
    const size_t all = (size_t)a.n_seq * a.c.nk * a.c.nb * Q8_BLOCK, at = ((size_t)seq * a.c.nk + h) * a.c.nb * Q8_BLOCK + p;
    const float before = a.w_splits == 1 && p < s.len ? a.w_in[at] : 0.0f;
    float total = 0.0f;
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            float v = sum[tt][j];
            v += dpp_f32<0xB1>(v);
            v += dpp_f32<0x4E>(v);
            v += dpp_f32<0x141>(v);
            v += dpp_f32<0x140>(v);
            v = xor_sum<16>(v);
            if (col == 16 * tt + j) total = v;
        }
    if (p >= s.end) return;
    if (a.w_splits == 1)
        a.w_out[at] = before + total;
    else
        a.w_part[split * all + at] = total;
}

// The shares added up, in their order: 4 tokens a thread.
__global__ __launch_bounds__(256) void attn_chunk_q8_weights_merge_kernel(const ChunkQ8Args a) {
    const uint32_t cap = a.c.nb * Q8_BLOCK;
    const size_t all = (size_t)a.n_seq * a.c.nk * cap, at = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (at >= all) return;
    const uint32_t seq = (uint32_t)(at / ((size_t)a.c.nk * cap));
    const int p = (int)(at % cap);
    const Q8Span s = q8_span(a.lengths, a.counts, seq, a.n, a.c.nb);
    if (p >= s.end) return;
    f32x4 sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t i = 0; i < a.w_splits; ++i) sum += *reinterpret_cast<const f32x4*>(a.w_part + i * all + at);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (p + j < s.end) a.w_out[at + j] = (p + j < s.len ? a.w_in[at + j] : 0.0f) + sum[j];
}

// ---------------------------------------------------------------------------------------------------- few rows --
//
// Up to 32 rows of a KV head (a few drafted tokens): bound by memory like a single token, and read like one, in units of
// blocks that a wave takes whole; the rows are the columns of one or two 16 x 16 x 32 products, each with its own last
// token.  Their queries are bf16 already, so fp16 holds them in one term: elements down to 2^-30 of the largest exactly.  A
// second kernel joins a sequence's units.
// Measured (32 / 8 heads): 2 x 5 tokens at 4000 12.8 us and 4.6 the join (17.1 both, 27 with weights), 1 at 8000 and its join 12.2.
template <int CT>
__global__ __launch_bounds__(DQ_WAVES * 64, 2) void attn_rows_q8_kernel(const ChunkQ8Args a) {
    constexpr int COLS = 16 * CT;
    // the queries (fp16 by q_to_fp16, and bf16 as they came), then the waves' outputs
    __shared__ __align__(16) float room[DQ_WAVES * COLS * DQ_ROW];
    __shared__ float qf[COLS], wml[DQ_WAVES][COLS][2];
    _Float16* const qs = reinterpret_cast<_Float16*>(room);
    uint16_t* const qb = reinterpret_cast<uint16_t*>(room) + COLS * DQ_QROW;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t h = blockIdx.x % a.c.nk, unit = blockIdx.x / a.c.nk;
    DecodeUnit u;
    if (!dq_find({a.lengths, a.counts, a.n, a.n_seq, a.c.nb, a.c.nk}, unit, false, u)) return;
    const int group = (int)a.group, rows = (int)a.n * group;
    const Q8Span s = q8_span(a.lengths, a.counts, u.seq, a.n, a.c.nb);
    int count = a.counts ? a.counts[u.seq] : (int)a.n;
    count = u.blocks == 0 ? 0 : (count < (int)a.n ? count : (int)a.n);
    const int b0 = u.part * u.chunk;
    const int b1 = b0 + u.chunk < u.blocks ? b0 + u.chunk : u.blocks;
    const int c = lane & 15, g4 = lane >> 4;
    const int tail_b = s.end % Q8_BLOCK ? s.end / Q8_BLOCK : -1;
    const bool has_tail = tail_b >= b0 && tail_b < b1;
    const int len = min(u.len, (int)(a.c.nb * Q8_BLOCK));
    auto row_at = [&](int row) {  // row t * group + g in q and out
        return (((size_t)u.seq * a.n + row / group) * a.nh + h * group + row % group) * Q8_D;
    };
    uint32_t qw[COLS / DQ_WAVES];
#pragma unroll
    for (int i = 0; i < COLS / DQ_WAVES; ++i) {
        const int row = wave + DQ_WAVES * i;
        qw[i] = row < count * group ? reinterpret_cast<const uint32_t*>(a.q + row_at(row))[lane] : 0u;
    }
    float smax = 0.0f;
    for (int i = b0 + wave + DQ_WAVES * lane; i < b1; i += DQ_WAVES * 64)
        if (i != tail_b) smax = fmaxf(smax, a.c.vs[a.c.scale_at(u.seq, (uint32_t)i, h)]);
    const int krow = ((c >> 2) * 16 + (c & 3)) * Q8_D + g4 * 16;
    const int vrow = c * Q8_BLOCK + g4 * 16;
    uint4 kr[8], vr[8];
    float ks = 0.0f, vs = 0.0f;
    auto load_k = [&](int b) {
        const int8_t* p = a.c.k + a.c.block_at(u.seq, (uint32_t)b, h) + krow;
#pragma unroll
        for (int n = 0; n < 8; ++n) kr[n] = load_nt_u4(p + (n >> 1) * 4 * Q8_D + (n & 1) * 64);
        ks = a.c.ks[a.c.scale_at(u.seq, (uint32_t)b, h)];
    };
    auto load_v = [&](int b) {
        const int8_t* p = a.c.v + a.c.block_at(u.seq, (uint32_t)b, h) + vrow;
#pragma unroll
        for (int n = 0; n < 8; ++n) vr[n] = load_nt_u4(p + n * 16 * Q8_BLOCK);
        vs = a.c.vs[a.c.scale_at(u.seq, (uint32_t)b, h)];
    };
    int b = b0 + wave;
    if (b < b1 && b != tail_b) {
        load_k(b);
        load_v(b);
    }
#pragma unroll
    for (int i = 0; i < COLS / DQ_WAVES; ++i) {  // dims 2 lane, 2 lane + 1
        const int row = wave + DQ_WAVES * i;
        const float x = __uint_as_float(qw[i] << 16), y = __uint_as_float(qw[i] & 0xffff0000u);
        const uint32_t e = q_exponent(wave_max(fmaxf(fabsf(x), fabsf(y))));
        const float down = q_to_fp16(e);
        const f16x2_t two = {(_Float16)(x * down), (_Float16)(y * down)};
        *reinterpret_cast<f16x2_t*>(qs + row * DQ_QROW + 2 * lane) = two;
        *reinterpret_cast<uint32_t*>(qb + row * DQ_QROW + 2 * lane) = qw[i];
        if (lane == 0) qf[row] = q_from_fp16(e) * a.scale_log2;
    }
    __syncthreads();
    smax = wave_max(smax);
    float m[CT], l[CT], qfac[CT];
    int last[CT];  // the last token that the column sees
    f32x4 o[CT][8];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        const int row = 16 * ct + c;
        m[ct] = -INFINITY;
        l[ct] = 0.0f;
        qfac[ct] = qf[row];
        last[ct] = row < count * group ? min(len + row / group, s.end - 1) : -1;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) o[ct][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const int first = count > 0 ? min(len, s.end - 1) : -1;  // what every row sees

    // scores of key tiles t0 .. of a block -> weights; tokens 16 g4 + 4 t + i
    auto soften = [&](auto& x, int ct, int t0, float f, int b) {
        constexpr int N = sizeof(x) / sizeof(x[0]);
        const int mine = last[ct] - b * Q8_BLOCK;
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[t][i] = 16 * g4 + 4 * (t0 + t) + i > mine ? -INFINITY : x[t][i] * f;
                top = fmaxf(top, x[t][i]);
            }
        top = fmaxf(m[ct], xor_max<32>(xor_max<16>(top)));
        const float base = top == -INFINITY ? 0.0f : top;
        const float keep = __builtin_amdgcn_exp2f(m[ct] - base);
        float sum = 0.0f;
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[t][i] = __builtin_amdgcn_exp2f(x[t][i] - base);
                sum += x[t][i];
            }
        l[ct] = fmaf(l[ct], keep, sum);
        m[ct] = top;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) o[ct][dt] *= keep;
    };

    for (; b < b1 && b != tail_b; b += DQ_WAVES) {
        f32x4 x[CT][4];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int t = 0; t < 4; ++t) x[ct][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            f16x8 q[CT][2];
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    q[ct][i] = *reinterpret_cast<const f16x8*>(qs + (16 * ct + c) * DQ_QROW + 64 * j + 16 * g4 + 8 * i);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const uint4 kk = kr[2 * t + j];
                const f16x8 k0 = codes_f16x8(kk.x, kk.y), k1 = codes_f16x8(kk.z, kk.w);
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    x[ct][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, q[ct][0], x[ct][t], 0, 0, 0);
                    x[ct][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, q[ct][1], x[ct][t], 0, 0, 0);
                }
            }
        }
        const float fk = ks;
        const int next = b + DQ_WAVES;
        const bool more = next < b1 && next != tail_b;
        if (more) load_k(next);
        const float fv = vs * (DQ_P_SCALE / (smax > 0.0f ? smax : 1.0f));
        const bool edge = b * Q8_BLOCK + Q8_BLOCK - 1 > first;
        f16x8 p[CT][2];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            soften(x[ct], ct, 0, fk * qfac[ct], b);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float w = x[ct][e / 4][e % 4] * fv;
                if (edge && x[ct][e / 4][e % 4] == 0.0f) w = 0.0f;  // (where the block is broken and the row does not see it)
                p[ct][e / 8][e % 8] = (_Float16)w;
            }
        }
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
            const f16x8 v0 = codes_f16x8(vr[dt].x, vr[dt].y), v1 = codes_f16x8(vr[dt].z, vr[dt].w);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                o[ct][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, p[ct][0], o[ct][dt], 0, 0, 0);
                o[ct][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, p[ct][1], o[ct][dt], 0, 0, 0);
            }
        }
        if (more) load_v(next);
    }
    float unscale = (smax > 0.0f ? smax : 1.0f) * (1.0f / DQ_P_SCALE);
    if (has_tail) {  // tile `wave` of the unfinished block, as in the kernel of one token
        const size_t tail = a.c.tail_at(u.seq, h);
        const int ahead = s.end % Q8_BLOCK - 16 * g4 - 4 * wave;  // of a lane's 4 value tokens, those that there are
        const uint32_t live0 = ahead <= 0 ? 0u : ahead == 1 ? 0xffffu : 0xffffffffu;
        const uint32_t live1 = ahead <= 2 ? 0u : ahead == 3 ? 0xffffu : 0xffffffffu;
        uint4 tk[4];
        uint2 tv[8];
#pragma unroll
        for (int n = 0; n < 4; ++n) tk[n] = load_u4(a.c.kt + tail + krow + wave * 4 * Q8_D + 64 * (n >> 1) + 8 * (n & 1));
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            tv[n] = *reinterpret_cast<const uint2*>(a.c.vt + tail + vrow + n * 16 * Q8_BLOCK + 4 * wave);
            tv[n] = make_uint2(tv[n].x & live0, tv[n].y & live1);
        }
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            f32x4 x[1] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
            for (int n = 0; n < 4; ++n)
                x[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    as_bf16x8(tk[n]),
                    as_bf16x8(*reinterpret_cast<const uint4*>(qb + (16 * ct + c) * DQ_QROW + 64 * (n >> 1) + 16 * g4 + 8 * (n & 1))),
                    x[0], 0, 0, 0);
            soften(x, ct, wave, a.scale_log2, tail_b);
            // A NaN or an infinity would make the outputs of rows that do not see its token NaN too (0 times it): it is taken for 0,
            // and the rows that see it become NaN in its dim.
            uint32_t largest = 0;  // (here, where the values have come)
#pragma unroll
            for (int n = 0; n < 8; ++n) largest = max(largest, max(bf16_abs_max(tv[n].x), bf16_abs_max(tv[n].y)));
            if (ct == 0 && __any(largest >= 0x7f800000u)) {
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    int first = Q8_BLOCK;  // of dim 16 n + c
#pragma unroll
                    for (int e = 3; e >= 0; --e)
                        if (bf16_drop_broken(e < 2 ? tv[n].x : tv[n].y, e & 1)) first = 16 * g4 + 4 * wave + e;
                    first = min(first, __shfl_xor(first, 16));
                    first = min(first, __shfl_xor(first, 32));
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int from = __shfl(first, 4 * g4 + i);
#pragma unroll
                        for (int cc = 0; cc < CT; ++cc)
                            if (from <= last[cc] - tail_b * Q8_BLOCK) o[cc][n][i] = __uint_as_float(0x7fc00000u);
                    }
                }
            }
            bf16x4 ph, pl;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                ph[e] = (__bf16)x[0][e];
                pl[e] = (__bf16)(x[0][e] - (float)ph[e]);
            }
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) o[ct][dt] *= unscale;
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) {
                const t2h_v4i16 v = __builtin_bit_cast(t2h_v4i16, tv[dt]);
                o[ct][dt] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(v, __builtin_bit_cast(t2h_v4i16, ph), o[ct][dt], 0, 0, 0);
                o[ct][dt] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(v, __builtin_bit_cast(t2h_v4i16, pl), o[ct][dt], 0, 0, 0);
            }
        }
        unscale = 1.0f;
    }

    // the waves' states joined
    __syncthreads();
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        const float sum = xor_sum<32>(xor_sum<16>(l[ct]));
        const int row = 16 * ct + c;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt)
            *reinterpret_cast<f32x4*>(room + (wave * COLS + row) * DQ_ROW + 16 * dt + 4 * g4) = o[ct][dt] * unscale;
        if (g4 == 0) {
            wml[wave][row][0] = m[ct];
            wml[wave][row][1] = sum;
        }
    }
    __syncthreads();
    const int waves = !has_tail && b1 - b0 < DQ_WAVES ? b1 - b0 : DQ_WAVES;
    for (int i = tid; i < rows * (Q8_D / 4); i += DQ_WAVES * 64) {
        const int row = i / (Q8_D / 4), d = i % (Q8_D / 4) * 4;
        float M = -INFINITY, L = 0.0f;
        for (int w = 0; w < waves; ++w) M = fmaxf(M, wml[w][row][0]);
        const float base = M == -INFINITY ? 0.0f : M;
        f32x4 sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int w = 0; w < waves; ++w) {
            const float f = __builtin_amdgcn_exp2f(wml[w][row][0] - base);
            L = fmaf(f, wml[w][row][1], L);
            sum += *reinterpret_cast<const f32x4*>(room + (w * COLS + row) * DQ_ROW + d) * f;
        }
        if (u.count == 1) {
            if (L == 0.0f) sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};  // a row past the count: 0 times a broken block's scale is NaN
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            *reinterpret_cast<uint2*>(a.out + row_at(row) + d) =
                make_uint2(pack_bf16x2(sum[0] * inv, sum[1] * inv), pack_bf16x2(sum[2] * inv, sum[3] * inv));
            if (a.lse && d == 0) a.lse[((size_t)u.seq * a.c.nk + h) * rows + row] = M + log2f(L);
        } else {
            const size_t part = ((size_t)(u.first + (uint32_t)u.part) * a.c.nk + h) * rows + row;
            *reinterpret_cast<f32x4*>(a.part_o + part * Q8_D + d) = sum;
            if (d == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * part) = make_float2(M, L);
        }
    }
}

// The units of a (sequence, KV head) joined, 8 rows a thread block, 32 lanes a row: 5 us for 2 x 5 tokens at 4000, latency.
__global__ __launch_bounds__(256) void attn_rows_q8_merge_kernel(const ChunkQ8Args a) {
    const uint32_t rows = a.n * a.group, per = (rows + 7) / 8;
    const uint32_t h = blockIdx.x % a.c.nk, rest = blockIdx.x / a.c.nk;
    const uint32_t row = rest % per * 8 + (threadIdx.x >> 5), seq = rest / per;
    DecodeUnit u;
    dq_find({a.lengths, a.counts, a.n, a.n_seq, a.c.nb, a.c.nk}, seq, true, u);
    if (u.count <= 1 || row >= rows) return;
    const int d = (threadIdx.x & 31) * 4;
    constexpr uint32_t BATCH = 16;  // parts in flight
    float M = -INFINITY, L = 0.0f;
    f32x4 sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t i0 = 0; i0 < u.count; i0 += BATCH) {
        float2 ml[BATCH];
        f32x4 part[BATCH];
#pragma unroll
        for (uint32_t e = 0; e < BATCH; ++e) {
            const size_t at = ((size_t)(u.first + (i0 + e < u.count ? i0 + e : i0)) * a.c.nk + h) * rows + row;
            ml[e] = *reinterpret_cast<const float2*>(a.part_ml + 2 * at);
            part[e] = *reinterpret_cast<const f32x4*>(a.part_o + at * Q8_D + d);
        }
#pragma unroll
        for (uint32_t e = 0; e < BATCH; ++e) {
            if (i0 + e >= u.count) ml[e].x = -INFINITY;
            const float now = fmaxf(M, ml[e].x), base = now == -INFINITY ? 0.0f : now;
            const float keep = __builtin_amdgcn_exp2f(M - base), f = __builtin_amdgcn_exp2f(ml[e].x - base);
            L = fmaf(L, keep, f * ml[e].y);
            sum = sum * keep + part[e] * f;
            M = now;
        }
    }
    if (L == 0.0f) sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};  // (as above)
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    const uint32_t t = row / a.group, g = row % a.group;
    *reinterpret_cast<uint2*>(a.out + (((size_t)seq * a.n + t) * a.nh + h * a.group + g) * Q8_D + d) =
        make_uint2(pack_bf16x2(sum[0] * inv, sum[1] * inv), pack_bf16x2(sum[2] * inv, sum[3] * inv));
    if (a.lse && d == 0) a.lse[((size_t)seq * a.c.nk + h) * rows + row] = M + log2f(L);
}

// Whether a KV head's rows are columns of the products of single tokens: up to two tiles of 16 (three would not leave the
// registers a block's codes).  Measured against the kernel of 32-row waves (us a call, 32 / 8 heads): 1 token at 8000 12.2, 16.9;
// 8 at 8000 17.1, 17.9; 4 x 8 at 16000 37, 42; 16 x 5 at 4000 39, 42; 16 x 8 at 8000 62, 78; 32 x 5 at 8000 115, 161; but 5 at
// 1000 12.4, 12.1; 2 x 5 at 4000 17.1, 15.4; 2 x 8 at 4000 17.9, 15.5; 8 x 5 at 2000 21.0, 19.1, where the join's launch is 5 us.
static bool cq_few(uint32_t n, uint32_t nh, uint32_t nk) { return (uint64_t)n * (nh / nk) <= 32; }

// Waves a thread block: 8 share a block's conversion to 16 bits where that leaves two thread blocks for every CU.  Measured (us of
// 8 and of 4, 32 / 8 heads): 16000 tokens 1958, 2068; 8 x 2048 318, 318; 1901, 240 and 480 thread blocks, 56, 47; 1500 45, 38; at
// the border, 512 thread blocks, where those of 8 are one uneven round: 4096 tokens 169, 159; 2 x 2048 94, 87.
static uint32_t cq_waves(uint32_t n, uint32_t n_seq, uint32_t nh, uint32_t nk) {
    return ((uint64_t)n * (nh / nk) + 255) / 256 * n_seq * nk >= CQ_WIDE_GRID ? 8 : 4;
}

// Thread blocks that share a tile's keys, in a full cache each with 4 blocks of keys or more of those that a row of the chunk's
// middle sees: one a CU where there are not as many tiles; two a CU where that leaves each 8 blocks or more, 32 where it is what
// brings the join with it.  Measured (us, 32 / 8 heads unless named; one a CU, two): 100 tokens at 3000 24, 26; 64 at 8000 25, 29;
// 256 at 16000 89, 85; 512 at 8000 95, 87; and where one a CU is whole: 1000 at 0 26, 34; 2 x 512 at 2000 54, 59, at 4000 92, 93;
// 4 x 512 of 16 / 8 heads at 7000 147, 144; 2048 of 16 / 8 at 2048 81, 73.
// What the cache holds is not known here, its capacity stands for it: 100 tokens at 0 take 9 us at a capacity of 192 and 22 at 8192,
// where the keys have 16 parts of which 14 are empty.
static uint32_t cq_splits(uint32_t n, uint32_t n_seq, uint32_t nh, uint32_t nk, uint32_t nb) {
    const uint64_t rows = 32 * cq_waves(n, n_seq, nh, nk), tiles = ((uint64_t)n * (nh / nk) + rows - 1) / rows;
    const uint64_t grid = tiles * n_seq * nk, skip = n / (2 * Q8_BLOCK), most = nb > skip ? (nb - skip) / 4 : 0;
    if (grid == 0) return 1;
    const uint64_t one = 256 / grid, two = 512 / grid;
    const uint64_t want = two && nb / two >= (one > 1 ? 8 : 32) ? two : one;
    return (uint32_t)(want < most ? (want ? want : 1) : (most ? most : 1));
}

// Thread blocks that share the rows of a chunk's weights where there are few tokens: two rounds of the chip (for a causal
// chunk's share of the pairs) of 512 rows each or more, or one round of 128 or more.  Measured (us, 32 / 8 heads but for the
// last two): 2048 tokens at 0: 38 in rounds of 1024 thread blocks, 48 of 512, 196 unshared; 142 tokens at 4: 14 of 128 rows, 18
// of 256, 24 unshared; 2 x 300 of 40 / 8 at 3000: 37 of 512 rows in two rounds, 41 of 256; 300 of 16 / 2 at 2000: 18 of 128 rows
// in one round, 22 of 64, 26 of 512.  Here too the capacity stands for what the cache holds: 2048 tokens at 0, with their
// attention, 89 us at a capacity of 2112, 116 at 8192, 159 at 16384 and 243 from 32768 on, where nothing is shared.
static uint32_t cq_weight_splits(uint32_t n, uint32_t n_seq, uint32_t nh, uint32_t nk, uint32_t nb) {
    const uint64_t grid = ((uint64_t)nb + 3) / 4 * n_seq * nk, rows = (uint64_t)n * (nh / nk);
    const uint64_t large = 1024 / grid < rows / 512 ? 1024 / grid : rows / 512;
    const uint64_t small = 512 / grid < rows / 128 ? 512 / grid : rows / 128;
    const uint64_t splits = large > small ? large : small;
    return (uint32_t)(splits ? splits : 1);
}

// fp32 values of a chunk's weights: each row's softmax and the shares
static size_t cq_weight_values(uint32_t n, uint32_t n_seq, uint32_t nh, uint32_t nk, uint32_t s_cap) {
    const uint32_t splits = cq_weight_splits(n, n_seq, nh, nk, s_cap / Q8_BLOCK);
    return (size_t)n_seq * nh * n + (splits > 1 ? (size_t)splits * n_seq * nk * s_cap : 0);
}

}  // namespace t2h

using namespace t2h;

extern "C" size_t t2h_attn_decode_q8_workspace_bytes(uint32_t n_seq, uint32_t nh, uint32_t nk, uint32_t d, uint32_t s_cap,
                                                     int weights) {
    if (n_seq == 0 || nk == 0 || nh == 0 || nh % nk != 0 || nh / nk > Q8_MAX_GROUP || d != (uint32_t)Q8_D || s_cap == 0 ||
        s_cap % Q8_BLOCK != 0)
        return 0;
    const size_t parts = (size_t)dq_units(n_seq, nk, s_cap / Q8_BLOCK) * nh;
    return dq_counters(n_seq, nk) * 4 + (parts * (Q8_D + 2) * 4 + 15) / 16 * 16 + (weights ? (size_t)n_seq * nh * s_cap * 4 : 0);
}

extern "C" int t2h_attn_decode_q8(const float* q, uint64_t q_row, const float* k_new, uint64_t k_row, const float* v_new,
                                  uint64_t v_row, const float* q_norm_w, const float* k_norm_w, float eps, float theta,
                                  const int32_t* lengths, const int32_t* rope_offsets, void* const* cache, uint32_t s_cap,
                                  const float* weights, float* weights_out, void* out, uint32_t n_seq, uint32_t nh,
                                  uint32_t nk, uint32_t d, void* workspace, size_t workspace_bytes, void* stream) {
    DecodeQ8Args a;
    if (!q || !k_new || !v_new || !lengths || !out || !workspace) return T2H_ERR_NULL;
    if ((weights == nullptr) != (weights_out == nullptr) || (q_norm_w == nullptr) != (k_norm_w == nullptr)) return T2H_ERR_NULL;
    if (const int e = q8_cache(cache, s_cap, n_seq, nh, nk, d, a.c)) return e;
    if (q_row < (uint64_t)nh * d || k_row < (uint64_t)nk * d || v_row < (uint64_t)nk * d) return T2H_ERR_SHAPE;
    if (reinterpret_cast<uintptr_t>(out) & 3) return T2H_ERR_ALIGN;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return T2H_ERR_ALIGN;
    if (workspace_bytes < t2h_attn_decode_q8_workspace_bytes(n_seq, nh, nk, d, s_cap, weights != nullptr)) return T2H_ERR_WORKSPACE;
    a.q = q;
    a.k_new = k_new;
    a.v_new = v_new;
    a.q_row = (size_t)q_row;
    a.k_row = (size_t)k_row;
    a.v_row = (size_t)v_row;
    a.q_norm_w = q_norm_w;
    a.k_norm_w = k_norm_w;
    a.lengths = lengths;
    a.offsets = rope_offsets;
    a.w_in = weights;
    a.w_out = weights_out;
    a.out = reinterpret_cast<uint16_t*>(out);
    a.n_seq = n_seq;
    a.nh = nh;
    a.group = nh / nk;
    a.units = dq_units(n_seq, nk, a.c.nb);
    const size_t parts = (size_t)a.units * nh;
    a.done = reinterpret_cast<uint32_t*>(workspace);
    a.part_o = reinterpret_cast<float*>(workspace) + dq_counters(n_seq, nk);
    a.part_ml = a.part_o + parts * Q8_D;
    a.scores = weights ? a.part_o + (parts * (Q8_D + 2) + 3) / 4 * 4 : nullptr;
    a.eps = eps;
    a.scale_log2 = 1.4426950408889634f / sqrtf((float)Q8_D);
    a.rope = theta > 0.0f;
    a.log2_theta = a.rope ? log2((double)theta) : 0.0;
    const uint64_t grid = (uint64_t)a.units * nk;
    const uint64_t segments = ((uint64_t)s_cap + DQ_SEGMENT - 1) / DQ_SEGMENT;
    const uint64_t wgrid = (uint64_t)n_seq * nk * segments;
    if (grid > 0x7fffffffu || wgrid > 0x7fffffffu) return T2H_ERR_SHAPE;
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (!weights) {
        hipLaunchKernelGGL(attn_decode_q8_kernel<false>, dim3((uint32_t)grid), dim3(DQ_WAVES * 64), 0, st, a);
        T2H_LAUNCH_CHECK();
        return T2H_OK;
    }
    hipLaunchKernelGGL(attn_decode_q8_kernel<true>, dim3((uint32_t)grid), dim3(DQ_WAVES * 64), 0, st, a);
    T2H_LAUNCH_CHECK();
    hipLaunchKernelGGL(attn_decode_q8_weights_kernel, dim3((uint32_t)wgrid), dim3(256), 0, st, a);
    T2H_LAUNCH_CHECK();
    return T2H_OK;
}

extern "C" size_t t2h_flash_attn_prefill_q8_workspace_bytes(uint32_t n, uint32_t n_seq, uint32_t nh, uint32_t nk,
                                                            uint32_t s_cap, int weights) {
    if (n_seq == 0 || nk == 0 || nh == 0 || nh % nk != 0 || nh / nk > Q8_MAX_GROUP || s_cap == 0 || s_cap % Q8_BLOCK != 0) return 0;
    const size_t rows = (size_t)n_seq * nh * n;
    const size_t sums = weights ? cq_weight_values(n, n_seq, nh, nk, s_cap) * 4 : 0;
    if (cq_few(n, nh, nk)) return 16 + sums + (size_t)dq_units(n_seq, nk, s_cap / Q8_BLOCK) * nh * n * (Q8_D + 2) * 4;
    const uint32_t splits = cq_splits(n, n_seq, nh, nk, s_cap / Q8_BLOCK);
    return 16 + sums + (splits > 1 ? splits * rows * (Q8_D + 2) * 4 : 0);
}

extern "C" int t2h_flash_attn_prefill_q8(const void* q, void* const* cache, uint32_t s_cap, const int32_t* lengths,
                                         const int32_t* counts, const float* weights, float* weights_out, void* out,
                                         uint32_t n, uint32_t n_seq, uint32_t nh, uint32_t nk, uint32_t d, float scale,
                                         void* workspace, size_t workspace_bytes, void* stream) {
    ChunkQ8Args a;
    if (!lengths || (n && (!q || !out || !workspace))) return T2H_ERR_NULL;
    if ((weights == nullptr) != (weights_out == nullptr)) return T2H_ERR_NULL;
    if (const int e = q8_cache(cache, s_cap, n_seq, nh, nk, d, a.c)) return e;
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15)
        return T2H_ERR_ALIGN;
    if (n && workspace_bytes < t2h_flash_attn_prefill_q8_workspace_bytes(n, n_seq, nh, nk, s_cap, weights != nullptr))
        return T2H_ERR_WORKSPACE;
    a.q = reinterpret_cast<const uint16_t*>(q);
    a.out = reinterpret_cast<uint16_t*>(out);
    a.lengths = lengths;
    a.counts = counts;
    a.w_in = weights;
    a.w_out = weights_out;
    a.n = n;
    a.n_seq = n_seq;
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const uint64_t sums = ((uint64_t)n_seq * nk * s_cap + 1023) / 1024;
    if (sums > 0x7fffffffu) return T2H_ERR_SHAPE;
    if (n == 0) {  // no shares: the cached tokens' weights as they are
        if (weights == weights_out) return T2H_OK;
        a.w_part = nullptr;
        a.w_splits = 0;
        hipLaunchKernelGGL(attn_chunk_q8_weights_merge_kernel, dim3((uint32_t)sums), dim3(256), 0, st, a);
        T2H_LAUNCH_CHECK();
        return T2H_OK;
    }
    a.nh = nh;
    a.group = nh / nk;
    a.scale_log2 = 1.4426950408889634f * (scale > 0.0f ? scale : 1.0f / sqrtf((float)Q8_D));
    const uint64_t rows = (uint64_t)n_seq * nh * n, tile_rows = 32 * cq_waves(n, n_seq, nh, nk),
                   tiles = ((uint64_t)n * a.group + tile_rows - 1) / tile_rows;
    if (rows > 0x3fffffffu) return T2H_ERR_SHAPE;
    const bool few = cq_few(n, nh, nk);
    const uint32_t units = dq_units(n_seq, nk, a.c.nb);
    a.splits = few ? 1 : cq_splits(n, n_seq, nh, nk, a.c.nb);
    a.tiles = (uint32_t)tiles;
    float* at = reinterpret_cast<float*>(workspace);
    a.part_o = a.part_ml = a.lse = a.w_part = nullptr;
    a.w_splits = weights ? cq_weight_splits(n, n_seq, nh, nk, a.c.nb) : 1;
    if (a.w_splits > 1) {
        a.w_part = at;
        at += (size_t)a.w_splits * n_seq * nk * s_cap;
    }
    if (few || a.splits > 1) {
        const uint64_t parts = few ? (uint64_t)units * nh * n : a.splits * rows;
        a.part_o = at;
        a.part_ml = at + parts * Q8_D;
        at += parts * (Q8_D + 2);
    }
    if (weights) a.lse = at;
    const uint64_t grid = few ? (uint64_t)units * nk : tiles * n_seq * nk * a.splits;
    const uint64_t merge = few ? ((uint64_t)n * a.group + 7) / 8 * n_seq * nk : (rows + 7) / 8;
    const uint64_t wgrid = (uint64_t)n_seq * nk * ((a.c.nb + 3) / 4) * a.w_splits;
    if (grid > 0x7fffffffu || merge > 0x7fffffffu || wgrid > 0x7fffffffu) return T2H_ERR_SHAPE;
    if (few && n * a.group <= 16)
        hipLaunchKernelGGL(attn_rows_q8_kernel<1>, dim3((uint32_t)grid), dim3(DQ_WAVES * 64), 0, st, a);
    else if (few)
        hipLaunchKernelGGL(attn_rows_q8_kernel<2>, dim3((uint32_t)grid), dim3(DQ_WAVES * 64), 0, st, a);
    else if (tile_rows == 256)
        hipLaunchKernelGGL(attn_chunk_q8_kernel<8>, dim3((uint32_t)grid), dim3(512), 0, st, a);
    else
        hipLaunchKernelGGL(attn_chunk_q8_kernel<4>, dim3((uint32_t)grid), dim3(256), 0, st, a);
    T2H_LAUNCH_CHECK();
    if (few) {
        hipLaunchKernelGGL(attn_rows_q8_merge_kernel, dim3((uint32_t)merge), dim3(256), 0, st, a);
        T2H_LAUNCH_CHECK();
    } else if (a.splits > 1) {
        hipLaunchKernelGGL(attn_chunk_q8_merge_kernel, dim3((uint32_t)merge), dim3(256), 0, st, a);
        T2H_LAUNCH_CHECK();
    }
    if (weights) {
        hipLaunchKernelGGL(attn_chunk_q8_weights_kernel, dim3((uint32_t)wgrid), dim3(256), 0, st, a);
        T2H_LAUNCH_CHECK();
        if (a.w_splits > 1) {
            hipLaunchKernelGGL(attn_chunk_q8_weights_merge_kernel, dim3((uint32_t)sums), dim3(256), 0, st, a);
            T2H_LAUNCH_CHECK();
        }
    }
    return T2H_OK;
}
