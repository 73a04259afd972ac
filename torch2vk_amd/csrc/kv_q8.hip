// Writing, reading back and evicting the 8-bit KV cache (layout and rounding: kv_q8.h).
#include <math.h>

#include "kv_q8.h"
#include "kv_q8_args.h"

namespace t2h {

// ------------------------------------------------------------------------------------------------- chunk write --
//
// For every token t of a chunk, per head: RMSNorm over 128 dims and rotate-half RoPE at position length + offset + t of
// q and k; q goes out in bf16, k and v go to the cache.  Bound by memory: a token's q, k and v are read once in fp32.
// One launch holds two kinds of blocks: those of q (a wave takes 8 heads of a token), and one for each (sequence, cache
// block that the chunk touches, KV head), which holds the 64 tokens in registers because a finished block's scale needs
// all of them before the first is rounded.  Measured: 8 ragged prompts of 900 to 2048 tokens, 32 / 8 heads, 95 us for
// 446 MB, 4.7 TB/s (a large copy reaches 4.8); 512 tokens of 16 / 8 heads 8.1 us, the latency of a block's rows, angles and
// scale in turn.

struct Q8WriteArgs {
    const float* q;
    const float* k;
    const float* v;
    size_t q_row, k_row, v_row;
    const float* q_norm_w;
    const float* k_norm_w;
    float eps;
    double log2_theta;  // rope: whether to rotate
    int rope;
    const int32_t* lengths;
    const int32_t* counts;
    const int32_t* offsets;
    uint32_t n, n_seq, nh;
    uint32_t kv_blocks;  // cache blocks that n tokens can touch
    uint32_t kv_grid;    // kv_blocks * nk * n_seq
    uint16_t* q_out;
    KvQ8 c;
};

constexpr int Q8W_HEADS = 8;  // q heads a wave
constexpr int Q8W_WAVES = 8;  // a thread block

__device__ __forceinline__ void q8_write_q(const Q8WriteArgs& a, uint64_t unit) {
    const int lane = threadIdx.x & 63;
    const uint32_t groups = (a.nh + Q8W_HEADS - 1) / Q8W_HEADS;
    if (unit >= (uint64_t)a.n_seq * a.n * groups) return;
    const uint64_t row = unit / groups;
    const uint32_t h0 = (uint32_t)(unit - row * groups) * Q8W_HEADS;
    const uint32_t seq = (uint32_t)(row / a.n), t = (uint32_t)(row - (uint64_t)seq * a.n);
    uint16_t* out = a.q_out + (row * a.nh + h0) * Q8_D;
    const uint32_t heads = a.nh - h0 < Q8W_HEADS ? a.nh - h0 : Q8W_HEADS;
    const int len = a.lengths[seq];
    const int count = a.counts ? a.counts[seq] : (int)a.n;
    if (len < 0 || (int)t >= count) {  // padding
        for (uint32_t j = 0; j < heads; ++j) reinterpret_cast<uint32_t*>(out + j * Q8_D)[lane] = 0u;
        return;
    }
    float x0[Q8W_HEADS], x1[Q8W_HEADS];
#pragma unroll
    for (int j = 0; j < Q8W_HEADS; ++j) {
        const uint32_t h = h0 + (j < (int)heads ? j : heads - 1);  // past the last head: re-read it, store nothing
        const float* x = a.q + row * a.q_row + (size_t)h * Q8_D;
        x0[j] = x[lane];
        x1[j] = x[lane + 64];
    }
    const bool has_w = a.q_norm_w != nullptr;
    const float w0 = has_w ? a.q_norm_w[lane] : 1.0f, w1 = has_w ? a.q_norm_w[lane + 64] : 1.0f;
    float cs = 1.0f, sn = 0.0f;
    if (a.rope) rope_at(rope_turns(lane, a.log2_theta), len + (a.offsets ? a.offsets[seq] : 0) + (int)t, cs, sn);
#pragma unroll
    for (int j = 0; j < Q8W_HEADS; ++j) {
        if (j >= (int)heads) break;
        float r0, r1;
        q8_norm_rope(x0[j], x1[j], has_w, w0, w1, a.eps, cs, sn, r0, r1);
        out[j * Q8_D + lane] = (uint16_t)f32_to_bf16_bits(r0);
        out[j * Q8_D + lane + 64] = (uint16_t)f32_to_bf16_bits(r1);
    }
}

// One cache block of one head: tokens 64 b + 8 wave + i in wave `wave`, row i; a lane holds key dims lane and lane + 64
// and value dims 2 lane and 2 lane + 1, as bf16 pairs.
__device__ __forceinline__ void q8_write_block(const Q8WriteArgs& a, uint32_t seq, uint32_t h, Q8Span s, int b,
                                               uint32_t* kbytes, uint32_t* red) {
    constexpr int ROWS = Q8_BLOCK / Q8W_WAVES;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int p0 = b * Q8_BLOCK + wave * ROWS;
    const bool whole = (b + 1) * Q8_BLOCK <= s.end;
    const bool has_w = a.k_norm_w != nullptr;
    const float w0 = has_w ? a.k_norm_w[lane] : 1.0f, w1 = has_w ? a.k_norm_w[lane + 64] : 1.0f;
    const size_t tail = a.c.tail_at(seq, h);
    const int off = a.offsets ? a.offsets[seq] : 0;
    const size_t row0 = (size_t)seq * a.n + (size_t)((int64_t)p0 - a.lengths[seq]);  // of token p0, if that is new
    const float* kx = a.k + row0 * a.k_row + (size_t)h * Q8_D + lane;
    const float* vx = a.v + row0 * a.v_row + (size_t)h * Q8_D + 2 * lane;
    float k0[ROWS], k1[ROWS], v0[ROWS], v1[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        k0[i] = k1[i] = v0[i] = v1[i] = 0.0f;
        if (p0 + i >= s.len && p0 + i < s.end) {
            k0[i] = kx[i * a.k_row];
            k1[i] = kx[i * a.k_row + 64];
            v0[i] = vx[i * a.v_row];
            v1[i] = vx[i * a.v_row + 1];
        }
    }
    const double turns = a.rope ? rope_turns(lane, a.log2_theta) : 0.0;
    uint32_t kk[ROWS], vv[ROWS], kmax = 0, vmax = 0;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        __builtin_amdgcn_sched_barrier(0);  // a row at a time: 16 angles at once would take every register
        const int p = p0 + i, r = wave * ROWS + i;
        kk[i] = vv[i] = 0;
        if (p >= s.len && p < s.end) {
            float cs = 1.0f, sn = 0.0f, r0, r1;
            if (a.rope) rope_at(turns, p + off, cs, sn);
            q8_norm_rope(k0[i], k1[i], has_w, w0, w1, a.eps, cs, sn, r0, r1);
            kk[i] = pack_bf16x2(r0, r1);
            vv[i] = pack_bf16x2(v0[i], v1[i]);
        } else if (whole) {  // a token of the tail that this chunk completes
            kk[i] = (uint32_t)a.c.kt[tail + r * Q8_D + lane] | (uint32_t)a.c.kt[tail + r * Q8_D + lane + 64] << 16;
            vv[i] = (uint32_t)a.c.vt[tail + (2 * lane) * Q8_BLOCK + r] | (uint32_t)a.c.vt[tail + (2 * lane + 1) * Q8_BLOCK + r] << 16;
        }
        kmax = max(kmax, bf16_abs_max(kk[i]));
        vmax = max(vmax, bf16_abs_max(vv[i]));
    }
    if (!whole) {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int p = p0 + i, r = wave * ROWS + i;
            if (p < s.len || p >= s.end) continue;
            a.c.kt[tail + r * Q8_D + lane] = (uint16_t)kk[i];
            a.c.kt[tail + r * Q8_D + lane + 64] = (uint16_t)(kk[i] >> 16);
            a.c.vt[tail + (2 * lane) * Q8_BLOCK + r] = (uint16_t)vv[i];
            a.c.vt[tail + (2 * lane + 1) * Q8_BLOCK + r] = (uint16_t)(vv[i] >> 16);
        }
        return;
    }
    kmax = wave_max_u32(kmax);
    vmax = wave_max_u32(vmax);
    if (lane == 0) {
        red[wave] = kmax;
        red[Q8W_WAVES + wave] = vmax;
    }
    __syncthreads();
    for (int i = 0; i < Q8W_WAVES; ++i) {
        kmax = max(kmax, red[i]);
        vmax = max(vmax, red[Q8W_WAVES + i]);
    }
    float ks, kinv, vs, vinv;
    q8_scale(kmax, ks, kinv);
    q8_scale(vmax, vs, vinv);
    // keys: bytes through LDS, so that they leave as 16-byte stores
    uint8_t* kb = reinterpret_cast<uint8_t*>(kbytes) + wave * ROWS * Q8_D + lane;
    const size_t at = a.c.block_at(seq, (uint32_t)b, h);
    uint32_t lo[ROWS / 4], hi[ROWS / 4];
#pragma unroll
    for (int i = 0; i < ROWS; i += 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            kb[(i + e) * Q8_D] = (uint8_t)q8_code(__uint_as_float(kk[i + e] << 16), kinv);
            kb[(i + e) * Q8_D + 64] = (uint8_t)q8_code(__uint_as_float(kk[i + e] & 0xffff0000u), kinv);
        }
        lo[i / 4] = q8_pack4(__uint_as_float(vv[i] << 16), __uint_as_float(vv[i + 1] << 16), __uint_as_float(vv[i + 2] << 16),
                             __uint_as_float(vv[i + 3] << 16), vinv);
        hi[i / 4] = q8_pack4(__uint_as_float(vv[i] & 0xffff0000u), __uint_as_float(vv[i + 1] & 0xffff0000u),
                             __uint_as_float(vv[i + 2] & 0xffff0000u), __uint_as_float(vv[i + 3] & 0xffff0000u), vinv);
    }
    int8_t* vb = a.c.v + at + (size_t)(2 * lane) * Q8_BLOCK + wave * ROWS;
    *reinterpret_cast<uint2*>(vb) = make_uint2(lo[0], lo[1]);
    *reinterpret_cast<uint2*>(vb + Q8_BLOCK) = make_uint2(hi[0], hi[1]);
    __syncthreads();
    reinterpret_cast<uint4*>(a.c.k + at)[threadIdx.x] = reinterpret_cast<const uint4*>(kbytes)[threadIdx.x];
    if (threadIdx.x == 0) {
        a.c.ks[a.c.scale_at(seq, (uint32_t)b, h)] = ks;
        a.c.vs[a.c.scale_at(seq, (uint32_t)b, h)] = vs;
    }
}

__global__ __launch_bounds__(Q8W_WAVES * 64) void q8_write_kernel(const Q8WriteArgs a) {
    __shared__ __align__(16) uint32_t kbytes[Q8_BYTES / 4];
    __shared__ uint32_t red[2 * Q8W_WAVES];
    if (blockIdx.x >= a.kv_grid) {
        q8_write_q(a, (uint64_t)(blockIdx.x - a.kv_grid) * Q8W_WAVES + (threadIdx.x >> 6));
        return;
    }
    const uint32_t h = blockIdx.x % a.c.nk;
    const uint32_t rest = blockIdx.x / a.c.nk;
    const uint32_t j = rest % a.kv_blocks, seq = rest / a.kv_blocks;
    const Q8Span s = q8_span(a.lengths, a.counts, seq, a.n, a.c.nb);
    if (s.len >= s.end) return;
    const int first = s.len / Q8_BLOCK, last = (s.end - 1) / Q8_BLOCK;
    const int b = first + (int)j;
    if (b > last) return;
    // The block that the old tail's rows belong to is completed before the chunk's own rest becomes the tail: where both
    // happen, one thread block does them in that order.
    const bool chained = last > first && s.len % Q8_BLOCK != 0 && s.end % Q8_BLOCK != 0;
    if (chained && b == last) return;
    q8_write_block(a, seq, h, s, b, kbytes, red);
    if (chained && j == 0) {
        __syncthreads();
        q8_write_block(a, seq, h, s, last, kbytes, red);
    }
}

// ------------------------------------------------------------------------------------------------- read back --
//
// The cache's values as the token-major bf16 rows [n_seq][s_cap][nk][128] of the framework's other caches, code times
// scale rounded once; zeros from the length on.  Bound by the bf16 rows that it writes: 38 us for 8
// sequences of 4096 tokens and a tail, 8 heads: 67 MB read and 137 written, 5.4 TB/s.

struct Q8ReadArgs {
    KvQ8 c;
    const int32_t* lengths;
    uint16_t* k_out;
    uint16_t* v_out;
};

// Eight codes times a scale as bf16.
__device__ __forceinline__ uint4 q8_rows(uint32_t w0, uint32_t w1, float s) {
    return make_uint4(pack_bf16x2(q8_value(w0, 0) * s, q8_value(w0, 1) * s), pack_bf16x2(q8_value(w0, 2) * s, q8_value(w0, 3) * s),
                      pack_bf16x2(q8_value(w1, 0) * s, q8_value(w1, 1) * s), pack_bf16x2(q8_value(w1, 2) * s, q8_value(w1, 3) * s));
}

__global__ __launch_bounds__(256) void q8_read_kernel(const Q8ReadArgs a) {
    __shared__ uint32_t vb[Q8_D][Q8_BLOCK / 4 + 1];
    const uint32_t h = blockIdx.x % a.c.nk;
    const uint32_t rest = blockIdx.x / a.c.nk;
    const uint32_t b = rest % a.c.nb, seq = rest / a.c.nb;
    const int cap = (int)(a.c.nb * Q8_BLOCK);
    const int given = a.lengths[seq];
    const int len = given < 0 ? 0 : (given < cap ? given : cap);
    const int tid = threadIdx.x;
    const int p0 = (int)b * Q8_BLOCK;
    const bool whole = p0 + Q8_BLOCK <= len;
    const size_t at = a.c.block_at(seq, b, h), tail = a.c.tail_at(seq, h);
    const size_t out = (((size_t)seq * cap + p0) * a.c.nk + h) * Q8_D, step = (size_t)a.c.nk * Q8_D;  // token p0; a token
    if (whole) {
        // keys: 16 codes of a row a thread, twice
        uint4 kc[2], vc[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            kc[i] = load_u4(a.c.k + at + (tid + 256 * i) * 16);
            vc[i] = load_u4(a.c.v + at + (tid + 256 * i) * 16);
        }
        const float ks = a.c.ks[a.c.scale_at(seq, b, h)], vs = a.c.vs[a.c.scale_at(seq, b, h)];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int n = tid + 256 * i;
            uint32_t* row = &vb[n >> 2][4 * (n & 3)];
            row[0] = vc[i].x, row[1] = vc[i].y, row[2] = vc[i].z, row[3] = vc[i].w;
            uint4* to = reinterpret_cast<uint4*>(a.k_out + out + (n >> 3) * step + 16 * (n & 7));
            to[0] = q8_rows(kc[i].x, kc[i].y, ks);
            to[1] = q8_rows(kc[i].z, kc[i].w, ks);
        }
        __syncthreads();
        // values: 4 tokens of 8 dims a thread, transposed in registers
        const int d = (tid & 15) * 8, quad = tid >> 4;
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = vb[d + j][quad];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = pack_bf16x2(q8_value(w[2 * j], t) * vs, q8_value(w[2 * j + 1], t) * vs);
            *reinterpret_cast<uint4*>(a.v_out + out + (4 * quad + t) * step + d) = make_uint4(o[0], o[1], o[2], o[3]);
        }
        return;
    }
    const int lane = tid & 63, wave = tid >> 6;
    for (int i = wave; i < Q8_BLOCK; i += 4) {
        uint32_t kk = 0, vv = 0;  // dims 2 lane, 2 lane + 1
        if (p0 + i < len) {
            kk = reinterpret_cast<const uint32_t*>(a.c.kt + tail + i * Q8_D)[lane];
            vv = (uint32_t)a.c.vt[tail + (2 * lane) * Q8_BLOCK + i] | (uint32_t)a.c.vt[tail + (2 * lane + 1) * Q8_BLOCK + i] << 16;
        }
        reinterpret_cast<uint32_t*>(a.k_out + out + i * step)[lane] = kk;
        reinterpret_cast<uint32_t*>(a.v_out + out + i * step)[lane] = vv;
    }
}

// --------------------------------------------------------------------------------------------------- eviction --
//
// Per (sequence, KV head), of the F whole blocks' tokens 64 min(F, keep) stay: the first `sink`, the last `recent`, then
// by accumulated weight (ties: the lowest index; a NaN ranks above every number), in the order of the tokens.
// The choice is a radix selection of the last weight that stays, 11 + 11 + 10 bits of an order-preserving key, each
// digit one pass over the weights and a histogram in LDS; then ballots give each token its place.  A second kernel moves
// the tokens: block by block it gathers 64 of them, finds their new scale and rounds them again.
//
// Measured: 8 sequences of 9000 to 16300 tokens, 8 heads, brought to 64 blocks: selection 23 us, one thread block a head, bound
// by the chain of three digits and by what one CU issues (60000 tokens, both kernels: 73 us with the keys in registers, 112 with
// keys read again for every pass); moving 56 us, 145 MB read and 70 written, 3.8 TB/s.  A token's values are a byte of each of
// its block's 128 rows, so that all rows of a block with any token that stays are read, while its keys are 128 bytes in a row.
// Taking those rows through LDS whole, with loads straight into it, was 4 % faster where all of a large batch's blocks lie
// close (32 of 16000: 365 us for 379) and 4 % slower at 8 sequences; through registers it was slower throughout.

struct Q8EvictArgs {
    KvQ8 c, o;  // from, to
    const int32_t* lengths;
    const float* w_in;
    float* w_out;
    int32_t* kept;  // [n_seq][nk][64 keep]
    int32_t* lengths_out;
    uint32_t keep, sink, recent;
    uint32_t most;   // output blocks that a head can have
    int same;        // output and input are one cache: o is the workspace
    float* w_back;   // where weights_out and weights are one: they, w_out being the workspace
    size_t w_row;    // of a head in w_out
};

__device__ __forceinline__ int q8_length(const int32_t* lengths, uint32_t seq, uint32_t nb) {
    const int cap = (int)(nb * Q8_BLOCK), given = lengths[seq];
    return given < 0 ? 0 : (given < cap ? given : cap);
}

__device__ __forceinline__ uint32_t evict_key(const float* w, int t, int full, const Q8EvictArgs& a) {
    if (t < (int)a.sink || t >= full - (int)a.recent) return 0xffffffffu;
    const float x = w[t] + 0.0f;  // -0 ranks as 0
    if (x != x) return 0xfffffffeu;
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int EV_THREADS = 1024;
constexpr int EV_WAVES = EV_THREADS / 64;
constexpr int EV_SMALL = 16384;  // tokens that 16 keys a lane hold; 64 hold 65536, the most that the registers of 16 waves do

template <int EV_BATCH>
__global__ __launch_bounds__(EV_THREADS) void q8_evict_select_kernel(const Q8EvictArgs a) {
    __shared__ uint32_t hist[2048];
    __shared__ uint32_t wsum[EV_WAVES][2];
    __shared__ uint32_t found[2];
    const uint32_t h = blockIdx.x % a.c.nk, seq = blockIdx.x / a.c.nk;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int len = q8_length(a.lengths, seq, a.c.nb);
    const int blocks = len / Q8_BLOCK, full = blocks * Q8_BLOCK;
    const int most = (int)a.keep * Q8_BLOCK;
    const int stay = full < most ? full : most;
    int32_t* kept = a.kept + (size_t)blockIdx.x * most;
    if (h == 0 && tid == 0) a.lengths_out[seq] = a.lengths[seq] < 0 ? a.lengths[seq] : len - full + stay;
    for (int i = (stay < full ? stay : 0) + tid; i < most; i += EV_THREADS) kept[i] = i < stay ? i : -1;
    if (stay == full) return;
    const float* w = a.w_in + (size_t)blockIdx.x * a.c.nb * Q8_BLOCK;

    // each wave takes a run of tokens, EV_BATCH rows of 64 at a time in registers; up to 1024 EV_BATCH tokens are loaded once
    const int per = ((full + EV_WAVES - 1) / EV_WAVES + 63) / 64 * 64;
    const int t0 = wave * per + lane, t1 = wave * per + per < full ? wave * per + per : full;
    const bool once = per <= EV_BATCH * 64;
    uint32_t key[EV_BATCH];
    auto load = [&](int base) {
#pragma unroll
        for (int e = 0; e < EV_BATCH; ++e) {
            const int t = t0 + base + 64 * e;
            key[e] = t < t1 ? evict_key(w, t, full, a) : 0u;
        }
    };
    load(0);
    uint32_t prefix = 0, need = (uint32_t)stay;  // of the tokens whose key begins with prefix, `need` stay
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
        const uint32_t mask = pass == 0 ? 0u : ~0u << (shift + bits), digits = (1u << bits) - 1u;
        for (int i = tid; i < 2048; i += EV_THREADS) hist[i] = 0;
        __syncthreads();
        for (int base = 0; base < per; base += EV_BATCH * 64) {
            if (!once) load(base);
#pragma unroll
            for (int e = 0; e < EV_BATCH; ++e) {
                if (base + 64 * e >= per) break;
                if (t0 + base + 64 * e < t1 && (key[e] & mask) == prefix) atomicAdd(&hist[(key[e] >> shift) & digits], 1u);
            }
        }
        __syncthreads();
        // bins from the top: thread i holds bins 2047 - 2 i and 2046 - 2 i
        const uint32_t c0 = hist[2047 - 2 * tid], c1 = hist[2046 - 2 * tid];
        const uint32_t run = wave_scan_u32(c0 + c1);
        if (lane == 63) wsum[wave][0] = run;
        __syncthreads();
        uint32_t before = run - c0 - c1;
#pragma unroll
        for (int i = 0; i < EV_WAVES; ++i) before += i < wave ? wsum[i][0] : 0u;
        if (before < need && need <= before + c0) {
            found[0] = 2047u - 2u * (uint32_t)tid;
            found[1] = need - before;
        } else if (before + c0 < need && need <= before + c0 + c1) {
            found[0] = 2046u - 2u * (uint32_t)tid;
            found[1] = need - before - c0;
        }
        __syncthreads();
        prefix |= found[0] << shift;
        need = found[1];
    }
    // prefix is the smallest key that stays, and `need` of the tokens that have it
    uint32_t above = 0, equal = 0;
    for (int base = 0; base < per; base += EV_BATCH * 64) {
        if (!once) load(base);
#pragma unroll
        for (int e = 0; e < EV_BATCH; ++e) {
            if (base + 64 * e >= per) break;
            const bool in = t0 + base + 64 * e < t1;
            above += __popcll(__ballot(in && key[e] > prefix));
            equal += __popcll(__ballot(in && key[e] == prefix));
        }
    }
    __syncthreads();
    if (lane == 0) {
        wsum[wave][0] = above;
        wsum[wave][1] = equal;
    }
    __syncthreads();
    above = equal = 0;
#pragma unroll
    for (int i = 0; i < EV_WAVES; ++i) {
        above += i < wave ? wsum[i][0] : 0u;
        equal += i < wave ? wsum[i][1] : 0u;
    }
    const uint64_t below = (1ull << lane) - 1;
    for (int base = 0; base < per; base += EV_BATCH * 64) {
        if (!once) load(base);
#pragma unroll
        for (int e = 0; e < EV_BATCH; ++e) {
            if (base + 64 * e >= per) break;
            const int t = t0 + base + 64 * e;
            const bool in = t < t1;
            const uint64_t ma = __ballot(in && key[e] > prefix), me = __ballot(in && key[e] == prefix);
            const uint32_t a0 = above + __popcll(ma & below), e0 = equal + __popcll(me & below);
            if (in && (key[e] > prefix || (key[e] == prefix && e0 < need))) kept[a0 + (e0 < need ? e0 : need)] = t;
            above += __popcll(ma);
            equal += __popcll(me);
        }
    }
}

// Keys (blockIdx.y 0, with the weights) or values (1): one output block of one head.  Where the output is the input's own
// memory, what is written here lies in the workspace and the kernel below brings it back, so that all blocks are made at once:
// a thread block that walks a head's blocks in order needs no second memory, but takes 115 us for 32 blocks of 8 heads, 20 here.
__global__ __launch_bounds__(256, 7) void q8_evict_move_kernel(const Q8EvictArgs a) {
    __shared__ int from[Q8_BLOCK];
    __shared__ float fs[Q8_BLOCK];
    __shared__ uint32_t red[4];
    const uint32_t h = blockIdx.x % a.c.nk;
    const uint32_t rest = blockIdx.x / a.c.nk;
    const int b = (int)(rest % a.most);
    const uint32_t seq = rest / a.most;
    const bool values = blockIdx.y != 0;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int len = q8_length(a.lengths, seq, a.c.nb);
    const int blocks = len / Q8_BLOCK;
    const int stay = blocks < (int)a.keep ? blocks : (int)a.keep;
    const size_t head = (size_t)seq * a.c.nk + h;
    const float* w_in = a.w_in + head * a.c.nb * Q8_BLOCK;
    float* w_out = a.w_out + head * a.w_row;
    const bool all = stay == blocks;  // nothing leaves: blocks are copied as they are
    const bool move = !(all && a.same);
    if (!values) {
        if (b < stay && tid < Q8_BLOCK) w_out[b * Q8_BLOCK + tid] = w_in[a.kept[(head * a.keep + b) * Q8_BLOCK + tid]];
        const int r = len - blocks * Q8_BLOCK;
        if (b == 0 && tid < r) w_out[stay * Q8_BLOCK + tid] = w_in[blocks * Q8_BLOCK + tid];
    }
    if (b == 0 && !a.same && a.lengths[seq] >= 0) {  // the tail's rows
        const uint4* src = reinterpret_cast<const uint4*>((values ? a.c.vt : a.c.kt) + a.c.tail_at(seq, h));
        uint4* dst = reinterpret_cast<uint4*>((values ? a.o.vt : a.o.kt) + a.o.tail_at(seq, h));
        for (int i = tid; i < Q8_BYTES * 2 / 16; i += 256) dst[i] = src[i];
    }
    if (b < stay && move) {
        if (tid < Q8_BLOCK) {
            const int t = a.kept[(head * a.keep + b) * Q8_BLOCK + tid];
            from[tid] = t;
            fs[tid] = (values ? a.c.vs : a.c.ks)[a.c.scale_at(seq, (uint32_t)t / Q8_BLOCK, h)];
        }
        __syncthreads();
        uint32_t top = 0;
        const size_t to = a.o.block_at(seq, (uint32_t)b, h);
        float inv, s;
        if (!values) {
            const int r = tid >> 2, part = tid & 3;
            const int t = from[r];
            const float f = fs[r];
            const uint4* src = reinterpret_cast<const uint4*>(a.c.k + a.c.block_at(seq, (uint32_t)t / Q8_BLOCK, h) +
                                                              (t % Q8_BLOCK) * Q8_D + part * 32);
            uint4 x[2] = {src[0], src[1]};
            uint32_t* u = reinterpret_cast<uint32_t*>(x);
#pragma unroll
            for (int i = 0; i < 32; ++i) top = max(top, abs_bits(q8_value(u[i / 4], i % 4) * f));
#pragma unroll
            for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(u[i]));
            top = wave_max_u32(top);
            if (lane == 0) red[wave] = top;
            __syncthreads();
            q8_scale(max(max(red[0], red[1]), max(red[2], red[3])), s, inv);
            if (all) s = f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!all)
                    u[i] = q8_pack4(q8_value(u[i], 0) * f, q8_value(u[i], 1) * f, q8_value(u[i], 2) * f, q8_value(u[i], 3) * f, inv);
            uint4* dst = reinterpret_cast<uint4*>(a.o.k + to + r * Q8_D + part * 32);
            dst[0] = x[0];
            dst[1] = x[1];
        } else {
            // a lane is a token, a wave 32 dims: 64 tokens of a dim are a few short runs of bytes
            const int t = from[lane];
            const float f = fs[lane];
            const int8_t* src = a.c.v + a.c.block_at(seq, (uint32_t)t / Q8_BLOCK, h) + (size_t)wave * 32 * Q8_BLOCK + t % Q8_BLOCK;
            uint32_t u[8];  // 4 dims a word: the kernel waits for memory, and more registers would be fewer waves that do
            {
                uint8_t x[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) x[i] = (uint8_t)src[i * Q8_BLOCK];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    u[i] = (uint32_t)x[4 * i] | (uint32_t)x[4 * i + 1] << 8 | (uint32_t)x[4 * i + 2] << 16 |
                           (uint32_t)x[4 * i + 3] << 24;
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) top = max(top, abs_bits(q8_value(u[i / 4], i % 4) * f));
#pragma unroll
            for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(u[i]));  // (unpacked again below, not kept)
            top = wave_max_u32(top);
            if (lane == 0) red[wave] = top;
            __syncthreads();
            q8_scale(max(max(red[0], red[1]), max(red[2], red[3])), s, inv);
            if (all) s = f;
            // a dim's 4 tokens leave as one word: byte stores would take a cycle of the address unit for each lane
            int8_t* dst = a.o.v + to + (size_t)wave * 32 * Q8_BLOCK + lane;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                int w = (all ? (int)(u[i / 4] >> (8 * (i % 4))) : q8_code(q8_value(u[i / 4], i % 4) * f, inv)) & 255;
                w |= __builtin_amdgcn_update_dpp(0, w, 0xB1, 0xf, 0xf, true) << 8;   // lane ^ 1
                w |= __builtin_amdgcn_update_dpp(0, w, 0x4E, 0xf, 0xf, true) << 16;  // lane ^ 2
                if ((lane & 3) == 0) *reinterpret_cast<int*>(dst + i * Q8_BLOCK) = w;
            }
        }
        if (tid == 0) (values ? a.o.vs : a.o.ks)[a.o.scale_at(seq, (uint32_t)b, h)] = s;
    }
}

// An output block of one head, and its weights, from the workspace to where they belong.
__global__ __launch_bounds__(256) void q8_evict_back_kernel(const Q8EvictArgs a) {
    const uint32_t h = blockIdx.x % a.c.nk;
    const uint32_t rest = blockIdx.x / a.c.nk;
    const int b = (int)(rest % a.most);
    const uint32_t seq = rest / a.most;
    const int tid = threadIdx.x;
    const int len = q8_length(a.lengths, seq, a.c.nb);
    const int blocks = len / Q8_BLOCK;
    if (blocks <= (int)a.keep) return;  // nothing has left
    const int stay = (int)a.keep;
    const size_t head = (size_t)seq * a.c.nk + h;
    if (a.same) {
        const size_t at = a.o.block_at(seq, (uint32_t)b, h), to = a.c.block_at(seq, (uint32_t)b, h);
        uint4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = load_u4((i < 2 ? a.o.k : a.o.v) + at + ((i & 1) * 256 + tid) * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>((i < 2 ? a.c.k : a.c.v) + to + ((i & 1) * 256 + tid) * 16) = x[i];
        if (tid == 0) {
            a.c.ks[a.c.scale_at(seq, (uint32_t)b, h)] = a.o.ks[a.o.scale_at(seq, (uint32_t)b, h)];
            a.c.vs[a.c.scale_at(seq, (uint32_t)b, h)] = a.o.vs[a.o.scale_at(seq, (uint32_t)b, h)];
        }
    }
    if (a.w_back) {
        const float* w = a.w_out + head * a.w_row;
        float* to = a.w_back + head * a.c.nb * Q8_BLOCK;
        if (tid < Q8_BLOCK) to[b * Q8_BLOCK + tid] = w[b * Q8_BLOCK + tid];
        if (b == 0 && tid < len - blocks * Q8_BLOCK) to[stay * Q8_BLOCK + tid] = w[stay * Q8_BLOCK + tid];
    }
}

}  // namespace t2h

using namespace t2h;

extern "C" int t2h_qk_norm_rope_cache_q8(const float* q, uint64_t q_row, const float* k, uint64_t k_row, const float* v,
                                         uint64_t v_row, const float* q_norm_w, const float* k_norm_w, float eps,
                                         float theta, const int32_t* lengths, const int32_t* counts,
                                         const int32_t* rope_offsets, uint32_t n, uint32_t n_seq, uint32_t nh, uint32_t nk,
                                         uint32_t d, void* q_out, void* const* cache, uint32_t s_cap, void* stream) {
    Q8WriteArgs a;
    if (!q || !k || !v || !lengths || !q_out) return T2H_ERR_NULL;
    if ((q_norm_w == nullptr) != (k_norm_w == nullptr)) return T2H_ERR_NULL;
    if (const int e = q8_cache(cache, s_cap, n_seq, nh, nk, d, a.c)) return e;
    if (q_row < (uint64_t)nh * d || k_row < (uint64_t)nk * d || v_row < (uint64_t)nk * d) return T2H_ERR_SHAPE;
    if (reinterpret_cast<uintptr_t>(q_out) & 3) return T2H_ERR_ALIGN;
    if (n == 0) return T2H_OK;
    const uint64_t kv_blocks = ((uint64_t)n + 2 * Q8_BLOCK - 2) / Q8_BLOCK;
    const uint64_t kv_grid = kv_blocks * nk * n_seq;
    const uint64_t units = (uint64_t)n_seq * n * ((nh + Q8W_HEADS - 1) / Q8W_HEADS);
    if (n > 0x3fffffffu || kv_grid + (units + Q8W_WAVES - 1) / Q8W_WAVES > 0x7fffffffu) return T2H_ERR_SHAPE;
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_row = (size_t)q_row;
    a.k_row = (size_t)k_row;
    a.v_row = (size_t)v_row;
    a.q_norm_w = q_norm_w;
    a.k_norm_w = k_norm_w;
    a.eps = eps;
    a.rope = theta > 0.0f;
    a.log2_theta = a.rope ? log2((double)theta) : 0.0;
    a.lengths = lengths;
    a.counts = counts;
    a.offsets = rope_offsets;
    a.n = n;
    a.n_seq = n_seq;
    a.nh = nh;
    a.kv_blocks = (uint32_t)kv_blocks;
    a.kv_grid = (uint32_t)kv_grid;
    a.q_out = reinterpret_cast<uint16_t*>(q_out);
    hipLaunchKernelGGL(q8_write_kernel, dim3((uint32_t)(kv_grid + (units + Q8W_WAVES - 1) / Q8W_WAVES)), dim3(Q8W_WAVES * 64), 0,
                       reinterpret_cast<hipStream_t>(stream), a);
    T2H_LAUNCH_CHECK();
    return T2H_OK;
}

extern "C" int t2h_kv_cache_q8_dequantize(void* const* cache, uint32_t s_cap, const int32_t* lengths, uint32_t n_seq,
                                          uint32_t nk, uint32_t d, void* k_out, void* v_out, void* stream) {
    Q8ReadArgs a;
    if (!lengths || !k_out || !v_out) return T2H_ERR_NULL;
    if (const int e = q8_cache(cache, s_cap, n_seq, nk, nk, d, a.c)) return e;
    if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15) return T2H_ERR_ALIGN;
    a.lengths = lengths;
    a.k_out = reinterpret_cast<uint16_t*>(k_out);
    a.v_out = reinterpret_cast<uint16_t*>(v_out);
    const uint64_t grid = (uint64_t)n_seq * a.c.nb * nk;
    if (grid > 0x7fffffffu) return T2H_ERR_SHAPE;
    hipLaunchKernelGGL(q8_read_kernel, dim3((uint32_t)grid), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), a);
    T2H_LAUNCH_CHECK();
    return T2H_OK;
}

// Bytes of the parts of an eviction's workspace: codes, scales, weights.
struct Q8EvictRoom {
    size_t codes, scales, weights;
    Q8EvictRoom(uint32_t keep, uint32_t n_seq, uint32_t nk, uint32_t s_cap) {
        const size_t most = keep < s_cap / Q8_BLOCK ? keep : s_cap / Q8_BLOCK, heads = (size_t)n_seq * nk;
        codes = heads * most * Q8_BYTES;
        scales = (heads * most * 4 + 15) / 16 * 16;
        weights = heads * (most + 1) * Q8_BLOCK * 4;
    }
};

extern "C" size_t t2h_kv_cache_q8_evict_workspace_bytes(uint32_t keep_blocks, uint32_t n_seq, uint32_t nk, uint32_t s_cap) {
    if (keep_blocks == 0 || n_seq == 0 || nk == 0 || s_cap == 0 || s_cap % Q8_BLOCK != 0) return 0;
    const Q8EvictRoom room(keep_blocks, n_seq, nk, s_cap);
    return 2 * room.codes + 2 * room.scales + room.weights;
}

extern "C" int t2h_kv_cache_q8_evict(void* const* cache, uint32_t s_cap, const int32_t* lengths, const float* weights,
                                     uint32_t keep_blocks, uint32_t sink, uint32_t recent, uint32_t n_seq, uint32_t nk,
                                     uint32_t d, void* const* cache_out, uint32_t s_cap_out, float* weights_out,
                                     int32_t* kept, int32_t* lengths_out, void* workspace, size_t workspace_bytes,
                                     void* stream) {
    Q8EvictArgs a;
    if (!lengths || !weights || !weights_out || !kept || !lengths_out) return T2H_ERR_NULL;
    if (const int e = q8_cache(cache, s_cap, n_seq, nk, nk, d, a.c)) return e;
    if (const int e = q8_cache(cache_out, s_cap_out, n_seq, nk, nk, d, a.o)) return e;
    if (keep_blocks == 0 || keep_blocks > 0x1000000u || lengths_out == lengths) return T2H_ERR_ARG;
    if ((uint64_t)sink + recent > (uint64_t)keep_blocks * Q8_BLOCK) return T2H_ERR_ARG;
    // a cache of the output's capacity holds what stays and a tail
    if ((uint64_t)s_cap_out < s_cap && s_cap_out < ((uint64_t)keep_blocks + 1) * Q8_BLOCK) return T2H_ERR_SHAPE;
    const bool same = a.c.k == a.o.k;
    if (same != (a.c.v == a.o.v) || same != (a.c.ks == a.o.ks) || same != (a.c.vs == a.o.vs) ||
        same != (a.c.kt == a.o.kt) || same != (a.c.vt == a.o.vt))
        return T2H_ERR_ARG;
    const bool in_place = same || weights == weights_out;
    if (in_place && s_cap != s_cap_out) return T2H_ERR_SHAPE;
    if (in_place && !workspace) return T2H_ERR_NULL;
    if (in_place && (reinterpret_cast<uintptr_t>(workspace) & 15)) return T2H_ERR_ALIGN;
    if (in_place && workspace_bytes < t2h_kv_cache_q8_evict_workspace_bytes(keep_blocks, n_seq, nk, s_cap))
        return T2H_ERR_WORKSPACE;
    a.lengths = lengths;
    a.w_in = weights;
    a.w_out = weights_out;
    a.kept = kept;
    a.lengths_out = lengths_out;
    a.keep = keep_blocks;
    a.sink = sink;
    a.recent = recent;
    a.most = keep_blocks < a.c.nb ? keep_blocks : a.c.nb;
    a.same = same;
    a.w_back = nullptr;
    a.w_row = (size_t)s_cap_out;
    const Q8EvictRoom room(keep_blocks, n_seq, nk, s_cap);
    int8_t* const at = reinterpret_cast<int8_t*>(workspace);
    if (same) {
        a.o.k = at;
        a.o.v = at + room.codes;
        a.o.ks = reinterpret_cast<float*>(at + 2 * room.codes);
        a.o.vs = reinterpret_cast<float*>(at + 2 * room.codes + room.scales);
        a.o.nb = a.most;
    }
    if (weights == weights_out) {
        a.w_back = weights_out;
        a.w_out = reinterpret_cast<float*>(at + 2 * room.codes + 2 * room.scales);
        a.w_row = ((size_t)a.most + 1) * Q8_BLOCK;
    }
    const uint64_t grid = (uint64_t)n_seq * a.most * nk;
    if (grid > 0x7fffffffu) return T2H_ERR_SHAPE;
    if (s_cap <= EV_SMALL)
        hipLaunchKernelGGL(q8_evict_select_kernel<16>, dim3(n_seq * nk), dim3(EV_THREADS), 0, reinterpret_cast<hipStream_t>(stream), a);
    else
        hipLaunchKernelGGL(q8_evict_select_kernel<64>, dim3(n_seq * nk), dim3(EV_THREADS), 0, reinterpret_cast<hipStream_t>(stream), a);
    T2H_LAUNCH_CHECK();
    hipLaunchKernelGGL(q8_evict_move_kernel, dim3((uint32_t)grid, 2), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), a);
    T2H_LAUNCH_CHECK();
    if (in_place) {
        hipLaunchKernelGGL(q8_evict_back_kernel, dim3((uint32_t)grid), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), a);
        T2H_LAUNCH_CHECK();
    }
    return T2H_OK;
}
