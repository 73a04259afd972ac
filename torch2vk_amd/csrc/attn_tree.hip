// Attention of a tree of drafted tokens over a bf16 KV cache: q/k norm and RoPE of the nodes, their rows into the cache, and
// softmax(q . k / sqrt(d)) . v over the cached tokens, a node's ancestors and itself.
#include <math.h>

#include "kv_q8.h"
#include "lds_dma.h"
#include "tree.h"

namespace t2h {

typedef __bf16 ta_bf16x8 __attribute__((ext_vector_type(8)));
typedef float ta_f32x16 __attribute__((ext_vector_type(16)));
typedef float ta_f32x4 __attribute__((ext_vector_type(4)));

constexpr int TA_D = 128;
constexpr uint32_t TA_CUS = 256;
constexpr int TA_MAX_GROUP = 16;
constexpr uint32_t TA_MOST = (1u << 29) - 64;  // tokens of a sequence: tiles of 32 are counted in 24 bits (275 GB of one KV head)
constexpr int TA_ROW_BYTES = TA_D * 2;
constexpr int TP_NODES = 16, TP_GROUPS = TREE_MAX / TP_NODES;  // nodes of a thread block that writes K and V rows
constexpr float TA_RESCALE = 8.0f;  // log2 headroom of the lazily updated running maximum

// What a thread block of the attention works on: tiles [tile0, tile1) of a sequence's tokens.
struct TreeUnit {
    int seq;  // -1: none
    int tile0, tile1;
    int len, count;          // cached tokens, nodes
    int first, parts, part;  // where the sequence's parts begin, how many they are, and which this is
};

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
    // workspace
    uint16_t* qh;      // [n_seq][nk][n * group][128] rotated queries, and what their rounding to bf16 left
    uint16_t* ql;
    uint64_t* line;    // [n_seq][n] sets of seen nodes
    uint16_t* vt;      // [n_seq][nk][n + 1][128] the nodes' values; zeros where there is none or it is not finite
    uint32_t* broken;  // [n_seq][nk][TP_GROUPS] whether a value of 16 nodes is not finite
    uint64_t* which;   // [n_seq][nk][TP_GROUPS][128][3] then: the nodes whose value in a dim is NaN, infinite, -infinite
    uint32_t* done;    // [n_seq][nk] units that have left their parts; zero between calls
    TreeUnit* units;   // [n_units]
    int2* of_seq;      // [n_seq] first part, parts
    float* part_ml;    // [n_units * nk][rows][2] log2 maximum, sum
    float* part_o;     // [n_units * nk][rows][128]
    uint32_t n_units, row_tiles, rows;  // rows: of a KV head, in whole tiles
    uint32_t keys, least;               // tokens a tile; the least tiles a unit
    float us_turn, us_tile, us_shared, us_join, us_part;  // what tree_chunk goes by
    uint32_t kv_blocks, q_blocks;
};

// ------------------------------------------------------------------------------------------ before the attention --
//
// One launch of three kinds of thread blocks: the units' table, the nodes' K and V rows of a (sequence, KV head), and the
// queries.  5.5 us for 26 nodes, 6.8 for 4 x 64: latency, of the lengths, the rows and the angles in 64 bits one after another.

constexpr int TP_HEADS = 4;  // q heads a wave

// Tiles that a sequence's cached tokens and nodes fill; none where there are no nodes.
__device__ __forceinline__ uint32_t tree_tiles(const TreeAttnArgs& a, uint32_t i, int& len, int& count) {
    len = a.lengths[i];
    count = tree_count_at(a.counts, i, a.n, len, a.s_cap);
    if (count == 0) len = 0;
    return count > 0 ? ((uint32_t)(len + count) + a.keys - 1) / a.keys : 0u;
}

__device__ __forceinline__ uint32_t wave_total_u32(uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)wave_scan_u32(v), 63); }

__device__ __forceinline__ uint32_t div_up(uint32_t x, uint32_t by) {  // x < 2^24
    uint32_t q = (uint32_t)((float)(x + by - 1) * __builtin_amdgcn_rcpf((float)by));
    const int r = (int)(x + by - 1 - q * by);
    q = r < 0 ? q - 1 : q;
    return r >= (int)by ? q + 1 : q;
}

// Tiles a unit.  Each lane weighs the longest sequence in another number of units, by what a turn of the chip costs besides tiles,
// what a tile costs where its thread block is alone and what it costs where all are bound by memory, and a join by its parts.
// `mine`: tiles of sequence `lane`, the others' are looked up.
__device__ uint32_t tree_chunk(const TreeAttnArgs& a, uint32_t mine) {
    const uint32_t lane = threadIdx.x & 63;
    int len, count;
    uint32_t total = lane < a.n_seq ? mine : 0, most = total;
    for (uint32_t i = lane + 64; i < a.n_seq; i += 64) {
        const uint32_t t = tree_tiles(a, i, len, count);
        total += t;
        most = most > t ? most : t;
    }
    total = wave_total_u32(total);
    most = wave_max_u32(most);
    if (most == 0) return 1;
    uint32_t c = div_up(most, lane < 32 ? lane + 1 : 32 + (lane - 31) * 7);
    c = c > a.least ? c : a.least;
    uint32_t units = 0;
    for (uint32_t i = 0; i < a.n_seq; ++i) {
        const uint32_t t = i < 64 ? (uint32_t)__builtin_amdgcn_readlane((int)mine, (int)i) : tree_tiles(a, i, len, count);
        units += t > c ? div_up(t, c) : 1u;
    }
    const float blocks = (float)(a.nk * a.row_tiles) * (1.0f / TA_CUS), turns = ceilf((float)units * blocks);
    // (8 thread blocks read a tile of 64 KiB in 0.7 us each, 64 in 1.5, 256 in 2.6: about the power 0.42 of the chip's share)
    const float busy = (float)units * blocks / turns, share = a.us_shared * __builtin_amdgcn_exp2f(__builtin_amdgcn_logf(busy) * 0.42f);
    const float alone = turns * (a.us_turn + (float)min(c, most) * fmaxf(a.us_tile, share)), together = a.us_turn + (float)total * blocks * a.us_shared;
    float cost = fmaxf(alone, together) + (c < most ? a.us_join + a.us_part * (float)div_up(most, c) : 0.0f);
    if (units > a.n_units) cost = INFINITY;
    const uint64_t best = __ballot(cost == -wave_max(-cost));
    const uint32_t chunk = (uint32_t)__builtin_amdgcn_readlane((int)c, __builtin_ctzll(best));
    return chunk;  // (one unit a sequence is never too many)
}

// Units of a whole chunk come first, the sequences' last, shorter ones behind them, so that what the chip ends with is short.
__device__ void tree_table(const TreeAttnArgs& a) {
    const uint32_t lane = threadIdx.x;
    if (lane >= 64) return;
    int len = 0, count = 0;
    const uint32_t chunk = tree_chunk(a, lane < a.n_seq ? tree_tiles(a, lane, len, count) : 0u);
    uint32_t fulls = 0;
    for (uint32_t i = lane; i < a.n_seq; i += 64) fulls += tree_tiles(a, i, len, count) / chunk;
    fulls = wave_total_u32(fulls);
    uint32_t full_at = 0, rest_at = fulls, part_at = 0;
    for (uint32_t base = 0; base < a.n_seq; base += 64) {
        const uint32_t i = base + lane;
        uint32_t tiles = 0;
        len = count = 0;
        if (i < a.n_seq) tiles = tree_tiles(a, i, len, count);
        const uint32_t full = tiles / chunk, rest = i < a.n_seq && (tiles % chunk || tiles == 0) ? 1u : 0u;
        const uint32_t full_up = wave_scan_u32(full), rest_up = wave_scan_u32(rest);
        if (i < a.n_seq) {
            const uint32_t first = part_at + full_up - full + rest_up - rest, parts = full + rest;
            a.of_seq[i] = make_int2((int)first, (int)parts);
            TreeUnit u;
            u.seq = (int)i;
            u.len = len;
            u.count = count;
            u.first = (int)first;
            u.parts = (int)parts;
            for (uint32_t p = 0; p < parts; ++p) {
                u.tile0 = (int)(p * chunk);
                u.tile1 = (int)min(p * chunk + chunk, tiles);
                u.part = (int)p;
                a.units[p < full ? full_at + full_up - full + p : rest_at + rest_up - rest] = u;
            }
        }
        full_at += (uint32_t)__builtin_amdgcn_readlane((int)full_up, 63);
        rest_at += (uint32_t)__builtin_amdgcn_readlane((int)rest_up, 63);
        part_at += (uint32_t)__builtin_amdgcn_readlane((int)(full_up + rest_up), 63);
    }
    for (uint32_t u = rest_at + lane; u < a.n_units; u += 64) a.units[u].seq = -1;
}

// The same unit by its number, worked out by one wave.
__device__ bool tree_find(const TreeAttnArgs& a, uint32_t unit, TreeUnit& u) {
    const uint32_t lane = threadIdx.x & 63;
    if (a.n_seq == 1) {
        const uint32_t tiles = tree_tiles(a, 0, u.len, u.count);
        const uint32_t chunk = tree_chunk(a, tiles);
        u.seq = u.first = 0;
        u.part = (int)unit;
        u.parts = tiles ? (int)((tiles + chunk - 1) / chunk) : 1;
        u.tile0 = (int)(unit * chunk);
        u.tile1 = (int)min(unit * chunk + chunk, tiles);
        return (int)unit < u.parts;
    }
    int len = 0, count = 0;
    const uint32_t mine = lane < a.n_seq ? tree_tiles(a, lane, len, count) : 0u;
    const uint32_t chunk = tree_chunk(a, mine);
    uint32_t fulls = lane < a.n_seq ? mine / chunk : 0u;
    int l, c;
    for (uint32_t i = lane + 64; i < a.n_seq; i += 64) fulls += tree_tiles(a, i, l, c) / chunk;
    fulls = wave_total_u32(fulls);
    uint32_t full_at = 0, rest_at = 0;
    for (uint32_t base = 0; base < a.n_seq; base += 64) {
        const uint32_t i = base + lane;
        uint32_t tiles = mine;
        if (base) tiles = i < a.n_seq ? tree_tiles(a, i, len, count) : 0u;
        const uint32_t full = tiles / chunk, rest = i < a.n_seq && (tiles % chunk || tiles == 0) ? 1u : 0u;
        const uint32_t full_up = full_at + wave_scan_u32(full), rest_up = rest_at + wave_scan_u32(rest);
        const bool whole = unit < fulls;
        const uint64_t hit = whole ? __ballot(unit >= full_up - full && unit < full_up) : __ballot(rest && unit - fulls == rest_up - 1);
        if (hit) {
            const int at = __builtin_ctzll(hit);
            u.seq = (int)base + at;
            u.len = __builtin_amdgcn_readlane(len, at);
            u.count = __builtin_amdgcn_readlane(count, at);
            const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)(full_up - full), at),
                           n_full = (uint32_t)__builtin_amdgcn_readlane((int)full, at),
                           n_rest = (uint32_t)__builtin_amdgcn_readlane((int)rest, at),
                           all = (uint32_t)__builtin_amdgcn_readlane((int)tiles, at);
            u.first = (int)(first + (uint32_t)__builtin_amdgcn_readlane((int)(rest_up - rest), at));
            u.parts = (int)(n_full + n_rest);
            u.part = (int)(whole ? unit - first : n_full);
            u.tile0 = u.part * (int)chunk;
            u.tile1 = (int)min((uint32_t)u.tile0 + chunk, all);
            return true;
        }
        full_at = (uint32_t)__builtin_amdgcn_readlane((int)full_up, 63);
        rest_at = (uint32_t)__builtin_amdgcn_readlane((int)rest_up, 63);
    }
    return false;
}

// Which of 32 tokens a row sees, from the one `at` places behind the cached ones: those before are seen, nodes by their set.
__device__ __forceinline__ uint32_t tree_seen(uint64_t line, int at) {
    const uint32_t nodes = at < 64 ? (uint32_t)(line >> (at & 63)) : 0u;
    const uint32_t before = at > -32 ? ((uint32_t)line << (-at & 31)) | ((1u << (-at & 31)) - 1u) : 0xffffffffu;
    return at >= 0 ? nodes : before;
}

// A pair of weights as two bf16 terms each: the upper half of their bits, and the rest, rounded, with 2^-20 of the weight on top: so
// that it is positive too and both products of an infinite value are infinite.
__device__ __forceinline__ uint32_t tree_split(float p0, float p1, uint32_t& rest) {
    const uint32_t b0 = __float_as_uint(p0), b1 = __float_as_uint(p1);
    constexpr float MORE = 1.0f + 0x1p-20f;
    rest = pack_bf16x2(fmaf(p0, MORE, -__uint_as_float(b0 & 0xffff0000u)), fmaf(p1, MORE, -__uint_as_float(b1 & 0xffff0000u)));
    return __builtin_amdgcn_perm(b1, b0, 0x07060302u);
}

__device__ __forceinline__ uint64_t readlane64(uint64_t x, int lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)x, lane);
}

// Which nodes' bf16 values, two a lane, are NaN, infinite, -infinite; those become zeros.
__device__ __forceinline__ void tree_take_broken(uint32_t& v, int node, uint64_t (&bad)[2][3]) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const uint32_t x = v >> (16 * e) & 0xffffu;
        if ((x & 0x7f80u) == 0x7f80u) {
            bad[e][x & 0x7fu ? 0 : x >> 15 ? 2 : 1] |= 1ull << node;
            v &= e ? 0xffffu : 0xffff0000u;
        }
    }
}

// 16 nodes of a (sequence, KV head), four a wave.
__device__ void tree_kv_rows(const TreeAttnArgs& a, uint32_t block) {
    __shared__ uint64_t found[4][TA_D][3];
    constexpr int EACH = TP_NODES / 4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t groups = (a.n + TP_NODES - 1) / TP_NODES, group = block % groups, head = block / groups;
    const uint32_t seq = head / a.nk, h = head % a.nk;
    const int i0 = (int)group * TP_NODES + wave * EACH;
    float k0[EACH], k1[EACH], v0[EACH], v1[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const size_t row = (size_t)seq * a.n + min(i0 + e, (int)a.n - 1);
        const float* kx = a.k_new + row * a.k_row + (size_t)h * TA_D + lane;
        const float* vx = a.v_new + row * a.v_row + (size_t)h * TA_D + 2 * lane;
        k0[e] = kx[0];
        k1[e] = kx[64];
        v0[e] = vx[0];
        v1[e] = vx[1];
    }
    const int len = a.lengths[seq];
    const int count = tree_count_at(a.counts, seq, a.n, len, a.s_cap);
    const uint64_t lines = tree_lineage(a.parents, seq, a.n, count);
    const bool has_w = a.k_norm_w != nullptr;
    const float w0 = has_w ? a.k_norm_w[lane] : 1.0f, w1 = has_w ? a.k_norm_w[lane + 64] : 1.0f;
    const double turns = a.rope ? rope_turns(lane, a.log2_theta) : 0.0;
    uint32_t* const vt = reinterpret_cast<uint32_t*>(a.vt + (size_t)head * (a.n + 1) * TA_D);
    uint64_t bad[2][3] = {{0, 0, 0}, {0, 0, 0}};
    if (group == 0 && wave == 3) vt[a.n * 64 + lane] = 0u;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int i = i0 + e;
        if (i >= (int)a.n) break;
        const uint64_t line = readlane64(lines, i);
        if (line == 0) {
            vt[i * 64 + lane] = 0u;
            continue;
        }
        const size_t slot = ((size_t)len + i) * a.nk + h;
        float cs = 1.0f, sn = 0.0f, r0, r1;
        if (a.rope) rope_at(turns, len + __popcll(line) - 1, cs, sn);
        q8_norm_rope(k0[e], k1[e], has_w, w0, w1, a.eps, cs, sn, r0, r1);
        uint16_t* const y = a.k_cache + seq * a.k_seq + slot * TA_D + lane;
        y[0] = (uint16_t)f32_to_bf16_bits(r0);
        y[64] = (uint16_t)f32_to_bf16_bits(r1);
        uint32_t v = pack_bf16x2(v0[e], v1[e]);
        reinterpret_cast<uint32_t*>(a.v_cache + seq * a.v_seq + slot * TA_D)[lane] = v;
        tree_take_broken(v, i, bad);
        vt[i * 64 + lane] = v;
    }
    const bool any = (bad[0][0] | bad[0][1] | bad[0][2] | bad[1][0] | bad[1][1] | bad[1][2]) != 0;
    const int all = __syncthreads_or(any);
    if (threadIdx.x == 0) a.broken[head * TP_GROUPS + group] = all ? 1u : 0u;
    if (!all) return;
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int k = 0; k < 3; ++k) found[wave][2 * lane + e][k] = bad[e][k];
    __syncthreads();
    for (int i = threadIdx.x; i < TA_D * 3; i += 256) {
        const int d = i / 3, k = i % 3;
        a.which[((size_t)head * TP_GROUPS + group) * TA_D * 3 + i] = found[0][d][k] | found[1][d][k] | found[2][d][k] | found[3][d][k];
    }
}

__device__ void tree_q_rows(const TreeAttnArgs& a, uint64_t unit) {
    const int lane = threadIdx.x & 63;
    const uint32_t parts = (a.nh + TP_HEADS - 1) / TP_HEADS;
    if (unit >= (uint64_t)a.n_seq * a.n * parts) return;
    const uint32_t row = (uint32_t)(unit / parts), h0 = (uint32_t)(unit % parts) * TP_HEADS;
    const uint32_t seq = row / a.n, i = row % a.n;
    float x0[TP_HEADS], x1[TP_HEADS];
#pragma unroll
    for (int j = 0; j < TP_HEADS; ++j) {
        const uint32_t h = h0 + j < a.nh ? h0 + j : h0;
        const float* x = a.q + row * a.q_row + (size_t)h * TA_D;
        x0[j] = x[lane];
        x1[j] = x[lane + 64];
    }
    const int len = a.lengths[seq];
    const int count = tree_count_at(a.counts, seq, a.n, len, a.s_cap);
    const uint64_t line = readlane64(tree_lineage(a.parents, seq, a.n, count), (int)i);
    if (h0 == 0 && lane == 0) a.line[row] = line;
    if (line == 0) return;  // what lies in the workspace stays: it reaches no output
    float cs = 1.0f, sn = 0.0f;
    if (a.rope) rope_at(rope_turns(lane, a.log2_theta), len + __popcll(line) - 1, cs, sn);
    const bool has_w = a.q_norm_w != nullptr;
    const float w0 = has_w ? a.q_norm_w[lane] : 1.0f, w1 = has_w ? a.q_norm_w[lane + 64] : 1.0f;
#pragma unroll
    for (int j = 0; j < TP_HEADS; ++j) {
        const uint32_t h = h0 + j;
        if (h >= a.nh) break;
        float r[2];
        q8_norm_rope(x0[j], x1[j], has_w, w0, w1, a.eps, cs, sn, r[0], r[1]);
        const size_t at = (((size_t)seq * a.nk + h / a.group) * a.n * a.group + i * a.group + h % a.group) * TA_D + lane;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t hi = f32_to_bf16_bits(r[e]);
            a.qh[at + 64 * e] = (uint16_t)hi;
            a.ql[at + 64 * e] = (uint16_t)f32_to_bf16_bits(r[e] - bf16_bits_to_f32(hi));
        }
    }
}

__global__ __launch_bounds__(256) void tree_rows_kernel(const TreeAttnArgs a) {
    if (blockIdx.x == 0) return tree_table(a);
    if (blockIdx.x <= a.kv_blocks) return tree_kv_rows(a, blockIdx.x - 1);
    tree_q_rows(a, (uint64_t)(blockIdx.x - 1 - a.kv_blocks) * 4 + (threadIdx.x >> 6));
}

// ----------------------------------------------------------------------------------------------- the attention --
//
// A thread block takes a unit's tiles of one KV head and the rows (node, q head) of that head, NWR waves of 32 rows by NWK waves
// of 32 keys.  Tiles go straight from the cache into LDS, STAGES of them in turn.
//   * S^T = K . Q^T on v_mfma_f32_32x32x16_bf16, q in two bf16 terms: a lane then holds 16 scores of one row, and their
//     weights, in one bf16 term or two, are the B operand of
//   * O^T += V^T . P^T, whose A operand the transposing LDS read hands out.
// 16-byte pieces of a row lie in LDS at their place XOR f(row), so that neither product's reads meet in a bank: f is the
// row's low four bits for keys (16 rows, one piece each) and twice two of them for values (4 rows, 4 pieces each).
// q's second term costs half as many products again; with one term outputs would be off by half of bf16's step in q.  So would
// they be in the weights, whose sum is of the unrounded ones: 0.0023 of the outputs' size for 0.0017 of their own rounding.  Up to
// 128 rows, what a step with few drafts has, a second term makes them as the one-token step's, whose weights are in 32 bits (us,
// 32 / 8 heads: 12 nodes at 4000 21.0 -> 21.3, 26 at 4100 25.0 -> 25.7, 2 x 26 at 8000 33.7 -> 36.1, 8 x 26 77 -> 86).  More rows
// are bound by the matrix cores, and weights are rounded once there, as a prompt's are (4 x 64 at 15000 113 for 133, 2 x 63 at
// 2000 with 32 / 4 heads 35.0 for 36.7).
// By rows of a KV head (32 / 8 heads, us with all launches): up to 64, 4 waves of keys and 64 KiB tiles twice, 12 nodes at 4000
// 21.3 (as 128 rows 22.4, as 256, rounded once, 22.5); up to 128, 4 times 32 KiB, 26 nodes at 4100 25.7, 8 x 26 at 8000 86 (as
// 256, rounded once: 82); more, 8 times 16 KiB, 4 x 50 to 64 at 15000 114, of which the attention is 95: 850 TFLOP/s of the three
// products.  There the matrix cores are 49 % and the vector units 43 % busy.  The next tile's scores between one's exponentials
// gave the same 97, 64 rows a wave, to halve what is read from LDS, 133: the queries no longer fit the registers that a product
// reads.

// A sum with the values that were zeros in the products.
__device__ __forceinline__ float tree_put_broken(float x, uint64_t nan, uint64_t inf, uint64_t minus) {
    if (nan) x += __uint_as_float(0x7fc00000u);
    if (inf) x += INFINITY;
    if (minus) x -= INFINITY;
    return x;
}

template <int NWR, int NWK, int STAGES>
struct TreeShape {
    static constexpr int WAVES = NWR * NWK, KEYS = 32 * NWK, PER = 16 / NWR;  // loads of 1 KiB a wave and tile
    static constexpr int STAGE = KEYS * 2 * TA_ROW_BYTES;
    static constexpr bool TWO = NWR < 8;  // weights in two terms
    static constexpr int OROW = TA_D + 4;  // fp32 row of the join, padded
    static constexpr int JOIN = WAVES * 32 * OROW * 4;
    static constexpr int LDS = STAGES * STAGE > JOIN ? STAGES * STAGE : JOIN;
};

template <int NWR, int NWK, int STAGES>
__global__ __launch_bounds__(NWR * NWK * 64) __attribute__((amdgpu_waves_per_eu(1, NWR * NWK / 4)))
void tree_attn_kernel(const TreeAttnArgs a) {
    using S = TreeShape<NWR, NWK, STAGES>;
    __shared__ __align__(1024) uint8_t lds[S::LDS];
    __shared__ float wml[S::WAVES][32][2];
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wave % NWR, wk = wave / NWR;
    // the row tiles of a unit one after another on one of the 8 XCDs
    uint32_t rt = 0, uh = blockIdx.x;
    if (a.row_tiles > 1) {
        const uint32_t per = a.n_units * a.nk;
        if (per % 8 == 0) {
            const uint32_t j = blockIdx.x / 8;
            rt = j % a.row_tiles;
            uh = j / a.row_tiles * 8 + blockIdx.x % 8;
        } else {
            rt = blockIdx.x / per;
            uh = blockIdx.x % per;
        }
    }
    const uint32_t unit = uh / a.nk, h = uh % a.nk;
    const TreeUnit u = a.units[unit];
    if (u.seq < 0) return;
    const int group = (int)a.group, len = u.len, rows = u.count * group;  // the sequence's rows of this head
    const int r0 = (int)rt * NWR * 32;
    const size_t head = (size_t)u.seq * a.nk + h;
    const int tiles = rows > r0 ? u.tile1 - u.tile0 : 0;
    const uint16_t* const kb = a.k_cache + u.seq * a.k_seq + (size_t)h * TA_D;
    const uint16_t* const vb = a.v_cache + u.seq * a.v_seq + (size_t)h * TA_D;
    const uint16_t* const vt = a.vt + head * (a.n + 1) * TA_D;
    const size_t step = (size_t)a.nk * TA_D;  // elements from a token to the next

    // loads of this wave: pieces of rows 4 q + lane / 16, q = q0 ..
    const uint32_t base = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)&lds[0]);
    constexpr int HALF = S::PER / 2;
    const int q0 = wave * HALF;
    const int lr = lane >> 4, lp = lane & 15;
    const int kcol = 8 * (lp ^ lr), vcol = 8 * (lp ^ (lr << 2));  // a key's piece also goes by the row's next two bits: 4 (q % 4)
    auto load = [&](int it) {
        const int t0 = (u.tile0 + it) * S::KEYS;
        const uint32_t at = base + (uint32_t)(it % STAGES) * S::STAGE;
        if (t0 + S::KEYS <= len) {
            const uint16_t* const kp = kb + (size_t)(t0 + lr) * step;
            const uint16_t* const vp = vb + (size_t)(t0 + lr) * step + vcol;
#pragma unroll
            for (int i = 0; i < HALF; ++i) {
                const int q = q0 + i;
                lds_dma16(kp + (size_t)(4 * q) * step + (kcol ^ (32 * (q & 3))), at + q * 1024);
            }
#pragma unroll
            for (int i = 0; i < HALF; ++i) {
                const int q = q0 + i;
                lds_dma16(vp + (size_t)(4 * q) * step, at + S::KEYS * TA_ROW_BYTES + q * 1024);
            }
        } else {
            // the tile of the last cached tokens or of nodes: their values come from the copy without what is not finite, and what
            // lies behind them is its row of zeros (keys there: any row of the cache, the scores are masked)
#pragma unroll
            for (int i = 0; i < HALF; ++i) {
                const int q = q0 + i, t = min(t0 + 4 * q + lr, (int)a.s_cap - 1);
                lds_dma16(kb + (size_t)t * step + (kcol ^ (32 * (q & 3))), at + q * 1024);
            }
#pragma unroll
            for (int i = 0; i < HALF; ++i) {
                const int q = q0 + i, t = t0 + 4 * q + lr;
                const uint16_t* const p = t < len ? vb + (size_t)t * step : vt + (size_t)min(t - len, (int)a.n) * TA_D;
                lds_dma16(p + vcol, at + S::KEYS * TA_ROW_BYTES + q * 1024);
            }
        }
    };

    ta_f32x16 o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.0f;
    float m_run = -INFINITY, l_part = 0.0f;
    const int row = r0 + 32 * wr + (lane & 31);  // this lane's
    const bool busy = r0 + 32 * wr < rows;       // whether this wave has any
    if (tiles > 0) {
        load(0);
        const int qr = row < rows ? row : rows - 1;
        const uint16_t* const qhp = a.qh + (head * a.n * group + qr) * TA_D + 8 * half;
        const uint16_t* const qlp = a.ql + (head * a.n * group + qr) * TA_D + 8 * half;
        ta_bf16x8 qh[8], ql[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            qh[s] = *reinterpret_cast<const ta_bf16x8*>(qhp + 16 * s);
            ql[s] = *reinterpret_cast<const ta_bf16x8*>(qlp + 16 * s);
        }
        const uint64_t line = a.line[(size_t)u.seq * a.n + qr / group];
        // (the compiler does not count the loads into LDS: everything that it counts has landed before the loop)
        wait_vm<0>();
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 1; i < STAGES - 1; ++i)
            if (i < tiles) load(i);

        // where this lane reads: a key's row and pieces, a value's 8 bytes in 4 rows (and 8 rows on)
        const int krow = 32 * wk + (lane & 31), n16 = lane & 15;
        const uint32_t ka = (uint32_t)krow * TA_ROW_BYTES;
        const int vr = 32 * wk + 4 * half + (n16 >> 2), vpiece = 2 * ((lane >> 4) & 1) + ((n16 & 3) >> 1);
        const uint32_t va = S::KEYS * TA_ROW_BYTES + (uint32_t)vr * TA_ROW_BYTES + 8 * (n16 & 1);
        for (int it = 0; it < tiles; ++it) {
            const int left = tiles - 1 - it;
            if (left >= STAGES - 2) wait_vm<S::PER * (STAGES - 2)>();
            else wait_vm<0>();
            wait_lgkm0();
            wave_barrier();
            if (it + STAGES - 1 < tiles) load(it + STAGES - 1);
            if (busy) {
                const uint8_t* const stage = &lds[(it % STAGES) * S::STAGE];
                ta_f32x16 s;
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll
                for (int st = 0; st < 8; ++st) {
                    const ta_bf16x8 kf = *reinterpret_cast<const ta_bf16x8*>(stage + ka + (((2 * st + half) ^ (krow & 15)) << 4));
                    s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qh[st], s, 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, ql[st], s, 0, 0, 0);
                }
                const int t0 = (u.tile0 + it) * S::KEYS + 32 * wk;
                if (t0 + 32 > len) {
                    const uint32_t seen = tree_seen(line, t0 + 4 * half - len);
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[e] = seen & 1u << (8 * (e >> 2) + (e & 3)) ? s[e] : -INFINITY;
                }
                float mt = -INFINITY;
#pragma unroll
                for (int e = 0; e < 16; ++e) mt = fmaxf(mt, s[e]);
                mt = xor_max<32>(mt * a.scale_log2);
                const bool grow = mt > m_run + TA_RESCALE;
                const float m_new = grow ? mt : m_run;
                const float alpha = grow ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.0f;
                const float msub = m_new == -INFINITY ? 0.0f : m_new;
                m_run = m_new;
                uint32_t pk[8], pl[8];
                float lsum = 0.0f;
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale_log2, -msub));
                    const float p1 = __builtin_amdgcn_exp2f(fmaf(s[e + 1], a.scale_log2, -msub));
                    lsum += p0 + p1;
                    pk[e / 2] = S::TWO ? tree_split(p0, p1, pl[e / 2]) : pack_bf16x2(p0, p1);
                }
                l_part = fmaf(l_part, alpha, lsum);
                if (__builtin_amdgcn_ballot_w64(grow) != 0) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[i][e] *= alpha;
                }
#pragma unroll
                for (int stp = 0; stp < 2; ++stp) {
                    const ta_bf16x8 pf =
                        __builtin_bit_cast(ta_bf16x8, make_uint4(pk[4 * stp], pk[4 * stp + 1], pk[4 * stp + 2], pk[4 * stp + 3]));
                    ta_bf16x8 pr;
                    if (S::TWO) pr = __builtin_bit_cast(ta_bf16x8, make_uint4(pl[4 * stp], pl[4 * stp + 1], pl[4 * stp + 2], pl[4 * stp + 3]));
                    const uint8_t* const v = stage + va + 16 * stp * TA_ROW_BYTES;
#pragma unroll
                    for (int db = 0; db < 4; ++db) {
                        const uint32_t at = (uint32_t)((4 * db + vpiece) ^ ((vr & 3) << 2)) << 4;
                        const uint2 x = lds_read_tr16_b64(reinterpret_cast<const uint16_t*>(v + at));
                        const uint2 y = lds_read_tr16_b64(reinterpret_cast<const uint16_t*>(v + at + 8 * TA_ROW_BYTES));
                        const ta_bf16x8 vf = __builtin_bit_cast(ta_bf16x8, make_uint4(x.x, x.y, y.x, y.y));
                        o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf, o[db], 0, 0, 0);
                        if (S::TWO) o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pr, o[db], 0, 0, 0);
                    }
                }
            }
        }
    }

    // join the waves of the same rows
    const float l = xor_sum<32>(l_part);
    wait_lgkm0();
    __syncthreads();
    float* const os = reinterpret_cast<float*>(lds);
    if (half == 0) {
        wml[wave][lane][0] = m_run;
        wml[wave][lane][1] = l;
    }
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<ta_f32x4*>(os + (wave * 32 + (lane & 31)) * S::OROW + 32 * db + 8 * g + 4 * half) =
                ta_f32x4{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
    __syncthreads();
    const bool whole = u.parts == 1;
    // values that are not finite were zeros in the products; they come to the rows that see them here, in the nodes' own unit
    const int node0 = max(u.tile0 * S::KEYS - len, 0), node1 = min(u.tile1 * S::KEYS - len, TREE_MAX);
    uint32_t broken = 0;  // groups of nodes
    if (node1 > node0)
        for (uint32_t g = 0; g < (a.n + TP_NODES - 1) / TP_NODES; ++g) broken |= (a.broken[head * TP_GROUPS + g] & 1u) << g;
    const uint64_t here = broken ? (~0ull >> (TREE_MAX - (node1 - node0))) << node0 : 0;
    const int all = (int)a.n * group;  // rows of the output, nodes or not
    for (int i = tid; i < NWR * 32 * 32; i += S::WAVES * 64) {
        const int r = i >> 5, d = (i & 31) * 4, at = r0 + r;
        if (at >= (whole ? all : rows)) break;
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int w = 0; w < NWK; ++w) M = fmaxf(M, wml[w * NWR + (r >> 5)][r & 31][0]);
        const float msub = M == -INFINITY ? 0.0f : M;
        ta_f32x4 sum = ta_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < NWK; ++w) {
            const int from = w * NWR + (r >> 5);
            const float f = __builtin_amdgcn_exp2f(wml[from][r & 31][0] - msub);
            L = fmaf(f, wml[from][r & 31][1], L);
            sum += *reinterpret_cast<const ta_f32x4*>(os + (from * 32 + (r & 31)) * S::OROW + d) * f;
        }
        const int node = at / group;
        const uint64_t line = a.line[(size_t)u.seq * a.n + node];
        for (uint32_t rest = broken; rest; rest &= rest - 1) {
            const uint64_t* const w = a.which + ((head * TP_GROUPS + __builtin_ctz(rest)) * TA_D + d) * 3;
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] = tree_put_broken(sum[e], line & here & w[3 * e], line & here & w[3 * e + 1], line & here & w[3 * e + 2]);
        }
        if (whole) {
            const float inv = line ? 1.0f / L : 0.0f;
            uint2 y = make_uint2(0u, 0u);
            if (line) y = make_uint2(pack_bf16x2(sum[0] * inv, sum[1] * inv), pack_bf16x2(sum[2] * inv, sum[3] * inv));
            *reinterpret_cast<uint2*>(a.out + (((size_t)u.seq * a.n + node) * a.nh + h * group + at % group) * TA_D + d) = y;
        } else {
            const size_t part = ((size_t)(u.first + u.part) * a.nk + h) * a.rows + at;
            *reinterpret_cast<ta_f32x4*>(a.part_o + part * TA_D + d) = sum;
            if (d == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * part) = make_float2(M, L);
        }
    }
}

// Joins the units of a sequence, a wave a row: a lane holds a unit's maximum and sum, and four dims of every other unit's row.
// All of up to 32 units are on their way at once.  5.0 us for 26 nodes of 32 heads and 9.3 for 4 x 64 (33 MB, 3.5 TB/s).
constexpr int TJ_BATCH = 16;

template <int N>
__device__ __forceinline__ void tree_join_rows(const float* part_o, size_t first, size_t step, int p0, int parts, float f, ta_f32x4& o) {
    const int lane = threadIdx.x & 63, half = lane >> 5, d = (lane & 31) * 4;
    ta_f32x4 x[N];
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = *reinterpret_cast<const ta_f32x4*>(part_o + (first + min(p0 + 2 * e + half, parts - 1) * step) * TA_D + d);
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const float f0 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), (p0 + 2 * e) & 63)),
                    f1 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), (p0 + 2 * e + 1) & 63));
        const bool in = p0 + 2 * e + half < parts;
        if (in) o += x[e] * (half ? f1 : f0);
    }
}

__global__ __launch_bounds__(256) void tree_join_kernel(const TreeAttnArgs a) {
    const int lane = threadIdx.x & 63;
    const uint32_t unit = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (unit >= a.n_seq * a.n * a.nh) return;
    const uint32_t seq = unit / (a.n * a.nh), i = unit / a.nh % a.n, head = unit % a.nh, h = head / a.group;
    const int2 parts = a.of_seq[seq];
    const uint64_t line = a.line[(size_t)seq * a.n + i];
    if (parts.y <= 1) return;
    if (line == 0) {
        reinterpret_cast<uint32_t*>(a.out + (size_t)unit * TA_D)[lane] = 0u;
        return;
    }
    const size_t first = ((size_t)parts.x * a.nk + h) * a.rows + (size_t)i * a.group + head % a.group, step = (size_t)a.nk * a.rows;
    float M = -INFINITY, L = 0.0f;
    ta_f32x4 o = ta_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int p0 = 0; p0 < parts.y; p0 += 64) {
        const bool in = p0 + lane < parts.y;
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * (first + min(p0 + lane, parts.y - 1) * step));
        const float m = in ? ml.x : -INFINITY;
        const float now = fmaxf(M, wave_max(m)), msub = now == -INFINITY ? 0.0f : now;
        const float keep = __builtin_amdgcn_exp2f(M - msub), f = in ? __builtin_amdgcn_exp2f(m - msub) : 0.0f;
        L = fmaf(L, keep, wave_sum(in ? f * ml.y : 0.0f));
        o *= keep;
        M = now;
        if (parts.y <= 8) {
            tree_join_rows<4>(a.part_o, first, step, 0, parts.y, f, o);
        } else {
            for (int p = p0; p < min(p0 + 64, parts.y); p += 2 * TJ_BATCH) tree_join_rows<TJ_BATCH>(a.part_o, first, step, p, parts.y, f, o);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = xor_sum<32>(o[e]) / L;
    if (lane < 32)
        *reinterpret_cast<uint2*>(a.out + (size_t)unit * TA_D + lane * 4) = make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
}

// ------------------------------------------------------------------------------------- the attention of few rows --
//
// Up to 32 rows a KV head: all in one launch.  Every thread block norms and rotates the head's queries itself, while its first
// tiles are on their way, and finds its unit in the lengths; the one that holds the nodes also brings their K and V into the
// cache and reads them from LDS.  8 waves, 16 keys each, that wait for nothing but their own loads in the loop: two waves a SIMD
// hide each other's latency.  Both products on v_mfma_f32_16x16x32_bf16 and _16x16x16_, CB blocks of 16 rows as their columns:
// S^T's accumulators hold 4 keys a lane, whose weights, in two bf16 terms (with one 10.2 for 10.6 us at 8 nodes and 500, 68.4 for
// 70.0 at 16 x 5, the same at 32 x 4 and 16000), are the operand of the second product, and a transposing LDS read hands out 4 keys
// of a dim.
// The last unit of a (sequence, KV head) to leave its part joins them: parts go past the caches that the chip's parts do not
// share (agent scope), and are there before the count is raised.
// 32 x 4 nodes at 16000: 360 us, 5.7 TB/s (three launches: 486); 8 at 500: 10.6 us (three launches: 14.8), which is one step
// after another: lengths, the table's sums, queries' norm and angles, a tile, two joins.  16 rows as 32: 23.7 for 19.7 us at 1 x 8
// of 16 / 8 heads at 8000.

constexpr int TF_WAVES = 8, TF_KEYS = 16 * TF_WAVES;
constexpr int TF_QROW = TA_D + 8;  // bf16 row of queries in LDS, padded
constexpr int TF_OROW = TA_D + 4;  // fp32 row of the join, padded
constexpr int TF_STAGE = TF_KEYS * 2 * TA_ROW_BYTES;
constexpr int TF_PART = (TA_D + 4) * 4;  // bytes of a row's part: maximum, sum, nothing, then the row

typedef uint32_t ta_u32x4 __attribute__((ext_vector_type(4)));
typedef short ta_s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t ta_lds;
constexpr int TF_AGENT = 16;  // cache policy of buffer loads and stores: agent scope

template <int CB>
__global__ __launch_bounds__(TF_WAVES * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void tree_few_kernel(const TreeAttnArgs a) {
    constexpr int ROWS = 16 * CB, EACH = ROWS / TF_WAVES;  // rows, and most nodes, of a wave
    constexpr int QS = 2 * ROWS * TF_QROW * 2, ANGLES = ROWS * 64 * 8;
    constexpr bool APART = CB == 1;  // the queries' two terms and the nodes' angles have room of their own, or before the loop the
                                     // second stage's, which is then loaded later
    static_assert(TF_WAVES * ROWS * TF_OROW * 4 <= 2 * TF_STAGE + 4096 * CB, "the join's rows fit the stages");
    constexpr int LDS = TF_WAVES * ROWS * TF_OROW * 4 > 2 * TF_STAGE ? TF_WAVES * ROWS * TF_OROW * 4 : 2 * TF_STAGE;
    __shared__ __align__(1024) uint8_t lds[LDS];
    __shared__ __align__(16) uint8_t own[APART ? QS + ANGLES : 16];
    __shared__ __align__(16) uint8_t fresh[2][(ROWS + 1) * TA_ROW_BYTES];  // the nodes' keys and values, and a row of zeros
    __shared__ float wml[TF_WAVES][ROWS][2];
    __shared__ uint32_t found[TA_D][3], arrived;
    uint16_t* const qs = reinterpret_cast<uint16_t*>(APART ? own : lds + TF_STAGE);
    float2* const angles = reinterpret_cast<float2*>((APART ? own : lds + TF_STAGE) + QS);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t unit = blockIdx.x / a.nk, h = blockIdx.x % a.nk;
    const int group = (int)a.group, all = (int)a.n * group;  // rows of the head, nodes or not
    TreeUnit u;
    if (!tree_find(a, unit, u)) return;  // every wave of the thread block finds the same
    u.seq = __builtin_amdgcn_readfirstlane(u.seq);
    u.tile0 = __builtin_amdgcn_readfirstlane(u.tile0);
    u.tile1 = __builtin_amdgcn_readfirstlane(u.tile1);
    u.first = __builtin_amdgcn_readfirstlane(u.first);
    u.parts = __builtin_amdgcn_readfirstlane(u.parts);
    u.part = __builtin_amdgcn_readfirstlane(u.part);
    const uint32_t seq = (uint32_t)u.seq;
    const int len = __builtin_amdgcn_readfirstlane(u.len), count = __builtin_amdgcn_readfirstlane(u.count);
    const int rows = count * group, tiles = u.tile1 - u.tile0;
    const size_t head = (size_t)seq * a.nk + h;
    const bool has_nodes = u.tile1 * TF_KEYS > len && count > 0;
    const uint16_t* const kb = a.k_cache + seq * a.k_seq + (size_t)h * TA_D;
    const uint16_t* const vb = a.v_cache + seq * a.v_seq + (size_t)h * TA_D;
    const size_t step = (size_t)a.nk * TA_D;

    // the wave's 16 keys and values of a tile, 4 rows a load; 16-byte pieces lie at their place XOR f(row): a key's row's four
    // bits, twice three of a value's row
    const uint32_t base = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(ta_lds*)&lds[0]);
    const int lr = lane >> 4, lp = lane & 15;
    const int kcol = 8 * (lp ^ lr), vcol = 8 * (lp ^ (lr << 1));
    auto load = [&](int it) {
        const int first = (u.tile0 + it) * TF_KEYS + 16 * wave, t0 = first + lr;
        const uint32_t at = __builtin_amdgcn_readfirstlane(base + (uint32_t)(it & 1) * TF_STAGE + wave * 16 * TA_ROW_BYTES);
        if (first + 16 <= len) {
            const uint16_t* const kp = kb + (size_t)t0 * step;
            const uint16_t* const vp = vb + (size_t)t0 * step;
#pragma unroll
            for (int i = 0; i < 4; ++i) lds_dma16(kp + (size_t)(4 * i) * step + (kcol ^ (32 * i)), at + i * 1024);
#pragma unroll
            for (int i = 0; i < 4; ++i) lds_dma16(vp + (size_t)(4 * i) * step + (vcol ^ (64 * (i & 1))), at + TF_KEYS * TA_ROW_BYTES + i * 1024);
        } else {  // rows from the length on are read from `fresh`: here the last slot's stand for them
#pragma unroll
            for (int i = 0; i < 4; ++i) lds_dma16(kb + (size_t)min(t0 + 4 * i, (int)a.s_cap - 1) * step + (kcol ^ (32 * i)), at + i * 1024);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                lds_dma16(vb + (size_t)min(t0 + 4 * i, (int)a.s_cap - 1) * step + (vcol ^ (64 * (i & 1))), at + TF_KEYS * TA_ROW_BYTES + i * 1024);
        }
    };
    // the loads that the prologue waits for, then the tiles'
    float x0[EACH], x1[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int r = min(wave + TF_WAVES * e, all - 1);
        const float* x = a.q + ((size_t)seq * a.n + r / group) * a.q_row + (size_t)(h * group + r % group) * TA_D + lane;
        x0[e] = x[0];
        x1[e] = x[64];
    }
    const bool has_w = a.q_norm_w != nullptr;
    const float qw0 = has_w ? a.q_norm_w[lane] : 1.0f, qw1 = has_w ? a.q_norm_w[lane + 64] : 1.0f;
    float k0[EACH], k1[EACH], v0[EACH], v1[EACH], kw0 = 1.0f, kw1 = 1.0f;
    if (has_nodes) {
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const size_t row = (size_t)seq * a.n + min(wave + TF_WAVES * e, (int)a.n - 1);
            const float* kx = a.k_new + row * a.k_row + (size_t)h * TA_D + lane;
            const float* vx = a.v_new + row * a.v_row + (size_t)h * TA_D + 2 * lane;
            k0[e] = kx[0];
            k1[e] = kx[64];
            v0[e] = vx[0];
            v1[e] = vx[1];
        }
        if (has_w) {
            kw0 = a.k_norm_w[lane];
            kw1 = a.k_norm_w[lane + 64];
        }
    }
    const uint64_t lines = tree_lineage(a.parents, seq, a.n, count);
    if (tiles > 0) load(0);
    if (APART && tiles > 1) load(1);

    // the nodes' angles, then the rows
    if (a.rope && tiles > 0) {
        const double turns = rope_turns(lane, a.log2_theta);
        for (int i = wave; i < count; i += TF_WAVES) {
            float cs, sn;
            rope_at(turns, len + __popcll(readlane64(lines, i)) - 1, cs, sn);
            angles[i * 64 + lane] = make_float2(cs, sn);
        }
    }
    if (has_nodes)
        for (int i = tid; i < TA_D * 3; i += TF_WAVES * 64) found[i / 3][i % 3] = 0u;
    __syncthreads();
    uint64_t bad[2][3] = {{0, 0, 0}, {0, 0, 0}};
    if (tiles > 0) {
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const int r = wave + TF_WAVES * e;
            if (r >= rows) break;
            const float2 angle = a.rope ? angles[r / group * 64 + lane] : make_float2(1.0f, 0.0f);
            float y[2];
            q8_norm_rope(x0[e], x1[e], has_w, qw0, qw1, a.eps, angle.x, angle.y, y[0], y[1]);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t hi = f32_to_bf16_bits(y[k]);
                qs[r * TF_QROW + lane + 64 * k] = (uint16_t)hi;
                qs[(ROWS + r) * TF_QROW + lane + 64 * k] = (uint16_t)f32_to_bf16_bits(y[k] - bf16_bits_to_f32(hi));
            }
        }
        if (has_nodes) {
            // pieces of a row lie where a tile's row of that number has them; rows that are no nodes are zeros
            auto key_at = [&](int i, int d) { return i * TA_D + ((d >> 3 ^ (i & 15)) << 3 | (d & 7)); };
            uint16_t* const fk = reinterpret_cast<uint16_t*>(fresh[0]);
            uint32_t* const fv = reinterpret_cast<uint32_t*>(fresh[1]);
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                const int i = wave + TF_WAVES * e;
                if (i >= (int)a.n) break;
                uint32_t v = 0;
                float r0 = 0.0f, r1 = 0.0f;
                if (readlane64(lines, i)) {
                    const float2 angle = a.rope ? angles[i * 64 + lane] : make_float2(1.0f, 0.0f);
                    q8_norm_rope(k0[e], k1[e], has_w, kw0, kw1, a.eps, angle.x, angle.y, r0, r1);
                    v = pack_bf16x2(v0[e], v1[e]);
                    // (where the nodes lie across two units both have them; one writes)
                    if (len + i >= u.tile0 * TF_KEYS && len + i < u.tile1 * TF_KEYS) {
                        const size_t slot = ((size_t)len + i) * step + (size_t)h * TA_D;
                        uint16_t* const y = a.k_cache + seq * a.k_seq + slot + lane;
                        y[0] = (uint16_t)f32_to_bf16_bits(r0);
                        y[64] = (uint16_t)f32_to_bf16_bits(r1);
                        reinterpret_cast<uint32_t*>(a.v_cache + seq * a.v_seq + slot)[lane] = v;
                    }
                    tree_take_broken(v, i, bad);
                }
                fk[key_at(i, lane)] = (uint16_t)f32_to_bf16_bits(r0);
                fk[key_at(i, lane + 64)] = (uint16_t)f32_to_bf16_bits(r1);
                fv[i * 64 + ((lane >> 2 ^ (i & 7) << 1) << 2 | (lane & 3))] = v;
            }
            if (wave == 0) fv[a.n * 64 + lane] = 0u;
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int k = 0; k < 3; ++k)
                    if (bad[e][k]) atomicOr(&found[2 * lane + e][k], (uint32_t)bad[e][k]);
        }
    }
    const int broken = __syncthreads_or((bad[0][0] | bad[0][1] | bad[0][2] | bad[1][0] | bad[1][1] | bad[1][2]) != 0);

    ta_f32x4 o[CB][8];
    float m_run[CB], l_part[CB];
#pragma unroll
    for (int b = 0; b < CB; ++b) {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[b][i] = ta_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        m_run[b] = -INFINITY;
        l_part[b] = 0.0f;
    }
    if (tiles > 0) {
        // dims 32 s + 8 (lane / 16) .. of row 16 b + lane % 16
        ta_bf16x8 qh[CB][4], ql[CB][4];
        uint32_t line[CB];
#pragma unroll
        for (int b = 0; b < CB; ++b) {
            const int r = min(16 * b + lp, rows - 1);
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                qh[b][s] = *reinterpret_cast<const ta_bf16x8*>(qs + r * TF_QROW + 32 * s + 8 * lr);
                ql[b][s] = *reinterpret_cast<const ta_bf16x8*>(qs + (ROWS + r) * TF_QROW + 32 * s + 8 * lr);
            }
            line[b] = (uint32_t)__shfl((int)lines, r / group);  // up to 32 nodes
        }
        // every load that the compiler counts has landed; the second stage is free
        wait_vm<0>();
        wait_lgkm0();
        asm volatile("" ::: "memory");
        if (!APART) {
            __syncthreads();
            if (tiles > 1) load(1);
        }
        const int vj = 4 * lr + (lp >> 2), vpiece = (lp & 3) >> 1;
        const uint32_t fresh_at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(ta_lds*)&fresh[0][0]);
        for (int it = 0; it < tiles; ++it) {
            const int t0 = (u.tile0 + it) * TF_KEYS + 16 * wave;
            if (it + 1 < tiles) wait_vm<8>();
            else wait_vm<0>();
            asm volatile("" ::: "memory");
            if (t0 < len + count) {
                const bool edge = t0 + 16 > len;
                const uint32_t stage = base + (uint32_t)(it & 1) * TF_STAGE + wave * 16 * TA_ROW_BYTES;
                // where this lane reads: a key's row and a value's, of the tile or of the nodes
                uint32_t ka = stage + (uint32_t)lp * TA_ROW_BYTES, kf = (uint32_t)lp;
                uint32_t va = stage + TF_KEYS * TA_ROW_BYTES + (uint32_t)vj * TA_ROW_BYTES, vf = (uint32_t)vj & 7;
                if (edge) {
                    const int jk = min(t0 + lp - len, (int)a.n), jv = min(t0 + vj - len, (int)a.n);
                    if (jk >= 0) {
                        ka = fresh_at + (uint32_t)jk * TA_ROW_BYTES;
                        kf = (uint32_t)jk & 15;
                    }
                    if (jv >= 0) {
                        va = fresh_at + (uint32_t)(ROWS + 1 + jv) * TA_ROW_BYTES;
                        vf = (uint32_t)jv & 7;
                    }
                }
                ta_bf16x8 kr[4];
#pragma unroll
                for (int s = 0; s < 4; ++s) kr[s] = *(const __attribute__((address_space(3))) ta_bf16x8*)(ta_lds*)(uintptr_t)(ka + (((4 * s + lr) ^ kf) << 4));
                uint2 vr[8];
#pragma unroll
                for (int d = 0; d < 8; ++d) {
                    const uint32_t at = va + (((uint32_t)(2 * d + vpiece) ^ (vf << 1)) << 4) + 8 * (lp & 1);
                    vr[d] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) t2h_v4i16*)(ta_lds*)(uintptr_t)at));
                }
#pragma unroll
                for (int b = 0; b < CB; ++b) {
                    ta_f32x4 sh = ta_f32x4{0.0f, 0.0f, 0.0f, 0.0f}, sl = sh;
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        sh = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kr[s], qh[b][s], sh, 0, 0, 0);
                        sl = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kr[s], ql[b][s], sl, 0, 0, 0);
                    }
                    sh += sl;
                    if (edge) {
                        const uint32_t seen = tree_seen(line[b], t0 + 4 * lr - len);
#pragma unroll
                        for (int e = 0; e < 4; ++e) sh[e] = seen & 1u << e ? sh[e] : -INFINITY;
                    }
                    float mt = fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3])) * a.scale_log2;
                    mt = xor_max<32>(xor_max<16>(mt));
                    const bool grow = mt > m_run[b] + TA_RESCALE;
                    const float m_new = grow ? mt : m_run[b], alpha = grow ? __builtin_amdgcn_exp2f(m_run[b] - m_new) : 1.0f;
                    const float msub = m_new == -INFINITY ? 0.0f : m_new;
                    m_run[b] = m_new;
                    float pe[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) pe[e] = __builtin_amdgcn_exp2f(fmaf(sh[e], a.scale_log2, -msub));
                    l_part[b] = fmaf(l_part[b], alpha, (pe[0] + pe[1]) + (pe[2] + pe[3]));
                    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) o[b][i] *= alpha;
                    }
                    uint2 ph, pl;
                    ph.x = tree_split(pe[0], pe[1], pl.x);
                    ph.y = tree_split(pe[2], pe[3], pl.y);
#pragma unroll
                    for (int d = 0; d < 8; ++d) {
                        const ta_s16x4 vf = __builtin_bit_cast(ta_s16x4, vr[d]);
                        o[b][d] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(vf, __builtin_bit_cast(ta_s16x4, ph), o[b][d], 0, 0, 0);
                        o[b][d] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(vf, __builtin_bit_cast(ta_s16x4, pl), o[b][d], 0, 0, 0);
                    }
                }
            }
            wait_lgkm0();  // the buffer is read before it is loaded again
            asm volatile("" ::: "memory");
            if (it + 2 < tiles) load(it + 2);
        }
    }

    // join the waves: lane holds dims 16 d + 4 (lane / 16) .. of row 16 b + lane % 16
    wait_lgkm0();
    __syncthreads();
    float* const os = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int b = 0; b < CB; ++b) {
        const float l = xor_sum<32>(xor_sum<16>(l_part[b]));
        if (lr == 0) {
            wml[wave][16 * b + lp][0] = m_run[b];
            wml[wave][16 * b + lp][1] = l;
        }
#pragma unroll
        for (int d = 0; d < 8; ++d) *reinterpret_cast<ta_f32x4*>(os + (wave * ROWS + 16 * b + lp) * TF_OROW + 16 * d + 4 * lr) = o[b][d];
    }
    __syncthreads();
    const bool whole = u.parts == 1;
    const int node0 = max(u.tile0 * TF_KEYS - len, 0), node1 = min(u.tile1 * TF_KEYS - len, 32);
    const uint32_t here = broken && node1 > node0 ? (~0u >> (32 - (node1 - node0))) << node0 : 0;
    auto put = [&](int r, int d, ta_f32x4 sum, float L, bool node) {
        uint2 y = make_uint2(0u, 0u);
        if (node) {
            const float inv = 1.0f / L;
            y = make_uint2(pack_bf16x2(sum[0] * inv, sum[1] * inv), pack_bf16x2(sum[2] * inv, sum[3] * inv));
        }
        *reinterpret_cast<uint2*>(a.out + (((size_t)seq * a.n + r / group) * a.nh + h * group + r % group) * TA_D + d) = y;
    };
    // this (sequence, head)'s parts, rows of ROWS each
    constexpr int PART = ROWS * TF_PART;
    uint8_t* const parts = reinterpret_cast<uint8_t*>(a.part_o) + ((size_t)u.first * a.nk + (size_t)h * u.parts) * PART;
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(parts, 0, u.parts * PART, 0x00027000);
    for (int i = tid; i < ROWS * 32; i += TF_WAVES * 64) {
        const int r = i >> 5, d = (i & 31) * 4;
        if (r >= (whole ? all : rows)) break;
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int w = 0; w < TF_WAVES; ++w) M = fmaxf(M, wml[w][r][0]);
        const float msub = M == -INFINITY ? 0.0f : M;
        ta_f32x4 sum = ta_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < TF_WAVES; ++w) {
            const float f = __builtin_amdgcn_exp2f(wml[w][r][0] - msub);
            L = fmaf(f, wml[w][r][1], L);
            sum += *reinterpret_cast<const ta_f32x4*>(os + (w * ROWS + r) * TF_OROW + d) * f;
        }
        const uint32_t line = (uint32_t)__shfl((int)lines, r / group);  // (of a wave's two rows the first one's lanes are there)
        if (line & here) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                sum[e] = tree_put_broken(sum[e], line & here & found[d + e][0], line & here & found[d + e][1], line & here & found[d + e][2]);
        }
        if (whole) {
            put(r, d, sum, L, line != 0);
        } else {
            const int at = u.part * PART + r * TF_PART;
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(ta_u32x4, sum), rsrc, at + 16 + d * 4, 0, TF_AGENT);
            if (d == 0) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(ta_u32x4, ta_f32x4{M, L, 0.0f, 0.0f}), rsrc, at, 0, TF_AGENT);
        }
    }
    if (whole) return;
    __builtin_amdgcn_s_waitcnt(0);
    asm volatile("" ::: "memory");
    __syncthreads();
    if (tid == 0) {
        arrived = __hip_atomic_fetch_add(&a.done[head], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u;
        if (arrived == (uint32_t)u.parts) __hip_atomic_store(&a.done[head], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (arrived != (uint32_t)u.parts) return;
    // slices of the parts, where rows are few; 8 parts of a slice on their way at a time
    const int pieces = rows * 32, slices = TF_WAVES * 64 / pieces > 0 ? TF_WAVES * 64 / pieces : 1;
    constexpr int BATCH = 8, TURNS = (ROWS * 32 + TF_WAVES * 64 - 1) / (TF_WAVES * 64);
    float M[TURNS], L[TURNS];
    ta_f32x4 sum[TURNS];
#pragma unroll
    for (int k = 0; k < TURNS; ++k) {
        M[k] = -INFINITY;
        L[k] = 0.0f;
        sum[k] = ta_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const int slice = tid / pieces;  // (in one turn only where there are several)
    for (int n0 = slice; n0 < u.parts && slice < slices; n0 += slices * BATCH) {
        ta_u32x4 ml[TURNS][BATCH], x[TURNS][BATCH];
#pragma unroll
        for (int k = 0; k < TURNS; ++k) {
            const int i = min(tid - slice * pieces + k * TF_WAVES * 64, pieces - 1);
#pragma unroll
            for (int e = 0; e < BATCH; ++e) {
                const int at = min(n0 + slices * e, u.parts - 1) * PART + (i >> 5) * TF_PART;
                ml[k][e] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, TF_AGENT);
                x[k][e] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, at + 16 + (i & 31) * 16, 0, TF_AGENT);
            }
        }
#pragma unroll
        for (int k = 0; k < TURNS; ++k)
#pragma unroll
            for (int e = 0; e < BATCH; ++e) {
                if (n0 + slices * e >= u.parts) break;
                const ta_f32x4 q = __builtin_bit_cast(ta_f32x4, ml[k][e]);
                const float now = fmaxf(M[k], q[0]), msub = now == -INFINITY ? 0.0f : now;
                const float keep = __builtin_amdgcn_exp2f(M[k] - msub), f = __builtin_amdgcn_exp2f(q[0] - msub);
                L[k] = fmaf(L[k], keep, f * q[1]);
                sum[k] = sum[k] * keep + __builtin_bit_cast(ta_f32x4, x[k][e]) * f;
                M[k] = now;
            }
    }
    if (slices == 1) {
#pragma unroll
        for (int k = 0; k < TURNS; ++k) {
            const int i = tid + k * TF_WAVES * 64;
            const bool node = __shfl((int)lines, min(i, pieces - 1) / 32 / group) != 0;
            if (i < pieces) put(i >> 5, (i & 31) * 4, sum[k], L[k], node);
        }
    } else {
        const int i = tid - slice * pieces, r = i >> 5, d = (i & 31) * 4;
        if (slice < slices) {
            *reinterpret_cast<ta_f32x4*>(os + (slice * rows + r) * TF_OROW + d) = sum[0];  // (slices times rows are up to 16)
            if (d == 0) {
                wml[slice & 7][(slice >> 3) * 8 + r][0] = M[0];
                wml[slice & 7][(slice >> 3) * 8 + r][1] = L[0];
            }
        }
        __syncthreads();
        if (tid < pieces) {
            float top = -INFINITY, under = 0.0f;
            for (int n = 0; n < slices; ++n) top = fmaxf(top, wml[n & 7][(n >> 3) * 8 + r][0]);
            const float msub = top == -INFINITY ? 0.0f : top;
            ta_f32x4 y = ta_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            for (int n = 0; n < slices; ++n) {
                const float f = __builtin_amdgcn_exp2f(wml[n & 7][(n >> 3) * 8 + r][0] - msub);
                under = fmaf(f, wml[n & 7][(n >> 3) * 8 + r][1], under);
                y += *reinterpret_cast<const ta_f32x4*>(os + (n * rows + r) * TF_OROW + d) * f;
            }
            put(r, d, y, under, __shfl((int)lines, r / group) != 0);
        }
    }
    // rows that are no nodes
    for (int i = rows * 32 + tid; i < all * 32; i += TF_WAVES * 64) put(i / 32, i % 32 * 4, ta_f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 1.0f, false);
}

// ------------------------------------------------------------------------------------------------------ launch --

// Rows of a KV head that one thread block takes: 16, 32, 64, 128 or 256, for more of them several.
static uint32_t ta_tile_rows(uint32_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256; }

struct TreeSizes {
    uint32_t tile_rows, row_tiles, rows, keys, least, units;
    float us_turn, us_tile, us_shared, us_join, us_part;
    size_t done, qh, ql, line, vt, broken, which, table, of_seq, part_ml, part_o, end;
};

static TreeSizes ta_sizes(uint32_t n_seq, uint32_t n, uint32_t nh, uint32_t nk, uint32_t s_cap) {
    TreeSizes s = {};
    const uint32_t rows = n * (nh / nk);
    s.tile_rows = ta_tile_rows(rows);
    s.row_tiles = (rows + s.tile_rows - 1) / s.tile_rows;
    s.rows = s.row_tiles * s.tile_rows;
    s.keys = s.tile_rows <= 64 ? 128 : s.tile_rows == 128 ? 64 : 32;
    s.least = s.tile_rows <= 64 ? 1 : s.tile_rows == 128 ? 4 : 8;
    // measured, in us (a tile of 64 KiB a CU where all read: 6.4 TB/s)
    s.us_shared = 2.6f * (float)s.keys / 128.0f;
    s.us_turn = s.tile_rows <= 16 ? 8.0f : s.tile_rows == 32 ? 10.0f : 9.0f;
    s.us_tile = s.tile_rows <= 16 ? 0.7f : s.tile_rows == 32 ? 1.0f : s.tile_rows == 64 ? 1.2f : s.tile_rows == 128 ? 0.62f : 1.05f;
    s.us_join = s.tile_rows <= 16 ? 1.3f : 2.0f;
    s.us_part = s.tile_rows <= 16 ? 0.35f : s.tile_rows == 32 ? 0.4f : 0.05f;
    const uint32_t slots = TA_CUS / (nk * s.row_tiles) > 1 ? TA_CUS / (nk * s.row_tiles) : 1;
    const uint64_t most = (uint64_t)n_seq * ((s_cap + s.keys - 1) / s.keys), some = slots > n_seq + slots / 2 ? slots : n_seq + slots / 2;
    s.units = (uint32_t)(most < some ? most : some);
    size_t at = 0;
    const size_t counters = (size_t)n_seq * nk;  // first, and as many for every shape up to 16384 of them: calls may share a workspace
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    const size_t q = (size_t)n_seq * n * nh * TA_D * 2, heads = (size_t)n_seq * nk, parts = (size_t)s.units * nk * s.rows;
    s.done = take((counters > 16384 ? counters : 16384) * 4);
    if (s.tile_rows <= 32) {  // one launch
        s.part_o = take(parts * (TA_D + 4) * 4);
        s.end = at;
        return s;
    }
    s.qh = take(q);
    s.ql = take(q);
    s.line = take((size_t)n_seq * n * 8);
    s.vt = take(heads * (n + 1) * TA_D * 2);
    s.broken = take(heads * TP_GROUPS * 4);
    s.which = take(heads * TP_GROUPS * TA_D * 24);
    s.table = take((size_t)s.units * sizeof(TreeUnit));
    s.of_seq = take((size_t)n_seq * 8);
    s.part_ml = take(parts * 8);
    s.part_o = take(parts * TA_D * 4);
    s.end = at;
    return s;
}

}  // namespace t2h

using namespace t2h;

static bool ta_shape(uint32_t n_seq, uint32_t n, uint32_t nh, uint32_t nk, uint32_t s_cap) {
    return n_seq != 0 && n <= (uint32_t)TREE_MAX && nk != 0 && nh != 0 && nh % nk == 0 && s_cap != 0 && s_cap <= TA_MOST;
}

extern "C" size_t t2h_attn_tree_workspace_bytes(uint32_t n_seq, uint32_t n, uint32_t nh, uint32_t nk, uint32_t d,
                                                uint32_t s_cap) {
    if (!ta_shape(n_seq, n, nh, nk, s_cap) || n == 0 || nh / nk > TA_MAX_GROUP || d != TA_D) return 0;
    return ta_sizes(n_seq, n, nh, nk, s_cap).end;
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
    const TreeSizes s = ta_sizes(n_seq, n, nh, nk, s_cap);
    if (workspace_bytes < s.end) return T2H_ERR_WORKSPACE;
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
    uint8_t* const ws = reinterpret_cast<uint8_t*>(workspace);
    a.done = reinterpret_cast<uint32_t*>(ws + s.done);
    a.qh = reinterpret_cast<uint16_t*>(ws + s.qh);
    a.ql = reinterpret_cast<uint16_t*>(ws + s.ql);
    a.line = reinterpret_cast<uint64_t*>(ws + s.line);
    a.vt = reinterpret_cast<uint16_t*>(ws + s.vt);
    a.broken = reinterpret_cast<uint32_t*>(ws + s.broken);
    a.which = reinterpret_cast<uint64_t*>(ws + s.which);
    a.units = reinterpret_cast<TreeUnit*>(ws + s.table);
    a.of_seq = reinterpret_cast<int2*>(ws + s.of_seq);
    a.part_ml = reinterpret_cast<float*>(ws + s.part_ml);
    a.part_o = reinterpret_cast<float*>(ws + s.part_o);
    a.n_units = s.units;
    a.row_tiles = s.row_tiles;
    a.rows = s.rows;
    a.keys = s.keys;
    a.least = s.least;
    a.us_turn = s.us_turn;
    a.us_tile = s.us_tile;
    a.us_shared = s.us_shared;
    a.us_join = s.us_join;
    a.us_part = s.us_part;
    const uint64_t waves = (uint64_t)n_seq * n * ((nh + TP_HEADS - 1) / TP_HEADS), kv = (uint64_t)n_seq * nk * ((n + TP_NODES - 1) / TP_NODES);
    const uint64_t grid = (uint64_t)s.units * nk * s.row_tiles, joins = ((uint64_t)n_seq * n * nh + 3) / 4;
    if (kv + waves > 0x3fffffffu || grid > 0x7fffffffu || joins > 0x3fffffffu) return T2H_ERR_SHAPE;
    a.kv_blocks = (uint32_t)kv;
    a.q_blocks = (uint32_t)((waves + 3) / 4);
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const dim3 g((uint32_t)grid);
    if (s.tile_rows <= 32) {
        if (s.tile_rows == 16) hipLaunchKernelGGL(tree_few_kernel<1>, g, dim3(TF_WAVES * 64), 0, st, a);
        else hipLaunchKernelGGL(tree_few_kernel<2>, g, dim3(TF_WAVES * 64), 0, st, a);
        T2H_LAUNCH_CHECK();
        return T2H_OK;
    }
    hipLaunchKernelGGL(tree_rows_kernel, dim3(1 + a.kv_blocks + a.q_blocks), dim3(256), 0, st, a);
    T2H_LAUNCH_CHECK();
    if (s.tile_rows == 64) hipLaunchKernelGGL((tree_attn_kernel<2, 4, 2>), g, dim3(512), 0, st, a);
    else if (s.tile_rows == 128) hipLaunchKernelGGL((tree_attn_kernel<4, 2, 4>), g, dim3(512), 0, st, a);
    else hipLaunchKernelGGL((tree_attn_kernel<8, 1, 8>), g, dim3(512), 0, st, a);
    T2H_LAUNCH_CHECK();
    if (s.units > n_seq) {
        hipLaunchKernelGGL(tree_join_kernel, dim3((uint32_t)joins), dim3(256), 0, st, a);
        T2H_LAUNCH_CHECK();
    }
    return T2H_OK;
}
