// Which drafted tokens of a tree the target's probabilities accept, the token that follows them, and the accepted nodes' rows
// in the cache (definitions: include/t2h.h, "trees of drafted tokens").
#include <math.h>
#include <type_traits>

#include "tree.h"

namespace t2h {

// ------------------------------------------------------------------------------------------------ verification --
//
// Two launches.  The first reads every node's row of logits once, a wave a piece of E * 64 of them, and leaves the piece's largest
// logit and the sum of exp((l - largest) / T), or where that logit is.  In the second every thread block joins the rows' pieces
// and walks down the tree; then its waves sum their segments of the row where the walk ended, and the last thread block of a
// sequence to get there draws the next token: the segment in which the running sum passes the border, then its logits.
// The borders between the tokens of a large vocabulary lie 10^-5 of the sum apart: that row's sums and exponentials are in 64
// bits (relative errors of 10^-12), since 32 would now and then draw a token's neighbour.
// The first launch's exponentials and a piece's sum are in 32 bits, which decides a child's acceptance wherever its number lies
// further from the border than they are off (V_OFF).  Nearer than that, or where rejected children leave so little of the row
// that the difference of two such sums says nothing, all waves sum what is left of the row in 64 bits, and that decides: one
// decision in 10^4 at random numbers, for 35 us, 65 with a draft's row.
// Where drafts are drawn the next token's mass is max(p - q, 0) = max(w / Z - v / Y, 0), and Z / Y is known from 32-bit sums only
// when the second pass begins.  The sums of w and v of the tokens that have any mass by that, and of all w and v, are kept apart;
// the last thread block has Z / Y in 64 bits.  Segments with a token whose w / v lies within V_BAND of the former, one in 10^3
// where rows are not nearly alike, are marked and summed again by the latter, all of them where the two lie further apart.
// The first launch is bound by HBM where rows are many (32 x 16 of 151936 in fp32: 42 us, 5.8 TB/s), else by its latency (8 rows
// 3.4 us).  The second is latency: pieces, walk, the row again, the join of its sums and a segment, one after another: 3.7 us
// where it is greedy, 12.4 drawn, 21.6 with drafts' rows for 16 sequences.  All rows in 64 bits took 31 us for 15.7 with 26 nodes.

struct VerifyArgs {
    const void* logits;
    const void* draft;
    size_t row_stride, draft_stride;
    const int64_t* tokens;
    const int32_t* parents;
    const int32_t* counts;
    const float* uniforms;
    float temperature;
    const float* temperatures;
    int32_t* path;
    int32_t* kept;
    int64_t* next_token;
    uint32_t n, n_seq, vocab;
    uint32_t pieces;  // of a row
    uint2* part;      // [rows][pieces], the draft's rows behind the target's: bits of the largest logit; of the sum, or its index
    uint32_t chunks;  // thread blocks a sequence in the second launch, of per_block segments
    uint32_t per_block;
    uint32_t* done;   // [n_seq] of those that have left their sums; zero between calls
    double* left;     // [n_seq][segments][4] sums of the row where the walk ended
};

constexpr int V_TABLE = 32;

// 2^(j / 32)
__device__ const double V_POWERS[V_TABLE] = {
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002,
};

// exp(y ln 2 / 32) of N numbers y <= 0: 2^(j / 32) from the table, and the Taylor series of what is left, |z| <= ln 2 / 64, up to
// z^4 (the next term is 10^-12).  What is less than 2^-1000, and NaN, gives 0.
template <int N>
__device__ __forceinline__ void exp_steps(double (&y)[N], const double* table) {
    constexpr double C = 0.02166084939249829;     // ln 2 / 32
    constexpr double MAGIC = 6755399441055744.0;  // 1.5 2^52: a sum with it is rounded to a whole number, in its low word
    int steps[N];
    double power[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        y[e] = fmax(y[e], -32001.0);
        const double z = y[e] + MAGIC;
        y[e] -= z - MAGIC;
        steps[e] = (int)__double2loint(z);
        power[e] = table[steps[e] & (V_TABLE - 1)];
    }
    __builtin_amdgcn_sched_barrier(0);  // (the table's reads all on their way)
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const double r = y[e];
        double p = fma(C * C * C * C / 24.0, r, C * C * C / 6.0);
        p = fma(p, r, C * C / 2.0);
        p = fma(p, r, C);
        p = fma(p, r, 1.0) * power[e];
        y[e] = steps[e] <= -32000 ? 0.0 : __hiloint2double(__double2hiint(p) + ((steps[e] >> 5) << 20), __double2loint(p));
    }
}

__device__ __forceinline__ float verify_temperature(const VerifyArgs& a, uint32_t seq) {  // 0: greedy
    const float t = a.temperatures ? a.temperatures[seq] : a.temperature;
    return t > 0.0f ? t : 0.0f;
}
__device__ __forceinline__ double verify_steps(float t) { return 46.16624130844683 / (double)t; }
__device__ __forceinline__ float verify_factor(float t) { return fminf(1.4426950408889634f / t, 3.4e38f); }

template <bool BF16>
__device__ __forceinline__ float verify_logit(const void* base, size_t at) {
    return BF16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(base)[at]) : static_cast<const float*>(base)[at];
}

template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_f64(double v) {
    return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, ROWS, 0xf, false),
                            __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ double readlane_f64(double x, int lane) {
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(x), lane), __builtin_amdgcn_readlane(__double2loint(x), lane));
}

// Sums over the lanes up to each: within rows of 16, then over the rows.
__device__ __forceinline__ double wave_scan_f64(double v) {
    v += dpp_f64<0x111, 0xf>(v);  // 1 lane up
    v += dpp_f64<0x112, 0xf>(v);
    v += dpp_f64<0x114, 0xf>(v);
    v += dpp_f64<0x118, 0xf>(v);
    v += dpp_f64<0x142, 0xa>(v);  // a row's last lane to the odd rows
    v += dpp_f64<0x143, 0xc>(v);  // lane 31 to the upper half
    return v;
}
__device__ __forceinline__ double wave_sum_f64(double v) { return readlane_f64(wave_scan_f64(v), 63); }
__device__ __forceinline__ uint32_t wave_min_u32(uint32_t v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = min(v, (uint32_t)__shfl_xor((int)v, off));
    return v;
}

template <bool BF16, int E>
__global__ __launch_bounds__(256) void verify_rows_kernel(const VerifyArgs a) {
    constexpr int PER = BF16 ? 8 : 4, LOADS = E / PER;  // logits a load of 16 bytes
    const int lane = threadIdx.x & 63;
    const uint32_t unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t r = unit / a.pieces, piece = unit % a.pieces, rows = a.n_seq * a.n;
    const bool draft = r >= rows;
    if (r >= rows + (a.draft ? a.n_seq * (a.n - 1) : 0)) return;
    const uint32_t per = draft ? a.n - 1 : a.n, row = draft ? r - rows : r, seq = row / per;
    const uint8_t* const base = draft ? static_cast<const uint8_t*>(a.draft) + (size_t)row * a.draft_stride * (BF16 ? 2 : 4)
                                      : static_cast<const uint8_t*>(a.logits) + (size_t)row * a.row_stride * (BF16 ? 2 : 4);
    if ((int)(row % per) >= tree_count(a.counts, seq, a.n) - (draft ? 1 : 0)) return;
    const float t = verify_temperature(a, seq);
    const uint32_t first = piece * (E * 64) + lane * PER;
    float x[E];
    if ((piece + 1) * (E * 64) <= a.vocab) {
        uint4 w[LOADS];
#pragma unroll
        for (int v = 0; v < LOADS; ++v) w[v] = load_u4_ua(base + (size_t)(first + v * (64 * PER)) * (BF16 ? 2 : 4));
#pragma unroll
        for (int v = 0; v < LOADS; ++v) {
            const uint32_t words[4] = {w[v].x, w[v].y, w[v].z, w[v].w};
#pragma unroll
            for (int e = 0; e < PER; ++e)
                x[v * PER + e] = BF16 ? __uint_as_float(e & 1 ? words[e / 2] & 0xffff0000u : words[e / 2] << 16) : __uint_as_float(words[e & 3]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t at = first + (e / PER) * (64 * PER) + e % PER;
            x[e] = verify_logit<BF16>(base, min(at, a.vocab - 1));  // (no load waits for another)
        }
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (first + (e / PER) * (64 * PER) + e % PER >= a.vocab) x[e] = -INFINITY;
    }
    float top = -INFINITY;  // (of a NaN and a number the number)
#pragma unroll
    for (int e = 0; e < E; ++e) top = fmaxf(top, x[e]);
    top = wave_max(top);
    uint32_t second;
    if (t == 0.0f) {
        second = 0xffffffffu;
#pragma unroll
        for (int e = E - 1; e >= 0; --e)
            if (x[e] == top) second = first + (e / PER) * (64 * PER) + e % PER;
        second = wave_min_u32(second);
    } else {
        float sum = 0.0f;  // up to 64 terms a lane: as good as its terms
        if (top == INFINITY) {
#pragma unroll
            for (int e = 0; e < E; ++e) sum += x[e] == INFINITY ? 1.0f : 0.0f;
        } else if (top > -INFINITY) {
            const float c = verify_factor(t);
#pragma unroll
            for (int e = 0; e < E; ++e) sum += __builtin_amdgcn_exp2f(fmaxf((x[e] - top) * c, -200.0f));
        }
        second = __float_as_uint(wave_sum(sum));
    }
    if (lane == 0) a.part[(size_t)r * a.pieces + piece] = make_uint2(__float_as_uint(top), second);
}

// Relative errors of the 32-bit exponentials and sums, in units of 2^-24: an exponent of -a (to the base 2) is off by 4 of its own
// roundings, 2.8 a in the exponential, which has 2 more.  In a sum over up to 2^31 tokens the mean of a by weight is at most 31
// (what the row lacks of the largest entropy); up to 63 additions a lane, 6 across, a product for each of two steps: 170.  One
// weight: a up to 100, 282.  Those below 2^-100 of the largest are taken as unknown.
constexpr double V_OFF = 0x1p-15, V_SMALL = 0x1p-100;
// and of those in 64 bits: 1.2 10^-12 of the series, and additions
constexpr double V_OFF64 = 0x1p-36;
// The quotient of two rows' 32-bit sums is off by up to 2 10^-7 (rows of 1000 to 151936, spreads of 0.01 to 5, temperatures of 0.3
// to 1.5), a tenth of this; where it is off by more than half of it, that is seen.
constexpr double V_BAND = 0x1p-19;

constexpr int VF_WAVES = 16, VF_THREADS = VF_WAVES * 64;
constexpr int VF_EACH = 8;                        // logits a lane
constexpr uint32_t VF_SEGMENT = 64 * VF_EACH;     // a wave

struct VerifyState {
    float top[2 * TREE_MAX];   // the rows' largest logits, the draft's behind the target's
    double sum[2 * TREE_MAX];  // and sums
    int64_t best[TREE_MAX];
    int gone[TREE_MAX];        // tokens that the walk rejected where it ended
    int n_gone, cur, kept;
    bool asks;                 // whether the walk waits for the row's sums in 64 bits
    double w[VF_WAVES], v[VF_WAVES];  // those, wave by wave
    double u;                  // the number that draws the next token
};

__device__ __forceinline__ int64_t readlane_i64(int64_t x, int lane) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 |
                     (uint32_t)__builtin_amdgcn_readlane((int)x, lane));
}

// Rows' largest logits and sums, or those logits' indexes, from their pieces: a wave two rows at a time.
__device__ __forceinline__ void verify_join(const VerifyArgs& a, uint32_t seq, int count, int rows, float t, VerifyState& st) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr int AHEAD = 3;  // 64 pieces each: those of 151936 logits, where they are small
    const float c = t > 0.0f ? verify_factor(t) : 0.0f;
    for (int i0 = wave; i0 < rows; i0 += 2 * VF_WAVES) {
        uint2 p[2][AHEAD];
        const uint2* part[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int i = min(i0 + k * VF_WAVES, rows - 1);
            const size_t row = i < count ? (size_t)seq * a.n + i : (size_t)a.n_seq * a.n + (size_t)seq * (a.n - 1) + (i - count);
            part[k] = a.part + row * a.pieces;
#pragma unroll
            for (int g = 0; g < AHEAD; ++g) p[k][g] = part[k][min((uint32_t)(lane + 64 * g), a.pieces - 1)];
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int i = i0 + k * VF_WAVES;
            if (i >= rows) break;
            float top = -INFINITY;
#pragma unroll
            for (int g = 0; g < AHEAD; ++g) top = fmaxf(top, __uint_as_float(p[k][g].x));
            for (uint32_t q = lane + 64 * AHEAD; q < a.pieces; q += 64) top = fmaxf(top, __uint_as_float(part[k][q].x));
            top = wave_max(top);
            double sum = 0.0;
            uint32_t best = 0xffffffffu;
            auto add = [&](uint2 q, bool in) {
                const float x = __uint_as_float(q.x);
                if (t == 0.0f) {
                    if (x == top) best = min(best, q.y);  // (a piece twice is no harm here)
                } else {
                    const float w = top == INFINITY ? (x == INFINITY ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(fmaxf((x - top) * c, -200.0f));
                    sum += in && x > -INFINITY ? (double)(__uint_as_float(q.y) * w) : 0.0;
                }
            };
#pragma unroll
            for (int g = 0; g < AHEAD; ++g) add(p[k][g], (uint32_t)(lane + 64 * g) < a.pieces);
            for (uint32_t q = lane + 64 * AHEAD; q < a.pieces; q += 64) add(part[k][q], true);
            if (t == 0.0f) best = wave_min_u32(best);
            else sum = wave_sum_f64(sum);
            if (lane == 0) {
                const int to = i < count ? i : TREE_MAX + i - count;
                st.top[to] = top;
                st.sum[to] = sum;
                if (i < count) st.best[i] = top == -INFINITY ? -1 : (int64_t)best;
            }
        }
    }
}

// A node as a lane of the walking wave sees it, with the logits of its token after its parent.
struct VerifyNode {
    int up;
    int64_t token;
    float x, y, u;
};

template <bool BF16, bool DRAWN>
__device__ __forceinline__ VerifyNode verify_node(const VerifyArgs& a, uint32_t seq, int count, float t) {
    const int lane = threadIdx.x & 63;
    VerifyNode v = {lane - 1, -1, -INFINITY, -INFINITY, 0.0f};
    if (lane >= count) return v;
    const size_t at = (size_t)seq * a.n + lane;
    v.token = a.tokens[at];
    if (a.parents) v.up = a.parents[at];
    if (t == 0.0f) return v;
    v.u = fminf(fmaxf(a.uniforms[at], 0.0f), 0.99999994f);  // NaN as 0
    if (v.up >= 0 && v.up < lane && v.token >= 0 && v.token < (int64_t)a.vocab) {
        v.x = verify_logit<BF16>(a.logits, ((size_t)seq * a.n + v.up) * a.row_stride + v.token);
        if (DRAWN) v.y = verify_logit<BF16>(a.draft, ((size_t)seq * (a.n - 1) + v.up) * a.draft_stride + v.token);
    }
    return v;
}

// exp((x - top) / T) in 32 bits, as the sums have it.
__device__ __forceinline__ double verify_share(float x, float top, double sum, float c) {
    if (!(x > -INFINITY) || !(sum > 0.0)) return 0.0;
    return (double)(top == INFINITY ? (x == INFINITY ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(fmaxf((x - top) * c, -200.0f)));
}

// A logit's exp((x - top) / T) in 64 bits, bit for bit as a pass over its row has it.
__device__ __forceinline__ double verify_weight(float x, float top, double steps, const double* table) {
    if (top == INFINITY) return x == INFINITY ? 1.0 : 0.0;
    double y[1] = {((double)x - (double)top) * steps};
    exp_steps(y, table);
    return y[0];
}

// How far a walk has come.
struct VerifyPath {
    int cur, kept, mine;      // mine: lane j holds the path's entry j
    uint64_t gone, children;  // of cur: rejected ones, and those to be asked
    double rest, off;         // what the rejected ones leave of cur's sum, and how far off that may be
    double w, q;              // the lane's node: its weight, drawn: the weights of both rows, each times the other's sum
    bool mass;                // whether its token has any probability
};

__device__ __forceinline__ void verify_stand(VerifyPath& p, int at, int count, float t, const VerifyNode& v, const VerifyState& st) {
    p.cur = at;
    p.gone = 0;
    p.children = __ballot((int)(threadIdx.x & 63) > at && (int)(threadIdx.x & 63) < count && v.up == at);
    p.rest = t > 0.0f ? st.sum[at] : 0.0;
    p.off = V_OFF * p.rest;
}

template <bool DRAWN>
__device__ __forceinline__ void verify_start(VerifyPath& p, int count, float t, const VerifyNode& v, const VerifyState& st) {
    const int lane = threadIdx.x & 63;
    p.w = p.q = 0.0;
    p.mass = false;
    if (t > 0.0f && v.up >= 0 && v.up < lane && lane < count) {
        const float c = verify_factor(t), top = st.top[v.up];
        p.mass = top == INFINITY ? v.x == INFINITY : v.x > -INFINITY;
        p.w = verify_share(v.x, top, st.sum[v.up], c);
        if (DRAWN) {  // u q Y^-1 < p Z^-1 as u q Z < p Y
            const double z = st.sum[v.up], y = st.sum[TREE_MAX + v.up];
            p.q = verify_share(v.y, st.top[TREE_MAX + v.up], y, c) * (z > 0.0 ? z : 1.0);
            p.w *= y > 0.0 ? y : 1.0;
        }
    }
    p.kept = count > 0 ? 1 : 0;
    p.mine = lane == 0 && p.kept ? 0 : -1;
    p.cur = 0;
    p.gone = p.children = 0;
    if (p.kept) verify_stand(p, 0, count, t, v, st);
}

// One wave walks down a sequence's tree: to its end, or (true) to a child whose acceptance the 32-bit sums do not decide.  It is
// called again then, with what is left of the row in 64 bits, and of the draft's row.
template <bool DRAWN>
__device__ __forceinline__ bool verify_walk(VerifyPath& p, int count, float t, const VerifyNode& v, const VerifyState& st,
                                            const double* table, bool answered) {
    const int lane = threadIdx.x & 63;
    while (p.children) {
        const int c = __builtin_ctzll(p.children), cur = p.cur;
        const int64_t x = readlane_i64(v.token, c);
        const double u = (double)__int_as_float(__builtin_amdgcn_readlane(__float_as_int(v.u), c));
        bool yes = false;
        double wc = 0.0, off = V_OFF;
        if (t == 0.0f) {
            yes = st.best[cur] >= 0 && x == st.best[cur];
        } else if ((__ballot(p.mass) >> c & 1) && !(!DRAWN && __ballot((p.gone >> lane & 1) && v.token == x))) {
            double border;
            wc = readlane_f64(p.w, c);
            if (answered) {
                const double steps = verify_steps(t);
                double z = 0.0, y = 0.0;
                for (int i = 0; i < VF_WAVES; ++i) {
                    z += st.w[i];
                    if (DRAWN) y += st.v[i];
                }
                wc = verify_weight(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(v.x), c)), st.top[cur], steps, table);
                if (DRAWN) {
                    const float to = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v.y), c));
                    border = u * (verify_weight(to, st.top[TREE_MAX + cur], steps, table) * (z > 0.0 ? z : 1.0));
                    wc *= y > 0.0 ? y : 1.0;
                } else {
                    border = u * z;
                    p.rest = z;
                    p.off = V_OFF64 * z;
                    off = V_OFF64;
                }
            } else if (DRAWN) {
                border = u * readlane_f64(p.q, c);
                const double z = st.sum[cur], y = st.sum[TREE_MAX + cur];
                if (fabs(border - wc) <= 2.0 * V_OFF * (border + wc) + V_SMALL * (z * (y > 0.0 ? y : 1.0))) return true;
            } else {
                border = u * p.rest;
                if (fabs(border - wc) <= u * p.off + V_OFF * wc + V_SMALL * st.sum[cur]) return true;
            }
            yes = border < wc;
        }
        answered = false;
        p.children &= p.children - 1;
        if (yes) {
            if (lane == p.kept) p.mine = c;
            ++p.kept;
            verify_stand(p, c, count, t, v, st);
        } else {
            p.gone |= 1ull << c;
            p.rest -= wc;
            p.off += off * wc;
        }
    }
    return false;
}

__device__ __forceinline__ void put_f64(double* p, double x) {
    __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double get_f64(const double* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <bool BF16, bool DRAWN>
__global__ __launch_bounds__(VF_THREADS) void verify_finish_kernel(const VerifyArgs a) {
    __shared__ double table[V_TABLE];
    __shared__ VerifyState st;
    const uint32_t seq = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int count = tree_count(a.counts, seq, a.n);
    const float t = verify_temperature(a, seq);
    if (chunk != 0 && (count == 0 || t == 0.0f)) return;
    const double steps = t > 0.0f ? verify_steps(t) : 0.0;
    VerifyNode node;
    if (wave == 0) node = verify_node<BF16, DRAWN>(a, seq, count, t);
    if (tid >= VF_THREADS - V_TABLE) table[tid - (VF_THREADS - V_TABLE)] = V_POWERS[tid - (VF_THREADS - V_TABLE)];
    verify_join(a, seq, count, DRAWN && count > 0 ? 2 * count - 1 : count, t, st);
    __syncthreads();
    const uint32_t segments = (a.vocab + VF_SEGMENT - 1) / VF_SEGMENT;
    // the row where the walk stands, and the draft's there
    float top = 0.0f, qtop = 0.0f;
    size_t logits = 0;
    const void* draft = nullptr;
    int gone = -1;
    bool residual = false;
    auto stand = [&](int cur) {
        top = st.top[cur];
        logits = ((size_t)seq * a.n + cur) * a.row_stride;
        gone = lane < st.n_gone ? st.gone[lane] : -1;
        residual = DRAWN && cur < count - 1;
        draft = residual ? static_cast<const uint8_t*>(a.draft) + ((size_t)seq * (a.n - 1) + cur) * a.draft_stride * (BF16 ? 2 : 4)
                         : static_cast<const uint8_t*>(a.logits) + logits * (BF16 ? 2 : 4);  // (a row that is not looked at)
        qtop = residual ? st.top[TREE_MAX + cur] : 0.0f;
    };
    auto weigh = [&](const float (&x)[VF_EACH], float top, double (&w)[VF_EACH]) {
        if (top == INFINITY) {  // infinite logits share the probability
#pragma unroll
            for (int e = 0; e < VF_EACH; ++e) w[e] = x[e] == INFINITY ? 1.0 : 0.0;
        } else {
#pragma unroll
            for (int e = 0; e < VF_EACH; ++e) w[e] = ((double)x[e] - (double)top) * steps;
            exp_steps(w, table);
        }
    };
    // of segment s: exp((l - top) / T) of the target (without what the walk rejected) and of the draft, lane's tokens 64 e + lane
    auto segment = [&](uint32_t s, double (&w)[VF_EACH], double (&v)[VF_EACH]) {
        const uint32_t x0 = s * VF_SEGMENT + lane;
        float x[VF_EACH], y[VF_EACH];
#pragma unroll
        for (int e = 0; e < VF_EACH; ++e) {  // (no load waits for another)
            const uint32_t at = min(x0 + 64 * e, a.vocab - 1);
            x[e] = verify_logit<BF16>(a.logits, logits + at);
            if (DRAWN) y[e] = verify_logit<BF16>(draft, at);
        }
#pragma unroll
        for (int e = 0; e < VF_EACH; ++e)
            if (x0 + 64 * e >= a.vocab) x[e] = y[e] = -INFINITY;
        weigh(x, top, w);
        if (DRAWN) {
            if (residual) weigh(y, qtop, v);
        } else {
            for (uint64_t here = __ballot(gone >= 0 && (uint32_t)gone / VF_SEGMENT == s); here; here &= here - 1) {
                const int g = __builtin_amdgcn_readlane(gone, __builtin_ctzll(here)) - (int)x0;
#pragma unroll
                for (int e = 0; e < VF_EACH; ++e)
                    if (g == 64 * e) w[e] = 0.0;
            }
        }
    };
    VerifyPath path;
    if (wave == 0) verify_start<DRAWN>(path, count, t, node, st);
    for (bool answered = false;; answered = true) {
        if (wave == 0) {
            const bool asks = verify_walk<DRAWN>(path, count, t, node, st, table, answered);
            if (!DRAWN && (path.gone >> lane & 1))
                st.gone[__popcll(path.gone & ((1ull << lane) - 1))] = node.token >= 0 && node.token < (int64_t)a.vocab ? (int)node.token : -1;
            if (lane == 0) {
                st.asks = asks;
                st.cur = path.cur;
                st.kept = path.kept;
                st.u = (double)node.u;
                st.n_gone = DRAWN ? 0 : __popcll(path.gone);
            }
        }
        __syncthreads();
        if (__builtin_expect(!st.asks, 1)) break;
        stand(st.cur);
        double z = 0.0, y = 0.0, w[VF_EACH], v[VF_EACH];
        for (uint32_t s = wave; s < segments; s += VF_WAVES) {
            segment(s, w, v);
#pragma unroll
            for (int e = 0; e < VF_EACH; ++e) {
                z += w[e];
                if (DRAWN) y += v[e];
            }
        }
        z = wave_sum_f64(z);
        if (DRAWN) y = wave_sum_f64(y);
        if (lane == 0) {
            st.w[wave] = z;
            st.v[wave] = y;
        }
        __syncthreads();
    }
    if (wave == 0 && chunk == 0) {
        if (lane < (int)a.n) a.path[(size_t)seq * a.n + lane] = path.mine;
        if (lane == 0) a.kept[seq] = path.kept;
    }
    const int cur = st.cur;
    if (st.kept == 0 || t == 0.0f) {
        if (tid == 0) a.next_token[seq] = st.kept == 0 ? -1 : st.best[cur];
        return;
    }
    stand(cur);
    double w[VF_EACH], v[VF_EACH];
    const double near = residual && st.sum[TREE_MAX + cur] > 0.0 ? st.sum[cur] / st.sum[TREE_MAX + cur] : 0.0;  // Z / Y to 10^-7
    double* const left = a.left + (size_t)seq * segments * 4;
    for (uint32_t s = chunk * a.per_block + wave; s < min((chunk + 1) * a.per_block, segments); s += VF_WAVES) {
        double sum = 0.0, others = 0.0, all = 0.0, all_others = 0.0;
        bool close = false;
        segment(s, w, v);
        if (residual) {
#pragma unroll
            for (int e = 0; e < VF_EACH; ++e) {
                const bool some = w[e] > near * v[e];
                sum += some ? w[e] : 0.0;
                others += some ? v[e] : 0.0;
                close = close || fabs(w[e] - near * v[e]) < V_BAND * w[e];
                all += w[e];
                all_others += v[e];
            }
            others = wave_sum_f64(others);
            all = wave_sum_f64(all);
            all_others = wave_sum_f64(all_others);
        } else {
#pragma unroll
            for (int e = 0; e < VF_EACH; ++e) sum += w[e];
        }
        sum = wave_sum_f64(sum);
        if (residual && __ballot(close)) sum = -1.0;
        if (lane == 0) {
            put_f64(left + 4 * s, sum);
            if (residual) {
                put_f64(left + 4 * s + 1, others);
                put_f64(left + 4 * s + 2, all);
                put_f64(left + 4 * s + 3, all_others);
            }
        }
    }
    // the last thread block of a sequence to get here draws.  The sums are there before the count is raised.
    __builtin_amdgcn_s_waitcnt(0);
    asm volatile("" ::: "memory");
    __syncthreads();
    if (wave != 0) return;
    uint32_t arrived = 0;
    if (lane == 0) {
        arrived = __hip_atomic_fetch_add(&a.done[seq], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u;
        if (arrived == a.chunks) __hip_atomic_store(&a.done[seq], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if ((uint32_t)__builtin_amdgcn_readfirstlane((int)arrived) != a.chunks) return;

    // 64 * GROUPS segments at a time, lane's are 64 apart
    constexpr int GROUPS = 5;  // those of 151936 tokens
    auto get = [&](uint32_t s0, int k, double (&x)[GROUPS]) {
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) x[g] = get_f64(left + 4 * (size_t)min(s0 + 64 * g + lane, segments - 1) + k);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
            if (s0 + 64 * g + lane >= segments) x[g] = 0.0;
    };
    bool both = residual;
    double ratio = 0.0, total = 0.0;
    if (residual) {
        double z = 0.0, y = 0.0;
        bool marked = false;
        for (uint32_t s0 = 0; s0 < segments; s0 += 64 * GROUPS) {
            double p[GROUPS], q[GROUPS], sum[GROUPS];
            get(s0, 2, p);
            get(s0, 3, q);
            get(s0, 0, sum);
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                z += p[g];
                y += q[g];
                marked = marked || sum[g] < 0.0;
            }
        }
        z = wave_sum_f64(z);
        y = wave_sum_f64(y);
        ratio = y > 0.0 ? z / y : 0.0;
        const bool every = !(fabs(ratio - near) <= V_BAND / 2 * near);
        if (every || __ballot(marked)) {
            for (uint32_t s0 = 0; s0 < segments; s0 += 64) {
                const bool mine = s0 + lane < segments && (every || get_f64(left + 4 * (size_t)(s0 + lane)) < 0.0);
                for (uint64_t which = __ballot(mine); which; which &= which - 1) {
                    const uint32_t s = s0 + __builtin_ctzll(which);
                    segment(s, w, v);
                    double mass = 0.0;
#pragma unroll
                    for (int e = 0; e < VF_EACH; ++e) mass += w[e] > ratio * v[e] ? w[e] - ratio * v[e] : 0.0;
                    mass = wave_sum_f64(mass);
                    if (lane == 0) {
                        put_f64(left + 4 * (size_t)s, mass);
                        put_f64(left + 4 * (size_t)s + 1, 0.0);
                    }
                }
            }
            __builtin_amdgcn_s_waitcnt(0);  // they are read again below
            asm volatile("" ::: "memory");
        }
    }
    double m[GROUPS];
    auto masses = [&](uint32_t s0) {
        get(s0, residual && !both ? 2 : 0, m);
        if (both) {
            double q[GROUPS];
            get(s0, 1, q);
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) m[g] = m[g] > ratio * q[g] ? m[g] - ratio * q[g] : 0.0;
        }
    };
    for (;;) {
        for (uint32_t s0 = 0; s0 < segments; s0 += 64 * GROUPS) {
            masses(s0);
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) total += m[g];
        }
        total = wave_sum_f64(total);
        if (total > 0.0 || !both) break;
        both = false;  // nothing is left of the target's row beside the draft's: the row itself
    }
    if (!(total > 0.0)) {
        if (lane == 0) a.next_token[seq] = -1;
        return;
    }
    const double border = st.u * total;
    double before = 0.0;
    uint32_t at = 0;
    bool past = false;  // rounding may leave nothing past the border: then the last segment, and token, with any mass
    for (uint32_t s0 = 0; s0 < segments && !past; s0 += 64 * GROUPS) {
        if (segments > 64 * GROUPS) masses(s0);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            const double upto = before + wave_scan_f64(m[g]);
            const uint64_t some = __ballot(m[g] > 0.0), over = __ballot(m[g] > 0.0 && upto > border);
            if (past) continue;
            past = over != 0;
            if (past) {
                const int hit = __builtin_ctzll(over);
                at = s0 + 64 * g + hit;
                before = readlane_f64(upto - m[g], hit);
            } else {
                if (some) at = s0 + 64 * g + 63 - __builtin_clzll(some);
                before = readlane_f64(upto, 63);
            }
        }
    }
    segment(at, w, v);
    int64_t choice = -1;
    bool done = false;
#pragma unroll
    for (int e = 0; e < VF_EACH; ++e) {
        double x = w[e];
        if (both) x = x > ratio * v[e] ? x - ratio * v[e] : 0.0;
        const double upto = before + wave_scan_f64(x);
        const uint64_t some = __ballot(x > 0.0), over = past ? __ballot(x > 0.0 && upto > border) : 0;
        if (!done && some) choice = (int64_t)at * VF_SEGMENT + 64 * e + (over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some));
        done = done || over != 0;
        before = readlane_f64(upto, 63);
    }
    if (lane == 0) a.next_token[seq] = choice;
}

struct KeepArgs {
    uint16_t* cache[2];
    size_t layer[2], seq[2];
    uint32_t s_cap, n, n_seq, nk;
    const int32_t* path;
    const int32_t* kept;
    const int32_t* lengths;
};

// A thread block a (layer, sequence): 256 pieces of 16 bytes of the K and V rows at a time, KEEP_GROUPS groups of threads share
// the moves.  Rows move down only (path[j] > j): those of KEEP_GROUPS * KEEP_EACH moves are read before one of them is written,
// and a later move reads no row that an earlier one has written.  36 layers of 16 sequences, 8 to 20 rows each: 26 us, 2.4 TB/s, two
// turns of the chip, the second of 64 thread blocks (one row after another: 33 us; 4 times as many smaller thread blocks would do for
// few rows: 26 nodes 6.7 us for 3.9).
constexpr int KEEP_GROUPS = 4, KEEP_EACH = 4, KEEP_THREADS = 256 * KEEP_GROUPS;

__global__ __launch_bounds__(KEEP_THREADS) void tree_keep_kernel(const KeepArgs a) {
    __shared__ int from[TREE_MAX], to[TREE_MAX], moves_s;
    const uint32_t seq = blockIdx.x % a.n_seq, layer = blockIdx.x / a.n_seq;
    const int len = a.lengths[seq];
    if (threadIdx.x < 64) {
        const int j = (int)threadIdx.x, kept = min(max(a.kept[seq], 0), (int)a.n);
        const int p = j < kept ? a.path[(size_t)seq * a.n + j] : -1;
        const bool move = len >= 0 && p > j && p < (int)a.n && (uint64_t)(uint32_t)len + (uint32_t)p < a.s_cap;
        const uint64_t all = __ballot(move);
        if (move) {
            const int at = __popcll(all & ((1ull << j) - 1));
            from[at] = p;
            to[at] = j;
        }
        if (j == 0) moves_s = __popcll(all);
    }
    __syncthreads();
    const int moves = moves_s;
    if (moves == 0) return;
    const uint32_t row = a.nk * 16;  // pieces of a K or V row
    const int group = threadIdx.x >> 8;
    uint4* const k = reinterpret_cast<uint4*>(a.cache[0] + layer * a.layer[0] + seq * a.seq[0]) + (size_t)len * row;
    uint4* const v = reinterpret_cast<uint4*>(a.cache[1] + layer * a.layer[1] + seq * a.seq[1]) + (size_t)len * row;
    for (uint32_t c0 = 0; c0 < 2 * row; c0 += 256) {
        const uint32_t c = c0 + (threadIdx.x & 255), which = c < row ? 0 : 1, col = c - which * row;
        const bool in = c < 2 * row;
        uint4* const base = (which ? v : k) + (in ? col : 0);
        for (int m0 = 0; m0 < moves; m0 += KEEP_GROUPS * KEEP_EACH) {
            const int mine = m0 + group * KEEP_EACH;
            uint4 x[KEEP_EACH];
#pragma unroll
            for (int i = 0; i < KEEP_EACH; ++i) x[i] = base[(size_t)from[min(mine + i, moves - 1)] * row];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < KEEP_EACH; ++i)
                if (in && mine + i < moves) base[(size_t)to[mine + i] * row] = x[i];
            if (m0 + KEEP_GROUPS * KEEP_EACH < moves) __syncthreads();
        }
    }
}

// Logits a lane and piece: few where rows are few, so that they fill the chip.
static uint32_t verify_each(uint64_t rows, uint32_t vocab) { return rows * ((vocab + 1023) / 1024) <= 12288 ? 16 : 64; }

struct VerifySizes {
    uint32_t each, pieces, chunks, per_block;
    uint64_t rows;
    size_t done, part, left, end;
};

static VerifySizes verify_sizes(uint32_t n_seq, uint32_t n, uint32_t vocab, bool drawn) {
    VerifySizes s;
    s.rows = (uint64_t)n_seq * n + (drawn ? (uint64_t)n_seq * (n - 1) : 0);
    s.each = verify_each(s.rows, vocab);
    s.pieces = (vocab + s.each * 64 - 1) / (s.each * 64);
    // a segment a wave, more of them where the sequences' thread blocks would be more than the chip's CUs
    const uint64_t segments = (vocab + VF_SEGMENT - 1) / VF_SEGMENT, blocks = (segments + VF_WAVES - 1) / VF_WAVES;
    const uint64_t turns = (n_seq * blocks + 255) / 256 < blocks ? (n_seq * blocks + 255) / 256 : blocks;
    s.per_block = (uint32_t)turns * VF_WAVES;
    s.chunks = (uint32_t)((segments + s.per_block - 1) / s.per_block);
    s.done = 0;  // as many for every shape of up to 16384 sequences, so that calls of several shapes may share them
    s.part = ((size_t)(n_seq > 16384 ? n_seq : 16384) * 4 + 15) / 16 * 16;
    s.left = s.part + (size_t)s.rows * s.pieces * 8;
    s.end = s.left + (size_t)n_seq * segments * 32;
    return s;
}

}  // namespace t2h

using namespace t2h;

extern "C" size_t t2h_tree_verify_workspace_bytes(uint32_t n_seq, uint32_t n, uint32_t vocab, int drawn) {
    if (n_seq == 0 || n == 0 || n > (uint32_t)TREE_MAX || vocab == 0 || vocab > 0x7fffffffu) return 0;
    return verify_sizes(n_seq, n, vocab, drawn != 0).end;
}

extern "C" int t2h_tree_verify(const void* logits, uint64_t row_stride, const void* draft, uint64_t draft_stride, int dtype,
                               const int64_t* tokens, const int32_t* parents, const int32_t* counts, const float* uniforms,
                               float temperature, const float* temperatures, int32_t* path, int32_t* kept,
                               int64_t* next_token, uint32_t n, uint32_t n_seq, uint32_t vocab, void* workspace,
                               size_t workspace_bytes, void* stream) {
    if (!logits || !tokens || !path || !kept || !next_token || !workspace) return T2H_ERR_NULL;
    if (!uniforms && (temperatures || temperature > 0.0f)) return T2H_ERR_NULL;
    if (dtype != T2H_DTYPE_F32 && dtype != T2H_DTYPE_BF16) return T2H_ERR_DTYPE;
    if (n == 0 || n > (uint32_t)TREE_MAX || n_seq == 0 || vocab == 0 || vocab > 0x7fffffffu) return T2H_ERR_SHAPE;
    if (row_stride < vocab || (draft && draft_stride < vocab)) return T2H_ERR_SHAPE;
    if (!(temperature < INFINITY) || (draft && parents)) return T2H_ERR_ARG;
    const uint64_t elem = dtype == T2H_DTYPE_F32 ? 3 : 1;
    if ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(draft)) & elem) return T2H_ERR_ALIGN;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return T2H_ERR_ALIGN;
    const bool drawn = draft && n > 1;
    const VerifySizes s = verify_sizes(n_seq, n, vocab, drawn);
    if (workspace_bytes < s.end) return T2H_ERR_WORKSPACE;
    const uint64_t grid = (s.rows * s.pieces + 3) / 4, finish = (uint64_t)n_seq * s.chunks;
    if (grid > 0x3fffffffu || finish > 0x7fffffffu) return T2H_ERR_SHAPE;
    VerifyArgs a;
    a.logits = logits;
    a.draft = drawn ? draft : nullptr;
    a.row_stride = (size_t)row_stride;
    a.draft_stride = (size_t)draft_stride;
    a.tokens = tokens;
    a.parents = parents;
    a.counts = counts;
    a.uniforms = uniforms;
    a.temperature = temperature;
    a.temperatures = temperatures;
    a.path = path;
    a.kept = kept;
    a.next_token = next_token;
    a.n = n;
    a.n_seq = n_seq;
    a.vocab = vocab;
    a.pieces = s.pieces;
    a.chunks = s.chunks;
    a.per_block = s.per_block;
    uint8_t* const ws = reinterpret_cast<uint8_t*>(workspace);
    a.done = reinterpret_cast<uint32_t*>(ws + s.done);
    a.part = reinterpret_cast<uint2*>(ws + s.part);
    a.left = reinterpret_cast<double*>(ws + s.left);
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    auto launch = [&](auto bf16, auto each, auto with_draft) {
        constexpr bool BF16 = decltype(bf16)::value, DRAWN = decltype(with_draft)::value;
        hipLaunchKernelGGL((verify_rows_kernel<BF16, decltype(each)::value>), dim3((uint32_t)grid), dim3(256), 0, st, a);
        hipLaunchKernelGGL((verify_finish_kernel<BF16, DRAWN>), dim3((uint32_t)finish), dim3(VF_THREADS), 0, st, a);
    };
    auto with_each = [&](auto bf16, auto with_draft) {
        if (s.each == 16) launch(bf16, std::integral_constant<int, 16>{}, with_draft);
        else launch(bf16, std::integral_constant<int, 64>{}, with_draft);
    };
    auto with_type = [&](auto with_draft) {
        if (dtype == T2H_DTYPE_BF16) with_each(std::true_type{}, with_draft);
        else with_each(std::false_type{}, with_draft);
    };
    if (drawn) with_type(std::true_type{});
    else with_type(std::false_type{});
    T2H_LAUNCH_CHECK();
    return T2H_OK;
}

extern "C" int t2h_tree_keep(void* k_cache, uint64_t k_layer, uint64_t k_seq, void* v_cache, uint64_t v_layer, uint64_t v_seq,
                             uint32_t layers, uint32_t s_cap, const int32_t* path, const int32_t* kept,
                             const int32_t* lengths, uint32_t n, uint32_t n_seq, uint32_t nk, uint32_t d, void* stream) {
    if (!k_cache || !v_cache || !path || !kept || !lengths) return T2H_ERR_NULL;
    if (d != 128) return T2H_ERR_UNSUPPORTED;
    if (n == 0 || n > (uint32_t)TREE_MAX || n_seq == 0 || layers == 0 || nk == 0 || s_cap == 0) return T2H_ERR_SHAPE;
    const uint64_t seq = (uint64_t)s_cap * nk * d;
    if ((n_seq > 1 && (k_seq < seq || v_seq < seq)) || (layers > 1 && (k_layer < seq || v_layer < seq))) return T2H_ERR_SHAPE;
    const uint64_t strides = (n_seq > 1 ? k_seq | v_seq : 0) | (layers > 1 ? k_layer | v_layer : 0);
    if ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) | strides * 2) & 15) return T2H_ERR_ALIGN;
    const uint64_t grid = (uint64_t)layers * n_seq;
    if (grid > 0x7fffffffu || (uint64_t)nk * 16 > 0x7fffffffu) return T2H_ERR_SHAPE;
    KeepArgs a;
    a.cache[0] = reinterpret_cast<uint16_t*>(k_cache);
    a.cache[1] = reinterpret_cast<uint16_t*>(v_cache);
    a.layer[0] = (size_t)k_layer;
    a.layer[1] = (size_t)v_layer;
    a.seq[0] = (size_t)k_seq;
    a.seq[1] = (size_t)v_seq;
    a.s_cap = s_cap;
    a.n = n;
    a.n_seq = n_seq;
    a.nk = nk;
    a.path = path;
    a.kept = kept;
    a.lengths = lengths;
    hipLaunchKernelGGL(tree_keep_kernel, dim3((uint32_t)grid), dim3(KEEP_THREADS), 0, reinterpret_cast<hipStream_t>(stream), a);
    T2H_LAUNCH_CHECK();
    return T2H_OK;
}
