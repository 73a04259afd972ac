// Which drafted tokens of a tree the target's probabilities accept, the token that follows them, and the accepted nodes' rows
// in the cache (definitions: include/t2h.h, "trees of drafted tokens").
#include <math.h>
#include <type_traits>

#include "tree.h"

namespace t2h {

// ------------------------------------------------------------------------------------------------ verification --
//
// Two launches.  The first reads every node's row of logits once, a wave a piece of E * 64 of them, and leaves the piece's largest
// logit and the sum of exp((l - largest) / T).  The second joins a row's pieces, walks down the tree, and draws the token that
// follows from the row where the walk ended: the piece in which the running sum passes the border, then its logits once more.
// Where drafts were drawn it reads that row of both models again for max(p - q, 0), in thread blocks of their own.
// Sums and exponentials are in 64 bits, relative errors of 10^-14: the borders between the tokens of a large vocabulary lie
// 10^-5 of the sum apart, and 32 bits would draw its neighbour for a token now and then.

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
    uint32_t pieces;   // of a row
    double* part_sum;  // [rows][pieces], the draft's rows behind the target's
    uint2* part_top;   // bits of the largest logit; its index where the sequence is greedy
    uint32_t chunks;   // thread blocks that read a sequence's last row again
    uint32_t* done;    // [n_seq] of those that have left their sums; zero between calls
    double* left;      // [n_seq][chunks] sums of max(p - q, 0)
};

constexpr int V_TABLE = 32;

// 2^(j / 32), by the first lanes of a thread block.
__device__ __forceinline__ void exp_table(double* table) {
    if (threadIdx.x < V_TABLE) table[threadIdx.x] = exp2((double)threadIdx.x / V_TABLE);
}

// exp(x) of x = y ln 2 / 32, y <= 0: 2^(j / 32) from the table, and the Taylor series of what is left, |z| <= ln 2 / 64, up to
// z^5 (the next term is 2 10^-15).  Under 2^-1000 it is 0.
__device__ __forceinline__ double exp_steps(double y, const double* table) {
    constexpr double C = 0.02166084939249829;  // ln 2 / 32
    constexpr double MAGIC = 6755399441055744.0;  // 1.5 2^52: a sum with it is rounded to a whole number, in its low word
    y = fmax(y, -33000.0);
    const double z = y + MAGIC, r = y - (z - MAGIC);
    const int steps = (int)__double2loint(z), e = steps >> 5;
    double p = C * C * C * C * C / 120.0;
    p = fma(p, r, C * C * C * C / 24.0);
    p = fma(p, r, C * C * C / 6.0);
    p = fma(p, r, C * C / 2.0);
    p = fma(p, r, C);
    p = fma(p, r, 1.0);
    p *= table[steps & (V_TABLE - 1)];
    const double w = __hiloint2double(__double2hiint(p) + (e << 20), __double2loint(p));
    return e < -1000 ? 0.0 : w;
}

// exp((x - top) / T) with steps = 32 / (T ln 2); infinite logits share the probability.  x is not NaN.
__device__ __forceinline__ double verify_weight(float x, float top, double steps, const double* table) {
    if (top == INFINITY) return x == INFINITY ? 1.0 : 0.0;
    if (x == -INFINITY) return 0.0;
    return exp_steps(((double)x - (double)top) * steps, table);
}

__device__ __forceinline__ double verify_steps(const VerifyArgs& a, uint32_t seq) {  // 0: greedy
    const float t = a.temperatures ? a.temperatures[seq] : a.temperature;
    return t > 0.0f ? 46.16624130844683 / (double)t : 0.0;
}

// A logit as it counts: NaN as -infinity.
template <bool BF16>
__device__ __forceinline__ float verify_logit(const void* base, size_t at) {
    const float x = BF16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(base)[at]) : static_cast<const float*>(base)[at];
    return fmaxf(x, -INFINITY);
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
}

template <bool BF16, int E>
__global__ __launch_bounds__(256) void verify_rows_kernel(const VerifyArgs a) {
    constexpr int PER = BF16 ? 8 : 4, LOADS = E / PER;  // logits a load of 16 bytes
    __shared__ double table[V_TABLE];
    exp_table(table);
    __syncthreads();
    const int lane = threadIdx.x & 63;
    const uint32_t unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t r = unit / a.pieces, piece = unit % a.pieces, rows = a.n_seq * a.n;
    const bool draft = r >= rows;
    if (r >= rows + (a.draft ? a.n_seq * (a.n - 1) : 0)) return;
    const uint32_t per = draft ? a.n - 1 : a.n, row = draft ? r - rows : r, seq = row / per;
    if ((int)(row % per) >= tree_count(a.counts, seq, a.n) - (draft ? 1 : 0)) return;
    const uint8_t* const base = draft ? static_cast<const uint8_t*>(a.draft) + (size_t)row * a.draft_stride * (BF16 ? 2 : 4)
                                      : static_cast<const uint8_t*>(a.logits) + (size_t)row * a.row_stride * (BF16 ? 2 : 4);
    const uint32_t first = piece * (E * 64) + lane * PER;
    float x[E];
#pragma unroll
    for (int v = 0; v < LOADS; ++v) {
        const uint32_t at = first + v * (64 * PER);
        if (at + PER <= a.vocab) {
            const uint4 w = load_u4_ua(base + (size_t)at * (BF16 ? 2 : 4));
            const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < PER; ++e)
                x[v * PER + e] = BF16 ? __uint_as_float(e & 1 ? words[e / 2] & 0xffff0000u : words[e / 2] << 16) : __uint_as_float(words[e & 3]);
        } else {
#pragma unroll
            for (int e = 0; e < PER; ++e) x[v * PER + e] = at + e < a.vocab ? verify_logit<BF16>(base, at + e) : -INFINITY;
        }
    }
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        x[e] = fmaxf(x[e], -INFINITY);
        top = fmaxf(top, x[e]);
    }
    top = wave_max(top);
    const double steps = verify_steps(a, seq);
    const size_t part = (size_t)r * a.pieces + piece;
    if (steps == 0.0) {
        uint32_t best = 0xffffffffu;
#pragma unroll
        for (int e = E - 1; e >= 0; --e)
            if (x[e] == top) best = first + (e / PER) * (64 * PER) + e % PER;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) best = min(best, (uint32_t)__shfl_xor((int)best, off));
        if (lane == 0) a.part_top[part] = make_uint2(__float_as_uint(top), best);
        return;
    }
    double sum = 0.0;
    if (top == INFINITY) {
#pragma unroll
        for (int e = 0; e < E; ++e) sum += x[e] == INFINITY ? 1.0 : 0.0;
    } else if (top > -INFINITY) {
        const double dtop = (double)top;
#pragma unroll
        for (int e = 0; e < E; ++e) sum += exp_steps(((double)x[e] - dtop) * steps, table);
    }
    sum = wave_sum_f64(sum);
    if (lane == 0) {
        a.part_top[part] = make_uint2(__float_as_uint(top), 0u);
        a.part_sum[part] = sum;
    }
}

constexpr int VF_WAVES = 16, VF_THREADS = VF_WAVES * 64;

__device__ __forceinline__ double shfl_up_f64(double v, int by) { return __shfl_up(v, by); }

// Sums over a thread block's threads up to each; `room` holds VF_WAVES doubles and is free again after the next barrier.
__device__ __forceinline__ double block_scan(double v, double* room) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const double o = shfl_up_f64(v, off);
        if (lane >= off) v += o;
    }
    if (lane == 63) room[wave] = v;
    __syncthreads();
    double before = 0.0;
    for (int w = 0; w < wave; ++w) before += room[w];
    return before + v;
}

struct VerifyState {
    float top[2 * TREE_MAX];   // the rows' largest logits, the draft's behind the target's
    double sum[2 * TREE_MAX];  // and sums
    int64_t best[TREE_MAX];
    int64_t gone[TREE_MAX];    // tokens that the walk rejected where it ended
    int n_gone, cur, kept;
    double scan[2][VF_WAVES];
    uint32_t hit[2], last[2];
    double fresh[TREE_MAX];    // masses of the pieces that lost them, read anew
    double before, border, total;
    uint32_t arrived;
};

__device__ __forceinline__ double readlane_f64(double x, int lane) {
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(x), lane), __builtin_amdgcn_readlane(__double2loint(x), lane));
}
__device__ __forceinline__ int64_t readlane_i64(int64_t x, int lane) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 |
                     (uint32_t)__builtin_amdgcn_readlane((int)x, lane));
}

// A row's largest logit and sum (or its index) from its pieces, in every lane of a wave.
__device__ __forceinline__ void verify_join(const VerifyArgs& a, size_t row, double steps, const double* table, float& top,
                                            double& sum, uint32_t& best) {
    const int lane = threadIdx.x & 63;
    const uint2* const tops = a.part_top + row * a.pieces;
    top = -INFINITY;
    for (uint32_t i = lane; i < a.pieces; i += 64) top = fmaxf(top, __uint_as_float(tops[i].x));
    top = wave_max(top);
    sum = 0.0;
    best = 0xffffffffu;
    for (uint32_t i = lane; i < a.pieces; i += 64) {
        const uint2 t = tops[i];
        const float x = __uint_as_float(t.x);
        if (steps == 0.0) {
            if (x == top) best = min(best, t.y);
        } else {
            sum += a.part_sum[row * a.pieces + i] * verify_weight(x, top, steps, table);
        }
    }
    if (steps == 0.0) {
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) best = min(best, (uint32_t)__shfl_xor((int)best, off));
    } else {
        sum = wave_sum_f64(sum);
    }
}

__device__ __forceinline__ double verify_uniform(const VerifyArgs& a, uint32_t seq, int c) {
    return (double)fminf(fmaxf(a.uniforms[(size_t)seq * a.n + c], 0.0f), 0.99999994f);  // NaN as 0
}

// One wave walks down a sequence's tree.
template <bool BF16, bool DRAWN>
__device__ void verify_walk(const VerifyArgs& a, uint32_t seq, int count, double steps, const double* table, VerifyState& st,
                            bool writes) {
    const int lane = threadIdx.x & 63;
    int up = lane - 1;
    int64_t token = -1;
    double w = 0.0, q = 0.0, u = 0.0;
    if (lane < count) {
        if (a.parents) up = a.parents[(size_t)seq * a.n + lane];
        token = a.tokens[(size_t)seq * a.n + lane];
        if (lane > 0 && up >= 0 && up < lane && token >= 0 && token < (int64_t)a.vocab && steps != 0.0) {
            const size_t row = (size_t)seq * a.n + up;
            w = verify_weight(verify_logit<BF16>(a.logits, row * a.row_stride + token), st.top[up], steps, table);
            if (DRAWN) {
                const size_t draft = (size_t)seq * (a.n - 1) + up;
                const double z = st.sum[up], zq = st.sum[TREE_MAX + up];
                w = z > 0.0 ? w / z : 0.0;
                q = verify_weight(verify_logit<BF16>(a.draft, draft * a.draft_stride + token), st.top[TREE_MAX + up], steps, table);
                q = zq > 0.0 ? q / zq : 0.0;
            }
        }
        if (steps != 0.0) u = verify_uniform(a, seq, lane);
    }
    int cur = 0, kept = count > 0 ? 1 : 0, mine = lane == 0 && kept ? 0 : -1;  // lane j: the path's entry j
    uint64_t gone = 0;
    double rest = count > 0 && steps != 0.0 ? st.sum[0] : 0.0;
    for (bool more = kept != 0; more;) {
        more = false;
        uint64_t children = __ballot(lane > cur && lane < count && up == cur);
        while (children) {
            const int c = __builtin_ctzll(children);
            children &= children - 1;
            const int64_t x = readlane_i64(token, c);
            bool yes;
            double wc = 0.0;
            if (steps == 0.0) {
                yes = st.best[cur] >= 0 && x == st.best[cur];
            } else if (DRAWN) {
                yes = readlane_f64(u, c) * readlane_f64(q, c) < readlane_f64(w, c);
            } else {
                const bool again = __ballot((gone >> lane & 1) && token == x) != 0;
                wc = again ? 0.0 : readlane_f64(w, c);
                yes = readlane_f64(u, c) * rest < wc;
            }
            if (yes) {
                if (lane == kept) mine = c;
                ++kept;
                cur = c;
                gone = 0;
                rest = steps != 0.0 ? st.sum[cur] : 0.0;
                more = true;
                break;
            }
            rest -= wc;
            gone |= 1ull << c;
        }
    }
    if (writes) {
        if (lane < (int)a.n) a.path[(size_t)seq * a.n + lane] = mine;
        if (lane == 0) a.kept[seq] = kept;
    }
    if (gone >> lane & 1) st.gone[__popcll(gone & ((1ull << lane) - 1))] = token;
    if (lane == 0) {
        st.cur = cur;
        st.kept = kept;
        st.n_gone = DRAWN ? 0 : __popcll(gone);
        st.total = rest;
    }
}

template <bool BF16, int E, bool DRAWN>
__global__ __launch_bounds__(VF_THREADS) void verify_finish_kernel(const VerifyArgs a) {
    __shared__ double table[V_TABLE];
    __shared__ VerifyState st;
    const uint32_t seq = DRAWN ? blockIdx.x / a.chunks : blockIdx.x, chunk = DRAWN ? blockIdx.x % a.chunks : 0;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int count = tree_count(a.counts, seq, a.n);
    const double steps = verify_steps(a, seq);
    const uint32_t row0 = seq * a.n, rows = a.n_seq * a.n;
    exp_table(table);
    __syncthreads();
    for (int i = wave; i < (DRAWN ? 2 * count - 1 : count); i += VF_WAVES) {
        const bool draft = i >= count;
        const int node = draft ? i - count : i;
        float top;
        double sum;
        uint32_t best;
        verify_join(a, draft ? (size_t)rows + (size_t)seq * (a.n - 1) + node : (size_t)row0 + node, steps, table, top, sum, best);
        if (lane == 0) {
            st.top[draft ? TREE_MAX + node : node] = top;
            st.sum[draft ? TREE_MAX + node : node] = sum;
            if (!draft) st.best[node] = top == -INFINITY ? -1 : (int64_t)best;
        }
    }
    __syncthreads();
    if (wave == 0) verify_walk<BF16, DRAWN>(a, seq, count, steps, table, st, chunk == 0);
    if (tid == 0) {
        st.hit[0] = st.hit[1] = 0xffffffffu;
        st.last[0] = st.last[1] = 0;
        st.before = 0.0;
    }
    __syncthreads();
    const int cur = st.cur;
    if (st.kept == 0 || steps == 0.0) {
        if (chunk == 0 && tid == 0) a.next_token[seq] = st.kept == 0 ? -1 : st.best[cur];
        return;
    }
    const float top = st.top[cur];
    const size_t row = (size_t)(row0 + cur), logits = row * a.row_stride;
    // the mass that token x has in the row where the walk ended
    auto mass = [&](uint32_t x) {
        if (x >= a.vocab) return 0.0;
        for (int j = 0; j < st.n_gone; ++j)
            if (st.gone[j] == (int64_t)x) return 0.0;
        return verify_weight(verify_logit<BF16>(a.logits, logits + x), top, steps, table);
    };

    if (DRAWN && cur < count - 1) {
        // max(p - q, 0), a chunk a thread block
        const float qtop = st.top[TREE_MAX + cur];
        const double z = st.sum[cur], zq = st.sum[TREE_MAX + cur], iz = z > 0.0 ? 1.0 / z : 0.0, izq = zq > 0.0 ? 1.0 / zq : 0.0;
        const size_t draft = ((size_t)seq * (a.n - 1) + cur) * a.draft_stride;
        auto more = [&](uint32_t x) {
            if (x >= a.vocab) return 0.0;
            const double p = verify_weight(verify_logit<BF16>(a.logits, logits + x), top, steps, table) * iz;
            const double q = verify_weight(verify_logit<BF16>(a.draft, draft + x), qtop, steps, table) * izq;
            return p > q ? p - q : 0.0;
        };
        constexpr int EACH = 8;
        constexpr uint32_t CHUNK = VF_THREADS * EACH;
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < EACH; ++e) sum += more(chunk * CHUNK + e * VF_THREADS + tid);
        const double upto = block_scan(sum, st.scan[0]);
        if (tid == VF_THREADS - 1)
            __hip_atomic_store(&a.left[(size_t)seq * a.chunks + chunk], upto, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        // the last thread block of a sequence to get here draws.  A sum is there before the count is raised.
        __builtin_amdgcn_s_waitcnt(0);
        asm volatile("" ::: "memory");
        __syncthreads();
        if (tid == 0) {
            st.arrived = __hip_atomic_fetch_add(&a.done[seq], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u;
            if (st.arrived == a.chunks) __hip_atomic_store(&a.done[seq], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (st.arrived != a.chunks) return;
        if (tid == 0) {
            double total = 0.0;
            for (uint32_t c = 0; c < a.chunks; ++c)
                total += __hip_atomic_load(&a.left[(size_t)seq * a.chunks + c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            const double border = verify_uniform(a, seq, 0) * total;
            double before = 0.0;
            uint32_t at = 0;
            for (uint32_t c = 0; c < a.chunks; ++c) {
                const double x = __hip_atomic_load(&a.left[(size_t)seq * a.chunks + c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (x <= 0.0) continue;
                at = c;
                if (before + x > border) break;
                before += x;
            }
            st.total = total;
            st.before = before;
            st.border = border;
            st.cur = (int)at;
        }
        __syncthreads();
        if (st.total > 0.0) {
            const uint32_t at = (uint32_t)st.cur * CHUNK;
            for (int e = 0; e < EACH; ++e) {
                const uint32_t x = at + e * VF_THREADS + tid;
                const double v = more(x);
                const double to = st.before + block_scan(v, st.scan[e & 1]);
                if (v > 0.0) {
                    atomicMax(&st.last[0], x);
                    if (to > st.border) atomicMin(&st.hit[0], x);
                }
                __syncthreads();
                if (tid == VF_THREADS - 1) st.before = to;
                __syncthreads();
                if (st.hit[0] != 0xffffffffu) break;
            }
            if (tid == 0) a.next_token[seq] = st.hit[0] != 0xffffffffu ? st.hit[0] : st.last[0];
            return;
        }
        // nothing is left of the target's row beside the draft's: the row itself
        __syncthreads();
        if (tid == 0) st.before = 0.0;
        __syncthreads();
    } else if (DRAWN && chunk != 0) {
        return;
    }

    // 1. the pieces' masses: a piece that lost tokens is read anew where little is left of the row, so that no difference of two
    // near numbers is drawn from
    const double whole = st.sum[cur];
    const bool little = st.n_gone > 0 && st.total < whole * (1.0 / 1024.0);
    constexpr uint32_t PIECE = E * 64;
    if (little)
        for (int j = 0; j < st.n_gone; ++j) {
            const int64_t x = st.gone[j];
            double m = 0.0;
            if (x >= 0 && x < (int64_t)a.vocab)
                for (uint32_t i = tid; i < PIECE; i += VF_THREADS) m += mass((uint32_t)x / PIECE * PIECE + i);
            const double upto = block_scan(m, st.scan[j & 1]);
            if (tid == VF_THREADS - 1) st.fresh[j] = upto;
            __syncthreads();
        }
    auto piece_mass = [&](uint32_t i) {
        if (i >= a.pieces) return 0.0;
        const float t = __uint_as_float(a.part_top[row * a.pieces + i].x);
        double m = a.part_sum[row * a.pieces + i] * verify_weight(t, top, steps, table);
        for (int j = 0; j < st.n_gone; ++j) {
            const int64_t x = st.gone[j];
            if (x < 0 || x >= (int64_t)a.vocab || (uint32_t)x / PIECE != i) continue;
            if (little) return st.fresh[j];
            bool first = true;
            for (int k = 0; k < j; ++k) first = first && st.gone[k] != x;
            if (first) m -= verify_weight(verify_logit<BF16>(a.logits, logits + (size_t)x), top, steps, table);
        }
        return m > 0.0 ? m : 0.0;
    };
    double total = 0.0;
    for (uint32_t i0 = 0; i0 < a.pieces; i0 += VF_THREADS) total += piece_mass(i0 + tid);
    const double sums = block_scan(total, st.scan[0]);
    if (tid == VF_THREADS - 1) {
        st.total = sums;
        st.border = verify_uniform(a, seq, 0) * sums;
    }
    __syncthreads();
    if (!(st.total > 0.0)) {
        if (tid == 0) a.next_token[seq] = -1;
        return;
    }
    // 2. the piece, 3. the token
    for (uint32_t i0 = 0; i0 < a.pieces; i0 += VF_THREADS) {
        const double m = piece_mass(i0 + tid), upto = st.before + block_scan(m, st.scan[1]);
        if (m > 0.0) {
            atomicMax(&st.last[0], i0 + tid);
            if (upto > st.border) atomicMin(&st.hit[0], i0 + tid);
        }
        __syncthreads();
        const uint32_t hit = st.hit[0];
        if (hit == i0 + tid) st.before = upto - m;
        if (hit == 0xffffffffu && tid == VF_THREADS - 1) st.before = upto;
        __syncthreads();
        if (hit != 0xffffffffu) break;
    }
    const bool found = st.hit[0] != 0xffffffffu;
    const uint32_t at = (found ? st.hit[0] : st.last[0]) * PIECE;
    if (!found && tid == 0) st.border = INFINITY;  // rounding: the last token that has any
    __syncthreads();
    for (uint32_t x0 = at; x0 < at + PIECE; x0 += VF_THREADS) {
        const uint32_t x = x0 + tid;
        const double v = x < at + PIECE ? mass(x) : 0.0, upto = st.before + block_scan(v, st.scan[0]);
        if (v > 0.0) {
            atomicMax(&st.last[1], x);
            if (upto > st.border) atomicMin(&st.hit[1], x);
        }
        __syncthreads();
        if (tid == VF_THREADS - 1) st.before = upto;
        __syncthreads();
        if (st.hit[1] != 0xffffffffu) break;
    }
    if (tid == 0) a.next_token[seq] = st.hit[1] != 0xffffffffu ? st.hit[1] : st.last[1];
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
// and a later move reads no row that an earlier one has written.
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
    for (uint32_t c0 = 0; c0 < 2 * row; c0 += 256) {
        const uint32_t c = c0 + (threadIdx.x & 255), which = c < row ? 0 : 1, col = c - which * row;
        const bool in = c < 2 * row;
        uint4* const base = reinterpret_cast<uint4*>(a.cache[which] + layer * a.layer[which] + seq * a.seq[which]) + (size_t)len * row + (in ? col : 0);
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
    uint32_t each, pieces, chunks;
    uint64_t rows;
    size_t done, top, sum, left, end;
};

static VerifySizes verify_sizes(uint32_t n_seq, uint32_t n, uint32_t vocab, bool drawn) {
    VerifySizes s;
    s.rows = (uint64_t)n_seq * n + (drawn ? (uint64_t)n_seq * (n - 1) : 0);
    s.each = verify_each(s.rows, vocab);
    s.pieces = (vocab + s.each * 64 - 1) / (s.each * 64);
    s.chunks = drawn ? (vocab + VF_THREADS * 8 - 1) / (VF_THREADS * 8) : 1;
    s.done = 0;  // as many for every shape of up to 16384 sequences, so that calls of several shapes may share them
    s.top = ((size_t)(n_seq > 16384 ? n_seq : 16384) * 4 + 15) / 16 * 16;
    s.sum = s.top + (size_t)s.rows * s.pieces * 8;
    s.left = s.sum + (size_t)s.rows * s.pieces * 8;
    s.end = s.left + (drawn ? (size_t)n_seq * s.chunks * 8 : 0);
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
    uint8_t* const ws = reinterpret_cast<uint8_t*>(workspace);
    a.done = reinterpret_cast<uint32_t*>(ws + s.done);
    a.part_top = reinterpret_cast<uint2*>(ws + s.top);
    a.part_sum = reinterpret_cast<double*>(ws + s.sum);
    a.left = reinterpret_cast<double*>(ws + s.left);
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    auto launch = [&](auto bf16, auto each) {
        constexpr bool BF16 = decltype(bf16)::value;
        constexpr int E = decltype(each)::value;
        hipLaunchKernelGGL((verify_rows_kernel<BF16, E>), dim3((uint32_t)grid), dim3(256), 0, st, a);
        if (drawn)
            hipLaunchKernelGGL((verify_finish_kernel<BF16, E, true>), dim3((uint32_t)finish), dim3(VF_THREADS), 0, st, a);
        else
            hipLaunchKernelGGL((verify_finish_kernel<BF16, E, false>), dim3((uint32_t)finish), dim3(VF_THREADS), 0, st, a);
    };
    using std::integral_constant;
    const bool bf16 = dtype == T2H_DTYPE_BF16;
    if (s.each == 16) {
        if (bf16) launch(integral_constant<bool, true>{}, integral_constant<int, 16>{});
        else launch(integral_constant<bool, false>{}, integral_constant<int, 16>{});
    } else {
        if (bf16) launch(integral_constant<bool, true>{}, integral_constant<int, 64>{});
        else launch(integral_constant<bool, false>{}, integral_constant<int, 64>{});
    }
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
