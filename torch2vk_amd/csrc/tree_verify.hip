// Which drafted tokens of a tree the target's probabilities accept, the token that follows them, and the accepted nodes' rows
// in the cache (definitions: include/t2h.h, "trees of drafted tokens").
#include <math.h>

#include "tree.h"

namespace t2h {

struct VerifyArgs {
    const void* logits;
    const void* draft;
    size_t row_stride, draft_stride;
    int bf16;
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
    double* top;    // per row: the largest logit
    double* sum;    // and the sum of exp((l - top) / T)
    int64_t* best;  // its index, -1 where no token has any probability
};

// A logit as it counts: NaN as -infinity.
__device__ __forceinline__ float verify_logit(const void* base, size_t at, int bf16) {
    const float x = bf16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(base)[at]) : static_cast<const float*>(base)[at];
    return x == x ? x : -INFINITY;
}

// exp((x - top) / T); infinite logits share the probability.
__device__ __forceinline__ double verify_weight(float x, float top, double inv_t) {
    if (top == INFINITY) return x == INFINITY ? 1.0 : 0.0;
    if (x == -INFINITY) return 0.0;
    return exp(((double)x - (double)top) * inv_t);
}

__device__ __forceinline__ float verify_temperature(const VerifyArgs& a, uint32_t seq) {
    const float t = a.temperatures ? a.temperatures[seq] : a.temperature;
    return t > 0.0f ? t : 0.0f;
}

__device__ __forceinline__ double block_sum(double x, double* red) {
    red[threadIdx.x] = x;
    __syncthreads();
    for (int w = 128; w > 0; w >>= 1) {
        if ((int)threadIdx.x < w) red[threadIdx.x] += red[threadIdx.x + w];
        __syncthreads();
    }
    const double r = red[0];
    __syncthreads();
    return r;
}

// Row r of the target's, then of the draft's.
__global__ __launch_bounds__(256) void verify_rows_kernel(const VerifyArgs a) {
    __shared__ double red[256];
    __shared__ float tops[256];
    __shared__ uint32_t at[256];
    const uint32_t rows = a.n_seq * a.n;
    const bool draft = blockIdx.x >= rows;
    const uint32_t r = draft ? blockIdx.x - rows : blockIdx.x;
    const uint32_t seq = r / (draft ? a.n - 1 : a.n);
    const void* base = draft ? a.draft : a.logits;
    const size_t row = r * (draft ? a.draft_stride : a.row_stride);
    const float t = verify_temperature(a, seq);
    float top = -INFINITY;
    uint32_t best = 0xffffffffu;
    for (uint32_t i = threadIdx.x; i < a.vocab; i += 256) {
        const float x = verify_logit(base, row + i, a.bf16);
        if (x > top) {
            top = x;
            best = i;
        }
    }
    tops[threadIdx.x] = top;
    at[threadIdx.x] = best;
    __syncthreads();
    for (int i = 0; i < 256; ++i)
        if (better_pair(tops[i], at[i], top, best)) {
            top = tops[i];
            best = at[i];
        }
    double s = 0.0;
    if (t > 0.0f)
        for (uint32_t i = threadIdx.x; i < a.vocab; i += 256) s += verify_weight(verify_logit(base, row + i, a.bf16), top, 1.0 / t);
    s = block_sum(s, red);
    if (threadIdx.x == 0) {
        a.top[blockIdx.x] = top;
        a.sum[blockIdx.x] = s;
        a.best[blockIdx.x] = top == -INFINITY ? -1 : (int64_t)best;
    }
}

__device__ __forceinline__ float verify_uniform(const VerifyArgs& a, uint32_t seq, int c) {
    return fminf(fmaxf(a.uniforms[(size_t)seq * a.n + c], 0.0f), 0.99999994f);  // NaN as 0
}

__global__ __launch_bounds__(256) void verify_walk_kernel(const VerifyArgs a) {
    __shared__ double part[256];
    __shared__ int cur_s, kept_s, gone[TREE_MAX], n_gone_s;
    const uint32_t seq = blockIdx.x;
    const int count = tree_count(a.counts, seq, a.n);
    int32_t* const path = a.path + (size_t)seq * a.n;
    const int64_t* const tokens = a.tokens + (size_t)seq * a.n;
    const float t = verify_temperature(a, seq);
    const double inv_t = t > 0.0f ? 1.0 / t : 0.0;
    const uint32_t row0 = seq * a.n, rows = a.n_seq * a.n;
    auto weight = [&](int node, int64_t x) {
        if (x < 0 || x >= (int64_t)a.vocab) return 0.0;
        return verify_weight(verify_logit(a.logits, (row0 + node) * a.row_stride + x, a.bf16), (float)a.top[row0 + node], inv_t);
    };
    auto draft_row = [&](int node) { return seq * (a.n - 1) + node; };
    auto draft_weight = [&](int node, int64_t x) {
        if (x < 0 || x >= (int64_t)a.vocab) return 0.0;
        const uint32_t r = draft_row(node);
        return verify_weight(verify_logit(a.draft, r * a.draft_stride + x, a.bf16), (float)a.top[rows + r], inv_t);
    };
    if (threadIdx.x == 0) {
        int cur = 0, kept = count > 0 ? 1 : 0, n_gone = 0;
        if (kept) path[0] = 0;
        double rest = count > 0 ? a.sum[row0] : 0.0;
        for (int c = 1; c < count; ++c) {
            const int up = a.parents ? a.parents[(size_t)seq * a.n + c] : c - 1;
            if (up != cur) continue;
            const int64_t x = tokens[c];
            bool yes;
            if (t == 0.0f) {
                yes = a.best[row0 + cur] >= 0 && x == a.best[row0 + cur];
            } else if (a.draft) {
                const double z = a.sum[row0 + cur], zq = a.sum[rows + draft_row(cur)];
                const double p = z > 0.0 ? weight(cur, x) / z : 0.0, q = zq > 0.0 ? draft_weight(cur, x) / zq : 0.0;
                yes = (double)verify_uniform(a, seq, c) * q < p;
            } else {
                double w = weight(cur, x);
                for (int j = 0; j < n_gone; ++j)
                    if (tokens[gone[j]] == x) w = 0.0;
                yes = (double)verify_uniform(a, seq, c) * rest < w;
                if (!yes) {
                    rest -= w;
                    gone[n_gone++] = c;
                }
            }
            if (yes) {
                path[kept++] = c;
                cur = c;
                n_gone = 0;
                rest = a.sum[row0 + cur];
            } else if (a.draft) {
                break;
            }
        }
        for (int j = kept; j < (int)a.n; ++j) path[j] = -1;
        a.kept[seq] = kept;
        cur_s = cur;
        kept_s = kept;
        n_gone_s = n_gone;
    }
    __syncthreads();
    const int cur = cur_s;
    if (kept_s == 0) {
        if (threadIdx.x == 0) a.next_token[seq] = -1;
        return;
    }
    if (t == 0.0f) {
        if (threadIdx.x == 0) a.next_token[seq] = a.best[row0 + cur];
        return;
    }
    const double z = a.sum[row0 + cur];
    // the mass that token x has where the walk ended; `residual`: max(p - q, 0)
    auto mass = [&](uint32_t x, bool residual) {
        double w = z > 0.0 ? weight(cur, x) / z : 0.0;
        for (int j = 0; j < n_gone_s; ++j)
            if (tokens[gone[j]] == (int64_t)x) w = 0.0;
        if (residual) {
            const double zq = a.sum[rows + draft_row(cur)];
            const double q = zq > 0.0 ? draft_weight(cur, x) / zq : 0.0;
            w = w > q ? w - q : 0.0;
        }
        return w;
    };
    bool residual = a.draft && cur < count - 1;
    const uint32_t seg = (a.vocab + 255) / 256, lo = min(threadIdx.x * seg, a.vocab), hi = min(lo + seg, a.vocab);
    for (int pass = 0; pass < 2; ++pass) {
        double s = 0.0;
        for (uint32_t x = lo; x < hi; ++x) s += mass(x, residual);
        part[threadIdx.x] = s;
        __syncthreads();
        double total = 0.0;
        for (int i = 0; i < 256; ++i) total += part[i];
        if (total > 0.0 || !residual) break;
        residual = false;  // the two rows are the same
        __syncthreads();
    }
    if (threadIdx.x != 0) return;
    double total = 0.0;
    for (int i = 0; i < 256; ++i) total += part[i];
    const double border = (double)verify_uniform(a, seq, 0) * total;
    double run = 0.0;
    int64_t choice = -1;
    bool found = false;
    for (uint32_t i = 0; i < 256 && !found; ++i) {
        if (part[i] == 0.0 || (run + part[i] <= border && i < 255)) {
            run += part[i];
            continue;
        }
        for (uint32_t x = min(i * seg, a.vocab); x < min((i + 1) * seg, a.vocab) && !found; ++x) {
            const double w = mass(x, residual);
            if (w > 0.0) {
                run += w;
                choice = x;
                found = run > border;
            }
        }
    }
    if (choice < 0 && total > 0.0)  // the last token that has any
        for (uint32_t x = a.vocab; x-- > 0 && choice < 0;)
            if (mass(x, residual) > 0.0) choice = x;
    a.next_token[seq] = choice;
}

struct KeepArgs {
    uint16_t* cache[2];
    size_t layer[2], seq[2];
    uint32_t s_cap, n, n_seq, nk;
    const int32_t* path;
    const int32_t* kept;
    const int32_t* lengths;
};

constexpr int KEEP_BATCH = 8;

// A thread block a (layer, sequence, K or V), a thread 16 bytes of every row.  Rows move down only (path[j] >= j), so a row is
// read before it is written: within a thread in its order, and no thread reads another's bytes.
__global__ __launch_bounds__(256) void tree_keep_kernel(const KeepArgs a) {
    __shared__ int from[TREE_MAX];
    const uint32_t which = blockIdx.x & 1, rest = blockIdx.x >> 1, seq = rest % a.n_seq, layer = rest / a.n_seq;
    const int len = a.lengths[seq], kept = min(max(a.kept[seq], 0), (int)a.n);
    if (len < 0 || kept == 0) return;
    if (threadIdx.x < (uint32_t)kept) {
        const int j = (int)threadIdx.x, p = a.path[(size_t)seq * a.n + j];
        from[j] = p > j && p < (int)a.n && (uint64_t)(uint32_t)len + (uint32_t)p < a.s_cap ? p : j;
    }
    __syncthreads();
    const uint32_t row = a.nk * 16;  // 16-byte pieces
    uint4* const base = reinterpret_cast<uint4*>(a.cache[which] + layer * a.layer[which] + seq * a.seq[which]) + (size_t)len * row;
    for (uint32_t c = threadIdx.x; c < row; c += 256)
        for (int j0 = 0; j0 < kept; j0 += KEEP_BATCH) {
            uint4 x[KEEP_BATCH];
#pragma unroll
            for (int i = 0; i < KEEP_BATCH; ++i)
                if (j0 + i < kept && from[j0 + i] != j0 + i) x[i] = base[(size_t)from[j0 + i] * row + c];
#pragma unroll
            for (int i = 0; i < KEEP_BATCH; ++i)
                if (j0 + i < kept && from[j0 + i] != j0 + i) base[(size_t)(j0 + i) * row + c] = x[i];
        }
}

}  // namespace t2h

using namespace t2h;

extern "C" size_t t2h_tree_verify_workspace_bytes(uint32_t n_seq, uint32_t n, uint32_t vocab, int drawn) {
    if (n_seq == 0 || n == 0 || n > (uint32_t)TREE_MAX || vocab == 0 || vocab > 0x7fffffffu) return 0;
    return (size_t)n_seq * n * 24 * (drawn ? 2 : 1);
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
    if (workspace_bytes < t2h_tree_verify_workspace_bytes(n_seq, n, vocab, draft != nullptr)) return T2H_ERR_WORKSPACE;
    VerifyArgs a;
    a.logits = logits;
    a.draft = n > 1 ? draft : nullptr;
    a.row_stride = (size_t)row_stride;
    a.draft_stride = (size_t)draft_stride;
    a.bf16 = dtype == T2H_DTYPE_BF16;
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
    const uint64_t rows = (uint64_t)n_seq * n + (a.draft ? (uint64_t)n_seq * (n - 1) : 0);
    if (rows > 0x7fffffffu) return T2H_ERR_SHAPE;
    a.top = reinterpret_cast<double*>(workspace);
    a.sum = a.top + rows;
    a.best = reinterpret_cast<int64_t*>(a.sum + rows);
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(verify_rows_kernel, dim3((uint32_t)rows), dim3(256), 0, st, a);
    T2H_LAUNCH_CHECK();
    hipLaunchKernelGGL(verify_walk_kernel, dim3(n_seq), dim3(256), 0, st, a);
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
    const uint64_t grid = 2ull * layers * n_seq;
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
    hipLaunchKernelGGL(tree_keep_kernel, dim3((uint32_t)grid), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), a);
    T2H_LAUNCH_CHECK();
    return T2H_OK;
}
