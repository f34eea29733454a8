// hf_logits.cu -- routing from logits: sigmoid or softmax scores, a balance
// bias, expert groups, top-k, renormalised weights and the permutation into
// expert segments (hf_route_logits). topKScores (compute/moe_router.h:29-57) is
// the case of a sigmoid, one group and k <= 8.
//
// One warp per token; lane i holds experts i, i + 32, ... . Scores become
// order-preserving integer codes (0: not in the choice; 1: NaN; then the
// numbers), so one round of the choice is a scan of the lane's codes, a
// redux.sync and, among equal codes, the lowest id.
//
// Which expert ranks before which is decided as in 64-bit arithmetic, without
// paying for it: without a bias the score is monotone in the logit, so the
// logits' own codes rank exactly. With a bias the round runs on fp32 keys
// whose error is bounded, and a token whose consecutive picks (or whose last
// kept and first dropped group) are closer than twice that bound is redone on
// 64-bit keys. At 256 experts that is about one token in a few hundred.
//
// The permutation: tokens are cut into blocks; a block keeps, per expert, one
// bit per token, so a slot's rank in its segment is a popcount, whatever the
// order of the atomics. Up to 128 tokens one block does everything; beyond, a
// second launch adds the counts of the blocks before its own.
#include "hf_internal.cuh"

#include <math.h>

namespace hf {
namespace {

constexpr int kMaxRouteK = 32;      // one lane per pick
constexpr int kMaxRouteGroups = 32;
constexpr int kOneBlockT = 128;     // tokens one block routes and permutes in one launch
constexpr size_t kWsAlign = 256;

struct LogitArgs {
    const void* logits;  // [T x E]
    int bf16;
    const float* bias;   // [E] or null
    int T, E, k, score, n_group, topk_group, group_top, norm;
    float scale;
    int32_t* ids;
    float* w;
    int32_t* counts;
    int32_t* offsets;
    int32_t* perm;
    int32_t* blk;        // [blocks x E] tokens per expert of each block
    int tb;              // tokens per block
};

// ------------------------------------------------------------------ codes
__device__ __forceinline__ uint32_t code_of(float v) {
    if (v != v) return 1u;
    const uint32_t b = __float_as_uint(v + 0.0f);  // -0 ranks as +0
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t c) {
    if (c <= 1u) return c ? __uint_as_float(0x7fc00000u) : -INFINITY;
    return __uint_as_float((c & 0x80000000u) ? (c & 0x7fffffffu) : ~c);
}
__device__ __forceinline__ unsigned long long code_of(double v) {
    if (v != v) return 1ull;
    const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
    return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ double value_of(unsigned long long c) {
    if (c <= 1ull) return c ? __longlong_as_double(0x7ff8000000000000ll) : double(-INFINITY);
    return __longlong_as_double((long long)((c >> 63) ? (c & 0x7fffffffffffffffull) : ~c));
}
__device__ __forceinline__ uint32_t warp_max(uint32_t c) { return __reduce_max_sync(~0u, c); }
__device__ __forceinline__ unsigned long long warp_max(unsigned long long c) {
    const uint32_t hi = uint32_t(c >> 32);
    const uint32_t mh = __reduce_max_sync(~0u, hi);
    const uint32_t ml = __reduce_max_sync(~0u, hi == mh ? uint32_t(c) : 0u);
    return ((unsigned long long)mh << 32) | ml;
}

// How far a is above b beyond the roundings of two fp32 sums (2^-24 of each, and
// as much again of the parts added): negative when they could be either way.
__device__ __forceinline__ float above(float a, float b) {
    return (a - b) - 0x1p-22f * (fabsf(a) + fabsf(b));
}
__device__ __forceinline__ double above(double a, double b) { return a - b; }

// The lane holding the lowest id among the lanes whose best code is `m`; every
// lane gets that id.
template <typename C>
__device__ __forceinline__ int lowest_id(C best, C m, int id) {
    const unsigned cand = __ballot_sync(~0u, best == m);
    if ((cand & (cand - 1u)) == 0u) return __shfl_sync(~0u, id, __ffs(cand) - 1);
    return __reduce_min_sync(~0u, best == m ? id : 0x7fffffff);
}

template <int NPL, typename C>
__device__ __forceinline__ void lane_best(const C (&c)[NPL], int lane, C& best, int& id) {
    best = 0;
    id = lane;
#pragma unroll
    for (int j = 0; j < NPL; ++j)
        if (c[j] > best) {  // strict: the lane's lowest id on equal codes
            best = c[j];
            id = j * 32 + lane;
        }
}

// Drops the experts of the groups that are not kept (their codes become 0).
// `gc` are the codes whose values are summed for a group's score. *gap: how far
// the last kept group is above the best dropped one.
template <int NPL, typename C, typename F>
__device__ __forceinline__ void keep_groups(C (&c)[NPL], const C (&gc)[NPL], const LogitArgs& a,
                                            int lane, F* gap) {
    const int gs = a.E / a.n_group;
    C mine = 0;  // lane g: the code of group g's score
#pragma unroll 1
    for (int g = 0; g < a.n_group; ++g) {
        C t[NPL], best;
        int id;
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
            const int e = j * 32 + lane;
            t[j] = (e >= g * gs && e < (g + 1) * gs) ? gc[j] : C(0);
        }
        lane_best(t, lane, best, id);
        const C m1 = warp_max(best);
        F s = value_of(m1);
        if (a.group_top == 2 && gs > 1) {
            const int w = lowest_id(best, m1, id);
#pragma unroll
            for (int j = 0; j < NPL; ++j)
                if (j * 32 + lane == w) t[j] = 0;
            lane_best(t, lane, best, id);
            s = s + value_of(warp_max(best));
        }
        if (lane == g) mine = code_of(s);
    }
    // rank of lane's group: the groups before it
    int rank = 0;
#pragma unroll 1
    for (int g = 0; g < a.n_group; ++g) {
        const C o = __shfl_sync(~0u, mine, g);
        rank += (o > mine) || (o == mine && g < lane);
    }
    const bool in = lane < a.n_group && rank < a.topk_group;
    const unsigned kept = __ballot_sync(~0u, in);
    if (a.topk_group < a.n_group) {
        const unsigned last = __ballot_sync(~0u, lane < a.n_group && rank == a.topk_group - 1);
        const unsigned next = __ballot_sync(~0u, lane < a.n_group && rank == a.topk_group);
        *gap = above(value_of(__shfl_sync(~0u, mine, __ffs(last) - 1)),
                     value_of(__shfl_sync(~0u, mine, __ffs(next) - 1)));
    }
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const int e = j * 32 + lane;
        if (e < a.E && !((kept >> (e / gs)) & 1u)) c[j] = 0;
    }
}

// The k best codes in rank order: lane r gets the r-th pick's id. *gap: the
// smallest distance of consecutive ones (the first one left out included).
template <int NPL, typename C, typename F>
__device__ __forceinline__ int pick(C (&c)[NPL], int k, int lane, F* gap) {
    int mine = 0;
    F prev = 0;
#pragma unroll 1
    for (int r = 0; r <= k; ++r) {
        C best;
        int id;
        lane_best(c, lane, best, id);
        const C m = warp_max(best);
        if (m == 0) break;  // after k picks of k experts
        if (r) *gap = fmin(*gap, above(prev, value_of(m)));  // fmin passes over NaN (inf - inf)
        if (r == k) break;
        prev = value_of(m);
        const int w = lowest_id(best, m, id);
        if (lane == r) mine = w;
#pragma unroll
        for (int j = 0; j < NPL; ++j)
            if (j * 32 + lane == w) c[j] = 0;
    }
    return mine;
}

__device__ __forceinline__ float load_logit(const LogitArgs& a, size_t i) {
    return a.bf16 ? bf16_to_f32(static_cast<const uint16_t*>(a.logits)[i])
                  : static_cast<const float*>(a.logits)[i];
}

__device__ __forceinline__ float warp_max_f(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
    return v;
}

// The choice on 64-bit keys (rare: out of line, so that the common path keeps
// its registers).
template <int NPL>
__device__ __noinline__ int pick_exact(const LogitArgs& a, int t, int lane) {
    unsigned long long c[NPL];
    double mx = -INFINITY, sum = 0.0;
    if (a.score == HF_SCORE_SOFTMAX) {
        float m = -INFINITY;
        for (int e = lane; e < a.E; e += 32) m = fmaxf(m, load_logit(a, size_t(t) * a.E + e));
        mx = warp_max_f(m);
        for (int e = lane; e < a.E; e += 32) {
            const double l = load_logit(a, size_t(t) * a.E + e);
            sum += l == -INFINITY ? 0.0 : exp(l - mx);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    }
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const int e = j * 32 + lane;
        c[j] = 0;
        if (e < a.E) {
            const double l = load_logit(a, size_t(t) * a.E + e);
            double p;
            if (a.score == HF_SCORE_SIGMOID) p = 1.0 / (1.0 + exp(-l));
            else p = l == -INFINITY ? 0.0 : exp(l - mx) / sum;
            c[j] = code_of(p + (a.bias ? double(a.bias[e]) : 0.0));
        }
    }
    double gap = INFINITY;
    if (a.topk_group < a.n_group) keep_groups(c, c, a, lane, &gap);
    return pick(c, a.k, lane, &gap);
}

// Scores, choice and weights of token t. Lane r < k returns its pick's id.
template <int NPL>
__device__ __forceinline__ int route_token(const LogitArgs& a, int t, int lane) {
    float s[NPL];
    uint32_t c[NPL];
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const int e = j * 32 + lane;
        s[j] = e < a.E ? load_logit(a, size_t(t) * a.E + e) : -INFINITY;
        c[j] = e < a.E ? code_of(s[j]) : 0u;
    }
    if (a.score == HF_SCORE_SIGMOID) {
#pragma unroll
        for (int j = 0; j < NPL; ++j) s[j] = __fdiv_rn(1.0f, __fadd_rn(1.0f, expf(-s[j])));
    } else {
        float m = s[0];
#pragma unroll
        for (int j = 1; j < NPL; ++j) m = fmaxf(m, s[j]);
        m = warp_max_f(m);
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
            s[j] = s[j] == -INFINITY ? 0.0f : expf(s[j] - m);
            sum += s[j];
        }
        sum = warp_sum(sum);
        const float inv = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);  // 0: every logit is -inf
#pragma unroll
        for (int j = 0; j < NPL; ++j) s[j] = __fmul_rn(s[j], inv);
    }
    // The bound on a fp32 score's error, for scores up to smax. Sigmoid: expf
    // 2^-22, the sum, the quotient: < 2^-21 smax. Softmax: the exponent's
    // rounding (|x e^-x| <= 0.37, 2^-24 each), expf, a sum of 1024 terms in
    // NPL + 5 roundings, the reciprocal and product: < 2^-18 smax. Two keys can
    // be off by twice that (tol), two groups' sums of two by four times; the
    // roundings of the sums themselves are above()'s.
    const bool by_logit = a.bias == nullptr;
    const bool limited = a.topk_group < a.n_group;
    float tol = 0.0f;
    float gap = INFINITY, ggap = INFINITY;
    if (!by_logit || (limited && a.group_top == 2)) {
        uint32_t key[NPL];
        float smax = 0.0f;
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
            const int e = j * 32 + lane;
            key[j] = 0u;
            if (e < a.E) {
                const float v = by_logit ? s[j] : __fadd_rn(s[j], a.bias[e]);
                key[j] = code_of(v);
                smax = fmaxf(smax, s[j]);
            }
        }
        tol = warp_max_f(smax) * (a.score == HF_SCORE_SIGMOID ? 0x1p-20f : 0x1p-17f);
        if (!by_logit) {
#pragma unroll
            for (int j = 0; j < NPL; ++j) c[j] = key[j];
        }
        if (limited) keep_groups(c, key, a, lane, &ggap);
    } else if (limited) {
        keep_groups(c, c, a, lane, &ggap);
        ggap = INFINITY;  // the logits rank exactly
    }
    int mine = pick(c, a.k, lane, &gap);
    // not (gap > tol): a NaN or infinite difference is decided on 64-bit keys too
    if (!(ggap > 2.0f * tol) || (!by_logit && !(gap > tol))) mine = pick_exact<NPL>(a, t, lane);

    float ws = 0.0f;  // the pick's score: from the lane that holds it
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const float v = __shfl_sync(~0u, s[j], mine & 31);
        if (j == (mine >> 5)) ws = v;
    }
    if (lane >= a.k) ws = 0.0f;
    float sum = 0.0f;  // rank order, as topKScores sums
#pragma unroll 1
    for (int i = 0; i < a.k; ++i) sum = __fadd_rn(sum, __shfl_sync(~0u, ws, i));
    if (lane < a.k) {
        if (a.norm && !(sum <= 0.0f)) ws = __fdiv_rn(ws, sum);
        a.ids[size_t(t) * a.k + lane] = mine;
        a.w[size_t(t) * a.k + lane] = __fmul_rn(ws, a.scale);
    }
    return mine;
}

// ------------------------------------------------------------------ permutation
// Rank of token tl among the set bits of its expert's mask.
__device__ __forceinline__ int mask_rank(const uint32_t* m, int tl) {
    int r = 0;
    for (int q = 0; q < (tl >> 5); ++q) r += __popc(m[q]);
    return r + __popc(m[tl >> 5] & ((1u << (tl & 31)) - 1u));
}

// Exclusive scan of v over the block (every thread calls it); *total: the sum.
__device__ __forceinline__ int block_scan(int v, int* tot, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = int(blockDim.x) >> 5;
    int inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(~0u, inc, o);
        if (lane >= o) inc += y;
    }
    if (lane == 31) tot[warp] = inc;
    __syncthreads();
    if (warp == 0) {
        const int wv = lane < nw ? tot[lane] : 0;
        int wi = wv;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(~0u, wi, o);
            if (lane >= o) wi += y;
        }
        tot[lane] = wi - wv;
        if (lane == 31) tot[32] = wi;
    }
    __syncthreads();
    *total = tot[32];
    const int r = tot[warp] + inc - v;
    __syncthreads();
    return r;
}

// Offsets of the segments from per-expert totals, with `mine` (the tokens of
// earlier blocks) added into base[e]; the first block writes counts and offsets.
__device__ __forceinline__ void segment_bases(const LogitArgs& a, const int* total, int* base,
                                              bool write) {
    __shared__ int tot[33];
    int run = 0;
    for (int e0 = 0; e0 < a.E; e0 += blockDim.x) {
        const int e = e0 + int(threadIdx.x);
        const int c = e < a.E ? total[e] : 0;
        int sum;
        const int off = run + block_scan(c, tot, &sum);
        if (e < a.E) {
            base[e] += off;
            if (write) {
                a.counts[e] = c;
                a.offsets[e] = off;
            }
        }
        run += sum;
    }
    if (write && threadIdx.x == 0) {
        a.counts[a.E] = 0;  // the shared group
        a.offsets[a.E] = a.offsets[a.E + 1] = run;
    }
    __syncthreads();
}

__device__ __forceinline__ void set_masks(const LogitArgs& a, uint32_t* masks, int t0, int nt,
                                          int words) {
    for (int i = threadIdx.x; i < nt * a.k; i += blockDim.x) {
        const int tl = i / a.k;
        atomicOr(&masks[a.ids[size_t(t0) * a.k + i] * words + (tl >> 5)], 1u << (tl & 31));
    }
}

__device__ __forceinline__ void scatter(const LogitArgs& a, const uint32_t* masks, const int* base,
                                        int t0, int nt, int words) {
    for (int i = threadIdx.x; i < nt * a.k; i += blockDim.x) {
        const int slot = t0 * a.k + i, e = a.ids[slot];
        a.perm[base[e] + mask_rank(masks + e * words, i / a.k)] = slot;
    }
}

// Block b routes tokens [b * tb, ...) and counts them per expert; a launch of
// one block goes on to the permutation.
template <int NPL, int THREADS>
__global__ void __launch_bounds__(THREADS) k_route_logits(LogitArgs a) {
    extern __shared__ __align__(16) uint32_t sm[];
    const int words = a.tb / 32;
    uint32_t* masks = sm;                                         // [E][words]
    int* total = reinterpret_cast<int*>(sm + size_t(a.E) * words);  // [E]
    int* base = total + a.E;                                      // [E]
    const int t0 = blockIdx.x * a.tb, nt = min(a.tb, a.T - t0);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    griddep_launch_dependents();
    for (int i = threadIdx.x; i < a.E * words; i += blockDim.x) masks[i] = 0u;
    __syncthreads();
    for (int tl = warp; tl < nt; tl += THREADS / 32) {
        const int id = route_token<NPL>(a, t0 + tl, lane);
        if (lane < a.k) atomicOr(&masks[id * words + (tl >> 5)], 1u << (tl & 31));
    }
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
        int c = 0;
        for (int q = 0; q < words; ++q) c += __popc(masks[e * words + q]);
        if (gridDim.x > 1) a.blk[size_t(blockIdx.x) * a.E + e] = c;
        total[e] = c;
        base[e] = 0;
    }
    if (gridDim.x > 1) return;
    __syncthreads();
    segment_bases(a, total, base, true);
    scatter(a, masks, base, t0, nt, words);
}

__global__ void __launch_bounds__(1024) k_route_scatter(LogitArgs a, int nb) {
    extern __shared__ __align__(16) uint32_t sm[];
    const int words = a.tb / 32;
    uint32_t* masks = sm;
    int* total = reinterpret_cast<int*>(sm + size_t(a.E) * words);
    int* base = total + a.E;
    const int b = blockIdx.x, t0 = b * a.tb, nt = min(a.tb, a.T - t0);
    for (int i = threadIdx.x; i < a.E * words; i += blockDim.x) masks[i] = 0u;
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) total[e] = base[e] = 0;
    griddep_wait();  // the ids and counts of every block
    __syncthreads();
    // threads cover (slice of blocks, expert), so that the loads of a column
    // are spread over the block; integer sums, any order
    const int cols = min(a.E, int(blockDim.x)), slices = int(blockDim.x) / cols;
    const int slice = int(threadIdx.x) / cols;
    if (slice < slices) {
        for (int e = int(threadIdx.x) % cols; e < a.E; e += cols) {
            int all = 0, before = 0;
#pragma unroll 8
            for (int q = slice; q < nb; q += slices) {
                const int c = a.blk[size_t(q) * a.E + e];
                all += c;
                before += q < b ? c : 0;
            }
            atomicAdd(&total[e], all);
            atomicAdd(&base[e], before);
        }
    }
    set_masks(a, masks, t0, nt, words);
    __syncthreads();
    segment_bases(a, total, base, b == 0);
    scatter(a, masks, base, t0, nt, words);
}

__global__ void k_route_empty(LogitArgs a) {
    for (int e = threadIdx.x; e <= a.E + 1; e += blockDim.x) {
        if (e <= a.E) a.counts[e] = 0;
        a.offsets[e] = 0;
    }
}

// Tokens per block: 128 routed by one block; else 32 while that leaves at most
// two blocks per SM (a block's warps then have one token each), 128, and 512
// where the second launch would add up too many blocks' counts.
int tokens_per_block(int T) {
    if (T <= kOneBlockT) return kOneBlockT;
    if (T <= 2 * 148 * 32) return 32;
    return T <= 65536 ? 128 : 512;
}

int blocks_of(int T) {
    const int tb = tokens_per_block(T);
    return (T + tb - 1) / tb;
}

size_t ws_bytes(int T, int E) {
    if (T <= kOneBlockT) return 0;
    return (size_t(blocks_of(T)) * E * sizeof(int32_t) + kWsAlign - 1) / kWsAlign * kWsAlign;
}

template <int NPL>
hf_status launch(const LogitArgs& a, cudaStream_t st) {
    // registers: NPL scores and codes per lane (and 64-bit ones in the rare path)
    constexpr int kThreads = NPL <= 8 ? 1024 : 256;
    const int nb = blocks_of(a.T);
    const int smem = a.E * (a.tb / 32 + 2) * 4;
    const auto kern = k_route_logits<NPL, kThreads>;
    HF_CUDA(ensure_smem(reinterpret_cast<const void*>(kern), smem));
    kern<<<nb, kThreads, smem, st>>>(a);
    HF_CUDA(cudaGetLastError());
    if (nb > 1) {
        HF_CUDA(ensure_smem(reinterpret_cast<const void*>(k_route_scatter), smem));
        HF_CUDA(launch_pdl(k_route_scatter, dim3(nb), dim3(1024), size_t(smem), st, a, nb));
    }
    return HF_OK;
}

hf_status check_spec(const hf_route_spec* s, const char* fn) {
    const std::string f(fn);
    if (!s) return fail(HF_ERR_ARG, f + ": null spec");
    if (s->num_experts < 1 || s->num_experts > kMaxExperts)
        return fail(HF_ERR_ARG, f + ": num_experts must be in 1..1024");
    if (s->score != HF_SCORE_SIGMOID && s->score != HF_SCORE_SOFTMAX)
        return fail(HF_ERR_ARG, f + ": score must be HF_SCORE_SIGMOID or HF_SCORE_SOFTMAX");
    if (s->n_group < 1 || s->n_group > kMaxRouteGroups || s->num_experts % s->n_group)
        return fail(HF_ERR_ARG, f + ": n_group must be in 1..32 and divide num_experts");
    if (s->topk_group < 1 || s->topk_group > s->n_group)
        return fail(HF_ERR_ARG, f + ": topk_group must be in 1..n_group");
    if (s->group_top != 1 && s->group_top != 2)
        return fail(HF_ERR_ARG, f + ": group_top must be 1 or 2");
    if (s->top_k < 1 || s->top_k > kMaxRouteK ||
        s->top_k > s->topk_group * (s->num_experts / s->n_group))
        return fail(HF_ERR_ARG, f + ": top_k must be in 1..32 and at most the experts of the "
                                    "kept groups");
    return HF_OK;
}

}  // namespace
}  // namespace hf

using namespace hf;

extern "C" {

size_t hf_route_workspace_size(int T, const hf_route_spec* spec) {
    if (T <= 0 || check_spec(spec, "hf_route_workspace_size") != HF_OK) return 0;
    return ws_bytes(T, spec->num_experts);
}

hf_status hf_route_logits(const void* logits, hf_dtype dtype, const float* bias, int T,
                          const hf_route_spec* spec, const hf_moe_routing* r, void* workspace,
                          size_t workspace_bytes, hf_stream stream) {
    HF_TRY(check_spec(spec, "hf_route_logits"));
    if (dtype != HF_BF16 && dtype != HF_F32)
        return fail(HF_ERR_ARG, "hf_route_logits: logits must be bf16 or f32");
    if (T < 0 || (long long)T * spec->top_k > 0x7fffffffll)
        return fail(HF_ERR_ARG, "hf_route_logits: T >= 0 and T * top_k below 2^31");
    if (!r || !r->counts || !r->offsets || (T && (!logits || !r->topk_ids || !r->topk_weights || !r->perm)))
        return fail(HF_ERR_ARG, "hf_route_logits: null pointer");
    if (r->margins || r->slot_out)
        return fail(HF_ERR_ARG, "hf_route_logits: margins and slot_out are not written");
    const size_t need = T ? ws_bytes(T, spec->num_experts) : 0;
    if (need) {
        if (!workspace || reinterpret_cast<uintptr_t>(workspace) % kWsAlign)
            return fail(HF_ERR_ARG, "hf_route_logits: workspace must be 256-byte aligned");
        if (workspace_bytes < need)
            return fail(HF_ERR_ARG, "hf_route_logits: workspace smaller than hf_route_workspace_size");
    }
    LogitArgs a{};
    a.logits = logits;
    a.bf16 = dtype == HF_BF16;
    a.bias = bias;
    a.T = T;
    a.E = spec->num_experts;
    a.k = spec->top_k;
    a.score = spec->score;
    a.n_group = spec->n_group;
    a.topk_group = spec->topk_group;
    a.group_top = spec->group_top;
    a.norm = spec->norm;
    a.scale = spec->scale;
    a.ids = r->topk_ids;
    a.w = r->topk_weights;
    a.counts = r->counts;
    a.offsets = r->offsets;
    a.perm = r->perm;
    a.blk = static_cast<int32_t*>(workspace);
    const cudaStream_t st = as_cuda(stream);
    if (T == 0) {
        k_route_empty<<<1, 256, 0, st>>>(a);
        HF_CUDA(cudaGetLastError());
        return HF_OK;
    }
    a.tb = tokens_per_block(T);
    const int npl = (a.E + 31) / 32;
    if (npl <= 1) return launch<1>(a, st);
    if (npl <= 2) return launch<2>(a, st);
    if (npl <= 4) return launch<4>(a, st);
    if (npl <= 8) return launch<8>(a, st);
    if (npl <= 16) return launch<16>(a, st);
    return launch<32>(a, st);
}

}  // extern "C"
