// hf_logits.cu -- routing from logits: sigmoid or softmax scores, a balance
// bias, expert groups, top-k, renormalised weights and the permutation into
// expert segments (hf_route_logits). topKScores (compute/moe_router.h:29-57) is
// the case of a sigmoid, one group and k <= 8.
//
// One warp per token; lane i holds experts i, i + 32, ... . Keys become
// order-preserving integers (0: not in the choice; then NaN; then the numbers)
// whose lowest bits are replaced by the expert's place in its lane, inverted:
// one integer maximum then finds the best key and, among equal ones, the lowest
// id. A lane sorts its keys once (min / max network); a round of the choice is a
// redux.sync over the lanes' first keys, and the winner moves its list up.
//
// Which expert ranks before which is decided as in 64-bit arithmetic, without
// paying for it. Without a bias the score is monotone in the logit, so the
// logits rank exactly (up to the replaced bits). With a bias the keys are fp32
// sums whose error is bounded. Where consecutive picks are closer than the bound
// the choice goes on until one is clearly below, and the candidates (one a lane)
// are ranked again by their 64-bit keys: at 256 experts about one token in two
// hundred. A token whose last kept and first dropped group are that close is
// redone in 64 bits from its logits.
//
// The permutation: tokens are cut into blocks; a block keeps, per expert, one
// bit per token, so a slot's rank in its segment is a popcount, whatever the
// order of the atomics. Up to 16 tokens one block does everything; beyond, a
// second launch adds the counts of the blocks before its own.
//
// 16384 tokens, E = 256, k = 8, bias: 30.6 us, of which routing 21 to 25, bound by
// issue slots (825 instructions a token, 61 % of the slots used; the rounds of the
// choice are the largest part). The logits' 16.8 MB would take 2.6.
#include "hf_internal.cuh"

#include <math.h>

#include <algorithm>

namespace hf {
namespace {

constexpr int kMaxRouteK = 32;      // one lane per pick
constexpr int kMaxRouteGroups = 32;
// Tokens that one block routes and permutes in one launch. E = 256, k = 8, us in one
// launch and in two: 16 tokens 6.6 and 6.9 (with groups 9.1 and 8.7), 24 tokens 8.1
// and 6.7.
constexpr int kOneBlockT = 16;
// Blocks of tokens above which their counts are scanned first. us with and without
// the scan: 147 blocks (16384 x 64) 18.4 and 17.0, 512 (262144 x 64) 180 and 182,
// 586 (300000 x 256) 277 and 296, 1954 (1000000 x 64) 654 and 705.
constexpr int kScanBlocks = 512;
constexpr size_t kWsAlign = 256;
// Dynamic shared memory that needs no opt-in: 48 KB with the kernels' static 144 bytes.
constexpr int kPlainSmem = 47 * 1024;

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
// -inf is 0x007fffff (and 0x000f... in 64 bits); NaN takes kNanCode below it,
// above the place bits.
constexpr uint32_t kNanCode = 0x40u;
__device__ __forceinline__ uint32_t code_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);  // -0 ranks as +0
    const uint32_t c = b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
    return v == v ? c : kNanCode;
}
// Of a code with its place bits cleared: -inf's own code is then the lowest NaN
// pattern, so everything up to it reads as -inf.
__device__ __forceinline__ float value_of(uint32_t c) {
    if (c <= 0x007fffffu) return c == kNanCode ? __uint_as_float(0x7fc00000u) : -INFINITY;
    return __uint_as_float((c & 0x80000000u) ? (c & 0x7fffffffu) : ~c);
}
__device__ __forceinline__ unsigned long long code_of(double v) {
    if (v != v) return kNanCode;
    const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
    return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ double value_of(unsigned long long c) {
    if (c <= 0x000fffffffffffffull)
        return c == kNanCode ? __longlong_as_double(0x7ff8000000000000ll) : double(-INFINITY);
    return __longlong_as_double((long long)((c >> 63) ? (c & 0x7fffffffffffffffull) : ~c));
}
__device__ __forceinline__ uint32_t warp_max(uint32_t c) { return __reduce_max_sync(~0u, c); }
__device__ __forceinline__ unsigned long long warp_max(unsigned long long c) {
    const uint32_t hi = uint32_t(c >> 32);
    const uint32_t mh = __reduce_max_sync(~0u, hi);
    const uint32_t ml = __reduce_max_sync(~0u, hi == mh ? uint32_t(c) : 0u);
    return ((unsigned long long)mh << 32) | ml;
}

// Low bits of a code that hold the expert's place j in its lane (as NPL - 1 - j).
template <int NPL>
struct Place {
    static constexpr int kBits = NPL == 1 ? 0 : NPL == 2 ? 1 : NPL == 4 ? 2 : NPL == 8 ? 3
                                 : NPL == 16 ? 4 : 5;
    static constexpr uint32_t kMask = (1u << kBits) - 1u;
};

template <int NPL>
__device__ __forceinline__ uint32_t packed(uint32_t code, int j) {
    return (code & ~Place<NPL>::kMask) | uint32_t(NPL - 1 - j);
}
template <int NPL>
__device__ __forceinline__ float value_at(uint32_t packed_code) {
    return value_of(packed_code & ~Place<NPL>::kMask);
}

// How far the key of code a is above that of code b, beyond what the fp32 sums
// (2^-23 of each) and the replaced bits (2^(kBits - 23)) may hide: not positive
// when either could be the larger.
template <int NPL>
__device__ __forceinline__ float beyond(float diff, float size) {
    constexpr float kRel = float(2 + (1 << Place<NPL>::kBits)) * 0x1p-23f;
    return diff - kRel * size;
}
template <int NPL>
__device__ __forceinline__ float above(uint32_t a, uint32_t b) {
    const float x = value_at<NPL>(a), y = value_at<NPL>(b);
    return beyond<NPL>(x - y, fabs(x) + fabs(y));
}

// Descending sort of a lane's codes: Batcher's merge exchange.
template <int NPL>
__device__ __forceinline__ void sort_lane(uint32_t (&c)[NPL]) {
#pragma unroll
    for (int p = 1; p < NPL; p <<= 1)
#pragma unroll
        for (int k = p; k >= 1; k >>= 1)
#pragma unroll
            for (int j = k % p; j + k < NPL; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < NPL && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const uint32_t hi = max(c[i + j], c[i + j + k]);
                        const uint32_t lo = min(c[i + j], c[i + j + k]);
                        c[i + j] = hi;
                        c[i + j + k] = lo;
                    }
}

// The best two of a group's n codes, read from place i on. (Equal keys count twice.)
template <typename C>
__device__ __forceinline__ void best_two(const C* g, int n, int i, C* b1, C* b2) {
    C m1 = 0, m2 = 0;
#pragma unroll 4
    for (int q = 0; q < n; ++q) {
        const C v = g[i];
        m2 = max(m2, min(m1, v));
        m1 = max(m1, v);
        if (++i == n) i = 0;
    }
    *b1 = m1;
    *b2 = m2;
}

// Rank of the lane's group by its score's code and its number.
template <typename C>
__device__ __forceinline__ int group_rank(C code, int n_group, int lane) {
    int rank = 0;
#pragma unroll 4
    for (int g = 0; g < n_group; ++g) {
        const C o = __shfl_sync(~0u, code, g);
        rank += (o > code) || (o == code && g < lane);
    }
    return rank;
}

// Drops the experts of the groups that are not kept (their codes become 0).
// `gc` are the packed codes whose values are summed for a group's score; lane g
// scans group g's codes in the warp's scratch `scr` [E], from a place of its own
// so that groups of 32 do not meet in one bank. *gap: how far the last kept group
// is above the best dropped one.
template <int NPL>
__device__ __forceinline__ void keep_groups(uint32_t (&c)[NPL], const uint32_t (&gc)[NPL],
                                            const LogitArgs& a, int lane, uint32_t* scr,
                                            float* gap) {
    const int gs = a.E / a.n_group;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < NPL; ++j)
        if (j * 32 + lane < a.E) scr[j * 32 + lane] = gc[j];
    __syncwarp();
    uint32_t code = 0;  // of the score of group `lane`
    float size = 0.0f;  // and the magnitudes that were added
    if (lane < a.n_group) {
        uint32_t b1, b2;
        best_two(scr + lane * gs, gs, lane % gs, &b1, &b2);
        float s = value_at<NPL>(b1);
        size = fabsf(s);
        if (a.group_top == 2) {
            const float s2 = value_at<NPL>(b2);
            s = s + s2;
            size = size + fabsf(s2);
        }
        code = code_of(s);
    }
    const int rank = group_rank(code, a.n_group, lane);
    const unsigned kept = __ballot_sync(~0u, lane < a.n_group && rank < a.topk_group);
    const unsigned last = __ballot_sync(~0u, lane < a.n_group && rank == a.topk_group - 1);
    const unsigned next = __ballot_sync(~0u, lane < a.n_group && rank == a.topk_group);
    const int ll = __ffs(last) - 1, ln = __ffs(next) - 1;
    *gap = beyond<NPL>(value_of(__shfl_sync(~0u, code, ll)) - value_of(__shfl_sync(~0u, code, ln)),
                       __shfl_sync(~0u, size, ll) + __shfl_sync(~0u, size, ln));
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const int e = j * 32 + lane;
        if (e < a.E && !((kept >> (e / gs)) & 1u)) c[j] = 0;
    }
}

// Takes the best code of the warp out of the lanes' sorted lists: its packed code
// (0 when none is left), and the id in *id.
template <int NPL>
__device__ __forceinline__ uint32_t take_best(uint32_t (&c)[NPL], int lane, int* id) {
    const uint32_t m = warp_max(c[0]);
    // equal codes have equal places, so the lowest lane has the lowest id
    const int w = __ffs(__ballot_sync(~0u, c[0] == m)) - 1;
    *id = (NPL - 1 - int(m & Place<NPL>::kMask)) * 32 + w;
    const bool mine = lane == w;
#pragma unroll
    for (int j = 0; j + 1 < NPL; ++j) c[j] = mine ? c[j + 1] : c[j];
    if (mine) c[NPL - 1] = 0;
    return m;
}

// Whether code b (<= a) is not clearly below a: the codes are equal but for the
// place (`exact`), or not more than tol apart; a NaN difference (inf - inf)
// counts as close.
template <int NPL>
__device__ __forceinline__ bool is_close(uint32_t a, uint32_t b, bool exact, float tol) {
    constexpr uint32_t place = Place<NPL>::kMask;
    return exact ? (a | place) == (b | place) : !(above<NPL>(a, b) > tol);
}

// Ranks n candidates (lane r < n: an id and its code) by code and id: lane r
// gets the id of rank r.
__device__ __forceinline__ int rank_again(unsigned long long code, int id, int n, int lane) {
    int rank = 0, mine = 0;
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        const unsigned long long o = __shfl_sync(~0u, code, i);
        const int oid = __shfl_sync(~0u, id, i);
        rank += o > code || (o == code && oid < id);
    }
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        const int ri = __shfl_sync(~0u, rank, i), oid = __shfl_sync(~0u, id, i);
        if (ri == lane) mine = oid;
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

// Maximum of token t's logits, and in 64 bits the sum of their exponentials.
__device__ __forceinline__ double softmax_sum(const LogitArgs& a, int t, int lane, double* mx) {
    float m = -INFINITY;
    for (int e = lane; e < a.E; e += 32) m = fmaxf(m, load_logit(a, size_t(t) * a.E + e));
    *mx = warp_max_f(m);
    double sum = 0.0;
#pragma unroll 1
    for (int e = lane; e < a.E; e += 32) {
        const double l = load_logit(a, size_t(t) * a.E + e);
        sum += l == -INFINITY ? 0.0 : exp(l - *mx);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    return sum;
}

__device__ __forceinline__ double key64(const LogitArgs& a, int t, int e, double mx, double sum) {
    const double l = load_logit(a, size_t(t) * a.E + e);
    double p;
    if (a.score == HF_SCORE_SIGMOID) p = 1.0 / (1.0 + exp(-l));
    else p = l == -INFINITY ? 0.0 : exp(l - mx) / sum;
    return p + (a.bias ? double(a.bias[e]) : 0.0);
}

// The candidates' order by logit, or by 64-bit key.
__device__ __noinline__ int refine(const LogitArgs& a, int t, int lane, int id, int n) {
    unsigned long long code;
    if (a.bias == nullptr) {
        code = code_of(load_logit(a, size_t(t) * a.E + id));
    } else {
        double mx = 0.0, sum = 1.0;
        if (a.score == HF_SCORE_SOFTMAX) sum = softmax_sum(a, t, lane, &mx);
        code = code_of(key64(a, t, id, mx, sum));
    }
    return rank_again(code, id, n, lane);
}

// The whole choice in 64 bits (groups too close to tell apart, more candidates
// than lanes): whole codes, so that equal keys and scores are the only ties, and the
// lowest id or group takes those. scr: the warp's row of E codes.
template <int NPL>
__device__ __noinline__ int pick_exact(const LogitArgs& a, int t, int lane,
                                       unsigned long long* scr) {
    unsigned long long c[NPL];  // 0: not in the choice
    // without a bias logits rank, but for the sums of two scores
    const bool by_logit = a.bias == nullptr, by_score = !by_logit || a.group_top == 2;
    const auto logit_code = [&](int e) {
        return (unsigned long long)code_of(load_logit(a, size_t(t) * a.E + e)) << 32;
    };
    double mx = 0.0, sum = 1.0;
    if (by_score && a.score == HF_SCORE_SOFTMAX) sum = softmax_sum(a, t, lane, &mx);
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const int e = j * 32 + lane;
        if (e >= a.E) c[j] = 0;
        else c[j] = by_score ? code_of(key64(a, t, e, mx, sum)) : logit_code(e);
    }
    unsigned kept = ~0u;
    const int gs = a.E / a.n_group;
    if (a.topk_group < a.n_group) {
        __syncwarp();
#pragma unroll
        for (int j = 0; j < NPL; ++j)
            if (j * 32 + lane < a.E) scr[j * 32 + lane] = c[j];
        __syncwarp();
        unsigned long long code = 0;
        if (lane < a.n_group) {
            unsigned long long b1, b2;
            best_two(scr + lane * gs, gs, lane % gs, &b1, &b2);
            code = a.group_top == 2 ? code_of(value_of(b1) + value_of(b2)) : b1;
        }
        const int rank = group_rank(code, a.n_group, lane);
        kept = __ballot_sync(~0u, lane < a.n_group && rank < a.topk_group);
    }
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const int e = j * 32 + lane;
        if (e >= a.E || !((kept >> (e / gs)) & 1u)) c[j] = 0;
        else if (by_logit && by_score) c[j] = logit_code(e);
    }
    int mine = 0;
#pragma unroll 1
    for (int r = 0; r < a.k; ++r) {
        unsigned long long m = 0;
        int at = 0;
#pragma unroll
        for (int j = 0; j < NPL; ++j)
            if (c[j] > m) {
                m = c[j];
                at = j;
            }
        const unsigned long long best = warp_max(m);
        const unsigned id = __reduce_min_sync(~0u, m == best ? unsigned(at * 32 + lane) : ~0u);
        if (lane == r) mine = int(id);
#pragma unroll
        for (int j = 0; j < NPL; ++j)
            if (id == unsigned(j * 32 + lane)) c[j] = 0;
    }
    return mine;
}

// Scores, choice and weights of token t. Lane r < k returns its pick's id.
template <int NPL>
__device__ __forceinline__ int route_token(const LogitArgs& a, const float (&bias)[NPL], int t,
                                           int lane, unsigned long long* scr) {
    const bool by_logit = a.bias == nullptr;
    const bool limited = a.topk_group < a.n_group;
    const bool softmax = a.score == HF_SCORE_SOFTMAX;
    float l[NPL];
    uint32_t c[NPL];
    // (uniform branches around whole loops: a choice inside one is made per expert)
    if (a.bf16) {
        const uint16_t* p = static_cast<const uint16_t*>(a.logits) + size_t(t) * a.E + lane;
#pragma unroll
        for (int j = 0; j < NPL; ++j)
            l[j] = j * 32 + lane < a.E ? bf16_to_f32(p[j * 32]) : -INFINITY;
    } else {
        const float* p = static_cast<const float*>(a.logits) + size_t(t) * a.E + lane;
#pragma unroll
        for (int j = 0; j < NPL; ++j) l[j] = j * 32 + lane < a.E ? p[j * 32] : -INFINITY;
    }
    float top = l[0];
#pragma unroll
    for (int j = 1; j < NPL; ++j) top = fmaxf(top, l[j]);
    top = warp_max_f(top);
    const float m = top == -INFINITY ? 0.0f : top;  // exp(-inf - 0) = 0
    float inv = 1.0f;
    if (softmax) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < NPL; ++j) sum += __expf(l[j] - m);
        sum = warp_sum(sum);
        inv = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);  // 0: every logit is -inf
    }
    float tol = 0.0f, ggap = INFINITY;
    if (!by_logit || (limited && a.group_top == 2)) {
        // Keys on the fast exponential (2 + 1.2 |x| units of 2^-23). Bounds on a
        // score's error, for the largest score smax. Sigmoid: s (1 - s) times the
        // exponential's, which is largest at the largest logit, and the sum and
        // quotient: < smax (2^-21 + 2^-22 |top|, the latter where top < 0).
        // Softmax: the exponent's rounding and the exponential's stay below 3 units
        // (e^-x (2 + 1.2 x) <= 2), the sum's error below 3 and NPL + 5 roundings:
        // < 2^-18 smax. Two keys can be off by twice that (tol), two groups' sums
        // of two by four times; the roundings of the sums are above()'s.
        float s[NPL];
        if (softmax) {
#pragma unroll
            for (int j = 0; j < NPL; ++j) s[j] = fmaf(__expf(l[j] - m), inv, bias[j]);
            tol = inv * 0x1p-17f;
        } else {
#pragma unroll
            for (int j = 0; j < NPL; ++j)
                s[j] = __fdividef(1.0f, 1.0f + __expf(-l[j])) + bias[j];
            tol = __fdividef(1.0f, 1.0f + __expf(-top)) *
                      (0x1p-20f + fmaxf(-top, 0.0f) * 0x1p-21f) +
                  0x1p-120f;  // quotients below 2^-126 come out as 0
        }
        uint32_t key[NPL];
#pragma unroll
        for (int j = 0; j < NPL; ++j)
            key[j] = j * 32 + lane < a.E ? packed<NPL>(code_of(s[j]), j) : 0u;
        if (by_logit) {
#pragma unroll
            for (int j = 0; j < NPL; ++j)
                c[j] = j * 32 + lane < a.E ? packed<NPL>(code_of(l[j]), j) : 0u;
            keep_groups(c, key, a, lane, reinterpret_cast<uint32_t*>(scr), &ggap);
        } else {
#pragma unroll
            for (int j = 0; j < NPL; ++j) c[j] = key[j];
            if (limited) keep_groups(c, c, a, lane, reinterpret_cast<uint32_t*>(scr), &ggap);
        }
    } else {
#pragma unroll
        for (int j = 0; j < NPL; ++j)
            c[j] = j * 32 + lane < a.E ? packed<NPL>(code_of(l[j]), j) : 0u;
        if (limited) keep_groups(c, c, a, lane, reinterpret_cast<uint32_t*>(scr), &ggap);
    }
    sort_lane(c);
    int mine = 0;
    uint32_t mc = 0;  // lane r < k: the r-th pick and its code
#pragma unroll 1
    for (int r = 0; r < a.k; ++r) {
        int id;
        const uint32_t m1 = take_best(c, lane, &id);
        if (lane == r) {
            mine = id;
            mc = m1;
        }
    }
    uint32_t left = warp_max(c[0]);  // the first one left out (0: none)
    // Logits rank exactly but for the replaced bits, which bf16 logits leave 0.
    const bool ranked = by_logit && a.bf16;
    const uint32_t before = __shfl_up_sync(~0u, mc, 1);
    bool close = lane > 0 && lane < a.k && is_close<NPL>(before, mc, by_logit, tol);
    uint32_t last = __shfl_sync(~0u, mc, a.k - 1);
    bool open = left && is_close<NPL>(last, left, by_logit, tol);
    if (limited && !(ggap > 2.0f * tol) && !(ranked && a.group_top == 1)) {
        mine = pick_exact<NPL>(a, t, lane, scr);
    } else if (!ranked && (__any_sync(~0u, close) || open)) {
        int n = a.k;  // candidates: on until one is clearly below
        while (open && n < 32) {
            int id;
            last = take_best(c, lane, &id);
            if (lane == n) mine = id;
            ++n;
            left = warp_max(c[0]);
            open = left && is_close<NPL>(last, left, by_logit, tol);
        }
        mine = open ? pick_exact<NPL>(a, t, lane, scr) : refine(a, t, lane, mine, n);
    }

    // the picks' scores once more, accurately
    const float lp = load_logit(a, size_t(t) * a.E + (lane < a.k ? mine : 0));
    float ws;
    if (softmax) ws = __fmul_rn(expf(lp - m), inv);
    else ws = __fdiv_rn(1.0f, __fadd_rn(1.0f, expf(-lp)));
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

// ids: of the block's tokens [nt x k]
__device__ __forceinline__ void scatter(const LogitArgs& a, const uint32_t* masks, const int* base,
                                        const int* ids, int t0, int nt, int words) {
    for (int i = threadIdx.x; i < nt * a.k; i += blockDim.x) {
        const int e = ids[i];
        a.perm[base[e] + mask_rank(masks + e * words, i / a.k)] = t0 * a.k + i;
    }
}

// Block b routes tokens [b * tb, ...) and counts them per expert; a launch of
// one block goes on to the permutation.
template <int NPL, int THREADS>
__global__ void __launch_bounds__(THREADS) k_route_logits(LogitArgs a) {
    extern __shared__ __align__(16) uint32_t sm[];
    const int words = (a.tb + 31) / 32;
    // groups: a scratch row of 64-bit codes per warp, in front
    auto* scr = reinterpret_cast<unsigned long long*>(sm) + size_t(threadIdx.x >> 5) * a.E;
    uint32_t* masks = sm + (a.topk_group < a.n_group ? size_t(blockDim.x >> 5) * a.E * 2 : 0);
    int* total = reinterpret_cast<int*>(masks + size_t(a.E) * words);  // [E]; masks [E][words]
    int* base = total + a.E;                                      // [E]
    const int t0 = blockIdx.x * a.tb, nt = min(a.tb, a.T - t0);
    int* s_ids = base + a.E;                                      // [tb][k] (one block)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    griddep_launch_dependents();
    float bias[NPL];
#pragma unroll
    for (int j = 0; j < NPL; ++j)
        bias[j] = a.bias && j * 32 + lane < a.E ? a.bias[j * 32 + lane] : 0.0f;
    for (int i = threadIdx.x; i < a.E * words; i += blockDim.x) masks[i] = 0u;
    __syncthreads();
    for (int tl = warp; tl < nt; tl += int(blockDim.x >> 5)) {
        const int id = route_token<NPL>(a, bias, t0 + tl, lane, scr);
        if (lane < a.k) {
            atomicOr(&masks[id * words + (tl >> 5)], 1u << (tl & 31));
            if (gridDim.x == 1) s_ids[tl * a.k + lane] = id;
        }
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
    scatter(a, masks, base, s_ids, t0, nt, words);
}

// Very long batches: blk becomes its exclusive prefix over the blocks (row nb: the
// totals), so that the scatter need not add up every block's counts. A lane has an
// expert, a warp one of 32 slices of the blocks.
__global__ void __launch_bounds__(1024) k_route_scan(LogitArgs a, int nb) {
    __shared__ int sums[32][32];
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
    const int per = (nb + 31) / 32, q0 = min(slice * per, nb), q1 = min(q0 + per, nb);
    int run = 0;
    if (e < a.E) {
#pragma unroll 8
        for (int q = q0; q < q1; ++q) run += a.blk[size_t(q) * a.E + e];
    }
    sums[slice][lane] = run;
    __syncthreads();
    run = 0;
    for (int s = 0; s < slice; ++s) run += sums[s][lane];
    if (e >= a.E) return;
#pragma unroll 8
    for (int q = q0; q < q1; ++q) {
        int32_t* p = a.blk + size_t(q) * a.E + e;
        const int c = *p;
        *p = run;
        run += c;
    }
    if (slice == 31) a.blk[size_t(nb) * a.E + e] = run;
}

// Per-expert tokens of all blocks, and of those before b. Threads cover (slice of
// blocks, V experts); integer sums, any order.
template <int V>
__device__ __forceinline__ void add_counts(const LogitArgs& a, int nb, int b, int* total, int* base) {
    const int cols = min(a.E / V, int(blockDim.x)), slices = int(blockDim.x) / cols;
    const int slice = int(threadIdx.x) / cols;
    if (slice >= slices) return;
    for (int c = int(threadIdx.x) % cols; c < a.E / V; c += cols) {
        int all[V] = {}, before[V] = {};
#pragma unroll 4
        for (int q = slice; q < nb; q += slices) {
            int v[V];
            const int32_t* p = a.blk + size_t(q) * a.E + c * V;
            if constexpr (V == 4) {
                const int4 x = *reinterpret_cast<const int4*>(p);
                v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
            } else {
                v[0] = p[0];
            }
#pragma unroll
            for (int e = 0; e < V; ++e) {
                all[e] += v[e];
                before[e] += q < b ? v[e] : 0;
            }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
            atomicAdd(&total[c * V + e], all[e]);
            atomicAdd(&base[c * V + e], before[e]);
        }
    }
}

// `scanned`: after k_route_scan.
__global__ void __launch_bounds__(1024) k_route_scatter(LogitArgs a, int nb, int scanned) {
    extern __shared__ __align__(16) uint32_t sm[];
    const int words = (a.tb + 31) / 32;
    uint32_t* masks = sm;
    int* total = reinterpret_cast<int*>(sm + size_t(a.E) * words);
    int* base = total + a.E;
    const int b = blockIdx.x, t0 = b * a.tb, nt = min(a.tb, a.T - t0);
    for (int i = threadIdx.x; i < a.E * words; i += blockDim.x) masks[i] = 0u;
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) total[e] = base[e] = 0;
    griddep_wait();  // the ids and counts of every block
    __syncthreads();
    if (scanned) {
        for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
            total[e] = a.blk[size_t(nb) * a.E + e];
            base[e] = a.blk[size_t(b) * a.E + e];
        }
    } else if (a.E % 4 == 0) {
        add_counts<4>(a, nb, b, total, base);
    } else {
        add_counts<1>(a, nb, b, total, base);
    }
    set_masks(a, masks, t0, nt, words);
    __syncthreads();
    segment_bases(a, total, base, b == 0);
    scatter(a, masks, base, a.ids + size_t(t0) * a.k, t0, nt, words);
}

__global__ void k_route_empty(LogitArgs a) {
    for (int e = threadIdx.x; e <= a.E + 1; e += blockDim.x) {
        if (e <= a.E) a.counts[e] = 0;
        a.offsets[e] = 0;
    }
}

// Tokens per block: all of up to 16 tokens in one; else as many as leave one block
// per SM, in steps of 8, 512 at most (the second launch adds up the counts of all
// blocks).
int tokens_per_block(int T) {
    if (T <= kOneBlockT) return kOneBlockT;
    return std::min(512, ((T + 147) / 148 + 7) / 8 * 8);
}

int blocks_of(int T) {
    const int tb = tokens_per_block(T);
    return (T + tb - 1) / tb;
}

size_t ws_bytes(int T, int E) {
    if (T <= kOneBlockT) return 0;
    return (size_t(blocks_of(T) + 1) * E * sizeof(int32_t) + kWsAlign - 1) / kWsAlign * kWsAlign;
}

template <int NPL>
hf_status launch(const LogitArgs& a, cudaStream_t st) {
    // registers: NPL scores and codes per lane (and 64-bit ones in the rare path)
    constexpr int kThreads = NPL <= 8 ? 1024 : 256;
    const int nb = blocks_of(a.T);
    const int smem = a.E * ((a.tb + 31) / 32 + 2) * 4;
    const auto kern = k_route_logits<NPL, kThreads>;
    // a warp per token, or per equal number of tokens; eight warps at least (they
    // also count and permute)
    const int most = kThreads / 32, tokens = std::min(a.T, a.tb), turns = (tokens + most - 1) / most;
    const int threads = std::max(8, (tokens + turns - 1) / turns) * 32;
    const int own = smem + (nb == 1 ? a.T * a.k * 4 : 0) +
                    (a.topk_group < a.n_group ? threads / 32 * a.E * 8 : 0);
    if (own > kPlainSmem) HF_CUDA(ensure_smem(reinterpret_cast<const void*>(kern), own));
    kern<<<nb, threads, own, st>>>(a);
    HF_CUDA(cudaGetLastError());
    if (nb > 1) {
        if (smem > kPlainSmem)
            HF_CUDA(ensure_smem(reinterpret_cast<const void*>(k_route_scatter), smem));
        const int scan = nb > kScanBlocks;
        if (scan) {
            k_route_scan<<<(a.E + 31) / 32, 1024, 0, st>>>(a, nb);
            HF_CUDA(cudaGetLastError());
        }
        HF_CUDA(launch_pdl(k_route_scatter, dim3(nb), dim3(nb > 16 ? 1024 : 256), size_t(smem), st,
                           a, nb, scan));
    }
    return HF_OK;
}

hf_status check_spec(const hf_route_spec* s, const char* fn) {
    const auto refuse = [&](const char* why) {
        return fail(HF_ERR_ARG, std::string(fn) + ": " + why);
    };
    if (!s) return refuse("null spec");
    if (s->num_experts < 1 || s->num_experts > kMaxExperts)
        return refuse("num_experts must be in 1..1024");
    if (s->score != HF_SCORE_SIGMOID && s->score != HF_SCORE_SOFTMAX)
        return refuse("score must be HF_SCORE_SIGMOID or HF_SCORE_SOFTMAX");
    if (s->n_group < 1 || s->n_group > kMaxRouteGroups || s->num_experts % s->n_group)
        return refuse("n_group must be in 1..32 and divide num_experts");
    if (s->topk_group < 1 || s->topk_group > s->n_group)
        return refuse("topk_group must be in 1..n_group");
    if (s->group_top != 1 && s->group_top != 2)
        return refuse("group_top must be 1 or 2");
    if (s->top_k < 1 || s->top_k > kMaxRouteK ||
        s->top_k > s->topk_group * (s->num_experts / s->n_group))
        return refuse("top_k must be in 1..32 and at most the experts of the kept groups");
    return HF_OK;
}

}  // namespace
}  // namespace hf

using namespace hf;

extern "C" {

size_t hf_route_workspace_size(int T, const hf_route_spec* spec) {
    if (T <= 0 || T > kMaxExtent || check_spec(spec, "hf_route_workspace_size") != HF_OK) return 0;
    return ws_bytes(T, spec->num_experts);
}

hf_status hf_route_logits(const void* logits, hf_dtype dtype, const float* bias, int T,
                          const hf_route_spec* spec, const hf_moe_routing* r, void* workspace,
                          size_t workspace_bytes, hf_stream stream) {
    HF_TRY(check_spec(spec, "hf_route_logits"));
    if (dtype != HF_BF16 && dtype != HF_F32)
        return fail(HF_ERR_ARG, "hf_route_logits: logits must be bf16 or f32");
    if (T < 0 || (long long)T * spec->top_k > kMaxExtent)
        return fail(HF_ERR_ARG, "hf_route_logits: T >= 0 and T * top_k at most 2^31 - 4096");
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
    a.group_top = a.E == a.n_group ? 1 : spec->group_top;  // a group of one has no second key
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
