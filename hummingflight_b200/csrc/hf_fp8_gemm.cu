// hf_fp8_gemm.cu -- the block-scaled product of e4m3 rows and e4m3 weight rows
// on the tensor cores, for one weight matrix or one per expert segment:
//   out[p, n] = sum_b sx[p, b] sw[n / 128, b] sum_{j in block b} xq[p, j] w[n, j]
//
// Orientation: the MMA's M = 128 weight rows, N = positions (tokens), both
// K-major, so the row-major weights feed the tensor cores as they lie and a
// segment of any length costs MMA columns in steps of 16 only. A tile is two
// blocks of 128 weight rows (gate and up rows of the same intermediate columns,
// or 256 output columns) x up to BN positions.
//
// The scales change every 128 columns of K, so the tensor memory accumulator
// holds one block of 128 (four kind::f8f6f4 steps of 32) and is then read back,
// multiplied by the position's and the weight block's scale and added to fp32
// registers. Two or four accumulator buffers let the MMAs of the next blocks run
// meanwhile.
//
// Warps: 0 TMA producer, 1 MMA issuer and TMEM owner, 2 scales (it writes the
// products of both scales per position into a ring in shared memory), 4-11
// accumulation and epilogue (two per TMEM lane quadrant, alternate 16-column
// chunks). One CTA per SM, tiles dealt round-robin; the tiles that share weight
// rows have adjacent ids, so their CTAs read those rows from L2 together.
// Every wait is bounded (hf_sm100.cuh).
//
// The gate/up epilogue evaluates silu(g) * u, takes the maximum over the tile's
// 128 intermediate columns (one block) per position and writes e4m3 values and
// the scale, so the intermediate never leaves the SM in more than 8 bits.
#include <algorithm>
#include <atomic>
#include <map>
#include <mutex>

#include "hf_fp8.cuh"
#include "hf_sm100.cuh"

namespace hf {
namespace {

using namespace sm100;

constexpr int kThreads = 384;
constexpr int kAccWarps = 8;
// Mean positions per segment up to which the weights are the MMA's M, and up to
// which a tile takes 32 positions instead of 64. 32 experts of 6144 x 2048, the
// three kernels' us: mean 4: 226 (32), 234 (64), 378 (pair); 48: 274, 279, 386;
// 64: 277, 293, 384; 96: 392, 389, 394; 128: 490, 420, 394. One matrix, 64
// rows x 12288 -> 6144: 24.6 (32), 22.3 (64).
constexpr int kNarrowRows = 96;
constexpr int kNarrow32 = 48;
constexpr int kScaleSlots = 4;
constexpr uint32_t kABytes = 128 * 128;  // 128 weight rows x 128 bytes
constexpr uint64_t kWaitNs = 2000ull * 1000 * 1000;
// What a warp that gave up waits for its copies or MMAs in flight, all together: a
// thousand times what they take. (Barriers that also wait for copies never asked for
// do not complete.)
constexpr uint64_t kDrainNs = 20ull * 1000 * 1000;

template <int BN>
struct Cfg {
    static constexpr int kStageBytes = 2 * kABytes + BN * 128;
    static constexpr int kCols = 2 * BN;                     // TMEM columns of one buffer
    static constexpr int kBufs = 4;
    static constexpr uint32_t kTmemCols = kBufs * kCols;     // a power of two, 128..512
    static constexpr int kBoxB = 32;                         // position rows of one TMA box
    static constexpr int kScaleBytes = kScaleSlots * 2 * BN * 4;
    static constexpr int kRedBytes = 5 * BN * 4;             // maxima of 4 quadrants, 1 / scale
    static constexpr int kBarBytes = 512;
    static constexpr int kFixed = kScaleBytes + kRedBytes + kBarBytes;
    // the plan: offsets and tile prefix of up to 1024 segments
    static constexpr int kStages0 = (227 * 1024 - 1024 - kFixed - 2 * 1025 * 4) / kStageBytes;
    static constexpr int kStages = kStages0 > 8 ? 8 : kStages0;
    static_assert((2 * kStages + kBufs + 2 * kScaleSlots + 2) * 8 + 8 <= kBarBytes, "barriers");
    static_assert(kStageBytes % 1024 == 0 && kStages >= 3, "stages");
    static int smem(int G) { return 1024 + kStages * kStageBytes + kFixed + 2 * (G + 1) * 4; }
};

struct Tile {
    int row0, n;      // first position, positions
    int m0;           // first weight row of block 0 in its matrix
    int kb0, kb1;     // blocks of K
    long long out0;   // first output row (behind the planes of earlier runs of K)
    int a0, a1;       // TMA rows of the two blocks
    const float* s0;  // weight scales of the two blocks, [kb]
    const float* s1;
};

__device__ __forceinline__ int find_segment(const int* pref, int G, int u) {
    int lo = 0, hi = G - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (pref[mid] <= u) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Segment offsets (clipped to the rows) and the prefix of their tiles, into
// shared memory; the whole block calls it.
template <int BN>
__device__ __forceinline__ void load_plan(const Fp8Args& a, int MB, int* off, int* pref) {
    const int lane = threadIdx.x & 31;
    if (a.offsets) {
        for (int g = threadIdx.x; g <= a.G; g += blockDim.x)
            off[g] = min(max(a.offsets[g], 0), a.rows);
    } else if (threadIdx.x == 0) {
        off[0] = 0;
        off[1] = a.rows;
    }
    __syncthreads();
    if (threadIdx.x >= 64 && threadIdx.x < 96) {  // warp 2
        int run = 0;
        for (int g0 = 0; g0 < a.G; g0 += 32) {
            const int g = g0 + lane;
            const int c = g < a.G ? max(off[g + 1] - off[g], 0) : 0;
            int inc = (c + BN - 1) / BN * MB;
            const int v = inc;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(~0u, inc, o);
                if (lane >= o) inc += y;
            }
            if (g < a.G) pref[g] = run + inc - v;
            run += __shfl_sync(~0u, inc, 31);
        }
        if (lane == 0) pref[a.G] = run;
    }
}

template <bool GLU, int BN>
__device__ __forceinline__ void decode(const Fp8Args& a, const int* off, const int* pref, int KB,
                                       int u, Tile& t) {
    t.kb0 = 0;
    t.kb1 = KB;
    t.out0 = 0;
    if (!GLU && a.nsplit > 1) {  // runs of K of one tile are adjacent
        const int ks = u % a.nsplit;
        u /= a.nsplit;
        t.kb0 = ks * a.kbper;
        t.kb1 = min(KB, t.kb0 + a.kbper);
        t.out0 = (long long)ks * a.rows;
    }
    const int g = find_segment(pref, a.G, u);
    const int c = off[g + 1] - off[g];
    const int nt = (c + BN - 1) / BN, nw = (c + nt - 1) / nt;  // equal widths
    const int local = u - pref[g], mi = local / nt, ni = local % nt;
    t.row0 = off[g] + ni * nw;
    t.out0 += t.row0;
    t.n = min(nw, c - ni * nw);
    t.m0 = mi * (GLU ? 128 : 256);
    t.a0 = g * a.a_stride + a.a_base + t.m0;
    t.a1 = t.a0 + (GLU ? a.N : 128);
    const int rb = t.m0 / kFp8Block;
    t.s0 = a.sw + g * a.sw_stride + size_t(rb) * KB;
    // past the last row block of the matrix nothing is stored: any scale does
    if (GLU) t.s1 = t.s0 + a.sw_up;
    else t.s1 = t.m0 + 128 < a.N ? t.s0 + KB : t.s0;
}

__device__ __forceinline__ void drain_wait(uint64_t* bar, uint32_t parity, uint64_t deadline) {
    while (!mbar_try_wait(bar, parity))
        if (globaltimer() > deadline) return;
}

// Four accumulators += sums times scales. (Packed pairs, fma.rn.f32x2, run at the
// same rate and cost moves to pair the registers: in the pair kernel 324 us against
// 297 on 4096 x 12288 x 6144.)
__device__ __forceinline__ void add4(float* acc, const uint32_t* d, float4 s) {
    acc[0] = fmaf(__uint_as_float(d[0]), s.x, acc[0]);
    acc[1] = fmaf(__uint_as_float(d[1]), s.y, acc[1]);
    acc[2] = fmaf(__uint_as_float(d[2]), s.z, acc[2]);
    acc[3] = fmaf(__uint_as_float(d[3]), s.w, acc[3]);
}

// What a warp that gave up leaves in place of an output.
__device__ __forceinline__ void store_nan(const Fp8Args& a, long long row, int col) {
    if (col >= a.N) return;
    const size_t o = size_t(row) * a.N + col;
    if (a.out_f32) static_cast<uint32_t*>(a.out)[o] = 0x7fffffffu;
    else static_cast<uint16_t*>(a.out)[o] = 0x7fffu;  // bf16, FP16 or the upper half of 24 bits
}

// AUX: the outputs take Fp8Args::out_aux's form. (A kernel of its own: as a branch its
// unrolled code cost the plain form 4 us of 41 where each CTA has one tile.)
// HOOK: Fp8Args::wait_ns and stall hold. (A kernel of its own as well: a limit that is
// not a constant and the check of the block cost 64 x 6144 x 12288 0.8 us of 23.7, and
// the pair kernel up to 5 %.)
template <bool GLU, int BN, bool AUX, bool HOOK>
__global__ void __launch_bounds__(kThreads, 1)
    k_fp8_mma(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
              const Fp8Args a) {
    using C = Cfg<BN>;
    constexpr int S = C::kStages, NB = C::kBufs;
    constexpr int CH = BN / 32;  // 16-column chunks of one accumulation warp
    extern __shared__ __align__(1024) uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) &
                                               ~uintptr_t(1023));
    float* sc = reinterpret_cast<float*>(smem + S * C::kStageBytes);  // [slot][2][BN]
    uint32_t* red = reinterpret_cast<uint32_t*>(sc + kScaleSlots * 2 * BN);  // [4][BN]
    float* invs = reinterpret_cast<float*>(red + 4 * BN);                    // [BN]
    uint64_t* full = reinterpret_cast<uint64_t*>(invs + BN);
    uint64_t* done = full + S;      // a block's MMAs: its stage is free, its sums are ready
    uint64_t* tempty = done + S;
    uint64_t* sfull = tempty + NB;
    uint64_t* sempty = sfull + kScaleSlots;
    uint64_t* final_bar = sempty + kScaleSlots;
    uint64_t* stall_bar = final_bar + 1;  // never signalled (test hook)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(stall_bar + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* off = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(full) + C::kBarBytes);  // [G+1]
    int* pref = off + a.G + 1;                                                           // [G+1]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int KB = (a.K + kFp8Block - 1) / kFp8Block;
    const int MB = GLU ? (a.N + 127) / 128 : (a.N + 255) / 256;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&done[s], 1);
        }
        for (int b = 0; b < NB; ++b) mbar_init(&tempty[b], kAccWarps);
        for (int b = 0; b < kScaleSlots; ++b) {
            mbar_init(&sfull[b], 1);
            mbar_init(&sempty[b], kAccWarps);
        }
        mbar_init(final_bar, 1);
        mbar_init(stall_bar, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, C::kTmemCols);
        tmem_relinquish();
    }
    // the rows, the offsets, the workspace's earlier users; early: the producer's first
    // weights are on their way meanwhile, and each warp that needs the rest waits below
    if (!a.early) griddep_wait();
    if (a.clear_err && blockIdx.x == 0 && threadIdx.x == 0) *a.err = 0;
    load_plan<BN>(a, MB, off, pref);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int total = pref[a.G] * (GLU ? 1 : a.nsplit);
    const auto wait = [&](uint64_t* bar, uint32_t parity) {
        return mbar_wait_for(smem_u32(bar), parity, abort_flag, HOOK ? a.wait_ns : kWaitNs);
    };

    if (warp < 4) {
        if (warp == 0) {
            // ------------------------------------------------------ TMA producer
            tma_prefetch_desc(&tmA);
            tma_prefetch_desc(&tmB);
            const auto bytes = [](const Tile& t) {
                return 2 * kABytes + (t.n + C::kBoxB - 1) / C::kBoxB * C::kBoxB * 128;
            };
            const auto load_weights = [&](const Tile& t, uint32_t s, int kb) {
                uint8_t* st = smem + s * C::kStageBytes;
                mbar_arrive_expect_tx(&full[s], bytes(t));
                tma_load_2d(st, &tmA, &full[s], kb * 128, t.a0);
                tma_load_2d(st + kABytes, &tmA, &full[s], kb * 128, t.a1);
            };
            uint32_t it = 0, pre = 0;  // pre: stages whose weights are already requested
            if (a.early && int(blockIdx.x) < total) {
                Tile t;
                decode<GLU, BN>(a, off, pref, KB, int(blockIdx.x), t);
                pre = uint32_t(min(S, t.kb1 - t.kb0));
                if (elect_one())
                    for (uint32_t s = 0; s < pre; ++s) load_weights(t, s, t.kb0 + int(s));
                __syncwarp();
            }
            griddep_wait();
            griddep_launch_dependents();
            const uint32_t stall = HOOK && a.stall > 0 ? uint32_t(a.stall) - 1 : ~0u;
            bool ok = true;
            for (int u = blockIdx.x; u < total && ok; u += gridDim.x) {
                Tile t;
                decode<GLU, BN>(a, off, pref, KB, u, t);
                const int nb = (t.n + C::kBoxB - 1) / C::kBoxB;
                for (int kb = t.kb0; kb < t.kb1; ++kb, ++it) {
                    const uint32_t s = it % S;
                    if (!wait(&done[s], ((it / S) & 1) ^ 1) ||
                        (HOOK && it == stall && !wait(stall_bar, 0))) {
                        ok = false;
                        break;
                    }
                    if (elect_one()) {
                        if (it >= pre) load_weights(t, s, kb);
                        uint8_t* at = smem + s * C::kStageBytes + 2 * kABytes;
                        for (int j = 0; j < nb; ++j)
                            tma_load_2d(at + j * C::kBoxB * 128, &tmB, &full[s], kb * 128,
                                        t.row0 + j * C::kBoxB);
                    }
                    __syncwarp();
                }
            }
            if (!ok) {  // every issued load lands before the CTA leaves
                const uint64_t dl = globaltimer() + kDrainNs;
                const uint32_t first = it > uint32_t(S) ? it - S : 0;
                it = max(it, pre);
                for (uint32_t i = first; i < it; ++i) drain_wait(&full[i % S], (i / S) & 1, dl);
            }
        } else if (warp == 1) {
            // ------------------------------------------------------ MMA issuer
            griddep_wait();  // so that its waits are timed from there
            uint32_t it = 0;
            bool ok = true;
            for (int u = blockIdx.x; u < total && ok; u += gridDim.x) {
                Tile t;
                decode<GLU, BN>(a, off, pref, KB, u, t);
                const uint32_t idesc = idesc_e4m3_m128(uint32_t(t.n + 15) & ~15u);
                for (int kb = t.kb0; kb < t.kb1; ++kb, ++it) {
                    const uint32_t s = it % S, b = it % NB;
                    if (!wait(&tempty[b], ((it / NB) & 1) ^ 1) || !wait(&full[s], (it / S) & 1)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t st = smem_u32(smem + s * C::kStageBytes);
                        const uint32_t d = tmem_base + b * C::kCols;
#pragma unroll
                        for (int ai = 0; ai < 2; ++ai)
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk)
                                mma_f8(d + ai * BN, desc_k_sw128(st + ai * kABytes) + 2 * kk,
                                       desc_k_sw128(st + 2 * kABytes) + 2 * kk, idesc, kk != 0);
                        mma_commit(&done[s]);
                    }
                    __syncwarp();
                }
            }
            if (elect_one()) mma_commit(final_bar);  // once every MMA issued above is done
            __syncwarp();
            drain_wait(final_bar, 0, globaltimer() + kDrainNs);
        } else if (warp == 2) {
            // ------------------------------------------------------ scales
            constexpr int PL = BN / 32;
            griddep_wait();
            uint32_t it = 0;
            bool ok = true;
            for (int u = blockIdx.x; u < total && ok; u += gridDim.x) {
                Tile t;
                decode<GLU, BN>(a, off, pref, KB, u, t);
                float x[PL], w0 = t.s0[t.kb0], w1 = t.s1[t.kb0];
                const float* xp[PL];
#pragma unroll
                for (int j = 0; j < PL; ++j) {
                    const int c = j * 32 + lane;
                    xp[j] = c < t.n ? a.sx + size_t(t.row0 + c) * KB : nullptr;
                    x[j] = xp[j] ? xp[j][t.kb0] : 0.0f;
                }
                for (int kb = t.kb0; kb < t.kb1; ++kb, ++it) {
                    float xn[PL], v0 = 0.0f, v1 = 0.0f;  // the next block's, in flight
                    const bool more = kb + 1 < t.kb1;
#pragma unroll
                    for (int j = 0; j < PL; ++j) xn[j] = more && xp[j] ? xp[j][kb + 1] : 0.0f;
                    if (more) {
                        v0 = t.s0[kb + 1];
                        v1 = t.s1[kb + 1];
                    }
                    const uint32_t q = it % kScaleSlots;
                    if (!wait(&sempty[q], ((it / kScaleSlots) & 1) ^ 1)) {
                        ok = false;
                        break;
                    }
                    float* p = sc + q * 2 * BN;
#pragma unroll
                    for (int j = 0; j < PL; ++j) {
                        const int c = j * 32 + lane;
                        p[c] = x[j] * w0;
                        p[BN + c] = x[j] * w1;
                        x[j] = xn[j];
                    }
                    w0 = v0;
                    w1 = v1;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sfull[q]);
                }
            }
        }
    } else {
        // ---------------------------------------------------------- accumulation
        const int q = warp & 3, h = (warp - 4) >> 2;
        const int r = q * 32 + lane;
        const uint32_t lanes = tmem_base + (uint32_t(q * 32) << 16);
        griddep_wait();
        uint32_t it = 0;
        bool ok = true;
        for (int u = blockIdx.x; u < total; u += gridDim.x) {
            Tile t;
            decode<GLU, BN>(a, off, pref, KB, u, t);
            // chunks of 16 columns at (2 i + h) * 16
            const int nc = t.n > h * 16 ? (t.n - h * 16 + 31) / 32 : 0;
            float g[CH][16], v[CH][16];
#pragma unroll
            for (int i = 0; i < CH; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) g[i][j] = v[i][j] = 0.0f;
            for (int kb = t.kb0; kb < t.kb1; ++kb, ++it) {
                const uint32_t b = it % NB, sl = it % kScaleSlots;
                if (!wait(&done[it % S], (it / S) & 1) ||
                    !wait(&sfull[sl], (it / kScaleSlots) & 1)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t ta = lanes + b * C::kCols + h * 16;
                const float* p = sc + sl * 2 * BN + h * 16;
                uint32_t d0[2][16], d1[2][16];
                if (nc > 0) {
                    tmem_ld16(ta, d0[0]);
                    tmem_ld16(ta + BN, d1[0]);
                    tmem_ld_wait_regs(d0[0], d1[0]);
                }
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    if (i < nc) {
                        if (i + 1 < nc) {
                            tmem_ld16(ta + (i + 1) * 32, d0[(i + 1) & 1]);
                            tmem_ld16(ta + BN + (i + 1) * 32, d1[(i + 1) & 1]);
                        }
#pragma unroll
                        for (int j = 0; j < 16; j += 4) {
                            const float4 s0 = *reinterpret_cast<const float4*>(p + i * 32 + j);
                            const float4 s1 = *reinterpret_cast<const float4*>(p + BN + i * 32 + j);
                            const uint32_t(&e0)[16] = d0[i & 1];
                            const uint32_t(&e1)[16] = d1[i & 1];
                            add4(&g[i][j], &e0[j], s0);
                            add4(&v[i][j], &e1[j], s1);
                        }
                        if (i + 1 < nc) tmem_ld_wait_regs(d0[(i + 1) & 1], d1[(i + 1) & 1]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&tempty[b]);
                    mbar_arrive(&sempty[sl]);
                }
            }
            if (!ok) {
                // NaN for this tile and the rest. GLU: through the maxima and scales, and
                // the barriers below, where the half's other warps may wait, are met.
                // (NaN in the sums and the ordinary epilogue: 64 x 6144 x 12288 24.8 us
                // instead of 23.7, since the accumulators outlive the loop over blocks.)
#pragma unroll 1
                for (; u < total; u += gridDim.x) {
                    decode<GLU, BN>(a, off, pref, KB, u, t);
                    if constexpr (GLU) {
                        for (int c = lane; c < BN; c += 32)
                            if (((c >> 4) & 1) == h) red[q * BN + c] = 0x7fffffffu;
                        named_bar_sync(1 + h, 128);
                        for (int c = r; c < BN / 2; c += 128) {
                            const int col = ((c >> 4) * 2 + h) * 16 + (c & 15);
                            invs[col] = __uint_as_float(0x7fffffffu);
                            if (col < t.n)
                                a.mid_s[size_t(t.row0 + col) * ((a.N + 127) / 128) + t.m0 / 128] =
                                    __uint_as_float(0x7fffffffu);
                        }
                        named_bar_sync(1 + h, 128);
                    } else {
#pragma unroll 1
                        for (int c = h * 16; c < t.n; c += (c & 15) == 15 ? 17 : 1) {
                            store_nan(a, t.out0 + c, t.m0 + r);
                            store_nan(a, t.out0 + c, t.m0 + 128 + r);
                        }
                    }
                }
                break;
            }
            if constexpr (GLU) {
                // silu(g) * u, and its maximum over the 128 rows per position
                const bool rv = t.m0 + r < a.N;
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    if (i < nc) {
                        uint32_t top = 0;
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            g[i][j] = rv ? swiglu_fast(g[i][j], v[i][j]) : 0.0f;
                            const uint32_t x = __reduce_max_sync(
                                ~0u, __float_as_uint(g[i][j]) & 0x7fffffffu);
                            if (lane == j) top = x;
                        }
                        if (lane < 16) red[q * BN + (2 * i + h) * 16 + lane] = top;
                    }
                }
                named_bar_sync(1 + h, 128);
                for (int c = r; c < nc * 16; c += 128) {
                    const int col = ((c >> 4) * 2 + h) * 16 + (c & 15);
                    const uint32_t top = max(max(red[col], red[BN + col]),
                                             max(red[2 * BN + col], red[3 * BN + col]));
                    float inv;
                    const float s = block_scale(__uint_as_float(top), inv);
                    invs[col] = inv;
                    if (col < t.n)
                        a.mid_s[size_t(t.row0 + col) * ((a.N + 127) / 128) + t.m0 / 128] = s;
                }
                named_bar_sync(1 + h, 128);
                if (rv) {
#pragma unroll
                    for (int i = 0; i < CH; ++i) {
#pragma unroll
                        for (int j = 0; j < 16; j += 2) {
                            const int c = (2 * i + h) * 16 + j;
                            if (i < nc && c < t.n) {
                                uint16_t e;
                                asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;"
                                    : "=h"(e)
                                    : "f"(g[i][j + 1] * invs[c + 1]), "f"(g[i][j] * invs[c]));
                                uint8_t* o = a.mid_q + size_t(t.row0 + c) * a.N + t.m0 + r;
                                o[0] = uint8_t(e);
                                if (c + 1 < t.n) o[a.N] = uint8_t(e >> 8);
                            }
                        }
                    }
                }
            } else if constexpr (AUX) {
#pragma unroll
                for (int i = 0; i < CH; ++i)
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int c = (2 * i + h) * 16 + j;
                        if (i < nc && c < t.n) {
                            const size_t o = size_t(t.out0 + c) * a.N + t.m0 + r;
                            const uint32_t y0 = __float_as_uint(g[i][j]), y1 = __float_as_uint(v[i][j]);
                            uint16_t* y = static_cast<uint16_t*>(a.out) + o;
                            if (t.m0 + r < a.N) {
                                y[0] = uint16_t(y0 >> 16);
                                a.out_aux[o] = uint8_t(y0 >> 8);
                            }
                            if (t.m0 + 128 + r < a.N) {
                                y[128] = uint16_t(y1 >> 16);
                                a.out_aux[o + 128] = uint8_t(y1 >> 8);
                            }
                        }
                    }
            } else {
#pragma unroll
                for (int i = 0; i < CH; ++i)
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int c = (2 * i + h) * 16 + j;
                        if (i < nc && c < t.n) {
                            const float y0 = g[i][j], y1 = v[i][j];
                            const size_t o = size_t(t.out0 + c) * a.N + t.m0 + r;
                            const bool r0 = t.m0 + r < a.N, r1 = t.m0 + 128 + r < a.N;
                            if (a.out_f32) {
                                float* y = static_cast<float*>(a.out) + o;
                                if (r0) y[0] = y0;
                                if (r1) y[128] = y1;
                            } else {
                                __nv_bfloat16* y = static_cast<__nv_bfloat16*>(a.out) + o;
                                if (r0) y[0] = __float2bfloat16_rn(y0);
                                if (r1) y[128] = __float2bfloat16_rn(y1);
                            }
                        }
                    }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, C::kTmemCols);
    }
    if (threadIdx.x == 0 && *abort_flag) atomicOr(a.err, 1);
}

// Four lanes' rows of four 16-byte chunks, transposed: lane l (of four) gets
// chunk l of each of the four rows, c[j] from row j.
__device__ __forceinline__ void transpose4(uint4 (&c)[4]) {
    const int l = threadIdx.x & 3;
    uint32_t(&w)[16] = *reinterpret_cast<uint32_t(*)[16]>(&c[0]);
    // two butterfly steps: exchange chunk bit b with lane bit b
#pragma unroll
    for (int b = 1; b <= 2; b <<= 1) {
        const bool hi = l & b;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j & b) continue;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t& lo_w = w[4 * j + k];
                uint32_t& hi_w = w[4 * (j + b) + k];
                const uint32_t got = __shfl_xor_sync(~0u, hi ? lo_w : hi_w, b);
                if (hi) lo_w = got;
                else hi_w = got;
            }
        }
    }
}

// Bits of the largest finite magnitude of the first n of 32 values.
__device__ __forceinline__ uint32_t row_top(const float* v, int n) {
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < 32; ++j) m = fmaxf(m, fabsf(v[j]));  // passes over NaN
    uint32_t top = __float_as_uint(m);
    if (top >= 0x7f800000u || n < 32) {  // Inf, or columns past the last
        top = 0;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            const uint32_t b = __float_as_uint(v[j]) & 0x7fffffffu;
            if (j < n && b < 0x7f800000u) top = max(top, b);
        }
    }
    return top;
}

// A warp's 32 x 32 block of outputs: lane l holds position row + l (of which n
// exist), columns [col, col + 32). Rows that start on a 16-byte boundary leave
// as 64-byte runs of four lanes, so that a store instruction touches 8 rows and
// not 32 (which bounded the epilogue); others value by value (N = 12287 instead of
// 12288: 752 us against 289 on 4096 x 6144, bf16).
template <bool AUX>
__device__ __forceinline__ void store32(const Fp8Args& a, long long row, int n, int col,
                                        const float* v) {
    const int lane = threadIdx.x & 31, size = a.out_f32 ? 4 : 2;
    uint8_t* base = static_cast<uint8_t*>(a.out) + (row * a.N + col) * size;
    const bool whole = col + 32 <= a.N && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0 &&
                       (a.N * size) % 16 == 0;
    if (whole) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            if (half && !a.out_f32) break;
            uint4 c[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (a.out_f32) {
                    const float* f = v + half * 16 + 4 * j;
                    c[j] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]),
                                      __float_as_uint(f[2]), __float_as_uint(f[3]));
                } else {
                    uint32_t w[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float lo = v[8 * j + 2 * k], hi = v[8 * j + 2 * k + 1];
                        if constexpr (AUX) {
                            const __half2 b = __floats2half2_rn(lo, hi);
                            w[k] = *reinterpret_cast<const uint32_t*>(&b);
                        } else {
                            const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
                            w[k] = *reinterpret_cast<const uint32_t*>(&b);
                        }
                    }
                    c[j] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            transpose4(c);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = (lane & ~3) + j;
                if (r < n)
                    *reinterpret_cast<uint4*>(base + (long long)r * a.N * size + half * 64 +
                                              (lane & 3) * 16) = c[j];
            }
        }
    } else if (lane < n) {
        base += (long long)lane * a.N * size;
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (col + j < a.N) {
                if (a.out_f32) reinterpret_cast<float*>(base)[j] = v[j];
                else if constexpr (AUX) reinterpret_cast<__half*>(base)[j] = __float2half_rn(v[j]);
                else reinterpret_cast<__nv_bfloat16*>(base)[j] = __float2bfloat16_rn(v[j]);
            }
    }
}

// ------------------------------------------------------------------ long segments
// A pair of CTAs (cta_group::2): M = 256 positions, 128 per CTA, N = 256 weight
// rows (128 gate and 128 up rows, or 256 output columns), of which each CTA
// loads 128. One CTA that loads 256 weight rows for its 128 positions needs 94
// bytes per clock and SM from L2 at the MMA's rate, more than L2 gives; the
// pair needs 63.
//
// An accumulator lane is one position, so a thread needs two scales per block:
// its position's times that of either weight block. Warp 2 writes these products
// to a ring in shared memory, eight blocks of K at a time.
//
// 4096 x 12288 x 6144: 290 us in a burst (2.1 PFLOP/s; the same product with whole-
// tensor scales, from the library, runs at 2.6 to 3.0), 338 in a long stream, under
// the power cap. In a burst a block of K takes about twice the 515 clocks of its
// MMAs (the chain below); on short K the output rows count (K = 2048: 119 us, 96
// without them).
//
// The MMA's N is cut in two halves of 128 (64 rows of either weight block: that
// is what N = 128 takes from each CTA's shared memory). Each half has two
// buffers, an issuing warp and four accumulation warps (64 columns of both weight
// blocks a thread) of its own. The chain MMA -> commit -> read-back -> release ->
// MMA of one buffer costs about 1000 clocks, half of them barrier latencies (a
// commit 200, a cluster arrive 120, a wait 50 each); two independent halves overlap
// their chains.
//
// Warps: 0 TMA producer, 1 and 3 MMA issuers of the halves (leader CTA; 1 owns
// TMEM), 2 scales, 4-11 accumulation, with the registers that the first four give
// up: 4 * 32 * 56 + 8 * 32 * 224 of the launch's 384 * 168.
constexpr int kPairThreads = 384;
constexpr int kPairWarps = 8;
constexpr int kPairStages = 6;
constexpr int kPairStage = 2 * kABytes;  // 128 positions, 128 weight rows
constexpr int kPairBar = 256;
constexpr int kPairBox = 64;             // position rows of one TMA box
constexpr int kPairGroup = 8;            // blocks of K per scale slot
constexpr int kPairSlots = 2;
constexpr int kPairScale = kPairGroup * 2 * 128 * 4;  // bytes of a slot
inline int pair_smem(int G) {
    return 1024 + kPairStages * kPairStage + kPairBar + kPairSlots * kPairScale + 2 * 128 * 4 +
           2 * (G + 1) * 4;
}

template <bool GLU, bool AUX, bool HOOK>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    k_fp8_pair(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
               const Fp8Args a) {
    constexpr int S = kPairStages;
    extern __shared__ __align__(1024) uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) &
                                               ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S * kPairStage);
    uint64_t* done = full + S;        // [half][stage] MMAs: sums ready, operands read
    uint64_t* tempty = done + 2 * S;  // [half][buffer]
    uint64_t* sfull = tempty + 4;
    uint64_t* sempty = sfull + kPairSlots;
    uint64_t* final_bar = sempty + kPairSlots;
    uint64_t* stall_bar = final_bar + 1;  // never signalled (test hook)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(stall_bar + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    static_assert((3 * S + 4 + 2 * kPairSlots + 2) * 8 + 8 <= kPairBar, "barriers");
    float* sc = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(full) + kPairBar);
    uint32_t* red = reinterpret_cast<uint32_t*>(sc + kPairSlots * kPairScale / 4);
    int* off = reinterpret_cast<int*>(red + 2 * 128);
    int* pref = off + a.G + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = int(cluster_rank());
    const int KB = (a.K + kFp8Block - 1) / kFp8Block;
    const int MB = GLU ? (a.N + 127) / 128 : (a.N + 255) / 256;
    const int first = int(blockIdx.x >> 1), step = int(gridDim.x >> 1);

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&done[s], 1);
            mbar_init(&done[S + s], 1);
        }
        for (int b = 0; b < 4; ++b) mbar_init(&tempty[b], kPairWarps);  // both CTAs' of a half
        for (int b = 0; b < kPairSlots; ++b) {
            mbar_init(&sfull[b], 1);
            mbar_init(&sempty[b], kPairWarps);
        }
        mbar_init(final_bar, 2);
        mbar_init(stall_bar, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, 512);
        tmem_relinquish_pair();
    }
    griddep_wait();  // the rows, the offsets, the workspace's earlier users
    if (a.clear_err && blockIdx.x == 0 && threadIdx.x == 0) *a.err = 0;
    load_plan<256>(a, MB, off, pref);
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // the peer's barriers exist before any remote arrive
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int total = pref[a.G] * (GLU ? 1 : a.nsplit);
    griddep_launch_dependents();
    // No barrier that the peer arrives on hands over data in ordinary memory (TMA
    // and the MMAs write and read shared memory, tcgen05 fences order the tensor
    // memory), so every wait orders this CTA's accesses only.
    const auto wait = [&](uint32_t bar, uint32_t parity) {
        return mbar_wait_for(bar, parity, abort_flag, HOOK ? a.wait_ns : kWaitNs);
    };
    const uint32_t full_at = smem_u32(full), done_at = smem_u32(done);

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0) {
            // ------------------------------------------------------ TMA producer
            tma_prefetch_desc(&tmA);
            tma_prefetch_desc(&tmB);
            uint32_t s = 0, ph = 1, issued = 0;
            const uint32_t stall =
                HOOK && (a.stall > 0 || (a.stall < 0 && rank)) ? uint32_t(abs(a.stall)) - 1 : ~0u;
            bool ok = true;
            for (int u = first; u < total && ok; u += step) {
                Tile t;
                decode<GLU, 256>(a, off, pref, KB, u, t);
                const int n0 = min(t.n, 128), n1 = t.n - n0;
                const int nb0 = (n0 + kPairBox - 1) / kPairBox, nb1 = (n1 + kPairBox - 1) / kPairBox;
                const int nb = rank ? nb1 : nb0, row = t.row0 + rank * 128;
                const int wrow = rank ? t.a1 : t.a0;
                const uint32_t bytes = 2 * kABytes + (nb0 + nb1) * kPairBox * 128;
                for (int kb = t.kb0; kb < t.kb1; ++kb, ++issued) {
                    if (!wait(done_at + s * 8, ph) || !wait(done_at + (S + s) * 8, ph) ||
                        (HOOK && issued == stall && !wait(smem_u32(stall_bar), 0))) {
                        ok = false;
                        break;
                    }
                    if (elect_one()) {
                        uint8_t* at = smem + s * kPairStage;
                        const uint32_t fb = cluster_addr(&full[s], 0);
                        if (rank == 0) mbar_arrive_expect_tx(&full[s], bytes);
                        for (int j = 0; j < nb; ++j)
                            tma_load_2d_pair(at + j * kPairBox * 128, &tmB, fb, kb * 128,
                                             row + j * kPairBox);
                        tma_load_2d_pair(at + kABytes, &tmA, fb, kb * 128, wrow);
                    }
                    __syncwarp();
                    if (++s == S) {
                        s = 0;
                        ph ^= 1;
                    }
                }
            }
            if (!ok) {  // every issued load lands before the pair leaves
                // (both CTAs' loads count on the leader's barriers: the other waits its time)
                const uint64_t dl = globaltimer() + kDrainNs;
                const uint32_t from = issued > uint32_t(S) ? issued - S : 0;
                if (rank == 0)
                    for (uint32_t i = from; i < issued; ++i) drain_wait(&full[i % S], (i / S) & 1, dl);
                else
                    while (globaltimer() < dl) {}
            }
        } else if (warp != 2) {
            // ------------------------------------------------------ MMA issuers
            if (rank == 0) {
                const int hf = warp >> 1;  // warp 1: half 0, warp 3: half 1
                const uint32_t idesc = idesc_e4m3_m256(128);
                const uint64_t ad = desc_k_sw128(smem_u32(smem));
                const uint64_t bd = desc_k_sw128(smem_u32(smem) + kABytes + hf * (kABytes / 2));
                const uint32_t te_at = smem_u32(tempty + hf * 2);
                uint32_t s = 0, ph = 0, b = 0, bph = 1;
                bool ok = true;
                for (int u = first; u < total && ok; u += step) {
                    const int k0 = GLU ? 0 : u % a.nsplit * a.kbper;
                    const int nk = GLU ? KB : min(KB - k0, a.kbper);
                    for (int kb = 0; kb < nk; ++kb) {
                        if (!wait(full_at + s * 8, ph) || !wait(te_at + b * 8, bph)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        if (elect_one()) {
                            const uint32_t d = tmem_base + b * 256 + hf * 128;
                            const uint32_t o = s * (kPairStage >> 4);
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk)
                                mma_f8_pair(d, ad + o + 2 * kk, bd + o + 2 * kk, idesc, kk != 0);
                            mma_commit_both(&done[hf * S + s]);
                        }
                        __syncwarp();
                        if (++s == S) {
                            s = 0;
                            ph ^= 1;
                        }
                        bph ^= b;
                        b ^= 1;
                    }
                }
                if (elect_one()) mma_commit_pair(smem_u32(final_bar));  // every MMA above is done
                __syncwarp();
                drain_wait(final_bar, 0, globaltimer() + kDrainNs);
            }
        } else if (warp == 2) {
            // ------------------------------------------------------ scales
            const bool vec = KB % 4 == 0 && (GLU || a.kbper % 4 == 0) &&
                             (reinterpret_cast<uintptr_t>(a.sx) & 15) == 0;
            uint32_t is = 0;
            bool ok = true;
            for (int u = first; u < total && ok; u += step) {
                Tile t;
                decode<GLU, 256>(a, off, pref, KB, u, t);
                const int n = min(128, t.n - rank * 128);
                for (int k0 = t.kb0; k0 < t.kb1; k0 += kPairGroup, ++is) {
                    const uint32_t q = is % kPairSlots;
                    float* o = sc + q * (kPairScale / 4) + lane;
#pragma unroll 1
                    for (int part = 0; part < kPairGroup; part += 4) {
                        const int kb = k0 + part;
                        float4 x[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int r = j * 32 + lane;
                            x[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            if (r < n && kb < KB) {
                                const float* p = a.sx + size_t(t.row0 + rank * 128 + r) * KB + kb;
                                if (vec) {
                                    x[j] = *reinterpret_cast<const float4*>(p);
                                } else {
                                    x[j].x = p[0];
                                    if (kb + 1 < KB) x[j].y = p[1];
                                    if (kb + 2 < KB) x[j].z = p[2];
                                    if (kb + 3 < KB) x[j].w = p[3];
                                }
                            }
                        }
                        if (part == 0 &&
                            !wait(smem_u32(&sempty[q]), ((is / kPairSlots) & 1) ^ 1)) {
                            ok = false;
                            break;
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool in = kb + e < KB;
                            const float w0 = in ? t.s0[kb + e] : 0.0f;
                            const float w1 = in ? t.s1[kb + e] : 0.0f;
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const float v = e == 0 ? x[j].x : e == 1 ? x[j].y : e == 2 ? x[j].z : x[j].w;
                                o[e * 256 + j * 32] = v * w0;
                                o[e * 256 + 128 + j * 32] = v * w1;
                            }
                        }
                        o += 4 * 256;
                    }
                    if (!ok) break;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sfull[q]);
                }
            }
        }
    } else {
        // ---------------------------------------------------------- accumulation
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int q = warp & 3, h = (warp - 4) >> 2;
        const int r = q * 32 + lane;
        // half h: columns [0, 64) are block 0's, [64, 128) block 1's
        const uint32_t lanes = tmem_base + (uint32_t(q * 32) << 16) + h * 128;
        const uint32_t te_at = cluster_addr(&tempty[h * 2], 0);  // the leader's
        const uint32_t ready_at = done_at + h * S * 8;
        const uint32_t sf_at = smem_u32(sfull);
        // ring positions: stage and its phase, buffer, scale slot and its phase
        uint32_t s = 0, ph = 0, b = 0, sl = 0, sph = 0;
        bool ok = true;
        for (int u = first; u < total; u += step) {
            Tile t;
            decode<GLU, 256>(a, off, pref, KB, u, t);
            const int n = t.n - rank * 128;  // this CTA's positions
            const bool work = q * 32 < n, rv = r < n;
            // columns [64 h, 64 h + 64) of either block
            float acc[2][64];
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int j = 0; j < 64; ++j) acc[c][j] = 0.0f;
            const auto release = [&] {  // the buffer goes back
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_remote_cta(te_at + b * 8);
                b ^= 1;
                if (++s == S) {
                    s = 0;
                    ph ^= 1;
                }
            };
            for (int k0 = t.kb0; k0 < t.kb1 && ok; k0 += kPairGroup) {
                if (!wait(sf_at + sl * 8, sph)) {
                    ok = false;
                    break;
                }
                const float* ps = sc + sl * (kPairScale / 4) + r;
                const int ng = min(kPairGroup, t.kb1 - k0);
                if (work) {
#pragma unroll 1
                    for (int e = 0; e < ng; ++e, ps += 256) {
                        const float s0 = ps[0], s1 = ps[128];
                        if (!wait(ready_at + s * 8, ph)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint32_t ta = lanes + b * 256;
                        uint32_t d[2][16];
                        tmem_ld16(ta, d[0]);
                        tmem_ld_wait_reg16(d[0]);
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            if (c < 7) tmem_ld16(ta + (c + 1) * 16, d[(c + 1) & 1]);
                            else release();  // all read: the last multiply-adds can follow
                            float(&y)[64] = acc[c >> 2];
#pragma unroll
                            for (int j = 0; j < 16; ++j)
                                y[(c & 3) * 16 + j] = fmaf(__uint_as_float(d[c & 1][j]),
                                                           c < 4 ? s0 : s1, y[(c & 3) * 16 + j]);
                            if (c < 7) tmem_ld_wait_reg16(d[(c + 1) & 1]);
                        }
                    }
                } else {  // no position of this warp: it keeps step only
#pragma unroll 1
                    for (int e = 0; e < ng && ok; ++e) {
                        ok = wait(ready_at + s * 8, ph);
                        if (ok) release();
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sempty[sl]);
                sph ^= sl;
                sl ^= 1;
            }
            if (!ok) {  // NaN for this tile and the rest (and the barriers below, where the
                        // other half's warp may wait, are met)
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int j = 0; j < 64; ++j) acc[c][j] = __uint_as_float(0x7fffffffu);
            }
            const size_t row = size_t(t.row0 + rank * 128 + r);
            if constexpr (GLU) {
                // silu(g) * u of this thread's 64 columns; the other 64 of the block are
                // the other half's warp's
                const int left = a.N - t.m0 - h * 64;  // columns before the end
                uint32_t top = 0;
#pragma unroll
                for (int j = 0; j < 64; ++j) {
                    const float m = j < left ? swiglu_fast(acc[0][j], acc[1][j]) : 0.0f;
                    top = max(top, __float_as_uint(m) & 0x7fffffffu);
                    acc[0][j] = m;
                }
                red[h * 128 + r] = top;
                named_bar_sync(1 + q, 64);
                const uint32_t both = max(red[r], red[128 + r]);
                named_bar_sync(1 + q, 64);  // both have read before the next tile writes
                float inv;
                const float s = block_scale(__uint_as_float(both), inv);
                if (rv && h == 0) a.mid_s[row * ((a.N + 127) / 128) + t.m0 / 128] = s;
                uint4 o[4];
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float* m = &acc[0][v * 16 + e * 4];
                        w[e] = pack4_e4m3(m[0] * inv, m[1] * inv, m[2] * inv, m[3] * inv);
                    }
                    o[v] = make_uint4(w[0], w[1], w[2], w[3]);
                }
                transpose4(o);  // 64-byte runs of four lanes, as in store32
                const int col = (lane & 3) * 16, r0 = r & ~3;
                uint8_t* y = a.mid_q + (row - r + r0) * a.N + t.m0 + h * 64 + col;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (r0 + j < n && col < left) *reinterpret_cast<uint4*>(y + size_t(j) * a.N) = o[j];
            } else if (work) {
                const long long p = t.out0 + rank * 128 + q * 32;
                if constexpr (AUX) {
                    const int yb = (a.N + kYBlock - 1) / kYBlock;
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int col = t.m0 + c * 128 + h * 64;
                        uint32_t e[2];
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            float* y = &acc[c][k * 32];
                            e[k] = y_exponent(row_top(y, a.N - col - k * 32));
                            const float inv = y_inverse(e[k]);
#pragma unroll
                            for (int j = 0; j < 32; ++j) y[j] *= inv;
                        }
                        // two together (a byte each touched as many sectors again: 670 us
                        // instead of 636)
                        uint8_t* ye = a.out_aux + size_t(p + lane) * yb + col / kYBlock;
                        if (rv && yb % 2 == 0 && col < a.N) {  // col / kYBlock is even
                            *reinterpret_cast<uint16_t*>(ye) = uint16_t(e[0] | e[1] << 8);
                        } else if (rv) {
                            if (col < a.N) ye[0] = uint8_t(e[0]);
                            if (col + 32 < a.N) ye[1] = uint8_t(e[1]);
                        }
                    }
                }
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    store32<AUX>(a, p, n - q * 32, t.m0 + (c >> 1) * 128 + h * 64 + (c & 1) * 32,
                                 &acc[c >> 1][(c & 1) * 32]);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // no remote arrive or TMEM write targets a finished CTA
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 512);
    }
    if (threadIdx.x == 0 && *abort_flag) atomicOr(a.err, 1);
}

// CTAs of a pair kernel that can be resident at once (an SM without a partner
// in its GPC cannot host a pair), per kernel and device.
int pair_grid(const void* kern, int smem, int dev) {
    static std::mutex mu;
    static std::map<std::pair<const void*, int>, int> cache;
    std::lock_guard<std::mutex> lk(mu);
    int& grid = cache[{kern, dev}];
    if (grid == 0) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(unsigned(num_sms(dev) & ~1));
        cfg.blockDim = dim3(kPairThreads);
        cfg.dynamicSmemBytes = size_t(smem);
        int clusters = 0;
        if (cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg) != cudaSuccess || clusters <= 0) {
            cudaGetLastError();
            clusters = num_sms(dev) / 2;
        }
        grid = std::min(2 * clusters, num_sms(dev) & ~1);
    }
    return grid;
}

template <bool GLU, bool AUX, bool HOOK>
hf_status launch_pair(const Fp8Args& a, cudaStream_t st) {
    int dev = 0;
    HF_CUDA(cudaGetDevice(&dev));
    const auto kern = k_fp8_pair<GLU, AUX, HOOK>;
    const void* kp = reinterpret_cast<const void*>(kern);
    const int smem = pair_smem(a.G);
    HF_CUDA(ensure_smem(kp, pair_smem(kMaxExperts)));
    CUtensorMap A, B;
    HF_TRY(make_map_u8(&A, a.w, a.K, a.a_rows, a.K, 128));
    HF_TRY(make_map_u8(&B, a.xq, a.K, a.rows, a.K, kPairBox));
    HF_CUDA(launch_pdl(kern, dim3(unsigned(pair_grid(kp, pair_smem(kMaxExperts), dev))),
                       dim3(kPairThreads), size_t(smem), st, A, B, a));
    return HF_OK;
}

template <bool GLU, int BN, bool AUX, bool HOOK>
hf_status launch_one(const Fp8Args& a, cudaStream_t st) {
    using C = Cfg<BN>;
    int dev = 0;
    HF_CUDA(cudaGetDevice(&dev));
    const auto kern = k_fp8_mma<GLU, BN, AUX, HOOK>;
    const int smem = C::smem(a.G);
    HF_CUDA(ensure_smem(reinterpret_cast<const void*>(kern), smem));
    CUtensorMap A, B;
    HF_TRY(make_map_u8(&A, a.w, a.K, a.a_rows, a.K, 128));
    HF_TRY(make_map_u8(&B, a.xq, a.K, a.rows, a.K, C::kBoxB));
    HF_CUDA(launch_pdl(kern, dim3(unsigned(num_sms(dev))), dim3(kThreads), size_t(smem), st, A, B, a));
    return HF_OK;
}

}  // namespace

// The runs of K of a product: with few tiles for the GPU's places (148 CTAs, or
// 74 pairs), each tile's blocks of K are dealt to several CTAs that write fp32
// planes, which the next launch adds in order. The number with the least modelled
// time, in us: rounds x (blocks x their time + 0.35 for a tile's end), and for the
// planes 3 (a launch) + 0.1 each + their bytes, written and read once. A block takes
// 0.7 where the weights stream from memory to every place; where some are idle less,
// down to what one CTA can load (tiles of 32 positions 0.45, of 64 0.55; a pair's
// MMAs take 0.7). Measured, cold, one run / the chosen number: 64 x 6144 x 12288
// 65.6 / 31, 1 x 2048 x 6144 26.7 / 14.4, 64 x 24576 x 1536 20.5 (two runs: 28.7),
// 128 x 6144 x 12288 (pairs) 55 / 35, 512 x 6144 x 6144 34.8 (two runs: 45).
Fp8Split fp8_split(long long tiles, int bn, int K, double plane_bytes) {
    const int KB = (K + kFp8Block - 1) / kFp8Block;
    const bool pair = bn == 256;
    const int slots = pair ? 74 : 148, mult = pair ? 4 : 1;
    const double least_block = pair ? 0.7 : bn == 64 ? 0.55 : 0.45;
    const double plane_us = plane_bytes * 2.0 / (pair ? 5e6 : 2.5e6);  // TB/s: 5, by columns 2.5
    Fp8Split best{1, KB};
    double least = 1e30;
    for (int n = 1; n <= 16 && n <= KB; ++n) {
        const int per = ((KB + n - 1) / n + mult - 1) / mult * mult;
        if ((KB + per - 1) / per != n) continue;  // no empty run
        const long long rounds = tiles * n / slots, rest = tiles * n % slots;
        double cost = rounds * (per * 0.7 + 0.35) + (n == 1 ? 0.0 : 3.0 + n * (0.1 + plane_us));
        if (rest) cost += per * std::max(least_block, 0.7 * rest / slots) + 0.35;
        if (cost < least) {
            least = cost;
            best = Fp8Split{n, per};
        }
    }
    return best;
}

int fp8_tile_rows(int mean) { return mean > kNarrowRows ? 256 : mean > kNarrow32 ? 64 : 32; }

Fp8Split fp8_gemm_split(int T, int N, int K) {
    const int bn = fp8_tile_rows(T);
    return fp8_split((long long)((N + 255) / 256) * ((T + bn - 1) / bn), bn, K, 4.0 * T * N);
}

__global__ void __launch_bounds__(256) k_sum_planes(const float* planes, int n, long long count,
                                                    void* out, int out_f32) {
    griddep_wait();
    griddep_launch_dependents();  // the next launch sets itself up meanwhile
    const long long quads = count / 4, rest = count - quads * 4;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i < quads) {
        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int s = 0; s < n; ++s) {
            const float* p = planes + s * count + i * 4;
            float4 v;
            if (count % 4 == 0) {
                v = *reinterpret_cast<const float4*>(p);
            } else {
                v = make_float4(p[0], p[1], p[2], p[3]);
            }
            y.x += v.x; y.y += v.y; y.z += v.z; y.w += v.w;
        }
        const bool vec = (reinterpret_cast<uintptr_t>(out) & 15) == 0;
        const float r[4] = {y.x, y.y, y.z, y.w};
        if (out_f32) {
            float* o = static_cast<float*>(out) + i * 4;
            if (vec) *reinterpret_cast<float4*>(o) = y;
            else
                for (int e = 0; e < 4; ++e) o[e] = r[e];
        } else {
            __nv_bfloat16* o = static_cast<__nv_bfloat16*>(out) + i * 4;
            if (vec) {
                const __nv_bfloat162 a = __floats2bfloat162_rn(y.x, y.y);
                const __nv_bfloat162 b = __floats2bfloat162_rn(y.z, y.w);
                *reinterpret_cast<uint2*>(o) = make_uint2(*reinterpret_cast<const uint32_t*>(&a),
                                                          *reinterpret_cast<const uint32_t*>(&b));
            } else {
                for (int e = 0; e < 4; ++e) o[e] = __float2bfloat16_rn(r[e]);
            }
        }
    } else if (i < quads + rest) {
        const long long c = quads * 4 + (i - quads);
        float y = 0.0f;
        for (int s = 0; s < n; ++s) y += planes[s * count + c];
        if (out_f32) static_cast<float*>(out)[c] = y;
        else static_cast<__nv_bfloat16*>(out)[c] = __float2bfloat16_rn(y);
    }
}

hf_status launch_fp8_gemm(const Fp8Args& args, float* planes, cudaStream_t st) {
    Fp8Args a = args;
    const Fp8Split sp = fp8_gemm_split(a.rows, a.N, a.K);
    a.nsplit = sp.n;
    a.kbper = sp.per;
    if (sp.n > 1) {
        a.out = planes;
        a.out_f32 = 1;
    }
    HF_TRY(launch_fp8_product(a, false, st));
    if (sp.n > 1) {
        const long long count = (long long)a.rows * a.N, n = count / 4 + count % 4;
        HF_CUDA(launch_pdl(k_sum_planes, dim3(unsigned((n + 255) / 256)), dim3(256), 0, st,
                           static_cast<const float*>(planes), sp.n, count, args.out,
                           args.out_f32));
    }
    return HF_OK;
}

template <bool GLU, bool AUX, bool HOOK>
hf_status launch_tiles(const Fp8Args& a, cudaStream_t st) {
    const int bn = fp8_tile_rows((a.rows + a.G - 1) / a.G);
    if (bn == 256) return launch_pair<GLU, AUX, HOOK>(a, st);
    if (bn == 64) return launch_one<GLU, 64, AUX, HOOK>(a, st);
    return launch_one<GLU, 32, AUX, HOOK>(a, st);
}

template <bool HOOK>
hf_status launch_form(const Fp8Args& a, bool glu, cudaStream_t st) {
    if (glu) return launch_tiles<true, false, HOOK>(a, st);
    return a.out_aux ? launch_tiles<false, true, HOOK>(a, st) : launch_tiles<false, false, HOOK>(a, st);
}

namespace {
std::atomic<unsigned long long> g_wait_ns{kWaitNs};
std::atomic<int> g_stall{0};
}  // namespace
void set_fp8_wait(unsigned long long ns) { g_wait_ns = ns ? std::min(ns, 1ull << 62) : kWaitNs; }
void set_fp8_stall(int block) { g_stall = block; }

hf_status launch_fp8_product(Fp8Args a, bool glu, cudaStream_t st) {
    a.wait_ns = g_wait_ns;
    a.stall = g_stall;
    return a.wait_ns != kWaitNs || a.stall ? launch_form<true>(a, glu, st)
                                           : launch_form<false>(a, glu, st);
}

}  // namespace hf
