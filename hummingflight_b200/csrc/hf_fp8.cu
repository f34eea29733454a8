// hf_fp8.cu -- FP8 operators: quantised rows, the block-scaled product and the
// routed SwiGLU experts (include/hf_fp8.h).
//
// A value is q * s: q in e4m3, s an fp32 scale per 128 columns of a row or per
// 128 x 128 block of a weight.
#include <algorithm>

#include "hf_fp8.cuh"

namespace hf {
namespace {

constexpr size_t kAlign = 256;
constexpr int kMaxK = 32;  // picks per token
size_t up(size_t v) { return (v + kAlign - 1) / kAlign * kAlign; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
int blocks128(int n) { return (n + kFp8Block - 1) / kFp8Block; }

// ------------------------------------------------------------------ quantise
// One pass bound by memory: 16 threads own a block of 128 columns, 8 columns
// (16 or 32 bytes) each, so the maximum is four shuffles and every load and store
// is whole sectors; a thread has kQuantBatch blocks' loads in flight.
// 16384 x 6144 bf16: 57 us, 5.3 TB/s of 6.5 measured.
struct QuantArgs {
    const void* x;
    long long ldx;
    int rows, K, nb;
    uint8_t* q;
    float* s;
    // experts: the row of slot perm[p]'s token goes to position p, pos[slot] = p
    const int32_t* perm;
    int k, n_tok;
    int32_t* pos;
    int* err;  // error word, cleared by the first block
};
constexpr int kQuantBatch = 4;

// 16 bytes that are read once. These kernels may start while the launch that writes
// what they read still runs, so the read-only path (.nc), which holds for memory that
// nobody writes while the kernel lives, is not theirs; nor may a load move ahead of
// griddep_wait.
__device__ __forceinline__ uint4 ld_once_u4(const void* p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "l"(p)
                 : "memory");
    return r;
}

// 8 columns as they lie in memory.
template <bool XF32>
struct Raw8 {
    uint4 v[XF32 ? 2 : 1];
    __device__ __forceinline__ void load(const void* x, long long i) {
        if constexpr (XF32) {
            const float* p = static_cast<const float*>(x) + i;
            v[0] = ld_once_u4(p);
            v[1] = ld_once_u4(p + 4);
        } else {
            v[0] = ld_once_u4(static_cast<const uint16_t*>(x) + i);
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < (XF32 ? 2 : 1); ++i) v[i] = make_uint4(0, 0, 0, 0);
    }
};

// A thread's 8 columns of a block: values and scale. The 16 threads of `half`
// call it together. Magnitudes order as their bits (NaN above Inf), bf16 ones two
// to a register.
__device__ __forceinline__ uint2 scaled8(const float (&f)[8], uint32_t m, float* scale) {
    float inv;
    *scale = block_scale(__uint_as_float(m), inv);
    return make_uint2(pack4_e4m3(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv),
                      pack4_e4m3(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
}
__device__ __forceinline__ uint2 quantize8(const float (&f)[8], unsigned half, float* scale) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(f[j]) & 0x7fffffffu);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(half, m, o));
    return scaled8(f, m, scale);
}
template <bool XF32>
__device__ __forceinline__ uint2 quantize8(const Raw8<XF32>& r, unsigned half, float* scale) {
    float f[8];
    if constexpr (XF32) {
        const uint4 a = r.v[0], b = r.v[1];
        const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(u[j]);
        return quantize8(f, half, scale);
    } else {
        const uint4 a = r.v[0];
        unpack8(a, f);
        uint32_t m = __vmaxu2(__vmaxu2(a.x & 0x7fff7fffu, a.y & 0x7fff7fffu),
                     __vmaxu2(a.z & 0x7fff7fffu, a.w & 0x7fff7fffu));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(half, m, o));
        m = max(m & 0xffff0000u, m << 16);
        return scaled8(f, m, scale);
    }
}

// Rows one behind the other and whole blocks: the blocks are one array.
template <bool XF32>
__global__ void __launch_bounds__(256) k_quantize_flat(const void* x, long long blocks, uint8_t* q,
                                                       float* s) {
    const int sub = threadIdx.x & 15;
    const unsigned half = 0xffffu << (threadIdx.x & 16);
    const long long step = (long long)gridDim.x * 16;
    for (long long i0 = (long long)blockIdx.x * 16 + (threadIdx.x >> 4); i0 < blocks;
         i0 += step * kQuantBatch) {
        Raw8<XF32> r[kQuantBatch];
#pragma unroll
        for (int u = 0; u < kQuantBatch; ++u)
            if (i0 + u * step < blocks) r[u].load(x, (i0 + u * step) * kFp8Block + sub * 8);
#pragma unroll
        for (int u = 0; u < kQuantBatch; ++u) {
            const long long i = i0 + u * step;
            if (i >= blocks) break;  // the 16 threads of a block agree
            float sc;
            reinterpret_cast<uint2*>(q)[i * 16 + sub] = quantize8(r[u], half, &sc);
            if (sub == 0) s[i] = sc;
        }
    }
}

// Any pitch, ragged last blocks, gathered rows.
template <bool XF32>
__global__ void __launch_bounds__(256) k_quantize(QuantArgs a) {
    griddep_wait();
    griddep_launch_dependents();  // behind the wait: see Fp8Args::early
    if (a.err && blockIdx.x == 0 && threadIdx.x == 0) *a.err = 0;
    const int sub = threadIdx.x & 15;
    const unsigned half = 0xffffu << (threadIdx.x & 16);
    const long long blocks = (long long)a.rows * a.nb, step = (long long)gridDim.x * 16;
    for (long long i = (long long)blockIdx.x * 16 + (threadIdx.x >> 4); i < blocks; i += step) {
        int p, b;
        if (blocks < 0x7fffffffll) {  // 32-bit division
            p = int(unsigned(i) / unsigned(a.nb));
            b = int(unsigned(i) - unsigned(p) * unsigned(a.nb));
        } else {
            p = int(i / a.nb);
            b = int(i - (long long)p * a.nb);
        }
        const int c = b * kFp8Block + sub * 8;
        int row = p;
        if (a.perm) {
            const int slot = a.perm[p];
            row = slot / a.k;
            if (slot < 0 || row >= a.n_tok) continue;  // the 16 threads agree
            if (c == 0) a.pos[slot] = p;
        }
        Raw8<XF32> r;
        if (c < a.K) r.load(a.x, row * a.ldx + c);
        else r.zero();
        float s;
        const uint2 q = quantize8(r, half, &s);
        if (c < a.K) *reinterpret_cast<uint2*>(a.q + size_t(p) * a.K + c) = q;
        if (sub == 0) a.s[size_t(p) * a.nb + b] = s;
    }
}

// pos[perm[p]] = p. A slot that perm does not name keeps what the workspace holds (a
// position of an earlier call, say), so pos is read through position_of only.
__global__ void __launch_bounds__(256) k_positions(const int32_t* perm, int n, int32_t* pos,
                                                   int* err) {
    const int p = blockIdx.x * 256 + threadIdx.x;
    if (p == 0) *err = 0;
    if (p >= n) return;
    const int slot = perm[p];
    if (slot >= 0 && slot < n) pos[slot] = p;
}

// The position that perm gives a slot, or ~0. n: positions.
__device__ __forceinline__ unsigned position_of(const int32_t* pos, const int32_t* perm, unsigned n,
                                                unsigned slot) {
    const unsigned p = unsigned(pos[slot]);
    return p < n && unsigned(perm[p]) == slot ? p : ~0u;
}

// Token-major gather of large batches: a block of a token's row is read and
// quantised once and written to the positions of its k slots (k times fewer reads
// than position by position).
template <bool XF32>
__global__ void __launch_bounds__(256) k_quantize_tokens(QuantArgs a) {
    const int sub = threadIdx.x & 15;
    const unsigned half = 0xffffu << (threadIdx.x & 16);
    const int t = blockIdx.x, n = a.n_tok * a.k;
    __shared__ int32_t at[kMaxK];
    if (int(threadIdx.x) < a.k)
        at[threadIdx.x] = int(position_of(a.pos, a.perm, unsigned(n), t * a.k + threadIdx.x));
    __syncthreads();
    for (int b0 = threadIdx.x >> 4; b0 < a.nb; b0 += 16 * kQuantBatch) {
        Raw8<XF32> r[kQuantBatch];
#pragma unroll
        for (int u = 0; u < kQuantBatch; ++u) {
            const int c = (b0 + u * 16) * kFp8Block + sub * 8;
            if (c < a.K) r[u].load(a.x, t * a.ldx + c);
            else r[u].zero();
        }
#pragma unroll
        for (int u = 0; u < kQuantBatch; ++u) {
            const int b = b0 + u * 16, c = b * kFp8Block + sub * 8;
            if (b >= a.nb) continue;
            float s;
            const uint2 q = quantize8(r[u], half, &s);
            for (int i = 0; i < a.k; ++i) {
                const int p = at[i];
                if (unsigned(p) >= unsigned(n)) continue;
                if (c < a.K) *reinterpret_cast<uint2*>(a.q + size_t(p) * a.K + c) = q;
                if (sub == 0) a.s[size_t(p) * a.nb + b] = s;
            }
        }
    }
}

// Positions from which the experts' gather goes by tokens. H = 6144, k = 8, us by
// positions and by tokens (two launches): 512 positions 4.8 and 6.6, 2048: 12.7
// and 7.9, 8192: 43.8 and 16.3, 32768: 161 and 45.
constexpr int kTokenMajor = 1024;

hf_status launch_quantize(const QuantArgs& a, bool f32, int dev, cudaStream_t st) {
    if (a.perm && a.rows >= kTokenMajor && a.k > 1) {
        k_positions<<<(a.rows + 255) / 256, 256, 0, st>>>(a.perm, a.rows, a.pos, a.err);
        HF_CUDA(cudaGetLastError());
        if (f32) k_quantize_tokens<true><<<a.n_tok, 256, 0, st>>>(a);
        else k_quantize_tokens<false><<<a.n_tok, 256, 0, st>>>(a);
        HF_CUDA(cudaGetLastError());
        return HF_OK;
    }
    const long long blocks = (long long)a.rows * a.nb;
    const long long most = num_sms(dev) * 8ll;
    // one array of blocks, or rows: 16384 x 6144 bf16 56 and 71 us, 1024 x 6144 4.4 and 5.6
    if (!a.perm && a.ldx == a.K && a.K % kFp8Block == 0) {
        const int grid = int(std::min((blocks + 15) / 16, most));
        if (f32) k_quantize_flat<true><<<grid, 256, 0, st>>>(a.x, blocks, a.q, a.s);
        else k_quantize_flat<false><<<grid, 256, 0, st>>>(a.x, blocks, a.q, a.s);
    } else {
        const int grid = int(std::min((blocks + 15) / 16, 2 * most));
        HF_CUDA(launch_pdl(f32 ? k_quantize<true> : k_quantize<false>, dim3(unsigned(grid)),
                           dim3(256), 0, st, a));
    }
    HF_CUDA(cudaGetLastError());
    return HF_OK;
}

// The intermediate of few positions, whose gate/up product ran in several runs of
// K: silu(g) * u of the summed planes [n x rows x 2 I] (gate columns, then up),
// quantised. 16 threads a block of 128 columns.
__global__ void __launch_bounds__(256) k_swiglu_planes(const float* planes, int n, int rows, int I,
                                                       int nb, uint8_t* q, float* s) {
    const int sub = threadIdx.x & 15;
    const unsigned half = 0xffffu << (threadIdx.x & 16);
    const int i = blockIdx.x * 16 + (threadIdx.x >> 4);
    griddep_wait();
    griddep_launch_dependents();  // behind the wait: see Fp8Args::early
    if (i >= rows * nb) return;  // the 16 threads of a block agree
    const int p = i / nb, b = i % nb, c = b * kFp8Block + sub * 8;
    float f[8] = {};
    if (c < I) {
        float g[8] = {}, u[8] = {};
#pragma unroll 4
        for (int r = 0; r < n; ++r) {
            const float4* v = reinterpret_cast<const float4*>(
                planes + (size_t(r) * rows + p) * 2 * I + c);
            const float4* w = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(v) + I);
            const float4 a0 = v[0], a1 = v[1], b0 = w[0], b1 = w[1];
            g[0] += a0.x; g[1] += a0.y; g[2] += a0.z; g[3] += a0.w;
            g[4] += a1.x; g[5] += a1.y; g[6] += a1.z; g[7] += a1.w;
            u[0] += b0.x; u[1] += b0.y; u[2] += b0.z; u[3] += b0.w;
            u[4] += b1.x; u[5] += b1.y; u[6] += b1.z; u[7] += b1.w;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = swiglu(g[j], u[j]);
    }
    float sc;
    const uint2 v = quantize8(f, half, &sc);
    if (c < I) *reinterpret_cast<uint2*>(q + size_t(p) * I + c) = v;
    if (sub == 0) s[size_t(p) * nb + b] = sc;
}

// ------------------------------------------------------------------ combine
// out[t] = resid[t] + sum_i w[t, i] y[pos(t, i)], rank order, fp32: the
// reference's separate multiply and add per pick.
__device__ __forceinline__ void unpack(const uint4 v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
}

// A thread takes 16 bytes of a token's columns, all of its picks' loads in flight
// before the first is used. T = 16384, k = 8, H = 6144: 369 us for bf16 outputs (5.0 TB/s),
// 602 for fp32 ones (6.0).
// Y: the expert outputs are fp32, in n planes (runs of K) that are added in order, or 24
// bits or FP16 (Fp8Args::out_aux). A slot without a position in the segments [offsets[0],
// offsets[E]) counts as 0: its y was not written.
enum class Y { f32, b24, f16 };
template <Y Form, bool F32, int kBatch>
__global__ void __launch_bounds__(256, kBatch == 2 ? 8 : 4)
    k_fp8_combine(const void* y, const uint8_t* aux, int n, const int32_t* pos,
                  const int32_t* perm, const int32_t* offsets, int E, const float* w, int T, int k,
                  int H, const void* resid, void* out) {
    constexpr bool Y32 = Form == Y::f32;
    constexpr int V = Y32 ? 4 : 8;
    const int t = blockIdx.x, c = (blockIdx.y * 256 + threadIdx.x) * V;
    // lane i: the position and weight of pick i (a slot that perm names is one it has
    // at that position; k_positions). They are older than the down product, which lets
    // this launch start behind its own wait (Fp8Args::early), and are read ahead of its end.
    const unsigned rows = unsigned(T) * unsigned(k);
    const int lane = threadIdx.x & 31, slot = t * k + lane;
    const unsigned p = lane < k ? unsigned(pos[slot]) : ~0u;
    const float wl = lane < k ? w[slot] : 0.0f;
    const int has = p < rows ? perm[p] : -1, first = offsets[0], end = offsets[E];
    const unsigned named = __ballot_sync(~0u, has == slot && int(p) >= first && int(p) < end);
    griddep_wait();
    griddep_launch_dependents();
    float acc[V] = {};
    for (int j0 = 0; j0 < k; j0 += kBatch) {
        uint4 v[kBatch];
        uint2 low[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const unsigned at = __shfl_sync(~0u, p, j0 + j);
            const bool in = ((named >> (j0 + j)) & 1u) && c < H;
            v[j] = in ? ld_once_u4(static_cast<const char*>(y) + (size_t(at) * H + c) * (Y32 ? 4 : 2))
                      : make_uint4(0, 0, 0, 0);
            low[j] = make_uint2(0, 0);
            if constexpr (Form == Y::b24)
                if (in) low[j] = *reinterpret_cast<const uint2*>(aux + size_t(at) * H + c);
            if constexpr (Form == Y::f16)
                if (in) low[j].x = aux[size_t(at) * ((H + kYBlock - 1) / kYBlock) + c / kYBlock];
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            if (j0 + j >= k) break;
            const float wj = __shfl_sync(~0u, wl, j0 + j);
            const unsigned at = __shfl_sync(~0u, p, j0 + j);
            if (!((named >> (j0 + j)) & 1u)) continue;
            float f[V];
            if constexpr (Form == Y::b24) {
                unpack24(v[j], low[j], f);
            } else if constexpr (Form == Y::f16) {
                unpack16(v[j], low[j].x, f);
            } else {
                unpack(v[j], f);
                for (int r = 1; r < n && c < H; ++r) {
                    float g[V];
                    unpack(ld_once_u4(static_cast<const float*>(y) +
                                    (size_t(r) * rows + at) * H + c), g);
#pragma unroll
                    for (int e = 0; e < V; ++e) f[e] += g[e];
                }
            }
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] = __fadd_rn(acc[e], __fmul_rn(wj, f[e]));
        }
    }
    if (c >= H) return;
    const size_t o = size_t(t) * H + c;
    if constexpr (F32) {
        static_assert(Y32, "fp32 outputs come from fp32 expert outputs");
        if (resid) {
            float f[V];
            unpack(*reinterpret_cast<const uint4*>(static_cast<const float*>(resid) + o), f);
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] = __fadd_rn(f[e], acc[e]);
        }
        *reinterpret_cast<float4*>(static_cast<float*>(out) + o) =
            make_float4(acc[0], acc[1], acc[2], acc[3]);
    } else {
        uint32_t b[V / 2];
        if (resid) {
#pragma unroll
            for (int e = 0; e < V / 2; ++e) {
                const uint32_t h = reinterpret_cast<const uint32_t*>(
                    static_cast<const uint16_t*>(resid) + o)[e];
                acc[2 * e] = __fadd_rn(bf16lo(h), acc[2 * e]);
                acc[2 * e + 1] = __fadd_rn(bf16hi(h), acc[2 * e + 1]);
            }
        }
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(acc[2 * e], acc[2 * e + 1]);
            b[e] = *reinterpret_cast<const uint32_t*>(&h);
        }
        uint16_t* d = static_cast<uint16_t*>(out) + o;
        if constexpr (V == 8) *reinterpret_cast<uint4*>(d) = make_uint4(b[0], b[1], b[2], b[3]);
        else *reinterpret_cast<uint2*>(d) = make_uint2(b[0], b[1]);
    }
}

template <Y Form, bool F32>
hf_status launch_fp8_combine(const void* y, const uint8_t* aux, int n, const int32_t* pos,
                             const int32_t* perm, const int32_t* offsets, int E, const float* w,
                             int T, int k, int H, const void* resid, void* out, cudaStream_t st) {
    constexpr int v = Form == Y::f32 ? 4 : 8;
    // one or two picks: two loads in flight a thread, 32 registers and not 60. The whole
    // call with one expert of 16384 rows, fp32 onto fp32, us: 1170, with eight 1467
    HF_CUDA(launch_pdl(k <= 2 ? k_fp8_combine<Form, F32, 2> : k_fp8_combine<Form, F32, 8>,
                       dim3(unsigned(T), unsigned((H / v + 255) / 256)), dim3(256), 0, st, y, aux, n,
                       pos, perm, offsets, E, w, T, k, H, resid, out));
    return HF_OK;
}

// ------------------------------------------------------------------ workspaces
// Runs of K of the experts' products: few positions make few tiles (at most one
// per position and row block of the weights). H = 6144, I = 2048, us without runs and
// with: 128 positions of 2 experts 68 and 39, 500 of 1: 57 and 50, 1000 of 1: 75 and
// 82; the planes' bytes grow with the positions and the tiles fill the GPU by then.
constexpr int kFewPositions = 512;

struct ExpertsWs {
    Fp8Split up, down;  // runs of the gate/up and down products
    bool few;           // the gate/up product writes planes, one for each run
    Y form;             // of the down product's rows
    size_t pos, xq, sx, gu, mq, ms, y, aux, total;
};

ExpertsWs experts_ws(int T, int k, int E, int H, int I, bool f32) {
    ExpertsWs w{};
    const size_t n = size_t(T) * k;
    w.up = Fp8Split{1, blocks128(H)};
    w.down = Fp8Split{1, blocks128(I)};
    if (n <= kFewPositions) {
        const int mean = int((n + E - 1) / E), bn = fp8_tile_rows(mean);
        const long long active = std::min<long long>(n, E) * ((mean + bn - 1) / bn);
        w.down = fp8_split(active * ((H + 255) / 256), bn, I, 4.0 * n * H);
        if (I % kFp8Block == 0) {  // gate and up rows then have one run of scale blocks
            w.up = fp8_split(active * (I / 128), bn, H, 8.0 * n * I);
            w.few = w.up.n > 1;
        }
    }
    size_t o = kAlign;  // the error word
    const auto take = [&](size_t bytes) {
        const size_t at = o;
        o += hf::up(bytes);
        return at;
    };
    w.pos = take(n * 4);
    w.xq = take(n * H);
    w.sx = take(n * blocks128(H) * 4);
    w.gu = take(w.few ? size_t(w.up.n) * n * 2 * I * 4 : 0);
    w.mq = take(n * I);
    w.ms = take(n * blocks128(I) * 4);
    w.form = f32 || w.down.n > 1 ? Y::f32 : fp8_pairs(int((n + E - 1) / E)) ? Y::f16 : Y::b24;
    w.y = take(size_t(w.down.n) * n * H * (w.form == Y::f32 ? 4 : 2));
    w.aux = take(w.form == Y::f32 ? 0 : w.form == Y::b24 ? n * H : n * ((H + kYBlock - 1) / kYBlock));
    w.total = o;
    return w;
}

bool bad_type(hf_dtype t) { return t != HF_BF16 && t != HF_F32; }

// x rows: 16-byte aligned pointer and pitch, rows of at least K elements
bool bad_rows(const void* x, hf_dtype t, long long ldx, int K) {
    return !aligned16(x) || ldx < K || ldx % (t == HF_F32 ? 4 : 8);
}

}  // namespace
}  // namespace hf

using namespace hf;

extern "C" {

hf_status hf_fp8_quantize(const void* x, hf_dtype x_dtype, long long ldx, int T, int K, uint8_t* q,
                          float* scales, hf_stream stream) {
    if (T < 0 || K <= 0 || K % 16 || std::max(T, K) > kMaxExtent)
        return fail(HF_ERR_ARG, "hf_fp8_quantize: T >= 0 and K a positive multiple of 16, both at "
                                "most 2^31 - 4096");
    if (bad_type(x_dtype)) return fail(HF_ERR_ARG, "hf_fp8_quantize: rows must be bf16 or f32");
    if (T == 0) return HF_OK;
    if (!x || !q || !scales) return fail(HF_ERR_ARG, "hf_fp8_quantize: null pointer");
    if (bad_rows(x, x_dtype, ldx, K))
        return fail(HF_ERR_ARG, "hf_fp8_quantize: x and its pitch must be 16-byte aligned, the "
                                "pitch at least K");
    if (!aligned16(q)) return fail(HF_ERR_ARG, "hf_fp8_quantize: q must be 16-byte aligned");
    int dev = 0;
    HF_CUDA(cudaGetDevice(&dev));
    QuantArgs a{};
    a.x = x;
    a.ldx = ldx;
    a.rows = T;
    a.K = K;
    a.nb = blocks128(K);
    a.q = q;
    a.s = scales;
    return launch_quantize(a, x_dtype == HF_F32, dev, as_cuda(stream));
}

size_t hf_fp8_gemm_workspace_size(int T, int N, int K) {
    if (T <= 0 || N <= 0 || K <= 0 || std::max({T, N, K}) > kMaxExtent) return 0;
    const Fp8Split sp = fp8_gemm_split(T, N, K);
    return kAlign + (sp.n > 1 ? up(size_t(sp.n) * T * N * sizeof(float)) : 0);
}

hf_status hf_fp8_gemm(const uint8_t* xq, const float* sx, const uint8_t* wq, const float* sw, int T,
                      int N, int K, void* out, hf_dtype out_dtype, void* workspace,
                      size_t workspace_bytes, hf_stream stream) {
    if (T < 0 || N <= 0 || K <= 0 || K % 16 || std::max({T, N, K}) > kMaxExtent)
        return fail(HF_ERR_ARG, "hf_fp8_gemm: T >= 0, N > 0 and K a positive multiple of 16, all "
                                "at most 2^31 - 4096");
    if (bad_type(out_dtype)) return fail(HF_ERR_ARG, "hf_fp8_gemm: out must be bf16 or f32");
    if (T == 0) return HF_OK;
    if (!xq || !sx || !wq || !sw || !out || !workspace)
        return fail(HF_ERR_ARG, "hf_fp8_gemm: null pointer");
    if (!aligned16(xq) || !aligned16(wq))
        return fail(HF_ERR_ARG, "hf_fp8_gemm: xq and wq must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(workspace) % kAlign)
        return fail(HF_ERR_ARG, "hf_fp8_gemm: workspace must be 256-byte aligned");
    if (workspace_bytes < hf_fp8_gemm_workspace_size(T, N, K))
        return fail(HF_ERR_ARG, "hf_fp8_gemm: workspace smaller than hf_fp8_gemm_workspace_size");
    Fp8Args a{};
    a.xq = xq;
    a.sx = sx;
    a.w = wq;
    a.a_rows = N;
    a.sw = sw;
    a.G = 1;
    a.rows = T;
    a.N = N;
    a.K = K;
    a.out = out;
    a.out_f32 = out_dtype == HF_F32;
    a.err = static_cast<int*>(workspace);
    a.clear_err = 1;
    return launch_fp8_gemm(a, reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kAlign),
                           as_cuda(stream));
}

size_t hf_fp8_moe_experts_workspace_size(int T, int top_k, int E, int H, int I,
                                         hf_dtype out_dtype) {
    if (T <= 0 || top_k <= 0 || top_k > kMaxK || E <= 0 || E > kMaxExperts || H <= 0 || I <= 0 ||
        (long long)T * top_k > kMaxExtent || 3ll * E * std::max(H, I) > kMaxExtent)
        return 0;
    return experts_ws(T, top_k, E, H, I, out_dtype == HF_F32).total;
}

hf_status hf_fp8_moe_experts(const uint8_t* experts, const float* scales, int E, int H, int I,
                             const void* x, hf_dtype x_dtype, long long ldx, int T, int top_k,
                             const hf_moe_routing* r, const void* resid, void* out,
                             hf_dtype out_dtype, void* workspace, size_t workspace_bytes,
                             hf_stream stream) {
    const auto refuse = [](const char* why) {
        return fail(HF_ERR_ARG, std::string("hf_fp8_moe_experts: ") + why);
    };
    if (E < 1 || E > kMaxExperts) return refuse("E must be in 1..1024");
    if (H <= 0 || I <= 0 || H % 16 || I % 16)
        return refuse("H and I must be positive multiples of 16");
    if (3ll * E * std::max(H, I) > kMaxExtent)
        return refuse("3 * E * max(H, I) must be at most 2^31 - 4096");
    if (top_k < 1 || top_k > kMaxK) return refuse("top_k must be in 1..32");
    if (T < 0 || (long long)T * top_k > kMaxExtent)
        return refuse("T >= 0 and T * top_k at most 2^31 - 4096");
    if (bad_type(x_dtype) || bad_type(out_dtype))
        return refuse("x and out must be bf16 or f32");
    if (T == 0) return HF_OK;
    if (!experts || !scales || !x || !out || !workspace || !r || !r->topk_weights || !r->offsets ||
        !r->perm)
        return refuse("null pointer");
    if (bad_rows(x, x_dtype, ldx, H))
        return refuse("x and its pitch must be 16-byte aligned, the pitch at least H");
    if (!aligned16(experts) || !aligned16(out) || (resid && !aligned16(resid)))
        return refuse("pointers must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(workspace) % kAlign)
        return refuse("workspace must be 256-byte aligned");
    const bool f32 = out_dtype == HF_F32;
    const ExpertsWs L = experts_ws(T, top_k, E, H, I, f32);
    if (workspace_bytes < L.total)
        return refuse("workspace smaller than hf_fp8_moe_experts_workspace_size");
    if (resid && resid != out) {
        const uintptr_t p = reinterpret_cast<uintptr_t>(resid), q = reinterpret_cast<uintptr_t>(out);
        const uintptr_t bytes = size_t(T) * H * (f32 ? 4 : 2);
        if (p < q + bytes && q < p + bytes)
            return refuse("resid and out overlap without being the same buffer");
    }
    int dev = 0;
    HF_CUDA(cudaGetDevice(&dev));
    const cudaStream_t st = as_cuda(stream);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const int n = T * top_k, hb = blocks128(H), ib = blocks128(I);

    QuantArgs qa{};
    qa.x = x;
    qa.ldx = ldx;
    qa.rows = n;
    qa.K = H;
    qa.nb = hb;
    qa.q = ws + L.xq;
    qa.s = reinterpret_cast<float*>(ws + L.sx);
    qa.perm = r->perm;
    qa.k = top_k;
    qa.n_tok = T;
    qa.pos = reinterpret_cast<int32_t*>(ws + L.pos);
    qa.err = reinterpret_cast<int*>(ws);
    HF_TRY(launch_quantize(qa, x_dtype == HF_F32, dev, st));

    // gate/up: an expert's block is 3 I rows of H; down: 3 H rows of I
    Fp8Args a{};
    a.xq = qa.q;
    a.sx = qa.s;
    a.w = experts;
    a.a_rows = 3ll * E * I;
    a.a_stride = 3 * I;
    a.sw = scales;
    a.sw_stride = 3ll * ib * hb;
    a.offsets = r->offsets;
    a.G = E;
    a.rows = n;
    a.K = H;
    a.nsplit = L.up.n;  // 1 unless few
    a.kbper = L.up.per;
    a.err = qa.err;
    a.early = 1;
    uint8_t* mq = ws + L.mq;
    float* ms = reinterpret_cast<float*>(ws + L.ms);
    if (L.few) {
        float* gu = reinterpret_cast<float*>(ws + L.gu);
        a.N = 2 * I;
        a.out = gu;
        a.out_f32 = 1;
        HF_TRY(launch_fp8_product(a, false, st));
        HF_CUDA(launch_pdl(k_swiglu_planes, dim3(unsigned((n * ib + 15) / 16)), dim3(256), 0, st,
                           static_cast<const float*>(gu), L.up.n, n, I, ib, mq, ms));
    } else {
        a.N = I;
        a.sw_up = (long long)ib * hb;
        a.mid_q = mq;
        a.mid_s = ms;
        HF_TRY(launch_fp8_product(a, true, st));
    }
    a.xq = mq;
    a.sx = ms;
    a.a_rows = 3ll * E * H;
    a.a_stride = 3 * H;
    a.a_base = 2 * H;
    a.sw = scales + 2ll * ib * hb;
    a.N = H;
    a.K = I;
    a.nsplit = L.down.n;
    a.kbper = L.down.per;
    a.out = ws + L.y;
    a.out_f32 = L.form == Y::f32;
    a.out_aux = a.out_f32 ? nullptr : ws + L.aux;
    HF_TRY(launch_fp8_product(a, false, st));
    const auto combine = f32                ? launch_fp8_combine<Y::f32, true>
                         : L.form == Y::f32 ? launch_fp8_combine<Y::f32, false>
                         : L.form == Y::b24 ? launch_fp8_combine<Y::b24, false>
                                            : launch_fp8_combine<Y::f16, false>;
    return combine(ws + L.y, ws + L.aux, L.down.n, qa.pos, r->perm, r->offsets, E, r->topk_weights,
                   T, top_k, H, resid, out, st);
}

hf_status hf_fp8_set_wait_timeout(uint64_t ns) {
    set_fp8_wait(ns);
    return HF_OK;
}

hf_status hf_fp8_debug_stall(int block) {
    if (block < -kMaxExtent) return fail(HF_ERR_ARG, "hf_fp8_debug_stall: block out of range");
    set_fp8_stall(block);
    return HF_OK;
}

hf_status hf_fp8_status(const void* workspace, hf_stream stream) {
    if (!workspace) return fail(HF_ERR_ARG, "hf_fp8_status: null workspace");
    HF_CUDA(cudaStreamSynchronize(as_cuda(stream)));
    int word = 0;
    HF_CUDA(cudaMemcpy(&word, workspace, sizeof(int), cudaMemcpyDeviceToHost));
    if (word) return fail(HF_ERR_TIMEOUT, "FP8 product: a bounded wait ran out of time");
    return HF_OK;
}

}  // extern "C"
