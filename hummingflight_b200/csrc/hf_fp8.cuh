// hf_fp8.cuh -- e4m3 helpers and the interface between the FP8 host code and
// its kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "hf_fp8.h"
#include "hf_internal.cuh"

namespace hf {

constexpr int kFp8Block = HF_FP8_BLOCK;

// Four floats (|v| <= 448, or NaN) as e4m3, rounded to nearest even; a in the
// lowest byte.
__device__ __forceinline__ uint32_t pack4_e4m3(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return uint32_t(lo) | (uint32_t(hi) << 16);
}

// Two e4m3 values as halves (exact: every e4m3 value is an FP16 one).
__device__ __forceinline__ uint32_t unpack2_e4m3(uint16_t v) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(v));
    return h;
}

// Scale of a block whose largest magnitude is m: the smallest power of two with
// m <= 448 s (448 = 1.75 * 2^8), at least 2^-126; 1 for a block of zeros; NaN
// for one that holds Inf or NaN. inv: 1 / s, a power of two as well.
__device__ __forceinline__ float block_scale(float m, float& inv) {
    const uint32_t b = __float_as_uint(m);
    if (b >= 0x7f800000u) {
        inv = __uint_as_float(0x7fc00000u);
        return inv;
    }
    if (b == 0u) {
        inv = 1.0f;
        return 1.0f;
    }
    // biased exponent of s: that of m less 8, one more above 1.75
    const int e = int(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    const int se = e < 1 ? 1 : e;
    inv = __uint_as_float(uint32_t(254 - se) << 23);
    return __uint_as_float(uint32_t(se) << 23);
}

// Expert outputs on their way to a bf16 sum (bf16 rows would put a second rounding of
// the output's size under it): two arrays, in one of two forms.
// Few positions a segment (k_fp8_mma): 24 bits of the fp32 number, 16 of them
// significant, its upper half and the next byte. The rest is cut off (2^-15 of the
// value; numbers of 16 bits, Inf and NaN stay as they are).
// CTA pairs, where the rows' bytes count: FP16 times a power of two per kYBlock columns
// of a position, whose exponents are the second array. The block's largest magnitude
// lies in [2^14, 2^15), so nothing overflows, and what is up to 2^28 smaller still has
// all 11 bits.
// 16384 tokens, k = 8, 256 experts of 6144 x 2048, ms: bf16 rows 8.34, FP16 8.65, 24 bits
// 8.94. 64 rows of one expert, us: bf16 rows 41, 24 bits 42, FP16 (maxima across the
// warp) 45.
constexpr int kYBlock = 32;

// Biased exponent of a block's factor, from the bits of its largest finite magnitude.
__device__ __forceinline__ uint32_t y_exponent(uint32_t top) {
    const int e = int(top >> 23) - 14;
    return top == 0u ? 127u : uint32_t(e < 1 ? 1 : e);
}
__device__ __forceinline__ float y_inverse(uint32_t e) { return __uint_as_float((254u - e) << 23); }
__device__ __forceinline__ float y_factor(uint32_t e) { return __uint_as_float(e << 23); }

// Eight numbers from their upper halves and third bytes.
__device__ __forceinline__ void unpack24(const uint4 hi, const uint2 lo, float (&f)[8]) {
    const uint32_t h[4] = {hi.x, hi.y, hi.z, hi.w}, l[2] = {lo.x, lo.y};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        // bytes: half i of h, byte i of l, 0
        const uint32_t w = __byte_perm(l[i >> 2], h[i >> 1], ((i & 1) ? 0x7600 : 0x5400) | (i & 3) << 4);
        f[i] = __uint_as_float(w & 0xffffff00u);
    }
}
// Eight numbers from FP16 and their block's exponent.
__device__ __forceinline__ void unpack16(const uint4 v, uint32_t e, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = h.x * y_factor(e);
        f[2 * i + 1] = h.y * y_factor(e);
    }
}

// ------------------------------------------------------------------ products
// Rows of e4m3 activations (positions) against weight rows. One group (offsets
// null: all rows) or G groups: group g multiplies positions [offsets[g],
// offsets[g+1]) by its own matrix.
struct Fp8Args {
    const uint8_t* xq;      // [rows x K]
    const float* sx;        // [rows x ceil(K/128)]
    const uint8_t* w;       // view of K-wide rows: row n of group g at g * a_stride + a_base + n
    long long a_rows;       // rows of the view
    int a_stride, a_base;
    const float* sw;        // scales [ceil(N/128) x ceil(K/128)] of group g at sw + g * sw_stride
    long long sw_stride;
    const int32_t* offsets; // [G + 1] or null
    int G, rows, N, K;
    // product: out [rows x N] in bf16 or f32, or (out_aux given) 16 bits of each in out
    // and in out_aux the third bytes [rows x N] or exponents [rows x ceil(N/kYBlock)]
    void* out;
    int out_f32;
    uint8_t* out_aux;
    // runs of K: run s takes blocks [s * kbper, ...) and writes rows [s * rows, ...)
    // of out (fp32 when there are several)
    int nsplit, kbper;
    // gate/up: the up rows follow the N gate rows, their scales sw_up floats
    // further; silu(g) * u quantised into mid_q [rows x N], mid_s [rows x ceil(N/128)]
    long long sw_up;
    uint8_t* mid_q;
    float* mid_s;
    int* err;               // error word: set when a bounded wait gives up
    int clear_err;          // the first kernel of a call clears it
    // limit of a wait, ns (set by launch_fp8_product), and the test hook: the copies
    // stop ahead of a CTA's stall-th block of K (0: never) and wait on a barrier that
    // nothing signals; stall < 0: those of a pair's second CTA only
    unsigned long long wait_ns;
    int stall;
    // 1: the launch before this one is of the same call and lets this one start only
    // after its own griddep_wait, so everything ahead of the call is done: offsets and
    // weights can be read before this kernel's griddep_wait
    int early;
};
hf_status launch_fp8_product(Fp8Args a, bool glu, cudaStream_t st);
void set_fp8_wait(unsigned long long ns);  // 0: the default
void set_fp8_stall(int block);
// Positions of a tile, by the mean per segment (256: the pair kernel's).
int fp8_tile_rows(int mean);
inline bool fp8_pairs(int mean) { return fp8_tile_rows(mean) == 256; }
struct Fp8Split {
    int n, per;  // runs, blocks of K in each
};
// tiles: of bn positions (32, 64, or 256 for CTA pairs); plane_bytes: of one run
Fp8Split fp8_split(long long tiles, int bn, int K, double plane_bytes);
// One group, with its runs of K chosen by size; planes: fp32 [n x T x N] when n > 1.
Fp8Split fp8_gemm_split(int T, int N, int K);
hf_status launch_fp8_gemm(const Fp8Args& a, float* planes, cudaStream_t st);

}  // namespace hf
