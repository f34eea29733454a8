// hf_fp8_gemm.cu -- the block-scaled product of e4m3 rows and e4m3 weight rows:
//   out[p, n] = sum_b sx[p, b] sw[n / 128, b] sum_{j in block b} xq[p, j] w[n, j]
//
// 64 positions x 64 weight rows per block, the operands widened to fp32 in
// shared memory in steps of 32 columns, each block of 128 columns summed in
// fp32 and then scaled.
#include "hf_fp8.cuh"

namespace hf {
namespace {

__global__ void __launch_bounds__(256) k_fp8_tile(Fp8Args a) {
    if (a.err && !a.offsets && blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0) *a.err = 0;
    __shared__ float xs[32][65], ws[32][65];
    const int g = blockIdx.y, kb = (a.K + kFp8Block - 1) / kFp8Block;
    const int n0 = blockIdx.x * 64, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int p0 = 0, p1 = a.rows;
    if (a.offsets) {
        p0 = max(0, a.offsets[g]);
        p1 = min(a.rows, a.offsets[g + 1]);
    }
    const uint8_t* w = a.w + g * a.w_stride;
    const float* sw = a.sw + g * a.sw_stride + size_t(n0 / kFp8Block) * kb;
    for (int m0 = p0 + blockIdx.z * 64; m0 < p1; m0 += gridDim.z * 64) {
        float acc[4][4] = {};
        for (int b = 0; b < kb; ++b) {
            float part[4][4] = {};
            for (int c0 = b * kFp8Block; c0 < min(a.K, (b + 1) * kFp8Block); c0 += 32) {
                __syncthreads();
                for (int i = threadIdx.x; i < 64 * 16; i += 256) {
                    const int r = i / 16, c = (i % 16) * 2;
                    uint32_t hx = 0, hw = 0;
                    if (m0 + r < p1 && c0 + c < a.K)
                        hx = unpack2_e4m3(*reinterpret_cast<const uint16_t*>(
                            a.xq + size_t(m0 + r) * a.K + c0 + c));
                    if (n0 + r < a.N && c0 + c < a.K)
                        hw = unpack2_e4m3(*reinterpret_cast<const uint16_t*>(
                            w + size_t(n0 + r) * a.K + c0 + c));
                    const float2 fx = __half22float2(*reinterpret_cast<const __half2*>(&hx));
                    const float2 fw = __half22float2(*reinterpret_cast<const __half2*>(&hw));
                    xs[c][r] = fx.x;
                    xs[c + 1][r] = fx.y;
                    ws[c][r] = fw.x;
                    ws[c + 1][r] = fw.y;
                }
                __syncthreads();
#pragma unroll 8
                for (int c = 0; c < 32; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            part[i][j] = fmaf(xs[c][ty * 4 + i], ws[c][tx * 4 + j], part[i][j]);
            }
            const float s = sw[b];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int p = m0 + ty * 4 + i;
                const float si = p < p1 ? a.sx[size_t(p) * kb + b] * s : 0.0f;
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(part[i][j], si, acc[i][j]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int p = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
                if (p >= p1 || n >= a.N) continue;
                const size_t o = size_t(p) * a.ld_out + n;
                if (a.out_f32) static_cast<float*>(a.out)[o] = acc[i][j];
                else static_cast<__nv_bfloat16*>(a.out)[o] = __float2bfloat16_rn(acc[i][j]);
            }
    }
}

}  // namespace

hf_status launch_fp8_product(const Fp8Args& a, cudaStream_t st) {
    const int mt = (a.rows + 63) / 64;
    const dim3 grid(unsigned((a.N + 63) / 64), unsigned(a.G), unsigned(mt < 8 ? mt : 8));
    k_fp8_tile<<<grid, 256, 0, st>>>(a);
    HF_CUDA(cudaGetLastError());
    return HF_OK;
}

}  // namespace hf
