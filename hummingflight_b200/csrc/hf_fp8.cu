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
// 16 threads own one block of 128 columns, 8 columns each.
struct QuantArgs {
    const void* x;
    long long ldx;
    int rows, K, nb;
    uint8_t* q;
    float* s;
    // gather (experts): the row of slot perm[p]'s token goes to position p;
    // null: row t of x to row t of q
    const int32_t* perm;
    int k, n_tok;
    int32_t* pos;  // [slots] position of each slot
    int* err;      // error word, cleared by the first block
};

template <bool XF32>
__global__ void __launch_bounds__(256) k_quantize(QuantArgs a) {
    if (a.err && blockIdx.x == 0 && threadIdx.x == 0) *a.err = 0;
    const int sub = threadIdx.x & 15;
    const unsigned half = 0xffffu << (threadIdx.x & 16);
    const long long blocks = (long long)a.rows * a.nb;
    for (long long i = (long long)blockIdx.x * 16 + (threadIdx.x >> 4); i < blocks;
         i += (long long)gridDim.x * 16) {
        const int p = int(i / a.nb), b = int(i % a.nb);
        int row = p;
        if (a.perm) {
            const int slot = a.perm[p];
            if (slot < 0 || slot / a.k >= a.n_tok) continue;
            row = slot / a.k;
            if (b == 0 && sub == 0) a.pos[slot] = p;
        }
        const int c = b * kFp8Block + sub * 8;
        float v[8] = {};
        if (c < a.K) load8<XF32>(a.x, row * a.ldx + c, v);
        uint32_t m = 0;  // magnitudes order as their bits; NaN is above Inf
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(half, m, o));
        float inv;
        const float s = block_scale(__uint_as_float(m), inv);
        if (c < a.K)
            *reinterpret_cast<uint2*>(a.q + size_t(p) * a.K + c) =
                make_uint2(pack4_e4m3(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                           pack4_e4m3(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
        if (sub == 0) a.s[size_t(p) * a.nb + b] = s;
    }
}

hf_status launch_quantize(const QuantArgs& a, bool f32, int dev, cudaStream_t st) {
    const long long groups = ((long long)a.rows * a.nb + 15) / 16;
    const int grid = int(std::min<long long>(groups, num_sms(dev) * 16));
    if (f32) k_quantize<true><<<grid, 256, 0, st>>>(a);
    else k_quantize<false><<<grid, 256, 0, st>>>(a);
    HF_CUDA(cudaGetLastError());
    return HF_OK;
}

// ------------------------------------------------------------------ combine
// out[t] = resid[t] + sum_i w[t, i] y[pos(t, i)], rank order, fp32: the
// reference's separate multiply and add per pick.
template <bool F32>
__device__ __forceinline__ void load4(const void* p, size_t i, float (&v)[4]) {
    if constexpr (F32) {
        const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    } else {
        const uint2 a = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
        v[0] = bf16lo(a.x); v[1] = bf16hi(a.x); v[2] = bf16lo(a.y); v[3] = bf16hi(a.y);
    }
}

template <bool F32>
__global__ void __launch_bounds__(256) k_fp8_combine(const void* y, const int32_t* pos,
                                                     const float* w, int T, int k, int H,
                                                     const void* resid, void* out) {
    const long long n = (long long)T * (H / 4);
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256ll) {
        const int t = int(i / (H / 4)), c = int(i % (H / 4)) * 4;
        float acc[4] = {}, v[4];
        for (int j = 0; j < k; ++j) {
            const float wj = w[size_t(t) * k + j];
            const unsigned at = unsigned(pos[size_t(t) * k + j]);
            if (at >= unsigned(T * k)) continue;  // a slot that perm does not name
            load4<F32>(y, size_t(at) * H + c, v);
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[q] = __fadd_rn(acc[q], __fmul_rn(wj, v[q]));
        }
        const size_t o = size_t(t) * H + c;
        if (resid) {
            load4<F32>(resid, o, v);
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[q] = __fadd_rn(v[q], acc[q]);
        }
        if constexpr (F32) {
            *reinterpret_cast<float4*>(static_cast<float*>(out) + o) =
                make_float4(acc[0], acc[1], acc[2], acc[3]);
        } else {
            const __nv_bfloat162 a = __floats2bfloat162_rn(acc[0], acc[1]);
            const __nv_bfloat162 b = __floats2bfloat162_rn(acc[2], acc[3]);
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + o) =
                make_uint2(*reinterpret_cast<const uint32_t*>(&a),
                           *reinterpret_cast<const uint32_t*>(&b));
        }
    }
}

// ------------------------------------------------------------------ workspaces
struct ExpertsWs {
    size_t pos, xq, sx, mq, ms, y, total;
};

ExpertsWs experts_ws(int T, int k, int H, int I, bool f32) {
    ExpertsWs w{};
    const size_t n = size_t(T) * k;
    size_t o = kAlign;  // the error word
    const auto take = [&](size_t bytes) {
        const size_t at = o;
        o += up(bytes);
        return at;
    };
    w.pos = take(n * 4);
    w.xq = take(n * H);
    w.sx = take(n * blocks128(H) * 4);
    w.mq = take(n * I);
    w.ms = take(n * blocks128(I) * 4);
    w.y = take(n * H * (f32 ? 4 : 2));
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
    if (T < 0 || K <= 0 || K % 16)
        return fail(HF_ERR_ARG, "hf_fp8_quantize: T >= 0 and K a positive multiple of 16");
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
    if (T <= 0 || N <= 0 || K <= 0) return 0;
    const Fp8Split sp = fp8_split(T, N, K);
    return kAlign + (sp.n > 1 ? up(size_t(sp.n) * T * N * sizeof(float)) : 0);
}

hf_status hf_fp8_gemm(const uint8_t* xq, const float* sx, const uint8_t* wq, const float* sw, int T,
                      int N, int K, void* out, hf_dtype out_dtype, void* workspace,
                      size_t workspace_bytes, hf_stream stream) {
    if (T < 0 || N <= 0 || K <= 0 || K % 16)
        return fail(HF_ERR_ARG, "hf_fp8_gemm: T >= 0, N > 0 and K a positive multiple of 16");
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
    if (T <= 0 || top_k <= 0 || E <= 0 || H <= 0 || I <= 0) return 0;
    return experts_ws(T, top_k, H, I, out_dtype == HF_F32).total;
}

hf_status hf_fp8_moe_experts(const uint8_t* experts, const float* scales, int E, int H, int I,
                             const void* x, hf_dtype x_dtype, long long ldx, int T, int top_k,
                             const hf_moe_routing* r, const void* resid, void* out,
                             hf_dtype out_dtype, void* workspace, size_t workspace_bytes,
                             hf_stream stream) {
    const std::string f("hf_fp8_moe_experts");
    if (E < 1 || E > kMaxExperts) return fail(HF_ERR_ARG, f + ": E must be in 1..1024");
    if (H <= 0 || I <= 0 || H % 16 || I % 16)
        return fail(HF_ERR_ARG, f + ": H and I must be positive multiples of 16");
    if (top_k < 1 || top_k > kMaxK) return fail(HF_ERR_ARG, f + ": top_k must be in 1..32");
    if (T < 0 || (long long)T * top_k > 0x7fffffffll)
        return fail(HF_ERR_ARG, f + ": T >= 0 and T * top_k below 2^31");
    if (bad_type(x_dtype) || bad_type(out_dtype))
        return fail(HF_ERR_ARG, f + ": x and out must be bf16 or f32");
    if (T == 0) return HF_OK;
    if (!experts || !scales || !x || !out || !workspace || !r || !r->topk_weights || !r->offsets ||
        !r->perm)
        return fail(HF_ERR_ARG, f + ": null pointer");
    if (bad_rows(x, x_dtype, ldx, H))
        return fail(HF_ERR_ARG, f + ": x and its pitch must be 16-byte aligned, the pitch at "
                                    "least H");
    if (!aligned16(experts) || !aligned16(out) || (resid && !aligned16(resid)))
        return fail(HF_ERR_ARG, f + ": pointers must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(workspace) % kAlign)
        return fail(HF_ERR_ARG, f + ": workspace must be 256-byte aligned");
    const bool f32 = out_dtype == HF_F32;
    const ExpertsWs L = experts_ws(T, top_k, H, I, f32);
    if (workspace_bytes < L.total)
        return fail(HF_ERR_ARG, f + ": workspace smaller than hf_fp8_moe_experts_workspace_size");
    if (resid && resid != out) {
        const uintptr_t p = reinterpret_cast<uintptr_t>(resid), q = reinterpret_cast<uintptr_t>(out);
        const uintptr_t bytes = size_t(T) * H * (f32 ? 4 : 2);
        if (p < q + bytes && q < p + bytes)
            return fail(HF_ERR_ARG, f + ": resid and out overlap without being the same buffer");
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
    a.sw_up = (long long)ib * hb;
    a.offsets = r->offsets;
    a.G = E;
    a.rows = n;
    a.N = I;
    a.K = H;
    a.nsplit = 1;
    a.kbper = hb;
    a.mid_q = ws + L.mq;
    a.mid_s = reinterpret_cast<float*>(ws + L.ms);
    a.err = qa.err;
    HF_TRY(launch_fp8_product(a, true, st));
    a.xq = a.mid_q;
    a.sx = a.mid_s;
    a.a_rows = 3ll * E * H;
    a.a_stride = 3 * H;
    a.a_base = 2 * H;
    a.sw = scales + 2ll * ib * hb;
    a.N = H;
    a.K = I;
    a.kbper = ib;
    a.out = ws + L.y;
    a.out_f32 = f32;
    HF_TRY(launch_fp8_product(a, false, st));
    const int grid = num_sms(dev) * 8;
    if (f32)
        k_fp8_combine<true><<<grid, 256, 0, st>>>(ws + L.y, qa.pos, r->topk_weights, T, top_k, H,
                                                  resid, out);
    else
        k_fp8_combine<false><<<grid, 256, 0, st>>>(ws + L.y, qa.pos, r->topk_weights, T, top_k, H,
                                                   resid, out);
    HF_CUDA(cudaGetLastError());
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
