// Attention of the newest tokens over a paged cache of 8-bit codes with one scale for each (block, K/V head)
// (diopiQuantizedPagedAttention). With K/V rows j of request i in block b_j, codes kc, vc and scales ks, vs:
//     x_j = softmax_scale * ks[b_j] * (q . kc_j),   out = sum_j softmax(x)_j * vs[b_j] * vc_j
// New token t of n sees the first L - (n - 1 - t) tokens; a row that sees none gives zeros.
//
// quant_plain_kernel: any width, strides and block size; one CTA to a query row, a warp to every fourth token.
#include "decode_common.cuh"

namespace b200 {
namespace k {

namespace {

__device__ __forceinline__ float code_value(uint8_t c, bool e4m3) {
    if (!e4m3) return static_cast<float>(static_cast<int8_t>(c));
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(c)));
    return __half2float(__ushort_as_half(static_cast<uint16_t>(h & 0xffffu)));
}

// Tokens of request i, never negative and never more than its row of the table names.
__device__ __forceinline__ int quant_len(const QuantAttnArgs& a, int i) {
    const int64_t cap = static_cast<int64_t>(a.cols) * a.block_size;
    const int64_t L = load_index(a.lens, i);
    return static_cast<int>(imin64(imax64(L, 0), cap));
}

constexpr int kPlainWarps = 4;
constexpr int kPlainRegs = 16;   // head_dim <= 512

template <typename T>
__global__ void __launch_bounds__(32 * kPlainWarps) quant_plain_kernel(const QuantAttnArgs a) {
    __shared__ float s_ml[kPlainWarps][2];
    __shared__ float s_o[kPlainWarps][32 * kPlainRegs];
    const int i = blockIdx.x, hq = blockIdx.y % a.Hq, t = blockIdx.y / a.Hq;
    const int h = hq / (a.Hq / a.Hkv);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int L = quant_len(a, i) - (a.n - 1 - t);
    const T* q = static_cast<const T*>(a.q) + static_cast<int64_t>(i) * a.q_s0 + static_cast<int64_t>(t) * a.q_s1 + static_cast<int64_t>(hq) * a.q_s2;
    const uint8_t* kb = static_cast<const uint8_t*>(a.cache[0]) + static_cast<int64_t>(h) * a.c_s2[0];
    const uint8_t* vb = static_cast<const uint8_t*>(a.cache[1]) + static_cast<int64_t>(h) * a.c_s2[1];
    float qr[kPlainRegs], o[kPlainRegs];
#pragma unroll
    for (int r = 0; r < kPlainRegs; ++r) {
        const int d = lane + 32 * r;
        qr[r] = d < a.D ? Cvt<T>::to_f(q[d]) * a.softmax_scale * kLog2e : 0.f;
        o[r] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int j = warp; j < L; j += kPlainWarps) {
        const int64_t b = load_index(a.table, i, j / a.block_size);
        if (b < 0 || b >= a.blocks) {
            if (lane == 0) report_status(a.status, 1);
            continue;
        }
        const int p = j % a.block_size;
        const float ks = a.scale[0][b * a.s_s0[0] + static_cast<int64_t>(h) * a.s_s1[0]], vs = a.scale[1][b * a.s_s0[1] + static_cast<int64_t>(h) * a.s_s1[1]];
        const uint8_t* kr = kb + b * a.c_s0[0] + static_cast<int64_t>(p) * a.c_s1[0];
        const uint8_t* vr = vb + b * a.c_s0[1] + static_cast<int64_t>(p) * a.c_s1[1];
        float x = 0.f;
#pragma unroll
        for (int r = 0; r < kPlainRegs; ++r) {
            const int d = lane + 32 * r;
            if (d < a.D) x = fmaf(qr[r], code_value(kr[d * a.c_s3[0]], a.e4m3), x);
        }
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
        x *= ks;
        const float mn = fmaxf(m, x);
        const float al = exp2f(m - mn), w = exp2f(x - mn);
        m = mn;
        l = fmaf(l, al, w);
#pragma unroll
        for (int r = 0; r < kPlainRegs; ++r) {
            const int d = lane + 32 * r;
            if (d < a.D) o[r] = fmaf(o[r], al, w * vs * code_value(vr[d * a.c_s3[1]], a.e4m3));
        }
    }
    if (lane == 0) {
        s_ml[warp][0] = m;
        s_ml[warp][1] = l;
    }
#pragma unroll
    for (int r = 0; r < kPlainRegs; ++r) s_o[warp][lane + 32 * r] = o[r];
    __syncthreads();
    float M = -INFINITY, Ls = 0.f, w[kPlainWarps];
#pragma unroll
    for (int k = 0; k < kPlainWarps; ++k) M = fmaxf(M, s_ml[k][0]);
#pragma unroll
    for (int k = 0; k < kPlainWarps; ++k) {
        w[k] = s_ml[k][0] == -INFINITY ? 0.f : exp2f(s_ml[k][0] - M);   // a warp that saw no token
        Ls = fmaf(s_ml[k][1], w[k], Ls);
    }
    const float inv = Ls == 0.f ? 0.f : 1.f / Ls;
    T* out = static_cast<T*>(a.out) + static_cast<int64_t>(i) * a.o_s0 + static_cast<int64_t>(t) * a.o_s1 + static_cast<int64_t>(hq) * a.o_s2;
    for (int d = threadIdx.x; d < a.D; d += 32 * kPlainWarps) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < kPlainWarps; ++k) v = fmaf(s_o[k][d], w[k], v);
        out[d] = Cvt<T>::from_f(v * inv);
    }
}

}  // namespace

int64_t quantized_attention_workspace_bytes(const QuantAttnArgs& a, int sm_count, int max_smem) { return 0; }

const char* launch_quantized_attention(const QuantAttnArgs& a, void* ws, int sm_count, int max_smem, cudaStream_t st) {
    const dim3 grid(a.B, a.n * a.Hq);
    if (a.dt == Dt::F16)
        quant_plain_kernel<__half><<<grid, 32 * kPlainWarps, 0, st>>>(a);
    else if (a.dt == Dt::BF16)
        quant_plain_kernel<__nv_bfloat16><<<grid, 32 * kPlainWarps, 0, st>>>(a);
    else
        quant_plain_kernel<float><<<grid, 32 * kPlainWarps, 0, st>>>(a);
    return "plain";
}

}  // namespace k
}  // namespace b200
