// The matrix product of blocks of 8-bit floating point.
//
//   y[m, n] = sum_b sa[m, b] sb[n / 128, b] sum_{k in block b} a[m, k] w[n, k] (+ bias[n])
//
// Each block's sum is exact products added in fp32; the scales multiply it once
// per block of 128, and the blocks are added in fp32 in order.
#include "fp8_types.cuh"
#include "kernels.h"

namespace wq {
namespace {

constexpr int kTile = 64;   // output tile, 4 x 4 values per thread
constexpr int kStep = 32;   // contraction values per shared-memory step

template <typename O>
__global__ void __launch_bounds__(256) fp8_gemm_kernel(const Fp8Gemm g) {
    __shared__ float as[kStep][kTile + 4], ws[kStep][kTile + 4];
    const int64_t m0 = (int64_t)blockIdx.y * kTile, n0 = (int64_t)blockIdx.x * kTile;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[4][4] = {};
    for (int64_t k0 = 0; k0 < g.K; k0 += kStep) {
        const int64_t kb = k0 / kFp8Block;
        for (int i = threadIdx.x; i < kTile * kStep; i += 256) {
            const int r = i / kStep, k = i % kStep;
            const int64_t m = m0 + r, kk = k0 + k;
            float v = 0.0f;
            if (m < g.M && kk < g.K)
                v = e4m3x2_values(g.a.codes[m * g.a.ld + kk]).x * g.a.scales[m * g.a.s_row + kb * g.a.s_col];
            as[k][r] = v;
        }
        for (int i = threadIdx.x; i < kTile * kStep; i += 256) {
            const int r = g.transpose ? i % kTile : i / kStep, k = g.transpose ? i / kTile : i % kStep;
            const int64_t n = n0 + r, kk = k0 + k;
            float v = 0.0f;
            if (n < g.N && kk < g.K) {
                const int64_t wr = g.transpose ? kk : n, wc = g.transpose ? n : kk;
                v = e4m3x2_values(g.w.codes[wr * g.w.ld + wc]).x *
                    g.w.scales[(wr / kFp8Block) * g.w.s_row + (wc / kFp8Block) * g.w.s_col];
            }
            ws[k][r] = v;
        }
        __syncthreads();
#pragma unroll 8
        for (int k = 0; k < kStep; ++k) {
            float av[4], wv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                av[i] = as[k][ty * 4 + i];
                wv[i] = ws[k][tx * 4 + i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(av[i], wv[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
            if (m < g.M && n < g.N) {
                const float b = load_any(g.bias, g.bias_type, n);
                static_cast<O*>(g.out)[m * g.ldo + n] = from_f32<O>(acc[i][j] + b);
            }
        }
}

}  // namespace

size_t fp8_gemm_workspace_bytes(int64_t, int64_t, int64_t) { return 0; }

cudaError_t launch_fp8_gemm(const Fp8Gemm& g, void*, cudaStream_t s) {
    const dim3 grid((unsigned)((g.N + kTile - 1) / kTile), (unsigned)((g.M + kTile - 1) / kTile));
    if (g.out_type == kF16) fp8_gemm_kernel<__half><<<grid, 256, 0, s>>>(g);
    else if (g.out_type == kBf16) fp8_gemm_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(g);
    else fp8_gemm_kernel<float><<<grid, 256, 0, s>>>(g);
    return cudaGetLastError();
}

}  // namespace wq
