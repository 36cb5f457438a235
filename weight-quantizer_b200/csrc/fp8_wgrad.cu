// The weight gradient of a linear layer from the 8-bit checkpoint of its input.
//
//   dw[n, k] (+)= sum_m dy[m, n] c[m, k] s[m, k / 128]
#include "fp8_types.cuh"
#include "kernels.h"

namespace wq {
namespace {

constexpr int kTile = 64;   // output tile, 4 x 4 values per thread
constexpr int kStep = 32;   // rows of dy and x per shared-memory step

template <typename O>
__global__ void __launch_bounds__(256) fp8_wgrad_kernel(const Fp8WeightGrad g) {
    __shared__ float ds[kStep][kTile + 4], xs[kStep][kTile + 4];
    const int64_t n0 = (int64_t)blockIdx.y * kTile, k0 = (int64_t)blockIdx.x * kTile;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[4][4] = {};
    for (int64_t m0 = 0; m0 < g.M; m0 += kStep) {
        for (int i = threadIdx.x; i < kTile * kStep; i += 256) {
            const int r = i / kTile, c = i % kTile;
            const int64_t m = m0 + r, n = n0 + c, k = k0 + c;
            ds[r][c] = m < g.M && n < g.N ? load_any(g.dy, g.dy_type, m * g.ldy + n) : 0.0f;
            xs[r][c] = m < g.M && k < g.K ? e4m3x2_values(g.a.codes[m * g.a.ld + k]).x *
                                                g.a.scales[m * g.a.s_row + (k / kFp8Block) * g.a.s_col]
                                          : 0.0f;
        }
        __syncthreads();
#pragma unroll 8
        for (int r = 0; r < kStep; ++r) {
            float dv[4], xv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                dv[i] = ds[r][ty * 4 + i];
                xv[i] = xs[r][tx * 4 + i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(dv[i], xv[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t n = n0 + ty * 4 + i, k = k0 + tx * 4 + j;
            if (n < g.N && k < g.K) {
                O* o = static_cast<O*>(g.out) + n * g.ldo + k;
                *o = from_f32<O>(g.accumulate ? to_f32<O>(*o) + acc[i][j] : acc[i][j]);
            }
        }
}

}  // namespace

size_t fp8_weight_grad_workspace_bytes(int64_t, int64_t, int64_t, int) { return 0; }

cudaError_t launch_fp8_weight_grad(const Fp8WeightGrad& g, void*, cudaStream_t s) {
    const dim3 grid((unsigned)((g.K + kTile - 1) / kTile), (unsigned)((g.N + kTile - 1) / kTile));
    if (g.out_type == kF16) fp8_wgrad_kernel<__half><<<grid, 256, 0, s>>>(g);
    else if (g.out_type == kBf16) fp8_wgrad_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(g);
    else fp8_wgrad_kernel<float><<<grid, 256, 0, s>>>(g);
    return cudaGetLastError();
}

}  // namespace wq
