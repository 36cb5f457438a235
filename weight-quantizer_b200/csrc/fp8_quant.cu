// Blocks of 8-bit floating point: quantize, the reverse, and the column sums
// of a layer's upstream gradient (its bias gradient).
//
//   block b of x (128 values of a row, or a 128 x 128 tile):
//     s_b = 2^k, the least k >= -117 with max|x| <= 448 * 2^k   (1 if the block is 0)
//     c   = e4m3(x / s_b), nearest, ties to even; x / s_b is exact (a shift of
//           the exponent), so each code is the e4m3 value nearest to x / s_b
//
// Why a power of two: the codes are floating point, so a scale up to twice as
// large costs no relative precision above the least codes, while the division
// and the product code * scale become exact: the weight gradient reads
// code * scale as a bf16 operand without a rounding.
//
// Bytes per value: the input's 2 or 4, 1 for the code, 4/128 (rows) or 4/16384 (tiles) for
// the scale. Tiles are bound by them (28672 x 8192 fp32 205 us, 179 at the copy rate), rows by
// instructions, the shuffles, vote and scale of each eight values (4096 x 8192 bf16 24 us,
// 15.5 at the copy rate).
#include "fp8_types.cuh"
#include "kernels.h"
#include "launch.h"
#include "tc_ptx.cuh"

#include <type_traits>

namespace wq {
namespace {

// Eight consecutive values of a row, as they are in memory; `n` of them exist (the
// others are 0). VEC: the eight are 16-byte aligned in memory.
template <typename T>
struct Eight {
    static constexpr int WORDS = 8 * (int)sizeof(T) / 4;
    uint32_t w[WORDS];
    __device__ __forceinline__ float at(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        const uint32_t h = w[i >> 1];
        if constexpr (std::is_same<T, __nv_bfloat16>::value)   // a bf16 is the upper half of its fp32
            return __uint_as_float(i & 1 ? h & 0xffff0000u : h << 16);
        return __half2float(__ushort_as_half((unsigned short)(i & 1 ? h >> 16 : h & 0xffffu)));
    }
};
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int n, Eight<T>& v) {
    if (VEC && n >= 8) {
#pragma unroll
        for (int i = 0; i < Eight<T>::WORDS / 4; ++i) {
            const uint4 r = ld_stream_v4(reinterpret_cast<const uint4*>(p) + i);
            v.w[4 * i] = r.x, v.w[4 * i + 1] = r.y, v.w[4 * i + 2] = r.z, v.w[4 * i + 3] = r.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < Eight<T>::WORDS; ++i) v.w[i] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i < n) {
                if constexpr (sizeof(T) == 4) v.w[i] = __float_as_uint(to_f32<T>(p[i]));
                else v.w[i >> 1] |= (uint32_t)reinterpret_cast<const unsigned short*>(p)[i] << (16 * (i & 1));
            }
        }
    }
}

// The largest magnitude of a block, held as its bits, which order magnitudes as
// whole numbers (two 16-bit values in a word, or one fp32): no conversions, and a
// value that is not finite shows as bits of at least the infinity's.
template <typename T>
struct Top {
    static constexpr bool WIDE = sizeof(T) == 4;
    static constexpr uint32_t INF =
        WIDE ? 0x7f800000u : (std::is_same<T, __nv_bfloat16>::value ? 0x7f807f80u : 0x7c007c00u);
    static __device__ __forceinline__ uint32_t of(uint32_t w) { return w & (WIDE ? 0x7fffffffu : 0x7fff7fffu); }
    static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) {
        return WIDE ? (a > b ? a : b) : __vmaxu2(a, b);
    }
    // each magnitude that is not finite replaced by 0
    static __device__ __forceinline__ uint32_t finite(uint32_t a) {
        return WIDE ? (a >= INF ? 0u : a) : a & __vcmpltu2(a, INF);
    }
    static __device__ __forceinline__ bool all_finite(uint32_t a) {
        return WIDE ? a < INF : __vcmpltu2(a, INF) == 0xffffffffu;
    }
    static __device__ __forceinline__ float value(uint32_t a) {   // the larger half's
        if constexpr (WIDE) return __uint_as_float(a);
        const uint32_t h = (a >> 16) > (a & 0xffffu) ? a >> 16 : a & 0xffffu;
        if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(h << 16);
        return __half2float(__ushort_as_half((unsigned short)h));
    }
};
template <typename T>
__device__ __forceinline__ uint32_t top8(const Eight<T>& v) {
    uint32_t m = Top<T>::of(v.w[0]);
#pragma unroll
    for (int i = 1; i < Eight<T>::WORDS; ++i) m = Top<T>::max(m, Top<T>::of(v.w[i]));
    return m;
}
template <typename T>
__device__ __forceinline__ uint32_t top8_finite(const Eight<T>& v) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < Eight<T>::WORDS; ++i) m = Top<T>::max(m, Top<T>::finite(Top<T>::of(v.w[i])));
    return m;
}

// Codes of eight values; `n` of them are written. vec: 8-byte aligned. all_finite:
// no NaN or infinity is among them, which saves the test of each.
template <typename T>
__device__ __forceinline__ void store8(uint8_t* p, int n, const Eight<T>& v, float inv, bool vec, bool all_finite) {
    uint32_t w[2];
    if (all_finite) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            w[i] = e4m3x2_finite(v.at(4 * i) * inv, v.at(4 * i + 1) * inv) |
                   (e4m3x2_finite(v.at(4 * i + 2) * inv, v.at(4 * i + 3) * inv) << 16);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            w[i] = e4m3x2(v.at(4 * i) * inv, v.at(4 * i + 1) * inv) |
                   (e4m3x2(v.at(4 * i + 2) * inv, v.at(4 * i + 3) * inv) << 16);
    }
    if (vec && n >= 8) {
        *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else {
        const uint64_t u = (uint64_t)w[0] | ((uint64_t)w[1] << 32);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = (uint8_t)(u >> (8 * i));
    }
}

constexpr int kRowsPerCta = 16;     // one half-warp per row
constexpr int kBlocksPerThread = 4; // consecutive blocks of the row in flight

// One scale per 128 values of a row: 16 lanes hold a block (8 values each). A
// CTA takes 16 rows, so that the scales of one block column, which lie side by
// side for consecutive rows, are written as 64 contiguous bytes.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) fp8_rows_kernel(const T* __restrict__ x, int64_t rows, int64_t cols,
                                                       int64_t ldx, uint8_t* __restrict__ codes, int64_t ldc,
                                                       bool vec_out, float* __restrict__ scales, int64_t s_row,
                                                       int64_t s_col, unsigned int* zero, int64_t zeros) {
    // what follows may start once every CTA is past the work before this launch
    grid_wait();
    launch_dependents();
    for (int64_t i = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x; i < zeros;
         i += (int64_t)gridDim.x * gridDim.y * 256)
        zero[i] = 0;
    const int64_t row = (int64_t)blockIdx.x * kRowsPerCta + (threadIdx.x >> 4);
    const int sub = threadIdx.x & 15;
    const int64_t nb = (cols + kFp8Block - 1) / kFp8Block;
    const int64_t j0 = (int64_t)blockIdx.y * kBlocksPerThread;
    const bool live = row < rows;
    Eight<T> v[kBlocksPerThread];
#pragma unroll
    for (int i = 0; i < kBlocksPerThread; ++i) {
        const int64_t c = (j0 + i) * kFp8Block + sub * 8;
        const int64_t left = live ? cols - c : 0;
        load8<T, VEC>(x + row * ldx + c, left >= 8 ? 8 : (left > 0 ? (int)left : 0), v[i]);
    }
#pragma unroll
    for (int i = 0; i < kBlocksPerThread; ++i) {
        uint32_t m = top8(v[i]);
        const bool fine = __all_sync(0xffffffffu, Top<T>::all_finite(m));
        if (!fine) m = top8_finite(v[i]);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = Top<T>::max(m, __shfl_xor_sync(0xffffffffu, m, o));
        const int e = fp8_scale_exponent(Top<T>::value(m));
        const int64_t j = j0 + i;
        const int64_t c = j * kFp8Block + sub * 8;
        const int64_t left = live ? cols - c : 0;
        if (left > 0) store8(codes + row * ldc + c, left >= 8 ? 8 : (int)left, v[i], pow2i(-e), vec_out, fine);
        if (live && j < nb && sub == 0) scales[row * s_row + j * s_col] = pow2i(e);
    }
}

// One scale per 128 x 128 tile: a CTA holds the tile in registers (half-warp
// h has rows h, h + 16, ...), so the input is read once.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) fp8_tiles_kernel(const T* __restrict__ x, int64_t rows, int64_t cols,
                                                        int64_t ldx, uint8_t* __restrict__ codes, int64_t ldc,
                                                        bool vec_out, float* __restrict__ scales, int64_t s_row,
                                                        int64_t s_col, int64_t nb) {
    __shared__ uint32_t red[8];
    const int64_t bi = blockIdx.x / nb, bj = blockIdx.x - bi * nb;
    const int sub = threadIdx.x & 15;
    const int64_t r0 = bi * kFp8Block + (threadIdx.x >> 4);
    const int64_t c = bj * kFp8Block + sub * 8;
    const int64_t left = cols - c;
    const int n = left >= 8 ? 8 : (left > 0 ? (int)left : 0);
    Eight<T> v[8];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t r = r0 + 16 * i;
        load8<T, VEC>(x + r * ldx + c, r < rows ? n : 0, v[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) m = Top<T>::max(m, top8(v[i]));
    const bool fine = __syncthreads_and(Top<T>::all_finite(m)) != 0;
    if (!fine) {
        m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = Top<T>::max(m, top8_finite(v[i]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = Top<T>::max(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) m = Top<T>::max(m, red[w]);
    const int e = fp8_scale_exponent(Top<T>::value(m));
    const float inv = pow2i(-e);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t r = r0 + 16 * i;
        if (r < rows && n > 0) store8(codes + r * ldc + c, n, v[i], inv, vec_out, fine);
    }
    if (threadIdx.x == 0) scales[bi * s_row + bj * s_col] = pow2i(e);
}

// code * scale (4 and 24 bits) rounded once to T. A scale that is a power of two has an
// exact product in fp32. Of others the product is cut off, for the 16-bit types, and its
// last bit set where anything was: that never falls on the middle of two 16-bit values,
// as a product rounded to fp32 first may.
template <typename T, bool POWER>
__device__ __forceinline__ T value_of(float code, float scale) {
    if (sizeof(T) == 4 || POWER) return from_f32<T>(code * scale);
    const uint32_t cut = __float_as_uint(__fmul_rz(code, scale));
    const bool exact = __fmul_rd(code, scale) == __fmul_ru(code, scale);
    return from_f32<T>(__uint_as_float(exact ? cut : cut | 1u));
}
// out = code * scale, rounded once to the output type. vec: four codes are aligned to their
// 4 bytes, and four values to theirs. 28672 x 8192 to bf16 262 us (2.7 TB/s; scales that are
// no powers of two 291), to fp32 275 us (4.3 TB/s): index divisions and conversions, not bytes.
template <typename T>
__global__ void __launch_bounds__(256) fp8_values_kernel(const uint8_t* __restrict__ codes, int64_t rows,
                                                         int64_t cols, int64_t ldc, int block_rows,
                                                         const float* __restrict__ scales, int64_t s_row,
                                                         int64_t s_col, T* __restrict__ out, int64_t ldo,
                                                         int64_t quads, bool vec) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < rows * quads;
         i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / quads, c = (i - r * quads) * 4;
        const float s = __ldg(scales + (block_rows == 1 ? r : r / kFp8Block) * s_row + (c / kFp8Block) * s_col);
        const int n = cols - c < 4 ? (int)(cols - c) : 4;
        const uint8_t* from = codes + r * ldc + c;
        T* at = out + r * ldo + c;
        uint32_t w = 0;
        if (vec && n == 4) w = __ldg(reinterpret_cast<const uint32_t*>(from));
        else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k < n) w |= (uint32_t)from[k] << (8 * k);
        }
        const float2 lo = e4m3x2_values(w), hi = e4m3x2_values(w >> 16);
        alignas(16) T v[4];
        if (sizeof(T) == 4 || (__float_as_uint(s) & 0x7fffffu) == 0) {
            v[0] = value_of<T, true>(lo.x, s), v[1] = value_of<T, true>(lo.y, s);
            v[2] = value_of<T, true>(hi.x, s), v[3] = value_of<T, true>(hi.y, s);
        } else {
            v[0] = value_of<T, false>(lo.x, s), v[1] = value_of<T, false>(lo.y, s);
            v[2] = value_of<T, false>(hi.x, s), v[3] = value_of<T, false>(hi.y, s);
        }
        if (vec && n == 4) {
            using Four = typename std::conditional<sizeof(T) == 4, uint4, uint2>::type;
            *reinterpret_cast<Four*>(at) = *reinterpret_cast<const Four*>(v);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k < n) at[k] = v[k];
        }
    }
}

// out[n] = sum_m x[m, n] in fp32: a CTA takes 64 columns, 8 threads side by side
// (8 columns each) times 64 row lanes; each thread adds its rows in order, then the
// lanes are added in order (the same bits on every call). There are few CTAs, so each
// thread has eight loads in flight.
constexpr int kSumLanes = 64;
template <typename T, typename O, bool VEC>
__global__ void __launch_bounds__(8 * kSumLanes) column_sum_kernel(const T* __restrict__ x, int64_t rows, int64_t cols,
                                                                   int64_t ldx, O* __restrict__ out) {
    __shared__ float part[kSumLanes][65];
    const int sub = threadIdx.x & 7, lane = threadIdx.x >> 3;
    const int64_t c = (int64_t)blockIdx.x * 64 + sub * 8;
    const int64_t left = cols - c;
    const int n = left >= 8 ? 8 : (left > 0 ? (int)left : 0);
    float acc[8] = {};
    constexpr int AHEAD = sizeof(T) == 4 ? 4 : 8;
    for (int64_t r = lane; r < rows; r += AHEAD * kSumLanes) {
        Eight<T> v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int64_t at = r + i * kSumLanes;
            load8<T, VEC>(x + at * ldx + c, at < rows ? n : 0, v[i]);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[k] += v[i].at(k);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) part[lane][sub * 8 + k] = acc[k];
    __syncthreads();
    if (threadIdx.x < 64 && (int64_t)blockIdx.x * 64 + threadIdx.x < cols) {
        float s = 0.0f;
#pragma unroll 16
        for (int l = 0; l < kSumLanes; ++l) s += part[l][threadIdx.x];
        out[(int64_t)blockIdx.x * 64 + threadIdx.x] = from_f32<O>(s);
    }
}

template <typename T>
cudaError_t quantize_t(const Fp8Quantize& q, cudaStream_t s) {
    const T* x = static_cast<const T*>(q.x);
    const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (q.ldx * (int64_t)sizeof(T)) % 16 == 0;
    const bool vec_out = (reinterpret_cast<uintptr_t>(q.codes) & 7) == 0 && q.ldc % 8 == 0;
    const int64_t nb = (q.cols + kFp8Block - 1) / kFp8Block;
    if (q.block_rows == 1) {
        const dim3 grid((unsigned)((q.rows + kRowsPerCta - 1) / kRowsPerCta),
                        (unsigned)((nb + kBlocksPerThread - 1) / kBlocksPerThread));
        LaunchConfig cfg(grid, 256, 0, s);
        return cudaLaunchKernelEx(&cfg.c, vec ? fp8_rows_kernel<T, true> : fp8_rows_kernel<T, false>, x, q.rows, q.cols,
                                  q.ldx, q.codes, q.ldc, vec_out, q.scales, q.s_row, q.s_col, q.zero, q.zeros);
    } else {
        const unsigned grid = (unsigned)((q.rows + kFp8Block - 1) / kFp8Block * nb);
        if (vec)
            fp8_tiles_kernel<T, true><<<grid, 256, 0, s>>>(x, q.rows, q.cols, q.ldx, q.codes, q.ldc, vec_out,
                                                           q.scales, q.s_row, q.s_col, nb);
        else
            fp8_tiles_kernel<T, false><<<grid, 256, 0, s>>>(x, q.rows, q.cols, q.ldx, q.codes, q.ldc, vec_out,
                                                            q.scales, q.s_row, q.s_col, nb);
    }
    return cudaGetLastError();
}

template <typename T>
cudaError_t values_t(const Fp8Operand& a, T* out, int64_t ldo, cudaStream_t s) {
    const int64_t quads = (a.cols + 3) / 4;
    const int64_t want = (a.rows * quads + 255) / 256;
    const int64_t most = (int64_t)sm_count() * 32;
    const bool vec = (reinterpret_cast<uintptr_t>(a.codes) & 3) == 0 && a.ld % 4 == 0 &&
                     (reinterpret_cast<uintptr_t>(out) & (4 * sizeof(T) - 1)) == 0 && ldo % 4 == 0;
    fp8_values_kernel<T><<<(unsigned)(want < most ? want : most), 256, 0, s>>>(
        a.codes, a.rows, a.cols, a.ld, a.block_rows, a.scales, a.s_row, a.s_col, out, ldo, quads, vec);
    return cudaGetLastError();
}

template <typename T, typename O>
cudaError_t column_sum_t(const T* x, int64_t rows, int64_t cols, int64_t ldx, O* out, cudaStream_t s) {
    const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ldx * (int64_t)sizeof(T)) % 16 == 0;
    const unsigned grid = (unsigned)((cols + 63) / 64);
    if (vec)
        column_sum_kernel<T, O, true><<<grid, 8 * kSumLanes, 0, s>>>(x, rows, cols, ldx, out);
    else
        column_sum_kernel<T, O, false><<<grid, 8 * kSumLanes, 0, s>>>(x, rows, cols, ldx, out);
    return cudaGetLastError();
}

template <typename T>
cudaError_t column_sum_o(const T* x, int64_t rows, int64_t cols, int64_t ldx, void* out, int out_type,
                         cudaStream_t s) {
    if (out_type == kF16) return column_sum_t(x, rows, cols, ldx, static_cast<__half*>(out), s);
    if (out_type == kBf16) return column_sum_t(x, rows, cols, ldx, static_cast<__nv_bfloat16*>(out), s);
    return column_sum_t(x, rows, cols, ldx, static_cast<float*>(out), s);
}

}  // namespace

cudaError_t launch_fp8_quantize(const Fp8Quantize& q, cudaStream_t s) {
    if (q.x_type == kF16) return quantize_t<__half>(q, s);
    if (q.x_type == kBf16) return quantize_t<__nv_bfloat16>(q, s);
    return quantize_t<float>(q, s);
}

cudaError_t launch_fp8_values(const Fp8Operand& a, void* out, int out_type, int64_t ldo, cudaStream_t s) {
    if (out_type == kF16) return values_t(a, static_cast<__half*>(out), ldo, s);
    if (out_type == kBf16) return values_t(a, static_cast<__nv_bfloat16*>(out), ldo, s);
    return values_t(a, static_cast<float*>(out), ldo, s);
}

cudaError_t launch_column_sum(const void* x, int x_type, int64_t rows, int64_t cols, int64_t ldx, void* out,
                              int out_type, cudaStream_t s) {
    if (x_type == kF16) return column_sum_o(static_cast<const __half*>(x), rows, cols, ldx, out, out_type, s);
    if (x_type == kBf16) return column_sum_o(static_cast<const __nv_bfloat16*>(x), rows, cols, ldx, out, out_type, s);
    return column_sum_o(static_cast<const float*>(x), rows, cols, ldx, out, out_type, s);
}

}  // namespace wq
