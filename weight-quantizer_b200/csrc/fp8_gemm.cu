// The matrix product of blocks of 8-bit floating point.
//
//   y[m, n] = sum_b sa[m, b] sb[n / 128, b] sum_{k in block b} a[m, k] w[n, k] (+ bias[n])
//
// A block's sum over 128 products runs on the tensor cores (e4m3 x e4m3, fp32 in
// tensor memory); the scales cannot enter there, so each block's sum is read back
// and added to fp32 registers, times the product of its two scales.
#include "fp8_types.cuh"
#include "kernels.h"
#include "tc_ptx.cuh"

#include "launch.h"

namespace wq {
namespace {

// ---- large products: pairs of CTAs ------------------------------------------------
//
// A pair of CTAs (two SMs) makes a 256 x 256 tile of y with tcgen05.mma of
// cta_group::2: each CTA holds 128 rows of a and 128 of the tile's 256 columns of
// w in shared memory, and 128 rows x 256 columns of the block's sums in tensor
// memory, twice (512 columns), so that block b + 1 multiplies while block b is
// read back. Bytes from L2 per block and CTA: 32 KB for 128 x 256 x 128 products,
// half of what one CTA with a 128 x 128 tile would read.
//
// Warp 0 of each CTA loads (TMA, 128-byte swizzle: a block of 128 codes is one
// swizzled row), warp 1 of the even CTA issues the MMAs of both, and eight
// warps of each CTA hold the sums: warp e reads tensor-memory lanes 32 (e % 4)
// .. + 31 (a lane is a row of y, so its scale is one register) and columns
// 128 (e / 4) .. + 127 (one 128-column block, so sb is one value).
//
// The transposed weight needs no copy: rows of 128 codes along y's columns are
// the MMA's MN-major form of the same operand.

constexpr int kPairTile = 256;
constexpr int kPairStages = 6;                      // even: each issuing warp has its own
constexpr int kOperandBytes = 128 * 128;            // one operand of one CTA for one block
constexpr int kPairStage = 2 * kOperandBytes;
constexpr int kPairThreads = 384;
constexpr int kPairLaunchRegs = 168, kPairCtlRegs = 56, kPairSumRegs = 224;
static_assert(kPairCtlRegs + 2 * kPairSumRegs <= 3 * kPairLaunchRegs, "register split exceeds the launch's registers");

struct PairSmem {
    static constexpr int BAR = kPairStages * kPairStage;
    // full and done per stage (done: the block's MMAs are over, so its operands
    // may be replaced and its sums read); sums empty[2]
    static constexpr int TMEM_SLOT = BAR + 8 * (2 * kPairStages + 2);
    static constexpr int TOTAL = TMEM_SLOT + 16;
    static_assert(TOTAL + 1024 <= 227 * 1024, "stages exceed the shared memory of one CTA");
};

struct PairParams {
    const float* sa;
    int64_t sa_row, sa_col;
    const float* sw;
    int64_t sw_n, sw_k;      // strides of sw by column block of y and by inner block
    const void* bias;
    int bias_type;
    void* out;
    int out_type;
    int64_t ldo;
    int M, N, blocks;        // inner blocks of 128
    int tiles_m, tiles_n, band;
    bool wide_out;           // rows of out are 32-byte aligned
    unsigned int* fault;
};

// Tile t of the raster: bands of `band` row tiles; inside a band the row tiles
// run fastest, so that the band's rows of a stay in L2 while w streams by once.
__device__ __forceinline__ void tile_of(int t, const PairParams& p, int& mt, int& nt) {
    const int per = p.band * p.tiles_n;
    const int b = t / per, in = t - b * per;
    const int bw = min(p.band, p.tiles_m - b * p.band);
    nt = in / bw;
    mt = b * p.band + (in - nt * bw);
}

// 32 columns (c .. c + 31) of row m of y from fp32 sums.
template <typename O>
__device__ __forceinline__ void store32(O* row, int64_t c, int64_t n, bool wide, const float (&v)[32], const void* bias,
                                        int bias_type) {
    float b[32];
    if (bias != nullptr) {
#pragma unroll
        for (int i = 0; i < 32; ++i) b[i] = c + i < n ? load_any(bias, bias_type, c + i) : 0.0f;
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) b[i] = -0.0f;   // leaves every value as it is
    }
    if (wide && c + 32 <= n) {
        constexpr int PER = 4 / (int)sizeof(O);       // values in a word
#pragma unroll
        for (int i = 0; i < 32; i += 8 * PER) {
            uint32_t w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                O e[PER];
#pragma unroll
                for (int j = 0; j < PER; ++j) e[j] = from_f32<O>(v[i + k * PER + j] + b[i + k * PER + j]);
                w[k] = *reinterpret_cast<const uint32_t*>(e);
            }
            st_32(row + c + i, w);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (c + i < n) row[c + i] = from_f32<O>(v[i] + b[i]);
    }
}

template <bool WT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    fp8_gemm_pair_kernel(const PairParams p, const __grid_constant__ CUtensorMap map_a,
                         const __grid_constant__ CUtensorMap map_w) {
    using L = PairSmem;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_addr(smem);
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // uniform
    const int rank = (int)cluster_rank();
    auto bar = [&](int i) -> uint32_t { return sbase + L::BAR + 8u * (uint32_t)i; };
    auto full = [&](int s) { return bar(s); };
    auto done = [&](int s) { return bar(kPairStages + s); };
    auto sums_empty = [&](int b) { return bar(2 * kPairStages + b); };
    launch_dependents();
    if (threadIdx.x == 0) {
        for (int s = 0; s < kPairStages; ++s) {
            mbar_init(full(s), 1);     // the even CTA's: its own arrival plus both CTAs' bytes
            mbar_init(done(s), 1);
        }
        for (int b = 0; b < 2; ++b)
            mbar_init(sums_empty(b), 16);   // the even CTA's: one arrival per summing warp of the pair
        fence_mbarrier_init();
    }
    if (warp == 1) tmem_alloc<2>(sbase + L::TMEM_SLOT, 512);
    tc_before();
    __syncthreads();
    cluster_sync();
    tc_after();
    grid_wait();   // nothing above reads global memory
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + L::TMEM_SLOT);
    const int pairs = (int)gridDim.x >> 1, first = (int)blockIdx.x >> 1;
    const int tiles = p.tiles_m * p.tiles_n;
    const int mine = first < tiles ? (tiles - 1 - first) / pairs + 1 : 0;
    const int64_t steps = (int64_t)mine * p.blocks;
    bool faulted = false;
    auto give_up = [&]() {
        faulted = true;
        atomicOr(p.fault, 1u);
    };

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPairCtlRegs));
        if (warp == 0) {
            // each CTA loads its 128 rows of a and its 128 columns of w; the
            // bytes count on the even CTA's barrier
            const uint32_t full0 = in_cta(full(0), 0);
            int s = 0;
            uint32_t ph = 1;
            for (int t = first; t < tiles; t += pairs) {
                int mt, nt;
                tile_of(t, p, mt, nt);
                const int m0 = mt * kPairTile + rank * 128, n0 = nt * kPairTile + rank * 128;
                for (int b = 0; b < p.blocks; ++b) {
                    if (!faulted && !mbar_wait_bounded(done(s), ph)) give_up();
                    __syncwarp();
                    if (elect_one()) {
                        const uint32_t f = full0 + 8u * (uint32_t)s;
                        const uint32_t dst = sbase + (uint32_t)(s * kPairStage);
                        if (rank == 0) mbar_arrive_expect_tx(full(s), 2 * kPairStage);
                        tma_box<2>(dst, &map_a, b * 128, m0, f);
                        if constexpr (WT) tma_box<2>(dst + kOperandBytes, &map_w, n0, b * 128, f);
                        else tma_box<2>(dst + kOperandBytes, &map_w, b * 128, n0, f);
                    }
                    __syncwarp();
                    if (++s == kPairStages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
            }
            // every copy this warp started has been read before the CTA goes
            // (a stage that was never filled passes at once)
            for (int i = 0; i < kPairStages; ++i) {
                if (!mbar_wait_bounded(done(s), ph)) atomicOr(p.fault, 1u);
                if (++s == kPairStages) {
                    s = 0;
                    ph ^= 1u;
                }
            }
        } else if ((warp == 1 || warp == 2) && rank == 0) {
            // even blocks by warp 1, odd ones by warp 2: a wait on a barrier takes
            // about 170 cycles beside the MMAs' own reads of shared memory, and one
            // warp's waits and its issue together take as long as a block's MMAs
            constexpr uint32_t idesc = mma_idesc(0, false, WT, 256, 256);
            const uint64_t desc0 = sw128_matrix(sbase);
            const int buf = warp - 1;
            const uint32_t d = tmem + (uint32_t)(buf * 256);
            int s = buf;
            uint32_t ph = 0;
            for (int64_t i = buf; i < steps; i += 2) {
                if (!faulted && !mbar_wait_bounded(full(s), ph)) give_up();
                const uint64_t da = desc0 + (uint64_t)(s * (kPairStage >> 4));
                const uint64_t dw = da + (uint64_t)(kOperandBytes >> 4);
                if (i >= 2 && !faulted && !mbar_wait_bounded(sums_empty(buf), (uint32_t)(((i >> 1) - 1) & 1)))
                    give_up();
                __syncwarp();
                tc_after();
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)   // 32 codes: 32 bytes of a row, or 32 rows of 128 bytes
                        mma_f8<2>(d, da + 2u * k, dw + (WT ? 256u : 2u) * k, idesc, k > 0);
                    mma_done<2>(done(s));
                }
                __syncwarp();
                s += 2;
                if (s >= kPairStages) {
                    s = buf;
                    ph ^= 1u;
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPairSumRegs));
        const int q = warp & 3, half = (warp - 4) >> 2;
        const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(half * 128);
        const uint32_t free0 = in_cta(sums_empty(0), 0);
        int64_t i = 0;
        int s = 0;
        uint32_t ph = 0;
        for (int t = first; t < tiles; t += pairs) {
            int mt, nt;
            tile_of(t, p, mt, nt);
            const int64_t m = (int64_t)mt * kPairTile + rank * 128 + q * 32 + lane;
            const int64_t n0 = (int64_t)nt * kPairTile + half * 128;
            const float* sa = p.sa + min(m, (int64_t)p.M - 1) * p.sa_row;
            const float* sw = p.sw + min(n0, (int64_t)p.N - 1) / 128 * p.sw_n;
            uint64_t acc[64];
#pragma unroll
            for (int c = 0; c < 64; ++c) acc[c] = 0;
            // the scales of the next three blocks are on their way
            float a1 = __ldg(sa), w1 = __ldg(sw), a2 = 0, w2 = 0, a3 = 0, w3 = 0;
            if (p.blocks > 1) a2 = __ldg(sa + p.sa_col), w2 = __ldg(sw + p.sw_k);
            if (p.blocks > 2) a3 = __ldg(sa + 2 * p.sa_col), w3 = __ldg(sw + 2 * p.sw_k);
            for (int b = 0; b < p.blocks; ++b, ++i) {
                const int buf = (int)(i & 1);
                const float sc = a1 * w1;
                a1 = a2, w1 = w2, a2 = a3, w2 = w3;
                if (b + 3 < p.blocks) a3 = __ldg(sa + (b + 3) * p.sa_col), w3 = __ldg(sw + (b + 3) * p.sw_k);
                const uint64_t sc2 = pack2(sc, sc);
                const uint32_t from = taddr + (uint32_t)(buf * 256);
                uint64_t v[32];
                if (!faulted && !mbar_wait_bounded(done(s), ph)) give_up();
                __syncwarp();
                tc_after();
                tmem_pairs(from, v);
#pragma unroll
                for (int c = 0; c < 32; ++c) fma2(acc[c], v[c], sc2);
                tmem_pairs(from + 64u, v);
                tc_before();
                __syncwarp();
                if (lane == 0) arrive_in_cluster(free0 + 8u * (uint32_t)buf);
#pragma unroll
                for (int c = 0; c < 32; ++c) fma2(acc[32 + c], v[c], sc2);
                if (++s == kPairStages) {
                    s = 0;
                    ph ^= 1u;
                }
            }
            if (m < p.M) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float v[32];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const float2 f = unpack2(acc[16 * c + k]);
                        v[2 * k] = f.x;
                        v[2 * k + 1] = f.y;
                    }
                    const int64_t col = n0 + 32 * c;
                    if (p.out_type == kBf16)
                        store32(static_cast<__nv_bfloat16*>(p.out) + m * p.ldo, col, p.N, p.wide_out, v, p.bias,
                                p.bias_type);
                    else if (p.out_type == kF16)
                        store32(static_cast<__half*>(p.out) + m * p.ldo, col, p.N, p.wide_out, v, p.bias, p.bias_type);
                    else
                        store32(static_cast<float*>(p.out) + m * p.ldo, col, p.N, p.wide_out, v, p.bias, p.bias_type);
                }
            }
        }
    }
    tc_before();
    __syncthreads();
    cluster_sync();   // the pair's MMAs, arrivals and reads of tensor memory are over
    tc_after();
    if (warp == 1) tmem_free<2>(tmem, 512);
}

// ---- host side ------------------------------------------------------------------------

int type_bytes(int t) { return t == kF32 ? 4 : 2; }

// y = bias, or 0, in every row: a product without inner values.
template <typename O>
__global__ void fill_rows_kernel(O* out, int64_t M, int64_t N, int64_t ldo, const void* bias, int bias_type) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < M * N; i += (int64_t)gridDim.x * blockDim.x)
        out[i / N * ldo + i % N] = from_f32<O>(load_any(bias, bias_type, i % N));
}

template <bool WT>
cudaError_t launch_pair(const Fp8Gemm& g, cudaStream_t s) {
    PairParams p;
    p.sa = g.a.scales;
    p.sa_row = g.a.s_row;
    p.sa_col = g.a.s_col;
    p.sw = g.w.scales;
    p.sw_n = WT ? g.w.s_col : g.w.s_row;
    p.sw_k = WT ? g.w.s_row : g.w.s_col;
    p.bias = g.bias;
    p.bias_type = g.bias_type;
    p.out = g.out;
    p.out_type = g.out_type;
    p.ldo = g.ldo;
    p.M = (int)g.M;
    p.N = (int)g.N;
    p.blocks = (int)((g.K + 127) / 128);
    p.tiles_m = (int)((g.M + kPairTile - 1) / kPairTile);
    p.tiles_n = (int)((g.N + kPairTile - 1) / kPairTile);
    // the rows of a band stay below 40 MB, well inside L2
    const int64_t per_tile = (int64_t)kPairTile * p.blocks * 128;
    int64_t band = ((int64_t)40 << 20) / per_tile;
    band = band < 1 ? 1 : band;
    const int64_t bands = (p.tiles_m + band - 1) / band;
    p.band = (int)((p.tiles_m + bands - 1) / bands);
    p.wide_out = (reinterpret_cast<uintptr_t>(g.out) & 31) == 0 && (g.ldo * type_bytes(g.out_type)) % 32 == 0;
    p.fault = fault_word();
    if (p.fault == nullptr) return cudaErrorInvalidDevicePointer;
    CUtensorMap ma, mw;
    if (!encode_codes(&ma, g.a.codes, g.a.cols, g.a.rows, g.a.ld, 128) ||
        !encode_codes(&mw, g.w.codes, g.w.cols, g.w.rows, g.w.ld, 128))
        return cudaErrorInvalidValue;
    const size_t smem = (size_t)PairSmem::TOTAL + 1024;
    auto kern = fp8_gemm_pair_kernel<WT>;
    static std::atomic<int> ready[kMaxDevices];
    cudaError_t e = prepare_kernel(reinterpret_cast<const void*>(kern), smem, kPairLaunchRegs, ready);
    if (e != cudaSuccess) return e;
    const int tiles = p.tiles_m * p.tiles_n;
    const int pairs = sm_count() / 2;
    LaunchConfig cfg(dim3(2u * (unsigned)(tiles < pairs ? tiles : pairs)), kPairThreads, smem, s);
    return cudaLaunchKernelEx(&cfg.c, kern, p, ma, mw);
}

}  // namespace

size_t fp8_gemm_workspace_bytes(int64_t, int64_t, int64_t) { return 0; }

cudaError_t launch_fp8_gemm(const Fp8Gemm& g, void*, cudaStream_t s) {
    if (g.K == 0) {
        const int64_t n = (g.M * g.N + 255) / 256;
        const unsigned grid = (unsigned)(n < 65536 ? n : 65536);
        if (g.out_type == kF16)
            fill_rows_kernel<<<grid, 256, 0, s>>>(static_cast<__half*>(g.out), g.M, g.N, g.ldo, g.bias, g.bias_type);
        else if (g.out_type == kBf16)
            fill_rows_kernel<<<grid, 256, 0, s>>>(static_cast<__nv_bfloat16*>(g.out), g.M, g.N, g.ldo, g.bias,
                                                  g.bias_type);
        else
            fill_rows_kernel<<<grid, 256, 0, s>>>(static_cast<float*>(g.out), g.M, g.N, g.ldo, g.bias, g.bias_type);
        return cudaGetLastError();
    }
    return g.transpose ? launch_pair<true>(g, s) : launch_pair<false>(g, s);
}

}  // namespace wq
