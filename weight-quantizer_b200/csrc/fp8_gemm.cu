// The matrix product of blocks of 8-bit floating point.
//
//   y[m, n] = sum_b sa[m, b] sb[n / 128, b] sum_{k in block b} a[m, k] w[n, k] (+ bias[n])
//
// A block's sum over 128 products runs on the tensor cores (e4m3 x e4m3, fp32 in
// tensor memory); scales of any fp32 value cannot enter there (the block-scaled MMA
// takes powers of two alone), so each block's sum is read back and added to fp32
// registers, times the product of its two scales.
#include "fp8_types.cuh"
#include "kernels.h"
#include "tc_ptx.cuh"

#include "launch.h"

#include <type_traits>

namespace wq {
namespace {

// ---- large products: pairs of CTAs ------------------------------------------------
//
// A pair of CTAs (two SMs) makes a 256 x TN tile of y with tcgen05.mma of
// cta_group::2: each CTA holds 128 rows of a and half of the tile's columns of w in
// shared memory, and 128 rows x TN columns of a block's sums in tensor memory, as
// often as fit (TN = 256 twice, TN = 128 four times), so that the next blocks
// multiply while one is read back. Bytes from L2 per block and CTA at TN = 256: 32 KB
// for 128 x 256 x 128 products.
//
// What bounds it: a block's hand-off. At TN = 256 a block takes 775 cycles, 512 of
// them MMAs: a buffer is seen free by the issuer 230 cycles after its release, the
// issue takes 100, the MMAs' latency is 300 beyond their time, and reading the sums
// takes 320, with two buffers in flight. (Three buffers of 160 columns took the
// summing warps 600 cycles for each 160 columns, more per column; four of 128
// columns, which fill the SMs better when there are few tiles, take about 0.6 of the
// wide tile's time.) Long products at full width also reach the board's power limit:
// 4096 x 28672 x 8192 runs at 1.5 GHz and 990 W, 0.90 to 0.95 ms = 2.0 to 2.1 PFLOP/s.
//
// In each CTA warp 0 loads (TMA, 128-byte swizzle: a block of 128 codes is one
// swizzled row) and warp 3 copies the scales. Warps 1 and 2 of the even CTA issue the
// MMAs of both, alternate blocks: a wait on a barrier takes up to 200 cycles beside
// the MMAs' own reads of shared memory, so one warp would spend a block's time on its
// waits. Warps 4-11 of each CTA hold the sums: warp 4 + e reads tensor-memory lanes
// 32 (e % 4) .. + 31 (a lane is a row of y, so its scale is one value) and half of the
// columns (of one column block of w).
//
// The transposed weight needs no copy: rows of 128 codes along y's columns are the
// MMA's MN-major form of the same operand.

constexpr int kPairRows = 256;
constexpr int kPairScaleSlots = 3;                  // blocks whose scales are on their way
constexpr int kPairScaleBytes = (128 + 4) * 4;      // a's of the CTA's rows, w's of its two column blocks
constexpr int kOutBytes = 4096;                     // a summing warp's part of y on its way out
constexpr int kOperandBytes = 128 * 128;            // one operand of one CTA for one block
constexpr int kPairThreads = 384;
constexpr int kPairLaunchRegs = 168, kPairCtlRegs = 56, kPairSumRegs = 224;
static_assert(kPairCtlRegs + 2 * kPairSumRegs <= 3 * kPairLaunchRegs, "register split exceeds the launch's registers");

// TN columns of y per tile: 256, or 128 where that fills the SMs better.
template <bool WT, int TN>
struct PairSmem {
    // a CTA's columns of w for one block: rows of 128 codes, or, of the transposed
    // weight, 128 rows of the 128 codes that a box of the swizzle holds (64 of them
    // used by the narrow tile)
    static constexpr int W_ROWS = WT ? 128 : TN / 2;
    static constexpr int STAGE = kOperandBytes + W_ROWS * 128;
    static constexpr int STAGES = STAGE > 24576 ? 6 : 8;   // even: each issuing warp has its own
    static constexpr int BUFS = 512 / TN;                  // even likewise
    static_assert(BUFS <= STAGES, "a stage's barrier would lap the summing warps");
    static constexpr int OUT = STAGES * STAGE;
    static constexpr int SCALES = OUT + 8 * kOutBytes;
    static constexpr int BAR = SCALES + kPairScaleSlots * kPairScaleBytes;
    // full and done per stage (done: the block's MMAs are over, so its operands
    // may be replaced and its sums read); sums empty per buffer; per scale slot
    // there, read
    static constexpr int TMEM_SLOT = BAR + 8 * (2 * STAGES + BUFS + 2 * kPairScaleSlots);
    static constexpr int FLAG = TMEM_SLOT + 8;
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
    int64_t ldo;
    int M, N, blocks;        // inner blocks of 128
    int tiles_m, tiles_n, band;
    bool tma_out;            // rows of out are 16-byte aligned
    int splits;              // parts of the inner blocks, each a tile's work for a pair of its own
    float* part;             // [tile][split][rank] sums of 128 x TN
    unsigned int* arrived;   // [tile][rank], zeroed before the launch
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

template <typename O>
__device__ __forceinline__ O ld_shared(uint32_t at) {
    if constexpr (sizeof(O) == 4) {
        uint32_t v;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
        return *reinterpret_cast<const O*>(&v);
    } else {
        uint16_t v;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at) : "memory");
        return *reinterpret_cast<const O*>(&v);
    }
}

// A warp's 32 rows (from m0) x C columns (from n0) of y out of its sums: a lane is
// a row. By way of shared memory (128 bytes of 32 rows at a time, swizzled) and a TMA
// store that ends at y's edges and drains while the next tile's blocks are summed:
// stores from registers held the tile's hand-off for 4300 cycles, every CTA's 64 KB
// at once.
template <typename O, int C>
__device__ __forceinline__ void put_tile(const PairParams& p, const CUtensorMap* map, uint32_t out, int lane,
                                         int64_t m0, int64_t n0, const uint64_t (&acc)[C / 2]) {
    constexpr int PER = 16 / (int)sizeof(O);      // values in 16 bytes
    constexpr int BOX = 8 * PER;                  // columns in 128 bytes
    const bool has_bias = p.bias != nullptr;
    auto value = [&](int c) {
        const float2 f = unpack2(acc[c / 2]);
        float v = c & 1 ? f.y : f.x;
        if (has_bias && n0 + c < p.N) v += load_any(p.bias, p.bias_type, n0 + c);
        return from_f32<O>(v);
    };
    auto stage = [&](int c0) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            uint32_t w[4];
            O e[PER];
#pragma unroll
            for (int j = 0; j < PER; ++j) e[j] = value(c0 + k * PER + j);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = reinterpret_cast<const uint32_t*>(e)[j];
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(out + lane * 128 + ((k ^ (lane & 7)) << 4)),
                         "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                         : "memory");
        }
    };
    if (p.tma_out) {
#pragma unroll
        for (int c0 = 0; c0 < C; c0 += BOX) {
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
            stage(c0);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                if (m0 < p.M && n0 + c0 < p.N) tma_store(map, (int)(n0 + c0), (int)m0, out);
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
        }
    } else {
        // rows that TMA cannot write: a row's neighbouring columns by the warp (single
        // elements of 32 rows per store took 416 us at 4096 x 11007 x 256, these 48)
        const int rows = (int)(p.M - m0 < 32 ? p.M - m0 : 32);
#pragma unroll
        for (int c0 = 0; c0 < C; c0 += BOX) {
            __syncwarp();
            stage(c0);
            __syncwarp();
            O* at = static_cast<O*>(p.out) + m0 * p.ldo + n0 + c0 + lane;
#pragma unroll 8
            for (int r = 0; r < rows; ++r, at += p.ldo) {
#pragma unroll
                for (int h = 0; h < BOX; h += 32) {
                    const int c = h + lane;
                    const O v = ld_shared<O>(out + r * 128 + (((c / PER) ^ (r & 7)) << 4) + c % PER * (int)sizeof(O));
                    if (n0 + c0 + c < p.N) at[h] = v;
                }
            }
        }
    }
}

template <bool WT, bool SPLIT, int TN, typename O>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    fp8_gemm_pair_kernel(const PairParams p, const __grid_constant__ CUtensorMap map_a,
                         const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_y) {
    using L = PairSmem<WT, TN>;
    constexpr int NS = L::STAGES, NB = L::BUFS, C = TN / 2;   // C: columns of w of one CTA, and of a summing warp
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_addr(smem);
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // uniform
    const int rank = (int)cluster_rank();
    auto bar = [&](int i) -> uint32_t { return sbase + L::BAR + 8u * (uint32_t)i; };
    auto full = [&](int s) { return bar(s); };
    auto done = [&](int s) { return bar(NS + s); };
    auto sums_empty = [&](int b) { return bar(2 * NS + b); };
    auto scaled = [&](int c) { return bar(2 * NS + NB + c); };
    auto scales_read = [&](int c) { return bar(2 * NS + NB + kPairScaleSlots + c); };
    launch_dependents();
    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(full(s), 1);     // the even CTA's: its own arrival plus both CTAs' bytes
            mbar_init(done(s), 1);
        }
        for (int b = 0; b < NB; ++b)
            mbar_init(sums_empty(b), 16);   // the even CTA's: one arrival per summing warp of the pair
        for (int c = 0; c < kPairScaleSlots; ++c) {
            mbar_init(scaled(c), 32);
            mbar_init(scales_read(c), 8);
        }
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
    // items of work: tiles, or parts of their inner blocks
    const int splits = SPLIT ? p.splits : 1;
    const int items = p.tiles_m * p.tiles_n * splits;
    auto from_block = [&](int item) { return SPLIT ? item % splits * p.blocks / splits : 0; };
    auto to_block = [&](int item) { return SPLIT ? (item % splits + 1) * p.blocks / splits : p.blocks; };
    int64_t steps = 0;
    for (int i = first; i < items; i += pairs) steps += to_block(i) - from_block(i);
    bool faulted = false;
    auto give_up = [&]() {
        faulted = true;
        atomicOr(p.fault, 1u);
    };

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPairCtlRegs));
        if (warp == 0) {
            // each CTA loads its 128 rows of a and its columns of w; the
            // bytes count on the even CTA's barrier
            const uint32_t full0 = in_cta(full(0), 0);
            int s = 0;
            uint32_t ph = 1;
            for (int t = first; t < items; t += pairs) {
                int mt, nt;
                tile_of(t / splits, p, mt, nt);
                const int m0 = mt * kPairRows + rank * 128, n0 = nt * TN + rank * C;
                const int b1 = to_block(t);
                for (int b = from_block(t); b < b1; ++b) {
                    if (!faulted && !mbar_wait_bounded(done(s), ph)) give_up();
                    __syncwarp();
                    if (elect_one()) {
                        const uint32_t f = full0 + 8u * (uint32_t)s;
                        const uint32_t dst = sbase + (uint32_t)(s * L::STAGE);
                        if (rank == 0) mbar_arrive_expect_tx(full(s), 2 * L::STAGE);
                        tma_box<2>(dst, &map_a, b * 128, m0, f);
                        if constexpr (WT) tma_box<2>(dst + kOperandBytes, &map_w, n0, b * 128, f);
                        else tma_box<2>(dst + kOperandBytes, &map_w, b * 128, n0, f);
                    }
                    __syncwarp();
                    if (++s == NS) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
            }
            // every copy this warp started has been read before the CTA goes
            // (a stage that was never filled passes at once)
            for (int i = 0; i < NS; ++i) {
                if (!mbar_wait_bounded(done(s), ph)) atomicOr(p.fault, 1u);
                if (++s == NS) {
                    s = 0;
                    ph ^= 1u;
                }
            }
        } else if ((warp == 1 || warp == 2) && rank == 0) {
            // even blocks by warp 1, odd ones by warp 2: a wait on a barrier takes
            // about 170 cycles beside the MMAs' own reads of shared memory, and one
            // warp's waits and its issue together take as long as a block's MMAs
            constexpr uint32_t idesc = mma_idesc(0, false, WT, kPairRows, TN);
            const uint64_t desc0 = sw128_matrix(sbase);
            int s = warp - 1, buf = warp - 1;
            uint32_t ph = 0, free_ph = 1;   // (a fresh barrier's other phase counts as complete)
            for (int64_t i = warp - 1; i < steps; i += 2) {
                const uint64_t da = desc0 + (uint64_t)(s * (L::STAGE >> 4));
                const uint64_t dw = da + (uint64_t)(kOperandBytes >> 4);
                if (!try_wait_both(full(s), ph, sums_empty(buf), free_ph)) {
                    if (!faulted && !mbar_wait_bounded(full(s), ph)) give_up();
                    if (!faulted && !mbar_wait_bounded(sums_empty(buf), free_ph)) give_up();
                }
                __syncwarp();
                tc_after();
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)   // 32 codes: 32 bytes of a row, or 32 rows of 128 bytes
                        mma_f8<2>(tmem + (uint32_t)(buf * TN), da + 2u * k, dw + (WT ? 256u : 2u) * k, idesc, k > 0);
                    mma_done<2>(done(s));
                }
                __syncwarp();
                s += 2;
                if (s >= NS) {
                    s -= NS;
                    ph ^= 1u;
                }
                buf += 2;
                if (buf >= NB) {
                    buf -= NB;
                    free_ph ^= 1u;
                }
            }
        } else if (warp == 3) {
            // each block's scales, by asynchronous copies (loaded into registers by the
            // summing warps they were waited for: three blocks ahead was too late for
            // scales that come from memory, and more cost registers)
            int c = 0;
            uint32_t ph = 1;
            for (int t = first; t < items; t += pairs) {
                int mt, nt;
                tile_of(t / splits, p, mt, nt);
                const int64_t m0 = (int64_t)mt * kPairRows + rank * 128 + lane;
                const int b0 = from_block(t), b1 = to_block(t);
                const float* sa = p.sa + m0 * p.sa_row + b0 * p.sa_col;
                const float* sw = p.sw + min((nt * TN + (lane & 1) * C) >> 7, (p.N - 1) >> 7) * p.sw_n + b0 * p.sw_k;
                for (int b = b0; b < b1; ++b) {
                    if (!faulted && !mbar_wait_bounded(scales_read(c), ph)) give_up();
                    __syncwarp();
                    const uint32_t to = sbase + (uint32_t)(L::SCALES + c * kPairScaleBytes);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const bool some = m0 + 32 * j < p.M;   // rows beyond the last: 0
                        cp_async4_s(to + (32 * j + lane) * 4, some ? sa + 32 * j * p.sa_row : p.sa, some);
                    }
                    if (lane < 2) cp_async4_s(to + (128 + lane) * 4, sw, true);
                    cp_async_arrive(scaled(c));
                    sa += p.sa_col;
                    sw += p.sw_k;
                    if (++c == kPairScaleSlots) {
                        c = 0;
                        ph ^= 1u;
                    }
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPairSumRegs));
        const int q = warp & 3, half = (warp - 4) >> 2;
        const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(half * C);
        const uint32_t free0 = in_cta(sums_empty(0), 0);
        int s = 0, c = 0;
        int64_t i = 0;
        uint32_t ph = 0, cph = 0;
        for (int t = first; t < items; t += pairs) {
            const int b0 = from_block(t), b1 = to_block(t);
            uint64_t acc[C / 2];
#pragma unroll
            for (int k = 0; k < C / 2; ++k) acc[k] = 0;
            for (int b = b0; b < b1; ++b) {
                if (!try_wait_both(done(s), ph, scaled(c), cph)) {
                    if (!faulted && !mbar_wait_bounded(scaled(c), cph)) give_up();
                    if (!faulted && !mbar_wait_bounded(done(s), ph)) give_up();
                }
                const int buf = (int)(i & (NB - 1));
                __syncwarp();
                tc_after();
                const float* scales = reinterpret_cast<const float*>(smem + L::SCALES + c * kPairScaleBytes);
                const float sc = scales[q * 32 + lane] * scales[128 + half];
                const uint64_t sc2 = pack2(sc, sc);
                const uint32_t from = taddr + (uint32_t)(buf * TN);
                uint64_t v[32];
                tmem_pairs(from, v);
                if constexpr (C == 128) {   // 64 columns at a time, for the registers
#pragma unroll
                    for (int k = 0; k < 32; ++k) fma2(acc[k], v[k], sc2);
                    tmem_pairs(from + 64u, v);
                }
                tc_before();
                __syncwarp();
                if (lane == 0) {
                    arrive_in_cluster(free0 + 8u * (uint32_t)buf);
                    mbar_arrive(scales_read(c));
                }
#pragma unroll
                for (int k = 0; k < 32; ++k) fma2(acc[C / 2 - 32 + k], v[k], sc2);
                ++i;
                if (++s == NS) {
                    s = 0;
                    ph ^= 1u;
                }
                if (++c == kPairScaleSlots) {
                    c = 0;
                    cph ^= 1u;
                }
            }
            bool write = true;
            if constexpr (SPLIT) {
                // the item's sums go to its slot, [column / 4][row][4]; the last of the
                // tile's items adds them in order
                const int64_t lane_at = ((int64_t)half * (C / 4) * 128 + q * 32 + lane) * 4;
                constexpr int64_t SLOT = 128 * TN;
                float4* mine = reinterpret_cast<float4*>(p.part + ((int64_t)t * 2 + rank) * SLOT + lane_at);
#pragma unroll
                for (int k = 0; k < C / 4; ++k) {
                    const float2 f = unpack2(acc[2 * k]), g = unpack2(acc[2 * k + 1]);
                    mine[k * 128] = make_float4(f.x, f.y, g.x, g.y);
                }
                named_barrier(1, 256);
                volatile uint32_t* flag = reinterpret_cast<volatile uint32_t*>(smem + L::FLAG);
                const int tile = t / splits;
                if (warp == 4 && lane == 0)
                    *flag = last_to_arrive(p.arrived + tile * 2 + rank, (unsigned)splits);
                named_barrier(1, 256);
                write = *flag != 0u;
                named_barrier(1, 256);   // the flag has been read
                if (write) {
#pragma unroll
                    for (int k = 0; k < C / 2; ++k) acc[k] = 0;
                    const uint64_t one = pack2(1.0f, 1.0f);
#pragma unroll 1
                    for (int sp = 0; sp < splits; ++sp) {
                        const float4* src = reinterpret_cast<const float4*>(
                            p.part + (((int64_t)tile * splits + sp) * 2 + rank) * SLOT + lane_at);
#pragma unroll
                        for (int k = 0; k < C / 4; ++k) {
                            const float4 f = __ldcg(src + k * 128);
                            fma2(acc[2 * k], pack2(f.x, f.y), one);
                            fma2(acc[2 * k + 1], pack2(f.z, f.w), one);
                        }
                    }
                }
            }
            int mt, nt;
            tile_of(t / splits, p, mt, nt);
            if (write)
                put_tile<O, C>(p, &map_y, sbase + (uint32_t)(L::OUT + (warp - 4) * kOutBytes), lane,
                            (int64_t)mt * kPairRows + rank * 128 + q * 32, (int64_t)nt * TN + half * C, acc);
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    cluster_sync();   // the pair's MMAs, arrivals and reads of tensor memory are over
    tc_after();
    if (warp == 1) tmem_free<2>(tmem, 512);
}

// ---- few rows: weights stream by, the work split evenly ------------------------------
//
// With few rows of a the bound is the weights' bytes (and, once they are in L2, the
// latency of each block). The MMA's rows (tensor-memory lanes) are 128 rows of w, its
// columns `bn` <= BN rows of a. The work is cut into units of 128 rows of w x one
// block, and every CTA takes an equal run of them, wherever tiles begin or end (224
// row tiles on 148 SMs would leave a quarter of them idle in the second round). A CTA
// that holds a whole tile writes y; the others put their sums into the workspace, and
// the last to arrive at a tile adds them in CTA order (a fixed order, whoever is last)
// and writes y.
//
// Two CTAs per SM for up to 32 rows, each with a ring of four units, one with eight
// for more: 148-192 KB in flight per SM either way. Warp 0 loads units (TMA) into the
// ring; warps 1 and 2 issue the MMAs of even and odd units; warp 3 copies the unit's
// scales (asynchronous 4-byte copies); the other warps add each unit's sums, times
// the scales, to registers. As many units' sums as the ring has stages fit in tensor
// memory, so no hand-off waits for another.
//
// One row through 28672 x 8192: 46.4 us; reading its 235 MB takes 35.9 us at the
// measured copy rate, and this ring of TMA loads without the products 37-41 us.

template <int BN>
struct Few {
    static constexpr int COLS = BN < 32 ? BN : 32;              // columns per summing warp
    static constexpr int SUM_WARPS = 4 * (BN / COLS);
    static constexpr int THREADS = 128 + 32 * SUM_WARPS;
    static constexpr int STAGE = kOperandBytes + BN * 128;
    // With few columns two CTAs share an SM: one's beginning and end (the first loads,
    // the partial sums) run beside the other's stream.
    static constexpr int CTAS = BN > 32 ? 1 : 2;
    static constexpr int STAGES = 206 * 1024 / CTAS / STAGE / 2 * 2;   // even likewise
    // Tensor-memory buffers: even, and no more than stages: a stage's barrier must not
    // complete twice before the summing warps have seen it once.
    static constexpr int BUFS = STAGES < 8 ? STAGES : 8;
    static_assert(BUFS <= STAGES, "a stage's barrier would lap the summing warps");
    static constexpr uint32_t TMEM = BUFS * BN;
    static constexpr int SCALES = STAGES * STAGE;               // per buffer BN of a, one of w
    static constexpr int SCALE_BYTES = (BN + 4) * 4;
    static constexpr int BAR = SCALES + BUFS * SCALE_BYTES;
    // full, done per stage; scales there, sums empty per buffer
    static constexpr int TMEM_SLOT = BAR + 8 * (2 * STAGES + 2 * BUFS);
    static_assert((TMEM & (TMEM - 1)) == 0 && TMEM >= 32 && TMEM * CTAS <= 512, "tensor memory is handed out in powers of two");
    static constexpr int FLAG = TMEM_SLOT + 8;
    static constexpr int TOTAL = TMEM_SLOT + 16;
    static_assert((TOTAL + 1024 + 1024) * CTAS <= 228 * 1024, "stages exceed the shared memory of an SM");
};

struct FewParams {
    const float* sa;
    int64_t sa_row, sa_col;
    const float* sw;
    int64_t sw_n, sw_k;
    const void* bias;
    int bias_type;
    void* out;
    int64_t ldo;
    int M, N, blocks;
    int bn;                  // rows of a in the MMA: M in steps of 16
    int64_t units;
    float* part;             // two slots of 128 x BN sums per CTA
    unsigned int* arrived;   // per tile, zeroed before the launch
    bool weights_ready;      // w was complete before the previous kernel let this one start
    unsigned int* fault;
};

__device__ __forceinline__ int64_t first_unit(int64_t cta, int64_t units, int64_t ctas) { return cta * units / ctas; }
__device__ __forceinline__ int64_t cta_of(int64_t unit, int64_t units, int64_t ctas) {
    return ((unit + 1) * ctas - 1) / units;
}

template <int BN, bool WT, typename O>
__global__ void __launch_bounds__(Few<BN>::THREADS, Few<BN>::CTAS)
    fp8_gemm_few_kernel(const FewParams p, const __grid_constant__ CUtensorMap map_a,
                        const __grid_constant__ CUtensorMap map_w) {
    using L = Few<BN>;
    constexpr int NS = L::STAGES, NB = L::BUFS;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_addr(smem);
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // uniform
    auto bar = [&](int i) -> uint32_t { return sbase + L::BAR + 8u * (uint32_t)i; };
    auto full = [&](int s) { return bar(s); };
    auto done = [&](int s) { return bar(NS + s); };
    auto scaled = [&](int b) { return bar(2 * NS + b); };
    auto sums_empty = [&](int b) { return bar(2 * NS + NB + b); };
    launch_dependents();
    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(full(s), 1);
            mbar_init(done(s), 1);
        }
        for (int b = 0; b < NB; ++b) {
            mbar_init(scaled(b), 32);
            mbar_init(sums_empty(b), L::SUM_WARPS);
        }
        fence_mbarrier_init();
    }
    if (warp == 1) tmem_alloc<1>(sbase + L::TMEM_SLOT, L::TMEM);
    tc_before();
    __syncthreads();
    tc_after();
    if (!p.weights_ready || warp != 0) grid_wait();   // nothing above reads global memory
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + L::TMEM_SLOT);
    const int64_t u0 = first_unit(blockIdx.x, p.units, gridDim.x), u1 = first_unit(blockIdx.x + 1, p.units, gridDim.x);
    bool faulted = false;
    auto wait = [&](uint32_t b, uint32_t parity) {
        if (!faulted && !mbar_wait_bounded(b, parity)) {
            faulted = true;
            atomicOr(p.fault, 1u);
        }
    };

    if (warp == 0) {
        const uint32_t bytes = (uint32_t)(kOperandBytes + p.bn * 128);
        int tile = (int)(u0 / p.blocks), b = (int)(u0 - (int64_t)tile * p.blocks);
        auto load_w = [&](int s, int tile, int b) {
            const int r0 = tile * 128;
            mbar_arrive_expect_tx(full(s), bytes);
            if constexpr (WT) tma_box<1>(sbase + (uint32_t)(s * L::STAGE), &map_w, r0, b * 128, full(s));
            else tma_box<1>(sbase + (uint32_t)(s * L::STAGE), &map_w, b * 128, r0, full(s));
        };
        auto load_a = [&](int s, int b) {
            tma_box<1>(sbase + (uint32_t)(s * L::STAGE + kOperandBytes), &map_a, b * 128, 0, full(s));
        };
        // the first round's weights may come before the previous kernel (which makes
        // a's codes) is over
        const int ahead = p.weights_ready ? (int)min((int64_t)NS, u1 - u0) : 0;
        {
            int t = tile, c = b;
            for (int s = 0; s < ahead; ++s) {
                if (elect_one()) load_w(s, t, c);
                __syncwarp();
                if (++c == p.blocks) c = 0, ++t;
            }
        }
        if (p.weights_ready) grid_wait();
        int s = 0;
        uint32_t ph = 1;
        for (int64_t u = u0; u < u1; ++u) {
            const bool loaded = u - u0 < ahead;
            if (!loaded) wait(done(s), ph);
            __syncwarp();
            if (elect_one()) {
                if (!loaded) load_w(s, tile, b);
                load_a(s, b);
            }
            __syncwarp();
            if (++b == p.blocks) b = 0, ++tile;
            if (++s == NS) {
                s = 0;
                ph ^= 1u;
            }
        }
        // every copy this warp started has been read before the CTA goes
        // (a stage that was never filled passes at once)
        for (int i = 0; i < NS; ++i) {
            if (!mbar_wait_bounded(done(s), ph)) atomicOr(p.fault, 1u);
            if (++s == NS) {
                s = 0;
                ph ^= 1u;
            }
        }
    } else if (warp < 3) {
        const uint32_t idesc = mma_idesc(0, WT, false, 128, p.bn);
        const uint64_t desc0 = sw128_matrix(sbase);
        int s = warp - 1, buf = warp - 1;
        uint32_t ph = 0, bph = 1;
        for (int64_t u = u0 + warp - 1; u < u1; u += 2) {
            if (!try_wait_both(full(s), ph, sums_empty(buf), bph)) {
                wait(full(s), ph);
                wait(sums_empty(buf), bph);
            }
            __syncwarp();
            tc_after();
            if (elect_one()) {
                const uint64_t dw = desc0 + (uint64_t)(s * (L::STAGE >> 4));
                const uint64_t da = dw + (uint64_t)(kOperandBytes >> 4);
#pragma unroll
                for (int k = 0; k < 4; ++k)   // 32 codes: 32 bytes of a row, or 32 rows of 128 bytes
                    mma_f8<1>(tmem + (uint32_t)(buf * BN), dw + (WT ? 256u : 2u) * k, da + 2u * k, idesc, k > 0);
                mma_done<1>(done(s));
            }
            __syncwarp();
            s += 2;
            if (s >= NS) {
                s -= NS;
                ph ^= 1u;
            }
            buf += 2;
            if (buf >= NB) {
                buf -= NB;
                bph ^= 1u;
            }
        }
    } else if (warp == 3) {
        // scales of the unit's block: a's rows of the tile (beyond the last: 0), and w's
        int tile = (int)(u0 / p.blocks), b = (int)(u0 - (int64_t)tile * p.blocks);
        int buf = 0;
        uint32_t bph = 1;
        for (int64_t u = u0; u < u1; ++u) {
            wait(sums_empty(buf), bph);
            __syncwarp();
            const uint32_t to = sbase + (uint32_t)(L::SCALES + buf * L::SCALE_BYTES);
#pragma unroll
            for (int i = 0; i < (BN + 31) / 32; ++i) {
                const int c = i * 32 + lane;
                const bool some = c < p.M;
                if (c < BN) cp_async4_s(to + c * 4, some ? p.sa + c * p.sa_row + b * p.sa_col : p.sa, some);
            }
            if (lane == 0) cp_async4_s(to + BN * 4, p.sw + tile * p.sw_n + b * p.sw_k, true);
            cp_async_arrive(scaled(buf));
            if (++b == p.blocks) b = 0, ++tile;
            if (++buf == NB) {
                buf = 0;
                bph ^= 1u;
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
        const int q = warp & 3, half = (warp - 4) >> 2;
        const int row = q * 32 + lane;
        constexpr int C = L::COLS;
        const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(half * C);
        int s = 0, buf = 0;
        uint32_t ph = 0, bph = 0;
        int64_t u = u0;
        while (u < u1) {
            // the part of a tile that this CTA holds
            const int tile = (int)(u / p.blocks);
            const int64_t t0 = (int64_t)tile * p.blocks, t1 = t0 + p.blocks;
            const int64_t from = u, to = min(u1, t1);
            uint64_t acc[C / 2];
#pragma unroll
            for (int c = 0; c < C / 2; ++c) acc[c] = 0;
            for (; u < to; ++u) {
                if (!try_wait_both(done(s), ph, scaled(buf), bph)) {
                    wait(done(s), ph);
                    wait(scaled(buf), bph);
                }
                __syncwarp();
                tc_after();
                const float* sc = reinterpret_cast<const float*>(smem + L::SCALES + buf * L::SCALE_BYTES);
                const float w = sc[BN];
                const uint64_t w2 = pack2(w, w);
                uint64_t by[C / 2];
#pragma unroll
                for (int c = 0; c < C / 4; ++c) {
                    const float4 f = *reinterpret_cast<const float4*>(sc + half * C + 4 * c);
                    by[2 * c] = mul2(pack2(f.x, f.y), w2);
                    by[2 * c + 1] = mul2(pack2(f.z, f.w), w2);
                }
                uint64_t v[C / 2];
                tmem_pairs(taddr + (uint32_t)(buf * BN), v);
#pragma unroll
                for (int c = 0; c < C / 2; ++c) fma2(acc[c], v[c], by[c]);
                tc_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(sums_empty(buf));
                if (++s == NS) {
                    s = 0;
                    ph ^= 1u;
                }
                if (++buf == NB) {
                    buf = 0;
                    bph ^= 1u;
                }
            }
            float4 y[C / 4];
#pragma unroll
            for (int c = 0; c < C / 4; ++c) {
                const float2 f = unpack2(acc[2 * c]), g = unpack2(acc[2 * c + 1]);
                y[c] = make_float4(f.x, f.y, g.x, g.y);
            }
            bool write = true;
            if (from != t0 || to != t1) {
                // slot [column / 4][row][4]: 16 bytes per lane, lanes side by side
                const int64_t ctas = gridDim.x;
                const int64_t lane_at = (half * (C / 4) * 128 + row) * 4;
                float4* mine = reinterpret_cast<float4*>(
                    p.part + (2 * (int64_t)blockIdx.x + (from == u0 ? 0 : 1)) * (128 * BN) + lane_at);
#pragma unroll
                for (int c = 0; c < C / 4; ++c) mine[c * 128] = y[c];
                named_barrier(1, 32 * L::SUM_WARPS);
                volatile uint32_t* flag = reinterpret_cast<volatile uint32_t*>(smem + L::FLAG);
                const int64_t c0 = cta_of(t0, p.units, ctas), c1 = cta_of(t1 - 1, p.units, ctas);
                if (warp == 4 && lane == 0) *flag = last_to_arrive(p.arrived + tile, (unsigned)(c1 - c0 + 1));
                named_barrier(1, 32 * L::SUM_WARPS);
                write = *flag != 0u;
                named_barrier(1, 32 * L::SUM_WARPS);   // the flag has been read
                if (write) {
#pragma unroll
                    for (int c = 0; c < C / 4; ++c) y[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    // (several CTAs' sums are on their way at once)
                    constexpr int AHEAD = C > 16 ? 1 : 3;
#pragma unroll 1
                    for (int64_t cta = c0; cta <= c1; cta += AHEAD) {
                        float4 part[AHEAD][C / 4];
#pragma unroll
                        for (int j = 0; j < AHEAD; ++j) {
                            if (cta + j <= c1) {
                                const int64_t b = first_unit(cta + j, p.units, ctas);
                                const float4* src = reinterpret_cast<const float4*>(
                                    p.part + (2 * (cta + j) + (b >= t0 ? 0 : 1)) * (128 * BN) + lane_at);
#pragma unroll
                                for (int c = 0; c < C / 4; ++c) part[j][c] = __ldcg(src + c * 128);
                            }
                        }
#pragma unroll
                        for (int j = 0; j < AHEAD; ++j) {
                            if (cta + j <= c1) {
#pragma unroll
                                for (int c = 0; c < C / 4; ++c) {
                                    y[c].x += part[j][c].x;
                                    y[c].y += part[j][c].y;
                                    y[c].z += part[j][c].z;
                                    y[c].w += part[j][c].w;
                                }
                            }
                        }
                    }
                }
            }
            const int n = tile * 128 + row;
            if (write && n < p.N) {
                const float bias = load_any(p.bias, p.bias_type, n);
                const int cols = min(C, p.M - half * C);
                O* at = static_cast<O*>(p.out) + (int64_t)half * C * p.ldo + n;
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const float4 f = y[c / 4];
                    const float v = c % 4 == 0 ? f.x : (c % 4 == 1 ? f.y : (c % 4 == 2 ? f.z : f.w));
                    if (c < cols) *at = from_f32<O>(v + bias);
                    at += p.ldo;
                }
            }
        }
    }
    tc_before();
    __syncthreads();
    tc_after();
    if (warp == 1) tmem_free<1>(tmem, L::TMEM);
}

// ---- host side ------------------------------------------------------------------------

// y = bias, or 0, in every row: a product without inner values.
template <typename O>
__global__ void fill_rows_kernel(O* out, int64_t M, int64_t N, int64_t ldo, const void* bias, int bias_type) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < M * N; i += (int64_t)gridDim.x * blockDim.x)
        out[i / N * ldo + i % N] = from_f32<O>(load_any(bias, bias_type, i % N));
}

// ---- plan ----

size_t round_up(size_t v) { return (v + 255) / 256 * 256; }
int64_t pair_tiles(int64_t M, int64_t N, int tn) { return ((M + kPairRows - 1) / kPairRows) * ((N + tn - 1) / tn); }
// The tile's columns, the parts that its inner blocks are cut into, and the time, in
// microseconds, by a model fitted to both on weights of 2304 x 768 to 28672 x 8192 at
// 65 to 4096 rows: 5, kWideUs or kNarrowUs for each round of blocks over the pairs of
// SMs (or the weights at 5.5 TB/s, if that is longer), and 16 + 2 for each part that
// a tile's blocks are cut into (at least four blocks, one pair each) where there are
// at most half as many tiles as pairs.
constexpr double kWideUs = 0.43, kNarrowUs = 0.26;
struct PairPlan {
    int tn, splits;
    double us;
};
PairPlan pair_plan(int64_t M, int64_t N, int64_t K) {
    const int64_t pairs = sm_count() / 2, blocks = (K + 127) / 128;
    const double stream = (double)N * (double)K / 5.5e6;
    PairPlan best{256, 1, 1e30};
    for (int tn = 256; tn >= 128; tn -= 128) {
        const int64_t tiles = pair_tiles(M, N, tn);
        int64_t most = pairs / tiles;
        if (most > blocks / 4) most = blocks / 4;
        if (most > 8) most = 8;
        for (const int64_t n : {(int64_t)1, most < 1 ? (int64_t)1 : most}) {
            const int64_t rounds = (tiles * n + pairs - 1) / pairs;
            const double run = (double)(rounds * ((blocks + n - 1) / n)) * (tn == 256 ? kWideUs : kNarrowUs);
            const double us = 5.0 + (run > stream ? run : stream) + (n > 1 ? 16.0 + 2.0 * (double)n : 0.0);
            if (us < best.us) best = PairPlan{tn, (int)n, us};
        }
    }
    return best;
}
size_t pair_arrived_bytes(int64_t M, int64_t N, int64_t K) {
    return round_up((size_t)pair_tiles(M, N, pair_plan(M, N, K).tn) * 2 * 4);
}
size_t pair_part_bytes(int64_t M, int64_t N, int64_t K) {
    const PairPlan plan = pair_plan(M, N, K);
    return (size_t)pair_tiles(M, N, plan.tn) * plan.splits * 2 * 128 * plan.tn * 4;
}

template <bool WT, bool SPLIT, int TN, typename O>
cudaError_t launch_pair_o(const Fp8Gemm& g, int splits, void* workspace, cudaStream_t s) {
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
    p.ldo = g.ldo;
    p.M = (int)g.M;
    p.N = (int)g.N;
    p.blocks = (int)((g.K + 127) / 128);
    p.tiles_m = (int)((g.M + kPairRows - 1) / kPairRows);
    p.tiles_n = (int)((g.N + TN - 1) / TN);
    // the rows of a band stay below 40 MB, well inside L2
    const int64_t per_tile = (int64_t)kPairRows * p.blocks * 128;
    int64_t band = ((int64_t)40 << 20) / per_tile;
    band = band < 1 ? 1 : band;
    const int64_t bands = (p.tiles_m + band - 1) / band;
    p.band = (int)((p.tiles_m + bands - 1) / bands);
    p.splits = splits;
    p.arrived = static_cast<unsigned int*>(workspace);
    p.part = SPLIT ? reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + pair_arrived_bytes(g.M, g.N, g.K))
                   : nullptr;
    p.fault = fault_word();
    if (p.fault == nullptr) return cudaErrorInvalidDevicePointer;
    CUtensorMap ma, mw, my = {};
    if (!encode_codes(&ma, g.a.codes, g.a.cols, g.a.rows, g.a.ld, 128) ||
        !encode_codes(&mw, g.w.codes, g.w.cols, g.w.rows, g.w.ld, PairSmem<WT, TN>::W_ROWS))
        return cudaErrorInvalidValue;
    constexpr CUtensorMapDataType DT = sizeof(O) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                       : std::is_same<O, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                        : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const int64_t out_pitch = g.M > 1 ? g.ldo * (int64_t)sizeof(O) : (g.N * (int64_t)sizeof(O) + 15) / 16 * 16;
    p.tma_out = (reinterpret_cast<uintptr_t>(g.out) & 15) == 0 && out_pitch % 16 == 0 &&
                encode_rows(&my, DT, (int)sizeof(O), g.out, g.N, g.M, out_pitch, 32);
    const size_t smem = (size_t)PairSmem<WT, TN>::TOTAL + 1024;
    auto kern = fp8_gemm_pair_kernel<WT, SPLIT, TN, O>;
    static std::atomic<int> ready[kMaxDevices];
    cudaError_t e = prepare_kernel(reinterpret_cast<const void*>(kern), smem, kPairLaunchRegs, ready);
    if (e != cudaSuccess) return e;
    const int64_t items = (int64_t)p.tiles_m * p.tiles_n * splits;
    const int64_t pairs = sm_count() / 2;
    if (items > 0x7fffffff) return cudaErrorInvalidValue;
    LaunchConfig cfg(dim3(2u * (unsigned)(items < pairs ? items : pairs)), kPairThreads, smem, s);
    return cudaLaunchKernelEx(&cfg.c, kern, p, ma, mw, my);
}

template <bool WT, bool SPLIT, int TN>
cudaError_t launch_pair_s(const Fp8Gemm& g, int splits, void* workspace, cudaStream_t s) {
    if (g.out_type == kF16) return launch_pair_o<WT, SPLIT, TN, __half>(g, splits, workspace, s);
    if (g.out_type == kBf16) return launch_pair_o<WT, SPLIT, TN, __nv_bfloat16>(g, splits, workspace, s);
    return launch_pair_o<WT, SPLIT, TN, float>(g, splits, workspace, s);
}

template <bool WT>
cudaError_t launch_pair(const Fp8Gemm& g, void* workspace, bool prepared, cudaStream_t s) {
    const PairPlan plan = pair_plan(g.M, g.N, g.K);
    if (plan.splits == 1)
        return plan.tn == 256 ? launch_pair_s<WT, false, 256>(g, 1, nullptr, s)
                              : launch_pair_s<WT, false, 128>(g, 1, nullptr, s);
    if (!prepared) {
        cudaError_t e = cudaMemsetAsync(workspace, 0, pair_arrived_bytes(g.M, g.N, g.K), s);
        if (e != cudaSuccess) return e;
    }
    return plan.tn == 256 ? launch_pair_s<WT, true, 256>(g, plan.splits, workspace, s)
                          : launch_pair_s<WT, true, 128>(g, plan.splits, workspace, s);
}

// ---- few rows: plan ----

constexpr int kFewMaxRows = 64;
int few_bn(int64_t M) { return (int)((M + 15) / 16 * 16); }
int few_width(int64_t M) { return M <= 16 ? 16 : (M <= 32 ? 32 : 64); }
int64_t few_tiles(int64_t N) { return (N + 127) / 128; }
// CTAs: as many as are resident, but with runs of six units and more (a shared tile
// costs two to four microseconds, a unit half of one), and at most 16 on a tile.
constexpr int64_t kFewMaxCtas = 512, kFewRun = 6;
int64_t few_ctas(int64_t N, int64_t K, int64_t resident) {
    const int64_t tiles = few_tiles(N), units = tiles * ((K + 127) / 128);
    int64_t n = (units + kFewRun - 1) / kFewRun;
    if (n < tiles) n = tiles;
    if (n > 16 * tiles) n = 16 * tiles;
    return n < resident ? n : resident;
}
int64_t few_resident(int64_t M) {
    const int64_t n = (int64_t)sm_count() * (M <= 32 ? 2 : 1);
    return n < kFewMaxCtas ? n : kFewMaxCtas;
}
size_t few_part_bytes(int64_t M, int64_t N, int64_t K) {
    return round_up((size_t)few_ctas(N, K, kFewMaxCtas) * 2 * 128 * (size_t)few_width(M) * 4);
}
size_t few_arrived_bytes(int64_t N) { return round_up((size_t)few_tiles(N) * 4); }

// Which of the two kernels: the shorter by the pairs' model above and this one, from
// memory, not L2: a call's fixed part, a unit's time for each unit of a CTA's run, and the
// CTAs that share a tile; two CTAs of an SM at up to 32 rows take a unit each in the time.
// Measured in a replayed graph over weights from memory, pairs / few rows: 28672 x 8192 at
// 16 rows 63 / 49, at 64 rows 64 / 53; at 64 rows 60000 x 4000 67 / 55, 1024 x 14336
// 32 / 20, 40000 x 2000 32 / 34, 11008 x 4096 21 / 22, 4096 x 4096 12 / 19. (Of 26 weights
// at 33 to 64 rows the rule takes the slower kernel for one, by 4%.)
double few_us(int64_t M, int64_t N, int64_t K) {
    const int64_t blocks = (K + 127) / 128, units = few_tiles(N) * blocks;
    const double run = (double)units / (double)few_ctas(N, K, few_resident(M));
    const double shared = (double)blocks / run;   // CTAs on a tile
    const double per_cta = shared > 1.0 ? shared : 0.0;
    if (M > 32) return 13.5 + run * 0.39 + per_cta * 0.6;
    return 8.0 + run * 0.86 + per_cta * (M <= 16 ? 0.5 : 0.7);
}
bool few_rows(int64_t M, int64_t N, int64_t K) { return M <= kFewMaxRows && few_us(M, N, K) <= pair_plan(M, N, K).us; }

template <int BN, bool WT, typename O>
cudaError_t launch_few_o(const Fp8Gemm& g, const FewParams& p, cudaStream_t s) {
    CUtensorMap ma, mw;
    if (!encode_codes(&ma, g.a.codes, g.a.cols, g.a.rows, g.a.ld, (uint32_t)p.bn) ||
        !encode_codes(&mw, g.w.codes, g.w.cols, g.w.rows, g.w.ld, 128))
        return cudaErrorInvalidValue;
    const size_t smem = (size_t)Few<BN>::TOTAL + 1024;
    auto kern = fp8_gemm_few_kernel<BN, WT, O>;
    static std::atomic<int> ready[kMaxDevices];
    cudaError_t e = prepare_kernel(reinterpret_cast<const void*>(kern), smem, 0, ready);
    if (e != cudaSuccess) return e;
    static_assert(Few<BN>::CTAS == (BN <= 32 ? 2 : 1), "few_resident counts the same");
    LaunchConfig cfg(dim3((unsigned)few_ctas(g.N, g.K, few_resident(g.M))), Few<BN>::THREADS, smem, s);
    return cudaLaunchKernelEx(&cfg.c, kern, p, ma, mw);
}

template <int BN, bool WT>
cudaError_t launch_few_t(const Fp8Gemm& g, const FewParams& p, cudaStream_t s) {
    if (g.out_type == kF16) return launch_few_o<BN, WT, __half>(g, p, s);
    if (g.out_type == kBf16) return launch_few_o<BN, WT, __nv_bfloat16>(g, p, s);
    return launch_few_o<BN, WT, float>(g, p, s);
}

template <bool WT>
cudaError_t launch_few(const Fp8Gemm& g, void* workspace, bool prepared, cudaStream_t s) {
    FewParams p;
    p.sa = g.a.scales;
    p.sa_row = g.a.s_row;
    p.sa_col = g.a.s_col;
    p.sw = g.w.scales;
    p.sw_n = WT ? g.w.s_col : g.w.s_row;
    p.sw_k = WT ? g.w.s_row : g.w.s_col;
    p.bias = g.bias;
    p.bias_type = g.bias_type;
    p.out = g.out;
    p.ldo = g.ldo;
    p.M = (int)g.M;
    p.N = (int)g.N;
    p.blocks = (int)((g.K + 127) / 128);
    p.bn = few_bn(g.M);
    p.units = few_tiles(g.N) * p.blocks;
    p.arrived = static_cast<unsigned int*>(workspace);
    p.part = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + few_arrived_bytes(g.N));
    p.weights_ready = prepared;
    p.fault = fault_word();
    if (p.fault == nullptr) return cudaErrorInvalidDevicePointer;
    if (!prepared) {
        cudaError_t e = cudaMemsetAsync(workspace, 0, few_arrived_bytes(g.N), s);
        if (e != cudaSuccess) return e;
    }
    switch (few_width(g.M)) {
        case 16: return launch_few_t<16, WT>(g, p, s);
        case 32: return launch_few_t<32, WT>(g, p, s);
        default: return launch_few_t<64, WT>(g, p, s);
    }
}

}  // namespace

size_t fp8_gemm_zeroed_bytes(int64_t M, int64_t N, int64_t K) {
    if (few_rows(M, N, K)) return few_arrived_bytes(N);
    return pair_plan(M, N, K).splits > 1 ? pair_arrived_bytes(M, N, K) : 0;
}

size_t fp8_gemm_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (few_rows(M, N, K)) return few_arrived_bytes(N) + few_part_bytes(M, N, K);
    return pair_plan(M, N, K).splits > 1 ? pair_arrived_bytes(M, N, K) + pair_part_bytes(M, N, K) : 0;
}

Fp8Plan fp8_gemm_plan(int64_t M, int64_t N, int64_t K) {
    if (few_rows(M, N, K)) return Fp8Plan{true, few_width(M), 1};
    const PairPlan plan = pair_plan(M, N, K);
    return Fp8Plan{false, plan.tn, plan.splits};
}

cudaError_t launch_fp8_gemm(const Fp8Gemm& g, void* workspace, bool prepared, cudaStream_t s) {
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
    if (few_rows(g.M, g.N, g.K))
        return g.transpose ? launch_few<true>(g, workspace, prepared, s) : launch_few<false>(g, workspace, prepared, s);
    return g.transpose ? launch_pair<true>(g, workspace, prepared, s) : launch_pair<false>(g, workspace, prepared, s);
}

}  // namespace wq
