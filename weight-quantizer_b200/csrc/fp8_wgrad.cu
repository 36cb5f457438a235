// The weight gradient of a linear layer from the 8-bit checkpoint of its input.
//
//   dw[n, k] (+)= sum_m dy[m, n] x^[m, k],   x^[m, k] = c[m, k] s[m, k / 128]
//
// The scale varies along the sum, so it cannot leave it: x^ enters the product as
// an operand. With power-of-two scales (quantize_fp8's) code * scale is exact in
// bf16, and dy is bf16 already, or is split into bf16 terms that add up to it (two
// for fp16, three for fp32): every product is exact. Other scales' code * scale is
// rounded to bf16 (by at most 2^-8 of each value), the only 16-bit operand type with
// the scales' range.
//
// Sums over 512 rows (256 and 128 with two and three terms) stay in tensor memory,
// then they are added to fp32 registers: the tensor core's own additions cut off what
// they add, and over all rows of a long batch that grows, all to one side. Relative
// error at 8192 rows of random signs 3.6e-6 without the spans and 1.6e-7 with them
// (1.3e-5 and 3.4e-7 where every product is positive). The least term of dy enters first,
// so that only the first term's additions cut at the sum's full size: with fp32 dy 5.9e-8
// at 64 rows and 2.7e-7 at 777, 3.8e-7 and 5.7e-7 the other way round.
#include "fp8_types.cuh"
#include "kernels.h"
#include "launch.h"
#include "tc_ptx.cuh"

namespace wq {
namespace {

// A pair of CTAs makes a 256 x TK tile of dw with tcgen05.mma of cta_group::2 on
// steps of 64 rows of dy and x. Both operands lie along the outer dimension in
// memory (MN-major), so dy goes from memory to the MMA as it is: warp 0 loads
// boxes of 64 rows x 64 columns. x^ is made by eight warps (4-11), which take turns
// by fours, so that each step of rows has two steps of time: codes (TMA) and scales
// (asynchronous copies) come into shared memory some steps ahead by warp 3, then
// e4m3 -> fp16 -> fp32, times the row's scale, to bf16 in the swizzled tile; a lane
// takes eight codes of each 64 columns, which are one 16-byte chunk of that tile, so
// that eight lanes fill a row without bank conflicts. Eight more warps
// (12-19) add the finished sums of a span to their registers: a lane is a row of
// dw, a warp has TK / 2 columns. TK is 256, or 128 where that fills the SMs better
// (a step of the narrow tile takes a little over half as long; 2304 x 768 is 27 wide
// tiles for 74 pairs, or 54 narrow ones). Where even the narrow tiles are fewer than
// half of the pairs, the rows are cut into parts (SPLIT): each pair writes its part's
// sums to the workspace, and the last to arrive at a tile adds them in order.

constexpr int kRows = 256;                     // rows of dw in a tile
constexpr int kStep = 64;                      // rows of dy and x per step
constexpr int kPlaneBytes = kStep * 128 * 2;   // 64 rows x 128 columns in bf16: one CTA's term of dy in one step
constexpr int kThreads = 640;
constexpr int kLaunchRegs = 96, kCtlRegs = 40, kMakeRegs = 56, kSumRegs = 160;
static_assert(kCtlRegs + 2 * kMakeRegs + 2 * kSumRegs <= 5 * kLaunchRegs, "register split exceeds the launch's registers");

// Codes on their way: 64 rows of 128 codes (128-byte swizzle) and their scales.
constexpr int kAhead = 6;
constexpr int kCodesBytes = kStep * 128;

// P terms of dy per step, then x^; the codes on their way, their scales.
template <int P, int TK>
struct Smem {
    // steps whose sums stay in tensor memory: some 32 MMAs whatever the terms
    static constexpr int SPAN = P == 1 ? 8 : (P == 2 ? 4 : 2);
    static constexpr int X_BYTES = kStep * (TK / 2) * 2;
    static constexpr int STAGE = P * kPlaneBytes + X_BYTES;
    static constexpr int STAGES = (222 * 1024 - kAhead * (kCodesBytes + kStep * 4)) / STAGE;
    static constexpr int CODES = STAGES * STAGE;
    static constexpr int SCALES = CODES + kAhead * kCodesBytes;
    static constexpr int BAR = SCALES + kAhead * kStep * 4;
    // full and done per stage; codes there and read; sums full[2], empty[2]
    static constexpr int TMEM_SLOT = BAR + 8 * (2 * STAGES + 2 * kAhead + 4);
    static constexpr int FLAG = TMEM_SLOT + 8;
    // a token to send, and where tokens go: one for each warp that makes a stage's x^
    static constexpr int TOKEN = TMEM_SLOT + 16;
    static constexpr int TOTAL = TOKEN + 16 * (1 + 4 * STAGES);
    static_assert(TOKEN % 16 == 0, "bulk copies are 16-byte aligned");
    static_assert(STAGES >= 2, "the MMAs of one step run while the next is made");
    static_assert(TOTAL + 1024 <= 227 * 1024, "stages exceed the shared memory of one CTA");
};

struct Params {
    const float* scales;
    int64_t s_row, s_col;
    void* out;
    int64_t ldo;
    int accumulate;
    int M, N, K, steps;
    int tiles_n, tiles_k, band;
    int splits;              // parts of the rows
    float* part;             // [tile][part][rank] sums of 128 x TK
    unsigned int* arrived;   // per tile and rank, zeroed before the launch
    unsigned int* fault;
};

// Tile t: bands of `band` column tiles of x; inside a band they run fastest, so
// that the band's columns of x stay in L2 while dy streams by once.
__device__ __forceinline__ void tile_of(int t, const Params& p, int& nt, int& kt) {
    const int per = p.band * p.tiles_n;
    const int b = t / per, in = t - b * per;
    const int bw = min(p.band, p.tiles_k - b * p.band);
    nt = in / bw;
    kt = b * p.band + (in - nt * bw);
}

// Columns c .. c + 15 of a row of dw whose rows lie 32 bytes apart.
template <typename O>
__device__ __forceinline__ void put16(O* at, const float (&v)[16], bool add) {
    constexpr int PER = 4 / (int)sizeof(O);       // values in a word
#pragma unroll
    for (int i = 0; i < 16; i += 8 * PER) {
        uint32_t w[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            O e[PER];
            if (add) *reinterpret_cast<uint32_t*>(e) = *reinterpret_cast<const uint32_t*>(at + i + q * PER);
#pragma unroll
            for (int j = 0; j < PER; ++j)
                e[j] = from_f32<O>(add ? to_f32<O>(e[j]) + v[i + q * PER + j] : v[i + q * PER + j]);
            w[q] = *reinterpret_cast<const uint32_t*>(e);
        }
        st_32(at + i, w);
    }
}

// The same 16 columns of a warp's 32 rows where rows lie otherwise, or end inside: a
// transposition inside the warp (bits of the lane change places with bits of the
// register), after which a lane has one column of 16 rows and a store fills 16
// neighbouring columns. Single elements of 32 rows per store took 752 us at
// 16 x 14336 x 8191 (fp32), these 216.
template <typename O>
__device__ __forceinline__ void put16_across(O* out, int64_t n0, int64_t c, int64_t rows, int64_t cols, int64_t ld,
                                             int lane, float (&v)[16], bool add) {
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) {
        const bool up = (lane & d) != 0;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            if (j & d) continue;
            const float got = __shfl_xor_sync(0xffffffffu, up ? v[j] : v[j + d], d);
            if (up) v[j] = got;
            else v[j + d] = got;
        }
    }
    const int64_t col = c + (lane & 15), n = n0 + (lane & 16);
    if (col >= cols) return;
    O* at = out + n * ld + col;
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (n + i < rows) {
            O* e = at + i * ld;
            *e = from_f32<O>(add ? to_f32<O>(*e) + v[i] : v[i]);
        }
}

// WIDE: rows of dw lie 32 bytes apart and K is a multiple of 16. (A kernel of its own: both
// ways in one cost registers: 695 us against 660 at 8192 x 11008 x 4096, 849 against 779
// where the result is added to dw, both under sustained power.)
template <int P, int TK, bool SPLIT, bool WIDE, typename O>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    fp8_wgrad_kernel(const Params p, const __grid_constant__ CUtensorMap map_dy,
                     const __grid_constant__ CUtensorMap map_x) {
    using L = Smem<P, TK>;
    constexpr int NS = L::STAGES;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_addr(smem);
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // uniform
    const int rank = (int)cluster_rank();
    auto bar = [&](int i) -> uint32_t { return sbase + L::BAR + 8u * (uint32_t)i; };
    auto full = [&](int s) { return bar(s); };
    auto done = [&](int s) { return bar(NS + s); };
    auto codes_full = [&](int a) { return bar(2 * NS + a); };
    auto codes_read = [&](int a) { return bar(2 * NS + kAhead + a); };
    auto sums_full = [&](int b) { return bar(2 * NS + 2 * kAhead + b); };
    auto sums_empty = [&](int b) { return bar(2 * NS + 2 * kAhead + 2 + b); };
    launch_dependents();
    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            // the even CTA's: its loader's arrival with both CTAs' bytes of dy and the
            // tokens of the odd CTA's four warps that made x^, and its own four
            mbar_init(full(s), 5);
            mbar_init(done(s), 1);
        }
        for (int a = 0; a < kAhead; ++a) {
            mbar_init(codes_full(a), 33);   // the codes' bytes, and every lane's copies of scales
            mbar_init(codes_read(a), 4);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(sums_full(b), 1);
            mbar_init(sums_empty(b), 16);
        }
        fence_mbarrier_init();
        *reinterpret_cast<uint4*>(smem + L::TOKEN) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
    }
    if (warp == 1) tmem_alloc<2>(sbase + L::TMEM_SLOT, 512);
    tc_before();
    __syncthreads();
    cluster_sync();
    tc_after();
    grid_wait();   // nothing above reads global memory
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + L::TMEM_SLOT);
    const int pairs = (int)gridDim.x >> 1, first = (int)blockIdx.x >> 1;
    // an item is a part of a tile's steps
    const int splits = SPLIT ? p.splits : 1;
    const int items = p.tiles_n * p.tiles_k * splits;
    auto from_step = [&](int item) -> int {
        return SPLIT ? (int)((int64_t)(item % splits) * p.steps / splits) : 0;
    };
    auto to_step = [&](int item) -> int {
        return SPLIT ? (int)((int64_t)(item % splits + 1) * p.steps / splits) : p.steps;
    };
    int64_t total = 0;   // this pair's steps
    if constexpr (SPLIT)
        for (int t = first; t < items; t += pairs) total += to_step(t) - from_step(t);
    else
        total = first < items ? (int64_t)((items - 1 - first) / pairs + 1) * p.steps : 0;
    bool faulted = false;
    auto give_up = [&]() {
        faulted = true;
        atomicOr(p.fault, 1u);
    };
    auto wait = [&](uint32_t b, uint32_t parity) {
        if (!faulted && !mbar_wait_bounded(b, parity)) give_up();
    };

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kCtlRegs));
        if (warp == 0) {
            const uint32_t full0 = in_cta(full(0), 0);
            int s = 0;
            uint32_t ph = 1;
            for (int t = first; t < items; t += pairs) {
                int nt, kt;
                tile_of(t / splits, p, nt, kt);
                const int n0 = nt * kRows + rank * 128, to = to_step(t);
                for (int i = from_step(t); i < to; ++i) {
                    wait(done(s), ph);
                    __syncwarp();
                    if (elect_one()) {
                        const uint32_t f = full0 + 8u * (uint32_t)s;
                        const uint32_t dst = sbase + (uint32_t)(s * L::STAGE);
                        if (rank == 0) mbar_arrive_expect_tx(full(s), 2 * P * kPlaneBytes + 4 * 16);
#pragma unroll
                        for (int pl = 0; pl < P; ++pl) {
                            // term pl of dy lies pl * M rows below the first; the rows
                            // of another term that a last step reaches into meet x^ = 0
                            const int y = pl * p.M + i * kStep;
                            tma_box<2>(dst + pl * kPlaneBytes, &map_dy, n0, y, f);
                            tma_box<2>(dst + pl * kPlaneBytes + kPlaneBytes / 2, &map_dy, n0 + 64, y, f);
                        }
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
        } else if (warp == 1 && rank == 0) {
            constexpr uint32_t idesc = mma_idesc(1, true, true, kRows, TK);
            const uint64_t desc0 = sw128_matrix(sbase, kPlaneBytes / 2);
            int s = 0, buf = 0;
            uint32_t ph = 0, reuse = 1;
            for (int t = first; t < items; t += pairs) {
                const int steps = to_step(t) - from_step(t);
                for (int i = 0; i < steps; ++i) {
                    const int in = i % L::SPAN;
                    if (in == 0) wait(sums_empty(buf), reuse);
                    // acquires the odd CTA's x^ too, which its warps' tokens release
                    if (!faulted && !mbar_wait_cluster(full(s), ph)) give_up();
                    __syncwarp();
                    tc_after();
                    const bool last = in == L::SPAN - 1 || i == steps - 1;
                    if (elect_one()) {
                        const uint64_t d0 = desc0 + (uint64_t)(s * (L::STAGE >> 4));
                        const uint64_t dx = d0 + (uint64_t)(P * (kPlaneBytes >> 4));
#pragma unroll
                        for (int pl = P - 1; pl >= 0; --pl)   // the least term first
#pragma unroll
                            for (int k = 0; k < kStep / 16; ++k)   // 16 rows of 128 bytes
                                mma_bf16(tmem + (uint32_t)(buf * TK), d0 + (uint64_t)(pl * (kPlaneBytes >> 4)) + 128u * k,
                                         dx + 128u * k, idesc, in > 0 || pl < P - 1 || k > 0);
                        mma_done<2>(done(s));
                        if (last) mma_done<2>(sums_full(buf));
                    }
                    __syncwarp();
                    if (last) {
                        buf ^= 1;
                        if (buf == 0) reuse ^= 1u;
                    }
                    if (++s == NS) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
            }
        } else if (warp == 3) {
            // each CTA's columns of codes (boxes of 128, of which the narrow tile uses 64),
            // and the scales of the block that they lie in
            int a = 0;
            uint32_t ph = 1;
            for (int t = first; t < items; t += pairs) {
                int nt, kt;
                tile_of(t / splits, p, nt, kt);
                const int k0 = kt * TK + rank * (TK / 2), to = to_step(t);
                const float* sc = p.scales + (min(k0, p.K - 1) >> 7) * p.s_col;
                for (int i = from_step(t); i < to; ++i) {
                    wait(codes_read(a), ph);
                    __syncwarp();
                    if (elect_one()) {
                        mbar_arrive_expect_tx(codes_full(a), kCodesBytes);
                        tma_box<1>(sbase + (uint32_t)(L::CODES + a * kCodesBytes), &map_x, k0, i * kStep, codes_full(a));
                    }
                    __syncwarp();
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int64_t m = (int64_t)i * kStep + h * 32 + lane;   // (rows beyond the last: scale 0)
                        cp_async4_s(sbase + (uint32_t)(L::SCALES + (a * kStep + h * 32 + lane) * 4),
                                    m < p.M ? sc + m * p.s_row : p.scales, m < p.M);
                    }
                    cp_async_arrive(codes_full(a));
                    if (++a == kAhead) {
                        a = 0;
                        ph ^= 1u;
                    }
                }
            }
            for (int i = 0; i < kAhead; ++i) {   // as warp 0 does
                if (!mbar_wait_bounded(codes_read(a), ph)) atomicOr(p.fault, 1u);
                if (++a == kAhead) {
                    a = 0;
                    ph ^= 1u;
                }
            }
        }
    } else if (warp < 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMakeRegs));
        const int q = warp & 3, turn = (warp - 4) >> 2;
        // this lane's rows row_of(j) of a step, j < 4, and its chunk of eight codes. (Two
        // rows that a half-warp reads at once are four apart: their chunks lie in
        // different halves of the swizzled 128 bytes.)
        const int sub = lane >> 3, chunk = lane & 7;
        const int row0 = q * 16 + (sub >> 1) + 4 * (sub & 1);
        auto row_of = [&](int j) { return row0 + 2 * (j & 1) + 8 * (j >> 1); };
        const uint32_t x_at = sbase + (uint32_t)(P * kPlaneBytes);
        const uint32_t full0 = in_cta(full(0), 0), tokens0 = in_cta(sbase + L::TOKEN + 16u, 0) + 16u * (uint32_t)q;
        int s = turn, a = turn;
        uint32_t ph = 1, aph = 0;
        for (int64_t left = (total + 1 - turn) >> 1; left > 0; --left) {
            uint2 code[4][2];         // eight codes of each 64 columns
            float scale[4];
            if (!try_wait_both(codes_full(a), aph, done(s), ph)) {
                wait(codes_full(a), aph);
                wait(done(s), ph);
            }
            __syncwarp();
            const unsigned char* from = smem + L::CODES + a * kCodesBytes;
            const float* sc = reinterpret_cast<const float*>(smem + L::SCALES) + a * kStep;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = row_of(j);
                const unsigned char* at = from + r * 128 + (chunk & 1) * 8;
                code[j][0] = *reinterpret_cast<const uint2*>(at + (((chunk >> 1) ^ (r & 7)) << 4));
                if constexpr (TK == 256)
                    code[j][1] = *reinterpret_cast<const uint2*>(at + (((4 + (chunk >> 1)) ^ (r & 7)) << 4));
                scale[j] = sc[r];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = row_of(j);
                const uint32_t at = x_at + (uint32_t)(s * L::STAGE + r * 128 + ((chunk ^ (r & 7)) << 4));
                const uint64_t by = pack2(scale[j], scale[j]);
#pragma unroll
                for (int h = 0; h < TK / 128; ++h) {
                    uint32_t o[4];
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const uint32_t w = b < 2 ? code[j][h].x : code[j][h].y;
                        const float2 c = e4m3x2_values(w >> (16 * (b & 1)));
                        const float2 f = unpack2(mul2(pack2(c.x, c.y), by));
                        const __nv_bfloat162 e = __floats2bfloat162_rn(f.x, f.y);
                        o[b] = *reinterpret_cast<const uint32_t*>(&e);
                    }
                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at + h * (kPlaneBytes / 2)),
                                 "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3])
                                 : "memory");
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                if (rank == 0) mbar_arrive(full(s));
                else token_to_cta(tokens0 + 64u * (uint32_t)s, sbase + L::TOKEN, full0 + 8u * (uint32_t)s);
                mbar_arrive(codes_read(a));
            }
            a += 2;
            if (a >= kAhead) {
                a -= kAhead;
                aph ^= 1u;
            }
            s += 2;
            if (s >= NS) {
                s -= NS;
                ph ^= 1u;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSumRegs));
        const int q = warp & 3, half = (warp - 12) >> 2;
        const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(half * (TK / 2));
        const uint32_t free0 = in_cta(sums_empty(0), 0);
        int buf = 0;
        uint32_t ph = 0;
        for (int t = first; t < items; t += pairs) {
            float acc[TK / 2];
#pragma unroll
            for (int c = 0; c < TK / 2; ++c) acc[c] = 0.0f;
            for (int left = to_step(t) - from_step(t); left > 0; left -= L::SPAN) {
                wait(sums_full(buf), ph);
                __syncwarp();
                tc_after();
#pragma unroll
                for (int c = 0; c < TK / 2; c += 16) {
                    uint64_t v[8];
                    tmem_pairs(taddr + (uint32_t)(buf * TK + c), v);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float2 f = unpack2(v[k]);
                        acc[c + 2 * k] += f.x;
                        acc[c + 2 * k + 1] += f.y;
                    }
                }
                tc_before();
                __syncwarp();
                if (lane == 0) arrive_in_cluster(free0 + 8u * (uint32_t)buf);
                buf ^= 1;
                if (buf == 0) ph ^= 1u;
            }
            bool write = true;
            if constexpr (SPLIT) {
                // the part's sums go to its slot, [column / 4][row][4]
                constexpr int64_t SLOT = 128 * TK;
                const int64_t lane_at = ((int64_t)half * (TK / 8) * 128 + q * 32 + lane) * 4;
                float4* mine = reinterpret_cast<float4*>(p.part + ((int64_t)t * 2 + rank) * SLOT + lane_at);
#pragma unroll
                for (int c = 0; c < TK / 8; ++c)
                    mine[c * 128] = make_float4(acc[4 * c], acc[4 * c + 1], acc[4 * c + 2], acc[4 * c + 3]);
                named_barrier(1, 256);
                volatile uint32_t* flag = reinterpret_cast<volatile uint32_t*>(smem + L::FLAG);
                const int tile = t / splits;
                if (warp == 12 && lane == 0)
                    *flag = last_to_arrive(p.arrived + tile * 2 + rank, (unsigned)splits);
                named_barrier(1, 256);
                write = *flag != 0u;
                named_barrier(1, 256);   // the flag has been read
                if (write) {
#pragma unroll
                    for (int c = 0; c < TK / 2; ++c) acc[c] = 0.0f;
#pragma unroll 1
                    for (int sp = 0; sp < splits; ++sp) {
                        const float4* src = reinterpret_cast<const float4*>(
                            p.part + (((int64_t)tile * splits + sp) * 2 + rank) * SLOT + lane_at);
#pragma unroll
                        for (int c = 0; c < TK / 8; ++c) {
                            const float4 f = __ldcg(src + c * 128);
                            acc[4 * c] += f.x;
                            acc[4 * c + 1] += f.y;
                            acc[4 * c + 2] += f.z;
                            acc[4 * c + 3] += f.w;
                        }
                    }
                }
            }
            int nt, kt;
            tile_of(t / splits, p, nt, kt);
            const int64_t n0 = (int64_t)nt * kRows + rank * 128 + q * 32;
            const int64_t k0 = (int64_t)kt * TK + half * (TK / 2);
            O* out = static_cast<O*>(p.out);
            if (WIDE ? write && n0 + lane < p.N : write && n0 < p.N) {
#pragma unroll
                for (int c = 0; c < TK / 2; c += 16) {
                    float v[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) v[k] = acc[c + k];
                    if (k0 + c < p.K) {
                        if constexpr (WIDE) put16<O>(out + (n0 + lane) * p.ldo + k0 + c, v, p.accumulate);
                        else put16_across<O>(out, n0, k0 + c, p.N, p.K, p.ldo, lane, v, p.accumulate);
                    }
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

// dy as bf16 terms that add up to it (fp16: 2, fp32: 3), each [M, ld] below the
// last: v cut off to bf16, then what is left (cut off, no term overflows and eight
// bits go into each). A value that is not finite has it in the first term and zeros
// below. bf16 input whose rows TMA cannot read (an odd stride or address) is copied as
// its one term. The product's counters are zeroed on the way.
template <typename T, int P>
__global__ void __launch_bounds__(256) split_terms_kernel(const T* __restrict__ dy, int64_t M, int64_t N, int64_t ldy,
                                                          __nv_bfloat16* __restrict__ out, int64_t ld, unsigned int* arrived,
                                                          int64_t n_arrived) {
    grid_wait();
    launch_dependents();
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n_arrived;
         i += (int64_t)gridDim.x * blockDim.x)
        arrived[i] = 0u;
    const int64_t quads = ld / 4;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < M * quads;
         i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t m = i / quads, n = (i - m * quads) * 4;
        __nv_bfloat16 term[P][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float v = n + k < N ? to_f32<T>(dy[m * ldy + n + k]) : 0.0f;
#pragma unroll
            for (int pl = 0; pl < P; ++pl) {
                term[pl][k] = __float2bfloat16_rz(v);
                const float h = __bfloat162float(term[pl][k]);
                v = fabsf(h) <= 3.402823466e38f ? v - h : 0.0f;
            }
        }
#pragma unroll
        for (int pl = 0; pl < P; ++pl)
            *reinterpret_cast<uint2*>(out + (pl * M + m) * ld + n) = *reinterpret_cast<const uint2*>(term[pl]);
    }
}

// dw = 0 where there are no rows (and nothing to add to).
template <typename O>
__global__ void zero_rows_kernel(O* out, int64_t N, int64_t K, int64_t ldo) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < N * K; i += (int64_t)gridDim.x * blockDim.x)
        out[i / K * ldo + i % K] = from_f32<O>(0.0f);
}

int terms_of(int type) { return type == kBf16 ? 1 : (type == kF16 ? 2 : 3); }
int64_t term_ld(int64_t N) { return (N + 7) / 8 * 8; }
int bytes_of(int type) { return type == kF32 ? 4 : 2; }

constexpr int64_t kMostSplits = 16;

bool rows_by_tma(const void* dy, int type, int64_t ldy) {
    return type == kBf16 && (reinterpret_cast<uintptr_t>(dy) & 15) == 0 && (ldy * 2) % 16 == 0;
}
bool wide_rows(const Fp8WeightGrad& g) {
    return (reinterpret_cast<uintptr_t>(g.out) & 31) == 0 && (g.ldo * bytes_of(g.out_type)) % 32 == 0 && g.K % 16 == 0;
}
size_t round_up(size_t v) { return (v + 255) / 256 * 256; }

// The tile's columns and the parts that its rows are cut into: the shortest by a model
// in microseconds, fitted at 512 to 8192 rows of 128 x 128 to 11008 x 4096: the rounds
// of steps over the pairs of SMs, a wide step taking 0.45 with one term, 0.65 with two
// and 0.92 with three, a narrow one 0.6 of that; parts cost 7 and 0.5 for each, for
// their sums written and read by the last pair to arrive. Without and with parts:
// 8192 x 128 x 128 (bf16 dy) 37 / 22, (fp32 dy) 62 / 22; 65536 x 256 x 256 260 / 39;
// 4096 x 768 x 768 22 / 21; 1024 x 512 x 512 (9.4) has none.
struct Plan {
    int tk, splits;
};
Plan plan_of(int64_t M, int64_t N, int64_t K, int dy_type) {
    const int64_t pairs = sm_count() / 2, rows = (N + kRows - 1) / kRows, steps = (M + kStep - 1) / kStep;
    const int terms = terms_of(dy_type);
    const double wide_us = terms == 1 ? 0.45 : (terms == 2 ? 0.65 : 0.92), narrow_us = 0.6 * wide_us;
    const int64_t wide = rows * ((K + 255) / 256), narrow = rows * ((K + 127) / 128);
    double best = wide_us * (double)((wide + pairs - 1) / pairs * steps);
    Plan plan{256, 1};
    const double one = narrow_us * (double)((narrow + pairs - 1) / pairs * steps);
    if (one < best) {
        best = one;
        plan = Plan{128, 1};
    }
    int64_t most = pairs / narrow;
    if (most > steps / 4) most = steps / 4;
    if (most > kMostSplits) most = kMostSplits;
    for (int64_t n = 2; n <= most; ++n) {
        const double us = narrow_us * (double)((steps + n - 1) / n) + 7.0 + 0.5 * (double)n;
        if (us < best) {
            best = us;
            plan = Plan{128, (int)n};
        }
    }
    return plan;
}
// The workspace: the counters and the parts' sums where there are parts, then the terms of
// dy where dy is not read as it is.
size_t terms_bytes(int64_t M, int64_t N, int type) {
    return round_up((size_t)terms_of(type) * (size_t)M * (size_t)term_ld(N) * 2);
}
int64_t plan_tiles(int64_t N, int64_t K, int tk) { return (N + kRows - 1) / kRows * ((K + tk - 1) / tk); }
size_t arrived_bytes(const Plan& plan, int64_t N, int64_t K) {
    return plan.splits == 1 ? 0 : round_up((size_t)plan_tiles(N, K, plan.tk) * 2 * 4);
}
size_t part_bytes(const Plan& plan, int64_t N, int64_t K) {
    return plan.splits == 1 ? 0 : (size_t)plan_tiles(N, K, plan.tk) * plan.splits * 2 * 128 * plan.tk * 4;
}

template <int P, int TK, bool SPLIT, bool WIDE, typename O>
cudaError_t launch_po(const Fp8WeightGrad& g, const void* dy, int64_t ld, int splits, unsigned char* counters,
                      cudaStream_t s) {
    Params p;
    p.scales = g.a.scales;
    p.s_row = g.a.s_row;
    p.s_col = g.a.s_col;
    p.out = g.out;
    p.ldo = g.ldo;
    p.accumulate = g.accumulate;
    p.M = (int)g.M;
    p.N = (int)g.N;
    p.K = (int)g.K;
    p.steps = (int)((g.M + kStep - 1) / kStep);
    p.tiles_n = (int)((g.N + kRows - 1) / kRows);
    p.tiles_k = (int)((g.K + TK - 1) / TK);
    // a band's columns of x stay below 40 MB, well inside L2
    int64_t band = ((int64_t)40 << 20) / (g.M * TK);
    band = band < 1 ? 1 : band;
    const int64_t bands = (p.tiles_k + band - 1) / band;
    p.band = (int)((p.tiles_k + bands - 1) / bands);
    p.splits = splits;
    p.arrived = SPLIT ? reinterpret_cast<unsigned int*>(counters) : nullptr;
    p.part = SPLIT ? reinterpret_cast<float*>(counters + arrived_bytes(Plan{TK, splits}, g.N, g.K)) : nullptr;
    p.fault = fault_word();
    if (p.fault == nullptr) return cudaErrorInvalidDevicePointer;
    CUtensorMap map, mx;
    if (!encode_rows(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, dy, g.N, P * g.M, ld * 2, kStep) ||
        !encode_codes(&mx, g.a.codes, g.a.cols, g.a.rows, g.a.ld, kStep))
        return cudaErrorInvalidValue;
    const size_t smem = (size_t)Smem<P, TK>::TOTAL + 1024;
    auto kern = fp8_wgrad_kernel<P, TK, SPLIT, WIDE, O>;
    static std::atomic<int> ready[kMaxDevices];
    cudaError_t e = prepare_kernel(reinterpret_cast<const void*>(kern), smem, kLaunchRegs, ready);
    if (e != cudaSuccess) return e;
    const int64_t items = (int64_t)p.tiles_n * p.tiles_k * splits;
    const int64_t pairs = sm_count() / 2;
    if (items > 0x7fffffff) return cudaErrorInvalidValue;
    LaunchConfig cfg(dim3(2u * (unsigned)(items < pairs ? items : pairs)), kThreads, smem, s);
    return cudaLaunchKernelEx(&cfg.c, kern, p, map, mx);
}

template <int P, typename O>
cudaError_t launch_tile(const Fp8WeightGrad& g, const void* dy, int64_t ld, const Plan& plan, unsigned char* counters,
                        cudaStream_t s) {
    // (parts make few tiles: one way of writing them serves)
    if (plan.splits > 1) return launch_po<P, 128, true, false, O>(g, dy, ld, plan.splits, counters, s);
    if (wide_rows(g))
        return plan.tk == 256 ? launch_po<P, 256, false, true, O>(g, dy, ld, 1, nullptr, s)
                              : launch_po<P, 128, false, true, O>(g, dy, ld, 1, nullptr, s);
    return plan.tk == 256 ? launch_po<P, 256, false, false, O>(g, dy, ld, 1, nullptr, s)
                          : launch_po<P, 128, false, false, O>(g, dy, ld, 1, nullptr, s);
}

template <int P>
cudaError_t launch_p(const Fp8WeightGrad& g, const void* dy, int64_t ld, const Plan& plan, unsigned char* counters,
                     cudaStream_t s) {
    if (g.out_type == kF16) return launch_tile<P, __half>(g, dy, ld, plan, counters, s);
    if (g.out_type == kBf16) return launch_tile<P, __nv_bfloat16>(g, dy, ld, plan, counters, s);
    return launch_tile<P, float>(g, dy, ld, plan, counters, s);
}

template <typename T, int P>
cudaError_t split_and_launch(const Fp8WeightGrad& g, unsigned char* counters, const Plan& plan, cudaStream_t s) {
    const int64_t ld = term_ld(g.N);
    __nv_bfloat16* terms = reinterpret_cast<__nv_bfloat16*>(counters + arrived_bytes(plan, g.N, g.K) +
                                                            part_bytes(plan, g.N, g.K));
    const int64_t want = (g.M * (ld / 4) + 255) / 256;
    const int64_t most = (int64_t)sm_count() * 16;
    LaunchConfig cfg(dim3((unsigned)(want < most ? want : most)), 256, 0, s);
    cudaError_t e = cudaLaunchKernelEx(&cfg.c, split_terms_kernel<T, P>, static_cast<const T*>(g.dy), g.M, g.N, g.ldy,
                                       terms, ld, reinterpret_cast<unsigned int*>(counters),
                                       (int64_t)(arrived_bytes(plan, g.N, g.K) / 4));
    if (e != cudaSuccess) return e;
    return launch_p<P>(g, terms, ld, plan, counters, s);
}

}  // namespace

bool fp8_weight_grad_reads(const void* dy, int dy_type, int64_t ldy) { return rows_by_tma(dy, dy_type, ldy); }

size_t fp8_weight_grad_workspace_bytes(int64_t M, int64_t N, int64_t K, int dy_type, bool terms) {
    const Plan plan = plan_of(M, N, K, dy_type);
    return arrived_bytes(plan, N, K) + part_bytes(plan, N, K) + (terms ? terms_bytes(M, N, dy_type) : 0);
}

Fp8Plan fp8_weight_grad_plan(int64_t M, int64_t N, int64_t K, int dy_type) {
    const Plan plan = plan_of(M, N, K, dy_type);
    return Fp8Plan{false, plan.tk, plan.splits};
}

cudaError_t launch_fp8_weight_grad(const Fp8WeightGrad& g, void* workspace, cudaStream_t s) {
    if (g.M == 0) {
        if (g.accumulate) return cudaSuccess;
        const int64_t n = (g.N * g.K + 255) / 256;
        const unsigned grid = (unsigned)(n < 65536 ? n : 65536);
        if (g.out_type == kF16) zero_rows_kernel<<<grid, 256, 0, s>>>(static_cast<__half*>(g.out), g.N, g.K, g.ldo);
        else if (g.out_type == kBf16)
            zero_rows_kernel<<<grid, 256, 0, s>>>(static_cast<__nv_bfloat16*>(g.out), g.N, g.K, g.ldo);
        else zero_rows_kernel<<<grid, 256, 0, s>>>(static_cast<float*>(g.out), g.N, g.K, g.ldo);
        return cudaGetLastError();
    }
    const Plan plan = plan_of(g.M, g.N, g.K, g.dy_type);
    unsigned char* counters = static_cast<unsigned char*>(workspace);
    if (g.dy_type == kF32) return split_and_launch<float, 3>(g, counters, plan, s);
    if (g.dy_type == kF16) return split_and_launch<__half, 2>(g, counters, plan, s);
    if (!rows_by_tma(g.dy, g.dy_type, g.ldy)) return split_and_launch<__nv_bfloat16, 1>(g, counters, plan, s);
    if (plan.splits > 1) {
        cudaError_t e = cudaMemsetAsync(counters, 0, arrived_bytes(plan, g.N, g.K), s);
        if (e != cudaSuccess) return e;
    }
    return launch_p<1>(g, g.dy, g.ldy, plan, counters, s);
}

}  // namespace wq
