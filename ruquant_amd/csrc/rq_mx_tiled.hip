// MXFP4 product for many tokens: tiles of rows x tokens, both operands through LDS.
//
// y[m][n] = sum over blocks b of 32 inputs of 2^(X_mb + X_nb - 254) sum_k x^[m][k] w[n][k]: the scaled MFMA does a run of two blocks for
// 32 x 32 outputs in one instruction, scales included, sums in fp32. Both operands lie in memory as the MFMA takes them (rq_mx.h), so a
// tile's loads are whole runs of 1 KiB that go to LDS without passing registers, a ring of R steps of 128 inputs ahead, and its reads of
// LDS are 16 bytes a lane in a row, free of conflicts. A step of a wavefront with RB x TB blocks reads 2 (RB + TB) fragments for 2 RB TB
// MFMAs: LDS delivers a fragment in 16 clocks (64 bytes each), in which the four SIMDs do one and a half MFMAs, so 4 x 2 blocks (12 reads in
// 192 clocks, 16 MFMAs in 170) are bound by LDS and MFMA nearly alike, and registers end there (128 accumulators and two steps' fragments
// of 256).
// 2048 tokens x 17408 x 5120: 85 us for the 512 tiles of 256 x 256 that are two rounds of the chip, 4.0 PFLOP/s, the MFMAs busy for 48 % of the
// cycles (a plain bf16 library product of 8192^3 here: 1.16), and 12 us for the rows behind them. 64 tokens x 17408 x 5120 is 12.2 us
// behind the quantiser's 3.2, 47 MB of weights at 3.9 TB/s.
// Tried and dropped: 16x16x128 MFMAs (4.4 to 5.5 PFLOP/s in registers against 7.0 to 7.8); the weights' fragments from L1 in place of
// LDS; deeper rings for the large forms.
#include <type_traits>

#include "rq_mx.h"

namespace rq {
namespace mx {
namespace {

// 64 lanes x 16 bytes to 1 KiB of LDS at `lds` (wave-uniform; the hardware adds lane * 16). Assembly, so that the count of
// outstanding loads is this file's (the waits of the steps); nothing is written to registers.
__device__ __forceinline__ void load_run(const uint8_t *from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(from), "s"(__builtin_amdgcn_readfirstlane((int) lds)) : "memory", "m0");
}
__device__ __forceinline__ void load_run(const uint8_t *base, uint32_t lane_off, uint32_t lds) {   // base: wave-uniform
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(lane_off), "s"(base), "s"(__builtin_amdgcn_readfirstlane((int) lds)) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
__device__ __forceinline__ void barrier() {
    asm volatile("s_barrier" : : : "memory");
}
__device__ __forceinline__ const uint8_t *uniform(const uint8_t *p) {
    const uint64_t b = (uint64_t) (uintptr_t) p;
    return reinterpret_cast<const uint8_t *>(
        (uintptr_t) ((uint64_t) (uint32_t) __builtin_amdgcn_readfirstlane((int) (uint32_t) b) |
                     (uint64_t) (uint32_t) __builtin_amdgcn_readfirstlane((int) (uint32_t) (b >> 32)) << 32));
}

// Wavefront (wr, wc) of 2 x WC has RB blocks of 32 rows x TB of 32 tokens. kGateUp: RB / 2 of each projection, so that a lane holds
// both values of a row of h. R: slots of the ring of steps in LDS.
template <int MODE, int RB, int TB, int WC, int R>
struct Tiled {
    static constexpr int kWaves = 2 * WC, kThreads = 64 * kWaves;
    static constexpr int kABlocks = 2 * RB, kBBlocks = WC * TB;
    static constexpr int kSlot = (kABlocks + kBBlocks) * 2048;   // one step of both operands
    // Behind the ring the scales, a part (two steps) a slot: row blocks, then token blocks, 256 bytes each, moved four at a time.
    static constexpr int kScaleRuns = (kABlocks + kBBlocks + 3) / 4, kScaleSlot = kScaleRuns * 1024, kScaleSlots = (R + 1) / 2;
    static constexpr int kScales = R * kSlot, kBytes = kScales + kScaleSlots * kScaleSlot;
    // 1 KiB each, of a wavefront per step, and of a part's scales (some are fetched twice so that all fetch as many)
    static constexpr int kARuns = 2 * kABlocks / kWaves, kBRuns = 2 * kBBlocks / kWaves, kRuns = kARuns + kBRuns;
    static constexpr int kPartRuns = (kScaleRuns + kWaves - 1) / kWaves;
    static_assert(2 * kABlocks % kWaves == 0 && 2 * kBBlocks % kWaves == 0, "split of the loads");
    static constexpr int kTileRows = MODE == kGateUp ? 32 * RB : 64 * RB;            // (of each matrix)
    static constexpr int kTileTokens = 32 * WC * TB;

    // what this wavefront moves
    const uint8_t *a_src[kARuns], *b_src[kBRuns];   // wave-uniform
    const uint8_t *s_src[kPartRuns];                // the lane's
    uint32_t       lds0, lane16;
    int            wave, wr, wc, lane, steps;
    const uint8_t *a_lds, *b_lds, *as_lds, *bs_lds;   // this lane's places in slot 0
    v16f           acc[RB][TB];
    v4i            A[RB][2];
    int            sA[RB];

    __device__ __forceinline__ void fetch_run(int t, int slot, int i) {
        const uint32_t to = lds0 + slot * kSlot;
        if (i < kARuns) load_run(a_src[i] + (int64_t) t * 2048, lane16, to + (wave * kARuns + i) * 1024);
        else load_run(b_src[i - kARuns] + (int64_t) t * 2048, lane16, to + (2 * kABlocks + wave * kBRuns + i - kARuns) * 1024);
    }
    static __device__ __forceinline__ int scale_slot(int part) { return part % kScaleSlots * kScaleSlot; }
    __device__ __forceinline__ void fetch_scales(int part) {
#pragma unroll
        for (int i = 0; i < kPartRuns; ++i)
            load_run(s_src[i] + (int64_t) part * 256, lds0 + kScales + scale_slot(part) + (i * kWaves + wave) % kScaleRuns * 1024);
    }
    __device__ __forceinline__ void read_a(int slot, int i) {
#pragma unroll
        for (int h = 0; h < 2; ++h) A[i][h] = *reinterpret_cast<const v4i *>(a_lds + slot * kSlot + (2 * i + h) * 1024);
    }
    __device__ __forceinline__ void read_b(v4i (&B)[TB][2], int slot, int i) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) B[i][h] = *reinterpret_cast<const v4i *>(b_lds + slot * kSlot + (2 * i + h) * 1024);
    }
    __device__ __forceinline__ void read_sa(int part, int i) { sA[i] = *reinterpret_cast<const int *>(as_lds + scale_slot(part) + i * 256); }
    __device__ __forceinline__ void read_sb(int (&sB)[TB], int part, int i) const {
        sB[i] = *reinterpret_cast<const int *>(bs_lds + scale_slot(part) + i * 256);
    }

    // Step t (t % 2 == J): its products from A and B, behind each row block's the read of its fragments of step t + 1, between them the
    // reads of step t + 1's activations into N and the fetch of step t + R - 1 into the slot of step t - 1. Who has passed this step's
    // barrier has issued the products of step t - 1, which waited for that slot's reads. The scales of part q are read by step 2 q - 1
    // and waited for by the products of step 2 q; part p is fetched with step 2 p, behind the barrier of step 2 p - R + 1, into the slot of part
    // p - S, whose reads are past from the barrier of step 2 (p - S) + 1 on: 2 S >= R. MORE: all of those steps exist.
    template <bool ACTIVE, int J, bool MORE>
    __device__ __forceinline__ void step(int t, int slot, const v4i (&B)[TB][2], v4i (&N)[TB][2], int (&sB)[TB], int (&sN)[TB]) {
        const int  next = slot + 1 == R ? 0 : slot + 1, last = slot == 0 ? R - 1 : slot - 1;
        const bool get = MORE || t + R - 1 < steps;
        // step t + 1 has arrived; those behind it need not have
        constexpr int kParts = (J + R - 2) / 2 - (J + 1) / 2;   // first steps of a part, which bring its scales, among those
        if (MORE || t + R - 2 < steps) wait_loads<(R - 3) * kRuns + kParts * kPartRuns>();
        else wait_loads<0>();
        barrier();
        if ((J + R - 1) % 2 == 0 && get) fetch_scales((t + R - 1) >> 1);
        if (!MORE && get) {
#pragma unroll
            for (int i = 0; i < kRuns; ++i) fetch_run(t + R - 1, last, i);
        }
#pragma unroll
        for (int r = 0; r < RB; ++r) {
            if constexpr (ACTIVE) {
#pragma unroll
                for (int b = 0; b < TB; ++b) acc[r][b] = mfma<2 * J>(A[r][0], B[b][0], acc[r][b], sA[r], sB[b]);
                // (past the last step: what the ring holds, for nobody)
#pragma unroll
                for (int i = r * TB / RB; i < (r + 1) * TB / RB; ++i) {
                    read_b(N, next, i);
                    if (J == 1) read_sb(sN, (t >> 1) + 1, i);
                }
            }
            if (MORE) {
#pragma unroll
                for (int i = r * kRuns / RB; i < (r + 1) * kRuns / RB; ++i) fetch_run(t + R - 1, last, i);
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (ACTIVE) {
#pragma unroll
                for (int b = 0; b < TB; ++b) acc[r][b] = mfma<2 * J + 1>(A[r][1], B[b][1], acc[r][b], sA[r], sB[b]);
                read_a(next, r);
                if (J == 1) read_sa((t >> 1) + 1, r);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (ACTIVE && J == 1) {
#pragma unroll
            for (int i = 0; i < TB; ++i) sB[i] = sN[i];
        }
    }

    // ACTIVE: this wavefront has tokens; otherwise it moves its share and keeps the barriers
    template <bool ACTIVE>
    __device__ __forceinline__ void loop() {
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int t = 0; t < TB; ++t) acc[r][t] = v16f{ 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0 };
#pragma unroll
        for (int t = 0; t < R - 1; ++t) {
            if (t < steps) {
                if (t % 2 == 0) fetch_scales(t >> 1);
#pragma unroll
                for (int i = 0; i < kRuns; ++i) fetch_run(t, t, i);
            }
        }
        if (steps >= R - 1) wait_loads<(R - 2) * kRuns + (R - 2) / 2 * kPartRuns>();
        else wait_loads<0>();
        barrier();
        v4i B[TB][2], N[TB][2];
        int sB[TB], sN[TB];
#pragma unroll
        for (int i = 0; i < RB; ++i) read_a(0, i), read_sa(0, i);
#pragma unroll
        for (int i = 0; i < TB; ++i) read_b(B, 0, i), read_sb(sB, 0, i);
        int  t = 0, slot = 0;
        auto next = [&]() __attribute__((always_inline)) { ++t, slot = slot + 1 == R ? 0 : slot + 1; };
        while (t + R < steps) {
            step<ACTIVE, 0, true>(t, slot, B, N, sB, sN), next();
            step<ACTIVE, 1, true>(t, slot, N, B, sB, sN), next();
        }
        while (true) {
            step<ACTIVE, 0, false>(t, slot, B, N, sB, sN), next();
            if (t >= steps) break;
            step<ACTIVE, 1, false>(t, slot, N, B, sB, sN), next();
            if (t >= steps) break;
        }
        wait_loads<0>();   // (none of this wavefront's loads lands in LDS behind this)
    }
};

// SPLIT: a.splits workgroups share a tile's inputs, a.split_steps steps each. Each wavefront leaves its sums, as they lie in its registers,
// in the workspace and counts itself in; the last of those that hold the same outputs adds them up, in the order of the inputs, so
// that the bits do not depend on who is last. The sums go past the XCDs' caches (atomic stores and loads of the device's scope) and
// are waited for before the count, so who sees the last count sees all sums. (With fences instead, which write a whole L2 back for every
// wavefront: 512 outputs of 17408 inputs, 64 tokens, 4 parts 13.7 us, 16 parts 17.2, 2048 outputs, 8 parts 29.4; so 13.6, 16.1, 16.4.
// Unshared 22.0 and 22.5.)
template <int MODE, int RB, int TB, int WC, int R, bool SPLIT>
__global__ __launch_bounds__(128 * WC, WC == 4 ? 2 : RB * TB <= 2 ? 2 : RB * TB <= 4 ? 3 : 2) void rq_mx_tiled_kernel(const ProductArgs a, const int row_tiles, const int token_tiles, const int across) {
    using G = Tiled<MODE, RB, TB, WC, R>;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    // Workgroups go to the XCDs in turn. Each XCD takes a run of the tiles in an order in which the token tiles run fastest, so that
    // those that share rows of the weight share an L2.
    const int total = row_tiles * token_tiles * (SPLIT ? a.splits : 1);
    // (A plain product's grid is one row: in the tiles that large ones take, outputs that made it too wide fit no memory, and the test costs 0.25 us. across: a
    // multiple of 8 where there is more than one row.)
    const int index = MODE == kDense ? (int) blockIdx.x : (int) blockIdx.y * across + (int) blockIdx.x;
    if (MODE != kDense && index >= total) return;
    const int xcd = index & 7, each = total >> 3, more = total & 7;
    const int place_of = xcd * each + min(xcd, more) + (index >> 3);
    const int v = SPLIT ? place_of / a.splits : place_of, part = SPLIT ? place_of - v * a.splits : 0;
    const int row_tile = v / token_tiles, token_tile = v - row_tile * token_tiles;
    Tile tile = { 0, 0, 0, 0 };
    if constexpr (MODE == kDense) {
        tile.first = token_tile * G::kTileTokens;
        tile.count = (int) (a.M - tile.first < G::kTileTokens ? a.M - tile.first : G::kTileTokens);
    } else {
        tile = a.tiles[token_tile];
        if (tile.count == 0) return;   // (past the last)
    }
    G g;
    g.lane = threadIdx.x & 63;
    g.wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
    // (a wavefront's number mod 4 is its SIMD: the two that a tile with half of its tokens leaves idle, or the four, are of all of them; with
    // four wavefronts the workgroups take turns)
    g.wr = g.wave & 1;
    g.wc = WC == 2 ? ((g.wave >> 1) ^ (index >> 3)) & 1 : g.wave >> 1;
    g.lane16 = g.lane * 16;
    const int step0 = SPLIT ? part * a.split_steps : 0;   // (a multiple of two: the scales' parts)
    g.steps = SPLIT ? min(a.split_steps, a.L.steps - step0) : a.L.steps;
    g.lds0 = (uint32_t) (uintptr_t) (__attribute__((address_space(3))) void *) lds;
    g.a_lds = lds + g.wr * RB * 2048 + g.lane * 16;
    g.b_lds = lds + (2 * G::kABlocks + g.wc * TB * 2) * 1024 + g.lane * 16;
    g.as_lds = lds + G::kScales + g.wr * RB * 256 + g.lane * 4;
    g.bs_lds = lds + G::kScales + (G::kABlocks + g.wc * TB) * 256 + g.lane * 4;
    constexpr int  kBlocks = G::kTileRows / 32;   // row blocks of the tile, per matrix
    const int      block0 = (MODE == kDense ? a.first_block : 0) + row_tile * kBlocks;
    const uint8_t *w = a.w + (int64_t) tile.expert * a.L.expert_bytes;
    const uint8_t *w2 = MODE == kGateUp ? a.w2 + (int64_t) tile.expert * a.L.expert_bytes : w;
    // row block i of the tile, in the order of its wavefronts: its matrix and place; blocks past the weight's repeat its last one
    auto place = [&](int i) __attribute__((always_inline)) {
        const int b = MODE == kGateUp ? block0 + i / RB * (RB / 2) + i % RB % (RB / 2 > 0 ? RB / 2 : 1) : block0 + i;
        return min(b, a.L.row_blocks - 1);
    };
    auto matrix = [&](int i) __attribute__((always_inline)) { return MODE == kGateUp && i % RB >= RB / 2 ? w2 : w; };
#pragma unroll
    for (int i = 0; i < G::kARuns; ++i) {
        const int run = g.wave * G::kARuns + i;
        g.a_src[i] = uniform(matrix(run >> 1) + (int64_t) place(run >> 1) * a.L.steps * 2048 + (run & 1) * 1024 + (int64_t) step0 * 2048);
    }
    // the tile's token blocks; those past the last repeat it, and those past the activations the activations' last
    const int token0 = tile.first >> 5, token_blocks = min((tile.count + 31) >> 5, a.P.row_blocks - token0);
    auto token_place = [&](int i) __attribute__((always_inline)) { return token0 + min(i, token_blocks - 1); };
#pragma unroll
    for (int i = 0; i < G::kBRuns; ++i) {
        const int run = g.wave * G::kBRuns + i;
        g.b_src[i] = uniform(a.panels + (int64_t) token_place(run >> 1) * a.P.steps * 2048 + (run & 1) * 1024 + (int64_t) step0 * 2048);
    }
#pragma unroll
    for (int i = 0; i < G::kPartRuns; ++i) {   // of four blocks, row blocks first (past the last one it again)
        const int r = min((i * G::kWaves + g.wave) % G::kScaleRuns * 4 + (g.lane >> 4), G::kABlocks + G::kBBlocks - 1);
        g.s_src[i] = (r < G::kABlocks ? matrix(r) + a.L.code_bytes + (int64_t) place(r) * a.L.chunks * 512
                                      : a.panels + a.P.code_bytes + (int64_t) token_place(r - G::kABlocks) * a.P.chunks * 512) + (g.lane & 15) * 16 + step0 * 128;
    }
    if (g.wc * TB * 32 < tile.count) g.template loop<true>();
    else g.template loop<false>();
    const int lane = g.lane, wr = g.wr, wc = g.wc;
    if constexpr (MODE == kGateUp) {
#pragma unroll
        for (int t = 0; t < TB; ++t) {
            const int token = (wc * TB + t) * 32 + (lane & 31);
#pragma unroll
            for (int q = 0; q < RB / 2; ++q) {
                const int b = block0 + wr * (RB / 2) + q;
                if (b < a.L.row_blocks) store_h(a, g.acc[q][t], g.acc[RB / 2 + q][t], lane, token < tile.count, tile.first + token, b);
            }
        }
    } else {
        // 32 tokens x 64 rows at a time through LDS (a region of the wavefront's own), so that a token's outputs leave as whole lines.
        // (Lines written in halves cost much: 2048 x 17408 outputs in bf16, 64 bytes a token and store, 38 us, in fp32 30.)
        constexpr int kStride = 68;
        static_assert(G::kWaves * 32 * kStride * 4 <= G::kBytes, "a region per wavefront");
        float    *mine = reinterpret_cast<float *>(lds) + g.wave * 32 * kStride;
        const int dtype = MODE == kDown ? RQ_F32 : a.out_dtype;
        // (the rows of this wavefront's tokens, a token a lane)
        int64_t row_at[TB];
#pragma unroll
        for (int t = 0; t < TB; ++t) {
            const int token = (wc * TB + t) * 32 + (lane & 31);
            row_at[t] = MODE == kDown ? (token < tile.count ? a.row_of[tile.first + token] : 0) : tile.first + token;
        }
        barrier();   // (the ring is not read any more)
        if (wc * TB * 32 >= tile.count) return;
        if constexpr (SPLIT) {
            constexpr int kPairs = RB * TB * 8;   // 512 bytes each
            const int     outputs = v * G::kWaves + 2 * wc + wr;   // (of the tile's: which wavefront has them differs by workgroup)
            auto         *sums = reinterpret_cast<uint64_t *>(a.sums) + (int64_t) outputs * a.splits * kPairs * 64 + lane;
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
                const float    lo = g.acc[i / 8 / TB][i / 8 % TB][i % 8 * 2], hi = g.acc[i / 8 / TB][i / 8 % TB][i % 8 * 2 + 1];
                const uint64_t x = (uint64_t) __float_as_uint(hi) << 32 | __float_as_uint(lo);
                __hip_atomic_store(sums + (part * kPairs + i) * 64, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            wait_loads<0>();   // (stores count alike: all of them are where every XCD sees them)
            int before = 0;
            if (lane == 0) before = __hip_atomic_fetch_add(a.arrived + outputs, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (__builtin_amdgcn_readfirstlane(before) != a.splits - 1) return;
            asm volatile("" : : : "memory");
            for (int p = 0; p < a.splits; ++p) {
                uint64_t x[kPairs];
#pragma unroll
                for (int i = 0; i < kPairs; ++i)
                    x[i] = __hip_atomic_load(sums + (p * kPairs + i) * 64, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
                for (int i = 0; i < kPairs; ++i) {
                    v16f       &c = g.acc[i / 8 / TB][i / 8 % TB];
                    const float lo = __uint_as_float((uint32_t) x[i]), hi = __uint_as_float((uint32_t) (x[i] >> 32));
                    c[i % 8 * 2] = p ? c[i % 8 * 2] + lo : lo;
                    c[i % 8 * 2 + 1] = p ? c[i % 8 * 2 + 1] + hi : hi;
                }
            }
        }
        // LANES of a token write 16 bytes each
        auto store = [&](auto lanes, int t, int r) __attribute__((always_inline)) {
            constexpr int kLanes = decltype(lanes)::value, kTokens = 64 / kLanes;
            const int     n = lane % kLanes * (dtype == RQ_F32 ? 4 : 8), first = (wc * TB + t) * 32;
            const int64_t n0 = (int64_t) (block0 + wr * RB + r) * 32 + n;
#pragma unroll
            for (int i = 0; i < 32 / kTokens; ++i) {
                const int     at = i * kTokens + lane / kLanes;
                const int64_t row = MODE == kDown ? __shfl((int) row_at[t], at) : tile.first + first + at;
                if (first + at < tile.count) store_out(dtype, a.y, row * a.ldy, n0, a.L.N, mine + at * kStride + n);
            }
        };
#pragma unroll
        for (int t = 0; t < TB; ++t) {
#pragma unroll
            for (int r = 0; r < RB; r += 2) {
                constexpr int kTwo = RB > 1 ? 2 : 1;   // row blocks at a time
                static_assert(RB % kTwo == 0, "row blocks in pairs");
#pragma unroll
                for (int q = 0; q < 4 * kTwo; ++q) {
                    const v16f &c = g.acc[r + q / 4][t];
                    *reinterpret_cast<v4f *>(mine + (lane & 31) * kStride + q * 8 + (lane >> 5) * 4) =
                        v4f{ c[q % 4 * 4], c[q % 4 * 4 + 1], c[q % 4 * 4 + 2], c[q % 4 * 4 + 3] };
                }
                __builtin_amdgcn_wave_barrier();
                if (dtype == RQ_F32) store(std::integral_constant<int, 8 * kTwo>{}, t, r);
                else store(std::integral_constant<int, 4 * kTwo>{}, t, r);
                __builtin_amdgcn_wave_barrier();
            }
        }
    }
}

constexpr int64_t kAcross = 1 << 20;   // workgroups in one dimension of a grid, which may have under 2^32 threads

template <int MODE, int RB, int TB, int WC, int R, bool SPLIT = false>
hipError_t launch(const ProductArgs &a, hipStream_t stream) {
    using G = Tiled<MODE, RB, TB, WC, R>;
    const int row_tiles = MODE == kDense ? a.row_tiles : (int) ((a.L.row_blocks * 32 + G::kTileRows - 1) / G::kTileRows);
    const int token_tiles = MODE == kDense ? (int) ((a.M + G::kTileTokens - 1) / G::kTileTokens) : a.most_tiles;
    const int64_t groups = (int64_t) row_tiles * token_tiles * (SPLIT ? a.splits : 1);
    if (groups > (MODE == kDense ? 0xFFFFFFFFll / G::kThreads : 0x7FFFFFFFll - kAcross)) return hipErrorInvalidConfiguration;
    const unsigned across = (unsigned) (MODE == kDense || groups < kAcross ? groups : kAcross);
    static std::atomic<uint64_t> allowed{ 0 };   // devices on which the kernel may have its LDS
    const hipError_t e = allow_lds(reinterpret_cast<const void *>(rq_mx_tiled_kernel<MODE, RB, TB, WC, R, SPLIT>), G::kBytes, allowed);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((rq_mx_tiled_kernel<MODE, RB, TB, WC, R, SPLIT>), dim3(across, (unsigned) ((groups + across - 1) / across)),
                       dim3(G::kThreads), G::kBytes, stream, a, row_tiles, token_tiles, (int) across);
    return hipGetLastError();
}

template <int MODE>
hipError_t launch_form(int form, const ProductArgs &a, hipStream_t stream) {
    if constexpr (MODE == kDense) {
        switch (form) {
            case 0: return a.splits > 1 ? launch<MODE, 1, 1, 2, 8, true>(a, stream) : launch<MODE, 1, 1, 2, 8>(a, stream);
            case 1: return launch<MODE, 2, 1, 2, 6>(a, stream);
            case 2: return launch<MODE, 2, 2, 2, 6>(a, stream);
            case 3: return launch<MODE, 2, 2, 2, 3>(a, stream);
            case 4: return launch<MODE, 2, 2, 4, 5>(a, stream);
            default: return launch<MODE, 4, 2, 4, 4>(a, stream);
        }
    } else {
        if (form == kForm64) return launch<MODE, 2, 1, 2, 6>(a, stream);
        if (form == kForm128) return launch<MODE, 2, 2, 2, 3>(a, stream);
        return launch<MODE, 4, 2, 2, 3>(a, stream);
    }
}

// The forms, and what their tiles take in microseconds: a step of 128 inputs with one tile on a compute unit, a step of every tile of
// many, and what stands in front of and behind the steps. Measured over K = 1024, 5120, 17408, N = 512 to 17408 and 20 to 2048 tokens:
// the form that these numbers choose is 1.7 % slower than the fastest of nine on average, 30 % at worst (deep rings cover the latency
// of few tiles, large tiles spare LDS and L2 where there are many); with what plan_product makes of them, from K = 256 and N = 64 on and 17
// to 512 tokens, within 5 % of the fastest form and split in 212 of 216 places, 9 % behind at worst.
struct Form {
    int    rows, tokens, resident;   // a tile; tiles that a compute unit holds (of the fourth form three, but two fit its times)
    double alone, full, fixed;
};
constexpr Form kForms[kTiledForms] = { { 64, 64, 2, .098, .155, 2.0 },   { 128, 64, 2, .131, .212, 2.2 },  { 128, 128, 1, .187, .358, 2.6 },
                                       { 128, 128, 2, .405, .310, 2.2 }, { 128, 256, 1, .295, .635, 4.0 }, { 256, 256, 1, .470, .866, 6.0 },
                                       { 256, 128, 2, 0, 0, 0 } };   // (the last one for the experts only)

}  // namespace

int tiled_rows(int form) { return kForms[form].rows; }
int tiled_tokens(int form) { return kForms[form].tokens; }
int tiled_resident(int form) { return kForms[form].resident; }
int64_t tiled_row_tiles(int mode, int form, int64_t N) {
    const int rows = mode == kGateUp ? kForms[form].rows / 2 : kForms[form].rows;
    return (N + rows - 1) / rows;
}
namespace {

double price(int form, int64_t tiles, int64_t steps) {
    const Form   &f = kForms[form];
    const int64_t load = (tiles + 255) / 256, rounds = (load + f.resident - 1) / f.resident;   // of the busiest compute unit
    const double  alone = f.alone * (double) rounds, full = load > 1 ? f.full * (double) load : 0;
    return (double) rounds * f.fixed + (double) steps * (full > alone ? full : alone);
}

}  // namespace

constexpr int64_t kUnsplitSteps = 24, kMostSplits = 16, kMostParts = 512;
// At least what any plan for up to M tokens takes.
int64_t product_sums_bytes(int64_t M, int64_t N, int64_t K) {
    if (K <= kUnsplitSteps * 128) return 0;
    const int64_t parts = up_to(N, 64) / 64 * (up_to(M, 64) / 64) * kMostSplits;
    return (parts < kMostParts ? parts : kMostParts) * (4 * 4096 + 16);   // (16: the counters of a tile's wavefronts)
}

// A product is one launch in the form of the least price, or two: as many row tiles as fill whole rounds of the chip in one form, and the
// rows behind them, which would leave most of it idle for a round, in another. (17408 x 5120 at 2048 tokens: 544 tiles of 256 x 256 are
// two rounds and 32 tiles.) Or, where the tiles are few and the inputs many, one whose tiles several workgroups share.
ProductPlan plan_product(int64_t M, int64_t N, int64_t K) {
    constexpr int    kPlain = kTiledForms - 1;
    constexpr double kLaunch = 2.0;
    const int64_t    rows = up_to(N, 64), steps = up_to(K, 128) / 128;
    auto token_tiles = [&](int f) { return (M + kForms[f].tokens - 1) / kForms[f].tokens; };
    auto row_tiles = [&](int f, int64_t n) { return (n + kForms[f].rows - 1) / kForms[f].rows; };
    double      least = 0;
    ProductPlan plan = { -1, -1, 0, 1, 0, 0, 0 };
    for (int f = 0; f < kPlain; ++f) {
        const int64_t tokens = token_tiles(f), all = row_tiles(f, rows);
        const double  whole = price(f, all * tokens, steps);
        if (plan.form < 0 || whole < least) least = whole, plan = { f, -1, all, 1, (int) steps, 0, 0 };
        const int64_t round = 256 * kForms[f].resident, rounds = all * tokens / round;
        for (int64_t k = rounds; k > 0 && k > rounds - 2; --k) {
            const int64_t n = k * round / tokens;   // row tiles
            if (n == 0 || n >= all) continue;
            const double some = price(f, n * tokens, steps) + kLaunch;
            for (int g = 0; g < kPlain; ++g) {
                const double p = some + price(g, row_tiles(g, rows - n * kForms[f].rows) * token_tiles(g), steps);
                if (p < least) least = p, plan = { f, g, n, 1, (int) steps, 0, 0 };
            }
        }
    }
    // (64 x 64 tiles only: larger ones have fewer wavefronts to join as much, and were never faster. The join's time from K = 17408 and 5120,
    // N = 256 to 9000 and 17 to 512 tokens; by it up to kUnsplitSteps never pay.)
    const int64_t tiles = row_tiles(0, rows) * token_tiles(0);
    for (int64_t parts = 2; steps > kUnsplitSteps && parts <= kMostSplits && tiles * parts <= kMostParts; ++parts) {
        const int64_t some = up_to((steps + parts - 1) / parts, 2), n = (steps + some - 1) / some;
        const double  p = price(0, tiles * n, some) + 0.6 + 0.3 * (double) n + 0.008 * (double) (tiles * n);
        if (n > 1 && p < least) least = p, plan = { 0, -1, row_tiles(0, rows), (int) n, (int) some, 0, 0 };
    }
    if (plan.splits > 1) {
        plan.arrived = (int) tiles * 4;   // wavefronts, of 32 x 32 outputs
        plan.sums_bytes = tiles * 4 * plan.splits * 4096;
    }
    return plan;
}

hipError_t launch_tiled_product(const ProductPlan &plan, const ProductArgs &a, hipStream_t stream) {
    ProductArgs one = a;
    one.first_block = 0;
    one.row_tiles = (int) plan.main_tiles;
    one.splits = plan.splits;
    one.split_steps = plan.split_steps;
    hipError_t e = launch_form<kDense>(plan.form, one, stream);
    if (e != hipSuccess || plan.rest < 0) return e;
    const int64_t done = plan.main_tiles * kForms[plan.form].rows;
    one.first_block = (int) (done / 32);
    one.row_tiles = (int) (((int64_t) a.L.row_blocks * 32 - done + kForms[plan.rest].rows - 1) / kForms[plan.rest].rows);
    return launch_form<kDense>(plan.rest, one, stream);
}

hipError_t launch_tiled(int mode, int form, const ProductArgs &a, hipStream_t stream) {
    return mode == kGateUp ? launch_form<kGateUp>(form, a, stream) : launch_form<kDown>(form, a, stream);
}

}  // namespace mx
}  // namespace rq
