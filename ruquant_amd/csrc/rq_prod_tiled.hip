// Products of many rows (int8, or grouped by expert): tiles of rows of the weight x rows of x, both operands through LDS.
//
// Loads go from memory to LDS without passing registers, rings of steps of 64 bytes ahead. The weight lies in memory as
// the matrix instructions take it. Rows of x lie as they are, wherever the call's indices say, so that nothing copies them together:
// a load takes 128 bytes, two steps, of each of 8 rows, and which 16 of those bytes go to which place of the row in LDS turns with the row,
// so that the reads of a fragment, the same bytes of 32 rows, meet different banks. (64 bytes of 16 rows, half lines: 128 x 128 272 -> 234 us, grouped
// bf16 299 -> 275.)
//
// What bounds it: a full chip of 256 x 256 tiles does 2.1 to 2.3 POP/s in int8 and 1.25 PFLOP/s in bf16, 2048 x 16384 x 5120 151 to 168 us by card, where a large library product
// does 2.1 to 2.5 and 1.38 to 1.57: the chip's clock falls to that (codes of zeros are done at 3.3). Small tiles wait for LDS, which delivers 64 bytes a clock
// (128 x 128: 48 KiB a step for 256 clocks of products), and for their first loads.
// Tried and dropped: the weight's fragments from memory straight into registers, four steps ahead (252 us for 162); 4 x 4 blocks by each of four wavefronts (175 for 165);
// 256 x 128 tiles, two a compute unit (188 for 166, and at best 5 % faster for experts of 125 rows); groups cut evenly into their tiles (no change).
#include <type_traits>

#include "rq_prod.h"

namespace rq {
namespace prod {
namespace {

__device__ __attribute__((aligned(16))) const uint8_t kZeros[16] = { 0 };

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

// Wavefront (wr, wc) of WR x WC has RB blocks of 32 rows x TB of 32 positions. In LDS S slots of pairs of steps of x and RA slots of steps of the weight.
template <int WT, int RB, int TB, int WR, int WC, int S, int RA>
struct Tiled {
    using Acc = typename Matrix<WT>::Acc;
    static constexpr int kWaves = WR * WC, kThreads = 64 * kWaves;
    static constexpr int kABlocks = WR * RB, kBBlocks = WC * TB;
    static constexpr int kSlotA = kABlocks * 2048, kSlotB = kBBlocks * 4096;   // a step of the weight, a pair of steps of x
    static constexpr int kRingA = RA * kSlotA, kRing = kRingA + S * kSlotB, kStride = 68, kOut = kWaves * 32 * kStride * 4;   // (of the outputs on their way out)
    static constexpr int kBytes = kRing > kOut ? kRing : kOut;
    static constexpr int kARuns = 2 * kABlocks / kWaves, kBRuns = 4 * kBBlocks / kWaves;   // 1 KiB each, of a wavefront per step and per pair of steps
    static_assert(2 * kABlocks % kWaves == 0 && 4 * kBBlocks % kWaves == 0, "split of the loads");
    static_assert(RA >= 3 && S >= 2 && kBytes <= 163840, "rings");
    static constexpr int kTileRows = 32 * WR * RB, kTileTokens = 32 * WC * TB;

    const uint8_t *a_src[kARuns];   // wave-uniform
    const uint8_t *b_src[kBRuns];   // the lane's
    bool           b_last[2];       // whether the lane's 16 bytes of the last pair of steps are of the row, for its even and odd runs
    uint32_t       lds0, lane16;
    int            wave, wr, wc, lane, steps;
    const uint8_t *a_lds;           // this lane's place in slot 0
    const uint8_t *b_lds[4];        // of the runs of a pair of steps
    Acc            acc[RB][TB];

    __device__ __forceinline__ void fetch_a(int t, int slot, int i) {
        load_run(a_src[i] + (int64_t) t * 2048, lane16, lds0 + slot * kSlotA + (wave * kARuns + i) * 1024);
    }
    // pair q of steps
    template <bool LAST>
    __device__ __forceinline__ void fetch_b(int q, int slot, int i) {
        const uint8_t *from = b_src[i] + (int64_t) q * 128;
        if (LAST && q == (steps - 1) >> 1 && !b_last[(wave * kBRuns + i) & 1]) from = kZeros;
        load_run(from, lds0 + kRingA + slot * kSlotB + (wave * kBRuns + i) * 1024);
    }
    __device__ __forceinline__ v4i read_a(int slot, int i, int h) const { return *reinterpret_cast<const v4i *>(a_lds + slot * kSlotA + (2 * i + h) * 1024); }
    template <int J>
    __device__ __forceinline__ v4i read_b(int slot, int i, int h) const {
        return *reinterpret_cast<const v4i *>(b_lds[2 * J + h] + slot * kSlotB + i * 4096);
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int t = 0; t < TB; ++t) acc[r][t] = Acc{ 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0 };
    }

    // Step t fetches the pair of steps that begins at t + 2 S - 2, if t is even, and behind it the weight's of t + RA - 1, each into the slot that step t - 1
    // was the last to use: who has passed step t's barrier has issued the products of step t - 1, which waited for its reads. In front of its barrier step t
    // waits for what step t + 1 needs, whose fragments it reads: `behind` counts what was fetched since, by the parity J of t, and need not be there.
    static constexpr bool kBoth = RB * TB <= 4;   // fragments of both operands are held twice
    static constexpr int even_steps(int J, int back) {   // of the `back` steps in front of t
        int n = 0;
        for (int k = 1; k <= back; ++k) n += (J + k) % 2 == 0;
        return n;
    }
    static constexpr int behind(int J) {
        const int a = RA - 3;                                // steps whose fetches all stand behind the weight's of t + 1
        const int b = 2 * S - 4;                             // J == 1: ... behind the pair of t + 1, the weight's beside it too
        const int by_a = a * kARuns + even_steps(J, a) * kBRuns, by_b = (b + 1) * kARuns + even_steps(J, b) * kBRuns;
        return J == 0 || by_a < by_b ? by_a : by_b;
    }
    // (a fetch past the last step is not made, and the count would be wrong)
    template <int J, bool MORE>
    __device__ __forceinline__ void wait_for_next(int t) const {
        if (MORE || (t + RA - 2 < steps && t + 2 * S - 3 < steps)) wait_loads<behind(J)>();
        else wait_loads<0>();
    }
    // i-th fetch of step t: x's first
    __device__ __forceinline__ void fetch_new(int i, int pairs, int t, int slot_a, int slot_b) {
        if (i < pairs) fetch_b<false>((t >> 1) + S - 1, slot_b, i);
        else fetch_a(t + RA - 1, slot_a, i - pairs);
    }
    // Where a wavefront has few blocks the reads stand in front, so that the rest of the step's products hide them; where it has eight, registers do not
    // hold both steps' A (NA is A), and a row block's is read behind its products. MORE: all of those steps exist, and the pair fetched is not the last.
    template <bool ACTIVE, int J, bool MORE>
    __device__ __forceinline__ void step(int t, int sa, int sb, v4i (&A)[RB][2], const v4i (&B)[TB][2], v4i (&NA)[RB][2], v4i (&NB)[TB][2]) {
        const int next_a = sa + 1 == RA ? 0 : sa + 1, last_a = sa == 0 ? RA - 1 : sa - 1;
        const int next_b = J == 0 ? sb : sb + 1 == S ? 0 : sb + 1, last_b = sb == 0 ? S - 1 : sb - 1;
        wait_for_next<J, MORE>(t);
        barrier();
        if (!MORE) {
            if (J == 0 && t + 2 * S - 2 < steps)
#pragma unroll
                for (int i = 0; i < kBRuns; ++i) fetch_b<true>((t >> 1) + S - 1, last_b, i);
            if (t + RA - 1 < steps)
#pragma unroll
                for (int i = 0; i < kARuns; ++i) fetch_a(t + RA - 1, last_a, i);
        }
        // One read or fetch behind each product, as far as there are products: a wavefront issues in order, and a run of fetches would leave the matrix
        // core idle while they queue.
        constexpr int kX = MORE && J == 0 ? kBRuns : 0, kNew = kX + (MORE ? kARuns : 0);
        if constexpr (!ACTIVE) {
#pragma unroll
            for (int i = 0; i < kNew; ++i) fetch_new(i, kX, t, last_a, last_b);
            return;
        }
#pragma unroll
        for (int r = 0; r < RB; ++r) {
            // of this row block's share: A's fragments of the row block in front (of all, where A is held twice), B's, fetches
            // (past the last step the fragments are what the rings hold, for nobody)
            const int a0 = kBoth ? 2 * RB * r / RB : r == 0 ? 0 : 2 * (r - 1), a1 = kBoth ? 2 * RB * (r + 1) / RB : 2 * r;
            const int b0 = 2 * TB * r / RB, b1 = 2 * TB * (r + 1) / RB, f0 = kNew * r / RB, f1 = kNew * (r + 1) / RB;
            const int ops = a1 - a0 + b1 - b0 + f1 - f0;
#pragma unroll
            for (int m = 0; m < 2 * TB; ++m) {
                const int h = m / TB, b = m % TB;
                acc[r][b] = Matrix<WT>::mfma(A[r][h], B[b][h], acc[r][b]);
#pragma unroll
                for (int k = ops * m / (2 * TB); k < ops * (m + 1) / (2 * TB); ++k) {
                    if (k < b1 - b0) {
                        const int i = b0 + k;
                        NB[i >> 1][i & 1] = read_b<1 - J>(next_b, i >> 1, i & 1);
                    } else if (k < b1 - b0 + a1 - a0) {
                        const int i = a0 + k - (b1 - b0);
                        NA[i >> 1][i & 1] = read_a(next_a, i >> 1, i & 1);
                    } else {
                        fetch_new(f0 + k - (b1 - b0) - (a1 - a0), kX, t, last_a, last_b);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if constexpr (!kBoth) {
#pragma unroll
            for (int h = 0; h < 2; ++h) NA[RB - 1][h] = read_a(next_a, RB - 1, h);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // ACTIVE: this wavefront has positions; otherwise it moves its share and keeps the barriers
    template <bool ACTIVE>
    __device__ __forceinline__ void loop() {
        clear();
        constexpr int kAhead = RA > 2 * S - 1 ? RA : 2 * S;
#pragma unroll
        for (int t = -kAhead; t < 0; ++t) {   // (as the steps in front of the first would)
            if (t % 2 == 0 && t / 2 + S - 1 >= 0 && t + 2 * S - 2 < steps)
#pragma unroll
                for (int i = 0; i < kBRuns; ++i) fetch_b<true>(t / 2 + S - 1, t / 2 + S - 1, i);
            if (t + RA - 1 >= 0 && t + RA - 1 < steps)
#pragma unroll
                for (int i = 0; i < kARuns; ++i) fetch_a(t + RA - 1, t + RA - 1, i);
        }
        wait_for_next<1, false>(-1);
        barrier();
        v4i A[RB][2], NA[kBoth ? RB : 1][2], B[TB][2], NB[TB][2];
        auto &A2 = [&]() -> v4i(&)[RB][2] {
            if constexpr (kBoth) return NA;
            else return A;
        }();
#pragma unroll
        for (int i = 0; i < 2 * RB; ++i) A[i >> 1][i & 1] = read_a(0, i >> 1, i & 1);
#pragma unroll
        for (int i = 0; i < 2 * TB; ++i) B[i >> 1][i & 1] = read_b<0>(0, i >> 1, i & 1);
        int  t = 0, sa = 0, sb = 0;
        auto next = [&](bool pair) __attribute__((always_inline)) {
            ++t, sa = sa + 1 == RA ? 0 : sa + 1;
            if (pair) sb = sb + 1 == S ? 0 : sb + 1;
        };
        while (t + RA < steps && t + 2 * S - 2 < ((steps - 1) & ~1)) {
            step<ACTIVE, 0, true>(t, sa, sb, A, B, A2, NB), next(false);
            step<ACTIVE, 1, true>(t, sa, sb, A2, NB, A, B), next(true);
        }
        while (true) {
            step<ACTIVE, 0, false>(t, sa, sb, A, B, A2, NB), next(false);
            if (t >= steps) break;
            step<ACTIVE, 1, false>(t, sa, sb, A2, NB, A, B), next(true);
            if (t >= steps) break;
        }
        wait_loads<0>();   // (none of this wavefront's loads lands in LDS behind this)
    }
};

// Workgroups go to the XCDs in turn: each takes a run of the tiles, so that those next to each other share an L2.
__device__ __forceinline__ int place_of(int index, int total) {
    const int xcd = index & 7, each = total >> 3, more = total & 7;
    return xcd * each + min(xcd, more) + (index >> 3);
}

// SPLIT: a.splits workgroups share a tile's bytes, a.split_steps steps each. Each wavefront leaves its sums, as they lie in its registers, in the
// workspace and counts itself in; the last of those that hold the same outputs adds them up, in the order of the bytes, so that the bits do
// not depend on who is last. The sums go past the XCDs' caches (atomic stores and loads of the device's scope) and are waited for before the count, so
// who sees the last count sees all sums.
template <int WT, int RB, int TB, int WR, int WC, int S, int RA, bool GROUPED, bool SPLIT>
__global__ __launch_bounds__(64 * WR * WC, RB * TB > 8 ? 1 : 2) void rq_tiled_kernel(const ProductArgs a, const int row_tiles, const int token_tiles,
                                                                                                 const int across) {
    using G = Tiled<WT, RB, TB, WR, WC, S, RA>;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int index = (int) blockIdx.y * across + (int) blockIdx.x;
    const int splits = SPLIT ? a.splits : 1;
    int       e = 0, first, count, row_tile, v;   // v: which tile of all, then which part of it
    if constexpr (GROUPED) {
        // The groups one behind the other; in a group, for each run of rows of its weight the tiles of its positions, which start together on one XCD
        // and read the weight together.
        constexpr int T = G::kTileTokens;
        auto units = [&](int n) { return (n + T - 1) / T * row_tiles * splits; };
        int  gfirst, gcount, place;
        v = -1;
        auto mine = [&](int total) { return index < total ? v = place_of(index, total) : -1; };
        if (!find_group<true>(a, units, mine, e, gfirst, gcount, place)) return;
        if (v / splits >= row_tiles * token_tiles) return;   // (more than there can be: the offsets overlap)
        place /= splits;
        const int tiles = (gcount + T - 1) / T, tile = place % tiles;
        row_tile = place / tiles;
        first = gfirst + tile * T;
        count = min(T, gcount - tile * T);
    } else {
        const int total = row_tiles * token_tiles * splits;
        if (index >= total) return;
        v = place_of(index, total);
        row_tile = v / splits / token_tiles;
        first = (v / splits - row_tile * token_tiles) * G::kTileTokens;
        count = (int) (a.P - first < G::kTileTokens ? a.P - first : G::kTileTokens);
    }
    const int part = SPLIT ? v % splits : 0;
    v /= splits;
    G g;
    g.lane = threadIdx.x & 63;
    g.wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
    g.wr = g.wave % WR;
    // (with four wavefronts the workgroups take turns in which SIMDs a tile with half of its positions leaves idle)
    g.wc = WR == 2 && WC == 2 ? ((g.wave >> 1) ^ (index >> 3)) & 1 : g.wave / WR;
    g.lane16 = g.lane * 16;
    const int step0 = SPLIT ? part * a.split_steps : 0;   // (even: the pairs of steps)
    g.steps = SPLIT ? min(a.split_steps, a.L.steps - step0) : a.L.steps;
    g.lds0 = (uint32_t) (uintptr_t) (__attribute__((address_space(3))) void *) lds;
    g.a_lds = lds + g.wr * RB * 2048 + g.lane * 16;
    // A row keeps its bytes 16 c .. + 15 at place c ^ (row / 2 % 8) of its 128: 16 rows' same bytes lie in 16 places of the banks' 256 bytes.
    {
        const int      row = g.lane & 31, turn = (row >> 1) & 7, half = g.lane >> 5;
        const uint8_t *b = lds + G::kRingA + g.wc * TB * 4096 + row * 128;
#pragma unroll
        for (int i = 0; i < 4; ++i) g.b_lds[i] = b + ((2 * i + half) ^ turn) * 16;
    }
    const int      block0 = a.first_block + row_tile * G::kABlocks;
    const uint8_t *w = a.w + (int64_t) e * a.L.expert_bytes;
#pragma unroll
    for (int i = 0; i < G::kARuns; ++i) {   // (blocks past the weight's repeat its last one)
        const int run = g.wave * G::kARuns + i, block = min(block0 + (run >> 1), a.L.row_blocks - 1);
        g.a_src[i] = uniform(w + ((int64_t) block * a.L.steps + step0) * 2048 + (run & 1) * 1024);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) g.b_last[i] = (int64_t) ((step0 + g.steps - 1) >> 1) * 128 + ((g.lane & 7) ^ (i * 4 + (g.lane >> 4))) * 16 < a.x_bytes;
#pragma unroll
    for (int i = 0; i < G::kBRuns; ++i) {   // (positions past the last repeat it)
        const int     run = g.wave * G::kBRuns + i, at = min(run * 8 + (g.lane >> 3), count - 1);
        const int64_t row = row_read(a, first + at);
        g.b_src[i] = a.x + (row < 0 ? 0 : row) * a.pitch + (int64_t) step0 * 64 + ((g.lane & 7) ^ ((run & 1) * 4 + (g.lane >> 4))) * 16;
    }
    // Which rows the outputs are, asked before the products (a position a lane; y's rows are fewer than 2^31).
    const int    lane = g.lane, wr = g.wr, wc = g.wc;
    const float *t_scales = reinterpret_cast<const float *>(w + a.L.code_bytes);
    int          out_at[TB];
    float        s_m[TB];      // of int8
    bool         in_there[TB];
#pragma unroll
    for (int t = 0; t < TB; ++t) {
        const int at = (wc * TB + t) * 32 + (lane & 31);
        out_at[t] = -1, s_m[t] = 0, in_there[t] = false;
        if (at < count) {
            out_at[t] = (int) row_written(a, first + at);
            const int64_t row = row_read(a, first + at);
            in_there[t] = row >= 0;
            if constexpr (WT == RQ_I8)
                if (row >= 0) s_m[t] = a.x_scales[row];
        }
    }
    if (wc * TB * 32 < count) g.template loop<true>();
    else g.template loop<false>();

    // 32 positions x 64 rows at a time through LDS (a region of the wavefront's own), in the output's type, so that a position's outputs
    // leave as whole lines and LDS moves no more than they are.
    barrier();   // (the ring is not read any more)
    if (wc * TB * 32 >= count) return;
    if constexpr (SPLIT) {
        constexpr int kPairs = RB * TB * 8;   // 512 bytes each
        const int     outputs = v * G::kWaves + WR * wc + wr;   // (of the tile's: which wavefront has them differs by workgroup)
        auto         *sums = reinterpret_cast<uint64_t *>(a.sums) + (int64_t) outputs * splits * kPairs * 64 + lane;
        auto          bits = [](auto x) __attribute__((always_inline)) { return __builtin_bit_cast(uint32_t, x); };
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            const auto    &c = g.acc[i / 8 / TB][i / 8 % TB];
            const uint64_t x = (uint64_t) bits(c[i % 8 * 2 + 1]) << 32 | bits(c[i % 8 * 2]);
            __hip_atomic_store(sums + (part * kPairs + i) * 64, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        wait_loads<0>();   // (stores count alike: all of them are where every XCD sees them)
        int before = 0;
        if (lane == 0) before = __hip_atomic_fetch_add(a.arrived + outputs, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (__builtin_amdgcn_readfirstlane(before) != splits - 1) return;
        asm volatile("" : : : "memory");
        for (int p = 0; p < splits; ++p) {
            constexpr int kBatch = kPairs < 16 ? kPairs : 16;   // (more, and the registers do not hold them)
#pragma unroll
            for (int i0 = 0; i0 < kPairs; i0 += kBatch) {
                uint64_t x[kBatch];
#pragma unroll
                for (int i = 0; i < kBatch; ++i)
                    x[i] = __hip_atomic_load(sums + (p * kPairs + i0 + i) * 64, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const int k = i0 + i;
                    auto     &c = g.acc[k / 8 / TB][k / 8 % TB];
                    using E = std::remove_reference_t<decltype(c[0] + c[0])>;
                    const E lo = __builtin_bit_cast(E, (uint32_t) x[i]), hi = __builtin_bit_cast(E, (uint32_t) (x[i] >> 32));
                    c[k % 8 * 2] = p ? c[k % 8 * 2] + lo : lo;
                    c[k % 8 * 2 + 1] = p ? c[k % 8 * 2 + 1] + hi : hi;
                }
            }
        }
    }
    auto write = [&](auto out) __attribute__((always_inline)) {
        constexpr int OT = decltype(out)::value;
        using T = typename Element<OT>::type;
        constexpr int kTwo = RB > 1 ? 2 : 1;                                  // row blocks at a time
        constexpr int kEach = 16 / (int) sizeof(T), kLanes = 32 * kTwo / kEach;   // a lane writes 16 bytes, so many lanes a position
        constexpr int kPlaces = 64 / kLanes, kPitch = 64 + kEach;             // (of elements: 16 bytes behind a position's 64)
        static_assert(RB % kTwo == 0, "row blocks in pairs");
        T *mine = reinterpret_cast<T *>(lds + g.wave * 32 * G::kStride * 4);
#pragma unroll
        for (int r = 0; r < RB; r += kTwo) {
            v4f tn[WT == RQ_I8 ? 4 * kTwo : 1];   // the scales of these rows
            if constexpr (WT == RQ_I8) {
#pragma unroll
                for (int q = 0; q < 4 * kTwo; ++q) {
                    const int block = min(block0 + wr * RB + r + q / 4, a.L.row_blocks - 1);
                    tn[q] = *reinterpret_cast<const v4f *>(t_scales + block * 32 + q % 4 * 8 + (lane >> 5) * 4);
                }
            }
#pragma unroll
            for (int t = 0; t < TB; ++t) {
#pragma unroll
                for (int q = 0; q < 4 * kTwo; ++q) {
                    const auto &c = g.acc[r + q / 4][t];
                    v4f         v;
                    if constexpr (WT == RQ_I8) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = (float) c[q % 4 * 4 + i] * tn[q][i] * s_m[t];
                    } else {
                        v = v4f{ c[q % 4 * 4], c[q % 4 * 4 + 1], c[q % 4 * 4 + 2], c[q % 4 * 4 + 3] };
                    }
                    if (!in_there[t]) v = v4f{ 0, 0, 0, 0 };
                    T *to = mine + (lane & 31) * kPitch + q * 8 + (lane >> 5) * 4;
                    if constexpr (OT == RQ_F32) *reinterpret_cast<v4f *>(to) = v;
                    else *reinterpret_cast<uint2 *>(to) = make_uint2(mx::pair_bits<OT>(v[0], v[1]), mx::pair_bits<OT>(v[2], v[3]));
                }
                __builtin_amdgcn_wave_barrier();
                const int     n = lane % kLanes * kEach;
                const int64_t n0 = (int64_t) (block0 + wr * RB + r) * 32 + n;
                T            *y = reinterpret_cast<T *>(a.y);
#pragma unroll
                for (int i = 0; i < 32 / kPlaces; ++i) {
                    const int     at = i * kPlaces + lane / kLanes;
                    const int64_t row = __shfl(out_at[t], at);
                    const T      *from = mine + at * kPitch + n;
                    if (row < 0 || n0 >= a.L.N) continue;
                    T *to = y + row * a.ldy + n0;
                    if (n0 + kEach <= a.L.N && ((uintptr_t) to & 15) == 0) {
                        *reinterpret_cast<v4i *>(to) = *reinterpret_cast<const v4i *>(from);
                    } else {
#pragma unroll
                        for (int k = 0; k < kEach; ++k)
                            if (n0 + k < a.L.N) to[k] = from[k];
                    }
                }
                __builtin_amdgcn_wave_barrier();
            }
        }
    };
    if (a.out_dtype == RQ_F32) write(std::integral_constant<int, RQ_F32>{});
    else if (a.out_dtype == RQ_F16) write(std::integral_constant<int, RQ_F16>{});
    else write(std::integral_constant<int, RQ_BF16>{});
}

constexpr int64_t kAcross = 1 << 20;   // workgroups in one dimension of a grid, which may have under 2^32 threads

template <int WT, int RB, int TB, int WR, int WC, int S, int RA, bool GROUPED, bool SPLIT = false>
hipError_t launch(const ProductArgs &a, hipStream_t stream) {
    using G = Tiled<WT, RB, TB, WR, WC, S, RA>;
    const int64_t row_tiles = a.row_tiles ? a.row_tiles : (a.L.row_blocks * 32 + G::kTileRows - 1) / G::kTileRows;
    const int64_t token_tiles = most_token_tiles(G::kTileTokens, a.P, GROUPED ? a.E : 0), groups = row_tiles * token_tiles * (SPLIT ? a.splits : 1);
    if (groups > 0x7FFFFFFFll - kAcross) return hipErrorInvalidConfiguration;
    const unsigned across = (unsigned) (groups < kAcross ? groups : kAcross);
    static std::atomic<uint64_t> allowed{ 0 };   // devices on which the kernel may have its LDS
    const hipError_t e = allow_lds(reinterpret_cast<const void *>(rq_tiled_kernel<WT, RB, TB, WR, WC, S, RA, GROUPED, SPLIT>), G::kBytes, allowed);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((rq_tiled_kernel<WT, RB, TB, WR, WC, S, RA, GROUPED, SPLIT>), dim3(across, (unsigned) ((groups + across - 1) / across)),
                       dim3(G::kThreads), G::kBytes, stream, a, (int) row_tiles, (int) token_tiles, (int) across);
    return hipGetLastError();
}

template <int WT, bool GROUPED>
hipError_t launch_form(int form, const ProductArgs &a, hipStream_t stream) {
    if (a.splits > 1) {
        switch (form) {
            case 0: return launch<WT, 1, 1, 2, 2, 4, 9, GROUPED, true>(a, stream);
            case 1: return launch<WT, 2, 1, 2, 2, 3, 7, GROUPED, true>(a, stream);
            default: return launch<WT, 2, 2, 2, 2, 3, 5, GROUPED, true>(a, stream);
        }
    }
    switch (form) {
        case 0: return launch<WT, 1, 1, 2, 2, 4, 9, GROUPED>(a, stream);
        case 1: return launch<WT, 2, 1, 2, 2, 3, 7, GROUPED>(a, stream);
        case 2: return launch<WT, 2, 2, 2, 2, 3, 4, GROUPED>(a, stream);
        case 3: return launch<WT, 2, 2, 2, 2, 3, 5, GROUPED>(a, stream);
        default: return launch<WT, 4, 2, 2, 4, 3, 4, GROUPED>(a, stream);
    }
}
template <bool GROUPED>
hipError_t launch_type(int weight_type, int form, const ProductArgs &a, hipStream_t stream) {
    if (weight_type == RQ_I8) return launch_form<RQ_I8, GROUPED>(form, a, stream);
    if (weight_type == RQ_F16) return launch_form<RQ_F16, GROUPED>(form, a, stream);
    return launch_form<RQ_BF16, GROUPED>(form, a, stream);
}

constexpr int kRowsOf[kForms] = { 64, 128, 128, 128, 256 }, kTokensOf[kForms] = { 64, 64, 128, 128, 256 };

}  // namespace

int tiled_rows(int form) { return kRowsOf[form]; }
int tiled_tokens(int form) { return kTokensOf[form]; }

hipError_t launch_tiled(int weight_type, int form, const ProductArgs &a, hipStream_t stream) {
    if (a.offsets) return launch_type<true>(weight_type, form, a, stream);
    return weight_type == RQ_I8 ? launch_form<RQ_I8, false>(form, a, stream) : hipErrorInvalidValue;
}

}  // namespace prod
}  // namespace rq
