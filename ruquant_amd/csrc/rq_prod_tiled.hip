// Products of many rows (int8, or grouped by expert): tiles of rows of the weight x rows of x, both operands through LDS.
//
// Loads go from memory to LDS without passing registers, a ring of R steps of 64 bytes of both operands ahead. The weight lies in memory as
// the matrix instructions take it. Rows of x lie as they are, wherever the call's indices say, so that nothing copies them together:
// a load takes 64 bytes of each of 16 rows, and which 16 of those 64 bytes go to which place of the row in LDS turns with the row, so
// that the reads of a fragment, the same bytes of 32 rows, meet different banks.
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

// Wavefront (wr, wc) of 2 x WC has RB blocks of 32 rows x TB of 32 positions. R: slots of the ring of steps in LDS.
template <int WT, int RB, int TB, int WC, int R>
struct Tiled {
    using Acc = typename Matrix<WT>::Acc;
    static constexpr int kWaves = 2 * WC, kThreads = 64 * kWaves;
    static constexpr int kABlocks = 2 * RB, kBBlocks = WC * TB;
    static constexpr int kSlot = (kABlocks + kBBlocks) * 2048;   // one step of both operands
    static constexpr int kRing = R * kSlot, kStride = 68, kOut = kWaves * 32 * kStride * 4;   // (of the outputs on their way out)
    static constexpr int kBytes = kRing > kOut ? kRing : kOut;
    static constexpr int kARuns = 2 * kABlocks / kWaves, kBRuns = 2 * kBBlocks / kWaves, kRuns = kARuns + kBRuns;   // 1 KiB each, of a wavefront per step
    static_assert(2 * kABlocks % kWaves == 0 && 2 * kBBlocks % kWaves == 0, "split of the loads");
    static_assert(R >= 3 && kBytes <= 163840, "ring");
    static constexpr int kTileRows = 64 * RB, kTileTokens = 32 * WC * TB;

    const uint8_t *a_src[kARuns];   // wave-uniform
    const uint8_t *b_src[kBRuns];   // the lane's
    bool           b_last;          // whether the lane's 16 bytes of the last step are of the row
    uint32_t       lds0, lane16;
    int            wave, wr, wc, lane, steps;
    const uint8_t *a_lds;           // this lane's place in slot 0
    const uint8_t *b_lds[2];        // of either run of a step
    Acc            acc[RB][TB];
    v4i            A[RB][2];

    template <bool LAST>
    __device__ __forceinline__ void fetch_run(int t, int slot, int i) {
        const uint32_t to = lds0 + slot * kSlot;
        if (i < kARuns) {
            load_run(a_src[i] + (int64_t) t * 2048, lane16, to + (wave * kARuns + i) * 1024);
        } else {
            const uint8_t *from = b_src[i - kARuns] + (int64_t) t * 64;
            if (LAST && t == steps - 1 && !b_last) from = kZeros;
            load_run(from, to + (2 * kABlocks + wave * kBRuns + i - kARuns) * 1024);
        }
    }
    __device__ __forceinline__ void read_a(int slot, int i) {
#pragma unroll
        for (int h = 0; h < 2; ++h) A[i][h] = *reinterpret_cast<const v4i *>(a_lds + slot * kSlot + (2 * i + h) * 1024);
    }
    __device__ __forceinline__ void read_b(v4i (&B)[TB][2], int slot, int i) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) B[i][h] = *reinterpret_cast<const v4i *>(b_lds[h] + slot * kSlot + i * 2048);
    }

    // Step t: its products from A and B, behind each row block's the read of its fragments of step t + 1, between them the reads of
    // step t + 1's rows of x into N and the fetch of step t + R - 1 into the slot of step t - 1. Who has passed this step's barrier has issued
    // the products of step t - 1, which waited for that slot's reads. MORE: all of those steps exist, and the one fetched is not the last.
    template <bool ACTIVE, bool MORE>
    __device__ __forceinline__ void step(int t, int slot, const v4i (&B)[TB][2], v4i (&N)[TB][2]) {
        const int  next = slot + 1 == R ? 0 : slot + 1, last = slot == 0 ? R - 1 : slot - 1;
        const bool get = MORE || t + R - 1 < steps;
        // step t + 1 has arrived; those behind it need not have
        if (MORE || t + R - 2 < steps) wait_loads<(R - 3) * kRuns>();
        else wait_loads<0>();
        barrier();
        if (!MORE && get) {
#pragma unroll
            for (int i = 0; i < kRuns; ++i) fetch_run<true>(t + R - 1, last, i);
        }
#pragma unroll
        for (int r = 0; r < RB; ++r) {
            if constexpr (ACTIVE) {
#pragma unroll
                for (int b = 0; b < TB; ++b) acc[r][b] = Matrix<WT>::mfma(A[r][0], B[b][0], acc[r][b]);
                // (past the last step: what the ring holds, for nobody)
#pragma unroll
                for (int i = r * TB / RB; i < (r + 1) * TB / RB; ++i) read_b(N, next, i);
            }
            if (MORE) {
#pragma unroll
                for (int i = r * kRuns / RB; i < (r + 1) * kRuns / RB; ++i) fetch_run<false>(t + R - 1, last, i);
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (ACTIVE) {
#pragma unroll
                for (int b = 0; b < TB; ++b) acc[r][b] = Matrix<WT>::mfma(A[r][1], B[b][1], acc[r][b]);
                read_a(next, r);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // ACTIVE: this wavefront has positions; otherwise it moves its share and keeps the barriers
    template <bool ACTIVE>
    __device__ __forceinline__ void loop() {
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int t = 0; t < TB; ++t) acc[r][t] = Acc{ 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0 };
#pragma unroll
        for (int t = 0; t < R - 1; ++t) {
            if (t < steps) {
#pragma unroll
                for (int i = 0; i < kRuns; ++i) fetch_run<true>(t, t, i);
            }
        }
        if (steps >= R - 1) wait_loads<(R - 2) * kRuns>();
        else wait_loads<0>();
        barrier();
        v4i B[TB][2], N[TB][2];
#pragma unroll
        for (int i = 0; i < RB; ++i) read_a(0, i);
#pragma unroll
        for (int i = 0; i < TB; ++i) read_b(B, 0, i);
        int  t = 0, slot = 0;
        auto next = [&]() __attribute__((always_inline)) { ++t, slot = slot + 1 == R ? 0 : slot + 1; };
        while (t + R + 1 < steps) {   // (both steps fetch one in front of the last)
            step<ACTIVE, true>(t, slot, B, N), next();
            step<ACTIVE, true>(t, slot, N, B), next();
        }
        while (true) {
            step<ACTIVE, false>(t, slot, B, N), next();
            if (t >= steps) break;
            step<ACTIVE, false>(t, slot, N, B), next();
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

template <int WT, int RB, int TB, int WC, int R, bool GROUPED>
__global__ __launch_bounds__(128 * WC, WC == 4 ? 2 : RB * TB <= 2 ? 2 : RB * TB <= 4 ? 3 : 1) void rq_tiled_kernel(const ProductArgs a, const int row_tiles, const int token_tiles,
                                                                                                 const int across) {
    using G = Tiled<WT, RB, TB, WC, R>;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int index = (int) blockIdx.y * across + (int) blockIdx.x;
    int       e = 0, first, count, row_tile;
    if constexpr (GROUPED) {
        // The tiles of the groups in a row, rows of the weight fastest: an XCD then reads the weights of its groups, and few others do.
        constexpr int T = G::kTileTokens;
        auto tiles = [](int n) { return (n + T - 1) / T; };
        int  gfirst, gcount, place, total;
        find_group(a, -1, tiles, e, gfirst, gcount, place, total);
        if (index >= total * row_tiles) return;
        const int v = place_of(index, total * row_tiles), tile = v / row_tiles;
        row_tile = v - tile * row_tiles;
        if (!find_group(a, tile, tiles, e, gfirst, gcount, place, total)) return;
        first = gfirst + place * T;
        count = min(T, gcount - place * T);
    } else {
        const int total = row_tiles * token_tiles;
        if (index >= total) return;
        const int v = place_of(index, total);
        row_tile = v / token_tiles;
        first = (v - row_tile * token_tiles) * G::kTileTokens;
        count = (int) (a.P - first < G::kTileTokens ? a.P - first : G::kTileTokens);
    }
    G g;
    g.lane = threadIdx.x & 63;
    g.wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
    g.wr = g.wave & 1;
    // (with four wavefronts the workgroups take turns in which SIMDs a tile with half of its positions leaves idle)
    g.wc = WC == 2 ? ((g.wave >> 1) ^ (index >> 3)) & 1 : g.wave >> 1;
    g.lane16 = g.lane * 16;
    g.steps = a.L.steps;
    g.lds0 = (uint32_t) (uintptr_t) (__attribute__((address_space(3))) void *) lds;
    g.a_lds = lds + g.wr * RB * 2048 + g.lane * 16;
    // Row j of 16 keeps its bytes 16 c .. + 15 at place c ^ (j / 4) of its 64: 16 rows' same bytes lie in 16 places of the banks' 256 bytes.
    {
        const int row = g.lane & 31, turn = (row >> 2) & 3, half = g.lane >> 5;
        const uint8_t *b = lds + (2 * G::kABlocks + g.wc * TB * 2) * 1024 + row * 64;
        g.b_lds[0] = b + (half ^ turn) * 16;
        g.b_lds[1] = b + ((2 + half) ^ turn) * 16;
    }
    const int      block0 = row_tile * G::kABlocks;
    const uint8_t *w = a.w + (int64_t) e * a.L.expert_bytes;
#pragma unroll
    for (int i = 0; i < G::kARuns; ++i) {   // (blocks past the weight's repeat its last one)
        const int run = g.wave * G::kARuns + i, block = min(block0 + (run >> 1), a.L.row_blocks - 1);
        g.a_src[i] = uniform(w + (int64_t) block * a.L.steps * 2048 + (run & 1) * 1024);
    }
    const int chunk = (g.lane & 3) ^ ((g.lane >> 4) & 3);
    g.b_last = (int64_t) (a.L.steps - 1) * 64 + chunk * 16 < a.x_bytes;
#pragma unroll
    for (int i = 0; i < G::kBRuns; ++i) {   // (positions past the last repeat it)
        const int     at = min((g.wave * G::kBRuns + i) * 16 + (g.lane >> 2), count - 1);
        const int64_t row = row_read(a, first + at);
        g.b_src[i] = a.x + (row < 0 ? 0 : row) * a.pitch + chunk * 16;
    }
    if (g.wc * TB * 32 < count) g.template loop<true>();
    else g.template loop<false>();

    // 32 positions x 64 rows at a time through LDS (a region of the wavefront's own), so that a position's outputs leave as whole lines.
    const int    lane = g.lane, wr = g.wr, wc = g.wc;
    float       *mine = reinterpret_cast<float *>(lds) + g.wave * 32 * G::kStride;
    const int    dtype = a.out_dtype;
    const float *t_scales = reinterpret_cast<const float *>(w + a.L.code_bytes);
    int          out_at[TB];   // (a position a lane; y's rows are fewer than 2^31)
    float        s_m[TB];      // of int8; and 0 for a row that is not there
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
    barrier();   // (the ring is not read any more)
    if (wc * TB * 32 >= count) return;
    // LANES of a position write 16 bytes each
    auto store = [&](auto lanes, int t, int r) __attribute__((always_inline)) {
        constexpr int kLanes = decltype(lanes)::value, kTokens = 64 / kLanes;
        const int     n = lane % kLanes * (dtype == RQ_F32 ? 4 : 8);
        const int64_t n0 = (int64_t) (block0 + wr * RB + r) * 32 + n;
#pragma unroll
        for (int i = 0; i < 32 / kTokens; ++i) {
            const int     at = i * kTokens + lane / kLanes;
            const int64_t row = __shfl(out_at[t], at);
            if (row >= 0) store_out(dtype, a.y, row * a.ldy, n0, a.L.N, mine + at * G::kStride + n);
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
                const auto &c = g.acc[r + q / 4][t];
                v4f         v;
                if constexpr (WT == RQ_I8) {
                    const int block = min(block0 + wr * RB + r + q / 4, a.L.row_blocks - 1);
                    const v4f tn = *reinterpret_cast<const v4f *>(t_scales + block * 32 + q % 4 * 8 + (lane >> 5) * 4);
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = (float) c[q % 4 * 4 + i] * tn[i] * s_m[t];
                } else {
                    v = v4f{ c[q % 4 * 4], c[q % 4 * 4 + 1], c[q % 4 * 4 + 2], c[q % 4 * 4 + 3] };
                }
                if (!in_there[t]) v = v4f{ 0, 0, 0, 0 };
                *reinterpret_cast<v4f *>(mine + (lane & 31) * G::kStride + q * 8 + (lane >> 5) * 4) = v;
            }
            __builtin_amdgcn_wave_barrier();
            if (dtype == RQ_F32) store(std::integral_constant<int, 8 * kTwo>{}, t, r);
            else store(std::integral_constant<int, 4 * kTwo>{}, t, r);
            __builtin_amdgcn_wave_barrier();
        }
    }
}

constexpr int64_t kAcross = 1 << 20;   // workgroups in one dimension of a grid, which may have under 2^32 threads

template <int WT, int RB, int TB, int WC, int R, bool GROUPED>
hipError_t launch(const ProductArgs &a, hipStream_t stream) {
    using G = Tiled<WT, RB, TB, WC, R>;
    const int64_t row_tiles = (a.L.row_blocks * 32 + G::kTileRows - 1) / G::kTileRows;
    int64_t       token_tiles = (a.P + G::kTileTokens - 1) / G::kTileTokens;
    if (GROUPED) token_tiles = a.P / G::kTileTokens + (a.P < a.E ? a.P : a.E);   // (at most: every group's last tile is not full)
    const int64_t groups = row_tiles * token_tiles;
    if (groups > 0x7FFFFFFFll - kAcross) return hipErrorInvalidConfiguration;
    const unsigned across = (unsigned) (groups < kAcross ? groups : kAcross);
    static std::atomic<uint64_t> allowed{ 0 };   // devices on which the kernel may have its LDS
    const hipError_t e = allow_lds(reinterpret_cast<const void *>(rq_tiled_kernel<WT, RB, TB, WC, R, GROUPED>), G::kBytes, allowed);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((rq_tiled_kernel<WT, RB, TB, WC, R, GROUPED>), dim3(across, (unsigned) ((groups + across - 1) / across)),
                       dim3(G::kThreads), G::kBytes, stream, a, (int) row_tiles, (int) token_tiles, (int) across);
    return hipGetLastError();
}

template <int WT, bool GROUPED>
hipError_t launch_form(int form, const ProductArgs &a, hipStream_t stream) {
    switch (form) {
        case 0: return launch<WT, 1, 1, 2, 8, GROUPED>(a, stream);
        case 1: return launch<WT, 2, 1, 2, 6, GROUPED>(a, stream);
        case 2: return launch<WT, 2, 2, 2, 4, GROUPED>(a, stream);
        default: return launch<WT, 4, 2, 4, 4, GROUPED>(a, stream);
    }
}
template <bool GROUPED>
hipError_t launch_type(int weight_type, int form, const ProductArgs &a, hipStream_t stream) {
    if (weight_type == RQ_I8) return launch_form<RQ_I8, GROUPED>(form, a, stream);
    if (weight_type == RQ_F16) return launch_form<RQ_F16, GROUPED>(form, a, stream);
    return launch_form<RQ_BF16, GROUPED>(form, a, stream);
}

constexpr int kRowsOf[kForms] = { 64, 128, 128, 256 }, kTokensOf[kForms] = { 64, 64, 128, 256 };

}  // namespace

int tiled_rows(int form) { return kRowsOf[form]; }
int tiled_tokens(int form) { return kTokensOf[form]; }

hipError_t launch_tiled(int weight_type, int form, const ProductArgs &a, hipStream_t stream) {
    if (a.offsets) return launch_type<true>(weight_type, form, a, stream);
    return weight_type == RQ_I8 ? launch_form<RQ_I8, false>(form, a, stream) : hipErrorInvalidValue;
}

}  // namespace prod
}  // namespace rq
