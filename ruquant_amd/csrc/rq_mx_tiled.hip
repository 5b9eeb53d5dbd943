// MXFP4 product for many tokens: tiles of rows x tokens, both operands through LDS.
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
    static constexpr int kScales = R * kSlot;                    // behind the ring: one chunk of their scales
    static constexpr int kBytes = kScales + (kABlocks + kBBlocks) * 512;
    // 1 KiB each, of a wavefront per step; runs of the scales per chunk (some are fetched twice so that all fetch as many)
    static constexpr int kARuns = 2 * kABlocks / kWaves, kBRuns = 2 * kBBlocks / kWaves, kRuns = kARuns + kBRuns;
    static constexpr int kScaleRuns = (kABlocks + kBBlocks) / 2, kScales1 = (kScaleRuns + kWaves - 1) / kWaves;
    static_assert(2 * kABlocks % kWaves == 0 && 2 * kBBlocks % kWaves == 0 && kBBlocks % 2 == 0, "split of the loads");
    static constexpr int kTileRows = MODE == kGateUp ? 32 * RB : 64 * RB;            // (of each matrix)
    static constexpr int kTileTokens = 32 * WC * TB;

    // what this wavefront moves
    const uint8_t *a_src[kARuns], *b_src[kBRuns];   // wave-uniform
    const uint8_t *s_src[kScales1];                 // the lane's
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
    __device__ __forceinline__ void fetch_scales(int c) {
#pragma unroll
        for (int i = 0; i < kScales1; ++i) load_run(s_src[i] + (int64_t) c * 512, lds0 + kScales + (i * kWaves + wave) % kScaleRuns * 1024);
    }
    __device__ __forceinline__ void read_a(int slot, int i) {
#pragma unroll
        for (int h = 0; h < 2; ++h) A[i][h] = *reinterpret_cast<const v4i *>(a_lds + slot * kSlot + (2 * i + h) * 1024);
    }
    __device__ __forceinline__ void read_b(v4i (&B)[TB][2], int slot, int i) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) B[i][h] = *reinterpret_cast<const v4i *>(b_lds + slot * kSlot + (2 * i + h) * 1024);
    }
    // the scales of inputs 256 half .. + 255 of the chunk in LDS
    __device__ __forceinline__ void read_sa(int half, int i) { sA[i] = *reinterpret_cast<const int *>(as_lds + i * 512 + half * 256); }
    __device__ __forceinline__ void read_sb(int (&sB)[TB], int half, int i) const {
        sB[i] = *reinterpret_cast<const int *>(bs_lds + i * 512 + half * 256);
    }

    // Step t = 4 c + J: its products from A and B, behind each row block's the read of its fragments of step t + 1, between them the
    // reads of step t + 1's activations into N and the fetch of step t + R - 1 into the slot of step t - 1 (whose reads the products
    // of step t - 1 have waited for, in every wavefront that has passed this step's barrier). The scales are read every second
    // step; those of the next chunk are fetched by the second step of a chunk, last of its loads, and read by the fourth. MORE: all
    // of those steps exist.
    template <int J, bool MORE>
    __device__ __forceinline__ void step(int t, int slot, const v4i (&B)[TB][2], v4i (&N)[TB][2], int (&sB)[TB], int (&sN)[TB]) {
        const int  next = slot + 1 == R ? 0 : slot + 1, last = slot == 0 ? R - 1 : slot - 1;
        const bool get = MORE || t + R - 1 < steps;
        // step t + 1 has arrived; those behind it need not have
        if (MORE || t + R - 2 < steps) wait_loads<(R - 3) * kRuns + (MORE && J == 2 ? kScales1 : 0)>();
        else wait_loads<0>();
        barrier();
        if (!MORE && get) {
#pragma unroll
            for (int i = 0; i < kRuns; ++i) fetch_run(t + R - 1, last, i);
        }
#pragma unroll
        for (int r = 0; r < RB; ++r) {
#pragma unroll
            for (int b = 0; b < TB; ++b) acc[r][b] = mfma<2 * (J & 1)>(A[r][0], B[b][0], acc[r][b], sA[r], sB[b]);
            // (past the last step: what the ring holds, for nobody)
#pragma unroll
            for (int i = r * TB / RB; i < (r + 1) * TB / RB; ++i) {
                read_b(N, next, i);
                if (J & 1) read_sb(sN, J == 1, i);
            }
            if (MORE) {
#pragma unroll
                for (int i = r * kRuns / RB; i < (r + 1) * kRuns / RB; ++i) fetch_run(t + R - 1, last, i);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int b = 0; b < TB; ++b) acc[r][b] = mfma<2 * (J & 1) + 1>(A[r][1], B[b][1], acc[r][b], sA[r], sB[b]);
            read_a(next, r);
            if (J & 1) read_sa(J == 1, r);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (J & 1) {
#pragma unroll
            for (int i = 0; i < TB; ++i) sB[i] = sN[i];
        }
        if (J == 1 && (MORE || t + 3 < steps)) fetch_scales((t >> 2) + 1);
    }

    __device__ __forceinline__ void loop() {
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int t = 0; t < TB; ++t) acc[r][t] = v16f{ 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0 };
        fetch_scales(0);
#pragma unroll
        for (int t = 0; t < R - 1; ++t) {
            if (t < steps) {
#pragma unroll
                for (int i = 0; i < kRuns; ++i) fetch_run(t, t, i);
            }
        }
        if (steps >= R - 1) wait_loads<(R - 2) * kRuns>();
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
        while (t + R + 2 < steps) {
            step<0, true>(t, slot, B, N, sB, sN), next();
            step<1, true>(t, slot, N, B, sB, sN), next();
            step<2, true>(t, slot, B, N, sB, sN), next();
            step<3, true>(t, slot, N, B, sB, sN), next();
        }
        while (true) {
            step<0, false>(t, slot, B, N, sB, sN), next();
            if (t >= steps) break;
            step<1, false>(t, slot, N, B, sB, sN), next();
            if (t >= steps) break;
            step<2, false>(t, slot, B, N, sB, sN), next();
            if (t >= steps) break;
            step<3, false>(t, slot, N, B, sB, sN), next();
            if (t >= steps) break;
        }
        wait_loads<0>();   // (none of this wavefront's loads lands in LDS behind this)
    }
};

template <int MODE, int RB, int TB, int WC, int R>
__global__ __launch_bounds__(128 * WC, WC == 4 ? 2 : RB * TB <= 4 ? 3 : 2) void rq_mx_tiled_kernel(const ProductArgs a, const int row_tiles, const int token_tiles) {
    using G = Tiled<MODE, RB, TB, WC, R>;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    // Workgroups go to the XCDs in turn. Each XCD takes a run of the tiles in an order in which the token tiles run fastest, so that
    // those that share rows of the weight share an L2.
    const int total = row_tiles * token_tiles;
    const int xcd = blockIdx.x & 7, each = total >> 3, more = total & 7;
    const int v = xcd * each + min(xcd, more) + (int) (blockIdx.x >> 3);
    const int row_tile = v / token_tiles, token_tile = v - row_tile * token_tiles;
    Tile tile = { 0, 0, 0, 0 };
    if constexpr (MODE == kDense) {
        tile.first = token_tile * G::kTileTokens;
        tile.count = (int) (a.M - tile.first < G::kTileTokens ? a.M - tile.first : G::kTileTokens);
    } else {
        if (token_tile >= *a.n_tiles) return;
        tile = a.tiles[token_tile];
    }
    G g;
    g.lane = threadIdx.x & 63;
    g.wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
    g.wr = g.wave / WC;
    g.wc = g.wave % WC;
    g.lane16 = g.lane * 16;
    g.steps = a.L.steps;
    g.lds0 = (uint32_t) (uintptr_t) (__attribute__((address_space(3))) void *) lds;
    g.a_lds = lds + g.wr * RB * 2048 + g.lane * 16;
    g.b_lds = lds + (2 * G::kABlocks + g.wc * TB * 2) * 1024 + g.lane * 16;
    g.as_lds = lds + G::kScales + g.wr * RB * 512 + g.lane * 4;
    g.bs_lds = lds + G::kScales + (G::kABlocks + g.wc * TB) * 512 + g.lane * 4;
    constexpr int  kBlocks = G::kTileRows / 32;   // row blocks of the tile, per matrix
    const int      block0 = row_tile * kBlocks;
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
        g.a_src[i] = uniform(matrix(run >> 1) + (int64_t) place(run >> 1) * a.L.steps * 2048 + (run & 1) * 1024);
    }
    // the tile's token blocks; those past the last repeat it, and those past the activations the activations' last
    const int token0 = tile.first >> 5, token_blocks = min((tile.count + 31) >> 5, a.P.row_blocks - token0);
    auto token_place = [&](int i) __attribute__((always_inline)) { return token0 + min(i, token_blocks - 1); };
#pragma unroll
    for (int i = 0; i < G::kBRuns; ++i) {
        const int run = g.wave * G::kBRuns + i;
        g.b_src[i] = uniform(a.a_codes + (int64_t) token_place(run >> 1) * a.P.steps * 2048 + (run & 1) * 1024);
    }
#pragma unroll
    for (int i = 0; i < G::kScales1; ++i) {   // of two row blocks, or of two token blocks
        const int  run = (i * G::kWaves + g.wave) % G::kScaleRuns;
        const bool rows = run < RB;
        const int  r = 2 * run + (g.lane >> 5);
        g.s_src[i] = (rows ? matrix(r) + a.L.code_bytes + (int64_t) place(r) * a.L.chunks * 512
                           : a.a_codes + a.P.code_bytes + (int64_t) token_place(r - 2 * RB) * a.P.chunks * 512) + (g.lane & 31) * 16;
    }
    g.loop();
    const int lane = g.lane, wr = g.wr, wc = g.wc;
    if constexpr (MODE == kGateUp) {
#pragma unroll
        for (int t = 0; t < TB; ++t) {
            const int token = (wc * TB + t) * 32 + (lane & 31);
#pragma unroll
            for (int q = 0; q < RB / 2; ++q) {
                const int b = block0 + wr * (RB / 2) + q;
                if (b < a.L.row_blocks) store_h<true>(a, g.acc[q][t], g.acc[RB / 2 + q][t], lane, token < tile.count, tile.first + token, b);
            }
        }
    } else {
        // 32 tokens x 64 rows at a time through LDS (a region of the wavefront's own), so that a token's outputs leave as whole lines.
        // (Lines written in halves cost much: 2048 x 17408 outputs in bf16, 64 bytes a token and store, 38 us, in fp32 30.)
        constexpr int kStride = 68;
        static_assert(RB % 2 == 0 && G::kWaves * 32 * kStride * 4 <= G::kBytes, "a region per wavefront");
        float    *mine = reinterpret_cast<float *>(lds) + g.wave * 32 * kStride;
        const int dtype = MODE == kDown ? RQ_F32 : a.out_dtype;
        barrier();   // (the ring is not read any more)
#pragma unroll
        for (int t = 0; t < TB; ++t) {
#pragma unroll
            for (int r = 0; r < RB; r += 2) {
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const v16f &c = g.acc[r + q / 4][t];
                    *reinterpret_cast<v4f *>(mine + (lane & 31) * kStride + q * 8 + (lane >> 5) * 4) =
                        v4f{ c[q % 4 * 4], c[q % 4 * 4 + 1], c[q % 4 * 4 + 2], c[q % 4 * 4 + 3] };
                }
                __builtin_amdgcn_wave_barrier();
                const int64_t n0 = (int64_t) (block0 + wr * RB + r) * 32;
                const int     wide = dtype == RQ_F32 ? 4 : 3;   // (log2 of the lanes of a token: 16 bytes each)
                const int     step = 64 >> wide, at0 = lane >> wide, n = (lane & ((1 << wide) - 1)) << (6 - wide);
                for (int at = at0; at < 32; at += step) {
                    const int token = (wc * TB + t) * 32 + at;
                    if (token < tile.count) {
                        const int64_t row = MODE == kDown ? a.row_of[tile.first + token] : tile.first + token;
                        store_out(dtype, a.y, row * a.ldy, n0 + n, a.L.N, mine + at * kStride + n);
                    }
                }
                __builtin_amdgcn_wave_barrier();
            }
        }
    }
}

template <int MODE, int RB, int TB, int WC, int R>
hipError_t launch(const ProductArgs &a, hipStream_t stream) {
    using G = Tiled<MODE, RB, TB, WC, R>;
    const int row_tiles = (int) ((a.L.row_blocks * 32 + G::kTileRows - 1) / G::kTileRows);
    const int token_tiles = MODE == kDense ? (int) ((a.M + G::kTileTokens - 1) / G::kTileTokens) : a.most_tiles;
    static const hipError_t set = hipFuncSetAttribute(reinterpret_cast<const void *>(rq_mx_tiled_kernel<MODE, RB, TB, WC, R>),
                                                      hipFuncAttributeMaxDynamicSharedMemorySize, G::kBytes);
    if (set != hipSuccess) return set;
    hipLaunchKernelGGL((rq_mx_tiled_kernel<MODE, RB, TB, WC, R>), dim3((unsigned) row_tiles * token_tiles), dim3(G::kThreads), G::kBytes, stream,
                       a, row_tiles, token_tiles);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_tiled(int mode, const ProductArgs &a, hipStream_t stream) {
    if (mode == kDense) return a.L.steps >= 64 ? launch<kDense, 4, 2, 4, 4>(a, stream) : launch<kDense, 2, 2, 2, 3>(a, stream);
    return mode == kGateUp ? launch<kGateUp, 4, 2, 2, 3>(a, stream) : launch<kDown, 4, 2, 2, 3>(a, stream);
}

}  // namespace mx
}  // namespace rq
