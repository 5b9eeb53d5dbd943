// MXFP4 product for many tokens: tiles of 128 rows x 128 tokens, both operands through LDS.
#include "rq_mx.h"

namespace rq {
namespace mx {
namespace {

constexpr int kThreads = 256;
constexpr int kTileRows = 128;
constexpr int kTok = kTiledTokens;
constexpr int kWeightBytes = kTileRows * 128;   // of a stage (256 inputs)
constexpr int kStage = kWeightBytes + kTok * 128;

__device__ __forceinline__ void to_lds(const uint8_t *from, uint8_t *to) {   // 16 bytes a lane, `to` + 16 * lane
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *) from,
                                     (__attribute__((address_space(3))) void *) to, 16, 0, 0);
}

// Wavefront (wr, wc) of four has 64 rows x 64 tokens. kGateUp: 32 rows of each projection, so that a lane holds both of a row.
template <int MODE>
__global__ __launch_bounds__(kThreads) void rq_mx_tiled_kernel(const ProductArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * kStage];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wr = wave >> 1, wc = wave & 1;
    Tile tile = { 0, 0, 0, 0 };
    if constexpr (MODE == kDense) {
        tile.first = blockIdx.y * kTok;
        tile.count = (int) (a.M - tile.first < kTok ? a.M - tile.first : kTok);
    } else {
        if ((int) blockIdx.y >= *a.n_tiles) return;
        tile = a.tiles[blockIdx.y];
    }
    constexpr int  kBlocks = MODE == kGateUp ? 4 : 8;   // row blocks of the tile, per matrix
    const int      block0 = blockIdx.x * kBlocks;
    const uint8_t *w = a.w + (int64_t) tile.expert * a.L.expert_bytes;
    const uint8_t *w2 = MODE == kGateUp ? a.w2 + (int64_t) tile.expert * a.L.expert_bytes : w;
    // row block i (0 .. 7) of the tile: its matrix and place; blocks past the weight's repeat its last one
    auto codes_of = [&](int i) __attribute__((always_inline)) {
        const int b = MODE == kGateUp ? block0 + (i >> 2) * 2 + (i & 1) : block0 + i;
        const uint8_t *base = MODE == kGateUp && (i & 2) ? w2 : w;
        return base + (int64_t) min(b, a.L.row_blocks - 1) * a.L.steps * 1024;
    };
    auto scales_of = [&](int i) __attribute__((always_inline)) {
        const int b = MODE == kGateUp ? block0 + (i >> 2) * 2 + (i & 1) : block0 + i;
        const uint8_t *base = MODE == kGateUp && (i & 2) ? w2 : w;
        return base + a.L.code_bytes + (int64_t) min(b, a.L.row_blocks - 1) * a.L.chunks * 256;
    };
    // what this lane moves: of weight blocks 2 wave and 2 wave + 1 both steps, of activation rows 32 wave .. + 31 a line each; a
    // row's eight pieces lie in LDS in an order that its number turns, so that the reads below spread over the banks
    const uint8_t *wsrc[2], *asrc[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) wsrc[i] = codes_of(2 * wave + i) + lane * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int     r = wave * 32 + i * 8 + (lane >> 3);
        const int     p = tile.first + min(r, tile.count - 1);
        const int64_t row = MODE == kGateUp ? a.row_of[p] : p;
        asrc[i] = a.a_codes + row * a.A.code_stride + (((lane & 7) ^ (r & 7)) * 16);
    }
    const uint8_t *ws[4], *as[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        ws[i] = scales_of(wr * 4 + i) + lane * 4;
        const int     p = tile.first + min(wc * 64 + i * 16 + (lane & 15), tile.count - 1);
        const int64_t row = MODE == kGateUp ? a.row_of[p] : p;
        as[i] = a.a_scales + row * a.A.scale_stride + (lane >> 4) * 4;
    }
    const int stages = (a.L.steps + 1) / 2;
    auto fetch = [&](int st) __attribute__((always_inline)) {
        uint8_t *to = lds + (st & 1) * kStage;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int s = min(2 * st + h, a.L.steps - 1);   // (an odd last step is fetched twice and used once)
                to_lds(wsrc[i] + (int64_t) s * 1024, to + ((2 * wave + i) * 2 + h) * 1024);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) to_lds(asrc[i] + (int64_t) st * 128, to + kWeightBytes + (wave * 4 + i) * 1024);
    };
    v4f acc[4][4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[r][t] = v4f{ 0, 0, 0, 0 };
    fetch(0);
    for (int st = 0; st < stages; ++st) {
        __syncthreads();
        if (st + 1 < stages) fetch(st + 1);
        const uint8_t *from = lds + (st & 1) * kStage;
        int sw[4], sa[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sw[i] = *reinterpret_cast<const int *>(ws[i] + (int64_t) (st >> 1) * 256) >> (16 * (st & 1));
            sa[i] = *reinterpret_cast<const int *>(as[i] + (int64_t) (st >> 1) * 16) >> (16 * (st & 1));
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (2 * st + h >= a.L.steps) break;
            v4i A[4], B[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                A[i] = reinterpret_cast<const v4i *>(from + ((wr * 4 + i) * 2 + h) * 1024)[lane];
                const int r = wc * 64 + i * 16 + (lane & 15);
                B[i] = *reinterpret_cast<const v4i *>(from + kWeightBytes + r * 128 + (((h * 4 + (lane >> 4)) ^ (r & 7)) * 16));
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int t = 0; t < 4; ++t) acc[r][t] = mfma(A[r], B[t], acc[r][t], sw[r] >> (8 * h), sa[t] >> (8 * h));
        }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int  token = wc * 64 + t * 16 + (lane & 15);
        const bool there = token < tile.count;
        if constexpr (MODE == kGateUp) {
            // rows 32 (2 blockIdx.x + wr) .. + 31: one block of h per token, of which this lane has two runs of four
            float    h[2][4];
            uint32_t top = 0;
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float g = acc[r][t][i], u = acc[r + 2][t][i];
                    h[r][i] = g / (1.0f + expf(-g)) * u;
                    top = max(top, __float_as_uint(h[r][i]) & 0x7FFFFFFFu);
                }
            top = max(top, (uint32_t) __shfl_xor((int) top, 16));
            top = max(top, (uint32_t) __shfl_xor((int) top, 32));
            const int X = block_scale(top);
            float     v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = h[i >> 2][i & 3];
            const uint32_t c = X == 255 ? 0u : pack8(v, scale_down(X));
            const int      b = blockIdx.x * 2 + wr;
            if (there && b < a.L.row_blocks / 2) {
                const int64_t p = tile.first + token;
                uint8_t      *to = a.h_codes + p * a.H.code_stride + b * 16 + (lane >> 4) * 2;
                *reinterpret_cast<uint16_t *>(to) = (uint16_t) c;
                *reinterpret_cast<uint16_t *>(to + 8) = (uint16_t) (c >> 16);
                if (lane < 16) store_h_scale(a, p, b, X);
            }
        } else if (there) {
            const int64_t row = MODE == kDown ? a.row_of[tile.first + token] : tile.first + token;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int64_t n = (int64_t) (block0 + wr * 4 + r) * 16 + (lane >> 4) * 4;
                for (int i = 0; i < 4; ++i) {
                    if (n + i >= a.L.N) break;
                    if (MODE == kDown || a.out_dtype == RQ_F32) reinterpret_cast<float *>(a.y)[row * a.ldy + n + i] = acc[r][t][i];
                    else if (a.out_dtype == RQ_F16) reinterpret_cast<__half *>(a.y)[row * a.ldy + n + i] = from_float<RQ_F16>(acc[r][t][i]);
                    else reinterpret_cast<__hip_bfloat16 *>(a.y)[row * a.ldy + n + i] = from_float<RQ_BF16>(acc[r][t][i]);
                }
            }
        }
    }
}

template <int MODE>
hipError_t launch(const ProductArgs &a, hipStream_t stream) {
    constexpr int kBlocks = MODE == kGateUp ? 4 : 8;
    const int64_t tiles = MODE == kDense ? (a.M + kTok - 1) / kTok : a.most_tiles;
    hipLaunchKernelGGL((rq_mx_tiled_kernel<MODE>), dim3((a.L.row_blocks + kBlocks - 1) / kBlocks, (unsigned) tiles), dim3(kThreads), 0,
                       stream, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_tiled(int mode, const ProductArgs &a, hipStream_t stream) {
    return mode == kDense ? launch<kDense>(a, stream) : mode == kGateUp ? launch<kGateUp>(a, stream) : launch<kDown>(a, stream);
}

}  // namespace mx
}  // namespace rq
