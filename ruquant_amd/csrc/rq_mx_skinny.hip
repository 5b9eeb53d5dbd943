// MXFP4 product for few tokens per weight: the weights stream from memory into registers, once.
//
// A workgroup owns RB blocks of 32 rows (kGateUp: of each projection), its wavefronts split the inputs, and their partial sums are
// joined through LDS in the wavefronts' order. The weight fragment is the MFMA's first operand, the tokens are its 32 columns.
#include "rq_mx.h"

namespace rq {
namespace mx {
namespace {

constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kDepth = 4;   // steps in flight per wavefront

template <int MODE, int RB, int TB>
__global__ __launch_bounds__(kThreads) void rq_mx_skinny_kernel(const ProductArgs a) {
    constexpr int kMat = MODE == kGateUp ? 2 : 1;
    constexpr int T = 32 * TB;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Tile tile = { 0, 0, 0, 0 };
    if constexpr (MODE == kDense) {
        tile.first = blockIdx.y * T;
        tile.count = (int) (a.M - tile.first < T ? a.M - tile.first : T);
    } else {
        if ((int) blockIdx.y >= *a.n_tiles) return;
        tile = a.tiles[blockIdx.y];
    }
    const int      block0 = blockIdx.x * RB;
    const uint8_t *w[kMat][RB], *ws[kMat][RB];
#pragma unroll
    for (int m = 0; m < kMat; ++m) {
        const uint8_t *base = (m ? a.w2 : a.w) + (int64_t) tile.expert * a.L.expert_bytes;
#pragma unroll
        for (int r = 0; r < RB; ++r) {
            w[m][r] = base + (int64_t) (block0 + r) * a.L.steps * 2048 + lane * 16;
            ws[m][r] = base + a.L.code_bytes + (int64_t) (block0 + r) * a.L.chunks * 512 + lane * 4;
        }
    }
    // this lane's token in each block of 32, as a row of the activations (a token past the count repeats the last one)
    const uint8_t *act[TB], *act_s[TB];
#pragma unroll
    for (int t = 0; t < TB; ++t) {
        const int     p = tile.first + min(t * 32 + (lane & 31), tile.count - 1);
        const int64_t row = MODE == kGateUp ? a.row_of[p] : p;
        act[t] = a.a_codes + row * a.A.code_stride + (lane >> 5) * 16;
        act_s[t] = a.a_scales + row * a.A.scale_stride + (lane >> 5) * 4;
    }
    const int s0 = (int) ((int64_t) a.L.steps * wave / kWaves), s1 = (int) ((int64_t) a.L.steps * (wave + 1) / kWaves);

    v16f acc[kMat][RB][TB];
#pragma unroll
    for (int m = 0; m < kMat; ++m)
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int t = 0; t < TB; ++t) acc[m][r][t] = v16f{ 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0 };

    struct Frag {
        v4i A[kMat][RB][2], B[TB][2];
        int sa[kMat][RB], sb[TB];
    };
    auto load = [&](Frag &f, int s) __attribute__((always_inline)) {
#pragma unroll
        for (int m = 0; m < kMat; ++m) {
#pragma unroll
            for (int r = 0; r < RB; ++r) {
#pragma unroll
                for (int h = 0; h < 2; ++h) f.A[m][r][h] = *reinterpret_cast<const v4i *>(w[m][r] + (int64_t) s * 2048 + h * 1024);
                f.sa[m][r] = *reinterpret_cast<const int *>(ws[m][r] + (s >> 1) * 256);
            }
        }
#pragma unroll
        for (int t = 0; t < TB; ++t) {
#pragma unroll
            for (int h = 0; h < 2; ++h) f.B[t][h] = *reinterpret_cast<const v4i *>(act[t] + (int64_t) s * 64 + h * 32);
            f.sb[t] = *reinterpret_cast<const int *>(act_s[t] + (s >> 1) * 8);
        }
    };
    auto multiply = [&](const Frag &f, int s) __attribute__((always_inline)) {
        const int by = (s & 1) * 16;
#pragma unroll
        for (int m = 0; m < kMat; ++m)
#pragma unroll
            for (int r = 0; r < RB; ++r) {
                const int sa = f.sa[m][r] >> by;
#pragma unroll
                for (int t = 0; t < TB; ++t) {
                    acc[m][r][t] = mfma<0>(f.A[m][r][0], f.B[t][0], acc[m][r][t], sa, f.sb[t] >> by);
                    acc[m][r][t] = mfma<1>(f.A[m][r][1], f.B[t][1], acc[m][r][t], sa, f.sb[t] >> by);
                }
            }
    };
    Frag ring[kDepth];
#pragma unroll
    for (int i = 0; i < kDepth; ++i)
        if (s0 + i < s1) load(ring[i], s0 + i);
    for (int s = s0; s < s1; s += kDepth) {
#pragma unroll
        for (int i = 0; i < kDepth; ++i) {
            if (s + i < s1) {
                multiply(ring[i], s + i);
                if (s + i + kDepth < s1) load(ring[i], s + i + kDepth);
            }
        }
    }

    // join: [wave][matrix, row block, token block][quad][lane] of four floats: rows 8 quad + 4 (lane / 32) + i, token lane % 32
    constexpr int kCells = kMat * RB * TB * 256;
    extern __shared__ __attribute__((aligned(16))) v4f part[];
#pragma unroll
    for (int m = 0; m < kMat; ++m)
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int t = 0; t < TB; ++t)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const v16f &c = acc[m][r][t];
                    part[wave * kCells + (((m * RB + r) * TB + t) * 4 + q) * 64 + lane] = v4f{ c[4 * q], c[4 * q + 1], c[4 * q + 2], c[4 * q + 3] };
                }
    __syncthreads();
    for (int c = threadIdx.x; c < kCells; c += kThreads) {
        v4f sum = part[c];
#pragma unroll
        for (int v = 1; v < kWaves; ++v) sum += part[v * kCells + c];
        if constexpr (MODE == kGateUp) {
            part[c] = sum;
        } else {
            const int l = c & 63, q = (c >> 6) & 3, t = (c >> 8) % TB, r = (c >> 8) / TB;
            const int token = t * 32 + (l & 31);
            if (token < tile.count) {
                const int64_t row = MODE == kDown ? a.row_of[tile.first + token] : tile.first + token;
                store_out(MODE == kDown ? RQ_F32 : a.out_dtype, a.y, row * a.ldy, (int64_t) (block0 + r) * 32 + q * 8 + (l >> 5) * 4, a.L.N, sum);
            }
        }
    }
    if constexpr (MODE == kGateUp) {
        __syncthreads();
        if (wave < RB * TB) {
            const int r = wave / TB, t = wave % TB;
            v16f      gate, up;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const v4f x = part[((r * TB + t) * 4 + q) * 64 + lane], y = part[(((RB + r) * TB + t) * 4 + q) * 64 + lane];
#pragma unroll
                for (int i = 0; i < 4; ++i) gate[4 * q + i] = x[i], up[4 * q + i] = y[i];
            }
            const int token = t * 32 + (lane & 31);
            store_h<false>(a, gate, up, lane, token < tile.count, tile.first + token, block0 + r);
        }
    }
}

template <int MODE, int RB, int TB>
hipError_t launch(const ProductArgs &a, hipStream_t stream) {
    constexpr int kBytes = kWaves * (MODE == kGateUp ? 2 : 1) * RB * TB * 4096;
    static const hipError_t set = hipFuncSetAttribute(reinterpret_cast<const void *>(rq_mx_skinny_kernel<MODE, RB, TB>),
                                                      hipFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (set != hipSuccess) return set;
    const int64_t tiles = MODE == kDense ? (a.M + 32 * TB - 1) / (32 * TB) : a.most_tiles;
    hipLaunchKernelGGL((rq_mx_skinny_kernel<MODE, RB, TB>), dim3(a.L.row_blocks / RB, (unsigned) tiles), dim3(kThreads), kBytes, stream, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_skinny(int mode, const ProductArgs &a, int tile_tokens, hipStream_t stream) {
    const bool one = tile_tokens == 32;
    if (mode == kDense) return one ? launch<kDense, 1, 1>(a, stream) : launch<kDense, 1, 2>(a, stream);
    if (mode == kDown) return one ? launch<kDown, 1, 1>(a, stream) : launch<kDown, 1, 2>(a, stream);
    return one ? launch<kGateUp, 1, 1>(a, stream) : launch<kGateUp, 1, 2>(a, stream);
}

}  // namespace mx
}  // namespace rq
