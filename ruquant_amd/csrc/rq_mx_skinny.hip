// MXFP4 product for few tokens per weight: the weights stream from memory into registers, once.
//
// A workgroup owns some row blocks of 16 rows, its wavefronts split the inputs, and their partial sums are joined through LDS in
// the wavefronts' order. The weight fragment is the MFMA's first operand, the tokens are its 16 columns.
#include "rq_mx.h"

namespace rq {
namespace mx {
namespace {

constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kDepth = 4;   // steps in flight per wavefront

// RB row blocks (kGateUp: RB of each projection), TB blocks of 16 tokens
template <int MODE, int RB, int TB>
__global__ __launch_bounds__(kThreads) void rq_mx_skinny_kernel(const ProductArgs a) {
    constexpr int kMat = MODE == kGateUp ? 2 : 1;
    constexpr int T = 16 * TB;
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
    const uint8_t *w[kMat];
    w[0] = a.w + (int64_t) tile.expert * a.L.expert_bytes;
    if constexpr (kMat == 2) w[1] = a.w2 + (int64_t) tile.expert * a.L.expert_bytes;

    // this lane's token in each block of 16, as a row of the activations (a token past the count repeats the last one)
    const uint8_t *act[TB], *act_s[TB];
#pragma unroll
    for (int t = 0; t < TB; ++t) {
        const int p = tile.first + min(t * 16 + (lane & 15), tile.count - 1);
        const int64_t row = MODE == kGateUp ? a.row_of[p] : p;
        act[t] = a.a_codes + row * a.A.code_stride + (lane >> 4) * 16;
        act_s[t] = a.a_scales + row * a.A.scale_stride + (lane >> 4) * 4;
    }
    const int s0 = (int) ((int64_t) a.L.steps * wave / kWaves), s1 = (int) ((int64_t) a.L.steps * (wave + 1) / kWaves);

    v4f acc[kMat][RB][TB];
#pragma unroll
    for (int m = 0; m < kMat; ++m)
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int t = 0; t < TB; ++t) acc[m][r][t] = v4f{ 0, 0, 0, 0 };

    struct Frag {
        v4i A[kMat][RB], B[TB];
        int sa[kMat][RB], sb[TB];
    };
    auto load = [&](Frag &f, int s) __attribute__((always_inline)) {
#pragma unroll
        for (int m = 0; m < kMat; ++m) {
#pragma unroll
            for (int r = 0; r < RB; ++r) {
                const int64_t b = block0 + r;
                f.A[m][r] = reinterpret_cast<const v4i *>(w[m] + (b * a.L.steps + s) * 1024)[lane];
                f.sa[m][r] = reinterpret_cast<const int *>(w[m] + a.L.code_bytes + (b * a.L.chunks + (s >> 2)) * 256)[lane] >> (8 * (s & 3));
            }
        }
#pragma unroll
        for (int t = 0; t < TB; ++t) {
            f.B[t] = *reinterpret_cast<const v4i *>(act[t] + (int64_t) s * 64);
            f.sb[t] = *reinterpret_cast<const int *>(act_s[t] + (s >> 2) * 16) >> (8 * (s & 3));
        }
    };
    auto multiply = [&](const Frag &f) __attribute__((always_inline)) {
#pragma unroll
        for (int m = 0; m < kMat; ++m)
#pragma unroll
            for (int r = 0; r < RB; ++r)
#pragma unroll
                for (int t = 0; t < TB; ++t) acc[m][r][t] = mfma(f.A[m][r], f.B[t], acc[m][r][t], f.sa[m][r], f.sb[t]);
    };
    Frag ring[kDepth];
#pragma unroll
    for (int i = 0; i < kDepth; ++i)
        if (s0 + i < s1) load(ring[i], s0 + i);
    for (int s = s0; s < s1; s += kDepth) {
#pragma unroll
        for (int i = 0; i < kDepth; ++i) {
            if (s + i < s1) {
                multiply(ring[i]);
                if (s + i + kDepth < s1) load(ring[i], s + i + kDepth);
            }
        }
    }

    // join: [wave][matrix][row block][token block][lane] of four floats, rows (lane / 16) * 4 + i, token lane % 16
    constexpr int kCells = kMat * RB * TB * 64;
    __shared__ v4f part[kWaves][kCells];
#pragma unroll
    for (int m = 0; m < kMat; ++m)
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int t = 0; t < TB; ++t) part[wave][((m * RB + r) * TB + t) * 64 + lane] = acc[m][r][t];
    __syncthreads();
    for (int c = threadIdx.x; c < kCells; c += kThreads) {
        v4f sum = part[0][c];
#pragma unroll
        for (int v = 1; v < kWaves; ++v) sum += part[v][c];
        if constexpr (MODE == kGateUp) {
            part[0][c] = sum;
        } else {
            const int l = c & 63, t = (c >> 6) % TB, r = (c >> 6) / TB;
            const int token = t * 16 + (l & 15);
            const int64_t n = (int64_t) (block0 + r) * 16 + (l >> 4) * 4;
            if (token < tile.count) {
                const int64_t row = MODE == kDown ? a.row_of[tile.first + token] : tile.first + token;
                for (int i = 0; i < 4; ++i) {
                    if (n + i >= a.L.N) break;
                    if (MODE == kDown || a.out_dtype == RQ_F32) reinterpret_cast<float *>(a.y)[row * a.ldy + n + i] = sum[i];
                    else if (a.out_dtype == RQ_F16) reinterpret_cast<__half *>(a.y)[row * a.ldy + n + i] = from_float<RQ_F16>(sum[i]);
                    else reinterpret_cast<__hip_bfloat16 *>(a.y)[row * a.ldy + n + i] = from_float<RQ_BF16>(sum[i]);
                }
            }
        }
    }
    if constexpr (MODE == kGateUp) {
        // h = silu(gate) * up, and its blocks of 32 rows (two row blocks) as activations of the down projection
        __syncthreads();
        for (int c = threadIdx.x; c < RB / 2 * T; c += kThreads) {
            const int token = c % T, pair = c / T;
            if (token >= tile.count) continue;
            float    h[32];
            uint32_t top = 0;
            for (int i = 0; i < 32; ++i) {
                const int cell = ((pair * 2 + (i >> 4)) * TB + (token >> 4)) * 64 + ((i >> 2) & 3) * 16 + (token & 15);
                const float g = part[0][cell][i & 3], u = part[0][RB * TB * 64 + cell][i & 3];
                h[i] = g / (1.0f + expf(-g)) * u;
                top = max(top, __float_as_uint(h[i]) & 0x7FFFFFFFu);
            }
            const int X = block_scale(top);
            uint32_t  code[4];
            for (int q = 0; q < 4; ++q) {
                float v[8];
                for (int i = 0; i < 8; ++i) v[i] = h[8 * q + i];
                code[q] = X == 255 ? 0u : pack8(v, scale_down(X));
            }
            const int64_t p = tile.first + token;
            const int     b = (block0 >> 1) + pair;   // block of the row of h
            *reinterpret_cast<uint4 *>(a.h_codes + p * a.H.code_stride + b * 16) = make_uint4(code[0], code[1], code[2], code[3]);
            store_h_scale(a, p, b, X);
        }
    }
}

template <int MODE, int RB, int TB>
hipError_t launch(const ProductArgs &a, hipStream_t stream) {
    const int64_t tiles = MODE == kDense ? (a.M + 16 * TB - 1) / (16 * TB) : a.most_tiles;
    hipLaunchKernelGGL((rq_mx_skinny_kernel<MODE, RB, TB>), dim3(a.L.row_blocks / RB, (unsigned) tiles), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_skinny(int mode, const ProductArgs &a, int tile_tokens, hipStream_t stream) {
    if (mode == kDense) {
        if (tile_tokens == 16) return launch<kDense, 2, 1>(a, stream);
        if (tile_tokens == 32) return launch<kDense, 2, 2>(a, stream);
        return launch<kDense, 2, 4>(a, stream);
    }
    if (mode == kDown) {
        if (tile_tokens == 16) return launch<kDown, 2, 1>(a, stream);
        if (tile_tokens == 32) return launch<kDown, 2, 2>(a, stream);
        return launch<kDown, 2, 4>(a, stream);
    }
    if (tile_tokens == 16) return launch<kGateUp, 2, 1>(a, stream);
    if (tile_tokens == 32) return launch<kGateUp, 2, 2>(a, stream);
    return launch<kGateUp, 2, 4>(a, stream);
}

}  // namespace mx
}  // namespace rq
