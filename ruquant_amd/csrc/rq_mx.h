// Shared definitions of the MXFP4 operators: layouts, element conversions and launch arguments.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/rq_mx4.h"

namespace rq {
namespace mx {

typedef int   v4i __attribute__((ext_vector_type(4)));
typedef int   v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));

inline int64_t up_to(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

// ---------------------------------------------------------------------------------------------------
// One MFMA (16x16x128, both operands fp4) takes from lane l of its first operand row l % 16 and inputs 32 (l / 16) .. + 31 of
// a run of 128 inputs: one block, 16 bytes of codes and one scale. A "step" below is such a run of 128, a "chunk" four steps.
//
// Prepared weight: per expert
//   codes : N / 16 row blocks x K / 128 steps x 64 lanes x 16 bytes (N padded to 64, K to 128, zeros): a wavefront reads a
//           fragment as 1 KiB of consecutive bytes, and a row block's steps follow one another.
//   scales: N / 16 row blocks x K / 512 chunks x 64 lanes x 4 bytes, the lane's scales of the chunk's four steps.
// Activations (workspace): rows of K / 2 bytes (K padded to 256: whole 128-byte lines), and per row and chunk 4 x 4 bytes of
//   scales, [block of a step][step]: the four bytes that a lane needs of a chunk are one word here too.
// ---------------------------------------------------------------------------------------------------
struct WeightLayout {
    int64_t N, K;
    int     row_blocks, steps, chunks;
    int64_t code_bytes, expert_bytes;   // of one expert
};
inline WeightLayout weight_layout(int64_t N, int64_t K) {
    WeightLayout L;
    L.N = N;
    L.K = K;
    L.row_blocks = (int) (up_to(N, 64) / 16);
    L.steps = (int) (up_to(K, 128) / 128);
    L.chunks = (int) (up_to(K, 512) / 512);
    L.code_bytes = (int64_t) L.row_blocks * L.steps * 1024;
    L.expert_bytes = L.code_bytes + (int64_t) L.row_blocks * L.chunks * 256;
    return L;
}

struct ActLayout {
    int64_t code_stride, scale_stride;   // bytes per row
};
inline ActLayout act_layout(int64_t K) { return { up_to(K, 256) / 2, up_to(K, 512) / 32 }; }

// ---- element types --------------------------------------------------------------------------------
template <int DT> struct Element;
template <> struct Element<RQ_F32> { using type = float; };
template <> struct Element<RQ_F16> { using type = __half; };
template <> struct Element<RQ_BF16> { using type = __hip_bfloat16; };

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__hip_bfloat16 v) {
    return __uint_as_float((uint32_t) __builtin_bit_cast(uint16_t, v) << 16);
}
__device__ __forceinline__ uint16_t bf16_bits(float f) {   // to the nearest, ties to even; NaN stays NaN
    const uint32_t u = __float_as_uint(f);
    return f != f ? 0x7FC0 : (uint16_t) ((u + 0x7FFF + ((u >> 16) & 1)) >> 16);
}
template <int DT>
__device__ __forceinline__ typename Element<DT>::type from_float(float f) {
    if constexpr (DT == RQ_F32) return f;
    else if constexpr (DT == RQ_F16) return __float2half(f);
    else return __builtin_bit_cast(__hip_bfloat16, bf16_bits(f));
}

// The scale byte of a block by its largest magnitude's bits (sign cleared): 255 for an infinity or NaN.
__device__ __forceinline__ int block_scale(uint32_t top_bits) {
    const int e = (int) (top_bits >> 23);
    return e >= 255 ? 255 : e > 2 ? e - 2 : 0;
}
// 2^(127 - X), what the block's elements are multiplied by; 0 for X = 255 (zero codes: 0 * NaN is taken care of by the caller)
__device__ __forceinline__ float scale_down(int X) { return __uint_as_float((uint32_t) (254 - X) << 23); }
// 2^(X - 127)
__device__ __forceinline__ float scale_value(int X) {
    return X == 255 ? __uint_as_float(0x7FC00000u) : X == 0 ? __uint_as_float(0x00400000u) : __uint_as_float((uint32_t) X << 23);
}
// four codes pairs of eight values in a block's units: to nearest even, saturating at 6, the first value in the lowest bits
__device__ __forceinline__ uint32_t pack8(const float (&v)[8], float down) {
    uint32_t u = 0;
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[0] * down, v[1] * down, 1.0f, 0);
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[2] * down, v[3] * down, 1.0f, 1);
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[4] * down, v[5] * down, 1.0f, 2);
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[6] * down, v[7] * down, 1.0f, 3);
    return u;
}

__device__ __forceinline__ v4f mfma(const v4i &a, const v4i &b, const v4f &c, int sa, int sb) {
    const v8i A = { a[0], a[1], a[2], a[3], 0, 0, 0, 0 };
    const v8i B = { b[0], b[1], b[2], b[3], 0, 0, 0, 0 };
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, c, 4, 4, 0, sa, 0, sb);
}

// ---- launches ---------------------------------------------------------------------------------------
// x -> activations in the workspace's form (rows m of `codes` / `scales`)
hipError_t launch_act_quantize(int dtype, const void *x, int64_t ldx, int64_t M, int64_t K, uint8_t *codes, uint8_t *scales,
                               hipStream_t stream);

// How a product's tokens are cut into tiles. A plain product has one segment of M tokens; the experts' products have one
// per expert, and the device knows how long they are.
struct Tile {
    int expert, first, count, pad;   // positions first .. first + count - 1 of the expert-sorted order
};

enum Mode { kDense = 0, kGateUp = 1, kDown = 2 };

struct ProductArgs {
    WeightLayout   L;
    const uint8_t *w, *w2;          // prepared weights; kGateUp: w the gate, w2 the up projection
    const uint8_t *a_codes, *a_scales;
    ActLayout      A;
    int64_t        M;               // tokens (kDense)
    const Tile    *tiles;           // kGateUp, kDown: the tiles, on the device
    const int     *n_tiles;         //   and how many there are
    int            most_tiles;      //   at most
    const int     *row_of;          // kGateUp: position -> row of the activations; kDown: position -> row of the output
    int            out_dtype;
    void          *y;               // kDense: the result; kDown: fp32 rows of the slots
    int64_t        ldy;
    uint8_t       *h_codes, *h_scales;   // kGateUp: activations of the down projection, rows by position
    ActLayout      H;
};
// The scale of block b of row p of the feed-forward's h. Behind the last block that the rows of h have (their padding to 64), the
// step's remaining scales are set too: the down projection multiplies them by zero codes, and a NaN would show.
__device__ __forceinline__ void store_h_scale(const ProductArgs &a, int64_t p, int b, int X) {
    uint8_t *to = a.h_scales + p * a.H.scale_stride + (b >> 4) * 16;
    to[(b & 3) * 4 + ((b >> 2) & 3)] = (uint8_t) X;
    if (b == a.L.row_blocks / 2 - 1) {
        for (int c = b + 1; c & 3; ++c) to[(c & 3) * 4 + ((c >> 2) & 3)] = 0;
    }
}
// few tokens per tile (up to 64; tile_tokens 16, 32 or 64): weights go from memory into registers
hipError_t launch_skinny(int mode, const ProductArgs &a, int tile_tokens, hipStream_t stream);
// many: both operands through LDS (tile_tokens 128)
hipError_t launch_tiled(int mode, const ProductArgs &a, hipStream_t stream);
constexpr int kTiledTokens = 128;

// sorts the slots by expert and cuts them into tiles of tile_tokens positions
struct SortArgs {
    const int32_t *ids;
    int            slots, top, E, tile_tokens;
    int           *token_of, *slot_of;   // by position: token, slot
    Tile          *tiles;
    int           *n_tiles;
};
hipError_t launch_sort(const SortArgs &a, hipStream_t stream);
inline int64_t most_tiles(int64_t slots, int64_t E, int tile_tokens) {
    const int64_t some = slots < E ? slots : E;
    return some + slots / tile_tokens;
}
// y[m] = sum_j weights[m][j] * rows[m * top + j], over the slots whose id is an expert's
hipError_t launch_combine(const float *rows, int64_t N, const int32_t *ids, const float *weights, int64_t M, int top, int E,
                          int out_dtype, void *y, int64_t ldy, hipStream_t stream);

struct RouteArgs {
    int            dtype;
    const void    *logits;
    int64_t        ldl, M;
    int            E, scoring, groups, top_groups, top, renormalize;
    const float   *bias;
    float          scale;
    int32_t       *ids;
    float         *weights;
};
hipError_t launch_route(const RouteArgs &a, hipStream_t stream);

}  // namespace mx
}  // namespace rq
