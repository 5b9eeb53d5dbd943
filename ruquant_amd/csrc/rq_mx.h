// Shared definitions of the MXFP4 operators: layouts, element conversions and launch arguments.
#pragma once

#include <atomic>

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
typedef float v16f __attribute__((ext_vector_type(16)));

inline int64_t up_to(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

// ---------------------------------------------------------------------------------------------------
// One MFMA (32x32x64, both operands fp4) takes from lane l of its first operand row l % 32 and inputs 32 (l / 32) .. + 31 of a run
// of 64 inputs: one block, 16 bytes of codes and one scale; the second operand's columns likewise. Lane l holds of the 32 x 32
// result column l % 32 and rows 8 (i / 4) + 4 (l / 32) + i % 4, i = 0 .. 15. (Over the chip this form reaches 7.6 PFLOP/s from one
// wavefront per SIMD, the 16x16x128 form with scales 4.7.) A "step" below is 128 inputs, two such runs, a "chunk" four steps.
//
// Prepared weight: per expert
//   codes : N / 32 row blocks x K / 64 runs x 64 lanes x 16 bytes (N padded to 64, K to 128, zeros): a wavefront reads a fragment
//           as 1 KiB of consecutive bytes, and a row block's runs follow one another.
//   scales: N / 32 row blocks x K / 256 x 64 lanes x 4 bytes (K padded to 512), the lane's scales of four runs.
// Activations (workspace), in one of two forms:
//   panels: as a weight of so many rows (the tiled product: its loads are whole runs of 1 KiB);
//   rows  : rows of K / 2 bytes (K padded to 256: whole 128-byte lines), and per row and 256 inputs 2 x 4 bytes of scales, [block of
//           a run][run] (a few tokens, which the lanes of one fragment read).
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
    L.row_blocks = (int) (up_to(N, 64) / 32);
    L.steps = (int) (up_to(K, 128) / 128);
    L.chunks = (int) (up_to(K, 512) / 512);
    L.code_bytes = (int64_t) L.row_blocks * L.steps * 2048;
    L.expert_bytes = L.code_bytes + (int64_t) L.row_blocks * L.chunks * 512;
    return L;
}
// place of block b's scale of a row in the row block's scales of the panel form
__host__ __device__ __forceinline__ int64_t panel_scale_at(int row, int64_t b) {
    return (b >> 3) * 256 + ((b & 1) * 32 + row) * 4 + ((b >> 1) & 3);
}
// place of block b's scale in a row of activations (row form)
__host__ __device__ __forceinline__ int64_t act_scale_at(int64_t b) { return (b >> 3) * 8 + (b & 1) * 4 + ((b >> 1) & 3); }

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
template <int DT>
__device__ __forceinline__ typename Element<DT>::type from_float(float f) {
    if constexpr (DT == RQ_F32) return f;
    else if constexpr (DT == RQ_F16) return __float2half(f);
    else return __builtin_bit_cast(__hip_bfloat16, (__bf16) f);   // (to the nearest, ties to even; one instruction for two)
}

// The largest of this lane's and its neighbours' in the group of four, and of both lanes l and l + 32 (cross-lane operations of the
// vector ALU: through LDS each costs a hundred clocks).
__device__ __forceinline__ uint32_t max_of_four(uint32_t v) {
    v = max(v, (uint32_t) __builtin_amdgcn_mov_dpp((int) v, 0xB1, 0xF, 0xF, true));
    return max(v, (uint32_t) __builtin_amdgcn_mov_dpp((int) v, 0x4E, 0xF, 0xF, true));
}
__device__ __forceinline__ uint32_t of_other_half(uint32_t v, bool upper) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);   // [0]: the lower half's, [1]: the upper half's
    return upper ? r[0] : r[1];
}
// The scale byte of a block by its largest magnitude's bits (sign cleared): 255 for an infinity or NaN.
__device__ __forceinline__ int block_scale(uint32_t top_bits) {
    const int e = (int) (top_bits >> 23);
    return e >= 255 ? 255 : e > 2 ? e - 2 : 0;
}
// 2^(X - 127)
__device__ __forceinline__ float scale_value(int X) {
    return X == 255 ? __uint_as_float(0x7FC00000u) : X == 0 ? __uint_as_float(0x00400000u) : __uint_as_float((uint32_t) X << 23);
}
// What the conversions divide by, 2^(X - 127), for X up to 254.
__device__ __forceinline__ float block_unit(int X) { return __uint_as_float(max((uint32_t) X << 23, 0x00400000u)); }
// The codes of eight values in a block of scale X, the first in the lowest bits: to nearest even, saturating at 6; zeros for X = 255.
__device__ __forceinline__ uint32_t pack8(const float (&v)[8], int X) {
    const float unit = block_unit(X);
    uint32_t    u = 0;
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[0], v[1], unit, 0);
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[2], v[3], unit, 1);
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[4], v[5], unit, 2);
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[6], v[7], unit, 3);
    return X == 255 ? 0u : u;
}

// Eight consecutive elements, in their own type: the 16-bit ones are compared and converted in pairs, half the instructions that
// fp32 copies of them take (2048 x 5120 in bf16 8.6 -> 7.6 us, 16384 rows of it by an order 31 -> 25).
template <int DT> struct Unit {
    using T = typename Element<DT>::type;
    static constexpr bool kWide = DT == RQ_F32;
    uint32_t w[kWide ? 8 : 4];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (uint32_t &x : w) x = 0;
    }
    template <bool VEC> __device__ __forceinline__ void load(const T *p) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < (kWide ? 2 : 1); ++i) {
                const uint4 x = reinterpret_cast<const uint4 *>(p)[i];
                w[4 * i] = x.x, w[4 * i + 1] = x.y, w[4 * i + 2] = x.z, w[4 * i + 3] = x.w;
            }
        } else if constexpr (kWide) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = reinterpret_cast<const uint32_t *>(p)[i];
        } else {
            const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = h[2 * i] | (uint32_t) h[2 * i + 1] << 16;
        }
    }
    // the bits of the largest magnitude as a float
    __device__ __forceinline__ uint32_t top() const {
        if constexpr (kWide) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
            return m;
        } else {
            typedef uint16_t u2 __attribute__((ext_vector_type(2)));
            u2 m = __builtin_bit_cast(u2, w[0] & 0x7FFF7FFFu);
#pragma unroll
            for (int i = 1; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u2, w[i] & 0x7FFF7FFFu));
            const uint32_t both = __builtin_bit_cast(uint32_t, m);
            const uint16_t most = (uint16_t) max(both & 0xFFFF, both >> 16);
            return __float_as_uint(to_float(__builtin_bit_cast(T, most)));
        }
    }
    __device__ __forceinline__ uint32_t pack(int X) const {
        if constexpr (kWide) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
            return pack8(v, X);
        } else {
            const float unit = block_unit(X);
            uint32_t    u = 0;
            if constexpr (DT == RQ_F16) {
                typedef _Float16 h2 __attribute__((ext_vector_type(2)));
                u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(u, __builtin_bit_cast(h2, w[0]), unit, 0);
                u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(u, __builtin_bit_cast(h2, w[1]), unit, 1);
                u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(u, __builtin_bit_cast(h2, w[2]), unit, 2);
                u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(u, __builtin_bit_cast(h2, w[3]), unit, 3);
            } else {
                typedef __bf16 b2 __attribute__((ext_vector_type(2)));
                u = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(u, __builtin_bit_cast(b2, w[0]), unit, 0);
                u = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(u, __builtin_bit_cast(b2, w[1]), unit, 1);
                u = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(u, __builtin_bit_cast(b2, w[2]), unit, 2);
                u = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(u, __builtin_bit_cast(b2, w[3]), unit, 3);
            }
            return X == 255 ? 0u : u;
        }
    }
};

// the product of a run of 64 inputs; J: which byte of the scales' words is this run's
template <int J>
__device__ __forceinline__ v16f mfma(const v4i &a, const v4i &b, const v16f &c, int sa, int sb) {
    const v8i A = { a[0], a[1], a[2], a[3], 0, 0, 0, 0 };
    const v8i B = { b[0], b[1], b[2], b[3], 0, 0, 0, 0 };
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B, c, 4, 4, J, sa, J, sb);
}

// Lets a kernel have so much dynamic LDS, once per device; `allowed` has a bit for each.
inline hipError_t allow_lds(const void *kernel, int bytes, std::atomic<uint64_t> &allowed) {
    int        dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (allowed.load(std::memory_order_relaxed) & bit) return hipSuccess;
    e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess) allowed.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// ---- launches ---------------------------------------------------------------------------------------
// x -> activations in row form
hipError_t launch_act_quantize(int dtype, const void *x, int64_t ldx, int64_t M, int64_t K, uint8_t *codes, uint8_t *scales,
                               hipStream_t stream);
// x -> activations in panel form: row r of the panels is row row_of[r] of x (none if negative), or row r if row_of is null. *rows
// (on the device; null: L.N) of them are looked at. What the panels hold behind the last row is left as it is. Sets zero[0 .. zeros - 1] to 0.
hipError_t launch_panel_quantize(int dtype, const void *x, int64_t ldx, const WeightLayout &L, const int *row_of, const int *rows,
                                 uint8_t *panels, int *zero, int zeros, hipStream_t stream);

// How a product's tokens are cut into tiles. A plain product has one segment of M tokens; the experts' products have one
// per expert, and the device knows how long they are.
struct Tile {
    int expert, first, count, pad;   // positions first .. first + count - 1 of the expert-sorted order
};

enum Mode { kDense = 0, kGateUp = 1, kDown = 2 };

struct ProductArgs {
    WeightLayout   L;
    const uint8_t *w, *w2;          // prepared weights; kGateUp: w the gate, w2 the up projection
    int            first_block, row_tiles;   // kDense: the row blocks of this launch start here
    const uint8_t *panels;          // the activations
    WeightLayout   P;
    int64_t        M;               // tokens (kDense)
    int            splits, split_steps;   // kDense: workgroups that share a tile, and the steps of 128 inputs of each
    float         *sums;            //   splits > 1: what they leave
    int           *arrived;         //   and how many have, by wavefront's outputs: zero before the launch
    const Tile    *tiles;           // kGateUp, kDown: the tiles, on the device
    int            most_tiles;      //   so many; those past the last one have no tokens
    const int     *row_of;          // kDown: position -> row of y
    int            out_dtype;
    void          *y;               // kDense: the result; kDown: rows of the slots, fp32
    int64_t        ldy;
    uint8_t       *h;               // kGateUp: the down projection's activations, panels by position
    WeightLayout   HP;
};
template <int DT>
__device__ __forceinline__ uint32_t pair_bits(float lo, float hi) {   // of a 16-bit type
    if constexpr (DT == RQ_F16) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, h2{ (_Float16) lo, (_Float16) hi });
    } else {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, b2{ (__bf16) lo, (__bf16) hi });
    }
}
// Four consecutive outputs n .. n + 3 of a row (`base` elements in), those in front of N.
__device__ __forceinline__ void store_out(int dtype, void *y, int64_t base, int64_t n, int64_t N, const v4f &v) {
    const int64_t at = base + n;
    if (n + 3 < N && (at & 3) == 0 && ((uintptr_t) y & 15) == 0) {
        if (dtype == RQ_F32) *reinterpret_cast<v4f *>(reinterpret_cast<float *>(y) + at) = v;
        else if (dtype == RQ_F16) *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(y) + at) = make_uint2(pair_bits<RQ_F16>(v[0], v[1]), pair_bits<RQ_F16>(v[2], v[3]));
        else *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(y) + at) = make_uint2(pair_bits<RQ_BF16>(v[0], v[1]), pair_bits<RQ_BF16>(v[2], v[3]));
        return;
    }
    for (int i = 0; i < 4; ++i) {
        if (n + i >= N) break;
        if (dtype == RQ_F32) reinterpret_cast<float *>(y)[at + i] = v[i];
        else if (dtype == RQ_F16) reinterpret_cast<__half *>(y)[at + i] = from_float<RQ_F16>(v[i]);
        else reinterpret_cast<__hip_bfloat16 *>(y)[at + i] = from_float<RQ_BF16>(v[i]);
    }
}
// 16 bytes of consecutive outputs from LDS: four in fp32, eight in the 16-bit types.
__device__ __forceinline__ void store_out(int dtype, void *y, int64_t base, int64_t n, int64_t N, const float *v) {
    const v4f x = *reinterpret_cast<const v4f *>(v);
    if (dtype == RQ_F32) {
        store_out(RQ_F32, y, base, n, N, x);
        return;
    }
    const v4f     z = *reinterpret_cast<const v4f *>(v + 4);
    const int64_t at = base + n;
    if (n + 7 < N && (at & 7) == 0 && ((uintptr_t) y & 15) == 0) {
        const uint4 w = dtype == RQ_F16 ? make_uint4(pair_bits<RQ_F16>(x[0], x[1]), pair_bits<RQ_F16>(x[2], x[3]), pair_bits<RQ_F16>(z[0], z[1]), pair_bits<RQ_F16>(z[2], z[3]))
                                        : make_uint4(pair_bits<RQ_BF16>(x[0], x[1]), pair_bits<RQ_BF16>(x[2], x[3]), pair_bits<RQ_BF16>(z[0], z[1]), pair_bits<RQ_BF16>(z[2], z[3]));
        *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(y) + at) = w;
        return;
    }
    store_out(dtype, y, base, n, N, x);
    store_out(dtype, y, base, n + 4, N, z);
}
// Block b (32 rows) of h = silu(gate) * up for the token in column lane % 32, from both lanes that hold it, as activations of the down
// projection in row p. Behind the last block that the rows of h have (their padding to 64), the step's remaining scales are set
// too: the down projection multiplies them by zero codes, and a NaN would show.
__device__ __forceinline__ void store_h(const ProductArgs &a, const v16f &gate, const v16f &up, int lane, bool there, int64_t p, int b) {
    float    h[16];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        h[i] = gate[i] / (1.0f + expf(-gate[i])) * up[i];
        top = max(top, __float_as_uint(h[i]) & 0x7FFFFFFFu);
    }
    const bool upper = lane >= 32;
    top = max(top, of_other_half(top, upper));
    const int X = block_scale(top);
    uint32_t  c[2];   // rows 8 q + 4 (lane / 32) .. + 3 in half-word q
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = h[8 * q + i];
        c[q] = pack8(v, X);
    }
    const uint32_t o[2] = { of_other_half(c[0], upper), of_other_half(c[1], upper) };
    if (lane < 32 && there) {
        const uint4 codes = make_uint4((c[0] & 0xFFFF) | o[0] << 16, c[0] >> 16 | (o[0] & 0xFFFF0000u), (c[1] & 0xFFFF) | o[1] << 16,
                                       c[1] >> 16 | (o[1] & 0xFFFF0000u));
        const int64_t block = p >> 5;
        const int     row = (int) p & 31;
        *reinterpret_cast<uint4 *>(a.h + (block * a.HP.steps * 2 + (b >> 1)) * 1024 + ((b & 1) * 32 + row) * 16) = codes;
        uint8_t *to = a.h + a.HP.code_bytes + block * a.HP.chunks * 512;
        to[panel_scale_at(row, b)] = (uint8_t) X;
        if (b == a.L.row_blocks - 1) {
            for (int k = b + 1; k & 3; ++k) to[panel_scale_at(row, k)] = 0;
        }
    }
}
// Few tokens (rq_mx_decode.hip): up to four that every workgroup quantises for itself, or up to 16 in row form (a_codes set). The
// experts of few tokens in two launches; their h is rows of h_stride bytes of codes by slot, and of h_stride / 16 scales.
struct DecodeArgs {
    WeightLayout   L;
    const uint8_t *w, *w2;
    const void    *x;
    bool           aligned;   // every row of x to 16 bytes
    int64_t        ldx, M;
    const uint8_t *a_codes, *a_scales;
    ActLayout      A;
    const int32_t *ids;
    const float   *weights;
    int            top, E;
    uint8_t       *h_codes, *h_scales;
    int64_t        h_stride;
    int            out_dtype;
    void          *y;
    int64_t        ldy;
};
// whether a product's tokens are quantised that way
bool decode_takes(int64_t M, int64_t K, int64_t N);
hipError_t launch_decode(int dtype, const DecodeArgs &a, hipStream_t stream);
hipError_t launch_decode_experts(int dtype, const DecodeArgs &gate_up, const DecodeArgs &down, hipStream_t stream);

// more tokens: both operands through LDS, in tiles of several forms
constexpr int kTiledForms = 7, kForm64 = 1, kForm128 = 3, kForm256 = 6;   // (the experts': 128 x 64, 128 x 128, 256 x 128 rows x tokens)
hipError_t launch_tiled(int mode, int form, const ProductArgs &a, hipStream_t stream);   // the experts'
// a plain one, planned by its size
struct ProductPlan {
    int     form, rest;           // rest: of the rows behind main_tiles row tiles, or -1
    int64_t main_tiles;
    int     splits, split_steps;
    int     arrived;              // counters, and bytes of sums, that splits > 1 takes
    int64_t sums_bytes;
};
ProductPlan plan_product(int64_t M, int64_t N, int64_t K);
int64_t     product_sums_bytes(int64_t M, int64_t N, int64_t K);   // for sums and counters of up to M tokens
hipError_t launch_tiled_product(const ProductPlan &plan, const ProductArgs &a, hipStream_t stream);
int tiled_rows(int form);   // of a tile
int tiled_tokens(int form);
int tiled_resident(int form);
int64_t tiled_row_tiles(int mode, int form, int64_t N);

// Sorts the slots by expert, every expert's from a multiple of 32 positions on, and cuts them into tiles of tile_tokens positions.
struct SortArgs {
    const int32_t *ids;
    int            slots, top, E, tile_tokens, positions;   // (positions: at most)
    int           *token_of, *slot_of;   // by position: token, slot; token -1 where there is none
    Tile          *tiles;
    int            most_tiles;           // the table's length: the tiles behind the last get a count of 0
    int           *used;                 // how many positions there are
};
hipError_t launch_sort(const SortArgs &a, hipStream_t stream);
inline int64_t most_positions(int64_t slots, int64_t E) {
    const int64_t some = slots < E ? slots : E;
    return up_to(slots + 31 * some, 32);
}
inline int64_t most_tiles(int64_t slots, int64_t E, int tile_tokens) {
    const int64_t some = slots < E ? slots : E;
    return some + slots / tile_tokens;
}
// y[m] = sum_j weights[m][j] * rows[m * top + j], over the slots whose id is an expert's; rows of N
hipError_t launch_combine(const float *rows, int64_t N, const int32_t *ids, const float *weights, int64_t M, int top, int E, int out_dtype, void *y,
                          int64_t ldy, hipStream_t stream);

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
