// Shared definitions of the int8 products and of the products grouped by expert: layouts, matrix instructions, launch arguments.
#pragma once

#include "../../include/rq_i8.h"
#include "rq_mx.h"

namespace rq {
namespace prod {

using mx::allow_lds;
using mx::Element;
using mx::from_float;
using mx::store_out;
using mx::to_float;
using mx::up_to;
using mx::v16f;
using mx::v4f;
using mx::v4i;
typedef int    v16i __attribute__((ext_vector_type(16)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

inline int type_bytes(int type) { return type == RQ_F32 ? 4 : type == RQ_I8 ? 1 : 2; }

// ---------------------------------------------------------------------------------------------------
// All three types are fed to the matrix cores in 16 bytes a lane: a 32x32x32 (int8) or 32x32x16 (16 bits) MFMA takes from lane l of
// either operand row l % 32 and bytes 16 (l / 32) .. + 15 of a run of 32 bytes of the row. Lane l holds of the 32 x 32 result column l % 32
// and rows 8 (i / 4) + 4 (l / 32) + i % 4, i = 0 .. 15. The 16x16 forms take row l % 16 and bytes 16 (l / 16) of a run of 64; lane l holds column
// l % 16 and rows 4 (l / 16) + i. (Which element of a run a byte stands for is the same for both operands, so it does not matter.)
//
// Prepared weight, per expert: N / 32 row blocks x steps of 64 bytes x 2 runs x 64 lanes x 16 bytes (rows and bytes padded with zeros), so a
// wavefront reads a fragment as 1 KiB of consecutive bytes; behind them, of int8, a scale for each row of the blocks.
// Activations stay rows, `pitch` bytes apart and on multiples of 16: what gathers them costs nothing then.
// ---------------------------------------------------------------------------------------------------
struct Panels {
    int64_t N, row_bytes;                // rows; bytes of a row that count
    int     row_blocks, steps;
    int64_t code_bytes, expert_bytes;    // of one expert
};
inline Panels panels(int type, int64_t N, int64_t K) {
    Panels L;
    L.N = N;
    L.row_bytes = K * type_bytes(type);
    L.row_blocks = (int) (up_to(N, 32) / 32);
    L.steps = (int) (up_to(L.row_bytes, 64) / 64);
    L.code_bytes = (int64_t) L.row_blocks * L.steps * 2048;
    L.expert_bytes = L.code_bytes + (type == RQ_I8 ? up_to((int64_t) L.row_blocks * 128, 256) : 0);
    return L;
}

template <int WT> struct Matrix;
template <> struct Matrix<RQ_I8> {
    using Acc = v16i;
    using Acc4 = v4i;
    static __device__ __forceinline__ Acc mfma(const v4i &a, const v4i &b, const Acc &c) { return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ Acc4 mfma16(const v4i &a, const v4i &b, const Acc4 &c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
};
template <> struct Matrix<RQ_BF16> {
    using Acc = v16f;
    using Acc4 = v4f;
    static __device__ __forceinline__ Acc mfma(const v4i &a, const v4i &b, const Acc &c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ Acc4 mfma16(const v4i &a, const v4i &b, const Acc4 &c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
    }
};
template <> struct Matrix<RQ_F16> {
    using Acc = v16f;
    using Acc4 = v4f;
    static __device__ __forceinline__ Acc mfma(const v4i &a, const v4i &b, const Acc &c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ Acc4 mfma16(const v4i &a, const v4i &b, const Acc4 &c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
    }
};

struct ProductArgs {
    Panels         L;
    const uint8_t *w;              // prepared
    const uint8_t *x;              // rows of x; for the tiles on multiples of 16 bytes
    int64_t        pitch, x_bytes; // of a row: distance, and how many there are to read (for the tiles a multiple of 16), with zeros behind them
    int64_t        K;              // launch_stream where it rounds: x is the call's own, `pitch` its row stride in elements, rows of K;
    bool           aligned;        //   whether they are on multiples of 16 bytes, and K of eight;
    int            chunk;          //   up to so many rows at a time (16 where it does not round)
    const float   *x_scales;       // of int8 rows
    int64_t        M;              // rows of x
    int64_t        P;              // positions
    const int32_t *offsets;        // null: one group of all positions
    int            E;
    const int32_t *rows, *out_rows;
    int            out_dtype;
    void          *y;
    int64_t        ldy, y_rows;
    int            first_block, row_tiles;   // tiles: the row blocks of this launch start here, and how many tiles they make (0: all)
    int            splits, split_steps;      //   workgroups that share a tile, and the steps of 64 bytes of each (even)
    uint32_t      *sums;                     //   splits > 1: what they leave
    int           *arrived;                  //   and how many have, by wavefront's outputs: zero before the launch
};

// The rows that position p reads and writes; -1: none.
__device__ __forceinline__ int64_t row_read(const ProductArgs &a, int64_t p) {
    if (!a.rows) return p < a.M ? p : -1;
    const int64_t r = a.rows[p];
    return r >= 0 && r < a.M ? r : -1;
}
__device__ __forceinline__ int64_t row_written(const ProductArgs &a, int64_t p) {
    if (!a.out_rows) return p < a.y_rows ? p : -1;
    const int64_t r = a.out_rows[p];
    return r >= 0 && r < a.y_rows ? r : -1;
}
// Group e's first position and how many it has. (Both ends are clamped on both sides: an offset may be any number, and the difference of two is not.)
__device__ __forceinline__ void group(const ProductArgs &a, int e, int &first, int &count) {
    const int P = (int) a.P;
    first = min(max(a.offsets[e], 0), P);
    count = max(min(max(a.offsets[e + 1], 0), P) - first, 0);
}
// Group e has units(its count) units, and all groups' stand in a row. Finds the group that has unit want(how many there are), and the place in it; all lanes
// of a wavefront take part, with the same numbers. False where no group has it. TOTAL: `want` looks at its argument (else it is 0).
template <bool TOTAL, typename U, typename W>
__device__ __forceinline__ bool find_group(const ProductArgs &a, U units, W want, int &e_, int &first_, int &count_, int &place_) {
    const int lane = threadIdx.x & 63;
    auto      scan = [&](int e0, int &first, int &count, int &mine) __attribute__((always_inline)) {   // of 64 groups: the units up to this lane's last
        first = count = 0;
        if (e0 + lane < a.E) group(a, e0 + lane, first, count);
        mine = units(count);
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(sum, o);
            if (lane >= o) sum += u;
        }
        return sum;
    };
    int  first, count, mine, wanted = 0;
    auto found = [&](int e0, int from) __attribute__((always_inline)) {
        const uint64_t here = __ballot(wanted >= from && wanted < from + mine);
        if (!here) return false;
        const int l = __builtin_ctzll(here);
        e_ = e0 + l;
        first_ = __builtin_amdgcn_readlane(first, l);
        count_ = __builtin_amdgcn_readlane(count, l);
        place_ = wanted - __builtin_amdgcn_readlane(from, l);
        return true;
    };
    if (a.E <= 64) {
        const int sum = scan(0, first, count, mine);
        wanted = want(__builtin_amdgcn_readlane(sum, 63));
        return found(0, sum - mine);
    }
    int total = 0;
    if (TOTAL)
        for (int e0 = 0; e0 < a.E; e0 += 64) total += __builtin_amdgcn_readlane(scan(e0, first, count, mine), 63);
    wanted = want(total);
    for (int e0 = 0, before = 0; e0 < a.E; e0 += 64) {
        const int sum = scan(e0, first, count, mine);
        if (found(e0, before + sum - mine)) return true;
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

// ---- loads and stores at any address (the card takes them, in pieces where they cross lines) ------------------
template <int N>
__device__ __forceinline__ void load_bytes(uint32_t (&w)[N], const void *p) { __builtin_memcpy(w, p, N * 4); }
__device__ __forceinline__ void store_bytes(void *p, const uint2 &v) { __builtin_memcpy(p, &v, 8); }

// ---- rounding of a row to int8 ------------------------------------------------------------------------
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v = max(v, (uint32_t) __shfl_xor((int) v, o));
    return v;
}
// From the bits of a row's largest magnitude: its scale, what the elements are multiplied by, and the codes' bits that count (none where the row holds
// an infinity or a NaN).
struct RowScale {
    float    s, r;
    uint32_t keep;
    __device__ __forceinline__ RowScale(uint32_t top) {
        s = __uint_as_float(top) * (1.0f / 127.0f);
        s = s > 0x1p-126f ? s : 0x1p-126f;
        r = 1.0f / s;
        keep = top < 0x7F800000u ? ~0u : 0u;
        if (!keep) s = __uint_as_float(0x7FC00000u);
    }
};
// The codes of eight elements. A code is the nearest whole number of x r: fma(x, r, 1.5 x 2^23) rounds the exact product once, to the nearest whole
// number, ties to even, and leaves it in the low bits; |x r| is at most 127 (1 + 2^-22).
__device__ __forceinline__ uint2 codes_of(const float (&v)[8], float r, uint32_t keep) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(fmaf(v[4 * h + i], r, 12582912.0f));
        const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000C0Cu);
        w[h] = (lo | hi) & keep;
    }
    return make_uint2(w[0], w[1]);
}

// ---- launches ---------------------------------------------------------------------------------------
// x -> codes in rows of `pitch` bytes, the places behind K zeros up to `padded` of them, and scales. Sets zero[0 .. zeros - 1] to 0.
hipError_t launch_i8_quantize(int dtype, const void *x, int64_t ldx, int64_t M, int64_t K, uint8_t *codes, int64_t pitch, int64_t padded,
                              float *scales, int *zero, int zeros, hipStream_t stream);
// rows of row_bytes bytes (distance ld_bytes) -> rows of `pitch` bytes, zeros behind them. Sets zero[0 .. zeros - 1] to 0, also where M is 0.
hipError_t launch_pack(const void *x, int64_t ld_bytes, int64_t M, int64_t row_bytes, uint8_t *to, int64_t pitch, int *zero, int zeros, hipStream_t stream);

// Few rows a group: weights from memory into registers. x_type: the type of the rows of x where it rounds them, else RQ_I8.
hipError_t launch_stream(int weight_type, int x_type, const ProductArgs &a, hipStream_t stream);
// How many rows at a time launch_stream rounds itself, of P in E groups (0: one); 0 where a launch in front is faster, or they do not fit.
int stream_rounds(int64_t P, int64_t K, int64_t N, int64_t E);

// more: both operands through LDS, in tiles of several forms
constexpr int kForms = 5;   // 64 x 64, 128 x 64, 128 x 128 (two a compute unit), 128 x 128 (one), 256 x 256 rows x positions
hipError_t launch_tiled(int weight_type, int form, const ProductArgs &a, hipStream_t stream);
int        tiled_rows(int form);
int        tiled_tokens(int form);
// tiles of T positions: of P in one group (E = 0), or at most, of P in E groups
inline int64_t most_token_tiles(int T, int64_t P, int64_t E) { return E == 0 ? (P + T - 1) / T : P / T + (P < E ? P : E); }

}  // namespace prod
}  // namespace rq
