// int8 quantiser and dequantiser, the rewriting of weights, and rows brought to multiples of 16 bytes.
//
// One pass over memory each, bound by it: 17408 x 5120 in fp32 is rounded in 83 to 103 us and taken back in 77, 446 MB each; 2048 x 5120 bf16 is rounded in 9, of which
// 6 are its 31 MB; a weight of 64 x 1280 x 5120 int8 is rewritten in 141 us, 839 MB. A row's threads keep it between the maximum and the codes. (1 to 17408 rows of 512 to
// 17408: 64 to 512 threads a row by its length are within 6 % of the fastest of fifteen shapes, rows of 5120 to 17408 in fp32 within 7.)
#include "rq_prod.h"

namespace rq {
namespace prod {
namespace {

// Eight elements of a row as they lie, zeros behind its end; 16-bit ones in pairs. VEC: on 16 bytes, and rows of a multiple of eight.
template <int DT> struct Eight {
    using T = typename Element<DT>::type;
    static constexpr bool kWide = DT == RQ_F32;
    uint32_t w[kWide ? 8 : 4];
    template <bool VEC> __device__ __forceinline__ void load(const T *x, int64_t K, int64_t k) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < (kWide ? 2 : 1); ++i) {
                const uint4 u = reinterpret_cast<const uint4 *>(x + k)[i];
                w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
            }
        } else if (k + 8 <= K) {
            load_bytes(w, x + k);
        } else if constexpr (kWide) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = k + i < K ? __float_as_uint(x[k + i]) : 0u;
        } else {
            const uint16_t *h = reinterpret_cast<const uint16_t *>(x) + k;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = (k + 2 * i < K ? h[2 * i] : 0u) | (k + 2 * i + 1 < K ? (uint32_t) h[2 * i + 1] << 16 : 0u);
        }
    }
    // the larger of `top`, the bits of a magnitude in this type, and those of the elements
    __device__ __forceinline__ uint32_t top(uint32_t t) const {
        if constexpr (kWide) {
#pragma unroll
            for (int i = 0; i < 8; ++i) t = max(t, w[i] & 0x7FFFFFFFu);
            return t;
        } else {
            typedef uint16_t u2 __attribute__((ext_vector_type(2)));
            u2 m = __builtin_bit_cast(u2, w[0] & 0x7FFF7FFFu);
#pragma unroll
            for (int i = 1; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u2, w[i] & 0x7FFF7FFFu));
            const uint32_t both = __builtin_bit_cast(uint32_t, m);
            return max(t, max(both & 0xFFFF, both >> 16));
        }
    }
    static __device__ __forceinline__ uint32_t as_float_bits(uint32_t t) {
        if constexpr (kWide) return t;
        else return __float_as_uint(to_float(__builtin_bit_cast(T, (uint16_t) t)));
    }
    __device__ __forceinline__ uint2 codes(const RowScale &q) const {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (kWide) v[i] = __uint_as_float(w[i]);
            else v[i] = to_float(__builtin_bit_cast(T, (uint16_t) (i & 1 ? w[i >> 1] >> 16 : w[i >> 1])));
        }
        return codes_of(v, q.r, q.keep);
    }
};

// A row by G threads, U units of eight elements of it held by each between its maximum and the codes; what is longer is read twice. VEC: rows of x on multiples of
// 16 bytes, K a multiple of 8. Codes go to rows of `pitch` bytes: on multiples of eight with zeros up to `padded`, or (padded 0) of K bytes in a row.
template <int DT, bool VEC, int G, int U>
__global__ __launch_bounds__(G < 256 ? 256 : G) void rq_i8_quantize_kernel(const typename Element<DT>::type *x, int64_t ldx, int64_t M, int64_t K,
                                                                           uint8_t *codes, int64_t pitch, int64_t padded, float *scales, int *zero, int zeros) {
    if (zeros && blockIdx.x == 0)
        for (int i = threadIdx.x; i < zeros; i += (int) blockDim.x) zero[i] = 0;
    constexpr int kRows = G < 256 ? 256 / G : 1, kWaves = G / 64;
    const int     t = threadIdx.x % G, lane = threadIdx.x & 63;
    const int64_t m = (int64_t) blockIdx.x * kRows + threadIdx.x / G;
    const bool    there = m < M;
    const auto   *row = x + (there ? m : 0) * ldx;
    Eight<DT>     v[U];
    uint32_t      top = 0;
    if (there) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t k = (int64_t) (u * G + t) * 8;
            if (k < K) v[u].template load<VEC>(row, K, k);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if ((int64_t) (u * G + t) * 8 < K) top = v[u].top(top);
        for (int64_t k = (int64_t) (U * G + t) * 8; k < K; k += G * 8) {
            Eight<DT> w;
            w.template load<VEC>(row, K, k);
            top = w.top(top);
        }
    }
    top = wave_max(top);
    if constexpr (kWaves > 1) {
        __shared__ uint32_t tops[G < 256 ? 4 : kWaves];
        if (lane == 0) tops[threadIdx.x >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kWaves; ++i) top = max(top, tops[threadIdx.x / G * kWaves + i]);
    }
    if (!there) return;
    const RowScale q(Eight<DT>::as_float_bits(top));
    if (t == 0) scales[m] = q.s;
    uint8_t *to = codes + m * pitch;
    auto     put = [&](int64_t k, const Eight<DT> &w) __attribute__((always_inline)) {
        const uint2 c = w.codes(q);
        if (VEC || k + 8 <= padded) {
            // (rows of K bytes are on multiples of eight where VEC is set, and padded rows always)
            *reinterpret_cast<uint2 *>(to + k) = c;
        } else if (k + 8 <= K) {
            store_bytes(to + k, c);
        } else {
            for (int i = 0; i < 8; ++i)
                if (k + i < K) to[k + i] = (uint8_t) ((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
        }
    };
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t k = (int64_t) (u * G + t) * 8;
        if (k < K) put(k, v[u]);
    }
    for (int64_t k = (int64_t) (U * G + t) * 8; k < K; k += G * 8) {
        Eight<DT> w;
        w.template load<VEC>(row, K, k);
        put(k, w);
    }
    for (int64_t k = (K + 7) / 8 * 8 + t * 8; k < padded; k += G * 8) *reinterpret_cast<uint2 *>(to + k) = make_uint2(0, 0);
}

// Eight elements a thread, a row a run of workgroups.
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void rq_i8_dequantize_kernel(const int8_t *codes, const float *scales, int64_t M, int64_t K,
                                                               typename Element<DT>::type *out, int64_t ldo) {
    const int64_t per_row = (K + 7) / 8, n = (int64_t) blockIdx.x * 256 + threadIdx.x;
    const int64_t m = n / per_row, k = (n - m * per_row) * 8;
    if (m >= M) return;
    const float   s = scales[m];
    const int8_t *from = codes + m * K + k;
    auto         *to = out + m * ldo + k;
    if (!VEC && k + 8 > K) {
        for (int i = 0; k + i < K; ++i) to[i] = from_float<DT>((float) from[i] * s);
        return;
    }
    uint32_t c[2], w[DT == RQ_F32 ? 8 : 4];
    float    v[8];
    load_bytes(c, from);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float) (int8_t) (c[i >> 2] >> (8 * (i & 3))) * s;
#pragma unroll
    for (int i = 0; i < (DT == RQ_F32 ? 8 : 4); ++i) {
        if constexpr (DT == RQ_F32) w[i] = __float_as_uint(v[i]);
        else w[i] = mx::pair_bits<DT>(v[2 * i], v[2 * i + 1]);
    }
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < (DT == RQ_F32 ? 2 : 1); ++i) reinterpret_cast<uint4 *>(to)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    } else {
        __builtin_memcpy(to, w, sizeof(w));
    }
}

// 16 bytes a thread; experts are the grid's y.
template <bool VEC>
__global__ __launch_bounds__(256) void rq_weight_prepare_kernel(const uint8_t *w, const float *scales, Panels L, uint8_t *prepared) {
    const int64_t  e = blockIdx.y;
    const uint8_t *from = w + e * L.N * L.row_bytes;
    uint8_t       *to = prepared + e * L.expert_bytes;
    const int64_t  pieces = L.code_bytes / 16, words = scales ? (int64_t) L.row_blocks * 32 : 0;
    for (int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x; i < pieces + words; i += (int64_t) gridDim.x * 256) {
        if (i >= pieces) {
            const int64_t n = i - pieces;
            reinterpret_cast<float *>(to + L.code_bytes)[n] = n < L.N ? scales[e * L.N + n] : 0.0f;
            continue;
        }
        const int     lane = (int) i & 63;
        const int64_t runs = 2 * (int64_t) L.steps, block = (i >> 6) / runs, run = (i >> 6) - block * runs;
        const int64_t row = block * 32 + (lane & 31), b = run * 32 + (lane >> 5) * 16;
        uint32_t      v[4] = { 0, 0, 0, 0 };
        if (row < L.N && b < L.row_bytes) {
            const uint8_t *p = from + row * L.row_bytes + b;
            if constexpr (VEC) {
                const uint4 u = *reinterpret_cast<const uint4 *>(p);
                v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
            } else if (b + 16 <= L.row_bytes) {
                load_bytes(v, p);
            } else {
                for (int j = 0; b + j < L.row_bytes; ++j) v[j >> 2] |= (uint32_t) p[j] << (8 * (j & 3));
            }
        }
        reinterpret_cast<uint4 *>(to)[i] = make_uint4(v[0], v[1], v[2], v[3]);
    }
}

// 16 bytes a thread
__global__ __launch_bounds__(256) void rq_pack_kernel(const uint8_t *x, int64_t ld, int64_t M, int64_t row_bytes, uint8_t *to, int64_t pitch, int *zero, int zeros) {
    if (zeros && blockIdx.x == 0)
        for (int i = threadIdx.x; i < zeros; i += 256) zero[i] = 0;
    const int64_t per_row = pitch / 16, n = (int64_t) blockIdx.x * 256 + threadIdx.x;
    const int64_t m = n / per_row, b = (n - m * per_row) * 16;
    if (m >= M) return;
    const uint8_t *p = x + m * ld + b;
    uint32_t       v[4] = { 0, 0, 0, 0 };
    if (b + 16 <= row_bytes) {
        load_bytes(v, p);
    } else {
        for (int j = 0; b + j < row_bytes; ++j) v[j >> 2] |= (uint32_t) p[j] << (8 * (j & 3));
    }
    *reinterpret_cast<uint4 *>(to + m * pitch + b) = make_uint4(v[0], v[1], v[2], v[3]);
}

constexpr int64_t kGrid = 1ll << 23;   // workgroups of a launch (of up to 512 threads, of which a grid has under 2^32)

template <int DT, bool VEC, int G, int U>
hipError_t quantize_rows(const void *x_, int64_t ldx, int64_t M, int64_t K, uint8_t *codes, int64_t pitch, int64_t padded, float *scales,
                         int *zero, int zeros, hipStream_t stream) {
    constexpr int kRows = G < 256 ? 256 / G : 1;
    constexpr int64_t kMost = kGrid / 2 * kRows;
    const auto   *x = reinterpret_cast<const typename Element<DT>::type *>(x_);
    for (int64_t m = 0; m < M; m += kMost) {
        const int64_t rows = M - m < kMost ? M - m : kMost;
        hipLaunchKernelGGL((rq_i8_quantize_kernel<DT, VEC, G, U>), dim3((unsigned) ((rows + kRows - 1) / kRows)), dim3(G < 256 ? 256 : G), 0, stream,
                           x + m * ldx, ldx, rows, K, codes + m * pitch, pitch, padded, scales + m, zero, m ? 0 : zeros);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}
template <int DT, bool VEC>
hipError_t quantize(const void *x, int64_t ldx, int64_t M, int64_t K, uint8_t *codes, int64_t pitch, int64_t padded, float *scales,
                    int *zero, int zeros, hipStream_t stream) {
    if (K <= 2048) return quantize_rows<DT, VEC, 64, 4>(x, ldx, M, K, codes, pitch, padded, scales, zero, zeros, stream);
    if (K <= 8192) return quantize_rows<DT, VEC, 256, 4>(x, ldx, M, K, codes, pitch, padded, scales, zero, zeros, stream);
    return quantize_rows<DT, VEC, 512, 4>(x, ldx, M, K, codes, pitch, padded, scales, zero, zeros, stream);
}
template <int DT>
hipError_t quantize(const void *x, int64_t ldx, int64_t M, int64_t K, uint8_t *codes, int64_t pitch, int64_t padded, float *scales,
                    int *zero, int zeros, hipStream_t stream) {
    const int  size = DT == RQ_F32 ? 4 : 2;
    const bool vec = (uintptr_t) x % 16 == 0 && (M == 1 || ldx * size % 16 == 0) && K % 8 == 0 && (uintptr_t) codes % 8 == 0;
    return vec ? quantize<DT, true>(x, ldx, M, K, codes, pitch, padded, scales, zero, zeros, stream)
               : quantize<DT, false>(x, ldx, M, K, codes, pitch, padded, scales, zero, zeros, stream);
}

template <int DT>
hipError_t dequantize(const void *codes_, const float *scales, int64_t M, int64_t K, void *out_, int64_t ldo, hipStream_t stream) {
    using T = typename Element<DT>::type;
    const int8_t *codes = reinterpret_cast<const int8_t *>(codes_);
    T            *out = reinterpret_cast<T *>(out_);
    const bool    vec = K % 8 == 0 && (uintptr_t) codes % 8 == 0 && (uintptr_t) out % 16 == 0 && (M == 1 || ldo * (int64_t) sizeof(T) % 16 == 0);
    const int64_t per_row = (K + 7) / 8, most = kGrid * 256 / per_row;   // (K up to 2^30: at least 16)
    for (int64_t m = 0; m < M; m += most) {
        const int64_t rows = M - m < most ? M - m : most;
        const dim3    grid((unsigned) ((rows * per_row + 255) / 256));
        if (vec) hipLaunchKernelGGL((rq_i8_dequantize_kernel<DT, true>), grid, dim3(256), 0, stream, codes + m * K, scales + m, rows, K, out + m * ldo, ldo);
        else hipLaunchKernelGGL((rq_i8_dequantize_kernel<DT, false>), grid, dim3(256), 0, stream, codes + m * K, scales + m, rows, K, out + m * ldo, ldo);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

hipError_t launch_i8_quantize(int dtype, const void *x, int64_t ldx, int64_t M, int64_t K, uint8_t *codes, int64_t pitch, int64_t padded,
                              float *scales, int *zero, int zeros, hipStream_t stream) {
    if (dtype == RQ_F32) return quantize<RQ_F32>(x, ldx, M, K, codes, pitch, padded, scales, zero, zeros, stream);
    if (dtype == RQ_F16) return quantize<RQ_F16>(x, ldx, M, K, codes, pitch, padded, scales, zero, zeros, stream);
    return quantize<RQ_BF16>(x, ldx, M, K, codes, pitch, padded, scales, zero, zeros, stream);
}

hipError_t launch_pack(const void *x, int64_t ld_bytes, int64_t M, int64_t row_bytes, uint8_t *to, int64_t pitch, int *zero, int zeros, hipStream_t stream) {
    const int64_t per_row = pitch / 16, most = kGrid * 256 / per_row;   // (pitch up to 2^18)
    for (int64_t m = 0; m < M || m == 0; m += most) {
        const int64_t rows = M - m < most ? M - m : most;
        hipLaunchKernelGGL(rq_pack_kernel, dim3((unsigned) ((rows * per_row + 255) / 256 + (rows == 0))), dim3(256), 0, stream,
                           (const uint8_t *) x + m * ld_bytes, ld_bytes, rows, row_bytes, to + m * pitch, pitch, zero, m ? 0 : zeros);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace prod
}  // namespace rq

using namespace rq::prod;

namespace {
bool float_dtype(int dtype) { return dtype == RQ_F32 || dtype == RQ_F16 || dtype == RQ_BF16; }
bool aligned_to(const void *p, size_t n) { return (uintptr_t) p % n == 0; }
constexpr int64_t kMostK = 1ll << 30;
}  // namespace

extern "C" int rq_i8_quantize(int dtype, const void *x, int64_t ldx, int64_t M, int64_t K, void *codes, float *scales, rq_stream_t stream) {
    if (!float_dtype(dtype) || K < 1 || K > kMostK || M < 0) return RQ_E_UNSUPPORTED;
    if (M == 0) return 0;
    if (!x || !aligned_to(x, type_bytes(dtype)) || !codes || !scales || !aligned_to(scales, 4) || (M > 1 && ldx < K)) return RQ_E_ARGUMENT;
    return launch_i8_quantize(dtype, x, ldx, M, K, (uint8_t *) codes, K, 0, scales, nullptr, 0, (hipStream_t) stream);
}

extern "C" int rq_i8_dequantize(int dtype, const void *codes, const float *scales, int64_t M, int64_t K, void *out, int64_t ldo,
                                rq_stream_t stream) {
    if (!float_dtype(dtype) || K < 1 || K > kMostK || M < 0) return RQ_E_UNSUPPORTED;
    if (M == 0) return 0;
    if (!out || !aligned_to(out, type_bytes(dtype)) || !codes || !scales || !aligned_to(scales, 4) || (M > 1 && ldo < K)) return RQ_E_ARGUMENT;
    const hipStream_t st = (hipStream_t) stream;
    if (dtype == RQ_F32) return dequantize<RQ_F32>(codes, scales, M, K, out, ldo, st);
    if (dtype == RQ_F16) return dequantize<RQ_F16>(codes, scales, M, K, out, ldo, st);
    return dequantize<RQ_BF16>(codes, scales, M, K, out, ldo, st);
}

extern "C" size_t rq_weight_prepared_bytes(int type, int64_t E, int64_t N, int64_t K) {
    if ((type != RQ_I8 && type != RQ_F16 && type != RQ_BF16) || E < 1 || E > RQ_GROUPED_MAX_E || N < 1 || N > (1 << 24) || K < 1 || K > RQ_I8_MAX_K) return 0;
    return (size_t) (E * panels(type, N, K).expert_bytes);
}

extern "C" int rq_weight_prepare(int type, const void *w, const float *scales, int64_t E, int64_t N, int64_t K, void *prepared,
                                 size_t prepared_bytes, rq_stream_t stream) {
    const size_t need = rq_weight_prepared_bytes(type, E, N, K);
    if (need == 0) return RQ_E_UNSUPPORTED;
    if (!w || !aligned_to(w, type_bytes(type)) || !prepared || !aligned_to(prepared, 256) || (type == RQ_I8) != (scales != nullptr) ||
        !aligned_to(scales, 4)) {
        return RQ_E_ARGUMENT;
    }
    if (prepared_bytes < need) return RQ_E_WORKSPACE;
    const Panels  L = panels(type, N, K);
    const int64_t x = (L.expert_bytes / 16 + 255) / 256;
    const dim3    grid((unsigned) (x < 4096 ? x : 4096), (unsigned) E);
    if (aligned_to(w, 16) && L.row_bytes % 16 == 0) {
        hipLaunchKernelGGL(rq_weight_prepare_kernel<true>, grid, dim3(256), 0, (hipStream_t) stream, (const uint8_t *) w, scales, L, (uint8_t *) prepared);
    } else {
        hipLaunchKernelGGL(rq_weight_prepare_kernel<false>, grid, dim3(256), 0, (hipStream_t) stream, (const uint8_t *) w, scales, L, (uint8_t *) prepared);
    }
    return hipGetLastError();
}
