// int8 quantiser and dequantiser, the rewriting of weights, and rows brought to multiples of 16 bytes.
//
// All of these are bound by memory.
#include "rq_prod.h"

namespace rq {
namespace prod {
namespace {

constexpr int kUnits = 4;   // of eight elements that a thread keeps between its row's maximum and the codes

template <int DT, bool VEC>
__device__ __forceinline__ void load_unit(const typename Element<DT>::type *x, int64_t K, int64_t k, float (&v)[8]) {
    using T = typename Element<DT>::type;
    if constexpr (VEC) {
        if constexpr (DT == RQ_F32) {
            const float4 a = reinterpret_cast<const float4 *>(x + k)[0], b = reinterpret_cast<const float4 *>(x + k)[1];
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
            const uint4    u = *reinterpret_cast<const uint4 *>(x + k);
            const uint32_t w[4] = { u.x, u.y, u.z, u.w };
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = to_float(__builtin_bit_cast(T, (uint16_t) w[i]));
                v[2 * i + 1] = to_float(__builtin_bit_cast(T, (uint16_t) (w[i] >> 16)));
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = k + i < K ? to_float(x[k + i]) : 0.0f;
    }
}
__device__ __forceinline__ uint32_t top_bits(const float (&v)[8], uint32_t top) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return top;
}
// A row a workgroup of G threads, or 256 / G rows where G < 256. VEC: rows of x on multiples of 16 bytes, K a multiple of 8. PITCH: codes go to rows of `pitch`
// bytes, on multiples of eight, with zeros up to `padded`; else to rows of K bytes in a row.
template <int DT, bool VEC, int G>
__global__ __launch_bounds__(G < 256 ? 256 : G) void rq_i8_quantize_kernel(const typename Element<DT>::type *x, int64_t ldx, int64_t M, int64_t K,
                                                                           uint8_t *codes, int64_t pitch, int64_t padded, float *scales, int *zero, int zeros) {
    if (zeros && blockIdx.x == 0)
        for (int i = threadIdx.x; i < zeros; i += (int) blockDim.x) zero[i] = 0;
    constexpr int kRows = G < 256 ? 256 / G : 1;
    const int     t = threadIdx.x % G, lane = threadIdx.x & 63;
    const int64_t m = (int64_t) blockIdx.x * kRows + threadIdx.x / G;
    const bool    there = m < M;
    const auto   *row = x + (there ? m : 0) * ldx;
    float         v[kUnits][8];
    uint32_t      top = 0;
    if (there) {
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int64_t k = (int64_t) (u * G + t) * 8;
            if (k < K) {
                load_unit<DT, VEC>(row, K, k, v[u]);
                top = top_bits(v[u], top);
            }
        }
        for (int64_t k = (int64_t) (kUnits * G + t) * 8; k < K; k += G * 8) {
            float w[8];
            load_unit<DT, VEC>(row, K, k, w);
            top = top_bits(w, top);
        }
    }
    top = wave_max(top);
    if constexpr (G > 64) {
        __shared__ uint32_t tops[G / 64];
        if (lane == 0) tops[threadIdx.x >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < G / 64; ++i) top = max(top, tops[i]);
    }
    if (!there) return;
    const RowScale q(top);
    if (t == 0) scales[m] = q.s;
    uint8_t *to = codes + m * pitch;
    auto     put = [&](int64_t k, const float(&w)[8]) __attribute__((always_inline)) {
        const uint2 c = codes_of(w, q.r, q.keep);
        if (VEC || k + 8 <= padded) {
            // (rows of K bytes are on multiples of eight where VEC is set, and padded rows always)
            *reinterpret_cast<uint2 *>(to + k) = c;
        } else {
            for (int i = 0; i < 8; ++i)
                if (k + i < K) to[k + i] = (uint8_t) ((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
        }
    };
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const int64_t k = (int64_t) (u * G + t) * 8;
        if (k < K) put(k, v[u]);
    }
    for (int64_t k = (int64_t) (kUnits * G + t) * 8; k < K; k += G * 8) {
        float w[8];
        load_unit<DT, VEC>(row, K, k, w);
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
    float         v[8];
    if constexpr (VEC) {
        const uint2 c = *reinterpret_cast<const uint2 *>(from);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float) (int8_t) ((i < 4 ? c.x : c.y) >> (8 * (i & 3))) * s;
        if constexpr (DT == RQ_F32) {
            reinterpret_cast<float4 *>(to)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4 *>(to)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            *reinterpret_cast<uint4 *>(to) = make_uint4(mx::pair_bits<DT>(v[0], v[1]), mx::pair_bits<DT>(v[2], v[3]),
                                                        mx::pair_bits<DT>(v[4], v[5]), mx::pair_bits<DT>(v[6], v[7]));
        }
    } else {
        for (int i = 0; i < 8; ++i)
            if (k + i < K) to[i] = from_float<DT>((float) from[i] * s);
    }
}

// 16 bytes a thread; experts are the grid's y and z.
template <bool VEC>
__global__ __launch_bounds__(256) void rq_weight_prepare_kernel(const uint8_t *w, const float *scales, Panels L, int64_t E, uint8_t *prepared) {
    const int64_t e = (int64_t) blockIdx.z * gridDim.y + blockIdx.y;
    if (e >= E) return;
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
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (b + j < L.row_bytes) v[j >> 2] |= (uint32_t) p[j] << (8 * (j & 3));
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
#pragma unroll
    for (int j = 0; j < 16; ++j)
        if (b + j < row_bytes) v[j >> 2] |= (uint32_t) p[j] << (8 * (j & 3));
    *reinterpret_cast<uint4 *>(to + m * pitch + b) = make_uint4(v[0], v[1], v[2], v[3]);
}

constexpr int64_t kGrid = 1ll << 23;   // workgroups of a launch (of up to 512 threads, of which a grid has under 2^32)

template <int DT, bool VEC, int G>
hipError_t quantize_rows(const void *x_, int64_t ldx, int64_t M, int64_t K, uint8_t *codes, int64_t pitch, int64_t padded, float *scales,
                         int *zero, int zeros, hipStream_t stream) {
    constexpr int kRows = G < 256 ? 256 / G : 1;
    constexpr int64_t kMost = kGrid / 2 * kRows;
    const auto   *x = reinterpret_cast<const typename Element<DT>::type *>(x_);
    for (int64_t m = 0; m < M; m += kMost) {
        const int64_t rows = M - m < kMost ? M - m : kMost;
        hipLaunchKernelGGL((rq_i8_quantize_kernel<DT, VEC, G>), dim3((unsigned) ((rows + kRows - 1) / kRows)), dim3(G < 256 ? 256 : G), 0, stream,
                           x + m * ldx, ldx, rows, K, codes + m * pitch, pitch, padded, scales + m, zero, m ? 0 : zeros);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}
template <int DT>
hipError_t quantize(const void *x, int64_t ldx, int64_t M, int64_t K, uint8_t *codes, int64_t pitch, int64_t padded, float *scales,
                    int *zero, int zeros, hipStream_t stream) {
    const int  size = DT == RQ_F32 ? 4 : 2;
    const bool vec = (uintptr_t) x % 16 == 0 && (M == 1 || ldx * size % 16 == 0) && K % 8 == 0 && (uintptr_t) codes % 8 == 0;
    if (K <= 2048) return vec ? quantize_rows<DT, true, 64>(x, ldx, M, K, codes, pitch, padded, scales, zero, zeros, stream)
                              : quantize_rows<DT, false, 64>(x, ldx, M, K, codes, pitch, padded, scales, zero, zeros, stream);
    if (K <= 8192) return vec ? quantize_rows<DT, true, 256>(x, ldx, M, K, codes, pitch, padded, scales, zero, zeros, stream)
                              : quantize_rows<DT, false, 256>(x, ldx, M, K, codes, pitch, padded, scales, zero, zeros, stream);
    return vec ? quantize_rows<DT, true, 512>(x, ldx, M, K, codes, pitch, padded, scales, zero, zeros, stream)
               : quantize_rows<DT, false, 512>(x, ldx, M, K, codes, pitch, padded, scales, zero, zeros, stream);
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
        hipLaunchKernelGGL(rq_weight_prepare_kernel<true>, grid, dim3(256), 0, (hipStream_t) stream, (const uint8_t *) w, scales, L, E, (uint8_t *) prepared);
    } else {
        hipLaunchKernelGGL(rq_weight_prepare_kernel<false>, grid, dim3(256), 0, (hipStream_t) stream, (const uint8_t *) w, scales, L, E, (uint8_t *) prepared);
    }
    return hipGetLastError();
}
