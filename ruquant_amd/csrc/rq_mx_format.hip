// MXFP4 quantiser, dequantiser and the rewriting of weights.
//
// A block's scale byte is the exponent field of its largest magnitude less two: the maximum of the numbers' bits, which order them, and no
// division. An element times a power of two is exact, and the conversion to e2m1 rounds it once. All of these are one pass over
// memory, bound by it: 17408 x 5120 in fp32 is quantised in 90 us and taken back in 79, 404 MB each, 4.5 and 5.1 TB/s (a plain copy: 4.95).
#include "rq_mx.h"

namespace rq {
namespace mx {
namespace {

constexpr int kThreads = 256;

// n / d and n % d for n < 2^31 by a multiplication
struct Divider {
    uint32_t d, mul;
    int      shift;
};
Divider make_divider(uint32_t d) {
    int s = 0;
    while ((1u << s) < d) ++s;
    return { d, (uint32_t) (((1ull << (31 + s)) + d - 1) / d), 31 + s };
}
__device__ __forceinline__ uint32_t divide(uint32_t n, const Divider &v) { return (uint32_t) (((uint64_t) n * v.mul) >> v.shift); }

// Eight elements a thread, so four lanes hold a block and its maximum crosses them in two steps. ACT: the workspace's form, rows
// padded with zeros; otherwise rows of K / 2 and K / 32 bytes.
template <int DT, bool VEC, bool ACT>
__global__ __launch_bounds__(kThreads) void rq_mx_quantize_kernel(const typename Element<DT>::type *x, int64_t ldx, uint32_t units,
                                                                  Divider per_row, int64_t K, uint8_t *codes, int64_t code_stride,
                                                                  uint8_t *scales, int64_t scale_stride) {
    const uint32_t n = blockIdx.x * kThreads + threadIdx.x;
    if (n >= units) return;   // (whole blocks: units is a multiple of four)
    const uint32_t m = divide(n, per_row), u = n - m * per_row.d;
    Unit<DT>       v;
    v.clear();
    if (!ACT || (int64_t) u * 8 < K) v.template load<VEC>(x + (int64_t) m * ldx + (int64_t) u * 8);
    const int      X = block_scale(max_of_four(v.top()));
    const uint32_t c = v.pack(X);
    if (!ACT || (int64_t) u * 4 < code_stride) *reinterpret_cast<uint32_t *>(codes + (int64_t) m * code_stride + (int64_t) u * 4) = c;
    if ((u & 3) == 0) {
        const uint32_t b = u >> 2;
        scales[(int64_t) m * scale_stride + (ACT ? act_scale_at(b) : b)] = (uint8_t) X;
    }
}

// The panel form: a workgroup has 32 rows x 256 elements, eight threads a row and run of 64, so that a wavefront reads eight rows'
// lines and writes two lines of codes; a thread's four scales are one word. The grid is the parts of a row, then the row blocks: the threads of a
// long call are more than one dimension of a grid may have.
constexpr int kPanelBlocks = 32768;
template <int DT, bool VEC>
__global__ __launch_bounds__(kThreads) void rq_mx_panel_quantize_kernel(const typename Element<DT>::type *x, int64_t ldx, WeightLayout L,
                                                                        const int *row_of, const int *rows, uint8_t *panels, int *zero, int zeros) {
    if (blockIdx.y == 0 && blockIdx.z == 0)
        for (int i = blockIdx.x * kThreads + threadIdx.x; i < zeros; i += gridDim.x * kThreads) zero[i] = 0;
    const int     parts = 2 * L.chunks;
    const int     block = blockIdx.z * kPanelBlocks + blockIdx.y, part = blockIdx.x;
    const int     row = threadIdx.x >> 3, u = threadIdx.x & 7;
    const int64_t r = (int64_t) block * 32 + row;
    if ((int64_t) block * 32 >= (rows ? *rows : L.N)) return;
    const int64_t m = r < L.N ? row_of ? row_of[r] : r : -1;
    if (m < 0) return;   // (all eight threads of a row)
    uint8_t *codes = panels + ((int64_t) block * L.steps * 2 + part * 4) * 1024 + ((u >> 2) * 32 + row) * 16 + (u & 3) * 4;
    uint32_t word = 0;
    Unit<DT> v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t k = (int64_t) part * 256 + j * 64 + u * 8;
        v[j].clear();
        if (k < L.K) v[j].template load<VEC>(x + m * ldx + k);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int X = block_scale(max_of_four(v[j].top()));
        if (part * 4 + j < 2 * L.steps) *reinterpret_cast<uint32_t *>(codes + j * 1024) = v[j].pack(X);
        word |= (uint32_t) X << (8 * j);
    }
    if ((u & 3) == 0)
        reinterpret_cast<uint32_t *>(panels + L.code_bytes + ((int64_t) block * parts + part) * 256)[(u >> 2) * 32 + row] = word;
}

template <int DT, bool VEC>
__global__ __launch_bounds__(kThreads) void rq_mx_dequantize_kernel(const uint8_t *codes, const uint8_t *scales, uint32_t units,
                                                                    Divider per_row, int64_t K, typename Element<DT>::type *out,
                                                                    int64_t ldo) {
    const uint32_t n = blockIdx.x * kThreads + threadIdx.x;
    if (n >= units) return;
    const uint32_t m = divide(n, per_row), u = n - m * per_row.d;
    const uint32_t c = *reinterpret_cast<const uint32_t *>(codes + (int64_t) m * (K / 2) + (int64_t) u * 4);
    const float    s = scale_value(scales[(int64_t) m * (K / 32) + (u >> 2)]);
    float          v[8];
    v2f            p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0);
    v[0] = p[0] * s, v[1] = p[1] * s;
    p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1);
    v[2] = p[0] * s, v[3] = p[1] * s;
    p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 2);
    v[4] = p[0] * s, v[5] = p[1] * s;
    p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 3);
    v[6] = p[0] * s, v[7] = p[1] * s;
    typename Element<DT>::type *o = out + (int64_t) m * ldo + (int64_t) u * 8;
    if constexpr (!VEC) {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = from_float<DT>(v[i]);
    } else if constexpr (DT == RQ_F32) {
        reinterpret_cast<float4 *>(o)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4 *>(o)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = (uint32_t) __builtin_bit_cast(uint16_t, from_float<DT>(v[2 * i])) |
                   (uint32_t) __builtin_bit_cast(uint16_t, from_float<DT>(v[2 * i + 1])) << 16;
        }
        *reinterpret_cast<uint4 *>(o) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// The prepared weight, 16 bytes of codes or four of scales a thread; experts are the grid's y and z. Bound by memory: a wavefront writes 1 KiB in a row
// and reads 32 bytes from each of 32 rows, whose lines the next ones share: 17408 x 5120 26 us, 95 MB, 3.6 TB/s, 64 experts of 1280 x 5120 97 us, 4.6.
__global__ __launch_bounds__(kThreads) void rq_mx_prepare_kernel(const uint8_t *codes, const uint8_t *scales, WeightLayout L, int64_t E,
                                                                 uint8_t *prepared) {
    const int64_t e = (int64_t) blockIdx.z * gridDim.y + blockIdx.y;
    if (e >= E) return;
    const int64_t pieces = L.code_bytes / 16, words = (int64_t) L.row_blocks * L.chunks * 128;
    const uint8_t *c = codes + e * L.N * (L.K / 2), *s = scales + e * L.N * (L.K / 32);
    uint8_t       *to = prepared + e * L.expert_bytes;
    for (int64_t i = (int64_t) blockIdx.x * kThreads + threadIdx.x; i < pieces + words; i += (int64_t) gridDim.x * kThreads) {
        const int lane = (int) (i < pieces ? i : i - pieces) & 63;
        if (i < pieces) {
            const int64_t block = (i >> 6) / (2 * L.steps), run = (i >> 6) - block * 2 * L.steps;
            const int64_t row = block * 32 + (lane & 31), k = run * 64 + (lane >> 5) * 32;
            uint4         v = make_uint4(0, 0, 0, 0);
            if (row < L.N && k < L.K) v = *reinterpret_cast<const uint4 *>(c + row * (L.K / 2) + k / 2);
            reinterpret_cast<uint4 *>(to)[i] = v;
        } else {
            const int64_t w = (i - pieces) >> 6;
            const int64_t block = w / (2 * L.chunks), part = w - block * 2 * L.chunks;   // (of 256 inputs)
            const int64_t row = block * 32 + (lane & 31);
            uint32_t      v = 0;
            for (int j = 0; j < 4; ++j) {
                const int64_t b = part * 8 + j * 2 + (lane >> 5);
                v |= (row < L.N && b < L.K / 32 ? (uint32_t) s[row * (L.K / 32) + b] : 127u) << (8 * j);
            }
            reinterpret_cast<uint32_t *>(to + L.code_bytes)[i - pieces] = v;
        }
    }
}

template <int DT, bool ACT>
hipError_t quantize(const void *x_, int64_t ldx, int64_t M, int64_t K, uint8_t *codes, uint8_t *scales, int64_t code_stride,
                    int64_t scale_stride, int64_t per_row, hipStream_t stream) {
    using T = typename Element<DT>::type;
    const T      *x = reinterpret_cast<const T *>(x_);
    const bool    vec = (uintptr_t) x % 16 == 0 && (M == 1 || ldx * (int64_t) sizeof(T) % 16 == 0);
    const Divider d = make_divider((uint32_t) per_row);
    const int64_t rows = (1ll << 30) / per_row;   // of one launch, for the division
    for (int64_t m = 0; m < M; m += rows) {
        const uint32_t units = (uint32_t) ((M - m < rows ? M - m : rows) * per_row);
        const dim3     grid((units + kThreads - 1) / kThreads);
        const T       *from = x + m * ldx;
        uint8_t       *c = codes + m * code_stride, *s = scales + m * scale_stride;
        if (vec) {
            hipLaunchKernelGGL((rq_mx_quantize_kernel<DT, true, ACT>), grid, dim3(kThreads), 0, stream, from, ldx, units, d, K, c,
                               code_stride, s, scale_stride);
        } else {
            hipLaunchKernelGGL((rq_mx_quantize_kernel<DT, false, ACT>), grid, dim3(kThreads), 0, stream, from, ldx, units, d, K, c,
                               code_stride, s, scale_stride);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <int DT>
hipError_t panel_quantize(const void *x_, int64_t ldx, const WeightLayout &L, const int *row_of, const int *rows, uint8_t *panels,
                          int *zero, int zeros, hipStream_t stream) {
    using T = typename Element<DT>::type;
    const T   *x = reinterpret_cast<const T *>(x_);
    const bool vec = (uintptr_t) x % 16 == 0 && ldx * (int64_t) sizeof(T) % 16 == 0;
    const int64_t blocks = (L.N + 31) / 32;
    const dim3    grid((unsigned) (2 * L.chunks), (unsigned) (blocks < kPanelBlocks ? blocks : kPanelBlocks), (unsigned) ((blocks + kPanelBlocks - 1) / kPanelBlocks));
    if (vec) hipLaunchKernelGGL((rq_mx_panel_quantize_kernel<DT, true>), grid, dim3(kThreads), 0, stream, x, ldx, L, row_of, rows, panels, zero, zeros);
    else hipLaunchKernelGGL((rq_mx_panel_quantize_kernel<DT, false>), grid, dim3(kThreads), 0, stream, x, ldx, L, row_of, rows, panels, zero, zeros);
    return hipGetLastError();
}

template <int DT>
hipError_t dequantize(const uint8_t *codes, const uint8_t *scales, int64_t M, int64_t K, void *out_, int64_t ldo, hipStream_t stream) {
    using T = typename Element<DT>::type;
    T            *out = reinterpret_cast<T *>(out_);
    const bool    vec = (uintptr_t) out % 16 == 0 && (M == 1 || ldo * (int64_t) sizeof(T) % 16 == 0);
    const Divider d = make_divider((uint32_t) (K / 8));
    const int64_t rows = (1ll << 30) / (K / 8);
    for (int64_t m = 0; m < M; m += rows) {
        const uint32_t units = (uint32_t) ((M - m < rows ? M - m : rows) * (K / 8));
        const dim3     grid((units + kThreads - 1) / kThreads);
        const uint8_t *c = codes + m * (K / 2), *s = scales + m * (K / 32);
        if (vec) {
            hipLaunchKernelGGL((rq_mx_dequantize_kernel<DT, true>), grid, dim3(kThreads), 0, stream, c, s, units, d, K, out + m * ldo, ldo);
        } else {
            hipLaunchKernelGGL((rq_mx_dequantize_kernel<DT, false>), grid, dim3(kThreads), 0, stream, c, s, units, d, K, out + m * ldo, ldo);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

hipError_t launch_act_quantize(int dtype, const void *x, int64_t ldx, int64_t M, int64_t K, uint8_t *codes, uint8_t *scales,
                               hipStream_t stream) {
    const ActLayout A = act_layout(K);
    const int64_t   per_row = up_to(K, 512) / 8;   // (the scales' padding is the longer one)
    if (dtype == RQ_F32) return quantize<RQ_F32, true>(x, ldx, M, K, codes, scales, A.code_stride, A.scale_stride, per_row, stream);
    if (dtype == RQ_F16) return quantize<RQ_F16, true>(x, ldx, M, K, codes, scales, A.code_stride, A.scale_stride, per_row, stream);
    return quantize<RQ_BF16, true>(x, ldx, M, K, codes, scales, A.code_stride, A.scale_stride, per_row, stream);
}

hipError_t launch_panel_quantize(int dtype, const void *x, int64_t ldx, const WeightLayout &L, const int *row_of, const int *rows,
                                 uint8_t *panels, int *zero, int zeros, hipStream_t stream) {
    if (dtype == RQ_F32) return panel_quantize<RQ_F32>(x, ldx, L, row_of, rows, panels, zero, zeros, stream);
    if (dtype == RQ_F16) return panel_quantize<RQ_F16>(x, ldx, L, row_of, rows, panels, zero, zeros, stream);
    return panel_quantize<RQ_BF16>(x, ldx, L, row_of, rows, panels, zero, zeros, stream);
}

}  // namespace mx
}  // namespace rq

using namespace rq::mx;

namespace {
bool known_dtype(int dtype) { return dtype == RQ_F32 || dtype == RQ_F16 || dtype == RQ_BF16; }
bool element_aligned(const void *p, int dtype) { return (uintptr_t) p % (dtype == RQ_F32 ? 4 : 2) == 0; }
// rows of K elements whose blocks are counted in 64 bits, but a row's own units in 32
bool good_row(int64_t K) { return K > 0 && K % RQ_MX4_BLOCK == 0 && K <= (1ll << 30); }
}  // namespace

extern "C" int rq_mx4_quantize(int dtype, const void *x, int64_t ldx, int64_t M, int64_t K, void *codes, void *scales, rq_stream_t stream) {
    if (!known_dtype(dtype) || !good_row(K) || M < 0) return RQ_E_UNSUPPORTED;
    if (M == 0) return 0;
    if (!x || !element_aligned(x, dtype) || !codes || !scales || (uintptr_t) codes % 4 || (M > 1 && ldx < K)) return RQ_E_ARGUMENT;
    uint8_t *c = (uint8_t *) codes, *s = (uint8_t *) scales;
    const hipStream_t st = (hipStream_t) stream;
    if (dtype == RQ_F32) return quantize<RQ_F32, false>(x, ldx, M, K, c, s, K / 2, K / 32, K / 8, st);
    if (dtype == RQ_F16) return quantize<RQ_F16, false>(x, ldx, M, K, c, s, K / 2, K / 32, K / 8, st);
    return quantize<RQ_BF16, false>(x, ldx, M, K, c, s, K / 2, K / 32, K / 8, st);
}

extern "C" int rq_mx4_dequantize(int dtype, const void *codes, const void *scales, int64_t M, int64_t K, void *out, int64_t ldo,
                                 rq_stream_t stream) {
    if (!known_dtype(dtype) || !good_row(K) || M < 0) return RQ_E_UNSUPPORTED;
    if (M == 0) return 0;
    if (!out || !element_aligned(out, dtype) || !codes || !scales || (uintptr_t) codes % 4 || (M > 1 && ldo < K)) return RQ_E_ARGUMENT;
    const uint8_t *c = (const uint8_t *) codes, *s = (const uint8_t *) scales;
    const hipStream_t st = (hipStream_t) stream;
    if (dtype == RQ_F32) return dequantize<RQ_F32>(c, s, M, K, out, ldo, st);
    if (dtype == RQ_F16) return dequantize<RQ_F16>(c, s, M, K, out, ldo, st);
    return dequantize<RQ_BF16>(c, s, M, K, out, ldo, st);
}

extern "C" size_t rq_mx4_prepared_bytes(int64_t E, int64_t N, int64_t K) {
    if (E < 1 || E > (1 << 20) || N < 1 || N > (1 << 24) || K < RQ_MX4_BLOCK || K % RQ_MX4_BLOCK || K > RQ_MX4_MAX_K) return 0;
    return (size_t) (E * weight_layout(N, K).expert_bytes);
}

extern "C" int rq_mx4_prepare(const void *codes, const void *scales, int64_t E, int64_t N, int64_t K, void *prepared,
                              size_t prepared_bytes, rq_stream_t stream) {
    const size_t need = rq_mx4_prepared_bytes(E, N, K);
    if (need == 0) return RQ_E_UNSUPPORTED;
    if (!codes || !scales || !prepared || (uintptr_t) codes % 256 || (uintptr_t) scales % 256) return RQ_E_ARGUMENT;
    if (prepared_bytes < need || (uintptr_t) prepared % 256) return RQ_E_WORKSPACE;
    const WeightLayout L = weight_layout(N, K);
    const int64_t      threads = L.expert_bytes / 16;
    const int64_t      x = (threads + kThreads - 1) / kThreads;
    const int64_t      y = E < 32768 ? E : 32768;
    const dim3         grid((unsigned) (x < 4096 ? x : 4096), (unsigned) y, (unsigned) ((E + y - 1) / y));
    hipLaunchKernelGGL(rq_mx_prepare_kernel, grid, dim3(kThreads), 0, (hipStream_t) stream, (const uint8_t *) codes,
                       (const uint8_t *) scales, L, E, (uint8_t *) prepared);
    return hipGetLastError();
}
