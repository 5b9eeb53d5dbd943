// MXFP4 products for up to 16 tokens, and the experts of few tokens: few launches, and weights from memory into registers.
//
// A call of this size is the stream of its weights and what stands in front of it and behind it, so a product is one launch: a
// workgroup fetches the tokens first and its first weights behind them, quantises the tokens into LDS while the weights are on
// their way, and its wavefronts split the inputs. (From some size on a launch in front quantises them: decode_takes.) The experts are two
// launches, too: gate and up of every slot, then the down projections of a token's slots with their weighted sum. 16x16x128 MFMAs: workgroups of 16 rows spread a small weight over
// twice as many compute units as the 32 rows of the other form would.
//
// Bound by the weights' stream where they are large, by the chain of a load, the rounding, the products and the join of the inputs' parts
// where they are not: one token x 5120: 5120 outputs (14 MB) 6.3 us, 17408 outputs (47 MB) 11.5 us, 4.1 TB/s; three tokens x 17408 x 5120
// 12.9 us behind a launch of 2.8 that rounds them. One token's 8 experts of 1280 x 5120: 14.0 + 9.5 us, 56 and 28 MB, 4.0 and 2.9 TB/s;
// with 8 of 64, 2, 3 and 4 tokens 38, 49 and 62 us.
#include "rq_mx.h"

namespace rq {
namespace mx {
namespace {

constexpr int kWaves = 8;   // of the experts' kernels
constexpr int kDecodeUnits = 512;   // most runs of 16 rows that are a workgroup each

// This lane's part of a 16-row fragment of a step: row lane % 16, block lane / 16 of the step's four.
struct Lane {
    int  lane, row, block;
    uint32_t code_off, scale_off, shift;   // in a step of a row block, in its word of scales, in that word
    __device__ __forceinline__ Lane() {
        lane = threadIdx.x & 63;
        row = lane & 15;
        block = lane >> 4;
        code_off = (block >> 1) * 1024 + (block & 1) * 512 + row * 16;
        scale_off = ((block & 1) * 32 + row) * 4;
        shift = (block >> 1) * 8;
    }
};
__device__ __forceinline__ v4f mfma16(const v4i &a, const v4i &b, const v4f &c, int sa, int sb) {
    const v8i A = { a[0], a[1], a[2], a[3], 0, 0, 0, 0 };
    const v8i B = { b[0], b[1], b[2], b[3], 0, 0, 0, 0 };
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, c, 4, 4, 0, sa, 0, sb);
}

// 16 rows of a weight
struct Rows {
    const uint8_t *codes, *scales;
    __device__ __forceinline__ Rows() {}
    __device__ __forceinline__ Rows(const uint8_t *weight, const WeightLayout &L, int unit, const Lane &l) {
        codes = weight + (int64_t) (unit >> 1) * L.steps * 2048 + (unit & 1) * 256 + l.code_off;
        scales = weight + L.code_bytes + (int64_t) (unit >> 1) * L.chunks * 512 + (unit & 1) * 64 + l.scale_off;
    }
    __device__ __forceinline__ v4i code(int s) const { return *reinterpret_cast<const v4i *>(codes + (int64_t) s * 2048); }
    __device__ __forceinline__ int scale(int s) const { return *reinterpret_cast<const int *>(scales + (int64_t) (s >> 1) * 256); }
};

// Tokens in LDS: codes of up to 128-padded rows, then their scales in the order of the blocks.
struct Tokens {
    uint8_t *codes, *scales;
    int      code_stride, scale_stride;
    __device__ __forceinline__ Tokens(uint8_t *lds, int T, int steps) {
        code_stride = steps * 64;
        scale_stride = steps * 4;
        codes = lds;
        scales = lds + T * code_stride;
    }
};

// Eight elements of a token from 8 u on (zeros past its end)
template <int DT>
__device__ __forceinline__ void load_unit(const typename Element<DT>::type *x, bool aligned, int K, int u, Unit<DT> &v) {
    v.clear();
    if (u * 8 >= K) return;
    if (aligned) v.template load<true>(x + u * 8);
    else v.template load<false>(x + u * 8);
}
// ... rounded by the four lanes that hold their block
template <int DT>
__device__ __forceinline__ void store_unit(uint8_t *codes, uint8_t *scales, int u, const Unit<DT> &v) {
    const int X = block_scale(max_of_four(v.top()));
    *reinterpret_cast<uint32_t *>(codes + u * 4) = v.pack(X);
    if ((u & 3) == 0) scales[u >> 2] = (uint8_t) X;
}

// MAT weights of NR runs of 16 rows against T tokens: this wavefront's share of the inputs. DEPTH steps of the weights are on their
// way while the tokens are quantised. ROWS: the tokens are in memory in row form instead (up to 16).
template <int DT, bool ROWS, int W, int MAT, int NR, int DEPTH>
__device__ __forceinline__ void stream(const Rows (&rows)[MAT][NR], const Lane &l, const DecodeArgs &a, const typename Element<DT>::type *x, int T,
                                       uint8_t *lds, v4f (&acc)[MAT][NR]) {
    constexpr int kThreads = 64 * W;
    const int    K = (int) a.L.K, steps = (K + 127) / 128, units = steps * 16;
    const Tokens tokens(lds, T, steps);
    const int    wave = threadIdx.x >> 6, u0 = threadIdx.x;
    const int    s0 = steps * wave / W, s1 = steps * (wave + 1) / W;
    Unit<DT> v[2];
    if constexpr (!ROWS) {   // (the first two units of the first token: all there is of a short one)
        if (u0 < units) load_unit<DT>(x, a.aligned, K, u0, v[0]);
        if (u0 + kThreads < units) load_unit<DT>(x, a.aligned, K, u0 + kThreads, v[1]);
        __builtin_amdgcn_sched_barrier(0);
    }
    const int      t = min(l.row, T - 1);   // (columns past the tokens repeat the last one)
    const uint8_t *b, *bs;
    if constexpr (ROWS) {
        b = a.a_codes + t * a.A.code_stride + l.block * 16;
        bs = a.a_scales + t * a.A.scale_stride + (l.block & 1) * 4 + (l.block >> 1);
    } else {
        b = tokens.codes + t * tokens.code_stride + l.block * 16;
        bs = tokens.scales + t * tokens.scale_stride + l.block;
    }
    v4i A[DEPTH][MAT][NR], B[ROWS ? DEPTH : 1];
    int S[DEPTH][MAT][NR], sb[ROWS ? DEPTH : 1];
    auto load = [&](int i, int s) __attribute__((always_inline)) {
#pragma unroll
        for (int m = 0; m < MAT; ++m)
#pragma unroll
            for (int r = 0; r < NR; ++r) A[i][m][r] = rows[m][r].code(s), S[i][m][r] = rows[m][r].scale(s);
        if constexpr (ROWS) B[i] = *reinterpret_cast<const v4i *>(b + s * 64), sb[i] = bs[(s >> 1) * 8 + (s & 1) * 2];
    };
#pragma unroll
    for (int i = 0; i < DEPTH; ++i)
        if (s0 + i < s1) load(i, s0 + i);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (!ROWS) {
        if (u0 < units) store_unit(tokens.codes, tokens.scales, u0, v[0]);
        if (u0 + kThreads < units) store_unit(tokens.codes, tokens.scales, u0 + kThreads, v[1]);
        for (int k = 0; k < T; ++k) {
            uint8_t *codes = tokens.codes + k * tokens.code_stride, *scales = tokens.scales + k * tokens.scale_stride;
            for (int u = k == 0 ? u0 + 2 * kThreads : u0; u < units; u += 2 * kThreads) {
                const bool more = u + kThreads < units;
                load_unit<DT>(x + k * a.ldx, a.aligned, K, u, v[0]);
                if (more) load_unit<DT>(x + k * a.ldx, a.aligned, K, u + kThreads, v[1]);
                store_unit(codes, scales, u, v[0]);
                if (more) store_unit(codes, scales, u + kThreads, v[1]);
            }
        }
        __syncthreads();
    }
    for (int s = s0; s < s1; s += DEPTH) {
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) {
            if (s + i < s1) {
                const v4i tb = ROWS ? B[ROWS ? i : 0] : *reinterpret_cast<const v4i *>(b + (s + i) * 64);
                const int ts = ROWS ? sb[ROWS ? i : 0] : bs[(s + i) * 4];
                const int shift = ((s + i) & 1) * 16 + l.shift;
#pragma unroll
                for (int m = 0; m < MAT; ++m)
#pragma unroll
                    for (int r = 0; r < NR; ++r) acc[m][r] = mfma16(A[i][m][r], tb, acc[m][r], S[i][m][r] >> shift, ts);
                if (s + i + DEPTH < s1) load(i, s + i + DEPTH);
            }
        }
    }
}

// The wavefronts' sums in their order. part: [wave][cell][token][block of four rows], four floats; cells of the tokens only.
template <int CELLS>
__device__ __forceinline__ void put_part(v4f *part, const v4f (&acc)[CELLS], const Lane &l, int T, int wave) {
    if (l.row < T) {
#pragma unroll
        for (int c = 0; c < CELLS; ++c) part[((wave * CELLS + c) * T + l.row) * 4 + l.block] = acc[c];
    }
}

template <int DT, bool ROWS, int W, int NR>
__global__ __launch_bounds__(64 * W, 4) void rq_mx_decode_kernel(const DecodeArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const Lane l;
    const int  wave = threadIdx.x >> 6, unit0 = blockIdx.x * NR;
    Rows       rows[1][NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) rows[0][r] = Rows(a.w, a.L, unit0 + r, l);
    v4f acc[1][NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) acc[0][r] = v4f{ 0, 0, 0, 0 };
    const int T = (int) a.M;
    stream<DT, ROWS, W, 1, NR, 8 / NR>(rows, l, a, reinterpret_cast<const typename Element<DT>::type *>(a.x), T, lds, acc);
    __syncthreads();   // (the tokens are not read any more)
    v4f *part = reinterpret_cast<v4f *>(lds);
    put_part<NR>(part, acc[0], l, T, wave);
    __syncthreads();
    const int cells = NR * T * 4;
    for (int c = threadIdx.x; c < cells; c += 64 * W) {
        v4f sum = part[c];
#pragma unroll
        for (int w = 1; w < W; ++w) sum += part[w * cells + c];
        const int t = (c >> 2) % T, r = (c >> 2) / T;
        store_out(a.out_dtype, a.y, t * a.ldy, (int64_t) (unit0 + r) * 16 + (c & 3) * 4, a.L.N, sum);
    }
}

// One block of 32 rows of h of the slot blockIdx.y: gate and up, silu(gate) * up, quantised.
template <int DT>
__global__ __launch_bounds__(64 * kWaves, 4) void rq_mx_decode_gate_up_kernel(const DecodeArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int slot = blockIdx.y, e = a.ids[slot];
    if (e < 0 || e >= a.E) return;
    const Lane l;
    const int  wave = threadIdx.x >> 6, unit0 = blockIdx.x * 2;
    Rows       rows[2][2];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r) rows[m][r] = Rows((m ? a.w2 : a.w) + (int64_t) e * a.L.expert_bytes, a.L, unit0 + r, l);
    v4f acc[2][2];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r) acc[m][r] = v4f{ 0, 0, 0, 0 };
    const typename Element<DT>::type *x = reinterpret_cast<const typename Element<DT>::type *>(a.x) + (int64_t) (slot / a.top) * a.ldx;
    stream<DT, false, kWaves, 2, 2, 3>(rows, l, a, x, 1, lds, acc);
    __syncthreads();
    v4f      *part = reinterpret_cast<v4f *>(lds);
    const v4f all[4] = { acc[0][0], acc[0][1], acc[1][0], acc[1][1] };
    put_part<4>(part, all, l, 1, wave);
    __syncthreads();
    if (threadIdx.x < 16) {
        v4f sum = part[threadIdx.x];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) sum += part[w * 16 + threadIdx.x];
        part[threadIdx.x] = sum;   // (cell 0 .. 7: 32 rows of the gate, 8 .. 15: of the up projection)
    }
    __syncthreads();
    if (threadIdx.x < 4) {
        const float *g = reinterpret_cast<const float *>(part) + threadIdx.x * 8, *u = g + 32;
        float        h[8];
        uint32_t     top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            h[i] = g[i] / (1.0f + expf(-g[i])) * u[i];
            top = max(top, __float_as_uint(h[i]) & 0x7FFFFFFFu);
        }
        top = max_of_four(top);
        const int X = block_scale(top), b = blockIdx.x, blocks = gridDim.x;
        reinterpret_cast<uint32_t *>(a.h_codes + (int64_t) slot * a.h_stride + b * 16)[threadIdx.x] = pack8(h, X);
        if (threadIdx.x == 0) {
            uint8_t *s = a.h_scales + (int64_t) slot * (a.h_stride >> 4);
            s[b] = (uint8_t) X;
            if (b == blocks - 1)   // (the last step's other blocks: multiplied by zero codes, where a NaN would show)
                for (int k = blocks; k & 3; ++k) s[k] = 0;
        }
    }
}

// 16 rows of the output of token blockIdx.y: the wavefronts share out its slots, or parts of their inputs where there are fewer slots
// than wavefronts, weigh their sums, and join them in the order of the wavefronts.
template <int DT>
__global__ __launch_bounds__(64 * kWaves, 4) void rq_mx_decode_down_kernel(const DecodeArgs a) {
    constexpr int kDepth = 5;   // (8: its registers leave one workgroup per compute unit)
    const Lane l;
    const int  wave = threadIdx.x >> 6, unit = blockIdx.x, m = blockIdx.y;
    const int  split = a.top >= kWaves ? 1 : kWaves / a.top, shares = a.top * split;
    const int  steps = (int) ((a.L.K + 127) / 128);
    v4f        total = { 0, 0, 0, 0 };
    for (int i = wave; i < shares; i += kWaves) {
        const int j = i / split, p = i - j * split, slot = m * a.top + j, e = a.ids[slot];
        if (e < 0 || e >= a.E) continue;
        const float    weight = a.weights[slot];
        const int      s0 = steps * p / split, s1 = steps * (p + 1) / split;
        const Rows     rows(a.w + (int64_t) e * a.L.expert_bytes, a.L, unit, l);
        const uint8_t *b = a.h_codes + (int64_t) slot * a.h_stride + l.block * 16;
        const uint8_t *bs = a.h_scales + (int64_t) slot * (a.h_stride >> 4) + l.block;
        v4i A[kDepth], B[kDepth];
        int S[kDepth], sb[kDepth];
        auto load = [&](int k, int s) __attribute__((always_inline)) {
            A[k] = rows.code(s), S[k] = rows.scale(s);
            B[k] = *reinterpret_cast<const v4i *>(b + s * 64), sb[k] = bs[s * 4];
        };
#pragma unroll
        for (int k = 0; k < kDepth; ++k)
            if (s0 + k < s1) load(k, s0 + k);
        v4f acc = { 0, 0, 0, 0 };
        for (int s = s0; s < s1; s += kDepth) {
#pragma unroll
            for (int k = 0; k < kDepth; ++k) {
                if (s + k < s1) {
                    acc = mfma16(A[k], B[k], acc, S[k] >> (((s + k) & 1) * 16 + l.shift), sb[k]);
                    if (s + k + kDepth < s1) load(k, s + k + kDepth);
                }
            }
        }
        total += weight * acc;
    }
    __shared__ v4f part[kWaves][4];
    if (l.row == 0) part[wave][l.block] = total;
    __syncthreads();
    if (threadIdx.x < 4) {
        v4f sum = part[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) sum += part[w][threadIdx.x];
        store_out(DT, a.y, m * a.ldy, (int64_t) unit * 16 + threadIdx.x * 4, a.L.N, sum);
    }
}

// LDS of the tokens, or of the partial sums behind them
int lds_bytes(int64_t T, int64_t K, int cells, int waves) {
    const int64_t tokens = T * ((K + 127) / 128) * 68, sums = (int64_t) waves * cells * T * 64;
    return (int) (tokens > sums ? tokens : sums);
}

template <int DT, bool ROWS>
hipError_t decode(const DecodeArgs &a, hipStream_t stream) {
    // 32 rows and four wavefronts a workgroup where that is enough of them for the chip, 16 and eight where it is not (K = 5120, N = 5120,
    // one token: 5.8 us with four, 5.1 with eight, 7.4 with sixteen; N = 17408 the same with four and eight)
    const int units = (int) ((a.L.N + 15) / 16);
    const int64_t K = ROWS ? 0 : a.L.K;
    if (units > kDecodeUnits) {
        hipLaunchKernelGGL((rq_mx_decode_kernel<DT, ROWS, 4, 2>), dim3((units + 1) / 2), dim3(256), lds_bytes(a.M, K, 2, 4), stream, a);
    } else {
        hipLaunchKernelGGL((rq_mx_decode_kernel<DT, ROWS, 8, 1>), dim3(units), dim3(512), lds_bytes(a.M, K, 1, 8), stream, a);
    }
    return hipGetLastError();
}

}  // namespace

bool decode_takes(int64_t M, int64_t K, int64_t N) {
    if (M > 4 || M * K > 65536) return false;
    // Every workgroup reads and rounds all of the tokens, against a launch of 2 us that does it once. (us, by every workgroup -> once:
    // N = 5120: K = 5120 2 tokens 5.9 -> 7.3, 4 tokens 7.7 -> 7.6, K = 17408 1 token 13.3 -> 14.5; N = 17408, K = 5120: 2 tokens
    // 12.6 -> 12.8, 4 tokens 15.9 -> 13.2)
    const int64_t units = (N + 15) / 16, workgroups = units > kDecodeUnits ? (units + 1) / 2 : units;
    return M * K * workgroups <= 6000000;
}

hipError_t launch_decode(int dtype, const DecodeArgs &a, hipStream_t stream) {
    if (a.a_codes) return decode<RQ_F32, true>(a, stream);
    return dtype == RQ_F32 ? decode<RQ_F32, false>(a, stream) : dtype == RQ_F16 ? decode<RQ_F16, false>(a, stream) : decode<RQ_BF16, false>(a, stream);
}

hipError_t launch_decode_experts(int dtype, const DecodeArgs &gate_up, const DecodeArgs &down, hipStream_t stream) {
    const dim3 grid(gate_up.L.row_blocks, (unsigned) (gate_up.M * gate_up.top));
    const int  bytes = lds_bytes(1, gate_up.L.K, 4, kWaves);
    if (dtype == RQ_F32) hipLaunchKernelGGL((rq_mx_decode_gate_up_kernel<RQ_F32>), grid, dim3(64 * kWaves), bytes, stream, gate_up);
    else if (dtype == RQ_F16) hipLaunchKernelGGL((rq_mx_decode_gate_up_kernel<RQ_F16>), grid, dim3(64 * kWaves), bytes, stream, gate_up);
    else hipLaunchKernelGGL((rq_mx_decode_gate_up_kernel<RQ_BF16>), grid, dim3(64 * kWaves), bytes, stream, gate_up);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const dim3 out((unsigned) ((down.L.N + 15) / 16), (unsigned) down.M);
    if (down.out_dtype == RQ_F32) hipLaunchKernelGGL((rq_mx_decode_down_kernel<RQ_F32>), out, dim3(64 * kWaves), 0, stream, down);
    else if (down.out_dtype == RQ_F16) hipLaunchKernelGGL((rq_mx_decode_down_kernel<RQ_F16>), out, dim3(64 * kWaves), 0, stream, down);
    else hipLaunchKernelGGL((rq_mx_decode_down_kernel<RQ_BF16>), out, dim3(64 * kWaves), 0, stream, down);
    return hipGetLastError();
}

}  // namespace mx
}  // namespace rq
