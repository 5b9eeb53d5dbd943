// Products of few rows a group (int8, or grouped by expert): weights from memory into registers.
//
// A call of this size is the stream of its weights. A workgroup has 32 rows of one weight and up to 16 rows of x at a time; its wavefronts
// split the row's bytes, each with DEPTH steps of 64 bytes on their way, and join their sums in LDS in their order. Rows of x that are still to be
// rounded are rounded by every workgroup for itself, into LDS, while its first weights are on their way: that saves a launch, where the rows are few.
//
// Bound by memory where weights are large, by the chain of a load, the products and the join where they are not. The kernel's own time, two weights in turn: one token x 5120 x 17408
// in int8 17.2 us, 89 MB at 5.1 TB/s, a large copy's rate (21.4 a call in a graph of calls, the next one's start among them); 13 x 4099 x 5121 10.3 us; 37 tokens' 111 rows of
// 1376 x 4096 in fp16, from 40 to 49 of 60 experts, 452 to 554 MB, 91 us. A group's rows go 16 at a time, one pass over its weight each: 512 rows x 5120 x 1280 in int8 184 us
// where one of 128 experts has them all, 159 where all have four. Tried:
// 16 wavefronts (2.4 times as long), 16 rows (more steps on their way, 10 to 60 % longer), 64 rows (as fast for groups, 10 to 25 % longer for one).
#include "rq_prod.h"

namespace rq {
namespace prod {
namespace {

__device__ __attribute__((aligned(16))) const uint8_t kZeros[16] = { 0 };

// LDS that every launch may have, and what of it a workgroup takes beside its rows.
constexpr int kMostLds = 65536, kFixedLds = 128;

// Eight elements of a row from k on, zeros behind its end.
template <int DT>
__device__ __forceinline__ void load_unit(const typename Element<DT>::type *x, bool aligned, int K, int k, float (&v)[8]) {
    using T = typename Element<DT>::type;
    uint32_t w[DT == RQ_F32 ? 8 : 4];
    if (k + 8 > K) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = k + i < K ? to_float(x[k + i]) : 0.0f;
        return;
    }
    if (aligned) {   // (on 16 bytes)
#pragma unroll
        for (int i = 0; i < (DT == RQ_F32 ? 2 : 1); ++i) {
            const uint4 u = reinterpret_cast<const uint4 *>(x + k)[i];
            w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
        }
    } else {
        load_bytes(w, x + k);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (DT == RQ_F32) v[i] = __uint_as_float(w[i]);
        else v[i] = to_float(__builtin_bit_cast(T, (uint16_t) (i & 1 ? w[i >> 1] >> 16 : w[i >> 1])));
    }
}

// WT: the weight's type; DT: RQ_F32, RQ_F16, RQ_BF16: rows of x of that type, to be rounded to int8; RQ_I8: rows as the products take them. W wavefronts; NR
// runs of 16 rows of the weight; GROUPED: blockIdx.y is a group that has rows.
template <int WT, int DT, int W, int NR, int DEPTH, bool GROUPED>
__global__ __launch_bounds__(64 * W) void rq_stream_kernel(const ProductArgs a) {
    using Acc4 = typename Matrix<WT>::Acc4;
    constexpr bool kRound = DT != RQ_I8;
    constexpr int  kKept = 3, kThreads = 64 * W;   // units of a row that a thread keeps while its maximum is found
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ uint32_t tops[2][W];
    __shared__ float    scale_of[16];
    static_assert(sizeof(tops) + sizeof(scale_of) <= kFixedLds, "LDS beside the rows");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quarter = lane >> 4;
    int       e = 0, first = 0, count = (int) a.P;
    if constexpr (GROUPED) {
        int place;
        if (!find_group<false>(a, [](int n) { return n > 0 ? 1 : 0; }, [](int) { return (int) blockIdx.y; }, e, first, count, place)) return;
    }
    const int      unit0 = blockIdx.x * NR, steps = a.L.steps;
    const int      s0 = steps * wave / W, s1 = steps * (wave + 1) / W;
    const uint8_t *weight = a.w + (int64_t) e * a.L.expert_bytes;
    // rows col of run unit0 + r, bytes 16 quarter .. of a step (a run past the weight's last repeats it: it is computed and not stored)
    const uint8_t *from[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        const int unit = min(unit0 + r, 2 * a.L.row_blocks - 1);
        from[r] = weight + (int64_t) (unit >> 1) * steps * 2048 + (unit & 1) * 256 + (quarter >> 1) * 1024 + (quarter & 1) * 512 + col * 16;
    }
    const float *t_scales = reinterpret_cast<const float *>(weight + a.L.code_bytes);
    const int    pitch = steps * 64 + 16;   // (of rows in LDS: the same bytes of 16 rows in 16 places of the banks)
    for (int t0 = 0; t0 < count; t0 += a.chunk) {
        const int T = min(a.chunk, count - t0);
        v4i       A[DEPTH][NR], B[kRound ? 1 : DEPTH];
        Acc4      acc[NR];
        const uint8_t *x = lds + min(col, T - 1) * pitch + quarter * 16;   // (columns past the rows repeat the last one)
        uint32_t       tail[4] = { 0, 0, 0, 0 };   // the row's bytes behind its last 16th, zeros behind them
        if constexpr (!kRound) {
            const int64_t row = row_read(a, first + t0 + min(col, T - 1));
            x = a.x + (row < 0 ? 0 : row) * a.pitch;
            if (a.x_bytes & 15)
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (j < (a.x_bytes & 15)) tail[j >> 2] |= (uint32_t) x[(a.x_bytes & ~15ll) + j] << (8 * (j & 3));
        }
        auto load = [&](int i, int s) __attribute__((always_inline)) {
#pragma unroll
            for (int r = 0; r < NR; ++r) A[i][r] = *reinterpret_cast<const v4i *>(from[r] + (int64_t) s * 2048);
            if constexpr (!kRound) {   // (a row's last bytes end anywhere, and behind them is another's memory)
                uint32_t w[4];
                load_bytes(w, a.x_bytes < 16 ? kZeros : x + min(s * 64 + quarter * 16, (int) a.x_bytes - 16));
                B[i] = v4i{ (int) w[0], (int) w[1], (int) w[2], (int) w[3] };
            }
        };
        // what was loaded, or the row's last bytes and zeros (looked at where it is used: a load that is looked at is waited for)
        auto whole = [&](const v4i &v, int s) __attribute__((always_inline)) {
            const int at = s * 64 + quarter * 16;
            v4i       r;
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = at + 16 <= a.x_bytes ? v[j] : at < a.x_bytes ? (int) tail[j] : 0;
            return r;
        };
        if constexpr (kRound) {
            using X = typename Element<DT>::type;
            const int K = (int) a.K, units = steps * 8;
            float     v[kKept][8];
            auto      row_at = [&](int t) __attribute__((always_inline)) { return row_read(a, first + t0 + t); };
            auto      begin = [&](int64_t row) __attribute__((always_inline)) {
                const X *p = reinterpret_cast<const X *>(a.x) + (row < 0 ? 0 : row) * a.pitch;
#pragma unroll
                for (int i = 0; i < kKept; ++i) {
                    const int k = ((int) threadIdx.x + i * kThreads) * 8;
                    if (k < K) load_unit<DT>(p, a.aligned, K, k, v[i]);
                }
                return p;
            };
            int64_t  row = row_at(0);
            const X *p = begin(row);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < DEPTH; ++i)
                if (s0 + i < s1) load(i, s0 + i);
            __builtin_amdgcn_sched_barrier(0);
            if (t0) __syncthreads();   // (the sums of the rows before, in the rows' place, are not read any more)
            for (int t = 0; t < T; ++t) {
                if (t) row = row_at(t), p = begin(row);
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < kKept; ++i) {
                    const int k = ((int) threadIdx.x + i * kThreads) * 8;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (k < K) top = max(top, __float_as_uint(v[i][j]) & 0x7FFFFFFFu);
                }
                for (int u = threadIdx.x + kKept * kThreads; u * 8 < K; u += kThreads) {
                    float w[8];
                    load_unit<DT>(p, a.aligned, K, u * 8, w);
#pragma unroll
                    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(w[j]) & 0x7FFFFFFFu);
                }
                top = wave_max(top);
                if (lane == 0) tops[t & 1][wave] = top;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < W; ++i) top = max(top, tops[t & 1][i]);
                const RowScale q(top);
                if (threadIdx.x == 0) scale_of[t] = row < 0 ? 0.0f : q.s;
                const uint32_t keep = row < 0 ? 0u : q.keep;
                uint8_t       *to = lds + t * pitch;
#pragma unroll
                for (int i = 0; i < kKept; ++i) {
                    const int u = threadIdx.x + i * kThreads;
                    if (u * 8 < K) *reinterpret_cast<uint2 *>(to + u * 8) = codes_of(v[i], q.r, keep);
                }
                for (int u = threadIdx.x + kKept * kThreads; u < units; u += kThreads) {
                    float w[8] = { 0, 0, 0, 0, 0, 0, 0, 0 };
                    if (u * 8 < K) load_unit<DT>(p, a.aligned, K, u * 8, w);
                    *reinterpret_cast<uint2 *>(to + u * 8) = codes_of(w, q.r, keep);
                }
#pragma unroll
                for (int i = 0; i < kKept; ++i) {   // (the places behind the row)
                    const int u = threadIdx.x + i * kThreads;
                    if (u * 8 >= K && u < units) *reinterpret_cast<uint2 *>(to + u * 8) = make_uint2(0, 0);
                }
            }
            __syncthreads();
        } else {
#pragma unroll
            for (int i = 0; i < DEPTH; ++i)
                if (s0 + i < s1) load(i, s0 + i);
        }
#pragma unroll
        for (int r = 0; r < NR; ++r) acc[r] = Acc4{ 0, 0, 0, 0 };
        for (int s = s0; s < s1; s += DEPTH) {
#pragma unroll
            for (int i = 0; i < DEPTH; ++i) {
                if (s + i < s1) {
                    const v4i b = kRound ? *reinterpret_cast<const v4i *>(x + (s + i) * 64) : whole(B[kRound ? 0 : i], s + i);
#pragma unroll
                    for (int r = 0; r < NR; ++r) acc[r] = Matrix<WT>::mfma16(A[i][r], b, acc[r]);
                    if (s + i + DEPTH < s1) load(i, s + i + DEPTH);
                }
            }
        }
        // [wavefront][run of rows][row of x][block of four rows], in the place of the rows
        Acc4 *part = reinterpret_cast<Acc4 *>(lds);
        if (kRound || t0) __syncthreads();   // (neither they nor the sums before are read any more)
#pragma unroll
        for (int r = 0; r < NR; ++r)
            if (col < T) part[((wave * NR + r) * T + col) * 4 + quarter] = acc[r];
        __syncthreads();
        const int cells = NR * T * 4;
        for (int c = threadIdx.x; c < cells; c += kThreads) {
            const int r = c / (T * 4), t = (c >> 2) % T, block = c & 3;
            Acc4      sum = part[c];
#pragma unroll
            for (int w = 1; w < W; ++w) sum += part[w * cells + c];
            const int64_t place = first + t0 + t, n = (int64_t) (unit0 + r) * 16 + block * 4, out = row_written(a, place), in = row_read(a, place);
            if (out < 0 || n >= a.L.N) continue;
            v4f v;
            if constexpr (WT == RQ_I8) {
                const v4f   tn = *reinterpret_cast<const v4f *>(t_scales + n);
                const float sm = kRound ? scale_of[t] : in < 0 ? 0.0f : a.x_scales[in];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = (float) sum[i] * tn[i] * sm;
            } else {
                v = sum;
            }
            if (in < 0) v = v4f{ 0, 0, 0, 0 };
            store_out(a.out_dtype, a.y, out * a.ldy, n, a.L.N, v);
        }
    }
}

int lds_bytes(int W, int NR, bool round, const ProductArgs &a) {
    const int T = (int) (a.P < a.chunk ? a.P : a.chunk), sums = W * NR * T * 64, rows = round ? T * (a.L.steps * 64 + 16) : 0;
    return sums > rows ? sums : rows;
}

template <int WT, int DT, bool GROUPED>
hipError_t stream(const ProductArgs &a, hipStream_t s) {
    const int64_t  units = (a.L.N + 15) / 16;
    const unsigned groups = GROUPED ? (unsigned) (a.P < a.E ? a.P : a.E) : 1;
    constexpr bool kRound = DT != RQ_I8;
    // Eight wavefronts a workgroup up to one workgroup a compute unit, four beyond. (us, eight -> four: one row of int8, K = 5120: N = 6592 9.9 -> 10.6, 8192 11.4 -> 11.6,
    // 12000 18.7 -> 15.9, 17408 22.8 -> 20.3; 6, 8 and 10 groups of one row, N = 1280 10.2 -> 10.8, 15.8 -> 12.6, 16.6 -> 16.6; bf16, 8 groups 22.6 -> 19.6)
    if (units * groups > 512) {
        hipLaunchKernelGGL((rq_stream_kernel<WT, DT, 4, 2, 4, GROUPED>), dim3((unsigned) ((units + 1) / 2), groups), dim3(256), lds_bytes(4, 2, kRound, a), s, a);
    } else {
        hipLaunchKernelGGL((rq_stream_kernel<WT, DT, 8, 2, 6, GROUPED>), dim3((unsigned) ((units + 1) / 2), groups), dim3(512), lds_bytes(8, 2, kRound, a), s, a);
    }
    return hipGetLastError();
}
template <bool GROUPED>
hipError_t stream(int weight_type, int x_type, const ProductArgs &a, hipStream_t s) {
    if constexpr (GROUPED) {
        if (weight_type == RQ_F16) return stream<RQ_F16, RQ_I8, GROUPED>(a, s);
        if (weight_type == RQ_BF16) return stream<RQ_BF16, RQ_I8, GROUPED>(a, s);
    } else if (weight_type != RQ_I8) {
        return hipErrorInvalidValue;
    }
    if (x_type == RQ_F32) return stream<RQ_I8, RQ_F32, GROUPED>(a, s);
    if (x_type == RQ_F16) return stream<RQ_I8, RQ_F16, GROUPED>(a, s);
    if (x_type == RQ_BF16) return stream<RQ_I8, RQ_BF16, GROUPED>(a, s);
    return stream<RQ_I8, RQ_I8, GROUPED>(a, s);
}

}  // namespace

int stream_rounds(int64_t P, int64_t K, int64_t N, int64_t E) {
    // (us a call in graphs of calls, weights from memory, rounded by every workgroup -> by a launch in front: K = 5120: N = 17408 1 row 21.4 -> 24.1, 2 rows 22.6 to 25.3 -> 25.1,
    // 4 28.3 -> 25.2; N = 5120 1 8.2 -> 10.4, 2 9.3 -> 10.6, 4 11.3 -> 10.7; N = 1024 1 6.7 -> 8.7, 2 7.7 -> 9.1, 4 9.7 -> 9.3; N = 30000 1 31.2 -> 33.6, 2 37.2 -> 32.4; N = 60000 1
    // 62.8 -> 58.2; K = 17408, N = 5120 1 23.5 -> 24.6; groups of 1 row, K = 5120, N = 1280: 8 13.1 -> 15.8, 16 22.6 -> 23.0; K = 1280, N = 5120 16 23.0 -> 22.6; that it stops at
    // eight rows costs some of those behind: 12 groups 16.7 -> 19.1, 16 of K = 2048, N = 512 6.8 -> 9.2)
    const int64_t most = (kMostLds - kFixedLds) / (up_to(K, 64) + 16), T = most < 16 ? most : 16;
    if (T == 0 || P > (E ? 8 : 2)) return 0;
    return P * K * ((N + 31) / 32) <= 6000000 ? (int) (T < P ? T : P) : 0;
}

hipError_t launch_stream(int weight_type, int x_type, const ProductArgs &a, hipStream_t s) {
    return a.offsets ? stream<true>(weight_type, x_type, a, s) : stream<false>(weight_type, x_type, a, s);
}

}  // namespace prod
}  // namespace rq
