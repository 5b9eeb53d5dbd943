// Products of few rows a group (int8, or grouped by expert): weights from memory into registers.
//
// A call of this size is the stream of its weights. A workgroup has 32 rows of one weight (or 16, where those are too few for the chip) and
// up to 16 rows of x at a time; its wavefronts split the row's bytes, each with DEPTH steps of 64 bytes on their way, and join their sums in LDS in
// their order.
#include "rq_prod.h"

namespace rq {
namespace prod {
namespace {

__device__ __attribute__((aligned(16))) const uint8_t kZeros[16] = { 0 };

// WT: the weight's type; W wavefronts; NR runs of 16 rows of the weight; GROUPED: blockIdx.y is a group that has rows.
template <int WT, int W, int NR, int DEPTH, bool GROUPED>
__global__ __launch_bounds__(64 * W) void rq_stream_kernel(const ProductArgs a) {
    using Acc4 = typename Matrix<WT>::Acc4;
    __shared__ Acc4 part[W][NR][16][4];   // [wavefront][run of rows][row of x][block of four rows]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quarter = lane >> 4;
    int       e = 0, first = 0, count = (int) a.P;
    if constexpr (GROUPED) {
        int place, total;
        if (!find_group(a, (int) blockIdx.y, [](int n) { return n > 0 ? 1 : 0; }, e, first, count, place, total)) return;
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
    for (int t0 = 0; t0 < count; t0 += 16) {
        const int      T = min(16, count - t0);
        const int64_t  row = row_read(a, first + t0 + min(col, T - 1));   // (columns past the rows repeat the last one)
        const uint8_t *x = a.x + (row < 0 ? 0 : row) * a.pitch + quarter * 16;
        v4i            A[DEPTH][NR], B[DEPTH];
        Acc4           acc[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) acc[r] = Acc4{ 0, 0, 0, 0 };
        auto load = [&](int i, int s) __attribute__((always_inline)) {
#pragma unroll
            for (int r = 0; r < NR; ++r) A[i][r] = *reinterpret_cast<const v4i *>(from[r] + (int64_t) s * 2048);
            B[i] = *reinterpret_cast<const v4i *>(s * 64 + quarter * 16 < a.x_bytes ? x + s * 64 : kZeros);
        };
#pragma unroll
        for (int i = 0; i < DEPTH; ++i)
            if (s0 + i < s1) load(i, s0 + i);
        for (int s = s0; s < s1; s += DEPTH) {
#pragma unroll
            for (int i = 0; i < DEPTH; ++i) {
                if (s + i < s1) {
#pragma unroll
                    for (int r = 0; r < NR; ++r) acc[r] = Matrix<WT>::mfma16(A[i][r], B[i], acc[r]);
                    if (s + i + DEPTH < s1) load(i, s + i + DEPTH);
                }
            }
        }
        if (t0) __syncthreads();   // (the sums of the rows before are not read any more)
#pragma unroll
        for (int r = 0; r < NR; ++r)
            if (col < T) part[wave][r][col][quarter] = acc[r];
        __syncthreads();
        for (int c = threadIdx.x; c < NR * T * 4; c += 64 * W) {
            const int r = c / (T * 4), t = (c >> 2) % T, block = c & 3;
            Acc4      sum = part[0][r][t][block];
#pragma unroll
            for (int w = 1; w < W; ++w) sum += part[w][r][t][block];
            const int64_t p = first + t0 + t, n = (int64_t) (unit0 + r) * 16 + block * 4, out = row_written(a, p), in = row_read(a, p);
            if (out < 0 || n >= a.L.N) continue;
            v4f v;
            if constexpr (WT == RQ_I8) {
                const v4f   tn = *reinterpret_cast<const v4f *>(t_scales + n);
                const float sm = in < 0 ? 0.0f : a.x_scales[in];
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

template <int WT, bool GROUPED>
hipError_t stream(const ProductArgs &a, hipStream_t s) {
    const int64_t  units = (a.L.N + 15) / 16;
    const unsigned groups = GROUPED ? (unsigned) (a.P < a.E ? a.P : a.E) : 1;
    if (units * groups > 1024) {
        hipLaunchKernelGGL((rq_stream_kernel<WT, 8, 2, 4, GROUPED>), dim3((unsigned) ((units + 1) / 2), groups), dim3(512), 0, s, a);
    } else {
        hipLaunchKernelGGL((rq_stream_kernel<WT, 8, 1, 8, GROUPED>), dim3((unsigned) units, groups), dim3(512), 0, s, a);
    }
    return hipGetLastError();
}
template <bool GROUPED>
hipError_t stream(int weight_type, const ProductArgs &a, hipStream_t s) {
    if (weight_type == RQ_I8) return stream<RQ_I8, GROUPED>(a, s);
    if (weight_type == RQ_F16) return stream<RQ_F16, GROUPED>(a, s);
    return stream<RQ_BF16, GROUPED>(a, s);
}

}  // namespace

hipError_t launch_stream(int weight_type, const ProductArgs &a, hipStream_t s) {
    return a.offsets ? stream<true>(weight_type, a, s) : stream<false>(weight_type, a, s);
}

}  // namespace prod
}  // namespace rq
