// Routing to experts: the choice, the order of the slots by expert, and the weighted sum of the experts' outputs.
#include "rq_mx.h"

namespace rq {
namespace mx {
namespace {

constexpr int kRouteThreads = 256;
constexpr float kLowest = -3.402823466e38f;

// A wavefront per token, expert e in lane e / V, slot e % V, V = values per lane.
template <int DT, int V>
__global__ __launch_bounds__(kRouteThreads) void rq_route_kernel(const RouteArgs a) {
    const int     lane = threadIdx.x & 63;
    const int64_t m = (int64_t) blockIdx.x * (kRouteThreads / 64) + (threadIdx.x >> 6);
    if (m >= a.M) return;
    const typename Element<DT>::type *x = reinterpret_cast<const typename Element<DT>::type *>(a.logits) + m * a.ldl;
    float s[V], c[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int   e = lane * V + j;
        const float f = e < a.E ? to_float(x[e]) : -INFINITY;
        s[j] = f != f ? -INFINITY : f;
    }
    if (a.scoring == 0) {
        float top = s[0];
#pragma unroll
        for (int j = 1; j < V; ++j) top = fmaxf(top, s[j]);
        for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        double sum = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            s[j] = s[j] == -INFINITY ? 0.0f : s[j] == top ? 1.0f : expf(s[j] - top);
            sum += (double) s[j];
        }
        for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
        const float by = (float) sum;
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = by > 0 ? s[j] / by : 0.0f;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = 1.0f / (1.0f + expf(-s[j]));
    }
    // what the choice goes by: numbers from the lowest finite one up; what cannot be chosen is minus infinity
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int e = lane * V + j;
        float     v = s[j];
        if (a.bias && e < a.E) v += a.bias[e];
        c[j] = e >= a.E ? -INFINITY : v > kLowest ? v : kLowest;   // (a NaN is not greater)
    }
    if (a.groups > 1) {
        // the groups' worth, a group per lane: its two largest values, found one expert at a time
        const int size = a.E / a.groups;
        float worth = -INFINITY;
        float one = -INFINITY, two = -INFINITY;
        for (int i = 0; i < size; ++i) {
            const int e = lane * size + i;
            float     v = -INFINITY;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float t = __shfl(c[j], (e / V) & 63);
                if (e % V == j) v = t;
            }
            if (v > one) two = one, one = v;
            else if (v > two) two = v;
        }
        if (lane < a.groups) {
            worth = size > 1 ? one + two : one;
            worth = worth > kLowest ? worth : kLowest;
        }
        // its place among the groups: how many are worth more, or as much in front of it
        int place = 0;
        for (int g = 0; g < a.groups; ++g) {
            const float v = __shfl(worth, g);
            place += v > worth || (v == worth && g < lane);
        }
        const int kept = lane < a.groups && place < a.top_groups;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int e = lane * V + j;
            const int k = __shfl(kept, (e / size) & 63);
            if (!k || e >= a.E) c[j] = -INFINITY;
        }
    }
    float chosen = 0, total = 0;
    int   id = 0;
    for (int i = 0; i < a.top; ++i) {
        float best = c[0];
        int   at = 0;
#pragma unroll
        for (int j = 1; j < V; ++j) {
            if (c[j] > best) best = c[j], at = j;
        }
        float all = best;
        for (int o = 32; o; o >>= 1) all = fmaxf(all, __shfl_xor(all, o));
        const int   from = __ffsll((unsigned long long) __ballot(best == all)) - 1;   // the lowest lane
        float       w = s[0];
#pragma unroll
        for (int j = 1; j < V; ++j) w = at == j ? s[j] : w;
        w = __shfl(w, from);
        const int e = __shfl(lane * V + at, from);
        if (lane == from) {
#pragma unroll
            for (int j = 0; j < V; ++j) c[j] = at == j ? -INFINITY : c[j];
        }
        total += w;
        if (lane == i) chosen = w, id = e;
    }
    if (lane < a.top) {
        const float w = a.renormalize ? (total > 0 ? chosen / total : 0.0f) : chosen;
        a.ids[m * a.top + lane] = id;
        a.weights[m * a.top + lane] = w * a.scale;
    }
}

template <int DT>
hipError_t route(const RouteArgs &a, hipStream_t stream) {
    const dim3 grid((unsigned) ((a.M + kRouteThreads / 64 - 1) / (kRouteThreads / 64)));
    const int  v = (a.E + 63) / 64;
    if (v <= 1) hipLaunchKernelGGL((rq_route_kernel<DT, 1>), grid, dim3(kRouteThreads), 0, stream, a);
    else if (v <= 2) hipLaunchKernelGGL((rq_route_kernel<DT, 2>), grid, dim3(kRouteThreads), 0, stream, a);
    else if (v <= 4) hipLaunchKernelGGL((rq_route_kernel<DT, 4>), grid, dim3(kRouteThreads), 0, stream, a);
    else if (v <= 8) hipLaunchKernelGGL((rq_route_kernel<DT, 8>), grid, dim3(kRouteThreads), 0, stream, a);
    else hipLaunchKernelGGL((rq_route_kernel<DT, 16>), grid, dim3(kRouteThreads), 0, stream, a);
    return hipGetLastError();
}

// One workgroup: counts the experts' slots, lays their tiles out and deals the slots to their places. The order of an expert's
// slots is that in which they arrive, and no result depends on it: every slot's row is computed by itself.
constexpr int kSortThreads = 1024;
__global__ __launch_bounds__(kSortThreads) void rq_sort_kernel(const SortArgs a) {
    __shared__ int count[RQ_ROUTE_MAX_E], first[RQ_ROUTE_MAX_E];
    const int t = threadIdx.x;
    for (int e = t; e < a.E; e += kSortThreads) count[e] = 0;
    __syncthreads();
    for (int i = t; i < a.slots; i += kSortThreads) {
        const int e = a.ids[i];
        if (e >= 0 && e < a.E) atomicAdd(&count[e], 1);
    }
    __syncthreads();
    // prefix sums of the positions (in 32s) and of the tiles, an expert a thread (E <= 1024)
    const int mine = t < a.E ? count[t] : 0, room = (mine + 31) & ~31, tiles = (mine + a.tile_tokens - 1) / a.tile_tokens;
    __shared__ int sum1[kSortThreads], sum2[kSortThreads];
    sum1[t] = room;
    sum2[t] = tiles;
    __syncthreads();
    for (int o = 1; o < kSortThreads; o <<= 1) {
        const int v = t >= o ? sum1[t - o] : 0, w = t >= o ? sum2[t - o] : 0;
        __syncthreads();
        sum1[t] += v;
        sum2[t] += w;
        __syncthreads();
    }
    if (t < a.E) {
        const int at = sum1[t] - room;
        first[t] = at;
        for (int i = 0; i < tiles; ++i) {
            Tile &to = a.tiles[sum2[t] - tiles + i];
            to.expert = t;
            to.first = at + i * a.tile_tokens;
            to.count = min(a.tile_tokens, mine - i * a.tile_tokens);
        }
        for (int i = mine; i < room; ++i) a.token_of[at + i] = -1;
    }
    if (t == kSortThreads - 1) {
        a.n_tiles[0] = sum2[t];
        a.n_tiles[1] = sum1[t];
    }
    __syncthreads();
    for (int i = t; i < a.slots; i += kSortThreads) {
        const int e = a.ids[i];
        if (e >= 0 && e < a.E) {
            const int p = atomicAdd(&first[e], 1);
            a.slot_of[p] = i;
            a.token_of[p] = i / a.top;
        }
    }
}

template <int DT>
__global__ __launch_bounds__(256) void rq_combine_kernel(const float *rows, int64_t N, const int32_t *ids, const float *weights,
                                                         int top, int E, typename Element<DT>::type *y, int64_t ldy) {
    const int64_t m = blockIdx.x;
    for (int64_t n = (int64_t) blockIdx.y * 256 + threadIdx.x; n < N; n += (int64_t) gridDim.y * 256) {
        float sum = 0;
        for (int j = 0; j < top; ++j) {
            const int e = ids[m * top + j];
            if (e >= 0 && e < E) sum += weights[m * top + j] * rows[(m * top + j) * N + n];
        }
        y[m * ldy + n] = from_float<DT>(sum);
    }
}

}  // namespace

hipError_t launch_route(const RouteArgs &a, hipStream_t stream) {
    if (a.dtype == RQ_F32) return route<RQ_F32>(a, stream);
    if (a.dtype == RQ_F16) return route<RQ_F16>(a, stream);
    return route<RQ_BF16>(a, stream);
}

hipError_t launch_sort(const SortArgs &a, hipStream_t stream) {
    hipLaunchKernelGGL(rq_sort_kernel, dim3(1), dim3(kSortThreads), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_combine(const float *rows, int64_t N, const int32_t *ids, const float *weights, int64_t M, int top, int E,
                          int out_dtype, void *y, int64_t ldy, hipStream_t stream) {
    const dim3 grid((unsigned) M, (unsigned) ((N + 1023) / 1024));
    if (out_dtype == RQ_F32) {
        hipLaunchKernelGGL((rq_combine_kernel<RQ_F32>), grid, dim3(256), 0, stream, rows, N, ids, weights, top, E, (float *) y, ldy);
    } else if (out_dtype == RQ_F16) {
        hipLaunchKernelGGL((rq_combine_kernel<RQ_F16>), grid, dim3(256), 0, stream, rows, N, ids, weights, top, E, (__half *) y, ldy);
    } else {
        hipLaunchKernelGGL((rq_combine_kernel<RQ_BF16>), grid, dim3(256), 0, stream, rows, N, ids, weights, top, E,
                           (__hip_bfloat16 *) y, ldy);
    }
    return hipGetLastError();
}

}  // namespace mx
}  // namespace rq
