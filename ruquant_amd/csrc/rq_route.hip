// Routing to experts: the choice, the order of the slots by expert, and the weighted sum of the experts' outputs.
#include "rq_mx.h"

namespace rq {
namespace mx {
namespace {

constexpr int   kRouteThreads = 256;
constexpr float kLowest = -3.402823466e38f;

// Over the wavefront by cross-lane operations of the vector ALU: quads, rows of 16, then rows 1 and 3 take their neighbour's, rows 2 and 3
// the lower half's, and lane 63 has all.
template <int CTRL, int ROWS>
__device__ __forceinline__ int moved(int v, int other) {
    return __builtin_amdgcn_update_dpp(other, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_max(int v) {
    constexpr int kLeast = -2147483647 - 1;   // (so that each step is one instruction)
    v = max(v, moved<0xB1, 0xF>(v, kLeast));
    v = max(v, moved<0x4E, 0xF>(v, kLeast));
    v = max(v, moved<0x141, 0xF>(v, kLeast));
    v = max(v, moved<0x140, 0xF>(v, kLeast));
    v = max(v, moved<0x142, 0xA>(v, kLeast));
    v = max(v, moved<0x143, 0xC>(v, kLeast));
    return __builtin_amdgcn_readlane(v, 63);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double added(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t) moved<CTRL, ROWS>((int) (uint32_t) b, 0), hi = (uint32_t) moved<CTRL, ROWS>((int) (uint32_t) (b >> 32), 0);
    return v + __builtin_bit_cast(double, (uint64_t) hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum(double v) {
    v = added<0xB1, 0xF>(v);
    v = added<0x4E, 0xF>(v);
    v = added<0x141, 0xF>(v);
    v = added<0x140, 0xF>(v);
    v = added<0x142, 0xA>(v);
    v = added<0x143, 0xC>(v);
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t) __builtin_amdgcn_readlane((int) (uint32_t) b, 63), hi = (uint32_t) __builtin_amdgcn_readlane((int) (uint32_t) (b >> 32), 63);
    return __builtin_bit_cast(double, (uint64_t) hi << 32 | lo);
}
// floats as whole numbers of the same order (no NaN, no -0)
__device__ __forceinline__ int ordered(float f) {
    const int b = __float_as_int(f);
    return b ^ ((b >> 31) & 0x7FFFFFFF);
}
__device__ __forceinline__ float unordered(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7FFFFFFF)); }
constexpr int kNever = -2147483647 - 1;   // in front of every number: what cannot be chosen

// A wavefront per token, experts V lane .. V lane + V - 1 in a lane. The choice is `top` rounds of a maximum over the wavefront, of whole
// numbers that have the order of the choices: the lowest lane and place that holds it is the lowest index. Bound by the vector ALU
// from some thousand tokens on (534 instructions a token of 256 experts, 8 of them from 4 of 8 groups, of which 190 are the rounds and 100 the
// sigmoid: 16384 tokens 16.6 us; their 17.8 MB would take 3.6), by its latency below (a token of 64 experts 2.4 us). The sums of exponentials are in 64 bits, so that no order
// of addition changes a choice between two equal scores.
template <int DT, int V>
__global__ __launch_bounds__(kRouteThreads) void rq_route_kernel(const RouteArgs a, const bool vec, const bool vec_bias) {
    using T = typename Element<DT>::type;
    const int     lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t m = (int64_t) blockIdx.x * (kRouteThreads / 64) + wave;
    if (m >= a.M) return;
    const T *x = reinterpret_cast<const T *>(a.logits) + m * a.ldl + lane * V;
    const int mine = min(max(a.E - lane * V, 0), V);   // experts of this lane
    float s[V], bias[V];
    int   c[V];
    // (loads of places past the last expert are of the last one: a branch for each would wait for one after the other)
    if (vec_bias) {
        typedef float B __attribute__((ext_vector_type(V > 1 ? V : 2)));
        const B b = reinterpret_cast<const B *>(a.bias)[mine ? lane : 0];
#pragma unroll
        for (int j = 0; j < V; ++j) bias[j] = b[j];
    } else if (a.bias) {
#pragma unroll
        for (int j = 0; j < V; ++j) bias[j] = a.bias[min(lane * V + j, a.E - 1)];
    }
    if (V > 1 && vec) {   // (whole lanes)
        if constexpr (DT == RQ_F32) {
            typedef float F __attribute__((ext_vector_type(V)));
            F f;
#pragma unroll
            for (int j = 0; j < V; ++j) f[j] = -INFINITY;
            if (mine) f = *reinterpret_cast<const F *>(x);
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] = f[j];
        } else {
            typedef uint16_t H __attribute__((ext_vector_type(V)));
            H h;
            if (mine) h = *reinterpret_cast<const H *>(x);
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] = mine ? to_float(__builtin_bit_cast(T, (uint16_t) h[j])) : -INFINITY;
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = to_float((x - lane * V)[min(lane * V + j, a.E - 1)]);
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = j < mine ? s[j] : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (!a.bias) bias[j] = 0;
        bias[j] = s[j] != s[j] ? s[j] : bias[j];   // (what the choice goes by is NaN then, and the score 0)
        s[j] = s[j] != s[j] ? -INFINITY : s[j];
    }
    if (a.scoring == 0) {
        int most = kNever;
#pragma unroll
        for (int j = 0; j < V; ++j) most = max(most, ordered(s[j]));
        const float top = unordered(wave_max(most));
        double      sum = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            s[j] = s[j] == -INFINITY ? 0.0f : s[j] == top ? 1.0f : expf(s[j] - top);
            sum += (double) s[j];
        }
        const float by = (float) wave_sum(sum);
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = by > 0 ? s[j] / by : 0.0f;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = 1.0f / (1.0f + expf(-s[j]));
    }
    // what the choice goes by: numbers from the lowest finite one up
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float v = s[j] + bias[j];
        c[j] = j < mine ? ordered(v > kLowest ? v : kLowest) : kNever;   // (a NaN is not greater)
    }
    if (a.groups > 1) {
        // 2^share lanes a group find its two largest; the groups' sums are compared by all of their lanes
        __shared__ int all[kRouteThreads / 64][64 * V];
        const int  size = a.E / a.groups, share = 31 - __clz(64 / a.groups), group = lane >> share, first = lane & ((1 << share) - 1);
        const bool own = size == V << share;   // the lanes of a group hold its experts
        int        one = kNever, two = kNever;
        auto       take = [&](int v) __attribute__((always_inline)) {
            two = max(two, min(one, v));
            one = max(one, v);
        };
        auto join = [&](int p, int q) __attribute__((always_inline)) {   // (p >= q)
            two = max(min(one, p), max(two, q));
            one = max(one, p);
        };
        if (own) {
#pragma unroll
            for (int j = 0; j < V; ++j) take(c[j]);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) all[wave][lane * V + j] = c[j];
            __builtin_amdgcn_wave_barrier();
            if (group < a.groups) {
                for (int i = first; i < size; i += 1 << share) take(all[wave][group * size + i]);
            }
        }
        if (share > 0) join(moved<0xB1, 0xF>(one, kNever), moved<0xB1, 0xF>(two, kNever));
        if (share > 1) join(moved<0x4E, 0xF>(one, kNever), moved<0x4E, 0xF>(two, kNever));
        if (share > 2) join(moved<0x141, 0xF>(one, kNever), moved<0x141, 0xF>(two, kNever));
        if (share > 3) join(moved<0x140, 0xF>(one, kNever), moved<0x140, 0xF>(two, kNever));
        if (share > 4) join(__shfl_xor(one, 16), __shfl_xor(two, 16));
        // (from half the lowest number up each, so that one number in front of nothing is more than two of those)
        const float worth = size > 1 ? fmaxf(unordered(one), 0.5f * kLowest) + fmaxf(unordered(two), 0.5f * kLowest) : unordered(one);
        int place = 0;   // groups that are worth more, or as much in front of it
        for (int g = 0; g < a.groups; ++g) {
            const float v = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(worth), g << share));
            place += v > worth || (v == worth && g < group);
        }
        const unsigned long long kept = __ballot(group < a.groups && place < a.top_groups);
        const float              per = 1.0f / (float) size;
        if (own) {
#pragma unroll
            for (int j = 0; j < V; ++j) c[j] = place < a.top_groups ? c[j] : kNever;
        }
#pragma unroll
        for (int j = 0; j < V && !own; ++j) {
            const int of = (int) (((float) (lane * V + j) + 0.5f) * per);   // (exact: under 1024, and half a unit away from whole numbers)
            if (!((kept >> (min(of, a.groups - 1) << share)) & 1)) c[j] = kNever;
        }
    }
    float  chosen = 0;
    double total = 0;   // (so that small scores beside a large one are not lost one after the other)
    int    id = 0;
    if constexpr (V > 1 && V <= 4) {
        // Each lane's experts in falling order, so that a round looks at its first and takes it off: 19 instructions for 30. (Neighbours are
        // compared, and change places where the second is larger: equal ones keep their order. V = 8 and 16 would sort as long as they save.)
        int order = 0, place[V];
#pragma unroll
        for (int j = 0; j < V; ++j) place[j] = j;
#pragma unroll
        for (int round = 0; round < V; ++round) {
#pragma unroll
            for (int j = round & 1; j + 1 < V; j += 2) {
                const bool swap = c[j] < c[j + 1];
                const int  most = max(c[j], c[j + 1]), least = min(c[j], c[j + 1]), p = place[j], q = place[j + 1];
                c[j] = most, c[j + 1] = least;
                place[j] = swap ? q : p, place[j + 1] = swap ? p : q;
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) order |= place[j] << (8 * j);
        for (int i = 0; i < a.top; ++i) {
            const int  best = wave_max(c[0]);
            const int  from = __builtin_ctzll(__ballot(c[0] == best));
            const int  e = from * V + (__builtin_amdgcn_readlane(order, from) & 255);
            const bool off = lane == from;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int here = c[j], next = j + 1 < V ? c[(j + 1) % V] : kNever;
                c[j] = off ? next : here;
            }
            order = off ? order >> 8 : order;
            id = lane == i ? e : id;
        }
        // the scores of the chosen, a lane each, and their sum in the order of choice
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float of = __shfl(s[j], id / V);
            chosen = id % V == j ? of : chosen;
        }
        for (int i = 0; i < a.top; ++i) total += (double) __int_as_float(__builtin_amdgcn_readlane(__float_as_int(chosen), i));
    } else {
        for (int i = 0; i < a.top; ++i) {
            int most = c[0];
#pragma unroll
            for (int j = 1; j < V; ++j) most = max(most, c[j]);
            const int best = wave_max(most);
            // (the lane and the place are the wavefront's, so the scalar unit finds them)
            unsigned long long has[V], any = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) has[j] = __ballot(c[j] == best), any |= has[j];
            const int from = __builtin_ctzll(any);
            int       at = 0;
            float     w = s[0];
#pragma unroll
            for (int j = V - 1; j > 0; --j) at = (has[j] >> from) & 1 ? j : at;
            at = (has[0] >> from) & 1 ? 0 : at;
#pragma unroll
            for (int j = 1; j < V; ++j) w = at == j ? s[j] : w;
            const float picked = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), from));
            const int   e = from * V + at;
#pragma unroll
            for (int j = 0; j < V; ++j) c[j] = lane == (at == j ? from : -1) ? kNever : c[j];
            total += (double) picked;
            if (lane == i) chosen = picked, id = e;
        }
    }
    if (lane < a.top) {
        const float sum = (float) total, w = a.renormalize ? (sum > 0 ? chosen / sum : 0.0f) : chosen;
        a.ids[m * a.top + lane] = id;
        a.weights[m * a.top + lane] = w * a.scale;
    }
}

template <int DT, int V>
void route_with(RouteArgs a, hipStream_t stream) {
    const int64_t bytes = (DT == RQ_F32 ? 4 : 2) * V, align = bytes < 16 ? bytes : 16;
    const bool    vec = a.E % V == 0 && (uintptr_t) a.logits % align == 0 && (a.M == 1 || a.ldl * (DT == RQ_F32 ? 4 : 2) % align == 0);
    const bool    vec_bias = V > 1 && a.bias && a.E % V == 0 && (uintptr_t) a.bias % (V < 4 ? 4 * V : 16) == 0;
    // (a launch has under 2^32 threads, and a token is 64 of them; the rows in front of a launch are a multiple of 16 bytes for any stride)
    constexpr int64_t kMost = 1 << 25;
    for (int64_t left = a.M; left > 0; left -= kMost) {
        a.M = left < kMost ? left : kMost;
        const dim3 grid((unsigned) ((a.M + kRouteThreads / 64 - 1) / (kRouteThreads / 64)));
        hipLaunchKernelGGL((rq_route_kernel<DT, V>), grid, dim3(kRouteThreads), 0, stream, a, vec, vec_bias);
        a.logits = reinterpret_cast<const typename Element<DT>::type *>(a.logits) + a.M * a.ldl;
        a.ids += a.M * a.top;
        a.weights += a.M * a.top;
    }
}
template <int DT>
hipError_t route(const RouteArgs &a, hipStream_t stream) {
    if (a.E <= 64) route_with<DT, 1>(a, stream);
    else if (a.E <= 128) route_with<DT, 2>(a, stream);
    else if (a.E <= 256) route_with<DT, 4>(a, stream);
    else if (a.E <= 512) route_with<DT, 8>(a, stream);
    else route_with<DT, 16>(a, stream);
    return hipGetLastError();
}

// One workgroup: counts the experts' slots, lays their tiles out and deals the slots to their places. The order of an expert's
// slots is that in which they arrive, and no result depends on it: every slot's row is computed by itself. A chain of passes over the ids by
// one compute unit: 16384 slots 14.5 us, 148 slots 6.2, of calls of 437 and 100.
constexpr int kSortThreads = 1024;
constexpr int kSortBatch = 8;   // ids in flight per thread
// Up to so many positions the slots are dealt in LDS and written in order: from this one workgroup a store of 64 places of memory
// takes 64 clocks. (16384 slots of 64 experts: 19 us dealt to memory directly.)
constexpr int kSortLds = 32768;

// sum over the threads in front of and with this one (all of the workgroup take part)
__device__ __forceinline__ int scan(int v, int *waves) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(v, o);
        if (lane >= o) v += u;
    }
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    for (int i = 0; i < wave; ++i) v += waves[i];
    return v;
}

__global__ __launch_bounds__(kSortThreads) void rq_sort_kernel(const SortArgs a) {
    __shared__ int count[RQ_ROUTE_MAX_E], waves[2][kSortThreads / 64];
    const int t = threadIdx.x;
    count[t] = 0;   // (E <= 1024)
    __syncthreads();
    for (int i0 = t; i0 < a.slots; i0 += kSortThreads * kSortBatch) {
        int e[kSortBatch];
#pragma unroll
        for (int k = 0; k < kSortBatch; ++k) e[k] = i0 + k * kSortThreads < a.slots ? a.ids[i0 + k * kSortThreads] : -1;
#pragma unroll
        for (int k = 0; k < kSortBatch; ++k)
            if (e[k] >= 0 && e[k] < a.E) atomicAdd(&count[e[k]], 1);
    }
    __syncthreads();
    // the positions (in 32s) and tiles in front of each expert, an expert a thread
    const int mine = t < a.E ? count[t] : 0, room = (mine + 31) & ~31, tiles = (mine + a.tile_tokens - 1) / a.tile_tokens;
    const int at = scan(room, waves[0]) - room, tile0 = scan(tiles, waves[1]) - tiles;
    if (t < a.E) {
        count[t] = at;
        for (int i = 0; i < tiles; ++i) {
            const Tile to = { t, at + i * a.tile_tokens, min(a.tile_tokens, mine - i * a.tile_tokens), 0 };
            a.tiles[tile0 + i] = to;
        }
        if (a.positions > kSortLds)
            for (int i = mine; i < room; ++i) a.token_of[at + i] = -1;
    }
    if (t == kSortThreads - 1) *a.used = at + room;
    __shared__ int last;
    if (t == kSortThreads - 1) last = tile0 + tiles;
    extern __shared__ int dealt[];
    const bool in_lds = a.positions <= kSortLds;
    __syncthreads();
    for (int i = last + t; i < a.most_tiles; i += kSortThreads) a.tiles[i] = Tile{ 0, 0, 0, 0 };
    for (int i0 = t; i0 < a.slots; i0 += kSortThreads * kSortBatch) {
        int e[kSortBatch], p[kSortBatch];
#pragma unroll
        for (int k = 0; k < kSortBatch; ++k) e[k] = i0 + k * kSortThreads < a.slots ? a.ids[i0 + k * kSortThreads] : -1;
#pragma unroll
        for (int k = 0; k < kSortBatch; ++k) p[k] = e[k] >= 0 && e[k] < a.E ? atomicAdd(&count[e[k]], 1) : -1;
#pragma unroll
        for (int k = 0; k < kSortBatch; ++k) {
            const int i = i0 + k * kSortThreads;
            if (p[k] < 0) continue;
            if (in_lds) dealt[p[k]] = i;
            else a.slot_of[p[k]] = i, a.token_of[p[k]] = i / a.top;
        }
    }
    if (!in_lds) return;
    // (the places behind an expert's last slot)
    if (t < a.E)
        for (int i = mine; i < room; ++i) dealt[at + i] = -1;
    __shared__ int positions;
    if (t == kSortThreads - 1) positions = at + room;
    __syncthreads();
    for (int p = t; p < positions; p += kSortThreads) {
        const int i = dealt[p];
        a.slot_of[p] = i;
        a.token_of[p] = i < 0 ? -1 : i / a.top;
    }
}

// y[m] = sum_j weights[m][j] * rows[m top + j] in the order of j, fp32; the slots' rows are loaded four at a time, four outputs a
// thread. Bound by memory: 2048 tokens x 8 rows of 5120, 73 us for 356 MB, 4.9 TB/s.
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void rq_combine_kernel(const float *rows, int64_t N, const int32_t *ids, const float *weights, int top, int E,
                                                         typename Element<DT>::type *y, int64_t ldy) {
    const int64_t m = blockIdx.x, n = ((int64_t) blockIdx.y * 256 + threadIdx.x) * 4;
    if (n >= N) return;
    v4f sum = { 0, 0, 0, 0 };
    for (int j0 = 0; j0 < top; j0 += 4) {
        v4f   v[4];
        float w[4];
        bool  there[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t slot = m * top + j0 + k;
            const int     e = j0 + k < top ? ids[slot] : -1;
            there[k] = e >= 0 && e < E;
            v[k] = v4f{ 0, 0, 0, 0 };
            w[k] = 0;
            if (there[k]) {
                w[k] = weights[slot];
                const float *row = rows + slot * N + n;
                if constexpr (VEC) {
                    v[k] = *reinterpret_cast<const v4f *>(row);
                } else {
                    for (int i = 0; i < 4; ++i)
                        if (n + i < N) v[k][i] = row[i];
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (there[k]) sum += w[k] * v[k];
    }
    store_out(DT, y, m * ldy, n, N, sum);
}

template <int DT>
hipError_t combine(const float *rows, int64_t N, const int32_t *ids, const float *weights, int64_t M, int top, int E, void *y, int64_t ldy,
                   hipStream_t stream) {
    auto      *out = reinterpret_cast<typename Element<DT>::type *>(y);
    const dim3 grid((unsigned) M, (unsigned) ((N + 1023) / 1024));
    if (N % 4 == 0) hipLaunchKernelGGL((rq_combine_kernel<DT, true>), grid, dim3(256), 0, stream, rows, N, ids, weights, top, E, out, ldy);
    else hipLaunchKernelGGL((rq_combine_kernel<DT, false>), grid, dim3(256), 0, stream, rows, N, ids, weights, top, E, out, ldy);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_route(const RouteArgs &a, hipStream_t stream) {
    if (a.dtype == RQ_F32) return route<RQ_F32>(a, stream);
    if (a.dtype == RQ_F16) return route<RQ_F16>(a, stream);
    return route<RQ_BF16>(a, stream);
}

hipError_t launch_sort(const SortArgs &a, hipStream_t stream) {
    static std::atomic<uint64_t> allowed{ 0 };
    const hipError_t e = allow_lds(reinterpret_cast<const void *>(rq_sort_kernel), kSortLds * (int) sizeof(int), allowed);
    if (e != hipSuccess) return e;
    const int bytes = a.positions <= kSortLds ? a.positions * (int) sizeof(int) : 0;
    hipLaunchKernelGGL(rq_sort_kernel, dim3(1), dim3(kSortThreads), bytes, stream, a);
    return hipGetLastError();
}

hipError_t launch_combine(const float *rows, int64_t N, const int32_t *ids, const float *weights, int64_t M, int top, int E, int out_dtype, void *y,
                          int64_t ldy, hipStream_t stream) {
    if (out_dtype == RQ_F32) return combine<RQ_F32>(rows, N, ids, weights, M, top, E, y, ldy, stream);
    if (out_dtype == RQ_F16) return combine<RQ_F16>(rows, N, ids, weights, M, top, E, y, ldy, stream);
    return combine<RQ_BF16>(rows, N, ids, weights, M, top, E, y, ldy, stream);
}

}  // namespace mx
}  // namespace rq
