// Sort of slots by expert: a stable counting sort, so that it is the same every time.
//
// Slots go in runs of kRun. A wavefront ranks 64 slots among those of the same expert by comparing the bits of their ids across its lanes, and
// adds them to its run's count of that expert in one step. One run is one launch; more are counted by a launch in front, and every run then adds up
// the counts of those in front of it, which are few and lie in the caches.
#include "rq_prod.h"

namespace rq {
namespace prod {
namespace {

constexpr int kSortThreads = 1024, kWaves = kSortThreads / 64;

struct SortArgs {
    const int32_t *ids;
    int            slots, top, E, run;   // run: slots of a workgroup
    int32_t       *offsets, *slots_out, *tokens;
    int           *counts;               // [run][E + 1]
};

// The lanes whose e is this lane's (0 .. 1024, so 11 bits).
__device__ __forceinline__ uint64_t peers(int e) {
    uint64_t same = ~0ull;
#pragma unroll
    for (int b = 0; b < 11; ++b) {
        const uint64_t set = __ballot((e >> b) & 1);
        same &= (e >> b) & 1 ? set : ~set;
    }
    return same;
}
__device__ __forceinline__ int expert_of(const SortArgs &a, int i) {
    const int e = a.ids[i];
    return e >= 0 && e < a.E ? e : a.E;
}

__global__ __launch_bounds__(kSortThreads) void rq_sort_count_kernel(const SortArgs a) {
    __shared__ int count[RQ_GROUPED_MAX_E + 1];
    for (int e = threadIdx.x; e <= a.E; e += kSortThreads) count[e] = 0;
    __syncthreads();
    const int i0 = blockIdx.x * a.run, i1 = min(i0 + a.run, a.slots);
    for (int i = i0 + (int) threadIdx.x; i < i1; i += kSortThreads) atomicAdd(&count[expert_of(a, i)], 1);
    __syncthreads();
    for (int e = threadIdx.x; e <= a.E; e += kSortThreads) a.counts[blockIdx.x * (a.E + 1) + e] = count[e];
}

// Sum over the threads up to this one; all of the workgroup take part.
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

// COUNTED: a.counts holds what every run has of every expert; otherwise there is one run. at[w][e]: where wavefront w's next slot of expert e goes.
// A wavefront has a row of 64 slots after the other, its share of the run.
template <bool COUNTED>
__global__ __launch_bounds__(kSortThreads) void rq_sort_place_kernel(const SortArgs a) {
    extern __shared__ int at[];   // [kWaves][E + 1]
    __shared__ int waves[kWaves], behind;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, E1 = a.E + 1;
    for (int i = t; i < kWaves * E1; i += kSortThreads) at[i] = 0;
    __syncthreads();
    const int i0 = blockIdx.x * a.run, i1 = min(i0 + a.run, a.slots);
    const int share = ((i1 - i0 + kWaves - 1) / kWaves + 63) & ~63;
    const int w0 = min(i0 + wave * share, i1), w1 = min(w0 + share, i1);
    for (int i = w0 + lane; i < w1; i += 64) atomicAdd(&at[wave * E1 + expert_of(a, i)], 1);
    __syncthreads();
    // expert t: how many slots there are, how many of them in the runs in front, and in this run's wavefronts
    int all = 0, front = 0;
    if (t < a.E) {
        if constexpr (COUNTED) {
            for (int r = 0; r < (int) gridDim.x; ++r) {
                const int c = a.counts[r * E1 + t];
                all += c;
                front += r < (int) blockIdx.x ? c : 0;
            }
        } else {
            for (int w = 0; w < kWaves; ++w) all += at[w * E1 + t];
        }
    }
    const int end = scan(all, waves);   // (E <= 1024 = the threads)
    if (t == kSortThreads - 1) behind = end;
    if (blockIdx.x == 0) {
        if (t < a.E) a.offsets[t + 1] = end;
        if (t == 0) a.offsets[0] = 0;
    }
    __syncthreads();
    if (t < a.E) {
        int to = end - all + front;
        for (int w = 0; w < kWaves; ++w) {
            const int c = at[w * E1 + t];
            at[w * E1 + t] = to;
            to += c;
        }
    }
    if (t == 0) {   // the slots of no expert: behind all others, as many in front of this run as its slots less those that have one
        int to = behind;
        if constexpr (COUNTED)
            for (int r = 0; r < (int) blockIdx.x; ++r) to += a.counts[r * E1 + a.E];
        for (int w = 0; w < kWaves; ++w) {
            const int c = at[w * E1 + a.E];
            at[w * E1 + a.E] = to;
            to += c;
        }
    }
    __syncthreads();
    for (int i = w0; i < w1; i += 64) {   // (this wavefront alone has its row of `at`)
        const bool     there = i + lane < w1;
        const int      e = there ? expert_of(a, i + lane) : 0x7FF;   // (a number that no expert has)
        const uint64_t same = peers(e), below = same & ((1ull << lane) - 1);
        if (there) {
            int      *cell = &at[wave * E1 + e];
            const int p = *cell + __builtin_popcountll(below);
            a.slots_out[p] = i + lane;
            a.tokens[p] = (i + lane) / a.top;
            __builtin_amdgcn_wave_barrier();
            if (below == 0) *cell = p + __builtin_popcountll(same);
            __builtin_amdgcn_wave_barrier();
        }
    }
}

constexpr int64_t kMaxSlots = 1 << 22;
constexpr int     kOneRun = 8192;
// Runs of at least kOneRun slots, at most 256 of them.
int run_of(int64_t slots) {
    const int64_t each = up_to((slots + 255) / 256, kSortThreads);
    return (int) (each > kOneRun ? each : kOneRun);
}
bool good(int64_t M, int top, int64_t E) {
    return M >= 0 && top >= 1 && top <= 1024 && M <= kMaxSlots / top && E >= 1 && E <= RQ_GROUPED_MAX_E;
}

}  // namespace
}  // namespace prod
}  // namespace rq

using namespace rq::prod;

extern "C" size_t rq_sort_workspace_bytes(int64_t M, int top, int64_t E) {
    if (!good(M, top, E)) return 0;
    const int64_t slots = M * top, run = run_of(slots), runs = (slots + run - 1) / run;
    return runs <= 1 ? 0 : (size_t) up_to(runs * (E + 1) * 4, 256);
}

extern "C" int rq_sort_slots(const int32_t *ids, int64_t M, int top, int64_t E, int32_t *offsets, int32_t *slots, int32_t *tokens,
                             void *workspace, size_t workspace_bytes, rq_stream_t stream) {
    if (!good(M, top, E)) return RQ_E_UNSUPPORTED;
    auto aligned4 = [](const void *p) { return (uintptr_t) p % 4 == 0; };
    if (!offsets || !aligned4(offsets) || (M > 0 && (!ids || !slots || !tokens || !aligned4(ids) || !aligned4(slots) || !aligned4(tokens)))) return RQ_E_ARGUMENT;
    const size_t need = rq_sort_workspace_bytes(M, top, E);
    if (need && (!workspace || (uintptr_t) workspace % 256 || workspace_bytes < need)) return RQ_E_WORKSPACE;
    const int      n = (int) (M * top), run = run_of(n), runs = n ? (n + run - 1) / run : 1;
    const SortArgs a = { ids, n, top, (int) E, run, offsets, slots, tokens, (int *) workspace };
    const int      bytes = kWaves * ((int) E + 1) * (int) sizeof(int);
    static std::atomic<uint64_t> allowed[2];
    const void *kernels[2] = { reinterpret_cast<const void *>(rq_sort_place_kernel<false>), reinterpret_cast<const void *>(rq_sort_place_kernel<true>) };
    const int   counted = runs > 1;
    hipError_t  e = allow_lds(kernels[counted], kWaves * (RQ_GROUPED_MAX_E + 1) * (int) sizeof(int), allowed[counted]);
    if (e != hipSuccess) return e;
    if (counted) {
        hipLaunchKernelGGL(rq_sort_count_kernel, dim3(runs), dim3(kSortThreads), 0, (hipStream_t) stream, a);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL(rq_sort_place_kernel<true>, dim3(runs), dim3(kSortThreads), bytes, (hipStream_t) stream, a);
    } else {
        hipLaunchKernelGGL(rq_sort_place_kernel<false>, dim3(1), dim3(kSortThreads), bytes, (hipStream_t) stream, a);
    }
    return hipGetLastError();
}
