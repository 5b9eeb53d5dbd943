// Sort of slots by expert: a stable counting sort, so that it is the same every time.
//
// A workgroup has a run of slots, a wavefront some rows of 64 of them, whose ids its lanes keep. A wavefront ranks 64 slots among those of the same
// expert by comparing the bits of their ids across its lanes, and adds them to its count of that expert in one step. One run is one launch; more are
// counted by a launch in front, and every run then adds up the counts of all, which are few and lie in the caches. 131072 slots of 256 experts 2.9 + 9.3 us, 8 slots 3.0:
// the chain of the ids' load, the counts, their sum over the wavefronts and experts, and the slots' places.
#include <type_traits>

#include "rq_prod.h"

namespace rq {
namespace prod {
namespace {

constexpr int kSortThreads = 1024, kWaves = kSortThreads / 64;

struct SortArgs {
    const int32_t *ids;
    int            slots, top, E;
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

// The ids of this wavefront's slots: row k of 64 begins at first + 64 k. Behind the last slot a number that no expert has.
constexpr int kNone = 0x7FF;
template <int PER>
__device__ __forceinline__ int load_experts(const SortArgs &a, int (&e)[PER]) {
    const int first = ((int) blockIdx.x * kWaves + ((int) threadIdx.x >> 6)) * 64 * PER, lane = threadIdx.x & 63;
#pragma unroll
    for (int k = 0; k < PER; ++k) e[k] = first + 64 * k + lane < a.slots ? expert_of(a, first + 64 * k + lane) : kNone;
    return first;
}

template <int PER>
__global__ __launch_bounds__(kSortThreads) void rq_sort_count_kernel(const SortArgs a) {
    __shared__ int count[RQ_GROUPED_MAX_E + 1];
    int            e[PER];
    load_experts<PER>(a, e);
    for (int i = threadIdx.x; i <= a.E; i += kSortThreads) count[i] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PER; ++k)
        if (e[k] != kNone) atomicAdd(&count[e[k]], 1);
    __syncthreads();
    for (int i = threadIdx.x; i <= a.E; i += kSortThreads) a.counts[blockIdx.x * (a.E + 1) + i] = count[i];
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
template <int PER, bool COUNTED>
__global__ __launch_bounds__(kSortThreads) void rq_sort_place_kernel(const SortArgs a) {
    extern __shared__ int at[];   // [kWaves][E + 1]; COUNTED: then [2][E + 1], all slots of an expert, and those of the runs in front
    __shared__ int waves[kWaves], behind;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, E1 = a.E + 1;
    int      *sums = at + kWaves * E1;
    int       e[PER];
    const int first = load_experts<PER>(a, e);
    for (int i = t; i < (COUNTED ? kWaves + 2 : kWaves) * E1; i += kSortThreads) at[i] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PER; ++k)
        if (e[k] != kNone) atomicAdd(&at[wave * E1 + e[k]], 1);
    if constexpr (COUNTED) {   // the runs in as many shares as the threads have columns for, eight loads on their way in each
        const int stride = (E1 + 63) & ~63, shares = max(1, kSortThreads / stride), runs = gridDim.x;
        for (int i = t; i < shares * stride; i += kSortThreads) {
            const int share = i / stride, c = i - share * stride, r1 = runs * (share + 1) / shares;
            if (c >= E1) continue;
            int all = 0, front = 0;
            for (int r = runs * share / shares; r < r1; r += 8) {
                int n[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) n[k] = r + k < r1 ? a.counts[(r + k) * E1 + c] : 0;
#pragma unroll
                for (int k = 0; k < 8; ++k) all += n[k], front += r + k < (int) blockIdx.x ? n[k] : 0;
            }
            atomicAdd(&sums[c], all);
            atomicAdd(&sums[E1 + c], front);
        }
    }
    __syncthreads();
    // expert t: how many slots there are, how many of them in the runs in front, and in this run's wavefronts
    int all = 0;
    if (t < a.E) {
        if constexpr (COUNTED) all = sums[t];
        else
            for (int w = 0; w < kWaves; ++w) all += at[w * E1 + t];
    }
    const int end = scan(all, waves);   // (E <= 1024 = the threads)
    if (t == kSortThreads - 1) behind = end;
    if (blockIdx.x == 0) {
        if (t < a.E) a.offsets[t + 1] = end;
        if (t == 0) a.offsets[0] = 0;
    }
    __syncthreads();
    for (int c = t; c < E1; c += kSortThreads) {   // (column E: the slots of no expert, behind all others)
        int to = (c < a.E ? end - all : behind) + (COUNTED ? sums[E1 + c] : 0);
        for (int w = 0; w < kWaves; ++w) {
            const int n = at[w * E1 + c];
            at[w * E1 + c] = to;
            to += n;
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PER; ++k) {   // (this wavefront alone has its row of `at`)
        const uint64_t same = peers(e[k]), below = same & ((1ull << lane) - 1);
        if (e[k] != kNone) {
            int      *cell = &at[wave * E1 + e[k]];
            const int p = *cell + __builtin_popcountll(below), i = first + 64 * k + lane;
            a.slots_out[p] = i;
            a.tokens[p] = i / a.top;
            __builtin_amdgcn_wave_barrier();
            if (below == 0) *cell = p + __builtin_popcountll(same);
            __builtin_amdgcn_wave_barrier();
        }
    }
}

constexpr int64_t kMaxSlots = 1 << 22;
// Rows of 64 slots that a wavefront has: short runs (2048 slots) where they are few.
constexpr int kShort = 2, kLong = 8;
constexpr int run_of(int per) { return kSortThreads * per; }
int           rows_of(int64_t slots) { return slots <= 64 * run_of(kShort) ? kShort : kLong; }
bool good(int64_t M, int top, int64_t E) {
    return M >= 0 && top >= 1 && top <= 1024 && M <= kMaxSlots / top && E >= 1 && E <= RQ_GROUPED_MAX_E;
}

}  // namespace
}  // namespace prod
}  // namespace rq

using namespace rq::prod;

extern "C" size_t rq_sort_workspace_bytes(int64_t M, int top, int64_t E) {
    if (!good(M, top, E)) return 0;
    // (as many runs as the call's or any smaller one's, so that it grows)
    const int64_t slots = M * top;
    if (slots <= run_of(kShort)) return 0;
    const int64_t few = slots < 64 * run_of(kShort) ? slots : 64 * run_of(kShort), a = (few + run_of(kShort) - 1) / run_of(kShort), b = (slots + run_of(kLong) - 1) / run_of(kLong);
    return (size_t) up_to((a > b ? a : b) * (E + 1) * 4, 256);
}

extern "C" int rq_sort_slots(const int32_t *ids, int64_t M, int top, int64_t E, int32_t *offsets, int32_t *slots, int32_t *tokens,
                             void *workspace, size_t workspace_bytes, rq_stream_t stream) {
    if (!good(M, top, E)) return RQ_E_UNSUPPORTED;
    auto aligned4 = [](const void *p) { return (uintptr_t) p % 4 == 0; };
    if (!offsets || !aligned4(offsets) || (M > 0 && (!ids || !slots || !tokens || !aligned4(ids) || !aligned4(slots) || !aligned4(tokens)))) return RQ_E_ARGUMENT;
    const size_t need = rq_sort_workspace_bytes(M, top, E);
    if (need && (!workspace || (uintptr_t) workspace % 256 || workspace_bytes < need)) return RQ_E_WORKSPACE;
    const int      n = (int) (M * top), per = rows_of(n), runs = n ? (n + run_of(per) - 1) / run_of(per) : 1;
    const SortArgs a = { ids, n, top, (int) E, offsets, slots, tokens, (int *) workspace };
    auto           run = [&](auto rows) {
        constexpr int PER = decltype(rows)::value;
        static std::atomic<uint64_t> allowed[2];
        const void *kernels[2] = { reinterpret_cast<const void *>(rq_sort_place_kernel<PER, false>), reinterpret_cast<const void *>(rq_sort_place_kernel<PER, true>) };
        const int   counted = runs > 1, bytes = (kWaves + 2 * counted) * ((int) E + 1) * (int) sizeof(int);
        hipError_t  e = allow_lds(kernels[counted], (kWaves + 2) * (RQ_GROUPED_MAX_E + 1) * (int) sizeof(int), allowed[counted]);
        if (e != hipSuccess) return e;
        if (counted) {
            hipLaunchKernelGGL(rq_sort_count_kernel<PER>, dim3(runs), dim3(kSortThreads), 0, (hipStream_t) stream, a);
            e = hipGetLastError();
            if (e != hipSuccess) return e;
            hipLaunchKernelGGL((rq_sort_place_kernel<PER, true>), dim3(runs), dim3(kSortThreads), bytes, (hipStream_t) stream, a);
        } else {
            hipLaunchKernelGGL((rq_sort_place_kernel<PER, false>), dim3(1), dim3(kSortThreads), bytes, (hipStream_t) stream, a);
        }
        return hipGetLastError();
    };
    return per == kShort ? run(std::integral_constant<int, kShort>{}) : run(std::integral_constant<int, kLong>{});
}
