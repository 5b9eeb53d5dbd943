// Entry points of the int8 product and of the products grouped by expert: argument checks, workspaces, order of launches.
#include <string.h>

#include "../../include/rq_i8_plan.h"
#include "rq_prod.h"

using namespace rq::prod;

namespace {

bool   float_dtype(int dtype) { return dtype == RQ_F32 || dtype == RQ_F16 || dtype == RQ_BF16; }
bool   aligned(const void *p, size_t n) { return (uintptr_t) p % n == 0; }
size_t pad256(int64_t n) { return (size_t) up_to(n, 256); }

constexpr int64_t kMaxPositions = 1 << 22;   // rows of a call

// Rows of x as the kernels read them: in the workspace (rounded, or brought to multiples of 16 bytes), or where they are.
// (An odd number of lines of 128 bytes apart: at some other distances the same bytes of many rows, which the tiles read together, lie in few of an L2's
// channels: 2048 tokens x 16384 x 5120 in tiles of 256 x 256 at 5120 bytes 162 us, at 5248 151, of 128 x 128 226 and 181; at 4096 and 4224 alike.)
int64_t packed_bytes(int weight_type, int64_t K) { return up_to(K * type_bytes(weight_type), 64); }
int64_t packed_pitch(int weight_type, int64_t K) { return (up_to(K * type_bytes(weight_type), 128) / 128 | 1) * 128; }
size_t  act_bytes(int weight_type, int64_t K, int64_t M) { return pad256(M * packed_pitch(weight_type, K)) + pad256(M * 4); }

// Sets a's rows of x; launches what brings them there, and zeros to a.arrived.
hipError_t take_rows(ProductArgs &a, int weight_type, int64_t K, int in_dtype, const void *x, int64_t ldx, const float *x_scales, int64_t M,
                     bool few, int counters, uint8_t *workspace, hipStream_t stream) {
    a.M = M, a.chunk = 16;
    const int64_t row_bytes = K * type_bytes(weight_type), pitch = packed_pitch(weight_type, K), padded = packed_bytes(weight_type, K);
    if (weight_type == RQ_I8 && in_dtype != RQ_I8) {
        float *scales = reinterpret_cast<float *>(workspace + pad256(M * pitch));
        a.x = workspace, a.pitch = pitch, a.x_bytes = padded, a.x_scales = scales;
        return launch_i8_quantize(in_dtype, x, ldx, M, K, workspace, pitch, padded, scales, a.arrived, counters, stream);
    }
    a.x_scales = x_scales;
    const int64_t ld_bytes = ldx * type_bytes(in_dtype);
    if (few || (aligned(x, 16) && (M == 1 || ld_bytes % 16 == 0) && row_bytes % 16 == 0)) {
        a.x = (const uint8_t *) x, a.pitch = ld_bytes, a.x_bytes = row_bytes;
        return counters ? launch_pack(nullptr, 0, 0, 0, nullptr, 16, a.arrived, counters, stream) : hipSuccess;
    }
    a.x = workspace, a.pitch = pitch, a.x_bytes = padded;
    return launch_pack(x, ld_bytes, M, row_bytes, workspace, pitch, a.arrived, counters, stream);
}

// What a product runs.
struct Plan {
    bool    few;                   // launch_stream
    int     form, rest;            // tiles; rest: of the rows behind main_tiles row tiles, or -1
    int64_t main_tiles;
    int     splits, split_steps;
    int     counters;              // and bytes of sums, that splits > 1 takes
    int64_t sums_bytes;
};
// The tiles' forms, and what they take in microseconds: a step of 64 bytes where every compute unit has a tile of its own, a step of 256 tiles where the chip is full
// of them (256 x 256: 2.1 POP/s, what a large int8 library product reaches here: the chip's clock falls to that, whatever the form), what stands in front of and behind the
// steps; and, where several workgroups share a tile, their join, per part, and per tile and part of 64 KiB. Fitted to 959 times of K = 1024 to 17408, N = 512 to
// 17408 and 8 to 2048 rows of int8 in one group: what they choose is 1 % slower than the fastest of sixteen forms and shares on average, 13 % at worst. Groups and 16-bit weights go
// by the same prices, as if all groups had as many rows: over 47 calls of 4 to 64 routed experts (int8, fp16, bf16, K and N = 256 to 5100, 22 to 1939 tokens) 2 % on average and 11 %
// at worst behind the fastest of the five forms.
struct Form {
    int    resident;   // tiles that a compute unit holds
    double alone, full, fixed, join, part, tile;
};
constexpr Form    kForm[kForms] = { { 2, .112, .132, 4.7, 2.4, .50, .011 },
                                    { 2, .142, .196, 5.1, 2.5, .57, .014 },
                                    { 2, .268, .343, 5.4, 0.9, .50, .031 },
                                    { 1, .212, .292, 5.9, 2.5, .80, .016 },
                                    { 1, .504, 1.03, 10.1, 0, 0, 0 } };
constexpr int     kMostSplits = 8, kMostShared = 256;   // workgroups that share a tile, tiles that are shared
constexpr int64_t kMostSums = 32 << 20;
constexpr bool    shared_form(int f) { return f == 0 || f == 1 || f == 3; }
int64_t           tile_bytes(int f) { return (int64_t) tiled_rows(f) * tiled_tokens(f) * 4; }

// of `tiles` tiles, each by `parts` workgroups of `steps` steps
double price(int f, double tiles, int64_t steps, int64_t parts) {
    const Form   &o = kForm[f];
    const double  all = tiles * (double) parts, load = (double) (int64_t) ((all + 255) / 256);   // of the busiest compute unit
    const int64_t rounds = ((int64_t) load + o.resident - 1) / o.resident;
    double        step = o.alone * (double) rounds;
    if (step < o.full * all / 256) step = o.full * all / 256;
    if (load > 1 && step < .75 * o.full * load) step = .75 * o.full * load;
    double t = o.fixed * (double) rounds + step * (double) steps;
    if (parts > 1) t += o.join + o.part * (double) parts + o.tile * all * (double) tile_bytes(f) / 65536;
    return t;
}
// (nothing is faster than its weights come from memory; of those that they bound, the one with the most room)
double bound_price(double p, double bytes) {
    const double memory = 2 + bytes / 4.6e6;
    return (p > memory ? p : memory) + .05 * p;
}
// At least what any plan for up to P positions takes: sums and counters.
int64_t sums_bytes(int64_t P, int64_t N, int64_t E) {
    const int64_t most = up_to(N, 128) / 128 * most_token_tiles(128, P, E) * kMostSplits * 65536;
    return (most < kMostSums ? most : kMostSums) + kMostShared * 16;
}
// Positions a group, on average, up to which they are few: the stream reads a weight again for every 16 of its group's. (us, stream -> tiles, int8, K = 5120, N = 1280: 32 of 64
// groups 43.1 -> 49.9; K = 512, N = 1000, 60 of 8 9.4 -> 10.4; fp16, K = 1376, N = 4096, 148 of 60 98.0 -> 98.6; K = 5120, N = 1280, 512 rows routed to 128 int8 142 -> 145, bf16 265 -> 266,
// 256 to 64 76 -> 82 and 140 -> 145.) And at most so many, since one group may have them all: 512 rows in one of 128 184 -> 27 and 308 -> 32, 256 in one of 64 94 -> 22.
constexpr int64_t kFewEach = 4, kMostFew = 512;
bool few_rows(int64_t P, int64_t E) { return P <= 16 || (P <= kFewEach * E && P <= kMostFew); }
// P positions, of E groups (0: one) of which the host knows no more.
Plan plan_product(int weight_type, int64_t K, int64_t N, int64_t P, int64_t E) {
    Plan plan = { few_rows(P, E), 0, -1, 0, 1, 0, 0, 0 };
    if (plan.few) return plan;
    const int64_t steps = up_to(K * type_bytes(weight_type), 64) / 64, groups = E == 0 ? 1 : P < E ? P : E;
    const double  each = (double) P / (double) groups, bytes = (double) groups * (double) (N * K * type_bytes(weight_type));
    auto row_tiles = [&](int f, int64_t rows) { return (rows + tiled_rows(f) - 1) / tiled_rows(f); };
    auto token_tiles = [&](int f) {   // (groups: expected)
        if (E == 0) return (double) most_token_tiles(tiled_tokens(f), P, 0);
        const double t = each / tiled_tokens(f) + .5;
        return (double) groups * (t > 1 ? t : 1);
    };
    double least = 0;
    for (int f = 0; f < kForms; ++f) {
        const double  tokens = token_tiles(f);
        const int64_t all = row_tiles(f, N);
        const double  p = bound_price(price(f, (double) all * tokens, steps, 1), bytes);
        if (f == 0 || p < least) least = p, plan = { false, f, -1, all, 1, 0, 0, 0 };
        if (shared_form(f)) {
            const int64_t tiles = all * most_token_tiles(tiled_tokens(f), P, E);
            for (int64_t parts = 2; parts <= kMostSplits && tiles <= kMostShared; ++parts) {
                const int64_t some = up_to((steps + parts - 1) / parts, 2), n = (steps + some - 1) / some, sums = tiles * n * tile_bytes(f);
                if (n < 2 || some < 8 || sums > kMostSums) break;
                const double q = bound_price(price(f, (double) all * tokens, some, n), bytes);
                if (q < least) least = q, plan = { false, f, -1, all, (int) n, (int) some, (int) tiles * 4, sums };
            }
        }
        // whole rounds of the chip in one form, the rows behind them, which would leave most of it idle for a round, in another
        const int64_t round = 256 * kForm[f].resident, rounds = E ? 0 : (int64_t) ((double) all * tokens) / round;
        for (int64_t k = rounds; k > 0 && k > rounds - 2; --k) {
            const int64_t n = k * round / (int64_t) tokens;   // row tiles
            if (n == 0 || n >= all) continue;
            for (int g = 0; g < kForms; ++g) {
                const double q = bound_price(price(f, (double) n * tokens, steps, 1) + 2.0 +
                                             price(g, (double) row_tiles(g, N - n * tiled_rows(f)) * token_tiles(g), steps, 1), bytes);
                if (q < least) least = q, plan = { false, f, g, n, 1, 0, 0, 0 };
            }
        }
    }
    return plan;
}
hipError_t launch_product(const Plan &p, int weight_type, const ProductArgs &a, hipStream_t stream) {
    if (p.few) return launch_stream(weight_type, RQ_I8, a, stream);
    ProductArgs one = a;
    one.splits = p.splits, one.split_steps = p.split_steps;
    one.first_block = 0, one.row_tiles = p.rest >= 0 ? (int) p.main_tiles : 0;
    const hipError_t e = launch_tiled(weight_type, p.form, one, stream);
    if (e != hipSuccess || p.rest < 0) return e;
    const int64_t done = p.main_tiles * tiled_rows(p.form);
    one.first_block = (int) (done / 32);
    one.row_tiles = (int) ((a.L.N - done + tiled_rows(p.rest) - 1) / tiled_rows(p.rest));
    return launch_tiled(weight_type, p.rest, one, stream);
}

// Sets a's rows of x as the call has them, if launch_stream rounds them itself.
bool stream_takes_floats(ProductArgs &a, int in_dtype, const void *x, int64_t ldx, int64_t M, int64_t K, int64_t E) {
    const int rows = stream_rounds(a.P, K, a.L.N, E);
    if (rows == 0) return false;
    a.x = (const uint8_t *) x, a.pitch = ldx, a.K = K, a.M = M, a.chunk = rows;
    a.aligned = aligned(x, 16) && K % 8 == 0 && (M == 1 || ldx * type_bytes(in_dtype) % 16 == 0);
    return true;
}

// Whether a call looks at no workspace, whatever the type of x and its alignment: few rows, taken as they lie or rounded where they are used.
bool alone(int weight_type, int64_t K, int64_t N, int64_t P, int64_t E) {
    return few_rows(P, E) && (weight_type != RQ_I8 || stream_rounds(P, K, N, E) > 0);
}

int run(ProductArgs &a, const Plan &plan, int weight_type, int64_t K, int in_dtype, const void *x, int64_t ldx, const float *x_scales, int64_t M,
        uint8_t *workspace, size_t workspace_bytes, hipStream_t stream) {
    const size_t rows = act_bytes(weight_type, K, M);
    if (!plan.few && workspace_bytes < rows + plan.sums_bytes + 4 * (size_t) plan.counters) return RQ_E_WORKSPACE;   // (a plan that sums_bytes does not cover)
    uint8_t *behind = workspace + rows;
    a.sums = (uint32_t *) behind;
    a.arrived = (int *) (behind + plan.sums_bytes);
    const hipError_t e = take_rows(a, weight_type, K, in_dtype, x, ldx, x_scales, M, plan.few, plan.counters, workspace, stream);
    return e != hipSuccess ? e : launch_product(plan, weight_type, a, stream);
}

}  // namespace

extern "C" size_t rq_i8_workspace_bytes(int64_t K, int64_t N, int64_t M) {
    if (rq_weight_prepared_bytes(RQ_I8, 1, N, K) == 0 || M < 0 || M > kMaxPositions) return 0;
    if (alone(RQ_I8, K, N, M, 0)) return 256;   // (not looked at)
    return act_bytes(RQ_I8, K, M) + pad256(sums_bytes(M, N, 0)) + 256;
}

extern "C" int rq_i8_mul_mat(const void *prepared, int64_t K, int64_t N, int in_dtype, const void *x, int64_t ldx, const float *x_scales,
                             int64_t M, int out_dtype, void *y, int64_t ldy, void *workspace, size_t workspace_bytes, rq_stream_t stream) {
    const size_t need = rq_i8_workspace_bytes(K, N, M);
    if (!(float_dtype(in_dtype) || in_dtype == RQ_I8) || !float_dtype(out_dtype) || need == 0) return RQ_E_UNSUPPORTED;
    if (M == 0) return 0;
    if (!prepared || !aligned(prepared, 256) || !x || !aligned(x, type_bytes(in_dtype)) || !y || !aligned(y, type_bytes(out_dtype)) ||
        (in_dtype == RQ_I8) != (x_scales != nullptr) || !aligned(x_scales, 4) || (M > 1 && (ldx < K || ldy < N))) {
        return RQ_E_ARGUMENT;
    }
    if (!alone(RQ_I8, K, N, M, 0) && (!workspace || !aligned(workspace, 256) || workspace_bytes < need)) return RQ_E_WORKSPACE;
    ProductArgs a = {};
    a.L = panels(RQ_I8, N, K);
    a.w = (const uint8_t *) prepared;
    a.P = a.y_rows = M;
    a.out_dtype = out_dtype;
    a.y = y;
    a.ldy = ldy;
    const hipStream_t st = (hipStream_t) stream;
    if (in_dtype != RQ_I8 && stream_takes_floats(a, in_dtype, x, ldx, M, K, 0)) return launch_stream(RQ_I8, in_dtype, a, st);
    const Plan plan = plan_product(RQ_I8, K, N, M, 0);
    return run(a, plan, RQ_I8, K, in_dtype, x, ldx, x_scales, M, (uint8_t *) workspace, workspace_bytes, st);
}

extern "C" size_t rq_grouped_workspace_bytes(int weight_type, int64_t E, int64_t K, int64_t N, int64_t M, int64_t P) {
    if (rq_weight_prepared_bytes(weight_type, E, N, K) == 0 || M < 0 || M > kMaxPositions || P < 0 || P > kMaxPositions) return 0;
    if (alone(weight_type, K, N, P, E)) return 256;
    return act_bytes(weight_type, K, M) + pad256(sums_bytes(P, N, E)) + 256;
}

extern "C" int rq_grouped_mul_mat(int weight_type, const void *prepared, int64_t E, int64_t K, int64_t N, int in_dtype, const void *x,
                                  int64_t ldx, const float *x_scales, int64_t M, const int32_t *offsets, int64_t P, const int32_t *rows,
                                  const int32_t *out_rows, int out_dtype, void *y, int64_t ldy, int64_t y_rows, void *workspace,
                                  size_t workspace_bytes, rq_stream_t stream) {
    const size_t need = rq_grouped_workspace_bytes(weight_type, E, K, N, M, P);
    const bool   fits = weight_type == RQ_I8 ? float_dtype(in_dtype) || in_dtype == RQ_I8 : in_dtype == weight_type;
    if (!fits || !float_dtype(out_dtype) || need == 0 || y_rows < 0 || y_rows > (1ll << 31) - 1) return RQ_E_UNSUPPORTED;
    if (P == 0 || y_rows == 0) return 0;
    if (!prepared || !aligned(prepared, 256) || M < 1 || !x || !aligned(x, type_bytes(in_dtype)) || !y || !aligned(y, type_bytes(out_dtype)) ||
        (in_dtype == RQ_I8) != (x_scales != nullptr) || !aligned(x_scales, 4) || !offsets || !aligned(offsets, 4) || !aligned(rows, 4) ||
        !aligned(out_rows, 4) || (M > 1 && ldx < K) || (y_rows > 1 && ldy < N)) {
        return RQ_E_ARGUMENT;
    }
    if (!alone(weight_type, K, N, P, E) && (!workspace || !aligned(workspace, 256) || workspace_bytes < need)) return RQ_E_WORKSPACE;
    ProductArgs a = {};
    a.L = panels(weight_type, N, K);
    a.w = (const uint8_t *) prepared;
    a.P = P;
    a.offsets = offsets;
    a.E = (int) E;
    a.rows = rows;
    a.out_rows = out_rows;
    a.out_dtype = out_dtype;
    a.y = y;
    a.ldy = ldy;
    a.y_rows = y_rows;
    const hipStream_t st = (hipStream_t) stream;
    if (weight_type == RQ_I8 && in_dtype != RQ_I8 && stream_takes_floats(a, in_dtype, x, ldx, M, K, E)) return launch_stream(RQ_I8, in_dtype, a, st);
    const Plan plan = plan_product(weight_type, K, N, P, E);
    return run(a, plan, weight_type, K, in_dtype, x, ldx, x_scales, M, (uint8_t *) workspace, workspace_bytes, st);
}

namespace {

void tell(const Plan &p, int rounds, int64_t plan[8]) {
    memset(plan, 0, 8 * sizeof(plan[0]));
    plan[0] = rounds ? RQ_I8_ROUNDS : p.few ? RQ_I8_STREAM : RQ_I8_TILES;
    plan[1] = rounds;
    if (plan[0] != RQ_I8_TILES) return;
    plan[1] = tiled_rows(p.form);
    plan[2] = tiled_tokens(p.form);
    plan[3] = p.main_tiles;
    if (p.rest >= 0) plan[4] = tiled_rows(p.rest), plan[5] = tiled_tokens(p.rest);
    plan[6] = p.splits;
    plan[7] = kForm[p.form].resident;
}

}  // namespace

extern "C" int rq_i8_product_plan(int64_t K, int64_t N, int in_dtype, int64_t M, int64_t plan[8]) {
    if (!plan) return RQ_E_ARGUMENT;
    if (!(float_dtype(in_dtype) || in_dtype == RQ_I8) || rq_i8_workspace_bytes(K, N, M) == 0 || M < 1) return RQ_E_UNSUPPORTED;
    tell(plan_product(RQ_I8, K, N, M, 0), in_dtype == RQ_I8 ? 0 : stream_rounds(M, K, N, 0), plan);
    return 0;
}

extern "C" int rq_grouped_plan(int weight_type, int64_t E, int64_t K, int64_t N, int in_dtype, int64_t M, int64_t P, int64_t plan[8]) {
    if (!plan) return RQ_E_ARGUMENT;
    const bool fits = weight_type == RQ_I8 ? float_dtype(in_dtype) || in_dtype == RQ_I8 : in_dtype == weight_type;
    if (!fits || rq_grouped_workspace_bytes(weight_type, E, K, N, M, P) == 0 || P < 1) return RQ_E_UNSUPPORTED;
    tell(plan_product(weight_type, K, N, P, E), weight_type != RQ_I8 || in_dtype == RQ_I8 ? 0 : stream_rounds(P, K, N, E), plan);
    return 0;
}
