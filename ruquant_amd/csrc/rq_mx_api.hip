// Entry points of the MXFP4 product, the routing and the experts' feed-forward: argument checks, workspaces, order of launches.
#include <string.h>

#include "../../include/rq_mx4_plan.h"
#include "rq_mx.h"

using namespace rq::mx;

namespace {

bool known_dtype(int dtype) { return dtype == RQ_F32 || dtype == RQ_F16 || dtype == RQ_BF16; }
bool aligned(const void *p, size_t n) { return (uintptr_t) p % n == 0; }
bool rows_aligned(const void *x, int64_t ld, int64_t M, int dtype) {
    return aligned(x, 16) && (M == 1 || ld * (dtype == RQ_F32 ? 4 : 2) % 16 == 0);
}
size_t dtype_bytes(int dtype) { return dtype == RQ_F32 ? 4 : 2; }
int64_t pad256(int64_t n) { return up_to(n, 256); }

constexpr int64_t kMaxTokens = 1 << 22;   // rows of a call; slots of an experts' call

// Whether the experts' weights are streamed slot by slot (rq_mx_decode.hip) or the slots are sorted and go in tiles: the first reads a weight again
// for every slot that has it, the second has three launches more. Prices in us by the bytes of an expert's three weights and how many experts the
// tokens can be expected to hit, from 14 sizes of K = 1024 to 5120, F = 256 to 4096, 8 to 256 experts, 1 to 32 a token, 1 to 24 tokens: the one that they
// choose is at worst 2 % slower than the other, and 4 % over nine more sizes (K = 768 to 6144, F = 192 to 17408, 4 to 512 experts). (us, slot by slot -> tiles, K x F, experts: 5120 x 1280: 8 of 64 1 token 24.3 -> 36.4, 6 tokens
// 83 -> 91, 8 105 -> 104, 12 152 -> 126; 8 of 8 2 tokens 31 -> 37, 4 48 -> 37; 32 of 64 4 tokens 200 -> 145; 2048 x 512: 8 of 256 16 tokens 46 -> 61, 8 of 8
// 8 tokens 19 -> 25, 16 31 -> 25; 4096 x 4096, 2 of 8: 4 tokens 43 -> 47, 8 68 -> 52; 1024 x 256, 4 of 32: 24 tokens 17 -> 23.)
constexpr int64_t kExpertsDecodeTokens = 24;   // (as far as was measured)
bool experts_decode(int64_t E, int64_t K, int64_t F, int64_t N, int64_t M, int top) {
    if (M > kExpertsDecodeTokens || K > 65536) return false;   // (K: a token in LDS)
    const double mb = (double) F * (2 * K + N) * 17 / 32 * 1e-6, share = top < E ? (double) top / (double) E : 1.0;
    double       missed = 1;
    for (int64_t m = 0; m < M; ++m) missed *= 1 - share;
    const double hit = (double) E * (1 - missed), again = (double) (M * top) - hit;
    const double first = mb / 5.6 > .06 ? mb / 5.6 : .06, more = mb / 10 > .06 ? mb / 10 : .06;   // of a slot: its weight from memory, and from a cache
    return 8 + hit * first + again * more + (double) (M * K) / 17000 <= 20 + hit * mb / 5;
}
// Products whose weights go from memory into registers (rq_mx_decode.hip): up to 16 tokens, fewer where the sizes make each more costly than
// the tiles' start. (us, here -> in tiles, at the fewest tokens that go to those: K = 17408: N = 64 9 tokens 11.6 -> 11.0, N = 5120 4 tokens
// 17.8 -> 16.6, N = 17408 2 tokens 29.2 -> 28.6; K = 8992, N = 5120 8 tokens 12.5 -> 12.7; K = 5120: N = 5120 14 tokens 10.5 -> 10.7, N = 9000
// 10 tokens 11.1 -> 10.8, N = 17408 6 tokens 14.9 -> 14.8; K = 1024, N = 17408: here up to 16 tokens, 7.8 -> 8.1)
bool few_tokens(int64_t M, int64_t K, int64_t N) { return M <= 16 && M * K * (N + 4096) <= 614400000; }
// ... and that each workgroup rounds for itself, so that no workspace is looked at
bool alone(int64_t M, int64_t K, int64_t N) { return few_tokens(M, K, N) && decode_takes(M, K, N); }

struct ExpertsPlan {
    bool    decode;               // slot by slot (rq_mx_decode.hip); otherwise sorted by expert and tiled
    int     tile_tokens;          // of both products
    int     form;                 // of the tiles of both
    int64_t slots, positions, tiles;
    WeightLayout XP, HP;
    size_t  x, h, h_scales, rows, token_of, slot_of, tile_table, used, total;   // offsets
};
ExpertsPlan experts_plan(int64_t E, int64_t K, int64_t F, int64_t N, int64_t M, int top) {
    ExpertsPlan p = {};
    p.slots = M * top;
    size_t at = 0;
    auto take = [&](int64_t bytes) {
        const size_t here = at;
        at += (size_t) pad256(bytes);
        return here;
    };
    p.decode = experts_decode(E, K, F, N, M, top);
    if (p.decode) {
        p.h = take(p.slots * (up_to(F, 256) / 2));
        p.h_scales = take(p.slots * (up_to(F, 256) / 32));
        p.total = at;
        return p;
    }
    // Tiles of 64 tokens up to 96 slots an expert; of 128 above, 256 rows of weights each where those are enough to keep the chip busy.
    // (us for the whole call, 64 -> 128 tokens x 128 rows -> 128 x 256, by experts x slots an expert: 5120 x 1280 64 x 62: 213 -> 216 -> 230,
    // 64 x 125: 292 -> 295 -> 275, 64 x 256: 511 -> 491 -> 444, 8 x 125: 54 -> 59 -> 65, 8 x 512: 128 -> 107 -> 111; 2048 x 512 60 x 136: 84 ->
    // 88 -> 80, 64 x 256: 146 -> 134 -> 131; 4096 x 4096 8 x 250: 130 -> 113 -> 126, 8 x 1000: 413 -> 340 -> 327. At worst 11 % behind the fastest.)
    const int64_t token_tiles = p.slots / 128 + ((p.slots < E ? p.slots : E) + 1) / 2;
    p.form = p.slots <= 96 * E ? kForm64 : tiled_row_tiles(kGateUp, kForm256, F) * token_tiles >= 768 ? kForm256 : kForm128;
    p.tile_tokens = tiled_tokens(p.form);
    p.tiles = most_tiles(p.slots, E, p.tile_tokens);
    p.positions = most_positions(p.slots, E);
    p.XP = weight_layout(p.positions, K);
    p.HP = weight_layout(p.positions, F);
    p.x = take(p.XP.expert_bytes);
    p.h = take(p.HP.expert_bytes);
    p.rows = take(p.slots * N * 4);   // (fp32: what a token's slots cancel is not lost)
    p.token_of = take(p.positions * 4);
    p.slot_of = take(p.positions * 4);
    p.tile_table = take(most_tiles(p.slots, E, tiled_tokens(kForm64)) * (int64_t) sizeof(Tile));   // (room for the smallest, so that it grows with M)
    p.used = take(4);
    p.total = at;
    return p;
}
bool good_experts(int64_t E, int64_t K, int64_t F, int64_t N, int64_t M, int top) {
    return E >= 1 && E <= RQ_ROUTE_MAX_E && top >= 1 && top <= RQ_ROUTE_MAX_TOP && M >= 0 && M * top <= kMaxTokens &&
           rq_mx4_prepared_bytes(E, F, K) != 0 && rq_mx4_prepared_bytes(E, N, F) != 0;
}

}  // namespace

extern "C" size_t rq_mx4_workspace_bytes(int64_t K, int64_t N, int64_t M) {
    if (rq_mx4_prepared_bytes(1, N, K) == 0 || M < 0 || M > kMaxTokens) return 0;
    if (alone(M, K, N)) return 256;   // (not looked at)
    const ActLayout A = act_layout(K);
    if (few_tokens(M, K, N)) return (size_t) (pad256(M * A.code_stride) + pad256(M * A.scale_stride)) + 256;
    return (size_t) (pad256(weight_layout(M, K).expert_bytes) + pad256(product_sums_bytes(M, N, K))) + 256;
}

extern "C" int rq_mx4_mul_mat(const void *prepared, int64_t K, int64_t N, int in_dtype, const void *x, int64_t ldx, int64_t M,
                              int out_dtype, void *y, int64_t ldy, void *workspace, size_t workspace_bytes, rq_stream_t stream) {
    const size_t need = rq_mx4_workspace_bytes(K, N, M);
    if (!known_dtype(in_dtype) || !known_dtype(out_dtype) || need == 0) return RQ_E_UNSUPPORTED;
    if (M == 0) return 0;
    if (!prepared || !aligned(prepared, 256) || !x || !aligned(x, dtype_bytes(in_dtype)) || !y || !aligned(y, dtype_bytes(out_dtype)) ||
        (M > 1 && (ldx < K || ldy < N))) {
        return RQ_E_ARGUMENT;
    }
    if (!alone(M, K, N) && (!workspace || !aligned(workspace, 256) || workspace_bytes < need)) return RQ_E_WORKSPACE;
    const hipStream_t st = (hipStream_t) stream;
    if (few_tokens(M, K, N)) {
        DecodeArgs d = {};
        d.L = weight_layout(N, K);
        d.x = x;
        d.aligned = rows_aligned(x, ldx, M, in_dtype);
        d.ldx = ldx;
        d.M = M;
        d.w = (const uint8_t *) prepared;
        d.out_dtype = out_dtype;
        d.y = y;
        d.ldy = ldy;
        if (!alone(M, K, N)) {
            d.A = act_layout(K);
            uint8_t *codes = (uint8_t *) workspace, *scales = codes + pad256(M * d.A.code_stride);
            d.a_codes = codes;
            d.a_scales = scales;
            const hipError_t e = launch_act_quantize(in_dtype, x, ldx, M, K, codes, scales, st);
            if (e != hipSuccess) return e;
        }
        return launch_decode(in_dtype, d, st);
    }
    ProductArgs a = {};
    a.L = weight_layout(N, K);
    a.w = (const uint8_t *) prepared;
    a.panels = (uint8_t *) workspace;
    a.M = M;
    a.out_dtype = out_dtype;
    a.y = y;
    a.ldy = ldy;
    a.P = weight_layout(M, K);
    const ProductPlan plan = plan_product(M, N, K);
    uint8_t          *sums = (uint8_t *) workspace + pad256(a.P.expert_bytes);
    a.sums = (float *) sums;
    a.arrived = (int *) (sums + plan.sums_bytes);
    const hipError_t e = launch_panel_quantize(in_dtype, x, ldx, a.P, nullptr, nullptr, (uint8_t *) workspace, a.arrived, plan.arrived, st);
    return e != hipSuccess ? e : launch_tiled_product(plan, a, st);
}

extern "C" int rq_route(int dtype, const void *logits, int64_t ldl, int64_t M, int64_t E, int scoring, const float *bias, int groups,
                        int top_groups, int top, int renormalize, float scale, int32_t *ids, float *weights, rq_stream_t stream) {
    if (!known_dtype(dtype) || E < 1 || E > RQ_ROUTE_MAX_E || top < 1 || top > RQ_ROUTE_MAX_TOP || M < 0 || M > (1ll << 31) ||
        (scoring != 0 && scoring != 1) || groups < 1 || groups > 64 || E % groups || top_groups < 1 || top_groups > groups ||
        top > top_groups * (E / groups)) {
        return RQ_E_UNSUPPORTED;
    }
    if (M == 0) return 0;
    if (!logits || !aligned(logits, dtype_bytes(dtype)) || (M > 1 && ldl < E) || !ids || !weights || !aligned(ids, 4) ||
        !aligned(weights, 4) || !aligned(bias, 4)) {
        return RQ_E_ARGUMENT;
    }
    const RouteArgs a = { dtype, logits, ldl, M, (int) E, scoring, groups, top_groups, top, renormalize, bias, scale, ids, weights };
    return launch_route(a, (hipStream_t) stream);
}

extern "C" size_t rq_mx4_experts_workspace_bytes(int64_t E, int64_t K, int64_t F, int64_t N, int64_t M, int top) {
    if (!good_experts(E, K, F, N, M, top)) return 0;
    return experts_plan(E, K, F, N, M, top).total + 256;
}

extern "C" int rq_mx4_experts(const void *gate, const void *up, const void *down, int64_t E, int64_t K, int64_t F, int64_t N,
                              int in_dtype, const void *x, int64_t ldx, int64_t M, const int32_t *ids, const float *weights, int top,
                              int out_dtype, void *y, int64_t ldy, void *workspace, size_t workspace_bytes, rq_stream_t stream) {
    if (!known_dtype(in_dtype) || !known_dtype(out_dtype) || !good_experts(E, K, F, N, M, top)) return RQ_E_UNSUPPORTED;
    if (M == 0) return 0;
    if (!gate || !up || !down || !aligned(gate, 256) || !aligned(up, 256) || !aligned(down, 256) || !x ||
        !aligned(x, dtype_bytes(in_dtype)) || !y || !aligned(y, dtype_bytes(out_dtype)) || !ids || !weights || !aligned(ids, 4) ||
        !aligned(weights, 4) || (M > 1 && (ldx < K || ldy < N))) {
        return RQ_E_ARGUMENT;
    }
    const ExpertsPlan p = experts_plan(E, K, F, N, M, top);
    if (!workspace || !aligned(workspace, 256) || workspace_bytes < p.total) return RQ_E_WORKSPACE;
    const hipStream_t st = (hipStream_t) stream;
    uint8_t *ws = (uint8_t *) workspace;
    if (p.decode) {
        DecodeArgs g = {};
        g.L = weight_layout(F, K);
        g.w = (const uint8_t *) gate;
        g.w2 = (const uint8_t *) up;
        g.x = x;
        g.aligned = rows_aligned(x, ldx, M, in_dtype);
        g.ldx = ldx;
        g.M = M;
        g.ids = ids;
        g.weights = weights;
        g.top = top;
        g.E = (int) E;
        g.h_stride = up_to(F, 256) / 2;
        g.h_codes = ws + p.h;
        g.h_scales = ws + p.h_scales;
        g.out_dtype = out_dtype;
        g.y = y;
        g.ldy = ldy;
        DecodeArgs d = g;
        d.L = weight_layout(N, F);
        d.w = (const uint8_t *) down;
        return launch_decode_experts(in_dtype, g, d, st);
    }
    SortArgs s;
    s.ids = ids;
    s.slots = (int) p.slots;
    s.top = top;
    s.E = (int) E;
    s.tile_tokens = p.tile_tokens;
    s.positions = (int) p.positions;
    s.token_of = (int *) (ws + p.token_of);
    s.slot_of = (int *) (ws + p.slot_of);
    s.tiles = (Tile *) (ws + p.tile_table);
    s.most_tiles = (int) p.tiles;
    s.used = (int *) (ws + p.used);
    hipError_t e = launch_sort(s, st);
    if (e == hipSuccess) e = launch_panel_quantize(in_dtype, x, ldx, p.XP, s.token_of, s.used, ws + p.x, nullptr, 0, st);
    ProductArgs a = {};
    a.L = weight_layout(F, K);
    a.w = (const uint8_t *) gate;
    a.w2 = (const uint8_t *) up;
    a.panels = ws + p.x;
    a.P = p.XP;
    a.tiles = s.tiles;
    a.most_tiles = (int) p.tiles;
    a.h = ws + p.h;
    a.HP = p.HP;
    if (e == hipSuccess) e = launch_tiled(kGateUp, p.form, a, st);
    ProductArgs d = a;
    d.L = weight_layout(N, F);
    d.w = (const uint8_t *) down;
    d.panels = a.h;
    d.P = p.HP;
    d.row_of = s.slot_of;
    d.y = ws + p.rows;
    d.ldy = N;
    if (e == hipSuccess) e = launch_tiled(kDown, p.form, d, st);
    if (e == hipSuccess) e = launch_combine((const float *) (ws + p.rows), N, ids, weights, M, top, (int) E, out_dtype, y, ldy, st);
    return e;
}

extern "C" int rq_mx4_product_plan(int64_t K, int64_t N, int64_t M, int64_t plan[8]) {
    if (!plan) return RQ_E_ARGUMENT;
    if (rq_mx4_workspace_bytes(K, N, M) == 0 || M < 1) return RQ_E_UNSUPPORTED;
    memset(plan, 0, 8 * sizeof(plan[0]));
    plan[0] = alone(M, K, N) ? RQ_MX4_ALONE : few_tokens(M, K, N) ? RQ_MX4_ROWS : RQ_MX4_TILES;
    if (plan[0] != RQ_MX4_TILES) return 0;
    const ProductPlan p = plan_product(M, N, K);
    plan[1] = tiled_rows(p.form);
    plan[2] = tiled_tokens(p.form);
    plan[3] = p.main_tiles;
    if (p.rest >= 0) plan[4] = tiled_rows(p.rest), plan[5] = tiled_tokens(p.rest);
    plan[6] = p.splits;
    plan[7] = tiled_resident(p.form);
    return 0;
}

extern "C" int rq_mx4_experts_plan(int64_t E, int64_t K, int64_t F, int64_t N, int64_t M, int top, int64_t plan[3]) {
    if (!plan) return RQ_E_ARGUMENT;
    if (!good_experts(E, K, F, N, M, top) || M < 1) return RQ_E_UNSUPPORTED;
    const ExpertsPlan p = experts_plan(E, K, F, N, M, top);
    plan[0] = p.decode ? RQ_MX4_ALONE : RQ_MX4_TILES;
    plan[1] = p.decode ? 0 : tiled_rows(p.form);
    plan[2] = p.decode ? 0 : p.tile_tokens;
    return 0;
}
