// Entry points of the MXFP4 product, the routing and the experts' feed-forward: argument checks, workspaces, order of launches.
#include "rq_mx.h"

using namespace rq::mx;

namespace {

bool known_dtype(int dtype) { return dtype == RQ_F32 || dtype == RQ_F16 || dtype == RQ_BF16; }
bool aligned(const void *p, size_t n) { return (uintptr_t) p % n == 0; }
size_t dtype_bytes(int dtype) { return dtype == RQ_F32 ? 4 : 2; }
int64_t pad256(int64_t n) { return up_to(n, 256); }

constexpr int64_t kMaxTokens = 1 << 22;   // rows of a call; slots of an experts' call

// Most elements that every workgroup of a product quantises for itself.
constexpr int64_t kFusedElements = 24576;
// Most tokens whose experts' weights are streamed slot by slot, without sorting.
constexpr int64_t kExpertsDecodeTokens = 4;
// tokens up to which a product streams its weights (rq_mx_skinny.hip)
constexpr int kSkinnyTokens = 64;

struct ExpertsPlan {
    int     tile_tokens;   // 32, 64: skinny; 128: tiled
    bool    panels;        // activations in panel form: by position, as the tiled product reads them
    int64_t slots, positions, tiles;
    WeightLayout XP, HP;
    size_t  x, x_scales, h, h_scales, rows, token_of, slot_of, tile_table, n_tiles, total;   // offsets
};
ExpertsPlan experts_plan(int64_t E, int64_t K, int64_t F, int64_t N, int64_t M, int top) {
    ExpertsPlan p;
    p.slots = M * top;
    const double per = (double) p.slots / (double) E;   // of an expert, on average
    p.tile_tokens = per <= 16 ? 32 : per <= 40 || M <= kExpertsDecodeTokens ? 64 : 128;
    p.panels = p.tile_tokens > kSkinnyTokens;
    p.tiles = most_tiles(p.slots, E, p.tile_tokens);
    p.positions = most_positions(p.slots, E);
    p.XP = weight_layout(p.positions, K);
    p.HP = weight_layout(p.positions, F);
    const ActLayout X = act_layout(K), H = act_layout(F);
    size_t at = 0;
    auto take = [&](int64_t bytes) {
        const size_t here = at;
        at += (size_t) pad256(bytes);
        return here;
    };
    p.x = take(p.panels ? p.XP.expert_bytes : M * X.code_stride);
    p.x_scales = take(p.panels ? 0 : M * X.scale_stride);
    p.h = take(p.panels ? p.HP.expert_bytes : p.positions * H.code_stride);
    p.h_scales = take(p.panels ? 0 : p.positions * H.scale_stride);
    p.rows = take(p.slots * N * 4);
    p.token_of = take(p.positions * 4);
    p.slot_of = take(p.positions * 4);
    p.tile_table = take(p.tiles * (int64_t) sizeof(Tile));
    p.n_tiles = take(8);
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
    const ActLayout A = act_layout(K);
    return (size_t) (M > kSkinnyTokens ? weight_layout(M, K).expert_bytes : pad256(M * A.code_stride) + pad256(M * A.scale_stride)) + 256;
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
    if (!workspace || !aligned(workspace, 256) || workspace_bytes < need) return RQ_E_WORKSPACE;
    const hipStream_t st = (hipStream_t) stream;
    if (M <= 16) {
        DecodeArgs d = {};
        d.L = weight_layout(N, K);
        d.x = x;
        d.ldx = ldx;
        d.M = M;
        d.w = (const uint8_t *) prepared;
        d.out_dtype = out_dtype;
        d.y = y;
        d.ldy = ldy;
        if (!decode_takes(in_dtype, x, ldx, M, K, kFusedElements)) {
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
    a.A = act_layout(K);
    a.w = (const uint8_t *) prepared;
    uint8_t *codes = (uint8_t *) workspace, *scales = codes + pad256(M * a.A.code_stride);
    a.a_codes = codes;
    a.a_scales = scales;
    a.M = M;
    a.out_dtype = out_dtype;
    a.y = y;
    a.ldy = ldy;
    if (M <= kSkinnyTokens) {
        const hipError_t e = launch_act_quantize(in_dtype, x, ldx, M, K, codes, scales, st);
        return e != hipSuccess ? e : launch_skinny(kDense, a, M <= 32 ? 32 : 64, st);
    }
    a.P = weight_layout(M, K);
    const hipError_t e = launch_panel_quantize(in_dtype, x, ldx, a.P, nullptr, nullptr, codes, st);
    return e != hipSuccess ? e : launch_tiled(kDense, a, st);
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
    if (decode_takes(in_dtype, x, ldx, 1, K, 65536) && (M == 1 || (M <= kExpertsDecodeTokens && ldx * (int64_t) dtype_bytes(in_dtype) % 16 == 0))) {
        DecodeArgs g = {};
        g.L = weight_layout(F, K);
        g.w = (const uint8_t *) gate;
        g.w2 = (const uint8_t *) up;
        g.x = x;
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
    s.n_tiles = (int *) (ws + p.n_tiles);
    hipError_t e = launch_sort(s, st);
    if (e == hipSuccess) {
        e = p.panels ? launch_panel_quantize(in_dtype, x, ldx, p.XP, s.token_of, s.n_tiles + 1, ws + p.x, st)
                     : launch_act_quantize(in_dtype, x, ldx, M, K, ws + p.x, ws + p.x_scales, st);
    }
    ProductArgs a = {};
    a.L = weight_layout(F, K);
    a.A = act_layout(K);
    a.w = (const uint8_t *) gate;
    a.w2 = (const uint8_t *) up;
    a.a_codes = ws + p.x;
    a.a_scales = ws + p.x_scales;
    a.tiles = s.tiles;
    a.n_tiles = s.n_tiles;
    a.most_tiles = (int) p.tiles;
    a.row_of = s.token_of;
    a.h_codes = ws + p.h;
    a.h_scales = ws + p.h_scales;
    a.H = act_layout(F);
    a.P = p.XP;
    a.HP = p.HP;
    if (e == hipSuccess) e = p.panels ? launch_tiled(kGateUp, a, st) : launch_skinny(kGateUp, a, p.tile_tokens, st);
    ProductArgs d = a;
    d.L = weight_layout(N, F);
    d.A = a.H;
    d.P = p.HP;
    d.w = (const uint8_t *) down;
    d.a_codes = a.h_codes;
    d.a_scales = a.h_scales;
    d.row_of = s.slot_of;
    d.y = ws + p.rows;
    d.ldy = N;
    if (e == hipSuccess) e = p.panels ? launch_tiled(kDown, d, st) : launch_skinny(kDown, d, p.tile_tokens, st);
    if (e == hipSuccess) e = launch_combine((const float *) (ws + p.rows), N, ids, weights, M, top, (int) E, out_dtype, y, ldy, st);
    return e;
}
