// Entry points of the int8 product and of the products grouped by expert: argument checks, workspaces, order of launches.
#include "rq_prod.h"

using namespace rq::prod;

namespace {

bool   float_dtype(int dtype) { return dtype == RQ_F32 || dtype == RQ_F16 || dtype == RQ_BF16; }
bool   aligned(const void *p, size_t n) { return (uintptr_t) p % n == 0; }
size_t pad256(int64_t n) { return (size_t) up_to(n, 256); }

constexpr int64_t kMaxPositions = 1 << 22;   // rows of a call

// Rows of x as the kernels read them: in the workspace (rounded, or brought to multiples of 16 bytes), or where they are.
int64_t packed_pitch(int weight_type, int64_t K) { return up_to(K * type_bytes(weight_type), 64); }
size_t  act_bytes(int weight_type, int64_t K, int64_t M) { return pad256(M * packed_pitch(weight_type, K)) + pad256(M * 4); }

// Sets a's rows of x; launches what brings them there.
hipError_t take_rows(ProductArgs &a, int weight_type, int64_t K, int in_dtype, const void *x, int64_t ldx, const float *x_scales, int64_t M,
                     uint8_t *workspace, hipStream_t stream) {
    a.M = M;
    const int64_t row_bytes = K * type_bytes(weight_type), pitch = packed_pitch(weight_type, K);
    if (weight_type == RQ_I8 && in_dtype != RQ_I8) {
        float *scales = reinterpret_cast<float *>(workspace + pad256(M * pitch));
        a.x = workspace, a.pitch = a.x_bytes = pitch, a.x_scales = scales;
        return launch_i8_quantize(in_dtype, x, ldx, M, K, workspace, pitch, pitch, scales, stream);
    }
    a.x_scales = x_scales;
    const int64_t ld_bytes = ldx * type_bytes(in_dtype);
    if (aligned(x, 16) && (M == 1 || ld_bytes % 16 == 0) && row_bytes % 16 == 0) {
        a.x = (const uint8_t *) x, a.pitch = ld_bytes, a.x_bytes = row_bytes;
        return hipSuccess;
    }
    a.x = workspace, a.pitch = a.x_bytes = pitch;
    return launch_pack(x, ld_bytes, M, row_bytes, workspace, pitch, stream);
}

}  // namespace

extern "C" size_t rq_i8_workspace_bytes(int64_t K, int64_t N, int64_t M) {
    if (rq_weight_prepared_bytes(RQ_I8, 1, N, K) == 0 || M < 0 || M > kMaxPositions) return 0;
    return act_bytes(RQ_I8, K, M) + 256;
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
    if (!workspace || !aligned(workspace, 256) || workspace_bytes < need) return RQ_E_WORKSPACE;
    ProductArgs a = {};
    a.L = panels(RQ_I8, N, K);
    a.w = (const uint8_t *) prepared;
    a.P = a.y_rows = M;
    a.out_dtype = out_dtype;
    a.y = y;
    a.ldy = ldy;
    const hipStream_t st = (hipStream_t) stream;
    const hipError_t  e = take_rows(a, RQ_I8, K, in_dtype, x, ldx, x_scales, M, (uint8_t *) workspace, st);
    if (e != hipSuccess) return e;
    if (M <= 16) return launch_stream(RQ_I8, a, st);
    return launch_tiled(RQ_I8, M <= 64 ? 0 : M <= 256 ? 2 : 3, a, st);
}

extern "C" size_t rq_grouped_workspace_bytes(int weight_type, int64_t E, int64_t K, int64_t N, int64_t M, int64_t P) {
    if (rq_weight_prepared_bytes(weight_type, E, N, K) == 0 || M < 0 || M > kMaxPositions || P < 0 || P > kMaxPositions) return 0;
    return act_bytes(weight_type, K, M) + 256;
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
    if (!workspace || !aligned(workspace, 256) || workspace_bytes < need) return RQ_E_WORKSPACE;
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
    const hipError_t  e = take_rows(a, weight_type, K, in_dtype, x, ldx, x_scales, M, (uint8_t *) workspace, st);
    if (e != hipSuccess) return e;
    if (P <= 8 * E) return launch_stream(weight_type, a, st);
    return launch_tiled(weight_type, P <= 48 * E ? 1 : 2, a, st);
}
