/*
 * C ABI of the MXFP4 operators (microscaled 4-bit floating point), the routing to experts and the experts' feed-forward
 * on MI355X (gfx950). Exported by the same library as rq_w4a4.h, with the same conventions: plain pointers and sizes, device
 * pointers are memory of the current HIP device, `stream` is a hipStream_t passed as void*, calls are asynchronous on it,
 * allocate nothing, synchronize nothing and can be captured in a graph. Return values: 0 = success; > 0 = a hipError_t;
 * < 0 = one of the RQ_E_* codes of rq_w4a4.h. These operators have no counterpart in the reference.
 *
 * MXFP4: 32 consecutive elements of a row share one scale. An element is e2m1 (sign, two exponent bits, one mantissa bit:
 * 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two per byte, the even element in the low half. A scale is a byte X that
 * stands for 2^(X - 127), or for NaN when it is 255. A tensor of R rows and K inputs (K a multiple of 32) is R x K/2 bytes of
 * codes and R x K/32 bytes of scales, rows contiguous.
 */
#ifndef RQ_MX4_H
#define RQ_MX4_H

#include "rq_w4a4.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types of activations and outputs */
#define RQ_F32  0
#define RQ_F16  1
#define RQ_BF16 2

#define RQ_MX4_BLOCK     32         /* elements per scale */
#define RQ_MX4_MAX_K     (1 << 20)  /* longest row of a product */
#define RQ_ROUTE_MAX_E   1024       /* most experts of a routing call */
#define RQ_ROUTE_MAX_TOP 32         /* most experts per token */

/* x (M rows of K elements, row stride ldx elements, any alignment of its type) -> codes (4-byte aligned) and scales. A block's X is the exponent of its largest magnitude
 * less 2 (at least 0), so that the largest element lies in [4, 8) units; elements are rounded to the nearest, ties to the even
 * code, and saturate at 6. A block with an infinity or a NaN gets the scale 255 and zero codes. */
int rq_mx4_quantize(int dtype, const void *x_dev, int64_t ldx, int64_t M, int64_t K, void *codes_dev, void *scales_dev,
                    rq_stream_t stream);

/* codes (4-byte aligned) and scales -> out (M rows of K elements, row stride ldo elements, any alignment of its type), rounded once to dtype. */
int rq_mx4_dequantize(int dtype, const void *codes_dev, const void *scales_dev, int64_t M, int64_t K, void *out_dev, int64_t ldo,
                      rq_stream_t stream);

/* The form in which the product reads a weight of N rows, or E weights of N rows each, one behind the other (E = 1: a single
 * one): rewritten once, at first use. codes / scales / prepared 256-byte aligned. 0 bytes: not a shape that the product takes. */
size_t rq_mx4_prepared_bytes(int64_t E, int64_t N, int64_t K);
int rq_mx4_prepare(const void *codes_dev, const void *scales_dev, int64_t E, int64_t N, int64_t K, void *prepared_dev,
                   size_t prepared_bytes, rq_stream_t stream);

/* y[m][n] = sum_k x^[m][k] w[n][k], x^ the activations after rq_mx4_quantize's rounding, sums in fp32, rounded once to out_dtype.
 * x: M rows, stride ldx elements, any alignment of its type; y: row stride ldy elements, no memory of x. workspace: 256-byte aligned,
 * rq_mx4_workspace_bytes, need not be initialised, not shared by calls that can overlap; where that is 256 (a few tokens, which
 * the product quantises as it reads them) it is not looked at and may be null. It grows with M: the most tokens' serves all. */
size_t rq_mx4_workspace_bytes(int64_t K, int64_t N, int64_t M);
int rq_mx4_mul_mat(const void *prepared_dev, int64_t K, int64_t N, int in_dtype, const void *x_dev, int64_t ldx, int64_t M,
                   int out_dtype, void *y_dev, int64_t ldy, void *workspace_dev, size_t workspace_bytes, rq_stream_t stream);

/* Each of M tokens chooses `top` of E experts by their logits (row stride ldl). The scores s are softmax(logits) (scoring 0; its sum
 * is held in 64 bits) or sigmoid(logits) (scoring 1); the choice goes by c = s + bias (bias may be null). With groups > 1 the
 * experts are `groups` runs of E / groups; only those of the top_groups groups whose two largest c have the largest sums can be
 * chosen. ids[m][j]: the experts with the largest c, in falling order, ties to the lowest index; weights[m][j] = s of the chosen
 * ones (without bias), divided by their sum (in 64 bits) if renormalize (0 where that is 0), times scale. A NaN logit scores 0 whatever its bias, and
 * is chosen behind every number, as an expert is whose bias is NaN or minus infinity; a group that holds a number is in front of one that
 * holds only such experts. */
int rq_route(int dtype, const void *logits_dev, int64_t ldl, int64_t M, int64_t E, int scoring, const float *bias_dev, int groups,
             int top_groups, int top, int renormalize, float scale, int32_t *ids_dev, float *weights_dev, rq_stream_t stream);

/* The experts' gated feed-forward: y[m] = sum_j weights[m][j] D_e h^, h = silu(G_e x^) * (U_e x^), e = ids[m][j], ^ the rounding of
 * rq_mx4_quantize, sums in fp32. gate, up: E prepared weights of F rows and K inputs; down: E of N rows and F inputs. ids and
 * weights: M x top, contiguous; an id outside 0 .. E - 1 adds nothing (its weight is not looked at).
 * y shares no memory with the inputs. The workspace's bytes serve every out_dtype and grow with M. */
size_t rq_mx4_experts_workspace_bytes(int64_t E, int64_t K, int64_t F, int64_t N, int64_t M, int top);
int rq_mx4_experts(const void *gate_dev, const void *up_dev, const void *down_dev, int64_t E, int64_t K, int64_t F, int64_t N,
                   int in_dtype, const void *x_dev, int64_t ldx, int64_t M, const int32_t *ids_dev, const float *weights_dev,
                   int top, int out_dtype, void *y_dev, int64_t ldy, void *workspace_dev, size_t workspace_bytes,
                   rq_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif
