/*
 * C ABI of the products in 8-bit integers, of the products grouped by expert (weights in int8, fp16 or bf16) and of the sort that
 * makes such groups, on MI355X (gfx950). Exported by the same library as rq_w4a4.h and rq_mx4.h, with the same conventions: plain pointers and
 * sizes, device pointers are memory of the current HIP device, `stream` is a hipStream_t passed as void*, calls are asynchronous on
 * it, allocate nothing, synchronize nothing and can be captured in a graph. Return values: 0 = success; > 0 = a hipError_t;
 * < 0 = one of the RQ_E_* codes of rq_w4a4.h; nothing is launched then. These operators have no counterpart in the reference.
 *
 * int8 rows: a row of K numbers is K codes and one fp32 scale s; a code c stands for c s. Rounding a row x: s = max |x| times the
 * fp32 number nearest to 1 / 127, in fp32, at least 2^-126; r = 1 / s in fp32; code = the whole number nearest to x r (the exact product), ties to
 * even, so -127 .. 127.
 * A row that holds an infinity or a NaN has a NaN scale and zero codes. Tensors hold codes row by row and scales by row.
 */
#ifndef RQ_I8_H
#define RQ_I8_H

#include "rq_mx4.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types, beside RQ_F32, RQ_F16 and RQ_BF16 of rq_mx4.h */
#define RQ_I8 3

#define RQ_I8_MAX_K      131071     /* longest row of a product: 2^14 of any two codes, so often, stay below 2^31 */
#define RQ_GROUPED_MAX_E 1024       /* most groups of a call */

/* x (M rows of K elements, row stride ldx elements, any alignment of its type; K up to 2^30) -> codes (M x K) and scales (M). */
int rq_i8_quantize(int dtype, const void *x_dev, int64_t ldx, int64_t M, int64_t K, void *codes_dev, float *scales_dev, rq_stream_t stream);

/* codes (M x K) and scales (M) -> out (row stride ldo elements, any alignment of its type): the fp32 products, rounded to dtype. */
int rq_i8_dequantize(int dtype, const void *codes_dev, const float *scales_dev, int64_t M, int64_t K, void *out_dev, int64_t ldo,
                     rq_stream_t stream);

/* The form in which the products read a weight of N rows, or E weights of N rows each, one behind the other: rewritten once, at first
 * use. type: RQ_I8 (codes, E x N scales) or RQ_F16, RQ_BF16 (elements; scales null). Any alignment of the type; prepared 256-byte aligned.
 * 0 bytes: not a shape that the products take. */
size_t rq_weight_prepared_bytes(int type, int64_t E, int64_t N, int64_t K);
int rq_weight_prepare(int type, const void *w_dev, const float *scales_dev, int64_t E, int64_t N, int64_t K, void *prepared_dev,
                      size_t prepared_bytes, rq_stream_t stream);

/* y[m][n] = s_m t_n sum_k a[m][k] w[n][k]: a and s the rows of x as rq_i8_quantize rounds them, w and t the weight's codes and scales. The
 * sum is exact; y = ((fp32 of it) t_n) s_m, each product in fp32, rounded to out_dtype. in_dtype RQ_I8: x holds codes already and
 * x_scales their scales (else null). x: row stride ldx elements, any alignment of its type; y: row stride ldy elements, no memory of x.
 * workspace: 256-byte aligned, rq_i8_workspace_bytes (for every type and alignment; it grows with M, so the most tokens' serves all), need not be
 * initialised, not shared by calls that can overlap; where that is 256 (few rows) it is not looked at and may be null. */
size_t rq_i8_workspace_bytes(int64_t K, int64_t N, int64_t M);
int rq_i8_mul_mat(const void *prepared_dev, int64_t K, int64_t N, int in_dtype, const void *x_dev, int64_t ldx, const float *x_scales_dev,
                  int64_t M, int out_dtype, void *y_dev, int64_t ldy, void *workspace_dev, size_t workspace_bytes, rq_stream_t stream);

/* Sorts slots by expert: ids (M x top, contiguous) -> offsets (E + 1), slots and tokens (M x top each). Slot i = m top + j has expert ids[i];
 * slots[p] is the p-th slot in the order of the experts, those of one expert in rising order, and tokens[p] = slots[p] / top. Expert e's are
 * offsets[e] .. offsets[e + 1] - 1; slots with an id outside 0 .. E - 1 stand behind offsets[E], in rising order too. Workspace: 256-byte aligned,
 * as above (null where its bytes are 0). */
size_t rq_sort_workspace_bytes(int64_t M, int top, int64_t E);
int rq_sort_slots(const int32_t *ids_dev, int64_t M, int top, int64_t E, int32_t *offsets_dev, int32_t *slots_dev, int32_t *tokens_dev,
                  void *workspace_dev, size_t workspace_bytes, rq_stream_t stream);

/* Products grouped by expert: of P positions in a row, those from offsets[e] up to offsets[e + 1] are multiplied by weight e of E.
 *   y[q(p)] = W_e x[r(p)],  r(p) = rows[p], or p where rows is null; q(p) = out_rows[p], or p where out_rows is null.
 * weight_type RQ_I8: x rounded and products scaled as by rq_i8_mul_mat, x of any float type or given as codes (in_dtype RQ_I8 with x_scales,
 * one for each of the M rows of x). RQ_F16, RQ_BF16: x of the weight's type; sums in fp32, rounded once to out_dtype.
 * x has M rows (one at least where there are positions), y y_rows. Offsets are any numbers and are clamped to 0 .. P; a group whose end is not behind its start is empty, and groups
 * do not overlap (a row of y that several would write holds one group's product or another's, or is left as it was). An index of rows
 * outside 0 .. M - 1 gives a row of zeros; one of out_rows outside 0 .. y_rows - 1 is not written, and no index of out_rows comes twice. Rows
 * of y that no position writes are left as they were. Sizes that the device alone knows (the groups') shape no launch. y shares no memory with the
 * inputs. Workspace as above: rq_grouped_workspace_bytes serves every type and alignment of x and grows with M and P. */
size_t rq_grouped_workspace_bytes(int weight_type, int64_t E, int64_t K, int64_t N, int64_t M, int64_t P);
int rq_grouped_mul_mat(int weight_type, const void *prepared_dev, int64_t E, int64_t K, int64_t N, int in_dtype, const void *x_dev,
                       int64_t ldx, const float *x_scales_dev, int64_t M, const int32_t *offsets_dev, int64_t P, const int32_t *rows_dev,
                       const int32_t *out_rows_dev, int out_dtype, void *y_dev, int64_t ldy, int64_t y_rows, void *workspace_dev,
                       size_t workspace_bytes, rq_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif
