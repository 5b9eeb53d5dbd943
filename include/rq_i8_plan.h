/*
 * What a call of rq_i8.h runs: the plans that the entry points themselves go by, for tools and for tests that mean one kernel. No GPU is
 * asked. Exported by the same library. 0, or RQ_E_UNSUPPORTED for sizes that the call refuses.
 */
#ifndef RQ_I8_PLAN_H
#define RQ_I8_PLAN_H

#include "rq_i8.h"

#ifdef __cplusplus
extern "C" {
#endif

/* plan[0] */
#define RQ_I8_ROUNDS 1  /* few rows, which every workgroup rounds to int8 for itself (x of a float type) */
#define RQ_I8_STREAM 2  /* few rows, as they lie or from a launch in front */
#define RQ_I8_TILES  3

/* RQ_I8_ROUNDS: plan[1] = rows at a time. RQ_I8_TILES: plan[1], plan[2] = rows of the weight and of x in a tile, plan[3] = row tiles of that form, plan[4], plan[5] =
 * the same of the tiles of the rows behind them (0: none), plan[6] = workgroups that share a tile, plan[7] = tiles that a compute unit holds. Else zeros. */
int rq_i8_product_plan(int64_t K, int64_t N, int in_dtype, int64_t M, int64_t plan[8]);
int rq_grouped_plan(int weight_type, int64_t E, int64_t K, int64_t N, int in_dtype, int64_t M, int64_t P, int64_t plan[8]);

#ifdef __cplusplus
}
#endif
#endif
