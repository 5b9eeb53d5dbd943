/*
 * What a call of rq_mx4.h runs: the plans that the entry points themselves go by, for tools and for tests that mean one kernel. No GPU is
 * asked. Exported by the same library. 0, or RQ_E_UNSUPPORTED for sizes that the call refuses.
 */
#ifndef RQ_MX4_PLAN_H
#define RQ_MX4_PLAN_H

#include "rq_mx4.h"

#ifdef __cplusplus
extern "C" {
#endif

/* plan[0] of a product, and of the experts (RQ_MX4_ALONE or RQ_MX4_TILES) */
#define RQ_MX4_ALONE 1  /* few tokens, which every workgroup rounds for itself */
#define RQ_MX4_ROWS  2  /* few tokens, rounded by a launch in front */
#define RQ_MX4_TILES 3

/* RQ_MX4_TILES: plan[1], plan[2] = rows and tokens of a tile, plan[3] = row tiles of that form, plan[4], plan[5] = rows and tokens of the tiles
 * of the rows behind them (0: none), plan[6] = workgroups that share a tile, plan[7] = workgroups of the form that a compute unit holds
 * (two forms have tiles of 128 x 128). Else zeros. */
int rq_mx4_product_plan(int64_t K, int64_t N, int64_t M, int64_t plan[8]);

/* RQ_MX4_TILES: plan[1], plan[2] = rows (of gate and up together) and tokens of a tile. Else zeros. */
int rq_mx4_experts_plan(int64_t E, int64_t K, int64_t F, int64_t N, int64_t M, int top, int64_t plan[3]);

#ifdef __cplusplus
}
#endif
#endif
