/* Expert routing C ABI of the MI355X (gfx950) Ornith library: the experts of
 * each row of a gate's logits and their weights, for contracts other than the
 * fixed one of ornith_router_topk_launch (ornith_moe.h).  No counterpart in the
 * reference, which leaves other contracts to its serving engine.
 *
 * Per row of logits l [M, E], with a bias b [E] or none:
 *   - score s_i = exp(l_i - mx) / sum of these over the row (softmax), or
 *     1 / (1 + exp(-l_i)) (sigmoid);
 *   - the experts are picked by c_i = s_i + b_i; without a bias by l_i, which
 *     has the order of s_i;
 *   - an expert takes part if l_i is neither -inf nor NaN and c_i neither;
 *   - of G groups of E/G consecutive experts the Gk with the largest group
 *     score stay: that is the largest c of its experts (group_top 1) or the sum
 *     of its two largest (group_top 2, without a bias of scores; of the one that
 *     takes part where there is one).  Ties to the lower group;
 *   - the k experts with the largest c in those groups, in descending order, ties
 *     to the lower id;
 *   - weight = scale s_i, or with renormalize scale s_i / (sum of the k s).
 * A row with fewer than k experts to pick ends with ids -1 of weight 0; the sum
 * is over those it has.
 * Scores, sums and comparisons are in fp64 (scores to 2^-44 of themselves; two
 * c within 2^-41 of each other may count as tied), weights rounded once to
 * fp32.  Experts at a logit of +inf share a softmax; a sigmoid's logit below
 * -700 counts as -700.  A row depends on no other row.
 * Flags (sticky): 1 a NaN logit or a NaN or +inf bias, 4 a row with fewer than k
 * experts to pick. */
#ifndef ORNITH_MI355X_ROUTE_H
#define ORNITH_MI355X_ROUTE_H
#include <stddef.h>
#include <stdint.h>
#include <hip/hip_runtime_api.h>
#ifdef __cplusplus
extern "C" {
#endif
#ifndef ORNITH_EXPORT
#define ORNITH_EXPORT __attribute__((visibility("default")))
#endif

enum { ORNITH_SCORE_SOFTMAX = 0, ORNITH_SCORE_SIGMOID = 1 };

/* logits of logits_type (0 bf16, 1 fp16, 2 fp32) [M, E], row stride ld >= E
 * elements, aligned to their element; bias fp32 [E] (nullable); weights fp32
 * [M, k]; ids int32 [M, k]; flags uint32 [1].
 * 1 <= E <= 1024, 1 <= G <= 64 a divisor of E, 1 <= Gk <= G, 1 <= k <= 32 and
 * k <= Gk E/G, scale finite.  M == 0 returns hipSuccess without touching memory. */
ORNITH_EXPORT hipError_t ornith_route_experts_launch(
    const void* logits, int logits_type, int M, int E, int64_t ld, const void* bias_f32, int score, int G, int Gk,
    int group_top, int k, int renormalize, float scale, void* weights_f32, void* ids_i32, void* flags_u32,
    hipStream_t stream);

#ifdef __cplusplus
}
#endif
#endif
