/* Sampling C ABI of the MI355X (gfx950) Ornith library: the stochastic
 * hand-off after a head, beside the greedy one (ornith_head.h).  No
 * counterpart in the reference, whose sampler is its serving engine's.
 *
 * One token per row of logits l [M, N], from the row's temperature T, top_k k,
 * top_p p, min_p q and one given uniform number u:
 *   - a logit takes part if it is neither -inf nor NaN; mx is the largest;
 *   - mass e_i = exp((l_i - mx) / T), 1 where l_i == mx;
 *   - in the order (value descending, column ascending) the row keeps the
 *     shortest of three prefixes: the first k (k <= 0: all), the least number
 *     whose mass is at least p times that of the first k (p == 1: all), and
 *     those with e_i >= q;
 *   - token = the first column, in ascending order, up to which the kept mass
 *     exceeds u times the kept mass S;  logprob = ln(e_token / S).
 * T == 0 is greedy (the first maximum, logprob 0; k, p, q and u do not matter,
 * in range or not).
 * Masses are computed to 2^-33 of themselves and rounded to whole numbers of
 * units of 2^-36 of the power of two above the largest of their 8192-column
 * part, so results depend on no order of additions and on no other row.  A token whose mass is below 2^-37 of its
 * part's largest is never drawn.
 *
 * Per-row settings are device memory, [M] each, a NULL pointer meaning off
 * (temperature 1, top_k 0, top_p 1, min_p 0); uniform is required.
 * Flags (sticky): 1 a NaN logit (it takes no part), 2 a setting out of range
 * (T < 0 or not finite, p outside (0, 1], q outside [0, 1], u outside [0, 1)),
 * 4 a row with no logit that takes part.  A row with flag 2 or 4 gets token -1
 * and a NaN logprob. */
#ifndef ORNITH_MI355X_SAMPLE_H
#define ORNITH_MI355X_SAMPLE_H
#include <stddef.h>
#include <stdint.h>
#include <hip/hip_runtime_api.h>
#ifdef __cplusplus
extern "C" {
#endif
#ifndef ORNITH_EXPORT
#define ORNITH_EXPORT __attribute__((visibility("default")))
#endif

/* logits_type of the launch */
enum { ORNITH_LOGITS_BF16 = 0, ORNITH_LOGITS_F16 = 1, ORNITH_LOGITS_F32 = 2 };

/* Workspace for calls of up to Mcap rows of N columns: 0 bytes (a NULL
 * workspace) up to 8192 columns, and no more for many rows than for the 64 or,
 * of shorter rows, up to 512 that share it.  Mcap >= 0, 0 <= N <= 2^20. */
ORNITH_EXPORT hipError_t ornith_logits_sample_get_layout(int Mcap, int N, size_t* workspace_bytes);

/* logits of logits_type [M, N], row stride ld >= N elements, aligned to their
 * element; uniform, temperature, top_p, min_p fp32 [M]; top_k int32 [M];
 * token int64 [M]; logprob fp32 [M] (nullable); flags uint32 [1].  Workspace
 * 256-byte aligned memory of the stream's device (its blocks meet there through
 * device atomics), private to the call until it has finished.  M == 0 returns
 * hipSuccess without touching memory; N == 0 gives every row token -1. */
ORNITH_EXPORT hipError_t ornith_logits_sample_launch(
    const void* logits, int logits_type, int M, int N, int64_t ld, const void* uniform_f32,
    const void* temperature_f32, const void* top_k_i32, const void* top_p_f32, const void* min_p_f32,
    void* workspace, size_t workspace_bytes, void* token_i64, void* logprob_f32, void* flags_u32,
    hipStream_t stream);

#ifdef __cplusplus
}
#endif
#endif
