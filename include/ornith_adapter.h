/* Low-rank adapter C ABI of the MI355X (gfx950) Ornith library: what the
 * adapters of many requests add to a shared projection's results, in one call.
 * No counterpart in the reference.
 *
 * For row t with slot a = ids[t] >= 0 and output column n of slice p:
 *   v[t, p, r] = sum_k x[t, k] A[a, p R + r, k]
 *   out[t, n]  = round( base[t, n] + scale[a] * sum_r B[a, n, r] v[t, p, r] )
 * and out[t, n] = base[t, n] for a row with ids[t] < 0 (no adapter).
 *
 * x, A and B are all bf16 or all fp16; base and out bf16, fp16 or fp32, out perhaps
 * base itself (the same rows), which leaves rows without an adapter untouched.
 * Each product is exact and summed in fp32; scale v enters the second product
 * as the sum of 16-bit numbers, off by at most 2^-17 of itself (bf16, 16-bit
 * results), by nothing from 2^-103 up (bf16, fp32 results), or by 2^-23 and 2^-38 of
 * the largest of its row and slice (fp16); one rounding to the output's type.  Where a
 * result so formed is not finite, it and those that share 16 bytes of its row are
 * formed again from v itself, in fp64: an infinity or NaN of A, B, x or base gives what
 * it gives in the formula, in its own rows and columns alone.  A row depends on no
 * other row's values; the order of its sums goes by the numbers of rows and of
 * columns.
 *
 * A merged projection (q, k and v, or gate and up) has S slices of consecutive
 * columns, R rows of A each; a plain one has one slice.  Slots with a smaller
 * rank than R leave the rest of A or B zero.
 *
 * Flags (sticky): 4 a non-finite result in fp32, 8 a non-finite 16-bit result,
 * 16 an id >= slots (its row is treated as one without an adapter). */
#ifndef ORNITH_MI355X_ADAPTER_H
#define ORNITH_MI355X_ADAPTER_H
#include <stddef.h>
#include <stdint.h>
#include <hip/hip_runtime_api.h>
#ifdef __cplusplus
extern "C" {
#endif
#ifndef ORNITH_EXPORT
#define ORNITH_EXPORT __attribute__((visibility("default")))
#endif

enum { ORNITH_ADAPTER_BF16 = 0, ORNITH_ADAPTER_F16 = 1, ORNITH_ADAPTER_F32 = 2 };
enum { ORNITH_ADAPTER_MAX_SLICES = 8, ORNITH_ADAPTER_MAX_SLOTS = 4096, ORNITH_ADAPTER_MAX_RANK = 512 };

/* Workspace for calls of up to Mcap rows with S * R rows of A (however they are
 * divided). */
ORNITH_EXPORT hipError_t ornith_adapter_get_layout(int Mcap, int S, int R, size_t* workspace_bytes);

/* x [M, K] of x_type with row stride ldx; A [slots, S R, K] and B [slots, N, R] of
 * x_type, with slot strides a_slot and b_slot and contiguous within a slot; scales
 * fp32 [slots]; ids int32 [M]; base and out [M, N] of out_type, row strides ldb and
 * ldo; slice_ends int32 [S], a host array, ascending, the last N.  Strides in
 * elements.  x, A and B 16-byte aligned with strides that are multiples of 8,
 * K and R multiples of 8; base and out aligned to their element; workspace
 * 256-byte aligned memory of the stream's device, private to the call until it
 * has finished, in need of no initial value.
 * 0 <= M, 0 <= N <= 2^20, 0 <= K <= 65536, 0 <= slots <= 4096, 8 <= R <= 512,
 * 1 <= S <= 8.  M or N == 0 returns hipSuccess without touching memory. */
ORNITH_EXPORT hipError_t ornith_adapter_launch(
    const void* x, int x_type, int64_t ldx, const void* a, int64_t a_slot, const void* b, int64_t b_slot,
    const void* scales_f32, const void* ids_i32, const void* base, int64_t ldb, void* out, int out_type, int64_t ldo,
    void* workspace, size_t workspace_bytes, void* flags_u32, int M, int N, int K, int R, int S,
    const int* slice_ends, int slots, hipStream_t stream);

#ifdef __cplusplus
}
#endif
#endif
