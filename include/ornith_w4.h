/* Plain 4-bit linear C ABI of the MI355X (gfx950) Ornith library: weights with
 * a scale, and perhaps a zero point, per group of inputs, applied to the rows
 * as they are (no Hadamard rotation, no activation quantisation - those are
 * the G256 linears of ornith_dense.h).  No counterpart in the reference.
 *
 *   out[m, n] = round( sum_g s[n, g] * sum_{k in g} x[m, k] * (c[n, k] - z[n, g]) )
 *
 * with codes c and zero points z in 0..15, groups of G = 32, 64, 128 or 256
 * consecutive k (the last may be short), rows x bf16 or fp16, products and
 * sums in fp32 (each x * c product is exact), one rounding to the output's
 * type.  Over 128 k the kernels sum x (16 + c), up to 31 * 128 |x|: rows below
 * 2^116 in magnitude cannot overflow inside a group; of larger bf16 rows a
 * finite result may come out as NaN (flag 4).  The other half, (16 + z) times
 * the group's sum of x, is subtracted, so the error before the last rounding is
 * absolute: below (139 + K/128) 2^-23 * 32 sum |s x| (seen: below 2^-25 * 32 sum
 * |s x|), also of columns whose codes are their zero points, where the result
 * is not always 0.  A row's result depends on no other row's values; the order of
 * its sums goes by the numbers of rows and columns. */
#ifndef ORNITH_MI355X_W4_H
#define ORNITH_MI355X_W4_H
#include <stddef.h>
#include <stdint.h>
#include <hip/hip_runtime_api.h>
#ifdef __cplusplus
extern "C" {
#endif
#ifndef ORNITH_EXPORT
#define ORNITH_EXPORT __attribute__((visibility("default")))
#endif

enum { ORNITH_W4_BF16 = 0, ORNITH_W4_F16 = 1, ORNITH_W4_F32 = 2 };

/* Banks as the launch reads them; sizes in 32-bit words.
 *   codes [ceil(N/16), ceil(K/128), 64, 4]: word j of lane 16 q + c holds column
 *         c's k = 128 b + 32 j + 8 q .. + 7, k + 2 i at bits 4 i and k + 2 i + 1
 *         at bits 16 + 4 i; codes past N or K are 8;
 *   meta  [ceil(N/16), ceil(K/128), 16, 128/G], for G = 256 [ceil(N/16),
 *         ceil(ceil(K/128)/2), 16, 1]: the scale as fp32 (bf16 and fp16 scales
 *         leave its low bits clear) with the zero point in bits 0..3; scales
 *         past N or K are 0.
 * 0 <= N <= 2^20, 0 <= K <= 65536, K % 8 == 0. */
ORNITH_EXPORT hipError_t ornith_w4_get_layout(int N, int K, int G, size_t* code_words, size_t* meta_words);

/* Banks from a checkpoint's rows: codes uint32 [N, K/8], eight low-first 4-bit
 * values per word; scales [N, ceil(K/G)] bf16 or fp16 (scale_type); zeros uint8
 * [N, ceil(K/G)] or NULL: 8 everywhere.  Code buffers 4- and 16-byte aligned,
 * meta 4; the outputs must not overlap anything.  Flags (sticky): 1 a scale that
 * is not finite, 2 a zero point above 15 (its low four bits are taken). */
ORNITH_EXPORT hipError_t ornith_w4_pack(const void* codes_u32, const void* scales, int scale_type,
                                        const void* zeros_u8, void* packed_codes, void* packed_meta,
                                        void* flags_u32, int N, int K, int G, hipStream_t stream);

/* out [M, N] of out_type (stride ldo >= N) from x [M, K] of x_type (bf16 or
 * fp16; stride ldx >= K).  x and ldx on the 16-byte grid; out aligned to its
 * element; packed codes 16 bytes, meta 4.  Any number of rows; made for the few
 * of a decode step.
 * Flags (sticky): 4 a non-finite sum, 8 a non-finite 16-bit result (fp32 ones
 * raise 4 alone).  M, N == 0
 * return hipSuccess without touching memory; K == 0 gives zeros. */
ORNITH_EXPORT hipError_t ornith_w4_launch(const void* x, int x_type, int64_t ldx, const void* packed_codes,
                                          const void* packed_meta, void* out, int out_type, int64_t ldo,
                                          void* flags_u32, int M, int N, int K, int G, hipStream_t stream);

#ifdef __cplusplus
}
#endif
#endif
