/*
 * naiwa_mxfp4.h -- MXFP4 expert weights: quantisation, the inverse, and the
 * layout that the expert products read.
 *
 * MXFP4 (the OCP microscaling format): the 32 values of a block along a row share
 * one scale byte s, worth 2^(s - 127) (s = 255: the whole block is NaN), and each
 * is a 4-bit E2M1 code: a sign over the magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6.
 * 17 bytes hold 32 values (4.25 bits a value).
 *
 * Tile order (NAIWA_MXFP4_T) of an [n, k] projection, n a multiple of 16, k of 32.
 * Rows go in strips of 16; K is padded to whole steps of 128 values with code 0.
 * A step of a strip is 1024 bytes: bytes 16 (16 b + r) .. + 15 hold block b (of the
 * step's 4) of row r, value 2 i in the low half of byte i and value 2 i + 1 in its
 * high half.  After every 4 steps, and after the last, come 256 scale bytes: byte
 * 4 (16 b + r) + j is the scale of block b, row r of the group's step j (unused
 * bytes 0).  A strip is 1024 t + 256 ceil(t / 4) bytes, t = ceil(k / 128), and strips
 * follow each other.  The layout is the library's own: lane 16 b + r of a wave finds
 * its operand of the matrix cores' scaled 16x16x128 product at 16 times its number, so
 * every load of weights is a whole contiguous kilobyte.
 *
 * The expert products take banks of this type through naiwa_moe_decode[_ex|_noalloc],
 * naiwa_moe_prefill, the layered stack, the partial cache (misses staged over PCIe) and
 * the prefill stream; see naiwa_moe.h.  The reference quantises experts with its fork's
 * tools (src/commands/quantize.rs) and has no MXFP4 path.
 */
#ifndef NAIWA_MXFP4_H
#define NAIWA_MXFP4_H

#include "naiwa_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Quantise `batch` [n, k] projections to tile order.  src: f32, bf16 or f16
 * (src_dtype) device rows ld values apart (0: k), projections src_stride values
 * apart (0: n * ld); dst: device bytes, projections dst_stride bytes apart (0:
 * naiwa_projection_bytes(NAIWA_MXFP4_T, n, k)).  A block's scale is s =
 * max(0, e - 2) with e the biased f32 exponent of its largest magnitude, so that
 * magnitude lands in [4, 8); values are rounded to the nearest code (ties to the even
 * one), above 6 to 6.  A block with a NaN or an infinity becomes NaN (s = 255, codes 0).
 * The same bytes on every run.
 * NAIWA_E_INVALID: n % 16, k % 32, ld < k, a stride under a projection, src, dst or
 * dst_stride no multiple of 16 bytes, ld or src_stride no multiple of 8 values.
 * NAIWA_E_UNSUPPORTED: another src_dtype, or past 2^31 - 1 groups of 16 rows x 512. */
int naiwa_mxfp4_quantize(const void* src, int src_dtype, int64_t batch, int64_t n, int64_t k, int64_t ld,
                         int64_t src_stride, void* dst, int64_t dst_stride, int64_t stream);

/* The values of `batch` tile-order projections, to f32 or bf16 (dst_dtype) rows:
 * exact in f32; bf16 rounds only what is subnormal there.  Arguments and errors as
 * above, src and dst exchanged. */
int naiwa_mxfp4_dequantize(const void* src, int64_t batch, int64_t n, int64_t k, int64_t src_stride, void* dst,
                           int dst_dtype, int64_t ld, int64_t dst_stride, int64_t stream);

/* Host memory: one [n, k] projection of GGML MXFP4 blocks as a GGUF file holds them
 * (type NAIWA_GGML_MXFP4, 17 bytes a block: the scale byte, then 16 bytes whose low
 * halves are values 0..15 and high halves values 16..31) to tile order.  dst holds
 * naiwa_projection_bytes(NAIWA_MXFP4_T, n, k) bytes and does not overlap src.
 * No device call. */
int naiwa_mxfp4_from_ggml(const void* src, int64_t n, int64_t k, void* dst);

#ifdef __cplusplus
}
#endif
#endif
