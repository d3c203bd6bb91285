/* vosk_amd_ops.h -- C ABI of libvosk.so's 8-bit operators.
 *
 * Not part of the reference interface.  The operators that the engine's 8-bit
 * acoustic model runs, on device memory of the caller's, for programs that run
 * layers of their own beside the engine: rows of floats to 8-bit codes, row
 * maps of paged frame caches, the matrix product over codes.
 *
 * Every call enqueues its kernels on `stream` (a hipStream_t; NULL: the
 * device's default stream) of `device` and returns; it allocates nothing,
 * waits for nothing, keeps nothing, and may be captured into a graph.  All
 * pointers are device memory except those marked host.  Returns 0, or < 0 for
 * arguments it refuses (nothing is enqueued; vamd_last_error() says why).
 * Calls on one stream run in order; calls on several threads and streams are
 * independent as long as their outputs are.
 */
#ifndef VOSK_AMD_OPS_H
#define VOSK_AMD_OPS_H

#ifdef __cplusplus
extern "C" {
#endif

/* element types of float operands */
#define VAMD_FLOAT32 0
#define VAMD_FLOAT16 1
#define VAMD_BFLOAT16 2

/* Bytes of a code row of k values: k rounded up to a multiple of 64 (the
 * columns past k hold zeros).  < 0 if k is not in [1, 131072]. */
int vamd_op_code_bytes(int k);

/* Rows of floats to 8-bit codes with a 32-bit scale for each row:
 *   scale = fl32(max |x| / 127), code = x / scale rounded half to even
 * exactly, so code * scale is within scale / 2 of x.  A row of zeros gets
 * scale 0; a row that holds an Inf or a NaN gets scale NaN and codes 0.
 * x: [m][k] of `type`, rows ldx elements apart.  codes: rows of
 * vamd_op_code_bytes(k) bytes, ldc bytes apart (16-byte aligned, ldc a
 * multiple of 16).  rows (or NULL): row i is written to row rows[i] of the
 * cache_rows rows of codes and scales; an entry outside them is skipped, and
 * entries inside them have to be distinct.  Without it row i goes to row i
 * (cache_rows >= m).  count (or NULL): rows from *count (device) on are
 * skipped (rows that frame_map has not written name old frames). */
int vamd_op_quantize_rows(int device, void *stream, const void *x, int type, long long m, int k,
                          long long ldx, const int *rows, const int *count, long long cache_rows,
                          signed char *codes, long long ldc, float *scales);

/* Row maps of a frame cache.  Stream r of `streams` has lengths[r] new frames
 * from time first[r] on (a negative length counts as 0) and gives
 * n = ceil(lengths[r] / step) output rows, row i at time first[r] + step * i.
 * starts [streams + 1]: the streams' first output rows and, last, the total.
 * rows [cap][taps]: entry j of an output row at time t is the cache row of
 * frame t + offsets[j] (host array, taps <= 16): with ring = pages * page,
 *   table[r][(f mod ring) / page] * page + f mod page     (mod: 0 .. ring-1)
 * table: [streams][pages] page numbers, rows ldt entries apart.  low / high
 * [streams] (or NULL) are the first and last frame that a stream has: a frame
 * outside them is replaced by the nearest inside (clamp != 0) or has no row
 * (clamp == 0).  An entry is -1 where there is no row: no such frame, a
 * negative page number, a frame `ring` or more before the newest one that the
 * stream's rows name (the ring cannot hold both), or a time outside 32 bits.
 * Output rows from the total on, and those past cap, are not written. */
int vamd_op_frame_map(int device, void *stream, const int *lengths, const int *first, int streams,
                      const int *table, long long ldt, int pages, int page, const int *offsets, int taps,
                      int step, const int *low, const int *high, int clamp, int *starts, int *rows,
                      long long cap);

/* The matrix product over codes:
 *   out[i][n] = epi(wscale[n] * sum_j scale[r(i,j)] * sum_k codes[r(i,j)][k] * w[n][j * kb + k])
 * with kb = vamd_op_code_bytes(k) and r(i,j) = rows[i][j] (rows == NULL: i, taps 1); an entry
 * outside [0, cache_rows) adds nothing.  Inner sums are exact, the rest is
 * 32-bit floats:  v = v + bias[n];  v = max(v, 0) if relu;  v = v * gain[n] +
 * shift[n];  v = residual_scale * residual[i][n] + v;  rounded to out_type.
 * bias, gain with shift, and residual may be NULL.  w: [n][taps * kb] codes,
 * rows ldw bytes apart; codes and w 16-byte aligned, lda and ldw multiples of
 * 16.  count (or NULL): output rows from *count (device) on are left as they
 * were.  out may be residual (the same rows), else it overlaps no input. */
int vamd_op_linear_int8(int device, void *stream, const signed char *codes, long long lda, const float *scale,
                        long long cache_rows, const int *rows, int taps, const int *count, const signed char *w,
                        long long ldw, const float *wscale, int m, int n, int k, const float *bias, int relu,
                        const float *gain, const float *shift, const void *residual, long long ldr,
                        int residual_type, float residual_scale, void *out, long long ldo, int out_type);

/* The same for m rows of floats (x as in vamd_op_quantize_rows; one tap):
 * quantised and multiplied in one call.  workspace: vamd_op_linear_workspace
 * (m, k) bytes, 16-byte aligned, used by this call alone until it has run. */
long long vamd_op_linear_workspace(int m, int k);
int vamd_op_linear_float(int device, void *stream, const void *x, int type, long long ldx, void *workspace,
                         const int *count, const signed char *w, long long ldw, const float *wscale, int m, int n, int k,
                         const float *bias, int relu, const float *gain, const float *shift, const void *residual,
                         long long ldr, int residual_type, float residual_scale, void *out, long long ldo,
                         int out_type);

#ifdef __cplusplus
}
#endif
#endif /* VOSK_AMD_OPS_H */
