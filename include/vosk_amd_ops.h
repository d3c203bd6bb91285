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
 * pointers inside the structures are device memory.  Returns 0, or < 0 for
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
 * exactly, so code * scale is within scale / 2 of x where scale is a normal
 * float (max |x| from 127 * 2^-126 on).  A smaller scale is rounded to a
 * multiple of 2^-149: codes end at -127 and 127 then, and a row whose scale
 * rounds to 0 (max |x| up to 63 * 2^-149) gets codes 0, as a row of zeros
 * does.  A row that holds an Inf or a NaN gets scale NaN and codes 0. */
typedef struct {
    const void *x;           /* rows of k of `type`, ldx elements apart */
    const int *rows;         /* or NULL: row i goes to row rows[i * ldrows] of codes and scales; an entry
                                outside their cache_rows rows is skipped, those inside have to be distinct */
    const int *from;         /* or NULL: row i is row from[i * ldfrom] of the x_rows rows of x; an entry
                                outside them is skipped */
    const int *count;        /* or NULL: rows from *count on are skipped (what frame_map leaves behind its
                                last row names old frames) */
    signed char *codes;      /* rows of vamd_op_code_bytes(k) bytes, ldc apart; 16-byte aligned rows */
    float *scales;
    long long m, ldx, cache_rows, ldc, ldrows, ldfrom, x_rows;
    int type, k;
} VamdQuantizeRows;
int vamd_op_quantize_rows(int device, void *stream, const VamdQuantizeRows *args);

/* Row maps of a frame cache.  Stream r of `streams` has lengths[r] new frames
 * from time first[r] on (a negative length counts as 0) and gives
 * n = ceil(lengths[r] / step) output rows, row i at time first[r] + step * i.
 * Entry j of an output row at time t is the cache row of frame
 * f = t + offsets[j]: with ring = pages * page,
 *   table[r][(f mod ring) / page] * page_stride + (f mod page) * frame_stride
 * (mod: 0 .. ring-1; page_stride = page and frame_stride = 1 for pages of
 * neighbouring rows, page_stride = 1 and frame_stride = streams for a ring of
 * one page in which the streams' rows of one time are neighbours).
 * low / high are the first and last frame that a stream has: a frame outside
 * them is replaced by the nearest inside (clamp != 0) or has no row.  An entry
 * is -1 where there is no row: no such frame, a negative page number, a frame
 * `ring` or more before the newest one that the stream's rows name (the ring
 * cannot hold both), a time outside 32 bits, a row past 2^31 - 1. */
typedef struct {
    const int *lengths, *first; /* [streams] */
    const int *table;        /* [streams][pages] page numbers, rows ldt entries apart */
    const int *low, *high;   /* [streams], or NULL */
    int *starts;             /* [streams + 1]: the streams' first output rows, and last the total */
    int *rows;               /* [cap][taps]; rows from the total on, and those past cap, are not written */
    long long ldt, cap;
    int streams, pages, page, page_stride, frame_stride, taps, step, clamp;
    int offsets[16];
} VamdFrameMap;
int vamd_op_frame_map(int device, void *stream, const VamdFrameMap *args);

/* The matrix product over codes:
 *   out[i][n] = epi(wscale[n] * sum_j scale[r(i,j)] * sum_k codes[r(i,j)][k] * w[n][j * kb + k])
 * with kb = vamd_op_code_bytes(k), codes and w in -127 .. 127, and r(i,j) = rows[i][j] (rows NULL: i, one
 * tap); an entry outside [0, cache_rows) adds nothing.  Inner sums are exact,
 * the rest is 32-bit floats:  v = v + bias[n];  v = max(v, 0) if relu;
 * v = v * gain[n] + shift[n];  v = residual_scale * residual[i][n] + v;
 * rounded to out_type.
 * With x (and codes and scale NULL) rows of floats take the place of codes:
 * they are quantised as by vamd_op_quantize_rows in the call, which may take a
 * workspace (vamd_op_linear_workspace).  rows then maps the cache_rows rows of
 * x; without it x has m rows.  Where the workspace is not 0 all cache_rows
 * rows are quantised, however few of them the map names: a large cache is
 * better kept in codes.  m is at most 2^30, n and the row strides ldr and ldo at
 * most 2^23. */
typedef struct {
    const signed char *codes; /* rows of kb bytes, lda apart; 16-byte aligned rows */
    const float *scale;      /* [cache_rows] */
    const int *rows;         /* [m][taps], rows ldrows entries apart, or NULL */
    const int *count;        /* or NULL: output rows from *count on are left as they were */
    const void *x;           /* rows of k of x_type, ldx elements apart, or NULL */
    void *workspace;         /* 16-byte aligned, this call's alone until it has run */
    const signed char *w;    /* [n][taps * kb] codes, rows ldw apart; 16-byte aligned rows */
    const float *wscale;     /* [n] */
    const float *bias;       /* [n], or NULL */
    const float *gain, *shift; /* [n], or both NULL */
    const void *residual;    /* [m][n] of residual_type, rows ldr elements apart, or NULL */
    void *out;               /* [m][n] of out_type, rows ldo apart; overlapping no input, but it may be residual
                                itself (address, type and stride) where out_to and res_from are both NULL or
                                the same map; refused where it overlaps residual otherwise */
    const int *out_to;       /* or NULL: output row i goes to row out_to[i * ldout_to] of the out_rows rows of
                                out; an entry outside is skipped, those inside have to be distinct */
    const int *res_from;     /* or NULL: row i's residual is row res_from[i * ldres_from] of the res_rows rows;
                                an entry outside adds nothing (with either, that matrix is below 2^31 bytes) */
    long long cache_rows, lda, ldx, ldw, ldr, ldo, ldrows, ldout_to, out_rows, ldres_from, res_rows;
    int m, n, k, taps, relu, x_type, residual_type, out_type;
    float residual_scale;
} VamdLinearInt8;
int vamd_op_linear_int8(int device, void *stream, const VamdLinearInt8 *args);
/* Bytes of workspace for m output rows, n columns and x_rows rows of k floats
 * (x_rows = m without a map): may be 0; < 0 for bad sizes. */
long long vamd_op_linear_workspace(int m, int n, int k, int taps, long long x_rows);

#ifdef __cplusplus
}
#endif
#endif /* VOSK_AMD_OPS_H */
