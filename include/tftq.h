/*
 * tftq -- FP8 (OCP e4m3fn) quantized-collective kernels for AMD MI355X (gfx950).
 *
 * C ABI of libtftq.so.  Plain pointers and sizes only; no torch types.
 * The three compute entry points replace the three launchers of the reference
 * (torchft/quantization.py): fused_quantize_into_fp8 (:531-588),
 * fused_reduce_fp8 (:638-686) and fused_dequantize_from_fp8 (:591-635).
 * The plan replaces _prepare_quantize_fp8 (:431-528).
 *
 * Conventions
 *  - every function returns 0 on success; a negative value is a TFTQ_E_* code,
 *    a positive value is a hipError_t.  Nothing aborts or throws.
 *  - a plan describes shapes, strides, element type and group size only.  It
 *    holds no address and belongs to no device: tensor addresses, the packed
 *    buffer, the device and the stream are arguments of every compute call.
 *  - `device` is the ordinal of the device that all device addresses of the
 *    call belong to; the library makes it current for the duration of the
 *    call and restores the caller's device before it returns.  -1 = the device
 *    that is current on the calling thread.
 *  - kernels are enqueued on `stream` (a hipStream_t passed as void*, NULL = the
 *    null stream) and the host is never synchronised.
 *  - functions are thread-safe; a plan is immutable and may be used from
 *    several threads, devices and streams at once.
 *  - the library allocates no device memory.  Lists of up to TFTQ_N_INLINE
 *    tensors need none beyond tensors and packed buffer (their descriptors
 *    travel in the kernel arguments); longer lists need two caller-owned device
 *    buffers, see "Long lists" below.
 *
 * Packed buffer (byte-for-byte the reference's, quantization.py:108-123,
 * 495-503), for tensor i of shape [m_i, n_i] and group size ws:
 *    row_bytes_i  = (ceil(n_i / 4) + 1) * 4
 *    slice_rows_i = ceil(m_i / ws)
 *    slot_off_i   = sum_{j<i} slice_rows_j * row_bytes_j
 *    slot_size    = sum_i slice_rows_i * row_bytes_i
 *    output_size  = ws * slot_size
 *    addr(i, r)   = (r / slice_rows_i) * slot_size + slot_off_i
 *                   + (r % slice_rows_i) * row_bytes_i
 *    at addr: [fp32 scale][n_i e4m3fn codes][zero padding to row_bytes_i]
 */
#ifndef TFTQ_H
#define TFTQ_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TFTQ_VERSION 2

/* element types of the tensors being (de)quantized (quantization.py:474-478) */
#define TFTQ_F32 0
#define TFTQ_F16 1
#define TFTQ_BF16 2

/* lists of at most this many tensors need no device memory for their descriptors */
#define TFTQ_N_INLINE 16

/* error codes (negative); positive return values are hipError_t */
#define TFTQ_E_ARG (-1)      /* bad argument (null pointer, ws <= 0, rank out of range ...) */
#define TFTQ_E_DTYPE (-2)    /* "Only fp32, fp16 and bf16 are supported" (:474-478) */
#define TFTQ_E_SHAPE (-3)    /* negative or too large dimension */
#define TFTQ_E_SIZE (-4)     /* "Output size does not match" (:621, :672) */
#define TFTQ_E_NOMEM (-5)    /* host allocation failed */
#define TFTQ_E_NOTABLE (-6)  /* a list longer than TFTQ_N_INLINE needs `table` (and `pointers`) */
#define TFTQ_E_ARCH (-7)     /* the device is not gfx950 */
#define TFTQ_E_TOOBIG (-8)   /* tftq_reduce_static: the list's table exceeds TFTQ_STATIC_TABLE_BYTES */
#define TFTQ_E_BUSY (-9)     /* tftq_reduce_static: a call on another stream of the device has not finished */

typedef struct tftq_plan tftq_plan;

/* library version (TFTQ_VERSION of the build) */
int tftq_version(void);

/* Identifies the sources the library was built from (a hash that the build passes in;
 * "unknown" without one).  Static storage. */
const char *tftq_build_id(void);

/* Text for a return value of this library (static storage). */
const char *tftq_strerror(int code);

/* 0 when device `device` (-1: the current one) can run the kernels (gfx950), else
 * TFTQ_E_ARCH or a hipError_t. */
int tftq_check_device(int device);

/*
 * Layout arithmetic of _prepare_quantize_fp8 (quantization.py:486-503), host
 * only.  shapes: [n_tensors][2] = (m, n); 1-D tensors are passed as (k, 1)
 * (:487-488).  slot_off (may be NULL) receives n_tensors byte offsets.
 */
int tftq_layout(int n_tensors, const int64_t *shapes, int ws, int64_t *slot_off,
                int64_t *slot_size, int64_t *output_size);

/*
 * Builds the work plan for one list of tensors: the layout above plus the
 * partition of all rows into workgroups for the three kernels.  Replaces the
 * shape, stride and offset tables that _prepare_quantize_fp8 uploads on every
 * call (quantization.py:505-515); the addresses (its fourth table) are an
 * argument of the compute calls.  Host only, no HIP call.
 *   dtype    TFTQ_F32 / TFTQ_F16 / TFTQ_BF16
 *   shapes   [n_tensors][2] (m, n)
 *   strides  [n_tensors][2] element strides (row, column); any values
 */
int tftq_plan_create(int dtype, int n_tensors, const int64_t *shapes, const int64_t *strides,
                     int ws, tftq_plan **out);
void tftq_plan_destroy(tftq_plan *plan);

int64_t tftq_plan_output_size(const tftq_plan *plan); /* bytes of the packed buffer */
int64_t tftq_plan_slot_size(const tftq_plan *plan);   /* output_size / ws */
int64_t tftq_plan_max_rows(const tftq_plan *plan);    /* i_max_row_num of the reference */
int tftq_plan_n_tensors(const tftq_plan *plan);

/*
 * Long lists (more than TFTQ_N_INLINE tensors).  The kernels read the
 * descriptors from device memory that the caller owns:
 *   table     tftq_plan_table_bytes() bytes, 256-byte aligned, holding a copy of
 *             tftq_plan_table_host(): descriptors and lookup index, no addresses.
 *             The same image serves every device, stream and list of tensors of
 *             these shapes; copy it once per device, any way you like, before
 *             the first kernel that uses it runs.
 *   pointers  8 * n_tensors bytes, 8-byte aligned: the tensors' addresses.  When a
 *             compute call is given `tensors` (host array), it first writes them
 *             here with small kernels on `stream` (the host array is read
 *             before the call returns; nothing blocks); with tensors == NULL it
 *             uses what `pointers` already holds.  One `pointers` buffer must
 *             not be written by calls that overlap in time.  All arguments are
 *             checked before the addresses are written; a call whose kernel launch
 *             then fails with a hipError_t has still rewritten `pointers`.
 * For short lists both are ignored (pass NULL) and tftq_plan_table_bytes() is 0.
 */
int64_t tftq_plan_table_bytes(const tftq_plan *plan);
const void *tftq_plan_table_host(const tftq_plan *plan);

/* Writes the n_tensors addresses of `tensors` (host array) to `pointers` (device) on
 * `stream`: what the compute calls do when they are given `tensors` for a long list. */
int tftq_upload_pointers(const tftq_plan *plan, const void *const *tensors, void *pointers,
                         int device, void *stream);

/*
 * fused_quantize_into_fp8 (quantization.py:531-588).  Reads the tensors,
 * writes every byte of packed[0 .. output_size): scales, codes, zero padding
 * and zero padding rows, so `packed` needs no prior memset (the reference
 * relies on torch.zeros, :567-571).  packed must be 4-byte aligned.
 *   tensors  host array [n_tensors]: device address of element (0,0) of each
 *            tensor (may be NULL for a long list whose `pointers` are current)
 */
int tftq_quantize(const tftq_plan *plan, const void *const *tensors, const void *table,
                  void *pointers, void *packed, int64_t packed_bytes, int device, void *stream);

/*
 * fused_reduce_fp8 (quantization.py:638-686).  packed holds ws slots, slot p =
 * peer p's quantization of this rank's row slice.  Sums the slots in fp32 in
 * the order rank, rank+1, ... (wrapping, :405-407), requantizes and overwrites
 * slot `rank` (scale and codes of every row, padding rows included).  is_avg
 * != 0 divides by ws (:682).  No tensor is touched (the reference's launcher
 * ignores their addresses too, :675-686).
 */
int tftq_reduce(const tftq_plan *plan, const void *table, void *packed, int64_t packed_bytes,
                int rank, int is_avg, int device, void *stream);

/*
 * fused_dequantize_from_fp8 (quantization.py:591-635).  Writes
 * cast(float(code) / scale) into the tensors (all m_i real rows).
 */
int tftq_dequantize(const tftq_plan *plan, void *const *tensors, const void *table,
                    void *pointers, const void *packed, int64_t packed_bytes, int device,
                    void *stream);

/*
 * fused_dequantize_from_fp8 followed by the caller's normalisation of the result,
 * `tensor /= num_participants` in the continuation of Manager.allreduce
 * (manager.py:450-452), in one pass over the tensors instead of two.  Writes
 * cast(float(cast(float(code) / scale)) * post_scale): the value is rounded to
 * the tensors' dtype as tftq_dequantize stores it, widened again and multiplied
 * in fp32, which is what torch's division of a GPU tensor by a host scalar
 * computes with post_scale = (float)(1.0 / divisor).  The bytes equal those of
 * tftq_dequantize followed by that division.
 */
int tftq_dequantize_scaled(const tftq_plan *plan, void *const *tensors, const void *table,
                           void *pointers, const void *packed, int64_t packed_bytes,
                           float post_scale, int device, void *stream);

/*
 * tftq_reduce for callers that cannot hand over device memory for `table` and may not
 * allocate: code under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc.  It has no counterpart in the reference.  For a long list the table image
 * is written, with small kernels on `stream`, into a fixed array of
 * TFTQ_STATIC_TABLE_BYTES bytes that the library's code object holds on every device
 * it runs on, and the reduce kernel reads it from there; lists whose table is larger
 * are refused with TFTQ_E_TOOBIG (90 to 190 bytes per tensor: lists of 2800 tensors always fit).
 * Short lists use no scratch memory at all.  The call allocates and frees nothing; it
 * costs one small kernel per 3584 bytes of table in front of the reduce kernel.  The
 * array's address on a device is looked up once, by tftq_check_device() for that device
 * or else by the first call there (which should then not run under stream capture).
 * All calls on one device share that array.  Calls on one stream are ordered by the stream.
 * A call on another stream than the last one, while the last one's kernel has not finished,
 * queues nothing and returns TFTQ_E_BUSY (wait for that stream, or make this one wait for it,
 * and call again); calls from several threads are taken one at a time.  Calls that a stream
 * capture records are not checked against each other or against later calls: replays of
 * graphs that hold such calls, and eager calls beside them, must be serialised by the
 * caller.  Results are those of tftq_reduce.
 */
#define TFTQ_STATIC_TABLE_BYTES (512 * 1024)
int tftq_reduce_static(const tftq_plan *plan, void *packed, int64_t packed_bytes, int rank,
                       int is_avg, int device, void *stream);

/*
 * 4-bit microscaled matrices (no counterpart in the reference): the weights, activations and
 * gradients of a linear layer whose products run on the 4-bit matrix cores.
 *
 * Blocks of 32 consecutive elements of a row share a scale 2^e, e = clamp(floor(log2 max|x|) - 2,
 * -127, 127), held as the byte e + 127; an element is the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 to
 * x / 2^e with its sign (ties to the even mantissa, larger values 6), held in 4 bits (sign, two
 * bits of exponent, one of mantissa), two to a byte, the first in the low half.  The last block of
 * a row may be shorter.  A block that holds an infinity or a NaN has the byte 255 and reads as NaN.
 *
 * A matrix [rows, cols] is one buffer of tftq_mx_bytes(rows, cols) bytes, 16-byte aligned, that the
 * caller owns.  With P = ceil(cols / 256) panels:
 *    codes   [P][rows][128]            columns 256 p to 256 p + 255 of every row, zero past the last one
 *    scales  [P][rows rounded up to an even number][8]   of those columns' blocks
 */
/* bytes of a matrix, or TFTQ_E_SHAPE: rows and columns are at most 2^31 - 1024, here and below, and
 * nothing else but memory bounds a matrix */
int64_t tftq_mx_bytes(int64_t rows, int64_t cols);

/*
 * Quantises x [rows, cols] (row_stride elements from row to row, columns contiguous) along its rows
 * into by_rows, a matrix [rows, cols], and along its columns into by_cols, a matrix [cols, rows]:
 * either may be NULL.  x is read once for both.
 */
int tftq_mx_quantize(int dtype, const void *x, int64_t rows, int64_t cols, int64_t row_stride, void *by_rows,
                     void *by_cols, int device, void *stream);

/* The values that a matrix [rows, cols] stands for, rounded once to `dtype`. */
int tftq_mx_dequantize(int dtype, const void *matrix, int64_t rows, int64_t cols, void *out, int64_t row_stride,
                       int device, void *stream);

/* out [m, n] = a [m, k] b [n, k]^T of two matrices, summed in fp32 and rounded once to `dtype`. */
int tftq_mx_product(int dtype, const void *a, int64_t m, const void *b, int64_t n, int64_t k, void *out,
                    int64_t row_stride, int device, void *stream);

/*
 * out [m, n] = Q(x) b^T: x [m, k] is quantised along its rows on the way, out has its type.  Few rows
 * (the tokens of a model that is served) take one kernel and no workspace; others quantise into
 * `workspace`, tftq_mx_linear_workspace bytes (TFTQ_E_DTYPE or TFTQ_E_SHAPE in place of a number of bytes)
 * for the same x, 16-byte aligned, which holds nothing between calls.
 */
int64_t tftq_mx_linear_workspace(int dtype, const void *x, int64_t m, int64_t row_stride, int64_t n, int64_t k);
int tftq_mx_linear(int dtype, const void *x, int64_t m, int64_t row_stride, const void *b, int64_t n, int64_t k,
                   void *out, int64_t out_stride, void *workspace, int64_t workspace_bytes, int device, void *stream);

/*
 * Newton-Schulz orthogonalisation of a list of matrices, and the step of the Muon optimiser (no
 * counterpart in the reference): what a replica does with the averaged gradients of its weight
 * matrices.  For every matrix u [rows, cols]:
 *    X = u / max(|u|_F, eps);  iterations times:  X = a X + (b (X X^T) + c (X X^T)^2) X
 * (of u^T where rows > cols).  Products run on the 16-bit matrix cores with fp32 sums; with `precise`
 * set every one is three, of high and low parts, and the result has the accuracy of fp32 products
 * (as has, in any case, that of a matrix with fewer than 192 rows or columns).
 */
typedef struct tftq_ns {
    int n;                          /* matrices; empty ones are left alone */
    const int64_t *shapes;          /* [n][2] rows, columns: at most 2^24 each, 2^35 elements with either rounded up to 64 */
    const void *const *in;          /* gradients; columns contiguous */
    const int64_t *in_stride;       /* [n] elements from row to row */
    int in_dtype;
    float *const *momenta;          /* NULL: u is the gradient.  Else m = momentum m + (1 - momentum) g, in place, */
    const int64_t *momenta_stride;  /* and u = m, or momentum m + (1 - momentum) g with nesterov */
    float momentum;
    int nesterov;
    void *const *out;
    const int64_t *out_stride;
    int out_dtype;
    const float *steps;             /* NULL: out = X.  Else [n], and out = keep out - step X */
    float keep;
    int iterations;                 /* at least 1 */
    const float *coefficients;      /* [iterations][3] a, b, c */
    float eps;
    int precise;
} tftq_ns;

/* bytes that tftq_newton_schulz needs for these matrices, or TFTQ_E_ARG / TFTQ_E_SHAPE: those of the up to 24 that
 * are worked on at once (8 to 12 bytes an element, 12 to 20 with `precise`; a caller who has less passes a shorter list) */
int64_t tftq_newton_schulz_workspace(int n, const int64_t *shapes, int precise);

/*
 * `what` and the host arrays it names are read before the call returns.  `workspace` is device
 * memory, 128-byte aligned, of workspace_bytes bytes (TFTQ_E_SIZE if too few), and holds nothing
 * between calls.  A gradient may be the matrix that `out` names when it has no momentum.
 */
int tftq_newton_schulz(const tftq_ns *what, void *workspace, int64_t workspace_bytes, int device, void *stream);

/*
 * Row operators of a training step (no counterpart in the reference).  Rows are contiguous runs of `cols` elements of
 * TFTQ_F32, TFTQ_F16 or TFTQ_BF16 at any address that is a multiple of the element's size; strides are elements from
 * row to row, and where none is given rows follow each other.  Rows, columns, tokens and choices are at most 2^31 - 65536
 * (TFTQ_E_SHAPE).  Sums are fp32 in an order that the arguments alone decide; results are rounded once.  Workspaces
 * are device memory, 16-byte aligned, at least as many bytes as the function beside says (TFTQ_E_SIZE), and hold
 * nothing between calls.  What a function writes overlaps nothing that it reads.
 *
 * Root-mean-square norm:  h = x + residual, rounded to the rows' type;  y = h w / sqrt(mean(h^2) + eps).
 *   x         x_group rows x_stride apart, and as many again x_group_stride behind their beginning, and so on (heads inside
 *             wider rows); x_group = rows for rows that are one stride apart
 *   residual  NULL for none; then h is x and the argument h has to be NULL
 *   weight    [cols] of weight_dtype (dtype or TFTQ_F32); NULL for ones
 *   y         [rows, cols]; or NULL, with codes [rows, cols] and scales [rows]: y in e4m3 codes that scales multiply,
 *             a row's largest magnitude / 448 (1 where that is below 2^-126).  Codes are the nearest to 448 h w / max |h w|, the
 *             even one of two that are as near (of scales above 2^-100, and of h that are no less than 2^-126 of the row's root mean square)
 * The sum of squares is fp32: rows of magnitudes beyond 1e18 pass its range.
 */
int tftq_rms_norm(int dtype, int weight_dtype, const void *x, int64_t x_stride, int64_t x_group, int64_t x_group_stride,
                  const void *residual, int64_t residual_stride, const void *weight, int64_t rows, int64_t cols, float eps,
                  void *h, void *y, void *codes, float *scales, int device, void *stream);
/*
 * Its gradients, from the h that was kept (x where there was no residual):
 * dx = d/dx of <dy, y> + dh (dh may be NULL), also the residual's; dweight [cols] of weight_dtype (a weight is needed then).  Either may be NULL.
 */
int64_t tftq_rms_norm_backward_workspace(int dtype, int64_t rows, int64_t cols);
int tftq_rms_norm_backward(int dtype, int weight_dtype, const void *dy, const void *dh, const void *h, int64_t h_stride,
                           int64_t h_group, int64_t h_group_stride, const void *weight, int64_t rows, int64_t cols, float eps,
                           void *dx, void *dweight, void *workspace, int64_t workspace_bytes, int device, void *stream);

/*
 * Dropout:  out = residual + x keep / (1 - q) for n elements, q = round(p 65536) / 65536; residual may be NULL.  Element i
 * is kept if its 16-bit number is at least q 65536: number i % 8 (low half of the first word first) of the block that
 * the Philox generator of four 32-bit words and ten rounds makes of the counter (i / 8, offset) and the key seed,
 * all 64-bit numbers with the low word first.  seed_at: NULL, or a device address to read the seed from.
 */
int tftq_dropout(int dtype, const void *x, const void *residual, int64_t n, double p, int64_t seed, const int64_t *seed_at,
                 int64_t offset, void *out, int device, void *stream);

/*
 * Embedding:  out[t] = scale table[ids[t]], zeros where ids[t] is not in [0, vocab).  ids: signed, id_bytes 4 or 8 each.
 * Gradient:  dtable[v] = scale sum of dy[t] over ids[t] = v, every row of dtable written; tokens with ids[t] = skip have none
 * (skip outside [0, vocab): no such).
 */
int tftq_embedding(int dtype, int id_bytes, const void *ids, int64_t n, const void *table, int64_t vocab, int64_t cols,
                   int64_t row_stride, float scale, void *out, int device, void *stream);
int64_t tftq_embedding_backward_workspace(int dtype, int64_t n, int64_t vocab, int64_t cols);
int tftq_embedding_backward(int dtype, int id_bytes, const void *ids, int64_t n, int64_t skip, const void *dy, int64_t vocab,
                            int64_t cols, float scale, void *dtable, void *workspace, int64_t workspace_bytes, int device,
                            void *stream);

/*
 * Tokens by expert: `choices` numbers of experts, signed, id_bytes 4 or 8 each; what is not in [0, experts) names none.
 *   position  [choices] the place of a choice: by expert, then in order; those of no expert behind all others
 *   order     [choices] the choice at a place
 *   offsets   [experts + 1] the first place of every expert; the last: how many places have an expert
 */
int64_t tftq_expert_sort_workspace(int64_t choices, int64_t experts);
int tftq_expert_sort(int id_bytes, const void *chosen, int64_t choices, int64_t experts, int32_t *order, int32_t *position,
                     int32_t *offsets, void *workspace, int64_t workspace_bytes, int device, void *stream);
/*
 * Rows to the places of their tokens' k choices each, and back.  position: [tokens][k] from the sort, `used` the address
 * of the last of its offsets.
 *   dispatch  out[position[t, s]] = x[t], elements of 1, 2 or 4 bytes; zeros in places of no expert
 *   combine   out[t] = sum over s of weights[t, s] rows[position[t, s]], without choices of no expert.
 *             weights of weight_dtype (dtype or TFTQ_F32), NULL for ones: the gradient of dispatch
 *   combine_backward  drows[position[t, s]] = weights[t, s] dy[t], zeros in places of no expert;
 *             dweights[t, s] = <dy[t], rows[position[t, s]]>, 0 for choices of no expert.  Either may be NULL
 */
int tftq_dispatch(int element_bytes, const void *x, int64_t x_stride, int64_t tokens, int64_t k, int64_t cols,
                  const int32_t *position, const int32_t *used, void *out, int device, void *stream);
int tftq_combine(int dtype, int weight_dtype, const void *rows, int64_t rows_stride, const void *weights, int64_t tokens,
                 int64_t k, int64_t cols, const int32_t *position, const int32_t *used, void *out, int device, void *stream);
int tftq_combine_backward(int dtype, int weight_dtype, const void *dy, int64_t dy_stride, const void *rows,
                          int64_t rows_stride, const void *weights, int64_t tokens, int64_t k, int64_t cols,
                          const int32_t *position, const int32_t *used, void *drows, void *dweights, int device, void *stream);

/* Values of 8-bit rows: out[r, c] = codes[r, c] scales[r], e4m3 codes, rounded once to dtype. */
int tftq_fp8_rows_dequantize(int dtype, const void *codes, const float *scales, int64_t rows, int64_t cols, void *out,
                             int device, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* TFTQ_H */
