/* pk_hip.h - the C ABI of libpkhip.so, libpktito's int8 product path on one
 * MI355X (gfx950).
 *
 * libpktito's backend seam is a table of function pointers (the reference's
 * backend/kernels.h:242-278, pk_kernels). The int8 path is two of them:
 *
 *   quantize   fp32 activations to int8, per column in blocks of qb, a scale
 *              a block                     (backend/kernels.h:47-58)
 *   gemm_q8    the int8 product with exact int32 sums and the fixed fp32
 *              epilogue                    (backend/kernels.h:60-78)
 *
 * This library computes both on the GPU with the reference's bits: the int8
 * activations, their scales and every fp32 output are those of the
 * reference's scalar ref backend (backend/ref/kernels.c:24-86) on the same
 * inputs. The entry points come in seven groups:
 *
 *   1. the drop-in: pk_hip_quantize and pk_hip_gemm_q8 take host pointers and
 *      the arguments of the table's quantize and gemm_q8, and return with the
 *      results in host memory, as the table's functions do;
 *   2. the upload: the model-load step that repacks each PK_Q8 matrix once
 *      into HBM (the reference binds matrices at core/model.c:345-363);
 *   3. the device-resident path: the same two operations on device pointers,
 *      asynchronous on a caller's stream, for callers that keep activations
 *      in HBM;
 *   4. the device-resident encoder layer: the passes the reference runs
 *      between its products, fused with their quantizes, and a whole layer
 *      in one call (core/encoder.c:108-368);
 *   5. the decoder's token steps: its T = 1 products fused into one launch a
 *      step (core/decoder.c:54-101);
 *   6. the cache of keys and values, for streams of live audio: the encoder's
 *      attention over frames kept in 4 bits between calls. Its outputs are
 *      computed in 32 bits, not held to a bit pattern (the reference has no
 *      cache);
 *   7. audio without an end: attention with a sliding window and sinks, over
 *      whole segments and over the cache, a step's tables made on the device,
 *      and how sure a recognizer is of its tokens. In 32 bits as well.
 *
 * Every function returns PK_HIP_OK or an error code (pk_hip_strerror names it,
 * pk_hip_last_error gives the calling thread's last message); nothing falls
 * back to the CPU. No function here prints.
 */
#ifndef PK_HIP_H
#define PK_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* The activations of one product: the reference's pk_act
 * (backend/kernels.h:41-45), field for field, so a pk_act * may be passed
 * wherever a pk_hip_act * is taken.
 *   q  [T][n] int8, column t at q + t * n
 *   d  [T][n / qb] fp32, each block's scale */
typedef struct {
    int8_t   *q;
    float    *d;
    uint32_t  n, qb, T;
} pk_hip_act;

enum {
    PK_HIP_OK = 0,
    PK_HIP_EINVAL = 1,      /* arguments outside the contract */
    PK_HIP_ENODEV = 2,      /* no usable gfx950 device */
    PK_HIP_ENOMEM = 3,      /* a device or pinned allocation failed */
    PK_HIP_EDEVICE = 4,     /* a HIP call or a kernel launch failed */
    PK_HIP_ENOTUP = 5,      /* gemm_q8's w is inside no uploaded matrix */
    PK_HIP_EROUND = 6,      /* the caller's rounding mode is one this entry does not take */
    PK_HIP_ETIMEOUT = 7,    /* a launch's bounded wait ran out (the launch ended, its results are not whole) */
};

/* The error code's name, and the calling thread's last error message. */
const char *pk_hip_strerror(int err);
const char *pk_hip_last_error(void);

/* Opens the device (the one current on the calling thread, else device 0)
 * once a process; later calls return the first call's result. Every other
 * function calls it. The environment's PKTITO_HIP_DISABLE=1 makes it fail
 * with PK_HIP_ENODEV, so a caller's no-device path can be tested anywhere. */
int pk_hip_init(void);

/* ------------------------------------------------------------ upload --- */

/* Repacks the PK_Q8 matrix q (rows x cols, the reference's core/pkf.h:28-41
 * layout) into HBM with its rows scales s, once, and records the host range
 * [q, q + rows * cols) so that gemm_q8 calls whose w points at any whole
 * panel inside it run on the device copy. rows % 16 == 0, cols % 32 == 0,
 * cols <= 16384 (core/model.c:354). Replaces nothing in the reference: it is
 * the step a GPU backend adds after core/model.c's load_file (:783-811). The
 * host bytes and scales must not change while the matrix is uploaded (a
 * model's are its mapped file's): gemm_q8 reads the device copies, the
 * scales too when its ws is the uploaded s at that panel. A range that
 * shares any byte with an uploaded matrix's is refused (PK_HIP_EINVAL),
 * also when two threads upload it at once: one of them is taken. */
int pk_hip_upload_q8(const int8_t *q, const float *s, uint32_t rows, uint32_t cols);

/* Frees the device copy of the matrix whose host bytes start at q
 * (core/model.c:868-883's pk_model_free gains this call); all of them.
 * These wait for host-pointer products (pk_hip_gemm_q8) in flight on other
 * threads; the device-resident entries below are asynchronous, so their
 * caller must not release a matrix while products on it are queued. */
int pk_hip_release_q8(const int8_t *q);
void pk_hip_release_all(void);

/* -------------------------------------------------------- the drop-in --- */

/* The table's quantize (backend/kernels.h:47-58, :256), on host pointers:
 * a->q, a->d and x are host memory; returns with q and d written. Follows
 * the calling thread's rounding mode as the reference's ref does (both
 * divisions, the product and rintf; backend/ref/kernels.c:24-58); the
 * device-pointer quantizes below round to nearest. */
int pk_hip_quantize(pk_hip_act *a, const float *x, size_t xs);

/* The table's gemm_q8 (backend/kernels.h:60-78, :257-258), on host pointers:
 * out[t * os + r] for r < rows, t < a->T, w the PK_Q8 panels of those rows
 * and ws, bias their scales and biases. Where w is a whole panel of an
 * uploaded matrix the device copy is used; any other w (a caller's own
 * buffer, as the reference's checkers pass) is copied to the device and
 * repacked for this call alone: slower, the same bits. The floats between
 * one column's outputs and the next are not touched. Any of the four IEEE
 * rounding modes the calling thread has set. A release of the matrix
 * waits until the call has returned. */
int pk_hip_gemm_q8(float *out, size_t os, const int8_t *w, const float *ws, const float *bias,
                   uint32_t rows, const pk_hip_act *a, int add);

/* ------------------------------------------- the device-resident path --- */

/* An uploaded matrix, found by its host bytes; NULL if none holds q. */
typedef struct pk_hip_q8 pk_hip_q8;
const pk_hip_q8 *pk_hip_q8_find(const int8_t *q);
/* Its device scales (rows floats), rows and cols. */
const float *pk_hip_q8_scales(const pk_hip_q8 *m);
uint32_t pk_hip_q8_rows(const pk_hip_q8 *m);
uint32_t pk_hip_q8_cols(const pk_hip_q8 *m);

/* quantize on device pointers (a->q, a->d, x), enqueued on stream (a
 * hipStream_t; NULL for the null stream). q and x 16-byte aligned, xs a
 * multiple of 4 floats. Round-to-nearest. */
int pk_hip_quantize_dev(pk_hip_act *a, const float *x, size_t xs, void *stream);

/* gemm_q8 on device pointers: out, ws, bias, a->q and a->d in device memory;
 * the weights are rows [r0, r0 + rows) of the uploaded matrix m (r0 and rows
 * multiples of 16). ws and bias point at row r0's scale and bias (ws may be
 * pk_hip_q8_scales(m) + r0). a->q 16-byte aligned. rmode is the IEEE
 * rounding of the epilogue: 0 to nearest, 1 upward, 2 downward, 3 toward
 * zero. Enqueued on stream; returns once launched. */
int pk_hip_gemm_q8_dev(float *out, size_t os, const pk_hip_q8 *m, uint32_t r0, uint32_t rows,
                       const float *ws, const float *bias, const pk_hip_act *a, int add,
                       int rmode, void *stream);

/* Packed activations, for callers whose quantized activations feed only
 * products: the frames in groups of 16 and each group's inputs in units of
 * 16 frames x 64 inputs laid out as the MFMA takes them, unit u of every
 * group before unit u + 1 (the repacked weights' layout), so that a
 * product's activation tiles are contiguous 1 KB reads. Same q bytes, same
 * d, same outputs as the row-major path. No counterpart in the reference,
 * whose pk_act is row-major (backend/kernels.h:41-45): an extension of the
 * device-resident path. */

/* Bytes a packed copy of T columns of n inputs takes. */
size_t pk_hip_packed_bytes(uint32_t n, uint32_t T);

/* quantize (blocks of the whole row, or of 32 or 64 inputs: the encoder's
 * modes; n <= 4096) writing d and the packed copy qp, and the row-major a->q
 * too unless it is NULL. Device pointers; qp 16-byte aligned and
 * pk_hip_packed_bytes(n, T) long. */
int pk_hip_quantize_packed_dev(pk_hip_act *a, int8_t *qp, const float *x, size_t xs, void *stream);

/* gemm_q8_dev with the activations read from the packed copy qp (a->q is
 * not read; a->d, n, qb and T are; qb the whole row, 32 or 64). */
int pk_hip_gemm_q8_packed_dev(float *out, size_t os, const pk_hip_q8 *m, uint32_t r0, uint32_t rows,
                              const float *ws, const float *bias, const pk_hip_act *a, const int8_t *qp,
                              int add, int rmode, void *stream);

/* The few-frame products (T <= 16, blocks of the whole row: the decoder's
 * per-row callers, core/decoder.c:53-63 and :83-101, and the skinny
 * configs) bound by streaming the weights once: with a workspace, the K
 * inputs of each 16-row panel are split over up to 8 workgroups, so a
 * matrix of few panels (1024 or 1040 rows: 64 or 65 panels) spreads its
 * weights over the chip's CUs instead of one CU a panel. The workgroups of
 * a panel hand their exact int32 sums over in the workspace and the last
 * one runs the epilogue once: the same bits as the entries above. No
 * counterpart in the reference (its CPU calls have no split to make).
 *
 * pk_hip_gemm_workspace(rows): the bytes of workspace a product of rows
 * channels takes. The workspace is device memory, 256-byte aligned and zero
 * before its first use: it starts with a counter a panel, which every call
 * leaves at zero again, then the partial sums, which a call writes before it
 * reads them. Calls that overlap in time (two streams) need workspaces of
 * their own. */
size_t pk_hip_gemm_workspace(uint32_t rows);

/* pk_hip_gemm_q8_dev and pk_hip_gemm_q8_packed_dev with that workspace
 * (work, work_bytes >= pk_hip_gemm_workspace(rows)); NULL: no split. Other
 * calls (T > 16, blocks of 32 or 64) run as the entries above and leave it
 * untouched. */
int pk_hip_gemm_q8_ws_dev(float *out, size_t os, const pk_hip_q8 *m, uint32_t r0, uint32_t rows,
                          const float *ws, const float *bias, const pk_hip_act *a, int add, int rmode,
                          void *work, size_t work_bytes, void *stream);
int pk_hip_gemm_q8_packed_ws_dev(float *out, size_t os, const pk_hip_q8 *m, uint32_t r0, uint32_t rows,
                                 const float *ws, const float *bias, const pk_hip_act *a, const int8_t *qp,
                                 int add, int rmode, void *work, size_t work_bytes, void *stream);

/* One segment of a grouped product: its own activations and outputs. */
typedef struct {
    float      *out;
    size_t      os;
    pk_hip_act  a;
} pk_hip_seg;

/* gemm_q8 of one matrix over nseg segments of activations in a single launch
 * (the ragged batch of segments of different lengths that the reference runs
 * as concurrent lanes, core/asr.c:346-570): each segment's outputs are the
 * bits pk_hip_gemm_q8_dev gives it alone. Device pointers throughout; the
 * segments share n and qb; nseg <= 64. */
int pk_hip_gemm_q8_grouped_dev(const pk_hip_q8 *m, uint32_t r0, uint32_t rows, const float *ws,
                               const float *bias, const pk_hip_seg *segs, uint32_t nseg, int add,
                               void *stream);

/* One product of a batch: an uploaded matrix's run of panels [r0, r0 + rows)
 * with its scales and bias at r0 (device), the packed activations qp of a
 * (a->q is not read), and the outputs out[t * os + r]. */
typedef struct {
    float             *out;
    size_t             os;
    const pk_hip_q8   *m;
    uint32_t           r0, rows;
    const float       *ws, *bias;
    pk_hip_act         a;
    const int8_t      *qp;
    int                add;
} pk_hip_job;

/* njobs <= 8 independent products in one launch, each job's outputs the bits
 * pk_hip_gemm_q8_packed_dev gives it alone. The reference runs such products
 * one after another (core/encoder.c:329-368: the attention's q, k and v of one
 * activation, and the positions' projection); a device-resident caller
 * launches them together. The jobs share n and qb (per-row, qb == n, or
 * blocks of 32 or 64); device pointers throughout. */
int pk_hip_gemm_q8_batch_dev(const pk_hip_job *jobs, uint32_t njobs, int rmode, void *stream);

/* ----------------------------------------- the device-resident layer --- */

/* The producers of the encoder's activations (core/encoder.c), each fused
 * with the quantize that follows it there and writing the packed copy qp
 * (pk_hip_packed_bytes(a->n, a->T) long) and a->d that the next product
 * reads; a->q is not written. Device pointers, 16-byte aligned; a->qb the
 * whole row, 32 or 64 (dwq: 32 or 64). Same bits as the reference's pass
 * followed by its quantize. No counterpart in the reference's kernel table:
 * these are its CPU passes between the products (core/encoder.c:108-176),
 * which a device-resident caller runs where the activations already are. */

/* normq (core/encoder.c:108-128): each of a->T frames of a->n floats at x
 * (frame t at x + t a->n) layer-normed by w, b, eps (backend/kernels.h:
 * 112-122) and quantized; a->n a multiple of 64 up to 4096. */
int pk_hip_normq_dev(pk_hip_act *a, int8_t *qp, const float *x, const float *w, const float *b, float eps,
                     void *stream);

/* siluq (core/encoder.c:130-156): SiLU of each frame (stride xs) then the
 * quantize; a->n a multiple of 32 up to 4096. */
int pk_hip_siluq_dev(pk_hip_act *a, int8_t *qp, const float *x, size_t xs, void *stream);

/* dw (core/encoder.c:158-176): GLU of u [T][2 a->n] (backend/kernels.h:
 * 140-142), the depthwise convolution of K <= 33 taps w [a->n][K] with bias
 * b and SiLU (backend/kernels.h:144-158), quantized; a->n a multiple of 64. */
int pk_hip_dwq_dev(pk_hip_act *a, int8_t *qp, const float *u, const float *w, const float *b, uint32_t K,
                   void *stream);

/* The layer norm in place over T rows of n floats (backend/kernels.h:
 * 112-122; core/encoder.c:86-99); n a multiple of 64 up to 4096. */
int pk_hip_layernorm_dev(float *x, uint32_t T, uint32_t n, const float *w, const float *b, float eps,
                         void *stream);

/* The attention's float part (core/encoder.c:280-327): H heads of D / H
 * dimensions (a multiple of 16; heads of a multiple of 64 run on the
 * tiled kernels, others on one thread an output: fine for the tiny models'
 * 16-wide heads, slow, with no tiling, for long inputs), o [T][D] from the
 * products' outputs q, k,
 * v [T][D] and the positions' p [2T - 1][D] with the biases u and v [D]:
 * Transformer-XL's scores, the softmax, the weighted values, each output
 * the chain pk_k_gemm_f32 and pk_k_softmax make. ws has
 * pk_hip_attention_workspace(T, H) bytes, where the scores live if the call
 * takes the separate kernels (the one kernel keeps them on the chip and
 * leaves ws alone); which of them a call takes is a matter of its sizes. */
size_t pk_hip_attention_workspace(uint32_t T, uint32_t H);
int pk_hip_attention_dev(float *o, const float *q, const float *k, const float *v, const float *p,
                         const float *bias_u, const float *bias_v, uint32_t T, uint32_t D, uint32_t H, void *ws,
                         size_t ws_bytes, void *stream);

/* pk_hip_attention_dev with its scores and row sums in a static scratch
 * array of the library (24 MiB on each GPU it runs on, held until the
 * process ends) instead of a workspace: no allocation of any kind, for
 * callers that cannot allocate (code under HIP graph capture, tight serving
 * loops, harnesses that forbid hipMalloc). No counterpart in the reference.
 * pk_hip_attention_workspace(T, H) must be at most 24 MiB (T up to 884 at 8
 * heads), else PK_HIP_EINVAL. Every call on one GPU shares the array; it
 * keeps the last call's contents, and each call rewrites every score it
 * reads. Outside stream capture a call's kernels wait for the previous
 * call's on that GPU (an event the library records after each call), so
 * calls on two streams or threads take turns. Under capture the call adds
 * no such wait: the caller orders a graph's replays against each other and
 * against other calls (replays of one graph on one stream are ordered). */
int pk_hip_attention_noalloc_dev(float *o, const float *q, const float *k, const float *v, const float *p,
                                 const float *bias_u, const float *bias_v, uint32_t T, uint32_t D, uint32_t H,
                                 void *stream);

/* One encoder layer's weights on the device (core/model.h:45-53): the
 * eleven matrices uploaded, the vectors as device pointers. D = d_model
 * (a multiple of 64 up to 4096), H heads of D / H (a multiple of 16),
 * F = ff_dim (a multiple of 64 up to 4096), K depthwise taps (<= 33). */
typedef struct {
    uint32_t D, H, F, K;
    float    eps;
    const float *ff1_nw, *ff1_nb, *att_nw, *att_nb, *conv_nw, *conv_nb;
    const float *ff2_nw, *ff2_nb, *out_nw, *out_nb;
    const pk_hip_q8 *ff1_up, *ff1_down, *ff2_up, *ff2_down;
    const pk_hip_q8 *q, *k, *v, *pos, *o;
    const float *bias_u, *bias_v;
    const pk_hip_q8 *pw1, *pw2;
    const float *dw, *dw_b;
} pk_hip_layer;

/* Bytes of device workspace pk_hip_layer_dev needs at T frames. */
size_t pk_hip_layer_workspace(const pk_hip_layer *L, uint32_t T, uint32_t qb);

/* One layer (core/encoder.c:321-368) in place on x [T][D] in HBM: the
 * positions' activations ape_qp / ape_d are 2T - 1 frames of D quantized in
 * blocks of qb (pk_hip_quantize_packed_dev once an encode, core/encoder.c:
 * 467-469); the layer's activations are quantized in blocks of qb (32 or
 * 64, the encoder's modes, core/encoder.c:50-56). Every kernel on stream,
 * nothing allocated: ws is ws_bytes >= pk_hip_layer_workspace(L, T, qb) of
 * device memory. The same bits as the reference's layer() over its ref
 * kernels. Calls that overlap on one workspace race. */
int pk_hip_layer_dev(const pk_hip_layer *L, float *x, uint32_t T, const int8_t *ape_qp, const float *ape_d,
                     uint32_t qb, void *ws, size_t ws_bytes, void *stream);

/* ------------------------------------------ the decoder's token steps --- */

/* The decoder's per-token products (core/decoder.c:54-101), each a quantize
 * of one row (one block) and a T = 1 product, latency-bound: each entry is
 * one launch (the joint two) that fuses what the reference runs as separate
 * calls. Device pointers; the matrices uploaded, cols <= 4096. Same bits as
 * the reference's calls over its ref kernels. No counterpart in the kernel
 * table: these are core/decoder.c's steps, for a caller whose prediction
 * state lives in HBM. */

/* gemv (core/decoder.c:54-63): x (m's cols floats) quantized whole and
 * multiplied: out[r] for every row r of m, plus bias[r] if bias, added to
 * out[r] if add. */
int pk_hip_gemv_dev(float *out, const pk_hip_q8 *m, const float *bias, const float *x, int add, void *stream);

/* One LSTM layer's step (core/decoder.c:68-75): gates = wx x + b, then
 * + wh h_in (the reference's two calls), then the cell (backend/kernels.h:
 * 180-187): c stepped in place, the new h to h_out (which must not be h_in).
 * wx and wh are [4P][P], x, h_in, h_out and c P floats, b 4P. */
int pk_hip_lstm_step_dev(float *h_out, float *c, const float *h_in, const float *x, const pk_hip_q8 *wx,
                         const pk_hip_q8 *wh, const float *b, void *stream);

/* The joint (core/decoder.c:81-101): the logits of jout (its rows) from
 * relu(f + gp) (jout's cols floats each) plus jout_b, and tok_dur[0] = the
 * first best token of logits [0, V], tok_dur[1] = the first best duration
 * index among the n_dur logits after them. */
int pk_hip_joint_dev(float *logit, uint32_t *tok_dur, const pk_hip_q8 *jout, const float *jout_b, const float *f,
                     const float *gp, uint32_t V, uint32_t n_dur, void *stream);

/* The decoder's weights on the device, for the search below: shapes and
 * durations by value, the matrices uploaded, the vectors device pointers
 * (core/model.h's prediction network and joint). */
#define PK_HIP_DEC_MAX_LAYERS 8
typedef struct {
    uint32_t P, L, J, V, n_dur, blank, max_symbols;
    int32_t  dur[64];                               /* n_dur <= 64 */
    const float *embed;                             /* [V + 1][P] */
    const pk_hip_q8 *wx[PK_HIP_DEC_MAX_LAYERS], *wh[PK_HIP_DEC_MAX_LAYERS];   /* [4P][P] */
    const float *b[PK_HIP_DEC_MAX_LAYERS];          /* 4P each, or NULL */
    const pk_hip_q8 *jpred, *jout;                  /* [J][P]; [rows][J], rows >= V + 1 + n_dur */
    const float *jpred_b, *jout_b;
} pk_hip_decoder;

/* TDT's greedy search over a segment (core/decoder.c:121-147 and pk_decode,
 * :158-173: the state zeroed, the blank's prediction first) in one launch on
 * the device: the LSTM layers, jpred, the joint, its argmax, the duration
 * step and the max_symbols rule, with no host round trip between frames.
 * f: T frames of the joint's encoder half, device, [T][J] (pk_joint_frames'
 * output). Returns once the search has ended, with *ntoks tokens in toks
 * (host, 3 int32 a token: id, frame, duration, as pk_tok), the reference's
 * tokens. cap must be at least T * max_symbols (the most a search can emit).
 * ws: pk_hip_search_workspace(d, cap) bytes of device memory, 256-byte
 * aligned. P and J multiples of 16 up to 1024, V + 1 <= 2048, L <= 8.
 * spin_limit: the iterations a grid-wide wait may take before the launch
 * gives up (0: the default, about a second); a launch that gives up ends
 * and the call returns PK_HIP_ETIMEOUT. Not for stream capture (the launch
 * is cooperative and the call synchronizes). No counterpart in the kernel
 * table: core/decoder.c's loop, for a caller whose frames live in HBM. */
size_t pk_hip_search_workspace(const pk_hip_decoder *d, uint32_t cap);
int pk_hip_search_dev(const pk_hip_decoder *d, const float *f, uint32_t T, int32_t *toks, uint32_t cap,
                      uint32_t *ntoks, void *ws, size_t ws_bytes, uint32_t spin_limit, void *stream);

/* ------------------------------------- the cache of keys and values --- */

/* A stream of live audio is encoded a chunk of frames at a time, and each
 * chunk attends to the frames before it, whose keys and values are kept here
 * between the calls, in 4 bits and in pages. The reference has no counterpart
 * (it encodes a segment in one piece, core/encoder.c:280-327); the attention
 * is that one's, restricted to a window and run over many streams in a call.
 *
 * A page holds PK_HIP_CACHE_PAGE frames of one stream, in every layer and
 * head; which page holds which frames is the caller's table (one table a
 * stream serves all layers). The pool of pages is the caller's device memory,
 * 16-byte aligned, pk_hip_cache_bytes long, its contents of no matter before
 * they are written: layers x pages x heads records of 64 dk + 256 bytes, dk =
 * 32, 64, 96 or 128 (csrc/cache_layout.h has a record's layout). heads is the
 * number of kept heads; an attention of H heads, H a multiple of it, shares
 * each among H / heads consecutive ones.
 *
 * A kept value is one of 0, 1/2, 1, 3/2, 2, 3, 4, 6 with a sign, times the
 * scale of its frame and head: the least bfloat16 whose six-fold is no less
 * than the head's largest magnitude. The nearest one is kept (of two as near,
 * the one with the even code). A head with a NaN, an infinity or a magnitude
 * of 2^127 or more, or with none of 2^-121 or more, is kept as zeros. */
#define PK_HIP_CACHE_PAGE 64
typedef struct {
    void     *data;
    uint32_t  layers, pages, heads, dk;
} pk_hip_cache;
/* 0 for sizes that are not taken (2^48 bytes at most) */
size_t pk_hip_cache_bytes(uint32_t layers, uint32_t pages, uint32_t heads, uint32_t dk);

/* The streams of a call, B of them, with the call's rows of all streams one
 * after another. Device memory, read when the kernels run, so that a captured
 * graph follows the streams as they grow:
 *   table  [B][max_pages]: page of the stream's frames [64 i, 64 i + 64) in
 *          entry i. An entry outside [0, pages) is a hole: its frames are not
 *          written, read as zeros and not attended (a page given up for a
 *          limited context).
 *   len    [B]: the stream's frames before this call's
 *   row0   [B + 1]: stream b's rows are [row0[b], row0[b + 1]), its frames
 *          [len[b], len[b] + T) with T = row0[b + 1] - row0[b], which may be 0
 * rows is the call's number of rows and max_T at least the longest stream's T
 * (rows a stream has beyond max_T or beyond rows take no part). Frames past 64
 * max_pages have no page: they are not kept, and their rows attend those that
 * the table holds; a len past 64 max_pages counts as that. Rows of no stream
 * are left as they were. No two streams of a call may have one row or write
 * one page. max_pages 1 to 2^24, B up to 65535 (with none, table and len may be
 * NULL), rows up to 2^21, and B x max_T x heads what a launch holds (refused
 * otherwise): in a write or read 2^28 pages of all streams and heads,
 * ceil((max_T + 63) / 64) a stream, in an attention 2^24 tiles of their rows. */
typedef struct {
    const int32_t *table, *len, *row0;
    uint32_t B, max_pages, rows, max_T;
} pk_hip_streams;

/* Writes the rows' keys and values, k and v [rows][heads * dk] (row r at k + r
 * ks, v + r vs), as the streams' frames [len, len + T) of one layer. k and v
 * 16-byte aligned, ks and vs multiples of 4. The other frames of a page keep
 * their values. */
int pk_hip_cache_append_dev(const pk_hip_cache *c, uint32_t layer, const float *k, size_t ks, const float *v,
                            size_t vs, const pk_hip_streams *st, void *stream);

/* The values kept for the streams' frames [len, len + T), into k and v (as
 * above): zeros for a hole's frames. */
int pk_hip_cache_read_dev(const pk_hip_cache *c, uint32_t layer, float *k, size_t ks, float *v, size_t vs,
                          const pk_hip_streams *st, void *stream);

/* The attention's positions: p [n][H * dk], the projected position of
 * distance r = (row's frame - attended frame) in row center - r (the encoder's
 * order, center T - 1 for a segment of T, core/encoder.c:280-327), and the
 * biases u and w [H * dk] of the content and the position scores. Device
 * pointers, 16-byte aligned. */
typedef struct {
    const float *p, *bias_u, *bias_w;
    uint32_t n, center;
} pk_hip_positions;

#define PK_HIP_UNLIMITED 0xffffffffu

/* The attention of the call's rows, q [rows][H * dk] (row r at q + r qs), to
 * the frames kept for their streams in one layer, their own among them (append
 * them first), o likewise. The row of frame t attends frames [t - left, t +
 * right] of those its stream has, [0, len + T): right 0 is causal,
 * PK_HIP_UNLIMITED the whole chunk. Scores are
 *   ((q + u) . k + (q + w) . p[center - (t - j)]) / sqrt(dk)
 * or q . k / sqrt(dk) with pos NULL. With pos, distances that p has no row for
 * are not attended: left is at most center, right at most n - 1 - center. A
 * row that attends nothing is zeros. o and q 16-byte aligned, os and qs
 * multiples of 4; o may be q with os = qs. ws: pk_hip_attention_cache_workspace(...) bytes of device
 * memory (of the same cache, streams' counts, H, pos, left and right),
 * 16-byte aligned, of no matter before and after; calls that overlap in time
 * need workspaces of their own (0 bytes: none is needed, or the sizes are not
 * taken; position scores take 2^48 bytes at most). Products and sums in 32
 * bits: what enters them is not rounded below that, and a position score's
 * products are held to 2^-24 of themselves, as 32-bit ones are, but for what of
 * a query, of a position's row or of a value is under 2^-122, which may be
 * dropped (of numbers under 2^-99, their last bits). Values of 2^100 and more
 * may pass the largest float in a sum. */
size_t pk_hip_attention_cache_workspace(const pk_hip_cache *c, const pk_hip_streams *st, uint32_t H,
                                        const pk_hip_positions *pos, uint32_t left, uint32_t right);
int pk_hip_attention_cache_dev(float *o, size_t os, const float *q, size_t qs, const pk_hip_cache *c, uint32_t layer,
                               const pk_hip_streams *st, uint32_t H, const pk_hip_positions *pos, uint32_t left,
                               uint32_t right, void *ws, size_t ws_bytes, void *stream);

/* Copies pages in every layer: pairs (host, 2 n) of a page of src and the page
 * of dst it goes to; src and dst have the same layers, heads and dk and may be
 * one cache. A fork copies a stream's last page, a compaction moves pages
 * down. With table (device, entries of it), entries that name a page moved
 * become the page it went to, as a compaction's streams need (src and dst one
 * cache, then). Refused: ids outside the pools, a page copied to twice, a page
 * both copied from and to, and with a table a page moved twice. */
int pk_hip_cache_move_dev(const pk_hip_cache *dst, const pk_hip_cache *src, const int32_t *pairs, uint32_t n,
                          int32_t *table, size_t entries, void *stream);

/* Which pages of a pool are in use, on the host (no device needed): each page
 * has a count of the streams that hold it. Safe from several threads.
 *   alloc    n pages nobody holds, the lowest, into ids; PK_HIP_ENOMEM and
 *            nothing taken if fewer are free
 *   share    one more holder for each of ids (a fork's whole pages)
 *   release  one fewer; a page without holders is free. Ids that are not held
 *            are refused, and then nothing is changed (an id may be named as
 *            often as it has holders)
 *   holders  a page's count; 0 for a free page or an id outside the pool
 *   compact  the pairs (from, to) that move every page in use below the
 *            number in use, at most cap of them; the pool's own counts move at
 *            once, so the caller's next calls are pk_hip_cache_move_dev with
 *            them and the tables (in stream order before any later write).
 *            Returns how many in *n.
 *   restore  the counts as before a compact that gave these pairs, for a move
 *            that was refused. Refused itself, and then nothing is changed,
 *            where a page that the compact freed is held again, or one that it
 *            filled is free */
typedef struct pk_hip_pool pk_hip_pool;
int pk_hip_pool_create(pk_hip_pool **pool, uint32_t pages);
void pk_hip_pool_destroy(pk_hip_pool *pool);
uint32_t pk_hip_pool_free_pages(const pk_hip_pool *pool);
int pk_hip_pool_alloc(pk_hip_pool *pool, int32_t *ids, uint32_t n);
int pk_hip_pool_share(pk_hip_pool *pool, const int32_t *ids, uint32_t n);
int pk_hip_pool_release(pk_hip_pool *pool, const int32_t *ids, uint32_t n);
uint32_t pk_hip_pool_holders(const pk_hip_pool *pool, int32_t id);
int pk_hip_pool_compact(pk_hip_pool *pool, int32_t *pairs, uint32_t cap, uint32_t *n);
int pk_hip_pool_restore(pk_hip_pool *pool, const int32_t *pairs, uint32_t n);

/* ------------------------------------------- audio without an end --- */

/* The attention of whole segments with a sliding window and sinks, for audio
 * too long for every frame to attend to every other: frame t of a segment of T
 * attends the frames j < T with j <= t + right and either j >= t - left or j <
 * sinks (the segment's first frames, which stay visible behind the window).
 * Scores are
 *   ((q + u) . k + (q + w) . p[center - min(t - j, left)]) / sqrt(dk)
 * (pk_hip_positions; a sink behind the window takes the position of
 * distance left) or q . k / sqrt(dk) with pos NULL; each row is the softmax's
 * weighted values, in one launch whose time goes by the window. With pos,
 * distances that p has no row for are not attended: left is at most center,
 * right at most n - 1 - center. left and right may be PK_HIP_UNLIMITED.
 * q and o are [rows][H * dk], k and v [rows][G * dk], H a multiple of G (each
 * kept head shared among H / G consecutive ones), dk 32, 64, 96 or 128; row r
 * of x at x + r * its stride (qs, ks, vs, os), 16-byte aligned, strides
 * multiples of 4, ks and vs up to 2^25. o may be q with os = qs; an o that shares memory with k, v or
 * the positions is refused (rows of one stride may lie between each other's; of
 * different strides they count as sharing memory wherever their ranges
 * overlap). Rows of no segment are left as they were. Products
 * and sums in 32 bits, not held to a bit pattern (pk_hip_attention_dev's are
 * the reference's, core/encoder.c:280-327, which has no window). A row's
 * outputs depend on the frames that it attends alone, whatever the others hold.
 * Frames whose score is -infinity have no part, and a row without others is 0.
 * Outputs whose sums or scores pass the greatest float on their way (values from
 * some 10^28 on) are right as well, each such row made by itself in 64 bits: a
 * call full of them takes about fifty times as long.
 *
 * The segments of a call: row0 [B + 1] in device memory, read when the kernel
 * runs, segment b's rows [row0[b], row0[b + 1]) of rows in all; max_T at least
 * the longest one's T (what is beyond max_T or beyond rows takes no part). No two
 * segments may have one row. B up to 65535, rows up to 2^21, and B x H x ceil(max_T / 16) under 2^24. */
typedef struct {
    const int32_t *row0;
    uint32_t B, rows, max_T;
} pk_hip_segments;
int pk_hip_attention_window_dev(float *o, size_t os, const float *q, size_t qs, const float *k, size_t ks,
                                const float *v, size_t vs, const pk_hip_segments *sg, uint32_t H, uint32_t G,
                                uint32_t dk, const pk_hip_positions *pos, uint32_t left, uint32_t right,
                                uint32_t sinks, void *stream);

/* The same over the cache (pk_hip_attention_cache_dev), for its streams' steps:
 * the row of frame t also attends its stream's frames j < sinks, j <= t + right,
 * that lie behind the window and whose page the stream holds; their position
 * scores take distance left's row. sinks 0, or a window that all frames are in,
 * is pk_hip_attention_cache_dev. Arguments, outputs and arithmetic are that
 * one's, with the workspace of this one's arguments. */
size_t pk_hip_attention_sinks_workspace(const pk_hip_cache *c, const pk_hip_streams *st, uint32_t H,
                                        const pk_hip_positions *pos, uint32_t left, uint32_t right, uint32_t sinks);
int pk_hip_attention_sinks_dev(float *o, size_t os, const float *q, size_t qs, const pk_hip_cache *c, uint32_t layer,
                               const pk_hip_streams *st, uint32_t H, const pk_hip_positions *pos, uint32_t left,
                               uint32_t right, uint32_t sinks, void *ws, size_t ws_bytes, void *stream);

/* The plan of a step of a cache's streams, made on the device: what each stream
 * brings in, and out come the descriptor that the cache's calls take
 * (pk_hip_streams), pages taken from a pool for new frames, and pages that the
 * window has left given back to it, with nothing for the host to wait for or to
 * send, so that a captured graph of plan, append and attention runs a stream's
 * steps one after another. It stands beside the host's pool (pk_hip_pool_*): a
 * cache's pages are one's or the other's, and pages of this one have one holder.
 *
 * B streams (places that requests come and go in), device memory throughout, 4
 * byte aligned, each a call's own while it runs:
 *   add    [B]: the frames that each stream brings; negative counts as 0
 *   fresh  [B], or NULL for none: not 0 where a stream begins anew: whatever
 *          pages its place held go back, and it brings its first frames (a
 *          stream that ends: fresh, and nothing added)
 *   state  [B][2], kept between calls: the stream's frames so far, and the column
 *          of its table before which the window has given back all but the
 *          sinks'; zeros at first
 *   pool   [2 + pages], kept: the number of the first free page's place, how many
 *          are free, and a ring of places of free pages' ids (at first 0, pages,
 *          and every id): a queue, taken from its front and given back to its end
 *   table  [B][max_pages], kept: as in pk_hip_streams; entries are written as
 *          pages are taken (the id) and given back (-1)
 *   len, row0   [B], [B + 1], written: as in pk_hip_streams, for this call's rows
 *   slot   [rows], or NULL, written: each row's place in the pool, 64 times its
 *          page and its frame's number in it; -1 for rows of no stream or page
 *   told   [4], written: the call's rows, frames asked for that got none (beyond
 *          max_T a stream, rows in all, or 64 max_pages frames of a stream; those
 *          of the last streams in order), pages that the pool did not have
 *          (their frames have a hole), pages free now
 * First, in the order of streams and columns, pages go back: those of columns
 * whose frames are all more than left behind the stream's first new one and that
 * hold no sink (left PK_HIP_UNLIMITED: none), and those of fresh streams. Then, in
 * that order, every column that the new frames begin gets a page. A window that
 * grows from one call to the next does not bring pages back, and sinks that
 * become fewer stay held until their stream ends. Numbers that no call leaves
 * (counts below 0 or too great, ids outside the pool) are read as the nearest
 * that can be, and never make it write outside of the arrays. max_pages 1 to
 * 2^24, B up to 65535 and B x max_pages up to 2^31, rows up to 2^21, max_T up to
 * rows, pages 1 to 2^24. */
typedef struct {
    int32_t *table, *len, *row0, *state, *pool, *slot, *told;
    uint32_t B, max_pages, rows, max_T, pages;
} pk_hip_plan;
int pk_hip_cache_plan_dev(const pk_hip_plan *p, const int32_t *add, const int32_t *fresh, uint32_t left,
                          uint32_t sinks, void *stream);

/* How sure a recognizer is of its tokens: for each of `rows` rows of cols logits
 * (row r at x + r xs; any 4-byte alignment and stride, so the tokens' or the
 * durations' columns of the joint's logits serve as they are,
 * core/decoder.c:81-101), where asked for,
 *   lp       [rows][m]: the log probabilities of the given tokens [rows][m] (-1
 *            is none and gets 0; any other id outside [0, cols) gets a NaN)
 *   entropy  [rows]: of the row's distribution, in nats
 *   top      [rows][k]: the k most probable ids, the most probable first, of
 *            equal logits the lowest id, NaN last; and with top_lp [rows][k]
 *            their log probabilities
 * Computed in 32 bits from the differences to the row's largest logit, whose own
 * term is left out of the sum and added by log1p: a token that is all but certain
 * keeps its small log probability. A logit may be -infinity (probability 0, log
 * probability -infinity); in a row with a NaN, with an infinity, or with nothing
 * but -infinity every probability and the entropy are NaN, and the order is the
 * logits' all the same. Outputs that share memory with the logits, the tokens
 * or each other are refused (seen as in pk_hip_attention_window_dev: an output
 * between the rows of logits is taken only with their stride). cols 1 to 2^20, k up to 32 and up to cols, rows up to 2^21 and
 * under 2^24 with a row's every 8192 columns counted. ws:
 * pk_hip_logprobs_workspace(rows, cols, k) bytes of device memory (0 for up to
 * 8192 columns), 16-byte aligned, of no matter before and after; calls that
 * overlap in time need workspaces of their own. */
size_t pk_hip_logprobs_workspace(uint32_t rows, uint32_t cols, uint32_t k);
int pk_hip_logprobs_dev(const float *x, size_t xs, uint32_t rows, uint32_t cols, const int32_t *tokens, uint32_t m,
                        float *lp, float *entropy, uint32_t k, int32_t *top, float *top_lp, void *ws, size_t ws_bytes,
                        void *stream);

/* Measurement aids, with no counterpart in the reference: the floors a
 * small product's time is read against. pk_hip_empty_dev launches an empty
 * kernel; pk_hip_stream_read_dev reads the bytes at p (16-byte aligned,
 * bytes a multiple of 16) with non-temporal 16-byte loads, one a thread
 * over as many workgroups as they need (at most 32768, four loads a thread
 * in flight beyond that), and writes *sink only if the loads' fold meets a
 * fixed constant (so nothing is written in practice; sink is device
 * memory). */
int pk_hip_empty_dev(void *stream);
int pk_hip_stream_read_dev(const void *p, size_t bytes, uint32_t *sink, void *stream);
/* A measurement aid with no counterpart in the reference: the int8 matrix
 * cores' rate, for checking the published peak on the machine.
 * workgroups of four waves each run iters rounds of eight independent
 * v_mfma_i32_16x16x64_i8 (32768 ops each) on registers, nothing loaded;
 * *sink as for pk_hip_stream_read_dev. */
int pk_hip_mfma_rate_dev(uint32_t workgroups, uint32_t iters, uint32_t *sink, void *stream);

/* The kernel variant the calling thread launched last, for profiling and
 * tests. */
const char *pk_hip_last_kernel(void);

/* Tests and tuning: the number of tilings of the per-column product, each
 * one's name (the name pk_hip_last_kernel gives its launches; "" past the
 * last), and forcing one of them for every later launch in the process (-1
 * restores the automatic choice); returns the index forced before. Not
 * thread-safe against launches in flight on other threads. Every tiling
 * computes the same bits. */
int pk_hip_tilings(void);
const char *pk_hip_tiling_name(int index);
int pk_hip_force_tiling(int index);

/* Tests and tuning: how many workgroups share a panel in every later split
 * few-frame product (1..8; fewer where the panel has fewer units), -1 the
 * automatic choice; returns the one forced before. All compute the same
 * bits. */
int pk_hip_force_split(int splits);

/* Tests and tuning: 0 makes every later search load its LSTM, jpred and
 * jout panels from memory each token even where they fit resident (in its
 * workgroups' registers, loaded once a launch: P and J up to 640, at most 2
 * LSTM layers, at most 2048 rows of jout), 1 restores that; returns the
 * previous setting. Both compute the same tokens; pk_hip_last_kernel says
 * which ran, "search_resident" or "search". */
int pk_hip_force_search_resident(int on);

/* Tests and tuning: forcing the packed quantize's kernel for every later
 * launch in the process: 0 one wave a column (or a wave a 1024-input chunk
 * of a column over 1024 inputs in blocks), 1 one workgroup a half
 * 16-column group, 2 one wave a whole column, -1 the automatic choice by size;
 * returns the one forced before. All compute the same bits. */
int pk_hip_force_quantize(int kind);

/* Tests and tuning: the attention's kernels for every later launch in the
 * process: 0 on the matrix cores (one-step fp32 MFMAs), in one kernel or in
 * separate ones by size (the default), 1 as VALU fma chains, 2 on the matrix
 * cores in separate kernels always; any other value is 1. Returns the one
 * set before. All compute the same bits. */
int pk_hip_force_attention(int kind);

#ifdef __cplusplus
}
#endif

#endif /* PK_HIP_H */
