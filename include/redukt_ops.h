/* redukt_ops.h — operators of libredukt_gpu.so on the caller's own device tensors.
 *
 * The plugin ABI (redukt_backend.h) steps the models that the library loads.  The entry
 * points below are the parts of such a layer as operators of their own, for programs that hold
 * activations, weights and recurrent states themselves: the gated delta rule for one token
 * and for whole sequences, the selective scan likewise and with its gradients, and the int8
 * and block-scaled 8-bit floating point products with the passes that make their codes, and the
 * drawing of tokens from logits.
 *
 * Contract:
 *   - no model is needed (nothing here touches what redukt_backend_init made), and calls from
 *     several threads do not meet: no entry point keeps or shares anything between calls;
 *   - INVALID_ARGUMENT also answers sizes whose launch would not fit (2^32 threads or more);
 *   - every pointer but an argument struct's is device memory of ONE device, which need not be
 *     the calling thread's current one (the current device is the same after the call);
 *   - a call enqueues its kernels on `stream`, a hipStream_t of that device as an opaque
 *     pointer (NULL: the device's default stream), and returns without waiting; it allocates,
 *     copies and synchronises nothing, so it may be captured into a graph.  Work that makes
 *     the inputs, on another stream, is ordered before it by the caller;
 *   - outputs must not overlap inputs, except where a call names the same state pool twice;
 *   - result codes are redukt_backend.h's: INVALID_ARGUMENT launches nothing and changes
 *     nothing, FORWARD_FAILED is a launch that the runtime refused;
 *   - the same inputs give the same bits, whatever else runs.
 */
#ifndef REDUKT_OPS_H
#define REDUKT_OPS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of activations and outputs. */
#define REDUKT_OP_BF16 0u
#define REDUKT_OP_F16 1u
#define REDUKT_OP_F32 2u

/* ---------------- the gated delta rule ----------------
 *
 * Each of hv value heads keeps a state S [dk][dv] in f32.  A token with key k and query q
 * [dk] (of key head h / (hv / hk)), value v [dv], log decay g and write strength beta makes
 *     S <- e^g S + beta k (v - e^g S^T k)^T        o = scale S^T q
 * in f32 arithmetic.  (The factors of delta_chunk's 16-bit outputs are taken with 16 bits: beside
 * its rounding to `dtype` such an output is off by at most 2^-15 of the magnitudes that it sums.
 * States and f32 outputs are as exact as f32 sums are.)  g may be -inf (the state is dropped).  The
 * rule is stable for |k| <= 1, g <= 0 and beta in [0, 2]; with REDUKT_DELTA_NORMALIZE, k and q are
 * divided by sqrt(sum of squares + 1e-6) first.
 *
 * A value that is not finite goes where the rule takes it: one of v into its column, one of k,
 * g or beta into its head, from its token on; one of q into its token.  What it reaches is then
 * not finite, inf or NaN.  To normalize, a key or query whose sum of squares passes f32's range
 * (a length of about 1.8e19) counts as one that is not finite.  In delta_chunk, a sum that passes
 * f32's range from finite inputs may also reach up to 63 tokens back (a stable rule has none, but
 * of values and states next to that range), and a decay over several tokens below 2^-126 is 0. */
#define REDUKT_DELTA_NORMALIZE 1u

typedef struct {
    uint32_t dtype;         /* of q, k, v and out */
    uint32_t rows;          /* tokens */
    uint32_t hk, hv;        /* key heads, value heads: hv a multiple of hk, at most 4,096 */
    uint32_t dk, dv;        /* dk 64 or 128; dv a multiple of 32, at most 256 */
    uint32_t flags;         /* REDUKT_DELTA_* */
    float scale;
    const void* q;          /* row t: hk * dk elements at q + t * q_stride */
    const void* k;          /* hk * dk */
    const void* v;          /* hv * dv */
    void* out;              /* hv * dv */
    int64_t q_stride, k_stride, v_stride, out_stride;   /* elements from a row to the next, at most 2^22 */
    const float* g;         /* row t: hv values at g + t * g_stride */
    const float* beta;
    int64_t g_stride, beta_stride;
} redukt_delta_rows;        /* q, k, v, out: 16-byte aligned, with strides of whole 16 bytes */

/* One token for each of `rows` entries (at most 65,536): entry i steps the state of slot
 * slots[i] (NULL: slot i; rows <= n_slots then) of states [n_slots][hv][dk][dv], in place.
 * A slot of -1 is a padded entry: its output row and every state are left as they are.  A
 * slot that is otherwise out of range, or that an earlier entry names, touches no state and
 * its output row becomes NaN. */
int32_t redukt_op_delta_step(const redukt_delta_rows* a, float* states, uint32_t n_slots, const int32_t* slots,
                             void* stream);

/* Whole sequences: sequence i (of n_seq, at most 65,536) is rows cu[i] to cu[i + 1] (cu: n_seq + 1
 * values, none decreasing, within 0 and `rows`; other values give unspecified outputs, but
 * nothing outside the arrays is touched).  It starts from slot slots[i] (NULL: i) of state_in
 * (NULL: zeros) and leaves its final state there in state_out (NULL: not wanted; a sequence
 * without rows hands its first state on).  The pools are the same, for an update in place, or
 * do not overlap.  Slots behave as above (-1: the sequence is left out); without state_out
 * several sequences may start from one slot.  Rows of no sequence are left as they are.
 * `workspace` holds redukt_op_delta_chunk_workspace(a, n_seq) bytes, 16-byte aligned, which
 * nothing else may use until the call's kernels are done. */
int32_t redukt_op_delta_chunk(const redukt_delta_rows* a, const int32_t* cu, uint32_t n_seq, const float* state_in,
                              float* state_out, uint32_t n_slots, const int32_t* slots, void* workspace,
                              uint64_t workspace_bytes, void* stream);

/* The bytes of workspace for these rows (only the sizes and the element type are read); 0 if
 * the sizes are not ones that delta_chunk takes, or need none. */
uint64_t redukt_op_delta_chunk_workspace(const redukt_delta_rows* a, uint32_t n_seq);

/* ---------------- the selective scan ----------------
 *
 * Each channel keeps a state h [n] in f32.  A token with input x, time step dt, gate z (of the
 * channel), B and C [n] (of the channel's group) makes, with s = ln(1 + e^(dt + dt_bias)),
 *     h <- e^(s a) h + s x B        out = (C . h + d x) z / (1 + e^-z)
 * in f32, rounded once to `dtype`; without z its factor is 1, without d or dt_bias they are 0.  A dt of
 * -inf leaves the state as it is.  The rule is stable for a <= 0.  (With a > 0, scan_chunk and scan_grad form powers over up to
 * 64 tokens at once: where one passes f32's range, states and gradients become inf or NaN, zeros among them, that token by
 * token would be finite.)  A value that is not finite goes where
 * the rule takes it: one of x or dt into its channel, one of B into its group's channels, from its
 * token on; one of C or z into its token.  A power below 2^-126 is 0. */
typedef struct {
    uint32_t dtype;         /* of x, dt, z, b, c and out */
    uint32_t rows;          /* tokens */
    uint32_t channels;      /* at most 1,048,576; with several groups a multiple of 64 each */
    uint32_t groups;        /* of B and C: channel i has those of group i / (channels / groups) */
    uint32_t n;             /* 8, 16, 32 or 64 */
    const void* x;          /* row t: `channels` elements at x + t * x_stride */
    const void* dt;
    const void* z;          /* or NULL */
    const void* b;          /* row t: groups * n elements */
    const void* c;
    void* out;
    int64_t x_stride, dt_stride, z_stride, b_stride, c_stride, out_stride;   /* elements from a row to the next, at most 2^22 */
    const float* a;         /* [channels][n] */
    const float* d;         /* [channels], or NULL */
    const float* dt_bias;   /* [channels], or NULL */
} redukt_scan_rows;         /* a and states: 16-byte aligned; the others: as their element types */

/* One token for each of `rows` entries (at most 65,536), as redukt_op_delta_step has it: entry i steps
 * slot slots[i] (NULL: i) of states [n_slots][channels][n] in place; -1 leaves the entry's output and
 * state as they are; a slot out of range, or that an earlier entry names, touches no state and its
 * output row becomes NaN. */
int32_t redukt_op_scan_step(const redukt_scan_rows* a, float* states, uint32_t n_slots, const int32_t* slots, void* stream);

/* Whole sequences: cu, slots, state_in, state_out, workspace and rows of no sequence are
 * redukt_op_delta_chunk's.  A sequence's results depend on nothing else in the call. */
int32_t redukt_op_scan_chunk(const redukt_scan_rows* a, const int32_t* cu, uint32_t n_seq, const float* state_in,
                             float* state_out, uint32_t n_slots, const int32_t* slots, void* workspace,
                             uint64_t workspace_bytes, void* stream);

/* The bytes of workspace for these rows (only the sizes are read); 0 if the sizes are not ones that
 * scan_chunk takes, or need none.  With pieces of 64 rows (32 from n = 32 on) at most 4 channels (n + 1) times the smaller of
 * 2 rows / piece and rows / piece + n_seq. */
uint64_t redukt_op_scan_chunk_workspace(const redukt_scan_rows* a, uint32_t n_seq);

/* What the backward pass reads and writes beside the rows: arrays like the ones that they are gradients
 * of, in their types. */
typedef struct {
    const void* dout;       /* row t: `channels` elements */
    void* dx;
    void* ddt;
    void* dz;               /* NULL without z */
    void* db;               /* row t: groups * n elements */
    void* dc;
    int64_t dout_stride, dx_stride, ddt_stride, dz_stride, db_stride, dc_stride;    /* at most 2^22 */
    float* da;              /* [channels][n], 16-byte aligned */
    float* dd;              /* [channels]; NULL without d */
    float* ddt_bias;        /* [channels]; NULL without dt_bias */
} redukt_scan_grads;

/* The gradients of sum(dout * out) + sum(dstate_out * last states) for the sequences cu from the states
 * state_in [n_seq][channels][n] (NULL: zeros), dstate_out alike (NULL: zeros); `out` of the rows is not
 * read.  dstate_in (NULL: not wanted; not one of the others) takes that of the first states.  Rows of no
 * sequence get gradients of zero.  Everything is formed anew from the inputs, sums over channels, tokens
 * and sequences in f32 in a fixed order.  workspace: redukt_op_scan_grad_workspace(a, n_seq) bytes, which are about
 * 4 channels (n + 2) for each sequence, 20 channels (n + 1) at most for each 64 rows (16 to 64 of them in small calls), and 8 n
 * for each row and 64 to 256 channels. */
int32_t redukt_op_scan_grad(const redukt_scan_rows* a, const redukt_scan_grads* g, const int32_t* cu, uint32_t n_seq,
                            const float* state_in, const float* dstate_out, float* dstate_in, void* workspace,
                            uint64_t workspace_bytes, void* stream);
uint64_t redukt_op_scan_grad_workspace(const redukt_scan_rows* a, uint32_t n_seq);

/* ---------------- int8 codes and their product ---------------- */

typedef struct {
    uint32_t dtype;         /* of x */
    uint32_t rows, cols;
    const void* x;          /* row r: cols elements at x + r * x_stride */
    int64_t x_stride;
    int8_t* codes;          /* row r: cols codes at codes + r * codes_stride */
    int64_t codes_stride;
    float* scales;          /* [rows] */
} redukt_quantize_rows;     /* any alignment that the element types have */

/* The library's int8 recipe, row by row: scale = max|x| / 127 (1 where that is 0; NaN does
 * not count), code = x * (1 / scale), each step rounded to f32, to the nearest whole number
 * with halves away from zero, at most 127 in size, 0 for NaN.  x = code * scale, but in rows
 * whose largest magnitude is between 9e-44 and 3.7e-37: there 1 / scale passes f32's range, and
 * what is not 0 becomes 127 or -127.  A row with an infinity has the scale inf and codes of 0. */
int32_t redukt_op_quantize_rows(const redukt_quantize_rows* a, void* stream);

typedef struct {
    uint32_t dtype;         /* of out */
    uint32_t m, n, k;       /* tokens, channels, columns; k at most 131,000 */
    const int8_t* x;        /* token i: k codes at x + i * x_stride */
    int64_t x_stride;
    const float* x_scales;  /* [m] */
    const int8_t* w;        /* channel j: k codes at w + j * w_stride */
    int64_t w_stride;
    const float* w_scales;  /* [n] */
    const float* bias;      /* [n], or NULL */
    void* out;              /* token i: n elements at out + i * out_stride */
    int64_t out_stride;
} redukt_int8_matmul;       /* any alignment that the element types have */

/* out[i][j] = (sum over c of x[i][c] * w[j][c]) * (x_scales[i] * w_scales[j]) + bias[j]: the sum
 * exact in 32-bit integers, the rest in f32, rounded once to `dtype`.  Fastest where x, w and
 * their strides are multiples of 16 bytes and k is a multiple of 16. */
int32_t redukt_op_int8_matmul(const redukt_int8_matmul* a, void* stream);

/* ---------------- e4m3 codes with a scale a block, and their product ---------------- */

typedef struct {
    uint32_t dtype;         /* of x */
    uint32_t rows, cols;
    uint32_t block_rows;    /* rows of a block of 128 columns: 1 (activations) or 128 (weights) */
    const void* x;          /* row r: cols elements at x + r * x_stride */
    int64_t x_stride;
    void* codes;            /* row r: cols bytes (OCP e4m3: no infinities, at most 448) at codes + r * codes_stride */
    int64_t codes_stride;
    float* scales;          /* [ceil(rows / block_rows)][ceil(cols / 128)] */
} redukt_quantize_blocks;   /* any alignment that the element types have; fastest where rows begin on 16 bytes */

/* Block by block: scale = max|x| / 448, at least 2^-126 (NaN does not count), code = x * (1 / scale) to
 * the nearest e4m3 value with halves to the even one, the scale, its inverse and the product each rounded
 * to f32; NaN stays NaN.  x = code * scale.  A block with an infinity has the scale inf, and codes that are 0, or
 * NaN for the infinities. */
int32_t redukt_op_quantize_blocks(const redukt_quantize_blocks* a, void* stream);

typedef struct {
    uint32_t dtype;         /* of out */
    uint32_t m, n, k;       /* tokens, channels, columns; k at most 1,048,576 */
    const void* x;          /* token i: k e4m3 codes at x + i * x_stride */
    int64_t x_stride;
    const float* x_scales;  /* [m][ceil(k / 128)] */
    const void* w;          /* channel j: k e4m3 codes at w + j * w_stride */
    int64_t w_stride;
    const float* w_scales;  /* [ceil(n / 128)][ceil(k / 128)] */
    const float* bias;      /* [n], or NULL */
    void* out;              /* token i: n elements at out + i * out_stride */
    int64_t out_stride;
} redukt_fp8_matmul;        /* any alignment that the element types have */

/* out[i][j] = sum over blocks b of 128 columns (sum over c in b of x[i][c] * w[j][c]) *
 * (x_scales[i][b] * w_scales[j / 128][b]) + bias[j], in an order that the sizes choose, rounded once to `dtype`.
 * f32 outputs: every product is exact, and sums are f32's.
 * 16-bit outputs: the products of columns 8 c to 8 c + 7 are added together, each cut off (toward zero) 13 bits
 * below the exponent of the largest of the eight; all other sums are f32's.  Beside its rounding such an output
 * is off by at most 7 * 2^-13 of the largest product of each eight, times the block's scales, summed over all
 * eights.  Of random codes that is 1.5e-5 of a result; where large products of one eight cancel each other, or
 * the bias cancels them, it can be all that the small ones beside them come to.  Ask for f32 outputs where
 * that matters.
 * Fastest where x, w and their strides are multiples of 16 bytes and k is a multiple of 16. */
int32_t redukt_op_fp8_matmul(const redukt_fp8_matmul* a, void* stream);

/* ---------------- drawing a token ---------------- */

typedef struct {
    uint32_t dtype;         /* of logits */
    uint32_t rows, vocab;   /* vocab 1 to 1,048,576 */
    const void* logits;     /* row r: vocab elements at logits + r * logits_stride */
    int64_t logits_stride;
    const float* u;         /* [rows]: random numbers in [0, 1) */
    float temperature;      /* for every row, unless there are `temperatures` [rows]; and so on */
    float top_p, min_p;
    int32_t top_k;
    const float* temperatures;
    const float* top_ps;
    const float* min_ps;
    const int32_t* top_ks;
    int32_t* tokens;        /* [rows] */
} redukt_sample;            /* any alignment that the element types have */

/* Draws one token of each row.  With l the row's logits and m the largest of them, token i weighs
 * W_i = 2^42 e^((l_i - m) / temperature), rounded to a whole number (2^42 where l_i = m; -inf and NaN weigh
 * nothing).  In the order of falling logits, equal ones by index, are kept: the first top_k (not over 0: all); of
 * these, those before which less than top_p of their sum has come, the first always (not below 1: all); of these, those
 * of W_i >= min_p 2^42 (not over 0: all; over 1: as 1).  The token is the first in the order of indexes up to which
 * the kept weights' sum is over u times the whole one (u below 0 or NaN: as 0; of 1 or more: as just below 1).
 * Sums are exact; a sum and a limit are compared as doubles, the limits each one product of doubles.
 * A temperature that is not over 0 takes the first of the largest logits.  A row without a logit over
 * -inf gets the token -1. */
int32_t redukt_op_sample(const redukt_sample* a, void* stream);

#ifdef __cplusplus
}
#endif
#endif
