/* redukt_ops.h — operators of libredukt_gpu.so on the caller's own device tensors.
 *
 * The plugin ABI (redukt_backend.h) steps the models that the library loads.  The entry
 * points below are the parts of such a layer as operators of their own, for programs that hold
 * activations, weights and recurrent states themselves: the gated delta rule for one token
 * and for whole sequences, and the int8 product with the pass that makes its codes.
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

#ifdef __cplusplus
}
#endif
#endif
