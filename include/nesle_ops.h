/*
 * nesle_ops.h -- C ABI of the policy-learning operators.
 *
 * Operators of a recurrent actor-critic on the batched core: the 8-bit product
 * that reads RAM observations as they are, the gated delta rule that gives the
 * policy a memory over time, and the Newton-Schulz orthogonalisation of matrix
 * updates.  No counterpart in the reference.
 *
 * All pointers are device memory of `device`, aligned to their elements (a
 * pointer that is not is an invalid argument).  Calls are asynchronous on
 * `stream` (a cudaStream_t as void*, NULL = the legacy default stream), allocate
 * nothing and can be captured in a CUDA graph; scratch memory is the caller's.
 * Status codes and nesle_last_error() are those of nesle_b200.h.
 */
#ifndef NESLE_OPS_H
#define NESLE_OPS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* An output of nesle_int8_linear or nesle_delta_step lies on the memory of another argument, or may: it is told from the first
 * and the last byte of each, and for rows as far apart as one another (two columns of one record) from their place in a row. */
#define NESLE_ERR_OVERLAP 4

#define NESLE_F32 0
#define NESLE_BF16 1
#define NESLE_F16 2

/* Times that a kernel of this file gave up on an internal wait on `device`
 * (its outputs are then invalid); 0 unless something is broken.  Synchronous. */
int nesle_ops_stalls(int device, uint32_t* count);

/* Symmetric quantisation of each row to 8 bits: scale = max|x| / 127, q =
 * round-half-even(x / scale) clamped to [-127, 127], both divisions in IEEE
 * fp32 (the clamp acts where the scale is subnormal); a row whose scale is zero
 * gets zeros.  A row that holds a NaN or an infinity gets that scale, and
 * zeros where x / scale is not a number.  Columns cols..ld_q-1 of q are set to
 * zero (ld_q - cols < 16).  ld_* in elements. */
int nesle_quantize_rows(const void* x, int dtype, uint64_t rows, uint64_t cols, int64_t ld_x, int8_t* q, int64_t ld_q,
                        float* scale, int device, void* stream);

typedef struct nesle_int8_args {
    const void* x;         /* [m][k] 8-bit integers, rows ld_x bytes apart */
    int x_unsigned;        /* x is uint8 (else int8) */
    int64_t ld_x;
    const float* x_scale;  /* [m], or NULL: x_scale_value for every token */
    float x_scale_value;
    const int8_t* w;       /* [n][ld_w] int8, zeros from k to ld_w; ld_w a multiple of 16, 16-byte aligned */
    const uint8_t* w_biased; /* [n][ld_w] the same weights + 128 (read where x is unsigned) */
    int64_t ld_w;
    const float* w_scale;  /* [n] */
    const float* bias;     /* [n] or NULL */
    void* y;               /* [m][n], rows ld_y elements apart */
    int y_dtype;           /* NESLE_F32, NESLE_BF16 or NESLE_F16 */
    int64_t ld_y;
    uint64_t m, k, n;
    int relu;
    void* workspace;       /* nesle_int8_workspace bytes, 16-byte aligned */
    uint64_t workspace_bytes;
    int device;
} nesle_int8_args;

/* y[m][n] = act(x_scale[m] w_scale[n] sum_k x[m][k] w[n][k] + bias[n]); the sum is exact in 32-bit integers, which
 * bounds k: 33,025 for unsigned x (255 * 255 k < 2^31), 131,071 for signed (128 * 128 k < 2^31).  y shares no memory with the
 * other arguments (NESLE_ERR_OVERLAP). */
int nesle_int8_linear(const nesle_int8_args* args, void* stream);
/* Scratch bytes that the call needs (0 where x is 16-byte aligned with rows a multiple of 16 bytes apart). */
uint64_t nesle_int8_workspace(const nesle_int8_args* args);

typedef struct nesle_orth_args {
    const void* x;       /* [batch][rows][cols], any strides (elements) */
    int dtype;           /* NESLE_F32, NESLE_BF16 or NESLE_F16 */
    int64_t stride_b, stride_r, stride_c;
    uint64_t batch, rows, cols;
    int steps;           /* products' rounds, at least 1 */
    double eps;          /* added to the norm */
    void* out;           /* [batch][rows][cols] bf16, contiguous, 16-byte aligned */
    void* workspace;     /* nesle_orth_workspace bytes, 256-byte aligned */
    uint64_t workspace_bytes;
    int device;
} nesle_orth_args;

/* Each matrix divided by its Frobenius norm plus eps, then `steps` times X <- aX + (bA + cA^2) X with A = X X^T (of the
 * smaller side) and (a, b, c) = (3.4445, -4.7750, 2.0315): the singular values move towards 1, the singular vectors stay.
 * Products carry 22 bits.  A matrix whose norm is far below eps keeps fewer, and ends as zero.  A NaN or an infinity makes
 * its matrix NaN. */
int nesle_orthogonalize(const nesle_orth_args* args, void* stream);
uint64_t nesle_orth_workspace(const nesle_orth_args* args);

/* The gated delta rule.  Strides are in elements; the last dimension of q, k and v has stride 1; q, k, v and o have one
 * type.  dk and dv are 1 to 128.  States are fp32, [n][h][dk][dv]. */
typedef struct nesle_delta_step_args {
    const void *q, *k, *v; /* [n][h][dk], [n][h][dk], [n][h][dv] */
    int64_t q_n, q_h, k_n, k_h, v_n, v_h;
    int dtype;
    const float *g, *beta; /* [n][h]: log of the decay, write strength */
    int64_t g_n, g_h, beta_n, beta_h;
    const uint8_t* reset;  /* [n], nonzero: the state counts as zero; or NULL */
    int64_t reset_n;
    float* state;          /* in and out; its dk x dv matrices are contiguous */
    int64_t state_n, state_h;
    void* o;               /* [n][h][dv], contiguous */
    uint64_t n, h, dk, dv;
    float scale;
    int device;
} nesle_delta_step_args;

/* One token of every env and head, with the state updated in place:
 * S0 = reset ? 0 : exp(g) S;  u = beta (v - S0^T k);  S = S0 + k u^T;  o = scale S^T q.
 * o shares no memory with the other arguments (NESLE_ERR_OVERLAP), and state none with the inputs: a head's q and k are read
 * while others' o and state are written.  The states' matrices do not overlap. */
int nesle_delta_step(const nesle_delta_step_args* args, void* stream);

typedef struct nesle_delta_args {
    const void *q, *k, *v; /* [t][n][h][dk], [t][n][h][dk], [t][n][h][dv] */
    int64_t q_t, q_n, q_h, k_t, k_n, k_h, v_t, v_n, v_h;
    int dtype;
    const float *g, *beta; /* [t][n][h] */
    int64_t g_t, g_n, g_h, beta_t, beta_n, beta_h;
    const uint8_t* reset;  /* [t][n], nonzero: token t starts an episode; or NULL */
    int64_t reset_t, reset_n;
    const float* state;    /* before the first token, contiguous; NULL for zeros */
    uint64_t t, n, h, dk, dv;
    float scale;
    void* o;               /* [t][n][h][dv], contiguous */
    float* final_state;    /* or NULL */
    float* errors;         /* nesle_delta_error_floats and nesle_delta_checkpoint_floats floats, 16-byte aligned, that the */
    float* checkpoints;    /* backward pass reads; both NULL where no gradient is wanted */
    /* backward only; contiguous */
    const void* d_o;       /* like o */
    const float* d_final;  /* or NULL for zeros */
    void *dq, *d_k, *d_v;
    float *dg, *dbeta;
    float* dstate;         /* or NULL */
    int device;
} nesle_delta_args;

/* The same over t tokens; and its gradients, of all inputs, from those of o and of the final state.  The backward call
 * takes the forward call's inputs, errors and checkpoints.  The gradient of g is zero at tokens that start an episode.
 * A token that is not finite leaves outputs before it as they are; gradients of its whole episode may not be finite. */
uint64_t nesle_delta_error_floats(const nesle_delta_args* args);
uint64_t nesle_delta_checkpoint_floats(const nesle_delta_args* args);
int nesle_delta_scan(const nesle_delta_args* args, void* stream);
/* Where a few long sequences would leave most of the GPU idle, nesle_delta_split_floats (of the sizes, type and device) is not 0, and a workspace of
 * so many floats (16-byte aligned for speed) lets the scan cut them into segments that run side by side.  NULL: one scan. */
uint64_t nesle_delta_split_floats(const nesle_delta_args* args);
int nesle_delta_scan_split(const nesle_delta_args* args, float* workspace, void* stream);
int nesle_delta_scan_backward(const nesle_delta_args* args, void* stream);

#ifdef __cplusplus
}
#endif
#endif
