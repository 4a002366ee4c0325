/* nesle_memory.h -- operators of a policy with memory, of libnesle_hip.so.
 *
 * Plain C over device pointers; work is enqueued on the caller's HIP stream
 * (nothing is allocated, nothing synchronises, no memset: every call may be
 * captured in a graph).  Status codes and nesle_last_error() are those of
 * nesle_hip.h.  No counterpart in the reference, whose policies see one
 * instant.
 *
 * Tensors are time-major: [steps][batch][heads][dim], a rollout of `batch`
 * consoles.  Queries, keys, values and gradients that the caller hands in may
 * be strided (a slice of one projection's output) as long as the elements of
 * a head lie next to each other; what a call writes is contiguous, and lies,
 * as states and workspaces do, on 16-byte boundaries.
 */
#ifndef NESLE_MEMORY_H
#define NESLE_MEMORY_H

#include <stdint.h>

#include "nesle_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of queries, keys, values, outputs and their gradients. */
#define NESLE_MEM_F32 0u
#define NESLE_MEM_BF16 1u

/* Largest head dimension (a multiple of 8) of the norm and of the rule. */
#define NESLE_QK_MAX_DIM 256u
#define NESLE_DELTA_MAX_DIM 128u
/* Tokens of one chunk of the rule: it keeps one state per chunk for the gradient. */
#define NESLE_DELTA_CHUNK 32u

/* A [steps][batch][heads][dim] tensor: strides in elements, the last one 1. */
typedef struct nesle_heads {
    const void* data;
    int64_t stride_t, stride_n, stride_h;
} nesle_heads;

/* ---- norms of queries and keys for each head, with the position rotation ----
 *
 * For each head x of q and k, with w the weight of its kind (null: 1):
 *   y = x * w / sqrt(mean(x^2) + eps)      (unit: sum(x^2) in place of mean)
 * then each pair (y[i], y[i + rotated/2]) (interleaved: (y[2i], y[2i + 1])) of
 * the first `rotated` elements is turned by the angle whose cosine and sine
 * are table[position][i] and table[position][rotated/2 + i].  Everything in
 * float32, rounded once on output.  A position outside 0..table_rows-1 makes
 * its rows NaN. */
typedef struct nesle_qk_args {
    uint32_t dtype;
    uint32_t steps, batch, q_heads, k_heads, dim;
    uint32_t rotated;            /* multiple of 8, 0..dim; 0: no rotation */
    uint32_t unit, interleaved;
    float eps;
    nesle_heads q, k;
    const float* q_weight;       /* [dim], or null */
    const float* k_weight;
    const int32_t* positions;    /* [steps][batch], or null without rotation */
    const float* table;          /* [table_rows][rotated] */
    uint32_t table_rows;
    void* q_out;                 /* forward */
    void* k_out;
    nesle_heads dq_out, dk_out;  /* gradient: of the outputs, in */
    void* dq;                    /*           of the inputs, out */
    void* dk;
    float* dq_weight;            /*           [dim] each; null where the weight is */
    float* dk_weight;
    float* scratch;              /*           nesle_qk_scratch_floats() floats */
} nesle_qk_args;

/* 0 where no scratch is needed, and for dimensions that the calls refuse. */
uint64_t nesle_qk_scratch_floats(const nesle_qk_args* args);
int nesle_qk_norm_rotate(const nesle_qk_args* args, void* stream);
int nesle_qk_norm_rotate_grad(const nesle_qk_args* args, void* stream);

/* ---- the gated delta rule --------------------------------------------------
 *
 * Each head of each console holds a state S [k_dim][v_dim] in float32.  One
 * token, with a = exp(g):
 *   S <- a S                                  (S <- 0 where resets != 0)
 *   S <- S + k (beta (v - S^T k))^T
 *   out = scale S^T q
 * A reset, and a gate whose exp(g) is zero in float32, drop the state by
 * selection: no value of it reaches a later token.  Value head h uses query
 * and key head h / (v_heads / k_heads). */
typedef struct nesle_delta_args {
    uint32_t dtype;
    uint32_t steps, batch, k_heads, v_heads, k_dim, v_dim;
    float scale;
    nesle_heads q, k, v;
    const float* g;              /* [steps][batch][v_heads] */
    const float* beta;           /* [steps][batch][v_heads] */
    const uint8_t* resets;       /* [steps][batch], or null */
    const float* state;          /* [batch][v_heads][k_dim][v_dim], or null: zeros */
    void* out;                   /* [steps][batch][v_heads][v_dim] */
    float* state_out;            /* as state; nesle_delta_step: may be state itself */
    float* saved;                /* forward writes, gradient reads; null where no gradient follows */
    nesle_heads dout;            /* gradient: of out, in */
    const float* dstate_out;     /*           of state_out, in; null: zeros */
    void* dq;                    /*           out */
    void* dk;
    void* dv;
    float* dg;
    float* dbeta;
    float* dstate;               /*           null: not wanted */
    float* scratch;              /* nesle_delta_forward: nesle_delta_forward_scratch_floats() floats;
                                    gradient: nesle_delta_scratch_floats(); unused where that is 0 */
} nesle_delta_args;

/* Floats of `saved`, and of `scratch` of the forward and of the gradient. */
uint64_t nesle_delta_saved_floats(const nesle_delta_args* args);
uint64_t nesle_delta_forward_scratch_floats(const nesle_delta_args* args);
uint64_t nesle_delta_scratch_floats(const nesle_delta_args* args);

/* One token (steps 1) for every console; state_out may be state (in place). */
int nesle_delta_step(const nesle_delta_args* args, void* stream);
/* A rollout in chunks of NESLE_DELTA_CHUNK tokens, and its gradient. */
int nesle_delta_forward(const nesle_delta_args* args, void* stream);
int nesle_delta_backward(const nesle_delta_args* args, void* stream);

/* ---- linear attention with a decay for each head ------------------------------
 *
 * Each head of each console holds a state S [k_dim][v_dim] in float32.  One
 * token, with a = exp(g) of its head:
 *   S <- a S                                  (S <- 0 where resets != 0)
 *   S <- S + k v^T
 *   out = scale S^T q
 * A reset, and a decay whose exp(g) is zero in float32, drop the state by
 * selection.  Value head h uses query and key head h / (v_heads / k_heads).
 * A g above 0 is taken as it is; from where exp(n g) overflows float32, for n
 * tokens of a chunk (64), or of the few chunks that a long walk is cut into,
 * without an episode's end among them, results are unspecified until one ends.
 * `saved` has the same size and layout whatever the strides of either call. */
#define NESLE_DECAY_MAX_DIM 128u

typedef struct nesle_decay_args {
    uint32_t dtype;
    uint32_t steps, batch, k_heads, v_heads, k_dim, v_dim;
    float scale;
    nesle_heads q, k, v;
    const float* g;              /* [v_heads] */
    const uint8_t* resets;       /* [steps][batch], or null */
    const float* state;          /* [batch][v_heads][k_dim][v_dim], or null: zeros */
    void* out;                   /* [steps][batch][v_heads][v_dim] */
    float* state_out;            /* as state; nesle_decay_step: may be state itself */
    float* saved;                /* forward writes, gradient reads; null where no gradient follows */
    nesle_heads dout;            /* gradient: of out, in */
    const float* dstate_out;     /*           of state_out, in; null: zeros */
    void* dq;                    /*           out */
    void* dk;
    void* dv;
    float* dg;                   /*           [v_heads]; null: not wanted */
    float* dstate;               /*           null: not wanted */
    float* scratch;              /* nesle_decay_forward: nesle_decay_forward_scratch_floats() floats;
                                    gradient: nesle_decay_scratch_floats(); unused where that is 0 */
} nesle_decay_args;

/* Floats of `saved`, and of `scratch` of the forward and of the gradient. */
uint64_t nesle_decay_saved_floats(const nesle_decay_args* args);
uint64_t nesle_decay_forward_scratch_floats(const nesle_decay_args* args);
uint64_t nesle_decay_scratch_floats(const nesle_decay_args* args);

/* One token (steps 1) for every console; state_out may be state (in place). */
int nesle_decay_step(const nesle_decay_args* args, void* stream);
/* A rollout in chunks, and its gradient. */
int nesle_decay_forward(const nesle_decay_args* args, void* stream);
int nesle_decay_backward(const nesle_decay_args* args, void* stream);

/* ---- layer norm ------------------------------------------------------------------
 *
 * For each row x of `dim` elements, with statistics in float32:
 *   y = (x - mean) / sqrt(mean((x - mean)^2) + eps) * weight + bias
 * (null: 1 and 0), rounded once on output.  Rows are [steps][batch][heads]. */
#define NESLE_NORM_MAX_DIM 16384u

typedef struct nesle_norm_args {
    uint32_t dtype;
    uint32_t steps, batch, heads, dim;
    float eps;
    nesle_heads x;
    const float* weight;         /* [dim], or null */
    const float* bias;           /* [dim], or null */
    void* y;                     /* forward */
    nesle_heads dy;              /* gradient: of y, in */
    void* dx;                    /*           of x, out */
    float* dweight;              /*           [dim] each; null: not wanted */
    float* dbias;
    float* scratch;              /*           nesle_norm_scratch_floats() floats */
} nesle_norm_args;

/* 0 where no scratch is needed, and for sizes that the calls refuse. */
uint64_t nesle_norm_scratch_floats(const nesle_norm_args* args);
int nesle_layer_norm(const nesle_norm_args* args, void* stream);
int nesle_layer_norm_grad(const nesle_norm_args* args, void* stream);

/* ---- sampling of actions from given random numbers --------------------------------
 *
 * For each row of `actions` scores, in float64 throughout:
 *   s = logits / temperature,  w = exp(s - max s)
 *   of the rows' actions in order of falling s, equal ones by rising index, w is
 *   set to 0 from the top_k-th on (top_k 0: nowhere); then where the sum of those
 *   before is no less than top_p times the sum of all; and where w < min_p
 *   action = the first, by index, at which the running sum of w exceeds
 *            uniform times the sum of all
 *   logprob = log(w[action] / sum w)
 * Temperature 0 takes the largest logit (the lowest index of equal ones), with
 * logprob 0.  A row without an answer gets action -1 and logprob NaN: one whose
 * logits hold NaN or +infinity or nothing above -infinity, whose uniform is NaN,
 * or whose own temperature, top_k, top_p or min_p is out of its range.  A uniform
 * below 0 counts as 0, one of 1 or more picks the last action that is left. */
#define NESLE_SAMPLE_MAX_ACTIONS 1024u

typedef struct nesle_sample_args {
    uint32_t dtype;
    uint32_t steps, batch, actions;
    nesle_heads logits;          /* [steps][batch][actions]; stride_h is not used */
    const float* uniform;        /* [steps][batch] */
    double temperature;          /* 0 or more, finite */
    double top_p;                /* above 0, up to 1 */
    double min_p;                /* 0 to 1 */
    uint32_t top_k;              /* 0 or as many actions as there are, or more: all */
    const float* temperatures;   /* [steps][batch] each, or null: the row's own */
    const int32_t* top_ks;
    const float* top_ps;
    const float* min_ps;
    int64_t* action;             /* [steps][batch] */
    float* logprob;
} nesle_sample_args;

int nesle_sample(const nesle_sample_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* NESLE_MEMORY_H */
