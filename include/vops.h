/*
 * vops: operators around the sampler on AMD Instinct MI355X (gfx950): beam search's selection over
 * vocabulary-wide logits, the reordering of the beams' states that follows it, and the distillation loss
 * on a teacher's top entries with its gradient. A library of its own (libvops.so) with a version of its
 * own. No counterpart in the engine, which decodes one sequence at a time and does not train.
 *
 * Conventions, as in vsampler.h: every buffer is caller-allocated device memory unless said otherwise, the
 * library never allocates or frees; work is enqueued on `stream` (a hipStream_t; NULL = the null stream)
 * and nothing synchronises the host; 0 on success, else a VOPS_E_* code with vops_last_error()
 * (thread-local, valid until the next call on the thread). Calls on different streams may run at once with
 * different workspaces and outputs.
 */
#ifndef VOPS_H
#define VOPS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define VOPS_ABI_VERSION 2 /* 2: vops_distill_args.temperature is a double */

enum vops_dtype { VOPS_BF16 = 0, VOPS_F32 = 1 };

enum vops_status {
  VOPS_OK = 0,
  VOPS_E_ARG = 1,       /* a null pointer, a bad size or a stride that does not fit */
  VOPS_E_DTYPE = 2,     /* dtype not in vops_dtype */
  VOPS_E_HIP = 3,       /* a HIP runtime call failed */
  VOPS_E_WORKSPACE = 4, /* workspace missing, too small or not 256-byte aligned */
  VOPS_E_DEVICE = 5     /* the current device is not a gfx950 GPU */
};

#define VOPS_MAX_VOCAB 524288
#define VOPS_MAX_BEAMS 64         /* vops_beam_select */
#define VOPS_MAX_CONTINUATIONS 64 /* its n */
#define VOPS_MAX_REORDER_BEAMS 32
#define VOPS_MAX_ENTRIES 1024     /* vops_distill */
#define VOPS_MAX_DISTILL_SEGMENTS 16777215 /* rows times a row's segments (1 to 64) in a call that goes by segments */
#define VOPS_MIN_TEMPERATURE 1e-6
#define VOPS_MAX_TEMPERATURE 1e6

int vops_abi_version(void);

/* 0 if `device` can run the kernels, else a VOPS_E_* code and a reason in why[0..n) (why may be NULL). */
int vops_query(int device, char* why, size_t n);

/* ---- beam search ------------------------------------------------------------------------------------ */

/* The n best continuations of each request, over its beams w and every id v:
 *   scores[b][w] + logits[b][w][v] - log sum_v' exp(logits[b][w][v'])
 * in descending order, equal scores by ascending beam, then descending logit, then ascending id. A finished
 * beam has one continuation, pad_id with the beam's own score. A beam whose score is not finite has none
 * (its row is not read), nor has a row with a NaN, a +inf or no finite logit, nor a logit of -inf. Where
 * there are fewer than n, the rest is score -inf, beam -1, token -1. Scores are worked out
 * and compared in fp64, equal ones being equal there. A row's sum of exponentials has fp64 terms near its
 * largest and fp32 terms (sums of up to 64) below: its log is off by at most 46 2^-23, for all continuations of
 * the row alike, so that only continuations of different rows that lie nearer than twice that may change
 * places. */
#define VOPS_BEAM_KEEP_SLOTS 1u /* the order of the outputs: a parent's best child takes the parent's place, \
                                 * the others the free places in their order (needs n = beams) */
typedef struct vops_beam_args {
  const void* logits; /* `dtype`; row (b, w) at element b * request_stride + w * beam_stride */
  int32_t dtype;
  int32_t requests; /* 0 .. 65535 */
  int32_t beams;    /* 1 .. VOPS_MAX_BEAMS */
  int32_t vocab;    /* 1 .. VOPS_MAX_VOCAB */
  int64_t request_stride; /* elements, >= 0 (0: one row for all) */
  int64_t beam_stride;
  const float* scores;     /* [requests, beams] */
  const uint8_t* finished; /* [requests, beams], 0 or 1; NULL: none */
  int32_t n;               /* 1 .. VOPS_MAX_CONTINUATIONS */
  int32_t pad_id;
  uint32_t flags;
  uint32_t reserved;
  float* out_scores;   /* [requests, n] */
  int32_t* out_beams;  /* the parents' beams */
  int32_t* out_tokens;
  void* workspace; /* vops_beam_workspace_bytes(), 256-byte aligned; calls that overlap need their own */
  size_t workspace_bytes;
} vops_beam_args;

size_t vops_beam_workspace_bytes(int32_t dtype, int32_t requests, int32_t beams, int32_t vocab, int32_t n);
int vops_beam_select(const vops_beam_args* args, void* stream);

/* ---- reordering states ------------------------------------------------------------------------------- */

/* One tensor of per-slot states, as the caller normalised it: per slot up to 3 outer dimensions (sizes 1
 * where there are fewer), each holding runs of contiguous bytes. The requests' lengths limit the run
 * (length_dim 3, `unit` bytes a position), one outer dimension (0 .. 2), or nothing (-1). No two of its
 * elements may overlap, and no other state of the plan may overlap them. */
typedef struct vops_state {
  void* data; /* slot 0 */
  int64_t slot_stride; /* bytes, as all strides here */
  int64_t stride[3];
  int64_t run; /* bytes of a whole run */
  int64_t unit;
  int32_t size[3];
  int32_t length_dim;
  int32_t max_length;
  int32_t reserved;
} vops_state;

/* In place: slot b * beams + w of every state takes what slot b * beams + parents[b][w] held, up to
 * lengths[b] positions (clamped to [0, max_length]) where the state has a length; what lies beyond keeps its
 * contents. A parent outside [0, beams) leaves its slot as it is (-1, as vops_beam_select writes it, among
 * them). One launch, any mapping, no second buffer. `states` is device memory holding n_states
 * descriptions; max_columns is the largest vops_state_columns() of them. lengths may be NULL when no state
 * has a length. */
int64_t vops_state_columns(const vops_state* state); /* host memory; -1: a description that is refused */
int vops_reorder(const vops_state* states, int32_t n_states, int64_t max_columns, int32_t requests, int32_t beams,
                 const int32_t* parents, const int32_t* lengths, void* stream);

/* ---- distillation ------------------------------------------------------------------------------------ */

/* Per row t, with z = student / temperature, q = softmax(z) and the teacher's entries (ids[t][k], distinct
 * in a row; outside [0, vocab): no entry):
 *   without VOPS_DISTILL_TAIL: p = softmax(teacher / temperature) over the row's entries;
 *   with it: p = exp(teacher), teacher being log-probabilities, and rest = max(0, 1 - sum p) is the share
 *   of the ids that are not listed.
 * loss[t] = weights[t] (sum p (log p - log q) + rest (log rest - log q_rest)), q_rest = 1 - the listed q.
 * grad[t] = d loss[t] / d student[t], rounded to the student's dtype. A row of weight 0 is not read; its
 * loss and gradient are 0. A row without entries has loss 0 and gradient 0, whatever its logits hold. */
#define VOPS_DISTILL_TAIL 1u
typedef struct vops_distill_args {
  const void* student; /* `dtype`, row t at t * row_stride */
  int32_t dtype;
  int32_t rows;    /* >= 0; refused where they make more than VOPS_MAX_DISTILL_SEGMENTS segments (16 million rows
                    * of up to 16384 bf16 or 8192 fp32 logits) */
  int32_t vocab;   /* 1 .. VOPS_MAX_VOCAB */
  int32_t entries; /* 1 .. VOPS_MAX_ENTRIES */
  int64_t row_stride; /* elements, >= 0 (0: one row for all) */
  const int32_t* ids;   /* [rows, entries] */
  const float* teacher; /* [rows, entries] */
  const float* weights; /* [rows]; NULL: 1 */
  double temperature;   /* VOPS_MIN_TEMPERATURE .. VOPS_MAX_TEMPERATURE */
  uint32_t flags;
  float* out_loss; /* [rows] */
  void* out_grad;  /* `dtype`, row t at t * grad_stride, not over the student; NULL: the loss alone */
  int64_t grad_stride;
  float* states; /* NULL, or [rows, 2 + entries]: what vops_distill_grad takes */
  void* workspace;
  size_t workspace_bytes; /* vops_distill_workspace_bytes(), 256-byte aligned */
} vops_distill_args;

size_t vops_distill_workspace_bytes(int32_t dtype, int32_t rows, int32_t vocab, int32_t entries);
int vops_distill(const vops_distill_args* args, void* stream);

/* out_grad alone, from the states that vops_distill wrote for the same student, ids, temperature and flags;
 * weights may be others (a backward pass: the weights times the incoming gradients; a row whose weight was 0
 * there has gradient 0 under any, NaN among them). teacher, out_loss and the workspace are not used. */
int vops_distill_grad(const vops_distill_args* args, void* stream);

const char* vops_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* VOPS_H */
