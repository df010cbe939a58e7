/*
 * vpaged: a paged key/value cache that sequences share, on AMD Instinct MI355X (gfx950): page tables built from the
 * sequences' lengths, the rotation of queries and keys with the keys' and values' way into their pages, and the
 * attention of sequences in groups that share a prefix. A library of its own (libvpaged.so) with a version of its own.
 * No counterpart in the engine, whose cache is contiguous and serves one sequence.
 *
 * Conventions, as in vops.h: every buffer is caller-allocated device memory, the library never allocates or frees;
 * work is enqueued on `stream` (a hipStream_t; NULL = the null stream) and nothing synchronises the host; 0 on
 * success, else a VPAGED_E_* code with vpaged_last_error() (thread-local, valid until the next call on the thread).
 * Calls on different streams may run at once with different plans, workspaces and outputs.
 *
 * A page holds page_size positions (a power of two). Position p of a sequence lies in page table[p / page_size], at
 * its place p % page_size; its slot is page * page_size + place.
 */
#ifndef VPAGED_H
#define VPAGED_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define VPAGED_ABI_VERSION 1

enum vpaged_dtype { VPAGED_BF16 = 0, VPAGED_F16 = 1 };

enum vpaged_status {
  VPAGED_OK = 0,
  VPAGED_E_ARG = 1,       /* a null pointer, a bad size or a stride that does not fit */
  VPAGED_E_DTYPE = 2,     /* dtype not in vpaged_dtype */
  VPAGED_E_HIP = 3,       /* a HIP runtime call failed */
  VPAGED_E_WORKSPACE = 4, /* plan or workspace missing, too small or not 256-byte aligned */
  VPAGED_E_DEVICE = 5     /* the current device is not a gfx950 GPU */
};

#define VPAGED_MAX_PAGE_SIZE 4096
#define VPAGED_MAX_HEAD_DIM 256
#define VPAGED_MAX_HEADS 1024
#define VPAGED_MAX_SEQUENCES 65536
#define VPAGED_MAX_QUERIES 65536
#define VPAGED_MAX_TOKENS 1073741823 /* vpaged_extend */

int vpaged_abi_version(void);

/* 0 if `device` can run the kernels, else a VPAGED_E_* code and a reason in why[0..n) (why may be NULL). */
int vpaged_query(int device, char* why, size_t n);

/* ---- page tables ------------------------------------------------------------------------------------- */

/* The state of a cache's pages: what each sequence holds, and a stack of the pages that nobody holds. Lengths outside
 * [0, max_pages * page_size] and a count outside [0, pages] are taken as the nearest inside. */
typedef struct vpaged_tables {
  int32_t* tables;     /* [sequences, max_pages] */
  int32_t* lengths;    /* [sequences] */
  int32_t* free_pages; /* [pages]: the first free_count are free, the last of them is taken first */
  int32_t* free_count; /* [1] */
  int32_t sequences;   /* 0 .. VPAGED_MAX_SEQUENCES */
  int32_t max_pages;   /* >= 1; sequences * max_pages < 2^31 */
  int32_t pages;       /* >= 1; pages * page_size < 2^31 */
  int32_t page_size;
} vpaged_tables;

/* Each sequence s grows by counts[s] positions (below 0: 0), the sequences in their order taking the pages that they
 * need. A sequence is served whole or not at all: not where its table would be too short, where its tokens lie past
 * `tokens`, or where the pages that it and those before it need are more than are free; served[s] says so (1 where it
 * asks for nothing, but 0 for all behind tokens that lie past `tokens`). The sequences' tokens lie one after the other,
 * counts[s] of each: slots, positions and sequence of the i-th, or -1 where there is none or its sequence is not served. */
size_t vpaged_extend_workspace_bytes(int32_t sequences, int32_t tokens);
int vpaged_extend(const vpaged_tables* t, const int32_t* counts, int32_t tokens, int32_t* out_slots,
                  int32_t* out_positions, int32_t* out_sequences, uint8_t* out_served, void* workspace,
                  size_t workspace_bytes, void* stream);

/* Sequence s is cut to lengths[s] positions where it is longer (below 0: 0), its last pages go back to the stack: in
 * the reverse order of their taking, so that what one call of vpaged_extend took is laid back as it was. */
int vpaged_shrink(const vpaged_tables* t, const int32_t* lengths, void* stream);

/* ---- rotation and storing ---------------------------------------------------------------------------- */

/* Token i at position p turns each pair (x1, x2) of its query and key heads' first `dim` elements by the angle
 * a = p * frequencies[j] (worked out in 64 bits):
 *   y1 = magnitude (x1 cos a - x2 sin a), y2 = magnitude (x2 cos a + x1 sin a)
 * where pair j is elements (j, j + dim / 2), or (2j, 2j + 1) where `interleaved`; the other elements stay. The turned
 * queries go to out_q, the turned keys and the values into their slots. A token at a position below 0 is none: its
 * row of out_q is 0, and nothing is stored. A slot outside the pages is not stored to. Slots are distinct. */
typedef struct vpaged_rotate_args {
  const void* q; /* `dtype`; token i's head h at i * q_stride + h * q_head_stride (elements), likewise k and v */
  const void* k;
  const void* v;
  int64_t q_stride, k_stride, v_stride;
  int64_t q_head_stride, k_head_stride, v_head_stride;
  void* out_q; /* [tokens, heads, head_dim], not over an input */
  void* k_pages; /* slot (page, place), head h at page * page_stride + place * place_stride + h * head_stride */
  void* v_pages; /* with the same strides */
  int64_t page_stride, place_stride, head_stride;
  const int32_t* positions; /* [tokens] */
  const int32_t* slots;     /* [tokens] */
  const double* frequencies; /* [dim / 2] */
  float magnitude;
  int32_t dtype;
  int32_t tokens;   /* >= 0 */
  int32_t heads;    /* 0 .. VPAGED_MAX_HEADS */
  int32_t kv_heads; /* 0 .. VPAGED_MAX_HEADS */
  int32_t head_dim; /* 1 .. VPAGED_MAX_HEAD_DIM */
  int32_t dim;      /* even, 0 .. head_dim */
  int32_t interleaved;
  int32_t pages;
  int32_t page_size;
} vpaged_rotate_args;

int vpaged_rotate_store(const vpaged_rotate_args* args, void* stream);

/* ---- attention --------------------------------------------------------------------------------------- */

/* Sequences s of `queries` new tokens each, in groups: group g's are [group_starts[g], group_starts[g + 1]), and they
 * share a prefix of prefix_lengths[g] positions. lengths[s] are a sequence's own positions behind it, its new tokens
 * the last of them: token t sees the prefix and own positions up to lengths[s] - queries + t. Where that is below 0
 * there is no such token, and its outputs are 0. What lies behind a sequence's length is not seen, whatever it holds; a
 * value that is not finite at a sequence's own position reaches all of the call's new tokens. Scores are fp32, weights
 * rounded to the values' type. Lengths outside what the tables hold are taken as the nearest inside; group_starts ascend
 * from 0 to sequences.
 *   out[s][t][h] = sum_j softmax_j(scale q[s][t][h] . k[j][h / (heads / kv_heads)]) v[j][h / (heads / kv_heads)] */
typedef struct vpaged_shape {
  int32_t dtype;
  int32_t sequences; /* 0 .. VPAGED_MAX_SEQUENCES */
  int32_t groups;    /* 0 .. VPAGED_MAX_SEQUENCES; 0: no prefixes */
  int32_t queries;   /* 1 .. VPAGED_MAX_QUERIES */
  int32_t heads;     /* a multiple of kv_heads, up to VPAGED_MAX_HEADS */
  int32_t kv_heads;
  int32_t head_dim;  /* a multiple of 8, 8 .. VPAGED_MAX_HEAD_DIM */
  int32_t page_size;
  int32_t max_pages;        /* columns of the sequences' tables */
  int32_t max_prefix_pages; /* of the groups' */
} vpaged_shape;

/* A step's plan, from the lengths on the device: which keys each workgroup takes. Layers of one shape share it, of
 * either type. A shape is refused (0 bytes) whose tiles of a head, or of all heads for each of 256 workgroups (512 for heads
 * of up to 128), or rows are 2^31 and more. */
size_t vpaged_plan_bytes(const vpaged_shape* shape); /* 0: a shape that is refused */
int vpaged_plan(const vpaged_shape* shape, const int32_t* lengths, const int32_t* prefix_lengths,
                const int32_t* group_starts, void* plan, size_t plan_bytes, void* stream);

typedef struct vpaged_attend_args {
  vpaged_shape shape; /* the plan's, with the type of q, the pages and out (a plan knows none) */
  int32_t pages;      /* of the cache; a table's entry outside them is taken as the nearest inside */
  float scale;        /* 2^-126 .. 2^64; scores are fp32, and those past it infinite */
  const void* q; /* sequence s, token t, head h at s * q_stride + t * q_token_stride + h * q_head_stride */
  int64_t q_stride, q_token_stride, q_head_stride; /* elements, multiples of 8, as all strides of q and pages */
  const void* k_pages; /* as in vpaged_rotate_args, 16-byte aligned */
  const void* v_pages;
  int64_t page_stride, place_stride, head_stride;
  const int32_t* tables;        /* [sequences, max_pages], rows table_stride apart */
  const int32_t* prefix_tables; /* [groups, max_prefix_pages] */
  int64_t table_stride, prefix_table_stride;
  void* out; /* [sequences, queries, heads, head_dim] */
  const void* plan;
  void* workspace; /* vpaged_attend_workspace_bytes(), 256-byte aligned; calls that overlap need their own */
  size_t workspace_bytes;
} vpaged_attend_args;

size_t vpaged_attend_workspace_bytes(const vpaged_shape* shape);
int vpaged_attend(const vpaged_attend_args* args, void* stream);

const char* vpaged_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* VPAGED_H */
