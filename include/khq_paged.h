/*
 * khq_paged.h -- C ABI of libkhq_paged.so: an uncompressed fp16 / bf16 KV
 * cache in pages, for many requests at once, on MI355X (gfx950).
 *
 * The multi-request counterpart of khq.h's uncompressed baseline
 * (launch_khq_gqa_attn_fp16, one token of one sequence over one contiguous
 * cache); the reference has no such cache.  A step of a server makes
 * khq_paged_plan once, and khq_qk_norm_rope and khq_paged_attn for each layer.
 *
 * As in khq.h: all pointers are device pointers owned by the caller, launches
 * are asynchronous on `stream` (NULL = the null stream) of the current device,
 * and the return code is 0, -100 for arguments that an entry refuses, -101 for
 * a workspace that is too small, else a positive hipError_t.  Every entry may
 * be captured into a HIP graph; lengths, tables and slots are read on the
 * device, so a replay follows what they hold by then.
 */
#ifndef KHQ_PAGED_H
#define KHQ_PAGED_H

#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

#define KHQ_FP16 0
#define KHQ_BF16 1

/* Sequences of one call at most. */
#define KHQ_PAGED_MAX_SEQ 4096

/* The pages of one layer.  Dim d of KV head h of token t of page p is at
 * k[p * page_stride + t * token_stride + h * head_stride + d], in elements,
 * and at the same place in v: pages [n_pages][page_size][H_kv][head_dim] and
 * [n_pages][H_kv][page_size][head_dim] alike.  k, v and the strides are
 * multiples of 16 bytes.  Slot p * page_size + t names token t of page p;
 * there are less than 2^31 slots. */
typedef struct khq_pages {
    void* k;
    void* v;
    long long page_stride, token_stride, head_stride;
    int n_pages, page_size, H_kv;
    int head_dim; /* 64, 128 or 256 */
    int dtype;    /* KHQ_FP16 or KHQ_BF16 */
} khq_pages;

/* Block tables and slots of one step from the requests' lengths.
 *
 * Request s holds kv_len[s] tokens, in the pages of row s of table
 * i32 [n_seq][table_ld].  q_len[s] > 0: that many tokens are appended;
 * 0: nothing (idle); < 0: it has ended, and its pages go back.  The free pages
 * are a ring free_pages i32 [n_pages]: state[1] of them from entry state[0] on,
 * wrapping.  New pages leave at its front, in the requests' order; those of
 * ended requests join at its end.
 *
 * A request is refused (nothing of it changes) if its tokens would pass
 * table_ld pages or row n_tok of the batch, or if it needs new pages and those
 * of all the requests up to it (refused ones for want of pages among them) are
 * more than there are.
 *
 * Written: the new entries of table; cu_q i32 [n_seq + 1], the first batch row
 * of each request (a refused one has its rows too), none past n_tok;
 * seq_kv i32 [n_seq], the tokens each request's attention runs over, the new
 * ones included (0 for a refused or ended one); kv_out i32 [n_seq] and
 * state_out i32 [2], what kv_len and state are after the step (they may be
 * those arrays themselves); status i32 [1], the number of refused requests;
 * and for each of the n_tok batch rows positions i32 [n_tok] and slots i32
 * [n_tok]: slot -1 for a row of a refused request or behind the last one (a
 * padded batch; its position is 0).
 *
 * A table or free-list entry outside [0, n_pages) gives slot -1. */
int khq_paged_plan(const int* q_len, const int* kv_len, int* table, int table_ld,
                   int* free_pages, const int* state, int n_seq, int n_pages, int page_size,
                   int n_tok, int* cu_q, int* seq_kv, int* kv_out, int* state_out, int* status,
                   int* positions, int* slots, hipStream_t stream);

/* Rows of an attention layer's front. */
typedef struct khq_rows {
    const void* q;         /* [n][H_q][head_dim], NULL: no queries */
    void* q_out;           /* may be q itself */
    const void* k;         /* [n][H_kv][head_dim], NULL: no keys */
    void* k_out;           /* normalised and rotated keys; may be k itself, NULL: none */
    void* k_normed;        /* normalised keys before the rotation; NULL: none */
    const void* v;         /* [n][H_kv][head_dim]; only with pages */
    const float* q_weight; /* f32 [head_dim], NULL: no weight */
    const float* k_weight;
    const int* positions;  /* i32 [n], NULL: pos0 + row */
    const int* slots;      /* i32 [n], with pages */
    /* element strides of a token and a head */
    long long q_token, q_head, q_out_token, q_out_head, k_token, k_head, k_out_token,
        k_out_head, k_normed_token, k_normed_head, v_token, v_head;
    double theta;
    float eps;
    int n, H_q, H_kv, head_dim, rotary_dim, pos0;
    int round_norm; /* 1: normalised values are rounded to the type before the rotation */
    int dtype;
} khq_rows;

/* RMS norm of each query and key head (x / sqrt(mean x^2 + eps), times the
 * weight) and the half-split rotation of its first rotary_dim dims (pairs
 * i, i + rotary_dim / 2; angle position * theta^(-2 i / rotary_dim)) in one
 * pass over n tokens; with pages, row i's rotated keys and its values go to
 * slot slots[i] (no write for a slot outside the cache; what a slot named twice
 * holds is not said).  The many-token form of khq_layer_attention_step's front.
 * rotary_dim: a multiple of 16, 0 for no rotation.  Outputs overlap no input but
 * their own, and pages whose slots share memory are refused. */
int khq_qk_norm_rope(const khq_rows* rows, const khq_pages* pages, hipStream_t stream);

/* Queries of one attention call. */
typedef struct khq_attn_rows {
    const void* q;    /* [n_tok][H_q][head_dim] */
    const void* gate; /* [n_tok][H_q][head_dim]: out is times sigmoid(gate); NULL: none */
    void* out;        /* [n_tok][H_q][head_dim] */
    const int* cu_q;  /* i32 [n_seq + 1]: sequence s has rows cu_q[s] .. cu_q[s + 1] - 1 */
    const int* seq_kv; /* i32 [n_seq]: its tokens in the cache, its rows' own included */
    const int* table; /* i32 [n_seq][table_ld] */
    void* ws;         /* f32 workspace, 16-byte aligned; NULL: the library's own */
    size_t ws_bytes;
    /* element strides of a token and a head */
    long long q_token, q_head, gate_token, gate_head, out_token, out_head;
    float scale;
    int n_tok, n_seq, H_q, table_ld;
    int max_q; /* the most rows a sequence has; what it says too low or high costs only time */
} khq_attn_rows;

/* Attention of the new tokens over the pages: row i of sequence s (of n_q
 * rows) sees the sequence's first seq_kv[s] - n_q + i + 1 tokens, so a single
 * row sees them all; query head h reads KV head h / (H_q / H_kv).  A row that
 * sees none is 0.  Rows of no sequence (a padded batch) are left as they were; a
 * sequence that starts or ends outside the batch has those inside, or none if it
 * starts below 0 or ends before it starts; what rows of two sequences hold is
 * not said.
 * A table entry outside [0, n_pages) among the tokens a row's sequence holds
 * makes rows that see it NaN; nothing outside the cache is read.
 *
 * Keys are split over the chip where rows are few, and the parts joined in a
 * fixed order: results do not change from run to run.  The parts live in ws;
 * with ws NULL in the library's workspace, which khq_workspace_reserve grows
 * before a capture: two graphs that share it must not run at once, and those
 * that may have a ws each (khq_paged_attn_ws_bytes says how large).  Calls of
 * several threads take the library's in turn.
 * n_tok * H_q is below 2^27, n_seq * H_kv at most 2^21, scale finite. */
int khq_paged_attn(const khq_attn_rows* rows, const khq_pages* pages, hipStream_t stream);

/* Bytes of workspace that khq_paged_attn uses for these sizes, whatever the
 * lengths on the device; negative for sizes that it refuses. */
long long khq_paged_attn_ws_bytes(int n_tok, int n_seq, int H_q, int H_kv, int head_dim, int max_q);

#ifdef __cplusplus
}
#endif

#endif /* KHQ_PAGED_H */
