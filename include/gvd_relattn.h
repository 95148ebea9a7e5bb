/*
 * gvd_relattn.h -- C-ABI of attention with a learned relative position bias by buckets (csrc/relattn_forward.hip, relattn_backward.hip).
 *
 * Plain C: raw DEVICE pointers, sizes, hipStream_t as void*.  Every function returns 0 on success or a negative code
 * (gvd_relattn_last_error() has the message, per thread).  Nothing is allocated, kept or synchronised; every launch is on `stream`; results
 * do not depend on the order in which workgroups run.
 *
 *     s_ij = scale q_i . k_j + table[bucket(j - (start_b + i)), h],   seen: j < len_b, and j <= start_b + i where causal
 *     out_i = sum_j softmax_j(s_ij) v_j;  zeros where i sees nothing
 *
 * A table entry at or below -10000 masks its bucket: i does not see j there.  An entry above 10000 counts as 10000.  Neither has a gradient.
 *
 * bucket(d) of a distance d: side = both ? buckets / 2 : buckets; n = both ? |d| : max(-d, 0); the last k < side with first[k] <= n, plus side where
 * both and d > 0.  Keys and values behind len_b are not read into any result.
 */
#ifndef GVD_RELATTN_H_INCLUDED
#define GVD_RELATTN_H_INCLUDED

#ifdef __cplusplus
extern "C" {
#endif

#define GVD_RELATTN_MAX_SIDE 128      /* buckets of one side */
#define GVD_RELATTN_MAX_REACH 1024    /* first[side - 1]: from this distance on all share a bucket */

typedef struct gvd_relattn_problem {
    int B, H, Nq, Nk, D;              /* batch, heads, queries, keys, channels of a head: 64 */
    int is_bf16;                      /* q, k, v, out, d_out, dq, dk, dv: 0 fp16, 1 bf16 */
    int table_type;                   /* table, dtable [buckets, H], contiguous: 0 float, 1 fp16, 2 bf16 */
    int buckets, both, causal;
    const int* first;                 /* HOST array of side whole numbers, first[0] = 0, not descending */
    float scale;                      /* > 0 */
    int q_start;                      /* position of query 0 where q_starts is NULL */
    const int* q_starts;              /* device int[B] or NULL; forward only */
    const int* kv_lens;               /* device int[B] or NULL; values outside 0 .. Nk are brought inside */
    /* element (batch b, row n, head h, channel d) lives at b * bs + n * rs + h * 64 + d; strides in elements, multiples of 8; k and v (dk and dv) share
     * theirs, and so do q and dq, out and d_out.  kv_bs = 0 shares one K / V between all batch entries (forward only). */
    long long q_bs, q_rs, kv_bs, kv_rs, o_bs, o_rs;
} gvd_relattn_problem;

/* Bytes of device workspace that gvd_relattn_fwd / gvd_relattn_bwd need for this problem (0 where none); negative: an error. */
long long gvd_relattn_fwd_workspace(const gvd_relattn_problem* p);
long long gvd_relattn_bwd_workspace(const gvd_relattn_problem* p);

/* lse: NULL, or float [B, H, Nq] that receives the log2-domain log-sum-exp of each row (+infinity where it sees nothing), which the backward needs. */
int gvd_relattn_fwd(const gvd_relattn_problem* p, const void* q, const void* k, const void* v, const void* table, void* out, float* lse,
                    void* workspace, void* stream);

/* Gradients of q, k, v and the table from d_out, with `out` and `lse` of the forward.  All of dq, dk, dv, dtable are written (rows of dk, dv behind
 * len_b with zeros).  d_out of a query that sees nothing goes into no result.  The table's gradient is summed in a fixed order. */
int gvd_relattn_bwd(const gvd_relattn_problem* p, const void* q, const void* k, const void* v, const void* table, const void* out, const void* d_out,
                    const float* lse, void* dq, void* dk, void* dv, void* dtable, void* workspace, void* stream);

const char* gvd_relattn_last_error(void);

#ifdef __cplusplus
}
#endif
#endif
