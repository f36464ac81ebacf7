/*
 * ophelia_seq.h -- C ABI of libophelia_seq.so: operators of a text-to-frames sequence model on device tensors, MI355X (gfx950).
 *
 * They stand beside the per-operator entry points of ophelia_hip.h and widen them to training and to device-resident use:
 *   oph_seq_embed*      modules.embed          (modules.py:15-44)      lookup with scaling, and its gradient
 *   oph_seq_recur*      modules.hc's gated mix (modules.py:196-203)    with the previous state in place of the layer's input
 *   oph_seq_attn*       networks.Attention     (networks.py:286-325)   without the monotonic window: any number of heads
 *
 * Conventions
 *   - every tensor pointer is DEVICE memory of `device`; the caller allocates inputs, outputs and workspaces.  A call only launches
 *     kernels on `stream` (a hipStream_t, NULL = the default stream): it neither allocates, copies nor synchronises, so it can be
 *     recorded into a graph.  A workspace may be reused as soon as the launches that were given it have run; two graphs or streams
 *     that can run at the same time need two.
 *   - the calling thread's current device is left as it was.
 *   - dtype: OPH_SEQ_F32 / BF16 / F16 is the type of every activation, gradient and table of a call; statistics, states and sums
 *     are float32.  Strides are in elements and not negative, any layout with unit stride in the last axis; element alignment suffices.
 *   - 0 on success, a negative oph_status (ophelia_hip.h) otherwise (bad arguments: nothing has been launched), and oph_seq_last_error() names
 *     the argument (per thread).  An empty call (no rows) is a success that writes nothing.
 *   - results do not depend on the launch: sums run in a fixed order, there are no floating-point atomics.
 */
#ifndef OPHELIA_SEQ_H
#define OPHELIA_SEQ_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define OPH_SEQ_ABI_VERSION 1
#define OPH_SEQ_F32 0
#define OPH_SEQ_BF16 1
#define OPH_SEQ_F16 2

int oph_seq_abi_version(void);
const char* oph_seq_last_error(void);

/* ---- cross attention --------------------------------------------------------------------------------------------------------
 * q (B,Tq,Hq,D), k, v (B,Tk,Hk,D), Hq a multiple of Hk: query head h reads key head h / (Hq/Hk).  D a multiple of 8, 8..256.
 *   s = scale * q.k over the valid keys, p = softmax(s), out = p.v, lse = log(sum(exp(s)))  (natural logarithm)
 * Keys: key n of sequence b is valid where n < k_lens[b] (NULL: Tk) and mask[b*mask_sb + n*mask_sn] != 0 (NULL: all).  What is not
 * valid is not used, whatever it holds (NaN included).  Queries t >= q_lens[b] (NULL: Tq) are not used either.
 * Rows without a valid query or key: out = 0, lse = -inf, and gradients 0.  Lengths outside 0..T are taken as the nearer bound.
 * out and lse (B,Hq,Tq) are contiguous; so are the gradients dq, dk, dv, of the shapes of q, k, v. */
typedef struct oph_seq_attn {
    const void *q, *k, *v;
    void* out;                       /* forward: written; gradient: the forward's result  */
    float* lse;                      /* the same                                          */
    const void* dout;                /* gradient only, as everything down to dv           */
    void *dq, *dk, *dv;
    const int32_t *q_lens, *k_lens;  /* (B) or NULL                                       */
    const uint8_t* mask;             /* (B,Tk) or NULL                                    */
    int64_t q_stride[3], k_stride[3], v_stride[3], dout_stride[3];   /* of B, T, H         */
    int64_t mask_stride[2];          /* of B, Tk                                          */
    void* workspace;                 /* oph_seq_attn_workspace() bytes, 16-byte aligned; NULL if 0 */
    size_t workspace_bytes;
    int32_t B, Tq, Tk, Hq, Hk, D, dtype;
    float scale;
} oph_seq_attn;
/* bytes of workspace that a call with these sizes and dtype needs; gradient: 0 forward, 1 gradient.  Negative: oph_status. */
int64_t oph_seq_attn_workspace(const oph_seq_attn* a, int gradient);
int oph_seq_attn_forward(const oph_seq_attn* a, int device, void* stream);
int oph_seq_attn_gradient(const oph_seq_attn* a, int device, void* stream);

/* ---- embedding ---------------------------------------------------------------------------------------------------------------
 * ids: n int32 or int64 (id_bytes 4 or 8).  lookup: out (n,units) contiguous = scale * table[id], table (vocab,units) of row stride
 * table_stride.  gradient: grad (vocab,units) contiguous = scale * sum of dout's rows whose id is the row, in float32, in an
 * order that only the call's sizes and dtype decide; rows that no id names are 0.  zero_pad: id 0 reads as zeros and gets no gradient (modules.py:38-40).  An id outside
 * 0..vocab-1 reads as zeros and adds to no row. */
int oph_seq_embed_lookup(const void* ids, int id_bytes, int64_t n, const void* table, int64_t table_stride, int vocab, int units,
                         float scale, int zero_pad, int dtype, void* out, int device, void* stream);
int64_t oph_seq_embed_workspace(int64_t n, int vocab, int units);
int oph_seq_embed_gradient(const void* ids, int id_bytes, int64_t n, const void* dout, int64_t dout_stride, int vocab, int units,
                           float scale, int zero_pad, int dtype, void* grad, void* workspace, size_t workspace_bytes, int device,
                           void* stream);

/* ---- gated linear recurrence ---------------------------------------------------------------------------------------------------
 * x, gate (B,T,C): a = sigmoid(gate), h_t = a_t h_{t-1} + (1 - a_t) x_t from h0 (B,C) float32 (NULL: 0); h (B,T,C) contiguous,
 * h_last (B,C) float32 = the state after the last step.  Steps t >= lens[b] (NULL: T) are not used, leave the state as it is, and
 * have h = 0 and gradients 0.  The gradient takes the forward's h; dh_last (NULL: 0), dh0 float32 (B,C); dx, dgate contiguous.
 * Its states are float32: h itself in OPH_SEQ_F32; in 16 bits, where h is rounded, they are formed again from x, gate and h0, and h's values
 * are not used.
 * h0 may be h_last's buffer (the state of a step-by-step decoder, updated in place). */
typedef struct oph_seq_recur {
    const void *x, *gate;
    const float* h0;
    void* h;                         /* forward: written; gradient: the forward's result, of stride h_stride */
    float* h_last;                   /* forward only                                                         */
    const void* dh;                  /* gradient only, as everything down to dh0                             */
    const float* dh_last;
    void *dx, *dgate;
    float* dh0;
    const int32_t* lens;
    int64_t x_stride[2], gate_stride[2], h_stride[2], dh_stride[2];   /* of B, T */
    void* workspace;                 /* oph_seq_recur_workspace() bytes, 16-byte aligned; NULL if 0 */
    size_t workspace_bytes;
    int32_t B, T, C, dtype;
} oph_seq_recur;
/* bytes of workspace that a call with these sizes and dtype needs; gradient: 0 forward, 1 gradient.  Negative: oph_status. */
int64_t oph_seq_recur_workspace(const oph_seq_recur* a, int gradient);
int oph_seq_recur_forward(const oph_seq_recur* a, int device, void* stream);
int oph_seq_recur_gradient(const oph_seq_recur* a, int device, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* OPHELIA_SEQ_H */
