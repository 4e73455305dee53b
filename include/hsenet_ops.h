/* libhsenet_ops.so — C ABI of the operators that stand beside the dual-encoder path of libhsenet_hip.so: rotary positions with several
 * axes, differential attention, AdamW over many tensors.  They are a library of their own so that the encoder library, whose measured
 * counters are tied to its content hash (hs_build_id), does not change when an operator is added.
 *
 * The conventions are those of hsenet_hip.h: raw DEVICE pointers, sizes and a hipStream_t (as void*); an int status (HS_OK or a negative
 * HS_ERR_*) is returned and nothing is launched on an error; no entry point allocates, frees or synchronises (graph-capture safe);
 * callers own every buffer, workspaces included.  Every call enqueues on the CURRENT device, whose stream `stream` has to be.
 * Strides are in elements.  dtype: HS_PREC_BF16, HS_PREC_F16 or HS_PREC_F32 (hsenet_hip.h). */
#ifndef HSENET_OPS_H
#define HSENET_OPS_H
#include "hsenet_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A consumer checks hs_ops_version() == HS_OPS_ABI_VERSION at load time.  hs_ops_build_id: content hash of the sources, headers and flags. */
#define HS_OPS_ABI_VERSION 1
int hs_ops_version(void);
const char* hs_ops_build_id(void);

/* ---- rotary positions with several axes (the slice, row and column of a token of a volume; time, height, width of a video).
 * A head's first 2 * pairs columns are `pairs` points (x, y) of a plane: columns (j, j + pairs), or (2j, 2j + 1) with interleaved != 0.
 * Point j is turned by the angle positions[axis[j]] * freq[j], held in 64 bits until it is reduced to one turn; `inverse` turns back
 * (the gradient of the turn).  Columns behind 2 * pairs are copied.  One or two tensors [B][N][heads[i]][dh] (q and k: heads[1] = 0
 * for one) in one launch, each with strides of its own; a column's stride is 1.  y may be x (in place, equal strides); apart from that
 * they do not overlap.  positions: int32, int64 or float32 [axes][B][N] (strides of 0 broadcast).  freq: double [pairs], axis: int32
 * [pairs], entries in [0, axes) (device).  dh is at most 4096, heads[0] + heads[1] at most 4096, their product at most 2^18. */
#define HS_POS_I32 0
#define HS_POS_I64 1
#define HS_POS_F32 2
#define HS_ROTARY_MAX_PAIRS 512
typedef struct hs_rotary_desc {
    uint32_t struct_size;      /* sizeof(hs_rotary_desc) of the caller's header */
    int B, N, dh, pairs, axes;
    int heads[2];
    int interleaved, inverse, dtype, pos_dtype;
    int64_t x_b[2], x_n[2], x_h[2];      /* strides of batch entry, token, head */
    int64_t y_b[2], y_n[2], y_h[2];
    int64_t pos_a, pos_b, pos_n;
} hs_rotary_desc;
int hs_rotary_axes(const hs_rotary_desc* desc, const void* x0, void* y0, const void* x1, void* y1, const void* positions,
                   const double* freq, const int32_t* axis, void* stream);

/* ---- differential attention: o = softmax(scale q1 k1^T) v - lam[h] softmax(scale q2 k2^T) v.
 * q: [B][Nq][2 H][d], heads 2h and 2h + 1 are the two queries of head h; k: [B][Nk][2 Hkv][d] likewise; v: [B][Nk][Hkv][2 d];
 * head h reads key head h / (H / Hkv).  d is 32, 64 or 128; scale between 1e-30 and 1e6; dtype bf16 or fp16; lam: fp32, lam[h * lam_stride] (0: one for all heads).
 * kv_len (device, or NULL: Nk): the first kv_len[b] keys of batch entry b count, 0 to Nk (values outside are clamped).  causal: query i of
 * entry b sees the keys j <= q_start[b] + i (q_start NULL: q_start0).  A query that sees no key gets zeros, and no gradient comes from it.
 * What lies in k and v behind kv_len[b], or at keys that no query of the entry sees, and in q and d_o at queries that see no key, is never used, whatever
 * it holds.
 * o: [B][Nq][H][2 d], dense.  For a backward pass: maps: dense [2][B][Nq][H][2 d], the two maps' own outputs; lse: fp32 [B][H][4][Nq].
 * The strides of q, k, v and of d_o (see below) are multiples of 8 elements, their bases 16-byte aligned, a column's stride is 1; tokens and heads
 * lie at most 2^24 elements apart. */
typedef struct hs_diff_attn_desc {
    uint32_t struct_size;
    int B, Nq, Nk, H, Hkv, d;
    int dtype, causal, q_start0, lam_stride;
    float scale;
    int64_t q_b, q_n, q_h;
    int64_t k_b, k_n, k_h;
    int64_t v_b, v_n, v_h;
    int64_t go_b, go_n, go_h;            /* d_o's strides (hs_diff_attn_bwd) */
} hs_diff_attn_desc;
/* bytes of workspace of the forward (0 where none is needed) and backward pass; both are 0 for a bad descriptor */
size_t hs_diff_attn_fwd_ws_bytes(const hs_diff_attn_desc* desc);
size_t hs_diff_attn_bwd_ws_bytes(const hs_diff_attn_desc* desc);
int hs_diff_attn_fwd(const hs_diff_attn_desc* desc, const void* q, const void* k, const void* v, const float* lam, const int32_t* q_start,
                     const int32_t* kv_len, void* o, void* maps, float* lse, void* ws, size_t ws_bytes, void* stream);
/* dq, dk, dv: dense, in the layouts of q, k, v; dlam: fp32 [H] (one number with lam_stride 0).  All are written whole.  No atomics: equal
 * inputs give equal bits.  fp16: the products' gradients are held times 2^4, the second map's for dk with lam in them, so
 * |P (dP - D)| max(1, |lam|) has to stay under 4094; so has 1 + |lam|, for dv. */
int hs_diff_attn_bwd(const hs_diff_attn_desc* desc, const void* q, const void* k, const void* v, const float* lam, const int32_t* q_start,
                     const int32_t* kv_len, const void* d_o, const void* maps, const float* lse, void* dq, void* dk, void* dv, float* dlam,
                     void* ws, size_t ws_bytes, void* stream);

/* ---- AdamW over many tensors: for every element
 *   p *= 1 - lr * weight_decay;  m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2;
 *   p -= lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
 * with t = the tensor's own step count.  p and g are of `dtype` (arithmetic in fp32, p rounded once at the end).  state_bits 32: m, v
 * fp32.  state_bits 8: blocks of HS_ADAMW_BLOCK consecutive elements (from the tensor's first) with an fp32 scale each, s_m = max |m| and
 * s_u = max sqrt(v) of the block: m is held as int8 c = sign(m) rint(127 sqrt(|m| / s_m)), standing for s_m (c / 127) |c / 127|, and sqrt(v)
 * as uint8 c = max(1 where v > 0, rint(255 sqrt(sqrt(v) / s_u))), standing for s_u (c / 255)^2.  A square-root scale keeps small moments
 * apart: the smallest step is 6e-5 (m) and 1.5e-5 (sqrt v) of the block's largest, and a v > 0 never becomes 0.  The step uses the new
 * moments before they are rounded to 8 bits.  A value that is not finite makes its block's scale NaN.
 * tensors: HOST array of `count` entries (read before the call returns).  step: device, 4 x 32 bits, 16-byte aligned: [0] int32 steps done (raised by
 * the call), [1..2] scratch; a capture replays with the count going on.  A tensor of 0 elements is allowed.  The tensors of one call are disjoint. */
#define HS_ADAMW_BLOCK 256
typedef struct hs_adamw_tensor {
    void* p; const void* g; void* m; void* v; float* m_scale; float* v_scale; int32_t* step; int64_t n;
} hs_adamw_tensor;
int hs_adamw_multi(const hs_adamw_tensor* tensors, int count, int dtype, int state_bits, double lr, double beta1, double beta2, double eps,
                   double weight_decay, void* stream);
/* the moments (m, v) that 8-bit states stand for: fp32 or bf16, one pair of outputs per entry (out_m = p, out_v = g of the table's entry;
 * step is not used). */
int hs_adamw_moments(const hs_adamw_tensor* tensors, int count, int out_dtype, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* HSENET_OPS_H */
