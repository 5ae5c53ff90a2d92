/* sabrewing_hip.h -- C ABI of the MI355X (gfx950) MoE-block backend,
 * libsabrewing_hip.so.  Plain pointers and sizes only.
 *
 * Three layers of entry points:
 *   1. lag_hip_*            the Laguna backend ABI, entry for entry: same
 *                           arguments, same 0 = ok / -1 = failure convention,
 *                           host activations, device weights from
 *                           lag_hip_upload (c/backend_cuda_laguna.h:25-75).
 *                           The Linux loader (libsabrewing_loader.so,
 *                           include/sabrewing_loader.h) exports them under the
 *                           reference's lag_cuda_* names for unmodified engines.
 *   2. lag_hip_*_g          the same entries for group-scaled int4 (one f32
 *                           scale per gs inputs, the fmt=4 layout of
 *                           c/quant.h:168-203); the reference's lag family is
 *                           per-row only.
 *   3. lag_hip_moe_forward  the whole MoE block with routing on the device
 *                           (router GEMV -> gate -> top-k -> group-by-expert
 *                           -> SwiGLU experts -> combine -> shared expert ->
 *                           residual), device activations, the descriptor of
 *                           c/moe_arch.h:33-41.
 *
 * Like the reference backend: one device and one stream per process (a second
 * lag_hip_init naming another device fails), results
 * valid on return for the host-pointer entries, not thread-safe.
 * COLI_GPU_FAIL_AFTER=N makes every compute entry fail after N successful
 * calls (the reference's fault-injection hook, c/backend_cuda.cu:684-693). */
#ifndef SABREWING_HIP_H
#define SABREWING_HIP_H
#include <stddef.h>
#include <stdint.h>
#ifdef __cplusplus
extern "C" {
#endif

/* ---------------- 1. Laguna backend ABI (replaces c/backend_cuda_laguna.h) ---------------- */
/* lag_cuda_init (c/backend_cuda_laguna.h:25): select device, create the stream. 0 = ok */
int    lag_hip_init(int dev);
/* lag_cuda_free_bytes / lag_cuda_total_bytes (:26-27) */
size_t lag_hip_free_bytes(void);
size_t lag_hip_total_bytes(void);
/* lag_cuda_upload / lag_cuda_free (:28-29): plain byte copy, NULL = error */
void  *lag_hip_upload(const void *h, size_t n);
void   lag_hip_free(void *d);
/* lag_cuda_matmul_bf16 (:32): y[S,O] = x[S,I] @ W^T, W device bf16 [O,I], x/y host f32 */
int    lag_hip_matmul_bf16(float *y, const float *x, const void *W, int S, int I, int O);
/* lag_cuda_matmul_q4 (:39): per-row int4 [O,I/2] + f32 scale [O], nibble-8 */
int    lag_hip_matmul_q4(float *y, const float *x, const void *packed, const void *scale, int S, int I, int O);
/* lag_cuda_expert_q4 (:44): out[D] = W2 @ silu_glu(W13 @ x), gate_up block-concatenated */
int    lag_hip_expert_q4(float *out, const float *x, const void *p13, const void *s13,
                         const void *p2, const void *s2, int I, int D);
/* lag_cuda_moe_experts (:51): out[D] = sum_k w[k] * expert(sel[k], x), layer blobs */
int    lag_hip_moe_experts(float *out, const float *x, const void *gu_q, const float *gu_s,
                           const void *dn_q, const float *dn_s, const int *sel, const float *w,
                           int K, int I, int D);
/* lag_cuda_moe_group (:70): acc[S,D] = rank-order sum over the packed groups */
int    lag_hip_moe_group(float *acc, const float *x, const void *gu_q, const float *gu_s,
                         const void *dn_q, const float *dn_s, const int *gexp, const int *gbeg,
                         const int *gcnt, int G, const int *grow, const int *rowof, const float *w,
                         int S, int K, int I, int D);

/* lag_cuda_matmul_q8 (:36): int8 weights [O,I] followed in the same buffer by
 * their f32 row scales [O] (c/backend_cuda_laguna.cu:125-126) */
int    lag_hip_matmul_q8(float *y, const float *x, const void *W, int S, int I, int O);
/* ink_cuda_matmul_q8 (c/backend_cuda_ink.h:27-28): the same with the scales in
 * their own buffer */
int    lag_hip_matmul_q8_s(float *y, const float *x, const void *q8, const void *scale, int S, int I, int O);
/* ink_cuda_matmul_bf16 (c/backend_cuda_ink.h:17-18): activations rounded to bf16
 * (c/backend_cuda_ink.cu:63-64), in the lane order of the CPU's matmul_h
 * (c/moe_matmul.h:66-89, vdpbf16ps); I % 32 != 0 takes the f32-activation
 * contract, as the CPU does */
int    lag_hip_matmul_bf16_rx(float *y, const float *x, const void *W, int S, int I, int O);
/* Numerics of the host-activation matmuls: every call, whatever its row count,
 * reproduces the reference CPU's SIMD contracts bit for bit -- matmul_bf16 the
 * 16 f32-activation lanes of c/moe_matmul.h:92-110, matmul_q4 (per-row scales)
 * matmul_q4_k's F32 lanes (c/moe_quant.h:85-109), matmul_q8 matmul_q8_k's F32
 * lanes (c/moe_quant.h:378-391), matmul_bf16_rx the vdpbf16ps lanes -- so a
 * token's result does not depend on how many rows share its call. */

/* ---------------- 2. group-scaled int4 forms (scale[o*ng + g], ng = I/gs) ---------------- */
int    lag_hip_matmul_q4_g(float *y, const float *x, const void *packed, const void *scale,
                           int S, int I, int O, int gs);
int    lag_hip_expert_q4_g(float *out, const float *x, const void *p13, const void *s13,
                           const void *p2, const void *s2, int I, int D, int gs);
int    lag_hip_moe_experts_g(float *out, const float *x, const void *gu_q, const float *gu_s,
                             const void *dn_q, const float *dn_s, const int *sel, const float *w,
                             int K, int I, int D, int gs);
int    lag_hip_moe_group_g(float *acc, const float *x, const void *gu_q, const float *gu_s,
                           const void *dn_q, const float *dn_s, const int *gexp, const int *gbeg,
                           const int *gcnt, int G, const int *grow, const int *rowof, const float *w,
                           int S, int K, int I, int D, int gs);

/* ---------------- 3. device-resident MoE block ---------------- */
enum { LAG_HIP_ROUTE_SIGMOID = 0, LAG_HIP_ROUTE_SOFTMAX = 1, LAG_HIP_ROUTE_SOFTPLUS = 2,
       LAG_HIP_ROUTE_SOFTMAX_OLMOE = 3, LAG_HIP_ROUTE_SOFTMAX_QWEN = 4, LAG_HIP_ROUTE_SQRT_SOFTPLUS = 5,
       LAG_HIP_ROUTE_INKLING = 6 };
enum { LAG_HIP_SHARED_NONE = 0, LAG_HIP_SHARED_UNSCALED = 1, LAG_HIP_SHARED_GATED = 3 };

/* MoeDesc (c/moe_arch.h:33-41) plus the layer shape.  route_act: SIGMOID and
 * SOFTMAX are moe_block's (c/moe_block.h:24-26); the others are extensions:
 * SOFTPLUS x > 20 ? x : log1pf(expf(x)) (c/moe_math.h:54); SOFTMAX_OLMOE the
 * OLMoE engine's routing (float-sum softmax, each probability divided by the
 * sum, c/olmoe.c:212-216, 607-632; norm_topk as moe_block's); SOFTMAX_QWEN
 * qwen35's moe_route (double-sum softmax, (float)(p / sum) in double, the
 * picks always renormalised in double, c/qwen35.c:558-589; norm_topk and the
 * correction bias unused); SQRT_SOFTPLUS sqrtf(softplusf(x)), DeepSeek-V4's
 * router score (c/deepseek.c:854), selected and weighted as moe_block's
 * sigmoid scores; INKLING the Inkling engine's moe() routing (c/inkling.c:
 * 1027-1043): a router of n_experts + n_shared rows, the routed sigmoids
 * selected by moe_topk with the correction bias, weights the sigmoids of the
 * K picks and of the n_shared shared gates, each * route_scale / (their float
 * sum), route_scale being the engine's route_scale * gate.global_scale formed
 * in float (norm_topk unused; the routed sum is not scaled again).  The
 * reference wires shared NONE and UNSCALED; GATED (moe_arch.h's
 * MOE_SHARED_GATED, with INKLING only) adds n_shared shared experts after the
 * routed ranks, each output times its gate's weight (c/inkling.c:1166-1183),
 * their matmuls in inkling's matmul_h contract (bf16 weights, bf16-rounded
 * activations): sg and su [n_shared*Is, D], sd [n_shared*D, Is]. */
typedef struct {
    int   n_experts, topk, route_act, use_corr_bias, norm_topk;
    float route_scale;
    int   shared_mode;
    int   hidden, moe_inter, shared_inter, gs;   /* D, I, Is; gs = 0: per-row int4 scale */
    int   router_bf16;                           /* router element type: 1 bf16, 0 f32 */
    int   n_shared;                              /* INKLING: shared gate rows / GATED experts (else 0) */
} LagHipMoeDesc;

/* Device pointers of one layer.  Experts in the reference container layout
 * (c/laguna.c:586-588; docs/laguna.md:34-44); router from lag_hip_router_upload. */
typedef struct {
    const void  *router;
    const float *corr_bias;     /* [E] e_score_correction_bias (selection only) or NULL */
    const float *logit_bias;    /* [E] added to the router logits (a router-hook wrapper) or NULL */
    const void  *gu_q;
    const float *gu_s;
    const void  *dn_q;
    const float *dn_s;
    const void  *sg, *su, *sd;  /* bf16 shared expert [Is,D],[Is,D],[D,Is] or NULL */
} LagHipMoeWeights;

/* Upload a router [E,D] (bf16 or f32, host) into the order the routing
 * kernel streams, in its own element type: experts in groups of 4
 * (E4 = 4*ceil(E/4), the padding experts zero), each group a run of 1 KB
 * slices, slice q holding the next P elements (P = 8 bf16 or 4 f32) of each
 * of its 64 chains c = 16*(e%4) + i%16 (chain element m = i/16):
 * element (e, i) at ((e/4 * D/(16P) + m/P) * 64 + c) * P + m%P.
 * NULL = error.  Free with lag_hip_free. */
void  *lag_hip_router_upload(const void *W, int E, int D, int w_bf16);
/* the same transform from a device router W [E,D] into device Wc
 * (E4*D elements) (0 = ok) */
int    lag_hip_router_chain(const void *W, void *Wc, int E, int D, int w_bf16);
/* out[S,D] += MoE(x[S,D]) for S tokens (device pointers), queued on the
 * backend stream; S == 1 runs the per-token path, S > 1 the grouped path
 * (bit-identical per token).  0 = ok. */
int    lag_hip_moe_forward(const LagHipMoeDesc *d, const LagHipMoeWeights *w, const float *x, float *out, int S);
/* lag_hip_moe_forward without any allocation.  No counterpart in the
 * reference: it is for callers that cannot allocate device memory (code under
 * HIP graph capture, tight serving loops, harnesses that forbid hipMalloc).
 * The scratch of the forward lives in a static device array of
 * LAG_HIP_NOALLOC_SCRATCH_BYTES on each device (held from library load until
 * the process ends) instead of the growing arena; the call makes no
 * hipMalloc/hipFree and no other allocation.  A shape whose scratch does not
 * fit returns -1 before any launch (lag_hip_last_error gives the bytes it
 * needed): the C2 layer (D=4096, E=256, K=10, I=Is=1024) fits up to S = 78
 * (up to S = 66 with lag_hip_set_q4_mode(1) on per-row scales, which also
 * keeps int8 activations and an f32 h).
 * Same results, bit for bit, as lag_hip_moe_forward.  Every call on a device
 * shares that device's array, so calls that overlap on one device race. */
#define LAG_HIP_NOALLOC_SCRATCH_BYTES ((size_t)24 << 20)
int    lag_hip_moe_forward_noalloc(const LagHipMoeDesc *d, const LagHipMoeWeights *w, const float *x, float *out, int S);
/* The device scratch bytes lag_hip_moe_forward(_noalloc) needs for S tokens of
 * this layer in the current q4 mode (0 = unsupported descriptor or shape).
 * Host arithmetic only: callable before lag_hip_init and without a device, so a
 * caller can size its batches to the fixed region above. */
size_t lag_hip_moe_forward_scratch_bytes(const LagHipMoeDesc *d, const LagHipMoeWeights *w, int S);
/* the same with host x/out; synchronous */
int    lag_hip_moe_block(const LagHipMoeDesc *d, const LagHipMoeWeights *w, const float *x, float *out, int S);
/* routing only (device pointers): logits [S,E] (may be NULL), sel [S,K], w [S,K];
 * INKLING: logits [S, E + n_shared], w [S, K + n_shared] (the picks' weights,
 * then the shared gates') */
int    lag_hip_route(const LagHipMoeDesc *d, const LagHipMoeWeights *w, const float *x, int S,
                     float *logits, int *sel, float *wts);
/* the last forward's expert groups: G (host out), gexp/gbeg/gcnt [G] host copies (one token:
 * G alone).  They lie in the backend's scratch: a later call that takes so much of it that it
 * reaches them, or makes it grow, ends them (another forward, a lag_hip_route of more tokens,
 * lag_hip_attn_paged of up to 256 rows, an entry with host pointers), as does the end of a
 * recording; G is 0 from then on. */
int    lag_hip_last_groups(int *G, int *gexp, int *gbeg, int *gcnt, int cap);

/* ---------------- stack glue (device pointers, queued on the backend stream) ----------------
 * A layer of a stack is h += MoE(rmsnorm(h, w_l)) (lag_hip_rmsnorm, then
 * lag_hip_moe_forward with x = the normed rows and out = h); a step ends in
 * rmsnorm, the head and a greedy pick. */
/* out[s] = x[s] / sqrt(mean(x[s]^2) + eps) * w, the squares summed in double
 * (rmsnorm_row, c/moe_math.h:58-62); out may be x.  0 = ok */
int    lag_hip_rmsnorm(const float *x, const float *w, float *out, int S, int D, float eps);
/* One stack layer in one call: xn = rmsnorm(h, norm_w, eps) as lag_hip_rmsnorm (the
 * same bits), then h += MoE(xn) as lag_hip_moe_forward.  No counterpart in the
 * reference (c/laguna.c:1156-1160 calls rmsnorm_row and the block separately); for
 * stack callers: without a shared expert and below 512 tokens the routing launch
 * applies the norm as it stages the rows, one launch fewer per layer.  0 = ok */
int    lag_hip_moe_forward_rmsnorm(const LagHipMoeDesc *d, const LagHipMoeWeights *w, const float *norm_w, float eps,
                                   float *xn, float *h, int S);
/* logits[S,V] = x[S,D] . head^T under the 16-lane contract of the head's
 * resmm -> matmul_bf16 (c/laguna.c:1156-1158; Wc from lag_hip_router_upload
 * of the [V,D] head), and with tok non-null tok[s] = the greedy pick of
 * argmax_logits (strict ascending scan: ties to the lowest index,
 * c/laguna.c:1159).  0 = ok */
int    lag_hip_head_argmax(const void *Wc, int w_bf16, const float *x, int S, int D, int V, float *logits, int *tok);
/* tok[s] = argmax_logits' pick over logits[s, 0..V) alone (c/laguna.c:1159).  0 = ok */
int    lag_hip_argmax(const float *logits, int S, int V, int *tok);

/* ---------------- attention over a paged cache (device pointers, queued on the backend stream) ----------------
 * The attention half of a layer's decode step: the projection's heads normalised, turned and
 * appended to the cache, then one new token of each row against its sequence's cells.  No
 * counterpart in the reference's lag table (its engines keep attention on the CPU). */
enum { LAG_HIP_KV_F32 = 0, LAG_HIP_KV_BF16 = 1, LAG_HIP_KV_F16 = 2 };
/* One layer's cache: pools of n_pages pages of page_size tokens (a power of two, 8 to 4096)
 * of n_heads heads of head_dim values (a multiple of 32, at most 256).  The values of head g,
 * slot i of page p begin at element p * page_stride + g * head_stride + i * token_stride of k
 * and of v; the strides are in elements and a head's values side by side, so a page may be
 * [head][token][value] or [token][head][value], and both pools may lie in one allocation.
 * Pools and strides are multiples of 16 bytes, and cells do not overlap. */
typedef struct {
    void   *k, *v;
    int     type;                               /* LAG_HIP_KV_* */
    int     n_pages, page_size, n_heads, head_dim;
    int64_t page_stride, head_stride, token_stride;
} LagHipKvCache;
/* The rows of a batch (device arrays): row s is the token at position pos[s] of sequence
 * seq[s] (seq NULL: sequence s), whose token t lies in page table[seq * max_pages +
 * t / page_size], slot t % page_size.  pos[s] < 0: a free place, no row.  max_pages *
 * page_size <= 2^30.  What the arrays hold is read on the device, at the time of the launch
 * or replay: a sequence outside [0, n_seqs), a position beyond the table or a page outside
 * the pool has no cell (nothing is written there and nothing attended to). */
typedef struct {
    const int *pos, *seq, *table;
    int n_seqs, max_pages;
} LagHipKvRows;
/* Rotary positions of the first `dims` values of each head (even, 0: none, at most head_dim):
 * pair i, values (i, i + dims/2) or, interleaved, (2i, 2i + 1), turns by pos * freq[i] radians
 * (freq: device, [dims/2] doubles, so that a caller scales them for long contexts as it
 * likes; the angle is taken in 64 bits), times factor. */
typedef struct {
    const double *freq;
    int   dims, interleaved;
    float factor;
} LagHipRope;
/* qkv [S][ld]: row s holds n_q_heads q heads, then n_heads k heads, then n_heads v heads.  q
 * and k heads are normalised, x / sqrt(mean(x^2) + eps) * q_norm or k_norm ([head_dim], NULL:
 * not), and turned; q to q_out [S][n_q_heads][head_dim], k and v rounded to nearest into the
 * row's cell.  n_q_heads is a multiple of n_heads, ld of 4; qkv and q_out are 16-byte aligned
 * and do not overlap.  A free place leaves q_out and the cache as they were; a row whose
 * position has no cell has its q in q_out and leaves the cache.  Two rows of one cell are the
 * caller's mistake (the cell holds values of both).  0 = ok */
int    lag_hip_qk_rope_append(const LagHipKvCache *c, const LagHipKvRows *r, const LagHipRope *rope, const float *qkv,
                              int64_t ld, const float *q_norm, const float *k_norm, float eps, int n_q_heads, float *q_out,
                              int S);
/* out[s][h] = sum_t p_t v_t, p the softmax of scale * q[s][h] . k_t over the cells t <= pos[s]
 * of row s (t > pos[s] - window with window > 0), head h reading cache head h / (n_q_heads /
 * n_heads); q and out [S][n_q_heads][head_dim], 16-byte aligned, not overlapping.  Sums and
 * the softmax in 32 bits.  A free place, or a row without any cell, gives zeros.  Rows of one
 * sequence at consecutive positions (a chunk of a prompt, already appended) each see what is
 * theirs to see.  max_pages * page_size (of f32 caches, or heads over 160, rounded up to
 * a multiple of 16) times S, or 64 if that is less, is below 2^36.
 * Infinities and NaN in a cell reach the rows that attend to it, as values without meaning,
 * and no others; cells that no row attends to may hold anything.  The same call gives the same
 * bits; how a row's cells are cut into parts, and with that its last bits, depends on the
 * batch's positions, S, n_q_heads, window and max_pages * page_size, not on what the other
 * rows' cells hold.  Its scratch is the arena's.  0 = ok */
int    lag_hip_attn_paged(const LagHipKvCache *c, const LagHipKvRows *r, const float *q, int n_q_heads, float scale,
                          int window, float *out, int S);
/* Trees of drafted tokens (device arrays), to be verified in one step: tree i's nodes are rows first[i] ..
 * first[i + 1] - 1 of the batch (first: [n_trees + 1], from 0 on and rising; at most max_nodes of a tree, itself at most 64).
 * base[i] cells of sequence seq[i] (NULL: sequence i) come before the tree, and node j's k and v lie in cell base[i] + j,
 * whatever its depth; bit j of sees[s] says that row s attends to node j of its tree (itself and its ancestors, as a
 * rule).  pos[s] (NULL where no window is used): the row's position, base plus its depth.  base[i] < 0: a free place.  Tables as
 * LagHipKvRows'.  What the arrays hold is read on the device: rows outside the batch, sequences and pages that lead
 * nowhere have no cells. */
typedef struct {
    const int *first, *base, *seq, *pos, *table;
    const uint64_t *sees;
    int n_trees, n_seqs, max_pages, max_nodes;
} LagHipTrees;
/* lag_hip_attn_paged for trees: out[s][h] = sum_t p_t v_t over the cells t < base of row s's tree (with window > 0 those with t >
 * max(pos[s], base) - window) and the cells base + j of the nodes that sees[s] names (whatever the window: a caller whose trees are
 * as deep as it clears the bits of ancestors that it leaves out).  A tree's cells are read once for all of its nodes.  q, out, scale and
 * the accuracy as there; S rows in all.  A row that attends to nothing, or of a free place, gives zeros; rows of no tree are left as they were.  An infinity or NaN in a cell reaches the rows that attend to it, as
 * outputs without meaning, and no others.  max_pages * page_size <= 2^30.  0 = ok */
int    lag_hip_attn_tree(const LagHipKvCache *c, const LagHipTrees *t, const float *q, int n_q_heads, float scale, int window,
                         float *out, int S);
/* lag_hip_qk_rope_append with positions of their own for the turn: row s's q and k turn by at[s], and its cell is that of
 * token r->pos[s] (a tree's node: cell base + j, position base + its depth).  0 = ok */
int    lag_hip_qk_rope_append_at(const LagHipKvCache *c, const LagHipKvRows *r, const int *at, const LagHipRope *rope,
                                 const float *qkv, int64_t ld, const float *q_norm, const float *k_norm, float eps, int n_q_heads,
                                 float *q_out, int S);
/* The accepted path of each tree: from node 0 on, the lowest later node whose parent (parent[s], an index in its tree) is
 * the path's last node and whose drafted token (draft[s]) is the one picked there (tok[s]), until there is none.  Writes
 * path [n_trees][max_nodes] (indices of the path's nodes, then -1), count [n_trees] (its length; a free place or a tree without
 * nodes: 0) and next [n_trees] (the pick at its last node; -1 without one), and moves the cells of the path's nodes together: node
 * path[i]'s k and v to cell base + i, in every one of n_layers caches (one geometry and type).  Cells behind base + count
 * hold what they held.  Cells that lead nowhere are left out.  A tree's cells are its own: no other tree of the call has a node or a path's
 * place in them (one tree of a sequence, in pages that no other holds).  What is written overlaps nothing that is read.  parent, draft, tok: [S].  sees and pos of t are not used.  0 = ok */
int    lag_hip_tree_commit(const LagHipKvCache *layers, int n_layers, const LagHipTrees *t, const int *parent, const int *draft,
                           const int *tok, int *path, int *count, int *next, int S);
/* Page src[i] of every one of n_layers caches (one geometry and type) to page dst[i], k and v:
 * a fork's last page, or pages moved together.  src and dst are host arrays, free to change
 * on return; a dst is named once and is no src.  0 = ok */
int    lag_hip_kv_copy_pages(const LagHipKvCache *layers, int n_layers, const int *src, const int *dst, int n);
/* ---- latent attention: a token's keys and values of all heads come from one vector ----
 * k_t[h] = (Wk[h] c_t, r_t) and v_t[h] = Wv[h] c_t, c_t a latent of `rank` values, r_t a rotary part of `rope_dims` that the
 * heads share.  The cache holds (c_t, r_t) alone.  Two forms of one attention: absorbed, for single new tokens (queries go
 * into the latent space, Wk[h]^T q, outputs come back from it, Wv[h] o: lag_hip_latent_heads before and after
 * lag_hip_attn_latent), and expanded, for a prompt (lag_hip_attn_latent_prompt).  No counterpart in the reference's lag table; the
 * GLM engine's attention slots (include/sabrewing_coli.h) are other entries.
 *
 * One layer's cache: n_pages pages of page_size tokens (a power of two, 8 to 4096), a cell's rank + rope_dims values side
 * by side at c + page * page_stride + slot * token_stride (elements; strides and c multiples of 16 bytes, cells do not overlap).
 * type: LAG_HIP_KV_BF16 or LAG_HIP_KV_F16.  rank: 128, 256, 384 or 512; rope_dims: a multiple of 16 up to 64, or 0. */
typedef struct {
    void   *c;
    int     type, n_pages, page_size, rank, rope_dims;
    int64_t page_stride, token_stride;
} LagHipLatentCache;
/* Heads of rows: the values of row s's head h begin at element s * row_stride + h * head_stride of p. */
typedef struct {
    void   *p;
    int64_t row_stride, head_stride;
} LagHipHeads;
/* S rows (positions and tables as for the paged cache).  ckv [S][ld_c]: rank values, normalised (c / sqrt(mean(c^2) + eps) * norm;
 * norm NULL: not), and rope_dims values, turned (rope NULL: not; its dims rope_dims), both rounded to nearest into the row's
 * cell.  q [S][ld_q]: n_heads heads of `nope` values and a rotary part of rope_dims, rounded to the cache's type: the first to q_nope, the
 * second, turned, to q_rope (for the absorbed form behind the rank values of each head, for the expanded one behind the
 * nope values of the same head).  nope: a multiple of 16 up to 256 or, with n_heads 0 and q NULL, unused.  ckv, q and what is written
 * are 16-byte aligned, strides of inputs multiples of 4 elements, of outputs of 8.  A free place leaves everything as it was, a position without a
 * cell the cache.  0 = ok */
int    lag_hip_latent_append(const LagHipLatentCache *c, const LagHipKvRows *r, const LagHipRope *rope, const float *ckv, int64_t ld_c,
                             const float *norm, float eps, const float *q, int64_t ld_q, int n_heads, int nope, const LagHipHeads *q_nope,
                             const LagHipHeads *q_rope, int S);
/* y[s][h] = W[h] x[s][h] for S rows of n_heads heads: x of n_in values and W [n_heads][n_out][n_in] in `type` (BF16 or
 * F16), sums in 32 bits, y of n_out values in f32 (y_f32) or rounded to the type.  n_in and n_out are multiples of 32 up to 1024.  A
 * head_stride of 0 gives every head the same x.  Pointers are 16-byte aligned, strides multiples of 8 elements; x and y do not overlap.
 * 0 = ok */
int    lag_hip_latent_heads(int type, const LagHipHeads *x, const void *W, int n_heads, int n_in, int n_out, const LagHipHeads *y, int y_f32,
                            int S);
/* out[s][h] = sum_t p_t c_t, p the softmax of scale * q[s][h] . (c_t, r_t) over the cells t <= pos[s]: q [S][n_heads][rank +
 * rope_dims] and out [S][n_heads][rank] in the cache's type, 16-byte aligned, not overlapping.  Sums and the softmax in 32 bits, its weights
 * rounded to the cache's type before the second product, the output once.  Free places, rows without a cell, cells that are no numbers,
 * repeated calls and scratch as for lag_hip_attn_paged.  n_heads up to 1024.  0 = ok */
int    lag_hip_attn_latent(const LagHipLatentCache *c, const LagHipKvRows *r, const void *q, int n_heads, float scale, void *out, int S);
/* The expanded form for S tokens of one sequence, at positions start .. start + S - 1, their cells already written: pages (device,
 * [n_seq_pages]) are the sequence's pages as its table row names them; wk [n_heads][nope][rank] and wv [n_heads][v_dim][rank] in the cache's
 * type; q [S][n_heads][nope + rope_dims] in the cache's type; out [S][n_heads][v_dim] in f32 (out_f32) or the cache's type: row s
 * attends to the tokens t <= start + s.  nope and v_dim: multiples of 32 up to 256.  Keys and values are made once a call, rounded to 11 bits
 * (f16, scaled by a power of two for each head: what is more than 2^20 below the largest of a head's, over all of the call's tokens, loses bits); sums and the softmax in 32 bits,
 * its weights in 11.  Cells that lead nowhere are not attended to; cells that are no numbers reach the rows that attend to them.  Everything
 * is 16-byte aligned; out overlaps nothing that is read.  start + S <= 2^22.  Its scratch is its own, and a recording of it keeps it:
 * 2 (rank + 64) bytes a token, and keys and values, 2 (nope + v_dim) bytes a token and head with each rounded up to 64, 128 or 256, of as many
 * heads at a time as a GiB holds, but of one at least (4 GiB for 2^22 tokens of 256 + 256).  It is allocated twice as large as a call needs
 * when it grows.  0 = ok */
int    lag_hip_attn_latent_prompt(const LagHipLatentCache *c, const int *pages, int n_seq_pages, int start, const void *wk, const void *wv, int nope,
                                  int v_dim, const void *q, int n_heads, float scale, void *out, int out_f32, int S);
/* x[i] += t[i] for n values: the residual after an output projection.  t may be x, or does
 * not overlap it.  0 = ok */
int    lag_hip_add(float *x, const float *t, size_t n);

/* ---------------- sampling ----------------
 * Settings of a batch's rows, device arrays [S], each may be NULL: temperature (NULL 1; <= 0
 * or NaN: the greedy pick of lag_hip_argmax), top_k (NULL, <= 0 or >= V: off), top_p (NULL,
 * >= 1 or NaN: off), min_p (NULL, <= 0 or NaN: off). */
typedef struct {
    const float *temperature;
    const int   *top_k;
    const float *top_p, *min_p;
} LagHipSample;
/* tok[s] = a token of logits[s, 0..V) drawn by u[s] in [0, 1): weights w_i = exp((l_i - max) /
 * temperature); of the tokens in order of falling logit (equal ones by rising index) the
 * first top_k, of those the shortest beginning with at least top_p of their weight (at least
 * one token), of those the weights >= min_p * the largest; the pick is the lowest index at which the
 * kept weights' sum in order of index exceeds u * their total.  Weights are whole numbers of
 * 2^-42 of the largest, so the sums are exact and the pick the same in every run and batch;
 * V <= 2^20.  -inf and NaN are never picked; a row that holds nothing else gives
 * lag_hip_argmax's pick.  0 = ok */
int    lag_hip_sample(const float *logits, int S, int V, const LagHipSample *p, const float *u, int *tok);

/* ---------------- memory, stream, timing ---------------- */
void  *lag_hip_alloc(size_t n);
int    lag_hip_h2d(void *dst, const void *src, size_t n);
int    lag_hip_d2h(void *dst, const void *src, size_t n);
int    lag_hip_d2d(void *dst, const void *src, size_t n);   /* async on the backend stream */
int    lag_hip_memset(void *dst, int v, size_t n);
int    lag_hip_sync(void);
void  *lag_hip_event_create(void);
int    lag_hip_event_record(void *ev);
float  lag_hip_event_elapsed_ms(void *start, void *end);
void   lag_hip_event_destroy(void *ev);

/* ---------------- graphs ----------------
 * Record the device-pointer entries (lag_hip_moe_forward, lag_hip_route,
 * lag_hip_d2d, the stack glue, attention, page copies and sampling) issued
 * between begin and end into one graph, replayed with a
 * single submission by lag_hip_graph_launch (async on the backend stream).
 * Pointers and shapes are fixed at recording; scratch must already be large
 * enough (issue the same shapes once first), else the entry fails.  A
 * finished recording owns the backend scratch it was recorded over until
 * lag_hip_graph_destroy (which waits for the stream, then frees it); later
 * calls of any size allocate their own, so they never disturb a live graph.
 * A recording begun right after another one gets fresh scratch of the same
 * capacity, so same-shaped graphs can be recorded back to back.  A destroy
 * issued while a recording is open takes effect when that recording ends.
 * No counterpart in the reference (its decode loop launches per layer): this
 * is the launch-overhead-free way to drive a decode step. */
int    lag_hip_graph_begin(void);
void  *lag_hip_graph_end(void);          /* NULL on failure */
int    lag_hip_graph_launch(void *g);
void   lag_hip_graph_destroy(void *g);

/* Kernel choice for the grouped expert GEMMs of lag_hip_moe_forward with
 * S > 1: 0 auto (the f16 MFMA when the batch's groups average >= 4.75 tokens,
 * else dot8), 1 dot8, 2 f16 MFMA.  Both give the same bits.  Returns the
 * previous mode, -1 for a bad one.  No counterpart in the reference (one
 * grouped kernel there, c/backend_cuda.cu:618-700): a tuning switch. */
int    lag_hip_set_grouped_kernel(int mode);

/* The int4 activation contract of lag_hip_moe_forward / lag_hip_moe_block for
 * per-row scales (gs == 0): 0 (default) this build's exact-integer digits,
 * 1 the reference's IDOT contract -- activations to int8 per 32-block
 * (amax/127, lrintf), exact int8 x int4 block dots, acc = fma(s_b, dot_b, acc)
 * in block order, x row scale (c/moe_quant.h:48-82, 141-182) -- which gives
 * the bits of the CPU tier under LAG_IDOT=1 (c/laguna.c:204-207).  Returns
 * the previous mode, -1 for a bad one; descriptors with gs > 0 ignore it (the
 * reference's grouped kernel has no IDOT form, c/quant.h:168-203). */
int    lag_hip_set_q4_mode(int mode);

/* per-kernel timing with events on the backend stream (the analogue of the
 * reference's COLI_CUDA_PROFILE=1, c/backend_cuda.cu:822-940) */
int    lag_hip_profile(int enable);
int    lag_hip_profile_count(void);
int    lag_hip_profile_read(int idx, char *name, int cap, double *total_ms, long long *launches);
void   lag_hip_profile_reset(void);

/* ---------------- synthetic data (bit-identical to the host generator) ---------------- */
int    lag_hip_gen_normal(float *out, int64_t n, uint64_t seed, uint64_t offset, double sigma, int to_bf16);
int    lag_hip_gen_bf16(uint16_t *out, int64_t n, uint64_t seed, uint64_t offset, double sigma);
int    lag_hip_gen_q4(uint8_t *q, float *s, uint64_t seed, double sigma, int64_t row0, int64_t nrows, int K, int gs);

/* ---------------- diagnostics ---------------- */
/* MFMA lane-layout probes (f16, bf16, int8) + libm evaluation on n host
 * inputs; out_host gets 768 + 3n floats (layout in k_route.hip).  0 = ran */
int    lag_hip_selftest(float *out_host, const float *xin_host, int n);
const char *lag_hip_last_error(void);

#ifdef __cplusplus
}
#endif
#endif
