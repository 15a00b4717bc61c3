/*
 * neuratensor_native.h -- C ABI of libneuratensor_native.so
 *
 * B200 (sm_100a) kernels for the FusedSpikeBlock inference path of
 * NeuraTensor 4.0.4.  Every entry point takes plain device pointers, sizes
 * and element strides, runs asynchronously on the given CUDA stream and
 * returns an nt_status code; it never aborts the process.  The caller owns
 * every buffer: inputs, outputs, state buffers and workspaces (sized with
 * the *_workspace_bytes queries).
 *
 * Concurrency: calls on different streams may run concurrently when they use
 * different workspaces and outputs, with two exceptions that are shared
 * per device: nt_rmsnorm_in_proj_noalloc's static scratch (overlapping calls
 * of that entry point race), and the device error word that every kernel
 * with a bounded wait may set (nt_get_error_flag reports the union of all
 * streams' flags since it was last cleared).  The launch counter is a process
 * total.
 *
 * Reference interfaces replaced (paths inside the NeuraTensor source tree):
 *   nt_lif_scan            LIFLayer.forward            neuratensor/core/snn.py:264-312
 *                          (_lif_sequential_scan :167-182, _lif_single_step :64-75)
 *   nt_selective_scan      SelectiveSSMLayer._discretize + _scan_sequential / _scan_single_step
 *                                                      neuratensor/core/ssm.py:106-139,145-221
 *   nt_ssm_forward         SelectiveSSMLayer.forward   neuratensor/core/ssm.py:313-349
 *   nt_sparse_out_proj     FusedSpikeBlock._sparse_out_proj  neuratensor/core/fused.py:149-165
 *   nt_rmsnorm_in_proj     FusedSpikeBlock.norm + in_proj    neuratensor/core/fused.py:118-119
 *   nt_block_forward       FusedSpikeBlock.forward     neuratensor/core/fused.py:101-147
 *   nt_window_attention    SlidingWindowAttention RoPE + SDPA neuratensor/core/model.py:148-178
 *   nt_attention_forward   SlidingWindowAttention.forward neuratensor/core/model.py:148-181
 *   nt_attention_output    SlidingWindowAttention o_proj + residual neuratensor/core/model.py:180-181
 *   nt_embedding           NeuraTensorModel.embedding  neuratensor/core/model.py:258
 *   nt_lm_head             NeuraTensorModel.norm + lm_head neuratensor/core/model.py:283-284
 *   nt_greedy_tokens       top-k = 1 sampling in NeuraTensorModel.generate model.py:344-359
 *   nt_rotary              apply_rotary at given positions model.py:119-126
 *   nt_logits_process      repetition penalty in NeuraTensorModel.generate model.py:336-342
 *   nt_lif_ssm_fused       LIF spikes driving the selective scan with given dt/B/C
 *                          (snn.py:167-182 feeding ssm.py:106-139,184-221)
 *
 * Layouts: activations are row-major [rows, channels] with unit channel
 * stride; "rows" are (batch, time) pairs in batch-major order.  Weights are
 * the nn.Linear weights, row-major [out_features, in_features].
 */
#ifndef NEURATENSOR_NATIVE_H
#define NEURATENSOR_NATIVE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define NT_ABI_VERSION 1

#if defined(__GNUC__)
#define NT_API __attribute__((visibility("default")))
#else
#define NT_API
#endif

typedef enum {
    NT_F32 = 0,   /* float32                                   */
    NT_BF16 = 1,  /* bfloat16                                  */
    NT_U8 = 2     /* uint8 (spike output of nt_lif_ssm_fused)  */
} nt_dtype;

typedef enum {
    NT_OK = 0,
    NT_ERR_ARG = 1,        /* bad shape, stride, null pointer or alignment          */
    NT_ERR_DTYPE = 2,      /* unsupported dtype combination                          */
    NT_ERR_ARCH = 3,       /* device is not sm_100                                   */
    NT_ERR_CUDA = 4,       /* CUDA runtime / launch error                            */
    NT_ERR_TIMEOUT = 5,    /* a bounded device-side wait expired (see error flag)    */
    NT_ERR_WORKSPACE = 6   /* workspace pointer null or smaller than required        */
} nt_status;

/* Library / device queries ------------------------------------------------ */
NT_API int nt_abi_version(void);
/* Message of the last failing call on this host thread ("" if none). */
NT_API const char* nt_last_error(void);
/* NT_OK when `device` is an sm_100 GPU this build can run on. */
NT_API int nt_device_supported(int device);
/* Reads (and optionally clears) the device error word that kernels set when
 * a bounded wait expires.  Synchronises the device.  *flags == 0 means no
 * kernel reported an error. */
NT_API int nt_get_error_flag(int device, unsigned* flags, int clear);
/* Checks the bounded-wait path (no counterpart in the reference, whose code
 * never waits on the device): one CTA waits on a barrier that nothing
 * completes, gives up after limit_ns of wall time (0..1e9), sets bit 16 of the
 * device error word and returns normally.  Every pipeline wait in this
 * library's kernels is bounded the same way (2 s), so a stalled producer shows
 * up as a flag and an error status instead of a hung GPU. */
NT_API int nt_bounded_wait_check(int64_t limit_ns, void* stream);
/* Kernels this library has launched in this process (all devices, all host
 * threads).  Reading it before and after a call counts that call's launches.
 * No counterpart in the reference, which launches no kernels of its own. */
NT_API unsigned long long nt_launch_count(void);

/* (a) LIF membrane recurrence -- LIFLayer.forward (snn.py:264-312).
 * Per channel c and step t:  V = beta[c]*V + x[t,c]  (a product then a sum,
 * each rounded to `dtype`), S = (V >= threshold[c]), V = V - threshold[c]*S.
 * x: [B,T,C] with element strides (x_sb, x_st, 1); spikes written as 0/1 in
 * `dtype` with strides (s_sb, s_st, 1).  beta, threshold: [C] in `dtype`.
 * mem_in: [B,C] in `dtype` or NULL for zeros (snn.py:286-287); mem_out: [B,C].
 * spike_count: optional device uint64 that is incremented by the number of
 * spikes (caller zeroes it). */
NT_API int nt_lif_scan(int dtype, int64_t B, int64_t T, int64_t C,
                const void* x, int64_t x_sb, int64_t x_st,
                const void* beta, const void* threshold,
                const void* mem_in, void* mem_out,
                void* spikes, int64_t s_sb, int64_t s_st,
                unsigned long long* spike_count, void* stream);

/* (b) selective scan -- SelectiveSSMLayer._discretize + _scan_sequential
 * (ssm.py:106-139,184-221).  A = -exp(log_A); A_bar = exp(A*dt);
 * B_bar = (A_bar-1)/A*B (dt*B where |A| < 1e-6); h = A_bar*h + B_bar*u;
 * y = sum_n C[n]*h[n] + D*u.  If gate != NULL the output is y*silu(gate)
 * (fused.py:130).  u, dt, gate, y: [B,T,d] contiguous in `dtype`;
 * Bm, Cm: [B,T,N] contiguous in `dtype`; log_A: [d,N], D: [d] in `dtype`.
 * state_in/state_out: [B,d,N] in `state_dtype` (state_in NULL = zeros); the
 * recurrence itself runs in float32.  d_state N <= 256. */
NT_API int nt_selective_scan(int dtype, int state_dtype, int64_t B, int64_t T, int64_t d, int64_t N,
                      const void* u, const void* dt, const void* Bm, const void* Cm,
                      const void* log_A, const void* D, const void* gate,
                      const void* state_in, void* state_out, void* y, void* stream);

/* SelectiveSSMLayer.forward (ssm.py:313-349): B = u W_B^T, C = u W_C^T,
 * dt = softplus(u W_dt^T + b_dt), then the scan above.  W_proj is the packed
 * projection weight [d + 2N, d] = rows of W_dt, then W_B, then W_C.
 * Workspace: nt_ssm_workspace_bytes(). */
NT_API int64_t nt_ssm_workspace_bytes(int dtype, int64_t B, int64_t T, int64_t d, int64_t N);
NT_API int nt_ssm_forward(int dtype, int state_dtype, int64_t B, int64_t T, int64_t d, int64_t N,
                   const void* u, const void* W_proj, const void* b_dt,
                   const void* log_A, const void* D,
                   const void* state_in, void* state_out, void* y,
                   void* workspace, int64_t workspace_bytes, void* stream);

/* (c) spike-sparse out_proj -- FusedSpikeBlock._sparse_out_proj
 * (fused.py:149-165).  o: [M,K], spikes: [M,K] (0/1), W: [Nout,K], out:
 * [M,Nout], all `dtype`, contiguous.  A row is active when any spike in it
 * is non-zero.  If 2*n_active > M every row is projected (dense branch);
 * otherwise only active rows are projected and inactive rows are zero.
 * n_active_out: optional device int64 receiving n_active.
 * Workspace: nt_sparse_out_proj_workspace_bytes(). */
NT_API int64_t nt_sparse_out_proj_workspace_bytes(int dtype, int64_t M, int64_t K, int64_t Nout);
NT_API int nt_sparse_out_proj(int dtype, int64_t M, int64_t K, int64_t Nout,
                       const void* o, const void* spikes, const void* W, void* out,
                       long long* n_active_out,
                       void* workspace, int64_t workspace_bytes, void* stream);

/* (d) RMSNorm + in_proj -- fused.py:118-119.  xn = RMSNorm(x) (eps = float32
 * machine epsilon, as nn.RMSNorm with eps=None), [h | gate] = xn W_in^T.
 * x: [M,dm]; gamma: [dm]; W_in: [2*di, dm]; h, gate: [M,di], all `dtype`.
 * Workspace: nt_rmsnorm_in_proj_workspace_bytes(). */
NT_API int64_t nt_rmsnorm_in_proj_workspace_bytes(int dtype, int64_t M, int64_t dm, int64_t di);
NT_API int nt_rmsnorm_in_proj(int dtype, int64_t M, int64_t dm, int64_t di,
                       const void* x, const void* gamma, const void* W_in,
                       void* h, void* gate,
                       void* workspace, int64_t workspace_bytes, void* stream);

/* RMSNorm + in_proj without a workspace (no counterpart in the reference).
 * Same computation and arguments as nt_rmsnorm_in_proj, minus the workspace:
 * the normalised activations go to a scratch array the library itself holds
 * in device memory (nt_noalloc_scratch_bytes() bytes per device, 32 MiB), for
 * callers that cannot allocate device memory, e.g. serving runtimes that
 * reserve HBM at start-up and forbid cudaMalloc afterwards.  Requires
 * M*d_model*sizeof(dtype) <= nt_noalloc_scratch_bytes() (else NT_ERR_ARG).
 * The first call on a device, made with that device current, looks up the
 * array's address; make it before any stream capture.  The address is cached
 * for the life of the process and does not survive a device reset
 * (cudaDeviceReset or a re-created primary context): do not call this entry
 * point after one.  Calls share the array: calls that overlap on the GPU race. */
NT_API size_t nt_noalloc_scratch_bytes(void);
NT_API int nt_rmsnorm_in_proj_noalloc(int dtype, int64_t M, int64_t dm, int64_t di,
                       const void* x, const void* gamma, const void* W_in,
                       void* h, void* gate, void* stream);

/* SlidingWindowAttention.forward (model.py:148-181), bf16, head_dim 64 or 128:
 * out = o_proj(attention(qkv(RMSNorm(x)))) + x, with the attention as in
 * nt_window_attention.  x, out: [B,T,dm]; norm_w: [dm]; W_qkv: [3*dm, dm];
 * W_o: [dm, dm]; cos_t, sin_t: [T, dm/n_heads] rotary tables.
 * Workspace: nt_attention_workspace_bytes(). */
NT_API int64_t nt_attention_workspace_bytes(int dtype, int64_t B, int64_t T, int64_t dm);
NT_API int nt_attention_forward(int dtype, int64_t B, int64_t T, int64_t dm, int64_t n_heads, int64_t window,
                                const void* x, const void* norm_w, const void* W_qkv, const void* W_o,
                                const void* cos_t, const void* sin_t, void* out,
                                void* workspace, int64_t workspace_bytes, void* stream);

/* The end of nt_attention_forward for attention that was taken elsewhere
 * (model.py:180-181): out = rnd(rnd(o W_o^T) + x).  o, x, out: [M, dm] in `dtype`;
 * W_o: [dm, dm].  out must not overlap the inputs. */
NT_API int nt_attention_output(int dtype, int64_t M, int64_t dm, const void* o, const void* W_o, const void* x,
                               void* out, void* stream);

/* Embedding gather -- NeuraTensorModel.embedding (model.py:258, nn.Embedding):
 * out[r, :] = W[ids[r], :] for r < M.  ids: [M] int64; W: [vocab, dm]; out:
 * [M, dm], both `dtype`.  An id outside [0, vocab) yields a zero row and sets
 * a flag in the device error word (nt_get_error_flag), where the reference
 * raises IndexError. */
NT_API int nt_embedding(int dtype, int64_t M, int64_t dm, int64_t vocab, const int64_t* ids, const void* W,
                        void* out, void* stream);

/* Greedy next tokens -- NeuraTensorModel.generate with top_k = 1, temperature 1,
 * top_p 1 and no repetition penalty (model.py:344-359): per row of logits
 * [B, vocab] (row stride ld elements, `dtype`), the reference keeps the entries
 * equal to the maximum and samples among them; this picks the
 * floor(u[r] * ties)-th tied index in index order, u: [B] float32 in [0, 1).
 * tokens: [B] int64 device output. */
NT_API int nt_greedy_tokens(int dtype, int64_t B, int64_t vocab, const void* logits, int64_t ld, const float* u,
                            int64_t* tokens, void* stream);

/* Final RMSNorm + tied lm_head -- NeuraTensorModel.norm + lm_head
 * (model.py:283-284): logits = RMSNorm(x) W^T, logits in `dtype` (bf16 logits
 * in bf16 mode).  x: [M, dm]; gamma: [dm]; W: [vocab, dm] (the embedding
 * matrix when tied); logits: [M, vocab].  Workspace: nt_lm_head_workspace_bytes(). */
NT_API int64_t nt_lm_head_workspace_bytes(int dtype, int64_t M, int64_t dm, int64_t vocab);
NT_API int nt_lm_head(int dtype, int64_t M, int64_t dm, int64_t vocab, const void* x, const void* gamma,
                      const void* W, void* logits, void* workspace, int64_t workspace_bytes, void* stream);

/* FusedSpikeBlock.forward in eval mode (fused.py:101-147):
 *   out = sparse_out_proj(SSM(LIF(in_proj(RMSNorm(x))_h)) * silu(gate)) * out_scale + x
 * x, out: [B,T,dm]; weights as in the module (W_proj packed as above);
 * beta = sigmoid(beta_logit) and threshold in `dtype`, [di];
 * mem_in/mem_out: [B,di] in `dtype` (mem_in NULL = zeros);
 * state_in/state_out: [B,di,N] in `state_dtype` (state_in NULL = zeros);
 * spike_count: device uint64, incremented by this block's spike count;
 * sparse: 1 = inference sparse out_proj (fused.py:133-134), 0 = dense.
 * Workspace: nt_block_workspace_bytes(). */
NT_API int64_t nt_block_workspace_bytes(int dtype, int64_t B, int64_t T, int64_t dm, int64_t di, int64_t N);
NT_API int nt_block_forward(int dtype, int state_dtype, int64_t B, int64_t T, int64_t dm, int64_t di,
                     int64_t N,
                     const void* x, const void* norm_w, const void* W_in,
                     const void* beta, const void* threshold,
                     const void* log_A, const void* D, const void* W_proj, const void* b_dt,
                     const void* W_out, const void* out_scale,
                     const void* mem_in, void* mem_out,
                     const void* state_in, void* state_out,
                     void* out, unsigned long long* spike_count, int sparse,
                     void* workspace, int64_t workspace_bytes, void* stream);

/* Standalone fused LIF + selective scan: the LIF spikes of x drive the scan
 * with caller-given dt/B/C.  x, delta, y: [B,L,d] bf16; Bm, Cm: [B,L,N] bf16;
 * log_A: [d,N], Dskip, beta, threshold: [d] float32; mem_in/mem_out: [B,d]
 * float32; state_in/state_out: [B,d,N] float32 (NULL inputs = zeros);
 * spikes: optional [B,L,d] output in `spike_dtype` (NT_U8 or NT_BF16);
 * spike_count: optional device uint64 (incremented).  All math in float32. */
NT_API int nt_lif_ssm_fused(int64_t B, int64_t L, int64_t d, int64_t N,
                     const void* x, const void* delta, const void* Bm, const void* Cm,
                     const float* log_A, const float* Dskip,
                     const float* beta, const float* threshold,
                     const float* mem_in, float* mem_out,
                     const float* state_in, float* state_out,
                     void* y, void* spikes, int spike_dtype,
                     unsigned long long* spike_count, void* stream);

/* Sliding-window causal attention with rotary embedding -- the middle of
 * SlidingWindowAttention.forward (model.py:159-178: q/k/v from the qkv
 * projection, apply_rotary on q and k (model.py:119-126), then
 * scaled_dot_product_attention with the causal window mask j in [i-window, i]).
 * bf16 only, head_dim (HD) 64 or 128.  qkv: [B*T, ld_qkv] rows, columns
 * [q | k | v] of n_heads*HD each; cos_t, sin_t: [T, HD] bf16 rotary tables
 * (the module's cached ones); out: [B*T, ld_out], head h in columns
 * h*HD .. h*HD+HD-1 (the transpose(1,2).reshape layout o_proj takes).
 * Softmax scale 1/sqrt(HD).  RoPE
 * rounds like the reference's bf16 ops; scores and softmax in float32, the
 * probabilities rounded to bf16 before the product with v. */
NT_API int nt_window_attention(int dtype, int64_t B, int64_t T, int64_t n_heads, int64_t head_dim,
                        int64_t window, const void* qkv, int64_t ld_qkv, const void* cos_t,
                        const void* sin_t, void* out, int64_t ld_out, void* stream);

/* Rotary positions on any tensor of heads (the rotation of apply_rotary,
 * model.py:119-126, at given positions).  x, y: [B,T,H,D] in `dtype` with
 * element strides (sb, st, sh, 1); x == y rotates in place.  The first R
 * dimensions of each head turn in R/2 pairs: (i, i + R/2) when interleaved == 0,
 * (2i, 2i + 1) otherwise; dimensions past R are copied.  Pair i of the token
 * at position p turns by the angle p * inv_freq[i], taken in float64:
 *   y1 = m (x1 cos - x2 sin),  y2 = m (x2 cos + x1 sin),  m = mscale,
 * in float32 with one rounding to `dtype`.  inverse != 0 turns backwards (the
 * gradient of the forward call with the same arguments).  y is x or does not
 * overlap it; D <= 2048.  positions: int64,
 * row b starts at positions + b*p_sb (p_sb = 0: shared by the batch);
 * inv_freq: [R/2] float32. */
NT_API int nt_rotary(int dtype, int64_t B, int64_t T, int64_t H, int64_t D, int64_t R, int interleaved,
                     int inverse, float mscale, const void* x, int64_t x_sb, int64_t x_st, int64_t x_sh,
                     const int64_t* positions, int64_t p_sb, const float* inv_freq,
                     void* y, int64_t y_sb, int64_t y_st, int64_t y_sh, void* stream);

/* The 8-bit attention cache (no counterpart in the reference, whose attention
 * is stateless across calls).  Codes are e4m3 bytes in pages of `page` tokens
 * (16, 32 or 64), [n_pages, Hkv, page, D] contiguous, D 64 or 128; every page
 * and head has one float32 scale, a power of two >= 2^-126, in
 * [n_pages, Hkv]; keys and values have their own.  Position p of sequence b
 * is slot p % page of page table[b, p / page] (int32, row stride table_sb,
 * n_blocks entries).  lengths[b] (int32) counts the tokens of sequence b with
 * the new ones; its counts[b] (int32, NULL: T) new tokens are rows 0..counts-1
 * of k, v and q and the last counts[b] positions.
 *
 * nt_kv_append writes rows t < counts[b] of k and v ([B,T,Hkv,D] in `dtype`,
 * element strides, unit stride in D).  Block scale: the smallest power of two
 * s with max|x| <= 448 s over the block's finite new values, and not below the
 * block's scale when the block holds older tokens; older codes are re-encoded
 * when it grows.  Codes: x / s rounded to nearest even, saturating; NaN stays
 * NaN.  Slots behind the new tokens are left as they are.  A page that is
 * written must belong to one sequence and stand once among its blocks; calls that
 * write the same pages must not overlap.  A sequence with counts outside [0, T],
 * lengths < counts or lengths past the table, and a page outside
 * [0, n_pages), is skipped and sets the bad-argument bit of the device error
 * word. */
NT_API int nt_kv_append(int dtype, int64_t B, int64_t T, int64_t Hkv, int64_t D, int64_t page, int64_t n_pages,
                        int64_t n_blocks, const void* k, int64_t k_sb, int64_t k_st, int64_t k_sh,
                        const void* v, int64_t v_sb, int64_t v_st, int64_t v_sh,
                        void* k_codes, float* k_scale, void* v_codes, float* v_scale,
                        const int32_t* table, int64_t table_sb, const int32_t* lengths, const int32_t* counts,
                        void* stream);

/* Attention of the new tokens over the cache.  q: [B,T,Hq,D] in `dtype`
 * (strides as above), Hq a multiple of Hkv; query head h reads cached head
 * h / (Hq / Hkv).  Row t < counts[b] stands at p = lengths[b] - counts[b] + t
 * and sees keys j <= p, and j >= p - window when window >= 0 (-1: no window).
 * out: [B,T,Hq,D] contiguous in `dtype`, softmax(scale q.k) v; rows
 * t >= counts[b], rows that see no key and sequences with bad counts or lengths
 * are zero.  Keys in a page outside [0, n_pages) are not seen and set the
 * bad-argument bit.  Scores and sums in float32.  Meant for one to a few new
 * tokens per sequence; any T is right.
 * Workspace: nt_kv_attention_workspace_bytes() (0 when no split is taken). */
NT_API int64_t nt_kv_attention_workspace_bytes(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                               int64_t page, int64_t n_blocks, int64_t window);
NT_API int nt_kv_attention(int dtype, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t page,
                           int64_t n_pages, int64_t n_blocks, int64_t window, float scale,
                           const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh,
                           const void* k_codes, const float* k_scale, const void* v_codes, const float* v_scale,
                           const int32_t* table, int64_t table_sb, const int32_t* lengths, const int32_t* counts,
                           void* out, void* workspace, int64_t workspace_bytes, void* stream);

/* Penalties, biases and masks on logits (NeuraTensorModel.generate's
 * repetition penalty, model.py:336-342, and what callers add to it), one pass
 * over [B, V] rows in `dtype` (row strides ld, ldo; out == logits allowed).
 * With c the count of v among tokens[b, 0..lengths[b]) (int64, row stride
 * tok_ld, lengths NULL: L) and g the count from prompt_lengths[b] (NULL: 0) on:
 *   x = repetition penalty r, where c > 0: x > 0 ? x/r : x*r, once, or c times
 *       with a rounding to `dtype` after each when each != 0 (generate's loop)
 *   x = x - frequency*g - presence*[g > 0]
 *   x = x + bias[b, j] for the last j with bias_ids[b, j] == v (int64, ids
 *       outside [0, V) are skipped)
 *   x = -inf where bit v % 32 of allowed[b, v / 32] is 0
 * in float32, one rounding to `dtype`; x/r is the product with 1/r rounded to
 * float32 (from the double when r is the scalar, as torch divides by a number).
 * Tokens outside [0, V) are skipped.  A penalty is a [B] float32 array, or the
 * scalar beside it when the pointer is NULL (1, 0, 0: none).  tokens, bias and
 * allowed may be NULL (L, NB 0).  allowed: uint32 words, row stride
 * allowed_ld (0: one row for the batch). */
NT_API int nt_logits_process(int dtype, int64_t B, int64_t V, const void* logits, int64_t ld,
                             const int64_t* tokens, int64_t tok_ld, int64_t L, const int32_t* lengths,
                             const int32_t* prompt_lengths, int each,
                             const float* repetition, double repetition_all, const float* frequency,
                             float frequency_all, const float* presence, float presence_all,
                             const int64_t* bias_ids, int64_t ids_ld, const float* bias, int64_t bias_ld, int64_t NB,
                             const uint32_t* allowed, int64_t allowed_ld, void* out, int64_t ldo, void* stream);

/* A step of a beam search over the above (no counterpart in the reference, whose
 * generate samples one continuation per prompt; model.py:301-370).
 *
 * nt_beam_select: the n best continuations of each of B items with K beams
 * (K, n <= 64; B K <= 65535).  logits: [B*K, V] rows in `dtype`, row stride ld;
 * scores: [B*K] float32, log-probabilities so far; finished (bytes, NULL: none)
 * and lengths (int32, tokens made so far; NULL without a length penalty): [B*K].
 * A live beam k offers every token v whose logit is not -inf, with
 *   s = scores[k] + (x[k,v] - log sum_u exp x[k,u]);
 * a finished one itself alone, with s = scores[k] and token `pad`.  A beam whose
 * score or logarithm is not finite (a NaN or +inf among its logits, nothing but
 * -inf) offers nothing.  Candidates rank by s / max(l, 1)^length_penalty, l =
 * lengths + 1 for a live beam and lengths for a finished one, in float64 except
 * for the sum of exponentials; a beam's own in the order of their logits; ties go
 * to the lower beam, then the lower token.  out_scores float32, out_rows int32 (the
 * row b K + k that a candidate goes on from), out_tokens int64: [B, n], best first;
 * with stay != 0 (n == K) the best child of a beam stands in that beam's place and
 * the others, best first, in the places left.  Where candidates run out: -inf, row
 * b K + place % K, `pad`.  The outputs overlap no input.
 * Workspace: nt_beam_select_workspace_bytes(). */
NT_API int64_t nt_beam_select_workspace_bytes(int dtype, int64_t B, int64_t K, int64_t V, int64_t n);
NT_API int nt_beam_select(int dtype, int64_t B, int64_t K, int64_t V, int64_t n, const void* logits, int64_t ld,
                          const float* scores, const unsigned char* finished, const int32_t* lengths,
                          double length_penalty, int64_t pad, int stay,
                          float* out_scores, int32_t* out_rows, int64_t* out_tokens,
                          void* workspace, int64_t workspace_bytes, void* stream);

/* Rows moved in place, for many tensors at once: row r of each takes what row
 * rows[r] held (int32 [R]; -1: it stays as it is).  rows[r] lies in r's group of
 * `group` <= 1024 consecutive rows, else the row stays and the bad-argument bit of the
 * device error word is set.  tensors: host array [n_tensors][3] of device address, bytes
 * of a row, bytes between rows; tensors do not overlap. */
NT_API int nt_reorder_rows(int64_t n_tensors, const int64_t* tensors, int64_t R, int64_t group,
                           const int32_t* rows, void* stream);

/* Sequences over a shared pool of pages.  table (int32 [R, n_blocks], row stride
 * table_sb, -1: no page), refs (int32 [n_pages]: how many table entries, and other
 * holders, have a page; 0: free) and lengths (int32 [R], R <= 1024) are rewritten in
 * place so that row r goes on from row parents[r] (-1: it ends, with length 0):
 *  1. the row takes the parent's length n and its entries of the blocks that hold
 *     positions [max(0, n - window), n) (window < 0: all); its other entries are -1,
 *     and the counts follow;
 *  2. of the rows whose last page is the same and not full, one keeps it when its
 *     count is their number: the first that goes on from itself, else the first; every
 *     other gets a new page, and copies[r] = (old page, new page), else (-1, -1);
 *  3. the blocks of positions [n, n + tokens) behind get new pages, but those wholly
 *     before n + tokens - window.
 * New pages are the free pages of lowest index, row by row (2. before 3., blocks in
 * order).  Where they run out, or the table ends, entries stay -1 and the bad-argument
 * bit of the device error word is set, as for a bad parent (it ends), length or page.
 * With group > 0 shared[g] (int32 [R / group]) is how many leading tokens, in whole
 * blocks, the rows of group g have in the same pages: 0 where one has ended.
 * Workspace: nt_kv_fork_workspace_bytes() (0 without groups). */
NT_API int64_t nt_kv_fork_workspace_bytes(int64_t R, int64_t n_blocks, int64_t group);
NT_API int nt_kv_fork(int64_t R, int64_t n_pages, int64_t n_blocks, int64_t page, int64_t tokens, int64_t window,
                      int64_t group, int32_t* table, int64_t table_sb, int32_t* refs, int32_t* lengths,
                      const int32_t* parents, int32_t* copies, int32_t* shared,
                      void* workspace, int64_t workspace_bytes, void* stream);

/* Pages copied within their pools, codes and scales of keys and values of every
 * layer: pages (int32 [n, 2]): from, to; (-1, -1) is skipped, a page outside
 * [0, n_pages) too, with the bad-argument bit.  layers: host array [n_layers][4] of
 * the device addresses of k codes, k scales, v codes, v scales (nt_kv_append).  No
 * page is written twice, or read and written. */
NT_API int nt_kv_copy_pages(int64_t n_layers, const int64_t* layers, int64_t n_pages, int64_t Hkv, int64_t page,
                            int64_t D, int64_t n, const int32_t* pages, void* stream);

/* nt_kv_attention for sequences that share their beginnings: the B sequences are
 * `groups` groups of B / groups consecutive ones, and the first shared[g] (int32)
 * positions of a group's sequences hold the same keys and values, in each one's own
 * pages, which may be the same; they are read once for all of them, from one's pages.
 * Results and everything else as nt_kv_attention (shared[g] < 0 counts as 0).
 * Workspace: nt_kv_attention_shared_workspace_bytes(). */
NT_API int64_t nt_kv_attention_shared_workspace_bytes(int dtype, int64_t B, int64_t groups, int64_t T, int64_t Hq, int64_t Hkv,
                                                      int64_t D, int64_t page, int64_t n_blocks, int64_t window);
NT_API int nt_kv_attention_shared(int dtype, int64_t B, int64_t groups, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                  int64_t page, int64_t n_pages, int64_t n_blocks, int64_t window, float scale,
                                  const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh,
                                  const void* k_codes, const float* k_scale, const void* v_codes, const float* v_scale,
                                  const int32_t* table, int64_t table_sb, const int32_t* lengths, const int32_t* counts,
                                  const int32_t* shared, void* out, void* workspace, int64_t workspace_bytes, void* stream);

/* The entry points of a generation step with their arguments in one array, for bindings
 * that pay for every argument they convert (a step makes several short calls
 * per layer): `words` holds the arguments in order, 8 bytes each, integers as
 * int64, pointers as their address, floats as double; n_words must be the entry
 * point's number of arguments. */
enum { NT_ENTRY_ROTARY = 0, NT_ENTRY_KV_APPEND = 1, NT_ENTRY_KV_ATTENTION = 2, NT_ENTRY_LOGITS_PROCESS = 3,
       NT_ENTRY_BEAM_SELECT = 4, NT_ENTRY_REORDER_ROWS = 5, NT_ENTRY_KV_FORK = 6, NT_ENTRY_KV_COPY_PAGES = 7,
       NT_ENTRY_KV_ATTENTION_SHARED = 8 };
NT_API int nt_call_packed(int entry, const void* words, int64_t n_words);

#ifdef __cplusplus
}
#endif

#endif /* NEURATENSOR_NATIVE_H */
