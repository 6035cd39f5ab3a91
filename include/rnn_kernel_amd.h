/*
 * rnn_kernel_amd — C ABI of the MI355X (gfx950) fp32 GRU training path.
 *
 * Conventions for every entry point:
 *   - all pointers are device pointers owned by the caller (PyTorch's caching
 *     allocator in the Python front end); the library never allocates device
 *     memory in these calls;
 *   - work is enqueued on `stream` (a hipStream_t, NULL = default stream) and
 *     is asynchronous: no host synchronisation happens inside;
 *   - the device is the calling thread's current HIP device;
 *   - the return value is 0 on success, otherwise a nonzero code; the message
 *     of the last failure on the calling thread is rka_last_error();
 *   - tensors are dense row-major fp32: x [B,T,I], y/dy [B,T,H] (batch
 *     first), h0/hn/dh0 [B,H], W_ih [3H,I], W_hh [3H,H], biases [3H], with
 *     nn.GRU's gate order r, z, n in row blocks [0,H), [H,2H), [2H,3H).
 *
 * The reference binds its kernels from Python with cuda-python
 * (cuLaunchCooperativeKernel on raw pointers, torch's current stream);
 * each entry point below names the reference launcher it replaces.
 */
#ifndef RNN_KERNEL_AMD_H
#define RNN_KERNEL_AMD_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Error codes (besides hipError_t values passed through). */
#define RKA_OK 0
#define RKA_ERR_INVALID_ARGUMENT 1001
#define RKA_ERR_WORKSPACE_TOO_SMALL 1002
#define RKA_ERR_UNSUPPORTED_DEVICE 1003
#define RKA_ERR_UNSUPPORTED_SHAPE 1004
#define RKA_ERR_TOO_LARGE_FOR_RESIDENT_LAUNCH 1005

/* Library ABI version. */
int rka_version(void);

/* Message of the last failed call on this thread ("" if none). */
const char* rka_last_error(void);

/* 1 if `device` is a gfx950 (MI355X-class) GPU this library was built for,
 * 0 otherwise (message in rka_last_error()).  Replaces the reference's
 * _validate_a100_device / is_a100_available capability checks
 * (src/rnn_kernel/a100/prod/gru.py:109-117,139-148). */
int rka_device_supported(int device);

/* Bytes of the per-layer gate cache ("reserve") that rka_gru_forward writes
 * in training mode and rka_gru_backward reads: [B,T,H,4] fp32, the unit's
 * (r, z, n, a_n) contiguous (one 16-byte access per unit and step).
 * Replaces the reference's gate_cache [B,T,4H] allocation
 * (src/rnn_kernel/a100/prod/gru.py:238), which keeps the four gates in
 * blocks of H; the size is the same. */
size_t rka_gru_reserve_bytes(int batch, int seq_len, int hidden_size);

/* Workspace bytes rka_gru_forward needs (input-gate buffer, exchange
 * buffers, flags). */
size_t rka_gru_forward_workspace_bytes(int batch, int seq_len, int input_size, int hidden_size);

/*
 * Forward of one GRU layer: input projection (fp32 MFMA GEMM) followed by the
 * persistent recurrence.  Writes y [B,T,H] and hn [B,H].  When `reserve` is
 * non-NULL (training) it also writes the gate cache there; when NULL
 * (inference) no cache is written.
 * Replaces F.linear + _launch_forward / _launch_forward_no_cache + the h_n
 * copy (src/rnn_kernel/a100/prod/gru.py:519-525,226-376,610-616).
 */
int rka_gru_forward(const float* x, const float* h0,
                    const float* w_ih, const float* w_hh,
                    const float* b_ih, const float* b_hh,
                    float* y, float* hn, float* reserve,
                    void* workspace, size_t workspace_bytes,
                    int batch, int seq_len, int input_size, int hidden_size,
                    void* stream);

/*
 * Inference through a stack of layers (layer 0 takes x, each later one the
 * previous layer's output): rka_gru_forward without a gate cache, layer by
 * layer, with one workspace.  h0 and hn are [num_layers,B,H], y the last
 * layer's output [B,T,H] (earlier layers' outputs pass through it too); weights
 * holds w_ih, w_hh, b_ih, b_hh of each layer in order (4 num_layers pointers,
 * read on the host during the call).
 */
size_t rka_gru_stack_forward_workspace_bytes(int num_layers, int batch, int seq_len, int input_size, int hidden_size);
int rka_gru_stack_forward(int num_layers, const float* x, const float* h0, const float* const* weights,
                          float* y, float* hn, void* workspace, size_t workspace_bytes,
                          int batch, int seq_len, int input_size, int hidden_size, void* stream);

/* Workspace bytes rka_gru_backward needs (gate-gradient buffer, exchange
 * buffers, split-K partials, flags). */
size_t rka_gru_backward_workspace_bytes(int batch, int seq_len, int input_size, int hidden_size);

/*
 * Backward of one GRU layer from the forward's y and reserve.
 * dy [B,T,H] may be NULL (zeros, gru.py:534-535); dhn [B,H] may be NULL (no
 * gradient on h_n, gru.py:552-554); dx may be NULL (input gradient not
 * needed).  Writes (does not accumulate) dx, dh0, dw_ih, dw_hh, db_ih, db_hh.
 * Replaces _launch_pack_hidden_prev + _launch_backward_sequence + the cuBLAS
 * gradient GEMMs (src/rnn_kernel/a100/prod/gru.py:531-580,379-487).
 */
int rka_gru_backward(const float* x, const float* h0,
                     const float* w_ih, const float* w_hh,
                     const float* y, const float* reserve,
                     const float* dy, const float* dhn,
                     float* dx, float* dh0,
                     float* dw_ih, float* dw_hh, float* db_ih, float* db_hh,
                     void* workspace, size_t workspace_bytes,
                     int batch, int seq_len, int input_size, int hidden_size,
                     void* stream);

/*
 * Building blocks (each is a stage of the two calls above, exported for
 * kernel-level parity tests and profiling).
 */

/* C[m,n] = sum_k A(m,k) B(n,k) (+ bias[n] if bias != NULL), fp32 MFMA.
 * A(m,k) = a[m*lda+k] if a_kmajor == 0 else a[k*lda+m];
 * B(n,k) = b[n*ldb+k] if b_kmajor == 0 else b[k*ldb+n].
 * Any alignment and leading dimension below 2^22 (else
 * RKA_ERR_UNSUPPORTED_SHAPE, nothing launched); operands whose contiguous
 * extent, leading dimension and base are multiples of 16 bytes take the
 * faster float4 paths, the others give the same results bit for bit.
 * Replaces the torch F.linear / matmul calls of gru.py:519-523,571-578. */
int rka_gemm_f32(int m, int n, int k,
                 const float* a, int lda, int a_kmajor,
                 const float* b, int ldb, int b_kmajor,
                 const float* bias, float* c, int ldc, void* stream);

/* Workspace bytes of the recurrence-only calls below. */
size_t rka_gru_recurrence_workspace_bytes(int batch, int hidden_size);

/* Persistent forward recurrence from precomputed input gates gx [B,T,3H]
 * (x W_ih^T + b_ih).  Writes y, hn and (if non-NULL) the reserve.
 * Replaces _launch_forward / _launch_forward_no_cache
 * (src/rnn_kernel/a100/prod/gru.py:226-376). */
int rka_gru_recurrence_forward(const float* gx, const float* h0,
                               const float* w_hh, const float* b_hh,
                               float* y, float* hn, float* reserve,
                               void* workspace, size_t workspace_bytes,
                               int batch, int seq_len, int hidden_size,
                               void* stream);

/* The same as rka_gru_recurrence_forward without a workspace, for callers
 * that cannot allocate device memory (code under HIP graph capture, tight
 * serving loops, harnesses that forbid allocation).  No counterpart in the
 * reference.  The exchange state lives in a static device array of the
 * library (4 MiB + 32 KiB + 256 B): it is part of the library's code
 * object, so every process that loads the library holds it on each device
 * the code object is loaded on, until the process ends, whether or not it
 * calls this entry point; the first call on a device only looks up its
 * address there.  The call allocates no device memory.  Limit: batch * hidden_size <= 262144 (2 B H 8-byte
 * words in 4 MiB); larger shapes return RKA_ERR_UNSUPPORTED_SHAPE without
 * launching; so is seq_len >= 2^24.  Every call on a GPU shares that GPU's
 * array: calls ordered on one stream are safe (each zeroes the state it uses
 * first); calls that overlap on one GPU (different streams or threads
 * without ordering) race.  Each call's exchange words carry its own call
 * number, so overlapping calls never take each other's values: they abort
 * (NaN outputs, counted by rka_recurrence_abort_count) instead. */
int rka_gru_recurrence_forward_noalloc(const float* gx, const float* h0,
                                       const float* w_hh, const float* b_hh,
                                       float* y, float* hn, float* reserve,
                                       int batch, int seq_len, int hidden_size,
                                       void* stream);

/* Persistent reverse-time recurrence.  Writes the gate gradients
 * g [B,T,4H] as blocks (da_n, dr^, dz^, dn^) and dh0.  dy / dhn may be NULL.
 * Replaces _launch_backward_sequence (src/rnn_kernel/a100/prod/gru.py:415-487),
 * whose G_i / G_h outputs are the column ranges [H,4H) and the rotation of
 * [0,3H) of g. */
int rka_gru_recurrence_backward(const float* dy, const float* dhn,
                                const float* reserve, const float* h0,
                                const float* y, const float* w_hh,
                                float* g, float* dh0,
                                void* workspace, size_t workspace_bytes,
                                int batch, int seq_len, int hidden_size,
                                void* stream);

/* GEMM tile families (for tuning and A/B tests; affects later calls on all
 * threads).  RKA_GEMM_TILES_AUTO: the tile of each product by a cost rule
 * (32x32 to 128x64 where 128x128 tiles would fill the CUs unevenly).
 * RKA_GEMM_TILES_128: 128x128 tiles everywhere.  Products that the rule gives
 * 128x128 tiles are the same bit for bit in both modes; the others differ by
 * float32 rounding (other k-slices and summation order).  No counterpart in
 * the reference (its products are cuBLAS calls,
 * src/rnn_kernel/a100/prod/gru.py:569-578). */
#define RKA_GEMM_TILES_AUTO 0
#define RKA_GEMM_TILES_128 1
int rka_set_gemm_tiles(int mode);

/* The form that products take in the present tile mode (host only: no GPU is
 * asked), for tests and tuning.  rka_describe_gemm: a rka_gemm_f32 call of this
 * size, `aligned` telling whether the contiguous dimension of both operands is
 * whole aligned float4.  rka_describe_weight_gradients: the pair dW_hh, dW_ih of
 * rka_gru_backward; writes the first min(n_out, 4) of {form, k-slices of dW_hh, of
 * dW_ih, 1 if its launch writes the results itself}.  No counterpart in the
 * reference (its products are cuBLAS calls). */
#define RKA_GEMM_FORM_RING 0   /* 128x128 tiles, fp32 matrix cores */
#define RKA_GEMM_FORM_SPLIT 1  /* 128x128 tiles, three bf16 pieces per value */
#define RKA_GEMM_FORM_128X64 2 /* register-staged tiles, fp32 matrix cores */
#define RKA_GEMM_FORM_64X64 3
#define RKA_GEMM_FORM_32X32 4
int rka_describe_gemm(int m, int n, int k, int a_kmajor, int aligned, int* form);
int rka_describe_weight_gradients(int batch, int seq_len, int input_size, int hidden_size, int* out, int n_out);

/* Poll rounds a recurrence kernel's wait for another workgroup's words
 * makes before it gives up (0 = the default, 2^24 rounds, about 2 s at the
 * fastest poll rate; at most 2^30).  Every recurrence grid is resident, so
 * a wait lasts about one timestep unless other kernels hold the CUs it
 * needs.  A wait that gives up aborts the launch: every workgroup leaves its time loop and
 * writes NaN into every output row it did not store (y and the reserve in
 * the forward, the gate-gradient rows in the backward) and into its final
 * states (hn, dh0), so the gradients computed from them (dW, db, dx) are
 * NaN as well; every value an aborted launch leaves is either NaN or the
 * value a complete run computes.  The call itself returns 0 (the kernels
 * are asynchronous); rka_recurrence_abort_count reports the abort.
 * Affects later launches on all threads.  No counterpart in the reference
 * (its recurrence kernels step with cooperative grid barriers, which wait
 * without a bound, and it refuses a grid that cannot be resident before
 * launching, src/rnn_kernel/a100/prod/gru.py:257-263); exported so tests
 * can drive the abort path from the host. */
int rka_set_spin_limit(int polls);

/* Failure injection for tests (-1 = off, the default): in every later
 * recurrence launch, the workgroup with block index `block` publishes its
 * exchange words where its partners never look for them, so their waits
 * give up (after the rka_set_spin_limit bound) and the launch aborts, every
 * kernel still exiting normally.  Affects later launches on all threads.
 * No counterpart in the reference; exported so tests can force the abort
 * path deterministically. */
int rka_set_stall_block(int block);

/* How recurrence workgroups publish their exchange words.
 * RKA_EXCHANGE_AUTO (the default): with plain stores, which stay in the
 * XCD's L2, when a start-up check finds every workgroup of the exchange
 * group on one XCD (the grid is laid out so that they are whenever it is
 * still resident with the group count rounded up to a multiple of 8), else
 * with agent-scope stores.  RKA_EXCHANGE_AGENT: always agent-scope stores
 * (slower; the same results bit for bit).  Affects later launches on all
 * threads.  No counterpart in the reference; exported so tests cover both
 * store paths at every shape. */
#define RKA_EXCHANGE_AUTO 0
#define RKA_EXCHANGE_AGENT 1
int rka_set_exchange_stores(int mode);

/* Number of recurrence calls on the current device that aborted (a wait
 * gave up, see rka_set_spin_limit) since the library was loaded.  A call is
 * one direction of one layer (rka_gru_forward, rka_gru_backward or a
 * recurrence-only entry point), counted once however many of its launches
 * (batch slices, time ranges) aborted.  Synchronises the device first, so
 * it covers every call enqueued before.  Host code checks it at its synchronisation points; the
 * Python front end raises RuntimeError when it has grown.  No counterpart
 * in the reference (whose launches cannot abort). */
int rka_recurrence_abort_count(unsigned long long* count);

/* Override the recurrence kernel choice for direction `dir` (0 forward,
 * 1 backward); affects later calls on all threads.  For tuning and tests.
 * kind 0: automatic (register-resident kernel when hidden_size <= 256, with
 *         the fewest batch rows per workgroup whose grid is resident, else
 *         four rows and one resident launch per batch slice; four rows and 32
 *         units per workgroup for 257 to 768, likewise; LDS-tiled above, or
 *         where the others' grid is not resident);
 * kind 1: LDS-tiled; units = hidden units per workgroup (a divisor of 64,
 *         0 = auto), param = wavefronts holding (row, unit) pairs (1, 2, 4,
 *         0 = auto);
 * kind 2: register-resident; units = 64 (or 0), param = batch rows per
 *         workgroup (1, 2, 4, 0 = auto). */
#define RKA_REC_AUTO 0
#define RKA_REC_TILED 1
#define RKA_REC_REGISTER 2
int rka_set_recurrence_config(int dir, int kind, int units, int param);

/* Describe the decomposition the next recurrence call would use for this
 * shape: writes the first min(n_out, 10) of {kind, groups (per launch),
 * slices, units, rows_per_group, pair_waves, chunk, lds_bytes, launches,
 * batch_per_launch} to out and returns 0 (n_out < 1 is an error).  A batch
 * whose grid would not be resident on an idle GPU runs as `launches`
 * launches over consecutive slices of batch_per_launch rows, each grid
 * resident (the reference refuses such a batch instead,
 * src/rnn_kernel/a100/prod/gru.py:257-263). */
int rka_describe_recurrence(int dir, int batch, int hidden_size, int* out, int n_out);

/* Evaluates the recurrence kernels' gate nonlinearities (the same device
 * functions) elementwise: sigmoid_out = sigmoid(x), tanh_out = tanh(x).
 * For accuracy tests of those functions; no reference counterpart. */
int rka_eval_gate_functions(const float* x, float* sigmoid_out, float* tanh_out, int n, void* stream);

/*
 * Measurement of the exchange the persistent recurrences step with (for
 * bench.py's roofline; no counterpart in the reference, whose recurrences
 * step with cooperative grid barriers, a100_gru_h256_kernels.cu:698-778).
 * `pairs` pairs of workgroups (eight wavefronts each, all polling; the two
 * sides of a pair eight block ids apart, so on one XCD) ping-pong a 64-bit
 * word `iters` times: plain store to publish, agent-scope loads to poll, as
 * the recurrences do.  Writes the mean round trip in ns and whether every
 * pair ran on one XCD.  Synchronous (it waits for the device and copies the
 * timings back); every wait is bounded and one that gives up is an error.
 * The workspace is device memory of rka_exchange_probe_workspace_bytes(pairs).
 */
size_t rka_exchange_probe_workspace_bytes(int pairs);
int rka_measure_exchange_latency(int pairs, int iters, void* workspace, size_t workspace_bytes,
                                 double* round_trip_ns, int* same_xcd);

/*
 * Measurement of the issue rate of non-packed fp32 FMAs (v_fmac_f32 with
 * VGPR operands, the form of the recurrences' W_hh products; for bench.py's
 * roofline, no counterpart in the reference).  Every CU runs one or two
 * 512-thread workgroups whose lanes advance 12 or 24 independent FMA chains;
 * writes the best of the four configurations as ns per wave64 instruction
 * per SIMD and as TFLOP/s over the device.  Synchronous.  The workspace is
 * device memory of rka_fma_probe_workspace_bytes() (0 if no device).
 */
size_t rka_fma_probe_workspace_bytes(void);
int rka_measure_fma_rate(void* workspace, size_t workspace_bytes, double* ns_per_instruction, double* tflops);

/*
 * Stage profiler (the native counterpart of the reference's per-phase CUDA
 * events, rnn_benchmark.py:642-694).  While enabled, every stage launch of
 * rka_gru_forward / rka_gru_backward is bracketed by a pair of hipEvents on
 * its stream; rka_profile_read() waits for the recorded events, returns the
 * summed milliseconds and launch counts per stage and clears the records.
 * Stage ids: 0 input GEMM, 1 forward recurrence, 2 backward recurrence,
 * 3 dW_hh and dW_ih split-K products (one launch), 4 their split-K
 * reductions into dW and db, 5 dx GEMM.  When dx is requested, the
 * reductions run in the dx GEMM's launch and are reported under stage 5
 * (stage 4 then has no launches).
 */
#define RKA_NUM_STAGES 6
int rka_profile_enable(int on);
int rka_profile_read(double ms_out[RKA_NUM_STAGES], int count_out[RKA_NUM_STAGES]);
const char* rka_profile_stage_name(int stage);

/*
 * Training-step operations on either side of the GRU in the reference's
 * benchmark harness (rnn_benchmark.py:510,525,636,722): the Linear(H, 1)
 * head, the mean-squared-error loss and the AdamW update, which the
 * reference runs as PyTorch ops (nn.Linear, F.mse_loss, torch.optim.AdamW).
 * Every reduction runs in a fixed order (bitwise reproducible).
 */

/* Workspace bytes of rka_mse_forward for n elements. */
size_t rka_mse_workspace_bytes(size_t n);

/* loss[0] = sum_i (pred_i - target_i)^2 / n  (F.mse_loss, reduction 'mean',
 * rnn_benchmark.py:636). */
int rka_mse_forward(const float* pred, const float* target, float* loss, void* workspace, size_t workspace_bytes,
                    size_t n, void* stream);

/* grad_pred_i = grad_loss[0] * 2 (pred_i - target_i) / n  (its backward). */
int rka_mse_backward(const float* pred, const float* target, const float* grad_loss, float* grad_pred, size_t n,
                     void* stream);

/* pred[r] = sum_h out[r, h] w[h] + b[0] for rows r < rows of out [rows, hidden]
 * (self.head = nn.Linear(hidden_size, 1); head(out).squeeze(-1),
 * rnn_benchmark.py:510,525). */
int rka_head_forward(const float* out, const float* w, const float* b, float* pred, int rows, int hidden,
                     void* stream);

/* Workspace bytes of rka_head_backward. */
size_t rka_head_backward_workspace_bytes(int rows, int hidden);

/* dout[r, h] = dpred[r] w[h] (skipped when dout is NULL),
 * dw[h] = sum_r dpred[r] out[r, h], db[0] = sum_r dpred[r]. */
int rka_head_backward(const float* out, const float* w, const float* dpred, float* dout, float* dw, float* db,
                      void* workspace, size_t workspace_bytes, int rows, int hidden, void* stream);

/* One AdamW step (torch.optim.AdamW: decoupled weight decay, bias-corrected
 * moments; rnn_benchmark.py:722) over `count` tensors: params[i], grads[i],
 * exp_avgs[i], exp_avg_sqs[i] are device pointers of numels[i] floats; the
 * pointer arrays themselves are host memory.  `step` counts from 1.  The
 * hyper-parameters are doubles: scalars such as 1 - beta2 are formed in
 * double and rounded to fp32 once, as torch forms them from Python floats. */
int rka_adamw_step(float* const* params, const float* const* grads, float* const* exp_avgs,
                   float* const* exp_avg_sqs, const size_t* numels, int count, double lr, double beta1,
                   double beta2, double eps, double weight_decay, int step, void* stream);

/*
 * The gated delta rule, a recurrence whose state is a matrix.  Per batch row and
 * value head, with the state S [key_dim, value_dim] in float32:
 *
 *   S~ = exp(g_t) S_{t-1};  e_t = v_t - S~^T k_t;  S_t = S~ + k_t (beta_t e_t)^T;
 *   o_t = scale S_t^T q_t.
 *
 * q, k [batch, tokens, key_heads, key_dim], v [batch, tokens, value_heads,
 * value_dim] and o (as v, dense) are of `dtype`; g (the logarithm of the decay, at
 * most 0; -infinity empties the state) and beta [batch, tokens, value_heads] of
 * `gate_dtype`.  Value head h uses key head h / (value_heads / key_heads).
 * key_dim is at most 256.  With `normalize` q and k are divided by
 * sqrt(|.|^2 + 1e-6) first.  States [batch, value_heads, key_dim, value_dim] are
 * dense float32.  `strides` is a host array of 15 element strides: (batch row,
 * token, head) of q, k, v, g and beta in turn; a head's elements are contiguous.
 * (No counterpart in the reference, whose one recurrence is the GRU.)
 */
#define RKA_DTYPE_F32 0
#define RKA_DTYPE_BF16 1

/* Workspace of the calls below, and what a forward saves for its backward
 * (0 for sizes that the calls refuse). */
size_t rka_gated_delta_forward_workspace_bytes(int batch, int tokens, int key_heads, int value_heads, int key_dim,
                                               int value_dim, int dtype);
size_t rka_gated_delta_reserve_bytes(int batch, int tokens, int key_heads, int value_heads, int key_dim, int value_dim);
size_t rka_gated_delta_backward_workspace_bytes(int batch, int tokens, int key_heads, int value_heads, int key_dim,
                                                int value_dim, int dtype);

/* Whole sequences.  initial_state NULL: zeros.  lengths (device, [batch], or NULL):
 * row b ends after lengths[b] tokens (clamped to 0 .. tokens); what lies behind is
 * not read, its outputs are 0.  `reserve` non-NULL saves what the backward needs. */
int rka_gated_delta_forward(const void* q, const void* k, const void* v, const void* g, const void* beta,
                            const float* initial_state, const int* lengths, void* o, float* final_state, void* reserve,
                            void* workspace, size_t workspace_bytes, int batch, int tokens, int key_heads,
                            int value_heads, int key_dim, int value_dim, const long long* strides, int dtype,
                            int gate_dtype, int normalize, double scale, void* stream);

/* Its gradients, dense, of the inputs' types; those of tokens behind a row's length
 * are 0.  grad_o and grad_final_state may be NULL (zeros), grad_initial_state NULL
 * (not wanted).  dq and dk are summed over the value heads that share a key head in a
 * fixed order. */
int rka_gated_delta_backward(const void* q, const void* k, const void* g, const void* beta, const int* lengths,
                             const void* reserve, const void* grad_o, const float* grad_final_state, void* grad_q,
                             void* grad_k, void* grad_v, void* grad_g, void* grad_beta, float* grad_initial_state,
                             void* workspace, size_t workspace_bytes, int batch, int tokens, int key_heads,
                             int value_heads, int key_dim, int value_dim, const long long* strides, int dtype,
                             int gate_dtype, int normalize, double scale, void* stream);

/* One token of each of `batch` requests (q, k [batch, key_heads, key_dim] and so on;
 * the token strides are not used).  state [num_slots, value_heads, key_dim, value_dim]
 * is updated in place: request b has state slots[b] (device, [batch]), or b if slots is
 * NULL.  Slots have to be distinct.  A negative slot is a request without a state
 * (padding of the batch): its output is 0; one from num_slots up gives NaN.  Neither
 * touches a state. */
int rka_gated_delta_step(const void* q, const void* k, const void* v, const void* g, const void* beta, float* state,
                         const int* slots, int num_slots, void* o, int batch, int key_heads, int value_heads,
                         int key_dim, int value_dim, const long long* strides, int dtype, int gate_dtype, int normalize,
                         double scale, void* stream);

/* The form that the chain over a call's chunks takes (host only), for tests and tuning.
 * Writes the first min(n_out, 3) of {32-wide steps over key_dim, blocks of 16 columns of a
 * state per workgroup, workgroups}. */
int rka_describe_gated_delta(int batch, int value_heads, int key_dim, int value_dim, int dtype, int* out, int n_out);

/*
 * The matrix product with its epilogue, y = act(x W^T + b) + r: x [rows, inputs],
 * W [outputs, inputs], b [outputs] or NULL, r [rows, outputs] or NULL and y [rows,
 * outputs], all of `dtype`; y and z are dense, the others' rows lie ldx, ldw and ldr
 * elements apart.  Those, inputs and outputs are at most 2^21.  Sums, bias, activation and residual are in float32.
 * (The reference's F.linear, src/rnn_kernel/a100/prod/gru.py:519-523, has neither.)
 */
#define RKA_ACT_NONE 0
#define RKA_ACT_RELU 1
#define RKA_ACT_GELU 2 /* z Phi(z), by the error function */
#define RKA_ACT_SILU 3
#define RKA_ACT_SIGMOID 4
#define RKA_ACT_LOGSIGMOID 5

size_t rka_linear_forward_workspace_bytes(int rows, int outputs, int inputs, int dtype);
size_t rka_linear_backward_workspace_bytes(int rows, int outputs, int inputs, int dtype);

/* `z` non-NULL receives x W^T + b (dense, of `dtype`) for the backward. */
int rka_linear_forward(const void* x, long long ldx, const void* weight, long long ldw, const void* bias,
                       const void* residual, long long ldr, void* y, void* z, void* workspace, size_t workspace_bytes,
                       int rows, int outputs, int inputs, int act, int dtype, void* stream);

/* dz = dy act'(z) (z may be NULL without an activation); grad_x = dz W, grad_weight =
 * dz^T x, grad_bias = the sum of dz's rows, each dense, or NULL if it is not wanted.
 * Every sum has a fixed order. */
int rka_linear_backward(const void* grad_y, long long ldy, const void* x, long long ldx, const void* weight, long long ldw,
                        const void* z, void* grad_x, void* grad_weight, void* grad_bias, void* workspace,
                        size_t workspace_bytes, int rows, int outputs, int inputs, int act, int dtype, void* stream);

/* The form that a product of these calls takes (host only), for tests and tuning.
 * `product`: 0 for x W^T, 1 for grad_x, 2 for grad_weight; `aligned`: whether addresses
 * and row strides are multiples of 16 bytes.  Writes the first min(n_out, 4) of {form, edge
 * of a tile, slices of the sum, workgroups}. */
#define RKA_LINEAR_FORM_ROWS 0    /* 16 columns to a workgroup, at most 32 rows */
#define RKA_LINEAR_FORM_COLUMNS 1 /* 16 rows to a workgroup, at most 32 columns */
#define RKA_LINEAR_FORM_DIRECT 2  /* tiles, operands from memory to LDS */
#define RKA_LINEAR_FORM_TILES 3   /* tiles, operands through registers */
int rka_describe_linear(int product, int rows, int outputs, int inputs, int dtype, int aligned, int* out, int n_out);

/*
 * Layer norm over rows: y = (x - mean) rstd weight + bias, rstd = 1 / sqrt(var + eps).  x
 * [rows, size], its rows ldx elements apart, y dense; weight and bias [size] or NULL; all of
 * `dtype`, statistics in float32.  size is at most 16384.  (The reference has no norm.)
 */
/* `mean` and `rstd` [rows] receive the statistics for the backward, or are both NULL. */
int rka_layer_norm_forward(const void* x, long long ldx, const void* weight, const void* bias, void* y, float* mean,
                           float* rstd, int rows, int size, double eps, int dtype, void* stream);
size_t rka_layer_norm_backward_workspace_bytes(int rows, int size, int dtype);
/* Its gradients, dense, or NULL if one is not wanted; the workspace is for those of weight
 * and bias, whose sums have a fixed order. */
int rka_layer_norm_backward(const void* grad_y, long long ldy, const void* x, long long ldx, const void* weight,
                            const float* mean, const float* rstd, void* grad_x, void* grad_weight, void* grad_bias,
                            void* workspace, size_t workspace_bytes, int rows, int size, int dtype, void* stream);

/*
 * The causal convolution of each channel over `width` tokens (2 to 8):
 * y_t = act(bias + sum_j weight[j] x_{t - width + 1 + j}), act RKA_ACT_NONE or RKA_ACT_SILU.
 * x [batch, tokens, channels] with dense channels, y [batch, tokens, channels] dense, weight
 * [channels, width], bias [channels] or NULL, states [batch, width - 1, channels] (the inputs
 * before the first token, or NULL for zeros; a row's last width - 1 inputs), all of `dtype`.
 * lengths as in rka_gated_delta_forward.  batch is at most 65535, tokens 2^20.  (The reference
 * has none.)
 */
int rka_causal_conv_forward(const void* x, long long x_batch_stride, long long x_token_stride, const void* weight,
                            const void* bias, const void* initial_state, const int* lengths, void* y, void* final_state,
                            int batch, int tokens, int channels, int width, int act, int dtype, void* stream);
size_t rka_causal_conv_backward_workspace_bytes(int batch, int tokens, int channels, int width);
/* Its gradients, dense, or NULL if one is not wanted.  grad_y and grad_final_state may be NULL
 * (zeros).  The workspace is for the gradients of weight and bias, whose sums have a fixed
 * order. */
int rka_causal_conv_backward(const void* grad_y, const void* grad_final_state, const void* x, long long x_batch_stride,
                             long long x_token_stride, const void* weight, const void* bias, const void* initial_state,
                             const int* lengths, void* grad_x, void* grad_weight, void* grad_bias, void* grad_initial_state,
                             void* workspace, size_t workspace_bytes, int batch, int tokens, int channels, int width, int act,
                             int dtype, void* stream);
/* One token of each of `batch` requests: x [batch, channels], its rows ldx apart; state
 * [num_slots, width - 1, channels] is updated in place, slots as in rka_gated_delta_step. */
int rka_causal_conv_step(const void* x, long long ldx, const void* weight, const void* bias, void* state, const int* slots,
                         int num_slots, void* y, int batch, int channels, int width, int act, int dtype, void* stream);

/*
 * The selective scan.  Per batch row, channel d of group g = d / (channels / groups) and state
 * n, the state h in float32 and s = dt + dt_bias, or with `softplus` log(1 + exp(.)) of it:
 *
 *   h_t = exp(s_t A[d, n]) h_{t-1} + s_t x_t B_t[g, n];
 *   y_t = (sum_n C_t[g, n] h_t + skip[d] x_t) silu(gate_t).
 *
 * x, dt, gate (or NULL: no gate) [batch, tokens, channels], B and C [batch, tokens, groups,
 * states] and y (dense) are of `dtype`; A [channels, states], skip and dt_bias [channels] (or
 * NULL) and the states [batch, channels, states] dense float32.  states is at most 64.
 * `strides` is a host array of 12 element strides: (batch row, token) of x, dt and gate, (batch
 * row, token, group) of B and C; channels and states are contiguous.  lengths as in
 * rka_gated_delta_forward.  tokens is at most 2^30, channels and the strides of a token 2^21; sizes of
 * which a launch would have 2^32 threads are refused (2^26 rows of up to 16 channels, 2^24 of up to
 * 64 by a forward with a reserve and the backward).  (No counterpart in the reference.)
 */
/* Workspace of the calls below, and what a forward saves for its backward (0 for sizes that
 * the calls refuse). */
size_t rka_selective_scan_forward_workspace_bytes(int batch, int tokens, int channels, int states, int groups);
size_t rka_selective_scan_reserve_bytes(int batch, int tokens, int channels, int states, int groups);
size_t rka_selective_scan_backward_workspace_bytes(int batch, int tokens, int channels, int states, int groups);

/* Whole sequences.  initial_state NULL: zeros.  `reserve` non-NULL saves what the backward
 * needs. */
int rka_selective_scan_forward(const void* x, const void* dt, const float* A, const void* B, const void* C, const float* skip,
                               const void* gate, const float* dt_bias, const float* initial_state, const int* lengths, void* y,
                               float* final_state, void* reserve, void* workspace, size_t workspace_bytes, int batch, int tokens,
                               int channels, int states, int groups, const long long* strides, int softplus, int dtype,
                               void* stream);

/* Its gradients, dense; those of tokens behind a row's length are 0.  grad_y and
 * grad_final_state may be NULL (zeros), grad_A, grad_skip, grad_dt_bias and grad_initial_state
 * NULL (not wanted); grad_gate is written where there is a gate.  Every sum has a fixed
 * order. */
int rka_selective_scan_backward(const void* x, const void* dt, const float* A, const void* B, const void* C, const float* skip,
                                const void* gate, const float* dt_bias, const int* lengths, const void* reserve,
                                const void* grad_y, const float* grad_final_state, void* grad_x, void* grad_dt, float* grad_A,
                                void* grad_B, void* grad_C, float* grad_skip, void* grad_gate, float* grad_dt_bias,
                                float* grad_initial_state, void* workspace, size_t workspace_bytes, int batch, int tokens,
                                int channels, int states, int groups, const long long* strides, int softplus, int dtype,
                                void* stream);

/* One token of each of `batch` requests (x [batch, channels] and so on; the token strides are
 * not used).  state [num_slots, channels, states] is updated in place, slots as in
 * rka_gated_delta_step. */
int rka_selective_step(const void* x, const void* dt, const float* A, const void* B, const void* C, const float* skip,
                       const void* gate, const float* dt_bias, float* state, const int* slots, int num_slots, void* y, int batch,
                       int channels, int states, int groups, const long long* strides, int softplus, int dtype, void* stream);

/*
 * The cross entropy of a product with a vocabulary: l = x W^T + b, loss = log sum exp(l) -
 * l[target] of each row, or their sum, or their mean over the rows with a target.  x [rows,
 * inputs] and W [outputs, inputs], their rows ldx and ldw elements apart, and b [outputs] or
 * NULL are of `dtype`; target [rows] 64-bit or 32-bit integers; the losses float32.  A row whose
 * target is ignore_index has no part in anything: its loss and gradient are 0 and its x is not
 * read; the mean of no rows is 0.  One whose target lies outside the vocabulary gives NaN.  The
 * logits are not kept: the backward makes them again, for a piece of the vocabulary at a
 * time.  rows, inputs, outputs and ldw are at most 2^21, and a launch has to take all logits (some
 * 2^38 in float32, 2^39 in bfloat16).  (The reference's one loss is F.mse_loss,
 * rnn_benchmark.py:636.)
 */
#define RKA_REDUCE_NONE 0
#define RKA_REDUCE_MEAN 1
#define RKA_REDUCE_SUM 2

/* What a forward leaves for its backward (its calls need it in any case), and workspaces (0
 * for sizes that the calls refuse). */
size_t rka_cross_entropy_reserve_bytes(int rows);
size_t rka_cross_entropy_forward_workspace_bytes(int rows, int inputs, int outputs, int dtype);
size_t rka_cross_entropy_backward_workspace_bytes(int rows, int inputs, int outputs, int dtype);

/* loss: [rows] without reduction, else one. */
int rka_cross_entropy_forward(const void* x, long long ldx, const void* weight, long long ldw, const void* bias,
                              const void* target, int target_is_64bit, long long ignore_index, float* loss, void* reserve,
                              void* workspace, size_t workspace_bytes, int rows, int inputs, int outputs, int reduction, int dtype,
                              void* stream);
/* grad_loss as loss.  The gradients are dense, or NULL if one is not wanted.  Every sum has a
 * fixed order. */
int rka_cross_entropy_backward(const float* grad_loss, const void* x, long long ldx, const void* weight, long long ldw,
                               const void* bias, const void* reserve, void* grad_x, void* grad_weight, void* grad_bias,
                               void* workspace, size_t workspace_bytes, int rows, int inputs, int outputs, int reduction, int dtype,
                               void* stream);

/* The forms that these calls take (host only), for tests and tuning.  `aligned`: whether the
 * weight's address and row stride are multiples of 16 bytes.  Writes the first min(n_out, 9) of
 * {RKA_LINEAR_FORM_DIRECT or _TILES of the logits and dl, edge of a tile of the forward's logits,
 * pieces of the vocabulary, columns of a piece at most, edges of dl's tiles and of grad_x's, its slices,
 * edge of grad_weight's, its slices}. */
int rka_describe_cross_entropy(int rows, int inputs, int outputs, int dtype, int aligned, int* out, int n_out);

#ifdef __cplusplus
}
#endif

#endif /* RNN_KERNEL_AMD_H */
