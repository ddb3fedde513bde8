// Public C interface of libptb200.so: every entry point of the native library, grouped by source file.
// Generated by `python -m prometorch_b200._gen_header` from the PTB_API definitions; do not edit by hand.
//
// All functions are `extern "C"`; tensors cross the boundary as device pointers, launches go to the stream given
// (0 = the legacy default stream).  Functions returning int return 0 on success and -1 on failure, in which case
// ptb_last_error() holds a message for the calling thread.  Kernels that wait (on a copy, a flag of a peer GPU)
// bound their waits and report through a device status word: 0 ok, 1 a bulk copy never completed, 2 a peer never
// published its flag, 3 an index fell outside its extent.
//
// The reference exposes its native layer as C++ headers (c10/, aten/, torch/csrc/); here the native layer is this
// C ABI, which the Python package binds with ctypes and which C or C++ programs can link directly.
#pragma once
#include <cuda_runtime.h>
#include "ptb200_types.h"

#ifdef __cplusplus
extern "C" {
#endif

// ---------------------------------------------------------------------------- collectives.cu
void ptb_set_collective_timeout_ms(int ms);

int ptb_get_collective_timeout_ms();

// bufs/flags: host arrays of `world` device pointers (this rank's view of every peer's buffer / flag block).
// numel must be a multiple of 8 (bf16) or 4 (fp32).  ticket: device word, zero.  seq: strictly increasing per flag block.
int ptb_ddp_allreduce(void* const* bufs, void* const* flags, int rank, int world, long long numel, int bf16, float scale, unsigned seq, unsigned* ticket, int* status, int n_ctas, cudaStream_t st);

// The same reduction of a bf16 bucket with the result cast to fp32: every rank's `master_bufs` buffer (fp32, `numel`
// elements, symmetric like the bucket) receives the reduced, scaled gradients; the bf16 bucket keeps its local values.
int ptb_ddp_allreduce_master(void* const* bufs, void* const* master_bufs, void* const* flags, int rank, int world, long long numel, float scale, unsigned seq, unsigned* ticket, int* status, int n_ctas, cudaStream_t st);

// parts: [world][slot_elems] bf16 (local memory); resid (optional) and out: [slot_elems] bf16.
int ptb_slot_sum(const void* parts, int world, long long slot_elems, const void* resid, void* out, cudaStream_t st);

// numel: elements of the full gradient (a multiple of 8 * world); acc: numel / world floats.
int ptb_fsdp_rs_accum(void* const* bufs, void* const* flags, int rank, int world, long long numel, float* acc, float scale, unsigned seq, unsigned* ticket, int* status, int n_ctas, cudaStream_t st);

int ptb_fsdp_rs_adamw(void* const* bufs, void* const* flags, int rank, int world, long long numel, float* master, float* m, float* v, void* shard_out, float lr, float beta1, float beta2, float eps, float wd, int step, float grad_scale, unsigned seq, unsigned* ticket, int* status, int n_ctas, cudaStream_t st);

int ptb_allgather(void* const* bufs, void* const* flags, int rank, int world, const void* shard, long long shard_bytes, unsigned seq, unsigned* ticket, int* status, int n_ctas, cudaStream_t st);

int ptb_peer_barrier(void* const* flags, int rank, int world, unsigned seq, unsigned* ticket, int* status, cudaStream_t st);

// ---------------------------------------------------------------------------- decode_engine.cu
const char* ptb_last_error();

// y = epilogue(W x).  Device pointers; w2/norm_w/resid/bias may be null.
int ptb_gemv(const void* w, const void* w2, int qtype, int rows, int cols, int rowbytes, int layout, const float* x, const float* norm_w, float eps, const float* bias, const float* resid, float* out, int epilogue, int act_gelu, int n_ctas, void* scratch /* >= 16 + 8*n_ctas bytes, zeroed */, int* status, cudaStream_t stream);

int ptb_attn_decode(const float* q, const float* k, const float* v, const float* q_norm, const float* k_norm, const float* cos, const float* sin, void* k_cache, void* v_cache, float* out, float* part_o, float* part_ml, unsigned* ticket, const int* ctrl, int n_kv_heads, int group, int head_dim, int max_seq, int neox, float eps, int window, cudaStream_t stream);

void* ptb_engine_create(const PtbModelDesc* m, const PtbLayerDesc* layers, void* ext_stream);

void ptb_engine_destroy(void* h);

// Capture one token into a graph (call once, before the first replay).
int ptb_engine_capture(void* h);

// External all-reduce flow (PTB_DECODE_FLOW=external under tensor parallelism).  A token is
//   enqueue_range(0, 4) | all-reduce x | (2) | all-reduce x | (3) | ... | lm_head | all-gather result | finish_token
// where the residual vector x is ptb_engine_buffer(h, 0) (hidden floats) and this rank's {id, value bits} pair is
// ptb_engine_buffer(h, 1).  Everything is enqueued on the engine stream, so the caller can capture it in a graph.
int ptb_engine_enqueue_range(void* h, int first, int count);

void* ptb_engine_buffer(void* h, int which);

// pairs: device array [world][2] of every rank's {id, value bits} (the all-gathered result buffers).
int ptb_engine_finish_token(void* h, const void* pairs, int world);

// Write {token, pos, self_feed} (and the log cursor) through pinned memory on the engine stream.
int ptb_engine_set_ctrl(void* h, int token, int pos, int self_feed, int reset_log);

// Enqueue `n` tokens (graph replays if captured, eager launches otherwise).  Asynchronous.
int ptb_engine_run(void* h, int n);

// Host-fed step, the serving loop: copy {token,pos} in from pinned memory, run one token, copy the
// sampled id back to pinned memory, wait.  Returns the id (or -1).
int ptb_engine_step(void* h, int token, int pos);

// Scripted run: feed `n` prompt tokens starting at position pos0, then keep generating from the
// arg-max.  Sets up the control block; follow with ptb_engine_run(h, n + n_new - 1).  log[n-1+i] is
// the i-th generated token.
int ptb_engine_begin_script(void* h, const int* tokens, int n, int pos0);

int ptb_engine_sync(void* h);

// Copy the first n logged token ids to host memory; returns how many steps have run since the log reset.
int ptb_engine_read_log(void* h, int* out, int n);

int ptb_engine_status(void* h);

// Copy the phase stamps of the last token ([kernels][8] uint64 nanoseconds) to `out`; returns the kernel count.
int ptb_engine_read_trace(void* h, unsigned long long* out, int max_kernels);

void* ptb_engine_stream(void* h);

void* ptb_engine_logits(void* h);

void* ptb_engine_hidden(void* h);

void* ptb_engine_result(void* h);

// Device addresses of layer `layer`'s fp16 K and V caches, each [kv_heads][max_seq][head_dim].
int ptb_engine_kv_cache(void* h, int layer, void** k, void** v);

long ptb_engine_launches_per_token(void* h);

int ptb_engine_kv_bytes(void* h, long* out);

// Geometry report for one GEMV (tests and notes): rows per tile, stages, grid, smem, tile bytes.
int ptb_gemv_plan(int qtype, int rows, int cols, int rowbytes, int layout, int paired, int n_ctas, int* out5);

// ---------------------------------------------------------------------------- dequant.cu
// w: a matrix of N rows x cols in a GEMV streaming layout -> out bf16 [N, cols] row-major.
// layout: 0 = [segment][row][segment bytes], 1 = tiles of 16 rows.
int ptb_dequant_weight(const void* w, int qtype, int layout, int N, int cols, void* out, cudaStream_t st);

// `n` matrices of the same width, one below the other in `out` [sum of rows, cols]: one launch where they are Q4_K or Q6_K in tiles of 16 rows.
int ptb_dequant_weights(const void* const* w, const int* qtypes, const int* rows, int n, int layout, int cols, void* out, cudaStream_t st);

// What stands between the packed projection of a prompt and its attention: norm of the q and k heads (weights fp32 [D] or null; add_one: they are
// stored less one), rotary positions from pos0 (pairs (j, j + D/2), or (2j, 2j + 1)), both in place and rounded once, and k and v into the
// fp16 cache [Hk, S, D].  qkv bf16 [T, (H + 2 Hk) D]; cos, sin fp32 [S, D/2]; D 64 or 128.
int ptb_prompt_heads(void* qkv, int T, int H, int Hk, int D, const float* q_norm, const float* k_norm, int add_one, float eps, const float* cos, const float* sin, int neox, int pos0, void* k_cache, void* v_cache, int S, cudaStream_t st);

// out[t] = scale * table[ids[t]] for T ids (device int32).  status: device word, set if an id is out of range.
int ptb_dequant_rows(const void* table, int qtype, int rowbytes, int cols, const int* ids, int T, float scale, int vocab, int* status, void* out, cudaStream_t st);

// ---------------------------------------------------------------------------- experts.cu
// Routing of n tokens over O >= E router outputs: z [splits][n] fp32 logits (rows of pitch ld, splits `stride` apart), correction [O].  `always`
// experts behind the E routed ones serve every token; K = top + always.  index [n, K]: the place of a token's i-th expert in the order by expert, -1
// for an output behind the routed experts; weight [n, K]: its sigmoid score over the sum of the chosen ones, times scale (softmax: its score times
// scale), 1 for the last `always`; token [n K]: the token of every place; offsets [E + always + 1].  work: 2 n K + E ints.
int ptb_expert_route(const float* z, int splits, long long stride, long long ld, const float* correction, int n, int E, int O, int always, int softmax, int top, float scale, int* index, float* weight, int* token, int* offsets, int* work, int* status, cudaStream_t st);

// The same from the rows themselves, for few tokens: h [n, W] (pitch ldh) and the router w [O, W], both bf16 or fp32.  work: 2 n K ints and n O floats;
// done: n + 1 unsigned that are zero between calls, used by one stream at a time.
int ptb_expert_route_rows(const void* h, long long ldh, const void* w, int W, const float* correction, int n, int E, int O, int always, int softmax, int top, float scale, int* index, float* weight, int* token, int* offsets, int* work, unsigned* done, int bf16, cudaStream_t st);

// out [rows, N] = A_e B_e^T for the rows of every expert e (offsets [E + 1]), in fp32 arithmetic; `gated`: B_e has 2 N rows and the result is
// silu(gate) * up.  Row r of A is a[token[r]] (token null: a[r]), pitch lda.  bf16 or fp32 operands and result.
int ptb_expert_gemm_simt(const void* a, const int* token, long long lda, const void* b, int gated, void* out, const int* offsets, int rows, int E, int N, int K, int bf16, int* status, cudaStream_t st);

// ---------------------------------------------------------------------------- experts_sm100.cu
// out [rows, W] = h[token[r]] (rows of h [tokens] of pitch ld), bf16, for the first `count` (on the device) of at most `rows` rows; W, ld multiples
// of eight, 16-byte aligned.
int ptb_expert_gather(const void* h, long long ld, const int* token, const int* count, void* out, int rows, int W, int tokens, int* status, cudaStream_t st);

// out [rows, N] = A_e B_e^T for the sorted rows a [rows, K] (pitch lda) of every expert e (offsets [E + 1] on the device), bf16; `gated`: B_e has 2 N
// rows, gate rows first, and the result is silu(gate) * up.  N, K, lda multiples of eight.  few: the shape for few rows per expert.
int ptb_expert_gemm(const void* a, long long lda, const void* b, int gated, void* out, const int* offsets, int rows, int E, int N, int K, int few, int n_sm, int* status, cudaStream_t st);

// ---------------------------------------------------------------------------- flash_attn.cu
int ptb_flash_attn_fwd(const void* q, const void* k, const void* v, void* o, float* lse, int B, int Tq, int Tk, int H, int Hk, int D, int causal, float scale, int q_offset, cudaStream_t st);

// delta[b, h, t] = sum_d dO * O (fp32 [B, H, Tq]): the row term of the softmax backward.  dq_zero (optional): an fp32
// [B, Tq, H, D] buffer cleared in the same pass (the dQ accumulator of the backward kernel).
int ptb_flash_attn_delta(const void* o, const void* dout, float* delta, int B, int Tq, int H, int D, float* dq_zero, cudaStream_t st);

// dq: fp32 [B,Tq,H,D] zero-initialised by the caller; delta: fp32 [B,H,Tq] scratch.
int ptb_flash_attn_bwd(const void* q, const void* k, const void* v, const void* o, const void* dout, const float* lse, float* delta, float* dq, void* dk, void* dv, void* unused, int B, int Tq, int Tk, int H, int Hk, int D, int causal, float scale, int q_offset, cudaStream_t st);

// ---------------------------------------------------------------------------- flash_attn_sm100.cu
// q [B, Tq, H, D], k/v [B, Tk, Hk, D] bf16 contiguous, D in {64, 128}; o like q; lse [B, H, Tq] fp32 (natural log).
// status: device int, set non-zero if a wait timed out.
int ptb_flash_attn_fwd_sm100(const void* q, const void* k, const void* v, void* o, float* lse, int B, int Tq, int Tk, int H, int Hk, int D, int causal, float scale, int q_offset, int* status, cudaStream_t st);

// Whether the forward of these sizes runs one tile of 128 rows per CTA on a GPU of n_sm SMs (packed sequences never do).
int ptb_flash_attn_one_tile(int B, int Tq, int H, int Hk, int n_sm);

// Sequences of different lengths packed by rows: sequence i has rows cu[i] .. cu[i + 1] (cu: device int [n_seq + 1], rows in all, none longer
// than max_len) of q, k and v, whose rows are ldq, ldk and ldv elements apart with the heads packed along them; o [rows, H, D].  One launch.
int ptb_flash_attn_varlen_fwd(const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv, void* o, const int* cu, int n_seq, int max_len, long long rows, int H, int Hk, int D, int causal, float scale, int* status, cudaStream_t st);

// Backward on tcgen05.  dq: fp32 [B, Tq, H, D] (cleared here, together with the delta pass); delta: fp32 [B, H, Tq] scratch.
// dk, dv: bf16 [gsplit][B, Tk, Hk, D]: with grouped-query heads the query heads of one KV head can be split over
// `gsplit` CTAs (a divisor of H / Hk) so that small problems fill the GPU; the caller sums the slices.
int ptb_flash_attn_bwd_sm100(const void* q, const void* k, const void* v, const void* o, const void* dout, const float* lse, float* delta, float* dq, void* dk, void* dv, int B, int Tq, int Tk, int H, int Hk, int D, int causal, float scale, int q_offset, int gsplit, int* status, cudaStream_t st);

// ---------------------------------------------------------------------------- gated_attn.cu
// After the packed projection qkv (pitch ld; q heads first, k and v heads at k_col and v_col): q_out [n, H, Dp] = RMS norm of the q heads (weight qw
// [D]; null: none) times gain[pos] (fp32 [positions]; null: 1), the k heads' norm (kw) and the values go to the page slot of (req, pos).  v_first (pitch v_first_ld, optional) mixes another layer's
// values in: v = (1 - lam) v + lam v_first.  Dp, Dvp: sizes as stored, multiples of 16; the pad is zero.
int ptb_head_norm_write(const void* qkv, long long ld, int k_col, int v_col, void* q_out, void* k_pages, void* v_pages, const float* qw, const float* kw, const float* gain, int positions, const void* v_first, long long v_first_ld, float lam, const int* pos, int pos_stride, const int* req, int req_stride, const int* page_table, int pt_stride, int n_pages, int n, int H, int G, int D, int Dp, int Dv, int Dvp, float eps, int* status, int bf16, cudaStream_t st);

// Floats of workspace the row kernels need for `nsplit` > 1.
long long ptb_gated_rows_work_floats(int n, int H, int Dvp, int nsplit);

// Query rows q [n, H, Dp], each at its own position of its own sequence, against the cached keys inside their window.  max_keys: the
// most keys any row sees; nsplit CTAs share a row's keys (at most GA_KEYS each).  out [n, H Dv] in the type of q.
int ptb_gated_attn_rows(const void* q, void* out, int n, int H, int G, int Dp, int Dv, int Dvp, const int* pos, int pos_stride, const int* req, int req_stride, const int* page_table, int pt_stride, int n_pages, const void* k_pages, const void* v_pages, const float* bias, int nb, const float* talk, int window, float scale, float cap, int max_keys, float* work, int nsplit, int* status, int bf16, cudaStream_t st);

// ---------------------------------------------------------------------------- gated_prefill.cu
// Whether ptb_gated_attn_tiles takes these sizes (else: ptb_gated_attn_rows).
int ptb_gated_tiles_supported(int H, int G, int Dp, int Dvp);

// Query tiles of a prompt pass, bf16.  tiles: [n_tiles][4] int32 on the device: first row of q / out, its position, rows (<= 32), row
// of the page table; a tile's rows stand at consecutive positions of one sequence whose keys and values are in the pages.
// weights: scratch of n_tiles * H * 32 * KW bf16, KW (a multiple of 64) at least 64 times the most 64-key blocks a tile sees; per: 32-key steps a CTA of the weights kernel takes.
// tensor_cores: 1 takes the tcgen05 weights kernel where it fits, 0 the mma.sync one.
// q [n_rows, H, Dp], out [n_rows, H Dv].
int ptb_gated_attn_tiles(const void* q, void* out, int n_rows, const int* tiles, int n_tiles, int H, int G, int Dp, int Dv, int Dvp, const int* page_table, int pt_stride, int n_pages, const void* k_pages, const void* v_pages, const float* bias, int nb, const float* talk, int window, float scale, float cap, void* weights, int KW, int per, int tensor_cores, int* status, cudaStream_t st);

// ---------------------------------------------------------------------------- gemm_sm100.cu
int ptb_gemm_bf16_ex(void* const* a_ptrs, int a_shards, int a_shard_rows, long long lda, int a_mn, void* const* b_ptrs, int b_shards, int b_shard_rows, long long ldb, int b_mn, void* C, long long ldc, void* const* c_peers, int c_shards, int out_shard_rows, int M, int N, int K, const float* bias, int flags, int* status, int n_sm, cudaStream_t st, const PtbStaging* stage_a, const PtbStaging* stage_b);

// 0: use the ordinary GEMM; otherwise the split count of the skinny path (1 or more; its result needs the reduce launch).
int ptb_gemm_pick_splits(int M, int N, int K, int n_sm);

// Skinny GEMM (M <= 128), K-major operands: C[M,N] bf16 = A[M,K] B[N,K]^T (+ bias, then act: 0 none, 1 GELU, 2 square of ReLU) with `splits` K-splits whose
// fp32 partials go through `work` ([splits][M][N] floats) and one reduce launch.  N must be a multiple of 4.
int ptb_gemm_bf16_splitk(const void* A, long long lda, const void* B, long long ldb, void* C, long long ldc, int M, int N, int K, const float* bias, int act, int splits, float* work, int* status, int n_sm, cudaStream_t st);

// Only the partials: work [splits'][M][N] fp32, where splits' (returned, >= 1) is the number of splits that really ran.
// The caller's next kernel sums them (e.g. ptb_paged_rope_write_partials).  Returns -1 on error.
int ptb_gemm_bf16_splitk_partials(const void* A, long long lda, const void* B, long long ldb, int M, int N, int K, int splits, float* work, int* status, int n_sm, cudaStream_t st);

// The same product followed, in the reduce launch, by `resid_out = P + resid_in` and `y = rmsnorm(resid_out) * norm_w`
// (all bf16, [M, N] contiguous; N <= 8192).
int ptb_gemm_bf16_splitk_add_norm(const void* A, long long lda, const void* B, long long ldb, int M, int N, int K, int splits, float* work, const void* resid_in, void* resid_out, const void* norm_w, float eps, void* y, int* status, int n_sm, cudaStream_t st);

// The same product with an fp32 result (no bias).
int ptb_gemm_bf16_splitk_f32(const void* A, long long lda, const void* B, long long ldb, float* C, long long ldc, int M, int N, int K, int splits, float* work, int* status, int n_sm, cudaStream_t st);

// The same product followed, in the reduce launch, by `x += P / rms(P) * g * w; xb = bf16(x)` (x fp32 [M, N] contiguous, w an
// optional fp32 vector; N <= 8192).
int ptb_gemm_bf16_splitk_post_norm(const void* A, long long lda, const void* B, long long ldb, int M, int N, int K, int splits, float* work, const float* w, float g, float eps, float* x, void* xb, int* status, int n_sm, cudaStream_t st);

// The packed gate/up projection (N = 2 I, gate columns first) followed by out[M, I] = act(gate) * up in the reduce launch.
int ptb_gemm_bf16_splitk_gated(const void* A, long long lda, const void* B, long long ldb, int M, int N, int K, int splits, float* work, int gelu, void* out, int* status, int n_sm, cudaStream_t st);

// C[M,N] (+)= op(A) op(B)^T with bf16 operands and fp32 accumulation, all operands local.
//   a_mn == 0: A is [M, K] row-major (pitch lda);  a_mn == 1: A is stored as [K, M] row-major.
//   b_mn == 0: B is [N, K] row-major (pitch ldb);  b_mn == 1: B is stored as [K, N] row-major.
//   flags: EPI_BIAS | EPI_ACCUM | EPI_OUT_F32 | EPI_GELU | EPI_RELU2.  status: device int, set non-zero if a wait timed out.
int ptb_gemm_bf16(const void* A, long long lda, int a_mn, const void* B, long long ldb, int b_mn, void* C, long long ldc, int M, int N, int K, const float* bias, int flags, int* status, int n_sm, cudaStream_t st);

// Floats of workspace with which ptb_gemm_bf16_ws cuts the tiles of the last wave along K (0: it would not).
long long ptb_gemm_work_floats(int M, int N, int K, int n_sm);

// Whether a plain product of these sizes runs on pairs of SMs, with the workspace that ptb_gemm_work_floats asks for or without one.
int ptb_gemm_on_pairs(int M, int N, int K, int n_sm, int with_work);

// The same with a workspace of `work_floats` floats (16-byte aligned) for partial sums.
int ptb_gemm_bf16_ws(const void* A, long long lda, int a_mn, const void* B, long long ldb, int b_mn, void* C, long long ldc, int M, int N, int K, const float* bias, int flags, float* work, long long work_floats, int* status, int n_sm, cudaStream_t st);

// ---------------------------------------------------------------------------- latent_attn.cu
// Query rows of latent attention, bf16; see PtbWindowAttn: k_pages holds the cache rows (G = 1, Dp elements, of which the first Dvp are the value), q
// [n, H, Dp], out [n, H, Dvp].  nsplit CTAs share a row's pages; above one, work is needed.
int ptb_latent_attn_rows(const PtbWindowAttn* args, cudaStream_t st);

// The cached rows of whole contexts: pieces [n_pieces] int4 (first row of out, row of the page table, page of the sequence, rows <= 64); out [rows,
// row], row a multiple of eight bf16 elements.
int ptb_latent_gather(const void* pages, int n_pages, int row, const int* page_table, int pt_stride, int pt_rows, const void* pieces, int n_pieces, void* out, int rows, int* status, cudaStream_t st);

// out[r, h os + n] = sum_k x[r, h xs + k] w[h, n, k] (times sigmoid(gate[r, h])) for n rows of H heads.  rot_at > 0 (a multiple of two): columns N ..
// rot_at of a head become zero, behind them come the `rot` elements of x that follow its K, rotated to the row's position, then zeros up to os.
int ptb_head_linear(const void* x, long long ldx, int xs, const void* w, int H, int N, int K, void* out, long long ldo, int os, int n, const void* gate, long long gate_ld, int rot_at, int rot, const float* cos, const float* sin, int positions, const int* pos, int pos_stride, int* status, int bf16, cudaStream_t st);

// ---------------------------------------------------------------------------- optim_kernels.cu
// Fused AdamKiller step over one parameter group.  tensors / tensors_b: the two tables (see above), same row order;
// partial: 3 * n_chunks floats; ts: 8 * n_tensors floats (readable afterwards: scale, beta1, 1 - beta1^t, step size, clip).
int ptb_multi_tensor_adamkiller(const void* tensors, const void* tensors_b, const void* chunks, int n_chunks, const int* chunk_start, int n_tensors, int grad_bf16, const float* h, const float* grad_scale, const int* skip, float* partial, float* ts, cudaStream_t stream);

// Fused Adafactor step of ONE parameter.  rows x cols: the matrix (rows = 1 for a vector, which keeps a full second moment in
// V and passes R = C = null).  scratch: rows + ceil(rows / 256) * cols + 2 * blocks floats with blocks = 592; ts: 8 floats.
int ptb_adafactor_step(float* p, const void* g, int grad_bf16, float* R, float* Cv, float* V, float* mom, void* lowp, int rows, int cols, const float* h, const float* grad_scale, const int* skip, float* scratch, float* ts, cudaStream_t stream);

// Fused LAMB step.  chunk_start: device int [n_tensors + 1] (prefix sums of the chunk counts, in table order);
// partial: 2 * n_chunks floats of scratch; trust: n_tensors floats (the trust ratios of this step, readable afterwards).
// Every row of the table needs all three state slots (moments and the update buffer).
int ptb_multi_tensor_lamb(const void* tensors, const void* chunks, int n_chunks, const int* chunk_start, int n_tensors, int grad_bf16, const float* h, const float* grad_scale, const int* skip, float* partial, float* trust, cudaStream_t stream);

int ptb_opt_chunk();

int ptb_opt_tensor_bytes();

// tensors: device array of OptTensor rows; chunks: device int2 array of n_chunks entries; h: 16 host floats.
int ptb_multi_tensor_opt(const void* tensors, const void* chunks, int n_chunks, int kind, int grad_bf16, const float* h, const float* grad_scale, const int* skip, cudaStream_t stream);

// Total gradient norm into out[0], clip coefficient into out[1]; found_inf (optional) is set to 1 if any
// gradient is inf/nan.  `partial` holds n_chunks floats of scratch.
int ptb_multi_tensor_grad_norm(const void* tensors, const void* chunks, int n_chunks, int grad_bf16, float* partial, float max_norm, float extra_scale, float* out, int* found_inf, cudaStream_t stream);

int ptb_multi_tensor_scale(const void* tensors, const void* chunks, int n_chunks, int grad_bf16, const float* scale, cudaStream_t stream);

// ---------------------------------------------------------------------------- paged_attn.cu
int ptb_paged_rope_write(void* qkv, int n, int H, int Hk, int D, const int* pos, const int* req, const int* page_table, int pt_stride, int n_pages, const float* cos, const float* sin, int max_pos, void* k_pages, void* v_pages, void* k_out, int* status, cudaStream_t st);

// The same, reading the projection as split-K partials `work` [splits][n][(H + 2 Hk) D] fp32 (what ptb_gemm_bf16_splitk_partials
// leaves) and writing the rotated q to q_out [n, H D] bf16: the sum of the partials costs no launch of its own.
int ptb_paged_rope_write_partials(const float* work, int splits, void* q_out, int n, int H, int Hk, int D, const int* pos, const int* req, const int* page_table, int pt_stride, int n_pages, const float* cos, const float* sin, int max_pos, void* k_pages, void* v_pages, int* status, cudaStream_t st);

// Floats of workspace ptb_paged_attn_decode needs (up to sixteen splits merge on the chip).
long long ptb_paged_attn_work_floats(int B, int H, int D, int nsplit);

// One new token per request attends to its pages.  q: [B, q_stride] bf16; out: [B, H D] bf16; lens: [B].
int ptb_paged_attn_decode(const void* q, long long q_stride, void* out, int B, int H, int Hk, int D, const int* lens, const int* page_table, int pt_stride, int n_pages, const void* k_pages, const void* v_pages, float scale, float* work, int nsplit, int* status, cudaStream_t st);

// ---------------------------------------------------------------------------- paged_tree.cu
// Floats of workspace that ptb_paged_attn_tree needs, for either type of pages.
long long ptb_paged_tree_work_floats(int B, int T, int H, int Hk, int D);

// T drafted tokens of each of B requests (the latest token among them) attend to their request's cached tokens and to one another.  q: [B, T, heads] bf16 with
// pitches in elements, head h at column h * D; out [B, T, H D]; lens [B]: cached tokens before the drafted ones, node i stands in slot lens[b] + i; nodes [B]
// (null: T), rows behind them come out as zeros, as do rows that see nothing; mask [B, T]: bit j, whether the node sees node j (null: a chain).  Pages
// [n_pages, Hk, 64, D]: bf16, or e4m3 with exponents [n_pages, Hk, 64].  D is 64 or 128, T at most 64, B at most 1024.
int ptb_paged_attn_tree(const void* q, long long q_batch, long long q_row, void* out, int B, int T, int H, int Hk, int D, const int* lens, const int* nodes, const void* mask, const int* page_table, int pt_stride, int n_pages, const void* k_pages, const void* v_pages, const void* k_exp, const void* v_exp, float scale, float* work, int* status, cudaStream_t st);

// ---------------------------------------------------------------------------- paged_write.cu
// Rotate q and k of `n` tokens (pairs (j, j + D/2)); q goes to q_out [n, H D], k and v to the page slots of (req, slot), slot null: the position, negative: not
// stored.  qkv: [n, ld] bf16; cos / sin: [max_pos, D/2] fp32; k_out optional [n, Hk, D]: the rotated keys.  k_exp and v_exp null: bf16 pages
// [n_pages, Hk, 64, D]; else e4m3 pages with one biased exponent byte for a token's keys (values) of a head.  D is 64 or 128.  Tokens of one slot are equal.
int ptb_paged_write(const void* qkv, long long ld, int n, int H, int Hk, int D, const int* pos, const int* slot, const int* req, const int* page_table, int pt_stride, int pt_rows, int n_pages, const float* cos, const float* sin, int max_pos, void* q_out, void* k_out, void* k_pages, void* v_pages, void* k_exp, void* v_exp, int* status, cudaStream_t st);

// The cache entries of each request's accepted drafted tokens, moved from slot lens[b] + path[b][j] to lens[b] + j for j in 1 .. count[b], in every
// layer.  pools: [4][layers] device pointers (keys, values, their exponents or null), row: bytes of a token's keys of a head; path [B, T] ascends.
int ptb_paged_keep(void* const* pools, int layers, int B, int T, int Hk, int row, int n_pages, const int* lens, const int* path, const int* count, const int* page_table, int pt_stride, int* status, cudaStream_t st);

// ---------------------------------------------------------------------------- prompt_layers.cu
// Floats of workspace that ptb_prompt_layers needs (T, H, heads, kv_heads, D, I and n_sm of the run are read).
long long ptb_prompt_work_floats(const PtbPromptRun* r);

// Runs `n` layers: the caches filled for positions 0 .. T - 1, and, where the last layer has a next norm, the normed rows left in r->h.
int ptb_prompt_layers(const PtbPromptLayer* layers, int n, const PtbPromptRun* r, cudaStream_t st);

// ---------------------------------------------------------------------------- recurrence.cu
// out [n, C] = silu(causal convolution of x [n, C] (pitch ld) + bias) with w [taps][C] and bias [C] (or null) fp32, the current token's tap last; `add`:
// out = x + the convolution + bias.  state [slots][taps - 1][C] in the type of x.  seqs [n_seqs] int4 (first row, rows, first position, slot): a prompt pass; null: one token per row.
int ptb_short_conv(const void* x, long long ld, const float* w, const float* bias, int add, int C, int taps, void* state, void* out, int n, int slots, const int* pos, int pos_stride, const int* req, int req_stride, const void* seqs, int n_seqs, int* status, int bf16, cudaStream_t st);

// A recurrent layer over the rows of a batch, token by token; see PtbRecurrence.
int ptb_recurrence(const PtbRecurrence* args, cudaStream_t st);

// out [n, per_row gs] (bf16 or fp32) = o / rms(o) * w * act(gate), act the sigmoid (0) or SiLU (1), o fp32 in groups of gs columns, w [gs] fp32, gate [n, per_row gs] with
// row pitch ld_gate in bf16 (gate_bf16) or fp32.  first: out = g / rms(g) * w with g = o act(gate) instead; w_row: w is [per_row gs].
int ptb_group_norm_gate(const float* o, const float* w, const void* gate, int gate_bf16, long long ld_gate, void* out, int n, int per_row, int gs, float eps, int act, int first, int w_row, int bf16, cudaStream_t st);

// ---------------------------------------------------------------------------- recurrence_chunk.cu
// Bytes of workspace of ptb_recurrence_chunked, or -1 for sizes it does not take (bf16, D and Dv up to 128).
long long ptb_recurrence_chunked_bytes(const PtbRecurrence* args);

// ptb_recurrence for a prompt pass, in chunks of 64 rows; see PtbRecurrence.
int ptb_recurrence_chunked(const PtbRecurrence* args, void* work, long long bytes, cudaStream_t st);

// ---------------------------------------------------------------------------- residual.cu
// x [n, W] fp32 += branch a (+ branch b, absent with yb null); h [n, W] (bf16 or fp32) = x / rms(x) * w unless w is null.  A branch: y in
// bf16 (f32 = 0) or as the sum of `splits` fp32 matrices `stride` apart, row pitch ld; times g; RMS-normed with the fp32 weight w[W]
// when that is given.  eps sits inside every root.  status: device int, set
// non-zero if a copy never arrived.
int ptb_residual_norm(float* x, const void* ya, int f32a, int splits_a, long long stride_a, long long ld_a, const float* wa, float ga, const void* yb, int f32b, int splits_b, long long stride_b, long long ld_b, const float* wb, float gb, float eps, const float* w, void* h, int n, int W, int bf16, int* status, cudaStream_t st);

// x [n, W] fp32 = table[ids[i * id_stride]] * scale; xb: its bf16 copy (bf16 != 0; the table has the same type).
int ptb_embed_residual(const int* ids, int id_stride, const void* table, int V, int W, float scale, int n, float* x, void* xb, int* status, int bf16, cudaStream_t st);

// x [n, W] fp32 += y / rms(y) * g * w, with y [n, W] (row pitch ldy) in bf16 or fp32; xb: the bf16 copy of the new x.  w: optional
// fp32 [W].  eps sits inside the root.
int ptb_post_norm_add(const void* y, long long ldy, const float* w, float g, float eps, float* x, void* xb, int n, int W, int bf16, cudaStream_t st);

// out [m, W] (bf16 or fp32) = x[index[i]] / rms * g * w for m rows of x [rows, W] fp32; index null: the first m rows.
int ptb_row_norm(const float* x, const long long* index, int rows, const float* w, float g, float eps, void* out, int m, int W, int* status, int bf16, cudaStream_t st);

// ---------------------------------------------------------------------------- rotary_write.cu
// x [n, *] (pitch ld): q, k and v rows at the three columns.  q_out [n, H maps, Dp]: q with the first `dims` elements of every map of every
// head rotated; k, rotated likewise, and v to the page slot of (req, pos).  Dp, Dvp: sizes as stored, multiples of 16; the pad is zero.
int ptb_rope_write(const void* x, long long ld, int q_col, int k_col, int v_col, void* q_out, void* k_pages, void* v_pages, const float* cos, const float* sin, int dims, int positions, const int* pos, int pos_stride, const int* req, int req_stride, const int* page_table, int pt_stride, int n_pages, int n, int H, int G, int maps, int D, int Dp, int Dv, int Dvp, int* status, int bf16, cudaStream_t st);

// x [n, *] (pitch ld): the queries' latent [q_rank] at dq_col, the keys' latent [rank] and the shared key part [rot_dim] at dkv_col.  cq [n, q_rank]
// = RMS norm of the first times q_w; to the page slot of (req, pos) the row [RMS norm of the second times kv_w, rotated third], padded with
// zeros to rank_p and row.
int ptb_latent_write(const void* x, long long ld, int dq_col, int dkv_col, int q_rank, int rank, int rot_dim, const float* q_w, const float* kv_w, float eps, const float* cos, const float* sin, int positions, void* cq, void* pages, int rank_p, int row, const int* pos, int pos_stride, const int* req, int req_stride, const int* page_table, int pt_stride, int n_pages, int n, int* status, int bf16, cudaStream_t st);

// q [n, H (D + dims)] bf16 (pitch ld) -> out [n, H, Do + Ro]: every head's own D elements, zeros up to Do, its rotated elements, zeros up to Ro.
int ptb_latent_q(const void* q, long long ld, void* out, int n, int H, int D, int Do, int Ro, const float* cos, const float* sin, int dims, int positions, const int* pos, int pos_stride, int* status, cudaStream_t st);

// ---------------------------------------------------------------------------- sampling.cu
// Bytes of scratch for a vocabulary of V entries (zero it once before the first call).
// How many candidates the sampler behind `scratch` has dropped since the scratch was zeroed (0 unless thousands of
// logits are tied at the top-k boundary); a non-zero count means some draws ignored tied candidates.
int ptb_sample_dropped(const void* scratch, unsigned* out);

long long ptb_sample_scratch_bytes(int V);

// history: device array of `hist_cap` ids of which the first n_hist are valid; the chosen id is appended.
// top_k in 1..64.  `u` uniform in [0, 1).  temperature <= 0 returns the arg-max after the penalty.
// Three launches: histogram of the penalised logits, collection of the bins that hold the k best, final sort + draw.
int ptb_sample_logits(const float* logits, int V, int* history, int n_hist, int hist_cap, float repeat_penalty, float temperature, int top_k, float top_p, float u, void* scratch, int* out, int* ctrl_token, cudaStream_t st);

// Sample `n` requests in three launches (grid row = request).  `reqs`: host array; `d_params`: device scratch of
// ptb_sample_batch_param_bytes(n) bytes that receives the kernel parameters (one stream-ordered copy).
long long ptb_sample_batch_param_bytes(int n);

int ptb_sample_logits_batch(const PtbSampleRequest* reqs, int n, int V, void* d_params, cudaStream_t st);

// ---------------------------------------------------------------------------- scan.cu
// Floats of scratch for ptb_linear_scan_fwd / _bwd.
long long ptb_linear_scan_scratch_floats(int B, int T, int D);

// h = scan(g, x) over dim 1 of [B, T, D] tensors (bf16 or fp32, contiguous).  agg: scratch of the size above.
int ptb_linear_scan_fwd(const void* g, const void* x, void* h, float* agg, int B, int T, int D, int bf16, cudaStream_t st);

// dx[t] = dh[t] + g[t+1] dx[t+1];  dg[t] = dx[t] * h[t-1].
int ptb_linear_scan_bwd(const void* g, const void* h, const void* dh, void* dx, void* dg, float* agg, int B, int T, int D, int bf16, cudaStream_t st);

// ---------------------------------------------------------------------------- streams.cu
// x [n][streams][W] fp32: every stream of token i is table[id] + pairs[row] + at[pos]; see PtbPairEmbed.
int ptb_pair_embed(const PtbPairEmbed* args, cudaStream_t s);

// The step between two sublayers of a decoder with several residual streams; see PtbStreamStep.
int ptb_stream_step(const PtbStreamStep* args, cudaStream_t s);

// ---------------------------------------------------------------------------- symm.cu
int ptb_symm_alloc(size_t bytes, void** ptr, void* handle64);

int ptb_symm_open(const void* handle64, void** ptr);

int ptb_symm_close(void* ptr);

int ptb_symm_free(void* ptr);

// Same-process variant (one process driving several GPUs, used by tests): enable peer access.
int ptb_enable_peer_access(int dev, int peer);

// ---------------------------------------------------------------------------- tanh_norm.cu
// x [n, W] fp32 += post(y); += table[ids]; out = pre(x); see PtbTanhResidual.
int ptb_tanh_residual(const PtbTanhResidual* args, cudaStream_t s);

// out [m, W] (bf16 or fp32) = tanh(alpha x[index[i]]) w + b for m rows of x [rows, W] fp32; index null: the first m rows.
int ptb_tanh_rows(const float* x, const long long* index, int rows, float alpha, const float* w, const float* b, void* out, int m, int W, int* status, int bf16, cudaStream_t s);

// out [m, V] = cap tanh(z / cap), z fp32 with row pitch ld.
int ptb_softcap(const float* z, float* out, int m, int V, long long ld, float cap, cudaStream_t s);

// ---------------------------------------------------------------------------- train_kernels.cu
int ptb_rmsnorm_fwd(const void* x, const void* w, void* y, float* rstd, long long rows, int H, float eps, const void* resid_in, void* resid_out, int bf16, cudaStream_t st);

// dw_partial: [n_ctas, H] fp32 scratch.
int ptb_rmsnorm_bwd(const void* x, const void* w, const void* dy, const float* rstd, void* dx, void* dw, float* dw_partial, int n_ctas, long long rows, int H, const void* dresid, int bf16, cudaStream_t st);

// out[c] = sum over rows of x [rows, ld] (N columns, a multiple of eight, as are ld and the base in elements): fp32 sums, rounded once.  partial: n_parts * N floats.
int ptb_colsum(const void* x, long long rows, int N, long long ld, float* partial, int n_parts, void* out, int bf16, cudaStream_t st);

// LayerNorm over the last H of [rows, H] (H a multiple of eight up to 1024); mean, rstd fp32 [rows].
int ptb_layernorm_fwd(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, long long rows, int H, float eps, int bf16, cudaStream_t st);

// Its gradients: dx [rows, H], dwb [2, H] (of w, then of b); partial: n_ctas * 2 * H floats.
int ptb_layernorm_bwd(const void* x, const void* w, const void* dy, const float* mean, const float* rstd, void* dx, void* dwb, float* partial, int n_ctas, long long rows, int H, int bf16, cudaStream_t st);

int ptb_rope(const void* x, void* y, const float* cos, const float* sin, long long B, int T_, int heads, int D, int neox, int backward, int pos_offset, int bf16, cudaStream_t st);

// Forward: qkv -> (q, k rotated; v).  Backward (backward != 0): (dq, dk, dv) -> dqkv with the inverse rotation.
// rows = B * T; cos/sin fp32 [>= pos_offset + T, D/2]; D a multiple of 16.
int ptb_qkv_rope_split(void* qkv, void* q, void* k, void* v, const float* cos, const float* sin, long long rows, int T_, int H, int Hk, int D, int neox, int pos_offset, int backward, int bf16, cudaStream_t st);

int ptb_gated_act_fwd(const void* gu, void* out, long long rows, int I, int gelu, int bf16, cudaStream_t st);

int ptb_gated_act_bwd(const void* gu, const void* dout, void* dgu, long long rows, int I, int gelu, int bf16, cudaStream_t st);

// logits [rows, ld] (V valid columns), target int64 [rows]; loss fp32 [rows]; dlogits may alias logits or be null.
int ptb_xent(const void* logits, const long long* target, float* loss, float* lse, void* dlogits, long long rows, int V, long long ld, float grad_scale, long long ignore_index, int bf16, cudaStream_t st);

// The same with the gradient of the mean over *count rows (a device int64, at least 1).
int ptb_xent_mean(const void* logits, const long long* target, float* loss, void* dlogits, long long rows, int V, long long ld, const long long* count, long long ignore_index, int bf16, cudaStream_t st);

// x[0 .. n) *= *g (a device fp32 scalar); x 16-byte aligned.
int ptb_scale_unless_one(void* x, long long n, const float* g, int bf16, cudaStream_t st);

int ptb_rmsnorm_bwd_static(const void* x, const void* w, const void* dy, const float* rstd, void* dx, void* dw, int n_ctas, long long rows, int H, const void* dresid, int bf16, cudaStream_t st);

// ---------------------------------------------------------------------------- verify.cu
// Bytes of workspace that ptb_verify_drafts needs.
long long ptb_verify_work_bytes(int B, int T, int V);

// Which drafted tokens of B requests stay.  logits [B, T, V] (bf16 or fp32; pitches of a request and of a row in elements), tokens, parents (null: a chain) and u [B, T], nodes [B] (null: T),
// probs (null, or the draft's probabilities [B, T, V] fp32, row i what node i's child was drawn from; chains only), temperature [B].  Writes path [B, T] (accepted nodes, -1 behind),
// count [B] (accepted drafted tokens; -1 for a request without nodes) and out [B, T] (their tokens, then the drawn one, -1 behind).
int ptb_verify_drafts(const void* logits, int bf16, long long l_batch, long long l_row, const float* probs, long long p_batch, long long p_row, const int* tokens, const int* parents, const int* nodes, const float* u, const float* temperature, void* work, int* path, int* count, int* out, int B, int T, int V, cudaStream_t st);

// ---------------------------------------------------------------------------- window_attn.cu
// After the packed projection x [n, *] (pitch ld; q, k and v rows at the three columns): q_out [n, H, Dp] = q / rms(q) * qw over all H D
// columns together; k, normed over its G D columns with kw, and v go to the page slot of (req, pos).  Dp, Dvp: sizes as stored,
// multiples of 16; the pad is zero.
int ptb_proj_norm_write(const void* x, long long ld, int q_col, int k_col, int v_col, void* q_out, void* k_pages, void* v_pages, const float* qw, const float* kw, const int* pos, int pos_stride, const int* req, int req_stride, const int* page_table, int pt_stride, int n_pages, int n, int H, int G, int D, int Dp, int Dv, int Dvp, float eps, int* status, int bf16, cudaStream_t st);

// Floats of workspace the row kernels need (heads: H times the number of maps) where nsplit or the number of maps is above one.
long long ptb_window_rows_work_floats(int n, int heads, int Dvp, int nsplit);

// Query rows, each at its own position of its own sequence, against the cached keys it sees; see PtbWindowAttn.  max_keys: the most keys
// any row sees; nsplit CTAs share a row's keys (at most WA_KEYS each).
int ptb_window_attn_rows(const PtbWindowAttn* args, cudaStream_t st);

// ---------------------------------------------------------------------------- window_attn_sm100.cu
// Query tiles of a prompt pass against the keys they see, bf16; see PtbWindowAttn.  From pages: sizes as stored up to 128, one or two maps.
// Flat (flat_rows > 0, one map): Dp and rot_dim are a head's own and the shared key size, at most 128 and 64; q is [n][H][Dq] with the own
// part in front, padded with zeros to a multiple of 64, and the shared part, padded to a multiple of 16, behind it.
int ptb_window_attn_tiles(const PtbWindowAttn* args, cudaStream_t st);

#ifdef __cplusplus
}
#endif
