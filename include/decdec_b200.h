/*
 * decdec_b200 - C ABI of the B200 (sm_100a) implementation of the DecDEC decode hot path.
 *
 * Every entry point is what a foreign-function binding of the reference's `decdec_ext` module would
 * bind for that function: plain pointers, sizes, a dtype tag and a CUDA stream; no torch types.
 * "Reference" below is SNU-ARC/DecDEC; citations are paths inside that repository.
 *
 * Conventions
 *   - all functions return 0 on success, a negative DECDEC_E_* code on failure;
 *     decdec_last_error() gives the message of the last failure on the calling thread;
 *   - `dtype` is DECDEC_FP32 / DECDEC_FP16 / DECDEC_BF16 and names the element type of activations,
 *     outputs, scales, LUTs, alpha and q_bias of that call;
 *   - a linear layer is y[N] = W[N,K] x[K]; K = in_features, N = out_features;
 *   - every compute entry point ACCUMULATES into y (y += ...), like the reference kernels;
 *   - `stream` is a cudaStream_t passed as void*; work is enqueued, never synchronised;
 *   - pointers named *_dev must be device-accessible, *_host must be host memory;
 *   - the library keeps one small accumulator workspace per (device, stream).  The first compute call on a
 *     device allocates (its own and sixteen spare ones, 2 MB each) and therefore must not happen during stream capture.
 *     A stream first seen while it is capturing takes a spare; when the spares are used up it shares the
 *     device's first workspace, and that graph must then not run concurrently with work on the owning stream.
 *     Calls that share a stream are ordered; calls on different streams use different workspaces.  Graphs captured on
 *     one stream share its workspace and must not be replayed at the same time.
 */
#ifndef DECDEC_B200_H
#define DECDEC_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { DECDEC_FP32 = 0, DECDEC_FP16 = 1, DECDEC_BF16 = 2 };

enum {
    DECDEC_OK = 0,
    DECDEC_E_INVALID = -1,      /* bad argument (shape, dtype, alignment, null pointer) */
    DECDEC_E_UNSUPPORTED = -2,  /* valid in the reference but not implemented here */
    DECDEC_E_CUDA = -3,         /* a CUDA runtime call failed */
    DECDEC_E_NOMEM = -4,        /* allocation failed */
    DECDEC_E_DEVICE = -5        /* an earlier launch on the stream gave up on a bounded wait (see decdec_stream_status) */
};

/* Launch geometry of a config; replaces the dict of read_dec_config (dec_config.cu:337-354). */
typedef struct decdec_config_info {
    int32_t num_chunks;            /* ceil(K / 1024) */
    int32_t chunk_size;            /* 1024 */
    int32_t k_chunk;               /* channels selected per chunk */
    int32_t channels_per_tb;       /* packed residual columns (8 outputs each) per DEC thread block */
    int32_t n_tb;                  /* DEC thread blocks actually launched */
    int32_t block_dim_x;           /* 256 */
    int32_t block_dim_y;           /* 1 */
    int32_t shared_memory_size;    /* dynamic shared memory of a DEC-only launch, bytes */
    int32_t reduced_shared_memory; /* always 0: the reduced mode of the reference does not exist here */
} decdec_config_info;

const char* decdec_last_error(void);

/* Version / build probe: returns the compute capability the kernels were compiled for (100). */
int decdec_compiled_arch(void);

/* ---- device-side failures.  NO COUNTERPART IN THE REFERENCE (it ignores launch and device errors,
 * dec_config.cu:204-208).  Every wait inside the kernels of this library is bounded; a thread block that gives up
 * stores a code into the error word of the (device, stream) workspace: 1 = a wait for a shared-memory stage ran
 * out (DECDEC_PIPE_WAIT_NS, default 50 ms), 2 = the launch did not get the shared-memory layout it was sized for,
 * 3 = a call on the 4-bit key/value cache met a page or a slot outside the cache, or a length beyond its block table (it neither reads nor
 * writes there).
 * The output of that launch is then incomplete.  The word lives in mapped host memory, so every later compute call
 * on that stream sees it without a copy and fails with DECDEC_E_DEVICE until the stream is reset.
 *   decdec_stream_status  *error_out = the word (0 = fine); does not synchronise.
 *   decdec_stream_reset   waits for the stream, clears the word and the accumulator workspace. */
int decdec_stream_status(void* stream, uint32_t* error_out);
int decdec_stream_reset(void* stream);

/* ---- context (reference: create_dec_context, dec_context.cu:62-103) ------------------------------
 * num_tb: thread blocks given to the compensation role.  selected_rows_dev / selected_acts_dev:
 * caller-owned device buffers of `buffer_size` int32 / dtype elements; after a fused call they hold
 * the selection, before an unfused call the caller writes the rows there.  The context borrows them. */
int decdec_create_context(uint32_t num_tb, int32_t* selected_rows_dev, void* selected_acts_dev,
                          uint32_t buffer_size, int dtype, uintptr_t* out_ctx);
/* The reference has no destructor for contexts (they leak); this one is an addition. */
int decdec_destroy_context(uintptr_t ctx);

/* ---- config (reference: create/update/destroy/read_dec_config, dec_config.cu:247-354) -------------
 * q_residual: int32 [K, N/8] (packed 4-bit residual, cheatsheet.py:99-125).  If q_residual_on_device
 * is 0 the data is copied into pinned, device-mapped host memory owned by the config and fetched
 * zero-copy at run time; otherwise the device pointer is used as is (the reference prints a warning).
 * reordered_scales: dtype [N], layout [nibble][N/8]; copied into device memory owned by the config.
 * thresholds_host: dtype [K] on the host, BORROWED: entries [0] and [k-1] are read at every launch
 * (decdec.cu:66-67), so the caller keeps it alive. */
int decdec_create_config(uintptr_t ctx, uint32_t k_chunk, const int32_t* q_residual, int q_residual_on_device,
                         uint32_t K, uint32_t N, const void* reordered_scales, int scales_on_device,
                         const void* thresholds_host, int dtype, uintptr_t* out_cfg);
int decdec_update_config(uintptr_t cfg, uintptr_t new_ctx, uint32_t k_chunk);
int decdec_destroy_config(uintptr_t cfg);
int decdec_read_config(uintptr_t cfg, decdec_config_info* out);

/* ---- compensation alone (reference: dec / unfused_dec, decdec.cu:139-146, :238-245) ---------------
 * x_dev: dtype [K]; y_dev: dtype [N], accumulated into.  `dec` selects k_chunk channels per 1024
 * (bucket rule of dec.cu:78-182, ascending channel index inside a bucket) and publishes them in the
 * context buffers; `unfused_dec` takes the k rows the caller wrote into selected_rows_dev. */
int decdec_dec(uintptr_t cfg, const void* x_dev, void* y_dev, uint32_t K, uint32_t N, int dtype, void* stream);
int decdec_unfused_dec(uintptr_t cfg, const void* x_dev, void* y_dev, uint32_t K, uint32_t N, int dtype, void* stream);

/* ---- base GEMVs ------------------------------------------------------------------------------------
 * anyprec (reference: anyprec_gemv, decdec.cu:324-333): qweight int32 [planes >= bitwidth, N, K/32],
 *   lut dtype [N, 2^bitwidth]; bitwidth 3..8; fp16/bf16 only.  `planes` is the size of dim 0.
 * lutgemm (reference: lutgemm_gemv, decdec.cu:485-496): qweight int32 [K/32, bitwidth, N],
 *   alpha dtype [K/group, bitwidth, N], q_bias dtype [K/group, N]; bitwidth 1..8; N % 8 == 0.
 * sqllm (reference: sqllm_gemv, decdec.cu:594-603): qweight int32 [K*bitwidth/32, N],
 *   lut dtype [N, 2^bitwidth]; bitwidth 3 or 4. */
int decdec_anyprec_gemv(const void* x_dev, void* y_dev, const int32_t* qweight, uint32_t planes, const void* lut,
                        uint32_t N, uint32_t K, int bitwidth, int dtype, void* stream);
int decdec_lutgemm_gemv(const void* x_dev, void* y_dev, const int32_t* qweight, const void* alpha, const void* q_bias,
                        uint32_t N, uint32_t K, int bitwidth, int group_size, int dtype, void* stream);
int decdec_sqllm_gemv(const void* x_dev, void* y_dev, const int32_t* qweight, const void* lut,
                      uint32_t N, uint32_t K, int bitwidth, int dtype, void* stream);

/* lutgemm GEMV that allocates nothing.  NO COUNTERPART IN THE REFERENCE.
 * Same arguments and result as decdec_lutgemm_gemv.  The accumulator workspace that the other entry
 * points obtain with cudaMalloc is replaced by a fixed array inside the library (held by every GPU
 * that loads the library until the process exits), so the call is usable by hosts that may not call
 * cudaMalloc at that point: plug-ins of an application that owns all device memory, and real-time loops
 * that forbid calls which may synchronise the device.  Limits and duties of the caller:
 *   - out_features <= 32768, otherwise DECDEC_E_UNSUPPORTED;
 *   - the first call on a device resolves the array's address; make it before any stream capture;
 *   - all calls on one GPU share the array: calls that overlap in time on the GPU race. */
int decdec_lutgemm_gemv_noalloc(const void* x_dev, void* y_dev, const int32_t* qweight, const void* alpha,
                                const void* q_bias, uint32_t N, uint32_t K, int bitwidth, int group_size, int dtype,
                                void* stream);

/* Dense weights of a binary-coded layer for the prefill GEMM.  NO COUNTERPART IN THE REFERENCE BINDING: the reference
 * builds this tensor with a chain of torch ops on every prefill call (end-to-end/LUTGEMMLinear.py:41-82).
 * out_dev dtype [K, N] (in_features x out_features, the right operand of `x @ W`), same arithmetic as that
 * expression: the planes' +-alpha are summed, rounded to dtype, and q_bias is added in dtype. */
int decdec_lutgemm_dequant(const int32_t* qweight, const void* alpha, const void* q_bias, void* out_dev,
                           uint32_t N, uint32_t K, int bitwidth, int group_size, int dtype, void* stream);

/* ---- tensor-parallel output exchange.  NO COUNTERPART IN THE REFERENCE (it has no tensor parallelism). -------
 * One-shot push all-reduce of the [n] partial outputs of a row-parallel projection over NVLink peer memory:
 * every rank stores its vector into every peer's buffer as 16-byte lines that carry the call number beside the
 * payload (no fence, no separate flag), waits (bounded) for the peers' lines and sums in rank order, in one
 * kernel per rank.  Replaces ncclAllReduce for these 8-16 KB vectors.
 *
 *   decdec_tp_create       allocates this rank's exchange buffer on the current device; ipc_handle_out (64 bytes,
 *                          may be null) receives its cudaIpcMemHandle_t for the other processes.
 *   decdec_tp_connect_ipc  handles = [world][64] bytes, entry `rank` ignored: opens the peers' buffers.
 *   decdec_tp_connect_ptrs same, for buffers that are already addressable (several GPUs in one process).
 *   decdec_tp_allreduce    y_dev[n] <- sum over ranks, in place, on `stream`.  All ranks must make the same
 *                          sequence of calls with the same n.  Capturable in a CUDA graph.  n <= max_n,
 *                          n*sizeof(dtype) a multiple of 16, y_dev 16-byte aligned.
 *   decdec_tp_status       calls completed and the error word (1 = a wait ran out: a peer's lines did not arrive
 *                          within DECDEC_TP_WAIT_POLLS polls, default 2^21, about a second; that block's part of y was left unsummed).
 *   decdec_tp_layout       byte offsets inside an exchange buffer (call counters [world][64] u32 of which the first
 *                          row is used, slots [2][world][stride]; a slot is a sequence of lines {u32 payload, u32 call,
 *                          u32 payload, u32 call}).
 */
int decdec_tp_layout(uint32_t world, uint32_t max_n, size_t* flags_off, size_t* slots_off, size_t* slot_stride, size_t* bytes);
int decdec_tp_create(uint32_t world, uint32_t rank, uint32_t max_n, uintptr_t* comm_out, unsigned char* ipc_handle_out);
int decdec_tp_local_ptr(uintptr_t comm, void** ptr_out);
int decdec_tp_connect_ipc(uintptr_t comm, const unsigned char* handles);
int decdec_tp_connect_ptrs(uintptr_t comm, const uintptr_t* peer_ptrs);
int decdec_tp_allreduce(uintptr_t comm, void* y_dev, uint32_t n, int dtype, void* stream);
int decdec_tp_status(uintptr_t comm, uint32_t* calls_out, uint32_t* error_out);
int decdec_tp_destroy(uintptr_t comm);

/* anyprec_dequant (reference: decdec.cu:386-393): out_dev dtype [N, K] dense weights. */
int decdec_anyprec_dequant(const int32_t* qweight, const void* lut, void* out_dev,
                           uint32_t N, uint32_t K, int bitwidth, int dtype, void* stream);

/* ---- fused: base GEMV + compensation in ONE launch (reference: dec_anyprec / dec_lutgemm /
 * dec_sqllm, decdec.cu:609-779, which fork the GEMV onto a second stream).  The first thread blocks
 * of the grid run the compensation role, the rest the GEMV; both add into the same fp32
 * accumulator, rounded once into y. */
int decdec_dec_anyprec(uintptr_t cfg, const void* x_dev, void* y_dev, const int32_t* qweight, uint32_t planes,
                       const void* lut, uint32_t N, uint32_t K, int bitwidth, int dtype, void* stream);
int decdec_dec_lutgemm(uintptr_t cfg, const void* x_dev, void* y_dev, const int32_t* qweight, const void* alpha,
                       const void* q_bias, uint32_t N, uint32_t K, int bitwidth, int group_size, int dtype, void* stream);
int decdec_dec_sqllm(uintptr_t cfg, const void* x_dev, void* y_dev, const int32_t* qweight, const void* lut,
                     uint32_t N, uint32_t K, int bitwidth, int dtype, void* stream);

/* ---- GEMV next to an SM-occupying busy kernel (reference: dummy_anyprec / dummy_lutgemm /
 * dummy_sqllm, decdec.cu:874-1013): `dummy_sm` blocks of 1024 threads spin for `dummy_iters`
 * iterations on `stream` while the GEMV runs on a library-owned side stream; joined before return. */
int decdec_dummy_anyprec(const void* x_dev, void* y_dev, const int32_t* qweight, uint32_t planes, const void* lut,
                         uint32_t N, uint32_t K, int bitwidth, int dtype, int dummy_sm, long long dummy_iters, void* stream);
int decdec_dummy_lutgemm(const void* x_dev, void* y_dev, const int32_t* qweight, const void* alpha, const void* q_bias,
                         uint32_t N, uint32_t K, int bitwidth, int group_size, int dtype, int dummy_sm,
                         long long dummy_iters, void* stream);
int decdec_dummy_sqllm(const void* x_dev, void* y_dev, const int32_t* qweight, const void* lut,
                       uint32_t N, uint32_t K, int bitwidth, int dtype, int dummy_sm, long long dummy_iters, void* stream);

/* ---- the 4-bit key/value cache and what stands around it.  NO COUNTERPART IN THE REFERENCE BINDING (its models keep a dense
 * 16-bit cache, end-to-end/model.py).
 *
 * The cache is uint8 [pages, kv_heads, bytes of a page], 16-byte aligned; a page of `page_size` tokens (a multiple of 16) is a run of
 * cells of 16 tokens.  A cell of a head of `head_dim` D (64, 128, 256) elements with `group_size` G (32, 64, 128, not above D) is
 * 16 (D + 8 D/G) bytes:
 *   key codes    8 D bytes    [D/128][token][4][word of 32][2] 16-bit words of four codes; element = 128 b + 32 w + 8 [4] + 4 [2] + code
 *   value codes  8 D bytes    [D/128][token/8][8][token%8/2][word of 64][2][token%2]; element = 128 b + 64 w + 32 [2] + 4 [8] + code
 *   key steps    64 D/G bytes [token][group] pairs (step, offset) of dtype
 *   value steps  64 D/G bytes the same
 * (a head of 64 is one block of two words of 32, one of 64).  An element is offset + step * code; append takes offset = least element of
 * the group, step = (largest - least) / 15 rounded to dtype, code = (x - offset) / step to the nearest, ties to even.  A group with an
 * infinity or a NaN reads back as NaN.  dtype is DECDEC_FP16 or DECDEC_BF16 except in decdec_rotary, which takes all three.
 *
 * Rows are [tokens][heads][head_dim] with strides in elements between tokens and heads; elements of a head are neighbours.  `*_wide`: 1 if
 * the integers are int64, 0 if int32.  A slot is page * page_size + place; a negative slot is skipped (gather: zeros).  Two rows of one
 * append must not share a slot.  A page or slot outside the cache, or a length beyond the block table, raises error 3 of the stream.
 *
 *   decdec_rotary       (a, b) -> ((a cos - b sin) factor, (b cos + a sin) factor) with the angle position * frequencies[i] (64 bits), for
 *                       the pairs i of the first `rotary_dim` elements: neighbours if `interleaved`, else rotary_dim/2 apart.  The rest is
 *                       copied.  Outputs may be the inputs themselves (same pointer and strides), not overlap them otherwise.
 *   decdec_kv4_plan     lengths[requests] tokens held, fresh[requests] tokens to come, table [requests][table_cols] of pages, free_pages with
 *                       free_count[0] pages left, the last taken first.  Gives each request the pages that it lacks (in order of requests,
 *                       entered in `table`), positions and slots of the new tokens one request after another (tokens entries; behind the
 *                       last: position 0, slot -1), query_starts[requests + 1], out_lengths, out_free_count[1] and status[1]: 0, or a sum
 *                       of 1 = too few free pages, 2 = a request is longer than its table row, 4 = more than `tokens` new tokens,
 *                       8 = a negative count; then nothing is given: slots -1, query_starts 0, lengths and free_count as they were.
 *                       Outputs must not overlap inputs.
 *   decdec_kv4_append   writes rows of keys and values to their slots.
 *   decdec_kv4_gather   reads them: contiguous [tokens][kv_heads][head_dim], offset + step * code rounded to dtype (and kept finite).
 *   decdec_kv4_attention  out = softmax(scale q k^T) v per query head (head h reads key head h / (heads / kv_heads)).  Request b has the
 *                       rows query_starts[b] .. query_starts[b+1] - 1 and lengths[b] tokens in the cache, its own among them: row i stands
 *                       at position lengths[b] - queries + i and sees the tokens up to its own, the last `window` of them if window > 0.  A
 *                       row that sees nothing gives zeros (lse -inf).  max_queries bounds the rows of a request and chooses the kernel;
 *                       requests with more are computed all the same.  Rows of no request (before the first, behind the last) stay as they are,
 *                       or are cleared if clear_rest.  lse, if not null: fp32 [rows][heads], the logarithm of the sum of exp(scaled scores).
 *                       Scores and sums are fp32: keys beyond 2^100, or values whose sum weighted by up to 2^8 a token passes 2^128, may come out
 *                       as infinities or NaN.
 *                       The workspace (bytes from _workspace, 16-byte aligned) holds nothing between calls; calls that may overlap in time
 *                       need one each. */
int decdec_rotary(const void* q, int64_t q_token, int64_t q_head, uint32_t q_heads, const void* k, int64_t k_token, int64_t k_head, uint32_t k_heads,
                  void* q_out, int64_t qo_token, int64_t qo_head, void* k_out, int64_t ko_token, int64_t ko_head, const void* positions,
                  int positions_wide, const double* frequencies, uint32_t tokens, uint32_t head_dim, uint32_t rotary_dim, int interleaved,
                  float factor, int dtype, void* stream);
int decdec_kv4_plan(const int32_t* lengths, const int32_t* fresh, uint32_t requests, int32_t* table, int64_t table_stride, uint32_t table_cols,
                    const int32_t* free_pages, uint32_t free_capacity, const int32_t* free_count, uint32_t page_size, uint32_t tokens,
                    int64_t* positions, int64_t* slots, int32_t* query_starts, int32_t* out_lengths, int32_t* out_free_count, int32_t* status,
                    void* stream);
int decdec_kv4_append(const void* k, int64_t k_token, int64_t k_head, const void* v, int64_t v_token, int64_t v_head, const void* slots, int slots_wide,
                      uint32_t tokens, void* cache, uint32_t pages, uint32_t page_size, uint32_t kv_heads, uint32_t head_dim, uint32_t group_size,
                      int dtype, void* stream);
int decdec_kv4_gather(const void* cache, uint32_t pages, uint32_t page_size, uint32_t kv_heads, uint32_t head_dim, uint32_t group_size,
                      const void* slots, int slots_wide, uint32_t tokens, void* k_out, void* v_out, int dtype, void* stream);
int decdec_kv4_attention_workspace(uint32_t requests, uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t group_size,
                                   uint32_t max_queries, int dtype, size_t* bytes);
int decdec_kv4_attention(const void* q, int64_t q_token, int64_t q_head, void* out, int64_t out_token, int64_t out_head, float* lse, const void* cache,
                         uint32_t pages, uint32_t page_size, const int32_t* table, int64_t table_stride, uint32_t table_cols, const int32_t* lengths,
                         const int32_t* query_starts, uint32_t requests, uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim,
                         uint32_t group_size, uint32_t max_queries, float scale, uint32_t window, int clear_rest, void* workspace,
                         size_t workspace_bytes, int dtype, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* DECDEC_B200_H */
