/*
 * sf_q4.h -- C ABI of the B200 (sm_100a) Q4Linear kernels.
 *
 * This is the drop-in boundary for siliconfer's int4 weight-only linear path.
 * Every pointer is a DEVICE pointer (cudaMalloc / torch CUDA storage) unless a
 * comment says otherwise, and every call is asynchronous on `stream`
 * (a cudaStream_t passed as void*; NULL = legacy default stream).  The caller
 * owns every buffer, as in the reference's C kernels
 * (siliconfer/kernels/neon/q4_gemv.h:17-62).  Shape errors are reported as a
 * status code instead of the reference binding's std::runtime_error
 * (siliconfer/kernels/neon/bindings.cpp:24-40, 98-140); sf_last_error() gives
 * the same message text.
 *
 * Storage format (unchanged from the reference, q4_gemv.h:5-12 and
 * siliconfer/kernels/neon/__init__.py:42-81):
 *   W       uint8 [N, K/2]  byte j of row i = w(i,2j) | w(i,2j+1) << 4
 *                           sym: two's-complement nibbles (-8..7)
 *                           asym: unsigned nibbles (0..15)
 *   scales  float [N, K/group_size]
 *   zeros   float [N, K/group_size] or NULL (NULL selects the symmetric layout)
 *   x / X   [T, K] row-major, dtype SF_F32 / SF_F16 / SF_BF16
 *   y / Y   [T, N] row-major, dtype SF_F32 / SF_F16 / SF_BF16
 */
#ifndef SF_Q4_H_
#define SF_Q4_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum {
  SF_OK = 0,
  SF_ERR_NULL = 1,        /* a required pointer is NULL                       */
  SF_ERR_SHAPE = 2,       /* N/K/T/group_size inconsistent                     */
  SF_ERR_DTYPE = 3,       /* unknown dtype code                                */
  SF_ERR_ALIGN = 4,       /* pointer alignment the kernel needs is not met     */
  SF_ERR_CUDA = 5,        /* a CUDA runtime call failed                        */
  SF_ERR_UNSUPPORTED = 6, /* valid request this build does not implement       */
  SF_ERR_TIMEOUT = 7,     /* a device-side bounded wait expired                */
  SF_ERR_COMM = 8,        /* tensor-parallel peer exchange failed              */
  SF_ERR_CAPTURE = 9,     /* library scratch must grow while the stream is being
                             captured: run the same shape once on that stream
                             before capturing                                  */
  SF_ERR_INDEX = 10       /* a kernel met a page, position or length outside its
                             tensor; the access was skipped                    */
} sf_status;

typedef enum { SF_F32 = 0, SF_F16 = 1, SF_BF16 = 2,
               SF_E4M3 = 3 /* 8-bit float, 3 significand bits; only where a comment names it */ } sf_dtype;

/* Human-readable text of a status code, and the detailed message of the last
   failing call on this host thread (mirrors bindings.cpp:27-39 wording). */
const char* sf_status_string(int status);
const char* sf_last_error(void);
int sf_version(void);

/* ---- reference-named entry points (fp32 activations in and out) ----------
 * Each replaces the reference C function of the same role:
 *   sf_q4_gemv_sym   <- q4_gemv_sym_neon   (q4_gemv.h:17-24;  bindings.cpp:45-55)
 *   sf_q4_gemv_scalar<- q4_gemv_sym_scalar (q4_gemv.h:27-33;  bindings.cpp:60-70)
 *   sf_q4_gemv_asym  <- q4_gemv_asym_neon  (q4_gemv.h:36-43;  bindings.cpp:75-92)
 *   sf_q4_gemm_sym   <- q4_gemm_sym_neon   (q4_gemv.h:46-53;  bindings.cpp:97-119)
 *   sf_q4_gemm_asym  <- q4_gemm_asym_neon  (q4_gemv.h:56-62;  bindings.cpp:124-150)
 * Argument order and meaning follow the reference; `stream` is appended.    */
int sf_q4_gemv_sym(const uint8_t* W, const float* scales, const float* x, float* y,
                   int out_f, int in_f, int group_size, void* stream);
int sf_q4_gemv_scalar(const uint8_t* W, const float* scales, const float* x, float* y,
                      int out_f, int in_f, int group_size, void* stream);
int sf_q4_gemv_asym(const uint8_t* W, const float* scales, const float* zeros,
                    const float* x, float* y, int out_f, int in_f, int group_size,
                    void* stream);
int sf_q4_gemm_sym(const uint8_t* W, const float* scales, const float* X, float* Y,
                   int out_f, int in_f, int T, int group_size, void* stream);
int sf_q4_gemm_asym(const uint8_t* W, const float* scales, const float* zeros,
                    const float* X, float* Y, int out_f, int in_f, int T,
                    int group_size, void* stream);

/* ---- general entry point used by Q4Linear ----------------------------------
 * Y[T,N] = X[T,K] @ dequant(W)^T (+ bias), fp32 accumulation.
 * Replaces Q4Linear.__call__'s kernel dispatch (siliconfer/model/q4_linear.py:
 * 57-66): zeros != NULL selects the asymmetric kernel, bias (fp32 [N], may be
 * NULL) is added after the product.  T <= 16 (T <= 8 at group size 32) runs
 * the decode GEMV kernel in one pass over W (above 8 tokens on a two-digit
 * activation grid: rounding at most 2^-15 of each group's max |x|); T >= 48
 * runs the prefill GEMM; in between, the decode kernel runs on chunks of 8
 * tokens.  flags: bit 0 = allow programmatic
 * dependent launch (the kernel may start streaming weights before the
 * previous kernel on `stream` has finished; x is read only after it has). */
int sf_q4_linear(const uint8_t* W, const float* scales, const float* zeros,
                 const float* bias, const void* X, int x_dtype, void* Y, int y_dtype,
                 int N, int K, int T, int group_size, int flags, void* stream);
#define SF_FLAG_PDL 1

/* ---- a decode step: many GEMVs in one persistent launch -------------------
 * The reference calls Q4Linear once per projection, seven times per layer
 * (siliconfer/model/layers.py:93-95, 133, 144; q4_linear.py:49-68).  Here a
 * caller describes the whole sequence once and replays it: one cooperative
 * launch streams every task's weights back to back, so HBM stays busy across
 * projection boundaries.
 * Ordering: a task with wait_before != 0 starts a new phase.  Every task of a
 * phase reads its X only after all tasks of the previous phase have written
 * their Y (bounded device-side waits on per-task completion counters), which
 * is how o_proj <- attention(q, k, v) is expressed.  Tasks of one phase run
 * concurrently.  Only the first phase's X must exist before the launch.
 * All tasks must share T (1..16; 1..8 at group size 32), the layout (zeros NULL or not) and the group
 * class (group_size % 128, % 64 or % 32 == 0); group_size a power of two in
 * 32..256, K % 32 == 0, W/scales/zeros/X 16-byte aligned.  `workspace` is
 * caller-owned device memory of sf_q4_step_workspace_bytes(tasks, ntasks)
 * bytes, 256-byte aligned, kept alive until sf_q4_step_destroy; it holds the
 * task table, the completion counters and the activations in integer form, so
 * two handles that run concurrently need two workspaces.
 * create() uploads the table synchronously; run() is asynchronous. */
typedef struct {
  const uint8_t* W;
  const float* scales;
  const float* zeros;   /* NULL: symmetric */
  const float* bias;    /* NULL: none */
  const void* X;        /* [T, K] of x_dtype */
  void* Y;              /* [T, N] of y_dtype */
  int N, K, T, group_size, x_dtype, y_dtype, wait_before;
  int epilogue;         /* 0, or SF_EPI_SWIGLU (see sf_q4_linear_swiglu; N = gate + up rows) */
  int bits;             /* weight bit width: 0 or 4 (packed [N, K/2]), 2 (packed [N, K/4], see
                           sf_q2_linear); every task of a step has the same */
} sf_q4_task;
#define SF_EPI_SWIGLU 1
size_t sf_q4_step_workspace_bytes(const sf_q4_task* tasks, int ntasks);
int sf_q4_step_create(const sf_q4_task* tasks, int ntasks, void* workspace, size_t workspace_bytes,
                      void** handle_out);
int sf_q4_step_run(void* handle, void* stream);
void sf_q4_step_destroy(void* handle);

/* ---- 2-bit weights ------------------------------------------------------
 * The reference quantizes to 2 bits (siliconfer/quant/primitives.py:154-245,
 * quantize_sym_int2 / quantize_asym_int2) and packs four values per byte
 * (pack_int2, primitives.py:383-404: element i in bits 2i..2i+1), but its
 * loader refuses to serve them (siliconfer/engine/q4_loader.py:142-154: no
 * int2 kernel).  This is that kernel: W uint8 [N, K/4]; symmetric q in
 * [-2, 1] (two's complement, zeros NULL) or asymmetric q in [0, 3] with fp32
 * zeros; y = X @ dequant(W)^T (+ bias), dequant (q - z) * s as in
 * dequantize_sym_int2 / dequantize_asym_int2 (primitives.py:184-245).
 * K % 64 == 0 and group_size 128 or 256; any T (the decode kernel: one
 * launch up to 16 tokens, chunks of 8 above). */
int sf_q2_linear(const uint8_t* W, const float* scales, const float* zeros, const float* bias,
                 const void* X, int x_dtype, void* Y, int y_dtype, int N, int K, int T,
                 int group_size, void* stream);

/* ---- MLP gate/up with the SwiGLU activation fused ------------------------
 * Replaces the gate/up half of siliconfer's MLP.__call__ (siliconfer/model/
 * layers.py:144: down_proj(silu(gate_proj(x)) * up_proj(x))): both
 * projections read x once, in one GEMV whose epilogue writes
 *   Y[T, N] = silu(X @ Wg^T + bg) * (X @ Wu^T + bu),  silu(v) = v / (1 + e^-v),
 * ready to be down_proj's input.  W, scales, zeros and bias hold the gate and
 * up triples INTERLEAVED in blocks of 16 rows: rows 32i .. 32i+15 are gate rows
 * 16i .. 16i+15, rows 32i+16 .. 32i+31 the same up rows (2N rows in all;
 * N % 16 == 0).  Decode sizes only (T <= 16, T <= 8 at group size 32; shape
 * rules of the decode kernel); other shapes return SF_ERR_UNSUPPORTED. */
int sf_q4_linear_swiglu(const uint8_t* W, const float* scales, const float* zeros,
                        const float* bias, const void* X, int x_dtype, void* Y, int y_dtype,
                        int N, int K, int T, int group_size, void* stream);
/* The same activation applied to an already computed product of the
 * interleaved rows: in [T, 2N] fp32 (the sf_q4_linear output of those rows,
 * bias not added), bias [2N] interleaved or NULL, out [T, N] of out_dtype. */
int sf_swiglu_interleaved(const float* in, void* out, int out_dtype, int T, int N, const float* bias,
                          void* stream);

/* sf_q4_linear for T <= 16 that allocates nothing.  No counterpart in the
 * reference (its kernels need no device scratch).  sf_q4_linear keeps a
 * library-owned scratch buffer per stream and grows it with cudaMalloc the
 * first time it sees a shape; this entry point is for callers that cannot let
 * a library allocate (a process that reserves the whole GPU for its own pool,
 * code where an allocation would stall or be refused).  It uses a fixed 4 MiB
 * buffer compiled into the library's device image instead:
 *   - limits: N <= 524288 rows, and the activation blocks (about
 *     3*T*K + 8*T*K/group_size bytes) must fit in 4032 KiB, e.g. T = 8 up to
 *     K = 160000 at group 128; larger requests fail with SF_ERR_SHAPE and a
 *     message naming the limit.  When the k-split partial sums would not fit,
 *     fewer k-splits are used.
 *   - the first call on each device looks the buffer up
 *     (cudaGetSymbolAddress); make that first call before any stream capture.
 *   - there is ONE buffer per device: calls that overlap in time on the same
 *     device (other streams, other host threads) race on it.  Order them,
 *     e.g. issue them all on one stream.
 * Same arguments, layouts and results as sf_q4_linear otherwise (no flags). */
int sf_q4_linear_static_scratch(const uint8_t* W, const float* scales, const float* zeros,
                                const float* bias, const void* X, int x_dtype, void* Y,
                                int y_dtype, int N, int K, int T, int group_size, void* stream);

/* ---- tensor parallelism across the GPUs of one node -----------------------
 * The reference has no parallel form of Q4Linear (siliconfer/model/
 * q4_linear.py:32-68 is single-device); these entry points replace the
 * row-parallel projections (o_proj, down_proj; siliconfer/model/layers.py:133,
 * 144) of a model sharded over P ranks, one process per GPU.  A
 * column-parallel projection (q/k/v/gate/up) needs no exchange: each rank calls
 * sf_q4_linear on its own block of rows.  A row-parallel rank owns a block of
 * whole groups along K and calls sf_q4_linear_allreduce, which runs the GEMV
 * into the rank's exchange buffer and sums the partials of all ranks over
 * NVLink peer memory (rank order: every rank gets bitwise the same Y).
 * Set-up (once per rank, collective):
 *   sf_tp_comm_init    allocates this rank's exchange buffer (flags, two
 *                      slots of slot_bytes, then arena_bytes for the
 *                      regions of fused step tasks, see
 *                      sf_q4_step_create_tp) and writes its CUDA IPC handle
 *                      (sf_tp_handle_bytes() bytes) to handle_out;
 *   (exchange the handles between ranks, e.g. torch.distributed all_gather)
 *   sf_tp_comm_connect opens every peer's buffer (handles: world x handle
 *                      bytes, in rank order).
 * Every rank must issue the same sequence of all-reduce calls.  Waits on
 * peers are bounded (about 2 s); on expiry the kernel returns early and
 * sf_q4_check_device_error() reports SF_ERR_TIMEOUT.  An expired wait
 * POISONS the communicator for good: the ranks' call epochs are out of step,
 * so the rank that gave up marks its buffer and every peer's flag.  A peer
 * that arrives late, and every later all-reduce or fused step on any rank,
 * then returns at once without summing anything, and
 * sf_q4_check_device_error() reports SF_ERR_COMM.  Destroy the communicator
 * and create it again (on every rank) to continue. */
size_t sf_tp_handle_bytes(void);
int sf_tp_comm_init(int rank, int world, size_t slot_bytes, size_t arena_bytes, void** comm_out,
                    void* handle_out);
int sf_tp_comm_connect(void* comm, const void* handles);
/* Y[count] = sum over ranks of partial (fp32, device, count floats; NULL =
   already in place) + bias[i % ncols]; out of out_dtype. */
int sf_tp_allreduce(void* comm, const float* partial, void* out, int out_dtype, const float* bias,
                    long long count, int ncols, void* stream);
/* Row-parallel Q4Linear shard: Y = allreduce(X[T,K_shard] @ dequant(W_shard)^T) + bias. */
int sf_q4_linear_allreduce(void* comm, const uint8_t* W, const float* scales, const float* zeros,
                           const float* bias, const void* X, int x_dtype, void* Y, int y_dtype,
                           int N, int K, int T, int group_size, void* stream);
void sf_tp_comm_destroy(void* comm);

/* A tensor-parallel decode step as ONE persistent launch, the all-reduces
 * fused into the GEMV kernel.  Same tasks as sf_q4_step_create plus a role
 * per task:
 *   SF_ROLE_GEMV        an ordinary GEMV (column-parallel projections);
 *   SF_ROLE_PUSH        a row-parallel shard: each finished 32-row tile of its
 *                       fp32 partial is stored into every rank's exchange
 *                       region over NVLink (peer stores), followed by a
 *                       per-tile flag; Y may be NULL;
 *   SF_ROLE_REDUCE + i  the all-reduce of earlier task i (a PUSH task of the
 *                       same N): waits (bounded) for every rank's flag of each
 *                       tile, sums the ranks in rank order (+ bias) and
 *                       writes Y of y_dtype.  Give it task i's W, scales,
 *                       zeros, X, K and group_size (unused) and its own Y,
 *                       bias and y_dtype.
 * Regions are carved from the communicator's arena at creation (the same
 * task lists on every rank give the same offsets), two parities per region
 * so that consecutive runs never overwrite data a peer is still reading.
 * Every rank must create the same step and run it the same number of times;
 * the launch is cooperative.  The workspace is sized by
 * sf_q4_step_workspace_bytes on the same task list. */
#define SF_ROLE_GEMV 0
#define SF_ROLE_PUSH 1
#define SF_ROLE_REDUCE 2
int sf_q4_step_create_tp(const sf_q4_task* tasks, const int* roles, int ntasks, void* comm,
                         void* workspace, size_t workspace_bytes, void** handle_out);

/* ---- decode attention over an int8-quantized KV cache --------------------
 * Replaces fused_quantized_attention_decode (siliconfer/kernels/metal/
 * q4_attention.py:200-260) over the cache of siliconfer/model/kv_cache.py:49-69:
 *   q        [B, H, D] of q_dtype (one decode token per sequence)
 *   k_codes  [B, Hkv, T, D] int8, k_scales [B, Hkv, T] fp32 (per-vector scale)
 *   v_codes, v_scales likewise
 *   out      [B, H, D] of out_dtype = softmax(q.k / sqrt(D)) . v, fp32 math.
 * H % Hkv == 0 (GQA; group sizes 1, 2, 4, 7, 8), D in {64, 128, 256}.
 * n_split <= 0 picks the T-split count (sf_kv_attention_splits); the
 * caller-owned workspace holds the splits' partial results and must have
 * sf_kv_attention_workspace_bytes(B, H, D, n_split) bytes. */
size_t sf_kv_attention_workspace_bytes(int B, int H, int D, int n_split);
int sf_kv_attention_splits(int B, int Hkv, int T);
int sf_kv_attention_decode(const void* q, int q_dtype, const int8_t* k_codes, const float* k_scales,
                           const int8_t* v_codes, const float* v_scales, void* out, int out_dtype,
                           int B, int H, int Hkv, int T, int D, int n_split, void* workspace,
                           size_t workspace_bytes, void* stream);

/* ==== 8-bit decoder operators ===============================================
 * Norm, linear, rotary, cache and attention of a decoder whose activations and
 * cache are held in e4m3.  No counterpart in the reference, whose activations
 * stay fp32 and whose cache is int8 per vector.  Strides are in elements; the
 * last dimension of every tensor is contiguous.  A call with no rows (T = 0)
 * launches nothing and returns SF_OK.
 *
 * ---- RMS norm with the residual's addition ---------------------------------
 *   h = x + residual (x when residual is NULL), in fp32
 *   y = h / sqrt(mean(h^2) + eps) * weight      (weight NULL: ones)
 * x, residual and h_out [T, K] of x_dtype (row strides ldx, ldr, K); weight
 * [K] of w_dtype; h_out may be x's or residual's own memory, and is NULL exactly
 * when residual is.  y of y_dtype [T, K], row stride ldy; for SF_E4M3, y holds
 * codes and scales [T, ceil(K/128)] receives, for each row and 128 columns,
 * max|y| / 448 (1 where that is 0, at least 2^-126), codes the e4m3 values
 * nearest to y / scale, a quotient rounded to fp32.  A group that holds an
 * infinity or NaN decodes to NaN.
 * sf_quantize_e4m3: the same codes and scales of x itself. */
int sf_rms_norm(const void* x, int x_dtype, long long ldx, const void* residual, long long ldr, void* h_out,
                const void* weight, int w_dtype, float eps, void* y, int y_dtype, long long ldy, float* scales,
                int T, int K, void* stream);
int sf_quantize_e4m3(const void* x, int x_dtype, long long ldx, uint8_t* codes, long long ldy, float* scales,
                     int T, int K, void* stream);

/* ---- linear over e4m3 rows and e4m3 weights ---------------------------------
 *   Y[t,n] = sum_kb xs[t,kb] * ws[n/128,kb] * sum_{k in block kb} X[t,k] * W[n,k] (+ bias[n])
 * X [T, K] codes (row stride ldx), xs [T, ceil(K/128)] fp32 as written by
 * sf_rms_norm / sf_quantize_e4m3; W [N, K] codes (row stride ldw), ws
 * [ceil(N/128), ceil(K/128)] fp32; bias [N] fp32 or NULL; Y [T, N] of y_dtype
 * (SF_F32 / SF_F16 / SF_BF16), contiguous.  fp32 accumulation.  X and W start
 * at multiples of 16 bytes, ldx and ldw are multiples of 16. */
int sf_fp8_linear(const uint8_t* X, long long ldx, const float* xs, const uint8_t* W, long long ldw, const float* ws,
                  const float* bias, void* Y, int y_dtype, int T, int N, int K, void* stream);

/* ---- rotary positions ---------------------------------------------------------
 * out[t,h,:] = x[t,h,:] with its first `rot` elements turned, pair by pair, by
 * the angle whose cosine and sine table[pos][j] and table[pos][rot/2 + j] hold:
 * pair j is elements (j, rot/2 + j), or (2j, 2j + 1) when interleaved != 0.
 * x [T, H, D] of dtype with token and head strides xts, xhs; out likewise (it may
 * be x itself); positions [T] int32 (pos64 = 0) or int64; table fp32
 * [max_pos, rot].  rot even, rot <= D.  A position outside [0, max_pos) gives
 * NaN in the turned elements and SF_ERR_INDEX at the next error check. */
int sf_rotary(const void* x, int dtype, long long xts, long long xhs, void* out, long long ots, long long ohs,
              const void* positions, int pos64, const float* table, int max_pos, int rot, int interleaved, int T,
              int H, int D, void* stream);

/* ---- a paged cache in e4m3 ------------------------------------------------------
 * k_codes, v_codes [num_pages, n_kv_heads, page_size, head_dim] e4m3, k_scales,
 * v_scales [num_pages, n_kv_heads] fp32: value = code * scale of its page and
 * head.  Token j of sequence b is slot j % page_size of page
 * block_table[b][j / page_size].  seq_lens [batch] counts the tokens INCLUDING
 * the call's new ones; the call's token rows are packed, sequence b's being
 * rows starts[b] .. starts[b+1]-1 (starts NULL: T / batch rows each), and are
 * the sequence's last tokens.  A sequence with fewer tokens than rows has padding
 * rows in front: nothing of them is written, their query is turned as at
 * position 0, and they see no key.  So have rows before starts[0] and from
 * starts[batch] on, which are no sequence's (a captured step replayed with fewer
 * tokens).  page_size 16, 32, 64, 128 or 256; head_dim 64, 96, 128 or 256;
 * batch <= 4096; pages_per_seq * page_size <= 2^31 - 1024.  block_table, seq_lens
 * and starts are int32 device arrays; a page or length outside its tensor is
 * skipped and reported as SF_ERR_INDEX by sf_q4_check_device_error.  So are starts that fall or leave
 * the T rows: an append skips the sequences concerned, and attention gives 0 for
 * the whole call. */
typedef struct {
  uint8_t* k_codes;
  float* k_scales;
  uint8_t* v_codes;
  float* v_scales;
  const int* block_table; /* [batch, pages_per_seq] */
  const int* seq_lens;    /* [batch] */
  const int* starts;      /* [batch + 1] or NULL */
  int num_pages, n_kv_heads, page_size, head_dim, batch, pages_per_seq;
} sf_paged_cache;

/* Writes k and v [T, n_kv_heads, D] of dtype (token and head strides) as the last
 * tokens of their sequences, k turned by its position first when table is not
 * NULL; with q != NULL, also q_out [T, H, D] (contiguous) = q turned likewise.
 * A page and head keeps one scale, 2^e with the least e >= -64 for which its
 * largest finite value is <= 448 * 2^e.  When rows are added to a page that holds
 * tokens and they need a larger e, its older codes are rewritten for it (exact
 * but where they become subnormal).  Infinities are stored as +-448 * 2^e, NaN as
 * NaN, and neither counts for the scale.  A position past the table's end is
 * turned to NaN and reported as SF_ERR_INDEX.  Two sequences of one call must not
 * write to the same page. */
int sf_paged_append(const sf_paged_cache* cache, const void* k, long long kts, long long khs, const void* v,
                    long long vts, long long vhs, const void* q, long long qts, long long qhs, void* q_out, int dtype,
                    int H, int T, const float* table, int max_pos, int rot, int interleaved, void* stream);

/* Attention of q [T, H, D] over these pages: row i of sequence b's n rows has
 * position p = seq_lens[b] - n + i and sees keys max(0, p - window + 1) .. p
 * (window <= 0: 0 .. p);
 *   out[t,h,:] = sum_j softmax_j(scale * q . k_j) v_j,  lse[t,h] = log sum_j e^(scale * q . k_j).
 * H % n_kv_heads == 0 (any group size).  Softmax weights are held as fine as the
 * finer of q_dtype and out_dtype; v_scales up to 2^100, beyond which small weights
 * leave fp32's range.  A row that sees no key gives 0, and lse
 * -inf.  out [T, H, D] of out_dtype, contiguous; lse [T, H] fp32 or NULL.  The
 * workspace belongs to the caller and needs
 * sf_paged_attention_workspace_bytes(head_dim) bytes, 16-byte aligned. */
size_t sf_paged_attention_workspace_bytes(int head_dim);
int sf_paged_attention(const sf_paged_cache* cache, const void* q, int q_dtype, long long qts, long long qhs, void* out,
                       int out_dtype, float* lse, int H, int T, float scale, int window, void* workspace,
                       size_t workspace_bytes, void* stream);

/* ---- norms and rotary positions of query and key heads ----------------------------
 *   y = x / sqrt(mean(x^2) + eps) * weight       over a head's D elements (eps < 0: y = x)
 *   out = y with its first rot elements turned, pair by pair (sf_rotary's pairs), pair j
 *   by the angle of table row positions[t][axes[j]]
 * q [T, H, D] and k [T, Hkv, D] of dtype with token and head strides, q_out and k_out
 * likewise (each may be its input itself); H or Hkv may be 0.  Weights [D] of w_dtype
 * (NULL: ones).  positions [T, axes_n] int32 (pos64 = 0) or int64, contiguous; axes
 * [rot / 2] uint8, may be NULL where axes_n is 1; axes_n at most 8.  fp32 arithmetic.
 * D a multiple of 16 up to 512, of 8 up to 256, or of 4 up to 128.  A position outside
 * [0, max_pos) or an axis outside [0, axes_n) gives NaN in the elements that it turns and
 * SF_ERR_INDEX at the next error check. */
int sf_qk_norm_rotary(const void* q, long long qts, long long qhs, void* q_out, long long qots, long long qohs, int H,
                      const void* k, long long kts, long long khs, void* k_out, long long kots, long long kohs, int Hkv,
                      int dtype, const void* q_weight, const void* k_weight, int w_dtype, double eps,
                      const void* positions, int pos64, int axes_n, const uint8_t* axes, const float* table, int max_pos,
                      int rot, int interleaved, int T, int D, void* stream);
/* The same for rows that hold the last tokens of sequences, as in a call on a paged cache: seq_lens [batch], starts
 * [batch + 1] or NULL (then T is a multiple of batch).  A row that holds none (padding) is turned as at position 0
 * whatever positions says.  starts that fall or leave the rows, and lengths below 0: SF_ERR_INDEX at the next check. */
int sf_qk_norm_rotary_rows(const void* q, long long qts, long long qhs, void* q_out, long long qots, long long qohs, int H,
                           const void* k, long long kts, long long khs, void* k_out, long long kots, long long kohs, int Hkv,
                           int dtype, const void* q_weight, const void* k_weight, int w_dtype, double eps,
                           const void* positions, int pos64, int axes_n, const uint8_t* axes, const float* table, int max_pos,
                           int rot, int interleaved, int T, int D, const int* seq_lens, const int* starts, int batch,
                           void* stream);

/* ---- a paged cache in 4 bits --------------------------------------------------------
 * The e4m3 cache's tokens, pages and rules (sf_paged_cache), with another content:
 * k_codes, v_codes uint8 [num_pages, n_kv_heads, page_size, head_dim / 2] and k_scales,
 * v_scales bf16 [num_pages, n_kv_heads, page_size, 4], a scale for each quarter of a
 * vector, all 16-byte aligned.  Element e of a vector lies in quarter
 * c = e / (D / 4) at place r = e % (D / 4); its code is bits 4c .. 4c + 3 of the vector's
 * 16-bit word r (low byte first) and stands for (code - 8) * scale[c].  Scales are at
 * least 0; a vector that holds an infinity or a NaN has four NaN scales. */
typedef struct {
  uint8_t* k_codes;
  void* k_scales;
  uint8_t* v_codes;
  void* v_scales;
  const int* block_table; /* [batch, pages_per_seq] */
  const int* seq_lens;    /* [batch] */
  const int* starts;      /* [batch + 1] or NULL */
  int num_pages, n_kv_heads, page_size, head_dim, batch, pages_per_seq;
} sf_paged4_cache;

/* sf_paged_append for this cache, with sf_qk_norm_rotary's norms, axes and positions for
 * q and k on the way (positions NULL: a token's place in its sequence; a padding row's
 * query is turned as at position 0 whatever positions says).  table NULL: nothing is
 * turned; eps < 0: nothing is normed.  For each quarter of a vector
 *   scale = max|y| / 7.5, rounded to fp32 and then to bf16, at least 2^-126
 *   code  = y / scale, rounded to the nearest whole number (ties to even) and limited to
 *           -8 .. 7, plus 8
 * with y in fp64 for keys and values.  Two rows of one call must not be the same token. */
int sf_paged4_append(const sf_paged4_cache* cache, const void* k, long long kts, long long khs, const void* v,
                     long long vts, long long vhs, const void* q, long long qts, long long qhs, void* q_out, int dtype,
                     int H, int T, const void* q_weight, const void* k_weight, int w_dtype, double eps,
                     const void* positions, int pos64, int axes_n, const uint8_t* axes, const float* table, int max_pos,
                     int rot, int interleaved, void* stream);

/* sf_paged_attention over this cache.  A row that sees a key or value vector with NaN
 * scales is NaN as a whole.  Scales up to 2^100, of values from 2^-60; smaller ones lose digits,
 * and values below 2^-80 may count as 0.  Scales may lie any number of powers of two apart
 * between tokens; within a vector, a quarter's scale 2^20 and more below the largest loses
 * digits.  16-bit queries and outputs: weights are fp16 numbers, and in long runs keys and
 * values are rounded to 11 bits, so that a score, and lse, is off by up to 2^-12 of
 * sum |q k| there. */
size_t sf_paged4_attention_workspace_bytes(int head_dim);
int sf_paged4_attention(const sf_paged4_cache* cache, const void* q, int q_dtype, long long qts, long long qhs, void* out,
                        int out_dtype, float* lse, int H, int T, float scale, int window, void* workspace,
                        size_t workspace_bytes, void* stream);

/* Device dequant to fp32/fp16/bf16 [N, K].  fp32 output is bit-exact with
   dequantize_sym / dequantize_asym (siliconfer/quant/primitives.py:54-75,
   117-140); fp16/bf16 are that value rounded to nearest even. */
int sf_q4_dequant(const uint8_t* W, const float* scales, const float* zeros, void* out,
                  int out_dtype, int N, int K, int group_size, void* stream);

/* Device RTN quantize + pack of an fp32 [N, K] weight, bit-exact with
   pack_weights_sym / pack_weights_asym (siliconfer/kernels/neon/__init__.py:
   42-81 -> siliconfer/quant/primitives.py:24-51, 82-114).  zeros == NULL
   selects symmetric packing. */
int sf_q4_quantize_pack(const float* W, uint8_t* packed, float* scales, float* zeros,
                        int N, int K, int group_size, void* stream);

/* Sticky device-side error word (set when a bounded wait inside a kernel
   expires, when a tensor-parallel kernel met a poisoned communicator, or when a
   paged-cache or rotary kernel met an index outside its tensor).
   Synchronous: reads and clears it.  Returns SF_OK, SF_ERR_TIMEOUT,
   SF_ERR_INDEX, or SF_ERR_COMM (poisoned communicator; takes precedence, then
   an expired wait). */
int sf_q4_check_device_error(void);

/* Number of kernels this library has launched since load (host counter). */
long long sf_q4_launch_count(void);

#ifdef __cplusplus
}
#endif
#endif /* SF_Q4_H_ */
