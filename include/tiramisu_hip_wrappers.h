/* C ABI of the runtime layer that generated Tiramisu host code calls to reach the GPU.
 *
 * This is the drop-in boundary of the HIP back-end: plain pointers and sizes, no C++ or
 * framework types.  Each entry point names the reference interface it replaces
 * (src/tiramisu_cuda_wrappers.cpp of the reference tree).  Failure model of the
 * reference is kept: a failing HIP call prints "Error at <function>: <reason>" on
 * stderr and ends the process with status 1, so successful calls return 0.
 *
 * Stream model: every call works on the calling thread's *current stream*.  It starts as
 * HIP's per-thread default stream (the reference compiles with
 * --default-stream per-thread, tiramisu_codegen_cuda.cpp:1745) and can be replaced
 * with tiramisu_hip_set_stream() by callers that time or overlap work.
 */
#ifndef TIRAMISU_HIP_WRAPPERS_H
#define TIRAMISU_HIP_WRAPPERS_H

#include <stdbool.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- memory (replaces tiramisu_cuda_malloc / tiramisu_cuda_free,
 *      tiramisu_cuda_wrappers.cpp:55-68).  Freed blocks are kept for the next request of the
 *      same size (generated functions allocate and free their temporaries on every call), up to
 *      TIRAMISU_HIP_POOL_BYTES of idle memory (default 16 GiB, 0 = no pooling); tiramisu_hip_free
 *      waits for the calling thread's stream before it takes a block back. ---- */
void *tiramisu_hip_malloc(uint64_t size);
int tiramisu_hip_free(void *ptr);

/* ---- copies (replace tiramisu_cuda_memcpy_to_device / _to_host / _to_symbol,
 *      tiramisu_cuda_wrappers.cpp:34-53).  Issued with hipMemcpyAsync on the current
 *      stream and completed before returning, like the reference's cudaMemcpy. ---- */
int tiramisu_hip_memcpy_to_device(void *to, void *from, uint64_t size);
int tiramisu_hip_memcpy_to_host(void *to, void *from, uint64_t size);
int tiramisu_hip_memcpy_to_symbol(void *to, void *from, uint64_t size);
/* Device-to-device copy; the reference prints such copies as device-to-host
 * (tiramisu_codegen_cuda.cpp:1416-1419), which its runtime tolerates by accident. */
int tiramisu_hip_memcpy_device_to_device(void *to, void *from, uint64_t size);

/* ---- synchronisation (replaces tiramisu_cuda_stream_synchronize,
 *      tiramisu_cuda_wrappers.cpp:164-169); the argument is ignored ---- */
int32_t tiramisu_hip_stream_synchronize(int32_t dummy);

/* ---- GEMM library call (replaces tiramisu_cublas_sgemm / tiramisu_cublas_dgemm,
 *      tiramisu_cuda_wrappers.cpp:74-162).  Row-major C = alpha*op(A)*op(B) + beta*C,
 *      A is MxK, B is KxN after op().  A leading dimension of 0 means tightly packed
 *      (ldA = transposeA ? M : K, ldB = transposeB ? K : N, ldC = N); offsets are in
 *      elements.  Runs this library's own MFMA kernels; no BLAS library is involved. ---- */
int tiramisu_hip_sgemm(float *A, float *B, float *C, uint64_t M, uint64_t N, uint64_t K, float alpha,
                       float beta, uint64_t ldA, uint64_t ldB, uint64_t ldC, uint64_t offsetA,
                       uint64_t offsetB, uint64_t offsetC, bool transposeA, bool transposeB);
int tiramisu_hip_dgemm(double *A, double *B, double *C, uint64_t M, uint64_t N, uint64_t K, double alpha,
                       double beta, uint64_t ldA, uint64_t ldB, uint64_t ldC, uint64_t offsetA,
                       uint64_t offsetB, uint64_t offsetC, bool transposeA, bool transposeB);
/* tiramisu_hip_sgemm for callers that cannot allocate device memory (code under HIP graph capture,
 * serving loops, harnesses that forbid hipMalloc).  No counterpart in the reference.  Same arguments,
 * same kernels, bit-identical results; the difference is where deep reductions (at most 128 tiles of
 * 64x64, no dimension of C below 32, K >= 2048: their K range is split over workgroups) keep their partial tiles and per-tile
 * counters: tiramisu_hip_sgemm takes them from a per-thread workspace that it allocates and grows with
 * hipMalloc, this entry point from a 4 MiB (+512 B of counters) array that lives in the library's code
 * object, one copy per GPU, held until the process ends.  It calls no hipMalloc / hipFree.  A problem
 * whose split needs more than the array holds (tiles x chunks x 16 KiB: e.g. 640 x 640 x 4096, 300
 * partial tiles) is refused: a message on stderr, return value 1, nothing launched -- the one case in
 * this library where a failure returns instead of ending the process.  All calls on one GPU share the
 * array: calls that overlap on one GPU (two streams, two threads) race; serialise them.  The counters
 * are cleared by a small kernel before every use.  Returns 0 on success. */
int tiramisu_hip_sgemm_static_scratch(float *A, float *B, float *C, uint64_t M, uint64_t N, uint64_t K, float alpha,
                                      float beta, uint64_t ldA, uint64_t ldB, uint64_t ldC, uint64_t offsetA,
                                      uint64_t offsetB, uint64_t offsetC, bool transposeA, bool transposeB);
/* Batch scope (no counterpart in the reference).  Between _begin and _end the calling thread's tiramisu_hip_sgemm
 * calls are gathered instead of launched; _end launches them in call order, runs of calls of one shape (sizes,
 * leading dimensions, transposition, alpha, beta) as ONE launch with a problem per blockIdx.z (up to 8 per launch).
 * The gathered calls must be independent of one another: generated code opens a scope around the GEMM call of a
 * statement that it runs for all iterations of a host loop tagged parallel.  The tile of a small product, and with it
 * the order of its sums, depends on how many calls share its launch (the last bits of the results may differ from
 * those of separate calls).  Scopes do not nest (_begin inside a
 * scope and _end outside one return 1); tiramisu_hip_sgemm_static_scratch and tiramisu_hip_dgemm are not gathered. */
int tiramisu_hip_batch_begin(void);
int tiramisu_hip_batch_end(void);

/* The scratch block that deep reductions of tiramisu_hip_sgemm use on the calling thread's current stream (partial
 * tiles and per-tile counters), or NULL before the first such call: one block per (host thread, stream, GPU), so that
 * calls of one thread on two streams may overlap.  No counterpart in the reference; for tests and diagnostics. */
void *tiramisu_hip_sgemm_workspace(void);

/* ---- memory the library keeps between calls.  No counterpart in the reference, whose generated code allocates and
 *      frees everything on every call. ---- */
/* Scratch that a generated function keeps from one call to the next (the third plane of a time-tiled stencil, the
 * hand-over area of the windowed convolution): one block per requesting site (generated code passes the address of
 * a static of its own), host thread, stream and GPU, at least `bytes` large, allocated at the first request and handed
 * out again at every later one.  *fresh (may be NULL) is 1 when this call allocated the block -- its contents are
 * undefined then -- and 0 when it is the block of the call before. */
void *tiramisu_hip_kept_scratch(const void *site, uint64_t bytes, int32_t *fresh);
/* Waits for the device, then gives back to HIP everything the library holds without anyone using it: the kept
 * scratch of all generated functions, the workspaces of tiramisu_hip_sgemm, the idle blocks of the pool behind
 * tiramisu_hip_malloc.  Returns the number of bytes released.  The caller makes sure that no generated function and
 * no GEMM call is running; later calls allocate again what they need. */
uint64_t tiramisu_hip_release_cached_memory(void);
/* What tiramisu_hip_release_cached_memory would release now. */
uint64_t tiramisu_hip_cached_memory_bytes(void);

/* ---- code objects and launches.  The reference links nvcc-compiled kernel wrappers
 *      (_kernel_N_wrapper, tiramisu_codegen_cuda.cpp:1288-1318) into the program; here
 *      generated host code is plain C++ that embeds a gfx950 code object and launches
 *      its kernels through these three calls. ---- */
/* Load a code object image (an .hsaco file's bytes) on the current device. */
void *tiramisu_hip_module_load(const void *image, uint64_t size);
/* Look a kernel up by name; exits with status 1 if the module does not define it. */
void *tiramisu_hip_module_get_function(void *module, const char *kernel_name);
/* Device address of a global variable of the module (a __constant__ array holding a buffer tagged
 * tag_gpu_constant()); exits with status 1 if the module does not define it or it is smaller
 * than `bytes`.  Replaces the `<buffer>_get_symbol()` host function the reference emits into its
 * .cu file (src/tiramisu_codegen_cuda.cpp:817-823); its result is what
 * tiramisu_hip_memcpy_to_symbol() takes as destination. */
void *tiramisu_hip_module_get_global(void *module, const char *name, uint64_t bytes);
/* Launch on the current stream.  args[i] points to the i-th kernel argument. */
int tiramisu_hip_launch(void *function, const uint32_t grid[3], const uint32_t block[3],
                        uint32_t dynamic_lds_bytes, void **args);

/* ---- host loops tagged parallel around GPU work.  The reference lowers such a loop to a Halide
 *      parallel loop (ForType::Parallel, tiramisu_codegen_halide.cpp:2104-2145): its iterations
 *      run on pool threads, each on its own per-thread default stream, and the program
 *      synchronises that stream before the iteration ends
 *      (benchmarks/DNN/blocks/LSTM/gpu_lib/generator.cpp:99-100, :133-135).  Here generated host
 *      code hands the loop body to this call: body(i, closure) runs once for every i in
 *      [first, last] on up to four pool threads, each with a stream of its own as its current
 *      stream.  The caller's stream is synchronised before the first iteration starts and every
 *      pool thread's stream before the call returns, so work before, inside and after the loop
 *      is ordered as in the serial loop; iterations must be independent of one another.
 *      Called from inside a parallel iteration, or with a single iteration, it runs the body
 *      in the calling thread. ---- */
void tiramisu_hip_parallel_for(int32_t first, int32_t last, void (*body)(int32_t, void *), void *closure);

/* ---- stream and timing helpers for wrappers and benchmarks (the reference's
 *      benchmarks bracket device work with get_time() calls,
 *      benchmarks/linear_algebra/blas/level3/sgemm/gpu/generator3.cpp:66-69) ---- */
/* Make `stream` (a hipStream_t) the calling thread's current stream; NULL restores the
 * per-thread default stream.  Pooled memory follows the stream rule of tiramisu_hip_free: a block
 * must be freed by a thread whose current stream is the one its last use was issued on (or after
 * that stream has been synchronised); freeing it from a thread on another stream may hand the
 * block out again while that work still runs. */
int tiramisu_hip_set_stream(void *stream);
void *tiramisu_hip_get_stream(void);
/* The handle under which tiramisu_hip_set_stream takes the device's null stream (torch's default stream, whose own handle is NULL). */
void *tiramisu_hip_null_stream(void);
/* Waits for the device's null stream (other libraries' default stream), whatever the calling thread's current one. */
int tiramisu_hip_null_stream_synchronize(void);
/* Calls a generated function (extern "C" int f(halide_buffer_t *...)) of up to eight arguments, all in GPU memory.  `description` holds for
 * every argument the code and the bits of its type, the number of its dimensions and their extents, outermost first.  `stream`: the kernels
 * run there, and the thread's stream is put back; NULL (another library's default stream): they run on the thread's own stream, and the call
 * waits for the device's null stream first and for that stream afterwards.  Returns what the function returns, -1 for more arguments. */
int tiramisu_hip_call(void *function, int32_t arguments, const uint64_t *pointers, const int32_t *description, void *stream);
/* A new stream that does not synchronise with the default stream (default priority), for callers that overlap
 * calls; destroy waits for the stream's work and, if it is the calling thread's current stream, restores the
 * per-thread default stream.  Scratch blocks that the runtime keeps per (thread, stream, GPU) stay allocated until
 * tiramisu_hip_release_cached_memory. */
void *tiramisu_hip_stream_create(void);
int tiramisu_hip_stream_destroy(void *stream);
void *tiramisu_hip_event_create(void);
int tiramisu_hip_event_record(void *event);              /* on the current stream */
float tiramisu_hip_event_elapsed_ms(void *start, void *stop); /* waits for `stop` */
int tiramisu_hip_event_destroy(void *event);
int tiramisu_hip_device_count(void);

/* ---- operators of a transformer's feed-forward sublayer on this build's own kernels, forward and backward (the reference has
 *      nothing of the kind).  All pointers are GPU memory; all launches go to the calling thread's stream and nothing waits.
 *      Matrices are row-major with their columns dense and `ld...` elements from row to row (0: dense rows too; gradients refuse rows of operands that
 *      overlap); results are dense and must not overlap inputs.  Weights are [outputs][inputs].  Operands may begin at any element; rows that the
 *      matrix kernels cannot load in place (odd strides of 16-bit elements) are moved to scratch first.  Sums are kept in 32 bits and rounded once.
 *      Types and activations are the numbers below.  Arguments that do not fit together, and calls whose scratch cannot be had, are refused: a message
 *      on stderr, return value 1, nothing launched.  Scratch (gradients ahead of an activation, partial sums, moved rows) is one block for each thread, stream
 *      and GPU, as large as the largest call there needed, until tiramisu_hip_release_cached_memory().  A call recorded into a graph uses at every replay the
 *      block that it was recorded with, which stays where it is: work on the stream of the recording, replays elsewhere and replays of
 *      other graphs recorded there have to wait for each other.  A source of scratch of one's own (below) is free of that. ---- */
enum tiramisu_hip_element_t { TIRAMISU_HIP_FLOAT32 = 0, TIRAMISU_HIP_FLOAT16 = 1, TIRAMISU_HIP_BFLOAT16 = 2, TIRAMISU_HIP_FLOAT8_E4M3 = 3 };
enum tiramisu_hip_activation_t {
    TIRAMISU_HIP_NONE = 0, TIRAMISU_HIP_RELU = 1, TIRAMISU_HIP_GELU = 2 /* erf */, TIRAMISU_HIP_GELU_TANH = 3, TIRAMISU_HIP_SILU = 4
};

/* sum = x + residual (both or neither; else x itself), rstd = 1 / sqrt(mean(sum^2) + eps) of each row, y = sum rstd weight, of the
 * sum ahead of its rounding.  x, residual, weight, sum: `type` (float32, float16, bfloat16); y: the same, or y_type float8_e4m3:
 * y / scale with scale = max|y| / 448 of each row (1 where that is zero, and for a row of no elements).  rstd may be null; of a row of no elements it is NaN, like its mean. */
int tiramisu_hip_rms_norm(const void *x, const void *residual, const void *weight, void *y, void *sum, float *scale, float *rstd,
                          uint64_t rows, uint64_t columns, uint64_t ldx, uint64_t ldr, float eps, int32_t type, int32_t y_type);
/* dx = rstd (g - sum rstd^2 mean(g sum)) + dsum with g = dy weight; dweight = sum over the rows of dy sum rstd.  dsum (the
 * gradient that arrives at the sum itself) may be null.  dx is the gradient of x and of the residual.  Deterministic. */
int tiramisu_hip_rms_norm_backward(const void *dy, const void *sum, const void *weight, const float *rstd, const void *dsum, void *dx,
                                   void *dweight, uint64_t rows, uint64_t columns, uint64_t ldy, uint64_t lds, uint64_t ldd, int32_t type);
/* q = x / scale in float8_e4m3, scale = max|x| / 448 of each row (1 where that is zero, and for a row of no elements). */
int tiramisu_hip_quantize_rows(const void *x, void *q, float *scale, uint64_t rows, uint64_t columns, uint64_t ldx, int32_t type);

/* z = x weight^T [x_scale of the row, weight_scale of the column] + bias; pre = z; y = activation(z) + residual.  x is M x K, weight N x K, both of
 * `type`: float16 or bfloat16 (then y_type is the same), or float8_e4m3 with scales (y_type float16 or bfloat16).  bias,
 * residual, y and pre are of y_type; bias, residual and pre may be null. */
int tiramisu_hip_linear(const void *x, const void *weight, const void *bias, const void *residual, const float *x_scale,
                        const float *weight_scale, void *y, void *pre, uint64_t M, uint64_t N, uint64_t K, uint64_t ldx, uint64_t ldw,
                        uint64_t ldr, int32_t activation, int32_t type, int32_t y_type);
/* dz = dy activation'(pre) (relu's slope at 0 is 0), dx = dz weight, dweight = dz^T x, dbias = sum over the rows of dz (the residual's gradient is dy).  Of
 * float16 or bfloat16 throughout; dz is rounded to that type ahead of the products.  dx, dweight, dbias may be null; pre is null where
 * the activation is none. */
int tiramisu_hip_linear_backward(const void *dy, const void *x, const void *weight, const void *pre, void *dx, void *dweight, void *dbias,
                                 uint64_t M, uint64_t N, uint64_t K, uint64_t ldy, uint64_t ldx, uint64_t ldw, uint64_t ldp, int32_t activation,
                                 int32_t type);
/* gate = x gate_weight^T, up = x up_weight^T (scaled like tiramisu_hip_linear), h = activation(gate) up, in one kernel.  gate and up are stored
 * where both are given (what the backward pass reads). */
int tiramisu_hip_gated_linear(const void *x, const void *gate_weight, const void *up_weight, const float *x_scale, const float *gate_scale,
                              const float *up_scale, void *h, void *gate, void *up, uint64_t M, uint64_t N, uint64_t K, uint64_t ldx, uint64_t ldg,
                              uint64_t ldu, int32_t activation, int32_t type, int32_t h_type);
/* dgate = dh up activation'(gate), dup = dh activation(gate), dx = dgate gate_weight + dup up_weight, dgate_weight = dgate^T x, dup_weight =
 * dup^T x.  dgate and dup are rounded to `type` ahead of the products.  dx may be null, and so may both weights' gradients. */
int tiramisu_hip_gated_linear_backward(const void *dh, const void *x, const void *gate_weight, const void *up_weight, const void *gate,
                                       const void *up, void *dx, void *dgate_weight, void *dup_weight, uint64_t M, uint64_t N, uint64_t K, uint64_t ldh,
                                       uint64_t ldx, uint64_t ldg, uint64_t ldu, uint64_t ld_gate, uint64_t ld_up, int32_t activation, int32_t type);
/* ---- operators of a feed-forward sublayer with experts, and of 4-bit weights: the rules above, the numbers of types and activations below them.
 *      Rows grouped by expert: `offsets` (groups + 1 of them, rising, in GPU memory; the host never reads them) say where each group's S places begin and end;
 *      places ahead of the first group's (a call for some of the experts: offsets and weights of these alone) and behind the last one's are rows of zeros in results, and give nothing
 *      to gradients.  `rows` (may be null: x holds the S places' rows, T = S) picks
 *      the row of x, of T, for each place; numbers that are none of x's give rows of zeros, whatever weights and scales hold (in dweight: dy times zeros).  Group g's weight is N x K, all of them one below the other. ---- */

/* The k largest of each token's `count` logits (ties to the lowest index, NaN above everything, minus infinity never), and their weights: softmax
 * over the chosen ones (normalise) or over all.  A place that no expert is left for has expert -1 and weight 0.  Places by expert, in order of token and rank: offsets
 * [count + 1], rows [tokens k] (token of a place; -1 behind the last), places [tokens][k] (of each choice; -1 for none).  logits: float32, float16, bfloat16; at most 1024 experts,
 * 16 choices, 2^24 tokens. */
int tiramisu_hip_route(const void *logits, int32_t *experts, float *weights, int32_t *offsets, int32_t *rows, int32_t *places, uint64_t tokens, uint64_t count, uint64_t k,
                       uint64_t ldl, int32_t normalise, int32_t type);
/* dlogits (dense, of their type) from the weights' gradient and the experts that were chosen (-1 and other numbers that are no expert: none). */
int tiramisu_hip_route_backward(const float *dweights, const void *logits, const int32_t *experts, void *dlogits, uint64_t tokens, uint64_t count, uint64_t k, uint64_t ldl,
                                int32_t normalise, int32_t type);
/* y[s] = x[rows[s]] weight[g]^T, scaled like tiramisu_hip_linear (x_scale of x's T rows, weight_scale [groups][N]).  At most 1024 groups. */
int tiramisu_hip_grouped_linear(const void *x, const void *weight, const int32_t *offsets, const int32_t *rows, const float *x_scale, const float *weight_scale, void *y,
                                uint64_t S, uint64_t T, uint64_t groups, uint64_t N, uint64_t K, uint64_t ldx, uint64_t ldw, int32_t type, int32_t y_type);
/* dx[s] = dy[s] weight[g] (of each place: the gradient of a row of x that several places picked is their sum), dweight[g] = sum over the group of dy[s]^T x[rows[s]], zeros
 * for a group without places.  Either may be null. */
int tiramisu_hip_grouped_linear_backward(const void *dy, const void *x, const void *weight, const int32_t *offsets, const int32_t *rows, void *dx, void *dweight, uint64_t S,
                                         uint64_t T, uint64_t groups, uint64_t N, uint64_t K, uint64_t ldy, uint64_t ldx, uint64_t ldw, int32_t type);
/* tiramisu_hip_gated_linear for grouped rows: h, and gate and up where both are given, of S places. */
int tiramisu_hip_grouped_gated_linear(const void *x, const void *gate_weight, const void *up_weight, const int32_t *offsets, const int32_t *rows, const float *x_scale,
                                      const float *gate_scale, const float *up_scale, void *h, void *gate, void *up, uint64_t S, uint64_t T, uint64_t groups, uint64_t N, uint64_t K,
                                      uint64_t ldx, uint64_t ldg, uint64_t ldu, int32_t activation, int32_t type, int32_t h_type);
/* ... and its gradients; dx of each place.  dgate and dup are rounded to `type` ahead of the products. */
int tiramisu_hip_grouped_gated_linear_backward(const void *dh, const void *x, const void *gate_weight, const void *up_weight, const void *gate, const void *up, const int32_t *offsets,
                                               const int32_t *rows, void *dx, void *dgate_weight, void *dup_weight, uint64_t S, uint64_t T, uint64_t groups, uint64_t N, uint64_t K,
                                               uint64_t ldh, uint64_t ldx, uint64_t ldg, uint64_t ldu, uint64_t ld_gate, uint64_t ld_up, int32_t activation, int32_t type);
/* y[t] = residual[t] + sum over j < k of weights[t][j] x[places[t][j]]; places outside of x's `rows` count as none.  weights (null: ones) in 32 bits, residual may be null;
 * the rest float16 or bfloat16. */
int tiramisu_hip_combine_rows(const void *x, const int32_t *places, const float *weights, const void *residual, void *y, uint64_t tokens, uint64_t k, uint64_t rows, uint64_t columns,
                              uint64_t ldx, uint64_t ldr, int32_t type);
/* dx[places[t][j]] = weights[t][j] dy[t] (each row is in `places` once at most), zeros where owners (the token of each row: tiramisu_hip_route's rows) name no token or one whose
 * places have left the row out;
 * dweights[t][j] = dy[t] . x[places[t][j]].  Either may be null. */
int tiramisu_hip_combine_rows_backward(const void *dy, const void *x, const int32_t *places, const int32_t *owners, const float *weights, void *dx, float *dweights, uint64_t tokens,
                                       uint64_t k, uint64_t rows, uint64_t columns, uint64_t ldy, uint64_t ldx, int32_t type);
/* Rows in 4 bits: e2m1 values (0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives), two to a byte with the first in the low half, (columns + 1) / 2 bytes a row, and for each 32 of a row the
 * power of two, as its exponent and 127 (e8m0), that is the smallest by which the largest of them is at most 6; 1 for zeros, 255 (NaN) where one is not finite.  Dense results. */
int tiramisu_hip_quantize_groups(const void *x, void *q, uint8_t *scale, uint64_t rows, uint64_t columns, uint64_t ldx, int32_t type);
/* tiramisu_hip_linear and tiramisu_hip_gated_linear with weights in 4 bits; ldq, ldg, ldu, lds, ldgs, ldus: bytes from row to row of values and scales.  x, bias, residual and results
 * are float16 or bfloat16; weights are multiplied as numbers of that type: exact in bfloat16 (6 x 2^126, 2 x 2^127 and what else is 2^128 or more, of
 * scales 253 and 254, is infinite) and within float16's range, beyond which they are infinite and below which rounded to multiples of 2^-24. */
int tiramisu_hip_four_bit_linear(const void *x, const void *q, const uint8_t *scale, const void *bias, const void *residual, void *y, uint64_t M, uint64_t N, uint64_t K, uint64_t ldx,
                                 uint64_t ldq, uint64_t lds, uint64_t ldr, int32_t activation, int32_t type);
int tiramisu_hip_four_bit_gated_linear(const void *x, const void *gate_q, const void *up_q, const uint8_t *gate_scale, const uint8_t *up_scale, void *h, uint64_t M, uint64_t N,
                                       uint64_t K, uint64_t ldx, uint64_t ldg, uint64_t ldu, uint64_t ldgs, uint64_t ldus, int32_t activation, int32_t type);
/* Where the calling thread's operator calls take their scratch from, exchanged with *source.  `take` is called once at most by a call, before it launches
 * anything, and returns GPU memory of at least `bytes` at a multiple of 256 which is the call's until what it puts on the thread's stream has run (for a call
 * recorded into a graph: until the graph is gone), or NULL, which refuses the call.  It must not throw.  take = NULL: the runtime's blocks, where every thread begins. */
struct tiramisu_hip_scratch_source { void *(*take)(uint64_t bytes, void *context); void *context; };
int tiramisu_hip_exchange_scratch_source(struct tiramisu_hip_scratch_source *source);
/* For generated code: no buffer in the place of one that may be left out, and what becomes of a refused call there -- the reference's failure
 * model, the process ends with status 1 behind the operator's message. */
float *tiramisu_hip_no_buffer(void);
int32_t *tiramisu_hip_no_numbers(void);
int tiramisu_hip_require(int32_t status);

/* ---- per-launch timing.  Between profile_start and profile_stop every tiramisu_hip_launch
 *      (and GEMM library call), from any thread, is bracketed by two events on its current
 *      stream; profile_stop waits for them and keeps one (kernel name, milliseconds) record
 *      per launch, readable until the next profile_start.  The reference has no counterpart:
 *      its benchmarks use nvprof (utils/run_gpu_bench.py). ---- */
int tiramisu_hip_profile_start(void);
int tiramisu_hip_profile_stop(void);                 /* returns the number of records */
const char *tiramisu_hip_profile_name(int record);
float tiramisu_hip_profile_ms(int record);

#ifdef __cplusplus
}
#endif
#endif
