/*
 * C ABI of the MI355X (gfx950) complex-GEMM library: plain pointers and sizes,
 * opaque handles, integer status codes. These entry points are what the C++
 * classes of the ccglib API bind to (include/ccglib/...): each section names the
 * reference interface it stands in for, as file:line in the reference tree.
 *
 * Conventions
 *  - Every function returns CCGLIB_OK (0) or a non-zero status; the text of the
 *    last failure on the calling thread is returned by ccglib_last_error().
 *  - `device` is a HIP device ordinal; `stream` is a hipStream_t passed as
 *    void* (NULL = the default stream). All run functions only enqueue work on
 *    that stream and return; they never synchronise, allocate or free, except
 *    the *_run_host variants, which stage the host buffer through a
 *    stream-ordered temporary.
 *  - Pointers given to run functions are device pointers unless the name says
 *    host. The library never owns caller buffers.
 *  - Enum arguments are plain ints holding the values of the reference enums
 *    (repeated below as CCGLIB_* constants).
 *  - Objects are not thread-safe; use one per thread or serialise calls.
 */
#ifndef CCGLIB_AMD_H_
#define CCGLIB_AMD_H_

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

#define CCGLIB_API __attribute__((visibility("default")))

/* status codes */
enum {
  CCGLIB_OK = 0,
  CCGLIB_ERROR_INVALID_ARGUMENT = 1, /* bad handle, null pointer, bad enum   */
  CCGLIB_ERROR_UNSUPPORTED = 2,      /* valid request the library cannot do  */
  CCGLIB_ERROR_RUNTIME = 3           /* a HIP call failed                    */
};

/* ValueType: include/ccglib/common/value_type.h:14-22 */
enum {
  CCGLIB_INT1 = 0,
  CCGLIB_INT32 = 1,
  CCGLIB_BFLOAT16 = 2,
  CCGLIB_FLOAT8E4M3 = 3,
  CCGLIB_FLOAT8E5M2 = 4,
  CCGLIB_FLOAT16 = 5,
  CCGLIB_FLOAT32 = 6
};
/* ComplexAxisLocation: include/ccglib/common/complex_order.h:12 */
enum { CCGLIB_COMPLEX_PLANAR = 0, CCGLIB_COMPLEX_INTERLEAVED = 1 };
/* Direction: include/ccglib/common/direction.h:6 */
enum { CCGLIB_FORWARD = 0, CCGLIB_BACKWARD = 1 };
/* MemOrder: include/ccglib/gemm/mem_order.h:6 */
enum { CCGLIB_ROW_MAJOR = 0, CCGLIB_COL_MAJOR = 1 };
/* Variant: include/ccglib/gemm/variant.h:6 */
enum { CCGLIB_BASIC = 0, CCGLIB_OPT = 1 };

typedef struct ccglib_gemm *ccglib_gemm_t;
typedef struct ccglib_transpose *ccglib_transpose_t;
typedef struct ccglib_packing *ccglib_packing_t;
typedef struct ccglib_pipeline *ccglib_pipeline_t;

/* Text of the last error raised on this thread ("" if none). */
CCGLIB_API const char *ccglib_last_error(void);
/* Library version string. */
CCGLIB_API const char *ccglib_version(void);

/* ------------------------------------------------------------------------
 * Process-wide options. No counterpart in the reference (whose only such
 * channel is its JIT macros, src/mma/GEMM.cpp:140-214): they select code paths
 * that produce the same results, for tests and for tuning. An option is read
 * when an object is created (HOST_CHUNK_BYTES: at every host Run); setting
 * one is not synchronised with other threads.
 *   INT1_POPCOUNT    0 (default): the 1-bit GEMM runs on the matrix cores (fp4
 *                    MFMA on +-1 values, exact); 1: XOR + population count on
 *                    the vector ALUs, which is otherwise only the fallback.
 *   BASIC_RETILE     1 (default): a basic-variant GEMM whose planar rows are not
 *                    whole 16-byte chunks owns a tiled copy of A and B and
 *                    re-tiles into it at every Run where that is faster than
 *                    reading the rows in place; so does one whose rows are whole
 *                    chunks and whose operands turn out not to be 16-byte
 *                    aligned; 0: such rows are always read in place (no extra
 *                    memory).
 *   HOST_CHUNK_BYTES 0 (default): ccglib_pipeline_run_host moves jobs of 8 MiB
 *                    or more in chunks of whole batches of about 32 MiB; any
 *                    other value: chunks of about that many bytes, whatever
 *                    the size of the job.
 *   GEMM_BLOCK_TILE  0 (default): GEMMs on tiled or whole-chunk planar
 *                    operands use 256 x 128 block tiles, 128 x 128 ones when
 *                    the larger would leave compute units idle (small
 *                    problems), 64 x 64 ones when those would too, or
 *                    192 x 256 ones (16-bit tiled input, planar C without
 *                    beta, M and N multiples of 64, K of more than 32) when
 *                    those fill the compute units well enough;
 *                    1: always 256 x 128 (32-bit input, which has no such
 *                    block: 128 x 128); 2: always 128 x 128; 3: 192 x 256
 *                    wherever that kernel applies, else as 0; 4: always
 *                    64 x 64; 5, 6, 7: waves of 32 x 32, 32 x 16, 16 x 16 that
 *                    share nothing, which 0 takes where 64 x 64 blocks leave
 *                    units idle too (8- and 1-bit input: 32 x 32 only; where no
 *                    such kernel applies, 32-bit input among that, as 4). The 192 x 256 block also serves 16-bit
 *                    interleaved rows read in place (the pipeline) when K is a
 *                    multiple of 32.
 *   EXPECT_UNALIGNED 0 (default): a basic-variant GEMM that meets operands that
 *                    are not 16-byte aligned allocates its tiled copies at that
 *                    Run, and a pipeline that reads rows in place creates the
 *                    pipeline with transposes that takes over for such buffers
 *                    at that Run (never while the stream is being captured
 *                    into a graph: the GEMM then reads the rows through
 *                    registers, the pipeline reports an error); 1: both are
 *                    allocated when the object is created, and no device Run
 *                    allocates.
 *   PIPELINE_ROUTE   0 (default): an opt-variant pipeline whose input rows are
 *                    16 bytes or longer (of the basic variant: ragged and 32-bit
 *                    interleaved rows) lets the GEMM read them in place
 *                    where that is faster than transposing them into tiles
 *                    first (small M N / (M + N); the break-even points are
 *                    measured ones), and transposes otherwise; 1: in place
 *                    wherever the GEMM can; 2: always through the transposes.
 *                    ccglib_pipeline_reads_in_place tells which one an object
 *                    took.
 *   REAL_BLOCK       0 (default): the block shape of a real product (ScaledGEMM,
 *                    ScaledLinear, Orthogonalize, FusedLinear, GroupedLinear,
 *                    whose K is not cut) and the parts that its K is
 *                    cut into are chosen by its sizes; otherwise 1 plus the
 *                    shape's number (the last one where there are fewer), plus
 *                    256 times the number of parts (0: chosen).
 * ---------------------------------------------------------------------- */
enum {
  CCGLIB_AMD_OPTION_INT1_POPCOUNT = 0,
  CCGLIB_AMD_OPTION_BASIC_RETILE = 1,
  CCGLIB_AMD_OPTION_HOST_CHUNK_BYTES = 2,
  CCGLIB_AMD_OPTION_GEMM_BLOCK_TILE = 3,
  CCGLIB_AMD_OPTION_EXPECT_UNALIGNED = 4,
  CCGLIB_AMD_OPTION_PIPELINE_ROUTE = 5,
  CCGLIB_AMD_OPTION_REAL_BLOCK = 6,
  CCGLIB_AMD_OPTION_COUNT = 7
};
CCGLIB_API int ccglib_amd_set_option(int option, size_t value);
CCGLIB_API int ccglib_amd_get_option(int option, size_t *value);

/* ------------------------------------------------------------------------
 * Complex GEMM  C[b] = alpha * A[b] * B[b]^T + beta * C[b]
 * Replaces ccglib::mma::GEMM: constructor include/ccglib/gemm/mma.h:42-49
 * (src/mma/GEMM.cpp:243-254), Run :50 (src/mma/GEMM.cpp:263-268),
 * GetDimensions :39-40 (src/mma/GEMM.cpp:270-275).
 *
 * Layouts (kernels/type_selector.h:224-241, kernels/gemm_kernel_float.cu:28-33):
 *   basic: A [B][2][M][K], B [B][2][N][K] (K in 32-bit words for 1-bit input)
 *   opt:   A [B][Mp/Mb][Kp/Kc][2][Mb][Kc], B likewise with Nb: the output of
 *          the transpose below with the chunk sizes of get_dimensions
 *   C:     planar [B][2][M][N] (row major) / [B][2][N][M] (column major);
 *          interleaved [B][M][N][2] / [B][N][M][2] (opt variant only)
 * Supported (type_in -> type_out): float16->float32|float16,
 * bfloat16->float32|bfloat16, float32->float32|float16|bfloat16,
 * float8e4m3->float32, float8e5m2->float32, int1->int32 (the reference's
 * matrix, kernels/type_selector.h:65-212). Accumulation is float32 (int32 for
 * 1-bit input).
 * a_order must be row major and b_order column major (as in the reference,
 * where anything else fails to compile: kernels/gemm_kernel_float.cu:20-25);
 * the error text keeps the token HIPRTC_ERROR_COMPILATION that the
 * reference's callers match on (test/gemm/mma.cpp:598-627).
 * 1-bit input: K must be a multiple of 32; alpha and beta are truncated to
 * integers (src/reference/GEMM.cpp:202-205).
 * C is read only when beta != 0.
 * K whose interleaved row (2 * K * bits / 8 bytes) does not fit 32 bits is
 * refused. Operands should be 16-byte aligned: basic-variant operands whose rows
 * are whole 16-byte chunks and that are not aligned are re-tiled into a workspace
 * the object owns (allocated at the first such Run). Rows that are not whole
 * chunks are read in place from any address, or re-tiled likewise where that is
 * faster (workspace allocated at creation; see CCGLIB_AMD_OPTION_BASIC_RETILE).
 * Opt-variant operands that are not aligned are refused by Run.
 * ---------------------------------------------------------------------- */
CCGLIB_API int ccglib_gemm_create(ccglib_gemm_t *gemm, size_t B, size_t M,
                                  size_t N, size_t K, int device, void *stream,
                                  int type_in, int type_out, int variant,
                                  int c_complex_axis_location, int c_mem_order,
                                  int a_mem_order, int b_mem_order,
                                  float alpha_re, float alpha_im, float beta_re,
                                  float beta_im);
/* Argument order (a, b, c) as in GEMM::Run. */
CCGLIB_API int ccglib_gemm_run(ccglib_gemm_t gemm, const void *d_a,
                               const void *d_b, void *d_c);
/* Which kernel Run launches for 16-byte aligned buffers, in words (kernel
 * function, block tile, operand layout). No counterpart in the reference, whose
 * one kernel per precision is fixed by its parameter tables (src/mma/Kernel*.cpp);
 * here the choice depends on the problem size, and benchmark output names it. */
CCGLIB_API int ccglib_gemm_kernel_name(ccglib_gemm_t gemm, char *name, size_t size);
CCGLIB_API int ccglib_gemm_destroy(ccglib_gemm_t gemm);
/* (m_per_block, n_per_block, k_chunk): the chunk sizes of the opt layout. */
CCGLIB_API int ccglib_gemm_get_dimensions(int type_in, int type_out,
                                          int variant, unsigned *m_per_block,
                                          unsigned *n_per_block,
                                          unsigned *k_chunk);

/* ------------------------------------------------------------------------
 * Transpose into the tiled layout of the opt GEMM.
 * Replaces ccglib::transpose::Transpose: constructor
 * include/ccglib/transpose/transpose.h:26-29
 * (src/transpose/Transpose.cpp:131-141), Run(device) :31
 * (src/transpose/Transpose.cpp:160-164), Run(host) :30 (a no-op in the
 * reference, src/transpose/Transpose.cpp:147-154; here it does the work).
 *   in  [B][2][M][N] (planar) or [B][M][N][2] (interleaved)
 *   out [B][Mp/Mc][Np/Nc][2][Mc][Nc], zero where m >= M or n >= N
 * nr_bits is 1, 8, 16 or 32; for 1 bit N and N_chunk count samples and must
 * be multiples of 32 (whole 32-bit words move).
 * ---------------------------------------------------------------------- */
CCGLIB_API int ccglib_transpose_create(ccglib_transpose_t *transpose, size_t B,
                                       size_t M, size_t N, size_t M_chunk,
                                       size_t N_chunk, size_t nr_bits,
                                       int device, void *stream,
                                       int input_complex_axis_location);
CCGLIB_API int ccglib_transpose_run(ccglib_transpose_t transpose,
                                    const void *d_input, void *d_output);
CCGLIB_API int ccglib_transpose_run_host(ccglib_transpose_t transpose,
                                         const void *h_input, void *d_output);
/* Both operands of one GEMM: the same as ccglib_transpose_run on each, in one
 * kernel launch where the two have the same batch size, row length N, N_chunk,
 * width and input layout and one has at most a quarter of the other's rows
 * (otherwise in two: operands of similar size measured 1-3 % faster one after
 * the other). No counterpart in the reference,
 * whose pipeline launches one transpose per operand
 * (src/pipeline/Pipeline.cpp:116-121); a small operand no longer pays for a
 * launch, ramp-up and tail of its own. Both objects must have been created
 * for the same device and stream. */
CCGLIB_API int ccglib_transpose_run_pair(ccglib_transpose_t transpose_a,
                                         const void *d_input_a, void *d_output_a,
                                         ccglib_transpose_t transpose_b,
                                         const void *d_input_b, void *d_output_b);
CCGLIB_API int ccglib_transpose_destroy(ccglib_transpose_t transpose);

/* ------------------------------------------------------------------------
 * Bit packing: N one-byte samples <-> N bits, LSB first in 32-bit words.
 * Replaces ccglib::packing::Packing: constructor
 * include/ccglib/packing/packing.h:35-38 (src/packing/Packing.cpp:136-141),
 * Run(device) :40 (src/packing/Packing.cpp:162-166), Run(host) :39
 * (src/packing/Packing.cpp:152-156).
 * forward: byte != 0 -> bit 1; interleaved input (re,im pairs) is packed as all
 * real bits followed by all imaginary bits (kernels/packing_kernel.cu:15-22).
 * backward: bits -> bytes of 0/1, planar only (create fails otherwise, as
 * src/packing/Packing.cpp:49-53). The packed buffer holds ceil(N/32) words.
 * ---------------------------------------------------------------------- */
CCGLIB_API int ccglib_packing_create(ccglib_packing_t *packing, size_t N,
                                     int direction, int device, void *stream,
                                     int input_complex_axis_location);
CCGLIB_API int ccglib_packing_run(ccglib_packing_t packing,
                                  const void *d_input, void *d_output);
CCGLIB_API int ccglib_packing_run_host(ccglib_packing_t packing,
                                       const void *h_input, void *d_output);
CCGLIB_API int ccglib_packing_destroy(ccglib_packing_t packing);

/* ------------------------------------------------------------------------
 * Pipeline: [pack] -> [transpose] -> GEMM with scratch buffers owned by the
 * object. Replaces ccglib::pipeline::Pipeline: constructor
 * include/ccglib/pipeline/pipeline.h:44-53 (src/pipeline/Pipeline.cpp:145-160),
 * Run(device) :54 (src/pipeline/Pipeline.cpp:183-188), Run(host) :41
 * (src/pipeline/Pipeline.cpp:162-176).
 * 1-bit input is one byte per sample and is packed first (interleaved input:
 * every batch on its own, real bits then imaginary bits; the reference packs
 * the whole buffer as one, kernels/packing_kernel.cu:15-22, which is the same
 * for B = 1. With K a multiple of 32 the bytes go straight into the GEMM's
 * 1-bit tiles; otherwise, and with CCGLIB_AMD_OPTION_INT1_POPCOUNT, through a
 * packed buffer, which for interleaved input and B > 1 needs M*K and N*K to be
 * multiples of 32); the
 * opt variant transposes A and B first. 8- and 16-bit interleaved input whose
 * rows are whole 16-byte chunks is read by the GEMM in place instead (no
 * transposes), and so is planar input of the opt variant with such rows when
 * the problem is small enough for the transposes to cost more than they save;
 * if a Run then gets pointers that are not 16-byte aligned, the
 * object builds the pipeline with transposes at that Run and uses it for such
 * calls. Argument order follows the reference constructor.
 * run_host copies a, b (and c when beta != 0) to the device, runs, copies c
 * back and returns when c is complete; sizes are those of the layouts above.
 * Jobs of 8 MiB or more with several batches move in chunks of whole batches
 * over two internal streams (ordered after the work already queued on the
 * object's stream), so that with page-locked host buffers the copies in, the
 * kernels and the copies out overlap; the result is the same either way.
 * ---------------------------------------------------------------------- */
CCGLIB_API int ccglib_pipeline_create(
    ccglib_pipeline_t *pipeline, size_t B, size_t M, size_t N, size_t K,
    int device, void *stream, int input_complex_axis_location,
    int output_complex_axis_location, int a_mem_order, int b_mem_order,
    int c_mem_order, int input_type, int output_type, int variant,
    float alpha_re, float alpha_im, float beta_re, float beta_im);
CCGLIB_API int ccglib_pipeline_run(ccglib_pipeline_t pipeline, const void *d_a,
                                   const void *d_b, void *d_c);
CCGLIB_API int ccglib_pipeline_run_host(ccglib_pipeline_t pipeline,
                                        const void *h_a, const void *h_b,
                                        void *h_c);
/* Whether the object's GEMM reads the caller's rows in place (1) or the tiles
 * that its transposes write (0); see the option PIPELINE_ROUTE. No counterpart
 * in the reference, which always transposes for the opt variant
 * (src/pipeline/Pipeline.cpp:53, :78-93). */
CCGLIB_API int ccglib_pipeline_reads_in_place(ccglib_pipeline_t pipeline, int *in_place);
CCGLIB_API int ccglib_pipeline_destroy(ccglib_pipeline_t pipeline);

/* ------------------------------------------------------------------------
 * The pipeline as one stateless call that allocates nothing.
 * No counterpart in the reference. It is for callers that cannot allocate
 * device memory: code under HIP graph capture, tight serving loops, harnesses
 * that forbid hipMalloc. ccglib_pipeline_create allocates the scratch of its
 * object (the packed and transposed copies of A and B); this call does the
 * work of create + run + destroy with that scratch in a static device array
 * of CCGLIB_AMD_STATIC_SCRATCH_BYTES, which every GPU the library's code is
 * loaded on holds until the process ends. It calls no hipMalloc / hipFree (nor
 * their stream-ordered forms) and creates no host objects. (The HIP runtime
 * loads a code object on a GPU when something in it is first used there: the
 * array comes to exist, and its bytes leave the device's free memory, at the
 * first call on that GPU, which therefore belongs before a graph capture. No
 * later call moves the device's free memory.)
 *   - Arguments as ccglib_pipeline_create followed by those of
 *     ccglib_pipeline_run; only enqueues on `stream`.
 *   - Route: [1-bit interleaved input: pack each batch] -> transpose A and B
 *     into the tiled layout (1-bit planar input: bytes packed straight into
 *     1-bit tiles) -> GEMM on the tiles, whatever the variant. The process-wide
 *     options do not apply.
 *   - The tiled copies (rows padded to 128, K to the chunk of get_dimensions)
 *     plus the packed copies must fit the array; otherwise
 *     CCGLIB_ERROR_UNSUPPORTED and nothing is enqueued. K must be positive
 *     (1-bit input: a multiple of 32).
 *   - All calls on one GPU share the array: calls whose kernels may overlap
 *     (different streams, no dependency) race. Calls on one stream are safe.
 *   - What fits the default of 32 MiB, with M', N' the rows padded to 128 and
 *     K' padded to the chunk: B (M' + N') K' <= 8 Mi (2^23) elements for 16-bit
 *     input, 16 Mi for fp8, 4 Mi for float32, 128 Mi samples for 1-bit planar
 *     input and about 64 Mi for 1-bit interleaved input (whose packed copies live
 *     in the array too). E.g. 16-bit: B = 16 of 256 x 256 x 1024, or one
 *     1024 x 1024 x 4096.
 *   - The size is a build option: compile the library with
 *     -DCCGLIB_AMD_STATIC_SCRATCH_BYTES=<bytes> (a multiple of 256;
 *     ccglib_amd/build.py reads the environment variable of the same name).
 *     ccglib_amd_static_scratch_bytes() returns what the loaded library was
 *     built with, which is the figure that binds - not this header's default.
 * ---------------------------------------------------------------------- */
#ifndef CCGLIB_AMD_STATIC_SCRATCH_BYTES
#define CCGLIB_AMD_STATIC_SCRATCH_BYTES ((size_t)32 << 20)
#endif
CCGLIB_API size_t ccglib_amd_static_scratch_bytes(void);
CCGLIB_API int ccglib_pipeline_run_static(
    size_t B, size_t M, size_t N, size_t K, int device, void *stream,
    int input_complex_axis_location, int output_complex_axis_location,
    int a_mem_order, int b_mem_order, int c_mem_order, int input_type,
    int output_type, int variant, float alpha_re, float alpha_im, float beta_re,
    float beta_im, const void *d_a, const void *d_b, void *d_c);

/* ------------------------------------------------------------------------
 * Real products of 8-bit values with block scales, what makes their operands,
 * a linear layer of them, and orthogonalised updates of weights. No
 * counterpart in the reference.
 *
 * Layout of an 8-bit matrix of R rows of C values (e4m3 or e5m2): the rows
 * lie ccglib_scaled_pitch(C) bytes apart (a multiple of 16), the bytes behind
 * a row's end are zero. Its scales are numbered first by the group of 128
 * values along the row, then by the row (SCALE_ROWS) or by 128 rows
 * (SCALE_BLOCKS):
 *     scales[ceil(C / 128)][ccglib_scaled_pitch(R or ceil(R / 128))]
 * float, or one byte that holds a power of two (e8m0: 2^(byte - 127), NaN for
 * the byte 255). A batch is such matrices one after the other. Values start
 * at a multiple of 16 bytes.
 * ---------------------------------------------------------------------- */
/* Groups of values that share a scale: 128 of a row, or 128 x 128 */
enum { CCGLIB_SCALE_ROWS = 0, CCGLIB_SCALE_BLOCKS = 1 };
/* What a scale is */
enum { CCGLIB_SCALE_FLOAT32 = 0, CCGLIB_SCALE_E8M0 = 1 };

typedef struct ccglib_quantize *ccglib_quantize_t;
typedef struct ccglib_scaled_gemm *ccglib_scaled_gemm_t;
typedef struct ccglib_scaled_linear *ccglib_scaled_linear_t;
typedef struct ccglib_orthogonalize *ccglib_orthogonalize_t;

/* n rounded up to the distance of rows, of values and of scales. */
CCGLIB_API size_t ccglib_scaled_pitch(size_t n);

/* B matrices of M x N (float32, float16, bfloat16; rows in_pitch values apart,
 * 0: N) to 8 bits. For each group, t the type's largest value (448, 57344):
 *     amax = max(2^-100, largest finite |x|)
 *     float32 scales: scale = amax / t, q = round(x * (t / amax))
 *     e8m0 scales:    scale = 2^ceil(log2(amax / t)), q = round(x / scale)
 * in 32 bits, q rounded to nearest, ties to even. NaN stays NaN; an infinity
 * stays one in e5m2 and is NaN in e4m3. run writes the matrix as it is
 * (d_out, d_scales), its transpose (d_out_t, d_scales_t: N rows of M values,
 * groups along M), or both; a pair that is not wanted is null. */
CCGLIB_API int ccglib_quantize_create(ccglib_quantize_t *quantize, size_t B, size_t M, size_t N, int device, void *stream,
                                      int type_in, int type_out, int group, int scale_type, size_t in_pitch);
CCGLIB_API int ccglib_quantize_run(ccglib_quantize_t quantize, const void *d_in, void *d_out, void *d_scales, void *d_out_t,
                                   void *d_scales_t);
CCGLIB_API int ccglib_quantize_destroy(ccglib_quantize_t quantize);

/* C[m][n] (+)= sum over groups g of 128 of K of
 *     scale_a[g][m] scale_b[g][n] sum over k in g of A[m][k] B[n][k]
 * for B matrices each of M x K and N x K, C M x N row-major (float32, float16,
 * bfloat16). Sums of groups are held in 32 bits and rounded once; inside a
 * group those of a float32 C are too, those of a 16-bit C are the 8-bit matrix
 * instruction's, which drops what lies 2^-13 below the largest of eight
 * neighbouring products (1e-5 to 9e-5 of the sum). Where B has a scale for
 * 128 x 128, scale_a scale_b is formed first, a float that may neither
 * overflow nor become denormal. accumulate: C, which is float32 then, is added
 * to. pitch_a, pitch_b: bytes between rows where they are not
 * ccglib_scaled_pitch(K) (0; multiples of 16); pitch_c: elements between rows of
 * C (0: N). K may be 0 (a sum of nothing). Scales of less than 4 GiB a group of K. */
CCGLIB_API int ccglib_scaled_gemm_create(ccglib_scaled_gemm_t *gemm, size_t B, size_t M, size_t N, size_t K, int device,
                                         void *stream, int type_a, int type_b, int type_c, int group_a, int group_b,
                                         int scale_type, int accumulate, size_t pitch_a, size_t pitch_b, size_t pitch_c);
CCGLIB_API int ccglib_scaled_gemm_run(ccglib_scaled_gemm_t gemm, const void *d_a, const void *d_scales_a, const void *d_b,
                                      const void *d_scales_b, void *d_c);
CCGLIB_API int ccglib_scaled_gemm_kernel_name(ccglib_scaled_gemm_t gemm, char *buffer, size_t size);
CCGLIB_API int ccglib_scaled_gemm_destroy(ccglib_scaled_gemm_t gemm);

/* A linear layer of K inputs and N outputs on M rows, y = x W^T, by products of
 * 8-bit copies: x (M x K) and dy (M x N) with scales for 128 values along the
 * summed index, W (N x K) for 128 x 128; x and W in e4m3, dy in gradient_type.
 * x, y, W, dy and dx are of `type`, dw is float32. set_weights keeps 8-bit
 * copies of W until it is called again, forward those of x until the next one;
 * backward, with the x and W of the last forward, computes
 *     dx = dy W,  dw = dy^T x  (accumulate_dw: dw += dy^T x);
 * d_dx or d_dw may be null. Once set_weights has been called again that W is
 * gone, and backward refuses to compute dx until the next forward.
 * training = 0: forward only, half the work of making the copies. */
CCGLIB_API int ccglib_scaled_linear_create(ccglib_scaled_linear_t *linear, size_t M, size_t N, size_t K, int device, void *stream,
                                           int type, int gradient_type, int scale_type, int training);
CCGLIB_API int ccglib_scaled_linear_set_weights(ccglib_scaled_linear_t linear, const void *d_w);
CCGLIB_API int ccglib_scaled_linear_forward(ccglib_scaled_linear_t linear, const void *d_x, void *d_y);
CCGLIB_API int ccglib_scaled_linear_backward(ccglib_scaled_linear_t linear, const void *d_dy, void *d_dx, void *d_dw,
                                             int accumulate_dw);
CCGLIB_API int ccglib_scaled_linear_destroy(ccglib_scaled_linear_t linear);

/* B updates G of M x N (float32, float16, bfloat16; rows in_pitch and out_pitch
 * values apart, 0: N), each made nearly orthogonal by a Newton-Schulz iteration:
 *     X = G / (|G| + epsilon), |.| the Frobenius norm
 *     steps times:  S = X X^T,  X = a X + (b S + c S S) X      (M <= N; else of G^T)
 * d_out may be d_in. bfloat16 updates are multiplied in fp16 (11 bits), others
 * in two fp16 for each value (22 bits); sums are 32 bits. A matrix that holds
 * NaN or an infinity becomes NaN. */
CCGLIB_API int ccglib_orthogonalize_create(ccglib_orthogonalize_t *orthogonalize, size_t B, size_t M, size_t N, int device,
                                           void *stream, int type, int steps, float a, float b, float c, float epsilon,
                                           size_t in_pitch, size_t out_pitch);
CCGLIB_API int ccglib_orthogonalize_run(ccglib_orthogonalize_t orthogonalize, const void *d_in, void *d_out);
CCGLIB_API int ccglib_orthogonalize_destroy(ccglib_orthogonalize_t orthogonalize);

/* ------------------------------------------------------------------------
 * Linear layers of 16-bit values with what stands around the product, the same
 * grouped by expert, and what brings rows to experts and back. No counterpart
 * in the reference. Values are float16 or bfloat16, sums 32 bits, rounded once.
 * Buffers start at a multiple of their element; rows whose distance and start
 * are multiples of 16 bytes are the fast ones. Outputs lie apart from all inputs,
 * but y may be the residual.
 * FusedLinear, GroupedLinear and Route hold scratch memory, so that the calls of
 * one object, and graphs captured of them, run one after the other.
 * ---------------------------------------------------------------------- */
/* act(z): z; max(z, 0); z/2 (1 + tanh(sqrt(2/pi) (z + 0.044715 z^3))); z / (1 + e^-z) */
enum { CCGLIB_ACTIVATION_NONE = 0, CCGLIB_ACTIVATION_RELU = 1, CCGLIB_ACTIVATION_GELU = 2, CCGLIB_ACTIVATION_SILU = 3 };

typedef struct ccglib_fused_linear *ccglib_fused_linear_t;
typedef struct ccglib_grouped_linear *ccglib_grouped_linear_t;
typedef struct ccglib_route *ccglib_route_t;
typedef struct ccglib_combine *ccglib_combine_t;

/* A linear layer of K inputs and N outputs on M rows, x [M][K], W [N][K]:
 *     forward:   z = x W^T + bias,  y = act(z) + residual
 *     backward:  dz = dy act'(z),  dx = dz W,
 *                dW (+)= dz^T x,  dbias (+)= sum over rows of dz
 * (the residual's gradient is dy). bias, residual and z may be null: z is
 * stored where the backward pass is to have it; without an activation that
 * needs none. act is taken of the sum before z is rounded, act' of the z that
 * was stored (relu' is 0 where z is NaN, whose act is NaN). Behind an activation dz is
 * rounded to 16 bits, as the matrix instructions want it: up to 2^-8 of its value
 * (bfloat16; float16 2^-11) in dx and dW, also where dW is float32; dbias is summed
 * without that. dx, dw, dbias: null if not wanted. dw and dbias are of
 * gradient_type, the values' type or float32; float32 ones may be added to
 * (accumulate). training = 0: forward only. x_pitch, w_pitch, y_pitch:
 * elements between rows of x and dx, of W and dW, of y, z, residual and dy (0: K, K, N).
 * kernel_name, product 0 to 2: that of y, of dx, of dW (small ones are one launch,
 * where both are wanted).
 * Up to 2^31 - 1 rows, N, K and distances up to 2^22; for training 65535 blocks of
 * 64 rows (4.1 million rows; an expert's last block may hold one). A layer for training holds
 * dz, 2 M N bytes, if it has an activation, and the sums of dbias, 4 N bytes a block of 64 rows (of 16
 * where there are few). They live for one backward call: forward and backward share nothing but
 * what the caller hands them. */
CCGLIB_API int ccglib_fused_linear_create(ccglib_fused_linear_t *linear, size_t M, size_t N, size_t K, int device, void *stream,
                                          int type, int activation, int gradient_type, int training, size_t x_pitch,
                                          size_t w_pitch, size_t y_pitch);
CCGLIB_API int ccglib_fused_linear_forward(ccglib_fused_linear_t linear, const void *d_x, const void *d_w, const void *d_bias,
                                           const void *d_residual, void *d_y, void *d_z);
CCGLIB_API int ccglib_fused_linear_backward(ccglib_fused_linear_t linear, const void *d_dy, const void *d_z, const void *d_x,
                                            const void *d_w, void *d_dx, void *d_dw, void *d_dbias, int accumulate);
CCGLIB_API int ccglib_fused_linear_kernel_name(ccglib_fused_linear_t linear, int product, char *buffer, size_t size);
CCGLIB_API int ccglib_fused_linear_destroy(ccglib_fused_linear_t linear);

/* The same with E weight matrices, W [E][N][K] and bias [E][N], for M rows that
 * are sorted by expert: rows offsets[e] to offsets[e + 1] - 1 are multiplied
 * with W[e]. offsets is device memory, E + 1 int32 that do not fall (what lies outside 0 to M counts
 * as the nearer end); an expert may have no rows, whose dW and dbias are zero then.
 * Rows in front of offsets[0] and from offsets[E] on are neither read nor written. (Offsets that fall leave
 * results unspecified, of these M rows and E experts only.) 1 to 1024 experts. */
CCGLIB_API int ccglib_grouped_linear_create(ccglib_grouped_linear_t *linear, size_t E, size_t M, size_t N, size_t K, int device,
                                            void *stream, int type, int activation, int gradient_type, int training,
                                            size_t x_pitch, size_t w_pitch, size_t y_pitch);
CCGLIB_API int ccglib_grouped_linear_forward(ccglib_grouped_linear_t linear, const void *d_x, const void *d_offsets,
                                             const void *d_w, const void *d_bias, const void *d_residual, void *d_y, void *d_z);
CCGLIB_API int ccglib_grouped_linear_backward(ccglib_grouped_linear_t linear, const void *d_dy, const void *d_z, const void *d_x,
                                              const void *d_offsets, const void *d_w, void *d_dx, void *d_dw, void *d_dbias,
                                              int accumulate);
CCGLIB_API int ccglib_grouped_linear_kernel_name(ccglib_grouped_linear_t linear, int product, char *buffer, size_t size);
CCGLIB_API int ccglib_grouped_linear_destroy(ccglib_grouped_linear_t linear);

/* Which k of E experts each of T tokens goes to. logits [T][E] (float32, float16,
 * bfloat16). run writes, for each token, largest first and of equal ones the
 * lower number first:
 *     experts [T][k]  int32
 *     weights [T][k]  float32: softmax of the k logits (normalize), or of all E
 *     offsets [E + 1] int32, slots [T][k] int32: where the token's rows lie when
 *                     all T k rows are sorted by expert, those of an expert in the order of tokens
 * NaN counts as the largest; a token whose logits are all -inf has weights of 0.
 * backward: dlogits [T][E] from dweights [T][k], with what run wrote; logits may
 * be null with normalize. 1 <= k <= 16, k <= E <= 1024, T < 2^24. */
CCGLIB_API int ccglib_route_create(ccglib_route_t *route, size_t T, size_t E, size_t k, int device, void *stream, int type,
                                   int normalize);
CCGLIB_API int ccglib_route_run(ccglib_route_t route, const void *d_logits, void *d_experts, void *d_weights, void *d_offsets,
                                void *d_slots);
CCGLIB_API int ccglib_route_backward(ccglib_route_t route, const void *d_logits, const void *d_experts, const void *d_weights,
                                     const void *d_dweights, void *d_dlogits);
CCGLIB_API int ccglib_route_destroy(ccglib_route_t route);

/* Rows of N values between T tokens and `rows` places (0: T k), slots [T][k] int32,
 * weights [T][k] float32 or null (1):
 *     run:       out[t] = sum over j of weights[t][j] y[slots[t][j]]
 *     spread:    y[slots[t][j]] = weights[t][j] x[t]
 *     backward:  dy[slots[t][j]] = weights[t][j] dout[t],  dweights[t][j] = <dout[t], y[slots[t][j]]>
 * (of run; dy or dweights may be null, y too without dweights. The gradient of spread's x is run of dy.)
 * A slot outside 0 to rows - 1 is passed over: it adds nothing, nothing is written for it, and
 * its dweights is 0. Slots that are written differ from each other; places that no slot names are left
 * as they are. y_pitch, out_pitch: elements between rows of y and dy, of x, out and dout (0: N). k <= 16, T < 2^24. */
CCGLIB_API int ccglib_combine_create(ccglib_combine_t *combine, size_t T, size_t k, size_t N, int device, void *stream, int type,
                                     size_t rows, size_t y_pitch, size_t out_pitch);
CCGLIB_API int ccglib_combine_run(ccglib_combine_t combine, const void *d_y, const void *d_slots, const void *d_weights, void *d_out);
CCGLIB_API int ccglib_combine_spread(ccglib_combine_t combine, const void *d_x, const void *d_slots, const void *d_weights, void *d_y);
CCGLIB_API int ccglib_combine_backward(ccglib_combine_t combine, const void *d_dout, const void *d_y, const void *d_slots,
                                       const void *d_weights, void *d_dy, void *d_dweights);
CCGLIB_API int ccglib_combine_destroy(ccglib_combine_t combine);

#ifdef __cplusplus
}
#endif
#endif /* CCGLIB_AMD_H_ */
