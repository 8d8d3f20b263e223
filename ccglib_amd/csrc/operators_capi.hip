// C ABI of the operators on 8-bit values with block scales and of the orthogonalised updates (declared in
// include/ccglib_amd.h): argument checking, object state and workspaces around the kernel launchers. None of them has a
// counterpart in the reference.
#include <cstdio>
#include <cstring>
#include <new>

#include "host_util.h"
#include "scaled_linear.h"

using namespace ccglib_amd;

namespace {

constexpr size_t kMostRows = 0x7fffffffu;     // rows, and values of a row, of any matrix here
constexpr size_t kMostPitch = (size_t)1 << 23;  // bytes: 256 rows are addressed with 32-bit offsets
constexpr size_t kMostBlocks = 0x7fffffffu;

bool is_group(int g) { return g == kScaleRows || g == kScaleBlocks; }
bool is_scale(int s) { return s == kScaleFloat32 || s == kScaleE8m0; }
int check_quantize(const QuantizeParams &p, size_t B, size_t M, size_t N) {
  if (!is_wide_float(p.type_in)) {
    return fail(CCGLIB_ERROR_UNSUPPORTED, "Quantize: input is float32, float16 or bfloat16 (type %d)", p.type_in);
  }
  if (!is_float8(p.type_out)) {
    return fail(CCGLIB_ERROR_UNSUPPORTED, "Quantize: output is float8e4m3 or float8e5m2 (type %d)", p.type_out);
  }
  if (!is_group(p.group) || !is_scale(p.scale_type)) {
    return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "enum argument out of range");
  }
  if (B > kMostRows || M > kMostRows || N > kMostRows) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "problem size out of range");
  if (p.in_pitch < N) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "Quantize: rows of %zu values at a distance of %zu", N, p.in_pitch);
  // (groups, and rows of all matrices, are counted in 32 bits)
  if (B && M && N && (ceil_div(M, 16) > kMostBlocks / B / ceil_div(N, kScaleGroup) || M > 0xffffffffu / B / ceil_div(N, kScaleGroup))) {
    return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "problem size out of range");
  }
  return CCGLIB_OK;
}

int check_gemm(const ScaledGemmParams &p, size_t B, size_t M, size_t N, size_t K) {
  if (!is_float8(p.type_a) || !is_float8(p.type_b)) {
    return fail(CCGLIB_ERROR_UNSUPPORTED, "ScaledGEMM: operands are float8e4m3 or float8e5m2 (types %d, %d)", p.type_a, p.type_b);
  }
  if (!is_wide_float(p.type_c)) {
    return fail(CCGLIB_ERROR_UNSUPPORTED, "ScaledGEMM: C is float32, float16 or bfloat16 (type %d)", p.type_c);
  }
  if (p.accumulate && p.type_c != kFloat32) {
    return fail(CCGLIB_ERROR_UNSUPPORTED, "ScaledGEMM: C that is added to is float32 (type %d)", p.type_c);
  }
  if (!is_group(p.group_a) || !is_group(p.group_b) || !is_scale(p.scale_type)) {
    return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "enum argument out of range");
  }
  if (B > kMostRows || M > kMostRows || N > kMostRows || K > kMostPitch) {
    return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "problem size out of range");
  }
  const size_t least = scaled_pitch(K);
  if (p.pitch_a < least || p.pitch_b < least || p.pitch_a % kScaledPad || p.pitch_b % kScaledPad || p.pitch_a > kMostPitch ||
      p.pitch_b > kMostPitch) {
    return fail(CCGLIB_ERROR_INVALID_ARGUMENT,
                "ScaledGEMM: rows of A and B lie a multiple of %zu bytes apart, %zu to %zu for this K (got %zu, %zu)", kScaledPad,
                least, kMostPitch, p.pitch_a, p.pitch_b);
  }
  if (p.pitch_c < N) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "ScaledGEMM: rows of C of %zu values at a distance of %zu", N, p.pitch_c);
  // (a row's scale is found by a 32-bit offset in the scales of its group of K)
  if (scaled_pitch(scale_rows(M, p.group_a)) * scale_size(p.scale_type) > 0xffffffffu ||
      scaled_pitch(scale_rows(N, p.group_b)) * scale_size(p.scale_type) > 0xffffffffu) {
    return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "problem size out of range: scales of a group of K take 4 GiB or more");
  }
  // (blocks of C times pieces of K, each at least 16 x 64 values, are counted in 32 bits)
  if (B && M && N && ceil_div(M, 16) > kMostBlocks / 64 / B / ceil_div(N, 64)) {
    return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "problem size out of range");
  }
  return CCGLIB_OK;
}

int check_launch(const ScaledGemmParams &p) {
  if (scaled_gemm_launches(p)) return CCGLIB_OK;
  return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "problem size out of range: more blocks of C than a launch takes");
}

int check_operand(const char *what, const void *values, const void *scales, int scale_type) {
  if (!values || !scales) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null pointer: %s", what);
  if (!aligned(values, 16)) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "%s: 8-bit values start at a multiple of 16 bytes", what);
  if (!aligned(scales, scale_size(scale_type))) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "%s: misaligned scales", what);
  return CCGLIB_OK;
}

size_t element(int type) { return (size_t)bits_of(type) / 8; }

}  // namespace

struct ccglib_quantize {
  QuantizeParams p;
  int device;
  hipStream_t stream;
};

struct ccglib_scaled_gemm {
  ScaledGemmParams p;
  int device;
  hipStream_t stream;
  Buffer workspace;
};

struct ccglib_scaled_linear {
  ScaledLinearParams p;
  int device;
  hipStream_t stream;
  bool have_weights = false;
  bool have_x = false, have_w = false;   // the copies of x and of W are those of the last forward
  Buffer memory;
};

struct ccglib_orthogonalize {
  OrthogonalizeParams p;
  int device;
  hipStream_t stream;
  Buffer workspace;
};

extern "C" {

size_t ccglib_scaled_pitch(size_t n) { return scaled_pitch(n); }

// ---- Quantize ----

int ccglib_quantize_create(ccglib_quantize_t *quantize, size_t B, size_t M, size_t N, int device, void *stream, int type_in,
                           int type_out, int group, int scale_type, size_t in_pitch) {
  if (!quantize) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null pointer: quantize");
  *quantize = nullptr;
  QuantizeParams p = {};
  p.batch = (unsigned)B;
  p.m = (unsigned)M;
  p.n = (unsigned)N;
  p.in_pitch = in_pitch ? in_pitch : N;
  p.type_in = type_in;
  p.type_out = type_out;
  p.group = group;
  p.scale_type = scale_type;
  if (int s = check_quantize(p, B, M, N)) return s;
  if (int s = check_device(device)) return s;
  auto *q = new (std::nothrow) ccglib_quantize{p, device, static_cast<hipStream_t>(stream)};
  if (!q) return fail(CCGLIB_ERROR_RUNTIME, "out of memory");
  *quantize = q;
  return CCGLIB_OK;
}

int ccglib_quantize_run(ccglib_quantize_t q, const void *d_in, void *d_out, void *d_scales, void *d_out_t, void *d_scales_t) {
  if (!q) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null handle");
  QuantizeParams p = q->p;
  if (p.batch == 0 || p.m == 0 || p.n == 0) return CCGLIB_OK;
  if (!d_in) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null pointer: input");
  if (!d_out && !d_out_t) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null pointer: output");
  if (!aligned(d_in, element(p.type_in))) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "Quantize: misaligned input");
  if (d_out || d_scales) {
    if (int s = check_operand("Quantize, output", d_out, d_scales, p.scale_type)) return s;
  }
  if (d_out_t || d_scales_t) {
    if (int s = check_operand("Quantize, transposed output", d_out_t, d_scales_t, p.scale_type)) return s;
  }
  p.in = d_in;
  p.out = d_out;
  p.scales = d_scales;
  p.out_t = d_out_t;
  p.scales_t = d_scales_t;
  DeviceGuard guard(q->device);
  HIP_TRY(guard.status());
  HIP_TRY(launch_quantize(p, q->stream));
  return CCGLIB_OK;
}

int ccglib_quantize_destroy(ccglib_quantize_t q) {
  delete q;
  return CCGLIB_OK;
}

// ---- ScaledGEMM ----

int ccglib_scaled_gemm_create(ccglib_scaled_gemm_t *gemm, size_t B, size_t M, size_t N, size_t K, int device, void *stream,
                              int type_a, int type_b, int type_c, int group_a, int group_b, int scale_type, int accumulate,
                              size_t pitch_a, size_t pitch_b, size_t pitch_c) {
  if (!gemm) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null pointer: gemm");
  *gemm = nullptr;
  ScaledGemmParams p = {};
  p.batch = (unsigned)B;
  p.m = (unsigned)M;
  p.n = (unsigned)N;
  p.k = (unsigned)K;
  p.pitch_a = pitch_a ? pitch_a : scaled_pitch(K);
  p.pitch_b = pitch_b ? pitch_b : scaled_pitch(K);
  p.pitch_c = pitch_c ? pitch_c : N;
  p.type_a = type_a;
  p.type_b = type_b;
  p.type_c = type_c;
  p.group_a = group_a;
  p.group_b = group_b;
  p.scale_type = scale_type;
  p.accumulate = accumulate != 0;
  if (int s = check_gemm(p, B, M, N, K)) return s;
  p.plan = plan_scaled_gemm(p);
  if (int s = check_launch(p)) return s;
  if (int s = check_device(device)) return s;
  DeviceGuard guard(device);
  HIP_TRY(guard.status());
  auto *g = new (std::nothrow) ccglib_scaled_gemm{p, device, static_cast<hipStream_t>(stream), {}};
  if (!g) return fail(CCGLIB_ERROR_RUNTIME, "out of memory");
  // counters (cleared), then partial sums
  const size_t counters = ceil_div(p.plan.counter_bytes, 256) * 256;
  if (int s = allocate(&g->workspace, counters + p.plan.partial_bytes, p.plan.counter_bytes)) {
    delete g;
    return s;
  }
  g->p.arrived = reinterpret_cast<unsigned *>(g->workspace.at(0));
  g->p.partial = reinterpret_cast<float *>(g->workspace.at(counters));
  *gemm = g;
  return CCGLIB_OK;
}

int ccglib_scaled_gemm_run(ccglib_scaled_gemm_t g, const void *d_a, const void *d_scales_a, const void *d_b,
                           const void *d_scales_b, void *d_c) {
  if (!g) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null handle");
  ScaledGemmParams p = g->p;
  if (p.batch == 0 || p.m == 0 || p.n == 0) return CCGLIB_OK;
  if (p.k > 0) {
    if (int s = check_operand("ScaledGEMM, A", d_a, d_scales_a, p.scale_type)) return s;
    if (int s = check_operand("ScaledGEMM, B", d_b, d_scales_b, p.scale_type)) return s;
  }
  if (!d_c) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null pointer: ScaledGEMM, C");
  if (!aligned(d_c, element(p.type_c))) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "ScaledGEMM: misaligned C");
  p.a = d_a;
  p.b = d_b;
  p.scales_a = d_scales_a;
  p.scales_b = d_scales_b;
  p.c = d_c;
  DeviceGuard guard(g->device);
  HIP_TRY(guard.status());
  HIP_TRY(launch_scaled_gemm(p, g->stream));
  return CCGLIB_OK;
}

int ccglib_scaled_gemm_kernel_name(ccglib_scaled_gemm_t g, char *buffer, size_t size) {
  if (!g || !buffer || size == 0) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null handle or buffer");
  snprintf(buffer, size, "%s", describe_scaled_gemm(g->p));
  return CCGLIB_OK;
}

int ccglib_scaled_gemm_destroy(ccglib_scaled_gemm_t g) {
  if (!g) return CCGLIB_OK;
  DeviceGuard guard(g->device);
  delete g;
  return CCGLIB_OK;
}

// ---- ScaledLinear ----

int ccglib_scaled_linear_create(ccglib_scaled_linear_t *linear, size_t M, size_t N, size_t K, int device, void *stream, int type,
                                int gradient_type, int scale_type, int training) {
  if (!linear) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null pointer: linear");
  *linear = nullptr;
  if (M > kMostPitch || N > kMostPitch || K > kMostPitch) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "problem size out of range");
  ScaledLinearParams p = scaled_linear_params(M, N, K, type, gradient_type, scale_type, training != 0);
  if (int s = check_quantize(p.x, 1, M, K)) return s;
  if (int s = check_quantize(p.w, 1, N, K)) return s;
  if (int s = check_quantize(p.dy, 1, M, N)) return s;
  if (int s = check_gemm(p.y, 1, M, N, K)) return s;
  if (int s = check_gemm(p.dx, 1, M, K, N)) return s;
  if (int s = check_gemm(p.dw, 1, N, K, M)) return s;
  plan_scaled_linear(&p);
  for (const ScaledGemmParams *product : {&p.y, &p.dx, &p.dw}) {
    if (int s = check_launch(*product)) return s;
  }
  if (int s = check_device(device)) return s;
  DeviceGuard guard(device);
  HIP_TRY(guard.status());
  auto *l = new (std::nothrow) ccglib_scaled_linear{p, device, static_cast<hipStream_t>(stream)};
  if (!l) return fail(CCGLIB_ERROR_RUNTIME, "out of memory");
  place_scaled_linear(&l->p, nullptr);
  if (int s = allocate(&l->memory, l->p.bytes, l->p.counter_bytes)) {
    delete l;
    return s;
  }
  place_scaled_linear(&l->p, l->memory.at(0));
  *linear = l;
  return CCGLIB_OK;
}

int ccglib_scaled_linear_set_weights(ccglib_scaled_linear_t l, const void *d_w) {
  if (!l) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null handle");
  if (!d_w && l->p.w.m && l->p.w.n) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null pointer: weights");
  if (!aligned(d_w, element(l->p.x.type_in))) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "ScaledLinear: misaligned weights");
  DeviceGuard guard(l->device);
  HIP_TRY(guard.status());
  QuantizeParams p = l->p.w;
  p.in = d_w;
  l->have_weights = l->have_w = false;
  HIP_TRY(launch_quantize(p, l->stream));
  l->have_weights = true;
  return CCGLIB_OK;
}

int ccglib_scaled_linear_forward(ccglib_scaled_linear_t l, const void *d_x, void *d_y) {
  if (!l) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null handle");
  if (!l->have_weights) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "ScaledLinear: forward before the weights were set");
  if ((!d_x && l->p.x.m && l->p.x.n) || (!d_y && l->p.y.m && l->p.y.n)) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null pointer: x or y");
  if (!aligned(d_x, element(l->p.x.type_in)) || !aligned(d_y, element(l->p.x.type_in))) {
    return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "ScaledLinear: misaligned x or y");
  }
  DeviceGuard guard(l->device);
  HIP_TRY(guard.status());
  QuantizeParams q = l->p.x;
  q.in = d_x;
  l->have_x = l->have_w = false;
  HIP_TRY(launch_quantize(q, l->stream));
  ScaledGemmParams p = l->p.y;
  p.c = d_y;
  HIP_TRY(launch_scaled_gemm(p, l->stream));
  l->have_x = l->have_w = true;
  return CCGLIB_OK;
}

int ccglib_scaled_linear_backward(ccglib_scaled_linear_t l, const void *d_dy, void *d_dx, void *d_dw, int accumulate_dw) {
  if (!l) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null handle");
  if (!l->p.training) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "ScaledLinear: backward of a layer that was created without training");
  if (!l->have_x) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "ScaledLinear: backward before forward");
  if (d_dx && !l->have_w) {
    return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "ScaledLinear: dx with the W of the last forward, but the weights were set since then");
  }
  if (!d_dx && !d_dw) return CCGLIB_OK;
  if (!d_dy && l->p.y.m && l->p.y.n) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null pointer: dy");
  if (!aligned(d_dy, element(l->p.x.type_in)) || !aligned(d_dx, element(l->p.x.type_in)) || !aligned(d_dw, 4)) {
    return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "ScaledLinear: misaligned dy, dx or dw");
  }
  DeviceGuard guard(l->device);
  HIP_TRY(guard.status());
  QuantizeParams q = l->p.dy;
  q.in = d_dy;
  if (!d_dx) q.out = q.scales = nullptr;
  if (!d_dw) q.out_t = q.scales_t = nullptr;
  HIP_TRY(launch_quantize(q, l->stream));
  if (d_dx) {
    ScaledGemmParams p = l->p.dx;
    p.c = d_dx;
    HIP_TRY(launch_scaled_gemm(p, l->stream));
  }
  if (d_dw) {
    ScaledGemmParams p = l->p.dw;
    p.c = d_dw;
    p.accumulate = accumulate_dw != 0;
    HIP_TRY(launch_scaled_gemm(p, l->stream));
  }
  return CCGLIB_OK;
}

int ccglib_scaled_linear_destroy(ccglib_scaled_linear_t l) {
  if (!l) return CCGLIB_OK;
  DeviceGuard guard(l->device);
  delete l;
  return CCGLIB_OK;
}

// ---- Orthogonalize ----

int ccglib_orthogonalize_create(ccglib_orthogonalize_t *orthogonalize, size_t B, size_t M, size_t N, int device, void *stream,
                                int type, int steps, float a, float b, float c, float epsilon, size_t in_pitch,
                                size_t out_pitch) {
  if (!orthogonalize) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null pointer: orthogonalize");
  *orthogonalize = nullptr;
  if (!is_wide_float(type)) {
    return fail(CCGLIB_ERROR_UNSUPPORTED, "Orthogonalize: matrices are float32, float16 or bfloat16 (type %d)", type);
  }
  if (steps < 1 || steps > 1000) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "Orthogonalize: 1 to 1000 steps (got %d)", steps);
  if (!(epsilon >= 0.f)) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "Orthogonalize: epsilon is not negative (got %g)", epsilon);
  constexpr size_t kMost = (size_t)1 << 20;   // (rows of 2^21 bytes)
  if (B > 65535 || M > kMost || N > kMost || (B && M && N && M * N > ((size_t)1 << 40) / B)) {
    return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "problem size out of range");
  }
  OrthogonalizeParams p = {};
  p.batch = (unsigned)B;
  p.m = (unsigned)M;
  p.n = (unsigned)N;
  p.in_pitch = in_pitch ? in_pitch : N;
  p.out_pitch = out_pitch ? out_pitch : N;
  if (p.in_pitch < N || p.out_pitch < N) {
    return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "Orthogonalize: rows of %zu values at a distance of %zu and %zu", N, p.in_pitch,
                p.out_pitch);
  }
  p.type = type;
  p.steps = steps;
  p.a = a;
  p.b = b;
  p.c = c;
  p.epsilon = epsilon;
  p.block_option = real_block_option;
  if (int s = check_device(device)) return s;
  DeviceGuard guard(device);
  HIP_TRY(guard.status());
  auto *o = new (std::nothrow) ccglib_orthogonalize{p, device, static_cast<hipStream_t>(stream), {}};
  if (!o) return fail(CCGLIB_ERROR_RUNTIME, "out of memory");
  if (B && M && N) {
    if (int s = allocate(&o->workspace, orthogonalize_workspace_bytes(p), orthogonalize_zeroed_bytes(p))) {
      delete o;
      return s;
    }
  }
  o->p.workspace = o->workspace.p;
  *orthogonalize = o;
  return CCGLIB_OK;
}

int ccglib_orthogonalize_run(ccglib_orthogonalize_t o, const void *d_in, void *d_out) {
  if (!o) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null handle");
  OrthogonalizeParams p = o->p;
  if (p.batch == 0 || p.m == 0 || p.n == 0) return CCGLIB_OK;
  if (!d_in || !d_out) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null pointer: input or output");
  if (!aligned(d_in, element(p.type)) || !aligned(d_out, element(p.type))) {
    return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "Orthogonalize: misaligned input or output");
  }
  p.in = d_in;
  p.out = d_out;
  DeviceGuard guard(o->device);
  HIP_TRY(guard.status());
  HIP_TRY(launch_orthogonalize(p, o->stream));
  return CCGLIB_OK;
}

int ccglib_orthogonalize_destroy(ccglib_orthogonalize_t o) {
  if (!o) return CCGLIB_OK;
  DeviceGuard guard(o->device);
  delete o;
  return CCGLIB_OK;
}

}  // extern "C"
