// C ABI of the 16-bit linear layers, of those grouped by expert, and of the routing between them (declared in
// include/ccglib_amd.h): argument checking, object state and workspaces around the kernel launchers. None of them has a
// counterpart in the reference.
#include <cstdio>
#include <new>

#include "host_util.h"
#include "linear.h"
#include "route.h"

using namespace ccglib_amd;

namespace {

constexpr size_t kMostRows = 0x7fffffffu;
constexpr size_t kMostPitch = (size_t)1 << 22;    // values: 256 rows are addressed with 32-bit offsets
constexpr size_t kMostTokens = ((size_t)1 << 24) - 1;   // (256 threads each in a launch)

size_t element(int type) { return (size_t)bits_of(type) / 8; }
bool is_half(int type) { return type == kFloat16 || type == kBfloat16; }

int check_linear(const char *who, const LinearParams &p, size_t groups, size_t M, size_t N, size_t K) {
  if (!is_half(p.type)) return fail(CCGLIB_ERROR_UNSUPPORTED, "%s: values are float16 or bfloat16 (type %d)", who, p.type);
  if (p.gradient_type != p.type && p.gradient_type != kFloat32) {
    return fail(CCGLIB_ERROR_UNSUPPORTED, "%s: gradients of weights are of the values' type or float32 (type %d)", who, p.gradient_type);
  }
  if (p.activation < kNone || p.activation > kSilu) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "enum argument out of range");
  if (groups < 1 || groups > kMostExperts) {
    return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "%s: 1 to %zu experts (got %zu)", who, kMostExperts, groups);
  }
  if (M > kMostRows || N > kMostPitch || K > kMostPitch) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "problem size out of range");
  if (p.x_pitch < K || p.w_pitch < K || p.y_pitch < N || p.x_pitch > kMostPitch || p.w_pitch > kMostPitch || p.y_pitch > kMostPitch) {
    return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "%s: rows of %zu, %zu and %zu values at distances of %zu, %zu and %zu (at most %zu)", who,
                K, K, N, p.x_pitch, p.w_pitch, p.y_pitch, kMostPitch);
  }
  return CCGLIB_OK;
}

struct Linear {
  LinearParams p;
  int device;
  hipStream_t stream;
  Buffer workspace;
};

template <class Handle>
int create_linear(Handle **out, const char *who, size_t groups, bool grouped, size_t M, size_t N, size_t K, int device, void *stream,
                  int type, int activation, int gradient_type, int training, size_t x_pitch, size_t w_pitch, size_t y_pitch) {
  LinearParams p = {};
  p.m = (unsigned)M;
  p.n = (unsigned)N;
  p.k = (unsigned)K;
  p.groups = (unsigned)groups;
  p.grouped = grouped;
  p.training = training != 0;
  p.type = type;
  p.gradient_type = gradient_type;
  p.activation = activation;
  p.x_pitch = x_pitch ? x_pitch : K;
  p.w_pitch = w_pitch ? w_pitch : K;
  p.y_pitch = y_pitch ? y_pitch : N;
  if (int s = check_linear(who, p, groups, M, N, K)) return s;
  plan_linear(&p);
  if (!linear_launches(p)) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "problem size out of range: more blocks than a launch takes");
  if (int s = check_device(device)) return s;
  DeviceGuard guard(device);
  HIP_TRY(guard.status());
  auto *l = new (std::nothrow) Handle;
  if (!l) return fail(CCGLIB_ERROR_RUNTIME, "out of memory");
  l->p = p;
  l->device = device;
  l->stream = static_cast<hipStream_t>(stream);
  if (int s = allocate(&l->workspace, p.bytes, p.zeroed)) {
    delete l;
    return s;
  }
  l->p.workspace = l->workspace.at(0);
  *out = l;
  return CCGLIB_OK;
}

// A buffer of `values` elements of `type`: it is there, and aligned to them.
int check_buffer(const char *who, const char *what, const void *p, bool wanted, int type) {
  if (!p && wanted) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null pointer: %s, %s", who, what);
  if (!aligned(p, element(type))) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "%s: misaligned %s", who, what);
  return CCGLIB_OK;
}

int forward(Linear *l, const char *who, const LinearForward &f) {
  const LinearParams &p = l->p;
  if (p.m == 0 || p.n == 0) return CCGLIB_OK;
  if (int s = check_buffer(who, "x", f.x, p.k > 0, p.type)) return s;
  if (int s = check_buffer(who, "weights", f.w, p.k > 0, p.type)) return s;
  if (int s = check_buffer(who, "bias", f.bias, false, p.type)) return s;
  if (int s = check_buffer(who, "residual", f.residual, false, p.type)) return s;
  if (int s = check_buffer(who, "y", f.y, true, p.type)) return s;
  if (int s = check_buffer(who, "z", f.z, false, p.type)) return s;
  if (int s = check_buffer(who, "offsets", f.offsets, p.grouped, kInt32)) return s;
  DeviceGuard guard(l->device);
  HIP_TRY(guard.status());
  HIP_TRY(launch_linear_forward(p, f, l->stream));
  return CCGLIB_OK;
}

int backward(Linear *l, const char *who, const LinearBackward &b) {
  const LinearParams &p = l->p;
  if (!p.training) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "%s: backward of a layer that was created without training", who);
  if (b.accumulate && p.gradient_type != kFloat32) {
    return fail(CCGLIB_ERROR_UNSUPPORTED, "%s: gradients that are added to are float32 (type %d)", who, p.gradient_type);
  }
  if (!b.dx && !b.dw && !b.dbias) return CCGLIB_OK;
  const bool rows = p.m > 0 && p.n > 0;
  if (int s = check_buffer(who, "dy", b.dy, rows, p.type)) return s;
  if (int s = check_buffer(who, "z", b.z, rows && p.activation != kNone, p.type)) return s;
  if (int s = check_buffer(who, "x", b.x, b.dw && p.m > 0 && p.k > 0, p.type)) return s;
  if (int s = check_buffer(who, "weights", b.w, b.dx && p.n > 0 && p.k > 0, p.type)) return s;
  if (int s = check_buffer(who, "dx", b.dx, false, p.type)) return s;
  if (int s = check_buffer(who, "dw", b.dw, false, p.gradient_type)) return s;
  if (int s = check_buffer(who, "dbias", b.dbias, false, p.gradient_type)) return s;
  if (int s = check_buffer(who, "offsets", b.offsets, p.grouped, kInt32)) return s;
  DeviceGuard guard(l->device);
  HIP_TRY(guard.status());
  HIP_TRY(launch_linear_backward(p, b, l->stream));
  return CCGLIB_OK;
}

int kernel_name(Linear *l, int product, char *buffer, size_t size) {
  if (!buffer || size == 0) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null handle or buffer");
  if (product < 0 || product > (l->p.training ? 2 : 0)) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "no such product: %d", product);
  snprintf(buffer, size, "%s", describe_linear(l->p, product));
  return CCGLIB_OK;
}

template <class Handle> int destroy(Handle *l) {
  if (!l) return CCGLIB_OK;
  DeviceGuard guard(l->device);
  delete l;
  return CCGLIB_OK;
}

}  // namespace

struct ccglib_fused_linear : Linear {};
struct ccglib_grouped_linear : Linear {};

struct ccglib_route {
  RouteParams p;
  int device;
  hipStream_t stream;
  Buffer workspace;
};

struct ccglib_combine {
  CombineParams p;
  int device;
  hipStream_t stream;
};

extern "C" {

// ---- FusedLinear ----

int ccglib_fused_linear_create(ccglib_fused_linear_t *linear, size_t M, size_t N, size_t K, int device, void *stream, int type,
                               int activation, int gradient_type, int training, size_t x_pitch, size_t w_pitch, size_t y_pitch) {
  if (!linear) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null pointer: linear");
  *linear = nullptr;
  return create_linear(linear, "FusedLinear", 1, false, M, N, K, device, stream, type, activation, gradient_type, training, x_pitch,
                       w_pitch, y_pitch);
}

int ccglib_fused_linear_forward(ccglib_fused_linear_t l, const void *d_x, const void *d_w, const void *d_bias, const void *d_residual,
                                void *d_y, void *d_z) {
  if (!l) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null handle");
  return forward(l, "FusedLinear", {d_x, d_w, d_bias, d_residual, nullptr, d_y, d_z});
}

int ccglib_fused_linear_backward(ccglib_fused_linear_t l, const void *d_dy, const void *d_z, const void *d_x, const void *d_w, void *d_dx,
                                 void *d_dw, void *d_dbias, int accumulate) {
  if (!l) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null handle");
  return backward(l, "FusedLinear", {d_dy, d_z, d_x, d_w, nullptr, d_dx, d_dw, d_dbias, accumulate != 0});
}

int ccglib_fused_linear_kernel_name(ccglib_fused_linear_t l, int product, char *buffer, size_t size) {
  if (!l) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null handle or buffer");
  return kernel_name(l, product, buffer, size);
}

int ccglib_fused_linear_destroy(ccglib_fused_linear_t l) { return destroy(l); }

// ---- GroupedLinear ----

int ccglib_grouped_linear_create(ccglib_grouped_linear_t *linear, size_t E, size_t M, size_t N, size_t K, int device, void *stream,
                                 int type, int activation, int gradient_type, int training, size_t x_pitch, size_t w_pitch,
                                 size_t y_pitch) {
  if (!linear) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null pointer: linear");
  *linear = nullptr;
  return create_linear(linear, "GroupedLinear", E, true, M, N, K, device, stream, type, activation, gradient_type, training, x_pitch,
                       w_pitch, y_pitch);
}

int ccglib_grouped_linear_forward(ccglib_grouped_linear_t l, const void *d_x, const void *d_offsets, const void *d_w, const void *d_bias,
                                  const void *d_residual, void *d_y, void *d_z) {
  if (!l) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null handle");
  return forward(l, "GroupedLinear", {d_x, d_w, d_bias, d_residual, static_cast<const int *>(d_offsets), d_y, d_z});
}

int ccglib_grouped_linear_backward(ccglib_grouped_linear_t l, const void *d_dy, const void *d_z, const void *d_x, const void *d_offsets,
                                   const void *d_w, void *d_dx, void *d_dw, void *d_dbias, int accumulate) {
  if (!l) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null handle");
  return backward(l, "GroupedLinear",
                  {d_dy, d_z, d_x, d_w, static_cast<const int *>(d_offsets), d_dx, d_dw, d_dbias, accumulate != 0});
}

int ccglib_grouped_linear_kernel_name(ccglib_grouped_linear_t l, int product, char *buffer, size_t size) {
  if (!l) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null handle or buffer");
  return kernel_name(l, product, buffer, size);
}

int ccglib_grouped_linear_destroy(ccglib_grouped_linear_t l) { return destroy(l); }

// ---- Route ----

int ccglib_route_create(ccglib_route_t *route, size_t T, size_t E, size_t k, int device, void *stream, int type, int normalize) {
  if (!route) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null pointer: route");
  *route = nullptr;
  if (!is_wide_float(type)) return fail(CCGLIB_ERROR_UNSUPPORTED, "Route: logits are float32, float16 or bfloat16 (type %d)", type);
  if (E < 1 || E > kMostExperts || k < 1 || k > kMostChosen || k > E) {
    return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "Route: 1 to %zu experts, of which 1 to %zu are chosen (got %zu, %zu)", kMostExperts,
                kMostChosen, E, k);
  }
  if (T > kMostTokens) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "problem size out of range");
  if (int s = check_device(device)) return s;
  RouteParams p = {};
  p.tokens = (unsigned)T;
  p.experts = (unsigned)E;
  p.chosen = (unsigned)k;
  p.type = type;
  p.normalize = normalize != 0;
  plan_route(&p);
  DeviceGuard guard(device);
  HIP_TRY(guard.status());
  auto *r = new (std::nothrow) ccglib_route{p, device, static_cast<hipStream_t>(stream), {}};
  if (!r) return fail(CCGLIB_ERROR_RUNTIME, "out of memory");
  if (int s = allocate(&r->workspace, route_workspace_bytes(p), 0)) {
    delete r;
    return s;
  }
  r->p.counts = static_cast<unsigned short *>(r->workspace.p);
  *route = r;
  return CCGLIB_OK;
}

int ccglib_route_run(ccglib_route_t r, const void *d_logits, void *d_experts, void *d_weights, void *d_offsets, void *d_slots) {
  if (!r) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null handle");
  const RouteParams &p = r->p;
  if (int s = check_buffer("Route", "logits", d_logits, p.tokens > 0, p.type)) return s;
  if (int s = check_buffer("Route", "experts", d_experts, p.tokens > 0, kInt32)) return s;
  if (int s = check_buffer("Route", "weights", d_weights, p.tokens > 0, kFloat32)) return s;
  if (int s = check_buffer("Route", "offsets", d_offsets, true, kInt32)) return s;
  if (int s = check_buffer("Route", "slots", d_slots, p.tokens > 0, kInt32)) return s;
  DeviceGuard guard(r->device);
  HIP_TRY(guard.status());
  HIP_TRY(launch_route(p, d_logits, static_cast<int *>(d_experts), static_cast<float *>(d_weights), static_cast<int *>(d_offsets),
                       static_cast<int *>(d_slots), r->stream));
  return CCGLIB_OK;
}

int ccglib_route_backward(ccglib_route_t r, const void *d_logits, const void *d_experts, const void *d_weights, const void *d_dweights,
                          void *d_dlogits) {
  if (!r) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null handle");
  const RouteParams &p = r->p;
  if (p.tokens == 0) return CCGLIB_OK;
  if (int s = check_buffer("Route", "logits", d_logits, !p.normalize, p.type)) return s;
  if (int s = check_buffer("Route", "experts", d_experts, true, kInt32)) return s;
  if (int s = check_buffer("Route", "weights", d_weights, true, kFloat32)) return s;
  if (int s = check_buffer("Route", "dweights", d_dweights, true, kFloat32)) return s;
  if (int s = check_buffer("Route", "dlogits", d_dlogits, true, p.type)) return s;
  DeviceGuard guard(r->device);
  HIP_TRY(guard.status());
  HIP_TRY(launch_route_backward(p, d_logits, static_cast<const int *>(d_experts), static_cast<const float *>(d_weights),
                                static_cast<const float *>(d_dweights), d_dlogits, r->stream));
  return CCGLIB_OK;
}

int ccglib_route_destroy(ccglib_route_t r) {
  if (!r) return CCGLIB_OK;
  DeviceGuard guard(r->device);
  delete r;
  return CCGLIB_OK;
}

// ---- Combine ----

int ccglib_combine_create(ccglib_combine_t *combine, size_t T, size_t k, size_t N, int device, void *stream, int type, size_t rows,
                          size_t y_pitch, size_t out_pitch) {
  if (!combine) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null pointer: combine");
  *combine = nullptr;
  if (!is_half(type)) return fail(CCGLIB_ERROR_UNSUPPORTED, "Combine: values are float16 or bfloat16 (type %d)", type);
  if (k < 1 || k > kMostChosen) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "Combine: 1 to %zu rows a token (got %zu)", kMostChosen, k);
  if (T > kMostTokens || N > kMostPitch || rows > kMostRows) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "problem size out of range");
  CombineParams p = {};
  p.tokens = (unsigned)T;
  p.chosen = (unsigned)k;
  p.n = (unsigned)N;
  p.rows = (unsigned)(rows ? rows : T * k);
  p.type = type;
  p.y_pitch = y_pitch ? y_pitch : N;
  p.out_pitch = out_pitch ? out_pitch : N;
  if (p.y_pitch < N || p.out_pitch < N || p.y_pitch > kMostPitch || p.out_pitch > kMostPitch) {
    return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "Combine: rows of %zu values at distances of %zu and %zu (at most %zu)", N, p.y_pitch,
                p.out_pitch, kMostPitch);
  }
  if (int s = check_device(device)) return s;
  auto *c = new (std::nothrow) ccglib_combine{p, device, static_cast<hipStream_t>(stream)};
  if (!c) return fail(CCGLIB_ERROR_RUNTIME, "out of memory");
  *combine = c;
  return CCGLIB_OK;
}

int ccglib_combine_run(ccglib_combine_t c, const void *d_y, const void *d_slots, const void *d_weights, void *d_out) {
  if (!c) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null handle");
  const CombineParams &p = c->p;
  if (p.tokens == 0 || p.n == 0) return CCGLIB_OK;
  if (int s = check_buffer("Combine", "y", d_y, true, p.type)) return s;
  if (int s = check_buffer("Combine", "slots", d_slots, true, kInt32)) return s;
  if (int s = check_buffer("Combine", "weights", d_weights, false, kFloat32)) return s;
  if (int s = check_buffer("Combine", "output", d_out, true, p.type)) return s;
  DeviceGuard guard(c->device);
  HIP_TRY(guard.status());
  HIP_TRY(launch_combine(p, d_y, static_cast<const int *>(d_slots), static_cast<const float *>(d_weights), d_out, c->stream));
  return CCGLIB_OK;
}

int ccglib_combine_spread(ccglib_combine_t c, const void *d_x, const void *d_slots, const void *d_weights, void *d_y) {
  if (!c) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null handle");
  const CombineParams &p = c->p;
  if (p.tokens == 0 || p.n == 0) return CCGLIB_OK;
  if (int s = check_buffer("Combine", "x", d_x, true, p.type)) return s;
  if (int s = check_buffer("Combine", "slots", d_slots, true, kInt32)) return s;
  if (int s = check_buffer("Combine", "weights", d_weights, false, kFloat32)) return s;
  if (int s = check_buffer("Combine", "y", d_y, true, p.type)) return s;
  DeviceGuard guard(c->device);
  HIP_TRY(guard.status());
  HIP_TRY(launch_combine_backward(p, d_x, nullptr, static_cast<const int *>(d_slots), static_cast<const float *>(d_weights), d_y,
                                  nullptr, c->stream));
  return CCGLIB_OK;
}

int ccglib_combine_backward(ccglib_combine_t c, const void *d_dout, const void *d_y, const void *d_slots, const void *d_weights,
                            void *d_dy, void *d_dweights) {
  if (!c) return fail(CCGLIB_ERROR_INVALID_ARGUMENT, "null handle");
  const CombineParams &p = c->p;
  if (p.tokens == 0 || (!d_dy && !d_dweights)) return CCGLIB_OK;
  if (int s = check_buffer("Combine", "dout", d_dout, p.n > 0, p.type)) return s;
  if (int s = check_buffer("Combine", "y", d_y, d_dweights && p.n > 0, p.type)) return s;
  if (int s = check_buffer("Combine", "slots", d_slots, true, kInt32)) return s;
  if (int s = check_buffer("Combine", "weights", d_weights, false, kFloat32)) return s;
  if (int s = check_buffer("Combine", "dy", d_dy, false, p.type)) return s;
  if (int s = check_buffer("Combine", "dweights", d_dweights, false, kFloat32)) return s;
  DeviceGuard guard(c->device);
  HIP_TRY(guard.status());
  HIP_TRY(launch_combine_backward(p, d_dout, d_dweights ? d_y : nullptr, static_cast<const int *>(d_slots),
                                  static_cast<const float *>(d_weights), d_dy, static_cast<float *>(d_dweights), c->stream));
  return CCGLIB_OK;
}

int ccglib_combine_destroy(ccglib_combine_t c) {
  delete c;
  return CCGLIB_OK;
}

}  // extern "C"
