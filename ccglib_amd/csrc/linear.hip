// 16-bit linear layers: which kernel each of their products runs as, their launches, and what the backward pass does
// before its products: dz = dy act'(z), rounded to the 16 bits that the matrix cores multiply, and the bias' gradient from the same
// values in 32.
#include <algorithm>
#include <cmath>
#include <cstdio>

#include "linear_backward.h"
#include "real_plan.h"

namespace ccglib_amd {
namespace {

using namespace linear;

// (the shapes of linear_gemm.h, in their order; see real_plan.h for the figures. These were fitted to y, dx and dW of 34 problems from
// 1 x 8192 x 8192 to 8192 x 8192 x 2048, some of odd sizes, in every shape and 1 to 16 parts: there the choice is 1.2 % behind the
// fastest shape and number of parts in the mean, 13 % at most.)
constexpr RealShape kShapes[] = {{256, 256, 512, 1, 0.99f, 1.82f, 8.2f, 0.97f, "256x256"},
                                 {64, 64, 256, 2, 0.30f, 0.55f, 4.8f, 2.6f, "64x64"},
                                 {64, 32, 256, 2, 0.26f, 0.49f, 4.7f, 4.1f, "32x64"},
                                 {128, 128, 512, 1, 0.395f, 0.57f, 6.4f, 1.33f, "128x128"},
                                 {192, 192, 512, 1, 0.615f, 1.01f, 8.7f, 0.83f, "192x192"},
                                 {128, 256, 512, 1, 0.55f, 0.97f, 7.5f, 0.82f, "256x128"},
                                 {256, 256, 512, 1, 0.99f, 1.82f, 8.2f, 0.97f, "256x256 (the last ones cut)"}};
constexpr int kShapeCount = sizeof kShapes / sizeof kShapes[0], kWholeShapes = kShapeCount - 1;
static_assert(kWholeShapes == kCutShape, "the last of them");
#define CCGLIB_SAME(ID, BX, BY, WX, WY, SLOTS, EU) \
  static_assert(kShapes[ID].bx == BX && kShapes[ID].by == BY && kShapes[ID].threads == 64 * WX * WY, \
                "the table is in the order of the shapes");
CCGLIB_LINEAR_SHAPES(CCGLIB_SAME)
#undef CCGLIB_SAME

#define HIP_PASS(expr)                         \
  do {                                         \
    const hipError_t e_ = (expr);              \
    if (e_ != hipSuccess) return e_;           \
  } while (0)

// x, y and k of a product
struct Extents {
  size_t nx, ny, k;
};
Extents extents(const LinearParams &p, int kind) {
  if (kind == kOutput) return {p.n, p.m, p.k};
  if (kind == kInput) return {p.k, p.m, p.n};
  return {p.k, p.n, p.m};
}

// Blocks that a product is launched with: where rows are grouped, as many as there can be however they are (a group's
// last block may hold one row).
size_t launched_blocks(const LinearParams &p, int kind, int shape) {
  const RealShape &s = kShapes[shape];
  const Extents e = extents(p, kind);
  const size_t x = ceil_div(e.nx, s.bx);
  if (!p.grouped) {
    const size_t blocks = x * ceil_div(e.ny, s.by);
    if (shape != kCutShape) return blocks;
    const LastRound last = last_round((unsigned)(blocks % kUnits));
    return blocks + (size_t)last.blocks * (last.cut - 1);
  }
  if (kind == kWeights) return p.groups * x * ceil_div(e.ny, s.by);
  const size_t some = std::min<size_t>(p.groups, p.m);      // (groups that have rows)
  return x * (some + (p.m - some) / s.by) + (shape == kCutShape ? kMostCut : 0);
}

// Microseconds of a product with K in one part.
double product_us(int shape, size_t blocks, size_t pieces) {
  blocks = std::max<size_t>(1, blocks);
  pieces = std::max<size_t>(1, pieces);
  if (shape != kCutShape) return real_gemm_us(kShapes[shape], blocks, pieces, 1);
  const LastRound last = last_round((unsigned)(blocks % kUnits));
  if (last.cut == 1) return real_gemm_us(kShapes[shape], blocks, pieces, 1);
  return real_gemm_us(kShapes[shape], blocks - last.blocks, pieces, 1) +
         real_gemm_us(kShapes[last.cut == 2 ? 5 : 3], (size_t)last.blocks * last.cut, pieces, 1);
}
// The shape that REAL_BLOCK asks for
int shape_of(size_t option) { return (int)std::min<size_t>(option % 256 - 1, kShapeCount - 1); }

// option: REAL_BLOCK. *expected: what it takes, where the shape is given.
RealGemmPlan plan_product(const LinearParams &p, int kind, size_t option, double *expected = nullptr) {
  const Extents e = extents(p, kind);
  if (!p.grouped) {
    const size_t pieces = std::max<size_t>(1, ceil_div(e.k, (size_t)kPiece));
    RealGemmPlan plan = plan_real_gemm(kShapes, kWholeShapes, 1, e.nx, e.ny, pieces, false, option);
    const RealShape &shape = kShapes[plan.shape];
    const double us = real_gemm_us(shape, real_blocks(shape, 1, e.nx, e.ny, false), pieces, plan.parts);
    if (expected) *expected = us;
    const RealShape &cut = kShapes[kCutShape];
    const size_t blocks = real_blocks(cut, 1, e.nx, e.ny, false);
    if (option ? shape_of(option) == kCutShape : product_us(kCutShape, blocks, pieces) < us && real_launches(cut, blocks + kMostCut)) {
      plan = {};
      plan.shape = kCutShape;
      plan.parts = 1;
      plan.pieces_per_part = (unsigned)pieces;
    }
    return plan;
  }
  // K is not cut: that of kWeights has as many lengths as there are groups, and the other products have blocks of many groups. How
  // many rows each group has is not known here: the mean of what even and uneven groups would take, and of a few blocks more or less, so
  // that no choice hangs on a round of blocks that is just full.
  RealGemmPlan plan;
  double best = 0.0;
  for (int s = 0; s < kShapeCount; ++s) {
    const RealShape &shape = kShapes[s];
    if (s == kCutShape && kind == kWeights) continue;      // (whose blocks take as long as their group's rows are many)
    if (option && s != (kind == kWeights && shape_of(option) == kCutShape ? 0 : shape_of(option))) continue;
    double us = 0.0;
    for (const bool uneven : {false, true}) {
      double weights = 0.0, blocks = 0.0;
      auto weight = [&](unsigned g) {      // (rows of a group: the logarithm of their number is about normal)
        const double q = (g + 0.5) / p.groups;
        return uneven ? std::pow(q / (1.0 - q), 0.4) : 1.0;
      };
      for (unsigned g = 0; g < p.groups; ++g) weights += weight(g);
      for (unsigned g = 0; g < p.groups; ++g) {
        const double rows = weight(g) / weights * p.m;
        blocks += kind == kWeights ? (double)ceil_div(e.ny, shape.by) : rows < 1.0 ? rows : std::ceil(rows / shape.by);
      }
      blocks *= (double)ceil_div(e.nx, shape.bx);
      const size_t pieces = kind == kWeights ? ceil_div((size_t)p.m, (size_t)p.groups * kPiece) : ceil_div(e.k, (size_t)kPiece);
      for (const double more : {0.95, 1.0, 1.05, 1.1}) {      // (those of kWeights are known)
        us += product_us(s, (size_t)(kind == kWeights ? blocks : blocks * more), pieces);
      }
    }
    if (best == 0.0 || us < best) {
      best = us;
      plan.shape = s;
    }
  }
  if (expected) *expected = best / 8;
  return plan;
}

// dx and dW in one launch (linear_backward.h): in a shape in which the units hold all blocks of both at once.
bool plan_together(LinearParams *p) {
  double best = 0.0;
  for (int s = 0; s < kShapeCount; ++s) {
    if (!backward_in_one(s) || (real_block_option && s != shape_of(real_block_option))) continue;
    double us[2];
    RealGemmPlan plan[2];
    size_t blocks = 0;
    for (int i = 0; i < 2; ++i) {
      plan[i] = plan_product(*p, i ? kWeights : kInput, real_block_option ? real_block_option : (size_t)s + 1, us + i);
      blocks += launched_blocks(*p, i ? kWeights : kInput, s) * plan[i].parts;
    }
    if (blocks > (size_t)kUnits * kShapes[s].per_unit) continue;
    const double longer = std::max(us[0], us[1]);
    if (best > 0.0 && longer >= best) continue;
    best = longer;
    p->plan[kInput] = plan[0];
    p->plan[kWeights] = plan[1];
  }
  return best > 0.0;
}

// Blocks of `rows` rows of a group: as many as there can be.
size_t row_blocks(const LinearParams &p, size_t rows) {
  if (!p.grouped) return ceil_div(p.m, rows);
  const size_t some = std::min<size_t>(p.groups, p.m);
  return some + (p.m - some) / rows;
}
// Blocks of linear_rows.hip: as many as there can be.
size_t few_rows_blocks(const LinearParams &p) { return linear_rows_blocks(p.n) * row_blocks(p, kRowsOfX); }

// Whether y is linear_rows.hip's. Its blocks of 16 x 16 read their operands from the caches again and again, but wait for no ring: about 2.6 us and
// 1.7 for each 1024 of K and 256 blocks, where gemm_linear takes 3.9 and 3.4 for 1024 of K whatever the blocks. us, linear_rows and gemm_linear, W
// in the caches (W out of memory):
//   up to 256 blocks    16 x 4096 x 4096 10.1 and 12.3 (12.6 and 13.4); K = 6144 14.0 and 14.5 (18.4 and 16.4)
//   512                 16 x 8192 x 2048 10.0 and 10.8 (11.8 and 11.8); 128 x 1000 x 3000 13.0 and 11.4 (14.0 and 11.7)
//   768                 128 x 1280 x 768 6.5 and 6.8 (6.7 and 6.8); x 1000 5.8 and 7.5; x 1024 7.8 and 7.5; x 1536 10.4 and 9.8
//   1024                256 x 1024 x 256 4.4 and 4.6; x 512 6.2 and 6.1 (6.3 and 6.0); x 768 8.0 and 6.9
//   1280                128 x 2560 x 256 (5.2 and 4.9); of experts, whose rows fill fewer blocks as a rule: 256 rows over 64 of 256 x 256 (5.2 and 5.3)
// (80 other sizes, 40 of them drawn: never more than 1 % behind the best shape of gemm_linear where it is taken.)
// Up to four rows with long sums are bound by W's bytes: 8192 x 8192 24.8 and 30.1 (27.4 and 27.7). Rows that are not whole chunks are read in halves:
// 59 and 33 (1 x 8191 x 8191), 5.0 and 6.7 (1 x 1000 x 577).
// An expert's W is read for every 16 of its rows, and how many it has is not known here. Up to 16 rows in all read it once: 16 over 64 experts of 2048 x 2048
// 24.5 and 22.0 where each has its own, 7.4 and 11.2 where one has all; over 16 of 4096 x 4096 90 and 102, 12.2 and 17.3. More rows of large W would be 5 % faster with
// usual loads and as many times slower as an expert has 16 of them: 256 over 128 of 4096 x 4096 634 and 656, all to one 142 and 40 (8192 x 8192 507 and 65);
// over 1024 of 512 x 512 100 and 71, all to one 57 and 31.
bool plan_few_rows(const LinearParams &p) {
  if (real_block_option) return false;
  const double rows = p.m, products = rows * p.n * p.k;
  if (p.x_pitch % 8 || p.w_pitch % 8) return products <= 10e6;
  if (p.grouped ? p.m <= (unsigned)kRowsOfX : p.m <= 4 && rows * p.k <= 32768) return true;
  const size_t rounds = ceil_div(few_rows_blocks(p), (size_t)kUnits);
  return rounds <= (p.grouped ? 5 : 4) && rounds * rounds * p.k <= 10000 && p.k <= 5000;
}

// ---- before the products of the backward pass ----

template <int TYPE> __device__ __forceinline__ void activation_gradient(int activation, const float (&z)[8], float (&g)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (activation == kRelu) {
      g[e] = z[e] > 0.f ? g[e] : 0.f;
    } else {
      // act(z) = z s(a(z)): act' = s + z a' s (1 - s), whose second part is nothing where s (1 - s) is (a' may be infinite there)
      const float a = activation == kGelu ? gelu_argument(z[e]) : z[e];
      const float slope = activation == kGelu ? __builtin_fmaf(3.f * kGelu3 * z[e], z[e], kGelu1) : 1.f;
      const float s = sigmoid(a), curve = s * (1.f - s);
      g[e] *= curve == 0.f ? s : __builtin_fmaf(z[e] * slope, curve, s);
    }
  }
}

// Copies of the last 16 values of up to three arrays of 16-bit values, 8 zeros behind them (linear_gemm.h: Tail).
constexpr size_t kTailBytes = 64;
struct TailArgs {
  const unsigned short *end[3];
  unsigned short *to[3];
  unsigned have[3];              // values in front of `end`, 16 at most
};
__device__ __forceinline__ void make_tails(const TailArgs &a) {
  const unsigned i = threadIdx.x % 32, t = threadIdx.x / 32;
  if (t < 3 && a.to[t]) a.to[t][i] = i < 16 && 16 - i <= a.have[t] ? *(a.end[t] - (16 - i)) : (unsigned short)0;
}
__global__ __launch_bounds__(128) void copy_tails(TailArgs a) { make_tails(a); }

struct GradientArgs {
  const char *dy, *z;
  size_t pitch;                  // elements, of dy and z
  char *dz;                      // null: not wanted
  size_t dz_pitch;
  float *sums;                   // [row block][n]; null: not wanted
  unsigned n, rows;
  int activation;
  // as linear::Args
  const int *offsets;
  unsigned groups;
};

// dz = dy act'(z) and, for each block of ROWS rows of a group, the sums of its columns. Bound by memory: 8192 x 4096, 201 MB, 43 us, 4.6 TB/s.
template <int TYPE, unsigned ROWS> __global__ __launch_bounds__(256) void linear_gradient(GradientArgs a, TailArgs tails) {
  using T = typename Value<TYPE>::type;
  __shared__ float joined[3][kGradientColumns];
  if (blockIdx.x == 0 && blockIdx.y == 0) make_tails(tails);
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned x = blockIdx.x * kGradientColumns + lane * 8, left = x < a.n ? a.n - x : 0;
  unsigned first = blockIdx.y * ROWS, until = first + ROWS < a.rows ? first + ROWS : a.rows;
  if (a.offsets) {
    RowBlocks<ROWS> blocks(a.offsets, a.groups, a.rows);
    if (blockIdx.y >= blocks.all()) return;
    const RowBlock r = blocks.find(blockIdx.y);
    first = r.rows.first + r.block * ROWS;
    until = r.rows.first + r.rows.count < first + ROWS ? r.rows.first + r.rows.count : first + ROWS;
  }
  float sum[8] = {};
#pragma unroll 4
  for (unsigned row = first + wave; row < until; row += 4) {
    if (left == 0) break;
    float g[8], z[8];
    load_row(reinterpret_cast<const T *>(a.dy) + (size_t)row * a.pitch + x, left, g);
    if (a.activation != kNone) {
      load_row(reinterpret_cast<const T *>(a.z) + (size_t)row * a.pitch + x, left, z);
      activation_gradient<TYPE>(a.activation, z, g);
    }
    if (a.dz) real::store_row(reinterpret_cast<T *>(a.dz) + (size_t)row * a.dz_pitch + x, left, g);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] += g[e];
  }
  if (!a.sums) return;
  if (wave > 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) joined[wave - 1][e * 64 + lane] = sum[e];
  }
  __syncthreads();
  if (wave == 0 && left) {
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] = (sum[e] + joined[0][e * 64 + lane]) + (joined[1][e * 64 + lane] + joined[2][e * 64 + lane]);
    real::store_row(a.sums + (size_t)blockIdx.y * a.n + x, left, sum);
  }
}

__global__ __launch_bounds__(256) void join_sums(JoinArgs a) {
  __shared__ float lds[256];
  join(a, lds, blockIdx.x);
}

// An operand of a product: an array of 16-bit values.
struct Operand {
  const void *p;
  size_t rows, columns, pitch;   // elements
};

// Collects the copies of ends that products need, and makes them.
class Tails {
 public:
  explicit Tails(char *memory) : memory_(memory) {}
  // k: the length of the sum, strided: whether the operand's rows are along it
  Tail of(const Operand &o, size_t k, bool strided) {
    const bool loose = o.pitch % 8 != 0 || (uintptr_t)o.p % 16 != 0;
    if (!loose || (!strided && k >= 8) || o.rows == 0 || o.columns == 0) return {};
    const size_t values = (o.rows - 1) * o.pitch + o.columns;
    const char *const end = static_cast<const char *>(o.p) + 2 * values;
    int i = 0;
    while (i < count_ && reinterpret_cast<const char *>(args_.end[i]) != end) ++i;
    char *const to = memory_ + i * kTailBytes;
    if (i == count_) {
      args_.end[i] = reinterpret_cast<const unsigned short *>(end);
      args_.to[i] = reinterpret_cast<unsigned short *>(to);
      ++count_;
    }
    // (operands may end together and start apart: W may be a row of x)
    args_.have[i] = std::max(args_.have[i], (unsigned)std::min<size_t>(16, values));
    return {to, end};
  }
  const TailArgs &args() const { return args_; }
  hipError_t launch(hipStream_t stream) const {
    if (count_ == 0) return hipSuccess;
    copy_tails<<<1, 128, 0, stream>>>(args_);
    return hipGetLastError();
  }

 private:
  char *memory_;
  TailArgs args_ = {};
  int count_ = 0;
};

// Half of an XCD's L2.
constexpr size_t kStaysInCaches = (size_t)2 << 20;

Args product_args(const LinearParams &p, int kind, const Operand &x, const Operand &y, const int *offsets, Tails *tails) {
  const Extents e = extents(p, kind);
  const RealGemmPlan &plan = p.plan[kind];
  const RealShape &s = kShapes[plan.shape];
  Args a = {};
  a.x = static_cast<const char *>(x.p);
  a.y = static_cast<const char *>(y.p);
  a.nx = (unsigned)e.nx;
  a.ny = (unsigned)e.ny;
  a.k = (unsigned)e.k;
  a.x_pitch = (unsigned)(2 * x.pitch);
  a.y_pitch = (unsigned)(2 * y.pitch);
  a.x_tail = tails->of(x, kind == kWeights && p.grouped ? 8 : e.k, kind != kOutput);
  a.y_tail = tails->of(y, kind == kWeights && p.grouped ? 8 : e.k, kind == kWeights);
  a.offsets = p.grouped ? offsets : nullptr;
  a.groups = p.groups;
  a.rows = p.m;
  a.x_group = 2 * (size_t)p.n * p.w_pitch;
  a.blocks_x = (unsigned)ceil_div(e.nx, s.bx);
  a.blocks_y = (unsigned)ceil_div(e.ny, s.by);
  a.parts = plan.parts;
  a.pieces_per_part = plan.pieces_per_part;
  a.rotate = kind != kWeights && 2 * e.ny * e.k <= kStaysInCaches;
  a.arrived = reinterpret_cast<unsigned *>(p.workspace + p.counters[kind]);
  a.partial = reinterpret_cast<float *>(p.workspace + p.partial[kind]);
  return a;
}

hipError_t launch_product(const LinearParams &p, int kind, const Args &a, const StoreParams &s, hipStream_t stream) {
  const RealGemmPlan &plan = p.plan[kind];
  const unsigned grid = (unsigned)(launched_blocks(p, kind, plan.shape) * plan.parts);
  if (grid == 0) return hipSuccess;
  if (p.type == kFloat16) {
    if (kind == kOutput) return launch_gemm<kFloat16, kOutput>(plan.shape, grid, a, s, stream);
    if (kind == kInput) return launch_gemm<kFloat16, kInput>(plan.shape, grid, a, s, stream);
    return launch_gemm<kFloat16, kWeights>(plan.shape, grid, a, s, stream);
  }
  if (kind == kOutput) return launch_gemm<kBfloat16, kOutput>(plan.shape, grid, a, s, stream);
  if (kind == kInput) return launch_gemm<kBfloat16, kInput>(plan.shape, grid, a, s, stream);
  return launch_gemm<kBfloat16, kWeights>(plan.shape, grid, a, s, stream);
}

// Whether y and z are stored past the caches: where these do not hold what the product reads and writes, so that what is stored would
// push out operands and residual that are still to be read (us, kept and past, with residual and z: 8192 x 4096 x 4096, 288 MiB, 251 and 217; 16384 x
// 2048 x 2048, 264 MiB, 163 and 128; 8192 x 8192 x 1024 with the residual alone, 288 MiB, 191 and 155; below 256 MiB 0 to 7 % either way, and the
// next layer finds y there). y alone, dx and dW gain nothing up to 256 MiB of their own (16383 rows over 16 experts of 4096 x 2048: 298 and 311).
bool past_caches(const LinearParams &p, const LinearForward &f) {
  const size_t x = (size_t)p.m * p.k, y = (size_t)p.m * p.n, w = (size_t)p.groups * p.n * p.k;
  if (!f.z && !f.residual) return 2 * y >= kPastCachesBytes;
  return 2 * (x + w + y * (1 + (f.z ? 1 : 0) + (f.residual ? 1 : 0))) >= kPastCachesBytes;
}

size_t dz_pitch(const LinearParams &p) { return ceil_div(p.n, (size_t)8) * 8; }

unsigned gradient_rows(const LinearParams &p) {
  return row_blocks(p, kManyRows) * ceil_div(p.n, (size_t)kGradientColumns) < 512 ? kFewRows : kManyRows;
}
size_t gradient_blocks(const LinearParams &p) { return row_blocks(p, gradient_rows(p)); }

template <unsigned ROWS> hipError_t launch_gradient(const LinearParams &p, const GradientArgs &g, const TailArgs &t, hipStream_t stream) {
  const dim3 grid((unsigned)ceil_div(p.n, (size_t)kGradientColumns), (unsigned)gradient_blocks(p));
  if (p.type == kFloat16) {
    linear_gradient<kFloat16, ROWS><<<grid, 256, 0, stream>>>(g, t);
  } else {
    linear_gradient<kBfloat16, ROWS><<<grid, 256, 0, stream>>>(g, t);
  }
  return hipGetLastError();
}
}  // namespace

void plan_linear(LinearParams *p) {
  const int kinds = p->training ? 3 : 1;
  size_t counters = 0, partial = 0;
  p->few_rows = plan_few_rows(*p);
  for (int kind = p->few_rows ? 1 : 0; kind < kinds; ++kind) {
    p->plan[kind] = plan_product(*p, kind, real_block_option);
  }
  p->together = p->training && plan_together(p);
  // (where dW runs beside dx it has counters and sums of its own)
  size_t apart = 0, apart_partial = 0;
  for (int kind = 0; kind < kinds; ++kind) {
    const RealGemmPlan &plan = p->plan[kind];
    if (kind == kWeights && p->together) {
      apart = ceil_div(counters, 256) * 256;
      apart_partial = ceil_div(partial, 256) * 256;
      counters = apart + plan.counter_bytes;
      partial = apart_partial + plan.partial_bytes;
    } else {
      counters = std::max(counters, plan.counter_bytes);
      partial = std::max(partial, plan.partial_bytes);
    }
  }
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += ceil_div(bytes, 256) * 256;
    return here;
  };
  p->zeroed = counters;
  take(counters);
  const size_t sums = take(partial);
  for (int kind = 0; kind < 3; ++kind) {
    p->counters[kind] = kind == kWeights ? apart : 0;
    p->partial[kind] = sums + (kind == kWeights ? apart_partial : 0);
  }
  p->dz = take(p->training && p->activation != kNone ? 2 * (size_t)p->m * dz_pitch(*p) : 0);
  p->sums = take(p->training ? 4 * gradient_blocks(*p) * p->n : 0);
  p->tails = take(3 * kTailBytes);
  p->bytes = at;
}

bool linear_launches(const LinearParams &p) {
  if (p.few_rows && few_rows_blocks(p) > 0xffffffffu / 256) return false;
  for (int kind = p.few_rows ? 1 : 0; kind < (p.training ? 3 : 1); ++kind) {
    const int shape = p.plan[kind].shape;
    if (!real_launches(kShapes[shape], launched_blocks(p, kind, shape) * p.plan[kind].parts)) return false;
  }
  if (!p.training) return true;
  // (blocks of rows are a grid's second axis, groups too)
  const size_t columns = ceil_div(p.n, (size_t)kGradientColumns);
  return gradient_blocks(p) <= 65535 && gradient_blocks(p) * columns <= 0xffffffu && join_workgroups(p.n, p.groups) <= 0xffffffu;
}

const char *describe_linear(const LinearParams &p, int kind) {
  static thread_local char name[128];
  if (kind == kOutput && p.few_rows) {
    snprintf(name, sizeof name, "linear_rows<%s>", p.type == kFloat16 ? "float16" : "bfloat16");
    return name;
  }
  static const char *const kinds[] = {"forward", "input's gradient", "weights' gradient"};
  const bool together = kind != kOutput && p.together;
  snprintf(name, sizeof name, "gemm_linear%s<%s, %s> %s block, K in %u%s", together ? "_backward" : "",
           p.type == kFloat16 ? "float16" : "bfloat16", kinds[kind], kShapes[p.plan[kind].shape].name, p.plan[kind].parts,
           together ? ", dx and dW in one launch" : "");
  return name;
}

hipError_t launch_linear_forward(const LinearParams &p, const LinearForward &f, hipStream_t stream) {
  if (p.m == 0 || p.n == 0) return hipSuccess;
  StoreParams s = {};
  s.out = static_cast<char *>(f.y);
  s.z = static_cast<char *>(f.z);
  s.bias = static_cast<const char *>(f.bias);
  s.residual = static_cast<const char *>(f.residual);
  s.pitch = p.y_pitch;
  s.activation = p.activation;
  s.past = past_caches(p, f);
  Tails tails(p.workspace + p.tails);
  const Operand x = {f.x, p.m, p.k, p.x_pitch}, w = {f.w, (size_t)p.groups * p.n, p.k, p.w_pitch};
  Args a = product_args(p, kOutput, w, x, f.offsets, &tails);
  if (p.few_rows) {      // (which reads no more than the rows)
    a.blocks_x = (unsigned)linear_rows_blocks(p.n);
    return launch_linear_rows(p.type, (unsigned)few_rows_blocks(p), a, s, stream);
  }
  HIP_PASS(tails.launch(stream));
  return launch_product(p, kOutput, a, s, stream);
}

hipError_t launch_linear_backward(const LinearParams &p, const LinearBackward &b, hipStream_t stream) {
  if (p.n == 0) {
    // (sums of nothing)
    if (!b.dx || p.m == 0 || p.k == 0) return hipSuccess;
  }
  const bool activated = p.activation != kNone, few = gradient_rows(p) == kFewRows;
  Operand dz = {b.dy, p.m, p.n, p.y_pitch};
  if (activated) dz = {p.workspace + p.dz, p.m, p.n, dz_pitch(p)};
  Tails tails(p.workspace + p.tails);
  const Operand x = {b.x, p.m, p.k, p.x_pitch}, w = {b.w, (size_t)p.groups * p.n, p.k, p.w_pitch};
  Args input = {}, weights = {};
  if (b.dx) input = product_args(p, kInput, w, dz, b.offsets, &tails);
  if (b.dw) weights = product_args(p, kWeights, x, dz, b.offsets, &tails);
  if (p.m && p.n && (b.dbias || (activated && (b.dx || b.dw)))) {
    GradientArgs g = {};
    g.dy = static_cast<const char *>(b.dy);
    g.z = static_cast<const char *>(b.z);
    g.pitch = p.y_pitch;
    g.dz = activated && (b.dx || b.dw) ? p.workspace + p.dz : nullptr;
    g.dz_pitch = dz_pitch(p);
    g.sums = b.dbias ? reinterpret_cast<float *>(p.workspace + p.sums) : nullptr;
    g.n = p.n;
    g.rows = p.m;
    g.activation = p.activation;
    g.offsets = p.grouped ? b.offsets : nullptr;
    g.groups = p.groups;
    HIP_PASS(few ? launch_gradient<kFewRows>(p, g, tails.args(), stream) : launch_gradient<kManyRows>(p, g, tails.args(), stream));
  } else {
    HIP_PASS(tails.launch(stream));
  }
  JoinArgs j = {};
  unsigned joins = 0;
  if (b.dbias && p.n) {
    j.sums = reinterpret_cast<const float *>(p.workspace + p.sums);
    j.db = static_cast<char *>(b.dbias);
    j.n = p.n;
    j.rows = p.m;
    j.blocks = (unsigned)gradient_blocks(p);
    j.few = few;
    j.type = p.gradient_type;
    j.accumulate = b.accumulate;
    j.offsets = p.grouped ? b.offsets : nullptr;
    j.groups = p.groups;
    joins = (unsigned)join_workgroups(p.n, p.groups);
  }
  StoreParams si = {}, sw = {};
  si.out = static_cast<char *>(b.dx);
  si.pitch = p.x_pitch;
  si.past = 2 * (size_t)p.m * p.k >= kPastCachesBytes;
  sw.out = static_cast<char *>(b.dw);
  sw.pitch = p.w_pitch;
  sw.group = (size_t)p.n * p.w_pitch;
  sw.wide = p.gradient_type == kFloat32;
  sw.past = (sw.wide ? 4 : 2) * (size_t)p.groups * p.n * p.k >= kPastCachesBytes;
  sw.accumulate = b.accumulate;
  const bool have_dx = b.dx && p.m && p.k, have_dw = b.dw && p.n && p.k;
  if (p.together && have_dx && have_dw) {
    BackwardArgs a = {input, weights, si, sw, j, 0, 0};
    const int shape = p.plan[kInput].shape;
    a.input_blocks = (unsigned)(launched_blocks(p, kInput, shape) * p.plan[kInput].parts);
    a.weights_blocks = (unsigned)(launched_blocks(p, kWeights, shape) * p.plan[kWeights].parts);
    const unsigned grid = a.input_blocks + a.weights_blocks + joins;
    if (p.type == kFloat16) return launch_backward<kFloat16>(shape, grid, a, stream);
    return launch_backward<kBfloat16>(shape, grid, a, stream);
  }
  if (joins) {
    join_sums<<<joins, 256, 0, stream>>>(j);
    HIP_PASS(hipGetLastError());
  }
  if (have_dx) HIP_PASS(launch_product(p, kInput, input, si, stream));
  if (have_dw) HIP_PASS(launch_product(p, kWeights, weights, sw, stream));
  return hipSuccess;
}

}  // namespace ccglib_amd
