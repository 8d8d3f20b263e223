// Parameter blocks of the operators on 8-bit values with block scales and of the orthogonalised updates, handed from
// the C ABI layer (operators_capi.hip) to the kernel launchers.
#ifndef CCGLIB_AMD_SCALED_H_
#define CCGLIB_AMD_SCALED_H_

#include "common.h"

namespace ccglib_amd {

enum : int { kScaleRows = 0, kScaleBlocks = 1 };
enum : int { kScaleFloat32 = 0, kScaleE8m0 = 1 };

constexpr size_t kScaleGroup = 128;   // values of a row that share a scale

// Rows of 8-bit values, and rows of scales, are padded to this many elements.
constexpr size_t kScaledPad = 16;
inline size_t scaled_pitch(size_t n) { return ceil_div(n, kScaledPad) * kScaledPad; }
inline size_t scale_rows(size_t rows, int group) { return group == kScaleRows ? rows : ceil_div(rows, kScaleGroup); }
inline bool is_float8(int type) { return type == kFloat8e4m3 || type == kFloat8e5m2; }
inline bool is_wide_float(int type) { return type == kFloat32 || type == kFloat16 || type == kBfloat16; }

struct QuantizeParams {
  const void *in;
  void *out, *scales;        // [batch][m][scaled_pitch(n)], [batch][ceil(n / 128)][scaled_pitch(scale rows of m)]; may be null
  void *out_t, *scales_t;    // the same of the transposes: may be null
  unsigned batch, m, n;
  size_t in_pitch;           // elements from row to row
  int type_in, type_out, group, scale_type;
};
hipError_t launch_quantize(const QuantizeParams &p, hipStream_t stream);

// What a product of given sizes runs as, and its workspace: partial sums (floats), and a counter for each block of C.
struct RealGemmPlan {
  int shape = 0;
  unsigned parts = 1, pieces_per_part = 0;
  size_t partial_bytes = 0, counter_bytes = 0;
};

// A block shape of the real products' kernel: columns and rows of a block, its threads, blocks that a compute unit holds, and what it costs
// (us): a piece of K where a unit has one block, and where every unit has as many as it holds; a block's start and end;
// joining parts of K, for each 64 x 64 sums.
struct RealShape {
  unsigned bx, by, threads, per_unit;
  float alone_us, full_us, block_us, join_us;
  const char *name;
};
// The option REAL_BLOCK: 0, or a shape's number + 1, plus 256 times the number of parts that K is cut into (0: chosen).
extern size_t real_block_option;

struct ScaledGemmParams {
  const void *a, *b, *scales_a, *scales_b;
  void *c;
  unsigned batch, m, n, k;
  size_t pitch_a, pitch_b, pitch_c;   // elements
  int type_a, type_b, type_c, group_a, group_b, scale_type;
  int accumulate;
  RealGemmPlan plan;
  unsigned *arrived;                  // the plan's counters, zero when a product starts (it leaves them so)
  float *partial;                     // the plan's partial sums
};
RealGemmPlan plan_scaled_gemm(const ScaledGemmParams &p);
hipError_t launch_scaled_gemm(const ScaledGemmParams &p, hipStream_t stream);
// Whether the plan is one that a launch takes.
bool scaled_gemm_launches(const ScaledGemmParams &p);
// Name of the kernel that the plan launches.
const char *describe_scaled_gemm(const ScaledGemmParams &p);

struct OrthogonalizeParams {
  const void *in;
  void *out;
  unsigned batch, m, n;               // of the input
  size_t in_pitch, out_pitch;
  int type;
  int steps;
  float a, b, c, epsilon;
  size_t block_option;                // REAL_BLOCK when the object was created
  void *workspace;
};
size_t orthogonalize_workspace_bytes(const OrthogonalizeParams &p);
// What of the workspace has to be zero before the first launch (from its start).
size_t orthogonalize_zeroed_bytes(const OrthogonalizeParams &p);
hipError_t launch_orthogonalize(const OrthogonalizeParams &p, hipStream_t stream);

}  // namespace ccglib_amd
#endif  // CCGLIB_AMD_SCALED_H_
