// Parameter blocks of the 16-bit linear layers (FusedLinear, and GroupedLinear with a weight matrix for each group of
// rows), handed from the C ABI layer (linear_capi.hip) to the kernel launchers.
#ifndef CCGLIB_AMD_LINEAR_H_
#define CCGLIB_AMD_LINEAR_H_

#include "scaled.h"

namespace ccglib_amd {

enum : int { kNone = 0, kRelu = 1, kGelu = 2, kSilu = 3 };

namespace linear {

// The products of a layer (linear_gemm.h)
enum Kind : int { kOutput = 0, kInput = 1, kWeights = 2 };

}  // namespace linear

struct LinearParams {
  unsigned m, n, k;                    // rows, outputs, inputs
  unsigned groups;                     // weight matrices
  bool grouped, training;
  int type, gradient_type, activation;
  size_t x_pitch, w_pitch, y_pitch;    // elements from row to row: of x and dx; W and dW; y, z, residual, dy
  RealGemmPlan plan[3];                // by Kind
  bool few_rows;                       // y is linear_rows.hip's, else gemm_linear's
  bool together;                       // dx and dW in one launch, where both are wanted
  // the workspace, and where in it (bytes): counters first, which are zero whenever a product starts; products that run one after the other
  // share theirs
  char *workspace;
  size_t zeroed, counters[3], partial[3], dz, sums, tails, bytes;
};

// Fills in the plans and the workspace's layout.
void plan_linear(LinearParams *p);
// Whether all products are launches that the runtime takes.
bool linear_launches(const LinearParams &p);
const char *describe_linear(const LinearParams &p, int kind);

struct LinearForward {
  const void *x, *w, *bias, *residual;
  const int *offsets;
  void *y, *z;
};
struct LinearBackward {
  const void *dy, *z, *x, *w;
  const int *offsets;
  void *dx, *dw, *dbias;
  bool accumulate;
};
hipError_t launch_linear_forward(const LinearParams &p, const LinearForward &f, hipStream_t stream);
hipError_t launch_linear_backward(const LinearParams &p, const LinearBackward &b, hipStream_t stream);

}  // namespace ccglib_amd
#endif  // CCGLIB_AMD_LINEAR_H_
