// Parameter blocks of the routing operators (Route: which k of E experts a row goes to, with what weights, and where; Combine: rows
// spread to those places and summed back), handed from the C ABI layer (linear_capi.hip) to the kernel launchers.
#ifndef CCGLIB_AMD_ROUTE_H_
#define CCGLIB_AMD_ROUTE_H_

#include "common.h"

namespace ccglib_amd {

constexpr size_t kMostExperts = 1024, kMostChosen = 16;

struct RouteParams {
  unsigned tokens, experts, chosen;
  int type;
  bool normalize;
  unsigned tile, tiles;          // tokens that a block counts, how many such blocks there are (1 at least)
  unsigned short *counts;        // [tiles][experts, in whole quads]; null where there is one tile
};
void plan_route(RouteParams *p);
size_t route_workspace_bytes(const RouteParams &p);
hipError_t launch_route(const RouteParams &p, const void *logits, int *experts, float *weights, int *offsets, int *slots,
                        hipStream_t stream);
hipError_t launch_route_backward(const RouteParams &p, const void *logits, const int *experts, const float *weights,
                                 const float *dweights, void *dlogits, hipStream_t stream);

struct CombineParams {
  unsigned tokens, chosen, n, rows;   // rows of y: slots are smaller
  int type;
  size_t y_pitch, out_pitch;          // elements from row to row
};
hipError_t launch_combine(const CombineParams &p, const void *y, const int *slots, const float *weights, void *out, hipStream_t stream);
// y null: dweights is not wanted
hipError_t launch_combine_backward(const CombineParams &p, const void *dout, const void *y, const int *slots, const float *weights,
                                   void *dy, float *dweights, hipStream_t stream);

}  // namespace ccglib_amd
#endif  // CCGLIB_AMD_ROUTE_H_
