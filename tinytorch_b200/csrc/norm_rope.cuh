// Declarations of the norm and rotation of queries and keys (norm_rope.cu).
#pragma once
#include "../../include/tt_fused.h"
#include "common.cuh"

namespace ttattn {

constexpr int kMaxAxes = TT_ATTN_MAX_ROPE_AXES;

// [0]: q, [1]: k throughout
struct NormRopeArgs {
  const void* x[2];
  const void* dy[2];  // backward: the outputs' gradients
  void* y[2];         // forward: the outputs; backward: the inputs' gradients (or null)
  const void* w[2];   // [D], or null: not normalised
  void* dw[2];        // backward: [D], or null
  float* part;        // backward: workspace [CTAs][D] for shares of dw, or null
  Str3 xs[2], dys[2], ys[2];
  int heads[2];
  int B, S;
  float eps;
  const float* cos;  // [rope_positions, D/2], or null: no rotation
  const float* sin;
  int rope_positions;
  bool interleaved;
  const int32_t* positions;  // [axes][B or 1][S]
  int64_t pos_axis, pos_b;   // element strides
  int axes;
  int axis_end[kMaxAxes];    // the first pair behind an axis's section
  int32_t* status;
  int split[2], ctas[2];     // set by the launcher: warps to a token (forward), CTAs
};

cudaError_t launch_norm_rope(int dtype, int D, const NormRopeArgs& a, int device, cudaStream_t stream);
cudaError_t launch_norm_rope_bwd(int dtype, int D, const NormRopeArgs& a, int device, cudaStream_t stream);
// CTAs of the backward, each of which takes D floats of workspace where a dw is asked for
void norm_rope_bwd_ctas(int B, int S, const int (&heads)[2], int (&ctas)[2]);

}  // namespace ttattn
