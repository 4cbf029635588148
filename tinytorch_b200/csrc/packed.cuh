// Packed sequences: what the planning kernel (packed_plan.cu) is asked for by the forward's and the backward's launcher.
#pragma once
#include <cuda.h>

#include "common.cuh"

namespace ttattn {

struct PackedPlan {
  const int32_t* cu_q;  // [n + 1] device
  const int32_t* cu_k;
  int n, total_q, total_k;
  int group, causal;
  uint64_t per_group;   // ceil(2^40 / group)
  // items: of the forward 1 << step_log query blocks (128 rows of one head of a group); of the backward a key tile of 128
  bool bwd;
  int step_log;
  int width_log;        // threads to a sequence
  int shift, levels;    // of the sort: key tiles (backward: steps) of a walk >> shift
  int kv_heads, slots;  // backward: places for shares of dK / dV, per kv head (0: no walk is divided)
  PackedEntry* items;
  PackedSplit* splits;
  int* n_items;         // [0] items, [1] divided key tiles
  int* sched;           // set to zero, or null
  int32_t* status;
  // tensor maps (see PackedMaps): from how many rows on a sequence takes those of the whole tensors; which go along with k; rows are dimension 1
  int long_rows[kPackedBwdMaps];
  const char* address[kPackedBwdMaps];
  int64_t row_bytes[kPackedBwdMaps];
  bool of_k[kPackedBwdMaps];
  int n_maps;
  // Sequences of up to `narrow` rows (forward: and keys; 0: none) have maps of their own, where there are such, whose boxes are so many rows of several
  // heads; forward: items of their own, so many; backward: so many steps for a query tile of all heads of a group
  int narrow, narrow_items;
  bool has_narrow[kPackedBwdMaps];
  CUtensorMap* maps;
  // rows behind the last sequence: zeros in these (of 16-byte multiples), and -inf in lse
  struct Rows {
    char* ptr;
    int64_t row_bytes, head_bytes;
    int heads, bytes;  // bytes of a row of one head
    bool of_k;
  } zero[3];
  int n_zero;
  float* lse;  // [heads of zero[0]][total_q]
};

// What sequences' maps are made of: the maps of the whole tensors and of one row, and those two with narrow boxes.
struct PackedMaps {
  CUtensorMap kind[4][kPackedBwdMaps];
  struct Layout {  // of those whose long_rows the driver has been asked for
    int rows, heads;
    int64_t row_stride, head_stride;
  } layout[kPackedBwdMaps] = {};
};

// A call over packed sequences.
struct PackedCall {
  const int32_t* cu_q;
  const int32_t* cu_k;
  int n, total_k;
  void* scratch;  // packed_plan_bytes
  float* shares;  // backward: [dK, dV][Hkv * slots][128][D], or null
};

// Upper bounds of what a plan takes in scratch memory.
size_t packed_items(int n, int total, int group, int step);
size_t packed_plan_bytes(int n, int total_q, int total_k, int group, bool bwd);
// Backward: the places that shares of divided walks take at most, per kv head.
int packed_slots(int n, int total_q, int total_k, int Hq, int Hkv);

// Adds the map of an operand [rows][H][D] (fp32: dense [H][rows][D]).
// narrow_heads: also one with boxes of p->narrow rows of so many heads.
cudaError_t packed_map(PackedPlan* p, PackedMaps* maps, int dtype, const void* ptr, int D, int rows, int H, const Str3& st, int box_rows, bool of_k, int narrow_heads = 0);

// Fills in items, maps and args from `scratch` and enqueues the planning kernel.
cudaError_t launch_packed_plan(PackedPlan p, const PackedMaps& maps, void* scratch, PackedArgs* args, cudaStream_t stream);

// The forward and the backward; a's B is 1, its Lq and Skv are the rows of all sequences.
cudaError_t launch_fwd_packed(int dtype, int D, const FwdArgs& a, const PackedCall& c, int device, cudaStream_t stream);
cudaError_t launch_bwd_packed(int dtype, int D, const BwdArgs& a, const PackedCall& c, int device, cudaStream_t stream);

}  // namespace ttattn
