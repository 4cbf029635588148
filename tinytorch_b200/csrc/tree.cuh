// Attention of drafted tokens, arranged in a tree, over a KV cache: what the kernels for 16-bit tensors (tree_tc.cu) and for fp32
// (tree_f32.cu) share.
//
// The rows of one (sequence, kv head) are its T drafts times the G query heads of the group, row t * G + g, in blocks of whole
// drafts.  Their keys are the tiles of the cache's valid rows, then those of the drafts themselves, of which a row sees what
// the mask says.  All tiles of all (sequence, kv head, block) stand in one line, the end of each walk counting
// for some more, and every CTA takes an equal piece of it: the whole machine reads to the end whatever the lengths are, and a
// walk is broken only where a piece ends.  A broken walk leaves unnormalised
// sums, maxima and weights in scratch memory, two at most to a CTA (one that it goes on with, one that it leaves to others),
// and a second kernel puts them together in order.
#pragma once
#include "common.cuh"

namespace ttattn {

struct TreeArgs {
  const void* q;   // [B, Hq, T, D]
  const void* kd;  // [B, Hkv, T, D]
  const void* vd;
  const void* kc;  // [B, Hkv, capacity, D]
  const void* vc;
  void* o;         // [B, Hq, T, D]
  float* lse;      // [B, Hq, T] or null
  Str3 qs, kds, vds, kcs, vcs, os;
  int B, Hq, Hkv, T, capacity;
  float scale;
  const int32_t* kv_lens;  // [B], or null: every row of the cache is valid
  const uint8_t* mask;     // [B or 1, T, T], non-zero: row (draft) sees column (draft); null: a chain
  int64_t mask_b, mask_t;
  int32_t* status;
  int block, n_blocks;  // drafts of a block, blocks
  int least;            // tiles of a CTA's piece, about, at least
  int ends;             // what the end of a walk counts for in the line, in tiles
  float* partial;       // [CTAs][2] of tree_partial_floats
  int4* pieces;         // [CTAs]: pieces of the walk that begins in this CTA and goes on, sequence, kv head, block
};

constexpr int kTreeRows = 128;  // rows of a partial result

// One partial result: [D / 4][rows][4] sums, then (maximum, in log2 units, and weight) of each row.
__host__ __device__ constexpr size_t tree_partial_floats(int D) { return static_cast<size_t>(kTreeRows) * (D + 2); }

// A CTA's part of one walk: tiles [j0, j0 + n) of n_all, the first n_ctx of which are the cache's.
struct TreeSegment {
  int b, hk, block, j0, n, n_all, n_ctx, len;
  int at;     // where it begins in the line
  int piece;  // the CTA's first, if it goes on with a walk (0), or the last, if it leaves one (1); -1: whole
};

template <int KT>
__device__ __forceinline__ int tree_tiles(const TreeArgs& a, int b, int* len) {
  int l = a.capacity;
  if (a.kv_lens) {
    l = a.kv_lens[b];
    l = l < 0 ? 0 : (l < a.capacity ? l : a.capacity);
  }
  *len = l;
  return (l + KT - 1) / KT + (a.T + KT - 1) / KT;
}

// Where a CTA's piece begins and ends in the line.
struct TreeWalk {
  int at, end;       // tiles of the line
  int line, ctas;    // tiles of the line; CTAs that have a piece
  int b, unit, j;    // the sequence, (kv head, block) and tile of `at`
  int n_all, len;

  // By all THREADS threads of the CTA, with THREADS / 32 + 2 integers of shared memory; the launch has as many CTAs as scratch
  // was planned for.
  template <int KT, int THREADS>
  __device__ void start(const TreeArgs& a, int* s_sum) {
    constexpr int kW = THREADS / 32;
    int* s_found = s_sum + kW;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, units = a.Hkv * a.n_blocks;
    // totals up to every sequence: in one go where there are no more sequences than threads
    int total = 0, l, upto = 0, n = 0;
    auto scan = [&](int base) {  // of the sequences base ...: `n` and `upto` of this thread's, and what all of them come to
      n = base + tid < a.B ? tree_tiles<KT>(a, base + tid, &l) + a.ends : 0;
      upto = n;
#pragma unroll
      for (int of = 1; of < 32; of <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, upto, of);
        if (lane >= of) upto += o;
      }
      __syncthreads();
      if (lane == 31) s_sum[warp] = upto;
      __syncthreads();
      int all = 0;
#pragma unroll
      for (int w = 0; w < kW; ++w) {
        const int x = s_sum[w];
        if (w < warp) upto += x;
        all += x;
      }
      return all;
    };
    for (int base = 0; base < a.B; base += THREADS) total += scan(base);
    line = total * units;  // (the launcher has seen to it that it fits 32 bits)
    ctas = line / a.least < static_cast<int>(gridDim.x) ? line / a.least + 1 : gridDim.x;
    const int me = static_cast<int>(blockIdx.x) < ctas ? blockIdx.x : ctas;
    at = static_cast<int>(static_cast<int64_t>(line) * me / ctas);
    end = me < ctas ? static_cast<int>(static_cast<int64_t>(line) * (me + 1) / ctas) : at;
    int before = 0;
    for (int base = 0; base < a.B; base += THREADS) {
      const int all = a.B > THREADS ? scan(base) : total;
      const int lo = (before + upto - n) * units, hi = (before + upto) * units;
      if (at >= lo && at < hi) s_found[0] = base + tid, s_found[1] = lo;
      before += all;
      if (at < before * units) break;  // (the same for every thread)
    }
    __syncthreads();
    b = unit = j = n_all = len = 0;
    if (at < end) {
      b = s_found[0];
      n_all = tree_tiles<KT>(a, b, &len);
      const int off = at - s_found[1];
      unit = off / (n_all + a.ends), j = off - unit * (n_all + a.ends);
    }
  }

  // The next part of a walk, or false.
  template <int KT>
  __device__ bool next(const TreeArgs& a, TreeSegment* s) {
    if (j >= n_all) {  // (the piece begins in the end of a walk)
      at += n_all + a.ends - j;
      advance<KT>(a);
    }
    if (at >= end) return false;
    s->b = b, s->hk = unit / a.n_blocks, s->block = unit - s->hk * a.n_blocks;
    s->j0 = j, s->n_all = n_all, s->len = len, s->n_ctx = (len + KT - 1) / KT;
    s->at = at;
    const int left = n_all - j, room = end - at;
    s->n = left < room ? left : room;
    s->piece = j > 0 ? 0 : (s->n < n_all ? 1 : -1);
    at += s->n + (s->n == left ? a.ends : 0);
    advance<KT>(a);
    return true;
  }
  template <int KT>
  __device__ void advance(const TreeArgs& a) {
    j = 0;
    if (++unit == a.Hkv * a.n_blocks) {
      unit = 0;
      if (++b < a.B) n_all = tree_tiles<KT>(a, b, &len);
    }
  }

  // CTAs that the walk takes which begins with this segment
  __device__ int pieces(const TreeSegment& s) const {
    return static_cast<int>((static_cast<int64_t>(s.at + s.n_all) * ctas - 1) / line) - static_cast<int>(blockIdx.x) + 1;
  }
};

// What draft t sees of the drafts: bit j of words[j / 32].
template <int WORDS>
__device__ __forceinline__ void tree_mask_row(const TreeArgs& a, int b, int t, uint32_t (&words)[WORDS]) {
  if (!a.mask) {
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
      const int n = t + 1 - w * 32;  // a chain: every draft up to itself
      words[w] = n >= 32 ? 0xffffffffu : (n > 0 ? (1u << n) - 1 : 0u);
    }
    return;
  }
  // the aligned vectors that hold the row, four bytes to four bits, shifted into place
  const uint8_t* row = a.mask + b * a.mask_b + t * a.mask_t;
  const int lead = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15);
  const uint4* p = reinterpret_cast<const uint4*>(row - lead);
  const int n_vec = (lead + a.T + 15) / 16;
  uint32_t raw[WORDS + 1];
#pragma unroll
  for (int w = 0; w < WORDS + 1; ++w) raw[w] = 0;
#pragma unroll
  for (int i = 0; i < WORDS * 2 + 1; ++i) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (i < n_vec) v = p[i];
    const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t set = ((((x[e] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | x[e]) >> 7) & 0x01010101u;
      raw[i / 2] |= ((set * 0x01020408u) >> 24) << ((i & 1) * 16 + e * 4);
    }
  }
#pragma unroll
  for (int w = 0; w < WORDS; ++w) {
    const int n = a.T - w * 32;
    words[w] = __funnelshift_r(raw[w], raw[w + 1], lead) & (n >= 32 ? 0xffffffffu : (n > 0 ? (1u << n) - 1 : 0u));
  }
}

// The plan, shared with the workspace query: drafts of a block, blocks; CTAs, each with two partial results.
void tree_plan(int dtype, int Hq, int Hkv, int T, int* block, int* n_blocks);
int tree_ctas(int dtype, int B, int Hq, int Hkv, int T, int capacity, int D);
size_t tree_scratch_bytes(int dtype, int B, int Hq, int Hkv, int T, int capacity, int D);
// longest line that a call can have; the launchers take up to 2^31 - 1
double tree_line(int dtype, int B, int Hq, int Hkv, int T, int capacity, int D);

cudaError_t launch_tree(int dtype, int D, TreeArgs a, void* scratch, int device, cudaStream_t stream);
cudaError_t launch_tree_tc(int dtype, int D, const TreeArgs& a, int ctas, cudaStream_t stream);
cudaError_t launch_tree_f32(int D, const TreeArgs& a, int ctas, cudaStream_t stream);

// Rows of accepted drafts behind the valid rows of a cache (cache_accept.cu).
struct AcceptArgs {
  const void* kd;  // [B, Hkv, T, D]
  const void* vd;
  void* kc;        // [B, Hkv, capacity, D]
  void* vc;
  Str3 kds, vds, kcs, vcs;
  int B, Hkv, T, capacity, N;
  const int32_t* kv_lens;  // [B]
  const int32_t* path;     // [B, N]
  const int32_t* counts;   // [B]
  int32_t* new_lens;       // [B]
  int32_t* status;
};
cudaError_t launch_cache_accept(int dtype, int D, const AcceptArgs& a, cudaStream_t stream);

}  // namespace ttattn
