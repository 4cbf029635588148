// The plan of an attention call over packed sequences, made on the device because the lengths are there.
//
// The attention kernels take a sequence's tiles through tensor maps of its own: copies of the whole tensors' maps
// whose base is the sequence's first row and whose extent is its length.  Loads behind the end then read zeros, never the next
// sequence's rows (which may hold infinities), and stores and reductions behind it are dropped, so that nothing in the kernels'
// loops knows of packing.  CTA 0 sorts the work items, the longest walks first, so that the CTAs of the attention kernel finish
// together; the other CTAs make the maps, a warp each, and clear the rows behind the last sequence.
#include "packed.cuh"

#include "ptx.cuh"

namespace ttattn {
namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32, kLevels = 4096, kTile = 128;

struct Seq {
  int q0, lq, k0, lk;
};
__device__ __forceinline__ Seq load_seq(const PackedPlan& p, int s) {
  const int q0 = p.cu_q[s], k0 = p.cu_k[s];
  return Seq{q0, p.cu_q[s + 1] - q0, k0, p.cu_k[s + 1] - k0};
}

// Items of a sequence, and the tiles that item i walks over.
__device__ __forceinline__ int items_of(const PackedPlan& p, const Seq& s) {
  if (p.bwd) return (s.lk + kTile - 1) / kTile;
  return ((s.lq + kTile - 1) / kTile * p.group + p.step - 1) / p.step;
}
__device__ __forceinline__ int walk_of(const PackedPlan& p, const Seq& s, int i) {  // (query tiles of one head; key tiles of the longer of a pair)
  const int shift = causal_shift(p.causal, s.lk, s.lq);
  if (p.bwd) {
    const int nq = (s.lq + kTile - 1) / kTile, first = i * kTile - shift;
    const int from = p.causal && first > 0 ? first / kTile : 0;
    return from < nq ? nq - from : 0;
  }
  const int nq = (s.lq + kTile - 1) / kTile, last = (i * p.step + p.step - 1) / p.group;
  int end = s.lk;
  if (p.causal) {
    const int seen = ((last < nq ? last : nq - 1) + 1) * kTile + shift;
    end = seen < 0 ? 0 : (seen < end ? seen : end);
  }
  return (end + kTile - 1) / kTile;
}

__global__ void __launch_bounds__(kThreads) packed_plan_kernel(const __grid_constant__ PackedPlan p) {
  __shared__ int s_level[kLevels];  // items of a level; then where its next one goes
  __shared__ int s_warp_sum[kWarps];
  __shared__ __align__(128) uint32_t s_map[kWarps][32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();

  // Offsets that fall, or lie outside the rows, would let sequences share rows: then there are no items, and every row is cleared.
  bool falls = false;
  for (int i = tid; i <= p.n; i += kThreads) {
    const int q = p.cu_q[i], k = p.cu_k[i];
    falls |= q < 0 || q > p.total_q || k < 0 || k > p.total_k;
    if (i < p.n) falls |= p.cu_q[i + 1] < q || p.cu_k[i + 1] < k;
  }
  const bool bad = __syncthreads_or(falls) != 0;

  if (blockIdx.x > 0) {
    const int64_t first = (static_cast<int64_t>(blockIdx.x) - 1) * kWarps + warp, step = (static_cast<int64_t>(gridDim.x) - 1) * kWarps;
    for (int64_t i = first; i < static_cast<int64_t>(p.n) * p.n_maps && !bad; i += step) {
      const int s = static_cast<int>(i / p.n_maps), m = static_cast<int>(i - static_cast<int64_t>(s) * p.n_maps);
      const Seq q = load_seq(p, s);
      const int row = p.of_k[m] ? q.k0 : q.q0, rows = p.of_k[m] ? q.lk : q.lq;
      if (rows <= 0) continue;
      s_map[warp][lane] = reinterpret_cast<const uint32_t*>(&p.base[m])[lane];
      __syncwarp();
      if (lane == 0) {
        const uint32_t at = ptx::smem_u32(s_map[warp]);
        ptx::tensormap_set_address(at, p.address[m] + row * p.row_bytes[m]);
        ptx::tensormap_set_extent<1>(at, static_cast<uint32_t>(rows));
      }
      __syncwarp();
      ptx::tensormap_release(p.maps + i, ptx::smem_u32(s_map[warp]));
      __syncwarp();
    }
    // rows in front of the first sequence and behind the last
    for (int z = 0; z < p.n_zero; ++z) {
      const PackedPlan::Rows& r = p.zero[z];
      const int total = r.of_k ? p.total_k : p.total_q;
      const int32_t* cu = r.of_k ? p.cu_k : p.cu_q;
      const int head = bad ? 0 : cu[0], tail = bad ? 0 : cu[p.n];
      const int64_t n = static_cast<int64_t>(head + total - tail) * r.heads;
      for (int64_t i = first; i < n; i += step) {
        int row = static_cast<int>(i / r.heads);
        const int h = static_cast<int>(i - static_cast<int64_t>(row) * r.heads);
        if (row >= head) row += tail - head;
        char* at = r.ptr + row * r.row_bytes + h * r.head_bytes;
        for (int b = lane * 16; b < r.bytes; b += 512) *reinterpret_cast<uint4*>(at + b) = make_uint4(0, 0, 0, 0);
        if (z == 0 && p.lse && lane == 0) p.lse[static_cast<int64_t>(h) * p.total_q + row] = -INFINITY;
      }
    }
    return;
  }

  // ------------------------------------------------------------------ the items --
  if (p.sched && tid == 0) *p.sched = 0;
  if (bad) {
    if (tid == 0) *p.n_items = 0;
    if (tid == 0 && p.status) atomicOr(p.status, kStatusBadOffsets);
    return;
  }
  for (int i = tid; i < kLevels; i += kThreads) s_level[i] = 0;
  __syncthreads();
  // With few sequences several warps share one.
  int per = 1;
  while (per < kWarps && p.n * per * 2 <= kWarps) per *= 2;
  const int mine = warp / per, teams = kWarps / per, id = (warp % per) * 32 + lane, width = per * 32;
  for (int s = mine; s < p.n; s += teams) {
    const Seq q = load_seq(p, s);
    const int n = items_of(p, q);
    for (int i = id; i < n; i += width) atomicAdd(&s_level[walk_of(p, q, i) >> p.shift], 1);
  }
  __syncthreads();
  // places of the levels, the highest first: thread t has four of them
  constexpr int kMine = kLevels / kThreads;
  int count[kMine], sum = 0;
#pragma unroll
  for (int i = 0; i < kMine; ++i) count[i] = s_level[kLevels - 1 - (tid * kMine + i)], sum += count[i];
  int upto = sum;
#pragma unroll
  for (int of = 1; of < 32; of <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, upto, of);
    if (lane >= of) upto += o;
  }
  if (lane == 31) s_warp_sum[warp] = upto;
  __syncthreads();
  if (warp == 0) {
    int w = s_warp_sum[lane];
#pragma unroll
    for (int of = 1; of < 32; of <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, w, of);
      if (lane >= of) w += o;
    }
    s_warp_sum[lane] = w;
    if (lane == 31) *p.n_items = w;
  }
  __syncthreads();
  int place = upto - sum + (warp > 0 ? s_warp_sum[warp - 1] : 0);
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    s_level[kLevels - 1 - (tid * kMine + i)] = place;
    place += count[i];
  }
  __syncthreads();
  for (int s = mine; s < p.n; s += teams) {
    const Seq q = load_seq(p, s);
    const int n = items_of(p, q);
    for (int i = id; i < n; i += width) {
      const int walk = walk_of(p, q, i);
      const int at = atomicAdd(&s_level[walk >> p.shift], 1);
      reinterpret_cast<int4*>(p.items + at)[0] = make_int4(q.q0, q.lq, q.k0, q.lk);
      reinterpret_cast<int4*>(p.items + at)[1] = make_int4(p.bwd ? i : i * p.step, s, walk, 0);
    }
  }
}

constexpr size_t round256(size_t n) { return (n + 255) & ~size_t(255); }

}  // namespace

// Every sequence has at most one item more than its rows fill.
size_t packed_items(int n, int total, int group, int step) {
  return (static_cast<size_t>(total) / kTile + n) * group / step + n + 1;
}

static size_t items_bytes(int n, int total_q, int total_k, int group, bool bwd) {
  return round256(sizeof(PackedEntry) * (bwd ? packed_items(n, total_k, 1, 1) : packed_items(n, total_q, group, 1)));
}

size_t packed_plan_bytes(int n, int total_q, int total_k, int group, bool bwd) {
  return 256 + items_bytes(n, total_q, total_k, group, bwd) +
         round256(sizeof(CUtensorMap) * static_cast<size_t>(n) * (bwd ? kPackedBwdMaps : kPackedFwdMaps));
}

cudaError_t launch_packed_plan(PackedPlan p, void* scratch, PackedArgs* args, cudaStream_t stream) {
  char* at = static_cast<char*>(scratch);
  p.n_items = reinterpret_cast<int*>(at);
  p.items = reinterpret_cast<PackedEntry*>(at + 256);
  p.maps = reinterpret_cast<CUtensorMap*>(at + 256 + items_bytes(p.n, p.total_q, p.total_k, p.group, p.bwd));
  p.shift = 0;
  while ((((p.bwd ? p.total_q : p.total_k) + kTile - 1) / kTile >> p.shift) >= kLevels) ++p.shift;
  *args = PackedArgs{p.items, p.n_items, p.maps};
  const int64_t warps = static_cast<int64_t>(p.n) * p.n_maps + (p.total_q + p.total_k) / 64;
  const int64_t most = 2 * kSms, ctas = (warps + kWarps - 1) / kWarps;
  return launch_early(packed_plan_kernel, dim3(1 + static_cast<unsigned>(ctas < 1 ? 1 : (ctas < most ? ctas : most))), dim3(kThreads), 0, stream, 1, p);
}

}  // namespace ttattn
