// The keys and values of accepted drafts, copied behind the valid rows of a cache.
//
// A copy of a few rows for each sequence: launch-bound (64 sequences, up to 12 rows of 8 heads, D = 128: 4.7 us).  Every warp finds for itself how many rows its sequence takes (the first draft that
// does not exist, or the first row that the cache has no room for, ends the path), so that no other kernel has to say so first.
#include "tree.cuh"

#include "ptx.cuh"

namespace ttattn {
namespace {

constexpr int kThreads = 256;

__global__ void __launch_bounds__(kThreads) cache_accept_kernel(const AcceptArgs a, int row_vectors, int elem) {
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const int b = blockIdx.y, lane = threadIdx.x & 31;
  const int32_t* path = a.path + static_cast<int64_t>(b) * a.N;
  int len = a.kv_lens[b];
  len = len < 0 ? 0 : (len < a.capacity ? len : a.capacity);
  int n = a.counts[b], wrong = n < 0 || n > a.N ? kStatusBadOffsets : 0;
  n = n < 0 ? 0 : (n < a.N ? n : a.N);
  for (int base = 0; base < n; base += 32) {
    const int i = base + lane;
    const int p = i < n ? path[i] : 0;
    const uint32_t bad = __ballot_sync(0xffffffffu, p < 0 || p >= a.T);
    if (bad) n = base + __ffs(bad) - 1, wrong |= kStatusBadOffsets;
  }
  if (n > a.capacity - len) n = a.capacity - len, wrong |= kStatusCacheFull;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.new_lens[b] = len + n;
    if (wrong && a.status) atomicOr(a.status, wrong);
  }
  // 16-byte vectors: of K and V, heads, rows of the path
  const int per = n * row_vectors, total = 2 * a.Hkv * per;
  for (int i = blockIdx.x * kThreads + threadIdx.x; i < total; i += gridDim.x * kThreads) {
    const int th = i / per, rest = i - th * per, row = rest / row_vectors, vec = rest - row * row_vectors;
    const bool v = th >= a.Hkv;
    const int h = v ? th - a.Hkv : th;
    const Str3 &from = v ? a.vds : a.kds, &to = v ? a.vcs : a.kcs;
    const char* src = static_cast<const char*>(v ? a.vd : a.kd) + (b * from.b + h * from.h + path[row] * from.s) * elem + vec * 16;
    char* dst = static_cast<char*>(v ? a.vc : a.kc) + (b * to.b + h * to.h + static_cast<int64_t>(len + row) * to.s) * elem + vec * 16;
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
  }
}

}  // namespace

cudaError_t launch_cache_accept(int dtype, int D, const AcceptArgs& a, cudaStream_t stream) {
  const int elem = dtype == TT_ATTN_F32 ? 4 : 2, row_vectors = D * elem / 16;
  const int64_t most = 2ll * a.Hkv * a.N * row_vectors, ctas = (most + kThreads - 1) / kThreads;
  return launch_early(cache_accept_kernel, dim3(static_cast<unsigned>(ctas < 1 ? 1 : (ctas < 64 ? ctas : 64)), a.B), dim3(kThreads), 0, stream, 1, a, row_vectors, elem);
}

}  // namespace ttattn
