// Drafted tokens over a KV cache: the fp32 kernel, the kernel that puts broken walks together, and the plan (see tree.cuh).
//
// fp32 has no tensor-core product of its own precision, so products are FMAs from shared memory: a CTA, one of two on an SM, holds a block of
// R = 8 or 32 rows and walks over tiles of 4096 / D keys (cp.async, a tile or two ahead, on into the next walk).  With 8 rows a tile's arithmetic is
// less than the time its keys take to arrive, with 32 rows, whose loads from shared memory set the pace, about twice that; more rows are more
// blocks, which find the keys in L2.  4 sequences of 500 to 1003 rows, 5 drafts, 16 heads, D = 64: 17.3 us, of which the keys' bytes take 4: each CTA's few tiles
// follow one another (with one CTA to an SM 1.2 more).
#include <type_traits>

#include "ptx.cuh"
#include "tma_host.cuh"
#include "tree.cuh"

namespace ttattn {
namespace {

constexpr int kThreads = 256;

template <int D, int R>
struct Cfg {
  static constexpr int KT = 4096 / D;                            // keys of a tile
  static constexpr int kStages = R == 8 ? 3 : 2;
  static constexpr int kPitch = D + 4, kPPitch = KT + 4;         // floats; rows of other lanes then lie in other banks
  static constexpr int kTile = KT * kPitch, kGroups = kThreads / KT;  // threads to a key: of R / kGroups rows each
  static constexpr int oQ = 2 * kStages * kTile, oP = oQ + kStages * R * kPitch, oSees = oP + R * kPPitch, oM = oSees + R * 4, oL = oM + R, oAlpha = oL + R,
                       oScratch = oAlpha + R;
  static constexpr int kSmem = (oScratch + kThreads / 32 + 2) * 4;
  static_assert(2 * (kSmem + 1024) <= 233472, "two CTAs must fit the shared memory of an SM");
};

template <int D, int R>
__global__ void __launch_bounds__(kThreads, 2) tree_f32_kernel(const TreeArgs a) {
  using C = Cfg<D, R>;
  constexpr int KT = C::KT, kPitch = C::kPitch, kPPitch = C::kPPitch, kStages = C::kStages;
  extern __shared__ __align__(16) float fsmem[];
  float *sK = fsmem, *sV = fsmem + kStages * C::kTile, *sP = fsmem + C::oP;
  uint32_t* sSees = reinterpret_cast<uint32_t*>(fsmem + C::oSees);
  float *sM = fsmem + C::oM, *sL = fsmem + C::oL, *sAlpha = fsmem + C::oAlpha;
  const int tid = threadIdx.x, group = a.Hq / a.Hkv;
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  TreeWalk walk;
  walk.start<KT, kThreads>(a, reinterpret_cast<int*>(fsmem + C::oScratch));
  if (tid == 0) a.pieces[blockIdx.x] = make_int4(0, 0, 0, 0);
  const float c = a.scale * kLog2e;
  // keys of a tile that exist; the others are zeros, whatever the cache holds there
  auto keys_of = [&](const TreeSegment& s, int tile) { return tile < s.n_ctx ? s.len - tile * KT : a.T - (tile - s.n_ctx) * KT; };
  auto rows_of = [&](const TreeSegment& s) {
    const int left = a.T - s.block * a.block;
    return (left < a.block ? left : a.block) * group;
  };
  // tile j of a segment to stage st; with the first one its rows of Q to buffer qb (of as many as there are stages: a segment may have one tile)
  auto load = [&](const TreeSegment& s, int j, int st, int qb) {
    const int tile = s.j0 + j, keys = keys_of(s, tile);
    const bool ctx = tile < s.n_ctx;
    const int row0 = (ctx ? tile : tile - s.n_ctx) * KT;
    const int64_t ks = ctx ? a.kcs.s : a.kds.s, vs = ctx ? a.vcs.s : a.vds.s;
    const float* k = ctx ? reinterpret_cast<const float*>(a.kc) + s.b * a.kcs.b + s.hk * a.kcs.h : reinterpret_cast<const float*>(a.kd) + s.b * a.kds.b + s.hk * a.kds.h;
    const float* v = ctx ? reinterpret_cast<const float*>(a.vc) + s.b * a.vcs.b + s.hk * a.vcs.h : reinterpret_cast<const float*>(a.vd) + s.b * a.vds.b + s.hk * a.vds.h;
#pragma unroll
    for (int i = tid; i < KT * (D / 4); i += kThreads) {
      const int key = i / (D / 4), c4 = i % (D / 4), n = key < keys ? 16 : 0;
      const int64_t row = n ? row0 + key : 0;
      const uint32_t at = (st * C::kTile + key * kPitch + c4 * 4) * 4;
      ptx::cp_async16(ptx::smem_u32(sK) + at, k + row * ks + c4 * 4, n);
      ptx::cp_async16(ptx::smem_u32(sV) + at, v + row * vs + c4 * 4, n);
    }
    if (j == 0) {
      const int rows = rows_of(s);
      for (int i = tid; i < R * (D / 4); i += kThreads) {
        const int r = i / (D / 4), c4 = i % (D / 4), rr = r < rows ? r : 0;
        ptx::cp_async16(ptx::smem_u32(fsmem + C::oQ + (qb * R + r) * kPitch + c4 * 4),
                        reinterpret_cast<const float*>(a.q) + s.b * a.qs.b + (s.hk * group + rr % group) * a.qs.h +
                            static_cast<int64_t>(s.block * a.block + rr / group) * a.qs.s + c4 * 4,
                        r < rows ? 16 : 0);
      }
    }
  };
  // The tiles are asked for one or two ahead, over the ends of segments.
  TreeWalk walk_ahead = walk;
  TreeSegment s, sa;
  bool left = walk_ahead.next<KT>(a, &sa);
  int ja = 0, stage_ahead = 0, q_ahead = 0;
  auto ask = [&]() {
    if (left) {
      load(sa, ja, stage_ahead, q_ahead);
      stage_ahead = stage_ahead + 1 == kStages ? 0 : stage_ahead + 1;
      if (++ja == sa.n) {
        left = walk_ahead.next<KT>(a, &sa);
        ja = 0, q_ahead = q_ahead + 1 == kStages ? 0 : q_ahead + 1;
      }
    }
    ptx::cp_async_commit();
  };
#pragma unroll
  for (int j = 0; j < kStages - 1; ++j) ask();
  int st = 0;
  for (int qb = 0; walk.next<KT>(a, &s); qb = qb + 1 == kStages ? 0 : qb + 1) {
    if (tid == 0 && s.piece == 1) a.pieces[blockIdx.x] = make_int4(walk.pieces(s), s.b, s.hk, s.block);
    const int draft0 = s.block * a.block, rows = rows_of(s);
    const float* sQ = fsmem + C::oQ + qb * R * kPitch;
    __syncthreads();  // the segment before has been read
    if (tid < R) {
      uint32_t words[4] = {0, 0, 0, 0};
      if (tid < rows && s.j0 + s.n > s.n_ctx) tree_mask_row<4>(a, s.b, draft0 + tid / group, words);
#pragma unroll
      for (int w = 0; w < 4; ++w) sSees[tid * 4 + w] = words[w];
      sM[tid] = -INFINITY, sL[tid] = 0.f;
    }
    // sums: 4 channels of kMine rows
    constexpr int kRowSets = kThreads / (D / 4), kMine = R / kRowSets > 0 ? R / kRowSets : 1;
    const int c4 = tid % (D / 4), set = tid / (D / 4);
    float4 acc[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);

    for (int j = 0; j < s.n; ++j) {
      ptx::cp_async_wait_but<kStages - 2>();
      __syncthreads();  // tile j is there; tile j - 1 has been read
      ask();
      const int tile = s.j0 + j, keys = keys_of(s, tile);
      {  // scores of one key and kRows rows
        constexpr int kRows = R / C::kGroups;
        const int key = tid % KT, rg = tid / KT;
        const float* k = sK + st * C::kTile + key * kPitch;
        const float* q = sQ + rg * kRows * kPitch;
        float4 x[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int d = 0; d < D; d += 4) {
          const float4 kv = *reinterpret_cast<const float4*>(k + d);
#pragma unroll
          for (int i = 0; i < kRows; ++i) {
            const float4 qv = *reinterpret_cast<const float4*>(q + i * kPitch + d);
            x[i].x = fmaf(qv.x, kv.x, x[i].x), x[i].y = fmaf(qv.y, kv.y, x[i].y), x[i].z = fmaf(qv.z, kv.z, x[i].z), x[i].w = fmaf(qv.w, kv.w, x[i].w);
          }
        }
        const int draft = (tile - s.n_ctx) * KT + key;
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const int r = rg * kRows + i;
          const bool sees = key < keys && (tile < s.n_ctx || ((sSees[r * 4 + draft / 32] >> (draft % 32)) & 1));
          sP[r * kPPitch + key] = sees ? ((x[i].x + x[i].y) + (x[i].z + x[i].w)) * c : -INFINITY;
        }
      }
      __syncthreads();
      {  // softmax, kLanes neighbouring threads to a row
        constexpr int kLanes = kThreads / R < 32 ? kThreads / R : 32, kEach = KT / kLanes;
        const int r = tid / kLanes, at = tid % kLanes;
        float x[kEach], top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int i = 0; i < kEach; ++i) x[i] = sP[r * kPPitch + at + i * kLanes], top = fmaxf(top, x[i]);
#pragma unroll
        for (int of = kLanes / 2; of >= 1; of >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, of));
        const float m = sM[r], mn = fmaxf(m, top), use = mn == -INFINITY ? 0.f : mn;  // (nothing seen so far: exponentials of -inf)
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          x[i] = ptx::ex2(x[i] - use), sum += x[i];
          sP[r * kPPitch + at + i * kLanes] = x[i];
        }
#pragma unroll
        for (int of = kLanes / 2; of >= 1; of >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, of);
        __syncwarp();
        if (at == 0) {
          const float alpha = m == -INFINITY ? 0.f : ptx::ex2(m - mn);
          sM[r] = mn, sL[r] = fmaf(sL[r], alpha, sum), sAlpha[r] = alpha;
        }
      }
      __syncthreads();
      if (set * kMine < R) {
        const float* v = sV + st * C::kTile + c4 * 4;
        const float* p = sP + set * kMine * kPPitch;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          const float al = sAlpha[set * kMine + i];
          acc[i].x *= al, acc[i].y *= al, acc[i].z *= al, acc[i].w *= al;
        }
#pragma unroll 4
        for (int key = 0; key < KT; key += 4) {
          float4 vv[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) vv[e] = *reinterpret_cast<const float4*>(v + (key + e) * kPitch);
#pragma unroll
          for (int i = 0; i < kMine; ++i) {
            const float4 pv = *reinterpret_cast<const float4*>(p + i * kPPitch + key);
            const float pe[4] = {pv.x, pv.y, pv.z, pv.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              acc[i].x = fmaf(pe[e], vv[e].x, acc[i].x), acc[i].y = fmaf(pe[e], vv[e].y, acc[i].y);
              acc[i].z = fmaf(pe[e], vv[e].z, acc[i].z), acc[i].w = fmaf(pe[e], vv[e].w, acc[i].w);
            }
          }
        }
      }
      st = st + 1 == kStages ? 0 : st + 1;
    }
    float* part = a.partial + (static_cast<size_t>(blockIdx.x) * 2 + (s.piece > 0 ? 1 : 0)) * tree_partial_floats(D);
    if (set * kMine < R) {
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int r = set * kMine + i;
        if (r >= rows) break;
        if (s.piece >= 0) {
          *reinterpret_cast<float4*>(part + c4 * (kTreeRows * 4) + r * 4) = acc[i];
        } else {
          const float inv = inverse_sum(sL[r]);
          *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.o) + s.b * a.os.b + (s.hk * group + r % group) * a.os.h +
                                     static_cast<int64_t>(draft0 + r / group) * a.os.s + c4 * 4) =
              make_float4(acc[i].x * inv, acc[i].y * inv, acc[i].z * inv, acc[i].w * inv);
        }
      }
    }
    if (tid < rows) {
      const float l = sL[tid], m = sM[tid];
      if (s.piece >= 0)
        *reinterpret_cast<float2*>(part + kTreeRows * D + tid * 2) = make_float2(l == 0.f ? -INFINITY : m, l);
      else if (a.lse)
        a.lse[(static_cast<int64_t>(s.b) * a.Hq + s.hk * group + tid % group) * a.T + draft0 + tid / group] = row_lse(m, l);
    }
  }
  ptx::cp_async_wait();
}

// The walk that begins in piece blockIdx.x and goes on, if there is one: its partial results in the order of the pieces.  A thread has
// four channels of a row; neighbouring threads neighbouring rows.  (Only rows that a block has get threads: 5 rows of D = 64 by 296 CTAs, not 2368.)
template <typename T, int D>
__global__ void __launch_bounds__(256) tree_combine_kernel(const TreeArgs a) {
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const int4 w = a.pieces[blockIdx.x];
  if (w.x < 2) return;
  const int group = a.Hq / a.Hkv, draft0 = w.w * a.block, drafts = a.T - draft0 < a.block ? a.T - draft0 : a.block;
  const int rows = a.block * group, at = blockIdx.y * 256 + threadIdx.x, c4 = at / rows, r = at - c4 * rows;
  if (c4 >= D / 4 || r >= drafts * group) return;
  // the walk's first piece is the last of its CTA, the others the first of theirs
  const float* part = a.partial + static_cast<size_t>(blockIdx.x) * 2 * tree_partial_floats(D);
  auto piece = [&](int i) { return part + (i == 0 ? 1 : 2 * i) * tree_partial_floats(D); };
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int kBatch = 8;  // pieces whose loads are in flight together
  for (int i0 = 0; i0 < w.x; i0 += kBatch) {
    float2 ml[kBatch];
    float4 x[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      ml[i] = make_float2(-INFINITY, 0.f);
      if (i0 + i < w.x) {
        const float* p = piece(i0 + i);
        ml[i] = reinterpret_cast<const float2*>(p + kTreeRows * D)[r];
        x[i] = *reinterpret_cast<const float4*>(p + c4 * (kTreeRows * 4) + r * 4);
      }
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) top = fmaxf(top, ml[i].x);
    const float alpha = m == -INFINITY ? 0.f : ptx::ex2(m - top);
    l *= alpha, o.x *= alpha, o.y *= alpha, o.z *= alpha, o.w *= alpha, m = top;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (ml[i].y == 0.f) continue;  // (no piece, or one that has seen no key)
      const float f = ptx::ex2(ml[i].x - m);
      l = fmaf(ml[i].y, f, l);
      o.x = fmaf(x[i].x, f, o.x), o.y = fmaf(x[i].y, f, o.y), o.z = fmaf(x[i].z, f, o.z), o.w = fmaf(x[i].w, f, o.w);
    }
  }
  const float inv = inverse_sum(l);
  const int head = w.z * group + r % group, draft = draft0 + r / group;
  T* dst = reinterpret_cast<T*>(a.o) + w.y * a.os.b + head * a.os.h + static_cast<int64_t>(draft) * a.os.s + c4 * 4;
  if constexpr (std::is_same_v<T, float>) {
    *reinterpret_cast<float4*>(dst) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  } else {
    constexpr bool BF = std::is_same_v<T, __nv_bfloat16>;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<BF>(o.x * inv, o.y * inv), pack2<BF>(o.z * inv, o.w * inv));
  }
  if (a.lse && c4 == 0) a.lse[(static_cast<int64_t>(w.y) * a.Hq + head) * a.T + draft] = row_lse(m, l);
}

constexpr size_t round256(size_t n) { return (n + 255) & ~size_t(255); }
int tile_keys(int dtype, int D) { return dtype == TT_ATTN_F32 ? 4096 / D : 128; }
// What the end of a walk counts for, in tiles.  16-bit: the exchange between the halves, the next walk's Q and its first scores take 4 to 6 us, in which
// some of the next tiles arrive; less with few rows.  Measured, us, for 0, 2, 4, 6, 9: 32 sequences of 1000 to 8160 rows, 32 drafts, 32/8 heads,
// D = 128: 142, 132, 126, 120, 117; 64 of 500 to 4000, 8 drafts (32 rows): 135, 111, 107, 108, 108; 40 of 100 to 2900, 16 drafts, 12/4
// heads, D = 64 (48 rows): 30.7 with 2, 26.9, 26.5, 28.2.
int walk_end(int dtype, int rows) { return dtype == TT_ATTN_F32 ? 0 : (rows > 64 ? 8 : 4); }
constexpr int kLeast = 2;  // tiles of a piece: below that a piece costs more to begin and to put together than it takes
constexpr int kF32Ctas = 2;  // of an SM

template <int D, int R>
cudaError_t launch_r(const TreeArgs& a, int ctas, cudaStream_t stream) {
  auto kern = tree_f32_kernel<D, R>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D, R>::kSmem);
  if (e != cudaSuccess) return e;
  return launch_early(kern, dim3(ctas), dim3(kThreads), Cfg<D, R>::kSmem, stream, 1, a);
}

template <typename T>
cudaError_t launch_combine(int D, const TreeArgs& a, int ctas, cudaStream_t stream) {
  const dim3 grid(ctas, (a.block * (a.Hq / a.Hkv) * (D / 4) + 255) / 256);
  return D == 64 ? launch_early(tree_combine_kernel<T, 64>, grid, dim3(256), 0, stream, 1, a)
                 : launch_early(tree_combine_kernel<T, 128>, grid, dim3(256), 0, stream, 1, a);
}

}  // namespace

void tree_plan(int dtype, int Hq, int Hkv, int T, int* block, int* n_blocks) {
  const int group = Hq / Hkv, most = dtype == TT_ATTN_F32 ? 32 : kTreeRows;
  const int fit = most / group < T ? most / group : T;  // (groups of more heads than rows are refused)
  *block = (T + (T + fit - 1) / fit - 1) / ((T + fit - 1) / fit);  // as equal as can be
  *n_blocks = (T + *block - 1) / *block;
}

double tree_line(int dtype, int B, int Hq, int Hkv, int T, int capacity, int D) {
  int block, n;
  tree_plan(dtype, Hq, Hkv, T, &block, &n);
  const int keys = tile_keys(dtype, D);
  return static_cast<double>(B) * Hkv * n * ((capacity + keys - 1) / keys + (T + keys - 1) / keys + walk_end(dtype, block * (Hq / Hkv)));
}

int tree_ctas(int dtype, int B, int Hq, int Hkv, int T, int capacity, int D) {
  const double pieces = tree_line(dtype, B, Hq, Hkv, T, capacity, D) / kLeast + 1;
  const int most = kSms * (dtype == TT_ATTN_F32 ? kF32Ctas : 1);
  return pieces < most ? static_cast<int>(pieces) : most;
}

size_t tree_scratch_bytes(int dtype, int B, int Hq, int Hkv, int T, int capacity, int D) {
  const size_t ctas = tree_ctas(dtype, B, Hq, Hkv, T, capacity, D);
  return round256(ctas * sizeof(int4)) + ctas * 2 * tree_partial_floats(D) * sizeof(float);
}

cudaError_t launch_tree_f32(int D, const TreeArgs& a, int ctas, cudaStream_t stream) {
  const bool few = a.block * (a.Hq / a.Hkv) <= 8;
  if (D == 64) return few ? launch_r<64, 8>(a, ctas, stream) : launch_r<64, 32>(a, ctas, stream);
  return few ? launch_r<128, 8>(a, ctas, stream) : launch_r<128, 32>(a, ctas, stream);
}

cudaError_t launch_tree(int dtype, int D, TreeArgs a, void* scratch, int device, cudaStream_t stream) {
  const int ctas = tree_ctas(dtype, a.B, a.Hq, a.Hkv, a.T, a.capacity, D);
  tree_plan(dtype, a.Hq, a.Hkv, a.T, &a.block, &a.n_blocks);
  a.least = kLeast, a.ends = walk_end(dtype, a.block * (a.Hq / a.Hkv));
  a.pieces = static_cast<int4*>(scratch);
  a.partial = reinterpret_cast<float*>(static_cast<char*>(scratch) + round256(ctas * sizeof(int4)));
  cudaError_t e = dtype == TT_ATTN_F32 ? launch_tree_f32(D, a, ctas, stream) : launch_tree_tc(dtype, D, a, ctas, stream);
  if (e != cudaSuccess) return e;
  if (dtype == TT_ATTN_F32) return launch_combine<float>(D, a, ctas, stream);
  return dtype == TT_ATTN_F16 ? launch_combine<__half>(D, a, ctas, stream) : launch_combine<__nv_bfloat16>(D, a, ctas, stream);
}

}  // namespace ttattn
