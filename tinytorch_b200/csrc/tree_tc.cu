// Drafted tokens over a KV cache for fp16 / bf16 on sm_100a tensor cores (see tree.cuh for how the work is divided).
//
// Bound by memory: every cache row is read once for the up to 128 rows of a block (2 D keys and values of 16 bits for 4 D
// operations a row), so the loop has to keep the loads going and to do a tile's two products and 128 x 128 exponentials in the time
// that its 64 KB (D = 128) take to arrive, 2800 cycles of an SM's share of the bandwidth.  The key tiles of a walk go to the
// two halves of the CTA in turn:
//   warp 8     producer: publishes the segments, loads Q (one 5-D box: heads of the group inside drafts) and streams K and V tiles
//              of 128 keys, the cache's and then the drafts', through a ring in the order in which the products take them; it runs ahead
//              across segments
//   warp 9     issuer: S_t = Q K^T and O_t += P_t V with tcgen05.mma, P_t from TMEM
//   warps 0-3 / 4-7: softmax of half t.  Thread r owns row r (TMEM lane): scores, running maximum and sum, P written over S;
//              warps without rows skip all of it but the barriers.  V rows behind a sequence's length may hold anything and are
//              zeroed in shared memory before the product.  The halves' accumulators, in the same lanes, are put together at the end of a
//              segment by both warpgroups, each for half of the channels.
// R: a block of up to 32 rows lies in the 128 lanes four times, of up to 64 twice, and each copy takes 32 or 64 keys of every tile (its P is zero
// for the others): a tile's exponentials then are the work of all four warps of a warpgroup, on all four of an SM's
// special-function units, instead of one warp's.  The copies are added up through shared memory at the end of a segment.
// Measured, us: 32 sequences of 1000 to 8160 rows, 32 drafts, 32/8 heads, D = 128, bf16: 117 with the combine kernel (the scan alone 5.7 TB/s; one walk a CTA,
// as it came: 150); one of 2000 rows, 8 drafts: 12.4 (before the copies of few rows 2 more); 16 of 16 drafts, D = 64: 52 (77).
// Every mbarrier wait is bounded.
#include <cuda.h>

#include <type_traits>

#include "ptx.cuh"
#include "tma_host.cuh"
#include "tree.cuh"

namespace ttattn {
namespace {

constexpr int BM = 128, BN = 128, kThreads = 384, kTmemCols = 512;
constexpr int kHalfBytes = BM * 128;  // a block of 64 channels of a tile
constexpr int kSoft = 2 * BM;
constexpr int kProducer = 8, kIssuer = 9;

template <int D, int R>
struct Cfg {
  static constexpr int kTile = BM * D * 2, kRing = (R == 1 ? 6 : 5) * 128 / D;  // tiles of the ring
  static constexpr int kLanes = BM / R, kKeys = BN / R;                          // lanes of a copy of the rows, its keys of a tile
  static constexpr int kAddUp = R == 1 ? 0 : 2 * (BM - kLanes) * 32 * 4;         // 32 channels of all copies but the first, for either warpgroup
  static constexpr int kSmem = kTile + kRing * kTile + 512 /* control block */ + 2 * BM * 8 /* statistics */ + kAddUp;
  static_assert(kSmem <= 232448, "exceeds the shared memory a CTA may request");
};

struct __align__(16) Ctl {
  uint64_t q_full, q_empty;
  uint64_t full[12], empty[12];
  uint64_t s_full[2], p_full[2], o_full[2];
  uint64_t seg_full[2], seg_empty[2];
  TreeSegment seg[2];
  int scratch[kThreads / 32 + 2];
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(Ctl) <= 512, "control block");

template <int D, bool BF16, int R>
__global__ void __launch_bounds__(kThreads, 1)
    tree_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const __grid_constant__ CUtensorMap tmKd, const __grid_constant__ CUtensorMap tmVd, const TreeArgs a) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  using C = Cfg<D, R>;
  constexpr int kTile = C::kTile, kRing = C::kRing, kHalves = D / 64, kLanes = C::kLanes, kKeys = C::kKeys;
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((ptx::smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0 && a.status) atomicOr(a.status, kStatusBadSmemAlign);
    return;
  }
  uint8_t* sQ = smem;
  uint8_t* ring = sQ + kTile;
  Ctl* ctl = reinterpret_cast<Ctl*>(ring + kRing * kTile);
  volatile int* abort_flag = &ctl->abort_flag;
  float2* s_stat = reinterpret_cast<float2*>(reinterpret_cast<uint8_t*>(ctl) + 512);  // [half][lane]
  float* s_add = reinterpret_cast<float*>(s_stat + 2 * BM);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = a.Hq / a.Hkv;

  if (warp == kProducer && lane == 0) {
    ptx::mbar_init(&ctl->q_full, 1);
    ptx::mbar_init(&ctl->q_empty, 1);
#pragma unroll
    for (int i = 0; i < kRing; ++i) {
      ptx::mbar_init(&ctl->full[i], 1);
      ptx::mbar_init(&ctl->empty[i], 1);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(&ctl->s_full[i], 1);
      ptx::mbar_init(&ctl->p_full[i], BM);
      ptx::mbar_init(&ctl->o_full[i], 1);
      ptx::mbar_init(&ctl->seg_full[i], 1);
      ptx::mbar_init(&ctl->seg_empty[i], 1 + kSoft);
    }
    ctl->abort_flag = 0;
    ptx::fence_barrier_init();
    ptx::tma_prefetch_desc(&tmQ);
    ptx::tma_prefetch_desc(&tmK);
    ptx::tma_prefetch_desc(&tmV);
    ptx::tma_prefetch_desc(&tmKd);
    ptx::tma_prefetch_desc(&tmVd);
  }
  if (warp == kIssuer) {
    ptx::tmem_alloc(&ctl->tmem_base, kTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = ctl->tmem_base;
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  TreeWalk walk;
  walk.start<BN, kThreads>(a, ctl->scratch);

  if (warp >= 8) {
    ptx::setmaxnreg_dec<72>();  // (216 + 216 + 72 registers: the 168 x 384 that the CTA was launched with)
    if (warp == kProducer && lane == 0) {
      // -------------------------------------------------------------- producer --
      int st = 0;
      uint32_t ph = 0;  // of the ring
      a.pieces[blockIdx.x] = make_int4(0, 0, 0, 0);
      bool ok = true;
      for (uint32_t i = 0; ok; ++i) {
        TreeSegment s;
        const bool some = walk.next<BN>(a, &s);
        if (!some) s.n = -1;
        const int slot = i & 1;
        if (!ptx::mbar_wait(&ctl->seg_empty[slot], ((i >> 1) & 1) ^ 1, abort_flag)) break;
        ctl->seg[slot] = s;
        ptx::mbar_arrive(&ctl->seg_full[slot]);
        if (!some) break;
        if (s.piece == 1) a.pieces[blockIdx.x] = make_int4(walk.pieces(s), s.b, s.hk, s.block);
        auto load = [&](const CUtensorMap* cache, const CUtensorMap* drafts, int j) {
          const int tile = s.j0 + j;
          if (!ptx::mbar_wait(&ctl->empty[st], ph ^ 1, abort_flag)) return false;
          ptx::mbar_arrive_expect_tx(&ctl->full[st], kTile);
          const CUtensorMap* map = tile < s.n_ctx ? cache : drafts;
          const int row = (tile < s.n_ctx ? tile : tile - s.n_ctx) * BN;
#pragma unroll
          for (int hf = 0; hf < kHalves; ++hf) ptx::tma_load_4d(ring + st * kTile + hf * kHalfBytes, map, &ctl->full[st], hf * 64, row, s.hk, s.b);
          if (++st == kRing) st = 0, ph ^= 1;
          return true;
        };
        // In the order of the products: K0 K1 V0 K2 V1 ...  The first two go under the segment before, whose last products still need its Q.
        for (int j = 0; j < 2 && j < s.n && ok; ++j) ok = load(&tmK, &tmKd, j);
        if (!ok || !ptx::mbar_wait(&ctl->q_empty, (i & 1) ^ 1, abort_flag)) break;
        ptx::mbar_arrive_expect_tx(&ctl->q_full, R * kHalves * group * a.block * 128);
#pragma unroll
        for (int c = 0; c < R; ++c)
#pragma unroll
          for (int hf = 0; hf < kHalves; ++hf)
            ptx::tma_load_5d(sQ + hf * kHalfBytes + c * kLanes * 128, &tmQ, &ctl->q_full, hf * 64, 0, s.block * a.block, s.hk, s.b);
        for (int j = 0; j < s.n && ok; ++j) {
          ok = load(&tmV, &tmVd, j);
          if (j + 2 < s.n && ok) ok = load(&tmK, &tmKd, j + 2);
        }
      }
    } else if (warp == kIssuer) {
      // ---------------------------------------------------------------- issuer --
      // The whole warp runs the loop; one elected lane issues.  Half t takes the tiles t, t + 2, ... of a segment, in the order
      // PV(0) QK(0)' PV(1) QK(1)': MMAs execute in issue order, so QK(t)' cannot pass the PV(t) that still reads P_t.
      const bool leader = ptx::elect_one();
      auto uwait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, ptx::mbar_wait(bar, parity, abort_flag)) != 0; };
      // (a negative scale is folded into the sign of Q: the softmax multiplies by a non-negative one)
      const uint32_t idesc_qk = ptx::make_idesc_f16(BM, BN, BF16 ? 1 : 0, 0, 0) | (a.scale < 0.f ? (1u << 13) : 0u);
      const uint32_t idesc_pv = ptx::make_idesc_f16(BM, D, BF16 ? 1 : 0, 0, 1);
      constexpr uint32_t kHi = ptx::smem_desc_hi_sw128(1024);
      const uint32_t qlo = ptx::smem_desc_lo(ptx::smem_u32(sQ), 16), klo = ptx::smem_desc_lo(ptx::smem_u32(ring), 16);
      const uint32_t vlo = ptx::smem_desc_lo(ptx::smem_u32(ring), kHalfBytes);
      int st = 0;  // the next tile of the ring
      uint32_t ph = 0, done0 = 0, done1 = 0;  // done: softmax iterations of each half (p_full phases)
      bool ok = true;
      for (uint32_t i = 0; ok; ++i) {
        const int slot = i & 1;
        if (!uwait(&ctl->seg_full[slot], (i >> 1) & 1)) break;
        const int n = ctl->seg[slot].n;
        __syncwarp();
        if (leader) ptx::mbar_arrive(&ctl->seg_empty[slot]);
        if (n < 0) break;
        auto qk = [&](int t, bool last) {
          const uint32_t b0 = klo + st * (kTile >> 4), d = tmem + t * BN;
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            const uint32_t off = ((ks >> 2) * kHalfBytes + (ks & 3) * 32) >> 4;
            if (leader) ptx::mma_ss2(d, qlo + off, kHi, b0 + off, kHi, idesc_qk, ks > 0 ? 1u : 0u);
          }
          if (leader) ptx::mma_commit(&ctl->s_full[t]);
          if (leader) ptx::mma_commit(&ctl->empty[st]);
          if (leader && last) ptx::mma_commit(&ctl->q_empty);
          if (++st == kRing) st = 0, ph ^= 1;
        };
        if (!(ok = uwait(&ctl->q_full, i & 1))) break;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (t >= n || !ok) continue;
          if (!(ok = uwait(&ctl->full[st], ph))) continue;
          ptx::tc_fence_after();
          qk(t, t == n - 1);
        }
        for (int j0 = 0; j0 < n && ok; j0 += 2) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int j = j0 + t;
            if (j >= n || !ok) continue;
            const bool more = j + 2 < n;
            // (the wait for P comes last: it is the one on the critical path)
            bool all = ptx::mbar_wait(&ctl->full[st], ph, abort_flag);  // V, and the K behind it
            if (more && all) all = st + 1 < kRing ? ptx::mbar_wait(&ctl->full[st + 1], ph, abort_flag) : ptx::mbar_wait(&ctl->full[0], ph ^ 1, abort_flag);
            if (all) all = ptx::mbar_wait(&ctl->p_full[t], (t == 0 ? done0 : done1) & 1, abort_flag);
            if (!(ok = __all_sync(0xffffffffu, all) != 0)) continue;
            ptx::tc_fence_after();
            (t == 0 ? done0 : done1) += 1;
            const uint32_t b0 = vlo + st * (kTile >> 4), d = tmem + 256 + t * D, a0 = tmem + t * BN;
#pragma unroll
            for (int ks = 0; ks < BN / 16; ++ks)
              if (leader) ptx::mma_ts2(d, a0 + ks * 8, b0 + ks * (2048 >> 4), kHi, idesc_pv, (j0 > 0 || ks > 0) ? 1u : 0u);
            if (leader && !more) ptx::mma_commit(&ctl->o_full[t]);
            if (leader) ptx::mma_commit(&ctl->empty[st]);
            if (++st == kRing) st = 0, ph ^= 1;
            if (more) qk(t, j + 3 == n);
          }
        }
      }
    }
  } else {
    ptx::setmaxnreg_inc<216>();
    // ------------------------------------------------------------- softmax --
    const int t = warp >> 2, r = tid & (BM - 1);
    const uint32_t lane_addr = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + t * BN + lane_addr, tO = tmem + 256 + t * D + lane_addr;
    const float c = fmaxf(fabsf(a.scale) * kLog2e, 1e-30f);  // > 0, so that a hidden score stays -inf
    const float2 c2 = make_float2(c, c);
    const int copy = r / kLanes, row = r % kLanes, col0 = copy * kKeys;  // this lane's copy of the block's rows, its row, and its keys of a tile
    uint32_t cnt = 0, used = 0, ends[2] = {0, 0};  // phases of s_full, ring position, phases of o_full
    uint32_t s[BN];
    auto part_of = [&](const TreeSegment& g) { return a.partial + (static_cast<size_t>(blockIdx.x) * 2 + (g.piece > 0 ? 1 : 0)) * tree_partial_floats(D); };
    bool ok = true;
    // Threads meet at named barriers within a segment: an expired wait is voted on, and all leave together.
    for (uint32_t i = 0;; ++i) {
      const int slot = i & 1;
      ok = ptx::mbar_wait(&ctl->seg_full[slot], (i >> 1) & 1, abort_flag);
      if (ptx::named_barrier_or(3, kSoft, !ok)) break;
      const TreeSegment g = ctl->seg[slot];
      ptx::mbar_arrive(&ctl->seg_empty[slot]);
      if (g.n < 0) break;
      const int draft0 = g.block * a.block, drafts = a.T - draft0 < a.block ? a.T - draft0 : a.block, rows = drafts * group;
      const bool mine = row < rows, warp_has = (warp & 3) * 32 % kLanes < rows;
      const int draft = draft0 + row / group, head = g.hk * group + row % group;
      uint32_t sees[kKeys / 32];  // of this copy's keys of the drafts' tile
#pragma unroll
      for (int i = 0; i < kKeys / 32; ++i) sees[i] = 0;
      if (mine && g.j0 + g.n == g.n_all && ((g.n - 1) & 1) == t) {
        uint32_t words[4];
        tree_mask_row<4>(a, g.b, draft, words);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i / (kKeys / 32) == copy) sees[i % (kKeys / 32)] = words[i];
      }

      float m_ref = mine ? -INFINITY : 0.f;  // reference maximum, in log2 units
      float2 l2 = make_float2(0.f, 0.f);
      const int n_t = (g.n + 1 - t) / 2;
      for (int jj = 0; jj < n_t && ok; ++jj) {
        const int j = 2 * jj + t, tile = g.j0 + j;
        ok = ptx::mbar_wait(&ctl->s_full[t], (cnt + jj) & 1, abort_flag);
        if (!ok) break;
        ptx::tc_fence_after();
        const int left = tile < g.n_ctx ? g.len - tile * BN : BN;  // valid keys of a tile of the cache
        if (left < BN) {
          // what lies behind the length may be infinite: exact zeros, so that 0 times it is 0
          const uint32_t at = used + 2 * j + (j == g.n - 1 ? 1 : 2);  // (where V of tile j lies in the order K0 K1 V0 K2 V1 ...)
          ok = ptx::mbar_wait(&ctl->full[at % kRing], (at / kRing) & 1, abort_flag);
          if (ok && r >= left) {
            uint8_t* v = ring + (at % kRing) * kTile + r * 128;
#pragma unroll
            for (int hf = 0; hf < kHalves; ++hf)
#pragma unroll
              for (int ch = 0; ch < 8; ++ch) *reinterpret_cast<uint4*>(v + hf * kHalfBytes + ch * 16) = make_uint4(0, 0, 0, 0);
          }
          ptx::fence_proxy_async_smem();
        }
        if (warp_has) {
#pragma unroll
          for (int cc = 0; cc < kKeys / 32; ++cc) ptx::tmem_ld32p(tS + col0 + cc * 32, s + cc * 32);
          ptx::tmem_wait_ld();
          if (tile >= g.n_ctx) {
#pragma unroll
            for (int e = 0; e < kKeys; ++e)
              if (!((sees[e / 32] >> (e % 32)) & 1)) s[e] = 0xff800000u;
          } else if (left < BN || !mine) {
            const int lim = mine ? left - col0 : 0;
#pragma unroll
            for (int e = 0; e < kKeys; ++e)
              if (e >= lim) s[e] = 0xff800000u;
          }
          // The maximum is only a reference for the exponentials: it is kept while a tile's sum shows that none is large.
          bool need_max = jj == 0;
          for (;;) {
            if (need_max) {
              float mx[8];
#pragma unroll
              for (int q = 0; q < 8; ++q) mx[q] = ptx::max3(__uint_as_float(s[q]), __uint_as_float(s[q + 8]), -INFINITY);
#pragma unroll
              for (int e = 16; e < kKeys; e += 16)
#pragma unroll
                for (int q = 0; q < 8; ++q) mx[q] = ptx::max3(mx[q], __uint_as_float(s[e + q]), __uint_as_float(s[e + q + 8]));
              const float x_max = ptx::max3(ptx::max3(mx[0], mx[1], mx[2]), ptx::max3(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7])) * c;
              if (jj == 0) {
                if (mine) m_ref = x_max;
              } else if (__any_sync(0xffffffffu, x_max > m_ref)) {
                const float m_new = fmaxf(m_ref, x_max);
                const float alpha = m_new == -INFINITY ? 1.f : ptx::ex2(m_ref - m_new);
                uint32_t x[32];
#pragma unroll
                for (int cc = 0; cc < D / 32; ++cc) {
                  ptx::tmem_ld32(tO + cc * 32, x);
                  ptx::tmem_wait_ld();
#pragma unroll
                  for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * alpha);
                  ptx::tmem_st32(tO + cc * 32, x);
                }
                l2.x *= alpha, l2.y *= alpha;
                m_ref = m_new;
              }
            }
            const float m_use = m_ref == -INFINITY ? 0.f : m_ref;  // (nothing seen so far: exponentials of -inf)
            const float2 nm2 = make_float2(-m_use, -m_use);
            float2 lt = make_float2(0.f, 0.f);
            constexpr int kPart = kKeys < 64 ? kKeys : 64;  // keys whose P is stored together
#pragma unroll
            for (int k0 = 0; k0 < kKeys; k0 += kPart) {
              uint32_t pk[kPart / 2];
#pragma unroll
              for (int e2 = 0; e2 < kPart; e2 += 2) {
                const float2 x = ptx::fma2(make_float2(__uint_as_float(s[k0 + e2]), __uint_as_float(s[k0 + e2 + 1])), c2, nm2);
                const float2 p = make_float2(ptx::ex2(x.x), ptx::ex2(x.y));
                lt = ptx::add2(lt, p);
                pk[e2 >> 1] = pack2<BF16>(p.x, p.y);
              }
              if constexpr (R == 4) ptx::tmem_st16(tS + copy * 16, pk);
              else ptx::tmem_st32(tS + copy * 32 + k0 / 2, pk);
            }
            if constexpr (R > 1) {  // the other copies' keys
              uint32_t zero[kKeys / 2];
#pragma unroll
              for (int i = 0; i < kKeys / 2; ++i) zero[i] = 0;
#pragma unroll
              for (int i = 1; i < R; ++i) {
                if constexpr (R == 4) ptx::tmem_st16(tS + (copy + i) % R * 16, zero);
                else ptx::tmem_st32(tS + (copy + i) % R * 32, zero);
              }
            }
            const float sum = lt.x + lt.y;
            const bool redo = !need_max && (!(sum <= 256.f) || m_ref == -INFINITY);
            if (!__any_sync(0xffffffffu, redo)) {
              l2 = ptx::add2(l2, lt);
              break;
            }
            need_max = true;
          }
          ptx::tmem_wait_st();
        }
        ptx::tc_fence_before();
        ptx::mbar_arrive(&ctl->p_full[t]);
      }
      cnt += n_t, used += 2 * g.n;

      // Both halves, in the same lanes: warpgroup t puts the channels [64 t, 64 t + 64) together (D = 64: warpgroup 0 all of them).  It holds them in
      // registers before the barrier, behind which the accumulators may be overwritten while it still works on them.
      const bool two = g.n > 1, puts = warp_has && (D == 128 || t == 0);
      const int c0 = D == 128 ? t * 64 : 0;
      if (ok) ok = ptx::mbar_wait(&ctl->o_full[0], ends[0] & 1, abort_flag);
      if (ok && two) ok = ptx::mbar_wait(&ctl->o_full[1], ends[1] & 1, abort_flag);
      ++ends[0], ends[1] += two;
      ptx::tc_fence_after();
      // (with tiles for both halves, the products that were waited for say that the other has read the statistics of the segment before)
      if (!two) ptx::named_barrier(3, kSoft);
      s_stat[t * BM + r] = make_float2(n_t > 0 ? m_ref : -INFINITY, l2.x + l2.y);
      if (puts) {
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          ptx::tmem_ld32p(tmem + 256 + lane_addr + c0 + cc * 32, s + cc * 32);
          if (two) ptx::tmem_ld32p(tmem + 256 + D + lane_addr + c0 + cc * 32, s + 64 + cc * 32);
        }
        ptx::tmem_wait_ld();
      }
      ptx::tc_fence_before();
      if (ptx::named_barrier_or(3, kSoft, !ok)) break;
      if (puts && mine) {
        // over the copies and halves of the row; one that has seen no key for it holds zeros, or nothing at all, and takes no part (weight 0; a NaN sum
        // counts whatever its weight is)
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * R; ++i) m = fmaxf(m, s_stat[i * kLanes + row].x);
        auto weight = [&](float ref) { return ref == -INFINITY ? 0.f : ptx::ex2(ref - m); };
#pragma unroll
        for (int i = 0; i < 2 * R; ++i) {
          const float2 x = s_stat[i * kLanes + row];
          l = fmaf(x.y, weight(x.x), l);
        }
        const float inv = g.piece >= 0 ? 1.f : inverse_sum(l);
        const float ua = weight(s_stat[r].x) * inv, ub = weight(s_stat[BM + r].x) * inv;
#pragma unroll
        for (int e = 0; e < 64; ++e) {
          float x = ua != 0.f ? __uint_as_float(s[e]) * ua : 0.f;
          if (two && ub != 0.f) x = fmaf(__uint_as_float(s[64 + e]), ub, x);
          s[e] = __float_as_uint(x);
        }
        if (t == 0 && copy == 0) {
          if (g.piece >= 0)
            *reinterpret_cast<float2*>(part_of(g) + kTreeRows * D + row * 2) = make_float2(l == 0.f ? -INFINITY : m, l);
          else if (a.lse)
            a.lse[(static_cast<int64_t>(g.b) * a.Hq + head) * a.T + draft] = row_lse(m, l);
        }
      }
      if constexpr (R > 1) {
        if (D == 128 || t == 0) {
          float* add = s_add + t * (BM - kLanes) * 32;
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {  // 32 channels at a time
            if (copy > 0 && mine) {
#pragma unroll
              for (int e = 0; e < 32; ++e) add[e * (BM - kLanes) + r - kLanes] = __uint_as_float(s[cc * 32 + e]);
            }
            ptx::named_barrier(1 + t, BM);
            if (copy == 0 && mine) {
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                float x = __uint_as_float(s[cc * 32 + e]);
#pragma unroll
                for (int i = 0; i < R - 1; ++i) x += add[e * (BM - kLanes) + i * kLanes + row];
                s[cc * 32 + e] = __float_as_uint(x);
              }
            }
            ptx::named_barrier(1 + t, BM);
          }
        }
      }
      if (puts && mine && copy == 0) {
        if (g.piece >= 0) {
          float* part = part_of(g);
#pragma unroll
          for (int ch = 0; ch < 16; ++ch)
            *reinterpret_cast<uint4*>(part + (c0 / 4 + ch) * (kTreeRows * 4) + row * 4) = make_uint4(s[ch * 4], s[ch * 4 + 1], s[ch * 4 + 2], s[ch * 4 + 3]);
        } else {
          T* orow = reinterpret_cast<T*>(a.o) + g.b * a.os.b + head * a.os.h + draft * a.os.s;
#pragma unroll
          for (int ch = 0; ch < 8; ++ch) {
            uint4 w;
            w.x = pack2<BF16>(__uint_as_float(s[ch * 8 + 0]), __uint_as_float(s[ch * 8 + 1]));
            w.y = pack2<BF16>(__uint_as_float(s[ch * 8 + 2]), __uint_as_float(s[ch * 8 + 3]));
            w.z = pack2<BF16>(__uint_as_float(s[ch * 8 + 4]), __uint_as_float(s[ch * 8 + 5]));
            w.w = pack2<BF16>(__uint_as_float(s[ch * 8 + 6]), __uint_as_float(s[ch * 8 + 7]));
            *reinterpret_cast<uint4*>(orow + c0 + ch * 8) = w;
          }
        }
      }
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (warp == kIssuer) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, kTmemCols);
  }
  if (tid == 0 && ctl->abort_flag && a.status) atomicOr(a.status, kStatusWaitExpired);
}

// Q as [B][kv head][draft][head of the group][D]: a box is all heads of the group, the drafts of a block and 64 channels.
bool make_map_q(CUtensorMap* m, int dtype, const TreeArgs& a, int D) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const int group = a.Hq / a.Hkv;
  cuuint64_t dims[5] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(group), static_cast<cuuint64_t>(a.T),
                        static_cast<cuuint64_t>(a.Hkv), static_cast<cuuint64_t>(a.B)};
  cuuint64_t strides[4] = {static_cast<cuuint64_t>(a.qs.h) * 2, static_cast<cuuint64_t>(a.qs.s) * 2, static_cast<cuuint64_t>(a.qs.h) * group * 2,
                           static_cast<cuuint64_t>(a.qs.b) * 2};
  cuuint32_t box[5] = {64, static_cast<cuuint32_t>(group), static_cast<cuuint32_t>(a.block), 1, 1};
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  return fn(m, dtype == TT_ATTN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, const_cast<void*>(a.q), dims, strides,
            box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool BF16, int R>
cudaError_t launch_r(int dtype, const TreeArgs& a, int ctas, cudaStream_t stream) {
  CUtensorMap tq, tk, tv, tkd, tvd;
  if (!make_map_q(&tq, dtype, a, D) || !make_map(&tk, dtype, a.kc, D, a.capacity, a.Hkv, a.B, a.kcs) ||
      !make_map(&tv, dtype, a.vc, D, a.capacity, a.Hkv, a.B, a.vcs) || !make_map(&tkd, dtype, a.kd, D, a.T, a.Hkv, a.B, a.kds) ||
      !make_map(&tvd, dtype, a.vd, D, a.T, a.Hkv, a.B, a.vds))
    return cudaErrorInvalidValue;
  auto kern = tree_tc_kernel<D, BF16, R>;
  constexpr int kSmem = Cfg<D, R>::kSmem;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  return launch_early(kern, dim3(ctas), dim3(kThreads), kSmem, stream, 1, tq, tk, tv, tkd, tvd, a);
}
template <int D, bool BF16>
cudaError_t launch_t(int dtype, const TreeArgs& a, int ctas, cudaStream_t stream) {
  const int rows = a.block * (a.Hq / a.Hkv);
  return rows <= 32 ? launch_r<D, BF16, 4>(dtype, a, ctas, stream)
         : rows <= 64 ? launch_r<D, BF16, 2>(dtype, a, ctas, stream) : launch_r<D, BF16, 1>(dtype, a, ctas, stream);
}

}  // namespace

cudaError_t launch_tree_tc(int dtype, int D, const TreeArgs& a, int ctas, cudaStream_t stream) {
  const bool bf = dtype == TT_ATTN_BF16;
  if (D == 128) return bf ? launch_t<128, true>(dtype, a, ctas, stream) : launch_t<128, false>(dtype, a, ctas, stream);
  return bf ? launch_t<64, true>(dtype, a, ctas, stream) : launch_t<64, false>(dtype, a, ctas, stream);
}

}  // namespace ttattn
