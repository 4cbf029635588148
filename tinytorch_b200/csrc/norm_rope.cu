// The RMS norm of every head of q and k and the rotation of its channel pairs to the token's position, in one pass.
//
//   n = x * rsqrt(mean(x^2) + eps),  y = n * w            (skipped where there is no weight)
//   (a, b) -> (a cos - b sin, b cos + a sin)              for every pair of channels (skipped where there are no tables)
//
// and its gradients: with u = the output's gradient, turned back by the same angles, r = rsqrt(mean(x^2) + eps) and g = u * w,
//   dw = sum over tokens and heads of r u x,   dx = r g - r^3 mean(g x) x
// r is computed again from x, which has to be read anyway: nothing but the inputs is kept for the backward.  All in fp32,
// with one rounding to the tensor type of each value stored.
//
// Bound by memory: x in and y out (backward: x and dy in, dx out), and next to that by instructions (262 and 362 a chunk of 2 KB in and out, 3 KB
// backward), which set the pace at D = 64 in 16 bits and in the fp32 backward.  In a loop, whose inputs are partly in L2: 8200 tokens of 32/8 heads, D = 128, bf16: forward 29 us (5.8
// TB/s; 172 MB that are not there 31.7, 5.4), backward 52 us (4.9 TB/s); 8192 of 16/16, D = 64, fp16: 13 (5.2) and 25 us (4.0); 4000 of 40/8, D = 64, fp32: 14
// (6.9) and 32 us (4.6).  A row of D channels belongs to D / 16
// neighbouring lanes, each with 8 channels of the first half and the same 8 of the second, so that a pair (i, i + D/2) or
// (2i, 2i + 1) never leaves a thread, every access is a 16-byte vector of a 64- or 128-byte run, and the means take two or
// three shuffles; the arithmetic is in packed pairs.  A warp takes 512 / D heads of one token at a time (a chunk), and an equal,
// contiguous share of all chunks of q or of k.  Rows, and the angles of every new token, come through shared memory (cp.async), kAhead chunks
// before they are needed and across tokens; nothing there is shared by more than a warp, and the bytes in flight cost no registers.
#include <type_traits>

#include "norm_rope.cuh"
#include "ptx.cuh"
#include "tma_host.cuh"

namespace ttattn {
namespace {

constexpr int kWarps = 4;  // per CTA
// Chunks in flight beside the one that is worked on (kAhead + 1 is a power of two), and CTAs of an SM.  Warps in flight count for more than bytes of a
// warp: with 3 and 7 chunks ahead 8200 tokens of 32/8 heads, D = 128, bf16, take 54 and 72 us backward, with 1 52; with 5 CTAs, whose
// registers spill, 81.
constexpr int kAhead = 1, kFwdCtas = 8, kBwdCtas = 4;

__device__ __forceinline__ float2 splat(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 neg2(float2 x) { return make_float2(-x.x, -x.y); }

// two neighbouring channels
template <typename T>
__device__ __forceinline__ float2 widen(uint32_t w) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
}

// How the D channels of a row lie in its D / 16 lanes: per half of the row, kVec vectors of kChannels channels, whose lanes follow one another.
template <typename T, int D>
struct Lay {
  static constexpr int kLanes = D / 16, kRows = 32 / kLanes, kChannels = 16 / sizeof(T), kVec = 8 / kChannels;
  static __device__ __forceinline__ int channel(int l, int vec) { return (vec * kLanes + l) * kChannels; }

  static __device__ __forceinline__ void widen4(const uint4 (&w)[kVec], float2 (&f)[4]) {
    if constexpr (std::is_same_v<T, float>) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f[2 * i] = make_float2(__uint_as_float(w[i].x), __uint_as_float(w[i].y));
        f[2 * i + 1] = make_float2(__uint_as_float(w[i].z), __uint_as_float(w[i].w));
      }
    } else {
      f[0] = widen<T>(w[0].x), f[1] = widen<T>(w[0].y), f[2] = widen<T>(w[0].z), f[3] = widen<T>(w[0].w);
    }
  }
  // A lane's pairs.  (i, i + D/2): those of its 8 channels of a half.  (2i, 2i + 1): four in its channels of the first half, four in those of the second.
  template <bool INTERLEAVED>
  static __device__ __forceinline__ int pair_of(int l, int i) {
    if constexpr (INTERLEAVED) return kVec == 2 ? i / 4 * (D / 4) + channel(l, i / 2 % 2) / 2 + i % 2 : i / 4 * (D / 4) + channel(l, 0) / 2 + i % 4;
    else return kVec == 2 ? channel(l, i / 4) + i % 4 : channel(l, 0) + i;
  }
  // ... of a token's cos or sin
  template <bool INTERLEAVED>
  static __device__ __forceinline__ void get_angles(const float* p, int l, float2 (&f)[4]) {
    if constexpr (INTERLEAVED && kVec == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = *reinterpret_cast<const float2*>(p + pair_of<INTERLEAVED>(l, 2 * i));
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 v = *reinterpret_cast<const float4*>(p + pair_of<INTERLEAVED>(l, 4 * i));
        f[2 * i] = make_float2(v.x, v.y), f[2 * i + 1] = make_float2(v.z, v.w);
      }
    }
  }
  // half of a row
  static __device__ __forceinline__ void store(T* row, int l, const float2 (&f)[4]) {
    if constexpr (std::is_same_v<T, float>) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        *reinterpret_cast<float4*>(row + channel(l, i)) = make_float4(f[2 * i].x, f[2 * i].y, f[2 * i + 1].x, f[2 * i + 1].y);
    } else {
      constexpr bool BF = std::is_same_v<T, __nv_bfloat16>;
      *reinterpret_cast<uint4*>(row + channel(l, 0)) =
          make_uint4(pack2<BF>(f[0].x, f[0].y), pack2<BF>(f[1].x, f[1].y), pack2<BF>(f[2].x, f[2].y), pack2<BF>(f[3].x, f[3].y));
    }
  }
};

// A CTA's shared memory: each warp's ring of rows (a lane reads back what it has asked for itself) and of tokens' angles (cos and sin of every pair), and
// the weight in fp32.
template <typename T, int D, int TENSORS>
struct Smem {
  using L = Lay<T, D>;
  static constexpr int kStage = TENSORS * 2 * L::kVec * 32, kRing = kWarps * (kAhead + 1) * kStage, kAngles = kWarps * (kAhead + 1) * D / 4;  // 16-byte vectors
  static constexpr int kBytes = (kRing + (TENSORS == 2 ? kAngles : 0)) * 16 + D * 4;
  uint4* ring;
  float* angles;
  float* weight;
  __device__ __forceinline__ explicit Smem(uint4* smem) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    ring = smem + warp * ((kAhead + 1) * kStage) + lane;
    angles = reinterpret_cast<float*>(smem + kRing) + warp * ((kAhead + 1) * D);
    weight = reinterpret_cast<float*>(smem + kRing + (TENSORS == 2 ? kAngles : 0));
  }
  __device__ __forceinline__ uint4* row(int stage, int tensor, int half) const { return ring + (stage * TENSORS * 2 + tensor * 2 + half) * (L::kVec * 32); }
  __device__ __forceinline__ void ask(int stage, int tensor, const T* from, int l) const {
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int i = 0; i < L::kVec; ++i) ptx::cp_async16(ptx::smem_u32(row(stage, tensor, half) + i * 32), from + half * (D / 2) + L::channel(l, i), 16);
  }
  __device__ __forceinline__ void get(int stage, int tensor, int half, float2 (&f)[4]) const {
    uint4 w[L::kVec];
#pragma unroll
    for (int i = 0; i < L::kVec; ++i) w[i] = row(stage, tensor, half)[i * 32];
    L::widen4(w, f);
  }
  __device__ __forceinline__ void get_weight(int half, int l, float2 (&f)[4]) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // four channels at a time
      const int c = L::kVec == 2 ? L::channel(l, i) : L::channel(l, 0) + i * 4;
      const float4 w = *reinterpret_cast<const float4*>(weight + half * (D / 2) + c);
      f[2 * i] = make_float2(w.x, w.y), f[2 * i + 1] = make_float2(w.z, w.w);
    }
  }
};

// The axis of a pair, and its position.
__device__ __forceinline__ int axis_of(const NormRopeArgs& a, int pair) {
  int x = 0;
#pragma unroll
  for (int e = 0; e + 1 < kMaxAxes; ++e) x += pair >= a.axis_end[e];
  return x;
}
__device__ __forceinline__ int position_of(const NormRopeArgs& a, const int (&pos)[kMaxAxes], int pair) {
  if (a.axes == 1) return pos[0];
  const int x = axis_of(a, pair);
  int p = pos[0];
#pragma unroll
  for (int e = 1; e < kMaxAxes; ++e) p = x == e ? pos[e] : p;
  return p;
}

// By a warp: a token's cos and sin to shared memory.  A position outside the tables turns nothing.
template <int D>
__device__ __forceinline__ void ask_angles(const NormRopeArgs& a, const int (&pos)[kMaxAxes], float* to, int lane) {
  bool outside = false;
  constexpr int N = D / 64;  // pairs of a lane
  const int pair = lane * N, p = position_of(a, pos, pair);
  if (p >= 0 && p < a.rope_positions && (N == 1 || a.axes == 1 || axis_of(a, pair) == axis_of(a, pair + N - 1))) {
    const int64_t at = static_cast<int64_t>(p) * (D / 2) + pair;
    ptx::cp_async_small<N * 4>(ptx::smem_u32(to + pair), a.cos + at);
    ptx::cp_async_small<N * 4>(ptx::smem_u32(to + D / 2 + pair), a.sin + at);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int q = position_of(a, pos, pair + i);
      if (q >= 0 && q < a.rope_positions) {
        const int64_t at = static_cast<int64_t>(q) * (D / 2) + pair + i;
        ptx::cp_async_small<4>(ptx::smem_u32(to + pair + i), a.cos + at);
        ptx::cp_async_small<4>(ptx::smem_u32(to + D / 2 + pair + i), a.sin + at);
      } else {
        to[pair + i] = 1.f, to[D / 2 + pair + i] = 0.f, outside = true;
      }
    }
  }
  if (outside && a.status) atomicOr(a.status, kStatusRopeRange);
}

// ... of a lane's pairs to registers
template <typename T, int D, bool INTERLEAVED>
__device__ __forceinline__ void load_angles(const NormRopeArgs& a, const int (&pos)[kMaxAxes], int l, float2 (&c)[4], float2 (&s)[4]) {
  if (a.axes == 1 && pos[0] >= 0 && pos[0] < a.rope_positions) {
    const int64_t at = static_cast<int64_t>(pos[0]) * (D / 2);
    Lay<T, D>::template get_angles<INTERLEAVED>(a.cos + at, l, c), Lay<T, D>::template get_angles<INTERLEAVED>(a.sin + at, l, s);
    return;
  }
  bool outside = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // neighbouring pairs, as a rule of one axis
    const int pair = Lay<T, D>::template pair_of<INTERLEAVED>(l, 2 * i), p = position_of(a, pos, pair), p1 = position_of(a, pos, pair + 1);
    const bool in = p >= 0 && p < a.rope_positions, in1 = p1 >= 0 && p1 < a.rope_positions;
    const int64_t at = static_cast<int64_t>(p) * (D / 2) + pair, at1 = static_cast<int64_t>(p1) * (D / 2) + pair + 1;
    if (p == p1 && in) {
      c[i] = __ldg(reinterpret_cast<const float2*>(a.cos + at)), s[i] = __ldg(reinterpret_cast<const float2*>(a.sin + at));
    } else {
      c[i] = make_float2(in ? __ldg(a.cos + at) : 1.f, in1 ? __ldg(a.cos + at1) : 1.f);
      s[i] = make_float2(in ? __ldg(a.sin + at) : 0.f, in1 ? __ldg(a.sin + at1) : 0.f);
      outside |= !in || !in1;
    }
  }
  if (outside && a.status) atomicOr(a.status, kStatusRopeRange);
}

// lo, hi: the lane's channels of the two halves; BACK: by the negative angles
template <bool INTERLEAVED, bool BACK>
__device__ __forceinline__ void rotate(const float2 (&c)[4], const float2 (&s)[4], float2 (&lo)[4], float2 (&hi)[4]) {
  if constexpr (INTERLEAVED) {
    // (c[0].x, c[0].y, c[1].x, c[1].y: the pairs of lo; then those of hi)
    auto turn = [](float2& p, float c, float s) {
      if (BACK) s = -s;
      p = ptx::fma2(p, splat(c), ptx::mul2(make_float2(p.y, p.x), make_float2(-s, s)));
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      turn(lo[2 * i], c[i].x, s[i].x), turn(lo[2 * i + 1], c[i].y, s[i].y);
      turn(hi[2 * i], c[2 + i].x, s[2 + i].x), turn(hi[2 * i + 1], c[2 + i].y, s[2 + i].y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = lo[i], y = hi[i], n = neg2(s[i]);
      lo[i] = ptx::fma2(y, BACK ? s[i] : n, ptx::mul2(x, c[i]));
      hi[i] = ptx::fma2(x, BACK ? n : s[i], ptx::mul2(y, c[i]));
    }
  }
}

template <int LANES>
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int of = LANES / 2; of >= 1; of >>= 1) x += __shfl_xor_sync(0xffffffffu, x, of);
  return x;
}

// A walk over the chunks of a warp's share, token by token: of q (t = 0) or k (t = 1).
struct Walk {
  int token, chunk, chunks;  // chunks: of a token
  __device__ __forceinline__ Walk(int64_t first, int per_token) : chunks(per_token) {
    token = static_cast<int>(first / per_token), chunk = static_cast<int>(first - static_cast<int64_t>(token) * per_token);
  }
  __device__ __forceinline__ bool next() {  // true: a new token
    if (++chunk < chunks) return false;
    chunk = 0, ++token;
    return true;
  }
};

// The rows of token `token` of a tensor
template <typename T>
__device__ __forceinline__ T* rows_of(const void* base, const Str3& st, int S, int token) {
  const int b = token / S;
  return reinterpret_cast<T*>(const_cast<void*>(base)) + b * st.b + (token - b * S) * st.s;
}

// What both passes have in common: shares, positions one token ahead, rows and angles kAhead chunks ahead.  `done` gets (ring stage, angle slot, token, head).
template <typename T, int D, int TENSORS, typename F>
__device__ __forceinline__ void stream(const NormRopeArgs& a, const Smem<T, D, TENSORS>& smem, int t, int64_t first, int n, F done) {
  using L = Lay<T, D>;
  const int lane = threadIdx.x & 31, l = lane % L::kLanes, sub = lane / L::kLanes, heads = a.heads[t];
  const int per_token = (heads + L::kRows - 1) / L::kRows;
  const bool rotated = a.cos != nullptr, normed = a.w[t] != nullptr;
  int pos[kMaxAxes];
  auto load_pos = [&](int token) {
    if (!rotated || token >= a.B * a.S) return;
    const int b = token / a.S;
#pragma unroll
    for (int e = 0; e < kMaxAxes; ++e) pos[e] = e < a.axes ? a.positions[e * a.pos_axis + b * a.pos_b + (token - b * a.S)] : 0;
  };
  Walk ahead(first, per_token), now = ahead;
  const T *x0, *x1;
  int asked = 0, slot_ahead = 0, slot = 0;
  auto new_token = [&]() {
    x0 = rows_of<const T>(TENSORS == 2 ? a.dy[t] : a.x[t], TENSORS == 2 ? a.dys[t] : a.xs[t], a.S, ahead.token);
    if (TENSORS == 2) x1 = rows_of<const T>(a.x[t], a.xs[t], a.S, ahead.token);
  };
  const int64_t h0 = TENSORS == 2 ? a.dys[t].h : a.xs[t].h, h1 = a.xs[t].h;
  auto ask = [&](bool turn) {
    if (asked < n) {
      const int h = ahead.chunk * L::kRows + sub;
      if (h < heads) {
        smem.ask(asked & kAhead, 0, x0 + h * h0, l);
        if (TENSORS == 2 && normed) smem.ask(asked & kAhead, 1, x1 + h * h1, l);
      }
      if (turn && rotated) {
        ask_angles<D>(a, pos, smem.angles + slot_ahead * D, lane);
        load_pos(ahead.token + 1);
      }
    }
    ptx::cp_async_commit();
    ++asked;
  };
  // (a share, and a token, begins here: its rows are asked for before its position is waited for)
  load_pos(ahead.token);
  new_token();
  bool turn = true;
  auto step = [&]() {
    ask(turn);
    turn = ahead.next();
    if (turn) slot_ahead = (slot_ahead + 1) & kAhead, new_token();
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) step();
  for (int i = 0; i < n; ++i) {
    __syncwarp();  // (a slot of angles may be filled again: all lanes have read it)
    step();
    ptx::cp_async_wait_but<kAhead>();
    __syncwarp();
    done(i & kAhead, slot, now.token, now.chunk * L::kRows + sub);
    if (now.next()) slot = (slot + 1) & kAhead;
  }
}

// Some chunks of one token to a warp, all of them if there are many tokens: the angles then stay in registers, and with 32 warps to an SM those that wait for
// their angles (two loads, one after the other, under the first rows) do not show.
template <typename T, int D, bool INTERLEAVED>
__global__ void __launch_bounds__(kWarps * 32, kFwdCtas) norm_rope_kernel(const NormRopeArgs a) {
  using L = Lay<T, D>;
  extern __shared__ uint4 raw[];
  const Smem<T, D, 1> smem(raw);
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const int t = static_cast<int>(blockIdx.x) >= a.ctas[0], lane = threadIdx.x & 31, l = lane % L::kLanes, sub = lane / L::kLanes, heads = a.heads[t];
  const T* w = reinterpret_cast<const T*>(a.w[t]);
  const uint32_t unit = (blockIdx.x - (t ? a.ctas[0] : 0)) * kWarps + (threadIdx.x >> 5);
  const uint32_t token = unit / a.split[t], part = unit - token * a.split[t], b = token / a.S, row = token - b * a.S;
  const int chunks = (heads + L::kRows - 1) / L::kRows, per = (chunks + a.split[t] - 1) / a.split[t], c0 = part * per;
  const int c1 = token >= static_cast<uint32_t>(a.B) * a.S ? c0 : (c0 + per < chunks ? c0 + per : chunks);
  int pos[kMaxAxes];
  if (a.cos && c0 < c1) {
#pragma unroll
    for (int e = 0; e < kMaxAxes; ++e) pos[e] = e < a.axes ? a.positions[e * a.pos_axis + b * a.pos_b + row] : 0;
  }
  const T* x = reinterpret_cast<const T*>(a.x[t]) + b * a.xs[t].b + row * a.xs[t].s;
  const int64_t xh = a.xs[t].h, yh = a.ys[t].h;
  auto ask = [&](int c) {
    const int h = c * L::kRows + sub;
    if (c < c1 && h < heads) smem.ask(c & kAhead, 0, x + h * xh, l);
    ptx::cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) ask(c0 + i);
  if (w) {
    for (int i = threadIdx.x; i < D; i += kWarps * 32) smem.weight[i] = to_f32<T>(w[i]);
    __syncthreads();
  }
  if (c0 >= c1) return;
  float2 cs[4], sn[4];
  if (a.cos) load_angles<T, D, INTERLEAVED>(a, pos, l, cs, sn);
  T* y = reinterpret_cast<T*>(a.y[t]) + b * a.ys[t].b + row * a.ys[t].s;
  for (int c = c0; c < c1; ++c) {
    ask(c + kAhead);
    ptx::cp_async_wait_but<kAhead>();
    float2 lo[4], hi[4];
    smem.get(c & kAhead, 0, 0, lo), smem.get(c & kAhead, 0, 1, hi);  // (of a head that does not exist: whatever lies there, which goes nowhere)
    if (w) {
      float2 sq = ptx::mul2(lo[0], lo[0]);
#pragma unroll
      for (int i = 1; i < 4; ++i) sq = ptx::fma2(lo[i], lo[i], sq);
#pragma unroll
      for (int i = 0; i < 4; ++i) sq = ptx::fma2(hi[i], hi[i], sq);
      const float2 r = splat(rsqrtf(row_sum<L::kLanes>(sq.x + sq.y) * (1.f / D) + a.eps));
      float2 wv[4];
      smem.get_weight(0, l, wv);
#pragma unroll
      for (int i = 0; i < 4; ++i) lo[i] = ptx::mul2(lo[i], ptx::mul2(wv[i], r));
      smem.get_weight(1, l, wv);
#pragma unroll
      for (int i = 0; i < 4; ++i) hi[i] = ptx::mul2(hi[i], ptx::mul2(wv[i], r));
    }
    if (a.cos) rotate<INTERLEAVED, false>(cs, sn, lo, hi);
    const int h = c * L::kRows + sub;
    if (h < heads) {
      T* to = y + h * yh;
      L::store(to, l, lo), L::store(to + D / 2, l, hi);
    }
  }
}

template <typename T, int D, bool INTERLEAVED>
__global__ void __launch_bounds__(kWarps * 32, kBwdCtas) norm_rope_bwd_kernel(const NormRopeArgs a) {
  using L = Lay<T, D>;
  extern __shared__ uint4 raw[];
  const Smem<T, D, 2> smem(raw);  // 0: dy, 1: x
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const int t = static_cast<int>(blockIdx.x) >= a.ctas[0], lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % L::kLanes, heads = a.heads[t];
  const T* w = reinterpret_cast<const T*>(a.w[t]);
  if (w) {
    for (int i = threadIdx.x; i < D; i += kWarps * 32) smem.weight[i] = to_f32<T>(w[i]);
    __syncthreads();
  }
  float2 dwl[4], dwh[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) dwl[i] = dwh[i] = splat(0.f);
  // equal shares of all chunks, to one
  const int64_t all = static_cast<int64_t>(a.B) * a.S * ((heads + L::kRows - 1) / L::kRows), warps = static_cast<int64_t>(a.ctas[t]) * kWarps;
  const int64_t me = static_cast<int64_t>(blockIdx.x - (t ? a.ctas[0] : 0)) * kWarps + warp, first = all * me / warps, n = all * (me + 1) / warps - first;
  if (n > 0) {
    int at = -1;
    T* dx = nullptr;
    stream<T, D, 2>(a, smem, t, first, static_cast<int>(n), [&](int stage, int slot, int token, int h) {
      if (token != at) {
        at = token;
        if (a.y[t]) dx = rows_of<T>(a.y[t], a.ys[t], a.S, at);
      }
      const bool there = h < heads;
      float2 ul[4], uh[4];
      smem.get(stage, 0, 0, ul), smem.get(stage, 0, 1, uh);
      if (a.cos) {
        float2 c[4], s[4];
        L::template get_angles<INTERLEAVED>(smem.angles + slot * D, l, c), L::template get_angles<INTERLEAVED>(smem.angles + slot * D + D / 2, l, s);
        rotate<INTERLEAVED, true>(c, s, ul, uh);
      }
      if (w) {
        float2 xl[4], xh[4], wv[4];
        smem.get(stage, 1, 0, xl), smem.get(stage, 1, 1, xh);
        if (!there) {  // (nothing was asked for: dw must not get what lies there)
#pragma unroll
          for (int i = 0; i < 4; ++i) ul[i] = uh[i] = xl[i] = xh[i] = splat(0.f);
        }
        float2 sq = splat(0.f), ux = splat(0.f);
#pragma unroll
        for (int i = 0; i < 4; ++i) sq = ptx::fma2(xl[i], xl[i], sq);
#pragma unroll
        for (int i = 0; i < 4; ++i) sq = ptx::fma2(xh[i], xh[i], sq);
        float2 pl[4], ph[4];  // u x
        smem.get_weight(0, l, wv);
#pragma unroll
        for (int i = 0; i < 4; ++i) pl[i] = ptx::mul2(ul[i], xl[i]), ux = ptx::fma2(pl[i], wv[i], ux), ul[i] = ptx::mul2(ul[i], wv[i]);
        smem.get_weight(1, l, wv);
#pragma unroll
        for (int i = 0; i < 4; ++i) ph[i] = ptx::mul2(uh[i], xh[i]), ux = ptx::fma2(ph[i], wv[i], ux), uh[i] = ptx::mul2(uh[i], wv[i]);
        float r = rsqrtf(row_sum<L::kLanes>(sq.x + sq.y) * (1.f / D) + a.eps);
        if (!there) r = 0.f;  // (without an eps it would be infinite)
        const float m = row_sum<L::kLanes>(ux.x + ux.y) * (1.f / D);
        const float2 r2 = splat(r), k2 = splat(-(r * m) * (r * r));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          dwl[i] = ptx::fma2(pl[i], r2, dwl[i]), dwh[i] = ptx::fma2(ph[i], r2, dwh[i]);
          ul[i] = ptx::fma2(xl[i], k2, ptx::mul2(ul[i], r2)), uh[i] = ptx::fma2(xh[i], k2, ptx::mul2(uh[i], r2));
        }
      }
      if (dx && there) {
        T* row = dx + h * a.ys[t].h;
        L::store(row, l, ul), L::store(row + D / 2, l, uh);
      }
    });
  }
  // this CTA's share of dw: over the rows of a warp, then its warps, always in the same order
  if (!a.part || !w) return;
  ptx::cp_async_wait();
  __syncthreads();
  float(*s_dw)[D] = reinterpret_cast<float(*)[D]>(raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int of = L::kLanes; of < 32; of <<= 1) {
      dwl[i].x += __shfl_xor_sync(0xffffffffu, dwl[i].x, of), dwl[i].y += __shfl_xor_sync(0xffffffffu, dwl[i].y, of);
      dwh[i].x += __shfl_xor_sync(0xffffffffu, dwh[i].x, of), dwh[i].y += __shfl_xor_sync(0xffffffffu, dwh[i].y, of);
    }
    if (lane < L::kLanes) {
      const int c = L::kVec == 2 ? L::channel(l, i / 2) + i % 2 * 2 : L::channel(l, 0) + i * 2;
      *reinterpret_cast<float2*>(&s_dw[warp][c]) = dwl[i], *reinterpret_cast<float2*>(&s_dw[warp][D / 2 + c]) = dwh[i];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < D; e += kWarps * 32) {
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) x += s_dw[i][e];
    a.part[static_cast<int64_t>(blockIdx.x) * D + e] = x;
  }
}

// dw of q and k: the sums of the CTAs' shares, 16 channels to a CTA (in x; y: q, k) and 64 threads to a channel
template <typename T>
__global__ void __launch_bounds__(1024) norm_rope_dw_kernel(const NormRopeArgs a, int D) {
  __shared__ float s[64][16];
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const int t = blockIdx.y, e = threadIdx.x % 16, r = threadIdx.x / 16, c = blockIdx.x * 16 + e;
  T* dw = reinterpret_cast<T*>(a.dw[t]);
  if (!dw) return;
  const float* p = a.part + static_cast<int64_t>(t ? a.ctas[0] : 0) * D + c;
  float x = 0.f;
#pragma unroll 8
  for (int i = r; i < a.ctas[t]; i += 64) x += p[static_cast<int64_t>(i) * D];
  s[r][e] = x;
  __syncthreads();
  if (r > 0) return;
#pragma unroll 16
  for (int i = 1; i < 64; ++i) x += s[i][e];
  dw[c] = from_f32<T>(x);
}

template <typename T, int D>
cudaError_t launch_fwd(NormRopeArgs a, int device, cudaStream_t stream) {
  // a warp to a token, or, with fewer tokens than warps that the machine holds, as many as it has chunks for
  const int64_t tokens = static_cast<int64_t>(a.B) * a.S, warps = static_cast<int64_t>(kFwdCtas) * kWarps * sm_count(device);
  int64_t ctas = 0;
  for (int t = 0; t < 2; ++t) {
    const int64_t n = (a.heads[t] + Lay<T, D>::kRows - 1) / Lay<T, D>::kRows;
    int64_t want = (warps + tokens - 1) / tokens;
    if (want > n) want = n;
    const int64_t per = (n + want - 1) / want;
    a.split[t] = static_cast<int>((n + per - 1) / per);
    const int64_t c = (tokens * a.split[t] + kWarps - 1) / kWarps;
    if (c > 0x3fffffff / kWarps) return cudaErrorInvalidValue;
    a.ctas[t] = static_cast<int>(c), ctas += c;
  }
  auto kern = a.interleaved ? norm_rope_kernel<T, D, true> : norm_rope_kernel<T, D, false>;
  constexpr int kBytes = Smem<T, D, 1>::kBytes;
  if (kBytes > 48 * 1024)
    if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes); e != cudaSuccess) return e;
  return launch_early(kern, dim3(static_cast<unsigned>(ctas)), dim3(kWarps * 32), kBytes, stream, 1, a);
}

template <typename T, int D>
cudaError_t launch_bwd(NormRopeArgs a, int device, cudaStream_t stream) {
  norm_rope_bwd_ctas(a.B, a.S, a.heads, a.ctas);
  auto kern = a.interleaved ? norm_rope_bwd_kernel<T, D, true> : norm_rope_bwd_kernel<T, D, false>;
  constexpr int kBytes = Smem<T, D, 2>::kBytes;
  if (kBytes > 48 * 1024)
    if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes); e != cudaSuccess) return e;
  cudaError_t e = launch_early(kern, dim3(a.ctas[0] + a.ctas[1]), dim3(kWarps * 32), kBytes, stream, 1, a);
  if (e != cudaSuccess || !a.part) return e;
  return launch_early(norm_rope_dw_kernel<T>, dim3(D / 16, 2), dim3(1024), 0, stream, 1, a, D);
}

template <bool BWD>
cudaError_t launch(int dtype, int D, const NormRopeArgs& a, int device, cudaStream_t stream) {
  auto go = [&](auto t) {
    using T = decltype(t);
    if constexpr (BWD) return D == 64 ? launch_bwd<T, 64>(a, device, stream) : launch_bwd<T, 128>(a, device, stream);
    else return D == 64 ? launch_fwd<T, 64>(a, device, stream) : launch_fwd<T, 128>(a, device, stream);
  };
  if (dtype == TT_ATTN_F32) return go(float{});
  if (dtype == TT_ATTN_F16) return go(__half{});
  return go(__nv_bfloat16{});
}

}  // namespace

// CTAs of the backward for q and k, by their heads: as many as are resident at once, or fewer for little work.  (A token's chunk costs a warp the same
// whether its heads fill it or not: one kv head at D = 64, where a chunk is eight, gets an eighth of q's CTAs and as many chunks: 56 us for 8192 tokens of 8/1 heads.)
void norm_rope_bwd_ctas(int B, int S, const int (&heads)[2], int (&ctas)[2]) {
  const int64_t rows = static_cast<int64_t>(B) * S * (heads[0] + heads[1]);
  int64_t all = (rows + 4 * kWarps - 1) / (4 * kWarps);  // (no fewer than four rows to a warp: a chunk at D = 128, half of one at D = 64)
  if (all > kBwdCtas * kSms) all = kBwdCtas * kSms;
  if (all < 2) all = 2;
  ctas[1] = static_cast<int>(all * heads[1] / (heads[0] + heads[1]));
  if (ctas[1] < 1) ctas[1] = 1;
  ctas[0] = static_cast<int>(all) - ctas[1];
  if (ctas[0] < 1) ctas[0] = 1;
}

cudaError_t launch_norm_rope(int dtype, int D, const NormRopeArgs& a, int device, cudaStream_t stream) {
  return launch<false>(dtype, D, a, device, stream);
}
cudaError_t launch_norm_rope_bwd(int dtype, int D, const NormRopeArgs& a, int device, cudaStream_t stream) {
  return launch<true>(dtype, D, a, device, stream);
}

}  // namespace ttattn
