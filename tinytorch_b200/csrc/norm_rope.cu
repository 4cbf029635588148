// The RMS norm of every head of q and k and the rotation of its channel pairs to the token's position, in one pass.
//
//   n = x * rsqrt(mean(x^2) + eps),  y = n * w            (skipped where there is no weight)
//   (a, b) -> (a cos - b sin, b cos + a sin)              for every pair of channels (skipped where there are no tables)
//
// and its gradients: with u = the output's gradient, turned back by the same angles,
//   dw = sum over tokens and heads of u * n,   dx = r (g - n mean(g n)),   g = u * w,  r = rsqrt(mean(x^2) + eps)
// r is computed again from x, which has to be read anyway: nothing but the inputs is kept for the backward.  All in fp32,
// with one rounding to the tensor type of each value stored.
//
// Bound by memory: x in and y out (backward: x and dy in, dx out).  A row of D channels belongs to D / 16 neighbouring
// lanes, each with 8 channels of the first and 8 of the second half, so that a pair (i, i + D/2) or (2i, 2i + 1) never leaves
// a thread, every access is a 16-byte vector of a 64- or 128-byte run, and the mean takes two or three shuffles.  A warp
// takes 512 / D heads of one token at a time and several such chunks in turn, two of them in flight: positions, angles and their
// 512 bytes a token are fetched once for all of these.  With few tokens the chunks are divided among more warps.
#include <type_traits>

#include "common.cuh"
#include "norm_rope.cuh"
#include "tma_host.cuh"

namespace ttattn {
namespace {

constexpr int kWarps = 4;  // per CTA
constexpr int kInFlight = 2;  // chunks whose rows are loaded together

// 8 channels of a row
template <typename T>
struct Vec8 {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (size_t i = 0; i < sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (size_t i = 0; i < sizeof(T) / 2; ++i) w[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const T* t = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_f32<T>(t[i]);
  }
};
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  Vec8<T> v;
  T* t = reinterpret_cast<T*>(v.w);
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = from_f32<T>(f[i]);
#pragma unroll
  for (size_t i = 0; i < sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = v.w[i];
}

// cos and sin of this lane's 8 pairs.  Pairs (i, i + D/2): i = 8 l ... 8 l + 7, the same channels of both halves.  Pairs
// (2i, 2i + 1): four in the lane's channels of the first half, four in those of the second.
struct Angles {
  float c[8], s[8];
};

// Four consecutive pairs, the first of them `pair`.  A position outside the tables turns nothing and is reported.
template <int D>
__device__ __forceinline__ void four_angles(const NormRopeArgs& a, const int (&pos)[kMaxAxes], int pair, float* c, float* s, bool& outside) {
  auto axis_of = [&](int i) {
    int x = 0;
#pragma unroll
    for (int e = 0; e + 1 < kMaxAxes; ++e) x += i >= a.axis_end[e];
    return x;
  };
  auto position = [&](int x) {
    int p = pos[0];
#pragma unroll
    for (int e = 1; e < kMaxAxes; ++e) p = x == e ? pos[e] : p;
    return p;
  };
  const int x0 = axis_of(pair), x3 = axis_of(pair + 3);
  if (x0 == x3) {  // (always, with one axis)
    const int p = position(x0);
    if (p >= 0 && p < a.rope_positions) {
      const int64_t at = static_cast<int64_t>(p) * (D / 2) + pair;
      const float4 cv = __ldg(reinterpret_cast<const float4*>(a.cos + at)), sv = __ldg(reinterpret_cast<const float4*>(a.sin + at));
      c[0] = cv.x, c[1] = cv.y, c[2] = cv.z, c[3] = cv.w;
      s[0] = sv.x, s[1] = sv.y, s[2] = sv.z, s[3] = sv.w;
    } else {
      outside = true;
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = 1.f, s[i] = 0.f;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = position(axis_of(pair + i));
    const bool in = p >= 0 && p < a.rope_positions;
    const int64_t at = static_cast<int64_t>(p) * (D / 2) + pair + i;
    c[i] = in ? __ldg(a.cos + at) : 1.f;
    s[i] = in ? __ldg(a.sin + at) : 0.f;
    outside |= !in;
  }
}

template <int D>
__device__ __forceinline__ void load_angles(const NormRopeArgs& a, int b, int row, int l, Angles& g) {
  int pos[kMaxAxes];
#pragma unroll
  for (int e = 0; e < kMaxAxes; ++e) pos[e] = e < a.axes ? __ldg(a.positions + e * a.pos_axis + b * a.pos_b + row) : 0;
  bool outside = false;
  four_angles<D>(a, pos, a.interleaved ? l * 4 : l * 8, g.c, g.s, outside);
  four_angles<D>(a, pos, a.interleaved ? D / 4 + l * 4 : l * 8 + 4, g.c + 4, g.s + 4, outside);
  if (outside && a.status) atomicOr(a.status, kStatusRopeRange);
}

// lo: channels 8 l .. 8 l + 7, hi: D/2 + those; `back`: by the negative angles
__device__ __forceinline__ void rotate(float (&lo)[8], float (&hi)[8], const Angles& g, bool interleaved, float back) {
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float sl = g.s[i] * back, sh = g.s[4 + i] * back;
      const float x = lo[2 * i], y = lo[2 * i + 1], u = hi[2 * i], v = hi[2 * i + 1];
      lo[2 * i] = x * g.c[i] - y * sl, lo[2 * i + 1] = y * g.c[i] + x * sl;
      hi[2 * i] = u * g.c[4 + i] - v * sh, hi[2 * i + 1] = v * g.c[4 + i] + u * sh;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = lo[i], y = hi[i], s = g.s[i] * back;
      lo[i] = x * g.c[i] - y * s, hi[i] = y * g.c[i] + x * s;
    }
  }
}

template <int LANES>
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int of = LANES / 2; of >= 1; of >>= 1) x += __shfl_xor_sync(0xffffffffu, x, of);
  return x;
}

// A warp's share of the work: the chunks [c0, c1) of heads of one token, of q (t = 0) or k (t = 1).
struct Unit {
  int b, row, c0, c1;
};
__device__ __forceinline__ Unit unit_of(const NormRopeArgs& a, int t, int64_t u, int heads_per_chunk) {
  const int64_t token = u / a.split[t];
  const int part = static_cast<int>(u - token * a.split[t]);
  Unit r;
  r.b = static_cast<int>(token / a.S), r.row = static_cast<int>(token - static_cast<int64_t>(r.b) * a.S);
  const int n = (a.heads[t] + heads_per_chunk - 1) / heads_per_chunk, per = (n + a.split[t] - 1) / a.split[t];
  r.c0 = part * per, r.c1 = r.c0 + per < n ? r.c0 + per : n;
  return r;
}

template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32) norm_rope_kernel(const NormRopeArgs a) {
  constexpr int LANES = D / 16, ROWS = 32 / LANES;
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const int lane = threadIdx.x & 31, l = lane % LANES, sub = lane / LANES;
  const int t = static_cast<int>(blockIdx.x) >= a.ctas[0];
  const int64_t u = static_cast<int64_t>(blockIdx.x - (t ? a.ctas[0] : 0)) * kWarps + (threadIdx.x >> 5);
  if (u >= static_cast<int64_t>(a.B) * a.S * a.split[t]) return;
  const Unit un = unit_of(a, t, u, ROWS);
  const T* x = reinterpret_cast<const T*>(a.x[t]) + un.b * a.xs[t].b + un.row * a.xs[t].s + l * 8;
  T* y = reinterpret_cast<T*>(a.y[t]) + un.b * a.ys[t].b + un.row * a.ys[t].s + l * 8;
  const T* w = reinterpret_cast<const T*>(a.w[t]);
  Vec8<T> v[kInFlight][2];
  auto load = [&](int c) {
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      const int h = (c + i) * ROWS + sub;
      if (c + i < un.c1 && h < a.heads[t]) v[i][0].load(x + h * a.xs[t].h), v[i][1].load(x + h * a.xs[t].h + D / 2);
      else v[i][0].zero(), v[i][1].zero();
    }
  };
  load(un.c0);
  Angles g;
  if (a.cos) load_angles<D>(a, un.b, un.row, l, g);
  for (int c = un.c0; c < un.c1; c += kInFlight) {
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      if (c + i >= un.c1) break;
      const int h = (c + i) * ROWS + sub;
      float lo[8], hi[8];
      v[i][0].get(lo), v[i][1].get(hi);
      if (w) {
        float sq = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) sq = fmaf(lo[e], lo[e], fmaf(hi[e], hi[e], sq));
        const float r = rsqrtf(row_sum<LANES>(sq) * (1.f / D) + a.eps);
        float wl[8], wh[8];
        Vec8<T> wv;
        wv.load(w + l * 8), wv.get(wl), wv.load(w + D / 2 + l * 8), wv.get(wh);
#pragma unroll
        for (int e = 0; e < 8; ++e) lo[e] *= r * wl[e], hi[e] *= r * wh[e];
      }
      if (a.cos) rotate(lo, hi, g, a.interleaved, 1.f);
      if (h < a.heads[t]) store8(y + h * a.ys[t].h, lo), store8(y + h * a.ys[t].h + D / 2, hi);
    }
    if (c + kInFlight < un.c1) load(c + kInFlight);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32) norm_rope_bwd_kernel(const NormRopeArgs a) {
  constexpr int LANES = D / 16, ROWS = 32 / LANES;
  __shared__ float s_dw[kWarps][D];
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % LANES, sub = lane / LANES;
  const int t = static_cast<int>(blockIdx.x) >= a.ctas[0];
  const int64_t units = static_cast<int64_t>(a.B) * a.S * a.split[t];
  const T* w = reinterpret_cast<const T*>(a.w[t]);
  float dwl[8], dwh[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) dwl[e] = dwh[e] = 0.f;
  for (int64_t u = static_cast<int64_t>(blockIdx.x - (t ? a.ctas[0] : 0)) * kWarps + warp; u < units; u += static_cast<int64_t>(a.ctas[t]) * kWarps) {
    const Unit un = unit_of(a, t, u, ROWS);
    const T* x = reinterpret_cast<const T*>(a.x[t]) + un.b * a.xs[t].b + un.row * a.xs[t].s + l * 8;
    const T* dy = reinterpret_cast<const T*>(a.dy[t]) + un.b * a.dys[t].b + un.row * a.dys[t].s + l * 8;
    T* dx = a.y[t] ? reinterpret_cast<T*>(a.y[t]) + un.b * a.ys[t].b + un.row * a.ys[t].s + l * 8 : nullptr;
    Angles g;
    if (a.cos) load_angles<D>(a, un.b, un.row, l, g);
    for (int c = un.c0; c < un.c1; c += kInFlight) {
      Vec8<T> v[kInFlight][2], d[kInFlight][2];
#pragma unroll
      for (int i = 0; i < kInFlight; ++i) {
        const int h = (c + i) * ROWS + sub;
        if (c + i < un.c1 && h < a.heads[t]) {
          d[i][0].load(dy + h * a.dys[t].h), d[i][1].load(dy + h * a.dys[t].h + D / 2);
          if (w) v[i][0].load(x + h * a.xs[t].h), v[i][1].load(x + h * a.xs[t].h + D / 2);
        } else {  // (rows of zeros: they add nothing to dw)
          v[i][0].zero(), v[i][1].zero(), d[i][0].zero(), d[i][1].zero();
        }
      }
#pragma unroll
      for (int i = 0; i < kInFlight; ++i) {
        if (c + i >= un.c1) break;
        const int h = (c + i) * ROWS + sub;
        float ul[8], uh[8];
        d[i][0].get(ul), d[i][1].get(uh);
        if (a.cos) rotate(ul, uh, g, a.interleaved, -1.f);
        if (w) {
          float nl[8], nh[8], wl[8], wh[8];
          v[i][0].get(nl), v[i][1].get(nh);
          float sq = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) sq = fmaf(nl[e], nl[e], fmaf(nh[e], nh[e], sq));
          float r = rsqrtf(row_sum<LANES>(sq) * (1.f / D) + a.eps);
          if (h >= a.heads[t]) r = 0.f;  // (no row: without an eps, r would be infinite)
          Vec8<T> wv;
          wv.load(w + l * 8), wv.get(wl), wv.load(w + D / 2 + l * 8), wv.get(wh);
          float gn = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            nl[e] *= r, nh[e] *= r;
            dwl[e] = fmaf(ul[e], nl[e], dwl[e]), dwh[e] = fmaf(uh[e], nh[e], dwh[e]);
            ul[e] *= wl[e], uh[e] *= wh[e];
            gn = fmaf(ul[e], nl[e], fmaf(uh[e], nh[e], gn));
          }
          gn = row_sum<LANES>(gn) * (1.f / D);
#pragma unroll
          for (int e = 0; e < 8; ++e) ul[e] = r * fmaf(-nl[e], gn, ul[e]), uh[e] = r * fmaf(-nh[e], gn, uh[e]);
        }
        if (dx && h < a.heads[t]) store8(dx + h * a.ys[t].h, ul), store8(dx + h * a.ys[t].h + D / 2, uh);
      }
    }
  }
  // this CTA's share of dw: over the rows of a warp, then its warps, always in the same order
  if (!a.part || !w) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
#pragma unroll
    for (int of = LANES; of < 32; of <<= 1) {
      dwl[e] += __shfl_xor_sync(0xffffffffu, dwl[e], of);
      dwh[e] += __shfl_xor_sync(0xffffffffu, dwh[e], of);
    }
    if (sub == 0) s_dw[warp][l * 8 + e] = dwl[e], s_dw[warp][D / 2 + l * 8 + e] = dwh[e];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < D; e += kWarps * 32) {
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) x += s_dw[i][e];
    a.part[static_cast<int64_t>(blockIdx.x) * D + e] = x;
  }
}

// dw of q (CTA 0) and k (CTA 1): the sum of the CTAs' shares
template <typename T, int D>
__global__ void __launch_bounds__(1024) norm_rope_dw_kernel(const NormRopeArgs a) {
  constexpr int R = 1024 / D;
  __shared__ float s[R][D];
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const int t = blockIdx.x, e = threadIdx.x % D, r = threadIdx.x / D;
  T* dw = reinterpret_cast<T*>(a.dw[t]);
  if (!dw) return;
  const float* p = a.part + static_cast<int64_t>(t ? a.ctas[0] : 0) * D + e;
  float x = 0.f;
#pragma unroll 8
  for (int i = r; i < a.ctas[t]; i += R) x += p[static_cast<int64_t>(i) * D];
  s[r][e] = x;
  __syncthreads();
  if (r > 0) return;
#pragma unroll
  for (int i = 1; i < R; ++i) x += s[i][e];
  dw[e] = from_f32<T>(x);
}

// How many warps divide the chunks of a token: one, with enough tokens to fill the machine (32 warps an SM).
void plan_units(NormRopeArgs* a, int D, int sms) {
  const int rows = 32 / (D / 16);
  const int64_t tokens = static_cast<int64_t>(a->B) * a->S > 0 ? static_cast<int64_t>(a->B) * a->S : 1;
  for (int t = 0; t < 2; ++t) {
    const int n = (a->heads[t] + rows - 1) / rows;
    int64_t want = (32ll * sms + tokens - 1) / tokens;
    if (want > n) want = n;
    const int per = static_cast<int>((n + want - 1) / want);  // chunks of a unit
    a->split[t] = (n + per - 1) / per;
  }
}

template <typename T, int D>
cudaError_t launch_fwd(NormRopeArgs a, int device, cudaStream_t stream) {
  plan_units(&a, D, sm_count(device));
  int64_t ctas = 0;
  for (int t = 0; t < 2; ++t) {
    const int64_t n = (static_cast<int64_t>(a.B) * a.S * a.split[t] + kWarps - 1) / kWarps;
    if (n > 0x3fffffff) return cudaErrorInvalidValue;
    a.ctas[t] = static_cast<int>(n), ctas += n;
  }
  return launch_early(norm_rope_kernel<T, D>, dim3(static_cast<unsigned>(ctas)), dim3(kWarps * 32), 0, stream, 1, a);
}

template <typename T, int D>
cudaError_t launch_bwd(NormRopeArgs a, int device, cudaStream_t stream) {
  plan_units(&a, D, sm_count(device));
  norm_rope_bwd_ctas(a.B, a.S, a.heads, a.ctas);
  cudaError_t e = launch_early(norm_rope_bwd_kernel<T, D>, dim3(a.ctas[0] + a.ctas[1]), dim3(kWarps * 32), 0, stream, 1, a);
  if (e != cudaSuccess || !a.part) return e;
  return launch_early(norm_rope_dw_kernel<T, D>, dim3(2), dim3(1024), 0, stream, 1, a);
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

// CTAs of the backward for q and k, by their heads: as many as are resident at once, or fewer for little work.
void norm_rope_bwd_ctas(int B, int S, const int (&heads)[2], int (&ctas)[2]) {
  const int64_t rows = static_cast<int64_t>(B) * S * (heads[0] + heads[1]);
  int64_t all = (rows + 2 * kWarps - 1) / (2 * kWarps);  // (no fewer than two rows to a warp)
  if (all > 8 * kSms) all = 8 * kSms;
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
