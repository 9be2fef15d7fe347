// The end of a block and the start of the next, in one pass over a token's D values, and its backward:
//
//   u = Norm(o) w1 + b1;   v = u act(gate);   z = residual + scale v;   n = Norm(z) w2 + b2
//   Norm: (a - mean) r, r = 1 / sqrt(var + eps) (layer), or a r, r = 1 / sqrt(mean(a^2) + eps)
//
//   d  = dz + r2 (g2 - mean(g2) - zh mean(g2 zh)),  g2 = dn w2, zh = Norm(z)        (no mean(g2) without the layer's mean)
//   d residual = d;  d scale = sum d v;  dv = d scale;  d gate = dv u act'(gate);  du = dv act(gate)
//   do = r1 (g1 - mean(g1) - oh mean(g1 oh)),  g1 = du w1, oh = Norm(o);  dw, db: sums over the tokens
//
// Bound by memory.  A token belongs to the fewest threads (a warp or a power of two of them) that hold it with eight values each,
// so that it is read once and its statistics are two passes over registers; tokens of up to 8192 values take sixteen.  The
// backward computes z again from what the forward read (not from the z it wrote, whose rounding would be in the sums), keeps the
// sums over tokens of its columns to itself over all its tokens and leaves them as one part per CTA for an ordered sum.
#include <algorithm>
#include <cstdio>
#include <type_traits>

#include "ttt_elem.cuh"
#include "ttt_sum_parts.h"

namespace {

using namespace ttt;

struct Plan {
  int width;      // threads of a token
  int side;       // tokens next to each other in a CTA
  int ctas;
  float* part;    // backward: [ctas * side][5][D]
};

// A thread holds a token's values in vectors of eight, as four pairs.  Where all rows start on 16-byte boundaries (kVec) a vector is
// eight neighbours, moved as such; otherwise its values are a token's width of threads apart, each moved by itself with the
// warp's others next to it, and some of the last vector's may not be there.
constexpr int N = 4;
using F = float2;

struct Cols {
  int lane, width, D;      // thread among the token's; those; values of a token
  template <bool kVec> __device__ __forceinline__ int at(int j, int e) const {      // column of value e of vector j
    return kVec ? (j * width + lane) * 8 + e : (j * 8 + e) * width + lane;
  }
  template <bool kVec> __device__ __forceinline__ bool in(int j, int e = 0) const { return at<kVec>(j, e) < D; }
};

__device__ __forceinline__ float& half_of(F& f, int e) { return e ? f.y : f.x; }
__device__ __forceinline__ float half_of(const F& f, int e) { return e ? f.y : f.x; }
__device__ __forceinline__ void fill(F (&f)[N], float v) {
#pragma unroll
  for (int k = 0; k < N; ++k) f[k] = both(v);
}

// eight neighbouring values as they lie in memory
template <class T> struct Raw {
  static constexpr int kPieces = static_cast<int>(sizeof(T)) / 2;      // of 16 bytes
  alignas(16) T v[8];
};
template <class T> __device__ __forceinline__ void widen(const Raw<T>& r, F (&f)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) f[k] = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(r.v)[k]);
    else if constexpr (std::is_same<T, __half>::value) f[k] = __half22float2(reinterpret_cast<const __half2*>(r.v)[k]);
    else f[k] = make_float2(r.v[2 * k], r.v[2 * k + 1]);
  }
}
// vector j of a row; values that are not there become `none`
template <bool kVec, class T> __device__ __forceinline__ void load(const T* row, const Cols& c, int j, F (&f)[N], float none = 0.f) {
  if constexpr (kVec) {
    Raw<T> r;
#pragma unroll
    for (int i = 0; i < Raw<T>::kPieces; ++i) reinterpret_cast<uint4*>(r.v)[i] = reinterpret_cast<const uint4*>(row + c.at<true>(j, 0))[i];
    widen(r, f);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) half_of(f[e / 2], e % 2) = c.in<false>(j, e) ? to_f32(row[c.at<false>(j, e)]) : none;
  }
}
template <bool kVec, class T> __device__ __forceinline__ void store(T* row, const Cols& c, int j, const F (&f)[N]) {
  if constexpr (kVec) {
    Raw<T> r;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) reinterpret_cast<__nv_bfloat162*>(r.v)[k] = __float22bfloat162_rn(f[k]);
      else if constexpr (std::is_same<T, __half>::value) reinterpret_cast<__half2*>(r.v)[k] = __float22half2_rn(f[k]);
      else r.v[2 * k] = f[k].x, r.v[2 * k + 1] = f[k].y;
    }
#pragma unroll
    for (int i = 0; i < Raw<T>::kPieces; ++i) reinterpret_cast<uint4*>(row + c.at<true>(j, 0))[i] = reinterpret_cast<const uint4*>(r.v)[i];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c.in<false>(j, e)) row[c.at<false>(j, e)] = from_f32<T>(half_of(f[e / 2], e % 2));
  }
}
// a weight's values, or `none` where there is no such weight
template <bool kVec> __device__ __forceinline__ void weights(const float* p, const Cols& c, int j, float none, F (&f)[N]) {
  if (p) load<kVec>(p, c, j, f, none);
  else fill(f, none);
}

// The gate: its value, and with kSlope its derivative.  GELU as x sigmoid(2 u): no 1 + tanh(u), which cancels on the left.  The
// derivative needs 1 - sigmoid without its cancellation on the right, which is e times sigmoid; the exponent is bounded there so
// that this is not infinity times 0.
template <int kKind, bool kSlope> __device__ __forceinline__ void gate_one(F x, F& v, F& s) {
  constexpr float k = 1.5957691216057308f, c = 0.044715f;      // 2 sqrt(2 / pi)
  F e;
  const F q = times(x, x);
  if constexpr (kKind == TTT_B200_ACT_GELU) e = times(times(x, all<F>(-k * kLog2e)), mac(q, all<F>(c), all<F>(1.f)));
  else e = times(x, all<F>(-kLog2e));
  if constexpr (kSlope) e = least(e, 126.f);
  e = ex2(e);
  const F g = rcp(plus(e, all<F>(1.f)));
  if constexpr (kKind == TTT_B200_ACT_SIGMOID) {
    v = g;
    if constexpr (kSlope) s = times(g, times(e, g));
  } else {
    v = times(x, g);
    if constexpr (kSlope) {
      F o = times(e, g);
      if constexpr (kKind == TTT_B200_ACT_GELU) o = times(o, mac(q, all<F>(3.f * c * k), all<F>(k)));
      s = mac(v, o, g);
    }
  }
}
template <bool kSlope> __device__ __forceinline__ void gate(int kind, const F (&x)[N], F (&v)[N], F (&s)[N]) {
  if (kind == TTT_B200_ACT_SILU) {
#pragma unroll
    for (int k = 0; k < N; ++k) gate_one<TTT_B200_ACT_SILU, kSlope>(x[k], v[k], s[k]);
  } else if (kind == TTT_B200_ACT_GELU) {
#pragma unroll
    for (int k = 0; k < N; ++k) gate_one<TTT_B200_ACT_GELU, kSlope>(x[k], v[k], s[k]);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) gate_one<TTT_B200_ACT_SIGMOID, kSlope>(x[k], v[k], s[k]);
  }
}

// The sums of two values over the threads of a token, in all of them.  `buf` alternates between calls: a barrier lies between two
// uses of the same half.  The lower half of a warp takes the first value, the upper the second, here and across the warps.
__device__ __forceinline__ float2 row_sum(float2 v, float2 (*smem)[32], int& buf, int width) {
  const bool up = threadIdx.x & 16;
  float s = (up ? v.y : v.x) + __shfl_xor_sync(0xffffffffu, up ? v.x : v.y, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (width > 32) {
    const int warp = threadIdx.x >> 5, warps = width >> 5, first = warp & -warps, i = threadIdx.x & 15;
    float* part = reinterpret_cast<float*>(smem[buf]);
    if (i == 0) part[2 * warp + up] = s;
    __syncthreads();
    s = i < warps ? part[2 * (first + i) + up] : 0.f;
    if (warps > 16) s += part[2 * (first + 16 + i) + up];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    buf ^= 1;
  }
  const float other = __shfl_xor_sync(0xffffffffu, s, 16);
  return up ? make_float2(other, s) : make_float2(s, other);
}

// A thread's values of a tensor's rows, token after token at a fixed distance; a tensor that is not there is all zeros.
//   kOwn     vectors of eight: the next row is copied into the thread's own places in shared memory while it works on this one: no
//            barrier, no registers, and past the L1, which keeps the weights
//   kWindow  single values: the next row's 16-byte blocks are copied by the token's threads together (the first and the last may hold
//            neighbours of the row as well), and each value is picked out at the row's offset; needs a barrier in front of `get`
//   kDirect  from global memory
enum { kDirect, kOwn, kWindow };
template <class T, bool kVec, int kMode> struct Feed {
  const T* base;      // NULL: no such tensor
  int64_t stride;
  uint32_t slot;      // shared address of the first stage, the same for all threads
  __host__ __device__ static constexpr uint32_t window(int D) { return (static_cast<uint32_t>(D) * sizeof(T) + 30) / 16 * 16; }
  // bytes of one stage
  __host__ __device__ static uint32_t bytes(int threads, int side, int D) {
    return kMode == kOwn ? 8 * static_cast<int>(sizeof(T)) * threads : kMode == kWindow ? side * window(D) : 0;
  }
  __device__ __forceinline__ Feed(const void* p, int64_t stride, uint32_t& smem, int side, int D) : base(static_cast<const T*>(p)), stride(stride), slot(smem) {
    if (base) smem += 2 * bytes(blockDim.x, side, D);
  }
  __device__ __forceinline__ static uint32_t place(int sub, int D) { return kMode == kOwn ? threadIdx.x * 16 : sub * window(D); }
  // row m into a stage
  __device__ __forceinline__ void ahead(long m, uint32_t to, const Cols& c, int sub) const {
    if (!base) return;
    to += slot + place(sub, c.D);
    if constexpr (kMode == kOwn) {      // (one vector to a thread)
      if (!c.in<true>(0)) return;
      const T* from = base + m * stride + c.at<true>(0, 0);
#pragma unroll
      for (int i = 0; i < Raw<T>::kPieces; ++i) cp_async16_at(to + i * 16 * blockDim.x, from + i * (16 / static_cast<int>(sizeof(T))));
    } else if constexpr (kMode == kWindow) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(base + m * stride), begin = at & ~static_cast<uintptr_t>(15);
      const int span = c.D * static_cast<int>(sizeof(T)) + static_cast<int>(at - begin);
      for (int o = 16 * c.lane; o < span; o += 16 * c.width) cp_async16_at(to + o, reinterpret_cast<const char*>(begin) + o, min(16, span - o));
    }
  }
  // vector j of row m, of which this thread has some
  __device__ __forceinline__ void get(long m, uint32_t from, const Cols& c, int j, int sub, F (&f)[N]) const {
    if (!base) {
      fill(f, 0.f);
    } else if constexpr (kMode == kOwn) {
      Raw<T> r;
#pragma unroll
      for (int i = 0; i < Raw<T>::kPieces; ++i) reinterpret_cast<uint4*>(r.v)[i] = shared_load16(slot + from + place(sub, c.D) + i * 16 * blockDim.x);
      widen(r, f);
    } else if constexpr (kMode == kWindow) {
      const uint32_t at = slot + from + place(sub, c.D) + (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(base + m * stride)) & 15);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        half_of(f[e / 2], e % 2) = c.in<false>(j, e) ? shared_load<T>(at + c.at<false>(j, e) * static_cast<int>(sizeof(T))) : 0.f;
    } else {
      load<kVec>(base + m * stride, c, j, f);
    }
  }
};

// What the threads of a token share: partial sums, in two halves that alternate (a barrier lies between two uses of the same
// one), and how many columns each of its warps has.
struct Shared {
  alignas(16) float2 part[2][32];
  float columns[32];
  float4 stats[2][32];      // backward: each warp's token's
};
template <bool kVec, int NV> __device__ __forceinline__ void count_columns(Shared& sh, const Cols& c) {
  if (threadIdx.x < 32) {
    const int first = 32 * static_cast<int>(threadIdx.x);
    int n = 0;      // of warp threadIdx.x of a token: NV runs of 256, or 8 NV of 32
    if (first < c.width) {
#pragma unroll
      for (int j = 0; j < (kVec ? NV : 8 * NV); ++j) n += min(max(c.D - (j * c.width + first) * (kVec ? 8 : 1), 0), kVec ? 256 : 32);
    }
    sh.columns[threadIdx.x] = static_cast<float>(n);
  }
  __syncthreads();
}

// Mean and 1 / deviation of a row with one barrier: each warp's mean and its squares about it, joined as
// sum over warps of (squares + columns (mean of the warp - mean)^2).
template <bool kVec, int NV>
__device__ __forceinline__ float2 statistics(const F (&a)[NV][N], const ttt_b200_block_args& p, const Cols& c, Shared& sh, int& buf) {
  const int width = c.width;
  const float inv = 1.f / static_cast<float>(p.D);
  float mean = 0.f;
  if (p.layer) {
    F s = all<F>(0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int k = 0; k < N; ++k) s = plus(s, a[j][k]);      // (zeros behind the last column)
    mean = fold(s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, o);
    mean *= rcp(fmaxf(sh.columns[c.lane >> 5], 1.f));
  }
  F sq = both(0.f);
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (c.in<kVec>(j)) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        F v = add2(a[j][k], both(-mean));
        if (!kVec) v = make_float2(c.in<kVec>(j, 2 * k) ? v.x : 0.f, c.in<kVec>(j, 2 * k + 1) ? v.y : 0.f);
        sq = fma2(v, v, sq);
      }
    }
  float q = fold(sq);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
  if (width > 32) {
    const int warp = threadIdx.x >> 5, warps = width >> 5, home = warp & -warps, i = threadIdx.x & 31;
    if (i == 0) sh.part[buf][warp] = make_float2(mean, q);
    __syncthreads();
    const float2 v = i < warps ? sh.part[buf][home + i] : make_float2(0.f, 0.f);      // a lane for each warp
    q = v.y;
    if (p.layer) {
      const float n = sh.columns[i];      // (0 behind the last warp)
      mean = n * v.x;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, o);
      mean *= inv;
      q = fmaf(n * (v.x - mean), v.x - mean, q);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
    buf ^= 1;
  }
  return make_float2(mean, rsqrtf(fmaf(q, inv, p.eps)));
}

template <class T, class R, bool kVec, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) block_forward_kernel(const ttt_b200_block_args p, const Plan q) {
  wait_for_predecessor();
  constexpr int kMode = kVec ? kOwn : kWindow, NV = 1;
  __shared__ Shared sh;
  extern __shared__ __align__(16) unsigned char stages[];
  uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(stages));
  int buf = 0;
  const int lane = threadIdx.x % q.width, sub = threadIdx.x / q.width;
  const Cols c = {lane, q.width, p.D};
  const long step = static_cast<long>(q.ctas) * q.side;
  const Feed<T, kVec, kMode> fo(p.o, p.o_stride, at, q.side, p.D), fg(p.gate, p.gate_stride, at, q.side, p.D);
  const Feed<R, kVec, kMode> fx(p.residual, p.residual_stride, at, q.side, p.D);
  const uint32_t small = Feed<T, kVec, kMode>::bytes(blockDim.x, q.side, p.D), large = Feed<R, kVec, kMode>::bytes(blockDim.x, q.side, p.D);
  auto ahead = [&](long m, int stage) {
    if (m < p.M) {
      fo.ahead(m, stage * small, c, sub);
      fg.ahead(m, stage * small, c, sub);
      fx.ahead(m, stage * large, c, sub);
    }
    cp_async_commit();
  };
  long m = static_cast<long>(blockIdx.x) * q.side + sub;
  ahead(m, 0);
  count_columns<kVec, NV>(sh, c);
  int stage = 0;
  for (long base = static_cast<long>(blockIdx.x) * q.side; base < p.M; base += step, stage ^= 1, m += step) {
    const bool live = m < p.M;
    cp_async_wait<0>();
    if constexpr (kMode == kWindow) __syncthreads();
    ahead(m + step, stage ^ 1);
    F a[NV][N], z[NV][N];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int k = 0; k < N; ++k) a[j][k] = z[j][k] = both(0.f);
      if (live && c.in<kVec>(j)) fo.get(m, stage * small, c, j, sub, a[j]);
    }
    float2 s1 = make_float2(0.f, 1.f), s2 = s1;
    if (p.post_weight) s1 = statistics<kVec, NV>(a, p, c, sh, buf);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!(live && c.in<kVec>(j))) continue;
      F w[N], b[N];
      if (p.post_weight) {
        weights<kVec>(p.post_weight, c, j, 0.f, w);
        weights<kVec>(p.post_bias, c, j, 0.f, b);
#pragma unroll
        for (int k = 0; k < N; ++k) a[j][k] = mac(times(plus(a[j][k], both(-s1.x)), both(s1.y)), w[k], b[k]);
      }
      if (p.gate) {
        F g[N];
        fg.get(m, stage * small, c, j, sub, g);
        gate<false>(p.activation, g, g, w);
#pragma unroll
        for (int k = 0; k < N; ++k) a[j][k] = times(a[j][k], g[k]);
      }
      fx.get(m, stage * large, c, j, sub, z[j]);
      weights<kVec>(p.scale, c, j, 1.f, w);
#pragma unroll
      for (int k = 0; k < N; ++k) z[j][k] = mac(w[k], a[j][k], z[j][k]);
      store<kVec>(static_cast<R*>(p.x) + m * p.D, c, j, z[j]);
    }
    if (p.pre_weight) {
      s2 = statistics<kVec, NV>(z, p, c, sh, buf);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (live && c.in<kVec>(j)) {
          F w[N], b[N];
          weights<kVec>(p.pre_weight, c, j, 0.f, w);
          weights<kVec>(p.pre_bias, c, j, 0.f, b);
#pragma unroll
          for (int k = 0; k < N; ++k) z[j][k] = mac(times(plus(z[j][k], both(-s2.x)), both(s2.y)), w[k], b[k]);
          store<kVec>(static_cast<T*>(p.n) + m * p.D, c, j, z[j]);
        }
      }
    }
    if (p.stats && live && lane == 0) reinterpret_cast<float4*>(p.stats)[m] = make_float4(s1.x, s1.y, s2.x, s2.y);
  }
}

// Sums over tokens of a thread's columns: in registers, or, of sixteen columns, in shared memory.
enum { kDw1, kDb1, kDsc, kDw2, kDb2, kSums };
template <bool kVec, int NV, bool kShared> struct Sums {
  F r[kShared ? 1 : kSums][NV][N];
  float* s;
  __device__ __forceinline__ F get(int k, int j, int i, const Cols& c) const {
    if constexpr (!kShared) return r[k][j][i];
    else if constexpr (kVec) return *reinterpret_cast<const F*>(s + k * c.D + c.at<true>(j, 2 * i));
    else return make_float2(c.in<false>(j, 2 * i) ? s[k * c.D + c.at<false>(j, 2 * i)] : 0.f, c.in<false>(j, 2 * i + 1) ? s[k * c.D + c.at<false>(j, 2 * i + 1)] : 0.f);
  }
  __device__ __forceinline__ void set(int k, int j, int i, const Cols& c, F v) {
    if constexpr (!kShared) {
      r[k][j][i] = v;
    } else if constexpr (kVec) {
      *reinterpret_cast<F*>(s + k * c.D + c.at<true>(j, 2 * i)) = v;
    } else {
      if (c.in<false>(j, 2 * i)) s[k * c.D + c.at<false>(j, 2 * i)] = v.x;
      if (c.in<false>(j, 2 * i + 1)) s[k * c.D + c.at<false>(j, 2 * i + 1)] = v.y;
    }
  }
  __device__ __forceinline__ void add(int k, int j, int i, const Cols& c, F v) { set(k, j, i, c, add2(get(k, j, i, c), v)); }
  __device__ __forceinline__ void add(int k, int j, int i, const Cols& c, F a, F b) { set(k, j, i, c, fma2(a, b, get(k, j, i, c))); }
};

template <class T, class R, bool kVec, int NV, bool kShared, int kThreads>
__global__ void __launch_bounds__(kThreads, kThreads < 512 ? 512 / kThreads : 1) block_backward_kernel(const ttt_b200_block_args p, const Plan q) {
  wait_for_predecessor();
  constexpr int kMode = kShared ? kDirect : kVec ? kOwn : kWindow;
  __shared__ Shared sh;
  extern __shared__ __align__(16) unsigned char stages[];
  uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(stages));
  int buf = 0;
  const int lane = threadIdx.x % q.width, sub = threadIdx.x / q.width;
  const Cols c = {lane, q.width, p.D};
  const long step = static_cast<long>(q.ctas) * q.side;
  const Feed<T, kVec, kMode> fo(p.o, p.o_stride, at, q.side, p.D), fg(p.gate, p.gate_stride, at, q.side, p.D);
  const Feed<T, kVec, kMode> fn(p.pre_weight ? p.grad_n : nullptr, p.gn_stride, at, q.side, p.D);
  const Feed<R, kVec, kMode> fx(p.pre_weight ? p.residual : nullptr, p.residual_stride, at, q.side, p.D);
  const Feed<R, kVec, kMode> fd(p.grad_x, p.gx_stride, at, q.side, p.D);
  const uint32_t small = Feed<T, kVec, kMode>::bytes(blockDim.x, q.side, p.D), large = Feed<R, kVec, kMode>::bytes(blockDim.x, q.side, p.D);
  const uint32_t stats = static_cast<uint32_t>(__cvta_generic_to_shared(&sh.stats[0][threadIdx.x >> 5]));
  auto ahead = [&](long m, int stage) {
    if (m < p.M) {
      if ((threadIdx.x & 31) == 0) cp_async16_at(stats + stage * static_cast<uint32_t>(sizeof(sh.stats[0])), p.stats + 4 * m);
      fo.ahead(m, stage * small, c, sub);
      fg.ahead(m, stage * small, c, sub);
      fn.ahead(m, stage * small, c, sub);
      fx.ahead(m, stage * large, c, sub);
      fd.ahead(m, stage * large, c, sub);
    }
    cp_async_commit();
  };
  const float inv = 1.f / static_cast<float>(p.D);
  Sums<kVec, NV, kShared> sums;
  sums.s = reinterpret_cast<float*>(stages);
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (!kShared || c.in<kVec>(j)) {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int k = 0; k < kSums; ++k) sums.set(k, j, i, c, both(0.f));
    }
  long m = static_cast<long>(blockIdx.x) * q.side + sub;
  ahead(m, 0);
  int stage = 0;
  for (long base = static_cast<long>(blockIdx.x) * q.side; base < p.M; base += step, stage ^= 1, m += step) {
    const bool live = m < p.M;
    cp_async_wait<0>();
    if constexpr (kMode == kWindow) __syncthreads();
    else __syncwarp();
    ahead(m + step, stage ^ 1);
    float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live) st = sh.stats[stage][threadIdx.x >> 5];
    F o[NV][N], z[NV][N], gn[NV][N], d2[NV][N];
    // u (with its norm: oh) and z again, as the forward had them; z is its normalised value
    F sx = both(0.f), sy = sx;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const bool in = live && c.in<kVec>(j);
#pragma unroll
      for (int i = 0; i < N; ++i) o[j][i] = both(0.f);
      if (in) fo.get(m, stage * small, c, j, sub, o[j]);
      if (p.post_weight) {
#pragma unroll
        for (int i = 0; i < N; ++i) o[j][i] = times(plus(o[j][i], both(-st.x)), both(st.y));
      }
      if (!p.pre_weight || !in) continue;
      F u[N], w[N], b[N];
#pragma unroll
      for (int i = 0; i < N; ++i) u[i] = o[j][i];
      if (p.post_weight) {
        weights<kVec>(p.post_weight, c, j, 0.f, w);
        weights<kVec>(p.post_bias, c, j, 0.f, b);
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = mac(o[j][i], w[i], b[i]);
      }
      if (p.gate) {
        fg.get(m, stage * small, c, j, sub, w);
        gate<false>(p.activation, w, w, b);
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = times(u[i], w[i]);
      }
      weights<kVec>(p.scale, c, j, 1.f, w);
      fx.get(m, stage * large, c, j, sub, z[j]);
#pragma unroll
      for (int i = 0; i < N; ++i) z[j][i] = times(plus(mac(w[i], u[i], z[j][i]), both(-st.z)), both(st.w));
      fn.get(m, stage * small, c, j, sub, gn[j]);
      weights<kVec>(p.pre_weight, c, j, 0.f, w);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        sums.add(kDw2, j, i, c, gn[j][i], z[j][i]);
        sums.add(kDb2, j, i, c, gn[j][i]);
        gn[j][i] = times(gn[j][i], w[i]);
        sx = plus(sx, gn[j][i]);
        sy = mac(gn[j][i], z[j][i], sy);
      }
    }
    float2 s = make_float2(fold(sx), fold(sy));
    float m1 = 0.f, m2 = 0.f;
    if (p.pre_weight) {
      s = row_sum(s, sh.part, buf, q.width);
      m1 = p.layer ? s.x * inv : 0.f;
      m2 = s.y * inv;
    }
    sx = sy = both(0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!(live && c.in<kVec>(j))) continue;
      fd.get(m, stage * large, c, j, sub, d2[j]);
      if (p.pre_weight) {
#pragma unroll
        for (int i = 0; i < N; ++i) d2[j][i] = mac(both(st.w), mac(z[j][i], both(-m2), plus(gn[j][i], both(-m1))), d2[j][i]);
      }
      if (p.grad_residual) store<kVec>(static_cast<R*>(p.grad_residual) + m * p.D, c, j, d2[j]);
      F u[N], w[N], b[N], v[N], g[N];
#pragma unroll
      for (int i = 0; i < N; ++i) u[i] = o[j][i];
      if (p.post_weight) {
        weights<kVec>(p.post_weight, c, j, 0.f, w);
        weights<kVec>(p.post_bias, c, j, 0.f, b);
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = mac(o[j][i], w[i], b[i]);
      }
      weights<kVec>(p.scale, c, j, 1.f, b);
      if (p.gate) {
        fg.get(m, stage * small, c, j, sub, g);
        gate<true>(p.activation, g, v, g);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          sums.add(kDsc, j, i, c, d2[j][i], times(u[i], v[i]));
          d2[j][i] = times(d2[j][i], b[i]);
          g[i] = times(times(d2[j][i], u[i]), g[i]);
          d2[j][i] = times(d2[j][i], v[i]);
        }
        store<kVec>(static_cast<T*>(p.grad_gate) + m * p.D, c, j, g);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          sums.add(kDsc, j, i, c, d2[j][i], u[i]);
          d2[j][i] = times(d2[j][i], b[i]);
        }
      }
      if (p.post_weight) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          sums.add(kDw1, j, i, c, d2[j][i], o[j][i]);
          sums.add(kDb1, j, i, c, d2[j][i]);
          d2[j][i] = times(d2[j][i], w[i]);
          sx = plus(sx, d2[j][i]);
          sy = mac(d2[j][i], o[j][i], sy);
        }
      }
    }
    if (p.post_weight) {
      s = row_sum(make_float2(fold(sx), fold(sy)), sh.part, buf, q.width);
      m1 = p.layer ? s.x * inv : 0.f;
      m2 = s.y * inv;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!(live && c.in<kVec>(j))) continue;
      if (p.post_weight) {
#pragma unroll
        for (int i = 0; i < N; ++i) d2[j][i] = times(both(st.y), mac(o[j][i], both(-m2), plus(d2[j][i], both(-m1))));
      }
      store<kVec>(static_cast<T*>(p.grad_o) + m * p.D, c, j, d2[j]);
    }
  }
  float* part = q.part + (static_cast<long>(blockIdx.x) * q.side + sub) * kSums * p.D;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (!c.in<kVec>(j)) continue;
#pragma unroll
    for (int k = 0; k < kSums; ++k) {
      F v[N];
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = sums.get(k, j, i, c);
      store<kVec>(part + static_cast<long>(k) * p.D, c, j, v);
    }
  }
}

// ---- host --------------------------------------------------------------------------------------------------------------
int fail(const char* msg) { return ttt_set_error(TTT_B200_ERR_BAD_ARGS, msg); }

int check(const ttt_b200_block_args* p) {
  if (!p) return fail("block norm: NULL argument struct");
  if (p->M < 0 || p->D < 1 || p->D > 8192) return fail("block norm: M >= 0 and 1 <= D <= 8192");
  if (p->dtype < TTT_B200_BF16 || p->dtype > TTT_B200_FP32) return fail("block norm: unknown element type");
  if (p->activation < TTT_B200_ACT_SILU || p->activation > TTT_B200_ACT_SIGMOID) return fail("block norm: activation is silu, gelu or sigmoid");
  if (!(p->eps >= 0.f)) return fail("block norm: eps must be >= 0");
  if ((p->post_bias && !p->post_weight) || (p->pre_bias && !p->pre_weight)) return fail("block norm: a bias without its weight");
  return TTT_B200_OK;
}

int sm_count() {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// threads of a token: the fewest that hold it with `values` each
int width_of(int D, int values) {
  int w = 32;
  while (w * values < D) w *= 2;
  return w;
}
constexpr int kWide = 4096;      // backward of wider rows: sixteen values to a thread, the sums over tokens in shared memory

// CTAs that are resident together and walk over the tokens: 1024 threads to an SM, backward 512.
void plan(Plan& q, const ttt_b200_block_args& p, bool backward) {
  const bool wide = p.D > kWide;
  q.width = width_of(p.D, wide && backward ? 16 : 8);
  q.side = std::max(1, 128 / q.width);
  const long most = static_cast<long>(sm_count()) * std::max(1, (backward ? 512 : 1024) / (q.width * q.side));
  q.ctas = static_cast<int>(std::min<long>(most, (p.M + q.side - 1) / q.side));
}

bool rows16(const void* p, int64_t stride, size_t es) { return aligned16(p) && stride * static_cast<int64_t>(es) % 16 == 0; }

bool vectors(const ttt_b200_block_args& p, bool backward) {
  const size_t es = p.dtype == TTT_B200_FP32 ? 4 : 2, rs = p.residual_fp32 ? 4 : es;
  bool ok = p.D % 8 == 0 && rows16(p.o, p.o_stride, es) && rows16(p.residual, p.residual_stride, rs) && rows16(p.gate, p.gate_stride, es);
  for (const float* w : {p.post_weight, p.post_bias, p.scale, p.pre_weight, p.pre_bias}) ok = ok && aligned16(w);
  if (backward)
    return ok && rows16(p.grad_x, p.gx_stride, rs) && rows16(p.grad_n, p.gn_stride, es) && aligned16(p.grad_o) && aligned16(p.grad_residual) &&
           aligned16(p.grad_gate);
  return ok && aligned16(p.x) && aligned16(p.n);
}

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return TTT_B200_OK;
  static thread_local char buf[160];
  snprintf(buf, sizeof buf, "%s: %s", what, cudaGetErrorString(e));
  return ttt_set_error(TTT_B200_ERR_LAUNCH, buf);
}

template <class K> int launch(K kernel, const Plan& q, size_t bytes, cudaStream_t s, const ttt_b200_block_args& p, const char* what) {
  if (bytes > 40 * 1024) {      // (with the static part 48 KB is the most without asking)
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (e != cudaSuccess) return ttt_set_error(TTT_B200_ERR_LAUNCH, cudaGetErrorString(e));
  }
  ttt_launch_overlapped(kernel, q.ctas, q.width * q.side, static_cast<uint32_t>(bytes), s, p, q);
  return launched(what);
}

template <class T, class R, bool kVec, int kThreads> int forward_as(const ttt_b200_block_args& p, const Plan& q, cudaStream_t s) {
  constexpr int kMode = kVec ? kOwn : kWindow;
  const int n = q.width * q.side;
  const size_t bytes = 2 * (Feed<T, kVec, kMode>::bytes(n, q.side, p.D) * (1 + (p.gate != nullptr)) +
                            Feed<R, kVec, kMode>::bytes(n, q.side, p.D) * (p.residual != nullptr));
  return launch(block_forward_kernel<T, R, kVec, kThreads>, q, bytes, s, p, "block norm");
}

template <class T, class R> int forward(const ttt_b200_block_args& p, cudaStream_t s) {
  Plan q = {};
  plan(q, p, false);
  const int n = q.width * q.side;
  const bool vec = vectors(p, false);
  if (n <= 128) return vec ? forward_as<T, R, true, 128>(p, q, s) : forward_as<T, R, false, 128>(p, q, s);
  if (n <= 256) return vec ? forward_as<T, R, true, 256>(p, q, s) : forward_as<T, R, false, 256>(p, q, s);
  return vec ? forward_as<T, R, true, 1024>(p, q, s) : forward_as<T, R, false, 1024>(p, q, s);
}

template <class T, class R, bool kVec, int NV, bool kShared, int kThreads> int backward_as(const ttt_b200_block_args& p, const Plan& q, cudaStream_t s) {
  constexpr int kMode = kShared ? kDirect : kVec ? kOwn : kWindow;
  const int n = q.width * q.side;
  const size_t bytes = kShared ? static_cast<size_t>(kSums) * p.D * sizeof(float)
                               : 2 * (Feed<T, kVec, kMode>::bytes(n, q.side, p.D) * (1 + (p.gate != nullptr) + (p.pre_weight && p.grad_n)) +
                                          Feed<R, kVec, kMode>::bytes(n, q.side, p.D) * ((p.pre_weight && p.residual) + (p.grad_x != nullptr)));
  return launch(block_backward_kernel<T, R, kVec, NV, kShared, kThreads>, q, bytes, s, p, "block norm backward");
}

template <class T, class R> int backward(const ttt_b200_block_args& p, cudaStream_t s) {
  Plan q = {};
  plan(q, p, true);
  q.part = static_cast<float*>(p.scratch);
  const bool vec = vectors(p, true);
  const int n = q.width * q.side;
  int rc;
  if (p.D > kWide) rc = vec ? backward_as<T, R, true, 2, true, 512>(p, q, s) : backward_as<T, R, false, 2, true, 512>(p, q, s);
  else if (n <= 128) rc = vec ? backward_as<T, R, true, 1, false, 128>(p, q, s) : backward_as<T, R, false, 1, false, 128>(p, q, s);
  else if (n <= 256) rc = vec ? backward_as<T, R, true, 1, false, 256>(p, q, s) : backward_as<T, R, false, 1, false, 256>(p, q, s);
  else rc = vec ? backward_as<T, R, true, 1, false, 512>(p, q, s) : backward_as<T, R, false, 1, false, 512>(p, q, s);
  if (rc) return rc;
  const long row = static_cast<long>(kSums) * p.D;
  float* dst[kSums] = {p.grad_post_weight, p.grad_post_bias, p.grad_scale, p.grad_pre_weight, p.grad_pre_bias};
  ttt_sum_job jobs[kSums];
  for (int k = 0; k < kSums; ++k)
    jobs[k] = {q.part + static_cast<long>(k) * p.D, dst[k], p.D, row, q.ctas * q.side, TTT_B200_FP32, 0};
  return ttt_sum_parts(jobs, kSums, s);
}

}  // namespace

extern "C" uint64_t ttt_b200_norm_gate_residual_scratch_bytes(const ttt_b200_block_args* p) {
  if (check(p) || p->M == 0) return 0;
  Plan q = {};
  plan(q, *p, true);
  return static_cast<uint64_t>(q.ctas) * q.side * kSums * p->D * sizeof(float);
}

extern "C" int ttt_b200_norm_gate_residual(const ttt_b200_block_args* p, void* stream) {
  if (int rc = check(p)) return rc;
  if (!p->o || !p->x || (p->pre_weight && !p->n)) return fail("block norm: null tensor pointer");
  if (p->stats && !aligned16(p->stats)) return fail("block norm: stats must be 16-byte aligned");
  if (p->M == 0) return fail("block norm: no tokens");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  TTT_WITH_TYPE(p->dtype, return p->residual_fp32 ? (forward<Elem, float>(*p, s)) : (forward<Elem, Elem>(*p, s)))
  return TTT_B200_OK;
}

extern "C" int ttt_b200_norm_gate_residual_backward(const ttt_b200_block_args* p, void* stream) {
  if (int rc = check(p)) return rc;
  if (!p->o || !p->stats || !p->grad_o || (!p->grad_x && !p->grad_n)) return fail("block norm backward: null tensor pointer");
  if (!aligned16(p->stats)) return fail("block norm backward: stats must be 16-byte aligned");
  if (p->M == 0) return fail("block norm backward: no tokens");
  if (!p->scratch || p->scratch_bytes < ttt_b200_norm_gate_residual_scratch_bytes(p) || !aligned16(p->scratch))
    return fail("block norm backward: scratch is missing, too small or not 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  TTT_WITH_TYPE(p->dtype, return p->residual_fp32 ? (backward<Elem, float>(*p, s)) : (backward<Elem, Elem>(*p, s)))
  return TTT_B200_OK;
}
