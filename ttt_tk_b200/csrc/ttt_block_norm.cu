// The end of a block and the start of the next, in one pass over a token's D values, and its backward:
//
//   u = Norm(o) w1 + b1;   v = u act(gate);   z = residual + scale v;   n = Norm(z) w2 + b2
//   Norm: (a - mean) r, r = 1 / sqrt(var + eps) (layer), or a r, r = 1 / sqrt(mean(a^2) + eps)
//
//   d  = dz + r2 (g2 - mean(g2) - zh mean(g2 zh)),  g2 = dn w2, zh = Norm(z)        (no mean(g2) without the layer's mean)
//   d residual = d;  d scale = sum d v;  dv = d scale;  d gate = dv u act'(gate);  du = dv act(gate)
//   do = r1 (g1 - mean(g1) - oh mean(g1 oh)),  g1 = du w1, oh = Norm(o);  dw, db: sums over the tokens
//
// A token belongs to the fewest threads (a warp or a power of two of them) that hold it with eight values each (backward of more
// than 4096: sixteen), so that it is read once and its statistics are two passes over registers.  The backward computes z again from
// what the forward read (not from the z it wrote, whose rounding would be in the sums), keeps the sums over tokens of its columns to
// itself over all its tokens and leaves them as one part per CTA for an ordered sum.
//
// Measured, fp32 residual stream, layer norms, all weights, tanh gate, 16384 x 2048 bf16: forward 97 us (4.8 TB/s), backward 191 us
// (3.9 TB/s); bf16 residual, RMS norms 77 us (4.4) and 185 us (2.9); rows of 2047 117 and 256 us; 4096 x 8192, layer norms, 114 us
// (2.9) and 372 us (1.4).  Not memory but issued instructions and the wait at a token's barriers hold them: 1024 threads to an SM
// forward (1280: 106 us, the L1 has less room for the weights), 512 backward (128 registers, 40 of them sums over tokens).  So the
// width is a constant of the kernel (118 -> 104 and 230 -> 211 us; rows of 2047 174 -> 118 and 349 -> 257).
#include <algorithm>
#include <cstdio>
#include <type_traits>

#include "ttt_elem.cuh"
#include "ttt_sum_parts.h"

namespace {

using namespace ttt;

struct Plan {
  int width;      // threads of a token
  int ctas;
  float* part;    // backward: [ctas * tokens next to each other][5][D]
};
constexpr int side_of(int width) { return width < 128 ? 128 / width : 1; }      // tokens next to each other in a CTA

// A thread holds a token's values in vectors of eight, as four pairs: V neighbours, a token's width of threads from the next V.
//   V = 8  where nothing but the weights is fp32
//   V = 4  with an fp32 residual stream: a warp's 16-byte accesses to fp32 are then whole lines, where eight neighbours took the L1
//          twice as many cycles.  16384 x 2048, forward and backward: 128 -> 118 and 262 -> 230 us; with a bf16 residual, whose
//          rows then take twice as many accesses, 78 -> 95 and 209 -> 241 us, so there V stays 8.
//   V = 1  where a row does not start on a boundary of V values
// The last runs of a token may not be there, unless its values fill its threads (kFull): no comparisons and selections then,
// forward and backward 104 -> 97 and 211 -> 191 us of the first, 79 -> 77 and 187 -> 185 of the second.
constexpr int N = 4;
using F = float2;

template <int kRun, int kWidth, bool kFull> struct Cols {
  static constexpr int V = kRun, width = kWidth, side = side_of(kWidth), threads = width * side;
  int lane, D;      // thread among the token's; values of a token
  __device__ __forceinline__ int at(int j, int e) const { return ((j * (8 / V) + e / V) * width + lane) * V + e % V; }      // column of value e of vector j
  __device__ __forceinline__ bool in(int j, int e = 0) const { return kFull || at(j, e - e % V) < D; }
};

__device__ __forceinline__ float& half_of(F& f, int e) { return e ? f.y : f.x; }
__device__ __forceinline__ float half_of(const F& f, int e) { return e ? f.y : f.x; }
__device__ __forceinline__ void fill(F (&f)[N], float v) {
#pragma unroll
  for (int k = 0; k < N; ++k) f[k] = both(v);
}

// V neighbouring values as they lie in memory, in pieces of up to 16 bytes
template <class T, int V> struct Raw {
  using Piece = typename std::conditional<V * sizeof(T) >= 16, uint4, uint2>::type;
  static constexpr int kPieces = V * sizeof(T) / sizeof(Piece);
  alignas(16) T v[V];
  __device__ __forceinline__ Piece& piece(int i) { return reinterpret_cast<Piece*>(v)[i]; }
  __device__ __forceinline__ F pair(int k) const {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) return __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(v)[k]);
    else if constexpr (std::is_same<T, __half>::value) return __half22float2(reinterpret_cast<const __half2*>(v)[k]);
    else return make_float2(v[2 * k], v[2 * k + 1]);
  }
  __device__ __forceinline__ void pair(int k, F f) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) reinterpret_cast<__nv_bfloat162*>(v)[k] = __float22bfloat162_rn(f);
    else if constexpr (std::is_same<T, __half>::value) reinterpret_cast<__half2*>(v)[k] = __float22half2_rn(f);
    else v[2 * k] = f.x, v[2 * k + 1] = f.y;
  }
};
// vector j of a row; values that are not there become `none`
template <class C, class T> __device__ __forceinline__ void load(const T* row, const C& c, int j, F (&f)[N], float none = 0.f) {
  constexpr int V = C::V;
  if constexpr (V > 1) {
#pragma unroll
    for (int e = 0; e < 8; e += V) {
      Raw<T, V> r;
      const bool in = V == 8 || c.in(j, e);      // (the first run of a vector is there)
      if (in) {
#pragma unroll
        for (int i = 0; i < r.kPieces; ++i) r.piece(i) = reinterpret_cast<const typename Raw<T, V>::Piece*>(row + c.at(j, e))[i];
      }
#pragma unroll
      for (int k = 0; k < V / 2; ++k) f[e / 2 + k] = in ? r.pair(k) : both(none);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) half_of(f[e / 2], e % 2) = c.in(j, e) ? to_f32(row[c.at(j, e)]) : none;
  }
}
template <class C, class T> __device__ __forceinline__ void store(T* row, const C& c, int j, const F (&f)[N]) {
  constexpr int V = C::V;
  if constexpr (V > 1) {
#pragma unroll
    for (int e = 0; e < 8; e += V) {
      if (V < 8 && !c.in(j, e)) continue;
      Raw<T, V> r;
#pragma unroll
      for (int k = 0; k < V / 2; ++k) r.pair(k, f[e / 2 + k]);
#pragma unroll
      for (int i = 0; i < r.kPieces; ++i) reinterpret_cast<typename Raw<T, V>::Piece*>(row + c.at(j, e))[i] = r.piece(i);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c.in(j, e)) row[c.at(j, e)] = from_f32<T>(half_of(f[e / 2], e % 2));
  }
}
// a weight's values, or `none` where there is no such weight
template <class C> __device__ __forceinline__ void weights(const float* p, const C& c, int j, float none, F (&f)[N]) {
  if (p) load(p, c, j, f, none);
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
template <class C> __device__ __forceinline__ float2 row_sum(float2 v, float2 (*smem)[32], int& buf) {
  const bool up = threadIdx.x & 16;
  float s = (up ? v.y : v.x) + __shfl_xor_sync(0xffffffffu, up ? v.x : v.y, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if constexpr (C::width > 32) {
    constexpr int warps = C::width / 32;
    static_assert(warps <= 16, "half a warp has a lane for each warp");
    const int warp = threadIdx.x >> 5, first = warp & -warps, i = threadIdx.x & 15;
    float* part = reinterpret_cast<float*>(smem[buf]);
    if (i == 0) part[2 * warp + up] = s;
    __syncthreads();
    s = part[2 * (first + i % warps) + up];
#pragma unroll
    for (int o = warps / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    buf ^= 1;
  }
  const float other = __shfl_xor_sync(0xffffffffu, s, 16);
  return up ? make_float2(other, s) : make_float2(s, other);
}

// A thread's values of a tensor's rows, token after token at a fixed distance; a tensor that is not there is all zeros.
//   kOwn     vectors: the next row is copied into the thread's own places in shared memory while it works on this one: no
//            barrier, no registers, and past the L1, which keeps the weights
//   kWindow  V = 1: the next row's 16-byte blocks are copied by the token's threads together (the first and the last may hold
//            neighbours of the row as well), and each value is picked out at the row's offset; needs a barrier in front of `get`
//   kDirect  from global memory
enum { kDirect, kOwn, kWindow };
template <class T, class C, int kMode> struct Feed {
  static constexpr int V = C::V;
  static constexpr int kRun = V * static_cast<int>(sizeof(T));      // kOwn: 8 or 16 bytes
  static_assert(kMode != kOwn || kRun == 8 || kRun == 16, "a run is one copy");
  const T* base;      // NULL: no such tensor
  int64_t stride;
  uint32_t slot;      // shared address of the first stage, the same for all threads
  __host__ __device__ static constexpr uint32_t window(int D) { return (static_cast<uint32_t>(D) * sizeof(T) + 30) / 16 * 16; }
  // bytes of one stage
  __host__ __device__ static constexpr uint32_t bytes(int D) {
    return kMode == kOwn ? 8 * static_cast<int>(sizeof(T)) * C::threads : kMode == kWindow ? C::side * window(D) : 0;
  }
  __device__ __forceinline__ Feed(const void* p, int64_t stride, uint32_t& smem, int D) : base(static_cast<const T*>(p)), stride(stride), slot(smem) {
    if (base) smem += 2 * bytes(D);
  }
  __device__ __forceinline__ static uint32_t place(int sub, int D) { return kMode == kOwn ? threadIdx.x * kRun : sub * window(D); }
  // row m into a stage
  __device__ __forceinline__ void ahead(long m, uint32_t to, const C& c, int sub) const {
    if (!base) return;
    to += slot + place(sub, c.D);
    if constexpr (kMode == kOwn) {      // (one vector to a thread)
#pragma unroll
      for (int e = 0; e < 8; e += V) {
        if (!c.in(0, e)) continue;
        const T* from = base + m * stride + c.at(0, e);
        if constexpr (kRun == 16) cp_async16_at(to + e / V * kRun * C::threads, from);
        else cp_async8_at(to + e / V * kRun * C::threads, from);
      }
    } else if constexpr (kMode == kWindow) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(base + m * stride), begin = at & ~static_cast<uintptr_t>(15);
      const int span = c.D * static_cast<int>(sizeof(T)) + static_cast<int>(at - begin);
      for (int o = 16 * c.lane; o < span; o += 16 * c.width) cp_async16_at(to + o, reinterpret_cast<const char*>(begin) + o, min(16, span - o));
    }
  }
  // vector j of row m, of which this thread has some
  __device__ __forceinline__ void get(long m, uint32_t from, const C& c, int j, int sub, F (&f)[N]) const {
    if (!base) {
      fill(f, 0.f);
    } else if constexpr (kMode == kOwn) {
#pragma unroll
      for (int e = 0; e < 8; e += V) {
        Raw<T, V> r;
        const uint32_t at = slot + from + place(sub, c.D) + e / V * kRun * C::threads;
        if constexpr (kRun == 16) r.piece(0) = shared_load16(at);
        else r.piece(0) = shared_load8(at);
#pragma unroll
        for (int k = 0; k < V / 2; ++k) f[e / 2 + k] = V == 8 || c.in(0, e) ? r.pair(k) : both(0.f);
      }
    } else if constexpr (kMode == kWindow) {
      const uint32_t at = slot + from + place(sub, c.D) + (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(base + m * stride)) & 15);
#pragma unroll
      for (int e = 0; e < 8; ++e) half_of(f[e / 2], e % 2) = c.in(j, e) ? shared_load<T>(at + c.at(j, e) * static_cast<int>(sizeof(T))) : 0.f;
    } else {
      load(base + m * stride, c, j, f);
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
template <int NV, class C> __device__ __forceinline__ void count_columns(Shared& sh, const C& c) {
  constexpr int V = C::V;
  if (threadIdx.x < 32) {
    const int first = 32 * static_cast<int>(threadIdx.x);
    int n = 0;      // of warp threadIdx.x of a token: runs of 32 threads' values
    if (first < c.width) {
#pragma unroll
      for (int j = 0; j < 8 / V * NV; ++j) n += min(max(c.D - (j * c.width + first) * V, 0), 32 * V);
    }
    sh.columns[threadIdx.x] = static_cast<float>(n);
  }
  __syncthreads();
}

// Mean and 1 / deviation of a row with one barrier: each warp's mean and its squares about it, joined as
// sum over warps of (squares + columns (mean of the warp - mean)^2).
template <int NV, class C>
__device__ __forceinline__ float2 statistics(const F (&a)[NV][N], const ttt_b200_block_args& p, const C& c, Shared& sh, int& buf) {
  constexpr int V = C::V;
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
    if (c.in(j)) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        F v = add2(a[j][k], both(-mean));
        if (2 * k + 1 >= V) v = make_float2(c.in(j, 2 * k) ? v.x : 0.f, c.in(j, 2 * k + 1) ? v.y : 0.f);      // (the first run is there)
        sq = fma2(v, v, sq);
      }
    }
  float q = fold(sq);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
  if constexpr (C::width > 32) {
    constexpr int warps = C::width / 32;
    const int warp = threadIdx.x >> 5, home = warp & -warps, i = threadIdx.x % warps;
    if ((threadIdx.x & 31) == 0) sh.part[buf][warp] = make_float2(mean, q);
    __syncthreads();
    const float2 v = sh.part[buf][home + i];      // a lane for each warp
    q = v.y;
    if (p.layer) {
      const float n = sh.columns[i];
      mean = n * v.x;
#pragma unroll
      for (int o = warps / 2; o > 0; o >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, o);
      mean *= inv;
      q = fmaf(n * (v.x - mean), v.x - mean, q);
    }
#pragma unroll
    for (int o = warps / 2; o > 0; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
    buf ^= 1;
  }
  return make_float2(mean, rsqrtf(fmaf(q, inv, p.eps)));
}

template <class T, class R, class C>
__global__ void __launch_bounds__(C::threads, 1024 / C::threads) block_forward_kernel(const ttt_b200_block_args p, const Plan q) {
  wait_for_predecessor();
  constexpr int kMode = C::V > 1 ? kOwn : kWindow, NV = 1;
  __shared__ Shared sh;
  extern __shared__ __align__(16) unsigned char stages[];
  uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(stages));
  int buf = 0;
  const int lane = threadIdx.x % C::width, sub = threadIdx.x / C::width;
  const C c = {lane, p.D};
  const long step = static_cast<long>(q.ctas) * C::side;
  const Feed<T, C, kMode> fo(p.o, p.o_stride, at, p.D), fg(p.gate, p.gate_stride, at, p.D);
  const Feed<R, C, kMode> fx(p.residual, p.residual_stride, at, p.D);
  const uint32_t small = Feed<T, C, kMode>::bytes(p.D), large = Feed<R, C, kMode>::bytes(p.D);
  auto ahead = [&](long m, int stage) {
    if (m < p.M) {
      fo.ahead(m, stage * small, c, sub);
      fg.ahead(m, stage * small, c, sub);
      fx.ahead(m, stage * large, c, sub);
    }
    cp_async_commit();
  };
  long m = static_cast<long>(blockIdx.x) * C::side + sub;
  ahead(m, 0);
  count_columns<NV>(sh, c);
  int stage = 0;
  for (long base = static_cast<long>(blockIdx.x) * C::side; base < p.M; base += step, stage ^= 1, m += step) {
    const bool live = m < p.M;
    cp_async_wait<0>();
    if constexpr (kMode == kWindow) __syncthreads();
    ahead(m + step, stage ^ 1);
    F a[NV][N], z[NV][N];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int k = 0; k < N; ++k) a[j][k] = z[j][k] = both(0.f);
      if (live && c.in(j)) fo.get(m, stage * small, c, j, sub, a[j]);
    }
    float2 s1 = make_float2(0.f, 1.f), s2 = s1;
    if (p.post_weight) s1 = statistics<NV>(a, p, c, sh, buf);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!(live && c.in(j))) continue;
      F w[N], b[N];
      if (p.post_weight) {
        weights(p.post_weight, c, j, 0.f, w);
        weights(p.post_bias, c, j, 0.f, b);
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
      weights(p.scale, c, j, 1.f, w);
#pragma unroll
      for (int k = 0; k < N; ++k) z[j][k] = mac(w[k], a[j][k], z[j][k]);
      store(static_cast<R*>(p.x) + m * p.D, c, j, z[j]);
    }
    if (p.pre_weight) {
      s2 = statistics<NV>(z, p, c, sh, buf);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (live && c.in(j)) {
          F w[N], b[N];
          weights(p.pre_weight, c, j, 0.f, w);
          weights(p.pre_bias, c, j, 0.f, b);
#pragma unroll
          for (int k = 0; k < N; ++k) z[j][k] = mac(times(plus(z[j][k], both(-s2.x)), both(s2.y)), w[k], b[k]);
          store(static_cast<T*>(p.n) + m * p.D, c, j, z[j]);
        }
      }
    }
    if (p.stats && live && lane == 0) reinterpret_cast<float4*>(p.stats)[m] = make_float4(s1.x, s1.y, s2.x, s2.y);
  }
}

// Sums over tokens of a thread's columns: in registers, or, of sixteen columns, in shared memory.
enum { kDw1, kDb1, kDsc, kDw2, kDb2, kSums };
template <class C, int NV, bool kShared> struct Sums {
  F r[kShared ? 1 : kSums][NV][N];
  float* s;
  __device__ __forceinline__ F get(int k, int j, int i, const C& c) const {
    if constexpr (!kShared) return r[k][j][i];
    else if constexpr (C::V > 1) return c.in(j, 2 * i) ? *reinterpret_cast<const F*>(s + k * c.D + c.at(j, 2 * i)) : both(0.f);
    else return make_float2(c.in(j, 2 * i) ? s[k * c.D + c.at(j, 2 * i)] : 0.f, c.in(j, 2 * i + 1) ? s[k * c.D + c.at(j, 2 * i + 1)] : 0.f);
  }
  __device__ __forceinline__ void set(int k, int j, int i, const C& c, F v) {
    if constexpr (!kShared) {
      r[k][j][i] = v;
    } else if constexpr (C::V > 1) {
      if (c.in(j, 2 * i)) *reinterpret_cast<F*>(s + k * c.D + c.at(j, 2 * i)) = v;
    } else {
      if (c.in(j, 2 * i)) s[k * c.D + c.at(j, 2 * i)] = v.x;
      if (c.in(j, 2 * i + 1)) s[k * c.D + c.at(j, 2 * i + 1)] = v.y;
    }
  }
  __device__ __forceinline__ void add(int k, int j, int i, const C& c, F v) { set(k, j, i, c, add2(get(k, j, i, c), v)); }
  __device__ __forceinline__ void add(int k, int j, int i, const C& c, F a, F b) { set(k, j, i, c, fma2(a, b, get(k, j, i, c))); }
};

template <class T, class R, class C, int NV, bool kShared>
__global__ void __launch_bounds__(C::threads, 512 / C::threads) block_backward_kernel(const ttt_b200_block_args p, const Plan q) {
  wait_for_predecessor();
  constexpr int kMode = kShared ? kDirect : C::V > 1 ? kOwn : kWindow;
  __shared__ Shared sh;
  extern __shared__ __align__(16) unsigned char stages[];
  uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(stages));
  int buf = 0;
  const int lane = threadIdx.x % C::width, sub = threadIdx.x / C::width;
  const C c = {lane, p.D};
  const long step = static_cast<long>(q.ctas) * C::side;
  const Feed<T, C, kMode> fo(p.o, p.o_stride, at, p.D), fg(p.gate, p.gate_stride, at, p.D);
  const Feed<T, C, kMode> fn(p.pre_weight ? p.grad_n : nullptr, p.gn_stride, at, p.D);
  const Feed<R, C, kMode> fx(p.pre_weight ? p.residual : nullptr, p.residual_stride, at, p.D);
  const Feed<R, C, kMode> fd(p.grad_x, p.gx_stride, at, p.D);
  const uint32_t small = Feed<T, C, kMode>::bytes(p.D), large = Feed<R, C, kMode>::bytes(p.D);
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
  Sums<C, NV, kShared> sums;
  sums.s = reinterpret_cast<float*>(stages);
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (!kShared || c.in(j)) {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int k = 0; k < kSums; ++k) sums.set(k, j, i, c, both(0.f));
    }
  long m = static_cast<long>(blockIdx.x) * C::side + sub;
  ahead(m, 0);
  int stage = 0;
  for (long base = static_cast<long>(blockIdx.x) * C::side; base < p.M; base += step, stage ^= 1, m += step) {
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
      const bool in = live && c.in(j);
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
        weights(p.post_weight, c, j, 0.f, w);
        weights(p.post_bias, c, j, 0.f, b);
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = mac(o[j][i], w[i], b[i]);
      }
      if (p.gate) {
        fg.get(m, stage * small, c, j, sub, w);
        gate<false>(p.activation, w, w, b);
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = times(u[i], w[i]);
      }
      weights(p.scale, c, j, 1.f, w);
      fx.get(m, stage * large, c, j, sub, z[j]);
#pragma unroll
      for (int i = 0; i < N; ++i) z[j][i] = times(plus(mac(w[i], u[i], z[j][i]), both(-st.z)), both(st.w));
      fn.get(m, stage * small, c, j, sub, gn[j]);
      weights(p.pre_weight, c, j, 0.f, w);
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
      s = row_sum<C>(s, sh.part, buf);
      m1 = p.layer ? s.x * inv : 0.f;
      m2 = s.y * inv;
    }
    sx = sy = both(0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!(live && c.in(j))) continue;
      fd.get(m, stage * large, c, j, sub, d2[j]);
      if (p.pre_weight) {
#pragma unroll
        for (int i = 0; i < N; ++i) d2[j][i] = mac(both(st.w), mac(z[j][i], both(-m2), plus(gn[j][i], both(-m1))), d2[j][i]);
      }
      if (p.grad_residual) store(static_cast<R*>(p.grad_residual) + m * p.D, c, j, d2[j]);
      F u[N], w[N], b[N], v[N], g[N];
#pragma unroll
      for (int i = 0; i < N; ++i) u[i] = o[j][i];
      if (p.post_weight) {
        weights(p.post_weight, c, j, 0.f, w);
        weights(p.post_bias, c, j, 0.f, b);
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = mac(o[j][i], w[i], b[i]);
      }
      weights(p.scale, c, j, 1.f, b);
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
        store(static_cast<T*>(p.grad_gate) + m * p.D, c, j, g);
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
      s = row_sum<C>(make_float2(fold(sx), fold(sy)), sh.part, buf);
      m1 = p.layer ? s.x * inv : 0.f;
      m2 = s.y * inv;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!(live && c.in(j))) continue;
      if (p.post_weight) {
#pragma unroll
        for (int i = 0; i < N; ++i) d2[j][i] = times(both(st.y), mac(o[j][i], both(-m2), plus(d2[j][i], both(-m1))));
      }
      store(static_cast<T*>(p.grad_o) + m * p.D, c, j, d2[j]);
    }
  }
  float* part = q.part + (static_cast<long>(blockIdx.x) * C::side + sub) * kSums * p.D;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (!c.in(j)) continue;
#pragma unroll
    for (int k = 0; k < kSums; ++k) {
      F v[N];
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = sums.get(k, j, i, c);
      store(part + static_cast<long>(k) * p.D, c, j, v);
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
  const int side = side_of(q.width);
  const long most = static_cast<long>(sm_count()) * ((backward ? 512 : 1024) / (q.width * side));
  q.ctas = static_cast<int>(std::min<long>(most, (p.M + side - 1) / side));
}

template <class R> constexpr int kRun = sizeof(R) == 4 ? 4 : 8;      // V of rows that start on its boundaries

// whether every row of every tensor starts on a boundary of `run` values
bool vectors(const ttt_b200_block_args& p, bool backward, int run) {
  const size_t es = p.dtype == TTT_B200_FP32 ? 4 : 2, rs = p.residual_fp32 ? 4 : es;
  auto rows = [run](const void* a, int64_t stride, size_t bytes) { return reinterpret_cast<uintptr_t>(a) % (run * bytes) == 0 && stride % run == 0; };
  bool ok = p.D % run == 0 && rows(p.o, p.o_stride, es) && rows(p.residual, p.residual_stride, rs) && rows(p.gate, p.gate_stride, es);
  for (const float* w : {p.post_weight, p.post_bias, p.scale, p.pre_weight, p.pre_bias}) ok = ok && aligned16(w);
  if (backward)
    return ok && rows(p.grad_x, p.gx_stride, rs) && rows(p.grad_n, p.gn_stride, es) && rows(p.grad_o, 0, es) && rows(p.grad_residual, 0, rs) &&
           rows(p.grad_gate, 0, es);
  return ok && rows(p.x, 0, rs) && rows(p.n, 0, es);
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
  ttt_launch_overlapped(kernel, q.ctas, q.width * side_of(q.width), static_cast<uint32_t>(bytes), s, p, q);
  return launched(what);
}

template <class T, class R, class C> int forward_as(const ttt_b200_block_args& p, const Plan& q, cudaStream_t s) {
  constexpr int kMode = C::V > 1 ? kOwn : kWindow;
  const size_t bytes = 2 * (Feed<T, C, kMode>::bytes(p.D) * (1 + (p.gate != nullptr)) + Feed<R, C, kMode>::bytes(p.D) * (p.residual != nullptr));
  return launch(block_forward_kernel<T, R, C>, q, bytes, s, p, "block norm");
}
template <class T, class R, int kWidth> int forward_of(const ttt_b200_block_args& p, const Plan& q, cudaStream_t s) {
  if (!vectors(p, false, kRun<R>)) return forward_as<T, R, Cols<1, kWidth, false>>(p, q, s);
  return p.D == 8 * kWidth ? forward_as<T, R, Cols<kRun<R>, kWidth, true>>(p, q, s) : forward_as<T, R, Cols<kRun<R>, kWidth, false>>(p, q, s);
}

template <class T, class R> int forward(const ttt_b200_block_args& p, cudaStream_t s) {
  Plan q = {};
  plan(q, p, false);
  switch (q.width) {
    case 32: return forward_of<T, R, 32>(p, q, s);
    case 64: return forward_of<T, R, 64>(p, q, s);
    case 128: return forward_of<T, R, 128>(p, q, s);
    case 256: return forward_of<T, R, 256>(p, q, s);
    case 512: return forward_of<T, R, 512>(p, q, s);
    default: return forward_of<T, R, 1024>(p, q, s);
  }
}

template <class T, class R, class C, int NV, bool kShared> int backward_as(const ttt_b200_block_args& p, const Plan& q, cudaStream_t s) {
  constexpr int kMode = kShared ? kDirect : C::V > 1 ? kOwn : kWindow;
  const size_t bytes = kShared ? static_cast<size_t>(kSums) * p.D * sizeof(float)
                               : 2 * (Feed<T, C, kMode>::bytes(p.D) * (1 + (p.gate != nullptr) + (p.pre_weight && p.grad_n)) +
                                      Feed<R, C, kMode>::bytes(p.D) * ((p.pre_weight && p.residual) + (p.grad_x != nullptr)));
  return launch(block_backward_kernel<T, R, C, NV, kShared>, q, bytes, s, p, "block norm backward");
}
template <class T, class R, int kWidth, int NV = 1> int backward_of(const ttt_b200_block_args& p, const Plan& q, cudaStream_t s) {
  if (!vectors(p, true, kRun<R>)) return backward_as<T, R, Cols<1, kWidth, false>, NV, (NV > 1)>(p, q, s);
  return p.D == 8 * NV * kWidth ? backward_as<T, R, Cols<kRun<R>, kWidth, true>, NV, (NV > 1)>(p, q, s)
                                : backward_as<T, R, Cols<kRun<R>, kWidth, false>, NV, (NV > 1)>(p, q, s);
}
template <class T, class R> int backward_kernel(const ttt_b200_block_args& p, const Plan& q, cudaStream_t s) {
  if (p.D > kWide) return backward_of<T, R, 512, 2>(p, q, s);
  switch (q.width) {
    case 32: return backward_of<T, R, 32>(p, q, s);
    case 64: return backward_of<T, R, 64>(p, q, s);
    case 128: return backward_of<T, R, 128>(p, q, s);
    case 256: return backward_of<T, R, 256>(p, q, s);
    default: return backward_of<T, R, 512>(p, q, s);
  }
}

template <class T, class R> int backward(const ttt_b200_block_args& p, cudaStream_t s) {
  Plan q = {};
  plan(q, p, true);
  q.part = static_cast<float*>(p.scratch);
  const int rc = backward_kernel<T, R>(p, q, s);
  if (rc) return rc;
  const long row = static_cast<long>(kSums) * p.D;
  float* dst[kSums] = {p.grad_post_weight, p.grad_post_bias, p.grad_scale, p.grad_pre_weight, p.grad_pre_bias};
  ttt_sum_job jobs[kSums];
  for (int k = 0; k < kSums; ++k)
    jobs[k] = {q.part + static_cast<long>(k) * p.D, dst[k], p.D, row, q.ctas * side_of(q.width), TTT_B200_FP32, 0};
  return ttt_sum_parts(jobs, kSums, s);
}

}  // namespace

extern "C" uint64_t ttt_b200_norm_gate_residual_scratch_bytes(const ttt_b200_block_args* p) {
  if (check(p) || p->M == 0) return 0;
  Plan q = {};
  plan(q, *p, true);
  return static_cast<uint64_t>(q.ctas) * side_of(q.width) * kSums * p->D * sizeof(float);
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
