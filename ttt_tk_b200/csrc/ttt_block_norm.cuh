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
// itself over all its tokens and leaves them as one part per CTA for an ordered sum.  The width is a constant of a kernel, so that
// addresses and reductions are too (16384 x 2048, fp32 residual, forward and backward: 118 -> 104 and 230 -> 211 us; rows of 2047
// 174 -> 118 and 349 -> 257).
#pragma once

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "ttt_elem.cuh"
#include "ttt_sum_parts.h"

namespace ttt {
namespace block {

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

// kParts kAll: post norm, gate, residual, scale and pre norm are all there, backward both gradients too.  Without a branch around every one of
// them the loads of one part overlap the arithmetic of another: 98 -> 89 and 192 -> 169 us of the first, 77 -> 67 and 185 -> 147 of the second.
// kBare: a residual and the next norm alone, which is a plain block's end (16384 x 2048 bf16, RMS norm: 49 -> 44 and 107 -> 83 us; rows of 2047,
// layer norm: 85 -> 76 and 154 -> 119).  kSome: whatever the pointers say.
enum { kSome, kAll, kBare };
template <int kRun, int kWidth, bool kFull, int kParts> struct Cols {
  static constexpr bool all = kParts == kAll, bare = kParts == kBare;
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
template <bool kThere = false, class C> __device__ __forceinline__ void weights(const float* p, const C& c, int j, float none, F (&f)[N]) {
  if (kThere || p) load(p, c, j, f, none);
  else fill(f, none);
}

// The gate: its value, and with kSlope its derivative.  GELU as x sigmoid(2 u): no 1 + tanh(u), which cancels on the left.  The
// derivative needs 1 - sigmoid without its cancellation on the right, which is e times sigmoid.  Far on the left e is bounded, so that
// this is not infinity times 0: at 2^127 the reciprocal is below the least normal number and so 0, and with it all that it enters
// (at 2^126 it is 2^-126, which x = -1e38 takes to -1).  GELU's x^2 is bounded where it meets a factor of 0, beyond |x| = 1e15.
template <int kKind, bool kSlope> __device__ __forceinline__ void gate_one(F x, F& v, F& s) {
  constexpr float k = 1.5957691216057308f, c = 0.044715f;      // 2 sqrt(2 / pi)
  F e;
  const F q = times(x, x);
  if constexpr (kKind == TTT_B200_ACT_GELU) e = times(times(x, all<F>(-k * kLog2e)), mac(q, all<F>(c), all<F>(1.f)));
  else e = times(x, all<F>(-kLog2e));
  if constexpr (kSlope) e = least(e, 127.f);
  e = ex2(e);
  const F g = rcp(plus(e, all<F>(1.f)));
  if constexpr (kKind == TTT_B200_ACT_SIGMOID) {
    v = g;
    if constexpr (kSlope) s = times(g, times(e, g));
  } else {
    v = times(x, g);
    if constexpr (kSlope) {
      F o = times(e, g);
      if constexpr (kKind == TTT_B200_ACT_GELU) o = times(o, mac(least(q, 1e30f), all<F>(3.f * c * k), all<F>(k)));
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
template <class T, class C, int kMode, bool kThere> struct Feed {
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
    if (kThere || base) smem += 2 * bytes(D);
  }
  __device__ __forceinline__ static uint32_t place(int sub, int D) { return kMode == kOwn ? threadIdx.x * kRun : sub * window(D); }
  // row m into a stage
  __device__ __forceinline__ void ahead(long m, uint32_t to, const C& c, int sub) const {
    if (!kThere && !base) return;
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
    if (!kThere && !base) {
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

// ---- host --------------------------------------------------------------------------------------------------------------
inline int check(const ttt_b200_block_args* p) {
  if (!p) return fail("block norm: NULL argument struct");
  if (p->M < 0 || p->D < 1 || p->D > 8192) return fail("block norm: M >= 0 and 1 <= D <= 8192");
  if (p->dtype < TTT_B200_BF16 || p->dtype > TTT_B200_FP32) return fail("block norm: unknown element type");
  if (p->activation < TTT_B200_ACT_SILU || p->activation > TTT_B200_ACT_SIGMOID) return fail("block norm: activation is silu, gelu or sigmoid");
  if (!(p->eps >= 0.f)) return fail("block norm: eps must be >= 0");
  if ((p->post_bias && !p->post_weight) || (p->pre_bias && !p->pre_weight)) return fail("block norm: a bias without its weight");
  return TTT_B200_OK;
}

// threads of a token: the fewest that hold it with `values` each
inline int width_of(int D, int values) {
  int w = 32;
  while (w * values < D) w *= 2;
  return w;
}
constexpr int kWide = 4096;      // backward of wider rows: sixteen values to a thread, the sums over tokens in shared memory

// CTAs that are resident together and walk over the tokens: 1024 threads to an SM, backward 512.
inline void plan(Plan& q, const ttt_b200_block_args& p, bool backward) {
  const bool wide = p.D > kWide;
  q.width = width_of(p.D, wide && backward ? 16 : 8);
  const int side = side_of(q.width);
  const long most = static_cast<long>(sm_count()) * ((backward ? 512 : 1024) / (q.width * side));
  q.ctas = static_cast<int>(std::min<long>(most, (p.M + side - 1) / side));
}

template <class R> constexpr int kRun = sizeof(R) == 4 ? 4 : 8;      // V of rows that start on its boundaries

// whether every row of every tensor starts on a boundary of `run` values
inline bool vectors(const ttt_b200_block_args& p, bool backward, int run) {
  const size_t es = p.dtype == TTT_B200_FP32 ? 4 : 2, rs = p.residual_fp32 ? 4 : es;
  auto rows = [run](const void* a, int64_t stride, size_t bytes) { return reinterpret_cast<uintptr_t>(a) % (run * bytes) == 0 && stride % run == 0; };
  bool ok = p.D % run == 0 && rows(p.o, p.o_stride, es) && rows(p.residual, p.residual_stride, rs) && rows(p.gate, p.gate_stride, es);
  for (const float* w : {p.post_weight, p.post_bias, p.scale, p.pre_weight, p.pre_bias}) ok = ok && aligned16(w);
  if (backward)
    return ok && rows(p.grad_x, p.gx_stride, rs) && rows(p.grad_n, p.gn_stride, es) && rows(p.grad_o, 0, es) && rows(p.grad_residual, 0, rs) &&
           rows(p.grad_gate, 0, es);
  return ok && rows(p.x, 0, rs) && rows(p.n, 0, es);
}

inline int parts_of(const ttt_b200_block_args& p) {
  if (p.residual && p.gate && p.post_weight && p.scale && p.pre_weight) return kAll;
  return p.residual && p.pre_weight && !p.gate && !p.post_weight && !p.scale ? kBare : kSome;
}

// More dynamic shared memory than 48 KB has to be asked for, per kernel and device.  All that there is is asked for, once: a limit of a
// call's own would be lowered by a smaller call of another host thread between this call's asking and its launch.
template <auto kKernel> int allow_shared() {
  static std::atomic<uint64_t> done{0};      // a bit for each device
  int dev = 0, most = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? uint64_t{1} << dev : 0;      // (beyond 64 devices: every time the same)
  if (e == cudaSuccess && (done.load(std::memory_order_acquire) & bit)) return TTT_B200_OK;
  cudaFuncAttributes own = {};
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&own, kKernel);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most - static_cast<int>(own.sharedSizeBytes));
  if (e != cudaSuccess) return ttt_set_error(TTT_B200_ERR_LAUNCH, cudaGetErrorString(e));
  done.fetch_or(bit, std::memory_order_release);
  return TTT_B200_OK;
}
template <auto kKernel> int launch(const Plan& q, size_t bytes, cudaStream_t s, const ttt_b200_block_args& p, const char* what) {
  if (bytes > 40 * 1024)      // (with the static part 48 KB is the most without asking)
    if (int rc = allow_shared<kKernel>()) return rc;
  ttt_launch_overlapped(kKernel, q.ctas, q.width * side_of(q.width), static_cast<uint32_t>(bytes), s, p, q);
  return launched(what);
}

}  // namespace block
}  // namespace ttt
