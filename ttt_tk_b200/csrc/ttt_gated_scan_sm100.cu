// Gated linear recurrence: forward for prompts and training, backward, and the step of single tokens.
//
//   s = sigmoid(gate + gate_bias);  log a = A[d] s, A <= 0 (without A: a = s);  b = sqrt(1 - a^2), 1 - a or 1;
//   i = sigmoid(input_gate + input_bias);  u = b i x;  h_t = a_t h_{t-1} + u_t;  y = h
//
// Backward, with G_t the gradient with respect to h_t and c_t = a_t G_t what it leaves for the token before:  G_t = dy_t + c_{t+1};
// dx = G b i;  d input_gate = G b x i (1 - i);  d log a = G (a h_{t-1} + i x db/dlog a), db/dlog a = -a^2 / b, -a or 0;
// d gate = d log a times A s (1 - s), without A times 1 - s;  dA = sum d log a s;  dh_{-1} = c_0.
//
// Bound by memory: a value is read three times 2 bytes and written once (bf16; backward four and three times), for some 40 fp32
// operations and six of the exponential unit.  A recurrence of steps h -> p h + q joins: two after one another are p2 p1, p2 q1 + q2.  So a
// warp has S tokens of 64 channels in registers (two neighbouring channels to a lane), the warps of a CTA have the tokens behind one another
// of a tile, each takes its tokens from zero, and all join what is in front of them over shared memory: one pass over the data, one barrier.
// Where channels and sequences do not fill the GPU the CTAs of a cluster have tiles behind one another and join over distributed
// shared memory, with one cluster barrier more.  The order of the joins is fixed.
// The backward starts each tile from the state that the forward left of it and joins both directions over the same barrier.
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

#include "ttt_elem.cuh"
#include "ttt_sum_parts.h"

namespace {

using namespace ttt;

using F = float2;
using E4 = __nv_fp8_e4m3;
constexpr int kTile = TTT_B200_GATED_INTERVAL;      // tokens of a CTA's tile, and between two checkpoints
constexpr int kCols = 64;                           // channels of a CTA

#ifndef TTT_FWD_CTAS
#define TTT_FWD_CTAS 2
#define TTT_BWD_CTAS 2
#define TTT_FWD_S 8
#define TTT_BWD_S 8
#endif
struct Plan {
  int tiles;      // CTAs (clusters) side by side: channels / 64
  int cluster;    // CTAs that have tiles behind one another
  int nck;        // tiles of a sequence
  float* part;    // backward: [B * cluster][3][D]
};

// ---- arithmetic, two channels at a time ----------------------------------------------------------------------------------------
// NaN stays NaN (fminf would drop it)
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float rsqrt_fast(float v) {
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ F neg(F a) { return mul2(a, both(-1.f)); }

// s = sigmoid(v) and, with kBoth, 1 - s without the cancellation on the right.  For 1 - s the exponent is bounded so that far on the left e s
// is a number: at 2^127 the reciprocal is below the least normal number and so s = 0 (and e s = 0: it only ever meets the factor s); at 2^126
// s = 2^-126 and e s = 1, which the form without A needs.
// `bias` comes times -log2 e.
template <bool kBoth> __device__ __forceinline__ void sigmoid(F v, F bias, float most, F& s, F& other) {
  F t = fma2(v, both(-kLog2e), bias);
  if constexpr (kBoth) t = make_float2(min_nan(t.x, most), min_nan(t.y, most));
  const F e = ex2(t);
  s = rcp(add2(e, both(1.f)));
  if constexpr (kBoth) other = mul2(e, s);
}

// exp(v) and 1 - exp(v) for v <= 0: v = k ln 2 + f, |f| <= ln 2 / 2, ln 2 in two parts (Cody and Waite), exp(f) - 1 = f + f^2 p(f) with the
// polynomial of fourth degree that is off by the least part of f (1.6e-8, fitted).  Both from one series: 1 - a keeps its digits where a is close to one, which is where these
// recurrences are, and the exponential unit, which is close to its limit, is left alone.  Where k comes to -127 the power's
// bits are those of 0: exp(v) is 0 from there on, as far as A makes v.
__device__ __forceinline__ void exp_both(F v, F& a, F& rest) {
  v = make_float2(max_nan(v.x, -88.f), max_nan(v.y, -88.f));
  constexpr float magic = 12582912.f;      // 1.5 2^23: the sum's last bits are the rounded integer
  const F k = fma2(v, both(kLog2e), both(magic)), kf = add2(k, both(-magic));
  F f = fma2(kf, both(-0.693145751953125f), v);
  f = fma2(kf, both(-1.42860682030941723e-6f), f);
  F q = fma2(f, both(1.3947017723694444e-3f), both(8.366910740733147e-3f));
  q = fma2(q, f, both(4.166627302765846e-2f));
  q = fma2(q, f, both(1.6666540503501892e-1f));
  q = fma2(q, f, both(0.5f));
  q = fma2(mul2(f, f), q, f);
  const F two = make_float2(__int_as_float((__float_as_int(k.x) << 23) + 0x3f800000), __int_as_float((__float_as_int(k.y) << 23) + 0x3f800000));
  q = mul2(q, two);      // exact but where it is below the normal numbers
  a = add2(q, two);
  rest = fma2(q, both(-1.f), fma2(two, both(-1.f), both(1.f)));
}

// What does not change over the tokens of a lane's channels.
struct Weights {
  F A, gate_bias, input_bias;
  int mix;
  bool has_a, gated;
};

// A token's a and w = b i, and for the backward  k = d log a / d gate, s, slope = i db/dlog a, rest = 1 - i.
template <bool kBack> struct Factors;
template <> struct Factors<false> {
  F a, w;
};
template <> struct Factors<true> {
  F a, w, k, s, slope, rest;
};
// kUsual: A, the root and an input gate, which leaves nothing to decide for each token.
template <bool kUsual, bool kBack, class Gate, class Input>
__device__ __forceinline__ void factors(const Weights& z, Gate gate, Input input, Factors<kBack>& f) {
  F rest, o;      // 1 - a, 1 - s
  if (kUsual || z.has_a) {
    F s;
    sigmoid<kBack>(gate, z.gate_bias, 127.f, s, o);
    const F la = mul2(s, z.A);
    exp_both(la, f.a, rest);
    if constexpr (kBack) f.s = s, f.k = mul2(la, o);
  } else {
    sigmoid<true>(gate, z.gate_bias, 126.f, f.a, rest);
    if constexpr (kBack) f.s = f.a, f.k = rest;
  }
  if (kUsual || z.mix == TTT_B200_MIX_SQRT) {
    const F q = mul2(rest, fma2(rest, both(-1.f), both(2.f)));      // 1 - a^2
    // where that is no normal number b is 0, and so is its slope
    if constexpr (kBack) {
      F r = make_float2(rsqrt_fast(q.x), rsqrt_fast(q.y));
      r = make_float2(q.x < 1.17549435e-38f ? 0.f : r.x, q.y < 1.17549435e-38f ? 0.f : r.y);
      f.w = mul2(q, r);
      f.slope = mul2(mul2(f.a, f.a), neg(r));
    } else {
      f.w = mul2(q, make_float2(rsqrt_fast(max_nan(q.x, 1.17549435e-38f)), rsqrt_fast(max_nan(q.y, 1.17549435e-38f))));
    }
  } else if (z.mix == TTT_B200_MIX_LINEAR) {
    f.w = rest;
    if constexpr (kBack) f.slope = neg(f.a);
  } else {
    f.w = both(1.f);
    if constexpr (kBack) f.slope = both(0.f);
  }
  if (kUsual || z.gated) {
    F i;
    sigmoid<kBack>(input(), z.input_bias, 126.f, i, o);
    f.w = mul2(f.w, i);
    if constexpr (kBack) f.slope = mul2(f.slope, i), f.rest = o;
  } else if constexpr (kBack) {
    f.rest = both(0.f);
  }
}

// ---- rows through shared memory ------------------------------------------------------------------------------------------------
template <class T> __device__ __forceinline__ F pair_of(uint32_t at) {      // shared address
  if constexpr (sizeof(T) == 4) {
    const uint2 r = shared_load8(at);
    return make_float2(__uint_as_float(r.x), __uint_as_float(r.y));
  } else if constexpr (sizeof(T) == 2) {
    uint32_t r;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(at) : "memory");
    if constexpr (std::is_same<T, __half>::value) return __half22float2(reinterpret_cast<__half2&>(r));
    else return __bfloat1622float2(reinterpret_cast<__nv_bfloat162&>(r));
  } else {
    uint16_t r;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(r) : "r"(at) : "memory");
    return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(r, __NV_E4M3)));
  }
}
template <class T> __device__ __forceinline__ float value_of(uint32_t at) {
  if constexpr (sizeof(T) == 1) {
    uint16_t r;
    asm volatile("{.reg .u8 t; ld.shared.u8 t, [%1]; cvt.u16.u8 %0, t;}" : "=h"(r) : "r"(at) : "memory");
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(r), __NV_E4M3)));
  } else {
    return shared_load<T>(at);
  }
}

// S rows of 64 channels of a tensor, copied ahead by a warp into its own place in shared memory.
//   kWhole    rows start on 16-byte boundaries: 16-byte pieces, pairs
//   otherwise the 16-byte blocks that a row touches (the first and the last may hold its neighbours too), from which values are picked one
//             by one at the row's offset
// 8-bit values come with their scales, two to a row (one for each 32 channels).
template <class T, int S, bool kWhole> struct Rows {
  static constexpr int es = sizeof(T), kBytes = kCols * es, kPitch = kWhole ? kBytes : kBytes + 16, kPieces = kPitch / 16;
  static constexpr bool kScaled = es == 1;
  static constexpr uint32_t kStage = S * kPitch + (kScaled ? S * 8 : 0);      // bytes
  static_assert(kStage % 16 == 0, "copies start on 16-byte boundaries");
  const char* base;      // channel d0 of the first token
  const float* scales;   // its scale
  int64_t step, scale_step;      // bytes from token to token; scales
  int cols;      // bytes of a row that there are
  int second;    // distance of the second 32 channels' scale, 0 or 1; -1: there are none
  __device__ __forceinline__ Rows(const void* p, int64_t batch, int64_t token, int b, int d0, int D, const float* sc = nullptr, int groups = 0, int group = 32, int T_ = 0) {
    base = static_cast<const char*>(p) + (b * batch + d0) * es;
    step = token * es;
    cols = min(D - d0, kCols) * es;
    if constexpr (kScaled) {
      scales = sc + static_cast<int64_t>(b) * T_ * groups + d0 / group;
      scale_step = groups;
      second = d0 + 32 < D ? (d0 + 32) / group - d0 / group : -1;
    }
  }
  // tokens t .. t + S - 1, those before `stop`, to the shared address `to`
  __device__ __forceinline__ void copy(uint32_t to, int t, int stop) const {
    const int lane = threadIdx.x & 31;
    if (kWhole && t + S <= stop && cols == kBytes) {      // all of them: nothing to compare
      static_assert(32 % kPieces == 0 || !kWhole, "a lane's pieces are below one another");
      const char* from = base + (t + lane / kPieces) * step + lane % kPieces * 16;
      to += lane * 16;
#pragma unroll
      for (int i = 0; i < (S * kPieces + 31) / 32; ++i) {
        if (S * kPieces % 32 && lane + 32 * i >= S * kPieces) break;
        cp_async16_at(to + 512 * i, from);
        from += 32 / kPieces * step;
      }
      if constexpr (kScaled) to -= lane * 16;
    } else {
#pragma unroll
      for (int i = 0; i < (S * kPieces + 31) / 32; ++i) {
        const int n = lane + 32 * i, row = n / kPieces, o = n % kPieces * 16;
        if (S * kPieces % 32 && n >= S * kPieces) break;
        const char* from = base + (t + row) * step;
        int have = cols - o;
        if constexpr (!kWhole) {
          const int off = static_cast<int>(reinterpret_cast<uintptr_t>(from) & 15);
          from -= off;
          have += off;
        }
        have = t + row < stop ? min(max(have, 0), 16) : 0;
        cp_async16_at(to + row * kPitch + o, have ? from + o : reinterpret_cast<const char*>(reinterpret_cast<uintptr_t>(base) & ~uintptr_t{15}), have);
      }
    }
    if constexpr (kScaled) {
      static_assert(S * 2 <= 32, "a lane for each scale");
      if (lane < 2 * S) {
        const bool in = t + lane / 2 < stop && !(lane % 2 && second < 0);
        cp_async4_at(to + S * kPitch + lane * 4, in ? scales + (t + lane / 2) * scale_step + (lane % 2 ? second : 0) : scales, in ? 4 : 0);
      }
    }
  }
  // this lane's two channels of token t (row i of those at `from`)
  __device__ __forceinline__ F get(uint32_t from, int i, int t) const {
    const int lane = threadIdx.x & 31;
    F v;
    if constexpr (kWhole) {
      v = pair_of<T>(from + i * kPitch + lane * 2 * es);
    } else {
      const uint32_t at = from + i * kPitch + (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(base) + t * step) & 15) + lane * 2 * es;
      v = make_float2(value_of<T>(at), value_of<T>(at + es));
    }
    if constexpr (kScaled) v = mul2(v, both(shared_load<float>(from + S * kPitch + i * 8 + lane / 16 * 4)));
    return v;
  }
};

// ---- a lane's two channels in global memory -------------------------------------------------------------------------------------------
template <bool kWhole> __device__ __forceinline__ F load2(const float* p, int d, int D, float none) {
  if (!p || d >= D) return both(none);
  if constexpr (kWhole) return *reinterpret_cast<const F*>(p + d);
  return make_float2(p[d], d + 1 < D ? p[d + 1] : none);
}
template <class T, bool kWhole> __device__ __forceinline__ void store2(T* p, int d, int D, F v) {
  if (d >= D) return;
  if constexpr (kWhole) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) *reinterpret_cast<__nv_bfloat162*>(p + d) = __float22bfloat162_rn(v);
    else if constexpr (std::is_same<T, __half>::value) *reinterpret_cast<__half2*>(p + d) = __float22half2_rn(v);
    else *reinterpret_cast<F*>(p + d) = v;
  } else {
    p[d] = from_f32<T>(v.x);
    if (d + 1 < D) p[d + 1] = from_f32<T>(v.y);
  }
}
template <bool kWhole> __device__ __forceinline__ Weights weights_of(const ttt_b200_gated_args& p, int d) {
  Weights z;
  z.A = load2<kWhole>(p.A, d, p.D, 0.f);
  z.A = make_float2(min_nan(z.A.x, 0.f), min_nan(z.A.y, 0.f));
  z.gate_bias = mul2(load2<kWhole>(p.gate_bias, d, p.D, 0.f), both(-kLog2e));
  z.input_bias = mul2(load2<kWhole>(p.input_bias, d, p.D, 0.f), both(-kLog2e));
  z.mix = p.mix;
  z.has_a = p.A != nullptr;
  z.gated = p.input_gate != nullptr;
  return z;
}

// ---- joins -----------------------------------------------------------------------------------------------------------------------------
// The warp that has written to the other CTAs releases what it wrote, and what the CTA's barrier in front has put in front of it; for the other
// warps there is nothing to wait for (a release waits for all of a warp's stores, those of y among them).
__device__ __forceinline__ void cluster_arrive(bool wrote) {
  if (wrote) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  else asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ int cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return static_cast<int>(r);
}
__device__ __forceinline__ void store_remote(const void* mine, int rank, float4 v) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(mine))), "r"(rank));
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
constexpr int kMostCluster = 16;
__device__ __forceinline__ F first2(float4 v) { return make_float2(v.x, v.y); }
__device__ __forceinline__ F second2(float4 v) { return make_float2(v.z, v.w); }
__device__ __forceinline__ float4 four(F a, F b) { return make_float4(a.x, a.y, b.x, b.y); }

// Steps p h + q of the warps of a tile and of the tiles of a cluster, in two halves that alternate (a barrier lies between two uses of
// the same one).
template <int W> struct Steps {
  float4 warp[2][W][32], tile[2][kMostCluster][32];
  F end[2][32];      // what a tile leaves, where a CTA has all of them
};

struct At {
  int tile, b, rank, d, lane, warp, len;
  template <class P> __device__ __forceinline__ At(const P& p, const Plan& q) {
    rank = q.cluster > 1 ? cluster_rank() : 0;
    const int i = blockIdx.x / q.cluster;
    tile = i % q.tiles;
    b = i / q.tiles;
    lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
    d = tile * kCols + 2 * lane;
    len = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
  }
};

constexpr int kStages = 2;

template <class T, bool kWhole, bool kUsual, int S, int W>
__global__ void __launch_bounds__(32 * W, TTT_FWD_CTAS) gated_forward_kernel(const ttt_b200_gated_args p, const Plan q) {
  static_assert(S * W == kTile, "the warps' tokens make a tile");
  wait_for_predecessor();
  using R = Rows<T, S, kWhole>;
  __shared__ Steps<W> join;
  extern __shared__ __align__(16) unsigned char rings[];
  const At at(p, q);
  const int d0 = at.tile * kCols, C = q.cluster;
  const Weights z = weights_of<kWhole>(p, at.d);
  const R rx(p.x, p.x_stride[0], p.x_stride[1], at.b, d0, p.D), rg(p.gate, p.gate_stride[0], p.gate_stride[1], at.b, d0, p.D),
      ri(p.input_gate, p.input_stride[0], p.input_stride[1], at.b, d0, p.D);
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(rings)) + at.warp * (kStages * 3 * R::kStage);
  const int hop = C * kTile, first = at.rank * kTile + at.warp * S;      // tokens from one tile of a CTA to its next; the warp's first
  const int rounds = (at.len + hop - 1) / hop;
  auto ahead = [&](int j) {
    if (j < rounds) {
      const uint32_t to = ring + j % kStages * (3 * R::kStage);
      rx.copy(to, first + j * hop, at.len);
      rg.copy(to + R::kStage, first + j * hop, at.len);
      if (kUsual || z.gated) ri.copy(to + 2 * R::kStage, first + j * hop, at.len);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int j = 0; j < kStages - 1; ++j) ahead(j);
  F carry = load2<kWhole>(p.state ? p.state + static_cast<long>(at.b) * p.D : nullptr, at.d, p.D, 0.f);
  T* y = static_cast<T*>(p.y) + static_cast<long>(at.b) * p.T * p.D;
  for (int j = 0; j < rounds; ++j) {
    const int t0 = first + j * hop, half = j & 1;
    cp_async_wait<kStages - 2>();
    __syncwarp();      // the rows have landed for all lanes, and all are through with the place that the next ones take
    ahead(j + kStages - 1);
    const uint32_t from = ring + j % kStages * (3 * R::kStage);
    F a[S], u[S], whole = both(1.f), own = both(0.f);
#pragma unroll
    for (int t = 0; t < S; ++t) {
      Factors<false> f;
      factors<kUsual, false>(z, rg.get(from + R::kStage, t, t0 + t), [&] { return ri.get(from + 2 * R::kStage, t, t0 + t); }, f);
      a[t] = f.a;
      u[t] = mul2(f.w, rx.get(from, t, t0 + t));
    }
    if (t0 + S > at.len) {
#pragma unroll
      for (int t = 0; t < S; ++t)
        if (t0 + t >= at.len) a[t] = both(1.f), u[t] = both(0.f);
    }
#pragma unroll
    for (int t = 0; t < S; ++t) {
      own = fma2(a[t], own, u[t]);
      whole = mul2(whole, a[t]);
    }
    join.warp[half][at.warp][at.lane] = four(whole, own);
    __syncthreads();
    F h = C > 1 || j == 0 ? carry : join.end[half ^ 1][at.lane];
    if (C > 1) {
      if (at.warp == 0) {
        F P = both(1.f), H = both(0.f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float4 v = join.warp[half][w][at.lane];
          P = mul2(P, first2(v));
          H = fma2(first2(v), H, second2(v));
        }
        for (int r = 0; r < C; ++r) store_remote(&join.tile[half][at.rank][at.lane], r, four(P, H));
      }
      cluster_arrive(at.warp == 0);
      cluster_wait();
      F next = carry;
      for (int r = 0; r < C; ++r) {
        if (r == at.rank) h = next;
        const float4 v = join.tile[half][r][at.lane];
        next = fma2(first2(v), next, second2(v));
      }
      carry = next;
    }
    if (at.warp == 0 && p.checkpoints && t0 < at.len)
      store2<float, kWhole>(p.checkpoints + (static_cast<long>(at.b) * q.nck + j * C + at.rank) * p.D, at.d, p.D, h);
#pragma unroll
    for (int w = 0; w < W - 1; ++w) {
      if (w >= at.warp) break;
      const float4 v = join.warp[half][w][at.lane];
      h = fma2(first2(v), h, second2(v));
    }
    T* to = y + static_cast<long>(t0) * p.D;
    if (t0 + S <= at.len) {
#pragma unroll
      for (int t = 0; t < S; ++t) {
        h = fma2(a[t], h, u[t]);
        store2<T, kWhole>(to, at.d, p.D, h);
        to += p.D;
      }
    } else {
#pragma unroll
      for (int t = 0; t < S; ++t) {
        h = fma2(a[t], h, u[t]);
        if (t0 + t < p.T) store2<T, kWhole>(to, at.d, p.D, t0 + t < at.len ? h : both(0.f));
        to += p.D;
      }
    }
    if (C == 1 && at.warp == W - 1) carry = join.end[half][at.lane] = h;
  }
  if (p.final_state && at.rank == 0 && at.warp == W - 1) store2<float, kWhole>(p.final_state + static_cast<long>(at.b) * p.D, at.d, p.D, carry);
  for (int t0 = first + rounds * hop; t0 < p.T; t0 += hop)
    for (int t = t0; t < min(t0 + S, p.T); ++t) store2<T, kWhole>(y + static_cast<long>(t) * p.D, at.d, p.D, both(0.f));
}

// T: the gradients' type; I: that of x and the gates, or 8-bit values
template <class T, class I, bool kWhole, bool kUsual, int S, int W>
__global__ void __launch_bounds__(32 * W, TTT_BWD_CTAS) gated_backward_kernel(const ttt_b200_gated_args p, const Plan q) {
  static_assert(S * W == kTile, "the warps' tokens make a tile");
  wait_for_predecessor();
  using R = Rows<I, S, kWhole>;
  using U = Rows<T, S, kWhole>;
  constexpr uint32_t kStage = 3 * R::kStage + U::kStage;
  __shared__ Steps<W> join;
  __shared__ F back[2][W][32];
  extern __shared__ __align__(16) unsigned char rings[];
  const At at(p, q);
  const int d0 = at.tile * kCols, C = q.cluster;
  const Weights z = weights_of<kWhole>(p, at.d);
  const bool gated = kUsual || z.gated;
  const int groups = p.group ? (p.D + p.group - 1) / p.group : 0;
  const R rx(p.x, p.x_stride[0], p.x_stride[1], at.b, d0, p.D, p.x_scales, groups, p.group, p.T),
      rg(p.gate, p.gate_stride[0], p.gate_stride[1], at.b, d0, p.D, p.gate_scales, groups, p.group, p.T),
      ri(p.input_gate, p.input_stride[0], p.input_stride[1], at.b, d0, p.D, p.input_scales, groups, p.group, p.T);
  const U ru(p.grad_y, p.gy_stride[0], p.gy_stride[1], at.b, d0, p.D);
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(rings)) + at.warp * (kStages * kStage);
  const int hop = C * kTile, first = at.rank * kTile + at.warp * S;
  const int rounds = (at.len + hop - 1) / hop;
  auto ahead = [&](int j) {
    if (j >= 0) {
      const uint32_t to = ring + j % kStages * kStage;
      rx.copy(to, first + j * hop, at.len);
      rg.copy(to + R::kStage, first + j * hop, at.len);
      if (gated) ri.copy(to + 2 * R::kStage, first + j * hop, at.len);
      ru.copy(to + 3 * R::kStage, first + j * hop, at.len);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int j = 0; j < kStages - 1; ++j) ahead(rounds - 1 - j);
  const long batch = static_cast<long>(at.b) * p.T * p.D;
  T *gx = static_cast<T*>(p.grad_x) + batch, *gg = static_cast<T*>(p.grad_gate) + batch, *gi = static_cast<T*>(p.grad_input) + batch;
  auto put = [&](long o, F x, F g, F i) {
    store2<T, kWhole>(gx + o, at.d, p.D, x);
    store2<T, kWhole>(gg + o, at.d, p.D, g);
    if (gated) store2<T, kWhole>(gi + o, at.d, p.D, i);
  };
  F carry = load2<kWhole>(p.grad_final_state ? p.grad_final_state + static_cast<long>(at.b) * p.D : nullptr, at.d, p.D, 0.f);
  F sum_a = both(0.f), sum_g = sum_a, sum_i = sum_a;
  for (int j = rounds - 1; j >= 0; --j) {
    const int t0 = first + j * hop, half = j & 1;
    const bool some = t0 - at.warp * S < at.len;      // of the tile's tokens (else there is no checkpoint)
    F h = load2<kWhole>(some ? p.checkpoints + (static_cast<long>(at.b) * q.nck + j * C + at.rank) * p.D : nullptr, at.d, p.D, 0.f);
    cp_async_wait<kStages - 2>();
    __syncwarp();
    ahead(j - kStages + 1);
    const uint32_t from = ring + j % kStages * kStage;
    // of a token: a; w = b i; what there is of d log a / G without the state, which joins it; d log a's factors in d gate and dA; d input / G
    F a[S], w[S], slope[S], k[S], s[S], in[S], whole = both(1.f), own = both(0.f), left = both(0.f);
#pragma unroll
    for (int t = 0; t < S; ++t) {
      Factors<true> f;
      factors<kUsual, true>(z, rg.get(from + R::kStage, t, t0 + t), [&] { return ri.get(from + 2 * R::kStage, t, t0 + t); }, f);
      const F x = rx.get(from, t, t0 + t);
      a[t] = f.a, w[t] = f.w, k[t] = f.k, s[t] = f.s;
      slope[t] = mul2(f.slope, x);
      in[t] = mul2(f.rest, mul2(f.w, x));
    }
    if (t0 + S > at.len) {
#pragma unroll
      for (int t = 0; t < S; ++t)
        if (t0 + t >= at.len) a[t] = both(1.f), w[t] = both(0.f);
    }
#pragma unroll
    for (int t = 0; t < S; ++t) {
      own = fma2(a[t], own, mul2(w[t], rx.get(from, t, t0 + t)));
      whole = mul2(whole, a[t]);
    }
#pragma unroll
    for (int t = S - 1; t >= 0; --t) left = mul2(a[t], add2(ru.get(from + 3 * R::kStage, t, t0 + t), left));
    join.warp[half][at.warp][at.lane] = four(whole, own);
    back[half][at.warp][at.lane] = left;
    __syncthreads();
    F c = C > 1 || j == rounds - 1 ? carry : join.end[half ^ 1][at.lane];
    if (C > 1) {
      if (at.warp == W - 1) {
        F P = both(1.f), Q = both(0.f);
#pragma unroll
        for (int v = W - 1; v >= 0; --v) {
          const F f = first2(join.warp[half][v][at.lane]);
          P = mul2(P, f);
          Q = fma2(f, Q, back[half][v][at.lane]);
        }
        for (int r = 0; r < C; ++r) store_remote(&join.tile[half][at.rank][at.lane], r, four(P, Q));
      }
      cluster_arrive(at.warp == W - 1);
    }
#pragma unroll
    for (int v = 0; v < W; ++v) {
      if (v >= at.warp) break;
      const float4 f = join.warp[half][v][at.lane];
      h = fma2(first2(f), h, second2(f));
    }
    // to h_{t-1}, and with it to d log a / G
#pragma unroll
    for (int t = 0; t < S; ++t) {
      const F kept = mul2(a[t], h);
      slope[t] = add2(kept, slope[t]);
      h = fma2(w[t], rx.get(from, t, t0 + t), kept);
    }
    if (C > 1) {
      cluster_wait();
      F next = carry;
      for (int r = C - 1; r >= 0; --r) {
        if (r == at.rank) c = next;
        const float4 v = join.tile[half][r][at.lane];
        next = fma2(first2(v), next, second2(v));
      }
      carry = next;
    }
#pragma unroll
    for (int v = W - 1; v > 0; --v) {
      if (v <= at.warp) break;
      c = fma2(first2(join.warp[half][v][at.lane]), c, back[half][v][at.lane]);
    }
    long o = static_cast<long>(t0 + S - 1) * p.D;
    auto one = [&](int t) {
      const F G = add2(ru.get(from + 3 * R::kStage, t, t0 + t), c);
      c = mul2(a[t], G);
      const F dl = mul2(G, slope[t]), dg = mul2(dl, k[t]), di = mul2(G, in[t]);
      sum_a = fma2(dl, s[t], sum_a);
      sum_g = add2(sum_g, dg);
      sum_i = add2(sum_i, di);
      put(o, mul2(G, w[t]), dg, di);
    };
    if (t0 + S <= at.len) {
#pragma unroll
      for (int t = S - 1; t >= 0; --t, o -= p.D) one(t);
    } else {
#pragma unroll
      for (int t = S - 1; t >= 0; --t, o -= p.D) {
        if (t0 + t < at.len) one(t);
        else if (t0 + t < p.T) put(o, both(0.f), both(0.f), both(0.f));
      }
    }
    if (C == 1 && at.warp == 0) carry = join.end[half][at.lane] = c;
  }
  if (p.grad_state && at.rank == 0 && at.warp == 0) store2<float, kWhole>(p.grad_state + static_cast<long>(at.b) * p.D, at.d, p.D, carry);
  for (int t0 = first + rounds * hop; t0 < p.T; t0 += hop)
    for (int t = t0; t < min(t0 + S, p.T); ++t) put(static_cast<long>(t) * p.D, both(0.f), both(0.f), both(0.f));
  // the warps' sums, in their order
  __shared__ F sums[3][W][32];
  sums[0][at.warp][at.lane] = sum_a;
  sums[1][at.warp][at.lane] = sum_g;
  sums[2][at.warp][at.lane] = sum_i;
  __syncthreads();
  if (at.warp < 3) {
    F s = sums[at.warp][0][at.lane];
#pragma unroll
    for (int w = 1; w < W; ++w) s = add2(s, sums[at.warp][w][at.lane]);
    if (at.warp == 0 && p.A) {      // A counts as 0 where it is above
      const F A = load2<kWhole>(p.A, at.d, p.D, 0.f);
      s = make_float2(A.x > 0.f ? 0.f : s.x, A.y > 0.f ? 0.f : s.y);
    }
    store2<float, kWhole>(q.part + (static_cast<long>(at.b) * C + at.rank) * 3 * p.D + static_cast<long>(at.warp) * p.D, at.d, p.D, s);
  }
}

// A row of the batch and 256 channels to a CTA.  Rows that name the same slot are taken in their order by the CTA of the first of
// them, so that no two CTAs touch a state.
template <class T, bool kWhole> __global__ void __launch_bounds__(128) gated_step_kernel(const ttt_b200_gated_args p, int tiles) {
  wait_for_predecessor();
  const int b0 = blockIdx.x / tiles, d = (blockIdx.x % tiles * 128 + threadIdx.x) * 2;
  T* ys = static_cast<T*>(p.y);
  int slot = b0, more = 0;
  if (p.slots) {
    slot = p.slots[b0];
    if (slot < 0 || slot >= p.rows) {
      store2<T, kWhole>(ys + static_cast<long>(b0) * p.D, d, p.D, both(0.f));
      return;
    }
    int before = 0, after = 0;
    for (int r = threadIdx.x; r < p.B; r += 128)
      if (r != b0 && p.slots[r] == slot) (r < b0 ? before : after) = 1;
    if (__syncthreads_or(before)) return;
    more = __syncthreads_or(after);
  }
  if (d >= p.D) return;
  auto two = [&](const void* base, int64_t stride, int b) {
    const T* r = static_cast<const T*>(base) + b * stride + d;
    if constexpr (kWhole) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(r));
      else if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(r));
      else return *reinterpret_cast<const F*>(r);
    } else {
      return make_float2(to_f32(r[0]), d + 1 < p.D ? to_f32(r[1]) : 0.f);
    }
  };
  const Weights z = weights_of<kWhole>(p, d);
  float* st = p.state_io + static_cast<long>(slot) * p.D;
  F h = load2<kWhole>(st, d, p.D, 0.f);
  for (int b = b0; b < p.B; ++b) {
    if (b != b0 && p.slots[b] != slot) continue;
    Factors<false> f;
    const F x = two(p.x, p.x_stride[0], b);
    factors<false, false>(z, two(p.gate, p.gate_stride[0], b), [&] { return two(p.input_gate, p.input_stride[0], b); }, f);
    h = fma2(f.a, h, mul2(f.w, x));
    store2<T, kWhole>(ys + static_cast<long>(b) * p.D, d, p.D, h);
    if (!more) break;
  }
  store2<float, kWhole>(st, d, p.D, h);
}

// ---- host --------------------------------------------------------------------------------------------------------------
int check(const ttt_b200_gated_args* p) {
  if (!p) return fail("gated scan: NULL argument struct");
  if (p->B < 0 || p->T < 0 || p->T > 1 << 30 || p->D < 1 || p->D > 1 << 30) return fail("gated scan: B, T >= 0, D >= 1, T and D at most 2^30");
  if (p->dtype < TTT_B200_BF16 || p->dtype > TTT_B200_FP32) return fail("gated scan: unknown element type");
  if (p->mix < TTT_B200_MIX_NONE || p->mix > TTT_B200_MIX_LINEAR) return fail("gated scan: mix is none, sqrt or linear");
  if (p->group && p->group != 32 && p->group != 64 && p->group != 128) return fail("gated scan: groups of 32, 64 or 128 values, or 0");
  return TTT_B200_OK;
}

bool rows16(const void* a, const int64_t* st, int es) { return aligned16(a) && st[0] * es % 16 == 0 && st[1] * es % 16 == 0; }
bool even(const void* a, int es) { return reinterpret_cast<uintptr_t>(a) % (2 * es) == 0; }
int size_of(const ttt_b200_gated_args& p) { return p.dtype == TTT_B200_FP32 ? 4 : 2; }
// whether lanes can take their two channels as a pair, and rows be copied in 16-byte pieces
bool whole(const ttt_b200_gated_args& p, bool backward) {
  const int es = size_of(p), in = p.group ? 1 : es;
  bool ok = p.D % 2 == 0 && rows16(p.x, p.x_stride, in) && rows16(p.gate, p.gate_stride, in) && (!p.input_gate || rows16(p.input_gate, p.input_stride, in));
  for (const float* v : {p.A, p.gate_bias, p.input_bias, p.state, static_cast<const float*>(p.final_state), static_cast<const float*>(p.checkpoints), p.grad_final_state,
                         static_cast<const float*>(p.grad_state)})
    ok = ok && even(v, 4);
  if (!backward) return ok && even(p.y, es);
  return ok && rows16(p.grad_y, p.gy_stride, es) && even(p.grad_x, es) && even(p.grad_gate, es) && even(p.grad_input, es);
}

// CTAs of a cluster: as many as leave two to three CTAs to an SM, and no more than there are tiles.
void plan(Plan& q, const ttt_b200_gated_args& p) {
  q.tiles = (p.D - 1) / kCols + 1;
  q.nck = (p.T - 1) / kTile + 1;
  const long columns = static_cast<long>(q.tiles) * p.B, sms = sm_count();
  for (q.cluster = 1; q.cluster < kMostCluster && q.cluster < q.nck && columns * q.cluster < sms; q.cluster *= 2) {}
#ifdef TTT_PROBE
  if (getenv("TTT_PROBE_C")) q.cluster = atoi(getenv("TTT_PROBE_C"));
#endif
}

template <auto kKernel> int launch(const Plan& q, const ttt_b200_gated_args& p, int threads, uint32_t bytes, cudaStream_t s, const char* what) {
  const long grid = static_cast<long>(p.B) * q.tiles * q.cluster;
  if (grid > 0x7fffffffL) return fail("gated scan: too many CTAs");
  if (bytes > 16 * 1024)      // (with the static part 48 KB is the most without asking)
    if (int rc = allow_shared<kKernel>()) return rc;
  if (q.cluster > 8)
    if (cudaError_t e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) return ttt_set_error(TTT_B200_ERR_LAUNCH, cudaGetErrorString(e));
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = q.cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = q.cluster > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kKernel, p, q);
  return launched(what);
}

bool usual(const ttt_b200_gated_args& p) { return p.A && p.input_gate && p.mix == TTT_B200_MIX_SQRT; }

template <class T, bool kWhole> int forward(const ttt_b200_gated_args& p, const Plan& q, cudaStream_t s) {
  constexpr int S = TTT_FWD_S, W = kTile / S;
  constexpr uint32_t bytes = W * kStages * 3 * Rows<T, S, kWhole>::kStage;
  return usual(p) ? launch<gated_forward_kernel<T, kWhole, true, S, W>>(q, p, 32 * W, bytes, s, "gated scan")
                  : launch<gated_forward_kernel<T, kWhole, false, S, W>>(q, p, 32 * W, bytes, s, "gated scan");
}
template <class T, class I, bool kWhole> int backward_of(const ttt_b200_gated_args& p, const Plan& q, cudaStream_t s) {
  constexpr int S = TTT_BWD_S, W = kTile / S;
  constexpr uint32_t bytes = W * kStages * (3 * Rows<I, S, kWhole>::kStage + Rows<T, S, kWhole>::kStage);
  return usual(p) ? launch<gated_backward_kernel<T, I, kWhole, true, S, W>>(q, p, 32 * W, bytes, s, "gated scan backward")
                  : launch<gated_backward_kernel<T, I, kWhole, false, S, W>>(q, p, 32 * W, bytes, s, "gated scan backward");
}
template <class T> int backward(const ttt_b200_gated_args& p, cudaStream_t s) {
  Plan q = {};
  plan(q, p);
  q.part = static_cast<float*>(p.scratch);
  int rc;
  if (p.group) rc = whole(p, true) ? backward_of<T, E4, true>(p, q, s) : backward_of<T, E4, false>(p, q, s);
  else rc = whole(p, true) ? backward_of<T, T, true>(p, q, s) : backward_of<T, T, false>(p, q, s);
  if (rc) return rc;
  const long D = p.D;
  const int parts = p.B * q.cluster;
  const ttt_sum_job jobs[] = {{q.part, p.grad_A, D, 3 * D, parts, TTT_B200_FP32, 0},
                              {q.part + D, p.grad_gate_bias, D, 3 * D, parts, TTT_B200_FP32, 0},
                              {q.part + 2 * D, p.grad_input_bias, D, 3 * D, parts, TTT_B200_FP32, 0}};
  return ttt_sum_parts(jobs, 3, s);
}
template <class T> int step(const ttt_b200_gated_args& p, cudaStream_t s) {
  const int es = size_of(p);
  auto rows = [&](const void* a, int64_t st) { return even(a, es) && st % 2 == 0; };
  bool ok = p.D % 2 == 0 && rows(p.x, p.x_stride[0]) && rows(p.gate, p.gate_stride[0]) && rows(p.input_gate, p.input_stride[0]) && even(p.y, es);
  for (const float* v : {p.A, p.gate_bias, p.input_bias, static_cast<const float*>(p.state_io)}) ok = ok && even(v, 4);
  const int tiles = (p.D + 255) / 256;
  const long grid = static_cast<long>(p.B) * tiles;
  if (grid > 0x7fffffffL) return fail("gated scan step: too many CTAs");
  ttt_launch_overlapped(ok ? gated_step_kernel<T, true> : gated_step_kernel<T, false>, static_cast<int>(grid), 128, 0, s, p, tiles);
  return launched("gated scan step");
}

}  // namespace

extern "C" uint64_t ttt_b200_gated_scan_scratch_bytes(const ttt_b200_gated_args* p) {
  if (check(p) || p->B == 0 || p->T == 0) return 0;
  Plan q = {};
  plan(q, *p);
  return static_cast<uint64_t>(p->B) * q.cluster * 3 * p->D * sizeof(float);
}

extern "C" int ttt_b200_gated_scan(const ttt_b200_gated_args* p, void* stream) {
  if (int rc = check(p)) return rc;
  if (!p->x || !p->gate || !p->y) return fail("gated scan: null tensor pointer");
  if (p->B == 0 || p->T == 0) return fail("gated scan: no tokens");
  if (p->group) return fail("gated scan: 8-bit inputs are for the backward pass");
  if (p->input_bias && !p->input_gate) return fail("gated scan: input_bias without input_gate");
  Plan q = {};
  plan(q, *p);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  TTT_WITH_TYPE(p->dtype, return whole(*p, false) ? (forward<Elem, true>(*p, q, s)) : (forward<Elem, false>(*p, q, s)))
  return TTT_B200_OK;
}

extern "C" int ttt_b200_gated_scan_backward(const ttt_b200_gated_args* p, void* stream) {
  if (int rc = check(p)) return rc;
  if (!p->x || !p->gate || !p->checkpoints || !p->grad_y || !p->grad_x || !p->grad_gate || (p->input_gate && !p->grad_input))
    return fail("gated scan backward: null tensor pointer");
  if (p->group && (!p->x_scales || !p->gate_scales || (p->input_gate && !p->input_scales))) return fail("gated scan backward: 8-bit inputs without scales");
  if (p->B == 0 || p->T == 0) return fail("gated scan backward: no tokens");
  if ((p->input_bias && !p->input_gate) || (p->grad_A && !p->A)) return fail("gated scan backward: a gradient or bias of what is not there");
  if (!p->scratch || p->scratch_bytes < ttt_b200_gated_scan_scratch_bytes(p) || !aligned16(p->scratch))
    return fail("gated scan backward: scratch is missing, too small or not 16-byte aligned");
  TTT_WITH_TYPE(p->dtype, return backward<Elem>(*p, static_cast<cudaStream_t>(stream)))
  return TTT_B200_OK;
}

extern "C" int ttt_b200_gated_scan_step(const ttt_b200_gated_args* p, void* stream) {
  if (int rc = check(p)) return rc;
  if (!p->x || !p->gate || !p->y || !p->state_io) return fail("gated scan step: null tensor pointer");
  if (p->B == 0) return fail("gated scan step: no rows");
  if (p->group) return fail("gated scan step: 8-bit inputs are for the backward pass");
  if (p->input_bias && !p->input_gate) return fail("gated scan step: input_bias without input_gate");
  if (p->slots ? p->rows < 1 : p->rows != p->B) return fail("gated scan step: the state has another number of rows");
  TTT_WITH_TYPE(p->dtype, return step<Elem>(*p, static_cast<cudaStream_t>(stream)))
  return TTT_B200_OK;
}
