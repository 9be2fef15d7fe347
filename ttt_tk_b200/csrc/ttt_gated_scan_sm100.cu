// Gated linear recurrence: forward for prompts and training, backward, and the step of single tokens.
//
//   s = sigmoid(gate + gate_bias);  log a = A[d] s, A <= 0 (without A: a = s);  b = sqrt(1 - a^2), 1 - a or 1;
//   i = sigmoid(input_gate + input_bias);  u = b i x;  h_t = a_t h_{t-1} + u_t;  y = h
//
// Backward, with G_t the gradient with respect to h_t and c_t = a_t G_t what it leaves for the token before:  G_t = dy_t + c_{t+1};
// dx = G b i;  d input_gate = G b x i (1 - i);  d log a = G (a h_{t-1} + i x db/dlog a), db/dlog a = -a^2 / b, -a or 0;
// d gate = d log a times A s (1 - s), without A times 1 - s;  dA = sum d log a s;  dh_{-1} = c_0.
//
// Of a token and pair of channels the forward reads 12 bytes and writes 4 (bf16; backward 16 and 12), for 10 operations of the exponential unit and some 80
// instructions (backward 180): with every SM full the unit, the heavy half of the fp32 pipe and the issue slots are each 60 % busy, the memory 65 %.
// A recurrence of steps h -> p h + q joins: two after one another are p2 p1, p2 q1 + q2.  So a warp has S tokens of 64 channels in registers (two
// neighbouring channels to a lane), the warps of a CTA have the tokens behind one another of a tile, each takes its tokens from zero, and all join
// what is in front of them over shared memory: one pass over the data, one barrier a tile.
// The backward starts every 64 tokens from the state that the forward left of them and joins both directions over the same barrier.
// Where channels and sequences do not fill the GPU the sequence is cut into chunks: a first kernel leaves what each chunk does to a state, and
// every chunk of the main one begins with the steps of those in front of it.  The order of the joins is fixed.
//
// Measured, bf16 with A, root and input gate, us (TB/s of the bytes above), forward / backward with the sum of its parts / the same from 8-bit inputs: 37 x 1024
// tokens of 2048 channels 147 (4.2) / 276 (3.9) / 292 (2.9); 8 x 4096 of 2048 148 / 275 / 292, 14 % of it SMs with one CTA for two; 4 x 2048 of 2048 45 / 81 /
// 85; 16384 of 1024, in chunks, 73 / 97 / 101, of which the chunks' steps are 31, 21 and 23.  Not faster: three or four CTAs to an SM (80 and 64
// registers: 147 -> 150 and 162); clusters of CTAs along the sequence, joined over distributed shared memory, in place of chunks (16384 of 1024 102, a
// tile ahead of the exchange 107); four tokens to a warp; constants as kernel arguments (154 -> 165).
#include <cuda_fp8.h>

#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "ttt_eight_bits.cuh"
#include "ttt_sum_parts.h"

namespace {

using namespace ttt;

using F = float2;
using E4 = __nv_fp8_e4m3;
constexpr int kEvery = TTT_B200_GATED_INTERVAL;     // tokens between two checkpoints
constexpr int S = 8;                                // tokens of a warp's part of a tile; a tile is W of them, 64 tokens or 128
constexpr int kCols = 64;                           // channels of a CTA

constexpr int kMostChunks = 32;                     // that a CTA joins the steps of

struct Plan {
  int tiles;      // CTAs side by side: channels / 64
  int nck;        // checkpoints of a sequence
  int warps;      // of a CTA
  int chunk;      // tiles that a CTA has
  int chunks;
  float* ends;    // [B][chunks][2][D]: p and q of a chunk's step p h + q
  float* part;    // backward: [B * chunks][3][D]
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
__device__ __forceinline__ float sqrt_fast(float v) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
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

// 2^v and 1 - 2^v for v <= 0: v = k + f, |f| <= 1/2, both exact, 2^f - 1 = f p(f) with the polynomial of fifth degree that is off by the least part
// of it (2.1e-08, fitted).  Both from one series: 1 - a keeps its digits where a is close to one, which is where these recurrences are, and the
// exponential unit, which is close to its limit, is left alone.  Where k comes to -127 the power's bits are those of 0: 2^v is 0 from there on, as far
// as A makes v.
__device__ __forceinline__ void exp2_both(F v, F& a, F& rest) {
  v = make_float2(max_nan(v.x, -127.f), max_nan(v.y, -127.f));
  constexpr float magic = 12582912.f;      // 1.5 2^23: the sum's last bits are the rounded integer
  const F k = add2(v, both(magic));
  const F f = add2(v, fma2(k, both(-1.f), both(magic)));
  F q = fma2(f, both(0.00015403512225020677f), both(0.0013390964595600963f));
  q = fma2(q, f, both(0.009618238545954227f));
  q = fma2(q, f, both(0.055503569543361664f));
  q = fma2(q, f, both(0.24022649228572845f));
  q = fma2(q, f, both(0.6931471824645996f));
  q = mul2(q, f);
  const F two = make_float2(__int_as_float((__float_as_int(k.x) << 23) + 0x3f800000), __int_as_float((__float_as_int(k.y) << 23) + 0x3f800000));
  q = mul2(q, two);      // exact but where it is below the normal numbers
  a = add2(q, two);
  rest = fma2(q, both(-1.f), fma2(two, both(-1.f), both(1.f)));
}

// What does not change over the tokens of a lane's channels.
struct Weights {
  F A, A2, gate_bias, input_bias;      // A2 = A log2 e
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
// What makes them up, a token at a time.
template <bool kBack> __device__ __forceinline__ void decay_of(const Weights& z, F gate, Factors<kBack>& f, F& rest) {      // rest: 1 - a
  F s, o;
  sigmoid<kBack>(gate, z.gate_bias, 127.f, s, o);
  exp2_both(mul2(s, z.A2), f.a, rest);
  if constexpr (kBack) f.s = s, f.k = mul2(mul2(s, z.A), o);
}
template <bool kBack> __device__ __forceinline__ void root_of(F rest, Factors<kBack>& f) {
  const F q = mul2(rest, fma2(rest, both(-1.f), both(2.f)));      // 1 - a^2
  if constexpr (kBack) {      // where that is no normal number b is 0, and so is its slope
    F r = make_float2(rsqrt_fast(q.x), rsqrt_fast(q.y));
    r = make_float2(q.x < 1.17549435e-38f ? 0.f : r.x, q.y < 1.17549435e-38f ? 0.f : r.y);
    f.w = mul2(q, r);
    f.slope = mul2(mul2(f.a, f.a), neg(r));
  } else {
    f.w = make_float2(sqrt_fast(q.x), sqrt_fast(q.y));
  }
}
template <bool kBack> __device__ __forceinline__ void let_in(const Weights& z, F input, Factors<kBack>& f) {
  F i, o;
  sigmoid<kBack>(input, z.input_bias, 126.f, i, o);
  f.w = mul2(f.w, i);
  if constexpr (kBack) f.slope = mul2(f.slope, i), f.rest = o;
}

// Those of S tokens; `gate` and `input` give a token's.  kUsual: A, the root and an input gate, which leaves nothing to decide (8 x 4096 x 2048 bf16 158 ->
// 148 us forward, 323 -> 288 backward at the time).  Otherwise each part is decided once for all of the tokens, whose arithmetic then overlaps as well (decided for each
// token, 16 x 2048 x 2048 bf16: without A and input gate, linear 111 -> 96 and 230 -> 222 us; with both and no mix 180 -> 145 and 302 -> 296).
template <bool kUsual, bool kBack, int S, class Gate, class Input>
__device__ __forceinline__ void factors(const Weights& z, Gate gate, Input input, Factors<kBack> (&f)[S]) {
  if constexpr (kUsual) {
#pragma unroll
    for (int t = 0; t < S; ++t) {
      F rest;
      decay_of(z, gate(t), f[t], rest);
      root_of(rest, f[t]);
      let_in(z, input(t), f[t]);
    }
  } else {
    F rest[S];
    if (z.has_a) {
#pragma unroll
      for (int t = 0; t < S; ++t) decay_of(z, gate(t), f[t], rest[t]);
    } else {
#pragma unroll
      for (int t = 0; t < S; ++t) {
        sigmoid<true>(gate(t), z.gate_bias, 126.f, f[t].a, rest[t]);
        if constexpr (kBack) f[t].s = f[t].a, f[t].k = rest[t];
      }
    }
    if (z.mix == TTT_B200_MIX_SQRT) {
#pragma unroll
      for (int t = 0; t < S; ++t) root_of(rest[t], f[t]);
    } else if (z.mix == TTT_B200_MIX_LINEAR) {
#pragma unroll
      for (int t = 0; t < S; ++t) {
        f[t].w = rest[t];
        if constexpr (kBack) f[t].slope = neg(f[t].a);
      }
    } else {
#pragma unroll
      for (int t = 0; t < S; ++t) {
        f[t].w = both(1.f);
        if constexpr (kBack) f[t].slope = both(0.f);
      }
    }
    if (z.gated) {
#pragma unroll
      for (int t = 0; t < S; ++t) let_in(z, input(t), f[t]);
    } else if constexpr (kBack) {
#pragma unroll
      for (int t = 0; t < S; ++t) f[t].rest = both(0.f);
    }
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

enum { kSingles, kPairs, kWholeRows };
// S rows of 64 channels of a tensor, copied ahead by a warp into its own place in shared memory.
//   kWhole    rows start on 16-byte boundaries: 16-byte pieces
//   kPairs    rows start on boundaries of two values: the 16-byte blocks that a row touches (the first and the last may hold its neighbours too), from which
//             pairs are picked at the row's offset
//   kSingles  the same, and values one by one
template <class T, int kMode> struct Rows {
  static constexpr bool kWhole = kMode == kWholeRows;
  static constexpr int es = sizeof(T), kBytes = kCols * es, kPitch = kWhole ? kBytes : kBytes + 16, kPieces = kPitch / 16;
  static constexpr uint32_t kStage = S * kPitch;      // bytes
  static_assert(kStage % 16 == 0, "copies start on 16-byte boundaries");
  const char* base;      // channel d0 of the first token
  int64_t step;          // bytes from token to token
  int cols;              // bytes of a row that there are
  __device__ __forceinline__ Rows(const void* p, const int64_t (&stride)[2], int b, int d0, int D)
      : base(static_cast<const char*>(p) + (b * stride[0] + d0) * es), step(stride[1] * es), cols(min(D - d0, kCols) * es) {}
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
  }
  // this lane's two channels of token t (row i of those at `from`)
  __device__ __forceinline__ F get(uint32_t from, int i, int t) const {
    const int lane = threadIdx.x & 31;
    if constexpr (kWhole) {
      return pair_of<T>(from + i * kPitch + lane * 2 * es);
    } else {
      const uint32_t at = from + i * kPitch + (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(base) + t * step) & 15) + lane * 2 * es;
      if constexpr (kMode == kPairs) return pair_of<T>(at);
      else return make_float2(value_of<T>(at), value_of<T>(at + es));
    }
  }
};
// The scales of 8-bit x, gate and input gate, next to one another for a token and each half of the channels; T of another size: there are none.
template <class T> struct Scales {
  static constexpr bool kThere = sizeof(T) == 1;
  static constexpr uint32_t kStage = kThere ? S * 2 * 16 : 0;
  const float* base[3];      // of channel d0 of the first token, or NULL
  int64_t step;
  int second;      // distance of the second 32 channels' scale, 0 or 1; -1: there are none
  __device__ __forceinline__ Scales(const ttt_b200_gated_args& p, int b, int d0) {
    if constexpr (kThere) {
      const int groups = (p.D + p.group - 1) / p.group;
      const int64_t at = static_cast<int64_t>(b) * p.T * groups + d0 / p.group;
      base[0] = p.x_scales + at;
      base[1] = p.gate_scales + at;
      base[2] = p.input_gate ? p.input_scales + at : nullptr;
      step = groups;
      second = d0 + 32 < p.D ? (d0 + 32) / p.group - d0 / p.group : -1;
    }
  }
  __device__ __forceinline__ void copy(uint32_t to, int t, int stop) const {
    if constexpr (kThere) {
      static_assert(S * 2 <= 32, "a lane for each half of a token");
      const int lane = threadIdx.x & 31;
      if (lane >= 2 * S) return;
      const bool in = t + lane / 2 < stop && !(lane % 2 && second < 0);
      const int64_t at = in ? (t + lane / 2) * step + (lane % 2 ? second : 0) : 0;
#pragma unroll
      for (int k = 0; k < 3; ++k)
        if (base[k]) cp_async4_at(to + lane * 16 + k * 4, base[k] + at, in ? 4 : 0);
    }
  }
  __device__ __forceinline__ float4 get(uint32_t from, int i) const {
    if constexpr (kThere) {
      const uint4 r = shared_load16(from + (i * 2 + (threadIdx.x & 31) / 16) * 16);
      return make_float4(__uint_as_float(r.x), __uint_as_float(r.y), __uint_as_float(r.z), 0.f);
    } else {
      return make_float4(1.f, 1.f, 1.f, 0.f);
    }
  }
  // x, at most what unpacking makes of it (16 instructions a tile and warp: 8 x 4096 x 2048 286 -> 288 us; bytes put right in shared memory behind a vote on the
  // scales 293); a gate that comes out infinite is as closed or open as it was
  static __device__ __forceinline__ F bounded(F v, float scale) {
    v = apply(v, scale);
    if constexpr (kThere) v = make_float2(at_most(v.x, kMostOf<float>), at_most(v.y, kMostOf<float>));
    return v;
  }
  static __device__ __forceinline__ F apply(F v, float scale) {
    if constexpr (kThere) return mul2(v, both(scale));
    else return v;
  }
};

// ---- a lane's two channels in global memory -------------------------------------------------------------------------------------------
template <int kMode> __device__ __forceinline__ F load2(const float* p, int d, int D, float none) {
  if (!p || d >= D) return both(none);
  if constexpr (kMode != kSingles) return *reinterpret_cast<const F*>(p + d);
  return make_float2(p[d], d + 1 < D ? p[d + 1] : none);
}
template <class T, int kMode> __device__ __forceinline__ void store2(T* p, int d, int D, F v) {
  if (d >= D) return;
  if constexpr (kMode != kSingles) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) *reinterpret_cast<__nv_bfloat162*>(p + d) = __float22bfloat162_rn(v);
    else if constexpr (std::is_same<T, __half>::value) *reinterpret_cast<__half2*>(p + d) = __float22half2_rn(v);
    else *reinterpret_cast<F*>(p + d) = v;
  } else {
    p[d] = from_f32<T>(v.x);
    if (d + 1 < D) p[d + 1] = from_f32<T>(v.y);
  }
}
template <int kMode> __device__ __forceinline__ Weights weights_of(const ttt_b200_gated_args& p, int d) {
  Weights z;
  z.A = load2<kMode>(p.A, d, p.D, 0.f);
  z.A = make_float2(min_nan(z.A.x, 0.f), min_nan(z.A.y, 0.f));
  z.A2 = make_float2(max_nan(z.A.x, -FLT_MAX / 2), max_nan(z.A.y, -FLT_MAX / 2));
  z.A2 = mul2(z.A2, both(kLog2e));
  z.gate_bias = mul2(load2<kMode>(p.gate_bias, d, p.D, 0.f), both(-kLog2e));
  z.input_bias = mul2(load2<kMode>(p.input_bias, d, p.D, 0.f), both(-kLog2e));
  z.mix = p.mix;
  z.has_a = p.A != nullptr;
  z.gated = p.input_gate != nullptr;
  return z;
}

// ---- joins -----------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ F first2(float4 v) { return make_float2(v.x, v.y); }
__device__ __forceinline__ F second2(float4 v) { return make_float2(v.z, v.w); }
__device__ __forceinline__ float4 four(F a, F b) { return make_float4(a.x, a.y, b.x, b.y); }

// p of a step over several tokens, a product that may be less than fp32 has: never 0, or an infinite h would leave the step as no number, where the tokens one by
// one leave it as it is.  (The least number times a finite h is at most 2^-21.)
__device__ __forceinline__ F some(F p) { return make_float2(max_nan(p.x, 0x1p-149f), max_nan(p.y, 0x1p-149f)); }

// Steps p h + q of the warps of a tile, in two halves that alternate (a barrier lies between two uses of the same one).
template <int W> struct Steps {
  float4 warp[2][W][32];
  F end[2][32];      // what a tile leaves
};

template <int W> struct At {
  static constexpr int kTile = S * W;
  int tile, b, chunk, d, lane, warp, len, first, last;      // `first`, `last`: tiles of the chunk that have tokens, and the one behind them
  __device__ __forceinline__ At(const ttt_b200_gated_args& p, const Plan& q, int chunks) {
    const int i = blockIdx.x / q.tiles;
    tile = blockIdx.x % q.tiles;
    chunk = i % chunks;
    b = i / chunks;
    lane = threadIdx.x & 31;
    warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);      // known to be the same for a warp: addresses in uniform registers
    d = tile * kCols + 2 * lane;
    len = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
    first = chunk * q.chunk;
    last = max(first, min(first + q.chunk, (len + kTile - 1) / kTile));
  }
  // behind the chunk's last tile
  __device__ __forceinline__ int end(const Plan& q, int p_T) const { return min((chunk + 1) * q.chunk, (p_T + kTile - 1) / kTile); }
};
// Of what stands in front of a chunk (backward: behind it) the steps, one after another.
template <int kMode, bool kBack, class W> __device__ __forceinline__ F join_chunks(const ttt_b200_gated_args& p, const Plan& q, const W& at, F h) {
  const int n = kBack ? q.chunks - 1 - at.chunk : at.chunk;
  const float* ends = q.ends + static_cast<long>(at.b) * q.chunks * 2 * p.D;
#pragma unroll 8
  for (int k = 0; k < n; ++k) {
    const float* e = ends + static_cast<long>(kBack ? q.chunks - 1 - k : k) * 2 * p.D;
    h = fma2(load2<kMode>(e, at.d, p.D, 1.f), h, load2<kMode>(e + p.D, at.d, p.D, 0.f));
  }
  return h;
}

constexpr int kStages = 2;

// Where channels and sequences do not fill the GPU: a chunk's step p h + q, forward (kBack: backward, of which q is c in front of the chunk for
// nothing behind it).  Each warp has tokens after one another, and nothing to wait for until the end.  What the main kernels compute of a token is
// computed here before: but for the last chunk (the first one).
template <class T, class I, int kMode, bool kUsual, bool kBack, int W>
__global__ void __launch_bounds__(32 * W, 16 / W) gated_ends_kernel(const ttt_b200_gated_args p, const Plan q) {
  wait_for_predecessor();
  using R = Rows<I, kMode>;
  using U = Rows<T, kMode>;
  constexpr uint32_t kStage = kBack ? R::kStage + U::kStage + Scales<I>::kStage : 3 * R::kStage;
  __shared__ float4 steps[W][32];
  extern __shared__ __align__(16) unsigned char rings[];
  At<W> at(p, q, q.chunks - 1);
  constexpr int kTile = At<W>::kTile;
  if constexpr (kBack) {      // all but the first
    at.first += q.chunk;
    ++at.chunk;
    at.last = max(at.first, min(at.first + q.chunk, (at.len + kTile - 1) / kTile));
  }
  const int d0 = at.tile * kCols;
  const Weights z = weights_of<kMode>(p, at.d);
  const R rx(p.x, p.x_stride, at.b, d0, p.D), rg(p.gate, p.gate_stride, at.b, d0, p.D), ri(p.input_gate, p.input_stride, at.b, d0, p.D);
  const U ru(p.grad_y, p.gy_stride, at.b, d0, p.D);
  const Scales<I> scales(p, at.b, d0);
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(rings)) + at.warp * (kStages * kStage);
  const int rounds = at.last - at.first, first = at.first * kTile + at.warp * rounds * S;
  auto ahead = [&](int j) {
    if (j < rounds) {
      const uint32_t to = ring + j % kStages * kStage;
      const int t = first + j * S;
      rg.copy(to, t, at.len);
      if constexpr (kBack) {
        ru.copy(to + R::kStage, t, at.len);
        scales.copy(to + R::kStage + U::kStage, t, at.len);
      } else {
        rx.copy(to + R::kStage, t, at.len);
        if (kUsual || z.gated) ri.copy(to + 2 * R::kStage, t, at.len);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int j = 0; j < kStages - 1; ++j) ahead(j);
  F whole = both(1.f), own = both(0.f);
  for (int j = 0; j < rounds; ++j) {
    cp_async_wait<kStages - 2>();
    __syncwarp();      // the rows have landed for all lanes, and all are through with the place that the next ones take
    ahead(j + kStages - 1);
    const uint32_t from = ring + j % kStages * kStage;
    const int t0 = first + j * S;
    F a[S], u[S];
    if constexpr (kBack) {
      auto gate = [&](int t) { return scales.apply(rg.get(from, t, t0 + t), scales.get(from + R::kStage + U::kStage, t).y); };
      if (kUsual || z.has_a) {
#pragma unroll
        for (int t = 0; t < S; ++t) {
          Factors<false> f;
          F rest;
          decay_of(z, gate(t), f, rest);
          a[t] = f.a;
        }
      } else {
#pragma unroll
        for (int t = 0; t < S; ++t) {
          F o;
          sigmoid<false>(gate(t), z.gate_bias, 0.f, a[t], o);
        }
      }
#pragma unroll
      for (int t = 0; t < S; ++t) u[t] = ru.get(from + R::kStage, t, t0 + t);
    } else {
      Factors<false> f[S];
      factors<kUsual>(z, [&](int t) { return rg.get(from, t, t0 + t); }, [&](int t) { return ri.get(from + 2 * R::kStage, t, t0 + t); }, f);
#pragma unroll
      for (int t = 0; t < S; ++t) {
        a[t] = f[t].a;
        u[t] = mul2(f[t].w, rx.get(from + R::kStage, t, t0 + t));
      }
    }
    if (t0 + S > at.len) {
#pragma unroll
      for (int t = 0; t < S; ++t)
        if (t0 + t >= at.len) a[t] = both(1.f), u[t] = both(0.f);
    }
#pragma unroll
    for (int t = 0; t < S; ++t) {
      whole = mul2(whole, a[t]);
      if constexpr (kBack) whole = some(whole);
      own = kBack ? fma2(whole, u[t], own) : fma2(a[t], own, u[t]);
    }
    whole = some(whole);
  }
  steps[at.warp][at.lane] = four(whole, own);
  __syncthreads();
  if (at.warp) return;
#pragma unroll
  for (int w = 1; w < W; ++w) {
    const float4 v = steps[w][at.lane];
    own = kBack ? fma2(whole, second2(v), own) : fma2(first2(v), own, second2(v));
    whole = some(mul2(whole, first2(v)));
  }
  float* e = q.ends + (static_cast<long>(at.b) * q.chunks + at.chunk) * 2 * p.D;
  store2<float, kMode>(e, at.d, p.D, whole);
  store2<float, kMode>(e + p.D, at.d, p.D, own);
}

template <class T, int kMode, bool kUsual, int W>
__global__ void __launch_bounds__(32 * W, 16 / W) gated_forward_kernel(const ttt_b200_gated_args p, const Plan q) {
  wait_for_predecessor();
  using R = Rows<T, kMode>;
  __shared__ Steps<W> join;
  extern __shared__ __align__(16) unsigned char rings[];
  const At<W> at(p, q, q.chunks);
  constexpr int kTile = At<W>::kTile;
  const int d0 = at.tile * kCols;
  const Weights z = weights_of<kMode>(p, at.d);
  const R rx(p.x, p.x_stride, at.b, d0, p.D), rg(p.gate, p.gate_stride, at.b, d0, p.D), ri(p.input_gate, p.input_stride, at.b, d0, p.D);
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(rings)) + at.warp * (kStages * 3 * R::kStage);
  const int first = at.first * kTile + at.warp * S, rounds = at.last - at.first;
  auto ahead = [&](int j) {
    if (j < rounds) {
      const uint32_t to = ring + j % kStages * (3 * R::kStage);
      rx.copy(to, first + j * kTile, at.len);
      rg.copy(to + R::kStage, first + j * kTile, at.len);
      if (kUsual || z.gated) ri.copy(to + 2 * R::kStage, first + j * kTile, at.len);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int j = 0; j < kStages - 1; ++j) ahead(j);
  F carry = load2<kMode>(p.state ? p.state + static_cast<long>(at.b) * p.D : nullptr, at.d, p.D, 0.f);
  carry = join_chunks<kMode, false>(p, q, at, carry);
  T* y = static_cast<T*>(p.y) + static_cast<long>(at.b) * p.T * p.D;
  for (int j = 0; j < rounds; ++j) {
    const int t0 = first + j * kTile, half = j & 1;
    cp_async_wait<kStages - 2>();
    __syncwarp();      // the rows have landed for all lanes, and all are through with the place that the next ones take
    ahead(j + kStages - 1);
    const uint32_t from = ring + j % kStages * (3 * R::kStage);
    F a[S], u[S], whole = both(1.f), own = both(0.f);
    Factors<false> f[S];
    factors<kUsual>(z, [&](int t) { return rg.get(from + R::kStage, t, t0 + t); }, [&](int t) { return ri.get(from + 2 * R::kStage, t, t0 + t); }, f);
#pragma unroll
    for (int t = 0; t < S; ++t) {
      a[t] = f[t].a;
      u[t] = mul2(f[t].w, rx.get(from, t, t0 + t));
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
    join.warp[half][at.warp][at.lane] = four(some(whole), own);
    __syncthreads();
    F h = j == 0 ? carry : join.end[half ^ 1][at.lane];
#pragma unroll
    for (int w = 0; w < W - 1; ++w) {
      if (w >= at.warp) break;
      const float4 v = join.warp[half][w][at.lane];
      h = fma2(first2(v), h, second2(v));
    }
    if (at.warp % (kEvery / S) == 0 && p.checkpoints && t0 < at.len)
      store2<float, kMode>(p.checkpoints + (static_cast<long>(at.b) * q.nck + t0 / kEvery) * p.D, at.d, p.D, h);
    T* to = y + static_cast<long>(t0) * p.D;
    if (t0 + S <= at.len) {
#pragma unroll
      for (int t = 0; t < S; ++t) {
        h = fma2(a[t], h, u[t]);
        store2<T, kMode>(to, at.d, p.D, h);
        to += p.D;
      }
    } else {
#pragma unroll
      for (int t = 0; t < S; ++t) {
        h = fma2(a[t], h, u[t]);
        if (t0 + t < p.T) store2<T, kMode>(to, at.d, p.D, t0 + t < at.len ? h : both(0.f));
        to += p.D;
      }
    }
    if (at.warp == W - 1) carry = join.end[half][at.lane] = h;
  }
  if (p.final_state && at.chunk == q.chunks - 1 && at.warp == W - 1) store2<float, kMode>(p.final_state + static_cast<long>(at.b) * p.D, at.d, p.D, carry);
  for (int j = at.last; j < at.end(q, p.T); ++j)
    for (int t = j * kTile + at.warp * S; t < min(j * kTile + at.warp * S + S, p.T); ++t) store2<T, kMode>(y + static_cast<long>(t) * p.D, at.d, p.D, both(0.f));
}

// kStages: tiles of rows in shared memory.  The next one's are on their way while a CTA works on one; of four fp32 tensors two CTAs to an SM have room for one
// tile (3 x 1001 x 1003 backward 50 -> 45 us), and a CTA that has the SM for itself for two (4 x 2048 x 2048 108 -> 99).
// T: the gradients' type; I: that of x and the gates, or 8-bit values
template <class T, class I, int kMode, bool kUsual, int W, int kStages>
__global__ void __launch_bounds__(32 * W, 16 / W) gated_backward_kernel(const ttt_b200_gated_args p, const Plan q) {
  wait_for_predecessor();
  using R = Rows<I, kMode>;
  using U = Rows<T, kMode>;
  constexpr uint32_t kStage = 3 * R::kStage + U::kStage + Scales<I>::kStage, kKept = S * 256;
  __shared__ Steps<W> join;
  __shared__ F back[2][W][32];
  extern __shared__ __align__(16) unsigned char rings[];
  const At<W> at(p, q, q.chunks);
  constexpr int kTile = At<W>::kTile;
  const int d0 = at.tile * kCols;
  const Weights z = weights_of<kMode>(p, at.d);
  const bool gated = kUsual || z.gated;
  const R rx(p.x, p.x_stride, at.b, d0, p.D), rg(p.gate, p.gate_stride, at.b, d0, p.D), ri(p.input_gate, p.input_stride, at.b, d0, p.D);
  const U ru(p.grad_y, p.gy_stride, at.b, d0, p.D);
  const Scales<I> scales(p, at.b, d0);
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(rings)) + at.warp * (kStages * kStage + kKept);
  const int first = at.first * kTile + at.warp * S, rounds = at.last - at.first;
  auto ahead = [&](int j) {
    if (j >= 0) {
      const uint32_t to = ring + j % kStages * kStage;
      rx.copy(to, first + j * kTile, at.len);
      rg.copy(to + R::kStage, first + j * kTile, at.len);
      if (gated) ri.copy(to + 2 * R::kStage, first + j * kTile, at.len);
      ru.copy(to + 3 * R::kStage, first + j * kTile, at.len);
      scales.copy(to + 3 * R::kStage + U::kStage, first + j * kTile, at.len);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int j = 0; j < kStages - 1; ++j) ahead(rounds - 1 - j);
  const long batch = static_cast<long>(at.b) * p.T * p.D;
  T *gx = static_cast<T*>(p.grad_x) + batch, *gg = static_cast<T*>(p.grad_gate) + batch, *gi = static_cast<T*>(p.grad_input) + batch;
  auto put = [&](long o, F x, F g, F i) {
    store2<T, kMode>(gx + o, at.d, p.D, x);
    store2<T, kMode>(gg + o, at.d, p.D, g);
    if (gated) store2<T, kMode>(gi + o, at.d, p.D, i);
  };
  // u = b i x of each token, for the second pass over a tile, in a place of the thread's own (worked out again from the rows: 8 x 4096 x 2048 288 us for 275)
  const uint32_t mine = ring + kStages * kStage + at.lane * 8;
  auto keep = [&](int t, F u) { asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(mine + t * 256), "f"(u.x), "f"(u.y) : "memory"); };
  F carry = load2<kMode>(p.grad_final_state ? p.grad_final_state + static_cast<long>(at.b) * p.D : nullptr, at.d, p.D, 0.f);
  carry = join_chunks<kMode, true>(p, q, at, carry);
  F sum_a = both(0.f), sum_g = sum_a, sum_i = sum_a;
  for (int j = rounds - 1; j >= 0; --j) {
    const int t0 = first + j * kTile, half = j & 1;
    const int ck = t0 / kEvery;
    F h = load2<kMode>(ck * kEvery < at.len ? p.checkpoints + (static_cast<long>(at.b) * q.nck + ck) * p.D : nullptr, at.d, p.D, 0.f);
    if constexpr (kStages == 1) {
      __syncwarp();      // all lanes are through with the rows in front
      ahead(j);
      cp_async_wait<0>();
      __syncwarp();
    } else {
      cp_async_wait<kStages - 2>();
      __syncwarp();
      ahead(j - kStages + 1);
    }
    const uint32_t from = ring + j % kStages * kStage;
    // of a token: a; w = b i; what there is of d log a / G without the state, which joins it; d log a's factors in d gate and dA; d input / G
    F a[S], w[S], slope[S], k[S], s[S], in[S], whole = both(1.f), own = both(0.f), left = both(0.f);
    Factors<true> f[S];
    const uint32_t sc = from + 3 * R::kStage + U::kStage;
    factors<kUsual>(z, [&](int t) { return scales.apply(rg.get(from + R::kStage, t, t0 + t), scales.get(sc, t).y); },
                    [&](int t) { return scales.apply(ri.get(from + 2 * R::kStage, t, t0 + t), scales.get(sc, t).z); }, f);
#pragma unroll
    for (int t = 0; t < S; ++t) {
      const F x = scales.bounded(rx.get(from, t, t0 + t), scales.get(sc, t).x), u = mul2(f[t].w, x);
      keep(t, u);
      a[t] = f[t].a, w[t] = f[t].w, k[t] = f[t].k, s[t] = f[t].s;
      slope[t] = mul2(f[t].slope, x);
      in[t] = mul2(f[t].rest, u);
      own = fma2(a[t], own, u);
      whole = mul2(whole, a[t]);
    }
    if (t0 + S > at.len) {      // once more, with the tokens that there are
      own = both(0.f), whole = both(1.f);
#pragma unroll
      for (int t = 0; t < S; ++t) {
        if (t0 + t >= at.len) a[t] = both(1.f), keep(t, both(0.f));
        own = fma2(a[t], own, pair_of<float>(mine + t * 256));
        whole = mul2(whole, a[t]);
      }
    }
#pragma unroll
    for (int t = S - 1; t >= 0; --t) left = mul2(a[t], add2(ru.get(from + 3 * R::kStage, t, t0 + t), left));
    join.warp[half][at.warp][at.lane] = four(some(whole), own);
    back[half][at.warp][at.lane] = left;
    __syncthreads();
    F c = j == rounds - 1 ? carry : join.end[half ^ 1][at.lane];
#pragma unroll
    for (int v = 0; v < kEvery / S - 1; ++v) {
      if (v >= at.warp % (kEvery / S)) break;
      const float4 f = join.warp[half][at.warp / (kEvery / S) * (kEvery / S) + v][at.lane];
      h = fma2(first2(f), h, second2(f));
    }
    // to h_{t-1}, and with it to d log a / G
#pragma unroll
    for (int t = 0; t < S; ++t) {
      const F kept = mul2(a[t], h);
      slope[t] = add2(kept, slope[t]);
      h = add2(pair_of<float>(mine + t * 256), kept);
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
    if (at.warp == 0) carry = join.end[half][at.lane] = c;
  }
  if (p.grad_state && at.chunk == 0 && at.warp == 0) store2<float, kMode>(p.grad_state + static_cast<long>(at.b) * p.D, at.d, p.D, carry);
  for (int j = at.last; j < at.end(q, p.T); ++j)
    for (int t = j * kTile + at.warp * S; t < min(j * kTile + at.warp * S + S, p.T); ++t) put(static_cast<long>(t) * p.D, both(0.f), both(0.f), both(0.f));
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
      const F A = load2<kMode>(p.A, at.d, p.D, 0.f);
      s = make_float2(A.x > 0.f ? 0.f : s.x, A.y > 0.f ? 0.f : s.y);
    }
    store2<float, kMode>(q.part + (static_cast<long>(at.b) * q.chunks + at.chunk) * 3 * p.D + static_cast<long>(at.warp) * p.D, at.d, p.D, s);
  }
}

// A row of the batch and 256 channels to a CTA.  Rows that name the same slot are taken in their order by the CTA of the first of
// them, so that no two CTAs touch a state.
template <class T, int kMode> __global__ void __launch_bounds__(128) gated_step_kernel(const ttt_b200_gated_args p, int tiles) {
  wait_for_predecessor();
  const int b0 = blockIdx.x / tiles, d = (blockIdx.x % tiles * 128 + threadIdx.x) * 2;
  T* ys = static_cast<T*>(p.y);
  int slot = b0, more = 0;
  if (p.slots) {
    slot = p.slots[b0];
    if (slot < 0 || slot >= p.rows) {
      store2<T, kMode>(ys + static_cast<long>(b0) * p.D, d, p.D, both(0.f));
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
    if constexpr (kMode != kSingles) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(r));
      else if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(r));
      else return *reinterpret_cast<const F*>(r);
    } else {
      return make_float2(to_f32(r[0]), d + 1 < p.D ? to_f32(r[1]) : 0.f);
    }
  };
  const Weights z = weights_of<kMode>(p, d);
  float* st = p.state_io + static_cast<long>(slot) * p.D;
  F h = load2<kMode>(st, d, p.D, 0.f);
  for (int b = b0; b < p.B; ++b) {
    if (b != b0 && p.slots[b] != slot) continue;
    Factors<false> f[1];
    const F x = two(p.x, p.x_stride[0], b);
    factors<false>(z, [&](int) { return two(p.gate, p.gate_stride[0], b); }, [&](int) { return two(p.input_gate, p.input_stride[0], b); }, f);
    h = fma2(f[0].a, h, mul2(f[0].w, x));
    store2<T, kMode>(ys + static_cast<long>(b) * p.D, d, p.D, h);
    if (!more) break;
  }
  store2<float, kMode>(st, d, p.D, h);
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

// how rows of values of `size` bytes start
int mode_of(const void* a, const int64_t* st, int size) {
  const uintptr_t all = reinterpret_cast<uintptr_t>(a) | static_cast<uintptr_t>(st[0] * size) | static_cast<uintptr_t>(st[1] * size);
  return all % 16 == 0 ? kWholeRows : all % (2 * size) == 0 ? kPairs : kSingles;
}
bool even(const void* a, int size) { return reinterpret_cast<uintptr_t>(a) % (2 * size) == 0; }
int size_of(const ttt_b200_gated_args& p) { return p.dtype == TTT_B200_FP32 ? 4 : 2; }
// what all rows that are read allow, and all that is written
int mode_of(const ttt_b200_gated_args& p, bool backward) {
  const int es = size_of(p), in = p.group ? 1 : es;
  bool ok = p.D % 2 == 0;
  for (const float* v : {p.A, p.gate_bias, p.input_bias, p.state, static_cast<const float*>(p.final_state), static_cast<const float*>(p.checkpoints), p.grad_final_state,
                         static_cast<const float*>(p.grad_state)})
    ok = ok && even(v, 4);
  ok = ok && (backward ? even(p.grad_x, es) && even(p.grad_gate, es) && even(p.grad_input, es) : even(p.y, es));
  if (!ok) return kSingles;
  int mode = std::min(mode_of(p.x, p.x_stride, in), mode_of(p.gate, p.gate_stride, in));
  if (p.input_gate) mode = std::min(mode, mode_of(p.input_gate, p.input_stride, in));
  return backward ? std::min(mode, mode_of(p.grad_y, p.gy_stride, es)) : mode;
}

// How many chunks a sequence is cut into, of how many tiles, and whether a CTA has 8 warps (two CTAs to an SM) or 16: by what a round of tiles takes, in
// tenths of a microsecond, measured with 2048 channels and more or fewer sequences.  A CTA of 8 warps that has an SM for itself 15 (it waits for itself), two
// of them or one of 16 warps 24; a turn of CTAs over the SMs starts in 20; the chunks' steps take 0.6 of that.
// 16384 tokens of 1024 channels, forward / backward us: one chunk 348 / 673, 8 chunks 89 / 126, 18 (by the rule) 73 / 97, 24 83 / 116;
// 2 x 2048 of 2048: one of 8 warps 51 / 95, of 16 45 / 79, 4 chunks (by the rule) 42 / 56, 8 44 / 60.
// All of these are bf16 with every part, whole rows; fp32, odd rows and forms with fewer parts go by the same costs, which were not measured for them.
void plan(Plan& q, const ttt_b200_gated_args& p, bool backward) {
  q.tiles = (p.D - 1) / kCols + 1;
  q.nck = (p.T - 1) / kEvery + 1;
  const long columns = static_cast<long>(q.tiles) * p.B, sms = sm_count();
  auto rounds_of = [&](long ctas, long rounds) { return ctas <= sms ? 35 + 15 * rounds : 15 + (24 * rounds + 20) * ((ctas + 2 * sms - 1) / (2 * sms)); };
  long best = rounds_of(columns, q.nck);
  q.warps = 8;
  q.chunk = q.nck;
  // (16 warps' rows of four fp32 tensors: the shared memory has room for one tile, and then 8 warps with two are faster)
  if (columns <= sms && p.T > 8 * S && !(backward && p.dtype == TTT_B200_FP32 && !p.group)) {
    const int rounds = (p.T - 1) / (16 * S) + 1;
    const long cost = 35 + 24L * rounds;
    if (cost < best) best = cost, q.warps = 16, q.chunk = rounds;
  }
  for (int n = 2; n <= std::min(kMostChunks, q.nck); ++n) {
    const int chunk = (q.nck + n - 1) / n, chunks = (q.nck + chunk - 1) / chunk;
    const long cost = rounds_of(columns * chunks, chunk) + rounds_of(columns * (chunks - 1), chunk) * 6 / 10 + 20;
    if (cost < best) best = cost, q.warps = 8, q.chunk = chunk;
  }
  const int tiles = (p.T - 1) / (q.warps * S) + 1;
  q.chunks = (tiles + q.chunk - 1) / q.chunk;
}
// scratch: the chunks' steps, and behind them the sums' parts
uint64_t ends_bytes(const Plan& q, const ttt_b200_gated_args& p) { return q.chunks > 1 ? (static_cast<uint64_t>(p.B) * q.chunks * 2 * p.D * sizeof(float) + 15) / 16 * 16 : 0; }

template <auto kKernel> int launch(long grid, const Plan& q, const ttt_b200_gated_args& p, int threads, uint32_t bytes, cudaStream_t s, const char* what) {
  if (grid > 0x7fffffffL) return fail("gated scan: too many CTAs");
  if (bytes > 16 * 1024)      // (with the static part 48 KB is the most without asking)
    if (int rc = allow_shared<kKernel>()) return rc;
  ttt_launch_overlapped(kKernel, static_cast<int>(grid), threads, bytes, s, p, q);
  return launched(what);
}

bool usual(const ttt_b200_gated_args& p) { return p.A && p.input_gate && p.mix == TTT_B200_MIX_SQRT; }

template <class T, int kMode, bool kUsual> int forward_as(const ttt_b200_gated_args& p, const Plan& q, cudaStream_t s) {
  constexpr uint32_t bytes = kStages * 3 * Rows<T, kMode>::kStage;      // of a warp
  const long columns = static_cast<long>(p.B) * q.tiles;
  if (q.warps == 16) return launch<gated_forward_kernel<T, kMode, kUsual, 16>>(columns, q, p, 512, 16 * bytes, s, "gated scan");
  if (q.chunks > 1)
    if (int rc = launch<gated_ends_kernel<T, T, kMode, kUsual, false, 8>>(columns * (q.chunks - 1), q, p, 256, 8 * bytes, s, "gated scan")) return rc;
  return launch<gated_forward_kernel<T, kMode, kUsual, 8>>(columns * q.chunks, q, p, 256, 8 * bytes, s, "gated scan");
}
template <class T> int forward(const ttt_b200_gated_args& p, cudaStream_t s) {
  Plan q = {};
  plan(q, p, false);
  q.ends = static_cast<float*>(p.scratch);
  switch (mode_of(p, false)) {
    case kWholeRows: return usual(p) ? forward_as<T, kWholeRows, true>(p, q, s) : forward_as<T, kWholeRows, false>(p, q, s);
    case kPairs: return usual(p) ? forward_as<T, kPairs, true>(p, q, s) : forward_as<T, kPairs, false>(p, q, s);
    default: return usual(p) ? forward_as<T, kSingles, true>(p, q, s) : forward_as<T, kSingles, false>(p, q, s);
  }
}
template <class T, class I, int kMode, bool kUsual> int backward_as(const ttt_b200_gated_args& p, const Plan& q, cudaStream_t s) {
  // of a warp
  constexpr uint32_t in = Rows<I, kMode>::kStage, up = Rows<T, kMode>::kStage + Scales<I>::kStage, kept = S * 256;
  constexpr uint32_t one = 3 * in + up + kept, two = 2 * (3 * in + up) + kept;
  constexpr bool kLarge = sizeof(T) == 4 && sizeof(I) == 4;
  const char* what = "gated scan backward";
  const long columns = static_cast<long>(p.B) * q.tiles, ctas = columns * q.chunks;
  if constexpr (!kLarge)
    if (q.warps == 16) return launch<gated_backward_kernel<T, I, kMode, kUsual, 16, 2>>(columns, q, p, 512, 16 * two, s, what);
  if (q.chunks > 1)
    if (int rc = launch<gated_ends_kernel<T, I, kMode, kUsual, true, 8>>(columns * (q.chunks - 1), q, p, 256, 8 * kStages * (in + up), s, what)) return rc;
  if constexpr (kLarge)
    if (ctas > sm_count()) return launch<gated_backward_kernel<T, I, kMode, kUsual, 8, 1>>(ctas, q, p, 256, 8 * one, s, what);
  return launch<gated_backward_kernel<T, I, kMode, kUsual, 8, 2>>(ctas, q, p, 256, 8 * two, s, what);
}
template <class T, class I> int backward_of(const ttt_b200_gated_args& p, const Plan& q, cudaStream_t s) {
  switch (mode_of(p, true)) {
    case kWholeRows: return usual(p) ? backward_as<T, I, kWholeRows, true>(p, q, s) : backward_as<T, I, kWholeRows, false>(p, q, s);
    case kPairs: return usual(p) ? backward_as<T, I, kPairs, true>(p, q, s) : backward_as<T, I, kPairs, false>(p, q, s);
    default: return usual(p) ? backward_as<T, I, kSingles, true>(p, q, s) : backward_as<T, I, kSingles, false>(p, q, s);
  }
}
template <class T> int backward(const ttt_b200_gated_args& p, cudaStream_t s) {
  Plan q = {};
  plan(q, p, true);
  q.ends = static_cast<float*>(p.scratch);
  q.part = reinterpret_cast<float*>(static_cast<char*>(p.scratch) + ends_bytes(q, p));
  if (int rc = p.group ? backward_of<T, E4>(p, q, s) : backward_of<T, T>(p, q, s)) return rc;
  const long D = p.D;
  const int parts = p.B * q.chunks;
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
  ttt_launch_overlapped(ok ? gated_step_kernel<T, kPairs> : gated_step_kernel<T, kSingles>, static_cast<int>(grid), 128, 0, s, p, tiles);
  return launched("gated scan step");
}

}  // namespace

extern "C" uint64_t ttt_b200_gated_scan_scratch_bytes(const ttt_b200_gated_args* p, int backward) {
  if (check(p) || p->B == 0 || p->T == 0) return 0;
  Plan q = {};
  plan(q, *p, backward);
  return ends_bytes(q, *p) + (backward ? static_cast<uint64_t>(p->B) * q.chunks * 3 * p->D * sizeof(float) : 0);
}

static int check_scratch(const ttt_b200_gated_args* p, int backward) {
  const uint64_t need = ttt_b200_gated_scan_scratch_bytes(p, backward);
  if (need && (!p->scratch || p->scratch_bytes < need || !aligned16(p->scratch))) return fail("gated scan: scratch is missing, too small or not 16-byte aligned");
  return TTT_B200_OK;
}

extern "C" int ttt_b200_gated_scan(const ttt_b200_gated_args* p, void* stream) {
  if (int rc = check(p)) return rc;
  if (!p->x || !p->gate || !p->y) return fail("gated scan: null tensor pointer");
  if (p->B == 0 || p->T == 0) return fail("gated scan: no tokens");
  if (p->group) return fail("gated scan: 8-bit inputs are for the backward pass");
  if (p->input_bias && !p->input_gate) return fail("gated scan: input_bias without input_gate");
  if (int rc = check_scratch(p, 0)) return rc;
  TTT_WITH_TYPE(p->dtype, return forward<Elem>(*p, static_cast<cudaStream_t>(stream)))
  return TTT_B200_OK;
}

extern "C" int ttt_b200_gated_scan_backward(const ttt_b200_gated_args* p, void* stream) {
  if (int rc = check(p)) return rc;
  if (!p->x || !p->gate || !p->checkpoints || !p->grad_y || !p->grad_x || !p->grad_gate || (p->input_gate && !p->grad_input))
    return fail("gated scan backward: null tensor pointer");
  if (p->group && (!p->x_scales || !p->gate_scales || (p->input_gate && !p->input_scales))) return fail("gated scan backward: 8-bit inputs without scales");
  if (p->B == 0 || p->T == 0) return fail("gated scan backward: no tokens");
  if ((p->input_bias && !p->input_gate) || (p->grad_A && !p->A)) return fail("gated scan backward: a gradient or bias of what is not there");
  if (int rc = check_scratch(p, 1)) return rc;
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
