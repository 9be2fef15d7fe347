// Activations in 8 bits and back, and the residual's addition with the next norm whose output leaves in 8 bits (format: ttt_eight_bits.cuh).
//
//   pack      scale = least power of two with max |v| <= 448 scale over a group;  q = e4m3(v / scale)
//   unpack    v = q scale, at most the largest value that there is
//   norm      z = residual + o;  n = Norm(z) weight + bias, and that as above, a scale to a group or to a token
//
// All bound by memory: 2 + 1 bytes a value (16 bits), the norm 2 + 2 + 2 + 1 or with an fp32 residual stream 2 + 4 + 4 + 1.  A thread has eight
// neighbouring values, one 16-byte access; the lanes of a group, four, eight or sixteen, exchange their largest magnitudes.
//
// Measured, bf16, calls back to back: 3 x 32768 x 2048 packed in 104 us and unpacked in 94 (5.9 and 6.5 TB/s); the norm of 16384 x 2048 with an fp32
// residual, a scale to 128, 57 us (6.4 TB/s), with a bf16 residual 44 (5.4 TB/s), with that, layer norm and a scale to a token 53 (4.4 TB/s; 75 % of the issue slots).
#include <algorithm>
#include <cmath>

#include "ttt_eight_bits.cuh"

namespace {

using namespace ttt;

constexpr int kMost = TTT_B200_PACK8_TENSORS;
// Of an SM (16384 x 2048, fp32 residual: 63 us; 1536, with registers spilled everywhere, 82).  At 1024 those of up to 512 columns spill where rows start on any boundary (4 to
// 56 bytes), with an fp32 residual on every boundary (8 to 32): four and two tokens to a CTA take their registers.
constexpr int kNormThreads = 1024;

// ---- pack and unpack ----------------------------------------------------------------------------------------------------------------
struct Many {
  ttt_b200_pack8_args a;
  uint32_t lanes;      // of a row: vectors of eight, whole groups
  uint32_t magic, shift;      // n / lanes for n < 2^31: the high word of n magic, shifted (Granlund and Montgomery 1994)
  int64_t vectors;     // lanes * rows
  bool flat;           // rows of whole groups: values and scales follow one another, whatever the row
  bool rows;           // and so do src's: no row is needed
};

// The row of vector i, and which of its lanes it is.
__device__ __forceinline__ int64_t row_of(const Many& q, int64_t i, int& lane) {
  const int64_t row = q.lanes == 1 ? i : q.vectors >> 31 ? i / q.lanes : __umulhi(static_cast<uint32_t>(i), q.magic) >> q.shift;
  lane = static_cast<int>(i - row * q.lanes);
  return row;
}

// A thread has several times eight values, a block of threads apart, all requested before the first are worked on: 2048 threads to an SM with 16 bytes each on
// their way are less than the memory's latency takes.  3 x 32768 x 2048 bf16, packed / unpacked us with one, two and four: 135 / 135, 125 / 116, 119 / 104; 16384 x
// 2047, whose values come one by one, 45 / 51, 44 / 54, 43 / 61; fp32 16384 x 2048 35 / 41, 33 / 41, 35 / 43.  Since rows of whole groups need no division to be
// found (`flat`), the first is 111 / 102.
template <class T, bool kWhole> constexpr int kEach = kWhole && sizeof(T) == 2 ? 4 : 2;

// Columns of a lane's eight values in a row.  Rows on 16-byte boundaries: neighbours, one access.  Others: of the 256 columns of a warp every 32nd, so that each
// of eight accesses is the warp's 32 neighbours (eight neighbours to a lane one by one: 16384 x 2047 bf16 packed in 51 us, unpacked in 97).
template <bool kWhole> __device__ __forceinline__ int column(int lane, int j) { return kWhole ? lane * 8 + j : (lane & ~31) * 8 + j * 32 + (lane & 31); }
template <bool kWhole, class T> __device__ __forceinline__ void take(const T* row, int lane, int D, Eight<T>& e) {
  if (kWhole && lane * 8 + 8 <= D) {
    e.load(row + lane * 8);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) e.v[j] = column<kWhole>(lane, j) < D ? row[column<kWhole>(lane, j)] : T();
  }
}
template <bool kWhole, class T> __device__ __forceinline__ void leave(T* row, int lane, int D, const Eight<T>& e) {
  if (kWhole && lane * 8 + 8 <= D) {
    e.store(row + lane * 8);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (column<kWhole>(lane, j) < D) row[column<kWhole>(lane, j)] = e.v[j];
  }
}

// Eight values to 8 bits, with the scales of their groups, of 8 L values each; all lanes of a warp together.  The scale of value j is that of
// group first + j / (a group's share of a lane's values).
template <bool kWhole, int L> __device__ __forceinline__ void to_eight(const float (&v)[8], int lane, int groups, bool there, float* scales, Eight<uint8_t>& b) {
  if constexpr (kWhole) {
    float most = magnitude(v);
#pragma unroll
    for (int o = L / 2; o; o /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    const uint32_t x = scale_exponent(most);
    const float inv = inverse_of(x);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = mul2(make_float2(v[2 * j], v[2 * j + 1]), both(inv));
      reinterpret_cast<uint16_t*>(b.v)[j] = static_cast<uint16_t>(two_bytes(f.x, f.y));
    }
    if (there && lane % L == 0 && lane / L < groups) scales[lane / L] = scale_of(x);
  } else {
    constexpr int kShare = L / 4;      // of a lane's values in a group of the warp's: 1, 2 or 4
#pragma unroll
    for (int g = 0; g < 8; g += kShare) {
      uint32_t most = 0;      // (magnitudes go by their bits)
#pragma unroll
      for (int j = g; j < g + kShare; ++j) most = max(most, fabsf(v[j]) < INFINITY ? __float_as_uint(fabsf(v[j])) : 0u);
      const uint32_t x = scale_exponent(__uint_as_float(__reduce_max_sync(0xffffffffu, most)));
      const float inv = inverse_of(x);
#pragma unroll
      for (int j = g; j < g + kShare; ++j) b.v[j] = static_cast<uint8_t>(two_bytes(v[j] * inv, 0.f));
      const int at = ((lane & ~31) * 8 + g * 32) / (8 * L);
      if (there && (lane & 31) == 0 && at < groups) scales[at] = scale_of(x);
    }
  }
}

// A gate that is closed, by a mask's infinity or its type's lowest value, is closed at -448 as well, and there its group's scale is 1: the others keep their
// digits down to 2^-6 (sigmoid and its like have no use for more), and an infinity comes back as no value that its neighbours make of it.  NaN stays.
template <class T> __device__ __forceinline__ void clamp(Eight<T>& e, int how) {
  const float low = how ? -448.f : -INFINITY, high = how == TTT_B200_CLAMP_BOTH ? 448.f : INFINITY;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      asm("max.NaN.f32 %0, %0, %1;" : "+f"(e.v[j]) : "f"(low));
      asm("min.NaN.f32 %0, %0, %1;" : "+f"(e.v[j]) : "f"(high));
    }
  } else {
    using P = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const P lows = {from_f32<T>(low), from_f32<T>(low)}, highs = {from_f32<T>(high), from_f32<T>(high)};
    P* p = reinterpret_cast<P*>(e.v);
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = __hmin2_nan(__hmax2_nan(p[j], lows), highs);
  }
}

// L lanes to a group.  kClamp: some tensor of the call is bounded; kernels of their own, since bounds for all cost those that need none
// (16384 x 2047 bf16 31.9 -> 35.1 us, 16384 x 2048 fp16 in groups of 32 16.0 -> 17.1; 3 x 32768 x 2048 bf16 103.8 without and 102.8 with).
template <class T, bool kWhole, int L, bool kClamp> __global__ void __launch_bounds__(256) pack8_kernel(const Many q) {
  wait_for_predecessor();
  constexpr int kN = kEach<T, kWhole>;
  const ttt_b200_pack8_args& a = q.a;
  const int k = blockIdx.y, groups = (a.D + 8 * L - 1) / (8 * L);
  const int64_t i0 = blockIdx.x * (256L * kN) + threadIdx.x;
  Eight<T> e[kN];
  int64_t row[kN];
  int lane[kN];
#pragma unroll
  for (int c = 0; c < kN; ++c) {
    const int64_t i = i0 + c * 256;
    if (kWhole && q.rows) {
      if (i < q.vectors) e[c].load(static_cast<const T*>(a.src[k]) + i * 8);
    } else {
      row[c] = row_of(q, i, lane[c]);
      take<kWhole>(static_cast<const T*>(a.src[k]) + row[c] * a.stride[k], lane[c], i < q.vectors ? a.D : 0, e[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < kN; ++c) {
    const int64_t i = i0 + c * 256;
    if constexpr (kClamp) clamp(e[c], a.clamp[k]);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_f32(e[c].v[j]);
    const bool there = i < q.vectors;
    Eight<uint8_t> b;
    if (kWhole && q.flat) {      // a row of all of them, as it were
      to_eight<kWhole, L>(v, threadIdx.x % L, 1, there, a.scales[k] + i / L, b);
      if (there) b.store(static_cast<uint8_t*>(a.values[k]) + i * 8);
    } else {
      to_eight<kWhole, L>(v, lane[c], groups, there, a.scales[k] + row[c] * groups, b);
      if (there) leave<kWhole>(static_cast<uint8_t*>(a.values[k]) + row[c] * a.D, lane[c], a.D, b);
    }
  }
}

template <class T, bool kWhole> __global__ void __launch_bounds__(256) unpack8_kernel(const Many q) {
  wait_for_predecessor();
  constexpr int kN = kEach<T, kWhole>;
  const ttt_b200_pack8_args& a = q.a;
  const int groups = a.group ? (a.D + a.group - 1) / a.group : 1, k = blockIdx.y, shift = a.group == 32 ? 5 : a.group == 64 ? 6 : a.group == 128 ? 7 : 31;
  const int64_t i0 = blockIdx.x * (256L * kN) + threadIdx.x;
  constexpr int kScales = kWhole ? 1 : 8;
  Eight<uint8_t> b[kN];
  float scale[kN][kScales] = {};
  int64_t row[kN];
  int lane[kN];
#pragma unroll
  for (int c = 0; c < kN; ++c) {
    const int64_t i = i0 + c * 256;
    if (kWhole && q.flat) {
      if (i < q.vectors) {
        b[c].load(static_cast<const uint8_t*>(a.values[k]) + i * 8);
        scale[c][0] = a.scales[k][i >> (shift - 3)];
      }
      continue;
    }
    row[c] = row_of(q, i, lane[c]);
    const int D = i < q.vectors ? a.D : 0;
    take<kWhole>(static_cast<const uint8_t*>(a.values[k]) + row[c] * a.D, lane[c], D, b[c]);
#pragma unroll
    for (int j = 0; j < kScales; ++j) {
      const int d = column<kWhole>(lane[c], j);
      scale[c][j] = d < D ? a.scales[k][row[c] * groups + (d >> shift)] : 0.f;
    }
  }
  auto give = [&](auto bound) {
#pragma unroll
    for (int c = 0; c < kN; ++c) {
      const int64_t i = i0 + c * 256;
      if (i >= q.vectors) continue;
      Eight<T> e;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = mul2(two_values(reinterpret_cast<const uint16_t*>(b[c].v)[j]), make_float2(scale[c][2 * j % kScales], scale[c][(2 * j + 1) % kScales]));
        e.v[2 * j] = from_f32<T>(bound(f.x));
        e.v[2 * j + 1] = from_f32<T>(bound(f.y));
      }
      if (kWhole && q.flat) e.store(static_cast<T*>(a.dst[k]) + i * 8);
      else leave<kWhole>(static_cast<T*>(a.dst[k]) + row[c] * a.D, lane[c], a.D, e);
    }
  };
  // a scale with which a value can be more than there is; looked for once for all of a thread's values (once for each eight 98 -> 103 us, 3 x 32768 x 2048)
  float most = 0.f;
#pragma unroll
  for (int c = 0; c < kN; ++c)
#pragma unroll
    for (int j = 0; j < kScales; ++j) most = fmaxf(most, scale[c][j]);
  if (most > kMostOf<T> / 448.f) give([](float v) { return at_most(v, kMostOf<T>); });
  else give([](float v) { return v; });
}

// ---- norm -----------------------------------------------------------------------------------------------------------------------------
// Threads of a token: the fewest, a power of two from a warp on, that hold it with eight values each, 256 columns to a warp.  A CTA walks over tokens with its
// columns' weights in registers and the next token's values on their way.
template <int kWidth> constexpr int kSide = kWidth < 128 ? 128 / kWidth : 1;
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// What the warps of a token share: (mean, squares about it) and the largest, tokens by turns: a barrier lies between two uses of the same place.
struct Shared {
  float2 part[2][32];
  float top[2][32];
};

// 1 / sqrt(v) as a sum: the fast one, and a step of Newton's with 1 - v r^2 from v r in two parts.  An error that all of a token's values have alike takes more of them
// over a border of their rounding to 4 bits than as many errors that differ.  Of 99 million values (16384 x 2048 twice, 16384 x 1920) 50 are not those of 64 bits; of
// a root and a division in 32 bits 54.
__device__ __forceinline__ float2 inverse_root(float v) {
  const float r = rsqrtf(v), p = v * r, e = fmaf(-p, r, 1.f) - fmaf(v, r, -p) * r;
  return make_float2(r, e < 1.f ? 0.5f * r * e : 0.f);      // (v = 0, infinite or NaN: r as it is)
}

// Mean and 1 / deviation (in two parts) of a token with one barrier: each warp's mean and its squares about it, joined as
// sum over warps of (squares + columns (mean of the warp - mean)^2).
// `inv`: 1 / D in two parts, since rounded to one all tokens would have its error (a division in its place: 16384 x 2048 bf16 43 -> 45 us).
template <int kWidth, bool kWhole> __device__ __forceinline__ float3 statistics(const float (&z)[8], const ttt_b200_norm8_args& p, float2 inv, int lane, Shared& sh, int turn) {
  auto columns = [&](int warp) { return static_cast<float>(min(max(p.D - warp * 256, 0), 256)); };
  float mean = 0.f, sq = 0.f;
  if (p.layer) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s += z[j];      // (zeros behind the last column)
    mean = warp_sum(s) / fmaxf(columns(lane / 32), 1.f);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float v = column<kWhole>(lane, j) < p.D ? z[j] - mean : 0.f;
    sq = fmaf(v, v, sq);
  }
  sq = warp_sum(sq);
  if constexpr (kWidth > 32) {
    constexpr int warps = kWidth / 32;
    const int warp = threadIdx.x / 32, home = warp & -warps, i = threadIdx.x % warps;
    if (threadIdx.x % 32 == 0) sh.part[turn][warp] = make_float2(mean, sq);
    __syncthreads();
    const float2 v = sh.part[turn][home + i];      // a lane for each warp
    sq = v.y;
    if (p.layer) {
      const float n = columns(i);
      mean = n * v.x;
#pragma unroll
      for (int o = warps / 2; o; o /= 2) mean += __shfl_xor_sync(0xffffffffu, mean, o);
      mean = fmaf(mean, inv.x, mean * inv.y);
      sq = fmaf(n * (v.x - mean), v.x - mean, sq);
    }
#pragma unroll
    for (int o = warps / 2; o; o /= 2) sq += __shfl_xor_sync(0xffffffffu, sq, o);
  }
  const float2 dev = inverse_root(fmaf(sq, inv.x, fmaf(sq, inv.y, p.eps)));
  return make_float3(mean, dev.x, dev.y);
}

// L lanes to a group; 0: the token has one scale
template <class T, class R, int kWidth, bool kWhole, int L>
__global__ void __launch_bounds__(kWidth* kSide<kWidth>, kNormThreads / (kWidth * kSide<kWidth>)) norm8_kernel(const ttt_b200_norm8_args p, const float2 inv) {
  wait_for_predecessor();
  constexpr int side = kSide<kWidth>;
  __shared__ Shared sh;
  const int lane = threadIdx.x % kWidth, sub = threadIdx.x / kWidth, groups = L ? (p.D + 8 * L - 1) / (8 * L) : 1;
  Eight<float> w;
#pragma unroll
  for (int j = 0; j < 8; ++j) w.v[j] = column<kWhole>(lane, j) < p.D ? p.weight[column<kWhole>(lane, j)] : 0.f;
  const int64_t step = static_cast<int64_t>(gridDim.x) * side;
  Eight<T> o;
  Eight<R> r;
  auto ask = [&](int64_t m) {
    if (m >= p.M) return;
    take<kWhole>(static_cast<const T*>(p.o) + m * p.o_stride, lane, p.D, o);
    if (p.residual) take<kWhole>(static_cast<const R*>(p.residual) + m * p.residual_stride, lane, p.D, r);
  };
  int64_t m = static_cast<int64_t>(blockIdx.x) * side + sub;
  ask(m);
  int turn = 0;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * side; base < p.M; base += step, m += step, turn ^= 1) {
    const bool live = m < p.M;
    float z[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) z[j] = !live ? 0.f : p.residual ? to_f32(r.v[j]) + to_f32(o.v[j]) : to_f32(o.v[j]);
    if (live && p.residual) {
#pragma unroll
      for (int j = 0; j < 8; ++j) r.v[j] = from_f32<R>(z[j]);
      leave<kWhole>(static_cast<R*>(p.x) + m * p.D, lane, p.D, r);
    }
    ask(m + step);
    const float3 s = statistics<kWidth, kWhole>(z, p, inv, lane, sh, turn);
#pragma unroll
    for (int j = 0; j < 8; ++j) {      // (0 behind the last column, as weight and bias)
      const float c = z[j] - s.x;
      z[j] = fmaf(c, s.y, c * s.z) * w.v[j];      // the large product exact: rounded once
    }
    if (p.bias) {
#pragma unroll
      for (int j = 0; j < 8; ++j) z[j] += column<kWhole>(lane, j) < p.D ? p.bias[column<kWhole>(lane, j)] : 0.f;
    }
    if (kWhole ? lane * 8 >= p.D : lane / 32 * 256 >= p.D) {
#pragma unroll
      for (int j = 0; j < 8; ++j) z[j] = 0.f;      // (0 times what a token of infinities has for a deviation)
    }
    Eight<uint8_t> q;
    if constexpr (L > 0) {
      to_eight<kWhole, L>(z, lane, groups, live, p.scales + m * groups, q);
    } else {
      float most = magnitude(z);
#pragma unroll
      for (int e = 16; e; e /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, e));
      if constexpr (kWidth > 32) {
        constexpr int warps = kWidth / 32;
        const int warp = threadIdx.x / 32;
        if (threadIdx.x % 32 == 0) sh.top[turn][warp] = most;
        __syncthreads();
        most = sh.top[turn][(warp & -warps) + threadIdx.x % warps];
#pragma unroll
        for (int e = warps / 2; e; e /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, e));
      }
      const uint32_t x = scale_exponent(most);
      const float inv = inverse_of(x);
#pragma unroll
      for (int j = 0; j < 4; ++j) reinterpret_cast<uint16_t*>(q.v)[j] = static_cast<uint16_t>(two_bytes(z[2 * j] * inv, z[2 * j + 1] * inv));
      if (live && lane == 0) p.scales[m] = scale_of(x);
    }
    if (!live) continue;
    leave<kWhole>(static_cast<uint8_t*>(p.values) + m * p.D, lane, p.D, q);
    if (p.stats && lane == 0) reinterpret_cast<float4*>(p.stats)[m] = make_float4(0.f, 1.f, s.x, s.y + s.z);
  }
}

// ---- host --------------------------------------------------------------------------------------------------------------------------------
bool known(int group) { return group == 32 || group == 64 || group == 128; }
template <class E> bool rows(const void* p, int64_t stride) { return reinterpret_cast<uintptr_t>(p) % std::min<size_t>(16, 8 * sizeof(E)) == 0 && stride % 8 == 0; }

int check(const ttt_b200_pack8_args* p, bool back) {
  if (!p) return fail("pack8: NULL argument struct");
  if (p->M < 0 || p->D < 1 || p->D > 1 << 30 || p->count < 1 || p->count > kMost) return fail("pack8: M >= 0, 1 <= D <= 2^30 and one to four tensors");
  if (p->dtype < TTT_B200_BF16 || p->dtype > TTT_B200_FP32) return fail("pack8: unknown element type");
  if (!known(p->group) && !(back && p->group == 0)) return fail("pack8: groups of 32, 64 or 128 values");
  for (int k = 0; k < p->count; ++k) {
    if (!p->values[k] || !p->scales[k] || !(back ? p->dst[k] : p->src[k])) return fail("pack8: null tensor pointer");
    if (!back && (p->clamp[k] < 0 || p->clamp[k] > TTT_B200_CLAMP_BOTH)) return fail("pack8: unknown clamp");
  }
  if (p->M == 0) return fail("pack8: no rows");
  return TTT_B200_OK;
}
template <class T, bool kWhole, bool kClamp> auto pack_kernel(int group) {
  return group == 32 ? pack8_kernel<T, kWhole, 4, kClamp> : group == 64 ? pack8_kernel<T, kWhole, 8, kClamp> : pack8_kernel<T, kWhole, 16, kClamp>;
}
template <class T> int run(Many& q, bool back, cudaStream_t s) {
  const ttt_b200_pack8_args& a = q.a;
  bool whole = true;
  for (int k = 0; k < a.count; ++k)
    whole = whole && rows<uint8_t>(a.values[k], a.D) && (back ? rows<T>(a.dst[k], a.D) : rows<T>(a.src[k], a.stride[k]));
  const int64_t unit = whole ? (back ? 1 : a.group / 8) : 32;      // lanes that a row has a multiple of: a group's, or a warp
  const int64_t lanes = (a.D + 8 * unit - 1) / (8 * unit) * unit;
  q.lanes = static_cast<uint32_t>(lanes);
  if (a.M > (255L << 31) / lanes) return fail("pack8: too many values");
  q.vectors = a.M * lanes;
  q.flat = whole && (back ? a.group && a.D % a.group == 0 : a.D == 8 * lanes);
  q.rows = q.flat && !back;
  for (int k = 0; k < a.count; ++k) q.rows = q.rows && (a.stride[k] == a.D || a.M == 1);
  int bits = 0;      // 2^bits >= lanes
  while (int64_t{1} << bits < lanes) ++bits;
  q.shift = bits ? bits - 1 : 0;
  q.magic = static_cast<uint32_t>(((uint64_t{1} << (31 + bits)) + lanes - 1) / lanes);
  const int each = whole ? kEach<T, true> : kEach<T, false>;
  const int64_t blocks = (q.vectors + 256 * each - 1) / (256 * each);
  if (blocks > 0x7fffffffL) return fail("pack8: too many values");
  const bool clamp = a.clamp[0] | a.clamp[1] | a.clamp[2] | a.clamp[3];
  auto kernel = back ? (whole ? unpack8_kernel<T, true> : unpack8_kernel<T, false>)
              : clamp ? (whole ? pack_kernel<T, true, true>(a.group) : pack_kernel<T, false, true>(a.group))
                      : (whole ? pack_kernel<T, true, false>(a.group) : pack_kernel<T, false, false>(a.group));
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks), a.count);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, q);
  return launched(back ? "unpack8" : "pack8");
}

template <class T, class R, int kWidth, bool kWhole> int norm_with(const ttt_b200_norm8_args& p, cudaStream_t s) {
  constexpr int side = kSide<kWidth>, threads = kWidth * side;
  const int ctas = static_cast<int>(std::min<int64_t>(static_cast<int64_t>(sm_count()) * (kNormThreads / threads), (p.M + side - 1) / side));
  const auto kernel = p.group == 0 ? norm8_kernel<T, R, kWidth, kWhole, 0> : p.group == 32 ? norm8_kernel<T, R, kWidth, kWhole, 4>
                    : p.group == 64 ? norm8_kernel<T, R, kWidth, kWhole, 8> : norm8_kernel<T, R, kWidth, kWhole, 16>;
  float inv = static_cast<float>(1.0 / p.D);
  if (inv > 1.0 / p.D) inv = std::nextafter(inv, 0.f);
  const float rest = std::max(static_cast<float>(1.0 / p.D - inv), 0x1p-149f);      // (above 0, so that infinite squares stay infinite)
  ttt_launch_overlapped(kernel, ctas, threads, 0, s, p, make_float2(inv, rest));
  return launched("norm8");
}
template <class T, class R, int kWidth> int norm_as(const ttt_b200_norm8_args& p, cudaStream_t s) {
  const bool whole = p.D % 8 == 0 && rows<T>(p.o, p.o_stride) && rows<R>(p.residual, p.residual_stride) && rows<R>(p.x, p.D) && rows<uint8_t>(p.values, p.D);
  return whole ? norm_with<T, R, kWidth, true>(p, s) : norm_with<T, R, kWidth, false>(p, s);
}
template <class T, class R> int norm(const ttt_b200_norm8_args& p, cudaStream_t s) {
  if (p.D <= 256) return norm_as<T, R, 32>(p, s);
  if (p.D <= 512) return norm_as<T, R, 64>(p, s);
  if (p.D <= 1024) return norm_as<T, R, 128>(p, s);
  if (p.D <= 2048) return norm_as<T, R, 256>(p, s);
  return p.D <= 4096 ? norm_as<T, R, 512>(p, s) : norm_as<T, R, 1024>(p, s);
}

}  // namespace

extern "C" int ttt_b200_pack8(const ttt_b200_pack8_args* p, void* stream) {
  if (int rc = check(p, false)) return rc;
  Many q = {};
  q.a = *p;
  TTT_WITH_TYPE(p->dtype, return run<Elem>(q, false, static_cast<cudaStream_t>(stream)))
  return TTT_B200_OK;
}

extern "C" int ttt_b200_unpack8(const ttt_b200_pack8_args* p, void* stream) {
  if (int rc = check(p, true)) return rc;
  Many q = {};
  q.a = *p;
  TTT_WITH_TYPE(p->dtype, return run<Elem>(q, true, static_cast<cudaStream_t>(stream)))
  return TTT_B200_OK;
}

extern "C" int ttt_b200_norm_residual_8bit(const ttt_b200_norm8_args* p, void* stream) {
  if (!p) return fail("norm8: NULL argument struct");
  if (p->M < 0 || p->D < 1 || p->D > 8192) return fail("norm8: M >= 0 and 1 <= D <= 8192");
  if (p->dtype < TTT_B200_BF16 || p->dtype > TTT_B200_FP32) return fail("norm8: unknown element type");
  if (p->group && !known(p->group)) return fail("norm8: groups of 32, 64 or 128 values, or 0 for the whole token");
  if (!(p->eps >= 0.f)) return fail("norm8: eps must be >= 0");
  if (!p->o || !p->weight || !p->values || !p->scales || (p->residual && !p->x)) return fail("norm8: null tensor pointer");
  if (p->stats && !aligned16(p->stats)) return fail("norm8: stats must be 16-byte aligned");
  if (p->M == 0) return fail("norm8: no tokens");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  TTT_WITH_TYPE(p->dtype, return p->residual_fp32 ? (norm<Elem, float>(*p, s)) : (norm<Elem, Elem>(*p, s)))
  return TTT_B200_OK;
}
