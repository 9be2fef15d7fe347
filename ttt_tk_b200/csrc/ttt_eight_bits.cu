// Activations in 8 bits and back, and the residual's addition with the next norm whose output leaves in 8 bits (format: ttt_eight_bits.cuh).
//
//   pack      scale = least power of two with max |v| <= 448 scale over a group;  q = e4m3(v / scale)
//   unpack    v = q scale
//   norm      z = residual + o;  n = Norm(z) weight + bias, and that as above, a scale to a group or to a token
//
// All bound by memory: 2 + 1 bytes a value (16 bits), the norm 2 + 2 + 2 + 1 or with an fp32 residual stream 2 + 4 + 4 + 1.  A thread has eight
// neighbouring values, one 16-byte access; the lanes of a group, four, eight or sixteen, exchange their largest magnitudes.
#include <algorithm>

#include "ttt_eight_bits.cuh"

namespace {

using namespace ttt;

constexpr int kMost = TTT_B200_PACK8_TENSORS;

// ---- pack and unpack ----------------------------------------------------------------------------------------------------------------
struct Many {
  ttt_b200_pack8_args a;
  uint32_t lanes;      // of a row: vectors of eight, whole groups
  int64_t vectors;     // lanes * rows
};

// L lanes to a group
template <class T, bool kWhole, int L> __global__ void __launch_bounds__(256) pack8_kernel(const Many q) {
  wait_for_predecessor();
  const ttt_b200_pack8_args& a = q.a;
  const int64_t i = blockIdx.x * 256L + threadIdx.x;      // (whole groups: their lanes leave together)
  if (i >= q.vectors) return;
  const int64_t row = q.vectors >> 32 ? i / q.lanes : static_cast<uint32_t>(i) / q.lanes;
  const int lane = static_cast<int>(i - row * q.lanes), n = a.D - lane * 8, k = blockIdx.y;
  Eight<T> e;
  const T* src = static_cast<const T*>(a.src[k]) + row * a.stride[k] + lane * 8;
  if (kWhole && n >= 8) e.load(src);
  else e.load(src, n);
  float v[8];
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v[j] = to_f32(e.v[j]);
    most = magnitude(most, v[j]);
  }
  const int64_t left = q.vectors - (i - threadIdx.x % 32);      // from the warp's first lane on
  const uint32_t live = left >= 32 ? 0xffffffffu : (1u << left) - 1;
#pragma unroll
  for (int o = L / 2; o; o /= 2) most = max(most, __shfl_xor_sync(live, most, o));
  const uint32_t x = scale_exponent(most);
  const float inv = inverse_of(x);
  Eight<uint8_t> b;
#pragma unroll
  for (int j = 0; j < 4; ++j) reinterpret_cast<uint16_t*>(b.v)[j] = static_cast<uint16_t>(two_bytes(v[2 * j] * inv, v[2 * j + 1] * inv));
  uint8_t* dst = static_cast<uint8_t*>(a.values[k]) + row * a.D + lane * 8;
  if (kWhole && n >= 8) b.store(dst);
  else b.store(dst, n);
  if (lane % L == 0) a.scales[k][row * (q.lanes / L) + lane / L] = scale_of(x);
}

template <class T, bool kWhole> __global__ void __launch_bounds__(256) unpack8_kernel(const Many q) {
  wait_for_predecessor();
  const ttt_b200_pack8_args& a = q.a;
  const int64_t i = blockIdx.x * 256L + threadIdx.x;
  if (i >= q.vectors) return;
  const int64_t row = q.vectors >> 32 ? i / q.lanes : static_cast<uint32_t>(i) / q.lanes;
  const int lane = static_cast<int>(i - row * q.lanes), n = a.D - lane * 8, k = blockIdx.y;
  const int groups = a.group ? (a.D + a.group - 1) / a.group : 1;
  const float scale = a.scales[k][row * groups + (a.group ? lane * 8 / a.group : 0)];
  Eight<uint8_t> b;
  const uint8_t* src = static_cast<const uint8_t*>(a.values[k]) + row * a.D + lane * 8;
  if (kWhole && n >= 8) b.load(src);
  else b.load(src, n);
  Eight<T> e;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = two_values(reinterpret_cast<const uint16_t*>(b.v)[j]);
    e.v[2 * j] = from_f32<T>(f.x * scale);
    e.v[2 * j + 1] = from_f32<T>(f.y * scale);
  }
  T* dst = static_cast<T*>(a.dst[k]) + row * a.D + lane * 8;
  if (kWhole && n >= 8) e.store(dst);
  else e.store(dst, n);
}

// ---- norm -----------------------------------------------------------------------------------------------------------------------------
// Threads of a token: the fewest, a power of two from a warp on, that hold it with eight values each.  A CTA walks over tokens with its
// columns' weights in registers and the next token's values on their way.
template <int kWidth> constexpr int kSide = kWidth < 128 ? 128 / kWidth : 1;
__device__ __forceinline__ float add_up(float a, float b) { return a + b; }

// a value joined over a token's threads, in all of them; `part`: a place for each warp, used again only behind another barrier
template <int kWidth, class V, class Op> __device__ __forceinline__ V over_token(V v, V* part, Op op) {
#pragma unroll
  for (int o = 16; o; o /= 2) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  if constexpr (kWidth > 32) {
    constexpr int warps = kWidth / 32;
    const int warp = threadIdx.x / 32, first = warp & -warps;
    if (threadIdx.x % 32 == 0) part[warp] = v;
    __syncthreads();
    v = part[first + threadIdx.x % warps];
#pragma unroll
    for (int o = warps / 2; o; o /= 2) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  }
  return v;
}

// 1 / sqrt(v), a step of Newton's behind the fast one: an error of all of a token's values alike takes more of them over a border of their rounding
// to 4 bits than as many errors that differ (16384 x 2048: 4 times the values that differ from those of 64 bits).
__device__ __forceinline__ float inverse_root(float v) {
  const float r = rsqrtf(v), e = fmaf(-v * r, r, 1.f);
  return e < 1.f ? fmaf(0.5f * r, e, r) : r;      // (v = 0, infinite or NaN: r as it is)
}

template <class T, class R, int kWidth, bool kWhole>
__global__ void __launch_bounds__(kWidth* kSide<kWidth>, 1024 / (kWidth * kSide<kWidth>)) norm8_kernel(const ttt_b200_norm8_args p) {
  wait_for_predecessor();
  constexpr int side = kSide<kWidth>;
  __shared__ float parts[2][2][32];      // mean, squares; tokens take turns
  __shared__ uint32_t tops[2][32];
  const int lane = threadIdx.x % kWidth, sub = threadIdx.x / kWidth, d = lane * 8, n = p.D - d;
  const float inv_d = 1.f / static_cast<float>(p.D);
  const int lanes = p.group / 8, groups = p.group ? (p.D + p.group - 1) / p.group : 1;
  Eight<float> w, b;
  w.load(p.weight + d, n);
  if (p.bias) b.load(p.bias + d, n);
  const int64_t step = static_cast<int64_t>(gridDim.x) * side;
  Eight<T> o;
  Eight<R> r;
  auto ask = [&](int64_t m) {
    if (m >= p.M) return;
    const T* po = static_cast<const T*>(p.o) + m * p.o_stride + d;
    if (kWhole && n >= 8) o.load(po);
    else o.load(po, n);
    if (p.residual) {
      const R* pr = static_cast<const R*>(p.residual) + m * p.residual_stride + d;
      if (kWhole && n >= 8) r.load(pr);
      else r.load(pr, n);
    }
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
      R* x = static_cast<R*>(p.x) + m * p.D + d;
      if (kWhole && n >= 8) r.store(x);
      else r.store(x, n);
    }
    ask(m + step);
    float mean = 0.f;
    if (p.layer) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) s += z[j];      // (zeros behind the last column)
      mean = over_token<kWidth>(s, parts[turn][0], add_up) * inv_d;
    }
    float sq = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      z[j] -= mean;
      if (kWhole ? n > 0 : j < n) sq = fmaf(z[j], z[j], sq);
    }
    const float dev = inverse_root(fmaf(over_token<kWidth>(sq, parts[turn][1], add_up), inv_d, p.eps));
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      z[j] = z[j] * dev * w.v[j];
      if (p.bias) z[j] += b.v[j];
      if (kWhole ? n > 0 : j < n) most = magnitude(most, z[j]);
    }
    if (p.group) {
      for (int e = lanes / 2; e; e /= 2) most = max(most, __shfl_xor_sync(0xffffffffu, most, e));
    } else {
      most = over_token<kWidth>(most, tops[turn], [](uint32_t a, uint32_t b) { return max(a, b); });
    }
    if (!live || n <= 0) continue;
    const uint32_t x = scale_exponent(most);
    const float inv = inverse_of(x);
    Eight<uint8_t> q;
#pragma unroll
    for (int j = 0; j < 4; ++j) reinterpret_cast<uint16_t*>(q.v)[j] = static_cast<uint16_t>(two_bytes(z[2 * j] * inv, z[2 * j + 1] * inv));
    uint8_t* dst = static_cast<uint8_t*>(p.values) + m * p.D + d;
    if (kWhole && n >= 8) q.store(dst);
    else q.store(dst, n);
    if (p.group ? lane % lanes == 0 : lane == 0) p.scales[m * groups + (p.group ? lane / lanes : 0)] = scale_of(x);
    if (p.stats && lane == 0) reinterpret_cast<float4*>(p.stats)[m] = make_float4(0.f, 1.f, mean, dev);
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
  for (int k = 0; k < p->count; ++k)
    if (!p->values[k] || !p->scales[k] || !(back ? p->dst[k] : p->src[k])) return fail("pack8: null tensor pointer");
  if (p->M == 0) return fail("pack8: no rows");
  return TTT_B200_OK;
}
template <class T> int run(Many& q, bool back, cudaStream_t s) {
  const ttt_b200_pack8_args& a = q.a;
  const int L = back ? 1 : a.group / 8;
  const int64_t lanes = (a.D + 8L * L - 1) / (8L * L) * L;
  q.lanes = static_cast<uint32_t>(lanes);
  if (a.M > (255L << 31) / lanes) return fail("pack8: too many values");
  q.vectors = a.M * lanes;
  const int64_t blocks = (q.vectors + 255) / 256;
  bool whole = true;
  for (int k = 0; k < a.count; ++k)
    whole = whole && rows<uint8_t>(a.values[k], a.D) && (back ? rows<T>(a.dst[k], a.D) : rows<T>(a.src[k], a.stride[k]));
  auto kernel = back ? (whole ? unpack8_kernel<T, true> : unpack8_kernel<T, false>)
              : L == 4 ? (whole ? pack8_kernel<T, true, 4> : pack8_kernel<T, false, 4>)
              : L == 8 ? (whole ? pack8_kernel<T, true, 8> : pack8_kernel<T, false, 8>)
                       : (whole ? pack8_kernel<T, true, 16> : pack8_kernel<T, false, 16>);
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

template <class T, class R, int kWidth> int norm_as(const ttt_b200_norm8_args& p, cudaStream_t s) {
  constexpr int side = kSide<kWidth>, threads = kWidth * side;
  const bool whole = p.D % 8 == 0 && rows<T>(p.o, p.o_stride) && rows<R>(p.residual, p.residual_stride) && rows<R>(p.x, p.D) && rows<uint8_t>(p.values, p.D);
  const int ctas = static_cast<int>(std::min<int64_t>(static_cast<int64_t>(sm_count()) * (1024 / threads), (p.M + side - 1) / side));
  ttt_launch_overlapped(whole ? norm8_kernel<T, R, kWidth, true> : norm8_kernel<T, R, kWidth, false>, ctas, threads, 0, s, p);
  return launched("norm8");
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
  Many q = {*p, 0, 0};
  TTT_WITH_TYPE(p->dtype, return run<Elem>(q, false, static_cast<cudaStream_t>(stream)))
  return TTT_B200_OK;
}

extern "C" int ttt_b200_unpack8(const ttt_b200_pack8_args* p, void* stream) {
  if (int rc = check(p, true)) return rc;
  Many q = {*p, 0, 0};
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
