// Selective state space scan: forward for prompts and training, backward, and the step of single tokens.
//
//   delta = softplus(dt + dt_bias)
//   h[d][n] <- exp(delta A[d][n]) h[d][n] + delta x[d] B[g][n]        g: the group of channel d
//   y[d]     = sum_n C[g][n] h[d][n] + D[d] x[d]
//
// Backward, with dh_t the gradient with respect to the state after token t and c_t = exp(delta_t A) dh_t what it leaves for
// the token before:  dh_t = C_t dy_t + c_{t+1};  dC = sum_d dy h;  dB = sum_d delta x dh;  dx = delta sum_n dh B + D dy;
// d delta = sum_n dh (A exp(delta A) h_{t-1} + x B);  dA = sum_t delta dh exp(delta A) h_{t-1};  dh_{-1} = c_0.
//
// What bounds it: not memory.  A (token, channel) is read and written in 6 bytes (bf16) and costs N exponentials and 5 N fp32
// operations.  The exponentials leave at 16 per cycle and SM, four instructions' worth of issue slots each, so the arithmetic
// is packed two to an instruction and the operands that lanes share (delta, B, C) come from shared memory in fp32.
//
// A thread owns four states of a channel (of two channels in the backward) and walks along the tokens; the LN lanes of a
// channel add their parts of y by exchanging halves over LN tokens at a time.  Channels, groups and sequences are independent.
// Where they do not fill the GPU the sequence is split into chunks as well: a first kernel carries each chunk's state from
// zero, a second one joins the chunks with exp(A sum delta), and the main kernel starts every chunk from its own state.  The
// backward does the same from the other end.
#include <algorithm>
#include <cstdio>

#include "ttt_elem.cuh"
#include "ttt_sum_parts.h"

namespace {

using namespace ttt;

constexpr int kTile = TTT_B200_SCAN_INTERVAL;      // tokens staged at a time, and between two checkpoints
static_assert(kTile == 16, "the kernels unroll over tiles of 16 tokens");

// How a CTA is made up for LN lanes per channel (up to 4 LN states); CH channels per thread.
template <int LN, int CH> struct Shape {
  static constexpr int NP = 4 * LN;                                     // states, padded
  static constexpr int TH = CH == 1 && LN > 4 ? 32 * LN : 128;
  static constexpr int DC = TH / LN * CH;                               // channels of a CTA
  static constexpr int CPW = 32 / LN;                                   // channels next to each other in a warp
};

struct Plan {
  int per;        // channels of a group
  int tiles;      // CTAs to a group's channels
  int chunk;      // tokens of a chunk, a multiple of kTile
  int chunks;
  int nck;        // checkpoints of a sequence
  bool vec_x, vec_dt, vec_gy, vec_b, vec_c, vec_n;      // 16-byte rows; whole float4 of states
  float* state;   // [B][chunks][D][N]: what a chunk starts from (backward: ends with)
  float* delta;   // [B][chunks][D]: sum of delta
  float* part_bc; // backward: [2][tiles][B][T][G][N]
  float* part_a;  // backward: [B][chunks][D][N]
  float* part_d;  // backward: [2][B][chunks][D]: grad_D, grad_dt_bias
};

struct Where {
  int b, c, g, tile, ch0, cols;
  long bc;        // b * chunks + c
  int len;        // tokens of the sequence
  __device__ Where(const ttt_b200_scan_args& p, const Plan& q, int dc) {
    long i = blockIdx.x;
    tile = static_cast<int>(i % q.tiles);
    i /= q.tiles;
    g = static_cast<int>(i % p.G);
    bc = i / p.G;
    c = static_cast<int>(bc % q.chunks);
    b = static_cast<int>(bc / q.chunks);
    ch0 = g * q.per + tile * dc;
    cols = min(q.per - tile * dc, dc);
    len = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
  }
};

// `rows` x `cols` elements -> [kTile][W], the rest zeros.
template <class T, int W, int TH> __device__ __forceinline__ void stage(T* dst, const T* src, int64_t stride, int rows, int cols, bool vec) {
  constexpr int PV = 16 / sizeof(T), PR = W / PV;
  if (vec) {
#pragma unroll
    for (int i0 = 0; i0 < kTile * PR; i0 += TH) {
      const int i = i0 + threadIdx.x;
      if (kTile * PR % TH != 0 && i >= kTile * PR) break;
      const int t = i / PR, c = i % PR * PV;
      const int n = t < rows ? min(max(cols - c, 0), PV) : 0;
      cp_async16(dst + t * W + c, n > 0 ? src + t * stride + c : src, n * static_cast<int>(sizeof(T)));
    }
  } else {
    for (int i = threadIdx.x; i < kTile * W; i += TH) {
      const int t = i / W, c = i % W;
      dst[i] = t < rows && c < cols ? src[t * stride + c] : from_f32<T>(0.f);
    }
  }
}

// delta and its derivative.  log1p(e) of e = exp(-|v|) in (0, 1] as 2 atanh(e / (2 + e)), whose series in s^2 <= 1/9 is cut
// where its next term is 2e-8 of the value; log(1 + e) itself would lose the small steps that matter most.
__device__ __forceinline__ float2 softplus(float v) {
  const float e = ex2(-fabsf(v) * kLog2e);
  const float s = e * rcp(2.f + e), q = s * s;
  float r = fmaf(q, 1.f / 13, 1.f / 11);
  r = fmaf(q, r, 1.f / 9);
  r = fmaf(q, r, 1.f / 7);
  r = fmaf(q, r, 1.f / 5);
  r = fmaf(q, r, 1.f / 3);
  r = fmaf(q, r, 1.f);
  return make_float2(fmaxf(v, 0.f) + 2.f * s * r, (v >= 0.f ? 1.f : e) * rcp(1.f + e));
}

// four states of a row [N] of fp32
__device__ __forceinline__ void load_states(const float* p, int n0, int N, bool vec, float (&h)[4]) {
  if (vec && n0 + 4 <= N) {
    const float4 v = *reinterpret_cast<const float4*>(p + n0);
    h[0] = v.x, h[1] = v.y, h[2] = v.z, h[3] = v.w;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) h[k] = n0 + k < N ? p[n0 + k] : 0.f;
  }
}
__device__ __forceinline__ void store_states(float* p, int n0, int N, bool vec, const float (&h)[4]) {
  if (vec && n0 + 4 <= N) {
    *reinterpret_cast<float4*>(p + n0) = make_float4(h[0], h[1], h[2], h[3]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (n0 + k < N) p[n0 + k] = h[k];
  }
}
__device__ __forceinline__ void split(const float4 v, float2 (&o)[2]) {
  o[0] = make_float2(v.x, v.y);
  o[1] = make_float2(v.z, v.w);
}

// ---- forward ---------------------------------------------------------------------------------------------------------
template <class T, int LN> struct FwdSmem {
  using S = Shape<LN, 1>;
  static constexpr int YW = S::DC + S::CPW;      // the y of a warp's channels and LN tokens in different banks
  alignas(16) T x[2][kTile * S::DC];
  alignas(16) T dt[2][kTile * S::DC];
  alignas(16) T b[2][kTile * S::NP];
  alignas(16) T c[2][kTile * S::NP];
  alignas(16) float2 u[kTile * S::DC];      // delta, delta x
  alignas(16) float fb[kTile * S::NP];
  alignas(16) float fc[kTile * S::NP];
  float y[kTile * YW];
};

template <class T, int LN> __global__ void __launch_bounds__(Shape<LN, 1>::TH) scan_forward_kernel(const ttt_b200_scan_args p, const Plan q) {
  using S = Shape<LN, 1>;
  constexpr int TH = S::TH, DC = S::DC, NP = S::NP, U = LN < 4 ? 4 : LN, YW = FwdSmem<T, LN>::YW;
  extern __shared__ __align__(16) unsigned char raw[];
  FwdSmem<T, LN>& m = *reinterpret_cast<FwdSmem<T, LN>*>(raw);
  const Where w(p, q, DC);
  const int lane = threadIdx.x & 31, li = lane % LN, ch = threadIdx.x / LN, n0 = 4 * li;
  const bool live = ch < w.cols;
  const long row = static_cast<long>(w.ch0 + ch) * p.N, DN = static_cast<long>(p.D) * p.N;

  float2 a2[2] = {}, h[2] = {};
  if (live) {
    float v[4];
    load_states(p.A + row, n0, p.N, q.vec_n, v);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] *= kLog2e;
    split(make_float4(v[0], v[1], v[2], v[3]), a2);
    const float* from = q.chunks > 1 ? q.state + w.bc * DN : p.state ? p.state + w.b * DN : nullptr;
    if (from) {
      load_states(from + row, n0, p.N, q.vec_n, v);
      split(make_float4(v[0], v[1], v[2], v[3]), h);
    }
  }
  // this thread's channel where elements are worked on one at a time
  const int ec = threadIdx.x % DC;
  const float bias = p.dt_bias && ec < w.cols ? p.dt_bias[w.ch0 + ec] : 0.f;
  const float skip = p.Dskip && ec < w.cols ? p.Dskip[w.ch0 + ec] : 0.f;

  const int begin = w.c * q.chunk, end = min(begin + q.chunk, p.T);
  const T* xs = static_cast<const T*>(p.x) + w.b * p.x_stride[0] + w.ch0;
  const T* ds = static_cast<const T*>(p.dt) + w.b * p.dt_stride[0] + w.ch0;
  const T* bs = static_cast<const T*>(p.Bm) + w.b * p.B_stride[0] + w.g * p.B_stride[2];
  const T* cs = static_cast<const T*>(p.Cm) + w.b * p.C_stride[0] + w.g * p.C_stride[2];
  T* ys = static_cast<T*>(p.y) + static_cast<long>(w.b) * p.T * p.D + w.ch0;
  auto fetch = [&](int t0, int buf) {
    const int rows = min(w.len - t0, kTile);
    if (t0 < end && rows > 0) {
      stage<T, DC, TH>(m.x[buf], xs + t0 * p.x_stride[1], p.x_stride[1], rows, w.cols, q.vec_x);
      stage<T, DC, TH>(m.dt[buf], ds + t0 * p.dt_stride[1], p.dt_stride[1], rows, w.cols, q.vec_dt);
      stage<T, NP, TH>(m.b[buf], bs + t0 * p.B_stride[1], p.B_stride[1], rows, p.N, q.vec_b);
      stage<T, NP, TH>(m.c[buf], cs + t0 * p.C_stride[1], p.C_stride[1], rows, p.N, q.vec_c);
    }
    cp_async_commit();
  };

  fetch(begin, 0);
  int buf = 0;
  for (int t0 = begin; t0 < end; t0 += kTile, buf ^= 1) {
    const int rows = min(w.len - t0, kTile);
    if (rows <= 0) {      // behind the sequence: zeros, and the state stays
      for (int i = threadIdx.x; i < kTile * DC; i += TH)
        if (t0 + i / DC < end && ec < w.cols) ys[static_cast<long>(t0 + i / DC) * p.D + ec] = from_f32<T>(0.f);
      continue;
    }
    cp_async_wait<0>();
    __syncthreads();      // the tile has landed, and no thread reads the other buffer any more
    fetch(t0 + kTile, buf ^ 1);
#pragma unroll
    for (int i0 = 0; i0 < kTile * DC; i0 += TH) {
      const int i = i0 + threadIdx.x;
      const float v = to_f32(m.dt[buf][i]) + bias;
      const float d = i / DC < rows ? (p.softplus ? softplus(v).x : v) : 0.f;
      m.u[i] = make_float2(d, d * to_f32(m.x[buf][i]));
    }
    for (int i = threadIdx.x; i < kTile * NP; i += TH) {
      m.fb[i] = to_f32(m.b[buf][i]);
      m.fc[i] = to_f32(m.c[buf][i]);
    }
    __syncthreads();
    if (p.checkpoints && live) {
      const float v[4] = {h[0].x, h[0].y, h[1].x, h[1].y};
      store_states(p.checkpoints + (static_cast<long>(w.b) * q.nck + t0 / kTile) * DN + row, n0, p.N, q.vec_n, v);
    }
#pragma unroll
    for (int s = 0; s < kTile; s += U) {
      float acc[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int t = s + k;
        const float2 du = m.u[t * DC + ch];
        float2 b[2], c[2];
        split(*reinterpret_cast<const float4*>(m.fb + t * NP + n0), b);
        split(*reinterpret_cast<const float4*>(m.fc + t * NP + n0), c);
        float2 y;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float2 e = mul2(both(du.x), a2[j]);
          h[j] = fma2(make_float2(ex2(e.x), ex2(e.y)), h[j], mul2(both(du.y), b[j]));
          y = j ? fma2(h[j], c[j], y) : mul2(h[j], c[j]);
        }
        acc[k] = y.x + y.y;
      }
      spread_sum<U, LN, 1>(acc, lane);
#pragma unroll
      for (int k = 0; k < U / LN; ++k) m.y[(s + li * (U / LN) + k) * YW + ch] = acc[k];
    }
    __syncthreads();
#pragma unroll
    for (int i0 = 0; i0 < kTile * DC; i0 += TH) {
      const int t = (i0 + threadIdx.x) / DC;
      if (t0 + t < end && ec < w.cols) {
        const float y = t < rows ? fmaf(skip, to_f32(m.x[buf][t * DC + ec]), m.y[t * YW + ec]) : 0.f;
        ys[static_cast<long>(t0 + t) * p.D + ec] = from_f32<T>(y);
      }
    }
  }
  if (p.final_state && w.c == q.chunks - 1 && live) {
    const float v[4] = {h[0].x, h[0].y, h[1].x, h[1].y};
    store_states(p.final_state + w.b * DN + row, n0, p.N, q.vec_n, v);
  }
}

// ---- a chunk's state by itself, from zero: forwards h <- a h + delta x B; backwards (kRev) c <- a (c + dy C) -----------
template <class T, int LN> struct StateSmem {
  using S = Shape<LN, 1>;
  alignas(16) T v[2][kTile * S::DC];      // x or dy
  alignas(16) T dt[2][kTile * S::DC];
  alignas(16) T n[2][kTile * S::NP];      // B or C
  alignas(16) float2 u[kTile * S::DC];
  alignas(16) float fn[kTile * S::NP];
};

template <class T, int LN, bool kRev>
__global__ void __launch_bounds__(Shape<LN, 1>::TH) scan_state_kernel(const ttt_b200_scan_args p, const Plan q) {
  using S = Shape<LN, 1>;
  constexpr int TH = S::TH, DC = S::DC, NP = S::NP;
  extern __shared__ __align__(16) unsigned char raw[];
  StateSmem<T, LN>& m = *reinterpret_cast<StateSmem<T, LN>*>(raw);
  const Where w(p, q, DC);
  const int li = threadIdx.x % LN, ch = threadIdx.x / LN, n0 = 4 * li;
  const bool live = ch < w.cols;
  const long row = static_cast<long>(w.ch0 + ch) * p.N, DN = static_cast<long>(p.D) * p.N;
  float2 a2[2] = {}, h[2] = {};
  if (live) {
    float v[4];
    load_states(p.A + row, n0, p.N, q.vec_n, v);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] *= kLog2e;
    split(make_float4(v[0], v[1], v[2], v[3]), a2);
  }
  const int ec = threadIdx.x % DC;
  const float bias = p.dt_bias && ec < w.cols ? p.dt_bias[w.ch0 + ec] : 0.f;
  const int64_t* vst = kRev ? p.gy_stride : p.x_stride;
  const int64_t* nst = kRev ? p.C_stride : p.B_stride;
  const T* vs = static_cast<const T*>(kRev ? p.grad_y : p.x) + w.b * vst[0] + w.ch0;
  const T* ds = static_cast<const T*>(p.dt) + w.b * p.dt_stride[0] + w.ch0;
  const T* ns = static_cast<const T*>(kRev ? p.Cm : p.Bm) + w.b * nst[0] + w.g * nst[2];
  const int begin = w.c * q.chunk, end = min(begin + q.chunk, w.len);
  const int count = end > begin ? (end - begin + kTile - 1) / kTile : 0;
  auto at = [&](int k) { return begin + (kRev ? count - 1 - k : k) * kTile; };
  auto fetch = [&](int k, int buf) {
    if (k < count) {
      const int t0 = at(k), rows = min(end - t0, kTile);
      stage<T, DC, TH>(m.v[buf], vs + t0 * vst[1], vst[1], rows, w.cols, kRev ? q.vec_gy : q.vec_x);
      stage<T, DC, TH>(m.dt[buf], ds + t0 * p.dt_stride[1], p.dt_stride[1], rows, w.cols, q.vec_dt);
      stage<T, NP, TH>(m.n[buf], ns + t0 * nst[1], nst[1], rows, p.N, kRev ? q.vec_c : q.vec_b);
    }
    cp_async_commit();
  };
  float total = 0.f;
  fetch(0, 0);
  for (int k = 0; k < count; ++k) {
    const int buf = k & 1, rows = min(end - at(k), kTile);
    cp_async_wait<0>();
    __syncthreads();
    fetch(k + 1, buf ^ 1);
#pragma unroll
    for (int i0 = 0; i0 < kTile * DC; i0 += TH) {
      const int i = i0 + threadIdx.x;
      const float v = to_f32(m.dt[buf][i]) + bias;
      const float d = i / DC < rows ? (p.softplus ? softplus(v).x : v) : 0.f;
      m.u[i] = make_float2(d, kRev ? to_f32(m.v[buf][i]) : d * to_f32(m.v[buf][i]));
    }
    for (int i = threadIdx.x; i < kTile * NP; i += TH) m.fn[i] = to_f32(m.n[buf][i]);
    __syncthreads();
#pragma unroll 4
    for (int s = 0; s < kTile; ++s) {
      const int t = kRev ? kTile - 1 - s : s;
      const float2 du = m.u[t * DC + ch];
      float2 b[2];
      split(*reinterpret_cast<const float4*>(m.fn + t * NP + n0), b);
      total += du.x;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 e = mul2(both(du.x), a2[j]);
        const float2 f = make_float2(ex2(e.x), ex2(e.y));
        h[j] = kRev ? mul2(f, fma2(both(du.y), b[j], h[j])) : fma2(f, h[j], mul2(both(du.y), b[j]));
      }
    }
  }
  if (live) {
    const float v[4] = {h[0].x, h[0].y, h[1].x, h[1].y};
    store_states(q.state + w.bc * DN + row, n0, p.N, q.vec_n, v);
    if (li == 0) q.delta[w.bc * p.D + w.ch0 + ch] = total;
  }
}

// The chunks' own states -> the states that they start from (kRev: that they end with), in place, in the order of time.
template <bool kRev> __global__ void __launch_bounds__(256) scan_join_kernel(const ttt_b200_scan_args p, const Plan q) {
  const long DN = static_cast<long>(p.D) * p.N;
  const long i = static_cast<long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= p.B * DN) return;
  const long b = i / DN, dn = i % DN, d = dn / p.N;
  const float a2 = p.A[dn] * kLog2e;
  const float* from = kRev ? p.grad_final_state : p.state;
  float h = from ? from[i] : 0.f;
  constexpr int kAhead = 8;
  for (int c0 = 0; c0 < q.chunks; c0 += kAhead) {
    float s[kAhead], f[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const long c = b * q.chunks + (kRev ? q.chunks - 1 - min(c0 + k, q.chunks - 1) : min(c0 + k, q.chunks - 1));
      s[k] = q.state[c * DN + dn];
      f[k] = ex2(a2 * q.delta[c * p.D + d]);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (c0 + k < q.chunks) {
        const long c = b * q.chunks + (kRev ? q.chunks - 1 - (c0 + k) : c0 + k);
        q.state[c * DN + dn] = h;
        h = fmaf(f[k], h, s[k]);
      }
  }
}

// ---- backward --------------------------------------------------------------------------------------------------------
constexpr int kSub = 4;      // tokens whose states and factors are in registers at a time

template <class T, int LN> struct BwdSmem {
  using S = Shape<LN, 2>;
  static constexpr int OW = S::DC + S::CPW;
  alignas(16) T x[2][kTile * S::DC];
  alignas(16) T dt[2][kTile * S::DC];
  alignas(16) T gy[2][kTile * S::DC];
  alignas(16) T b[2][kTile * S::NP];
  alignas(16) T c[2][kTile * S::NP];
  alignas(16) float4 u[kTile * S::DC];      // delta, delta x, dy, d delta / d dt
  alignas(16) float fb[kTile * S::NP];
  alignas(16) float fc[kTile * S::NP];
  alignas(16) float4 start[kTile / kSub][2][S::TH];      // each thread's states at the starts of the runs of kSub tokens
  float bc[kTile][S::TH / 32][2 * S::NP];     // each warp's part of dB and dC
  float o[2][kTile * OW];                   // sum_n dh A exp(delta A) h (in base 2), sum_n dh B
};

template <class T, int LN>
__global__ void __launch_bounds__(Shape<LN, 2>::TH, 3) scan_backward_kernel(const ttt_b200_scan_args p, const Plan q) {
  using S = Shape<LN, 2>;
  constexpr int TH = S::TH, DC = S::DC, NP = S::NP, CPW = S::CPW, OW = BwdSmem<T, LN>::OW, ND = 32 / LN;
  extern __shared__ __align__(16) unsigned char raw[];
  BwdSmem<T, LN>& m = *reinterpret_cast<BwdSmem<T, LN>*>(raw);
  const Where w(p, q, DC);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, li = lane % LN, dl = lane / LN, n0 = 4 * li;
  const int ch[2] = {warp * 2 * CPW + dl, warp * 2 * CPW + CPW + dl};
  const long DN = static_cast<long>(p.D) * p.N;
  long row[2];
  float2 a2[2][2] = {}, carry[2][2] = {}, da[2][2] = {};
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    row[e] = static_cast<long>(w.ch0 + ch[e]) * p.N;
    if (ch[e] >= w.cols) continue;
    float v[4];
    load_states(p.A + row[e], n0, p.N, q.vec_n, v);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] *= kLog2e;
    split(make_float4(v[0], v[1], v[2], v[3]), a2[e]);
    const float* from = q.chunks > 1 ? q.state + w.bc * DN : p.grad_final_state ? p.grad_final_state + w.b * DN : nullptr;
    if (from) {
      load_states(from + row[e], n0, p.N, q.vec_n, v);
      split(make_float4(v[0], v[1], v[2], v[3]), carry[e]);
    }
  }
  const int ec = threadIdx.x % DC;
  const bool elive = ec < w.cols;
  const float bias = p.dt_bias && elive ? p.dt_bias[w.ch0 + ec] : 0.f;
  const float skip = p.Dskip && elive ? p.Dskip[w.ch0 + ec] : 0.f;
  float sum_d = 0.f, sum_bias = 0.f;

  const int begin = w.c * q.chunk, end = min(begin + q.chunk, p.T);
  const T* xs = static_cast<const T*>(p.x) + w.b * p.x_stride[0] + w.ch0;
  const T* ds = static_cast<const T*>(p.dt) + w.b * p.dt_stride[0] + w.ch0;
  const T* gs = static_cast<const T*>(p.grad_y) + w.b * p.gy_stride[0] + w.ch0;
  const T* bs = static_cast<const T*>(p.Bm) + w.b * p.B_stride[0] + w.g * p.B_stride[2];
  const T* cs = static_cast<const T*>(p.Cm) + w.b * p.C_stride[0] + w.g * p.C_stride[2];
  const long out0 = static_cast<long>(w.b) * p.T * p.D + w.ch0;
  T* gxs = static_cast<T*>(p.grad_x) + out0;
  T* gds = static_cast<T*>(p.grad_dt) + out0;
  const long GN = static_cast<long>(p.G) * p.N, BTGN = static_cast<long>(p.B) * p.T * GN;
  float* pb = q.part_bc + w.tile * BTGN + static_cast<long>(w.b) * p.T * GN + w.g * p.N;
  float* pc = pb + q.tiles * BTGN;
  auto fetch = [&](int t0, int buf) {
    const int rows = min(w.len - t0, kTile);
    if (t0 >= begin && rows > 0) {
      stage<T, DC, TH>(m.x[buf], xs + t0 * p.x_stride[1], p.x_stride[1], rows, w.cols, q.vec_x);
      stage<T, DC, TH>(m.dt[buf], ds + t0 * p.dt_stride[1], p.dt_stride[1], rows, w.cols, q.vec_dt);
      stage<T, DC, TH>(m.gy[buf], gs + t0 * p.gy_stride[1], p.gy_stride[1], rows, w.cols, q.vec_gy);
      stage<T, NP, TH>(m.b[buf], bs + t0 * p.B_stride[1], p.B_stride[1], rows, p.N, q.vec_b);
      stage<T, NP, TH>(m.c[buf], cs + t0 * p.C_stride[1], p.C_stride[1], rows, p.N, q.vec_c);
    }
    cp_async_commit();
  };

  const int last = begin + (end - begin - 1) / kTile * kTile;
  fetch(last, 0);
  int buf = 0;
  for (int t0 = last; t0 >= begin; t0 -= kTile, buf ^= 1) {
    const int rows = min(w.len - t0, kTile);
    if (rows <= 0) {      // behind the sequence: zeros, and the gradient of the state passes through
      for (int i = threadIdx.x; i < kTile * DC; i += TH)
        if (t0 + i / DC < end && elive) {
          gxs[static_cast<long>(t0 + i / DC) * p.D + ec] = from_f32<T>(0.f);
          gds[static_cast<long>(t0 + i / DC) * p.D + ec] = from_f32<T>(0.f);
        }
      for (int i = threadIdx.x; i < kTile * NP; i += TH)
        if (t0 + i / NP < end && i % NP < p.N) {
          pb[(t0 + i / NP) * GN + i % NP] = 0.f;
          pc[(t0 + i / NP) * GN + i % NP] = 0.f;
        }
      fetch(t0 - kTile, buf ^ 1);
      continue;
    }
    float2 h0[2][2] = {};      // the state before the tile
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (ch[e] < w.cols) {
        float v[4];
        load_states(p.checkpoints + (static_cast<long>(w.b) * q.nck + t0 / kTile) * DN + row[e], n0, p.N, q.vec_n, v);
        split(make_float4(v[0], v[1], v[2], v[3]), h0[e]);
      }
    cp_async_wait<0>();
    __syncthreads();      // the tile has landed, and no thread reads the other buffer any more
    fetch(t0 - kTile, buf ^ 1);
#pragma unroll
    for (int i0 = 0; i0 < kTile * DC; i0 += TH) {
      const int i = i0 + threadIdx.x;
      const float v = to_f32(m.dt[buf][i]) + bias;
      float2 d = p.softplus ? softplus(v) : make_float2(v, 1.f);
      if (i / DC >= rows) d = make_float2(0.f, 0.f);
      m.u[i] = make_float4(d.x, d.x * to_f32(m.x[buf][i]), to_f32(m.gy[buf][i]), d.y);
    }
    for (int i = threadIdx.x; i < kTile * NP; i += TH) {
      m.fb[i] = to_f32(m.b[buf][i]);
      m.fc[i] = to_f32(m.c[buf][i]);
    }
    __syncthreads();
    {      // the states at the starts of the runs
      float2 h[2][2] = {{h0[0][0], h0[0][1]}, {h0[1][0], h0[1][1]}};
#pragma unroll 1
      for (int s = 0;; ++s) {
#pragma unroll
        for (int e = 0; e < 2; ++e) m.start[s][e][threadIdx.x] = make_float4(h[e][0].x, h[e][0].y, h[e][1].x, h[e][1].y);
        if (s == kTile / kSub - 1) break;
#pragma unroll
        for (int k = 0; k < kSub; ++k) {
          const int t = s * kSub + k;
          float2 b[2];
          split(*reinterpret_cast<const float4*>(m.fb + t * NP + n0), b);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float4 u = m.u[t * DC + ch[e]];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float2 x = mul2(both(u.x), a2[e][j]);
              h[e][j] = fma2(make_float2(ex2(x.x), ex2(x.y)), h[e][j], mul2(both(u.y), b[j]));
            }
          }
        }
      }
    }
#pragma unroll 1
    for (int s = kTile / kSub - 1; s >= 0; --s) {
      float2 f[2][kSub][2], h[2][kSub + 1][2];      // factors; states before token k of the run
#pragma unroll
      for (int e = 0; e < 2; ++e) split(m.start[s][e][threadIdx.x], h[e][0]);
#pragma unroll
      for (int k = 0; k < kSub; ++k) {
        const int t = s * kSub + k;
        float2 b[2];
        split(*reinterpret_cast<const float4*>(m.fb + t * NP + n0), b);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float4 u = m.u[t * DC + ch[e]];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 x = mul2(both(u.x), a2[e][j]);
            f[e][k][j] = make_float2(ex2(x.x), ex2(x.y));
            h[e][k + 1][j] = fma2(f[e][k][j], h[e][k][j], mul2(both(u.y), b[j]));
          }
        }
      }
#pragma unroll
      for (int k = kSub - 1; k >= 0; --k) {
        const int t = s * kSub + k;
        float2 b[2], c[2], vb[2], vc[2];
        split(*reinterpret_cast<const float4*>(m.fb + t * NP + n0), b);
        split(*reinterpret_cast<const float4*>(m.fc + t * NP + n0), c);
        float o[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float4 u = m.u[t * DC + ch[e]];
          float2 qa, gb;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 g = fma2(both(u.z), c[j], carry[e][j]);
            vb[j] = e ? fma2(both(u.y), g, vb[j]) : mul2(both(u.y), g);
            vc[j] = e ? fma2(both(u.z), h[e][k + 1][j], vc[j]) : mul2(both(u.z), h[e][k + 1][j]);
            gb = j ? fma2(g, b[j], gb) : mul2(g, b[j]);
            carry[e][j] = mul2(f[e][k][j], g);
            const float2 r = mul2(carry[e][j], h[e][k][j]);
            qa = j ? fma2(r, a2[e][j], qa) : mul2(r, a2[e][j]);
            da[e][j] = fma2(both(u.x), r, da[e][j]);
          }
          o[e] = qa.x + qa.y;
          o[2 + e] = gb.x + gb.y;
        }
        // dx and d delta: over the channel's lanes
        spread_sum<4, LN, 1>(o, lane);
        if constexpr (LN <= 4) {
#pragma unroll
          for (int r = 0; r < 4 / LN; ++r) {
            const int i = li * (4 / LN) + r;
            m.o[i >> 1][t * OW + (i & 1 ? ch[1] : ch[0])] = o[r];
          }
        } else {
          const int i = li / (LN / 4);
          if (li % (LN / 4) == 0) m.o[i >> 1][t * OW + (i & 1 ? ch[1] : ch[0])] = o[0];
        }
        // dB and dC: over the warp's channels
        float v[8] = {vb[0].x, vb[0].y, vb[1].x, vb[1].y, vc[0].x, vc[0].y, vc[1].x, vc[1].y};
        spread_sum<8, ND, LN>(v, lane);
        if constexpr (ND <= 8) {
#pragma unroll
          for (int r = 0; r < 8 / ND; ++r) {
            const int i = dl * (8 / ND) + r;
            m.bc[t][warp][(i >> 2) * NP + n0 + (i & 3)] = v[r];
          }
        } else {
          const int i = dl / (ND / 8);
          if (dl % (ND / 8) == 0) m.bc[t][warp][(i >> 2) * NP + n0 + (i & 3)] = v[0];
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int i0 = 0; i0 < kTile * DC; i0 += TH) {
      const int t = (i0 + threadIdx.x) / DC;
      if (t0 + t < end && elive) {
        const float4 u = m.u[t * DC + ec];
        const float x = to_f32(m.x[buf][t * DC + ec]), gb = m.o[1][t * OW + ec];
        const float gx = fmaf(u.x, gb, skip * u.z), gd = u.w * fmaf(kLn2, m.o[0][t * OW + ec], x * gb);
        const bool in = t < rows;
        gxs[static_cast<long>(t0 + t) * p.D + ec] = from_f32<T>(in ? gx : 0.f);
        gds[static_cast<long>(t0 + t) * p.D + ec] = from_f32<T>(in ? gd : 0.f);
        if (in) {
          sum_d = fmaf(u.z, x, sum_d);
          sum_bias += gd;
        }
      }
    }
    for (int i = threadIdx.x; i < kTile * NP * 2; i += TH) {
      const int t = i / (2 * NP), k = i % (2 * NP);
      float v = 0.f;
#pragma unroll
      for (int r = 0; r < S::TH / 32; ++r) v += m.bc[t][r][k];
      const int n = k % NP;
      if (t0 + t < end && n < p.N) (k < NP ? pb : pc)[(t0 + t) * GN + n] = t < rows ? v : 0.f;
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (ch[e] < w.cols) {
      const float v[4] = {da[e][0].x, da[e][0].y, da[e][1].x, da[e][1].y};
      store_states(q.part_a + w.bc * DN + row[e], n0, p.N, q.vec_n, v);
      if (w.c == 0 && p.grad_state) {
        const float g[4] = {carry[e][0].x, carry[e][0].y, carry[e][1].x, carry[e][1].y};
        store_states(p.grad_state + w.b * DN + row[e], n0, p.N, q.vec_n, g);
      }
    }
  __syncthreads();
  float* red = m.o[0];      // [TH] pairs: what the threads of a channel have summed
  red[threadIdx.x] = sum_d;
  red[TH + threadIdx.x] = sum_bias;
  __syncthreads();
  if (threadIdx.x < DC && elive) {
    for (int r = threadIdx.x + DC; r < TH; r += DC) {
      sum_d += red[r];
      sum_bias += red[TH + r];
    }
    const long BCD = static_cast<long>(p.B) * q.chunks * p.D, i = w.bc * p.D + w.ch0 + ec;
    q.part_d[i] = sum_d;
    q.part_d[BCD + i] = sum_bias;
  }
}

// ---- one token ---------------------------------------------------------------------------------------------------------
// A row of the batch and up to 128 / LN channels to a CTA, each state read and written once.  Rows that name the same slot are
// taken in their order by the CTA of the first of them, so that no two CTAs touch a state.
template <class T, int LN> __global__ void __launch_bounds__(128) scan_step_kernel(const ttt_b200_scan_args p, bool vec_n, int tiles) {
  constexpr int DC = 128 / LN;
  const int b0 = blockIdx.x / tiles, d = (blockIdx.x % tiles) * DC + threadIdx.x / LN;
  const int li = threadIdx.x % LN, n0 = 4 * li;
  const bool live = d < p.D;
  T* ys = static_cast<T*>(p.y);
  int slot = b0, more = 0;
  if (p.slots) {
    slot = p.slots[b0];
    if (slot < 0 || slot >= p.rows) {
      if (live && li == 0) ys[static_cast<long>(b0) * p.D + d] = from_f32<T>(0.f);
      return;
    }
    int before = 0, after = 0;
    for (int r = threadIdx.x; r < p.B; r += 128)
      if (r != b0 && p.slots[r] == slot) (r < b0 ? before : after) = 1;
    if (__syncthreads_or(before)) return;
    more = __syncthreads_or(after);
  }
  const int g = live ? d / (p.D / p.G) : 0;
  float a[4] = {}, h[4] = {};
  float* st = p.state_io + (static_cast<long>(slot) * p.D + d) * p.N;
  if (live) {
    load_states(p.A + static_cast<long>(d) * p.N, n0, p.N, vec_n, a);
    load_states(st, n0, p.N, vec_n, h);
  }
  const float bias = live && p.dt_bias ? p.dt_bias[d] : 0.f, skip = live && p.Dskip ? p.Dskip[d] : 0.f;
  for (int b = b0; b < p.B; ++b) {
    if (b != b0 && p.slots[b] != slot) continue;
    float y = 0.f, x = 0.f;
    if (live) {
      x = to_f32(static_cast<const T*>(p.x)[b * p.x_stride[0] + d]);
      const float v = to_f32(static_cast<const T*>(p.dt)[b * p.dt_stride[0] + d]) + bias;
      const float dl = p.softplus ? softplus(v).x : v;
      const T* bs = static_cast<const T*>(p.Bm) + b * p.B_stride[0] + g * p.B_stride[2];
      const T* cs = static_cast<const T*>(p.Cm) + b * p.C_stride[0] + g * p.C_stride[2];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (n0 + k < p.N) {
          h[k] = fmaf(ex2(dl * (a[k] * kLog2e)), h[k], dl * x * to_f32(bs[n0 + k]));
          y = fmaf(h[k], to_f32(cs[n0 + k]), y);
        }
    }
#pragma unroll
    for (int o = LN / 2; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    if (live && li == 0) ys[static_cast<long>(b) * p.D + d] = from_f32<T>(fmaf(skip, x, y));
    if (!more) break;
  }
  if (live) store_states(st, n0, p.N, vec_n, h);
}

// ---- host --------------------------------------------------------------------------------------------------------------
int lanes_of(int N) { return N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

int sm_count() {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

int fail(const char* msg) { return ttt_set_error(TTT_B200_ERR_BAD_ARGS, msg); }

int check(const ttt_b200_scan_args* p) {
  if (!p) return fail("ssm scan: NULL argument struct");
  if (p->B < 0 || p->T < 0 || p->D < 1 || p->G < 1 || p->N < 1 || p->N > 64)
    return fail("ssm scan: B, T >= 0, D, G >= 1 and 1 to 64 states");
  if (p->D % p->G) return fail("ssm scan: the groups must divide the channels");
  if (p->dtype < TTT_B200_BF16 || p->dtype > TTT_B200_FP32) return fail("ssm scan: unknown element type");
  return TTT_B200_OK;
}

// Tokens to a chunk: see the measurements at the forward's and backward's launch.
void plan_chunks(Plan& q, const ttt_b200_scan_args& p, bool backward) {
  const int LN = lanes_of(p.N), ch = backward ? 2 : 1;
  const int th = ch == 1 && LN > 4 ? 32 * LN : 128;
  const int dc = th / LN * ch;
  q.per = p.D / p.G;
  q.tiles = (q.per + dc - 1) / dc;
  q.nck = (p.T + kTile - 1) / kTile;
  const long ctas = static_cast<long>(p.B) * p.G * q.tiles, warps = ctas * (th / 32);
  const long want = static_cast<long>(sm_count()) * (backward ? 8 : 16);
  long chunks = 1;
  if (warps * 2 < want) chunks = std::min<long>((want + warps - 1) / warps, (q.nck + 3) / 4);
  chunks = std::max<long>(1, std::min<long>(chunks, 64));
  const int per = static_cast<int>((q.nck + chunks - 1) / chunks);
  q.chunk = std::max(per, 1) * kTile;
  q.chunks = std::max(1, (p.T + q.chunk - 1) / q.chunk);
}

size_t up(size_t n) { return (n + 15) / 16 * 16; }

// The scratch's parts, in order; `base` may be null to ask for the size.
size_t lay_out(Plan& q, const ttt_b200_scan_args& p, bool backward, float* base) {
  const size_t DN = static_cast<size_t>(p.D) * p.N, BC = static_cast<size_t>(p.B) * q.chunks;
  size_t at = 0;
  auto take = [&](size_t n) {
    float* r = base ? base + at : nullptr;
    at += up(n);
    return r;
  };
  q.state = q.chunks > 1 ? take(BC * DN) : nullptr;
  q.delta = q.chunks > 1 ? take(BC * p.D) : nullptr;
  if (backward) {
    q.part_bc = take(2 * static_cast<size_t>(q.tiles) * p.B * p.T * p.G * p.N);
    q.part_a = take(BC * DN);
    q.part_d = take(2 * BC * p.D);
  }
  return at * sizeof(float);
}

bool rows16(const void* p, const int64_t* st, int n, size_t es, long inner) {
  bool ok = aligned16(p) && inner * es % 16 == 0;
  for (int i = 0; i < n; ++i) ok = ok && st[i] * static_cast<int64_t>(es) % 16 == 0;
  return ok;
}

int prepare(Plan& q, const ttt_b200_scan_args& p, bool backward) {
  plan_chunks(q, p, backward);
  const size_t need = lay_out(q, p, backward, nullptr);
  if (need && (!p.scratch || p.scratch_bytes < need || !aligned16(p.scratch)))
    return fail("ssm scan: scratch is missing, too small or not 16-byte aligned");
  lay_out(q, p, backward, static_cast<float*>(p.scratch));
  const size_t es = p.dtype == TTT_B200_FP32 ? 4 : 2;
  // a group's first channel has to be aligned too where there are several
  const long inner = p.G > 1 ? q.per : 0;
  q.vec_x = rows16(p.x, p.x_stride, 2, es, inner);
  q.vec_dt = rows16(p.dt, p.dt_stride, 2, es, inner);
  q.vec_gy = backward && rows16(p.grad_y, p.gy_stride, 2, es, inner);
  q.vec_b = rows16(p.Bm, p.B_stride, 3, es, p.N);
  q.vec_c = rows16(p.Cm, p.C_stride, 3, es, p.N);
  q.vec_n = p.N % 4 == 0;
  for (const void* s : {static_cast<const void*>(p.A), static_cast<const void*>(p.state), static_cast<const void*>(p.final_state),
                        static_cast<const void*>(p.checkpoints), static_cast<const void*>(p.grad_final_state),
                        static_cast<const void*>(p.grad_state)})
    q.vec_n = q.vec_n && aligned16(s);
  return TTT_B200_OK;
}

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return TTT_B200_OK;
  static thread_local char buf[160];
  snprintf(buf, sizeof buf, "%s: %s", what, cudaGetErrorString(e));
  return ttt_set_error(TTT_B200_ERR_LAUNCH, buf);
}

template <class K> int launch(K kernel, size_t smem, long grid, int threads, cudaStream_t s, const ttt_b200_scan_args& p, const Plan& q) {
  if (grid > 0x7fffffffL) return fail("ssm scan: too many CTAs");
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return ttt_set_error(TTT_B200_ERR_LAUNCH, cudaGetErrorString(e));
  }
  kernel<<<static_cast<unsigned>(grid), threads, smem, s>>>(p, q);
  return launched("ssm scan");
}

template <class T, int LN> int forward(const ttt_b200_scan_args& p, const Plan& q, cudaStream_t s) {
  const long grid = static_cast<long>(p.B) * q.chunks * p.G * q.tiles;
  if (q.chunks > 1) {
    if (int rc = launch(scan_state_kernel<T, LN, false>, sizeof(StateSmem<T, LN>), grid, Shape<LN, 1>::TH, s, p, q)) return rc;
    const long n = static_cast<long>(p.B) * p.D * p.N;
    scan_join_kernel<false><<<static_cast<unsigned>((n + 255) / 256), 256, 0, s>>>(p, q);
  }
  return launch(scan_forward_kernel<T, LN>, sizeof(FwdSmem<T, LN>), grid, Shape<LN, 1>::TH, s, p, q);
}

template <class T, int LN> int backward(const ttt_b200_scan_args& p, const Plan& q, cudaStream_t s) {
  if (q.chunks > 1) {
    Plan f = q;      // one channel per thread here: other tiles of the same chunks
    f.tiles = (q.per + Shape<LN, 1>::DC - 1) / Shape<LN, 1>::DC;
    const long grid = static_cast<long>(p.B) * q.chunks * p.G * f.tiles;
    if (int rc = launch(scan_state_kernel<T, LN, true>, sizeof(StateSmem<T, LN>), grid, Shape<LN, 1>::TH, s, p, f)) return rc;
    const long n = static_cast<long>(p.B) * p.D * p.N;
    scan_join_kernel<true><<<static_cast<unsigned>((n + 255) / 256), 256, 0, s>>>(p, q);
  }
  const long grid = static_cast<long>(p.B) * q.chunks * p.G * q.tiles;
  if (int rc = launch(scan_backward_kernel<T, LN>, sizeof(BwdSmem<T, LN>), grid, Shape<LN, 2>::TH, s, p, q)) return rc;
  const long BTGN = static_cast<long>(p.B) * p.T * p.G * p.N, DN = static_cast<long>(p.D) * p.N, BCD = static_cast<long>(p.B) * q.chunks * p.D;
  const int bc = p.B * q.chunks;
  const ttt_sum_job jobs[] = {{q.part_bc, p.grad_B, BTGN, BTGN, q.tiles, p.dtype, 0},
                              {q.part_bc + q.tiles * BTGN, p.grad_C, BTGN, BTGN, q.tiles, p.dtype, 0},
                              {q.part_a, p.grad_A, DN, DN, bc, TTT_B200_FP32, 0},
                              {q.part_d, p.grad_D, p.D, p.D, bc, TTT_B200_FP32, 0},
                              {q.part_d + BCD, p.grad_dt_bias, p.D, p.D, bc, TTT_B200_FP32, 0}};
  return ttt_sum_parts(jobs, 5, s);
}

template <class T, int LN> int step(const ttt_b200_scan_args& p, cudaStream_t s) {
  const int tiles = (p.D + 128 / LN - 1) / (128 / LN);
  const bool vec = p.N % 4 == 0 && aligned16(p.A) && aligned16(p.state_io);
  const long grid = static_cast<long>(p.B) * tiles;
  if (grid > 0x7fffffffL) return fail("ssm scan: too many CTAs");
  scan_step_kernel<T, LN><<<static_cast<unsigned>(grid), 128, 0, s>>>(p, vec, tiles);
  return launched("ssm scan step");
}

#define TTT_WITH_LANES(N, call)                                                  \
  switch (lanes_of(N)) {                                                         \
    case 2: { constexpr int LN = 2; return call; }                               \
    case 4: { constexpr int LN = 4; return call; }                               \
    case 8: { constexpr int LN = 8; return call; }                               \
    default: { constexpr int LN = 16; return call; }                             \
  }

}  // namespace

extern "C" uint64_t ttt_b200_ssm_scan_scratch_bytes(const ttt_b200_scan_args* p, int backward) {
  if (check(p) || p->B == 0 || p->T == 0) return 0;
  Plan q = {};
  plan_chunks(q, *p, backward != 0);
  return lay_out(q, *p, backward != 0, nullptr);
}

extern "C" int ttt_b200_ssm_scan(const ttt_b200_scan_args* p, void* stream) {
  if (int rc = check(p)) return rc;
  if (!p->x || !p->dt || !p->A || !p->Bm || !p->Cm || !p->y) return fail("ssm scan: null tensor pointer");
  if (p->B == 0 || p->T == 0) return fail("ssm scan: no tokens");
  Plan q = {};
  if (int rc = prepare(q, *p, false)) return rc;
  TTT_WITH_TYPE(p->dtype, TTT_WITH_LANES(p->N, (forward<Elem, LN>(*p, q, static_cast<cudaStream_t>(stream)))))
  return TTT_B200_OK;
}

extern "C" int ttt_b200_ssm_scan_backward(const ttt_b200_scan_args* p, void* stream) {
  if (int rc = check(p)) return rc;
  if (!p->x || !p->dt || !p->A || !p->Bm || !p->Cm || !p->grad_y || !p->checkpoints || !p->grad_x || !p->grad_dt || !p->grad_A ||
      !p->grad_B || !p->grad_C)
    return fail("ssm scan backward: null tensor pointer");
  if (p->B == 0 || p->T == 0) return fail("ssm scan backward: no tokens");
  Plan q = {};
  if (int rc = prepare(q, *p, true)) return rc;
  TTT_WITH_TYPE(p->dtype, TTT_WITH_LANES(p->N, (backward<Elem, LN>(*p, q, static_cast<cudaStream_t>(stream)))))
  return TTT_B200_OK;
}

extern "C" int ttt_b200_ssm_scan_step(const ttt_b200_scan_args* p, void* stream) {
  if (int rc = check(p)) return rc;
  if (!p->x || !p->dt || !p->A || !p->Bm || !p->Cm || !p->y || !p->state_io) return fail("ssm scan step: null tensor pointer");
  if (p->B == 0) return fail("ssm scan step: no rows");
  if (p->slots ? p->rows < 1 : p->rows != p->B) return fail("ssm scan step: the state has another number of rows");
  TTT_WITH_TYPE(p->dtype, TTT_WITH_LANES(p->N, (step<Elem, LN>(*p, static_cast<cudaStream_t>(stream)))))
  return TTT_B200_OK;
}
