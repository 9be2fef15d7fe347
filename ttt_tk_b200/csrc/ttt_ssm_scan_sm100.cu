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
// A thread owns four states of two channels and walks along the tokens; the LN lanes of a
// channel add their parts of y by exchanging halves over LN tokens at a time.  Channels, groups and sequences are independent.
// Where they do not fill the GPU the sequence is split into chunks as well: a first kernel carries each chunk's state from
// zero, a second one joins the chunks with exp(A sum delta), and the main kernel starts every chunk from its own state.  The
// backward does the same from the other end.
//
// Measured, 4 x 2048 tokens of 1536 channels, 16 states, bf16 (24 chunks; 201 M exponentials, 45 us of their unit): states 67 us, join 5,
// forward 93; backward states 60, join 5, backward 255, sum of parts 11.  8192 tokens of 1024 channels: 45, 7 and 64 us.  The exponential
// unit is 79, 57, 80 and 49 % busy in states, forward, states and backward, the issue slots 52, 58, 52 and 58 %.
#include <algorithm>
#include <type_traits>

#include "ttt_elem.cuh"
#include "ttt_sum_parts.h"

namespace {

using namespace ttt;

constexpr int kTile = TTT_B200_SCAN_INTERVAL;      // tokens staged at a time, and between two checkpoints
static_assert(kTile == 16, "the kernels unroll over tiles of 16 tokens");

// How a CTA is made up for LN lanes per channel (up to 4 LN states); a thread has two channels.
constexpr int TH = 128;
template <int LN> struct Shape {
  static constexpr int NP = 4 * LN;               // states, padded
  static constexpr int DC = TH / LN * 2;          // channels of a CTA
  static constexpr int CPW = 32 / LN;             // channels next to each other in a warp
};

struct Plan {
  int per;        // channels of a group
  int tiles;      // CTAs to a group's channels
  int chunk;      // tokens of a chunk, a multiple of kTile
  int chunks;
  int nck;        // checkpoints of a sequence
  int vec_x, vec_dt, vec_gy, vec_b, vec_c;      // bytes that the rows are aligned for: 16, 4 or 0
  bool vec_n, vec_part, pairs;                  // whole float4 of states; outputs in pairs
  float* state;   // [B][chunks][D][N]: what a chunk starts from (backward: ends with)
  float* delta;   // [B][chunks][D]: sum of delta
  float* part_bc; // backward: [2][tiles][B][T][G][N], where a group has several tiles
  float* part_a;  // backward: [B][chunks][D][N]
  float* part_d;  // backward: [2][B][chunks][D]: grad_D, grad_dt_bias
};

struct Where {
  int b, c, g, tile, ch0, cols;
  long bc;        // b * chunks + c
  int len;        // tokens of the sequence
  // CTAs for `count` chunks of a sequence, from chunk `from` on
  __device__ Where(const ttt_b200_scan_args& p, const Plan& q, int dc, int count, int from) {
    long i = blockIdx.x;
    tile = static_cast<int>(i % q.tiles);
    i /= q.tiles;
    g = static_cast<int>(i % p.G);
    i /= p.G;
    c = from + static_cast<int>(i % count);
    b = static_cast<int>(i / count);
    bc = static_cast<long>(b) * q.chunks + c;
    ch0 = g * q.per + tile * dc;
    cols = min(q.per - tile * dc, dc);
    len = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
  }
};

// `rows` x `cols` elements -> [kTile][W], the rest zeros.  `piece`: the bytes that all rows are aligned for, 16 or 4 (asynchronous
// copies; 4 x 2048 x 1535 x 16 in fp32, forward: 296 us one by one, 194 by fours) or less.
template <class T, int W> __device__ __forceinline__ void stage(T* dst, const T* src, int64_t stride, int rows, int cols, int piece) {
  if (piece == 16) {
    constexpr int PV = 16 / sizeof(T), PR = W / PV;
#pragma unroll
    for (int i0 = 0; i0 < kTile * PR; i0 += TH) {
      const int i = i0 + threadIdx.x;
      if (kTile * PR % TH != 0 && i >= kTile * PR) break;
      const int t = i / PR, c = i % PR * PV;
      const int n = t < rows ? min(max(cols - c, 0), PV) : 0;
      cp_async16(dst + t * W + c, n > 0 ? src + t * stride + c : src, n * static_cast<int>(sizeof(T)));
    }
  } else if (piece == 4) {
    constexpr int PV = 4 / sizeof(T), PR = W / PV;
    const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
#pragma unroll 4
    for (int i = threadIdx.x; i < kTile * PR; i += TH) {
      const int t = i / PR, c = i % PR * PV;
      const int n = t < rows ? min(max(cols - c, 0), PV) : 0;
      cp_async4_at(to + 4 * i, n > 0 ? src + t * stride + c : src, n * static_cast<int>(sizeof(T)));
    }
  } else {
#pragma unroll 8
    for (int i = threadIdx.x; i < kTile * W; i += TH) {
      const int t = i / W, c = i % W;
      dst[i] = t < rows && c < cols ? src[t * stride + c] : from_f32<T>(0.f);
    }
  }
}

// delta of two values, and its derivative.  log1p(e) of e = exp(-|v|) in (0, 1] as 2 atanh(s), s = e / (2 + e), whose series in
// s^2 <= 1/9 is cut where its next term is 2e-8 of the value; log(1 + e) itself would lose the small steps that matter most.
__device__ __forceinline__ float2 softplus2(float2 v, float2* slope = nullptr) {
  const float2 e = make_float2(ex2(-fabsf(v.x) * kLog2e), ex2(-fabsf(v.y) * kLog2e));
  const float2 d = add2(e, both(2.f)), s = mul2(e, make_float2(rcp(d.x), rcp(d.y))), q = mul2(s, s);
  float2 r = fma2(q, both(1.f / 13), both(1.f / 11));
  r = fma2(q, r, both(1.f / 9));
  r = fma2(q, r, both(1.f / 7));
  r = fma2(q, r, both(1.f / 5));
  r = fma2(q, r, both(1.f / 3));
  r = fma2(q, r, both(1.f));
  if (slope) {
    const float2 o = add2(e, both(1.f));
    *slope = mul2(make_float2(v.x >= 0.f ? 1.f : e.x, v.y >= 0.f ? 1.f : e.y), make_float2(rcp(o.x), rcp(o.y)));
  }
  return fma2(add2(s, s), r, make_float2(fmaxf(v.x, 0.f), fmaxf(v.y, 0.f)));
}

// a or b, both worked out: a branch would keep the arithmetic in front of it from filling the gaps of the walk
__device__ __forceinline__ float2 choose(bool first, float2 a, float2 b) {
  float2 r;
  asm("{ .reg .pred q; setp.ne.s32 q, %6, 0; selp.f32 %0, %2, %4, q; selp.f32 %1, %3, %5, q; }"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "r"(static_cast<int>(first)));
  return r;
}

// two neighbouring elements in shared memory
template <class T> __device__ __forceinline__ float2 pair(const T* p) {
  if constexpr (sizeof(T) == 4) {
    return *reinterpret_cast<const float2*>(p);
  } else if constexpr (std::is_same<T, __half>::value) {
    return __half22float2(*reinterpret_cast<const __half2*>(p));
  } else {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p));
  }
}
// two neighbouring values of a row of an output: together where the host has found all its rows aligned for it
template <class T> __device__ __forceinline__ void put_pair(T* p, float2 v, bool together, bool first, bool second) {
  if (together) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(p) = v;
    else if constexpr (std::is_same<T, __half>::value) *reinterpret_cast<__half2*>(p) = __floats2half2_rn(v.x, v.y);
    else *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(v.x, v.y);
  } else {
    if (first) p[0] = from_f32<T>(v.x);
    if (second) p[1] = from_f32<T>(v.y);
  }
}
// A thread's share of a tile [kTile][W] of B or C, on its way to fp32.
template <class T, int W> struct Wide {
  static constexpr int kPairs = kTile * W / 2, kMine = (kPairs + TH - 1) / TH;
  float2 v[kMine];
  __device__ __forceinline__ void load(const T* src) {
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      const int i = k * TH + threadIdx.x;
      if (kPairs % TH == 0 || i < kPairs) v[k] = pair(src + 2 * i);
    }
  }
  __device__ __forceinline__ void store(float* dst) const {
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      const int i = k * TH + threadIdx.x;
      if (kPairs % TH == 0 || i < kPairs) *reinterpret_cast<float2*>(dst + 2 * i) = v[k];
    }
  }
};

// exp(delta A) of a pair of states, a2 = A log2(e).  The approximate exponential is 2e-8 low on average for the slow decays
// (arguments of -0.5 to -0.001), which a state of a thousand tokens adds up; the offset takes the average to a quarter of
// that and leaves exp(0) = 1, which tokens behind a sequence rely on.
constexpr float kCentre = 2.2e-8f;
// A log2(e), a number for every A that is one: the lowest would be infinite, and a delta of zero times it no number.
__device__ __forceinline__ float rate(float a) {
  const float r = a * kLog2e;
  return isinf(r) ? copysignf(3.402823466e38f, r) : r;
}
__device__ __forceinline__ float2 decay(float delta, float2 a2) {
  const float2 x = fma2(both(delta), a2, both(kCentre));
  return make_float2(ex2(x.x), ex2(x.y));
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

// A thread's two channels and four states.
template <int LN> struct Mine {
  int li, dl, n0, ch[2];
  long row[2];
  __device__ __forceinline__ Mine(const Where& w, int N) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    li = lane % LN;
    dl = lane / LN;
    n0 = 4 * li;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      ch[e] = (2 * warp + e) * Shape<LN>::CPW + dl;
      row[e] = static_cast<long>(w.ch0 + ch[e]) * N;
    }
  }
  // of a row [D][N]; a channel behind the last reads nothing
  template <bool kRate = false> __device__ __forceinline__ void read(const float* p, const Where& w, int N, bool vec, float2 (&h)[2][2]) const {
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (ch[e] < w.cols) {
        float v[4];
        load_states(p + row[e], n0, N, vec, v);
        if constexpr (kRate) {
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = rate(v[k]);
        }
        h[e][0] = make_float2(v[0], v[1]);
        h[e][1] = make_float2(v[2], v[3]);
      }
  }
  __device__ __forceinline__ void write(float* p, const Where& w, int N, bool vec, const float2 (&h)[2][2]) const {
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (ch[e] < w.cols) {
        const float v[4] = {h[e][0].x, h[e][0].y, h[e][1].x, h[e][1].y};
        store_states(p + row[e], n0, N, vec, v);
      }
  }
};

// Where elements are worked on one by one a thread has two neighbouring channels, the same in every row.
template <int DC> struct Pair {
  int c, t0;      // channel; first row, the next ones kStep further
  static constexpr int kStep = 2 * TH / DC, kRows = kTile / kStep;
  bool first, second, together;
  float2 bias, skip;
  __device__ __forceinline__ Pair(const ttt_b200_scan_args& p, const Plan& q, const Where& w) {
    c = threadIdx.x % (DC / 2) * 2;
    t0 = threadIdx.x / (DC / 2);
    first = c < w.cols;
    second = c + 1 < w.cols;
    together = second && q.pairs && w.ch0 % 2 == 0;
    bias = skip = both(0.f);
    if (p.dt_bias) bias = make_float2(first ? p.dt_bias[w.ch0 + c] : 0.f, second ? p.dt_bias[w.ch0 + c + 1] : 0.f);
    if (p.Dskip) skip = make_float2(first ? p.Dskip[w.ch0 + c] : 0.f, second ? p.Dskip[w.ch0 + c + 1] : 0.f);
  }
};

// ---- forward ---------------------------------------------------------------------------------------------------------
template <class T, int LN> struct FwdSmem {
  using S = Shape<LN>;
  static constexpr int YW = S::DC + S::CPW;      // the y of a warp's channels and LN tokens in different banks
  alignas(16) T x[2][kTile * S::DC];
  alignas(16) T dt[2][kTile * S::DC];
  alignas(16) T b[2][kTile * S::NP];
  alignas(16) T c[2][kTile * S::NP];
  alignas(16) float2 u[2][kTile * S::DC];      // delta, delta x
  alignas(16) float fb[2][kTile * S::NP];
  alignas(16) float fc[2][kTile * S::NP];
  alignas(16) float y[2][kTile * YW];          // D x, then y
};

// Four CTAs to an SM, here and in the state kernel, against three, whose 168 registers hold nearly all that 128 spill (us, forward kernel / state
// kernel): 4 x 2048 x 1536 x 16 in 24 chunks 93 / 67 against 105 / 68, 2 x 1000 x 768 x 64 48 / 31 against 53 / 34; but 8 states in fp32 98 / 54 against
// 85 / 50, and 8 x 2048 x 2048 x 16, which is not split, 307 against 299.
//
// One barrier to a tile: between two of them the states walk over tile k, tile k + 1 goes from its copy to fp32 (in registers
// first, so that its arithmetic fills the gaps of the walk), tile k - 1 leaves, and the copy of tile k + 2 is on its way.
template <class T, int LN> __global__ void __launch_bounds__(TH, 4) scan_forward_kernel(const ttt_b200_scan_args p, const Plan q) {
  wait_for_predecessor();
  using S = Shape<LN>;
  constexpr int DC = S::DC, NP = S::NP, U = LN < 4 ? 4 : LN, YW = FwdSmem<T, LN>::YW;
  extern __shared__ __align__(16) unsigned char raw[];
  FwdSmem<T, LN>& m = *reinterpret_cast<FwdSmem<T, LN>*>(raw);
  const Where w(p, q, DC, q.chunks, 0);
  const Mine<LN> me(w, p.N);
  const Pair<DC> el(p, q, w);
  const int lane = threadIdx.x & 31;
  const long DN = static_cast<long>(p.D) * p.N;

  const int begin = w.c * q.chunk, end = min(begin + q.chunk, p.T), stop = min(end, w.len);
  const int count = stop > begin ? (stop - begin + kTile - 1) / kTile : 0;
  const T* xs = static_cast<const T*>(p.x) + w.b * p.x_stride[0] + w.ch0;
  const T* ds = static_cast<const T*>(p.dt) + w.b * p.dt_stride[0] + w.ch0;
  const T* bs = static_cast<const T*>(p.Bm) + w.b * p.B_stride[0] + w.g * p.B_stride[2];
  const T* cs = static_cast<const T*>(p.Cm) + w.b * p.C_stride[0] + w.g * p.C_stride[2];
  T* ys = static_cast<T*>(p.y) + static_cast<long>(w.b) * p.T * p.D + w.ch0 + el.c;
  auto fetch = [&](int k) {
    if (k < count) {
      const int t0 = begin + k * kTile, rows = min(stop - t0, kTile), buf = k & 1;
      stage<T, DC>(m.x[buf], xs + t0 * p.x_stride[1], p.x_stride[1], rows, w.cols, q.vec_x);
      stage<T, DC>(m.dt[buf], ds + t0 * p.dt_stride[1], p.dt_stride[1], rows, w.cols, q.vec_dt);
      stage<T, NP>(m.b[buf], bs + t0 * p.B_stride[1], p.B_stride[1], rows, p.N, q.vec_b);
      stage<T, NP>(m.c[buf], cs + t0 * p.C_stride[1], p.C_stride[1], rows, p.N, q.vec_c);
    }
    cp_async_commit();
  };
  auto leave = [&](int k) {      // the y of a tile, with zeros behind the sequence
#pragma unroll
    for (int i = 0; i < el.kRows; ++i) {
      const int r = el.t0 + i * el.kStep, t = begin + k * kTile + r;
      if (t < end)
        put_pair(ys + static_cast<long>(t) * p.D, t < stop ? *reinterpret_cast<const float2*>(m.y[k & 1] + r * YW + el.c) : both(0.f),
                 el.together, el.first, el.second);
    }
  };
  struct Next {      // a tile on its way to fp32
    float2 x[Pair<DC>::kRows], dt[Pair<DC>::kRows];
    Wide<T, NP> b, c;
  };
  auto pick_up = [&](int k, Next& n) {
    const int buf = k & 1;
#pragma unroll
    for (int i = 0; i < el.kRows; ++i) {
      const int at = (el.t0 + i * el.kStep) * DC + el.c;
      n.x[i] = pair(m.x[buf] + at);
      n.dt[i] = pair(m.dt[buf] + at);
    }
    n.b.load(m.b[buf]);
    n.c.load(m.c[buf]);
  };
  auto work_out = [&](int k, Next& n) {
    const int rows = stop - (begin + k * kTile);
#pragma unroll
    for (int i = 0; i < el.kRows; ++i) {
      const float2 v = add2(n.dt[i], el.bias);
      n.dt[i] = choose(p.softplus, softplus2(v), v);
      n.dt[i] = choose(el.t0 + i * el.kStep < rows, n.dt[i], both(0.f));
    }
  };
  auto put_down = [&](int k, const Next& n) {
    const int buf = k & 1;
#pragma unroll
    for (int i = 0; i < el.kRows; ++i) {
      const int r = el.t0 + i * el.kStep;
      const float2 dx = mul2(n.dt[i], n.x[i]);
      *reinterpret_cast<float4*>(m.u[buf] + r * DC + el.c) = make_float4(n.dt[i].x, dx.x, n.dt[i].y, dx.y);
      *reinterpret_cast<float2*>(m.y[buf] + r * YW + el.c) = mul2(el.skip, n.x[i]);
    }
    n.b.store(m.fb[buf]);
    n.c.store(m.fc[buf]);
  };

  fetch(0);
  float2 a2[2][2] = {}, h[2][2] = {};
  me.template read<true>(p.A, w, p.N, q.vec_n, a2);
  if (q.chunks > 1) me.read(q.state + w.bc * DN, w, p.N, q.vec_n, h);
  else if (p.state) me.read(p.state + w.b * DN, w, p.N, q.vec_n, h);
  Next next;
  cp_async_wait<0>();
  __syncthreads();
  fetch(1);
  if (count > 0) {
    pick_up(0, next);
    work_out(0, next);
    put_down(0, next);
  }
  for (int k = 0; k < count; ++k) {
    cp_async_wait<0>();
    __syncthreads();      // tile k + 1 has landed, tile k is ready, and no thread is behind
    fetch(k + 2);
    if (k > 0) leave(k - 1);
    if (p.checkpoints) me.write(p.checkpoints + (static_cast<long>(w.b) * q.nck + begin / kTile + k) * DN, w, p.N, q.vec_n, h);
    pick_up(k + 1, next);      // (behind the last tile: what is there, for nothing)
    work_out(k + 1, next);
    const float2* u = m.u[k & 1];
    const float *fb = m.fb[k & 1] + me.n0, *fc = m.fc[k & 1] + me.n0;
    float* y = m.y[k & 1];
#pragma unroll
    for (int s = 0; s < kTile; s += U) {
      float acc[2][U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int t = s + i;
        float2 b[2], c[2];
        split(*reinterpret_cast<const float4*>(fb + t * NP), b);
        split(*reinterpret_cast<const float4*>(fc + t * NP), c);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 du = u[t * DC + me.ch[e]];
          float2 o;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            h[e][j] = fma2(decay(du.x, a2[e][j]), h[e][j], mul2(both(du.y), b[j]));
            o = j ? fma2(h[e][j], c[j], o) : mul2(h[e][j], c[j]);
          }
          acc[e][i] = o.x + o.y;
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        spread_sum<U, LN, 1>(acc[e], lane);
#pragma unroll
        for (int i = 0; i < U / LN; ++i) y[(s + me.li * (U / LN) + i) * YW + me.ch[e]] += acc[e][i];
      }
    }
    put_down(k + 1, next);
  }
  __syncthreads();
  if (count > 0) leave(count - 1);
  for (int k = count; begin + k * kTile < end; ++k) leave(k);
  if (p.final_state && w.c == q.chunks - 1) me.write(p.final_state + w.b * DN, w, p.N, q.vec_n, h);
}

// ---- a chunk's state by itself, from zero: forwards h <- a h + delta x B; backwards (kRev) c <- a (c + dy C) -----------
// Not that of the last chunk in the direction of the walk, which none starts from.
template <class T, int LN> struct StateSmem {
  using S = Shape<LN>;
  alignas(16) T v[2][kTile * S::DC];      // x or dy
  alignas(16) T dt[2][kTile * S::DC];
  alignas(16) T n[2][kTile * S::NP];      // B or C
  alignas(16) float2 u[2][kTile * S::DC];
  alignas(16) float fn[2][kTile * S::NP];
};

template <class T, int LN, bool kRev> __global__ void __launch_bounds__(TH, 4) scan_state_kernel(const ttt_b200_scan_args p, const Plan q) {
  wait_for_predecessor();
  using S = Shape<LN>;
  constexpr int DC = S::DC, NP = S::NP;
  extern __shared__ __align__(16) unsigned char raw[];
  StateSmem<T, LN>& m = *reinterpret_cast<StateSmem<T, LN>*>(raw);
  const Where w(p, q, DC, q.chunks - 1, kRev ? 1 : 0);
  const Mine<LN> me(w, p.N);
  const Pair<DC> el(p, q, w);
  const long DN = static_cast<long>(p.D) * p.N;
  const int64_t* vst = kRev ? p.gy_stride : p.x_stride;
  const int64_t* nst = kRev ? p.C_stride : p.B_stride;
  const T* vs = static_cast<const T*>(kRev ? p.grad_y : p.x) + w.b * vst[0] + w.ch0;
  const T* ds = static_cast<const T*>(p.dt) + w.b * p.dt_stride[0] + w.ch0;
  const T* ns = static_cast<const T*>(kRev ? p.Cm : p.Bm) + w.b * nst[0] + w.g * nst[2];
  const int begin = w.c * q.chunk, end = min(begin + q.chunk, w.len);
  const int count = end > begin ? (end - begin + kTile - 1) / kTile : 0;
  auto at = [&](int k) { return begin + (kRev ? count - 1 - k : k) * kTile; };
  auto fetch = [&](int k) {
    if (k < count) {
      const int t0 = at(k), rows = min(end - t0, kTile), buf = k & 1;
      stage<T, DC>(m.v[buf], vs + t0 * vst[1], vst[1], rows, w.cols, kRev ? q.vec_gy : q.vec_x);
      stage<T, DC>(m.dt[buf], ds + t0 * p.dt_stride[1], p.dt_stride[1], rows, w.cols, q.vec_dt);
      stage<T, NP>(m.n[buf], ns + t0 * nst[1], nst[1], rows, p.N, kRev ? q.vec_c : q.vec_b);
    }
    cp_async_commit();
  };
  struct Next {
    float2 v[Pair<DC>::kRows], dt[Pair<DC>::kRows];
    Wide<T, NP> n;
  };
  auto pick_up = [&](int k, Next& n) {
    const int buf = k & 1;
#pragma unroll
    for (int i = 0; i < el.kRows; ++i) {
      const int o = (el.t0 + i * el.kStep) * DC + el.c;
      n.v[i] = pair(m.v[buf] + o);
      n.dt[i] = pair(m.dt[buf] + o);
    }
    n.n.load(m.n[buf]);
  };
  auto work_out = [&](int k, Next& n) {
    const int rows = end - at(k);
#pragma unroll
    for (int i = 0; i < el.kRows; ++i) {
      const float2 v = add2(n.dt[i], el.bias);
      n.dt[i] = choose(p.softplus, softplus2(v), v);
      n.dt[i] = choose(el.t0 + i * el.kStep < rows, n.dt[i], both(0.f));
      if (!kRev) n.v[i] = mul2(n.dt[i], n.v[i]);
    }
  };
  auto put_down = [&](int k, const Next& n) {
    const int buf = k & 1;
#pragma unroll
    for (int i = 0; i < el.kRows; ++i)
      *reinterpret_cast<float4*>(m.u[buf] + (el.t0 + i * el.kStep) * DC + el.c) = make_float4(n.dt[i].x, n.v[i].x, n.dt[i].y, n.v[i].y);
    n.n.store(m.fn[buf]);
  };

  fetch(0);
  float2 a2[2][2] = {}, h[2][2] = {};
  me.template read<true>(p.A, w, p.N, q.vec_n, a2);
  float2 total = both(0.f);
  Next next;
  cp_async_wait<0>();
  __syncthreads();
  fetch(1);
  if (count > 0) {
    pick_up(0, next);
    work_out(0, next);
    put_down(0, next);
  }
  for (int k = 0; k < count; ++k) {
    cp_async_wait<0>();
    __syncthreads();
    fetch(k + 2);
    pick_up(k + 1, next);      // (behind the last tile: what is there, for nothing)
    work_out(k + 1, next);
    const float2* u = m.u[k & 1];
    const float* fn = m.fn[k & 1] + me.n0;
#pragma unroll
    for (int s = 0; s < kTile; ++s) {
      const int t = kRev ? kTile - 1 - s : s;
      float2 b[2];
      split(*reinterpret_cast<const float4*>(fn + t * NP), b);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 du = u[t * DC + me.ch[e]];
        (e ? total.y : total.x) += du.x;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float2 f = decay(du.x, a2[e][j]);
          h[e][j] = kRev ? mul2(f, fma2(both(du.y), b[j], h[e][j])) : fma2(f, h[e][j], mul2(both(du.y), b[j]));
        }
      }
    }
    put_down(k + 1, next);
  }
  me.write(q.state + w.bc * DN, w, p.N, q.vec_n, h);
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (me.li == 0 && me.ch[e] < w.cols) q.delta[w.bc * p.D + w.ch0 + me.ch[e]] = e ? total.y : total.x;
}

// 2^x h for x > kStep, h a state that a chunk's decay carries on.  A state that grows (A delta > 0) may do so by more than fp32 holds over a
// chunk and still be a number, if it is zero or small, so the exponent is taken in steps: three take the least number beyond the greatest.
constexpr float kStep = 126.f;
__device__ __forceinline__ float grown(float x, float h) {
#pragma unroll
  for (int i = 0; i < 3; ++i, x -= kStep) h *= ex2(fminf(fmaxf(x, 0.f), kStep));
  return h;
}

// The chunks' own states -> the states that they start from (kRev: that they end with), in place, in the order of time.
template <bool kRev> __global__ void __launch_bounds__(256) scan_join_kernel(const ttt_b200_scan_args p, const Plan q) {
  wait_for_predecessor();
  const long DN = static_cast<long>(p.D) * p.N;
  const long i = static_cast<long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= p.B * DN) return;
  const long b = i / DN, dn = i % DN, d = dn / p.N;
  const float a2 = rate(p.A[dn]);
  const float* from = kRev ? p.grad_final_state : p.state;
  float h = from ? from[i] : 0.f;
  constexpr int kAhead = 8;      // chunks requested ahead of those that are worked on
  auto chunk = [&](int c) { return b * q.chunks + (kRev ? q.chunks - 1 - c : c); };
  float s[kAhead], f[kAhead], e[kAhead], s2[kAhead], f2[kAhead];
  auto request = [&](int c0) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const long c = chunk(min(c0 + k, q.chunks - 2));      // (the last one's own state is not there and not needed)
      s2[k] = q.state[c * DN + dn];
      f2[k] = q.delta[c * p.D + d];
    }
  };
  request(0);
  for (int c0 = 0; c0 < q.chunks; c0 += kAhead) {
    bool grows = false;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      s[k] = s2[k];
      e[k] = fmaf(a2, f2[k], kCentre);
      f[k] = ex2(e[k]);
      grows = grows || e[k] > kStep;
    }
    request(c0 + kAhead);
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (c0 + k < q.chunks) {
        q.state[chunk(c0 + k) * DN + dn] = h;
        h = grows && e[k] > kStep ? grown(e[k], h) + s[k] : fmaf(f[k], h, s[k]);
      }
  }
}

// ---- backward --------------------------------------------------------------------------------------------------------
constexpr int kSub = 4;      // tokens whose states and factors are in registers at a time

template <class T, int LN> struct BwdSmem {
  using S = Shape<LN>;
  alignas(16) T x[2][kTile * S::DC];
  alignas(16) T dt[2][kTile * S::DC];
  alignas(16) T gy[2][kTile * S::DC];
  alignas(16) T b[2][kTile * S::NP];
  alignas(16) T c[2][kTile * S::NP];
  alignas(16) float4 u[kTile * S::DC];      // delta, delta x, dy, d delta / d dt; then sum_n dh A exp(delta A) h (in base 2) and
                                            // sum_n dh B in the place of delta x and dy, which only the warp of the channel reads
  alignas(16) float fb[kTile * S::NP];
  alignas(16) float fc[kTile * S::NP];
  alignas(16) float4 start[kTile / kSub - 1][2][TH];      // each thread's states at the starts of the later runs of kSub tokens
  alignas(16) float bc[kTile][TH / 32][2 * S::NP];     // each warp's part of dB and dC
};

// With up to 16 states the factors exp(delta A) are worked out once more on the way back instead of kept, and four CTAs fit an SM
// instead of three (4 x 2048 x 1536 x 16: 348 -> 332 us); with 64 the exponentials cost more than that gives (191 -> 208).
template <class T, int LN>
__global__ void __launch_bounds__(TH, LN <= 4 ? 4 : 3) scan_backward_kernel(const ttt_b200_scan_args p, const Plan q) {
  wait_for_predecessor();
  constexpr bool kKeep = LN > 4;
  using S = Shape<LN>;
  constexpr int DC = S::DC, NP = S::NP, ND = 32 / LN;
  extern __shared__ __align__(16) unsigned char raw[];
  BwdSmem<T, LN>& m = *reinterpret_cast<BwdSmem<T, LN>*>(raw);
  const Where w(p, q, DC, q.chunks, 0);
  const Mine<LN> me(w, p.N);
  const Pair<DC> el(p, q, w);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long DN = static_cast<long>(p.D) * p.N;
  float2 a2[2][2] = {}, carry[2][2] = {}, da[2][2] = {};
  me.template read<true>(p.A, w, p.N, q.vec_n, a2);
  if (q.chunks > 1) me.read(q.state + w.bc * DN, w, p.N, q.vec_n, carry);
  else if (p.grad_final_state) me.read(p.grad_final_state + w.b * DN, w, p.N, q.vec_n, carry);
  float2 sum_d = both(0.f), sum_bias = both(0.f);

  const int begin = w.c * q.chunk, end = min(begin + q.chunk, p.T);
  const T* xs = static_cast<const T*>(p.x) + w.b * p.x_stride[0] + w.ch0;
  const T* ds = static_cast<const T*>(p.dt) + w.b * p.dt_stride[0] + w.ch0;
  const T* gs = static_cast<const T*>(p.grad_y) + w.b * p.gy_stride[0] + w.ch0;
  const T* bs = static_cast<const T*>(p.Bm) + w.b * p.B_stride[0] + w.g * p.B_stride[2];
  const T* cs = static_cast<const T*>(p.Cm) + w.b * p.C_stride[0] + w.g * p.C_stride[2];
  const long out0 = static_cast<long>(w.b) * p.T * p.D + w.ch0 + el.c;
  T* gxs = static_cast<T*>(p.grad_x) + out0;
  T* gds = static_cast<T*>(p.grad_dt) + out0;
  const long GN = static_cast<long>(p.G) * p.N, BTGN = static_cast<long>(p.B) * p.T * GN;
  float* pb = q.part_bc + w.tile * BTGN + static_cast<long>(w.b) * p.T * GN + w.g * p.N;
  float* pc = pb + q.tiles * BTGN;
  T *tb = static_cast<T*>(p.grad_B) + static_cast<long>(w.b) * p.T * GN + w.g * p.N, *tc = static_cast<T*>(p.grad_C) + static_cast<long>(w.b) * p.T * GN + w.g * p.N;
  auto fetch = [&](int t0, int buf) {
    const int rows = min(w.len - t0, kTile);
    if (t0 >= begin && rows > 0) {
      stage<T, DC>(m.x[buf], xs + t0 * p.x_stride[1], p.x_stride[1], rows, w.cols, q.vec_x);
      stage<T, DC>(m.dt[buf], ds + t0 * p.dt_stride[1], p.dt_stride[1], rows, w.cols, q.vec_dt);
      stage<T, DC>(m.gy[buf], gs + t0 * p.gy_stride[1], p.gy_stride[1], rows, w.cols, q.vec_gy);
      stage<T, NP>(m.b[buf], bs + t0 * p.B_stride[1], p.B_stride[1], rows, p.N, q.vec_b);
      stage<T, NP>(m.c[buf], cs + t0 * p.C_stride[1], p.C_stride[1], rows, p.N, q.vec_c);
    }
    cp_async_commit();
  };

  const int last = begin + (end - begin - 1) / kTile * kTile;
  fetch(last, 0);
  int buf = 0;
  for (int t0 = last; t0 >= begin; t0 -= kTile, buf ^= 1) {
    const int rows = min(w.len - t0, kTile);
    if (rows <= 0) {      // behind the sequence: zeros, and the gradient of the state passes through
#pragma unroll
      for (int t = el.t0; t < kTile; t += el.kStep)
        if (t0 + t < end) {
          put_pair(gxs + static_cast<long>(t0 + t) * p.D, both(0.f), el.together, el.first, el.second);
          put_pair(gds + static_cast<long>(t0 + t) * p.D, both(0.f), el.together, el.first, el.second);
        }
      for (int i = threadIdx.x; i < kTile * NP; i += TH)
        if (t0 + i / NP < end && i % NP < p.N) {
          const long at = (t0 + i / NP) * GN + i % NP;
          if (q.tiles > 1) pb[at] = pc[at] = 0.f;
          else tb[at] = tc[at] = from_f32<T>(0.f);
        }
      fetch(t0 - kTile, buf ^ 1);
      continue;
    }
    float2 h0[2][2] = {};      // the state before the tile
    me.read(p.checkpoints + (static_cast<long>(w.b) * q.nck + t0 / kTile) * DN, w, p.N, q.vec_n, h0);
    cp_async_wait<0>();
    __syncthreads();      // the tile has landed, and no thread reads the other buffer any more
    fetch(t0 - kTile, buf ^ 1);
#pragma unroll
    for (int t = el.t0; t < kTile; t += el.kStep) {
      const float2 x = pair(m.x[buf] + t * DC + el.c), v = add2(pair(m.dt[buf] + t * DC + el.c), el.bias);
      const float2 gy = pair(m.gy[buf] + t * DC + el.c);
      float2 slope = both(1.f), d = p.softplus ? softplus2(v, &slope) : v;
      if (t >= rows) d = slope = both(0.f);
      const float2 dx = mul2(d, x);
      m.u[t * DC + el.c] = make_float4(d.x, dx.x, gy.x, slope.x);
      m.u[t * DC + el.c + 1] = make_float4(d.y, dx.y, gy.y, slope.y);
    }
    Wide<T, NP> wide;
    wide.load(m.b[buf]);
    wide.store(m.fb);
    wide.load(m.c[buf]);
    wide.store(m.fc);
    __syncthreads();
    {      // the states at the starts of the runs
      float2 h[2][2] = {{h0[0][0], h0[0][1]}, {h0[1][0], h0[1][1]}};
#pragma unroll 1
      for (int s = 0; s < kTile / kSub - 1; ++s) {
#pragma unroll
        for (int k = 0; k < kSub; ++k) {
          const int t = s * kSub + k;
          float2 b[2];
          split(*reinterpret_cast<const float4*>(m.fb + t * NP + me.n0), b);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 u = *reinterpret_cast<const float2*>(m.u + t * DC + me.ch[e]);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              h[e][j] = fma2(decay(u.x, a2[e][j]), h[e][j], mul2(both(u.y), b[j]));
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) m.start[s][e][threadIdx.x] = make_float4(h[e][0].x, h[e][0].y, h[e][1].x, h[e][1].y);
      }
    }
#pragma unroll 1
    for (int s = kTile / kSub - 1; s >= 0; --s) {
      float2 f[2][kKeep ? kSub : 1][2], h[2][kSub + 1][2];      // factors; states before token k of the run
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        h[e][0][0] = h0[e][0];
        h[e][0][1] = h0[e][1];
        if (s > 0) split(m.start[s - 1][e][threadIdx.x], h[e][0]);
      }
#pragma unroll
      for (int k = 0; k < kSub; ++k) {
        const int t = s * kSub + k;
        float2 b[2];
        split(*reinterpret_cast<const float4*>(m.fb + t * NP + me.n0), b);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 u = *reinterpret_cast<const float2*>(m.u + t * DC + me.ch[e]);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 r = decay(u.x, a2[e][j]);
            if constexpr (kKeep) f[e][k][j] = r;
            h[e][k + 1][j] = fma2(r, h[e][k][j], mul2(both(u.y), b[j]));
          }
        }
      }
#pragma unroll
      for (int k = kSub - 1; k >= 0; --k) {
        const int t = s * kSub + k;
        float2 b[2], c[2], vb[2], vc[2];
        split(*reinterpret_cast<const float4*>(m.fb + t * NP + me.n0), b);
        split(*reinterpret_cast<const float4*>(m.fc + t * NP + me.n0), c);
        float o[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 u = *reinterpret_cast<const float2*>(m.u + t * DC + me.ch[e]);
          const float gy = m.u[t * DC + me.ch[e]].z;
          float2 qa, gb;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 g = fma2(both(gy), c[j], carry[e][j]);
            vb[j] = e ? fma2(both(u.y), g, vb[j]) : mul2(both(u.y), g);
            vc[j] = e ? fma2(both(gy), h[e][k + 1][j], vc[j]) : mul2(both(gy), h[e][k + 1][j]);
            gb = j ? fma2(g, b[j], gb) : mul2(g, b[j]);
            carry[e][j] = mul2(kKeep ? f[e][kKeep ? k : 0][j] : decay(u.x, a2[e][j]), g);
            const float2 r = mul2(carry[e][j], h[e][k][j]);
            qa = j ? fma2(r, a2[e][j], qa) : mul2(r, a2[e][j]);
            da[e][j] = fma2(both(u.x), r, da[e][j]);
          }
          o[e] = qa.x + qa.y;
          o[2 + e] = gb.x + gb.y;
        }
        // dx and d delta: over the channel's lanes, which have all read the token's delta x and dy when one of them overwrites these
        spread_sum<4, LN, 1>(o, lane);
        __syncwarp();
        if constexpr (LN <= 4) {
#pragma unroll
          for (int r = 0; r < 4 / LN; ++r) {
            const int i = me.li * (4 / LN) + r;
            reinterpret_cast<float*>(m.u + t * DC + (i & 1 ? me.ch[1] : me.ch[0]))[1 + (i >> 1)] = o[r];
          }
        } else {
          const int i = me.li / (LN / 4);
          if (me.li % (LN / 4) == 0) reinterpret_cast<float*>(m.u + t * DC + (i & 1 ? me.ch[1] : me.ch[0]))[1 + (i >> 1)] = o[0];
        }
        // dB and dC: over the warp's channels
        float v[8] = {vb[0].x, vb[0].y, vb[1].x, vb[1].y, vc[0].x, vc[0].y, vc[1].x, vc[1].y};
        spread_sum<8, ND, LN>(v, lane);
        if constexpr (ND <= 8) {
#pragma unroll
          for (int r = 0; r < 8 / ND; ++r) {
            const int i = me.dl * (8 / ND) + r;
            m.bc[t][warp][(i >> 2) * NP + me.n0 + (i & 3)] = v[r];
          }
        } else {
          const int i = me.dl / (ND / 8);
          if (me.dl % (ND / 8) == 0) m.bc[t][warp][(i >> 2) * NP + me.n0 + (i & 3)] = v[0];
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int t = el.t0; t < kTile; t += el.kStep) {
      if (t0 + t >= end) break;
      const float4 u0 = m.u[t * DC + el.c], u1 = m.u[t * DC + el.c + 1];
      const float2 d = make_float2(u0.x, u1.x), slope = make_float2(u0.w, u1.w), qa = make_float2(u0.y, u1.y), gb = make_float2(u0.z, u1.z);
      const float2 x = pair(m.x[buf] + t * DC + el.c), gy = pair(m.gy[buf] + t * DC + el.c);
      const float2 gx = fma2(d, gb, mul2(el.skip, gy)), gd = mul2(slope, fma2(both(kLn2), qa, mul2(x, gb)));
      const bool in = t < rows;
      put_pair(gxs + static_cast<long>(t0 + t) * p.D, in ? gx : both(0.f), el.together, el.first, el.second);
      put_pair(gds + static_cast<long>(t0 + t) * p.D, in ? gd : both(0.f), el.together, el.first, el.second);
      if (in) {
        sum_d = fma2(gy, x, sum_d);
        sum_bias = add2(sum_bias, gd);
      }
    }
    for (int i = threadIdx.x; i < kTile * NP / 2; i += TH) {      // four values of dB or dC, over the warps
      const int t = i / (NP / 2), k = i % (NP / 2) * 4, n = k % NP;
      if (t0 + t >= end || n >= p.N) continue;
      float v[4] = {};
      if (t < rows) {
#pragma unroll
        for (int r = 0; r < TH / 32; ++r) {
          const float4 o = *reinterpret_cast<const float4*>(&m.bc[t][r][k]);
          v[0] += o.x, v[1] += o.y, v[2] += o.z, v[3] += o.w;
        }
      }
      if (q.tiles > 1) {
        store_states((k < NP ? pb : pc) + (t0 + t) * GN, n, p.N, q.vec_part, v);
      } else {      // all of the group's channels are here
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (n + r < p.N) (k < NP ? tb : tc)[(t0 + t) * GN + n + r] = from_f32<T>(v[r]);
      }
    }
  }
  me.write(q.part_a + w.bc * DN, w, p.N, q.vec_n, da);
  if (w.c == 0 && p.grad_state) me.write(p.grad_state + w.b * DN, w, p.N, q.vec_n, carry);
  __syncthreads();
  float2* red = reinterpret_cast<float2*>(m.u);      // [2][TH]: what the threads of a pair of channels have summed
  red[threadIdx.x] = sum_d;
  red[TH + threadIdx.x] = sum_bias;
  __syncthreads();
  if (threadIdx.x < DC / 2) {
    for (int r = threadIdx.x + DC / 2; r < TH; r += DC / 2) {
      sum_d = add2(sum_d, red[r]);
      sum_bias = add2(sum_bias, red[TH + r]);
    }
    const long BCD = static_cast<long>(p.B) * q.chunks * p.D;
    float* to = q.part_d + w.bc * p.D + w.ch0 + el.c;
    put_pair(to, sum_d, el.together, el.first, el.second);
    put_pair(to + BCD, sum_bias, el.together, el.first, el.second);
  }
}

// ---- one token ---------------------------------------------------------------------------------------------------------
// A row of the batch and up to 256 / LN channels to a CTA, two per thread, each state read and written once.  What does not depend on
// the slot is requested in front of it, and the state in front of the search for rows that share it: two round trips to memory in all.
// Rows that name the same slot are taken in their order by the CTA of the first of them, so that no two CTAs touch a state.
// kOne: a CTA's channels are of one group, whose B and C are then read once, and eight CTAs fit an SM instead of six (64 rows of
// 2048 x 16: 7.3 -> 6.1 us with the states in the L2, 7.1 from memory; 64 of 4096 x 64: 47 -> 38 us, which is 3.6 TB/s; ten or twelve CTAs, with
// registers spilled, are no faster).
template <class T, int LN, bool kOne> __global__ void __launch_bounds__(TH, 8) scan_step_kernel(const ttt_b200_scan_args p, bool vec_n, int tiles) {
  wait_for_predecessor();
  constexpr int DC = TH / LN;
  const int b0 = blockIdx.x / tiles, li = threadIdx.x % LN, n0 = 4 * li;
  int d[2];
  bool live[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    d[e] = (blockIdx.x % tiles * 2 + e) * DC + threadIdx.x / LN;
    live[e] = d[e] < p.D;
    if (!live[e]) d[e] = 0;      // (reads there, writes nothing)
  }
  T* ys = static_cast<T*>(p.y);
  const int per = p.D / p.G;
  struct Token {
    float x[2], dt[2], b[kOne ? 1 : 2][4], c[kOne ? 1 : 2][4];
  };
  auto read = [&](int b, Token& t) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      t.x[e] = to_f32(static_cast<const T*>(p.x)[b * p.x_stride[0] + d[e]]);
      t.dt[e] = to_f32(static_cast<const T*>(p.dt)[b * p.dt_stride[0] + d[e]]);
      if (kOne && e) continue;
      const int g = p.G > 1 ? (kOne ? static_cast<int>(blockIdx.x % tiles) * 2 * DC : d[e]) / per : 0;
      const T* bs = static_cast<const T*>(p.Bm) + b * p.B_stride[0] + g * p.B_stride[2] + n0;
      const T* cs = static_cast<const T*>(p.Cm) + b * p.C_stride[0] + g * p.C_stride[2] + n0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        t.b[e][k] = n0 + k < p.N ? to_f32(bs[k]) : 0.f;
        t.c[e][k] = n0 + k < p.N ? to_f32(cs[k]) : 0.f;
      }
    }
  };
  int slot = p.slots ? p.slots[b0] : b0, more = 0;
  Token t;
  read(b0, t);
  float a[2][4], bias[2], skip[2], h[2][4];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    load_states(p.A + static_cast<long>(d[e]) * p.N, n0, p.N, vec_n, a[e]);
    bias[e] = p.dt_bias ? p.dt_bias[d[e]] : 0.f;
    skip[e] = p.Dskip ? p.Dskip[d[e]] : 0.f;
  }
  if (p.slots && (slot < 0 || slot >= p.rows)) {
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (live[e] && li == 0) ys[static_cast<long>(b0) * p.D + d[e]] = from_f32<T>(0.f);
    return;
  }
  float* st = p.state_io + static_cast<long>(slot) * p.D * p.N;
#pragma unroll
  for (int e = 0; e < 2; ++e) load_states(st + static_cast<long>(d[e]) * p.N, n0, p.N, vec_n, h[e]);
  if (p.slots) {
    int found = 0;      // 1: in a row before, 2: in one behind
    for (int r = threadIdx.x; r < p.B; r += TH)
      if (r != b0 && p.slots[r] == slot) found |= r < b0 ? 1 : 2;
    if (__syncthreads_or(found)) {      // (rarely: which of the two)
      if (__syncthreads_or(found & 1)) return;
      more = 1;
    }
  }
  for (int b = b0;;) {
    float y[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float v = t.dt[e] + bias[e], dl = p.softplus ? softplus2(both(v)).x : v, dx = dl * t.x[e];
      y[e] = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        h[e][k] = fmaf(ex2(fmaf(dl, rate(a[e][k]), kCentre)), h[e][k], dx * t.b[kOne ? 0 : e][k]);
        y[e] = fmaf(h[e][k], t.c[kOne ? 0 : e][k], y[e]);
      }
    }
#pragma unroll
    for (int o = LN / 2; o > 0; o >>= 1) {
      y[0] += __shfl_xor_sync(0xffffffffu, y[0], o);
      y[1] += __shfl_xor_sync(0xffffffffu, y[1], o);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (live[e] && li == 0) ys[static_cast<long>(b) * p.D + d[e]] = from_f32<T>(fmaf(skip[e], t.x[e], y[e]));
    if (!more) break;
    do ++b;
    while (b < p.B && p.slots[b] != slot);
    if (b >= p.B) break;
    read(b, t);
  }
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (live[e]) store_states(st + static_cast<long>(d[e]) * p.N, n0, p.N, vec_n, h[e]);
}

// ---- host --------------------------------------------------------------------------------------------------------------
int lanes_of(int N) { return N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

int check(const ttt_b200_scan_args* p) {
  if (!p) return fail("ssm scan: NULL argument struct");
  if (p->B < 0 || p->T < 0 || p->T > 1 << 30 || p->D < 1 || p->D > 1 << 30 || p->G < 1 || p->N < 1 || p->N > 64)
    return fail("ssm scan: B, T >= 0, D, G >= 1, T and D at most 2^30, and 1 to 64 states");
  if (p->D % p->G) return fail("ssm scan: the groups must divide the channels");
  if (p->dtype < TTT_B200_BF16 || p->dtype > TTT_B200_FP32) return fail("ssm scan: unknown element type");
  return TTT_B200_OK;
}

// Tokens to a chunk.  Without chunks the kernels need an SM's worth of CTAs next to each other to cover their latencies; with them
// every token's exponentials are worked out once more, by the state kernel.  Measured at 2048 tokens of N = 16, us without / with
// chunks: forward of 96 CTAs 244 / 160, of 256 282 / 374; backward of 96 CTAs 680 / 332, of 256 928 / 799, of 384 1160 / 1390.  So the
// forward is split below one CTA to an SM, the backward below two: into six to sixteen CTAs to an SM, of these the count that leaves
// the fullest SM least to do (96 CTAs of 128 tiles, backward with 12, 13, 16, 24 chunks: 333, 354, 332, 330), and where there are not
// that many tiles into single ones (512 tokens of 256 channels: 62 -> 20).  At most 128, which the joining kernel walks over.
void plan_chunks(Plan& q, const ttt_b200_scan_args& p, bool backward) {
  const int dc = TH / lanes_of(p.N) * 2;
  q.per = p.D / p.G;
  q.tiles = (q.per + dc - 1) / dc;
  q.nck = (p.T + kTile - 1) / kTile;
  const long ctas = static_cast<long>(p.B) * p.G * q.tiles, sms = sm_count();
  int per = std::max(q.nck, 1);      // tiles of a chunk
  if (ctas < (backward ? 2 : 1) * sms && q.nck > 1) {
    const int least = (q.nck + 127) / 128;
    per = least;
    long best = 0;
    for (int t = least; t <= q.nck; ++t) {
      const long all = ctas * ((q.nck + t - 1) / t);
      if (all > 16 * sms) continue;
      if (all < 6 * sms) break;
      const long cost = (all + sms - 1) / sms * t;
      if (!best || cost <= best) best = cost, per = t;
    }
  }
  q.chunk = per * kTile;
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
    q.part_bc = take(q.tiles > 1 ? 2 * static_cast<size_t>(q.tiles) * p.B * p.T * p.G * p.N : 0);
    q.part_a = take(BC * DN);
    q.part_d = take(2 * BC * p.D);
  }
  return at * sizeof(float);
}

// 16, 4 or 0: what a tensor's rows, and those of its groups where there are several, are aligned for
int aligned_for(const void* p, const int64_t* st, int n, size_t es, long inner) {
  for (int bytes : {16, 4}) {
    bool ok = reinterpret_cast<uintptr_t>(p) % bytes == 0 && inner * es % bytes == 0;
    for (int i = 0; i < n; ++i) ok = ok && st[i] * static_cast<int64_t>(es) % bytes == 0;
    if (ok) return bytes;
  }
  return 0;
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
  q.vec_x = aligned_for(p.x, p.x_stride, 2, es, inner);
  q.vec_dt = aligned_for(p.dt, p.dt_stride, 2, es, inner);
  q.vec_gy = backward ? aligned_for(p.grad_y, p.gy_stride, 2, es, inner) : 0;
  q.vec_b = aligned_for(p.Bm, p.B_stride, 3, es, 0);
  q.vec_c = aligned_for(p.Cm, p.C_stride, 3, es, 0);
  q.vec_n = q.vec_part = p.N % 4 == 0;      // (the scratch is aligned)
  q.pairs = p.D % 2 == 0;
  for (const void* o : {static_cast<const void*>(p.y), static_cast<const void*>(p.grad_x), static_cast<const void*>(p.grad_dt)})
    q.pairs = q.pairs && reinterpret_cast<uintptr_t>(o) % (2 * es) == 0;
  for (const void* s : {static_cast<const void*>(p.A), static_cast<const void*>(p.state), static_cast<const void*>(p.final_state),
                        static_cast<const void*>(p.checkpoints), static_cast<const void*>(p.grad_final_state),
                        static_cast<const void*>(p.grad_state)})
    q.vec_n = q.vec_n && aligned16(s);
  return TTT_B200_OK;
}

template <class K> int launch(K kernel, size_t smem, long grid, cudaStream_t s, const ttt_b200_scan_args& p, const Plan& q) {
  if (grid > 0x7fffffffL) return fail("ssm scan: too many CTAs");
  if (smem > 40 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return ttt_set_error(TTT_B200_ERR_LAUNCH, cudaGetErrorString(e));
  }
  ttt_launch_overlapped(kernel, static_cast<int>(grid), TH, static_cast<uint32_t>(smem), s, p, q);
  return launched("ssm scan");
}

template <class T, int LN> int forward(const ttt_b200_scan_args& p, const Plan& q, cudaStream_t s) {
  const long row = static_cast<long>(p.B) * p.G * q.tiles, grid = row * q.chunks;
  if (q.chunks > 1) {
    if (int rc = launch(scan_state_kernel<T, LN, false>, sizeof(StateSmem<T, LN>), row * (q.chunks - 1), s, p, q)) return rc;
    const long n = static_cast<long>(p.B) * p.D * p.N;
    ttt_launch_overlapped(scan_join_kernel<false>, static_cast<int>((n + 255) / 256), 256, 0, s, p, q);
  }
  return launch(scan_forward_kernel<T, LN>, sizeof(FwdSmem<T, LN>), grid, s, p, q);
}

template <class T, int LN> int backward(const ttt_b200_scan_args& p, const Plan& q, cudaStream_t s) {
  const long row = static_cast<long>(p.B) * p.G * q.tiles, grid = row * q.chunks;
  if (q.chunks > 1) {
    if (int rc = launch(scan_state_kernel<T, LN, true>, sizeof(StateSmem<T, LN>), row * (q.chunks - 1), s, p, q)) return rc;
    const long n = static_cast<long>(p.B) * p.D * p.N;
    ttt_launch_overlapped(scan_join_kernel<true>, static_cast<int>((n + 255) / 256), 256, 0, s, p, q);
  }
  if (int rc = launch(scan_backward_kernel<T, LN>, sizeof(BwdSmem<T, LN>), grid, s, p, q)) return rc;
  const long BTGN = static_cast<long>(p.B) * p.T * p.G * p.N, DN = static_cast<long>(p.D) * p.N, BCD = static_cast<long>(p.B) * q.chunks * p.D;
  const int bc = p.B * q.chunks;
  const bool parts = q.tiles > 1;
  const ttt_sum_job jobs[] = {{q.part_bc, parts ? p.grad_B : nullptr, BTGN, BTGN, q.tiles, p.dtype, 0},
                              {q.part_bc + q.tiles * BTGN, parts ? p.grad_C : nullptr, BTGN, BTGN, q.tiles, p.dtype, 0},
                              {q.part_a, p.grad_A, DN, DN, bc, TTT_B200_FP32, 0},
                              {q.part_d, p.grad_D, p.D, p.D, bc, TTT_B200_FP32, 0},
                              {q.part_d + BCD, p.grad_dt_bias, p.D, p.D, bc, TTT_B200_FP32, 0}};
  return ttt_sum_parts(jobs, 5, s);
}

template <class T, int LN> int step(const ttt_b200_scan_args& p, cudaStream_t s) {
  const int tiles = (p.D + 2 * TH / LN - 1) / (2 * TH / LN);
  const bool vec = p.N % 4 == 0 && aligned16(p.A) && aligned16(p.state_io);
  const long grid = static_cast<long>(p.B) * tiles;
  if (grid > 0x7fffffffL) return fail("ssm scan: too many CTAs");
  const bool one = p.G == 1 || p.D / p.G % (2 * TH / LN) == 0;
  ttt_launch_overlapped(one ? scan_step_kernel<T, LN, true> : scan_step_kernel<T, LN, false>, static_cast<int>(grid), TH, 0, s, p, vec, tiles);
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
