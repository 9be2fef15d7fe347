// Short depthwise causal convolution: forward (prompts, training), backward, and the step of single tokens.
//
//   y[b][t][d] = act(bias[d] + sum_k w[d][k] x[b][t - K + 1 + k][d])
//   g = dy act'(pre);  dx[s] = sum_k w[d][k] g[s + K - 1 - k];  dw[d][k] = sum_t g[t] x[t - K + 1 + k];  db = sum_t g[t]
//
// Bound by memory: 2 K operations per value that is read and written once.  A thread owns two neighbouring channels (one where rows
// do not start on a pair's boundary) and walks along a run of tokens with the last K - 1 inputs in registers, so that an input is read
// once per run; the K - 1 in front of a run come from the cache.  Rows come through a warp's ring of four blocks of eight rows (two in fp32) in shared
// memory: a warp's row is 128 bytes, and it takes some 40 KB in flight to keep an SM's share of the memory busy, which registers do
// not hold.  The backward keeps the last K values of g as well and leaves dx with a delay of K - 1 tokens.
//
// Measured, 4 x 2048 tokens of 2048 channels, K = 4, silu: in bf16 forward 16.2 us (4.1 TB/s), backward 31 us (3.3 TB/s; 52 % of the issue
// slots, 68 instructions per token and pair), in fp32 20.3 and 45 us.  3 x 1001 x 1003 in fp32, K = 3, single channels: 5.9 us
// (4.1 TB/s) and 10.8 us (3.3 TB/s).  The step of
// 8 rows of 2048: 2.5 us, a launch.
#include <algorithm>
#include <type_traits>

#include "ttt_elem.cuh"
#include "ttt_sum_parts.h"

namespace {

using namespace ttt;

struct Plan {
  int groups;      // V channels each
  int run;         // tokens of a thread
  int runs;        // CTAs along a sequence, kWarps runs each
  long y_batch, y_head, y_token;      // strides of y (dy with heads)
  float* part;     // backward: [B][runs][K + 1][D]
};

constexpr int kWarps = 4;      // of a CTA: runs of tokens after one another, of the same 32 V channels

// What a thread works on.
struct At {
  int tile, group, row, b, run;      // `row`: the CTA among those of its channels, over all sequences
  __device__ __forceinline__ explicit At(const Plan& q) {
    const int tiles = (q.groups + 31) / 32;
    tile = blockIdx.x % tiles;
    row = blockIdx.x / tiles;
    b = row / q.runs;
    run = row % q.runs * kWarps + threadIdx.x / 32;
    group = tile * 32 + threadIdx.x % 32;
  }
};

// V = 1 or 2 neighbouring channels of a thread: their values as float or float2, and as they lie in memory.
template <int V> struct Channels;
template <> struct Channels<1> {
  using F = float;
};
template <> struct Channels<2> {
  using F = float2;
};
template <class T, int V> struct alignas(V * sizeof(T)) Raw {
  T v[V];
};
// 1 / (1 + exp(-v)); far on the left exp is infinite and the result 0
template <class F> __device__ __forceinline__ F sigmoid(F v) { return rcp(plus(ex2(times(v, all<F>(-kLog2e))), all<F>(1.f))); }
template <class T, int V> __device__ __forceinline__ typename Channels<V>::F wide(const Raw<T, V>& r) {
  if constexpr (V == 1) return to_f32(r.v[0]);
  else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __bfloat1622float2(reinterpret_cast<const __nv_bfloat162&>(r));
  else if constexpr (std::is_same<T, __half>::value) return __half22float2(reinterpret_cast<const __half2&>(r));
  else return make_float2(r.v[0], r.v[1]);
}
template <class T, int V> __device__ __forceinline__ Raw<T, V> narrow(typename Channels<V>::F f) {
  Raw<T, V> r;
  if constexpr (V == 1) r.v[0] = from_f32<T>(f);
  else if constexpr (std::is_same<T, __nv_bfloat16>::value) reinterpret_cast<__nv_bfloat162&>(r) = __float22bfloat162_rn(f);
  else if constexpr (std::is_same<T, __half>::value) reinterpret_cast<__half2&>(r) = __float22half2_rn(f);
  else r.v[0] = f.x, r.v[1] = f.y;
  return r;
}
template <class T, int V> __device__ __forceinline__ Raw<T, V> nothing() { return narrow<T, V>(all<typename Channels<V>::F>(0.f)); }
template <class T, int V> __device__ __forceinline__ Raw<T, V> load(const T* p) { return *reinterpret_cast<const Raw<T, V>*>(p); }
template <class T, int V> __device__ __forceinline__ void store(T* p, Raw<T, V> r) { *reinterpret_cast<Raw<T, V>*>(p) = r; }

// weights [k] and bias of a thread's channels, whose K V weights are next to each other
template <int K, int V>
__device__ __forceinline__ void load_weights(const ttt_b200_conv_args& p, int d, typename Channels<V>::F (&w)[K], typename Channels<V>::F& bias) {
  float f[K * V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const Raw<float, V> r = load<float, V>(p.weight + static_cast<long>(d) * K + k * V);
#pragma unroll
    for (int i = 0; i < V; ++i) f[k * V + i] = r.v[i];
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if constexpr (V == 2) w[k] = make_float2(f[k], f[K + k]);
    else w[k] = f[k];
  }
  bias = p.bias ? wide<float, V>(load<float, V>(p.bias + d)) : all<typename Channels<V>::F>(0.f);
}

// The input at position t, which may lie in front of the sequence (the state) but not behind it.
template <class T, int K, int V> __device__ __forceinline__ Raw<T, V> input(const ttt_b200_conv_args& p, int b, int d, int t) {
  if (t >= 0) return load<T, V>(static_cast<const T*>(p.x) + b * p.x_stride[0] + t * p.x_stride[1] + d);
  if (p.state && t >= 1 - K) return load<T, V>(static_cast<const T*>(p.state) + (static_cast<long>(b) * (K - 1) + t + K - 1) * p.D + d);
  return nothing<T, V>();
}

__device__ __forceinline__ int length_of(const ttt_b200_conv_args& p, int b) {
  return p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
}

constexpr int U = 8;      // tokens of a block, which are requested together

// The rows of a tensor that a warp walks along, a block of U tokens at a time, requested ahead of the block that is worked on; those
// from `stop` on are not read.  Pairs of channels go through a ring in shared memory (asynchronous 16-byte copies: what is
// in flight costs no registers), single channels through registers.
template <class T, int V> struct Rows;
template <class T> struct Rows<T, 2> {
  static constexpr bool kRing = true;
  static constexpr int kSlots = sizeof(T) == 2 ? 4 : 2, kWidth = 64, kBytes = kSlots * U * kWidth * sizeof(T);
  static constexpr int kPiece = 16 / sizeof(T), kPieces = kWidth / kPiece, kMine = U * kPieces / 32;      // pieces of a block, of a lane
  T* ring;
  const T *from, *next;      // of this lane's first piece: the first block's and the next one's
  int64_t stride;
  int bytes, t, stop, block;      // bytes of a piece; first token of the next block to request
  __device__ __forceinline__ Rows(void* smem, const T* tile, int64_t stride, int cols) : ring(static_cast<T*>(smem)), from(tile), stride(stride) {
    const int c = (threadIdx.x & 31) % kPieces * kPiece, n = min(max(cols - c, 0), kPiece);
    bytes = n * static_cast<int>(sizeof(T));
    if (n > 0) from += c;
  }
  __device__ __forceinline__ void aim(int begin, int stop_) {
    t = begin;
    stop = stop_;
    block = -1;
    next = from + (begin + (threadIdx.x & 31) / kPieces) * stride;
  }
  __device__ __forceinline__ void issue(int slot) {
    if (t < stop) {
      const int u = (threadIdx.x & 31) / kPieces;
      T* to = ring + slot * (U * kWidth) + (threadIdx.x & 31) * kPiece;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const bool in = t + u + i * (32 / kPieces) < stop;
        cp_async16(to + i * 32 * kPiece, in ? next + i * (32 / kPieces) * stride : from, in ? bytes : 0);
      }
      next += U * stride;
      t += U;
    }
  }
  __device__ __forceinline__ void advance() {
    ++block;
    issue((block + kSlots - 1) % kSlots);
  }
  // row u of the block; `at`: where there are that many before `stop`
  __device__ __forceinline__ Raw<T, 2> at(int u) const { return load<T, 2>(ring + (block % kSlots * U + u) * kWidth + 2 * (threadIdx.x & 31)); }
};
template <class T> struct Rows<T, 1> {
  static constexpr bool kRing = false;
  static constexpr int kBytes = 0;
  const T* next;      // of this lane's channel (behind the last channel: of the tile's first)
  int64_t stride;
  int t, stop;
  Raw<T, 1> now[U], then[U];
  __device__ __forceinline__ Rows(void*, const T* tile, int64_t stride, int cols)
      : next(tile + (static_cast<int>(threadIdx.x & 31) < cols ? threadIdx.x & 31 : 0)), stride(stride) {}
  __device__ __forceinline__ void ask() {
    if (t + U <= stop) {
#pragma unroll
      for (int u = 0; u < U; ++u) then[u] = load<T, 1>(next + u * stride);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (t + u < stop) then[u] = load<T, 1>(next + u * stride);
    }
    next += U * stride;
    t += U;
  }
  __device__ __forceinline__ void aim(int begin, int stop_) {
    t = begin;
    stop = stop_;
    next += begin * stride;
    ask();
  }
  __device__ __forceinline__ void advance() {
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = then[u];
    ask();
  }
  __device__ __forceinline__ Raw<T, 1> at(int u) const { return now[u]; }
};

// Tensors that are walked along together, to their first block and from block to block; all lanes of a warp together.  Copies are waited for
// by groups, whichever ring they are for, so a block of all rings is one group: kSlots - 2 blocks of each are on their way behind a wait.
template <class R, class... More> __device__ __forceinline__ void start(int begin, int stop, R& rows, More&... more) {
  rows.aim(begin, stop);
  (more.aim(begin, stop), ...);
  if constexpr (R::kRing) {
#pragma unroll
    for (int k = 0; k < R::kSlots - 1; ++k) {
      rows.issue(k);
      (more.issue(k), ...);
      cp_async_commit();
    }
  }
}
template <class R, class... More> __device__ __forceinline__ void turn(R& rows, More&... more) {
  if constexpr (R::kRing) {
    cp_async_wait<R::kSlots - 2>();
    __syncwarp();      // the block has landed for all lanes, and all are through with the one before, whose place the next one takes
  }
  rows.advance();      // (issues the last block of the ring)
  (more.advance(), ...);
  if constexpr (R::kRing) cp_async_commit();
}

template <class T, int K, int V, bool kSilu> __global__ void __launch_bounds__(32 * kWarps) conv_forward_kernel(const ttt_b200_conv_args p, const Plan q) {
  wait_for_predecessor();
  using F = typename Channels<V>::F;
  __shared__ __align__(16) unsigned char rings[kWarps][Rows<T, V>::kBytes + 16];
  const At at(q);
  const int b = at.b, d0 = at.tile * 32 * V, begin = min(at.run * q.run, p.T), end = min(begin + q.run, p.T);
  if (begin == end) return;
  const bool mine = at.group < q.groups;
  const int d = mine ? at.group * V : d0;      // (a lane behind the last channel reads the tile's first)
  const int len = length_of(p, b), stop = min(len, end);
  Rows<T, V> rows(rings[threadIdx.x / 32], static_cast<const T*>(p.x) + b * p.x_stride[0] + d0, p.x_stride[1], p.D - d0);
  start(begin, stop, rows);
  T* y = static_cast<T*>(p.y) + b * q.y_batch + d / 64 * q.y_head + d % 64;
  F w[K], bias, x[K];
  load_weights<K, V>(p, d, w, bias);
#pragma unroll
  for (int k = 0; k < K - 1; ++k) {
    const int t = begin - K + 1 + k;
    x[k] = wide<T, V>(t < len ? input<T, K, V>(p, b, d, t) : nothing<T, V>());
  }
  auto one = [&](const Raw<T, V>& row) {
    x[K - 1] = wide<T, V>(row);
    F v = bias;
#pragma unroll
    for (int k = 0; k < K; ++k) v = mac(w[k], x[k], v);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) x[k] = x[k + 1];
    return kSilu ? times(v, sigmoid(v)) : v;
  };
  for (int t0 = begin; t0 < end; t0 += U) {
    turn(rows);
    T* to = y + t0 * q.y_token;
    if (t0 + U <= stop) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const Raw<T, V> o = narrow<T, V>(one(rows.at(u)));
        if (mine) store<T, V>(to, o);
        to += q.y_token;
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const F v = one(t0 + u < stop ? rows.at(u) : nothing<T, V>());
        if (mine && t0 + u < end) store<T, V>(to, t0 + u < stop ? narrow<T, V>(v) : nothing<T, V>());
        to += q.y_token;
      }
    }
  }
  if (begin == 0 && p.final_state && mine) {
    T* f = static_cast<T*>(p.final_state) + static_cast<long>(b) * (K - 1) * p.D + d;
#pragma unroll
    for (int k = 0; k < K - 1; ++k) store<T, V>(f + static_cast<long>(k) * p.D, input<T, K, V>(p, b, d, len - K + 1 + k));
  }
}

template <class T, int K, int V, bool kSilu> __global__ void __launch_bounds__(32 * kWarps) conv_backward_kernel(const ttt_b200_conv_args p, const Plan q) {
  wait_for_predecessor();
  using F = typename Channels<V>::F;
  __shared__ __align__(16) unsigned char rings[2][kWarps][Rows<T, V>::kBytes + 16];
  __shared__ float sums[kWarps][K + 1][32 * V];
  const At at(q);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = at.b, d0 = at.tile * 32 * V, begin = min(at.run * q.run, p.T), end = min(begin + q.run, p.T);
  F dw[K], db = all<F>(0.f);
#pragma unroll
  for (int k = 0; k < K; ++k) dw[k] = db;
  if (begin < end) {
    const bool mine = at.group < q.groups;
    const int d = mine ? at.group * V : d0;      // (a lane behind the last channel reads the tile's first)
    const int len = length_of(p, b);
    // token t finishes the gradient of position t - K + 1, in front of the sequence the state's
    const int live = min(len, end + K - 1), whole = min(len, end);
    const bool heads = p.heads != 0;
    Rows<T, V> rows(rings[0][warp], static_cast<const T*>(p.x) + b * p.x_stride[0] + d0, p.x_stride[1], p.D - d0);
    Rows<T, V> ups(rings[1][warp], static_cast<const T*>(p.grad_y) + (heads ? b * q.y_batch + d0 / 64 * q.y_head + d0 % 64 : b * p.gy_stride[0] + d0),
                   heads ? q.y_token : p.gy_stride[1], p.D - d0);
    start(begin, live, rows, ups);
    const T* gf = p.grad_final_state ? static_cast<const T*>(p.grad_final_state) + static_cast<long>(b) * (K - 1) * p.D + d : nullptr;
    T* gx = static_cast<T*>(p.grad_x) + static_cast<long>(b) * p.T * p.D + d;
    T* gs = p.grad_state ? static_cast<T*>(p.grad_state) + static_cast<long>(b) * (K - 1) * p.D + d : nullptr;
    F w[K], bias, x[K], g[K];      // g[j] is g at token t - j
    load_weights<K, V>(p, d, w, bias);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int t = begin - K + 1 + k;
      g[k] = x[k] = all<F>(0.f);
      if (k < K - 1 && t < len) x[k] = wide<T, V>(input<T, K, V>(p, b, d, t));
    }
    // `in`: a token of the sequence; behind it g is zero, and the last inputs, whatever they are, are in no product with it
    auto one = [&](const Raw<T, V>& row, const Raw<T, V>& up, bool own, bool in) {
      x[K - 1] = wide<T, V>(row);
      F v = wide<T, V>(up);
      if constexpr (kSilu) {
        F pre = bias;
#pragma unroll
        for (int k = 0; k < K; ++k) pre = mac(w[k], x[k], pre);
        const F s = sigmoid(pre);
        v = times(v, mac(times(pre, s), mac(s, all<F>(-1.f), all<F>(1.f)), s));
      }
#pragma unroll
      for (int k = K - 1; k > 0; --k) g[k] = g[k - 1];
      if (!in) v = all<F>(0.f);
      g[0] = v;
      F o = times(w[0], g[0]);
#pragma unroll
      for (int k = 1; k < K; ++k) o = mac(w[k], g[k], o);
      if (own && in) {
        db = plus(db, v);
#pragma unroll
        for (int k = 0; k < K; ++k) dw[k] = mac(v, x[k], dw[k]);
      }
#pragma unroll
      for (int k = 0; k < K - 1; ++k) x[k] = x[k + 1];
      return o;
    };
    auto place = [&](int s, F o) {      // the gradient of position s, where it may be the state's or among the last K - 1 inputs
      if (!mine || (s < begin && !(begin == 0 && gs))) return;
      const int j = s - len + K - 1;
      if (gf && j >= 0 && j < K - 1) o = plus(o, wide<T, V>(load<T, V>(gf + static_cast<long>(j) * p.D)));
      store<T, V>(s >= 0 ? gx + static_cast<long>(s) * p.D : gs + static_cast<long>(s + K - 1) * p.D, narrow<T, V>(o));
    };
    for (int t0 = begin; t0 < end; t0 += U) {
      turn(rows, ups);
      if (t0 + U <= whole) {
        T* to = gx + static_cast<long>(t0 - K + 1) * p.D;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const Raw<T, V> o = narrow<T, V>(one(rows.at(u), ups.at(u), true, true));
          if (mine && (u >= K - 1 || t0 > begin)) store<T, V>(to, o);
          else if (mine && begin == 0 && gs) store<T, V>(gs + static_cast<long>(u) * p.D, o);      // (t0 = 0, and len is beyond)
          to += p.D;
        }
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (t0 + u < end) {
            const bool in = t0 + u < live;
            place(t0 + u - K + 1, one(in ? rows.at(u) : nothing<T, V>(), in ? ups.at(u) : nothing<T, V>(), true, in));
          }
      }
    }
    // the K - 1 tokens behind the run, for the gradients of its last inputs; where there are any the run ends with a block
    if (end < live) {
      turn(rows, ups);
    }
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      const bool in = end + k < live;
      place(end + k - K + 1, one(in ? rows.at(k) : nothing<T, V>(), in ? ups.at(k) : nothing<T, V>(), false, in));
    }
  }
#pragma unroll
  for (int k = 0; k < K; ++k) reinterpret_cast<F*>(sums[warp][k])[lane] = dw[k];
  reinterpret_cast<F*>(sums[warp][K])[lane] = db;
  __syncthreads();
  float* part = q.part + static_cast<long>(at.row) * (K + 1) * p.D;
  for (int i = threadIdx.x; i < (K + 1) * V * 32; i += 32 * kWarps) {
    const int c = i % (V * 32), k = i / (V * 32), ch = at.tile * 32 * V + c;
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) s += sums[v][k][c];
    if (ch < p.D) part[static_cast<long>(k) * p.D + ch] = s;
  }
}

// A row of the batch and 128 V channels to a CTA.  Rows that name the same slot are taken in their order by the CTA of the first of
// them, so that no two CTAs touch a state.
template <class T, int K, int V> __global__ void __launch_bounds__(128) conv_step_kernel(const ttt_b200_conv_args p, int tiles) {
  wait_for_predecessor();
  const int b0 = blockIdx.x / tiles, d = (blockIdx.x % tiles * 128 + threadIdx.x) * V;
  const bool live = d < p.D;
  T* ys = static_cast<T*>(p.y);
  int slot = b0, more = 0;
  if (p.slots) {
    slot = p.slots[b0];
    if (slot < 0 || slot >= p.rows) {
      if (live) store<T, V>(ys + static_cast<long>(b0) * p.D + d, nothing<T, V>());
      return;
    }
    int before = 0, after = 0;
    for (int r = threadIdx.x; r < p.B; r += 128)
      if (r != b0 && p.slots[r] == slot) (r < b0 ? before : after) = 1;
    if (__syncthreads_or(before)) return;
    more = __syncthreads_or(after);
  }
  if (!live) return;
  using F = typename Channels<V>::F;
  F w[K], bias;
  Raw<T, V> x[K];
  load_weights<K, V>(p, d, w, bias);
  T* st = static_cast<T*>(p.state_io) + static_cast<long>(slot) * (K - 1) * p.D + d;
#pragma unroll
  for (int k = 0; k < K - 1; ++k) x[k] = load<T, V>(st + static_cast<long>(k) * p.D);
  for (int b = b0; b < p.B; ++b) {
    if (b != b0 && p.slots[b] != slot) continue;
    x[K - 1] = load<T, V>(static_cast<const T*>(p.x) + b * p.x_stride[0] + d);
    F v = bias;
#pragma unroll
    for (int k = 0; k < K; ++k) v = mac(w[k], wide<T, V>(x[k]), v);
    if (p.activation == TTT_B200_ACT_SILU) v = times(v, sigmoid(v));
    store<T, V>(ys + static_cast<long>(b) * p.D + d, narrow<T, V>(v));
#pragma unroll
    for (int k = 0; k < K - 1; ++k) x[k] = x[k + 1];
    if (!more) break;
  }
#pragma unroll
  for (int k = 0; k < K - 1; ++k) store<T, V>(st + static_cast<long>(k) * p.D, x[k]);
}

// ---- host --------------------------------------------------------------------------------------------------------------
int check(const ttt_b200_conv_args* p) {
  if (!p) return fail("short conv: NULL argument struct");
  if (p->B < 0 || p->T < 0 || p->T > 1 << 30 || p->D < 1 || p->D > 1 << 30 || p->K < 2 || p->K > 4)
    return fail("short conv: B, T >= 0, D >= 1, T and D at most 2^30, and a width of 2, 3 or 4");
  if (p->dtype < TTT_B200_BF16 || p->dtype > TTT_B200_FP32) return fail("short conv: unknown element type");
  if (p->activation != TTT_B200_ACT_NONE && p->activation != TTT_B200_ACT_SILU) return fail("short conv: activation is none or silu");
  if (p->heads && (p->D % 64 || p->T % 64)) return fail("short conv: heads need multiples of 64 channels and tokens");
  return TTT_B200_OK;
}

// whether channels can be taken in pairs
bool paired(const ttt_b200_conv_args& p, const void* a, const int64_t* st) {
  const uintptr_t two = p.dtype == TTT_B200_FP32 ? 8 : 4;
  return reinterpret_cast<uintptr_t>(a) % two == 0 && (!st || (st[0] % 2 == 0 && st[1] % 2 == 0));
}
// and whether its rows can be copied in pieces of 16 bytes
bool rows16(const ttt_b200_conv_args& p, const void* a, const int64_t* st) {
  const int64_t es = p.dtype == TTT_B200_FP32 ? 4 : 2;
  return aligned16(a) && (!st || (st[0] * es % 16 == 0 && st[1] * es % 16 == 0));
}
bool paired_weights(const ttt_b200_conv_args& p) {
  return p.D % 2 == 0 && ((reinterpret_cast<uintptr_t>(p.weight) | reinterpret_cast<uintptr_t>(p.bias)) & 7) == 0;
}

// Tokens of a warp's run: as many as leave four to five CTAs to an SM, since each run reads K - 1 tokens more and has its weights to
// fetch.  Measured, us, forward / backward with its sum of parts, K = 4, bf16, with runs of 16, 32, 64, 128: 4 x 2048 tokens of 2048 channels
// 19.9 / 46.4, 18.1 / 38.7, 16.2 / 34.6, 18.0 / 36.0 (64 by the rule); 2048 tokens of 768 channels 5.0 / 11.0, 6.3 / 12.2, 7.0 / 14.3, 9.4 / 20.4
// (16 by the rule).
void plan_runs(Plan& q, const ttt_b200_conv_args& p, int V) {
  q.groups = p.D / V;
  const long tiles = (q.groups + 31) / 32, sms = sm_count();
  for (q.run = 128; q.run > 16; q.run /= 2)
    if (2 * tiles * p.B * ((p.T + q.run * kWarps - 1) / (q.run * kWarps)) >= 9 * sms) break;
  q.runs = (p.T + q.run * kWarps - 1) / (q.run * kWarps);
  q.y_batch = static_cast<long>(p.T) * p.D;
  q.y_head = p.heads ? 64L * p.T : 64;
  q.y_token = p.heads ? 64 : p.D;
}

template <class T, int K> int forward(const ttt_b200_conv_args& p, cudaStream_t s) {
  Plan q = {};
  const bool vec = paired_weights(p) && rows16(p, p.x, p.x_stride) && paired(p, p.y, nullptr) && paired(p, p.state, nullptr) &&
                   paired(p, p.final_state, nullptr);
  plan_runs(q, p, vec ? 2 : 1);
  const long grid = static_cast<long>(p.B) * q.runs * ((q.groups + 31) / 32);
  if (grid > 0x7fffffffL) return fail("short conv: too many CTAs");
  const bool silu = p.activation == TTT_B200_ACT_SILU;
  const auto kernel = vec ? (silu ? conv_forward_kernel<T, K, 2, true> : conv_forward_kernel<T, K, 2, false>)
                          : (silu ? conv_forward_kernel<T, K, 1, true> : conv_forward_kernel<T, K, 1, false>);
  ttt_launch_overlapped(kernel, static_cast<int>(grid), 32 * kWarps, 0, s, p, q);
  return launched("short conv");
}

template <class T, int K> int backward(const ttt_b200_conv_args& p, cudaStream_t s) {
  Plan q = {};
  const bool vec = paired_weights(p) && rows16(p, p.x, p.x_stride) && rows16(p, p.grad_y, p.heads ? nullptr : p.gy_stride) &&
                   paired(p, p.state, nullptr) && paired(p, p.grad_final_state, nullptr) && paired(p, p.grad_x, nullptr) &&
                   paired(p, p.grad_state, nullptr);
  plan_runs(q, p, vec ? 2 : 1);
  q.part = static_cast<float*>(p.scratch);
  const long grid = static_cast<long>(p.B) * q.runs * ((q.groups + 31) / 32);
  if (grid > 0x7fffffffL) return fail("short conv backward: too many CTAs");
  const bool silu = p.activation == TTT_B200_ACT_SILU;
  const auto kernel = vec ? (silu ? conv_backward_kernel<T, K, 2, true> : conv_backward_kernel<T, K, 2, false>)
                          : (silu ? conv_backward_kernel<T, K, 1, true> : conv_backward_kernel<T, K, 1, false>);
  ttt_launch_overlapped(kernel, static_cast<int>(grid), 32 * kWarps, 0, s, p, q);
  if (int rc = launched("short conv backward")) return rc;
  const long row = static_cast<long>(K + 1) * p.D, KD = static_cast<long>(K) * p.D;
  const int parts = p.B * q.runs;
  const ttt_sum_job jobs[] = {{q.part, p.grad_weight, KD, row, parts, TTT_B200_FP32, p.D},
                              {q.part + KD, p.grad_bias, p.D, row, parts, TTT_B200_FP32, 0}};
  return ttt_sum_parts(jobs, 2, s);
}

template <class T, int K> int step(const ttt_b200_conv_args& p, cudaStream_t s) {
  const int64_t st[2] = {p.x_stride[0], 0};
  const bool vec = paired_weights(p) && paired(p, p.x, st) && paired(p, p.y, nullptr) && paired(p, p.state_io, nullptr);
  const int tiles = (p.D / (vec ? 2 : 1) + 127) / 128;
  const long grid = static_cast<long>(p.B) * tiles;
  if (grid > 0x7fffffffL) return fail("short conv step: too many CTAs");
  ttt_launch_overlapped(vec ? conv_step_kernel<T, K, 2> : conv_step_kernel<T, K, 1>, static_cast<int>(grid), 128, 0, s, p, tiles);
  return launched("short conv step");
}

#define TTT_WITH_WIDTH(width, call)                            \
  switch (width) {                                             \
    case 2: { constexpr int K = 2; return call; }              \
    case 3: { constexpr int K = 3; return call; }              \
    default: { constexpr int K = 4; return call; }             \
  }

}  // namespace

extern "C" uint64_t ttt_b200_short_conv_scratch_bytes(const ttt_b200_conv_args* p) {
  if (check(p) || p->B == 0 || p->T == 0) return 0;
  Plan one = {}, two = {};      // single channels or pairs: the pointers say which
  plan_runs(one, *p, 1);
  plan_runs(two, *p, 2);
  return static_cast<uint64_t>(p->B) * std::max(one.runs, two.runs) * (p->K + 1) * p->D * sizeof(float);
}

extern "C" int ttt_b200_short_conv(const ttt_b200_conv_args* p, void* stream) {
  if (int rc = check(p)) return rc;
  if (!p->x || !p->weight || !p->y) return fail("short conv: null tensor pointer");
  if (p->B == 0 || p->T == 0) return fail("short conv: no tokens");
  TTT_WITH_TYPE(p->dtype, TTT_WITH_WIDTH(p->K, (forward<Elem, K>(*p, static_cast<cudaStream_t>(stream)))))
  return TTT_B200_OK;
}

extern "C" int ttt_b200_short_conv_backward(const ttt_b200_conv_args* p, void* stream) {
  if (int rc = check(p)) return rc;
  if (!p->x || !p->weight || !p->grad_y || !p->grad_x || !p->grad_weight) return fail("short conv backward: null tensor pointer");
  if (p->B == 0 || p->T == 0) return fail("short conv backward: no tokens");
  if (!p->scratch || p->scratch_bytes < ttt_b200_short_conv_scratch_bytes(p) || !aligned16(p->scratch))
    return fail("short conv backward: scratch is missing, too small or not 16-byte aligned");
  TTT_WITH_TYPE(p->dtype, TTT_WITH_WIDTH(p->K, (backward<Elem, K>(*p, static_cast<cudaStream_t>(stream)))))
  return TTT_B200_OK;
}

extern "C" int ttt_b200_short_conv_step(const ttt_b200_conv_args* p, void* stream) {
  if (int rc = check(p)) return rc;
  if (!p->x || !p->weight || !p->y || !p->state_io) return fail("short conv step: null tensor pointer");
  if (p->B == 0) return fail("short conv step: no rows");
  if (p->heads) return fail("short conv step: heads are for whole mini-batches");
  if (p->slots ? p->rows < 1 : p->rows != p->B) return fail("short conv step: the state has another number of rows");
  TTT_WITH_TYPE(p->dtype, TTT_WITH_WIDTH(p->K, (step<Elem, K>(*p, static_cast<cudaStream_t>(stream)))))
  return TTT_B200_OK;
}
