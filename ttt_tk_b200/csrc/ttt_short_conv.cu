// Short depthwise causal convolution: forward (prompts, training), backward, and the step of single tokens.
//
//   y[b][t][d] = act(bias[d] + sum_k w[d][k] x[b][t - K + 1 + k][d])
//   g = dy act'(pre);  dx[s] = sum_k w[d][k] g[s + K - 1 - k];  dw[d][k] = sum_t g[t] x[t - K + 1 + k];  db = sum_t g[t]
//
// Bound by memory: 2 K operations per value that is read and written once.  A thread owns V neighbouring channels (eight, as
// 16-byte accesses, or one where rows do not start on 16-byte boundaries) and walks along a run of tokens with the last K - 1
// inputs in registers, so that an input is read once per run; the K - 1 in front of a run come from the cache.  The backward
// keeps the last K values of g as well and leaves dx with a delay of K - 1 tokens.
#include <algorithm>
#include <cstdio>

#include "ttt_elem.cuh"
#include "ttt_sum_parts.h"

namespace {

using namespace ttt;

struct Plan {
  int groups;      // V channels each
  int run;         // tokens of a thread
  int runs;        // of a sequence; backward: of a CTA's warps together
  long y_batch, y_head, y_token;      // strides of y (dy with heads)
  float* part;     // backward: [B][runs][K + 1][D]
};

template <class T, int V> __device__ __forceinline__ void load(const T* p, float (&f)[V]) {
  if constexpr (V == 8) {
    load8(p, f);
  } else {
    static_assert(V == 1, "one channel or eight");
    f[0] = to_f32(*p);
  }
}
template <class T, int V> __device__ __forceinline__ void store(T* p, const float (&f)[V]) {
  if constexpr (V == 8) store8(p, f);
  else *p = from_f32<T>(f[0]);
}
template <int V> __device__ __forceinline__ void clear(float (&f)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = 0.f;
}

// weights [k][channel] and bias of a thread's channels
template <int K, int V> __device__ __forceinline__ void load_weights(const ttt_b200_conv_args& p, int d, float (&w)[K][V], float (&bias)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int k = 0; k < K; ++k) w[k][i] = p.weight[static_cast<long>(d + i) * K + k];
    bias[i] = p.bias ? p.bias[d + i] : 0.f;
  }
}

// The input at position t, which may lie in front of the sequence (the state) but not behind it.
template <class T, int K, int V> __device__ __forceinline__ void input(const ttt_b200_conv_args& p, int b, int d, int t, float (&f)[V]) {
  if (t >= 0) load<T, V>(static_cast<const T*>(p.x) + b * p.x_stride[0] + t * p.x_stride[1] + d, f);
  else if (p.state && t >= 1 - K) load<T, V>(static_cast<const T*>(p.state) + (static_cast<long>(b) * (K - 1) + t + K - 1) * p.D + d, f);
  else clear<V>(f);
}

__device__ __forceinline__ float sigmoid(float v) { return rcp(1.f + ex2(fminf(-v * kLog2e, 126.f))); }

__device__ __forceinline__ int length_of(const ttt_b200_conv_args& p, int b) {
  return p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
}

template <class T, int K, int V> __global__ void __launch_bounds__(128) conv_forward_kernel(const ttt_b200_conv_args p, const Plan q) {
  const long id = static_cast<long>(blockIdx.x) * 128 + threadIdx.x;
  const int d = static_cast<int>(id % q.groups) * V;
  const long bt = id / q.groups;
  const int b = static_cast<int>(bt / q.runs), r = static_cast<int>(bt % q.runs);
  if (b >= p.B) return;
  const int len = length_of(p, b), begin = r * q.run, end = min(begin + q.run, p.T);
  float w[K][V], bias[V], x[K][V];
  load_weights<K, V>(p, d, w, bias);
#pragma unroll
  for (int k = 0; k < K - 1; ++k) {
    if (begin - K + 1 + k < len) input<T, K, V>(p, b, d, begin - K + 1 + k, x[k]);
    else clear<V>(x[k]);
  }
  T* y = static_cast<T*>(p.y) + b * q.y_batch + d / 64 * q.y_head + d % 64;
  constexpr int U = 4;      // rows requested together
  for (int t0 = begin; t0 < end; t0 += U) {
    float in[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (t0 + u < min(len, end)) load<T, V>(static_cast<const T*>(p.x) + b * p.x_stride[0] + (t0 + u) * p.x_stride[1] + d, in[u]);
      else clear<V>(in[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u;
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        x[K - 1][i] = in[u][i];
        float v = bias[i];
#pragma unroll
        for (int k = 0; k < K; ++k) v = fmaf(w[k][i], x[k][i], v);
        if (p.activation == TTT_B200_ACT_SILU) v *= sigmoid(v);
        o[i] = t < len ? v : 0.f;
#pragma unroll
        for (int k = 0; k < K - 1; ++k) x[k][i] = x[k + 1][i];
      }
      if (t < end) store<T, V>(y + t * q.y_token, o);
    }
  }
  if (r == 0 && p.final_state) {
    T* f = static_cast<T*>(p.final_state) + static_cast<long>(b) * (K - 1) * p.D + d;
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      float v[V];
      input<T, K, V>(p, b, d, len - K + 1 + k, v);
      store<T, V>(f + static_cast<long>(k) * p.D, v);
    }
  }
}

constexpr int kWarps = 4;      // of a backward CTA: runs of tokens after one another, of the same 32 V channels

template <class T, int K, int V> __global__ void __launch_bounds__(32 * kWarps) conv_backward_kernel(const ttt_b200_conv_args p, const Plan q) {
  __shared__ float sums[kWarps][(K + 1) * V][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tiles = (q.groups + 31) / 32;
  const int group = blockIdx.x % tiles * 32 + lane, d = group * V;
  const long bt = blockIdx.x / tiles;
  const int b = static_cast<int>(bt / q.runs), r = static_cast<int>(bt % q.runs);
  const int begin = min((r * kWarps + warp) * q.run, p.T), end = min(begin + q.run, p.T);
  const bool live = group < q.groups;
  float dw[K][V], db[V];
#pragma unroll
  for (int k = 0; k < K; ++k) clear<V>(dw[k]);
  clear<V>(db);
  if (live && begin < end) {
    const int len = length_of(p, b);
    float w[K][V], bias[V], x[K][V], g[K][V];
    load_weights<K, V>(p, d, w, bias);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      clear<V>(g[k]);
      if (k < K - 1 && begin - K + 1 + k < len) input<T, K, V>(p, b, d, begin - K + 1 + k, x[k]);
      else clear<V>(x[k]);
    }
    const bool heads = p.heads != 0;
    const T* gy = static_cast<const T*>(p.grad_y) + (heads ? b * q.y_batch + d / 64 * q.y_head + d % 64 : b * p.gy_stride[0] + d);
    const long gy_token = heads ? q.y_token : p.gy_stride[1];
    const T* gf = p.grad_final_state ? static_cast<const T*>(p.grad_final_state) + static_cast<long>(b) * (K - 1) * p.D + d : nullptr;
    T* gx = static_cast<T*>(p.grad_x) + static_cast<long>(b) * p.T * p.D + d;
    T* gs = p.grad_state ? static_cast<T*>(p.grad_state) + static_cast<long>(b) * (K - 1) * p.D + d : nullptr;
    // g[j] is g at token t - j; token t finishes the gradient of position t - K + 1, in front of the sequence the state's
    const int stop = end + K - 1;
    constexpr int U = 4;
    for (int t0 = begin; t0 < stop; t0 += U) {
      float in[U][V], dy[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = t0 + u;
        if (t < min(len, stop)) {
          load<T, V>(static_cast<const T*>(p.x) + b * p.x_stride[0] + t * p.x_stride[1] + d, in[u]);
          load<T, V>(gy + t * gy_token, dy[u]);
        } else {
          clear<V>(in[u]);
          clear<V>(dy[u]);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = t0 + u;
        if (t >= stop) break;
        const bool own = t < end;
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          x[K - 1][i] = in[u][i];
          float v = dy[u][i];
          if (p.activation == TTT_B200_ACT_SILU) {
            float pre = bias[i];
#pragma unroll
            for (int k = 0; k < K; ++k) pre = fmaf(w[k][i], x[k][i], pre);
            const float s = sigmoid(pre);
            v *= fmaf(pre * s, 1.f - s, s);
          }
#pragma unroll
          for (int k = K - 1; k > 0; --k) g[k][i] = g[k - 1][i];
          g[0][i] = v;
          const float mine = own ? v : 0.f;
          db[i] += mine;
          o[i] = 0.f;
#pragma unroll
          for (int k = 0; k < K; ++k) {
            dw[k][i] = fmaf(mine, x[k][i], dw[k][i]);
            o[i] = fmaf(w[k][i], g[k][i], o[i]);
          }
#pragma unroll
          for (int k = 0; k < K - 1; ++k) x[k][i] = x[k + 1][i];
        }
        const int s = t - K + 1;
        if (s >= begin || (begin == 0 && gs)) {
          const int j = s - len + K - 1;      // its place among the last K - 1 inputs
          if (gf && j >= 0 && j < K - 1) {
            float f[V];
            load<T, V>(gf + static_cast<long>(j) * p.D, f);
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] += f[i];
          }
          store<T, V>(s >= 0 ? gx + static_cast<long>(s) * p.D : gs + static_cast<long>(s + K - 1) * p.D, o);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int k = 0; k < K; ++k) sums[warp][k * V + i][lane] = dw[k][i];
    sums[warp][K * V + i][lane] = db[i];
  }
  __syncthreads();
  float* part = q.part + bt * (K + 1) * p.D;
  for (int i = threadIdx.x; i < (K + 1) * V * 32; i += 32 * kWarps) {
    const int c = i % (V * 32), k = i / (V * 32), at = blockIdx.x % tiles * 32 * V + c;
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) s += sums[v][k * V + c % V][c / V];
    if (at < p.D) part[static_cast<long>(k) * p.D + at] = s;
  }
}

// A row of the batch and 128 V channels to a CTA.  Rows that name the same slot are taken in their order by the CTA of the first of
// them, so that no two CTAs touch a state.
template <class T, int K, int V> __global__ void __launch_bounds__(128) conv_step_kernel(const ttt_b200_conv_args p, int tiles) {
  const int b0 = blockIdx.x / tiles, d = (blockIdx.x % tiles * 128 + threadIdx.x) * V;
  const bool live = d < p.D;
  T* ys = static_cast<T*>(p.y);
  int slot = b0, more = 0;
  if (p.slots) {
    slot = p.slots[b0];
    if (slot < 0 || slot >= p.rows) {
      float o[V];
      clear<V>(o);
      if (live) store<T, V>(ys + static_cast<long>(b0) * p.D + d, o);
      return;
    }
    int before = 0, after = 0;
    for (int r = threadIdx.x; r < p.B; r += 128)
      if (r != b0 && p.slots[r] == slot) (r < b0 ? before : after) = 1;
    if (__syncthreads_or(before)) return;
    more = __syncthreads_or(after);
  }
  if (!live) return;
  float w[K][V], bias[V], x[K][V];
  load_weights<K, V>(p, d, w, bias);
  T* st = static_cast<T*>(p.state_io) + static_cast<long>(slot) * (K - 1) * p.D + d;
#pragma unroll
  for (int k = 0; k < K - 1; ++k) load<T, V>(st + static_cast<long>(k) * p.D, x[k]);
  for (int b = b0; b < p.B; ++b) {
    if (b != b0 && p.slots[b] != slot) continue;
    load<T, V>(static_cast<const T*>(p.x) + b * p.x_stride[0] + d, x[K - 1]);
    float o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float v = bias[i];
#pragma unroll
      for (int k = 0; k < K; ++k) v = fmaf(w[k][i], x[k][i], v);
      o[i] = p.activation == TTT_B200_ACT_SILU ? v * sigmoid(v) : v;
#pragma unroll
      for (int k = 0; k < K - 1; ++k) x[k][i] = x[k + 1][i];
    }
    store<T, V>(ys + static_cast<long>(b) * p.D + d, o);
    if (!more) break;
  }
#pragma unroll
  for (int k = 0; k < K - 1; ++k) store<T, V>(st + static_cast<long>(k) * p.D, x[k]);
}

// ---- host --------------------------------------------------------------------------------------------------------------
int fail(const char* msg) { return ttt_set_error(TTT_B200_ERR_BAD_ARGS, msg); }

int check(const ttt_b200_conv_args* p) {
  if (!p) return fail("short conv: NULL argument struct");
  if (p->B < 0 || p->T < 0 || p->D < 1 || p->K < 2 || p->K > 4) return fail("short conv: B, T >= 0, D >= 1 and a width of 2, 3 or 4");
  if (p->dtype < TTT_B200_BF16 || p->dtype > TTT_B200_FP32) return fail("short conv: unknown element type");
  if (p->activation != TTT_B200_ACT_NONE && p->activation != TTT_B200_ACT_SILU) return fail("short conv: activation is none or silu");
  if (p->heads && (p->D % 64 || p->T % 64)) return fail("short conv: heads need multiples of 64 channels and tokens");
  return TTT_B200_OK;
}

int sm_count() {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return TTT_B200_OK;
  static thread_local char buf[160];
  snprintf(buf, sizeof buf, "%s: %s", what, cudaGetErrorString(e));
  return ttt_set_error(TTT_B200_ERR_LAUNCH, buf);
}

bool rows16(const ttt_b200_conv_args& p, const void* a, const int64_t* st) {
  const int64_t es = p.dtype == TTT_B200_FP32 ? 4 : 2;
  return aligned16(a) && (!st || (st[0] * es % 16 == 0 && st[1] * es % 16 == 0));
}

void fill(Plan& q, const ttt_b200_conv_args& p, int V) {
  q.groups = p.D / V;
  q.y_batch = static_cast<long>(p.T) * p.D;
  q.y_head = p.heads ? 64L * p.T : 64;
  q.y_token = p.heads ? 64 : p.D;
}

// Backward: tokens of a warp's run.
void plan_backward(Plan& q, const ttt_b200_conv_args& p) {
  q.run = 32;
  q.runs = (p.T + q.run * kWarps - 1) / (q.run * kWarps);
}

template <class T, int K> int forward(const ttt_b200_conv_args& p, cudaStream_t s) {
  Plan q = {};
  const bool vec = p.D % 8 == 0 && rows16(p, p.x, p.x_stride) && rows16(p, p.y, nullptr) && rows16(p, p.state, nullptr) &&
                   rows16(p, p.final_state, nullptr);
  fill(q, p, vec ? 8 : 1);
  const long want = static_cast<long>(sm_count()) * 1024, tokens = static_cast<long>(p.B) * p.T * q.groups;
  q.run = tokens / 32 >= want ? 32 : tokens / 16 >= want ? 16 : 8;
  q.runs = (p.T + q.run - 1) / q.run;
  const long grid = (static_cast<long>(p.B) * q.runs * q.groups + 127) / 128;
  if (grid > 0x7fffffffL) return fail("short conv: too many CTAs");
  if (vec) conv_forward_kernel<T, K, 8><<<static_cast<unsigned>(grid), 128, 0, s>>>(p, q);
  else conv_forward_kernel<T, K, 1><<<static_cast<unsigned>(grid), 128, 0, s>>>(p, q);
  return launched("short conv");
}

template <class T, int K> int backward(const ttt_b200_conv_args& p, cudaStream_t s) {
  Plan q = {};
  const bool vec = p.D % 8 == 0 && rows16(p, p.x, p.x_stride) && rows16(p, p.grad_y, p.heads ? nullptr : p.gy_stride) &&
                   rows16(p, p.state, nullptr) && rows16(p, p.grad_final_state, nullptr) && rows16(p, p.grad_x, nullptr) &&
                   rows16(p, p.grad_state, nullptr);
  fill(q, p, vec ? 8 : 1);
  plan_backward(q, p);
  q.part = static_cast<float*>(p.scratch);
  const long grid = static_cast<long>(p.B) * q.runs * ((q.groups + 31) / 32);
  if (grid > 0x7fffffffL) return fail("short conv backward: too many CTAs");
  if (vec) conv_backward_kernel<T, K, 8><<<static_cast<unsigned>(grid), 32 * kWarps, 0, s>>>(p, q);
  else conv_backward_kernel<T, K, 1><<<static_cast<unsigned>(grid), 32 * kWarps, 0, s>>>(p, q);
  if (int rc = launched("short conv backward")) return rc;
  const long row = static_cast<long>(K + 1) * p.D, KD = static_cast<long>(K) * p.D;
  const int parts = p.B * q.runs;
  const ttt_sum_job jobs[] = {{q.part, p.grad_weight, KD, row, parts, TTT_B200_FP32, p.D},
                              {q.part + KD, p.grad_bias, p.D, row, parts, TTT_B200_FP32, 0}};
  return ttt_sum_parts(jobs, 2, s);
}

template <class T, int K> int step(const ttt_b200_conv_args& p, cudaStream_t s) {
  const int64_t st[2] = {p.x_stride[0], 0};
  const bool vec = p.D % 8 == 0 && rows16(p, p.x, st) && rows16(p, p.y, nullptr) && rows16(p, p.state_io, nullptr);
  const int tiles = (p.D / (vec ? 8 : 1) + 127) / 128;
  const long grid = static_cast<long>(p.B) * tiles;
  if (grid > 0x7fffffffL) return fail("short conv step: too many CTAs");
  if (vec) conv_step_kernel<T, K, 8><<<static_cast<unsigned>(grid), 128, 0, s>>>(p, tiles);
  else conv_step_kernel<T, K, 1><<<static_cast<unsigned>(grid), 128, 0, s>>>(p, tiles);
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
  Plan q = {};
  plan_backward(q, *p);
  return static_cast<uint64_t>(p->B) * q.runs * (p->K + 1) * p->D * sizeof(float);
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
