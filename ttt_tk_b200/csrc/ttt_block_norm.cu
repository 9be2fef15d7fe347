// The end of a block and the start of the next, in one pass over a token's D values, and its backward:
//
//   u = Norm(o) w1 + b1;   v = u act(gate);   z = residual + scale v;   n = Norm(z) w2 + b2
//   Norm: (a - mean) r, r = 1 / sqrt(var + eps) (layer), or a r, r = 1 / sqrt(mean(a^2) + eps)
//
//   d  = dz + r2 (g2 - mean(g2) - zh mean(g2 zh)),  g2 = dn w2, zh = Norm(z)        (no mean(g2) without the layer's mean)
//   d residual = d;  d scale = sum d v;  dv = d scale;  d gate = dv u act'(gate);  du = dv act(gate)
//   do = r1 (g1 - mean(g1) - oh mean(g1 oh)),  g1 = du w1, oh = Norm(o);  dw, db: sums over the tokens
//
// Bound by memory.  A token belongs to the fewest threads (a warp or a power of two of them) that hold it with eight values each,
// so that it is read once and its statistics are two passes over registers; tokens of up to 8192 values take sixteen.  The
// backward computes z again from what the forward read (not from the z it wrote, whose rounding would be in the sums), keeps the
// sums over tokens of its columns to itself over all its tokens and leaves them as one part per CTA for an ordered sum.
#include <algorithm>
#include <cstdio>

#include "ttt_elem.cuh"
#include "ttt_sum_parts.h"

namespace {

using namespace ttt;

struct Plan {
  int width;      // threads of a token
  int side;       // tokens next to each other in a CTA
  int ctas;
  float* part;    // backward: [ctas * side][5][D]
};

template <class T, int V> __device__ __forceinline__ void load(const T* p, float (&f)[V]) {
  if constexpr (V == 8) load8(p, f);
  else f[0] = to_f32(*p);
}
template <class T, int V> __device__ __forceinline__ void store(T* p, const float (&f)[V]) {
  if constexpr (V == 8) store8(p, f);
  else *p = from_f32<T>(f[0]);
}

struct Gate {
  float v, s;      // value and slope
};
__device__ __forceinline__ Gate act(int kind, float x) {
  // sigmoid of a and its complement; the exponent is bounded so that neither becomes 0 times infinity
  float a = x, da = 1.f;
  if (kind == TTT_B200_ACT_GELU) {      // x sigmoid(2 u): no 1 + tanh(u), which cancels on the left
    constexpr float k = 1.5957691216057308f, c = 0.044715f;      // 2 sqrt(2 / pi)
    const float q = x * x;
    a = k * x * fmaf(c, q, 1.f);
    da = k * fmaf(3.f * c, q, 1.f);
  }
  const float e = ex2(fminf(-a * kLog2e, 126.f)), s = rcp(1.f + e), o = e * s;
  if (kind == TTT_B200_ACT_SIGMOID) return {s, s * o};
  return {x * s, fmaf(x * s, o * da, s)};
}

// The sum of two values over the threads of a token, in all of them.  `buf` alternates between calls: a barrier lies between two
// uses of the same half.
__device__ __forceinline__ float2 row_sum(float2 v, float2 (*smem)[32], int& buf, int width) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if (width > 32) {
    const int warp = threadIdx.x >> 5, warps = width >> 5, first = warp / warps * warps;
    if ((threadIdx.x & 31) == 0) smem[buf][warp] = v;
    __syncthreads();
    v = make_float2(0.f, 0.f);
    for (int i = 0; i < warps; ++i) {
      const float2 a = smem[buf][first + i];
      v.x += a.x;
      v.y += a.y;
    }
    buf ^= 1;
  }
  return v;
}

// column of vector j of this thread
template <int V> __device__ __forceinline__ int column(int j, int lane, int width) { return (j * width + lane) * V; }

template <int V, int NV>
__device__ __forceinline__ float2 statistics(const float (&a)[NV][V], const ttt_b200_block_args& p, int lane, int width, float2 (*smem)[32], int& buf) {
  const float inv = 1.f / static_cast<float>(p.D);
  float mean = 0.f;
  if (p.layer) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (column<V>(j, lane, width) < p.D) {
#pragma unroll
        for (int i = 0; i < V; ++i) s += a[j][i];
      }
    mean = row_sum(make_float2(s, 0.f), smem, buf, width).x * inv;
  }
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (column<V>(j, lane, width) < p.D) {
#pragma unroll
      for (int i = 0; i < V; ++i) s = fmaf(a[j][i] - mean, a[j][i] - mean, s);
    }
  s = row_sum(make_float2(s, 0.f), smem, buf, width).x;
  return make_float2(mean, rsqrtf(fmaf(s, inv, p.eps)));
}

template <class T, class R, int V, int NV>
__global__ void __launch_bounds__(1024) block_forward_kernel(const ttt_b200_block_args p, const Plan q) {
  __shared__ float2 smem[2][32];
  int buf = 0;
  const int lane = threadIdx.x % q.width;
  const long m = static_cast<long>(blockIdx.x) * q.side + threadIdx.x / q.width;
  const bool live = m < p.M;
  float a[NV][V], z[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int d = column<V>(j, lane, q.width);
#pragma unroll
    for (int i = 0; i < V; ++i) a[j][i] = z[j][i] = 0.f;
    if (live && d < p.D) {
      load<T, V>(static_cast<const T*>(p.o) + m * p.o_stride + d, a[j]);
      if (p.residual) load<R, V>(static_cast<const R*>(p.residual) + m * p.residual_stride + d, z[j]);
      if (p.gate && !p.post_weight) {
        float g[V];
        load<T, V>(static_cast<const T*>(p.gate) + m * p.gate_stride + d, g);
#pragma unroll
        for (int i = 0; i < V; ++i) a[j][i] *= act(p.activation, g[i]).v;
      }
    }
  }
  float2 s1 = make_float2(0.f, 1.f), s2 = s1;
  if (p.post_weight) {
    // the gate is requested before the statistics, which wait for o
    float g[NV][V];
    if (p.gate) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int d = column<V>(j, lane, q.width);
        if (live && d < p.D) load<T, V>(static_cast<const T*>(p.gate) + m * p.gate_stride + d, g[j]);
      }
    }
    s1 = statistics<V, NV>(a, p, lane, q.width, smem, buf);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int d = column<V>(j, lane, q.width);
      if (live && d < p.D) {
        float w[V], b[V];
        load<float, V>(p.post_weight + d, w);
        if (p.post_bias) load<float, V>(p.post_bias + d, b);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          a[j][i] = fmaf((a[j][i] - s1.x) * s1.y, w[i], p.post_bias ? b[i] : 0.f);
          if (p.gate) a[j][i] *= act(p.activation, g[j][i]).v;
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int d = column<V>(j, lane, q.width);
    if (live && d < p.D) {
      float sc[V];
      if (p.scale) load<float, V>(p.scale + d, sc);
#pragma unroll
      for (int i = 0; i < V; ++i) z[j][i] = fmaf(p.scale ? sc[i] : 1.f, a[j][i], z[j][i]);
      store<R, V>(static_cast<R*>(p.x) + m * p.D + d, z[j]);
    }
  }
  if (p.pre_weight) {
    s2 = statistics<V, NV>(z, p, lane, q.width, smem, buf);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int d = column<V>(j, lane, q.width);
      if (live && d < p.D) {
        float w[V], b[V];
        load<float, V>(p.pre_weight + d, w);
        if (p.pre_bias) load<float, V>(p.pre_bias + d, b);
#pragma unroll
        for (int i = 0; i < V; ++i) z[j][i] = fmaf((z[j][i] - s2.x) * s2.y, w[i], p.pre_bias ? b[i] : 0.f);
        store<T, V>(static_cast<T*>(p.n) + m * p.D + d, z[j]);
      }
    }
  }
  if (p.stats && live && lane == 0) reinterpret_cast<float4*>(p.stats)[m] = make_float4(s1.x, s1.y, s2.x, s2.y);
}

// Sums over tokens of a thread's columns: in registers, or, of sixteen columns, in shared memory.
enum { kDw1, kDb1, kDsc, kDw2, kDb2, kSums };
template <int V, int NV, bool kShared> struct Sums {
  float r[kShared ? 1 : kSums][NV][V];
  float* s;
  int D;
  __device__ __forceinline__ void add(int k, int j, int i, int d, float v) {
    if constexpr (kShared) s[k * D + d + i] += v;
    else r[k][j][i] += v;
  }
  __device__ __forceinline__ float get(int k, int j, int i, int d) const {
    if constexpr (kShared) return s[k * D + d + i];
    else return r[k][j][i];
  }
};

template <class T, class R, int V, int NV, bool kShared>
__global__ void __launch_bounds__(512) block_backward_kernel(const ttt_b200_block_args p, const Plan q) {
  __shared__ float2 smem[2][32];
  extern __shared__ float shared_sums[];
  int buf = 0;
  const int lane = threadIdx.x % q.width, sub = threadIdx.x / q.width;
  const float inv = 1.f / static_cast<float>(p.D);
  Sums<V, NV, kShared> sums;
  sums.s = shared_sums;
  sums.D = p.D;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int d = column<V>(j, lane, q.width);
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int k = 0; k < kSums; ++k) {
        if constexpr (kShared) {
          if (d < p.D) shared_sums[k * p.D + d + i] = 0.f;
        } else {
          sums.r[k][j][i] = 0.f;
        }
      }
  }
  for (long base = static_cast<long>(blockIdx.x) * q.side; base < p.M; base += static_cast<long>(q.ctas) * q.side) {
    const long m = base + sub;
    const bool live = m < p.M;
    float o[NV][V], z[NV][V], g[NV][V], d2[NV][V], gn[NV][V];
    float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live) st = reinterpret_cast<const float4*>(p.stats)[m];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int d = column<V>(j, lane, q.width);
#pragma unroll
      for (int i = 0; i < V; ++i) o[j][i] = z[j][i] = g[j][i] = d2[j][i] = gn[j][i] = 0.f;
      if (live && d < p.D) {
        load<T, V>(static_cast<const T*>(p.o) + m * p.o_stride + d, o[j]);
        if (p.gate) load<T, V>(static_cast<const T*>(p.gate) + m * p.gate_stride + d, g[j]);
        if (p.residual && p.pre_weight) load<R, V>(static_cast<const R*>(p.residual) + m * p.residual_stride + d, z[j]);
        if (p.grad_x) load<R, V>(static_cast<const R*>(p.grad_x) + m * p.gx_stride + d, d2[j]);
        if (p.grad_n && p.pre_weight) load<T, V>(static_cast<const T*>(p.grad_n) + m * p.gn_stride + d, gn[j]);
      }
    }
    // u (with its norm: oh) and z again, as the forward had them; from here on z is its normalised value
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int d = column<V>(j, lane, q.width);
      if (!(live && d < p.D)) continue;
      float w[V], b[V], sc[V], w2[V];
      if (p.post_weight) load<float, V>(p.post_weight + d, w);
      if (p.post_bias) load<float, V>(p.post_bias + d, b);
      if (p.scale) load<float, V>(p.scale + d, sc);
      if (p.pre_weight) load<float, V>(p.pre_weight + d, w2);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (p.post_weight) o[j][i] = (o[j][i] - st.x) * st.y;
        if (p.pre_weight) {
          const float u = p.post_weight ? fmaf(o[j][i], w[i], p.post_bias ? b[i] : 0.f) : o[j][i];
          const float v = p.gate ? u * act(p.activation, g[j][i]).v : u;
          z[j][i] = (fmaf(p.scale ? sc[i] : 1.f, v, z[j][i]) - st.z) * st.w;
          sums.add(kDw2, j, i, d, gn[j][i] * z[j][i]);
          sums.add(kDb2, j, i, d, gn[j][i]);
          gn[j][i] *= w2[i];
          s.x += gn[j][i];
          s.y = fmaf(gn[j][i], z[j][i], s.y);
        }
      }
    }
    if (p.pre_weight) {
      s = row_sum(s, smem, buf, q.width);
      const float m1 = p.layer ? s.x * inv : 0.f, m2 = s.y * inv;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) d2[j][i] = fmaf(st.w, gn[j][i] - m1 - z[j][i] * m2, d2[j][i]);
    }
    s = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int d = column<V>(j, lane, q.width);
      if (!(live && d < p.D)) continue;
      if (p.grad_residual) store<R, V>(static_cast<R*>(p.grad_residual) + m * p.D + d, d2[j]);
      float w[V], b[V], sc[V];
      if (p.post_weight) load<float, V>(p.post_weight + d, w);
      if (p.post_bias) load<float, V>(p.post_bias + d, b);
      if (p.scale) load<float, V>(p.scale + d, sc);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float u = p.post_weight ? fmaf(o[j][i], w[i], p.post_bias ? b[i] : 0.f) : o[j][i];
        Gate a = {1.f, 0.f};
        if (p.gate) a = act(p.activation, g[j][i]);
        sums.add(kDsc, j, i, d, d2[j][i] * (u * a.v));
        const float dv = p.scale ? d2[j][i] * sc[i] : d2[j][i];
        g[j][i] = dv * u * a.s;
        float du = dv * a.v;
        if (p.post_weight) {
          sums.add(kDw1, j, i, d, du * o[j][i]);
          sums.add(kDb1, j, i, d, du);
          du *= w[i];
          s.x += du;
          s.y = fmaf(du, o[j][i], s.y);
        }
        d2[j][i] = du;
      }
      if (p.grad_gate) store<T, V>(static_cast<T*>(p.grad_gate) + m * p.D + d, g[j]);
    }
    float m1 = 0.f, m2 = 0.f;
    if (p.post_weight) {
      s = row_sum(s, smem, buf, q.width);
      m1 = p.layer ? s.x * inv : 0.f;
      m2 = s.y * inv;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int d = column<V>(j, lane, q.width);
      if (!(live && d < p.D)) continue;
      if (p.post_weight) {
#pragma unroll
        for (int i = 0; i < V; ++i) d2[j][i] = st.y * (d2[j][i] - m1 - o[j][i] * m2);
      }
      store<T, V>(static_cast<T*>(p.grad_o) + m * p.D + d, d2[j]);
    }
  }
  float* part = q.part + (static_cast<long>(blockIdx.x) * q.side + sub) * kSums * p.D;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int d = column<V>(j, lane, q.width);
    if (d >= p.D) continue;
#pragma unroll
    for (int k = 0; k < kSums; ++k) {
      float v[V];
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = sums.get(k, j, i, d);
      store<float, V>(part + static_cast<long>(k) * p.D + d, v);
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
constexpr int kWide = 4096;      // backward: from here on sixteen values to a thread, the sums over tokens in shared memory

void plan_backward(Plan& q, const ttt_b200_block_args& p) {
  q.width = width_of(p.D, p.D > kWide ? 16 : 8);
  q.side = std::max(1, 128 / q.width);
  const long most = static_cast<long>(sm_count()) * 2;
  q.ctas = static_cast<int>(std::min<long>(most, (p.M + q.side - 1) / q.side));
}

bool rows16(const void* p, int64_t stride, size_t es) { return aligned16(p) && stride * static_cast<int64_t>(es) % 16 == 0; }

bool vectors(const ttt_b200_block_args& p, bool backward) {
  const size_t es = p.dtype == TTT_B200_FP32 ? 4 : 2, rs = p.residual_fp32 ? 4 : es;
  bool ok = p.D % 8 == 0 && rows16(p.o, p.o_stride, es) && rows16(p.residual, p.residual_stride, rs) && rows16(p.gate, p.gate_stride, es);
  for (const float* w : {p.post_weight, p.post_bias, p.scale, p.pre_weight, p.pre_bias}) ok = ok && aligned16(w);
  if (backward)
    return ok && rows16(p.grad_x, p.gx_stride, rs) && rows16(p.grad_n, p.gn_stride, es) && aligned16(p.grad_o) && aligned16(p.grad_residual) &&
           aligned16(p.grad_gate);
  return ok && aligned16(p.x) && aligned16(p.n);
}

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return TTT_B200_OK;
  static thread_local char buf[160];
  snprintf(buf, sizeof buf, "%s: %s", what, cudaGetErrorString(e));
  return ttt_set_error(TTT_B200_ERR_LAUNCH, buf);
}

template <class T, class R> int forward(const ttt_b200_block_args& p, cudaStream_t s) {
  Plan q = {};
  q.width = width_of(p.D, 8);
  q.side = std::max(1, 128 / q.width);
  const long grid = (p.M + q.side - 1) / q.side;
  if (grid > 0x7fffffffL) return fail("block norm: too many tokens");
  q.ctas = static_cast<int>(grid);
  const int threads = q.width * q.side;
  if (vectors(p, false)) block_forward_kernel<T, R, 8, 1><<<q.ctas, threads, 0, s>>>(p, q);
  else block_forward_kernel<T, R, 1, 8><<<q.ctas, threads, 0, s>>>(p, q);
  return launched("block norm");
}

template <class T, class R, int V, int NV, bool kShared> int backward_as(const ttt_b200_block_args& p, const Plan& q, cudaStream_t s) {
  const auto kernel = block_backward_kernel<T, R, V, NV, kShared>;
  const size_t bytes = kShared ? static_cast<size_t>(kSums) * p.D * sizeof(float) : 0;
  if (bytes > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (e != cudaSuccess) return ttt_set_error(TTT_B200_ERR_LAUNCH, cudaGetErrorString(e));
  }
  kernel<<<q.ctas, q.width * q.side, bytes, s>>>(p, q);
  return launched("block norm backward");
}

template <class T, class R> int backward(const ttt_b200_block_args& p, cudaStream_t s) {
  Plan q = {};
  plan_backward(q, p);
  q.part = static_cast<float*>(p.scratch);
  const bool vec = vectors(p, true);
  int rc;
  if (p.D > kWide) rc = vec ? backward_as<T, R, 8, 2, true>(p, q, s) : backward_as<T, R, 1, 16, true>(p, q, s);
  else rc = vec ? backward_as<T, R, 8, 1, false>(p, q, s) : backward_as<T, R, 1, 8, false>(p, q, s);
  if (rc) return rc;
  const long row = static_cast<long>(kSums) * p.D;
  float* dst[kSums] = {p.grad_post_weight, p.grad_post_bias, p.grad_scale, p.grad_pre_weight, p.grad_pre_bias};
  ttt_sum_job jobs[kSums];
  for (int k = 0; k < kSums; ++k)
    jobs[k] = {q.part + static_cast<long>(k) * p.D, dst[k], p.D, row, q.ctas * q.side, TTT_B200_FP32, 0};
  return ttt_sum_parts(jobs, kSums, s);
}

}  // namespace

extern "C" uint64_t ttt_b200_norm_gate_residual_scratch_bytes(const ttt_b200_block_args* p) {
  if (check(p) || p->M == 0) return 0;
  Plan q = {};
  plan_backward(q, *p);
  return static_cast<uint64_t>(q.ctas) * q.side * kSums * p->D * sizeof(float);
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
