// The end of a block and the start of the next: backward.
//
// Measured with all parts, the kernel by itself (the sum of its parts is 4 to 7 us more, of rows of up to 512 values 13 to 24), 16384 x 2048 bf16: fp32
// residual stream, layer norms, tanh gate 155 us (4.8 TB/s), all in fp32 177 us (6.1); bf16 residual, RMS norms 141 us (3.8 TB/s), a residual and the
// next norm alone 81 us (5.0); rows of 2047 216 us (3.4) and 204 us (2.6).  Rows that do not fill their threads, fp32 residual: 16384 x 1536 153 us
// (3.6), 32768 x 768 142 us (3.9).  65536 x 512, whose kernels spill (up to 132 bytes), 171 us (4.3).  4096 x 8192, layer norms, sums in shared memory and
// nothing copied ahead: 282 us (2.6), with a bf16 residual 324 us (1.7).  512 threads to an SM, since a thread has 128 registers, 40 of them sums
// over tokens; each wait (two barriers a token, the L1 for the weights) shows.
#include "ttt_block_norm.cuh"

namespace {

using namespace ttt;
using namespace ttt::block;

// Sums over tokens of a thread's columns: in registers, or, of sixteen columns, in shared memory.
enum { kDw1, kDb1, kDsc, kDw2, kDb2, kSums };
template <class C, int NV, bool kShared> struct Sums {
  F r[kShared ? 1 : kSums][NV][N];
  float* s;
  __device__ __forceinline__ F get(int k, int j, int i, const C& c) const {
    if constexpr (!kShared) return r[k][j][i];
    else if constexpr (C::V > 1) return c.in(j, 2 * i) ? *reinterpret_cast<const F*>(s + k * c.D + c.at(j, 2 * i)) : both(0.f);
    else return make_float2(c.in(j, 2 * i) ? s[k * c.D + c.at(j, 2 * i)] : 0.f, c.in(j, 2 * i + 1) ? s[k * c.D + c.at(j, 2 * i + 1)] : 0.f);
  }
  __device__ __forceinline__ void set(int k, int j, int i, const C& c, F v) {
    if constexpr (!kShared) {
      r[k][j][i] = v;
    } else if constexpr (C::V > 1) {
      if (c.in(j, 2 * i)) *reinterpret_cast<F*>(s + k * c.D + c.at(j, 2 * i)) = v;
    } else {
      if (c.in(j, 2 * i)) s[k * c.D + c.at(j, 2 * i)] = v.x;
      if (c.in(j, 2 * i + 1)) s[k * c.D + c.at(j, 2 * i + 1)] = v.y;
    }
  }
  __device__ __forceinline__ void add(int k, int j, int i, const C& c, F v) { set(k, j, i, c, add2(get(k, j, i, c), v)); }
  __device__ __forceinline__ void add(int k, int j, int i, const C& c, F a, F b) { set(k, j, i, c, fma2(a, b, get(k, j, i, c))); }
};

template <class T, class R, class C, int NV, bool kShared>
__global__ void __launch_bounds__(C::threads, 512 / C::threads) block_backward_kernel(const ttt_b200_block_args p, const Plan q) {
  wait_for_predecessor();
  constexpr int kMode = kShared ? kDirect : C::V > 1 ? kOwn : kWindow;
  __shared__ Shared sh;
  extern __shared__ __align__(16) unsigned char stages[];
  uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(stages));
  int buf = 0;
  const int lane = threadIdx.x % C::width, sub = threadIdx.x / C::width;
  const C c = {lane, p.D};
  const long step = static_cast<long>(q.ctas) * C::side;
  constexpr bool kMore = C::all || C::bare;
  const bool post = !C::bare && (C::all || p.post_weight), gated = !C::bare && (C::all || p.gate), pre = kMore || p.pre_weight;
  const Feed<T, C, kMode, true> fo(p.o, p.o_stride, at, p.D);
  const Feed<T, C, kMode, C::all> fg(gated ? p.gate : nullptr, p.gate_stride, at, p.D);
  const Feed<T, C, kMode, kMore> fn(pre ? p.grad_n : nullptr, p.gn_stride, at, p.D);
  const Feed<R, C, kMode, kMore> fx(pre ? p.residual : nullptr, p.residual_stride, at, p.D);
  const Feed<R, C, kMode, kMore> fd(p.grad_x, p.gx_stride, at, p.D);
  const uint32_t small = Feed<T, C, kMode, true>::bytes(p.D), large = Feed<R, C, kMode, true>::bytes(p.D);
  const uint32_t stats = static_cast<uint32_t>(__cvta_generic_to_shared(&sh.stats[0][threadIdx.x >> 5]));
  auto ahead = [&](long m, int stage) {
    if (m < p.M) {
      if ((threadIdx.x & 31) == 0) cp_async16_at(stats + stage * static_cast<uint32_t>(sizeof(sh.stats[0])), p.stats + 4 * m);
      fo.ahead(m, stage * small, c, sub);
      fg.ahead(m, stage * small, c, sub);
      fn.ahead(m, stage * small, c, sub);
      fx.ahead(m, stage * large, c, sub);
      fd.ahead(m, stage * large, c, sub);
    }
    cp_async_commit();
  };
  const float inv = 1.f / static_cast<float>(p.D);
  Sums<C, NV, kShared> sums;
  sums.s = reinterpret_cast<float*>(stages);
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (!kShared || c.in(j)) {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int k = 0; k < kSums; ++k) sums.set(k, j, i, c, both(0.f));
    }
  long m = static_cast<long>(blockIdx.x) * C::side + sub;
  ahead(m, 0);
  int stage = 0;
  for (long base = static_cast<long>(blockIdx.x) * C::side; base < p.M; base += step, stage ^= 1, m += step) {
    const bool live = m < p.M;
    cp_async_wait<0>();
    if constexpr (kMode == kWindow) __syncthreads();
    else __syncwarp();
    ahead(m + step, stage ^ 1);
    float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live) st = sh.stats[stage][threadIdx.x >> 5];
    F o[NV][N], z[NV][N], gn[NV][N], d2[NV][N];
    // u (with its norm: oh) and z again, as the forward had them; z is its normalised value
    F sx = both(0.f), sy = sx;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const bool in = live && c.in(j);
#pragma unroll
      for (int i = 0; i < N; ++i) o[j][i] = both(0.f);
      if (in) fo.get(m, stage * small, c, j, sub, o[j]);
      if (post) {
#pragma unroll
        for (int i = 0; i < N; ++i) o[j][i] = times(plus(o[j][i], both(-st.x)), both(st.y));
      }
      if (!pre || !in) continue;
      F u[N], w[N], b[N];
#pragma unroll
      for (int i = 0; i < N; ++i) u[i] = o[j][i];
      if (post) {
        weights<C::all>(p.post_weight, c, j, 0.f, w);
        weights(p.post_bias, c, j, 0.f, b);
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = mac(o[j][i], w[i], b[i]);
      }
      if (gated) {
        fg.get(m, stage * small, c, j, sub, w);
        gate<false>(p.activation, w, w, b);
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = times(u[i], w[i]);
      }
      weights<C::all>(C::bare ? nullptr : p.scale, c, j, 1.f, w);
      fx.get(m, stage * large, c, j, sub, z[j]);
#pragma unroll
      for (int i = 0; i < N; ++i) z[j][i] = times(plus(mac(w[i], u[i], z[j][i]), both(-st.z)), both(st.w));
      fn.get(m, stage * small, c, j, sub, gn[j]);
      weights<kMore>(p.pre_weight, c, j, 0.f, w);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        sums.add(kDw2, j, i, c, gn[j][i], z[j][i]);
        sums.add(kDb2, j, i, c, gn[j][i]);
        gn[j][i] = times(gn[j][i], w[i]);
        sx = plus(sx, gn[j][i]);
        sy = mac(gn[j][i], z[j][i], sy);
      }
    }
    float2 s = make_float2(fold(sx), fold(sy));
    float m1 = 0.f, m2 = 0.f;
    if (pre) {
      s = row_sum<C>(s, sh.part, buf);
      m1 = p.layer ? s.x * inv : 0.f;
      m2 = s.y * inv;
    }
    sx = sy = both(0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!(live && c.in(j))) continue;
      fd.get(m, stage * large, c, j, sub, d2[j]);
      if (pre) {
#pragma unroll
        for (int i = 0; i < N; ++i) d2[j][i] = mac(both(st.w), mac(z[j][i], both(-m2), plus(gn[j][i], both(-m1))), d2[j][i]);
      }
      if (kMore || p.grad_residual) store(static_cast<R*>(p.grad_residual) + m * p.D, c, j, d2[j]);
      F u[N], w[N], b[N], v[N], g[N];
#pragma unroll
      for (int i = 0; i < N; ++i) u[i] = o[j][i];
      if (post) {
        weights<C::all>(p.post_weight, c, j, 0.f, w);
        weights(p.post_bias, c, j, 0.f, b);
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = mac(o[j][i], w[i], b[i]);
      }
      weights<C::all>(C::bare ? nullptr : p.scale, c, j, 1.f, b);
      if (gated) {
        fg.get(m, stage * small, c, j, sub, g);
        gate<true>(p.activation, g, v, g);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          sums.add(kDsc, j, i, c, d2[j][i], times(u[i], v[i]));
          d2[j][i] = times(d2[j][i], b[i]);
          g[i] = times(times(d2[j][i], u[i]), g[i]);
          d2[j][i] = times(d2[j][i], v[i]);
        }
        store(static_cast<T*>(p.grad_gate) + m * p.D, c, j, g);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (!C::bare) sums.add(kDsc, j, i, c, d2[j][i], u[i]);
          d2[j][i] = times(d2[j][i], b[i]);
        }
      }
      if (post) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          sums.add(kDw1, j, i, c, d2[j][i], o[j][i]);
          sums.add(kDb1, j, i, c, d2[j][i]);
          d2[j][i] = times(d2[j][i], w[i]);
          sx = plus(sx, d2[j][i]);
          sy = mac(d2[j][i], o[j][i], sy);
        }
      }
    }
    if (post) {
      s = row_sum<C>(make_float2(fold(sx), fold(sy)), sh.part, buf);
      m1 = p.layer ? s.x * inv : 0.f;
      m2 = s.y * inv;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!(live && c.in(j))) continue;
      if (post) {
#pragma unroll
        for (int i = 0; i < N; ++i) d2[j][i] = times(both(st.y), mac(o[j][i], both(-m2), plus(d2[j][i], both(-m1))));
      }
      store(static_cast<T*>(p.grad_o) + m * p.D, c, j, d2[j]);
    }
  }
  float* part = q.part + (static_cast<long>(blockIdx.x) * C::side + sub) * kSums * p.D;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (!c.in(j)) continue;
#pragma unroll
    for (int k = 0; k < kSums; ++k) {
      F v[N];
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = sums.get(k, j, i, c);
      store(part + static_cast<long>(k) * p.D, c, j, v);
    }
  }
}

template <class T, class R, class C, int NV, bool kShared> int backward_as(const ttt_b200_block_args& p, const Plan& q, cudaStream_t s) {
  constexpr int kMode = kShared ? kDirect : C::V > 1 ? kOwn : kWindow;
  const size_t bytes = kShared ? static_cast<size_t>(kSums) * p.D * sizeof(float)
                               : 2 * (Feed<T, C, kMode, true>::bytes(p.D) * (1 + (p.gate != nullptr) + (p.pre_weight && p.grad_n)) +
                                      Feed<R, C, kMode, true>::bytes(p.D) * ((p.pre_weight && p.residual) + (p.grad_x != nullptr)));
  return launch<block_backward_kernel<T, R, C, NV, kShared>>(q, bytes, s, p, "block norm backward");
}
template <class T, class R, int kWidth, int NV, int kParts> int backward_with(const ttt_b200_block_args& p, const Plan& q, cudaStream_t s) {
  if (!vectors(p, true, kRun<R>)) return backward_as<T, R, Cols<1, kWidth, false, kParts>, NV, (NV > 1)>(p, q, s);
  return p.D == 8 * NV * kWidth ? backward_as<T, R, Cols<kRun<R>, kWidth, true, kParts>, NV, (NV > 1)>(p, q, s)
                                : backward_as<T, R, Cols<kRun<R>, kWidth, false, kParts>, NV, (NV > 1)>(p, q, s);
}
template <class T, class R, int kWidth, int NV = 1> int backward_of(const ttt_b200_block_args& p, const Plan& q, cudaStream_t s) {
  switch (p.grad_x && p.grad_n ? parts_of(p) : kSome) {
    case kAll: return backward_with<T, R, kWidth, NV, kAll>(p, q, s);
    case kBare: return backward_with<T, R, kWidth, NV, kBare>(p, q, s);
    default: return backward_with<T, R, kWidth, NV, kSome>(p, q, s);
  }
}
template <class T, class R> int backward_kernel(const ttt_b200_block_args& p, const Plan& q, cudaStream_t s) {
  if (p.D > kWide) return backward_of<T, R, 512, 2>(p, q, s);
  switch (q.width) {
    case 32: return backward_of<T, R, 32>(p, q, s);
    case 64: return backward_of<T, R, 64>(p, q, s);
    case 128: return backward_of<T, R, 128>(p, q, s);
    case 256: return backward_of<T, R, 256>(p, q, s);
    default: return backward_of<T, R, 512>(p, q, s);
  }
}

template <class T, class R> int backward(const ttt_b200_block_args& p, cudaStream_t s) {
  Plan q = {};
  plan(q, p, true);
  q.part = static_cast<float*>(p.scratch);
  const int rc = backward_kernel<T, R>(p, q, s);
  if (rc) return rc;
  const long row = static_cast<long>(kSums) * p.D;
  float* dst[kSums] = {p.grad_post_weight, p.grad_post_bias, p.grad_scale, p.grad_pre_weight, p.grad_pre_bias};
  ttt_sum_job jobs[kSums];
  for (int k = 0; k < kSums; ++k)
    jobs[k] = {q.part + static_cast<long>(k) * p.D, dst[k], p.D, row, q.ctas * side_of(q.width), TTT_B200_FP32, 0};
  return ttt_sum_parts(jobs, kSums, s);
}

}  // namespace

extern "C" uint64_t ttt_b200_norm_gate_residual_scratch_bytes(const ttt_b200_block_args* p) {
  if (check(p) || p->M == 0) return 0;
  Plan q = {};
  plan(q, *p, true);
  return static_cast<uint64_t>(q.ctas) * side_of(q.width) * kSums * p->D * sizeof(float);
}

extern "C" int ttt_b200_norm_gate_residual_backward(const ttt_b200_block_args* p, void* stream) {
  if (int rc = check(p)) return rc;
  if (!p->o || !p->stats || !p->grad_o || (!p->grad_x && !p->grad_n) || (p->gate && !p->grad_gate) || (p->residual && !p->grad_residual)) return fail("block norm backward: null tensor pointer");
  if (!aligned16(p->stats)) return fail("block norm backward: stats must be 16-byte aligned");
  if (p->M == 0) return fail("block norm backward: no tokens");
  if (!p->scratch || p->scratch_bytes < ttt_b200_norm_gate_residual_scratch_bytes(p) || !aligned16(p->scratch))
    return fail("block norm backward: scratch is missing, too small or not 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  TTT_WITH_TYPE(p->dtype, return p->residual_fp32 ? (backward<Elem, float>(*p, s)) : (backward<Elem, Elem>(*p, s)))
  return TTT_B200_OK;
}
