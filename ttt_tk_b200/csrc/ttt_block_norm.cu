// The end of a block and the start of the next: forward.
//
// Measured with all parts, 16384 x 2048 bf16: fp32 residual stream, layer norms, tanh gate 87 us (5.4 TB/s), all in fp32 102 us (6.6); bf16
// residual, RMS norms 68 us (4.9 TB/s); rows of 2047 127 us (3.7) and 106 us (3.2); a bf16 residual and the next RMS norm alone 42 us (6.3 TB/s).  Rows
// that do not fill their threads, fp32 residual: 16384 x 1536 83 us (4.2), 32768 x 768 81 us (4.3); 4096 x 8192 100 us (4.7).  Issued instructions and
// the wait at a token's barriers are what is left above the memory: 1024 threads to an SM (1280: 106 us where 1024 had 97, since the L1 has less
// room for the weights).
#include "ttt_block_norm.cuh"

namespace {

using namespace ttt;
using namespace ttt::block;

template <class T, class R, class C>
__global__ void __launch_bounds__(C::threads, 1024 / C::threads) block_forward_kernel(const ttt_b200_block_args p, const Plan q) {
  wait_for_predecessor();
  constexpr int kMode = C::V > 1 ? kOwn : kWindow, NV = 1;
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
  const Feed<R, C, kMode, kMore> fx(p.residual, p.residual_stride, at, p.D);
  const uint32_t small = Feed<T, C, kMode, true>::bytes(p.D), large = Feed<R, C, kMode, true>::bytes(p.D);
  auto ahead = [&](long m, int stage) {
    if (m < p.M) {
      fo.ahead(m, stage * small, c, sub);
      fg.ahead(m, stage * small, c, sub);
      fx.ahead(m, stage * large, c, sub);
    }
    cp_async_commit();
  };
  long m = static_cast<long>(blockIdx.x) * C::side + sub;
  ahead(m, 0);
  count_columns<NV>(sh, c);
  int stage = 0;
  for (long base = static_cast<long>(blockIdx.x) * C::side; base < p.M; base += step, stage ^= 1, m += step) {
    const bool live = m < p.M;
    cp_async_wait<0>();
    if constexpr (kMode == kWindow) __syncthreads();
    ahead(m + step, stage ^ 1);
    F a[NV][N], z[NV][N];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int k = 0; k < N; ++k) a[j][k] = z[j][k] = both(0.f);
      if (live && c.in(j)) fo.get(m, stage * small, c, j, sub, a[j]);
    }
    float2 s1 = make_float2(0.f, 1.f), s2 = s1;
    if (post) s1 = statistics<NV>(a, p, c, sh, buf);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!(live && c.in(j))) continue;
      F w[N], b[N];
      if (post) {
        weights<C::all>(p.post_weight, c, j, 0.f, w);
        weights(p.post_bias, c, j, 0.f, b);
#pragma unroll
        for (int k = 0; k < N; ++k) a[j][k] = mac(times(plus(a[j][k], both(-s1.x)), both(s1.y)), w[k], b[k]);
      }
      if (gated) {
        F g[N];
        fg.get(m, stage * small, c, j, sub, g);
        gate<false>(p.activation, g, g, w);
#pragma unroll
        for (int k = 0; k < N; ++k) a[j][k] = times(a[j][k], g[k]);
      }
      fx.get(m, stage * large, c, j, sub, z[j]);
      weights<C::all>(C::bare ? nullptr : p.scale, c, j, 1.f, w);
#pragma unroll
      for (int k = 0; k < N; ++k) z[j][k] = mac(w[k], a[j][k], z[j][k]);
      store(static_cast<R*>(p.x) + m * p.D, c, j, z[j]);
    }
    if (pre) {
      s2 = statistics<NV>(z, p, c, sh, buf);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (live && c.in(j)) {
          F w[N], b[N];
          weights<kMore>(p.pre_weight, c, j, 0.f, w);
          weights(p.pre_bias, c, j, 0.f, b);
#pragma unroll
          for (int k = 0; k < N; ++k) z[j][k] = mac(times(plus(z[j][k], both(-s2.x)), both(s2.y)), w[k], b[k]);
          store(static_cast<T*>(p.n) + m * p.D, c, j, z[j]);
        }
      }
    }
    if (p.stats && live && lane == 0) reinterpret_cast<float4*>(p.stats)[m] = make_float4(s1.x, s1.y, s2.x, s2.y);
  }
}

template <class T, class R, class C> int forward_as(const ttt_b200_block_args& p, const Plan& q, cudaStream_t s) {
  constexpr int kMode = C::V > 1 ? kOwn : kWindow;
  const size_t bytes = 2 * (Feed<T, C, kMode, true>::bytes(p.D) * (1 + (p.gate != nullptr)) + Feed<R, C, kMode, true>::bytes(p.D) * (p.residual != nullptr));
  return launch<block_forward_kernel<T, R, C>>(q, bytes, s, p, "block norm");
}
template <class T, class R, int kWidth, int kParts> int forward_with(const ttt_b200_block_args& p, const Plan& q, cudaStream_t s) {
  if (!vectors(p, false, kRun<R>)) return forward_as<T, R, Cols<1, kWidth, false, kParts>>(p, q, s);
  return p.D == 8 * kWidth ? forward_as<T, R, Cols<kRun<R>, kWidth, true, kParts>>(p, q, s)
                           : forward_as<T, R, Cols<kRun<R>, kWidth, false, kParts>>(p, q, s);
}
template <class T, class R, int kWidth> int forward_of(const ttt_b200_block_args& p, const Plan& q, cudaStream_t s) {
  switch (parts_of(p)) {
    case kAll: return forward_with<T, R, kWidth, kAll>(p, q, s);
    case kBare: return forward_with<T, R, kWidth, kBare>(p, q, s);
    default: return forward_with<T, R, kWidth, kSome>(p, q, s);
  }
}

template <class T, class R> int forward(const ttt_b200_block_args& p, cudaStream_t s) {
  Plan q = {};
  plan(q, p, false);
  switch (q.width) {
    case 32: return forward_of<T, R, 32>(p, q, s);
    case 64: return forward_of<T, R, 64>(p, q, s);
    case 128: return forward_of<T, R, 128>(p, q, s);
    case 256: return forward_of<T, R, 256>(p, q, s);
    case 512: return forward_of<T, R, 512>(p, q, s);
    default: return forward_of<T, R, 1024>(p, q, s);
  }
}

}  // namespace

extern "C" int ttt_b200_norm_gate_residual(const ttt_b200_block_args* p, void* stream) {
  if (int rc = check(p)) return rc;
  if (!p->o || !p->x || (p->pre_weight && !p->n)) return fail("block norm: null tensor pointer");
  if (p->stats && !aligned16(p->stats)) return fail("block norm: stats must be 16-byte aligned");
  if (p->M == 0) return fail("block norm: no tokens");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  TTT_WITH_TYPE(p->dtype, return p->residual_fp32 ? (forward<Elem, float>(*p, s)) : (forward<Elem, Elem>(*p, s)))
  return TTT_B200_OK;
}
