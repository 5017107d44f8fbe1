// A block's end and the next one's beginning in one pass over the rows:
//   total = residual_scale * residual + branch_scale * gate * post(x),   normed = pre(total),
// post and pre a LayerNorm or an RMS norm each, or left out; the gate one row for each group of rows, or left out.
//
// Memory bounds it: x and the residual are read once, total and normed written once, and a row stays in registers between its two
// norms.  Statistics in fp32 from the values themselves (mean first, then the squares of what is left of it); `pre` sees the total
// before it is rounded to the residual's type.
#include "quant_row.hpp"
#include "attn_relpos_shared.hpp"

namespace samfast {

struct NormResidualArgs {
  const unsigned short* x;
  const void* residual;      // T or fp32, as total
  const unsigned short* gate;
  const unsigned short *gamma_post, *beta_post, *gamma_pre, *beta_pre;
  void* total;
  unsigned short* normed;    // null: no pre norm
  int64_t M, ldx, ld_res, group;  // rows that share a gate row
  int K;
  int post, rms;
  float eps_post, eps_pre, branch_scale, residual_scale, inv_K;
};

constexpr int kNormMaxWidth = 32768;

// E values from p on, of which the first n count (the others 0); n >= E everywhere but in a row's last piece
template <class T, int E>
SF_DEVICE void load_values(const unsigned short* p, int n, float* f) {
  if (n >= E) {
    unsigned int w[E / 2];
    __builtin_memcpy(w, p, E * 2);
#pragma unroll
    for (int j = 0; j < E / 2; ++j) {
      f[2 * j] = T::lo(w[j]);
      f[2 * j + 1] = T::hi(w[j]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = e < n ? T::from_bits(p[e]) : 0.f;
  }
}
template <class T, int E>
SF_DEVICE void load_values(const float* p, int n, float* f) {
  if (n >= E) {
    __builtin_memcpy(f, p, E * 4);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = e < n ? p[e] : 0.f;
  }
}
template <class T, int E>
SF_DEVICE void store_values(unsigned short* p, int n, const float* f) {
  unsigned int w[E / 2];
#pragma unroll
  for (int j = 0; j < E / 2; ++j) w[j] = T::pack2(f[2 * j], f[2 * j + 1]);
  if (n >= E) {
    __builtin_memcpy(p, w, E * 2);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < n) p[e] = (unsigned short)(w[e >> 1] >> (16 * (e & 1)));
  }
}
template <class T, int E>
SF_DEVICE void store_values(float* p, int n, const float* f) {
  if (n >= E) {
    __builtin_memcpy(p, f, E * 4);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < n) p[e] = f[e];
  }
}

// THREADS of a row: 64, a wavefront each and four rows to the workgroup; or the whole workgroup.  A thread holds NCH pieces of E values.
template <class T, class R, int THREADS, int E, int NCH>
__global__ __launch_bounds__(THREADS == 64 ? 256 : THREADS) void norm_residual_kernel(NormResidualArgs a) {
  constexpr int WAVES = THREADS / 64;
  __shared__ float part[WAVES > 1 ? 4 * WAVES : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = WAVES > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
  if (WAVES == 1 && row >= a.M) return;
  const int first = (WAVES > 1 ? (int)threadIdx.x : lane) * E;
  const unsigned short* xs = a.x + row * a.ldx;
  const R* rs = reinterpret_cast<const R*>(a.residual) + row * a.ld_res;
  const int K = a.K;

  int round = 0;
  auto sum = [&](float v) __attribute__((always_inline)) {
    v = wave_sum(v);
    if constexpr (WAVES > 1) {  // (a place of its own for each of the four sums: no barrier behind the reading)
      float* p = part + WAVES * round++;
      if (lane == 0) p[wave] = v;
      __syncthreads();
      v = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) v += p[w];
    }
    return v;
  };
  // f = the row's values; scaled to mean 0 (LayerNorm) and mean square 1, times gamma plus beta
  auto norm = [&](float (&f)[NCH][E], const unsigned short* gamma, const unsigned short* beta, float eps) __attribute__((always_inline)) {
    if (!a.rms) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) s += f[i][e];
      const float mean = sum(s) * a.inv_K;
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const int n = K - first - i * THREADS * E;
#pragma unroll
        for (int e = 0; e < E; ++e) f[i][e] = e < n ? f[i][e] - mean : 0.f;
      }
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) q = fmaf(f[i][e], f[i][e], q);
    const float scale = 1.0f / sqrtf(fmaf(sum(q), a.inv_K, eps));
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int d = first + i * THREADS * E, n = K - d;
      if (n <= 0) continue;
      float g[E], b[E];
      load_values<T, E>(gamma + d, n, g);
      if (beta) load_values<T, E>(beta + d, n, b);
#pragma unroll
      for (int e = 0; e < E; ++e) f[i][e] = beta ? fmaf(f[i][e] * scale, g[e], b[e]) : f[i][e] * scale * g[e];
    }
  };

  float f[NCH][E], r[NCH][E];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int d = first + i * THREADS * E, n = K - d;
#pragma unroll
    for (int e = 0; e < E; ++e) f[i][e] = r[i][e] = 0.f;
    if (n > 0) {
      load_values<T, E>(xs + d, n, f[i]);
      load_values<T, E>(rs + d, n, r[i]);
    }
  }
  if (a.post) norm(f, a.gamma_post, a.beta_post, a.eps_post);
  const unsigned short* gate = a.gate ? a.gate + row / a.group * K : nullptr;
  R* total = reinterpret_cast<R*>(a.total) + row * K;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int d = first + i * THREADS * E, n = K - d;
    if (n <= 0) continue;
    if (gate) {
      float g[E];
      load_values<T, E>(gate + d, n, g);
#pragma unroll
      for (int e = 0; e < E; ++e) f[i][e] *= g[e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) f[i][e] = fmaf(a.residual_scale, r[i][e], a.branch_scale * f[i][e]);
    store_values<T, E>(total + d, n, f[i]);
  }
  if (!a.normed) return;
  norm(f, a.gamma_pre, a.beta_pre, a.eps_pre);
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int d = first + i * THREADS * E, n = K - d;
    if (n > 0) store_values<T, E>(a.normed + row * K + d, n, f[i]);
  }
}

template <class T, class R>
static int launch_norm_residual(const NormResidualArgs& a, hipStream_t stream) {
  using std::integral_constant;
  auto go = [&](auto threads, auto e, auto nch) {
    constexpr int TH = decltype(threads)::value;
    const dim3 grid((unsigned int)(TH == 64 ? (a.M + 3) / 4 : a.M)), block(TH == 64 ? 256 : TH);
    hipLaunchKernelGGL((norm_residual_kernel<T, R, TH, decltype(e)::value, decltype(nch)::value>), grid, block, 0, stream, a);
    return check_launch("norm_residual_kernel");
  };
  using E4 = integral_constant<int, 4>;
  using E8 = integral_constant<int, 8>;
  using N1 = integral_constant<int, 1>;
  using N2 = integral_constant<int, 2>;
  using N4 = integral_constant<int, 4>;
  if (a.K <= 256) return go(integral_constant<int, 64>{}, E4{}, N1{});
  if (a.K <= 512) return go(integral_constant<int, 64>{}, E8{}, N1{});
  if (a.K <= 1024) return go(integral_constant<int, 256>{}, E4{}, N1{});
  if (a.K <= 2048) return go(integral_constant<int, 256>{}, E8{}, N1{});
  if (a.K <= 4096) return go(integral_constant<int, 256>{}, E8{}, N2{});
  if (a.K <= 8192) return go(integral_constant<int, 256>{}, E8{}, N4{});
  return go(integral_constant<int, 1024>{}, E8{}, N4{});
}

}  // namespace samfast

extern "C" int samfast_norm_residual(const void* x, int64_t ldx, const void* residual, int64_t ld_res, const void* gate, int64_t gate_rows,
                                     const void* post_gamma, const void* post_beta, float post_eps,
                                     const void* pre_gamma, const void* pre_beta, float pre_eps, int rms,
                                     float branch_scale, float residual_scale, void* total, void* normed,
                                     int64_t M, int K, int dtype, int residual_is_f32, void* stream) {
  using namespace samfast;
  using us = unsigned short;
  if (dtype != SAMFAST_BF16 && dtype != SAMFAST_F16) SF_FAIL(SAMFAST_E_UNSUPPORTED, "norm_residual: element type %d is neither SAMFAST_BF16 nor SAMFAST_F16", dtype);
  SF_REQUIRE(M >= 0 && K > 0 && K <= kNormMaxWidth, "norm_residual: bad shape M=%lld K=%d (K at most %d)", (long long)M, K, kNormMaxWidth);
  SF_REQUIRE(M < (1ll << 31), "norm_residual: M too large");
  SF_REQUIRE(M == 0 || (pre_gamma == nullptr) == (normed == nullptr), "norm_residual: the pre norm's weight and the normed rows go together");
  SF_REQUIRE((post_gamma || !post_beta) && (pre_gamma || !pre_beta), "norm_residual: a bias without its weight");
  SF_REQUIRE(!gate || (gate_rows >= 1 && M % gate_rows == 0), "norm_residual: %lld rows do not share %lld gate rows evenly", (long long)M, (long long)gate_rows);
  SF_REQUIRE(post_eps >= 0.f && pre_eps >= 0.f, "norm_residual: eps must not be negative");
  SF_REQUIRE(M == 0 || (x && residual && total), "norm_residual: null pointer");
  SF_REQUIRE(ldx >= K && ld_res >= K, "norm_residual: row strides must hold a row");
  if (M == 0) return SAMFAST_OK;
  NormResidualArgs a = {};
  a.x = (const us*)x;
  a.residual = residual;
  a.gate = (const us*)gate;
  a.gamma_post = (const us*)post_gamma;
  a.beta_post = (const us*)post_beta;
  a.gamma_pre = (const us*)pre_gamma;
  a.beta_pre = (const us*)pre_beta;
  a.total = total;
  a.normed = (us*)normed;
  a.M = M;
  a.ldx = ldx;
  a.ld_res = ld_res;
  a.group = gate ? M / gate_rows : 1;
  a.K = K;
  a.post = post_gamma != nullptr;
  a.rms = rms != 0;
  a.eps_post = post_eps;
  a.eps_pre = pre_eps;
  a.branch_scale = branch_scale;
  a.residual_scale = residual_scale;
  a.inv_K = 1.0f / (float)K;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == SAMFAST_F16) return residual_is_f32 ? launch_norm_residual<ElemF16, float>(a, s) : launch_norm_residual<ElemF16, us>(a, s);
  return residual_is_f32 ? launch_norm_residual<ElemBf16, float>(a, s) : launch_norm_residual<ElemBf16, us>(a, s);
}
