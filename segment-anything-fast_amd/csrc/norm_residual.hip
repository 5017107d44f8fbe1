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
  int64_t run;               // rows of a row's threads
  int K;
  int rms;
  float eps_post, eps_pre, branch_scale, residual_scale, inv_K;
};

constexpr int kNormMaxWidth = 32768;

// E values from p on, as they lie in memory; the first n of them in a row's last piece, the others 0
template <class V, int E>
struct Piece {
  unsigned int w[E * sizeof(V) / 4];
  SF_DEVICE void load(const V* p, int n) {
    if (n >= E) {
      __builtin_memcpy(w, p, sizeof(w));
      return;
    }
#pragma unroll
    for (unsigned int i = 0; i < sizeof(w) / 4; ++i) w[i] = 0;
#pragma unroll
    for (int e = 0; e < E - 1; ++e)
      if (e < n) {
        if constexpr (sizeof(V) == 4) w[e] = __float_as_uint(p[e]);
        else w[e / 2] |= (unsigned int)p[e] << (16 * (e & 1));
      }
  }
  template <class T>
  SF_DEVICE float get(int e) const {
    if constexpr (sizeof(V) == 4) return __uint_as_float(w[e]);
    else return e & 1 ? T::hi(w[e / 2]) : T::lo(w[e / 2]);
  }
  template <class T>
  SF_DEVICE void put(const float (&f)[E]) {
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      if constexpr (sizeof(V) == 4) {
        w[e] = __float_as_uint(f[e]);
        w[e + 1] = __float_as_uint(f[e + 1]);
      } else {
        w[e / 2] = T::pack2(f[e], f[e + 1]);
      }
    }
  }
  SF_DEVICE void store(V* p, int n) const {
    if (n >= E) {
      __builtin_memcpy(p, w, sizeof(w));
      return;
    }
#pragma unroll
    for (int e = 0; e < E - 1; ++e)
      if (e < n) {
        if constexpr (sizeof(V) == 4) p[e] = __uint_as_float(w[e]);
        else p[e] = (unsigned short)(w[e / 2] >> (16 * (e & 1)));
      }
  }
};

// THREADS of a row: 64, a wavefront each and four of them to the workgroup; or the whole workgroup.  A thread holds NCH pieces of E values.
// A row's threads go on to the rows behind it (a.run of them), keep the norms' weights and the gate in registers meanwhile and
// request the next row before they work on this one (but 1024 threads, whose 128 registers hold no more than the row).
template <class T, class R, int THREADS, int E, int NCH, bool BETAS>
__global__ __launch_bounds__(THREADS == 64 ? 256 : THREADS) void norm_residual_kernel(NormResidualArgs a) {
  typedef Piece<unsigned short, E> P;
  constexpr bool KEEP = THREADS < 1024;
  constexpr int KEPT = KEEP ? NCH : 1;
  constexpr int WAVES = THREADS / 64;
  __shared__ float part[2][WAVES > 1 ? 4 * WAVES : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row0 = (WAVES > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave) * a.run;
  const int64_t end = min(row0 + a.run, a.M);
  if (row0 >= end) return;
  const int first = (WAVES > 1 ? (int)threadIdx.x : lane) * E;
  const int K = a.K;
  auto at = [&](int i) __attribute__((always_inline)) { return first + i * THREADS * E; };

  P gamma_post[KEPT], beta_post[BETAS ? KEPT : 1], gamma_pre[KEPT], beta_pre[BETAS ? KEPT : 1], gate[KEPT];
  auto fetch = [&](P* to, const unsigned short* from) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < KEPT; ++i)
      if (at(i) < K) to[i].load(from + at(i), K - at(i));
  };
  auto piece = [&](const P* kept, const unsigned short* from, int i) __attribute__((always_inline)) {
    if constexpr (KEEP) return kept[i];
    P p;
    p.load(from + at(i), K - at(i));
    return p;
  };
  Piece<unsigned short, E> xn[NCH];
  Piece<R, E> rn[NCH];
  auto request = [&](int64_t row) __attribute__((always_inline)) {
    const unsigned short* xs = a.x + row * a.ldx;
    const R* rs = reinterpret_cast<const R*>(a.residual) + row * a.ld_res;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (at(i) < K) {
        xn[i].load(xs + at(i), K - at(i));
        rn[i].load(rs + at(i), K - at(i));
      } else {
        xn[i] = {};
        rn[i] = {};
      }
    }
  };
  request(row0);
  if (KEEP && a.gamma_post) fetch(gamma_post, a.gamma_post);
  if (KEEP && BETAS && a.beta_post) fetch(beta_post, a.beta_post);
  if (KEEP && a.gamma_pre) fetch(gamma_pre, a.gamma_pre);
  if (KEEP && BETAS && a.beta_pre) fetch(beta_pre, a.beta_pre);

  int round = 0;
  // (the wavefronts' shares lie in places of their own for each of a row's four sums, and in another set for the next row: one barrier is enough)
  auto sum = [&](float v, int set) __attribute__((always_inline)) {
    v = wave_sum(v);
    if constexpr (WAVES > 1) {
      float* p = part[set] + WAVES * round++;
      if (lane == 0) p[wave] = v;
      __syncthreads();
      v = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) v += p[w];
    }
    return v;
  };
  // f = the row's values; scaled to mean 0 (LayerNorm) and mean square 1, times gamma plus beta
  auto norm = [&](float (&f)[NCH][E], const P* gamma, const unsigned short* gamma_at, const P* beta, const unsigned short* beta_at, float eps,
                  int set) __attribute__((always_inline)) {
    if (!a.rms) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) s += f[i][e];
      const float mean = sum(s, set) * a.inv_K;
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) f[i][e] = at(i) + e < K ? f[i][e] - mean : 0.f;
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) q = fmaf(f[i][e], f[i][e], q);
    const float scale = 1.0f / sqrtf(fmaf(sum(q, set), a.inv_K, eps));
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (at(i) >= K) continue;  // (what lies there stays 0)
      const P g = piece(gamma, gamma_at, i);
#pragma unroll
      for (int e = 0; e < E; ++e) f[i][e] = f[i][e] * scale * g.template get<T>(e);
      if (BETAS && beta_at) {
        const P b = piece(beta, beta_at, i);
#pragma unroll
        for (int e = 0; e < E; ++e) f[i][e] += b.template get<T>(e);
      }
    }
  };

  int64_t gate_row = -1, gate_end = row0;  // the rows up to gate_end share the gate in registers
  for (int64_t row = row0; row < end; ++row) {
    float f[NCH][E];
    Piece<R, E> rc[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      rc[i] = rn[i];
#pragma unroll
      for (int e = 0; e < E; ++e) f[i][e] = xn[i].template get<T>(e);
    }
    if (a.gate && row >= gate_end) {
      gate_row = row / a.group;
      gate_end = (gate_row + 1) * a.group;
      if (KEEP) fetch(gate, a.gate + gate_row * K);
    }
    if (KEEP && row + 1 < end) request(row + 1);
    round = 0;
    const int set = (int)(row - row0) & 1;
    if (a.gamma_post) norm(f, gamma_post, a.gamma_post, beta_post, a.beta_post, a.eps_post, set);
    R* total = reinterpret_cast<R*>(a.total) + row * K;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (at(i) >= K) continue;
      P g = {};
      if (a.gate) g = piece(gate, a.gate + gate_row * K, i);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float v = a.gate ? f[i][e] * g.template get<T>(e) : f[i][e];
        f[i][e] = fmaf(a.residual_scale, rc[i].template get<T>(e), a.branch_scale * v);
        if (at(i) + e >= K) f[i][e] = 0.f;
      }
      Piece<R, E> o;
      o.template put<T>(f[i]);
      o.store(total + at(i), K - at(i));
    }
    if (a.normed) {
      norm(f, gamma_pre, a.gamma_pre, beta_pre, a.beta_pre, a.eps_pre, set);
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        if (at(i) >= K) continue;
        P o;
        o.template put<T>(f[i]);
        o.store(a.normed + row * K + at(i), K - at(i));
      }
    }
    if (!KEEP && row + 1 < end) request(row + 1);
  }
}

template <class T, class R, bool BETAS>
static int launch_norm_residual(NormResidualArgs a, hipStream_t stream) {
  using std::integral_constant;
  // `keep` rows' threads fill the CUs' registers: as many runs of rows as that, all of them as long as one another
  auto go = [&](auto threads, auto e, auto nch, int64_t keep) {
    constexpr int TH = decltype(threads)::value;
    a.run = (a.M + keep - 1) / keep;
    const int64_t runs = (a.M + a.run - 1) / a.run;
    const dim3 grid((unsigned int)(TH == 64 ? (runs + 3) / 4 : runs)), block(TH == 64 ? 256 : TH);
    hipLaunchKernelGGL((norm_residual_kernel<T, R, TH, decltype(e)::value, decltype(nch)::value, BETAS>), grid, block, 0, stream, a);
    return check_launch("norm_residual_kernel");
  };
  using E4 = integral_constant<int, 4>;
  using E8 = integral_constant<int, 8>;
  using N1 = integral_constant<int, 1>;
  using N2 = integral_constant<int, 2>;
  using N3 = integral_constant<int, 3>;
  using N4 = integral_constant<int, 4>;
  using N5 = integral_constant<int, 5>;
  using T1 = integral_constant<int, 64>;
  using T4 = integral_constant<int, 256>;
  using T16 = integral_constant<int, 1024>;
  if (a.K <= 256) return go(T1{}, E4{}, N1{}, 8192);
  if (a.K <= 512) return go(T1{}, E8{}, N1{}, 8192);
  if (a.K <= 768) return go(T1{}, E4{}, N3{}, 4096);
  if (a.K <= 1024) return go(T1{}, E8{}, N2{}, 4096);
  if (a.K <= 1280) return go(T1{}, E4{}, N5{}, 4096);
  if (a.K <= 2048) return go(T1{}, E8{}, N4{}, 3072);
  if (a.K <= 4096) return go(T4{}, E8{}, N2{}, 1024);
  if (a.K <= 8192) return go(T4{}, E8{}, N4{}, 768);
  return go(T16{}, E8{}, N4{}, 256);
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
  a.rms = rms != 0;
  a.eps_post = post_eps;
  a.eps_pre = pre_eps;
  a.branch_scale = branch_scale;
  a.residual_scale = residual_scale;
  a.inv_K = 1.0f / (float)K;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  auto go = [&](auto elem) {
    using T = decltype(elem);
    const bool betas = post_beta || pre_beta;
    if (residual_is_f32) return betas ? launch_norm_residual<T, float, true>(a, s) : launch_norm_residual<T, float, false>(a, s);
    return betas ? launch_norm_residual<T, us, true>(a, s) : launch_norm_residual<T, us, false>(a, s);
  };
  return dtype == SAMFAST_F16 ? go(ElemF16{}) : go(ElemBf16{});
}
