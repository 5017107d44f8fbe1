// A block's end and the next one's beginning in one pass over the rows:
//   total = residual_scale * residual + branch_scale * gate * post(x),   normed = pre(total),
// post and pre a LayerNorm or an RMS norm each, or left out; the gate one row for each group of rows, or left out.
//
// Memory bounds it: x and the residual are read once, total and normed written once, and a row stays in registers between its two
// norms.  Statistics in fp32 from the values themselves (mean first, then the squares of what is left of it); `pre` sees the total
// before it is rounded to the residual's type.
#include "quant_row.hpp"
#include "attn_relpos_shared.hpp"

#include <type_traits>

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
  int halves, rows;          // of a workgroup: halves of wavefronts to a row, rows
  int in_place;
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

SF_DEVICE float half_sum(float v) {  // over 32 lanes: wave_reduce without its last step
  v += dpp_f32<0xB1>(v);
  v += dpp_f32<0x4E>(v);
  v += dpp_f32<0x141>(v);
  v += dpp_f32<0x140>(v);
  typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
  const unsigned int b = __float_as_uint(v);
  const u32x2_t r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// 32 lanes hold 256 NCH values of a row, and as many halves of wavefronts as that takes, `halves`, make up a row's threads: with an odd number
// two rows share a workgroup and its middle wavefront (768 in pieces for a thread each: three halves).  A thread has NCH pieces of 16 bytes
// (of 8: 65536 x 1280 238 us for 150).  What was behind that, all of it with fewer rows in flight: two rows to a thread, which then
// share the norms' weights, 43008 x 2048 131 us for 133, but onto fp32, 21504 x 2048, 113 for 101; threads that go on to other rows with the weights kept in
// registers, 65536 x 1280 143-180, 5003 x 8192 onto fp32 110-130.  The weights come out of the caches.
// WHOLE: K is a multiple of the pieces.
template <class T, class R, int NCH, bool WHOLE>
__global__ __launch_bounds__(1024) void norm_residual_kernel(NormResidualArgs a) {
  constexpr int E = 8;
  typedef Piece<unsigned short, E> P;
  __shared__ float part[4][32];
  const int lane = threadIdx.x & 63, half = (int)threadIdx.x >> 5;
  const int mine = half >= a.halves;  // which of the workgroup's rows
  const int64_t row = (int64_t)blockIdx.x * a.rows + mine;
  const bool idle = half >= a.rows * a.halves || row >= a.M;  // (it meets the others at the barriers)
  const int threads = 32 * a.halves, K = idle ? 0 : a.K;
  const int first = ((int)threadIdx.x - mine * threads) * E;
  // Where piece i lies.  One that would end behind its row lies over the one before it, so that it is whole too (one value after the other, 44058 x 1999 took 245 us for 167); the
  // values that belong to that one, below owned(i), are not summed.
  auto owned = [&](int i) __attribute__((always_inline)) { return first + i * threads * E; };
  auto at = [&](int i) __attribute__((always_inline)) { return !WHOLE && K >= E && owned(i) < K ? min(owned(i), K - E) : owned(i); };
  auto counts = [&](int i, int e) __attribute__((always_inline)) { return WHOLE || at(i) + e >= owned(i); };
  auto length = [&](int i) __attribute__((always_inline)) { return WHOLE ? E : K - at(i); };

  // everything is requested before anything is waited for, if there are registers for it
  constexpr bool AHEAD = NCH <= 2;
  const unsigned short* gate = a.gate ? a.gate + row / a.group * K : nullptr;
  const unsigned short* const from[5] = {a.gamma_post, a.beta_post, gate, a.gamma_pre, a.beta_pre};
  P ahead[AHEAD ? 5 : 1][NCH];
  Piece<unsigned short, E> xw[NCH];
  Piece<R, E> rw[NCH];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    if (at(i) < K) {
      xw[i].load(a.x + row * a.ldx + at(i), length(i));
      rw[i].load(reinterpret_cast<const R*>(a.residual) + row * a.ld_res + at(i), length(i));
    } else {
      xw[i] = {};
      rw[i] = {};
    }
  }
  if constexpr (AHEAD) {
#pragma unroll
    for (int j = 0; j < 5; ++j)
#pragma unroll
      for (int i = 0; i < NCH; ++i)
        if (from[j] && at(i) < K) ahead[j][i].load(from[j] + at(i), length(i));
  }
  if (!WHOLE && a.in_place) {  // two threads read some of a row's values: before either of them writes
    __builtin_amdgcn_s_waitcnt(0x0f70);
    __syncthreads();
  }
  auto weights = [&](int j, int i) __attribute__((always_inline)) {
    if constexpr (AHEAD) return ahead[j][i];
    P p;
    p.load(from[j] + at(i), length(i));
    return p;
  };

  int round = 0;
  auto sum = [&](float v) __attribute__((always_inline)) {
    v = half_sum(v);
    float* p = part[round++];  // (a place of its own for each of the four sums: no barrier behind the reading)
    if ((lane & 31) == 0) p[half] = v;
    __syncthreads();
    return half_sum(!idle && (lane & 31) < a.halves ? p[mine * a.halves + (lane & 31)] : 0.f);  // (an idle half may have no place of its own)
  };
  // f = the row's values; scaled to mean 0 (LayerNorm) and mean square 1, times weights(j) plus weights(j + 1)
  float f[NCH][E];
  auto norm = [&](int j, float eps) __attribute__((always_inline)) {
    if (!a.rms) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) s += counts(i, e) ? f[i][e] : 0.f;
      const float mean = sum(s) * a.inv_K;
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) f[i][e] = at(i) + (WHOLE ? 0 : e) < K ? f[i][e] - mean : 0.f;
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) q = counts(i, e) ? fmaf(f[i][e], f[i][e], q) : q;
    const float scale = 1.0f / sqrtf(fmaf(sum(q), a.inv_K, eps));
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (at(i) >= K) continue;  // (what lies there stays 0)
      const P g = weights(j, i);
#pragma unroll
      for (int e = 0; e < E; ++e) f[i][e] = f[i][e] * scale * g.template get<T>(e);
      if (from[j + 1]) {
        const P b = weights(j + 1, i);
#pragma unroll
        for (int e = 0; e < E; ++e) f[i][e] += b.template get<T>(e);
      }
    }
  };

#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) f[i][e] = xw[i].template get<T>(e);
  if (a.gamma_post) norm(0, a.eps_post);
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    if (at(i) >= K) continue;
    if (gate) {
      const P g = weights(2, i);
#pragma unroll
      for (int e = 0; e < E; ++e) f[i][e] *= g.template get<T>(e);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      f[i][e] = fmaf(a.residual_scale, rw[i].template get<T>(e), a.branch_scale * f[i][e]);
      if (!WHOLE && at(i) + e >= K) f[i][e] = 0.f;
    }
    Piece<R, E> o;
    o.template put<T>(f[i]);
    o.store(reinterpret_cast<R*>(a.total) + row * K + at(i), length(i));
  }
  if (!a.normed) return;
  norm(3, a.eps_pre);
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    if (at(i) >= K) continue;
    P o;
    o.template put<T>(f[i]);
    o.store(a.normed + row * K + at(i), length(i));
  }
}

template <class T, class R>
static int launch_norm_residual(NormResidualArgs a, hipStream_t stream) {
  auto go = [&](auto nch) {
    constexpr int NCH = decltype(nch)::value;
    a.halves = (a.K + 256 * NCH - 1) / (256 * NCH);
    a.rows = a.halves % 2 == 1 && a.halves <= 15 ? 2 : 1;
    const dim3 grid((unsigned int)((a.M + a.rows - 1) / a.rows)), block((a.rows * a.halves + 1) / 2 * 64);
    SF_REQUIRE(launchable(grid.x, (int)block.x), "norm_residual: %lld rows are too many for a launch", (long long)a.M);
    if (a.K % 8 == 0) hipLaunchKernelGGL((norm_residual_kernel<T, R, NCH, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((norm_residual_kernel<T, R, NCH, false>), grid, block, 0, stream, a);
    return check_launch("norm_residual_kernel");
  };
  using N1 = std::integral_constant<int, 1>;
  using N2 = std::integral_constant<int, 2>;
  using N4 = std::integral_constant<int, 4>;
  if (a.K > 16384) return go(N4{});
  // One piece to a thread / two, us at 88 M values (half of them onto fp32): fp32 residuals 1280 103 / 119, 2048 101 / 120, 8192 106 / 117; half types with RMS
  // norms 333 197 / 152 (two rows share a wavefront), 1024 117 / 124, 1999 154 / 158, 4096 121 / 127, 5000 158 / 131, 8192 130 / 135, with LayerNorms 333 205 / 181, 512 129 /
  // 129, 768 136 / 144, 1280 152 / 144, 2048 132 / 130, 4096 142 / 131, 5000 203 / 146, 8192 145 / 146
  const bool two = a.K > 8192 || (sizeof(R) == 2 && (a.K > 4096 || (a.K > 1024 && !a.rms) || (a.K > 256 && a.K < 512)));
  return two ? go(N2{}) : go(N1{});
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
  // (of one row the stride is nothing, but an fp32 total over it still reaches values that other threads have to read)
  SF_REQUIRE(M == 0 || ((total != residual || M == 1 || ld_res == K) && (total != x || ((M == 1 || ldx == K) && !residual_is_f32))),
             "norm_residual: total lies where its rows are read in another layout");
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
  a.in_place = total == x || total == residual;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == SAMFAST_F16) return residual_is_f32 ? launch_norm_residual<ElemF16, float>(a, s) : launch_norm_residual<ElemF16, us>(a, s);
  return residual_is_f32 ? launch_norm_residual<ElemBf16, float>(a, s) : launch_norm_residual<ElemBf16, us>(a, s);
}
