// Linears with 4-bit weights over few rows, the steps of token generation: the weights are read once and bound it, the rows come out of the L2s.
//
// A workgroup has 16 NT columns, its wavefronts take turns over K in segments of 128.  A lane loads 16 bytes of codes, 32 adjacent k of one
// column; four lanes that hold one column exchange words (v_permlane32_swap, v_permlane16_swap) until each 16 x 16 x 32 matrix instruction
// multiplies 32 adjacent k, which belong to one group.  code - zero is exact in either type; a group's sum is scaled in fp32, so no weight is
// rounded.  The wavefronts' sums meet in LDS.
#include "linear_i4_shared.hpp"

namespace samfast {

// words j of the lanes of quarter q: word q of the lanes of quarter j
SF_DEVICE void i4_transpose(u32x4& w) {
  typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
  u32x2_t r = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false));
  const unsigned int a0 = r[0], a2 = r[1];
  r = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false));
  const unsigned int a1 = r[0], a3 = r[1];
  r = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane16_swap(a0, a1, false, false));
  w[0] = r[0];
  w[1] = r[1];
  r = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane16_swap(a2, a3, false, false));
  w[2] = r[0];
  w[3] = r[1];
}

// MT x 16 rows, NT x 16 columns; STEPS matrix instructions (of 32 k) to a group, 4 also for longer ones; DEPTH segments of a wavefront in flight
template <class T, int MT, int NT, int STEPS, int DEPTH>
__global__ __launch_bounds__(512, 2) void linear_i4_few_kernel(I4Args a) {
  constexpr int GROUPS = 4 / STEPS;  // of a segment
  extern __shared__ __attribute__((aligned(16))) float sums[];
  const int lane = threadIdx.x & 63, lr = lane & 15, lq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int n0 = blockIdx.x * 16 * NT;
  const int nseg = (a.K + 127) / 128;

  const unsigned char* codes[NT];
  const unsigned char* zeros[NT];
  int quad[NT];  // the lane's four output columns
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int col = min(n0 + 16 * j + lr, a.N - 1);
    codes[j] = a.codes + (int64_t)col * (a.K / 2) + 16 * lq;
    zeros[j] = a.zeros + col;
    quad[j] = n0 + 16 * j + 4 * lq;
  }
  const unsigned short* rows[MT];
  bool row_in[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    row_in[i] = 16 * i + lr < a.M;
    rows[i] = a.x + (int64_t)(row_in[i] ? 16 * i + lr : 0) * a.ldx + 8 * lq;
  }

  u32x4 cw[DEPTH][NT], xw[DEPTH][MT][4];
  u32x2 sw[DEPTH][NT][GROUPS];
  unsigned int zw[DEPTH][NT][GROUPS];
  auto load = [&](int seg, auto slot) __attribute__((always_inline)) {
    constexpr int S = decltype(slot)::value;
    const int k0 = seg * 128;
    const bool whole = k0 + 128 <= a.K;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const unsigned char* p = codes[j] + seg * 64;
      if (whole) {
        __builtin_memcpy(&cw[S][j], __builtin_assume_aligned(p, 4), 16);
      } else {
        cw[S][j] = u32x4{};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (k0 + 32 * lq + 8 * e < a.K) cw[S][j][e] = *reinterpret_cast<const unsigned int*>(p + 4 * e);
      }
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        const int64_t at = (int64_t)(min(k0 + 32 * STEPS * g, a.K - 1) / a.group) * a.N;
        if (quad[j] + 4 <= a.N) {
          __builtin_memcpy(&sw[S][j][g], a.scales + at + quad[j], 8);
        } else {
#pragma unroll
          for (int e = 0; e < 2; ++e)
            sw[S][j][g][e] = a.scales[at + min(quad[j] + 2 * e, a.N - 1)] | (unsigned int)a.scales[at + min(quad[j] + 2 * e + 1, a.N - 1)] << 16;
        }
        zw[S][j][g] = a.zeros ? zeros[j][at] : 8u;
      }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        xw[S][i][t] = u32x4{};
        if (row_in[i] && (whole || k0 + 32 * t + 8 * lq < a.K)) xw[S][i][t] = *reinterpret_cast<const u32x4*>(rows[i] + k0 + 32 * t);
      }
  };
  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{};
  auto multiply = [&](int seg, auto slot) __attribute__((always_inline)) {
    constexpr int S = decltype(slot)::value;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      u32x4 c = cw[S][j];
      i4_transpose(c);
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        if (g > 0 && seg * 128 + 32 * STEPS * g >= a.K) break;  // (uniform)
        const float z = (float)zw[S][j][g];
        f32x4 part[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) part[i] = f32x4{};
#pragma unroll
        for (int t = g * STEPS; t < (g + 1) * STEPS; ++t) {
          float f[8];
          i4_codes(c[t], f);
          u32x4 w;
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = T::pack2(f[2 * e] - z, f[2 * e + 1] - z);
#pragma unroll
          for (int i = 0; i < MT; ++i) part[i] = T::mfma16(w, xw[S][i][t], part[i]);
        }
        const float s[4] = {T::lo(sw[S][j][g][0]), T::hi(sw[S][j][g][0]), T::lo(sw[S][j][g][1]), T::hi(sw[S][j][g][1])};
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(part[i][e], s[e], acc[i][j][e]);
      }
    }
  };
  auto each_slot = [&](auto f) __attribute__((always_inline)) {
    f(std::integral_constant<int, 0>{});
    if constexpr (DEPTH > 1) f(std::integral_constant<int, 1>{});
    if constexpr (DEPTH > 2) f(std::integral_constant<int, 2>{});
    if constexpr (DEPTH > 3) f(std::integral_constant<int, 3>{});
  };
  each_slot([&](auto slot) __attribute__((always_inline)) {
    const int seg = wave + decltype(slot)::value * waves;
    if (seg < nseg) load(seg, slot);
  });
  for (int first = wave; first < nseg; first += DEPTH * waves) {
    each_slot([&](auto slot) __attribute__((always_inline)) {
      const int seg = first + decltype(slot)::value * waves;
      if (seg < nseg) {
        multiply(seg, slot);
        if (seg + DEPTH * waves < nseg) load(seg + DEPTH * waves, slot);
      }
    });
  }

  f32x4* mine = reinterpret_cast<f32x4*>(sums) + wave * MT * NT * 64;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) mine[(i * NT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int o = threadIdx.x; o < MT * NT * 64; o += blockDim.x) {
    f32x4 v = reinterpret_cast<const f32x4*>(sums)[o];
    for (int w = 1; w < waves; ++w) v += reinterpret_cast<const f32x4*>(sums)[w * MT * NT * 64 + o];
    const int l = o & 63, m = o / (64 * NT) * 16 + (l & 15), n = n0 + (o / 64 % NT) * 16 + 4 * (l >> 4);
    if (m >= a.M || n >= a.N) continue;
    unsigned short* y = a.y + (int64_t)m * a.ldy + n;
    float b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = a.bias ? a.bias[min(n + e, a.N - 1)] : 0.f;
    const u32x2 r = {T::pack2(v[0] + b[0], v[1] + b[1]), T::pack2(v[2] + b[2], v[3] + b[3])};
    if (n + 4 <= a.N) {
      __builtin_memcpy(y, &r, 8);
    } else {
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (n + e < a.N) y[e] = (unsigned short)(r[e >> 1] >> (16 * (e & 1)));
    }
  }
}

template <class T, int MT, int NT, int STEPS>
static int go_few(const I4Args& a, hipStream_t stream) {
  constexpr int DEPTH = MT * NT > 2 ? 1 : 2;
  const int nseg = (a.K + 127) / 128, waves = nseg < 8 ? nseg : 8;
  hipLaunchKernelGGL((linear_i4_few_kernel<T, MT, NT, STEPS, DEPTH>), dim3((unsigned int)((a.N + 16 * NT - 1) / (16 * NT))), dim3(64 * waves),
                     waves * MT * NT * 1024, stream, a);
  return check_launch("linear_i4_few_kernel");
}
template <class T, int MT, int NT>
static int go_few(const I4Args& a, hipStream_t stream) {
  if (a.group % 128 == 0) return go_few<T, MT, NT, 4>(a, stream);
  if (a.group % 64 == 0) return go_few<T, MT, NT, 2>(a, stream);
  return go_few<T, MT, NT, 1>(a, stream);
}
template <class T>
static int go_few(const I4Args& a, hipStream_t stream) {
  const bool wide = a.N >= 8192;
  if (a.M <= 16) return wide ? go_few<T, 1, 2>(a, stream) : go_few<T, 1, 1>(a, stream);
  if (a.M <= 32) return wide ? go_few<T, 2, 2>(a, stream) : go_few<T, 2, 1>(a, stream);
  return wide ? go_few<T, 4, 2>(a, stream) : go_few<T, 4, 1>(a, stream);
}

int launch_i4_few(const I4Args& a, bool f16, hipStream_t stream) { return f16 ? go_few<ElemF16>(a, stream) : go_few<ElemBf16>(a, stream); }

}  // namespace samfast
