// Linears with 4-bit weights over few rows, the steps of token generation: the weights are read once and bound it, the rows come out of the L2s.
//
// A workgroup has 16 NT columns, its wavefronts take turns over K, 256 at a time.  A lane loads 16 bytes of codes, 32 adjacent k of one
// column; four lanes that hold one column exchange words (v_permlane32_swap, v_permlane16_swap) until each 16 x 16 x 32 matrix instruction
// multiplies 32 adjacent k, which belong to one group.  The codes are exact in either type; a group's sum is scaled in fp32, and its zero times the
// group's sum of x taken off in fp32, so no weight is rounded.  The wavefronts' sums meet in LDS.
//
// us, calls that follow one another (a copy's time for the weights): 1 x 4096 -> 4096 5.2 (1.7), 1 x 8192 -> 8192 9.5 (6.7), with zeros and groups of 32 11.9
// (7.7); 24 rows of the last 16.3 to 16.7.  There 1.2 million lines of 128 bytes come out of the L2s, two thirds of them x, a workgroup's own rows for each; vector
// instructions, 380 for 256 k of two fragments of columns, take a third of the SIMDs' cycles, matrix instructions 23 %, and wavefronts, two to a SIMD, wait for 37 % of theirs.
#include "linear_i4_shared.hpp"

#include <type_traits>

namespace samfast {

template <class T>
struct I4Few;
template <>
struct I4Few<ElemBf16> {
  template <bool HI>
  static SF_DEVICE unsigned int two(unsigned int bytes) { return __builtin_bit_cast(unsigned int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(bytes, 512.f, HI)); }
};
template <>
struct I4Few<ElemF16> {
  template <bool HI>
  static SF_DEVICE unsigned int two(unsigned int bytes) { return __builtin_bit_cast(unsigned int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes, 512.f, HI)); }
};

// The eight codes of a word as numbers 0 to 15 of the element type, in the order of k: 9 instructions for 23 with i4_codes
template <class T>
SF_DEVICE u32x4 i4_numbers(unsigned int w) {
  const u32x2 bytes = i4_bytes(w);
  return u32x4{I4Few<T>::template two<false>(bytes[0]), I4Few<T>::template two<true>(bytes[0]), I4Few<T>::template two<false>(bytes[1]), I4Few<T>::template two<true>(bytes[1])};
}

// MT x 16 rows, NT x 16 columns; STEPS matrix instructions (of 32 k) to a group, 4 also for longer ones.
//
// A wavefront takes 256 k at a time, and the next ones are under way while it multiplies.  The rows of x go straight into LDS of its own, whole lines
// to a load, and from there into registers: fragments straight from memory are half lines, and 24 x 8192 x 8192 took 22 us instead of 14.  (Codes
// as fragments or as lines were level.)  Scales and zeros come four columns of a group to a lane, and are handed round by way of LDS: as each lane's own,
// a load for each group, groups of 32 took 19.6 us instead of 18.0 there (16.5 now).  The loop has no branches, and addresses are uniform bases with 32-bit offsets that are made once: with a K that
// may end anywhere inside it, the loads of all paths were waited for at each step, and 1 x 8192 x 8192 took 16 us instead of 11.  What is left of K goes
// through a loop of its own.
constexpr int kI4FewWaves = 8;

template <class T, int MT, int NT, int STEPS>
__global__ __launch_bounds__(64 * kI4FewWaves) void linear_i4_few_kernel(I4Args a) {
  constexpr int GROUPS = 4 / STEPS;  // of 128 k
  constexpr int XBYTES = MT * 16 * 512, OWN = XBYTES + 2048;
  static_assert(MT * NT * 1024 <= OWN && 2 * GROUPS * 4 * NT <= 64, "the sums fit into what the loads used, the scales into 64 lanes");
  __shared__ __attribute__((aligned(16))) unsigned char lds[kI4FewWaves * OWN];
  const int lane = threadIdx.x & 63, lr = lane & 15, lq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = (int)blockDim.x >> 6;
  const int own = (int)blockIdx.x * 16 * NT, n0 = min(own, a.N - 16 * NT);  // (the last columns lie over the ones before them)
  const int m0 = (int)blockIdx.y * 16 * MT;
  // This wavefront's 256 k.  Workgroups start at different ones: rows of codes lie a power of two apart as a rule, and the rows of x are
  // everybody's (1 x 8192 x 8192 16.4 us for 14.3).
  const int units = a.K / 256, count = units / waves + (wave < units % waves);
  const int shift = units > 0 ? (int)(blockIdx.x % (unsigned int)units) : 0;
  auto unit = [&](int i) __attribute__((always_inline)) {
    const int p = wave + waves * i + shift;
    return p < units ? p : p - units;
  };

  const unsigned char* codes = a.codes + (int64_t)n0 * (a.K / 2);
  const unsigned char* rows = reinterpret_cast<const unsigned char*>(a.x + (int64_t)m0 * a.ldx);
  unsigned char* mine = lds + wave * OWN;
  // A load puts eight rows' lines side by side; 16-byte piece c of row r stands at position c ^ ((r >> 1) & 7), where a fragment's read finds no two
  // of its pieces in one bank.  Rows behind the last are the last one's again.
  unsigned int row_off[2 * MT];
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) {
    const int r = 8 * i + (lane >> 3);
    row_off[i] = (unsigned int)min(r, a.M - 1 - m0) * (unsigned int)(2 * a.ldx) + (((lane & 7) ^ ((r >> 1) & 7)) << 4);
  }
  typedef __attribute__((address_space(1))) const void* gptr_t;
  typedef __attribute__((address_space(3))) void* lptr_t;
  auto lines = [&](const unsigned char* base, unsigned int offset, int at) __attribute__((always_inline)) {
    asm volatile("" : "+s"(base));
    __builtin_amdgcn_global_load_lds((gptr_t)(base + offset), (lptr_t)(mine + at), 16, 0, 0);
  };
  auto request = [&](int p) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i)
      if (m0 + 8 * i < a.M) {
#pragma unroll
        for (int l = 0; l < 4; ++l) lines(rows + p * 512 + l * 128, row_off[i], (l * 2 * MT + i) * 1024);
      }
  };
  // piece c (of 8) of row r in a block of 128-byte rows
  auto piece = [&](int at, int r, int c) __attribute__((always_inline)) {
    return *reinterpret_cast<const u32x4*>(mine + at + r * 128 + ((c ^ ((r >> 1) & 7)) << 4));
  };

  // 256 k of the weights: the codes of the lane's column; scales and zeros of four columns, 4 (lane % Q) and on, in the group lane / Q
  constexpr int Q = 4 * NT;
  struct Weights {
    u32x4 codes[2][NT];
    u32x2 scales;
    unsigned int zeros;
  };
  const int scale_step = min(lane / Q, 2 * GROUPS - 1) * STEPS;
  auto load_scales = [&](Weights& w, int step) __attribute__((always_inline)) {  // (groups behind the last: the last one's, not used)
    const int64_t at = (int64_t)i4_group(a, min(step + scale_step, (a.K - 1) / 32)) * a.N + n0 + 4 * (lane % Q);
    __builtin_memcpy(&w.scales, a.scales + at, 8);
    w.zeros = 0x08080808u;
    if (a.zeros) __builtin_memcpy(&w.zeros, a.zeros + at, 4);
  };
  auto hand_round = [&](const Weights& w) __attribute__((always_inline)) {
    f32x4 s = {T::lo(w.scales[0]), T::hi(w.scales[0]), T::lo(w.scales[1]), T::hi(w.scales[1])}, sz;
#pragma unroll
    for (int e = 0; e < 4; ++e) sz[e] = -s[e] * (float)((w.zeros >> (8 * e)) & 255u);  // (exact)
    f32x4* to = reinterpret_cast<f32x4*>(mine + XBYTES) + lane;
    to[0] = s;
    to[64] = sz;
  };
  auto load = [&](Weights& w, int p) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < NT; ++j)
        __builtin_memcpy(&w.codes[h][j], __builtin_assume_aligned(codes + p * 128 + (unsigned int)((16 * j + lr) * (a.K / 2) + 64 * h + 16 * lq), 4), 16);
    load_scales(w, 8 * p);
  };
  f32x4 acc[MT][NT];
  // The zeros' part of 256 k: the groups' sums of x, which all columns share, times -scale * zero, four groups to an instruction in fp32.  Row n of the
  // sums' first operand has ones for the group that lanes of quarter n / 4 take along, and all groups add to one register.  (As vector instructions on each
  // group's sum 24 x 8192 -> 8192 17.4 us for 16.4, in groups of 64 14.9 for 14.0; before the products 16.6.)
  constexpr unsigned int ones = T::kOne | T::kOne << 16;
  unsigned int picks[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) picks[q] = lr >> 2 == q ? ones : 0u;
  auto take_zeros_off = [&](const u32x4 (&x)[2][MT][4]) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < 2 * GROUPS; c += 4) {
      f32x4 sum[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) sum[i] = f32x4{};
#pragma unroll
      for (int q = 0; q < 4 && c + q < 2 * GROUPS; ++q)
#pragma unroll
        for (int s = (c + q) * STEPS; s < (c + q + 1) * STEPS; ++s)
#pragma unroll
          for (int i = 0; i < MT; ++i) sum[i] = T::mfma16(u32x4{picks[q], picks[q], picks[q], picks[q]}, x[s >> 2][i][s & 3], sum[i]);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const float sz = reinterpret_cast<const float*>(mine + XBYTES + 1024)[(c + lq) * 4 * Q + 16 * j + lr];
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(sz, sum[i][0], acc[i][j], 0, 0, 0);
      }
    }
  };
  // The products of 128 k, the h-th of those whose scales were handed round.  SIMPLE: code - zero is made before it is multiplied, with the lane's own
  // column's zero; else the codes are.
  auto multiply = [&](const u32x4 (&cw)[NT], const u32x4 (&x)[MT][4], int h, int seg, auto simple, unsigned int zeros = 0) __attribute__((always_inline)) {
    constexpr bool SIMPLE = decltype(simple)::value;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      u32x4 c = cw[j];
      i4_transpose(c);
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        if (SIMPLE && g > 0 && seg * 128 + 32 * STEPS * g >= a.K) break;  // (uniform; the groups behind the last may not weigh in, whatever its scale)
        f32x4 part[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) part[i] = f32x4{};
        const int from = (h * GROUPS + g) * Q + 4 * j;  // the lane that had the first four columns
        const f32x4 s = reinterpret_cast<const f32x4*>(mine + XBYTES)[from + lq];
        float z = 0.f;
        if constexpr (SIMPLE) z = (float)((__shfl(zeros, from + (lr >> 2), 64) >> (8 * (lr & 3))) & 255u);
#pragma unroll
        for (int t = g * STEPS; t < (g + 1) * STEPS; ++t) {
          u32x4 w;
          if constexpr (SIMPLE) {
            float f[8];
            i4_codes(c[t], f);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = T::pack2(f[2 * e] - z, f[2 * e + 1] - z);
          } else {
            w = i4_numbers<T>(c[t]);
          }
#pragma unroll
          for (int i = 0; i < MT; ++i) part[i] = T::mfma16(w, x[i][t], part[i]);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(part[i][e], s[e], acc[i][j][e]);
      }
    }
  };
  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{};
  };
  // 128 k that may end behind K
  auto careful = [&](int seg) __attribute__((always_inline)) {
    Weights w;
    u32x4 x[MT][4];
    load_scales(w, 4 * seg);
    hand_round(w);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      w.codes[0][j] = u32x4{};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (seg * 128 + 32 * lq + 8 * e < a.K)
          w.codes[0][j][e] = *reinterpret_cast<const unsigned int*>(codes + (int64_t)(16 * j + lr) * (a.K / 2) + seg * 64 + 16 * lq + 4 * e);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        x[i][t] = u32x4{};
        if (m0 + 16 * i + lr < a.M && seg * 128 + 32 * t + 8 * lq < a.K)
          x[i][t] = *reinterpret_cast<const u32x4*>(rows + (int64_t)(16 * i + lr) * (2 * a.ldx) + seg * 256 + 64 * t + 16 * lq);
      }
    multiply(w.codes[0], x, 0, seg, std::true_type{}, w.zeros);
  };

  clear();
  if (count > 0) {
    Weights next;
    request(unit(0));
    load(next, unit(0));
    for (int n = 0; n < count; ++n) {
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt 0: this wavefront's lines are in LDS
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      const Weights now = next;
      hand_round(now);
      u32x4 x[2][MT][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int t = 0; t < 4; ++t) x[h][i][t] = piece(((2 * h + t / 2) * 2 * MT + 2 * i) * 1024, lr, 4 * (t & 1) + lq);
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt 0: and out of it again
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      if (n + 1 < count) {
        request(unit(n + 1));
        load(next, unit(n + 1));
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) multiply(now.codes[h], x[h], h, 2 * unit(n) + h, std::false_type{});
      take_zeros_off(x);
    }
  }
  // An infinity in a row or a scale, or sums that overflow before the zero is taken off, end as a NaN or an infinity here; the simple
  // way then gives what the formula does.
  bool finite = true;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) finite = finite && (m0 + 16 * i + lr >= a.M || __builtin_fabsf(acc[i][j][e]) < __builtin_inff());
  if (__builtin_amdgcn_ballot_w64(!finite) != 0) {
    clear();
#pragma unroll 1
    for (int n = 0; n < 2 * count; ++n) careful(2 * unit(n >> 1) + (n & 1));
  }
  // what is left of K, the wavefronts that had less first
#pragma unroll 1
  for (int seg = 2 * units + (wave + waves - units % waves) % waves; seg < (a.K + 127) / 128; seg += waves) careful(seg);

  f32x4* sums = reinterpret_cast<f32x4*>(lds);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) sums[wave * MT * NT * 64 + (i * NT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int o = threadIdx.x; o < MT * NT * 64; o += blockDim.x) {
    f32x4 v = sums[o];
    for (int w = 1; w < waves; ++w) v += sums[w * MT * NT * 64 + o];
    const int l = o & 63, m = m0 + o / (64 * NT) * 16 + (l & 15), n = n0 + (o / 64 % NT) * 16 + 4 * (l >> 4);
    if (m >= a.M || n + 4 <= own) continue;
    unsigned short* y = a.y + (int64_t)m * a.ldy + n;
    float b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = a.bias ? a.bias[n + e] : 0.f;
    const u32x2 r = {T::pack2(v[0] + b[0], v[1] + b[1]), T::pack2(v[2] + b[2], v[3] + b[3])};
    if (n >= own) {
      __builtin_memcpy(y, &r, 8);
    } else {
#pragma unroll
      for (int e = 1; e < 4; ++e)
        if (n + e >= own) y[e] = (unsigned short)(r[e >> 1] >> (16 * (e & 1)));
    }
  }
}

template <class T, int MT, int NT>
static int go_few(const I4Args& a, hipStream_t stream) {
  const int units = (a.K + 255) / 256, waves = units < kI4FewWaves ? units : kI4FewWaves;
  const dim3 grid((unsigned int)((a.N + 16 * NT - 1) / (16 * NT)), (unsigned int)((a.M + 16 * MT - 1) / (16 * MT)));
  SF_REQUIRE(launchable(grid.x, 64 * waves), "linear_i4: %d outputs are too many for a launch", a.N);
  auto go = [&](auto steps) {
    hipLaunchKernelGGL((linear_i4_few_kernel<T, MT, NT, decltype(steps)::value>), grid, dim3(64 * waves), 0, stream, a);
    return check_launch("linear_i4_few_kernel");
  };
  if (a.group % 128 == 0) return go(std::integral_constant<int, 4>{});
  if (a.group % 64 == 0) return go(std::integral_constant<int, 2>{});
  return go(std::integral_constant<int, 1>{});
}
template <class T>
static int go_few(const I4Args& a, hipStream_t stream) {
  // One workgroup fits a CU (LDS).  32 columns each where 16 would need a second round of the 256 CUs: M x 8192 -> N, groups of 128, us with 16 / 32 columns,
  // M = 1, 16, 24: N = 4096 7.8 / 10.1, 9.1 / 11.4, 11.1 / 13.6; 5120 11.5 / 10.5, 13.4 / 11.5, 19.1 / 13.7; 8192 11.7 / 10.7, 13.6 / 12.1, 19.5 / 14.2; 16384
  // 19.5 / 16.9, 22.6 / 18.7, 36.5 / 25.7 (in a recording).  Of three rounds against two up to 16 rows are level, in groups of 32 they lose: 16 x 8192 -> 10240 20.3 / 23.0.
  const bool wide = a.N > 16 * 256;
  if (a.M <= 16) return wide ? go_few<T, 1, 2>(a, stream) : go_few<T, 1, 1>(a, stream);
  return wide ? go_few<T, 2, 2>(a, stream) : go_few<T, 2, 1>(a, stream);
}

int launch_i4_few(const I4Args& a, bool f16, hipStream_t stream) { return f16 ? go_few<ElemF16>(a, stream) : go_few<ElemBf16>(a, stream); }

}  // namespace samfast
