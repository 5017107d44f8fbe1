// Shared by the kernels of Linears with 4-bit weights: arguments, and the codes as numbers.
#pragma once

#include "samfast_internal.hpp"
#include "attn_relpos_shared.hpp"

namespace samfast {

// y[m, n] = sum over the groups g of s[g, n] * sum over k in g of x[m, k] (c[n, k] - z[g, n]), + bias[n].
struct I4Args {
  const unsigned short* x;       // (M, K), row stride ldx
  const unsigned char* codes;    // (N, K / 2): the lower half of a byte is the even k
  const unsigned short* scales;  // (groups, N)
  const unsigned char* zeros;    // (groups, N), or null: 8 throughout
  const float* bias;             // (N), or null
  unsigned short* y;             // (M, N), row stride ldy
  float* parts;                  // K split between workgroups: their sums (splits, M, N); else null
  int64_t ldx, ldy;
  int M, N, K, group;            // K % 8 == 0, group % 32 == 0
  unsigned int div_group;        // for i4_group
  int tiles_m, tiles_n;
};

// The group of the 32 inputs from 32 * step on: step / (group / 32), exact below 2^15 steps, which K <= kI4MaxInputs keeps
constexpr int kI4MaxInputs = 1 << 20;
static inline unsigned int i4_divider(int group) { return (unsigned int)((((uint64_t)1 << 31) + group / 32 - 1) / (group / 32)); }
SF_DEVICE int i4_group(const I4Args& a, int step) { return (int)__umulhi((unsigned int)(2 * step), a.div_group); }

// The eight codes of a word in the order of k, as floats 0 to 15: the even and the odd ones stand in bytes of their own for
// v_cvt_f32_ubyte.
SF_DEVICE void i4_codes(unsigned int w, float (&c)[8]) {
  const unsigned int even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    c[2 * b] = (float)((even >> (8 * b)) & 255u);
    c[2 * b + 1] = (float)((odd >> (8 * b)) & 255u);
  }
}

// The same as bytes.  As an e4m3 number a byte c below 16 is c / 512, subnormal or not: conversions with the scale 512 give c itself.
SF_DEVICE u32x2 i4_bytes(unsigned int w) {
  const unsigned int even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;
  return u32x2{__builtin_amdgcn_perm(odd, even, 0x05010400u), __builtin_amdgcn_perm(odd, even, 0x07030602u)};
}

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

int launch_i4_few(const I4Args& a, bool f16, hipStream_t stream);  // linear_i4_few.hip: up to SAMFAST_I4_FEW_ROWS rows

// linear_i4_dense.hip: the weights written out once, then the half types' product by turns.  The tile's columns / 32 and about how many us it
// takes; 0: not this way
int i4_dense_tile(int64_t M, int N, int K, double* time);
int64_t i4_dense_workspace(int64_t M, int N, int K);
int launch_i4_dense(const I4Args& a, bool f16, int tile, void* weights, hipStream_t stream);

}  // namespace samfast
