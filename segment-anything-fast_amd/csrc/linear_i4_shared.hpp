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
  int64_t ldx, ldy;
  int M, N, K, group;            // K % 8 == 0, group % 32 == 0
  int tiles_m, tiles_n;
};

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

int launch_i4_few(const I4Args& a, bool f16, hipStream_t stream);  // linear_i4_few.hip: up to SAMFAST_I4_FEW_ROWS rows

// linear_i4_dense.hip: the weights written out once, then the half types' product by turns.  The tile's columns / 32, 0: not this way
int i4_dense_tile(int64_t M, int N, int K);
int launch_i4_dense(const I4Args& a, bool f16, int tile, void* weights, hipStream_t stream);

}  // namespace samfast
