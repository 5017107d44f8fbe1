// Linears with 4-bit weights over many rows by the half types' product by turns (gemm_pingpong.hpp): the weights are written out in the
// element type, once per call, and that product reads them out of the caches.  It walks K by whole 64s: of rows that end inside one, and of their weights, copies
// with zeros behind them are made.
#include "gemm_pingpong.hpp"
#include "linear_i4_shared.hpp"

namespace samfast {

static inline int i4_padded(int K) { return (K + 63) / 64 * 64; }

// w[n, k] = (code - zero) * scale, rounded to the element type: eight codes a thread.  Behind N rows of weights, with `copies`, those of x.
template <class T>
__global__ __launch_bounds__(256) void i4_weights_kernel(I4Args a, unsigned short* w, int padded, int copies) {
  const unsigned int words = (unsigned int)padded / 8u;  // of a row
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / words;
  const int k = 8 * (int)(i - row * words);
  if (row >= a.N || k >= a.K) {
    u32x4 v = {};
    if (row >= (int64_t)a.N + copies) return;
    if (row >= a.N && k < a.K) v = *reinterpret_cast<const u32x4*>(a.x + (row - a.N) * a.ldx + k);
    reinterpret_cast<u32x4*>(w)[i] = v;
    return;
  }
  const int n = (int)row;
  const int64_t at = (int64_t)(k / a.group) * a.N + n;
  const float s = T::from_bits(a.scales[at]), z = a.zeros ? (float)a.zeros[at] : 8.f;
  float c[8];
  i4_codes(reinterpret_cast<const unsigned int*>(a.codes)[row * (a.K / 8) + k / 8], c);
  u32x4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = T::pack2((c[2 * e] - z) * s, (c[2 * e + 1] - z) * s);
  reinterpret_cast<u32x4*>(w)[i] = o;
}

// The time: two launches, weights and copies written and read, and pp_choose's cost, a unit of which takes 0.075 us where the GPU is nearly idle and 0.112 where
// it is busy throughout (power).  2048 x 4096 -> 4096 71 us, 4096 x 1280 -> 5120 52, of 1288 values 54.6, 65536 x 1280 -> 3840 478, 1024 x 8192 -> 8192 146 to 168
// from card to card, 5405 x 3832 -> 4828 181 (copies 17 of it).
int i4_dense_tile(int64_t M, int N, int K, double* time) {
  const int padded = i4_padded(K);
  if (padded < 320 || M < 256 || N >= 1 << 22 || !launchable(((int64_t)N + M) * (padded / 8) / 256 + 1, 256)) return 0;
  const PPChoice c = pp_choose(M, N, padded / 64, false, 8.1);
  if (c.tn == 0) return 0;
  const double fragments = c.tn == 10 ? 12.5 : c.tn == 8 ? 10.0 : 8.1;
  *time = 7.0 + (0.55 * N + (padded != K ? 0.57 * M : 0.0)) * padded / 1e6 + (0.075 + 0.037 * c.used) * (double)c.rounds * fragments * (padded / 64 + 8);
  return c.tn;
}

int64_t i4_dense_workspace(int64_t M, int N, int K) {
  const int padded = i4_padded(K);
  return 2 * (int64_t)padded * (N + (padded != K ? M : 0));
}

template <class T, class E>
static int go_dense(const I4Args& a, int tile, unsigned short* weights, hipStream_t stream) {
  const int padded = i4_padded(a.K), copies = padded != a.K ? a.M : 0;
  const int64_t words = ((int64_t)a.N + copies) * (padded / 8);
  hipLaunchKernelGGL(i4_weights_kernel<T>, dim3((unsigned int)((words + 255) / 256)), dim3(256), 0, stream, a, weights, padded, copies);
  if (const int rc = check_launch("i4_weights_kernel")) return rc;
  PPArgs p = {};
  p.x = reinterpret_cast<const unsigned char*>(copies ? weights + (int64_t)a.N * padded : a.x);
  p.w = reinterpret_cast<const unsigned char*>(weights);
  p.out = a.y;
  p.bias = a.bias;
  p.ldo = a.ldy;
  p.x_kstep = p.w_kstep = 64;
  p.x_pitch = (unsigned int)((copies ? padded : a.ldx) * 2);
  p.w_pitch = (unsigned int)(padded * 2);
  p.M = a.M;
  p.N = a.N;
  p.nk = padded / 64;
  p.group_m = 4;
  p.tiles_m = (a.M + 255) / 256;
  p.tiles_n = (a.N + 32 * tile - 1) / (32 * tile);
  const dim3 grid(pp_grid(p));
  if (tile == 6) hipLaunchKernelGGL((gemm_pingpong_kernel<E, PP_PLAIN, 6, false>), grid, dim3(512), 0, stream, p);
  else if (tile == 8) hipLaunchKernelGGL((gemm_pingpong_kernel<E, PP_PLAIN, 8, false>), grid, dim3(512), 0, stream, p);
  else hipLaunchKernelGGL((gemm_pingpong_kernel<E, PP_PLAIN, 10, false>), grid, dim3(512), 0, stream, p);
  return check_launch("gemm_pingpong_kernel");
}

int launch_i4_dense(const I4Args& a, bool f16, int tile, void* weights, hipStream_t stream) {
  unsigned short* w = reinterpret_cast<unsigned short*>(weights);
  return f16 ? go_dense<ElemF16, PPF16Bias32>(a, tile, w, stream) : go_dense<ElemBf16, PPBf16Bias32>(a, tile, w, stream);
}

}  // namespace samfast
