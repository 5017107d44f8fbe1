// Linears with 4-bit weights over many rows: a tiled matrix product that makes the weights of a tile, rounded to the element type, on
// their way into LDS.
#include "linear_i4_shared.hpp"

namespace samfast {

template <class T, int FM, int FN>
struct I4Tile {
  static constexpr int BM = 32 * FM, BN = 32 * FN;   // four wavefronts, two by two, of FM x FN fragments of 16 x 16
  static constexpr int STAGE = (BM + BN) * 128;      // one k tile of 64 of both operands
  static constexpr int KT = BN / 4;                  // values of a weight tile that a thread makes: 256 threads, 64 BN values
  static constexpr int WORDS = KT / 8;
  static constexpr int THREADS_ROW = 64 / KT;        // threads that share a row
};

// 16-byte piece c of LDS row r stands at position c ^ ((r >> 1) & 7): a fragment's read (16 rows, four pieces) touches every bank once
SF_DEVICE int i4_place(int row, int piece) { return row * 128 + ((piece ^ ((row >> 1) & 7)) << 4); }

// 16 bytes a lane from base + offset to lds + 16 lane; zeros where the offset is kOutside
constexpr unsigned int kOutside = 0x80000000u;
SF_DEVICE void piece_to_lds(const void* base, unsigned int offset, void* lds) {
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, 0x7fffffff, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)lds, 16, offset, 0, 0, 0);
}

template <class T, int FM, int FN>
__global__ __launch_bounds__(256, 2) void linear_i4_tiled_kernel(I4Args a) {
  using P = I4Tile<T, FM, FN>;
  __shared__ __attribute__((aligned(16))) unsigned char lds[2 * P::STAGE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave & 1, wn = wave >> 1, lr = lane & 15, lq = lane >> 4;

  // neighbours on an XCD share the weights' tile columns in groups of eight rows of tiles
  const unsigned int total = (unsigned int)a.tiles_m * (unsigned int)a.tiles_n;
  const unsigned int pid = xcd_contiguous_id(blockIdx.x, total);
  if (pid >= total) return;
  const unsigned int per_group = 8u * a.tiles_n, first_m = pid / per_group * 8u;
  const unsigned int rows = min((unsigned int)a.tiles_m - first_m, 8u), in_group = pid % per_group;
  const int m0 = (int)(first_m + in_group % rows) * P::BM, n0 = (int)(in_group / rows) * P::BN;

  // ---- x: 16-byte pieces straight into LDS; a piece outside the matrix gets an offset behind the buffer's end and arrives as zeros
  constexpr int XLOADS = P::BM / 32;
  unsigned int x_off[XLOADS];
  int x_k[XLOADS];
#pragma unroll
  for (int i = 0; i < XLOADS; ++i) {
    const int row = (wave + 4 * i) * 8 + (lane >> 3), piece = (lane & 7) ^ ((row >> 1) & 7);
    x_k[i] = piece * 8;
    x_off[i] = m0 + row < a.M ? (unsigned int)row * (unsigned int)(a.ldx * 2) + piece * 16 : kOutside;
  }
  const unsigned short* xt = a.x + (int64_t)m0 * a.ldx;
  auto load_x = [&](int k0, int stage) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < XLOADS; ++i) piece_to_lds(xt + k0, k0 + x_k[i] < a.K ? x_off[i] : kOutside, lds + stage + (wave + 4 * i) * 1024);
  };

  // ---- weights: a thread's KT codes of one row.  Row i of fragment j of a wavefront's 16 FN columns holds column
  // 4 FN (i / 4) + 4 j + i % 4, so that a lane ends with 4 FN adjacent ones.
  const int wrow = tid / P::THREADS_ROW, wk = tid % P::THREADS_ROW * P::KT;
  const int in_wave = wrow % (16 * FN), wi = in_wave % 16, wj = in_wave / 16;
  const int wcol = min(n0 + wrow / (16 * FN) * 16 * FN + 4 * FN * (wi >> 2) + 4 * wj + (wi & 3), a.N - 1);
  const unsigned char* wcodes = a.codes + (int64_t)wcol * (a.K / 2);
  unsigned int cw[P::WORDS];
  unsigned int csw, czw;
  auto load_w = [&](int k0) __attribute__((always_inline)) {
    const int k = k0 + wk;
    if (k + P::KT <= a.K) {
      __builtin_memcpy(cw, __builtin_assume_aligned(wcodes + k / 2, 4), P::KT / 2);
    } else {
#pragma unroll
      for (int j = 0; j < P::WORDS; ++j) {
        cw[j] = 0;
        if (k + 8 * j < a.K) __builtin_memcpy(&cw[j], __builtin_assume_aligned(wcodes + k / 2 + 4 * j, 4), 4);
      }
    }
    const int64_t at = (int64_t)(min(k, a.K - 1) / a.group) * a.N + wcol;
    csw = a.scales[at];
    czw = a.zeros ? a.zeros[at] : 8u;
  };
  auto make_w = [&](int k0, int stage) __attribute__((always_inline)) {
    const float s = T::from_bits((unsigned short)csw), z = (float)czw;
#pragma unroll
    for (int j = 0; j < P::WORDS; ++j) {
      float c[8];
      i4_codes(cw[j], c);
      u32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = T::pack2((c[2 * e] - z) * s, (c[2 * e + 1] - z) * s);
      if (k0 + wk + 8 * j >= a.K) w = u32x4{};
      *reinterpret_cast<u32x4*>(lds + stage + P::BM * 128 + i4_place(wrow, wk / 8 + j)) = w;
    }
  };

  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{};

  const int nk = (a.K + 63) / 64;
  load_x(0, 0);
  load_w(0);
  make_w(0, 0);
  auto meet = [&]() __attribute__((always_inline)) {  // what every wavefront has put into LDS, by either way, is there
    __builtin_amdgcn_s_waitcnt(0x0070);
    __syncthreads();
  };
  meet();
  for (int kt = 0; kt < nk; ++kt) {
    const int stage = (kt & 1) * P::STAGE, other = P::STAGE - stage;
    const bool more = kt + 1 < nk;
    if (more) {
      load_x((kt + 1) * 64, other);
      load_w((kt + 1) * 64);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 fx[FM], fw[FN];
#pragma unroll
      for (int i = 0; i < FM; ++i) fx[i] = *reinterpret_cast<const u32x4*>(lds + stage + i4_place((wm * FM + i) * 16 + lr, 4 * h + lq));
#pragma unroll
      for (int j = 0; j < FN; ++j) fw[j] = *reinterpret_cast<const u32x4*>(lds + stage + P::BM * 128 + i4_place((wn * FN + j) * 16 + lr, 4 * h + lq));
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = T::mfma16(fw[j], fx[i], acc[i][j]);
    }
    if (more) make_w((kt + 1) * 64, other);
    meet();
  }

  // ---- a lane holds row 16 i + lr and 4 FN adjacent columns
  const int n = n0 + wn * 16 * FN + 4 * FN * lq;
  float bias[4 * FN];
#pragma unroll
  for (int c = 0; c < 4 * FN; ++c) bias[c] = a.bias ? a.bias[min(n + c, a.N - 1)] : 0.f;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int m = m0 + (wm * FM + i) * 16 + lr;
    if (m >= a.M || n >= a.N) continue;
    unsigned short* y = a.y + (int64_t)m * a.ldy + n;
    unsigned int o[2 * FN];
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        o[2 * j + e] = T::pack2(acc[i][j][2 * e] + bias[4 * j + 2 * e], acc[i][j][2 * e + 1] + bias[4 * j + 2 * e + 1]);
    if (n + 4 * FN <= a.N) {
      __builtin_memcpy(y, o, 8 * FN);
    } else {
#pragma unroll
      for (int c = 0; c < 4 * FN; ++c)
        if (n + c < a.N) y[c] = (unsigned short)(o[c >> 1] >> (16 * (c & 1)));
    }
  }
}

// y = the parts' sums + bias: four columns a thread
template <class T>
__global__ __launch_bounds__(256) void i4_sum_kernel(I4Args a, int splits) {
  const int quads = (a.N + 3) / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)a.M * quads) return;
  const int m = (int)(i / quads), n = 4 * (int)(i - (int64_t)m * quads);
  float v[4] = {};
  const float* part = a.parts + (int64_t)m * a.N + n;
  if (n + 4 <= a.N) {
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      float p[4];
      __builtin_memcpy(p, part + (int64_t)s * a.M * a.N, 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += p[e];
    }
  } else {
    for (int s = 0; s < splits; ++s)
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (n + e < a.N) v[e] += part[(int64_t)s * a.M * a.N + e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] += a.bias ? a.bias[min(n + e, a.N - 1)] : 0.f;
  const u32x2 r = {T::pack2(v[0], v[1]), T::pack2(v[2], v[3])};
  unsigned short* y = a.y + (int64_t)m * a.ldy + n;
  if (n + 4 <= a.N) {
    __builtin_memcpy(y, &r, 8);
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (n + e < a.N) y[e] = (unsigned short)(r[e >> 1] >> (16 * (e & 1)));
  }
}

template <class T>
static int launch_i4_tiled(I4Args a, hipStream_t stream) {
  auto go = [&](auto fm, auto fn) {
    using P = I4Tile<T, decltype(fm)::value, decltype(fn)::value>;
    a.tiles_m = (a.M + P::BM - 1) / P::BM;
    a.tiles_n = (a.N + P::BN - 1) / P::BN;
    const dim3 grid((unsigned int)(((int64_t)a.tiles_m * a.tiles_n + 7) / 8 * 8));
    hipLaunchKernelGGL((linear_i4_tiled_kernel<T, decltype(fm)::value, decltype(fn)::value>), grid, dim3(256), 0, stream, a);
    return check_launch("linear_i4_tiled_kernel");
  };
  using F2 = std::integral_constant<int, 2>;
  using F4 = std::integral_constant<int, 4>;
  if ((int64_t)((a.M + 127) / 128) * ((a.N + 127) / 128) >= 256) return go(F4{}, F4{});
  return go(F2{}, F2{});
}

}  // namespace samfast

extern "C" int64_t samfast_linear_i4_workspace(int64_t M, int N, int K) {
  using namespace samfast;
  SF_REQUIRE(M >= 0 && N > 0 && K > 0, "linear_i4_workspace: bad shape M=%lld N=%d K=%d", (long long)M, N, K);
  return i4_dense_tile(M, N, K) ? (int64_t)N * K * 2 : 0;
}

extern "C" int samfast_linear_i4(const void* x, int64_t ldx, const uint8_t* codes, const void* scales, const uint8_t* zeros, const float* bias,
                                 void* y, int64_t ldy, void* workspace, int64_t M, int N, int K, int group, int dtype, void* stream) {
  using namespace samfast;
  if (dtype != SAMFAST_BF16 && dtype != SAMFAST_F16) SF_FAIL(SAMFAST_E_UNSUPPORTED, "linear_i4: element type %d is neither SAMFAST_BF16 nor SAMFAST_F16", dtype);
  SF_REQUIRE(M >= 0 && N > 0 && K > 0 && K % 8 == 0, "linear_i4: bad shape M=%lld N=%d K=%d (K must be a multiple of 8)", (long long)M, N, K);
  SF_REQUIRE(group > 0 && group % 32 == 0, "linear_i4: groups of %d inputs (must be a multiple of 32)", group);
  SF_REQUIRE(M < (1ll << 31) - 512 && N < (1 << 30) && K <= kI4MaxInputs && ldx < (1 << 22), "linear_i4: too large");
  SF_REQUIRE(((M + 63) / 64) * ((N + 63) / 64) < (1ll << 31) - 8, "linear_i4: too large");
  if (M == 0) return SAMFAST_OK;
  SF_REQUIRE(x && codes && scales && y, "linear_i4: null pointer");
  SF_REQUIRE(ldx >= K && ldx % 8 == 0 && ldy >= N, "linear_i4: row strides must hold a row, that of x be a multiple of 8");
  SF_REQUIRE(aligned16(x) && (reinterpret_cast<uintptr_t>(codes) & 3u) == 0 && (reinterpret_cast<uintptr_t>(bias) & 3u) == 0,
             "linear_i4: x must be 16-byte aligned, codes and bias 4-byte");
  I4Args a = {};
  a.x = reinterpret_cast<const unsigned short*>(x);
  a.codes = codes;
  a.scales = reinterpret_cast<const unsigned short*>(scales);
  a.zeros = zeros;
  a.bias = bias;
  a.y = reinterpret_cast<unsigned short*>(y);
  a.ldx = ldx;
  a.ldy = ldy;
  a.M = (int)M;
  a.N = N;
  a.K = K;
  a.group = group;
  a.div_group = i4_divider(group < K ? group : (K + 31) / 32 * 32);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int tile = i4_dense_tile(M, N, K);
  SF_REQUIRE(tile == 0 || (workspace && aligned16(workspace)), "linear_i4: this shape needs a 16-byte aligned workspace (samfast_linear_i4_workspace)");
  if (tile != 0 && ldy % 8 == 0 && ldy < (1 << 22) && aligned16(y)) return launch_i4_dense(a, dtype == SAMFAST_F16, tile, workspace, s);
  if (M <= SAMFAST_I4_FEW_ROWS && N >= 16) return launch_i4_few(a, dtype == SAMFAST_F16, s);
  return dtype == SAMFAST_F16 ? launch_i4_tiled<ElemF16>(a, s) : launch_i4_tiled<ElemBf16>(a, s);
}
