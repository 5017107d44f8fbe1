// Linears with 4-bit weights over more than a few rows, of any shape: a tiled matrix product whose wavefronts make their own weights.
#include "linear_i4_shared.hpp"

#include <type_traits>

namespace samfast {

// 16 bytes a lane from base + offset to lds + 16 lane; zeros where the offset is kOutside
constexpr unsigned int kOutside = 0x80000000u;
SF_DEVICE void piece_to_lds(const void* base, unsigned int offset, void* lds) {
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, 0x7fffffff, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)lds, 16, offset, 0, 0, 0);
}

// The eight weights (code - zero) * scale of a word in the order of k, rounded to the element type once: code - zero is exact.  zero * scale alone may
// overflow where no weight does, so it is not made (512 x 4096 -> 4096 31.2 us for 30.1 with code * scale - zero * scale as one instruction; with the difference
// in fp32, an instruction a weight instead of half, 31.7).
SF_DEVICE u32x4 i4_weights(ElemBf16, unsigned int w, float scale, float zero) {
  typedef ElemF16::f16x2 f16x2;
  const u32x2 bytes = i4_bytes(w);
  const f16x2 z = {(_Float16)zero, (_Float16)zero};
  float none = -0.0f;
  asm("" : "+v"(none));  // (a product of a half and a float is one instruction as an fma)
  u32x4 o;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes[h], 512.f, false) - z, hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes[h], 512.f, true) - z;
    o[2 * h] = ElemBf16::pack2(fmaf((float)lo[0], scale, none), fmaf((float)lo[1], scale, none));
    o[2 * h + 1] = ElemBf16::pack2(fmaf((float)hi[0], scale, none), fmaf((float)hi[1], scale, none));
  }
  return o;
}
SF_DEVICE u32x4 i4_weights(ElemF16, unsigned int w, float scale, float zero) {
  typedef ElemF16::f16x2 f16x2;
  const u32x2 bytes = i4_bytes(w);
  const f16x2 s = {(_Float16)scale, (_Float16)scale}, z = {(_Float16)zero, (_Float16)zero};
  u32x4 o;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    o[2 * h] = __builtin_bit_cast(unsigned int, (__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes[h], 512.f, false) - z) * s);
    o[2 * h + 1] = __builtin_bit_cast(unsigned int, (__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes[h], 512.f, true) - z) * s);
  }
  return o;
}

// Tiles of 16 MT rows and 16 NT COLS columns, K 128 at a time.  The rows of x are everybody's and go through LDS, one k tile ahead; the columns are
// one wavefront's each, so that a weight is made once in the workgroup and never leaves the registers.  With two SIDES as many wavefronts again take
// every other k tile, and the sides' sums meet in LDS.  (x and weights two k tiles ahead were level.)
//
// Making the weights bounds it: at 512 x 4096 -> 4096 vector instructions take 60 % of the SIMDs' cycles, matrix instructions 24 %, LDS reads 25 % of the
// CUs' cycles, without bank conflicts.
template <int MT, int NT, int COLS, int SIDES>
struct I4Tile {
  static constexpr int BM = 16 * MT, BN = 16 * NT * COLS, STAGE = BM * 256, THREADS = 64 * COLS * SIDES;
  static constexpr int LOADS = 4 * MT / COLS;  // of a wavefront for a k tile of x: eight rows' lines each
  static_assert(4 * MT % COLS == 0 && (SIDES == 1 || SIDES == 2) && (SIDES == 1 || COLS * MT * NT * 1024 <= 2 * SIDES * STAGE) && 2 * SIDES * STAGE <= 160 * 1024, "");
};

template <class T, int MT, int NT, int COLS, int SIDES>
__global__ __launch_bounds__(64 * COLS * SIDES, 2) void linear_i4_kernel(I4Args a) {
  using P = I4Tile<MT, NT, COLS, SIDES>;
  __shared__ __attribute__((aligned(16))) unsigned char lds[2 * SIDES * P::STAGE];
  const int lane = threadIdx.x & 63, lr = lane & 15, lq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % COLS, side = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / COLS;
  unsigned char* mine = lds + 2 * side * P::STAGE;

  // neighbours on an XCD share a column of tiles, eight rows of them at a time
  const unsigned int total = (unsigned int)a.tiles_m * (unsigned int)a.tiles_n;
  const unsigned int pid = xcd_contiguous_id(blockIdx.x, total);
  if (pid >= total) return;
  const unsigned int per_group = 8u * a.tiles_n, first_m = pid / per_group * 8u;
  const unsigned int rows = min((unsigned int)a.tiles_m - first_m, 8u), in_group = pid % per_group;
  const int m0 = (int)(first_m + in_group % rows) * P::BM, n0 = (int)(in_group / rows) * P::BN + wave * 16 * NT;
  // this workgroup's k tiles; the last one of all may end behind K
  const int tiles = (a.K + 127) / 128;
  const int first = (int)((int64_t)tiles * blockIdx.y / gridDim.y), end = (int)((int64_t)tiles * (blockIdx.y + 1) / gridDim.y);

  // ---- x: a load puts eight rows' lines side by side; 16-byte piece c of row r stands at position c ^ ((r >> 1) & 7), where a fragment's read finds
  // no two of its pieces in one bank.  What lies outside the matrix arrives as zeros.
  unsigned int x_off[P::LOADS];
  int x_k[P::LOADS];
#pragma unroll
  for (int i = 0; i < P::LOADS; ++i) {
    const int q = wave + COLS * i, row = 8 * (q % (2 * MT)) + (lane >> 3);
    x_k[i] = q / (2 * MT) * 64 + ((lane & 7) ^ ((row >> 1) & 7)) * 8;
    x_off[i] = m0 + row < a.M ? (unsigned int)row * (unsigned int)(a.ldx * 2) + 2 * x_k[i] : kOutside;
  }
  const unsigned short* xt = a.x + (int64_t)m0 * a.ldx;
  auto load_x = [&](int kt, int stage) __attribute__((always_inline)) {
    unsigned char* to = mine + stage * P::STAGE;
#pragma unroll
    for (int i = 0; i < P::LOADS; ++i) piece_to_lds(xt + kt * 128, kt * 128 + x_k[i] < a.K ? x_off[i] : kOutside, to + (wave + COLS * i) * 1024);
  };
  auto x_piece = [&](int stage, int i, int t) __attribute__((always_inline)) {
    const int row = 16 * i + lr, c = 4 * (t & 1) + lq;
    return *reinterpret_cast<const u32x4*>(mine + stage * P::STAGE + (t >> 1) * P::BM * 128 + row * 128 + ((c ^ ((row >> 1) & 7)) << 4));
  };

  // ---- weights: row r of fragment j holds column 4 NT (r / 4) + 4 j + r % 4, so that a lane ends with 4 NT adjacent ones.  A lane has its
  // column's 32 adjacent codes, and the scale and zero of the group that the 32 inputs of quarter lq belong to.
  struct Weights {
    u32x4 codes[NT];
    unsigned int scale[NT], zero[NT];
  };
  int col[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) col[j] = min(n0 + 4 * NT * (lr >> 2) + 4 * j + (lr & 3), a.N - 1);
  auto load_w = [&](Weights& w, int kt) __attribute__((always_inline)) {
    const int64_t at = (int64_t)i4_group(a, min(4 * kt + lq, (a.K - 1) / 32)) * a.N;
    const unsigned char* zeros = a.zeros ? a.zeros : a.codes;  // (without zeros: not used)
    const int64_t zero_at = a.zeros ? at : 0;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      __builtin_memcpy(&w.codes[j], __builtin_assume_aligned(a.codes + (int64_t)col[j] * (a.K / 2) + kt * 64 + 16 * lq, 4), 16);
      w.scale[j] = a.scales[at + col[j]];
      w.zero[j] = zeros[zero_at + col[j]];
    }
  };
  auto load_w_careful = [&](Weights& w, int kt) __attribute__((always_inline)) {  // the k tile that may end behind K
    const int64_t at = (int64_t)i4_group(a, min(4 * kt + lq, (a.K - 1) / 32)) * a.N;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      w.codes[j] = u32x4{};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (kt * 128 + 32 * lq + 8 * e < a.K) w.codes[j][e] = *reinterpret_cast<const unsigned int*>(a.codes + (int64_t)col[j] * (a.K / 2) + kt * 64 + 16 * lq + 4 * e);
      w.scale[j] = a.scales[at + col[j]];
      w.zero[j] = a.zeros ? a.zeros[at + col[j]] : 0;
    }
  };

  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{};
  const bool one_group = a.group % 128 == 0;  // for a whole k tile
  // (`left`: inputs from the k tile's first on.  Weights behind the last one are zeros: a zero point times a scale may overflow where no weight does)
  auto multiply = [&](const Weights& w, int stage, int left = 128) __attribute__((always_inline)) {
    u32x4 x[2][MT], f[4][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) x[0][i] = x_piece(stage, i, 0);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      u32x4 c = w.codes[j];
      i4_transpose(c);
      const unsigned int sz = w.scale[j] | (a.zeros ? w.zero[j] : 8u) << 24;  // (to the top: of a byte in a register nothing has to be cleared before it is loaded)
      unsigned int of[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) of[t] = sz;
      if (!one_group) {
#pragma unroll
        for (int t = 0; t < 4; ++t) of[t] = (unsigned int)__builtin_amdgcn_ds_bpermute(4 * (16 * t + lr), (int)sz);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f[t][j] = i4_weights(T{}, c[t], T::from_bits((unsigned short)of[t]), (float)(of[t] >> 24));
        if (32 * t + 8 * lq >= left) f[t][j] = u32x4{};
      }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (t < 3) {
#pragma unroll
        for (int i = 0; i < MT; ++i) x[(t + 1) & 1][i] = x_piece(stage, i, t + 1);
      }
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i][j] = T::mfma16(f[t][j], x[t & 1][i], acc[i][j]);
    }
  };

  const int whole = end == tiles && a.K % 128 != 0 ? end - 1 : end;
  auto meet = [&]() __attribute__((always_inline)) {  // all loads are there, for every wavefront, and all reads done
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0070);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  Weights w[2];
  auto ask = [&](auto stage, int kt) __attribute__((always_inline)) {
    constexpr int S = decltype(stage)::value;
    if (kt < end) load_x(kt, S);
    if (kt < whole) load_w(w[S], kt);
    __builtin_amdgcn_sched_barrier(0);
  };
  using S0 = std::integral_constant<int, 0>;
  using S1 = std::integral_constant<int, 1>;
  int kt = first + side;
  ask(S0{}, kt);
  if (first < whole) {
    auto step = [&](auto stage, auto other) __attribute__((always_inline)) {
      meet();
      ask(other, kt + SIDES);
      if (SIDES == 1 || kt < whole) multiply(w[decltype(stage)::value], decltype(stage)::value);
      kt += SIDES;
    };
    for (;;) {
      step(S0{}, S1{});
      if (kt - side >= whole) break;
      step(S1{}, S0{});
      if (kt - side >= whole) break;
    }
  }
  meet();
  if (whole < end && (whole - first) % SIDES == side) {  // its rows were requested with the others
    Weights last;
    load_w_careful(last, whole);
    multiply(last, (whole - first) / SIDES % 2, a.K - 128 * whole);
  }
  if constexpr (SIDES == 2) {
    meet();
    f32x4* sums = reinterpret_cast<f32x4*>(lds) + wave * MT * NT * 64 + lane;
    if (side == 1) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) sums[(i * NT + j) * 64] = acc[i][j];
    }
    meet();
    if (side == 1) return;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] += sums[(i * NT + j) * 64];
  }

  // ---- a lane holds row 16 i + lr and 4 NT adjacent columns
  const int n = n0 + 4 * NT * lq;
  if (n >= a.N) return;
  if (a.parts) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int m = m0 + 16 * i + lr;
      if (m >= a.M) continue;
      float* part = a.parts + ((int64_t)blockIdx.y * a.M + m) * a.N + n;
      if (n + 4 * NT <= a.N) {
#pragma unroll
        for (int j = 0; j < NT; ++j) __builtin_memcpy(part + 4 * j, &acc[i][j], 16);
      } else {
#pragma unroll
        for (int c = 0; c < 4 * NT; ++c)
          if (n + c < a.N) part[c] = acc[i][c / 4][c % 4];
      }
    }
    return;
  }
  float bias[4 * NT];
#pragma unroll
  for (int c = 0; c < 4 * NT; ++c) bias[c] = a.bias ? a.bias[min(n + c, a.N - 1)] : 0.f;
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = m0 + 16 * i + lr;
    if (m >= a.M) continue;
    unsigned short* y = a.y + (int64_t)m * a.ldy + n;
    unsigned int o[2 * NT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        o[2 * j + e] = T::pack2(acc[i][j][2 * e] + bias[4 * j + 2 * e], acc[i][j][2 * e + 1] + bias[4 * j + 2 * e + 1]);
    if (n + 4 * NT <= a.N) {
      __builtin_memcpy(y, o, 8 * NT);
    } else {
#pragma unroll
      for (int c = 0; c < 4 * NT; ++c)
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

// How a product is done, from its sizes alone (the workspace is asked for before the call): what takes least by these estimates in us, which lie within
// a fifth of the times measured, most within a tenth.  Measured in bf16, groups of 128 with zeros, calls that follow one another:
//   tiles: 4 + a k tile's time x k tiles x tiles to a CU, alone on it / not; + 3 and the sums' bytes at 6 TB/s where K is split.  32 x 64 / 64 x 64 /
//     128 x 128 tiles: 128 x 1280 -> 3840 7.7 / 8.8 / 17.6, 333 x 1000 -> 1003 7.4 / 8.6 / 15.6, 256 x 4096 -> 4096 24.9 / 20.3 / 23.8 (K in four), 512 x 4096 -> 4096
//     42 / 30.3 / 34 (K in four), 1024 x 1280 -> 3840 30 / 23.2 / 19.2, 1024 x 4096 -> 4096 79 / 58 / 47; 64 x 64 tiles, K whole / in four: 64 x 4096 -> 4096 20 / 12.1,
//     64 x 8192 -> 8192 36 / 21.5, 256 x 4096 -> 4096 20.3 / 25.5.
//   dense (linear_i4_dense.hip): by its own estimate.  128 x 128 tiles / dense: 4096 x 1280 -> 5120 72 / 52, 5405 x 3832 -> 4828 266 / 181, 8000 x 4096 -> 3001 239 / 160,
//     4096 x 1280 -> 5121 88 / 58, 10000 x 328 -> 4001 69 / 56, 2048 x 4096 -> 4096 82 / 71, 16384 x 1000 -> 1003 53 / 46, but 1024 x 4096 -> 4096 50 / 64, 512 x 8192 -> 8192
//     92 / 140, 4096 x 1280 -> 1280 26.7 / 27.3; 1024 x 8192 -> 8192 157 / 168 on one card and 162 / 146 on another (the second is taken).
// Up to SAMFAST_I4_FEW_ROWS rows linear_i4_few.hip: 24 x 4096 -> 4096 7.1, tiles with K in four 10.0.
struct I4Plan {
  int dense;   // columns / 32 of the dense product's tile, or 0
  int tile;    // 32 x 64, 64 x 64, 128 x 128
  int splits;  // of K
};
static I4Plan i4_plan(int64_t M, int N, int K) {
  I4Plan p = {0, 0, 1};
  if (M <= SAMFAST_I4_FEW_ROWS && N >= 16) return p;
  static const struct { int rows, cols, sides; double alone, beside; } kTiles[3] = {{32, 64, 2, 0.35, 0.30}, {64, 64, 2, 0.52, 0.42}, {128, 128, 1, 1.25, 1.0}};
  const int k_tiles = (K + 127) / 128;
  double least = 0.0;
  for (int t = 0; t < 3; ++t)
    for (int splits : {1, 2, 3, 4, 6, 8}) {
      const int sides = kTiles[t].sides;
      if (splits > 1 && k_tiles < 2 * splits) break;
      const int each = ((k_tiles + splits - 1) / splits + sides - 1) / sides * sides;
      const double blocks = (double)((M + kTiles[t].rows - 1) / kTiles[t].rows) * ((N + kTiles[t].cols - 1) / kTiles[t].cols) * splits / 256.0;
      const double time = 4.0 + each * (blocks <= 1.0 ? kTiles[t].alone : blocks <= 4.0 ? (double)(int)(blocks + 0.999) * kTiles[t].beside : blocks * kTiles[t].beside) +
                          (splits > 1 ? 3.0 + 8.0 * splits * (double)M * N / 6e6 : 0.0);
      if (least == 0.0 || time < least) {
        least = time;
        p = I4Plan{0, t, splits};
      }
    }
  double dense = 0.0;
  const int columns = i4_dense_tile(M, N, K, &dense);
  // (against the dense product the estimate of the largest tiles is too short: their ends, and the power limit from a round of them on; 16384 x 1000 -> 1003 53, 36 above)
  if (p.tile == 2) least = 1.18 * (least - 4.0) + 4.0 + 2.0 * fmax((double)((M + 127) / 128) * ((N + 127) / 128) / 256.0 - 1.0, 0.0);
  if (columns && dense < least) p = I4Plan{columns, 0, 1};
  return p;
}

template <class T>
static int launch_i4_tiled(I4Args a, const I4Plan& plan, hipStream_t stream) {
  auto go = [&](auto mt, auto nt, auto cols, auto sides) {
    using P = I4Tile<decltype(mt)::value, decltype(nt)::value, decltype(cols)::value, decltype(sides)::value>;
    a.tiles_m = (a.M + P::BM - 1) / P::BM;
    a.tiles_n = (a.N + P::BN - 1) / P::BN;
    const int64_t tiles = ((int64_t)a.tiles_m * a.tiles_n + 7) / 8 * 8;
    SF_REQUIRE(launchable(tiles, P::THREADS), "linear_i4: %lld tiles are too many for a launch", (long long)tiles);
    const dim3 grid((unsigned int)tiles, (unsigned int)plan.splits);
    hipLaunchKernelGGL((linear_i4_kernel<T, decltype(mt)::value, decltype(nt)::value, decltype(cols)::value, decltype(sides)::value>), grid,
                       dim3(P::THREADS), 0, stream, a);
    if (const int rc = check_launch("linear_i4_kernel")) return rc;
    if (!a.parts) return SAMFAST_OK;
    hipLaunchKernelGGL(i4_sum_kernel<T>, dim3((unsigned int)(((int64_t)a.M * ((a.N + 3) / 4) + 255) / 256)), dim3(256), 0, stream, a, plan.splits);
    return check_launch("i4_sum_kernel");
  };
  using C1 = std::integral_constant<int, 1>;
  using C2 = std::integral_constant<int, 2>;
  using C4 = std::integral_constant<int, 4>;
  using C8 = std::integral_constant<int, 8>;
  if (plan.tile == 0) return go(C2{}, C1{}, C4{}, C2{});
  if (plan.tile == 1) return go(C4{}, C1{}, C4{}, C2{});
  return go(C8{}, C1{}, C8{}, C1{});
}

}  // namespace samfast

extern "C" int64_t samfast_linear_i4_workspace(int64_t M, int N, int K) {
  using namespace samfast;
  SF_REQUIRE(M >= 0 && N > 0 && K > 0, "linear_i4_workspace: bad shape M=%lld N=%d K=%d", (long long)M, N, K);
  const I4Plan plan = i4_plan(M, N, K);
  return plan.dense ? i4_dense_workspace(M, N, K) : plan.splits > 1 ? (int64_t)plan.splits * M * N * 4 : 0;
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
  const I4Plan plan = i4_plan(M, N, K);
  SF_REQUIRE((plan.dense == 0 && plan.splits == 1) || (workspace && aligned16(workspace)),
             "linear_i4: this shape needs a 16-byte aligned workspace (samfast_linear_i4_workspace)");
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
  if (plan.dense && ldy < (1 << 22)) return launch_i4_dense(a, dtype == SAMFAST_F16, plan.dense, workspace, s);
  if (M <= SAMFAST_I4_FEW_ROWS && N >= 16) return launch_i4_few(a, dtype == SAMFAST_F16, s);
  if (plan.splits > 1) a.parts = reinterpret_cast<float*>(workspace);
  return dtype == SAMFAST_F16 ? launch_i4_tiled<ElemF16>(a, plan, s) : launch_i4_tiled<ElemBf16>(a, plan, s);
}
