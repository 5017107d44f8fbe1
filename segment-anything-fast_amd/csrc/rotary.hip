// Rotary positions: pairs of channels of the queries and keys turned by an angle position * frequency,
//   (a, b) -> (a cos - b sin, b cos + a sin) * magnitude,
// over the first `width` channels of a head, the others copied; one launch for queries and keys.
//
// Every value is read and written once, so memory bounds it.  An angle belongs to a token and a pair, not to a head: a workgroup takes a
// few tokens, makes their cosines and sines once and goes through all the heads with them.  The angle is a product in 64 bits, in turns,
// of which only the fraction goes on in 32: at position 10^6 the 24 bits of a float product leave 1/16 of a radian.
#include "samfast_internal.hpp"
#include "attn_relpos_shared.hpp"

#include <type_traits>

namespace samfast {

struct RotarySide {
  const unsigned short* in;
  unsigned short* out;
  int64_t in_b, in_h, in_t, out_b, out_h, out_t;  // elements between images, heads, tokens
};
struct RotaryArgs {
  RotarySide side[2];
  const int64_t* pos;   // axes positions a token
  const double* freq;   // axes * pairs, radians a position
  int64_t pos_b;
  float magnitude;
  int tokens, T, heads_q, heads, D, pairs, axes;
  int items;                  // pieces of a head
  int chunks, copies;         // halves: pieces of an axis, pieces that are only copied
  int block_tokens, block_heads;
  unsigned int div_items, div_turned, div_copies, div_heads, div_chunks;  // 2^32 / d, rounded up: x / d is the upper half of a product where x d < 2^32
};

constexpr int kRotaryThreads = 256;
constexpr int kRotaryPiece = 8;       // channels (halves: pairs) of a piece
constexpr int kRotaryItems = 2048;    // pieces of a workgroup, unless one head has more
constexpr int kRotaryTable = 1024;    // angles of a workgroup
constexpr int kRotaryMaxDim = 1024;
enum { kNeighbours, kHalves, kCopies };

SF_DEVICE u32x4 load_any(const unsigned short* p) {  // 16 bytes from any even address
  u32x4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
SF_DEVICE void store_any(unsigned short* p, u32x4 v) { __builtin_memcpy(p, &v, 16); }
// the first n of eight values, 1 <= n <= 8
SF_DEVICE u32x4 load_some(const unsigned short* p, int n) {
  if (n == 8) return load_any(p);
  u32x4 v = {};
#pragma unroll
  for (int e = 0; e < 7; ++e)
    if (e < n) v[e >> 1] |= (unsigned int)p[e] << (16 * (e & 1));
  return v;
}
SF_DEVICE void store_some(unsigned short* p, u32x4 v, int n) {
  if (n == 8) return store_any(p, v);
#pragma unroll
  for (int e = 0; e < 7; ++e)
    if (e < n) p[e] = (unsigned short)(v[e >> 1] >> (16 * (e & 1)));
}
template <class T>
SF_DEVICE float value(const u32x4& v, int e) { return e & 1 ? T::hi(v[e >> 1]) : T::lo(v[e >> 1]); }

template <class T, bool INTERLEAVED>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(RotaryArgs a) {
  __shared__ f32x2 table[kRotaryTable];  // cosine and sine
  const int t0 = (int)blockIdx.x * a.block_tokens;
  const int nt = min(a.block_tokens, a.tokens - t0);
  const unsigned int b0 = (unsigned int)t0 / (unsigned int)a.T, first = (unsigned int)t0 - b0 * (unsigned int)a.T;
  // image and token in it of this workgroup's token t
  auto place = [&](int t, int64_t& b, int64_t& n) __attribute__((always_inline)) {
    unsigned int over = 0, in = first + (unsigned int)t;
    if (in >= (unsigned int)a.T) {
      over = in / (unsigned int)a.T;
      in -= over * (unsigned int)a.T;
    }
    b = b0 + over;
    n = in;
  };
  const int h0 = blockIdx.y * a.block_heads, nh = min(a.block_heads, a.heads - h0);
  const int angles = a.axes * a.pairs;

  auto make_table = [&]() __attribute__((always_inline)) {
    for (int i = threadIdx.x; i < nt * angles; i += kRotaryThreads) {
      const int t = i / angles, p = i - t * angles;
      int64_t b, n;
      place(t, b, n);
      const double pos = (double)a.pos[b * a.pos_b + n * a.axes + (a.axes == 1 ? 0 : p / a.pairs)];
      double turns = pos * (a.freq[p] * 0.15915494309189535);  // 1 / 2 pi
      turns -= rint(turns);
      float s, c;
      sincospif(2.0f * (float)turns, &s, &c);
      table[i] = f32x2{c * a.magnitude, s * a.magnitude};
    }
    __syncthreads();
  };

  // The pieces of one kind, `items` of them to a head, UNROLL of a thread at a time with all their loads in flight; before the first are used,
  // `ready` is called.
  auto walk = [&](auto kind, unsigned int items, unsigned int div, auto ready) __attribute__((always_inline)) {
    constexpr int KIND = decltype(kind)::value;
    constexpr int UNROLL = KIND == kHalves ? 2 : 4;
    const unsigned int total = (unsigned int)(nt * nh) * items;
    bool first_round = true;
    for (unsigned int i0 = threadIdx.x; first_round || i0 < total; i0 += UNROLL * kRotaryThreads) {
      u32x4 x[UNROLL], y[UNROLL];
      unsigned short* out[UNROLL];
      int at[UNROLL], n[UNROLL], turned[UNROLL];  // first angle, channels (halves: pairs), neighbours: pairs from here on that are turned
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const unsigned int i = i0 + u * kRotaryThreads;
        n[u] = 0;
        if (i >= total) continue;
        const unsigned int row = items == 1 ? i : __umulhi(i, div);
        const int item = (int)(i - row * items);
        const int t = a.block_heads == 1 ? (int)row : (int)__umulhi(row, a.div_heads);  // (0 where heads are split: one token then)
        int h = h0 + (int)row - t * nh;
        int64_t b, token;
        place(t, b, token);
        const RotarySide& s = a.side[h >= a.heads_q];
        if (h >= a.heads_q) h -= a.heads_q;
        int d = item * kRotaryPiece;
        at[u] = t * angles + d / 2;
        turned[u] = angles - d / 2;
        if (KIND == kHalves) {
          const int axis = a.axes == 1 ? 0 : a.chunks == 1 ? item : (int)__umulhi((unsigned int)item, a.div_chunks);
          const int p = d - axis * a.chunks * kRotaryPiece;
          n[u] = min(kRotaryPiece, a.pairs - p);
          at[u] = t * angles + axis * a.pairs + p;
          d = 2 * axis * a.pairs + p;
        } else {
          if (KIND == kCopies) d += 2 * angles;
          n[u] = min(kRotaryPiece, a.D - d);
        }
        const unsigned short* in = s.in + b * s.in_b + h * s.in_h + token * s.in_t + d;
        out[u] = s.out + b * s.out_b + h * s.out_h + token * s.out_t + d;
        x[u] = load_some(in, n[u]);
        if (KIND == kHalves) y[u] = load_some(in + a.pairs, n[u]);
      }
      if (first_round) ready();
      first_round = false;
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        if (n[u] == 0) continue;
        if (KIND == kNeighbours) {
          u32x4 o;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const f32x2 w = table[j < turned[u] ? at[u] + j : 0];
            const float v0 = T::lo(x[u][j]), v1 = T::hi(x[u][j]);
            o[j] = j < turned[u] ? T::pack2(v0 * w[0] - v1 * w[1], v1 * w[0] + v0 * w[1]) : x[u][j];
          }
          store_some(out[u], o, n[u]);
        } else if (KIND == kHalves) {
          u32x4 ox, oy;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const f32x2 w0 = table[at[u] + min(2 * j, n[u] - 1)], w1 = table[at[u] + min(2 * j + 1, n[u] - 1)];
            const float x0 = T::lo(x[u][j]), x1 = T::hi(x[u][j]), y0 = T::lo(y[u][j]), y1 = T::hi(y[u][j]);
            ox[j] = T::pack2(x0 * w0[0] - y0 * w0[1], x1 * w1[0] - y1 * w1[1]);
            oy[j] = T::pack2(y0 * w0[0] + x0 * w0[1], y1 * w1[0] + x1 * w1[1]);
          }
          store_some(out[u], ox, n[u]);
          store_some(out[u] + a.pairs, oy, n[u]);
        } else {
          store_some(out[u], x[u], n[u]);
        }
      }
    }
  };
  if (INTERLEAVED) {
    walk(std::integral_constant<int, kNeighbours>{}, (unsigned int)a.items, a.div_items, make_table);
  } else {
    walk(std::integral_constant<int, kHalves>{}, (unsigned int)(a.axes * a.chunks), a.div_turned, make_table);
    if (a.copies > 0) walk(std::integral_constant<int, kCopies>{}, (unsigned int)a.copies, a.div_copies, [] {});
  }
}

static unsigned int divider(int d) { return (unsigned int)(((uint64_t)1 << 32) / (unsigned int)d + 1); }  // (d > 1)

template <class T>
static int launch_rotary(RotaryArgs a, bool interleaved, hipStream_t stream) {
  const dim3 grid((unsigned int)((a.tokens + a.block_tokens - 1) / a.block_tokens), (unsigned int)((a.heads + a.block_heads - 1) / a.block_heads));
  if (interleaved) hipLaunchKernelGGL((rotary_kernel<T, true>), grid, dim3(kRotaryThreads), 0, stream, a);
  else hipLaunchKernelGGL((rotary_kernel<T, false>), grid, dim3(kRotaryThreads), 0, stream, a);
  return check_launch("rotary_kernel");
}

}  // namespace samfast

extern "C" int samfast_rotary(const void* q, const void* k, void* q_out, void* k_out, const int64_t* positions, int64_t pos_sb, const double* frequencies,
                              int64_t B, int64_t T, int heads_q, int heads_k, int D, int pairs, int axes, int interleaved, float magnitude,
                              const int64_t* strides, int dtype, void* stream) {
  using namespace samfast;
  if (dtype != SAMFAST_BF16 && dtype != SAMFAST_F16) SF_FAIL(SAMFAST_E_UNSUPPORTED, "rotary: element type %d is neither SAMFAST_BF16 nor SAMFAST_F16", dtype);
  SF_REQUIRE(B >= 0 && T >= 0 && heads_q >= 0 && heads_k >= 0 && heads_q <= (1 << 20) && heads_k <= (1 << 20) && T < (1ll << 31),
             "rotary: bad shape B=%lld T=%lld heads=%d, %d", (long long)B, (long long)T, heads_q, heads_k);
  SF_REQUIRE(axes >= 1 && pairs >= 1 && D >= 1 && D <= kRotaryMaxDim && (int64_t)2 * axes * pairs <= D,
             "rotary: %d axes of %d pairs do not fit into %d channels (at most %d)", axes, pairs, D, kRotaryMaxDim);
  SF_REQUIRE(strides, "rotary: null strides");
  if (B == 0 || T == 0 || heads_q + heads_k == 0) return SAMFAST_OK;
  SF_REQUIRE(B < (1ll << 31) / T, "rotary: too many tokens");
  SF_REQUIRE((heads_q == 0 || (q && q_out)) && (heads_k == 0 || (k && k_out)) && positions && frequencies, "rotary: null pointer");
  RotaryArgs a = {};
  const void* in[2] = {q, k};
  void* out[2] = {q_out, k_out};
  for (int i = 0; i < 2; ++i) {
    const int64_t* s = strides + 6 * i;
    a.side[i] = RotarySide{(const unsigned short*)in[i], (unsigned short*)out[i], s[0], s[1], s[2], s[3], s[4], s[5]};
  }
  a.pos = positions;
  a.freq = frequencies;
  a.pos_b = pos_sb;
  a.tokens = (int)(B * T);
  a.magnitude = magnitude;
  a.T = (int)T;
  a.heads_q = heads_q;
  a.heads = heads_q + heads_k;
  a.D = D;
  a.pairs = pairs;
  a.axes = axes;
  const int angles = axes * pairs;
  a.chunks = (pairs + kRotaryPiece - 1) / kRotaryPiece;
  a.copies = (D - 2 * angles + kRotaryPiece - 1) / kRotaryPiece;
  a.items = interleaved ? (D + kRotaryPiece - 1) / kRotaryPiece : axes * a.chunks + a.copies;
  // a workgroup's share: kRotaryItems pieces, fewer where that leaves CUs without one
  int64_t share = (int64_t)a.tokens * a.heads * a.items / 1024;
  share = share < kRotaryThreads ? kRotaryThreads : share > kRotaryItems ? kRotaryItems : share;
  int64_t heads = share / a.items;
  a.block_heads = (int)(heads < 1 ? 1 : heads > a.heads ? a.heads : heads);
  const int parts = (a.heads + a.block_heads - 1) / a.block_heads;
  a.block_heads = (a.heads + parts - 1) / parts;
  int64_t tokens = parts > 1 ? 1 : share / ((int64_t)a.block_heads * a.items);
  if (tokens > kRotaryTable / angles) tokens = kRotaryTable / angles;
  a.block_tokens = (int)(tokens < 1 ? 1 : tokens);
  SF_REQUIRE(parts < 65536, "rotary: too many heads");
  a.div_items = a.items > 1 ? divider(a.items) : 0;
  a.div_turned = axes * a.chunks > 1 ? divider(axes * a.chunks) : 0;
  a.div_copies = a.copies > 1 ? divider(a.copies) : 0;
  a.div_heads = a.block_heads > 1 ? divider(a.block_heads) : 0;
  a.div_chunks = a.chunks > 1 ? divider(a.chunks) : 0;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return dtype == SAMFAST_F16 ? launch_rotary<ElemF16>(a, interleaved != 0, s) : launch_rotary<ElemBf16>(a, interleaved != 0, s);
}
