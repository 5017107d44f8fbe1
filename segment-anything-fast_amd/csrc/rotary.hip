// Rotary positions: pairs of channels of the queries and keys turned by an angle position * frequency,
//   (a, b) -> (a cos - b sin, b cos + a sin) * magnitude,
// over the first `width` channels of a head, the others copied; one launch for queries and keys.
//
// Every value is read and written once, so memory bounds it.  An angle belongs to a token and a pair, not to a head: a workgroup takes a
// few tokens, makes their cosines and sines once and turns the heads with them, 32 to 64 bytes to a thread, all of them requested before the table is made.  The angle is a product in 64 bits, in turns,
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
  int in_place;
  int tokens, T, heads_q, heads, D, pairs, axes;
  int items;                  // a head's pieces; halves: the first `turns` of them are turned, `chunks` for an axis, the others copied
  int chunks, turns;
  int block_tokens, block_heads;
  unsigned int div_items, div_heads;  // 2^32 / d, rounded up: x / d is the upper half of a product where x d < 2^32
};

constexpr int kRotaryThreads = 256;
constexpr int kRotaryPiece = 8;       // values of 16 bytes
constexpr int kRotaryTable = 1024;    // angles of a workgroup
constexpr int kRotaryMaxDim = 1024;
constexpr int kRotaryMaxAxes = 64;    // halves: a head has up to kRotaryMaxDim / 2 / kRotaryPiece + axes pieces, which a workgroup's threads have to hold
// cosine and sine of the workgroup's angle i: a lane reads PLANES adjacent ones, which lie apart so that its neighbours' lie side by side
template <int PLANES>
SF_DEVICE int table_at(int i) { return i % PLANES * (kRotaryTable / PLANES + 1) + i / PLANES; }

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

// EACH pieces of a thread
template <class T, bool INTERLEAVED, int EACH>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(RotaryArgs a) {
  constexpr int PLANES = INTERLEAVED ? 4 : 8;
  static_assert(kRotaryMaxDim / kRotaryPiece + kRotaryMaxAxes <= EACH * kRotaryThreads, "a workgroup has whole heads");
  __shared__ f32x2 table[kRotaryTable + PLANES];
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

  // What a thread has of a head at a time: kRotaryPiece channels (neighbours), or as many pairs of halves, lower and upper channels, or twice
  // as many channels that are only copied
  struct Where {
    const unsigned short* in;
    unsigned short* out;
    int angle, turned;  // its first angle, and how many pairs from there on are turned
    int n, second, n2;  // values of the first 16 bytes, where the second ones start, values of these
  };
  const unsigned int total = (unsigned int)(nt * nh * a.items);
  auto where = [&](unsigned int i) __attribute__((always_inline)) {
    Where w = {};
    if (i >= total) return w;
    const unsigned int row = a.items == 1 ? i : __umulhi(i, a.div_items);
    const int item = (int)(i - row * a.items);
    const int t = a.block_heads == 1 ? (int)row : (int)__umulhi(row, a.div_heads);  // (0 where heads are split: one token then)
    int h = h0 + (int)row - t * nh;
    int64_t b, token;
    place(t, b, token);
    const RotarySide& s = a.side[h >= a.heads_q];
    if (h >= a.heads_q) h -= a.heads_q;
    // (a piece that would end behind its like lies over the one before it, so that it is whole too: both write the same there)
    int d = item * kRotaryPiece;
    w.angle = t * angles;
    if (INTERLEAVED) {
      if (a.D % 2 == 0 && a.D >= kRotaryPiece) d = min(d, a.D - kRotaryPiece);
      w.n = min(kRotaryPiece, a.D - d);
      w.angle += d / 2;
      w.turned = angles - d / 2;
    } else if (item < a.turns) {
      const int axis = a.axes == 1 ? 0 : item / a.chunks;
      int p = d - axis * a.chunks * kRotaryPiece;
      if (a.pairs >= kRotaryPiece) p = min(p, a.pairs - kRotaryPiece);
      d = 2 * axis * a.pairs + p;
      w.angle += axis * a.pairs + p;
      w.turned = w.n = w.n2 = min(kRotaryPiece, a.pairs - p);
      w.second = a.pairs;
    } else {
      const int last = a.D - 2 * angles >= kRotaryPiece ? a.D - kRotaryPiece : a.D;
      d = 2 * angles + (item - a.turns) * 2 * kRotaryPiece;
      const int d2 = min(d + kRotaryPiece, last);
      w.n2 = d + kRotaryPiece < a.D ? min(kRotaryPiece, a.D - d2) : 0;
      d = min(d, last);
      w.n = min(kRotaryPiece, a.D - d);
      w.second = d2 - d;
    }
    w.in = s.in + b * s.in_b + h * s.in_h + token * s.in_t + d;
    w.out = s.out + b * s.out_b + h * s.out_h + token * s.out_t + d;
    return w;
  };

  // all loads are under way before the table is made
  u32x4 x[EACH], y[EACH];
  Where w[EACH];
#pragma unroll
  for (int u = 0; u < EACH; ++u) {
    w[u] = where(threadIdx.x + u * kRotaryThreads);
    x[u] = y[u] = u32x4{};
    if (w[u].n > 0) x[u] = load_some(w[u].in, w[u].n);
    if (!INTERLEAVED && w[u].n2 > 0) y[u] = load_some(w[u].in + w[u].second, w[u].n2);
  }
  for (int i = threadIdx.x; i < nt * angles; i += kRotaryThreads) {
    const int t = i / angles, p = i - t * angles;
    int64_t b, n;
    place(t, b, n);
    const double pos = (double)a.pos[b * a.pos_b + n * a.axes + (a.axes == 1 ? 0 : p / a.pairs)];
    double turns = pos * (a.freq[p] * 0.15915494309189535);  // 1 / 2 pi
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * (float)turns, &s, &c);
    table[table_at<PLANES>(i)] = f32x2{c * a.magnitude, s * a.magnitude};
  }
  if (a.in_place) __builtin_amdgcn_s_waitcnt(0x0f70);  // (what two threads read is read before either of them writes)
  __syncthreads();
#pragma unroll
  for (int u = 0; u < EACH; ++u) {
    if (w[u].n == 0) continue;
    if (INTERLEAVED) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool turned = j < w[u].turned;
        const f32x2 c = table[table_at<PLANES>(turned ? w[u].angle + j : 0)];
        const float v0 = T::lo(x[u][j]), v1 = T::hi(x[u][j]);
        if (turned) x[u][j] = T::pack2(v0 * c[0] - v1 * c[1], v1 * c[0] + v0 * c[1]);
      }
    } else if (w[u].turned > 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x2 c0 = table[table_at<PLANES>(w[u].angle + min(2 * j, w[u].turned - 1))];
        const f32x2 c1 = table[table_at<PLANES>(w[u].angle + min(2 * j + 1, w[u].turned - 1))];
        const float x0 = T::lo(x[u][j]), x1 = T::hi(x[u][j]), y0 = T::lo(y[u][j]), y1 = T::hi(y[u][j]);
        x[u][j] = T::pack2(x0 * c0[0] - y0 * c0[1], x1 * c1[0] - y1 * c1[1]);
        y[u][j] = T::pack2(y0 * c0[0] + x0 * c0[1], y1 * c1[0] + x1 * c1[1]);
      }
    }
    store_some(w[u].out, x[u], w[u].n);
    if (!INTERLEAVED && w[u].n2 > 0) store_some(w[u].out + w[u].second, y[u], w[u].n2);
  }
}

static unsigned int divider(int d) { return (unsigned int)(((uint64_t)1 << 32) / (unsigned int)d + 1); }  // (d > 1)

// Pieces of a thread.  Neighbours 2 / 4: 16 x 4096 tokens, 32 heads of 80 194 / 127 us, 8 x 4096, 40 of 128 162 / 124; halves 1 / 2 / 4: 129 / 143 /
// 143, 126 / 125 / 129, 30011 tokens, 28 heads, 64 of 96 channels 59 / 64 / 67.
constexpr int kRotaryNeighbours = 4, kRotaryHalves = 1;

template <class T>
static int launch_rotary(RotaryArgs a, bool interleaved, hipStream_t stream) {
  const dim3 grid((unsigned int)((a.tokens + a.block_tokens - 1) / a.block_tokens), (unsigned int)((a.heads + a.block_heads - 1) / a.block_heads));
  if (interleaved) hipLaunchKernelGGL((rotary_kernel<T, true, kRotaryNeighbours>), grid, dim3(kRotaryThreads), 0, stream, a);
  else hipLaunchKernelGGL((rotary_kernel<T, false, kRotaryHalves>), grid, dim3(kRotaryThreads), 0, stream, a);
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
  SF_REQUIRE(axes <= kRotaryMaxAxes, "rotary: %d axes (at most %d)", axes, kRotaryMaxAxes);
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
  a.in_place = q_out == q || (k && k_out == k);
  a.T = (int)T;
  a.heads_q = heads_q;
  a.heads = heads_q + heads_k;
  a.D = D;
  a.pairs = pairs;
  a.axes = axes;
  const int angles = axes * pairs;
  a.chunks = (pairs + kRotaryPiece - 1) / kRotaryPiece;
  a.turns = axes * a.chunks;
  a.items = interleaved ? (D + kRotaryPiece - 1) / kRotaryPiece : a.turns + (D - 2 * angles + 2 * kRotaryPiece - 1) / (2 * kRotaryPiece);
  // a workgroup's share: what its threads hold at most, fewer where that leaves CUs without one
  const int64_t most = (interleaved ? kRotaryNeighbours : kRotaryHalves) * kRotaryThreads;
  int64_t share = (int64_t)a.tokens * a.heads * a.items / 1024;
  share = share < kRotaryThreads ? kRotaryThreads : share > most ? most : share;
  int64_t heads = share / a.items;
  a.block_heads = (int)(heads < 1 ? 1 : heads > a.heads ? a.heads : heads);
  const int parts = (a.heads + a.block_heads - 1) / a.block_heads;
  a.block_heads = (a.heads + parts - 1) / parts;
  int64_t tokens = parts > 1 ? 1 : share / ((int64_t)a.block_heads * a.items);
  if (tokens > kRotaryTable / angles) tokens = kRotaryTable / angles;
  a.block_tokens = (int)(tokens < 1 ? 1 : tokens);
  SF_REQUIRE(parts < 65536, "rotary: too many heads");
  a.div_items = a.items > 1 ? divider(a.items) : 0;
  a.div_heads = a.block_heads > 1 ? divider(a.block_heads) : 0;
  SF_REQUIRE(launchable((a.tokens + a.block_tokens - 1) / a.block_tokens, kRotaryThreads), "rotary: too many tokens");
  for (int i = 0; i < 2; ++i) {
    const RotarySide& t = a.side[i];
    SF_REQUIRE(!t.out || t.out != t.in || (t.out_b == t.in_b && t.out_h == t.in_h && t.out_t == t.in_t), "rotary: in place, but in another layout");
  }
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return dtype == SAMFAST_F16 ? launch_rotary<ElemF16>(a, interleaved != 0, s) : launch_rotary<ElemBf16>(a, interleaved != 0, s);
}
