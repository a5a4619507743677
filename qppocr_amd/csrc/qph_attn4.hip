// Attention over the 4-bit key / value cache (format: qph_fp4.h).
//
// For a new token at position p of its sequence and a query head of the
// cache's head h, over the visible keys j:
//   s_j = scale q . k_j,  m = max s_j,  o = sum exp(s_j - m) v_j / sum exp(s_j - m)
// in one pass over the cache with a running m (the sums so far are multiplied
// by exp(m_old - m_new) when it grows).
//
// A wave holds 16 NQ rows (a row is one new token and one query head of h) as
// the columns of its MFMAs and walks the keys in tiles of 32:
//   S^T [16 keys][16 rows] = K [16][32 d] Q^T [32 d][16]   (D: lane's row, 4 keys)
//   O^T [16 d][16 rows]   += V^T [16 d][32 keys] P^T [32 keys][16]
// The sum over keys (or d) inside an MFMA may take them in any order that both
// operands share, and both orders are chosen so that nothing moves between
// lanes: lane group g holds, of a 32-key tile, the keys 4 g .. 4 g + 3 and
// 16 + 4 g .. 16 + 4 g + 3, which are those of its four S values of either
// half, so exp(s - m) is the second product's operand where it stands; and it
// reads dh / 4 neighbouring d of a key, W = dh / 32 words of codes.  Of a
// value row lane i reads bytes W i .. W i + W - 1, the 2 W elements d = 2 W i + m
// that become row i of product m.  Codes turn into bfloat16 in registers, one
// instruction for two.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "qph_fp4.h"

namespace qph {

struct Attn4 {
  const unsigned char *kc, *ks, *vc, *vs;
  int64_t n_pages;
  int shift;
  int heads, group;               // the cache's heads, query heads to each
  const void* q;
  void* out;
  float* lse;                     // [tokens][heads * group], or NULL
  int64_t qt, qh, ot, oh;         // strides of a token and a head
  int64_t tokens;
  int batch;
  const int32_t* table;
  int64_t table_stride;
  int max_pages;
  const int32_t* lens;
  const int32_t* starts;          // or NULL: `news` tokens a sequence
  int news;
  float scale;
  int causal, window;
  int row_tiles, splits;          // grid: row tiles x splits x heads x batch
  int64_t chunk;                  // keys a split
  float* part_o;                  // [split][token][query head][dh], splits > 1
  float* part_ml;                 // [split][token][query head][2]
};

constexpr int64_t kMaxKeys = 0x7fffff00;     // of one sequence: positions stay in 31 bits

// The maximum of a wave with more rows is a bound, set 2^8 past the largest score
// so far and moved where a score passes it, so that the sums are seldom scaled
// and the lanes of a column seldom compared.  (Past it, not at it: no term is
// above 1, and the sums overflow no sooner than they would with the maximum.)
constexpr float kLazy = 8.0f;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// The maximum is kept as a score m; the terms are 2^(s c - m c), c = |scale|
// log2 e.  With m c rounded, a term is one fused operation and all terms of the
// row are off by the same factor 2^r, r up to half a unit of m c, which the
// sums share.  Past this bound 2^r is more than 2^(1/32), later out of float32's
// range, and the row's terms are 2^((s - m) c), whose largest is 1: such a row
// is walked again with its m known.  (In every tile both cost more: 5 to 7 % of a
// chunk's time as a branch or as a difference ahead of the product.)
constexpr float kFar = 1048576.0f;

__device__ __forceinline__ bool is_far(float mc) { return fabsf(mc) >= kFar; }

// log2 of the factor from sums with the maximum `was` to sums with `top`; was <= top,
// top not -infinity.
__device__ __forceinline__ float rescale(float was, float top, float c) {
  const float wc = was * c, tc = top * c;
  if (is_far(wc)) return is_far(tc) ? (was - top) * c : __builtin_fmaf(was, c, -tc);
  return is_far(tc) ? -__builtin_fmaf(top, c, -wc) : wc - tc;
}

// log of the sum of the row's exponentials; l the sum of its terms.
__device__ __forceinline__ float log_sum(float m, float l, float scale) {
  const float mc = m * (scale * kLog2e);
  return (is_far(mc) ? m * scale : mc * kLn2) + logf(l);
}

// The larger over the four lanes of one column (lane ^ 16, lane ^ 32).
__device__ __forceinline__ float column_max(float v) {
  u32x2 a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

__device__ __forceinline__ float column_sum(float v) {
  u32x2 a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// What a lane reads of a row of dh = 32 W elements.
template <int W>
struct Lane {
  static constexpr bool odd = W == 3 || W == 6;        // its part straddles two blocks
  static constexpr int kblocks = W == 8 || odd ? 2 : 1;   // scales of its W words of a key
  static constexpr int vblocks = odd ? 2 : 1;             // and of its W bytes of a value
  static constexpr int vwords = (W + 3) / 4;           // words that hold W bytes
};

// Page numbers of the two halves of a 32-key tile, by scalar loads: they are
// asked for two tiles ahead, and waiting for them does not wait for the
// vector loads in flight.
struct PageIds {
  int id[2];
};

typedef const __attribute__((address_space(4))) int32_t* ScalarI32;

__device__ __forceinline__ PageIds page_ids(const Attn4& a, ScalarI32 table, int j0, int khi) {
  PageIds p;
#pragma unroll
  for (int u = 0; u < 2; u++) {
    // (past the last key: the last one's page again, an entry that exists)
    const int j = min(j0 + 16 * u, khi - 1);
    p.id[u] = table[j >> a.shift];
  }
  return p;
}

// Where the halves lie; a page outside the pool holds no keys (page 0 is read
// in its place, and masked).
struct Pages {
  int64_t row[2];
  bool there[2];
};

__device__ __forceinline__ Pages find_pages(const Attn4& a, const PageIds& ids, int j0, int h) {
  Pages p;
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const int page = ids.id[u], j = j0 + 16 * u;
    p.there[u] = page >= 0 && page < a.n_pages;
    p.row[u] = (((int64_t)(p.there[u] ? page : 0) * a.heads + h) << a.shift) +
               (j & ((1 << a.shift) - 1));
  }
  return p;
}

// A lane's part of 32 keys and values: W words of two keys, W bytes of eight
// values, and their scales.
template <int W>
struct KeyTile {
  unsigned w[2][W], s[2][Lane<W>::kblocks];
};

template <int W>
struct ValueTile {
  unsigned w[8][Lane<W>::vwords], s[8][Lane<W>::vblocks];
};

// A lane's place in a tile's half, in bytes: the loads take a uniform base and
// this.
template <int W>
struct Place {
  static constexpr unsigned span = W == 3 ? 4 : W == 6 ? 8 : W;   // bytes that a value load takes
  unsigned k, ks, ks1, v, vs, vs1, shift;
  __device__ __forceinline__ Place(unsigned li, unsigned kg) {
    k = li * (16 * W) + kg * (4 * W);
    ks = li * W + W * kg / 4;
    ks1 = li * W + (W * kg + W - 1) / 4;
    // (W of 3 or 6 bytes by a word, or two, that stays inside the row)
    const unsigned at = min(W * li, 16 * W - span);
    v = kg * (64 * W) + at;
    shift = 8 * (W * li - at);
    vs = kg * (4 * W) + W * li / 16;
    vs1 = kg * (4 * W) + (W * li + W - 1) / 16;
  }
};

template <int W>
__device__ __forceinline__ void load_keys(const Attn4& a, const Pages& pg, const Place<W>& at,
                                          KeyTile<W>& t) {
#pragma unroll
  for (int u = 0; u < 2; u++) {
    __builtin_memcpy(t.w[u], a.kc + pg.row[u] * (16 * W) + at.k, 4 * W);
    const unsigned char* s = a.ks + pg.row[u] * W;
    t.s[u][0] = s[at.ks];
    if constexpr (Lane<W>::kblocks > 1) t.s[u][1] = s[at.ks1];
  }
}

template <int W>
__device__ __forceinline__ void load_values(const Attn4& a, const Pages& pg, const Place<W>& at,
                                            ValueTile<W>& t) {
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const unsigned char* p = a.vc + pg.row[e / 4] * (16 * W) + at.v;
    const unsigned char* s = a.vs + pg.row[e / 4] * W;
    constexpr unsigned row = 16 * W;
    const unsigned r = e % 4;
    if constexpr (W == 1) t.w[e][0] = p[r * row];
    else if constexpr (W == 2) t.w[e][0] = *(const unsigned short*)(p + r * row);
    else __builtin_memcpy(t.w[e], p + r * row, sizeof t.w[e]);
    t.s[e][0] = s[at.vs + r * W];
    if constexpr (Lane<W>::vblocks > 1) t.s[e][1] = s[at.vs1 + r * W];
  }
}

// (Registers: three waves a SIMD hide more of the loads than the last of them
// are worth; 32 sequences of 4096 keys, float16: 43 us so, 48 with two.)
template <typename E, int W, int NQ, int WS>
__global__ __launch_bounds__(256, NQ == 1 && W <= 4 && E::terms < 3 ? 3 : 1) void attn4_kernel(Attn4 a) {
  // The exponentials' terms in the second product: all 24 bits for float32.  For
  // the two-byte types 16 bits, the one rounding between q and out, far below
  // the output's own 8 or 11: against 64 bits the error stays that of rounding
  // the output (relative 1.70e-3 in a bfloat16 batch either way), 0.3 % of the
  // elements become the neighbour of the nearest number (0.03 % with three
  // terms, 0.06 % in torch's float32).  Three terms cost 16 % of a chunk's time
  // (325 and 378 us), 8 % of a long cache's in float16, 2 % of a batch's; the
  // first term rounded instead of cut off halves the 0.3 % for 2.5 % of a chunk's.
  // The sums l are of the terms themselves, not of these.
  constexpr int T = E::terms, PT = T < 2 ? 2 : T;
  constexpr int DH = 32 * W;
  extern __shared__ float lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, kg = lane >> 4;
  unsigned id = blockIdx.x;
  const int rt0 = id % a.row_tiles; id /= a.row_tiles;
  const int split = id % a.splits; id /= a.splits;
  const int h = id % a.heads;
  const int b = id / a.heads;

  // this sequence's new tokens and cached keys, inside what the caller's
  // buffers hold whatever the device arrays say
  int64_t t0, t1;
  if (a.starts) {
    t0 = min(max((int64_t)a.starts[b], (int64_t)0), a.tokens);
    t1 = min(max((int64_t)a.starts[b + 1], t0), a.tokens);
  } else {
    t0 = (int64_t)b * a.news;
    t1 = t0 + a.news;
  }
  const int news = (int)(t1 - t0);
  const int room = (int)min((int64_t)a.max_pages << a.shift, kMaxKeys);
  const int len = min(max(a.lens[b], 0), room);
  const int64_t rows = (int64_t)news * a.group;
  const ScalarI32 table = (ScalarI32)(a.table + b * a.table_stride);
  const int first = len - news;          // position of the first new token
  const int base = a.window > 0 ? (int)max((int64_t)0, (int64_t)first - a.window + 1) & ~31 : 0;
  const int from = (int)min(base + split * a.chunk, (int64_t)room);
  const int to = split == a.splits - 1 ? room : (int)min(from + a.chunk, (int64_t)room);

  for (int64_t tile = WS == 4 ? rt0 : (int64_t)rt0 * 4 + wave; tile * 16 * NQ < rows;
       tile += (int64_t)a.row_tiles * (WS == 4 ? 1 : 4)) {
    // (a row has seen a key if and only if its sum is not 0: the largest score's
    // term is 1 or near it, and NaN is not 0 either)
    // rows of this wave: query fragments, visible keys [lo, hi)
    bf16x8 qf[NQ][T][W];
    int64_t tok[NQ];
    int lo[NQ], hi[NQ], head[NQ];
    bool live[NQ];
    int wlo = room, whi = 0;
    const float sign = a.scale < 0.0f ? -1.0f : 1.0f;
#pragma unroll
    for (int q = 0; q < NQ; q++) {
      const int64_t r = tile * 16 * NQ + 16 * q + li;
      live[q] = r < rows;
      const int64_t rr = live[q] ? r : rows - 1;
      const int i = (int)(rr / a.group);
      head[q] = h * a.group + (int)(rr - (int64_t)i * a.group);
      tok[q] = t0 + i;
      const int pos = first + i;
      hi[q] = a.causal ? min(len, max(pos + 1, 0)) : len;
      lo[q] = a.window > 0 ? (int)max((int64_t)0, (int64_t)pos - a.window + 1) : 0;
      if (!live[q]) lo[q] = hi[q] = 0;
      if (lo[q] < hi[q]) { wlo = min(wlo, lo[q]); whi = max(whi, hi[q]); }
      const typename E::type* p = (const typename E::type*)a.q + tok[q] * a.qt + head[q] * a.qh;
#pragma unroll
      for (int n = 0; n < W; n++) {
        float v[8];
        bf16x8 f[T];
        load8<E>(p + 8 * (W * kg + n), v);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] *= sign;
        split8<T>(v, f);
#pragma unroll
        for (int t = 0; t < T; t++) qf[q][t][n] = f[t];
      }
    }
#pragma unroll
    for (int d = 1; d < 16; d *= 2) {
      wlo = min(wlo, __shfl_xor(wlo, d));
      whi = max(whi, __shfl_xor(whi, d));
    }
    const float c = fabsf(a.scale) * kLog2e;
    const int klo = __builtin_amdgcn_readfirstlane(max(wlo & ~31, from));
    const int khi = __builtin_amdgcn_readfirstlane(min(whi, to));

    const Place<W> place(li, kg);
    f32x4 o[NQ][2 * W];
    float m[NQ], l[NQ], shift[NQ];     // shift: what a second walk takes off the scores

    // minimum and maximum of the live rows' borders: between them a tile needs no masks
    int all_lo = 0, all_hi = khi;
#pragma unroll
    for (int q = 0; q < NQ; q++)
      if (live[q]) { all_lo = max(all_lo, lo[q]); all_hi = min(all_hi, hi[q]); }
#pragma unroll
    for (int d = 1; d < 16; d *= 2) {
      all_lo = max(all_lo, __shfl_xor(all_lo, d));
      all_hi = min(all_hi, __shfl_xor(all_hi, d));
    }
    all_lo = __builtin_amdgcn_readfirstlane(max(all_lo, from));
    all_hi = __builtin_amdgcn_readfirstlane(all_hi);

    // (the bound's distance as a score; it vanishes beside a far one)
    const float lazy = fminf(kLazy / c, FLT_MAX);
    bool careful = false;      // second run
    auto compute = [&](const KeyTile<W>& kt, ValueTile<W>& vt, const Pages& pg, int j0) __attribute__((always_inline)) {
      f32x4 s[2][NQ];
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const int g0 = W * kg / 4;
        const float s0 = scale_of_byte(kt.s[u][0]);
        const float s1 = Lane<W>::kblocks > 1 ? scale_of_byte(kt.s[u][Lane<W>::kblocks - 1]) : s0;
#pragma unroll
        for (int q = 0; q < NQ; q++) s[u][q] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int n = 0; n < W; n++) {
          const bf16x8 kf = fp4_word(kt.w[u][n], (W * kg + n) / 4 == g0 ? s0 : s1);
#pragma unroll
          for (int q = 0; q < NQ; q++)
#pragma unroll
            for (int t = T - 1; t >= 0; t--) s[u][q] = mfma16(kf, qf[q][t][n], s[u][q]);
        }
      }
      // masks, only where a border lies in the tile or a page is none
      if (j0 < all_lo || j0 + 32 > all_hi || !(pg.there[0] && pg.there[1])) {
#pragma unroll
        for (int q = 0; q < NQ; q++)
#pragma unroll
          for (int u = 0; u < 2; u++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
              const int j = j0 + 16 * u + 4 * kg + r;
              const bool see = pg.there[u] && j >= max(lo[q], from) && j < min(hi[q], to);
              s[u][q][r] = see ? s[u][q][r] - shift[q] : -INFINITY;
            }
        // the values of keys that no row sees, whatever stands there, are zeros
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int j = j0 + 16 * (e / 4) + 4 * kg + e % 4;
          if (!pg.there[e / 4] || j < wlo || j >= khi) {
#pragma unroll
            for (int i = 0; i < Lane<W>::vblocks; i++) vt.s[e][i] = 127;
#pragma unroll
            for (int i = 0; i < Lane<W>::vwords; i++) vt.w[e][i] = 0;
          }
        }
      }
      // running maximum, exponentials
      bf16x8 pf[NQ][PT];
#pragma unroll
      for (int q = 0; q < NQ; q++) {
        float mx = s[0][q][0];
#pragma unroll
        for (int e = 1; e < 8; e++) mx = fmaxf(mx, s[e / 4][q][e % 4]);
        float top = m[q];
        bool grows;
        if constexpr (NQ == 1) {
          top = fmaxf(top, column_max(mx));
          grows = top > m[q];
        } else {
          grows = mx > m[q];
        }
        if (__any(grows)) {
          if constexpr (NQ > 1) {
            const float most = column_max(mx);
            if (most > top) top = fminf(most + lazy, fmaxf(most, FLT_MAX));
          }
          const float keep = exp2_(m[q] * c - (top == -INFINITY ? 0.0f : top * c));
          m[q] = top;
          l[q] *= keep;
#pragma unroll
          for (int x = 0; x < 2 * W; x++)
#pragma unroll
            for (int r = 0; r < 4; r++) o[q][x][r] *= keep;
        }
        const float mc = m[q] == -INFINITY ? 0.0f : m[q] * c;
        float p[8], sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          p[e] = exp2_(__builtin_fmaf(s[e / 4][q][e % 4], c, -mc));
          sum += p[e];
        }
        l[q] += sum;
        split8<PT, false>(p, pf[q]);
      }
      if (careful) {
        bf16x8 ones[NQ];
#pragma unroll
        for (int q = 0; q < NQ; q++)
#pragma unroll
          for (int e = 0; e < 8; e++) ones[q][e] = s[e / 4][q][e % 4] == -INFINITY ? (__bf16)0.0f : (__bf16)1.0f;
#pragma unroll
        for (int x = 0; x < 2 * W; x++) {
          const bool half = Lane<W>::vblocks > 1 && (W * li + x / 2) / 16 != W * li / 16;
          bf16x8 nan;
#pragma unroll
          for (int e = 0; e < 8; e++)
            nan[e] = (half ? vt.s[e][Lane<W>::vblocks - 1] : vt.s[e][0]) > 252 ? (__bf16)1.0f : (__bf16)0.0f;
#pragma unroll
          for (int q = 0; q < NQ; q++) {
            const f32x4 hit = mfma16(nan, ones[q], f32x4{0, 0, 0, 0});
#pragma unroll
            for (int r = 0; r < 4; r++)
              if (hit[r] != 0.0f) o[q][x][r] = NAN;
          }
        }
#pragma unroll
        for (int e = 0; e < 8; e++)
#pragma unroll
          for (int i = 0; i < Lane<W>::vblocks; i++)
            if (vt.s[e][i] > 252) vt.s[e][i] = 0;
      }
      // values
      float vsc[8][Lane<W>::vblocks];
#pragma unroll
      for (int e = 0; e < 8; e++)
#pragma unroll
        for (int i = 0; i < Lane<W>::vblocks; i++)
          vsc[e][i] = scale_of_byte(vt.s[e][i]);
      if constexpr (Lane<W>::odd) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          if constexpr (W == 3) {
            vt.w[e][0] >>= place.shift;
          } else {
            const unsigned long long v = ((unsigned long long)vt.w[e][1] << 32 | vt.w[e][0]) >> place.shift;
            vt.w[e][0] = (unsigned)v;
            vt.w[e][1] = (unsigned)(v >> 32);
          }
        }
      }
#pragma unroll
      for (int y = 0; y < W; y++) {
        unsigned pr[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const bool half = Lane<W>::vblocks > 1 && (W * li + y) / 16 != W * li / 16;
          const float sc = half ? vsc[e][Lane<W>::vblocks - 1] : vsc[e][0];
          const unsigned w = vt.w[e][y / 4];
          pr[e] = y % 4 == 0 ? fp4_pair<0>(w, sc) : y % 4 == 1 ? fp4_pair<1>(w, sc)
                : y % 4 == 2 ? fp4_pair<2>(w, sc) : fp4_pair<3>(w, sc);
        }
        u32x4 lo4, hi4;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          lo4[e] = __builtin_amdgcn_perm(pr[2 * e + 1], pr[2 * e], 0x05040100u);
          hi4[e] = __builtin_amdgcn_perm(pr[2 * e + 1], pr[2 * e], 0x07060302u);
        }
#pragma unroll
        for (int q = 0; q < NQ; q++)
#pragma unroll
          for (int t = PT - 1; t >= 0; t--) {
            o[q][2 * y] = mfma16(__builtin_bit_cast(bf16x8, lo4), pf[q][t], o[q][2 * y]);
            o[q][2 * y + 1] = mfma16(__builtin_bit_cast(bf16x8, hi4), pf[q][t], o[q][2 * y + 1]);
          }
      }
    };

    // Tiles of 32 keys, the next one's loads in flight while one is computed (with
    // more rows a wave the values' come late, behind the keys' products: their
    // registers are needed, and there is enough to compute until then).
    // Keys are walked a second time, for what would cost the first one more in
    // every tile.  A value block of NaN must not reach the rows that do not see
    // its key, but 0 * NaN does: where the result holds a NaN, such blocks are
    // zeros the second time, and the rows that see them get their NaN from a
    // product of ones.  (So do scale bytes 253 and 254, whose numbers overflow;
    // the format has none.)  And a row whose maximum ends past kFar has it taken
    // off its scores; one whose maximum was so far past it on the way that a sum
    // overflowed (the rescaling has made that a NaN) starts with its last maximum.
    const int step = WS == 4 ? 128 : 32;
#pragma unroll
    for (int q = 0; q < NQ; q++) {
      m[q] = -INFINITY;
      shift[q] = 0.0f;
    }
    while (true) {
#pragma unroll
      for (int q = 0; q < NQ; q++) {
        l[q] = 0.0f;
#pragma unroll
        for (int x = 0; x < 2 * W; x++) o[q][x] = f32x4{0, 0, 0, 0};
      }
      int j0 = klo + (WS == 4 ? 32 * wave : 0);
      if (j0 < khi) {
        constexpr bool late = NQ > 1;
        KeyTile<W> ka, kb;
        ValueTile<W> va, vb;
        Pages pa = find_pages(a, page_ids(a, table, j0, khi), j0, h), pb;
        load_keys<W>(a, pa, place, ka);
        if (!late) load_values<W>(a, pa, place, va);
        PageIds ids = page_ids(a, table, j0 + step, khi);
        while (true) {
          if (late) load_values<W>(a, pa, place, va);
          pb = find_pages(a, ids, j0 + step, h);
          load_keys<W>(a, pb, place, kb);
          if (!late) load_values<W>(a, pb, place, vb);
          ids = page_ids(a, table, j0 + 2 * step, khi);
          __builtin_amdgcn_sched_barrier(0);
          compute(ka, va, pa, j0);
          j0 += step;
          if (j0 >= khi) break;
          if (late) load_values<W>(a, pb, place, va);
          pa = find_pages(a, ids, j0 + step, h);
          load_keys<W>(a, pa, place, ka);
          if (!late) load_values<W>(a, pa, place, va);
          ids = page_ids(a, table, j0 + 2 * step, khi);
          __builtin_amdgcn_sched_barrier(0);
          compute(kb, late ? va : vb, pb, j0);
          j0 += step;
          if (j0 >= khi) break;
        }
      }
      if (careful) break;
#pragma unroll
      for (int q = 0; q < NQ; q++) {
        careful |= m[q] != -INFINITY && is_far(m[q] * c);
#pragma unroll
        for (int x = 0; x < 2 * W; x++)
#pragma unroll
          for (int r = 0; r < 4; r++) careful |= o[q][x][r] != o[q][x][r];
      }
      careful = __any(careful);
      if (!careful) break;
      all_lo = INT32_MAX;        // the masks' part of every tile takes the maximum off
#pragma unroll
      for (int q = 0; q < NQ; q++) {
        const float sum = column_sum(l[q]);
        const bool far = m[q] != -INFINITY && is_far(m[q] * c);
        shift[q] = far ? m[q] : 0.0f;
        m[q] = far ? 0.0f : sum != sum ? m[q] : -INFINITY;
      }
    }
#pragma unroll
    for (int q = 0; q < NQ; q++) m[q] += shift[q];

    // the sums of a row: over the lanes of its column, then (WS = 4) over the
    // workgroup's waves, in their order
#pragma unroll
    for (int q = 0; q < NQ; q++) l[q] = column_sum(l[q]);
    if constexpr (WS == 4) {
      float* ml = lds;                          // [4][NQ * 16][2]
      float* ol = lds + 4 * NQ * 32;            // [4 waves][NQ * 2W * 4][64]
      __syncthreads();                          // (an earlier tile's reads)
      if (kg == 0) {
#pragma unroll
        for (int q = 0; q < NQ; q++) {
          ml[((wave * NQ + q) * 16 + li) * 2] = m[q];
          ml[((wave * NQ + q) * 16 + li) * 2 + 1] = l[q];
        }
      }
#pragma unroll
      for (int q = 0; q < NQ; q++)
#pragma unroll
        for (int x = 0; x < 2 * W; x++)
#pragma unroll
          for (int r = 0; r < 4; r++)
            ol[((wave * NQ + q) * 8 * W + r * 2 * W + x) * 64 + lane] = o[q][x][r];
      __syncthreads();
#pragma unroll
      for (int q = 0; q < NQ; q++) {
        float wm[4], top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++) {
          wm[w] = ml[((w * NQ + q) * 16 + li) * 2];
          top = fmaxf(top, wm[w]);
        }
#pragma unroll
        for (int w = 0; w < 4; w++) {
          wm[w] = top == -INFINITY ? 0.0f : exp2_(rescale(wm[w], top, c));
          sum += wm[w] * ml[((w * NQ + q) * 16 + li) * 2 + 1];
        }
        m[q] = top;
        l[q] = sum;
        // wave r takes the rows d = 2 W (4 kg + r) + x of every lane group
#pragma unroll
        for (int x = 0; x < 2 * W; x++) {
          float v = 0.0f;
#pragma unroll
          for (int w = 0; w < 4; w++)
            v += wm[w] * ol[((w * NQ + q) * 8 * W + wave * 2 * W + x) * 64 + lane];
          o[q][x][0] = v;
        }
      }
    }
    constexpr int NR = WS == 4 ? 1 : 4;
    // (out of the compiler's sight, which otherwise holds the stores' addresses through
    // the walk: one long cache in float16 41.4 us, 40.6 so)
    int kgs = kg;
    if constexpr (WS == 4) asm volatile("" : "+v"(kgs));
#pragma unroll
    for (int q = 0; q < NQ; q++) {
      if (!live[q]) continue;
      const int64_t at = tok[q] * (a.heads * a.group) + head[q];
      if (a.splits > 1) {
        const int64_t part = (int64_t)split * a.tokens * (a.heads * a.group) + at;
        if (kg == 0 && (WS == 1 || wave == 0)) {
          a.part_ml[2 * part] = m[q];
          a.part_ml[2 * part + 1] = l[q];
        }
        if (l[q] == 0.0f) continue;
#pragma unroll
        for (int r = 0; r < NR; r++) {
          float* p = a.part_o + part * DH + 2 * W * (4 * kgs + (WS == 4 ? wave : r));
#pragma unroll
          for (int x = 0; x < 2 * W; x++) p[x] = o[q][x][r];
        }
      } else {
        const float inv = l[q] == 0.0f ? 0.0f : 1.0f / l[q];
        if (a.lse && kg == 0 && (WS == 1 || wave == 0))
          a.lse[at] = l[q] == 0.0f ? -INFINITY : log_sum(m[q], l[q], fabsf(a.scale));
#pragma unroll
        for (int r = 0; r < NR; r++) {
          typename E::type* p = (typename E::type*)a.out + tok[q] * a.ot + head[q] * a.oh +
                                2 * W * (4 * kgs + (WS == 4 ? wave : r));
          typename E::type t[2 * W];
#pragma unroll
          for (int x = 0; x < 2 * W; x++) t[x] = (typename E::type)(o[q][x][r] * inv);
          __builtin_memcpy(p, t, sizeof t);
        }
      }
    }
  }
}

// Joins the splits of a row.  JW = 4: a workgroup a row, its waves take the
// splits in turn, sixteen loads in flight, and their sums are added in the
// waves' order (64 splits of 32 rows: 5 us, against 41 with a wave a row that
// walks them).  JW = 1, up to 8 splits: a wave a row (4 splits of 2048 rows:
// 7 us against 16).
template <typename E, int JW>
__global__ __launch_bounds__(256) void attn4_join_kernel(Attn4 a, int dh) {
  constexpr int U = JW == 4 ? 16 : 8;
  __shared__ float sum4[JW == 4 ? 4 : 1][256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int qheads = a.heads * a.group;
  const int64_t all = a.tokens * qheads;
  for (int64_t row = JW == 4 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave; row < all;
       row += (int64_t)gridDim.x * (JW == 4 ? 1 : 4)) {
    const int64_t t = row / qheads;
    if (a.starts && (t < a.starts[0] || t >= a.starts[a.batch])) continue;
    float m = -INFINITY, l = 0.0f;
    if (lane < a.splits) {
      m = a.part_ml[2 * (lane * all + row)];
      l = a.part_ml[2 * (lane * all + row) + 1];
    }
    float top = m;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
    const float w = top == -INFINITY ? 0.0f : exp2_(rescale(m, top, fabsf(a.scale) * kLog2e));
    float sum = w * l;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
    // splits without keys have stored nothing
    const unsigned long long some = __ballot(l != 0.0f);
    f32x4 v = {0, 0, 0, 0};
    const float* p = a.part_o + row * dh + 4 * lane;
    for (int s0 = JW == 4 ? wave : 0; s0 < a.splits; s0 += U * JW) {
      f32x4 u[U];
#pragma unroll
      for (int i = 0; i < U; i++) {
        const int s = s0 + JW * i;
        u[i] = f32x4{0, 0, 0, 0};
        if (s < a.splits && (some >> s & 1) && 4 * lane < dh) u[i] = *(const f32x4*)(p + s * all * dh);
      }
#pragma unroll
      for (int i = 0; i < U; i++) {
        const float ws = __shfl(w, min(s0 + JW * i, 63));
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] += ws * u[i][e];
      }
    }
    if (a.lse && lane == 0 && (JW == 1 || wave == 0))
      a.lse[row] = some ? log_sum(top, sum, fabsf(a.scale)) : -INFINITY;
    const float inv = some ? 1.0f / sum : 0.0f;
    typename E::type* out = (typename E::type*)a.out + t * a.ot + (row % qheads) * a.oh;
    if constexpr (JW == 4) {
      *(f32x4*)&sum4[wave][4 * lane] = v;
      __syncthreads();
      const int d = threadIdx.x;
      if (d < dh)
        out[d] = (typename E::type)((((sum4[0][d] + sum4[1][d]) + sum4[2][d]) + sum4[3][d]) * inv);
      __syncthreads();
    } else if (4 * lane < dh) {
      typename E::type y[4];
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] = (typename E::type)(v[e] * inv);
      __builtin_memcpy(out + 4 * lane, y, sizeof y);
    }
  }
}

// ------------------------------------------------------------ host: the plan

struct Attn4Plan {
  int nq, ws;          // column tiles a wave; 4: the waves of a workgroup share their rows
  int row_tiles;       // workgroups along the rows of a sequence and head
  int splits;
  int64_t chunk;
  size_t workspace;
};

static Attn4Plan attn4_plan(const qph_cache4* c, const qph_attn4* p) {
  Attn4Plan r{};
  const int64_t rows = std::min<int64_t>((int64_t)p->max_new * (p->heads / c->heads), 1 << 30);
  const int64_t keys = p->window > 0
                           ? std::min<int64_t>(p->max_len, (int64_t)p->window + p->max_new + 31)
                           : p->max_len;
  const int64_t seqs = (int64_t)p->batch * c->heads;
  // Waves with 32 rows of their own where they fill the card and their registers
  // do (up to 128 elements a head, 64 in float32), waves of a workgroup that
  // share 16 rows and split the keys otherwise.  us with 32 rows and with 16,
  // bfloat16: a chunk of 1024 tokens, 32 / 8 heads of 128 over 4000 keys (512
  // waves) 138 and 147, of 512 tokens over 2000 (256 waves) 72 and 48, 16 of 64
  // tokens, 16 / 4 heads of 64 (512 waves of little work) 56 and 32.
  const bool many = (p->dtype != QPH_F32 ? c->dh <= 128 : c->dh <= 64) && rows >= 1024 &&
                    (rows + 63) / 64 * seqs >= 512;
  r.nq = many ? 2 : 1;
  r.ws = many ? 1 : 4;
  const int64_t tiles = (rows + 16 * r.nq - 1) / (16 * r.nq);
  // max_new is a bound for every sequence, and one long prompt among single tokens
  // leaves most of the workgroups that it would make empty: past a million in all
  // (some rounds of the card, whatever their work) they take further tiles in turn.
  r.row_tiles = (int)std::clamp<int64_t>(r.ws == 4 ? tiles : (tiles + 3) / 4, 1,
                                         std::max<int64_t>(1, ((int64_t)1 << 20) / seqs));
  r.splits = 1;
  r.chunk = (int64_t)1 << 40;
  const int64_t blocks = r.row_tiles * seqs;
  // Splits along the keys: up to six workgroups a CU, of 512 keys or more (of
  // 256 where that leaves CUs without one).  us with a bound of 1024, this one
  // and 2048 workgroups: 64 sequences of 0 to 16384 keys, 8 heads, 160, 138 and
  // 155; 128 of 1000 to 2000 keys 55, 57 and 65.  512 keys against 256: 64
  // sequences of 512 to 1024 keys 18 and 25 to 30; one of 2000 keys 12 and 11.
  const int64_t least = keys / 512 >= (255 + blocks) / blocks ? 512 : 256;
  if (r.ws == 4 && 2 * blocks <= 1536 && keys > 2 * least) {
    int64_t n = std::min<int64_t>({1536 / blocks, (keys + least - 1) / least, 64});
    r.chunk = ((keys + n - 1) / n + 127) / 128 * 128;
    n = (keys + r.chunk - 1) / r.chunk;
    if (n > 1) r.splits = (int)n;
    else r.chunk = (int64_t)1 << 40;
  }
  if (r.splits > 1) r.workspace = (size_t)r.splits * p->tokens * p->heads * (c->dh + 2) * 4;
  return r;
}

template <typename E, int W, int NQ, int WS>
static int launch_attn4_one(const Attn4& a, hipStream_t s) {
  const size_t lds = WS == 4 ? (size_t)4 * NQ * (32 + 2 * W * 4 * 64) * 4 : 0;
  if (lds > 65536) QPH_TRY(allow_full_lds((const void*)attn4_kernel<E, W, NQ, WS>));
  const int64_t blocks = (int64_t)a.row_tiles * a.splits * a.heads * a.batch;
  hipLaunchKernelGGL((attn4_kernel<E, W, NQ, WS>), dim3((unsigned)blocks), dim3(256), lds, s, a);
  return launch_check("attn4_kernel");
}

template <typename E, int W>
static int launch_attn4_w(const Attn4& a, const Attn4Plan& p, hipStream_t s) {
  if constexpr (W <= (E::terms == 3 ? 2 : 4)) {
    if (p.nq == 2) return launch_attn4_one<E, W, 2, 1>(a, s);
  }
  return launch_attn4_one<E, W, 1, 4>(a, s);
}

template <typename E>
static int launch_attn4(const Attn4& a, const Attn4Plan& p, int dh, hipStream_t s) {
  switch (dh) {
    case 32: QPH_TRY((launch_attn4_w<E, 1>(a, p, s))); break;
    case 64: QPH_TRY((launch_attn4_w<E, 2>(a, p, s))); break;
    case 96: QPH_TRY((launch_attn4_w<E, 3>(a, p, s))); break;
    case 128: QPH_TRY((launch_attn4_w<E, 4>(a, p, s))); break;
    case 192: QPH_TRY((launch_attn4_w<E, 6>(a, p, s))); break;
    default: QPH_TRY((launch_attn4_w<E, 8>(a, p, s))); break;
  }
  if (a.splits == 1) return QPH_OK;
  const int64_t rows = a.tokens * a.heads * a.group;
  const bool wide = a.splits > 8;
  const dim3 grid((unsigned)std::min<int64_t>(wide ? rows : (rows + 3) / 4, 1 << 20));
  if (wide) hipLaunchKernelGGL((attn4_join_kernel<E, 4>), grid, dim3(256), 0, s, a, dh);
  else hipLaunchKernelGGL((attn4_join_kernel<E, 1>), grid, dim3(256), 0, s, a, dh);
  return launch_check("attn4_join_kernel");
}

static int attn4_check(const qph_cache4* c, const qph_attn4* p, int* shift) {
  QPH_TRY(cache4_check(c, "attention_cache4", shift));
  if (!p) return fail(QPH_EINVAL, "attention_cache4: NULL arguments");
  if (!dtype_valid(p->dtype)) return fail(QPH_EINVAL, "attention_cache4: unknown element type");
  if (p->tokens < 0 || p->batch < 0 || p->max_new < 0 || p->max_len < 0 || p->max_pages < 0 ||
      p->window < 0)
    return fail(QPH_EINVAL, "attention_cache4: negative size");
  if (p->heads <= 0 || p->heads % c->heads)
    return fail(QPH_EINVAL, "attention_cache4: query heads are no multiple of the cache's heads");
  if (p->heads > 65536) return fail(QPH_EUNSUPPORTED, "attention_cache4: more than 65536 query heads");
  // (device code takes subnormal numbers as zeros, and uses scale log2 e)
  if (!std::isnormal(p->scale) || !std::isfinite(p->scale * kLog2e))
    return fail(QPH_EINVAL, "attention_cache4: scale is zero, subnormal or too large");
  if (p->batch > INT32_MAX / c->heads || p->max_pages > INT32_MAX)
    return fail(QPH_EUNSUPPORTED, "attention_cache4: more than 2^31 - 1 sequences' heads or pages");
  if (!p->starts && p->batch && p->tokens != p->batch * (int64_t)p->max_new)
    return fail(QPH_EINVAL, "attention_cache4: without starts, tokens must be batch * max_new");
  if (p->tokens > ((int64_t)1 << 31) || (int64_t)p->tokens * p->heads > ((int64_t)1 << 33))
    return fail(QPH_EUNSUPPORTED, "attention_cache4: too many rows for one call");
  return QPH_OK;
}

}  // namespace qph

using namespace qph;

extern "C" {

QPH_API int qph_attention_cache4_workspace(const qph_cache4* cache, const qph_attn4* args,
                                           size_t* bytes) {
  if (!bytes) return fail(QPH_EINVAL, "attention_cache4_workspace: NULL argument");
  *bytes = 0;
  int shift = 0;
  QPH_TRY(attn4_check(cache, args, &shift));
  if (args->tokens == 0 || args->batch == 0) return QPH_OK;
  *bytes = attn4_plan(cache, args).workspace;
  return QPH_OK;
}

QPH_API int qph_attention_cache4(qph_ctx* ctx, const qph_cache4* cache, const qph_attn4* args) {
  int shift = 0;
  QPH_TRY(attn4_check(cache, args, &shift));
  const bool none = args->tokens == 0 || args->batch == 0;
  if (!none && (!args->q || !args->out || !args->lens || (!args->page_table && args->max_pages)))
    return fail(QPH_EINVAL, "attention_cache4: NULL argument");
  const Attn4Plan p = none ? Attn4Plan{} : attn4_plan(cache, args);
  if (p.workspace && (!args->workspace || args->workspace_bytes < p.workspace))
    return fail(QPH_EINVAL, "attention_cache4: workspace of " + std::to_string(args->workspace_bytes) +
                                " bytes, needs " + std::to_string(p.workspace));
  if ((uintptr_t)args->workspace % 16)
    return fail(QPH_EINVAL, "attention_cache4: workspace is not 16-byte aligned");
  if ((int64_t)p.row_tiles * p.splits * cache->heads * args->batch > kMaxGroups)
    return fail(QPH_EUNSUPPORTED, "attention_cache4: batch too large for one call");
  if (!ctx) return fail(QPH_EINVAL, "null context");
  if (none) return QPH_OK;
  Attn4 a{};
  a.kc = (const unsigned char*)cache->k_codes; a.ks = (const unsigned char*)cache->k_scales;
  a.vc = (const unsigned char*)cache->v_codes; a.vs = (const unsigned char*)cache->v_scales;
  a.n_pages = cache->n_pages;
  a.shift = shift;
  a.heads = cache->heads;
  a.group = args->heads / cache->heads;
  a.q = args->q; a.out = args->out; a.lse = args->lse;
  a.qt = args->q_strides[0]; a.qh = args->q_strides[1];
  a.ot = args->out_strides[0]; a.oh = args->out_strides[1];
  a.tokens = args->tokens;
  a.batch = (int)args->batch;
  a.table = args->page_table;
  a.table_stride = args->table_stride;
  a.max_pages = (int)args->max_pages;
  a.lens = args->lens;
  a.starts = args->starts;
  a.news = args->max_new;
  a.scale = args->scale;
  a.causal = args->causal != 0;
  a.window = args->window;
  a.row_tiles = p.row_tiles;
  a.splits = p.splits;
  a.chunk = p.chunk;
  if (p.splits > 1) {
    a.part_o = (float*)args->workspace;
    a.part_ml = a.part_o + (size_t)p.splits * args->tokens * args->heads * cache->dh;
  }
  OnDevice dev(ctx);
  QPH_TRY(dev.rc());
  if (args->dtype == QPH_F32) return launch_attn4<F32>(a, p, cache->dh, ctx->stream);
  if (args->dtype == QPH_F16) return launch_attn4<F16>(a, p, cache->dh, ctx->stream);
  return launch_attn4<BF16>(a, p, cache->dh, ctx->stream);
}

}  // extern "C"
