// What the kernels of attention over the 4-bit cache share (qph_attn4.hip,
// qph_mask4.hip): their arguments, a row's softmax in parts, a lane's loads of
// keys and values, the joining of splits.
#pragma once

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

// Joins the splits of a (device workspaces) into its outputs; nothing where there is one.
int attn4_join(const Attn4& a, int dtype, int dh, hipStream_t s);
// Checks the arguments of an attention but its pointers (host); sets *shift to log2 of
// the page size.
int attn4_check(const qph_cache4* c, const qph_attn4* p, const char* what, int* shift);
// The kernel's arguments of checked ones, but its grid and splits.
Attn4 attn4_args(const qph_cache4* cache, const qph_attn4* args, int shift);

}  // namespace qph
