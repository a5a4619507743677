// Attention over the 4-bit cache where a row sees more than a run of keys: a window
// and a sequence's first tokens beside it, or the context and the drafted tokens on
// its own path of a tree.
//
// For a new token and a query head, over the keys j that the row sees:
//   s_j = scale q . k_j,  m = max s_j,  o = sum exp(s_j - m) v_j / sum exp(s_j - m)
// with the operand layouts, the running maximum and the second walk of
// qph_attn4.hip.  Two forms:
//
// Few rows of a sequence and head: the waves of a workgroup share 16 NQ rows and take
// the tiles of 32 keys in turn, codes to registers to operands.  Bound by the codes' way
// from memory: one token of 32 sequences with 4100 of their keys (8 heads of 128) 143 MB in
// 36.7 us, 3.9 TB/s where a large copy runs at 4.6.
//
// Many (mask4_shared_kernel): each wave has 16 NQ rows of its own, so every tile is
// needed by all waves, and its codes are turned into operands once, by way of LDS.  Bound
// by what the SIMDs issue beside their products and by LDS: 1024 new tokens of two
// sequences with windows of 2000 (bfloat16, 32 heads of 128 over 8) 68 GF in 89 us, 770
// TFLOP/s where a large library product runs at 1134; a round of 64 keys takes about 5000
// cycles, of which the matrix unit has work for 2050, the vector instructions of two waves
// fill 2600 and the operands' reads of LDS 2300.
//
// Keys are walked as two runs of tiles: the first tokens, and what lies in the
// window of any row of the workgroup, up to the last key.  A tile inside every row's
// window and before every row's border needs no masks.
#pragma once

#include <type_traits>

#include "qph_attn4.h"

namespace qph {

struct Mask4 {
  Attn4 a;
  int sinks;                      // first tokens that stay visible (0 without a window)
  const unsigned* tree;           // [tokens][words], or NULL
  int words;                      // of 32 bits
};

// What a workgroup works on: a sequence's head, from a row tile on, and of its keys (the two
// runs counted as one) those from va to vb, which are split number `split` of them.
struct Part4 {
  int b, h, rt0, split;
  int64_t va, vb;
};

// The four bits of a tree's row from drafted token d on (none before the first and past the
// words).  Without branches, so that the loads of several go out together.
__device__ __forceinline__ unsigned path_bits(const unsigned* row, int words, int d) {
  const int e = max(d, 0), w = e >> 5;
  const unsigned lo = row[min(w, words - 1)], hi = row[min(w + 1, words - 1)];
  const unsigned long long both = (unsigned long long)(w + 1 < words ? hi : 0u) << 32 | (w < words ? lo : 0u);
  const unsigned v = (unsigned)(both >> (e & 31));
  return d >= 0 ? v : d > -4 ? v << -d : 0u;
}

// A workgroup's sequence and head, and its tiles of keys.
struct Walk4 {
  int64_t t0, rows, r0;
  int news, len, first;           // first: the first new token's position, the context's keys
  int h, split, rt0;
  bool tree;
  int window, causal, sinks;
  ScalarI32 table;
  int a0, a1, s32;                // this split of the first tokens
  int64_t bfrom, bto;             // and of the rest
  int ghi, glo, n1, b0, tiles;    // of a row tile: keys that some row sees
  int i0;                         // its first row's token,
  unsigned rem;                   // and query head of this cache head

  __device__ __forceinline__ Walk4(const Mask4& g, const Part4& part) {
    const Attn4& a = g.a;
    const int b = part.b;
    h = part.h; rt0 = part.rt0; split = part.split;
    // inside what the caller's buffers hold whatever the device arrays say
    int64_t t1;
    if (a.starts) {
      t0 = min(max((int64_t)a.starts[b], (int64_t)0), a.tokens);
      t1 = min(max((int64_t)a.starts[b + 1], t0), a.tokens);
    } else {
      t0 = (int64_t)b * a.news;
      t1 = t0 + a.news;
    }
    news = (int)(t1 - t0);
    const int room = (int)min((int64_t)a.max_pages << a.shift, kMaxKeys);
    len = min(max(a.lens[b], 0), room);
    rows = (int64_t)news * a.group;
    table = (ScalarI32)(a.table + b * a.table_stride);
    first = len - news;
    tree = g.tree != nullptr;
    window = a.window; causal = a.causal; sinks = g.sinks;
    // the two runs of the whole sequence, [0, s32) and from `base` on, counted as one
    // (a path's end stands at first - 1 at least, which is that of no tokens)
    s32 = (min(sinks, len) + 31) & ~31;
    const int base = window > 0 ? max(s32, window_from((int64_t)first - tree) & ~31) : 0;
    const int64_t va = part.va, vb = part.vb;
    a0 = (int)min(va, (int64_t)s32); a1 = (int)min(vb, (int64_t)s32);
    bfrom = base + max(va - s32, (int64_t)0); bto = base + max(vb - s32, (int64_t)0);
  }

  // The first key inside the window of a token at position p.
  __device__ __forceinline__ int window_from(int64_t p) const {
    return window > 0 ? (int)max((int64_t)0, p - window + 1) : 0;
  }

  // The key behind the last that a token at position p sees (a tree's: of the context).
  __device__ __forceinline__ int border(int64_t p) const {
    return tree ? max(first, 0) : causal ? (int)min((int64_t)len, max(p + 1, (int64_t)0)) : len;
  }

  // The token of row r0 + d (a row tile has few rows and group is 65536 at most).
  __device__ __forceinline__ int token(unsigned d, unsigned group) const { return i0 + (int)((rem + d) / group); }

  // The tiles of rows r0 to r1.
  __device__ __forceinline__ void tiles_of(int64_t from, int64_t r1, unsigned group) {
    r0 = from;
    i0 = (int)(from / group);
    rem = (unsigned)(from - (int64_t)i0 * group);
    ghi = tree ? len : border((int64_t)first + token((unsigned)(r1 - r0), group));
    glo = window_from(tree ? (int64_t)first - 1 : (int64_t)first + i0);
    n1 = (max(min(a1, ghi) - a0, 0) + 31) >> 5;
    b0 = (int)max(bfrom, (int64_t)(glo & ~31));
    const int n2 = bfrom >= ghi ? 0 : (max((int)min(bto, (int64_t)ghi) - b0, 0) + 31) >> 5;
    tiles = n1 + n2;
  }

  __device__ __forceinline__ int key_of(int t) const { return t < n1 ? a0 + 32 * t : b0 + 32 * (t - n1); }
};

// The part of a workgroup where all splits have as many keys.  Neighbouring workgroups go to
// the card's eight dies in turn: heads are next to each other, so that the row tiles of one
// find its keys in their die's cache, and splits come last, so that those without keys (of
// shorter sequences) are no die's more than another's (32 ragged sequences of 8 heads, 8
// splits: 454 us with splits next to each other, 154 so).
__device__ __forceinline__ Part4 part_of_block(const Attn4& a) {
  Part4 p;
  unsigned id = blockIdx.x;
  p.h = id % a.heads; id /= a.heads;
  p.b = id % a.batch; id /= a.batch;
  p.rt0 = id % a.row_tiles;
  p.split = id / a.row_tiles;
  p.va = p.split * a.chunk;
  p.vb = p.split == a.splits - 1 ? INT64_MAX / 2 : p.va + a.chunk;
  return p;
}

// In pairs of tiles: the least share, and what a part costs beside its own (its queries, the
// first loads, its sums; 32 ragged sequences of 8 heads: 207 us counted as nothing, 151 as
// 3, 135 as 6, 136 as 10).
constexpr int64_t kLeastShare = 4;
constexpr unsigned kPartCost = 6;


// The next part of a workgroup's even share: of the pairs of tiles of all sequences and heads,
// kPartCost places ahead of each and one after the other, those from `at` (-1: none yet) to
// `end`.  Each lane counts a sequence's (at most 64); one whose rows see no keys has a pair all
// the same, so that they are stored.  `parts` is the number of splits that the keys of the
// part's sequence and head have in all.  False: none is left.
__device__ __forceinline__ bool next_part(const Mask4& g, int64_t& at, int64_t& end, Part4& part, int& parts) {
  const Attn4& a = g.a;
  const int lane = threadIdx.x & 63;
  unsigned mine = 0;
  if (lane < a.batch) {
    const Walk4 w(g, Part4{lane, 0, 0, 0, 0, INT64_MAX / 2});
    const int hi = w.tree ? w.len : w.border((int64_t)w.first + w.news - 1);
    const int64_t tiles = w.s32 / 32 + ((max((int64_t)hi - w.bfrom, (int64_t)0) + 31) >> 5);
    mine = w.news ? max((unsigned)((tiles + 1) >> 1), 1u) + kPartCost : 0u;
  }
  unsigned upto = mine, most = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const unsigned before = __shfl_up(upto, d);
    upto += lane >= d ? before : 0u;
    most = max(most, (unsigned)__shfl_xor(most, d));
  }
  const unsigned n = a.heads;
  const int64_t all = (int64_t)(unsigned)__builtin_amdgcn_readlane(upto, 63) * n;
  most = __builtin_amdgcn_readfirstlane(most);
  const int64_t share = max(max((all + gridDim.x - 1) / gridDim.x, (int64_t)(most + a.splits - 2) / (a.splits - 1)),
                            kLeastShare);
  if (at < 0) {
    at = blockIdx.x * share;
    end = min(at + share, all);
  }
  if (at >= end) return false;
  const int64_t from = (int64_t)(upto - mine) * n;
  part.b = __builtin_ctzll(__ballot(from <= at && at < (int64_t)upto * n));
  unsigned len = __builtin_amdgcn_readlane(mine, part.b);
  const int64_t first = (int64_t)__builtin_amdgcn_readlane(upto - mine, part.b) * n;
  part.h = (int)((at - first) / len);
  part.rt0 = 0;
  const int64_t head = first + (int64_t)part.h * len + kPartCost;
  len -= kPartCost;
  at = max(at, head);
  if (at >= end) return false;
  const int64_t x0 = at - head, x1 = min((int64_t)len, x0 + (end - at));
  const int64_t before = head / share;
  part.split = (int)(blockIdx.x - before);
  parts = (int)((head + len - 1) / share - before) + 1;
  part.va = 64 * x0;
  part.vb = x1 == len ? INT64_MAX / 2 : 64 * x1;
  at += x1 - x0;
  return true;
}

// (for scalar registers: the compiler does not see that all lanes have the same)
__device__ __forceinline__ int64_t same_in_all(int64_t v) {
  return (int64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)v) |
         (int64_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32;
}

struct EvenState {
  int64_t at, end;
  Part4 part;
};

// Says of the splits from `parts` on that a sequence's rows have no keys in them.
__device__ __forceinline__ void unused_splits(const Mask4& g, const Part4& part, int parts) {
  const Attn4& a = g.a;
  const Walk4 w(g, part);
  const int qheads = a.heads * a.group;
  for (int s = parts; s < a.splits; s++)
    for (int64_t r = threadIdx.x; r < w.rows; r += blockDim.x) {
      const int64_t t = r / a.group;
      float* ml = a.part_ml + 2 * (s * a.tokens * qheads + (w.t0 + t) * qheads + part.h * a.group + (r - t * a.group));
      ml[0] = -INFINITY;
      ml[1] = 0.0f;
    }
}

// The rows of a wave, 16 to a column tile, and what each sees.
template <int NQ>
struct Rows4 {
  int tok[NQ], head[NQ];          // tok: from the sequence's first
  int lo[NQ], hi[NQ];             // of the context
  bool live[NQ];
  int all_lo, all_hi;             // tiles between need no masks

  // Rows from w.r0 + d0 on.
  __device__ __forceinline__ Rows4(const Mask4& g, const Walk4& w, unsigned d0, int li) {
    const Attn4& a = g.a;
    const unsigned group = (unsigned)a.group, left = (unsigned)min(w.rows - w.r0, (int64_t)1 << 30);
#pragma unroll
    for (int q = 0; q < NQ; q++) {
      const unsigned d = d0 + 16 * q + li;
      live[q] = d < left;
      const unsigned dd = live[q] ? d : left - 1;
      const int i = w.token(dd, group);
      head[q] = w.h * a.group + (int)((w.rem + dd) % group);
      tok[q] = i;
      int64_t pos = (int64_t)w.first + i;
      if (w.tree && w.window > 0) {
        // a path's end stands as many places behind the context as it has tokens
        const unsigned* path = g.tree + (w.t0 + i) * g.words;
        int depth = 0;
#pragma unroll 4
        for (int x = 0; x < g.words && 32 * x < w.news; x++) {
          const int left = w.news - 32 * x;
          depth += __popc(left < 32 ? path[x] & ((1u << left) - 1) : path[x]);
        }
        pos = (int64_t)w.first + depth - 1;
      }
      hi[q] = live[q] ? w.border(pos) : 0;
      lo[q] = w.window_from(pos);
    }
    const unsigned d1 = min(left, d0 + 16 * NQ) - 1;
    all_lo = w.window_from((int64_t)w.first + (w.tree ? w.news - 1 : w.token(d1, group)));
    all_hi = min(w.ghi, w.border((int64_t)w.first + w.token(min(d0, left - 1), group)));
  }

  __device__ __forceinline__ bool sees_all(const Walk4& w, int j0) const {
    return (j0 >= all_lo || j0 + 32 <= w.sinks) && j0 + 32 <= all_hi;
  }

  // Scores of the keys from j0 on, less `shift`, or -infinity where a row sees none.
  __device__ __forceinline__ void mask(const Mask4& g, const Walk4& w, int j0, int kg, bool there0,
                                       bool there1, const float (&shift)[NQ], f32x4 (&s)[2][NQ]) const {
    unsigned bits[NQ][2];
#pragma unroll
    for (int q = 0; q < NQ; q++) bits[q][0] = bits[q][1] = 0;
    if (w.tree && j0 + 32 > w.first) {
#pragma unroll
      for (int q = 0; q < NQ; q++)
#pragma unroll
        for (int u = 0; u < 2; u++)
          bits[q][u] = path_bits(g.tree + (w.t0 + tok[q]) * g.words, g.words, j0 + 16 * u + 4 * kg - w.first);
    }
#pragma unroll
    for (int q = 0; q < NQ; q++)
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int j = j0 + 16 * u + 4 * kg + r;
          const bool near = (j < hi[q]) & ((j >= lo[q]) | (j < w.sinks));
          const bool see = (u ? there1 : there0) & (j < w.len) & (near | (live[q] & (bits[q][u] >> r & 1)));
          s[u][q][r] = see ? s[u][q][r] - shift[q] : -INFINITY;
        }
  }
};

// Queries of the wave's rows as bfloat16 terms.
template <typename E, int W, int NQ>
__device__ __forceinline__ void load_queries(const Attn4& a, const Walk4& w, const Rows4<NQ>& rows, int kg,
                                             bf16x8 (&qf)[NQ][E::terms][W]) {
  const float sign = a.scale < 0.0f ? -1.0f : 1.0f;
#pragma unroll
  for (int q = 0; q < NQ; q++) {
    const typename E::type* p = (const typename E::type*)a.q + (w.t0 + rows.tok[q]) * a.qt + rows.head[q] * a.qh;
#pragma unroll
    for (int n = 0; n < W; n++) {
      float v[8];
      bf16x8 f[E::terms];
      load8<E>(p + 8 * (W * kg + n), v);
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] *= sign;
      split8<E::terms>(v, f);
#pragma unroll
      for (int t = 0; t < E::terms; t++) qf[q][t][n] = f[t];
    }
  }
}

// A lane's operand out of the keys' codes that it has loaded.
template <int W>
__device__ __forceinline__ bf16x8 key_operand(const KeyTile<W>& kt, int kg, int u, int n) {
  const float s0 = scale_of_byte(kt.s[u][0]);
  const float s1 = Lane<W>::kblocks > 1 ? scale_of_byte(kt.s[u][Lane<W>::kblocks - 1]) : s0;
  return fp4_word(kt.w[u][n], (W * kg + n) / 4 == W * kg / 4 ? s0 : s1);
}

// The values of keys that no row of the workgroup sees, whatever stands there, are zeros.
template <int W>
__device__ __forceinline__ void clear_unseen(const Walk4& w, ValueTile<W>& vt, bool there0, bool there1, int j0,
                                             int kg) {
  if (j0 >= w.glo && j0 + 32 <= w.ghi && there0 && there1) return;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const int j = j0 + 16 * (e / 4) + 4 * kg + e % 4;
    if (!(e / 4 ? there1 : there0) || j >= w.ghi || (j < w.glo && j >= w.sinks)) {
#pragma unroll
      for (int i = 0; i < Lane<W>::vblocks; i++) vt.s[e][i] = 127;
#pragma unroll
      for (int i = 0; i < Lane<W>::vwords; i++) vt.w[e][i] = 0;
    }
  }
}

// take(x, words): operand x of the values' product, in bfloat16 or (H) float16.
template <int W, bool H, typename F>
__device__ __forceinline__ void value_operands(ValueTile<W>& vt, const Place<W>& place, int li, F&& take) {
  float vsc[8][Lane<W>::vblocks];
#pragma unroll
  for (int e = 0; e < 8; e++)
#pragma unroll
    for (int i = 0; i < Lane<W>::vblocks; i++) vsc[e][i] = scale_of_byte(vt.s[e][i]);
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
      if constexpr (H)
        pr[e] = y % 4 == 0 ? fp4_pair_f16<0>(w, sc) : y % 4 == 1 ? fp4_pair_f16<1>(w, sc)
              : y % 4 == 2 ? fp4_pair_f16<2>(w, sc) : fp4_pair_f16<3>(w, sc);
      else
        pr[e] = y % 4 == 0 ? fp4_pair<0>(w, sc) : y % 4 == 1 ? fp4_pair<1>(w, sc)
              : y % 4 == 2 ? fp4_pair<2>(w, sc) : fp4_pair<3>(w, sc);
    }
    u32x4 lo4, hi4;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      lo4[e] = __builtin_amdgcn_perm(pr[2 * e + 1], pr[2 * e], 0x05040100u);
      hi4[e] = __builtin_amdgcn_perm(pr[2 * e + 1], pr[2 * e], 0x07060302u);
    }
    take(2 * y, lo4);
    take(2 * y + 1, hi4);
  }
}

// A wave's sums: for each row the largest score or its bound, the sum of the terms
// (of this lane's keys) and the sums of the values.
template <int W, int NQ>
struct Sums4 {
  f32x4 o[NQ][2 * W];
  float m[NQ], l[NQ];
  float c, lazy;                  // |scale| log2 e; the bound's distance as a score

  __device__ __forceinline__ explicit Sums4(const Attn4& a) {
    c = fabsf(a.scale) * kLog2e;
    lazy = fminf(kLazy / c, FLT_MAX);         // (it vanishes beside a far one)
#pragma unroll
    for (int q = 0; q < NQ; q++) m[q] = -INFINITY;
    clear();
  }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int q = 0; q < NQ; q++) {
      l[q] = 0.0f;
#pragma unroll
      for (int x = 0; x < 2 * W; x++) o[q][x] = f32x4{0, 0, 0, 0};
    }
  }

  // Takes column tile q's scores into its maximum.
  __device__ __forceinline__ void raise(int q, const f32x4 (&s)[2][NQ]) {
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
    if (__any(grows)) raise_to(q, NQ > 1 ? column_max(mx) : top);
  }

  // The same with the column's largest score at hand.
  __device__ __forceinline__ void raise_to(int q, float most) {
    float top = m[q];
    if constexpr (NQ > 1) {
      if (most > top) top = fminf(most + lazy, fmaxf(most, FLT_MAX));
    } else {
      top = fmaxf(top, most);
    }
    const float keep = exp2_(m[q] * c - (top == -INFINITY ? 0.0f : top * c));
    m[q] = top;
    l[q] *= keep;
#pragma unroll
    for (int x = 0; x < 2 * W; x++)
#pragma unroll
      for (int r = 0; r < 4; r++) o[q][x][r] *= keep;
  }

  __device__ __forceinline__ float offset(int q) const { return m[q] == -INFINITY ? 0.0f : m[q] * c; }

  // Whether the keys have to be walked a second time.
  __device__ __forceinline__ bool unsure() const {
    bool again = false;
#pragma unroll
    for (int q = 0; q < NQ; q++) {
      again |= m[q] != -INFINITY && is_far(m[q] * c);
#pragma unroll
      for (int x = 0; x < 2 * W; x++)
#pragma unroll
        for (int r = 0; r < 4; r++) again |= o[q][x][r] != o[q][x][r];
    }
    return __any(again);
  }
};

// One tile from a wave's own registers, in bfloat16 terms.  `careful`: the second walk,
// which keys are walked for what would cost the first one more in every tile (the
// reasons stand at attn4_kernel's): blocks of NaN in the values are zeros, and the rows
// that see them get their NaN from a product of ones; a row whose maximum ended past
// kFar has it taken off its scores (shift), one whose sum overflowed on the way starts
// with its last maximum.
template <typename E, int W, int NQ, bool careful>
__device__ __forceinline__ void own_tile(const Mask4& g, const Walk4& w, const Rows4<NQ>& rows,
                                         const bf16x8 (&qf)[NQ][E::terms][W], const KeyTile<W>& kt,
                                         ValueTile<W>& vt, const Pages& pg, int j0, int li, int kg,
                                         const Place<W>& place, const float (&shift)[NQ], Sums4<W, NQ>& sums) {
  // (terms of the probabilities: as in attn4_kernel)
  constexpr int T = E::terms, PT = T < 2 ? 2 : T;
  f32x4 s[2][NQ];
  bf16x8 pf[NQ][PT];
#pragma unroll
  for (int u = 0; u < 2; u++) {
#pragma unroll
    for (int q = 0; q < NQ; q++) s[u][q] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int n = 0; n < W; n++) {
      const bf16x8 kf = key_operand<W>(kt, kg, u, n);
#pragma unroll
      for (int q = 0; q < NQ; q++)
#pragma unroll
        for (int t = T - 1; t >= 0; t--) s[u][q] = mfma16(kf, qf[q][t][n], s[u][q]);
    }
  }
  if (careful || !(rows.sees_all(w, j0) && pg.there[0] && pg.there[1]))
    rows.mask(g, w, j0, kg, pg.there[0], pg.there[1], shift, s);
#pragma unroll
  for (int q = 0; q < NQ; q++) {
    sums.raise(q, s);
    const float mc = sums.offset(q);
    float p[8], sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      p[e] = exp2_(__builtin_fmaf(s[e / 4][q][e % 4], sums.c, -mc));
      sum += p[e];
    }
    sums.l[q] += sum;
    split8<PT, false>(p, pf[q]);
  }
  clear_unseen<W>(w, vt, pg.there[0], pg.there[1], j0, kg);
  if constexpr (careful) {
    bf16x8 ones[NQ];
#pragma unroll
    for (int q = 0; q < NQ; q++)
#pragma unroll
      for (int e = 0; e < 8; e++)
        ones[q][e] = s[e / 4][q][e % 4] == -INFINITY ? (__bf16)0.0f : (__bf16)1.0f;
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
          if (hit[r] != 0.0f) sums.o[q][x][r] = NAN;
      }
    }
#pragma unroll
    for (int e = 0; e < 8; e++)
#pragma unroll
      for (int i = 0; i < Lane<W>::vblocks; i++)
        if (vt.s[e][i] > 252) vt.s[e][i] = 0;
  }
  value_operands<W, false>(vt, place, li, [&](int x, u32x4 v) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < NQ; q++)
#pragma unroll
      for (int t = PT - 1; t >= 0; t--)
        sums.o[q][x] = mfma16(__builtin_bit_cast(bf16x8, v), pf[q][t], sums.o[q][x]);
  });
}

// The second walk of tiles t0, t0 + step, ...; the maxima it starts with (and what it
// took off) in sums.m and shift.
template <typename E, int W, int NQ>
__device__ __forceinline__ void walk_again(const Mask4& g, const Walk4& w, const Rows4<NQ>& rows,
                                           const bf16x8 (&qf)[NQ][E::terms][W], int t0, int step, int li, int kg,
                                           const Place<W>& place, float (&shift)[NQ], Sums4<W, NQ>& sums) {
#pragma unroll
  for (int q = 0; q < NQ; q++) {
    const float sum = column_sum(sums.l[q]);
    const bool far = sums.m[q] != -INFINITY && is_far(sums.m[q] * sums.c);
    shift[q] = far ? sums.m[q] : 0.0f;
    sums.m[q] = far ? 0.0f : sum != sum ? sums.m[q] : -INFINITY;
  }
  sums.clear();
  for (int t = t0; t < w.tiles; t += step) {
    KeyTile<W> kt;
    ValueTile<W> vt;
    const int j = w.key_of(t);
    const Pages pg = find_pages(g.a, page_ids(g.a, w.table, j, w.ghi), j, w.h);
    load_keys<W>(g.a, pg, place, kt);
    load_values<W>(g.a, pg, place, vt);
    own_tile<E, W, NQ, true>(g, w, rows, qf, kt, vt, pg, j, li, kg, place, shift, sums);
  }
}

// A row's results, or its part of them: the lane has the elements 2 W (4 kg + r) + x, of
// o[x][r] where NR is 4, of o[x][0] and r = wave where it is 1.
template <typename E, int W, int NQ, int NR>
__device__ __forceinline__ void store_rows(const Attn4& a, const Walk4& w, const Rows4<NQ>& rows, int kg, int wave,
                                           const float (&m)[NQ], const float (&l)[NQ], const f32x4 (&o)[NQ][2 * W]) {
#pragma unroll
  for (int q = 0; q < NQ; q++) {
    if (!rows.live[q]) continue;
    const int64_t tok = w.t0 + rows.tok[q];
    const int64_t at = tok * (a.heads * a.group) + rows.head[q];
    if (a.splits > 1) {
      const int64_t part = (int64_t)w.split * a.tokens * (a.heads * a.group) + at;
      if (kg == 0 && (NR == 4 || wave == 0)) {
        a.part_ml[2 * part] = m[q];
        a.part_ml[2 * part + 1] = l[q];
      }
      if (l[q] == 0.0f) continue;
#pragma unroll
      for (int r = 0; r < NR; r++) {
        float* p = a.part_o + part * (32 * W) + 2 * W * (4 * kg + (NR == 4 ? r : wave));
#pragma unroll
        for (int x = 0; x < 2 * W; x++) p[x] = o[q][x][r];
      }
    } else {
      // (a row has seen a key if and only if its sum is not 0: the largest score's
      // term is 1 or near it, and NaN is not 0 either)
      const float inv = l[q] == 0.0f ? 0.0f : 1.0f / l[q];
      if (a.lse && kg == 0 && (NR == 4 || wave == 0))
        a.lse[at] = l[q] == 0.0f ? -INFINITY : log_sum(m[q], l[q], fabsf(a.scale));
#pragma unroll
      for (int r = 0; r < NR; r++) {
        typename E::type* p = (typename E::type*)a.out + tok * a.ot + rows.head[q] * a.oh +
                              2 * W * (4 * kg + (NR == 4 ? r : wave));
        typename E::type t[2 * W];
#pragma unroll
        for (int x = 0; x < 2 * W; x++) t[x] = (typename E::type)(o[q][x][r] * inv);
        __builtin_memcpy(p, t, sizeof t);
      }
    }
  }
}

// ------------------------------------------------------------- few rows

// Waves of a workgroup: four, and up to twelve where registers leave room for three a SIMD
// (a longer row of waves in place of workgroups that split the keys saves their join).
template <int NQ>
constexpr int mask4_few_waves(int terms, int w) { return NQ == 1 && w <= 4 && terms < 3 ? 12 : 4; }

// Waves a SIMD that the compiler keeps registers free for.  Two where it would take a few
// past half of them by itself (bfloat16, heads of 128, 32 rows: 68 us, 88 without; of 192, 16
// rows: 78 and 94); with more terms of such heads it would keep values in memory (float16 of
// 256: 173 and 107, float32 of 192: 168 and 115).
template <int NQ>
constexpr int mask4_few_simd(int terms, int w) {
  return mask4_few_waves<NQ>(terms, w) > 4 ? 3 : (terms < 3 && NQ == 2 && w == 4) || (terms == 1 && w >= 6) ? 2 : 1;
}

template <typename E, int W, int NQ>
__global__ __launch_bounds__(64 * mask4_few_waves<NQ>(E::terms, W), mask4_few_simd<NQ>(E::terms, W)) void
mask4_few_kernel(Mask4 g) {
  const Attn4& a = g.a;
  constexpr int R = 16 * NQ;
  extern __shared__ u32x4 lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, kg = lane >> 4;
  const int waves = mask4_few_waves<NQ>(E::terms, W) > 4 ? blockDim.x >> 6 : 4;
  Walk4 w(g, part_of_block(a));
  const Place<W> place(li, kg);
  for (int64_t tile = w.rt0; tile * R < w.rows; tile += a.row_tiles) {
    w.tiles_of(tile * R, min(w.rows, tile * R + R) - 1, a.group);
    const Rows4<NQ> rows(g, w, 0, li);
    bf16x8 qf[NQ][E::terms][W];
    load_queries<E, W, NQ>(a, w, rows, kg, qf);
    Sums4<W, NQ> sums(a);
    float shift[NQ];
#pragma unroll
    for (int q = 0; q < NQ; q++) shift[q] = 0.0f;

    // This wave's tiles t, t + waves, ...; the next one's loads in flight while one is computed
    // (with more rows a wave the values' come late, behind the keys' products).
    int t = wave;
    if (t < w.tiles) {
      constexpr bool late = NQ > 1;
      KeyTile<W> ka, kb;
      ValueTile<W> va, vb;
      int j0 = w.key_of(t);
      Pages pa = find_pages(a, page_ids(a, w.table, j0, w.ghi), j0, w.h), pb;
      load_keys<W>(a, pa, place, ka);
      if (!late) load_values<W>(a, pa, place, va);
      int j1 = w.key_of(min(t + waves, w.tiles - 1));
      PageIds ids = page_ids(a, w.table, j1, w.ghi);
      while (true) {
        if (late) load_values<W>(a, pa, place, va);
        pb = find_pages(a, ids, j1, w.h);
        load_keys<W>(a, pb, place, kb);
        if (!late) load_values<W>(a, pb, place, vb);
        const int j2 = w.key_of(min(t + 2 * waves, w.tiles - 1));
        ids = page_ids(a, w.table, j2, w.ghi);
        __builtin_amdgcn_sched_barrier(0);
        own_tile<E, W, NQ, false>(g, w, rows, qf, ka, va, pa, j0, li, kg, place, shift, sums);
        t += waves;
        if (t >= w.tiles) break;
        if (late) load_values<W>(a, pb, place, va);
        pa = find_pages(a, ids, j2, w.h);
        load_keys<W>(a, pa, place, ka);
        if (!late) load_values<W>(a, pa, place, va);
        j0 = w.key_of(min(t + 2 * waves, w.tiles - 1));
        ids = page_ids(a, w.table, j0, w.ghi);
        __builtin_amdgcn_sched_barrier(0);
        own_tile<E, W, NQ, false>(g, w, rows, qf, kb, late ? va : vb, pb, j1, li, kg, place, shift, sums);
        t += waves;
        if (t >= w.tiles) break;
        j1 = j0;
        j0 = j2;
      }
    }
    if (sums.unsure()) walk_again<E, W, NQ>(g, w, rows, qf, wave, waves, li, kg, place, shift, sums);
    auto& o = sums.o;
    auto& m = sums.m;
    auto& l = sums.l;
    // the sums of a row: over the lanes of its column, then over the workgroup's waves,
    // in their order
#pragma unroll
    for (int q = 0; q < NQ; q++) {
      m[q] += shift[q];
      l[q] = column_sum(l[q]);
    }
    float* ml = (float*)lds;                  // [waves][NQ * 16][2]
    float* ol = ml + waves * NQ * 32;         // [waves][NQ * 2W * 4][64]
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
    if (wave > 3) continue;
#pragma unroll
    for (int q = 0; q < NQ; q++) {
      float top = -INFINITY;
      for (int v = 0; v < waves; v++) top = fmaxf(top, ml[((v * NQ + q) * 16 + li) * 2]);
      m[q] = top;
      l[q] = 0.0f;
      // wave r takes the rows d = 2 W (4 kg + r) + x of every lane group
#pragma unroll
      for (int x = 0; x < 2 * W; x++) o[q][x][0] = 0.0f;
#pragma unroll 4
      for (int v = 0; v < waves; v++) {
        const float* from = ml + ((v * NQ + q) * 16 + li) * 2;
        const float wm = top == -INFINITY ? 0.0f : exp2_(rescale(from[0], top, sums.c));
        l[q] += wm * from[1];
#pragma unroll
        for (int x = 0; x < 2 * W; x++)
          o[q][x][0] += wm * ol[((v * NQ + q) * 8 * W + wave * 2 * W + x) * 64 + lane];
      }
    }
    store_rows<E, W, NQ, 1>(a, w, rows, kg, wave, m, l, o);
  }
}

// ------------------------------------------------------------ many rows

__device__ __forceinline__ f32x4 mfma16h(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// The products' types.  With float16 queries the scores are float16 products, and
// with queries of either two-byte type the second products are: one term of a
// bfloat16 row's probabilities (11 bits: the row is rounded to 8; with two, chunks with
// sinks 119 us for 95 and ragged trees 232 for 185), two of a float16 row's.  Probabilities
// stand 2^14 higher there, so that float16 holds them down to 2^-28 in full and to 2^-38 at all.
// That is of the bound, which stands up to 2^8 past the row's largest where a wave has two
// column tiles: smaller ones, and the rests of a float16 row's below 2^-9 of the largest, are
// off by half of 2^-30 of the largest.  Keys or values past what float16 holds, and NaN, send
// all rows of the workgroup through the second walk, which is in bfloat16 terms, as all of
// float32 is: a choice between two products in every tile has the sums held twice.  (One such
// block in a call: 1024 tokens of two prompts 281 us for 97, ragged trees of 32 sequences 200
// for 134, 100 tokens behind 131071 1118 for 405.)
template <typename E> struct Shared4 { static constexpr int kterms = E::terms, pterms = 3; };
template <> struct Shared4<F16> { static constexpr int kterms = 1, pterms = 2; };
template <> struct Shared4<BF16> { static constexpr int kterms = 1, pterms = 1; };

constexpr float kHigh = 14.0f;

// The scale byte of a block whose codes (this lane's word of them) are `codes`, for
// float16: any for zeros with a scale below its range.  (Past the range it stays, zeros or
// not: a written block of NaN has the mark 255 and zeros for codes.)
__device__ __forceinline__ unsigned f16_scale(unsigned s, unsigned codes) {
  return s >= 104u || codes & 0x77777777u ? s : 127u;
}

__device__ __forceinline__ bool f16_holds(unsigned s) { return s - 104u <= 36u; }

// By the registers of a wave (terms of the type, dh / 32): its column tiles, and the waves
// of a workgroup, two a SIMD or one.
constexpr int mask4_nq(int terms, int w) { return (terms == 3 ? w <= 2 : w <= 4) ? 2 : 1; }
constexpr int mask4_waves(int terms, int w) { return terms == 3 && w > 4 ? 4 : 8; }

// The kernel's arguments, read from memory here: the compiler loads all of them at the
// kernel's start, and those that are used late or seldom would take registers until then.
__device__ __forceinline__ const Mask4& late_args() {
  const Mask4* p = (const Mask4*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *p;
}

// What a maker has on its way of a tile, in LDS as it lies in the cache: the codes of
// 32 keys (or values), then their scales; a load is 64 x 16 or 64 x 4 bytes.
template <int W>
struct Raw4 {
  static constexpr int loads = (W + 1) / 2, codes = loads * 1024, bytes = codes + 256;
};

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"   // m0 is reserved; nothing else uses it here
// Loads to LDS that the compiler does not count (it would wait for them at every read
// of LDS): waited for by wait_vmcnt<0>() ahead of the reads.
__device__ __forceinline__ void lds_fetch16(unsigned to, const void* from) {
  __asm__ volatile(QPH_M0 "global_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "m0", "memory");
}

__device__ __forceinline__ void lds_fetch4(unsigned to, const void* from) {
  __asm__ volatile(QPH_M0 "global_load_lds_dword %1, off" ::"s"(to), "v"(from) : "m0", "memory");
}
#pragma clang diagnostic pop

// Starts the loads of a tile's keys or values (codes, scales: the cache's), whose halves
// start at the rows r0 and r1 of the pool.
template <int W>
__device__ __forceinline__ void fetch_tile(int64_t r0, int64_t r1, const unsigned char* codes,
                                           const unsigned char* scales, unsigned to, int lane) {
#pragma unroll
  for (int i = 0; i < Raw4<W>::loads; i++) {
    // (lanes past the tile, where W is odd, fetch its last bytes again)
    const int f = W % 2 ? min(64 * i + lane, 32 * W - 1) : 64 * i + lane;
    const bool u = f >= 16 * W;
    lds_fetch16(to + 1024 * i, codes + (u ? r1 : r0) * (16 * W) + 16 * (f - (u ? 16 * W : 0)));
  }
  const int f = min(lane, 8 * W - 1);
  const bool u = f >= 4 * W;
  lds_fetch4(to + Raw4<W>::codes, scales + (u ? r1 : r0) * W + 4 * (f - (u ? 4 * W : 0)));
}

// A lane's part of fetched keys.
template <int W>
__device__ __forceinline__ void take_keys(const unsigned char* raw, int li, int kg, KeyTile<W>& t) {
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const int key = 16 * u + li;
#pragma unroll
    for (int n = 0; n < W; n++) t.w[u][n] = ((const unsigned*)raw)[key * 4 * W + W * kg + n];
    const unsigned char* s = raw + Raw4<W>::codes + key * W;
    t.s[u][0] = s[W * kg / 4];
    if constexpr (Lane<W>::kblocks > 1) t.s[u][1] = s[(W * kg + W - 1) / 4];
  }
}

// And of values, the lane's bytes lowest (what is past them is not used).
template <int W>
__device__ __forceinline__ void take_values(const unsigned char* raw, int li, int kg, ValueTile<W>& t) {
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const int key = 16 * (e / 4) + 4 * kg + e % 4;
    const unsigned char* p = raw + key * 16 * W + W * li;
    const unsigned char* s = raw + Raw4<W>::codes + key * W;
    if constexpr (W == 1) {
      t.w[e][0] = *p;
    } else if constexpr (W == 2) {
      t.w[e][0] = *(const unsigned short*)p;
    } else if constexpr (Lane<W>::odd) {
      const unsigned* q = (const unsigned*)(raw + key * 16 * W) + W * li / 4;
      const unsigned long long v = ((unsigned long long)q[1] << 32 | q[0]) >> (8 * (W * li % 4));
      t.w[e][0] = (unsigned)v;
      if constexpr (Lane<W>::vwords > 1) t.w[e][1] = (unsigned)(v >> 32);
    } else {
#pragma unroll
      for (int i = 0; i < Lane<W>::vwords; i++) t.w[e][i] = ((const unsigned*)p)[i];
    }
    t.s[e][0] = s[W * li / 16];
    if constexpr (Lane<W>::vblocks > 1) t.s[e][1] = s[(W * li + W - 1) / 16];
  }
}

// A wave's rows of the row tile from r0 on by themselves, and whatever they meet: in
// careful walks alone, the first of which finds the maxima.  (A function of its own:
// seldom, and it would take registers from the kernel.)
template <typename E, int W, int NQ>
__device__ __noinline__ void slow_rows(const Mask4* g, int b, int h, int rt0, int split, int64_t va, int64_t vb,
                                       int64_t r0, int R) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, kg = lane >> 4;
  r0 = same_in_all(r0);
  Walk4 w(*g, Part4{(int)same_in_all(b), (int)same_in_all(h), (int)same_in_all(rt0), (int)same_in_all(split),
                    same_in_all(va), same_in_all(vb)});
  if (r0 + 16 * NQ * wave >= w.rows) return;
  const Place<W> place(li, kg);
  w.tiles_of(r0, min(w.rows, r0 + R) - 1, g->a.group);
  const Rows4<NQ> rows(*g, w, 16 * NQ * wave, li);
  bf16x8 qf[NQ][E::terms][W];
  load_queries<E, W, NQ>(g->a, w, rows, kg, qf);
  Sums4<W, NQ> sums(g->a);
  float shift[NQ];
  for (int i = 0; i < 2; i++) {
    walk_again<E, W, NQ>(*g, w, rows, qf, 0, 1, li, kg, place, shift, sums);
    bool far = false;
#pragma unroll
    for (int q = 0; q < NQ; q++) far |= (sums.m[q] != -INFINITY && is_far(sums.m[q] * sums.c)) || sums.l[q] != sums.l[q];
    if (!__any(far)) break;
  }
#pragma unroll
  for (int q = 0; q < NQ; q++) {
    sums.m[q] += shift[q];
    sums.l[q] = column_sum(sums.l[q]);
  }
  store_rows<E, W, NQ, 4>(g->a, w, rows, kg, 0, sums.m, sums.l, sums.o);
}

// Waves of a workgroup work on the same tiles, each on 16 NQ rows of its own.  Turning
// codes into operands takes more vector instructions than the softmax of 16 rows, so
// it is done once a tile: the first four waves each turn the keys or the values of
// one tile of a pair, and leave the operands in LDS as the lanes will read them (16
// bytes a lane, lane after lane: no bank conflict either way).
//
// A round, between two barriers: the second product of a pair of tiles and the first
// of the next pair, whose scores then lie in the registers of the pair before (so the
// matrix unit has work while the exponentials of the other tile are taken); keys of the
// pair after that and values of the next are turned; and the codes of one pair more
// are on their way.  (Two halves of the waves in opposite phases, one multiplying while the
// other turns codes and takes exponentials, were slower: 119 us for 96.)
template <typename E, int W, int NQ, bool EVEN>
__global__ __launch_bounds__(64 * mask4_waves(E::terms, W), mask4_waves(E::terms, W) / 4) void
mask4_shared_kernel(Mask4 g) {
  const Attn4& a = g.a;
  constexpr int KT = Shared4<E>::kterms, PT = Shared4<E>::pterms;
  constexpr bool KH = E::terms == 2, VH = E::terms < 3;     // float16 products
  constexpr int kHalf = 2 * W * 64;                         // 16-byte words of a tile's keys or values
  extern __shared__ u32x4 lds[];                            // keys [2][2], values [2][2]
  int* flags = (int*)(lds + 8 * kHalf);                     // [4][2], or [waves]; 16 words
  const int waves = blockDim.x >> 6;
  const int R = 16 * NQ * waves;
  // (EVEN: what is left of the share and the part at hand, kept here: they would take
  // registers that the walk needs)
  EvenState* state = (EvenState*)(flags + 16);
  if constexpr (EVEN) {
    if (threadIdx.x == 0) state->at = -1;
    __syncthreads();
  }
  while (true) {
    // (what follows from the lane is found anew each time, for the registers' sake)
    int thread = threadIdx.x;
    if constexpr (EVEN) asm volatile("" : "+v"(thread));
    const int lane = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    const int li = lane & 15, kg = lane >> 4;
    const int slot = wave >> 1;
    const bool keys = !(wave & 1), maker = wave < 4;
    Part4 part;
    if constexpr (EVEN) {
      int parts;
      int64_t at = same_in_all(state->at), end = same_in_all(state->end);
      const bool some = next_part(late_args(), at, end, part, parts);
      __syncthreads();                    // (the last part's reads of LDS too)
      if (!some) break;
      // (in scalar registers, and with them all that follows from it: float32 trees of 32
      // sequences 140 us, 201 where the compiler held them in each lane)
      part = Part4{(int)same_in_all(part.b), (int)same_in_all(part.h), 0, (int)same_in_all(part.split),
                   same_in_all(part.va), same_in_all(part.vb)};
      if (thread == 0) *state = EvenState{at, end, part};
      if (part.va == 0) unused_splits(late_args(), part, parts);
    } else {
      part = part_of_block(a);
    }
    Walk4 w(g, part);
    bool again = false;
    if ((int64_t)w.rt0 * R < w.rows) {
      w.tiles_of((int64_t)w.rt0 * R, min(w.rows, (int64_t)w.rt0 * R + R) - 1, a.group);
      const unsigned d0 = 16 * NQ * wave;
      const bool idle = w.r0 + d0 >= w.rows;
      const int pairs = (w.tiles + 1) >> 1;
      const Rows4<NQ> rows(g, w, d0, li);
      // queries: as they are, or (float32) in bfloat16 terms
      bf16x8 qf[NQ][KT][W];
      if constexpr (KH) {
        const _Float16 sign = a.scale < 0.0f ? (_Float16)-1.0f : (_Float16)1.0f;
#pragma unroll
        for (int q = 0; q < NQ; q++)
#pragma unroll
          for (int n = 0; n < W; n++) {
            f16x8 v;
            __builtin_memcpy(&v, (const _Float16*)a.q + (w.t0 + rows.tok[q]) * a.qt + rows.head[q] * a.qh +
                                     8 * (W * kg + n), 16);
            qf[q][0][n] = __builtin_bit_cast(bf16x8, v * sign);
          }
      } else {
        load_queries<E, W, NQ>(a, w, rows, kg, qf);
      }
      Sums4<W, NQ> sums(a);
      float shift[NQ];
#pragma unroll
      for (int q = 0; q < NQ; q++) shift[q] = 0.0f;

      // A maker's tile on its way; where the halves of its next 32 tiles lie, one to a lane (a
      // row of the pool, and whether the page is one in the highest bit).
      unsigned char* raw = (unsigned char*)(flags + 64) + (wave & 3) * Raw4<W>::bytes;
      const unsigned raw_at = __builtin_amdgcn_readfirstlane(
          (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)raw);
      const unsigned char *codes = keys ? a.kc : a.vc, *scales = keys ? a.ks : a.vs;
      const int off = keys ? 2 : 1;         // pairs that its operands are made ahead
      const int mine = maker ? (w.tiles - slot + 1) >> 1 : 0;      // its tiles
      unsigned row_lo = 0, row_hi = 0;
      int on = 0;                           // which halves of the tile on its way lie on pages
      bool odd = false;                     // it has met what float16 does not hold
      auto fetch = [&](int pair) __attribute__((always_inline)) {
        if (pair >= mine) return;
        if ((pair & 31) == 0) {
          const int t = min(2 * (pair + (lane >> 1)) + slot, w.tiles - 1);
          const int j = w.key_of(t) + 16 * (lane & 1);
          const Attn4& c = late_args().a;
          const int page = ((const int32_t*)w.table)[min(j, w.ghi - 1) >> c.shift];
          const bool there = page >= 0 && page < c.n_pages;
          const int64_t row = (((int64_t)(there ? page : 0) * c.heads + w.h) << c.shift) + (j & ((1 << c.shift) - 1));
          row_lo = (unsigned)row;
          row_hi = (unsigned)(row >> 32) | (there ? 0x80000000u : 0u);
        }
        const int at = 2 * (pair & 31);
        const unsigned h0 = __builtin_amdgcn_readlane(row_hi, at), h1 = __builtin_amdgcn_readlane(row_hi, at + 1);
        const unsigned l0 = __builtin_amdgcn_readlane(row_lo, at), l1 = __builtin_amdgcn_readlane(row_lo, at + 1);
        on = (int)(h0 >> 31 | (h1 >> 31) << 1);
        // (the reads of what lies there have ended: their values are used)
        fetch_tile<W>((int64_t)(h0 & 0x7fffffffu) << 32 | l0, (int64_t)(h1 & 0x7fffffffu) << 32 | l1, codes, scales,
                      raw_at, lane);
      };
      auto make = [&](int pair) __attribute__((always_inline)) {
        if (!maker || pair >= pairs) return;
        // (its addresses are found anew each time: they would take registers from the products)
        int lane = threadIdx.x & 63;
        if constexpr (EVEN) asm volatile("" : "+v"(lane));
        const int li = lane & 15, kg = lane >> 4;
        u32x4* to = lds + ((keys ? 0 : 4) + 2 * (pair & 1) + slot) * kHalf + lane;
        const bool there = pair < mine;
        wait_vmcnt<0>();
        __asm__ volatile("" ::: "memory");
        if (keys) {
          if (lane == 0) flags[2 * (pair & 3) + slot] = there ? on : 0;
          KeyTile<W> kt;
          take_keys<W>(raw, li, kg, kt);
#pragma unroll
          for (int u = 0; u < 2; u++)
#pragma unroll
            for (int n = 0; n < W; n++) {
              if constexpr (KH) {
                const unsigned s0 = kt.s[u][0], s1 = kt.s[u][Lane<W>::kblocks - 1];
                const unsigned sc = f16_scale((W * kg + n) / 4 == W * kg / 4 ? s0 : s1, kt.w[u][n]);
                odd |= there && !f16_holds(sc);
                to[(u * W + n) * 64] = __builtin_bit_cast(u32x4, fp4_word_f16(kt.w[u][n], scale_of_byte(sc)));
              } else {
                to[(u * W + n) * 64] = __builtin_bit_cast(u32x4, key_operand<W>(kt, kg, u, n));
              }
            }
        } else {
          ValueTile<W> vt;
          take_values<W>(raw, li, kg, vt);
          // (of a tile that is none: zeros, as of keys that no row sees)
          clear_unseen<W>(w, vt, there && (on & 1), there && (on & 2), w.key_of(2 * pair + slot), kg);
          if constexpr (VH) {
            unsigned lo = 255, hi = 0;
#pragma unroll
            for (int e = 0; e < 8; e++)
#pragma unroll
              for (int i = 0; i < Lane<W>::vblocks; i++) {
                lo = min(lo, vt.s[e][i]);
                hi = max(hi, vt.s[e][i]);
              }
            if (__any(!f16_holds(lo) || !f16_holds(hi))) {
#pragma unroll
              for (int e = 0; e < 8; e++)
#pragma unroll
                for (int i = 0; i < Lane<W>::vblocks; i++) {
                  unsigned codes = 0;
#pragma unroll
                  for (int x = 0; x < Lane<W>::vwords; x++) codes |= vt.w[e][x];
                  vt.s[e][i] = f16_scale(vt.s[e][i], codes);
                  odd |= !f16_holds(vt.s[e][i]);
                }
            }
          }
          Place<W> place(li, kg);
          place.shift = 0;
          value_operands<W, VH>(vt, place, li, [&](int x, u32x4 v) __attribute__((always_inline)) { to[x * 64] = v; });
        }
        __asm__ volatile("" ::: "memory");
      };

      f32x4 s[2][2][NQ];                     // scores of a pair
      float mc[NQ];
      u32x4 kf[2 * W], vf[2][W];
      auto read_keys = [&](int buffer, int i) __attribute__((always_inline)) {
        const u32x4* from = lds + (2 * buffer + i) * kHalf + lane;
#pragma unroll
        for (int x = 0; x < 2 * W; x++) kf[x] = from[x * 64];
      };
      auto read_values = [&](int buffer, int i, int half) __attribute__((always_inline)) {
        const u32x4* from = lds + (4 + 2 * buffer + i) * kHalf + half * W * 64 + lane;
#pragma unroll
        for (int x = 0; x < W; x++) vf[half][x] = from[x * 64];
      };
      auto scores = [&](int i) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int q = 0; q < NQ; q++) s[i][u][q] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int n = 0; n < W; n++)
#pragma unroll
          for (int u = 0; u < 2; u++)
#pragma unroll
            for (int q = 0; q < NQ; q++) {
              const u32x4 k = kf[u * W + n];
              if constexpr (KH) {
                s[i][u][q] = mfma16h(__builtin_bit_cast(f16x8, k), __builtin_bit_cast(f16x8, qf[q][0][n]), s[i][u][q]);
              } else {
#pragma unroll
                for (int t = KT - 1; t >= 0; t--)
                  s[i][u][q] = mfma16(__builtin_bit_cast(bf16x8, k), qf[q][t][n], s[i][u][q]);
              }
            }
      };
      auto terms = [&](int i, bf16x8 (&pf)[NQ][PT]) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < NQ; q++) {
          float p[8], sum = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; e++) {
            p[e] = exp2_(__builtin_fmaf(s[i][e / 4][q][e % 4], sums.c, -mc[q]));
            sum = e ? sum + p[e] : p[e];
          }
          sums.l[q] += sum;
          if constexpr (VH) {
            f16x8 f;
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] = (_Float16)p[e];
            pf[q][0] = __builtin_bit_cast(bf16x8, f);
            if constexpr (PT > 1) {
              f16x8 f1;
#pragma unroll
              for (int e = 0; e < 8; e++) f1[e] = (_Float16)(p[e] - (float)f[e]);
              pf[q][1] = __builtin_bit_cast(bf16x8, f1);
            }
          } else {
            split8<PT, false>(p, pf[q]);
          }
        }
      };
      auto add_values = [&](const bf16x8 (&pf)[NQ][PT], int half) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < W; x++)
#pragma unroll
          for (int q = 0; q < NQ; q++)
#pragma unroll
            for (int t = PT - 1; t >= 0; t--) {
              f32x4& o = sums.o[q][half * W + x];
              if constexpr (VH)
                o = mfma16h(__builtin_bit_cast(f16x8, vf[half][x]), __builtin_bit_cast(f16x8, pf[q][t]), o);
              else
                o = mfma16(__builtin_bit_cast(bf16x8, vf[half][x]), pf[q][t], o);
            }
      };

      // what the first round needs, and the loads of the next
      fetch(0);
      make(0);
      if (keys) {
        fetch(1);
        make(1);
      }
      fetch(off);
      // pairs of tiles that need no masks (where they lie on pages): behind the first tokens
      const int clear0 = w.n1 + ((max(rows.all_lo - w.b0, 0) + 31) >> 5), clear1 = w.n1 + ((rows.all_hi - w.b0) >> 5);
      __syncthreads();
      if (!idle) {
        read_keys(0, 0);
        scores(0);
        read_keys(0, 1);
        scores(1);
      }
      __syncthreads();
      for (int pair = 0; pair < pairs; pair++) {
        const int on0 = flags[2 * (pair & 3)], on1 = flags[2 * (pair & 3) + 1];
        make(pair + off);
        fetch(pair + off + 1);
        if (!idle) {
          const int buffer = pair & 1;
          // masks and maxima of the pair's scores
          const int there0 = __builtin_amdgcn_readfirstlane(on0), there1 = __builtin_amdgcn_readfirstlane(on1);
          if (2 * pair < clear0 || 2 * pair + 2 > clear1 || (there0 & there1) != 3) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const int there = i ? there1 : there0;
              rows.mask(late_args(), w, w.key_of(2 * pair + i), kg, there & 1, there & 2, shift, s[i]);
            }
          }
          bool grows = false;
          float mx[NQ];
#pragma unroll
          for (int q = 0; q < NQ; q++) {
            mx[q] = s[0][0][q][0];
#pragma unroll
            for (int e = 1; e < 16; e++) mx[q] = fmaxf(mx[q], s[e / 8][e / 4 % 2][q][e % 4]);
            grows |= mx[q] > sums.m[q];
          }
          // (all lanes or none; said as each lane's own choice, for which the compiler scales
          // the sums where they are: else it copies all of them every round, 5% of the time)
          const bool some = __any(grows);
          if (grows | some) {
#pragma unroll
            for (int q = 0; q < NQ; q++) sums.raise_to(q, column_max(mx[q]));
          }
#pragma unroll
          for (int q = 0; q < NQ; q++) mc[q] = sums.offset(q) - (VH ? kHigh : 0.0f);
          // The pair's terms and their products with the values; between them the next
          // pair's scores (the last round's are of nothing and not used).  Operands are
          // read a step ahead of their products.
          bf16x8 p0[NQ][PT], p1[NQ][PT];
          read_keys(buffer ^ 1, 0);
          __builtin_amdgcn_sched_barrier(0);
          terms(0, p0);
          read_values(buffer, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
          scores(0);
          read_values(buffer, 0, 1);
          __builtin_amdgcn_sched_barrier(0);
          add_values(p0, 0);
          add_values(p0, 1);
          read_keys(buffer ^ 1, 1);
          __builtin_amdgcn_sched_barrier(0);
          terms(1, p1);
          read_values(buffer, 1, 0);
          __builtin_amdgcn_sched_barrier(0);
          scores(1);
          read_values(buffer, 1, 1);
          __builtin_amdgcn_sched_barrier(0);
          add_values(p1, 0);
          add_values(p1, 1);
        }
        __syncthreads();
      }
      again = sums.unsure();
      if constexpr (VH) {
        if (lane == 0) flags[wave] = 0;
        if (odd) flags[wave] = 1;
        __syncthreads();
        for (int i = 0; i < waves; i++) again |= flags[i] != 0;
        again = __any(again);
      }
      if (!idle && !again) {
#pragma unroll
        for (int q = 0; q < NQ; q++) {
          sums.l[q] = column_sum(sums.l[q]);
          if constexpr (VH) {
            sums.l[q] *= 0x1p-14f;
#pragma unroll
            for (int x = 0; x < 2 * W; x++)
#pragma unroll
              for (int r = 0; r < 4; r++) sums.o[q][x][r] *= 0x1p-14f;
          }
        }
        // (found anew: out of the compiler's sight, which would keep them through the walk)
        int lanes = li;
        asm volatile("" : "+v"(lanes));
        const Rows4<NQ> at(late_args(), w, d0, lanes);
        store_rows<E, W, NQ, 4>(late_args().a, w, at, kg, 0, sums.m, sums.l, sums.o);
      }
    }
    // rows to be walked again, and those of a sequence with more than max_new bounds
    const Mask4& late = late_args();
    for (int64_t tile = (int64_t)w.rt0 + (again ? 0 : late.a.row_tiles); tile * R < w.rows; tile += late.a.row_tiles) {
      const Part4 p = EVEN ? state->part : part_of_block(late.a);
      slow_rows<E, W, NQ>(&late, p.b, p.h, p.rt0, p.split, p.va, p.vb, tile * R, R);
    }
    if constexpr (!EVEN) break;
  }
}

// How a call is run: waves of a workgroup that share tiles (0: few rows), column tiles
// a wave.
struct Mask4Plan {
  int nq, waves, few, even;       // (few: waves that share few rows; even: even shares)
  int row_tiles, splits;
  int64_t chunk;
  size_t workspace;
};

template <typename E, int W, int NQ>
static int launch_mask4_few(const Mask4& g, int few, hipStream_t s) {
  const size_t lds = (size_t)few * NQ * (32 + 2 * W * 4 * 64) * 4;
  if (lds > 65536) QPH_TRY(allow_full_lds((const void*)mask4_few_kernel<E, W, NQ>));
  const int64_t blocks = (int64_t)g.a.row_tiles * g.a.splits * g.a.heads * g.a.batch;
  hipLaunchKernelGGL((mask4_few_kernel<E, W, NQ>), dim3((unsigned)blocks), dim3(64 * few), lds, s, g);
  return launch_check("mask4_few_kernel");
}

template <typename E, int W, int NQ, bool EVEN>
static int launch_mask4_shared(const Mask4& g, int waves, hipStream_t s) {
  const size_t lds = (size_t)16 * W * 1024 + 256 + 4 * Raw4<W>::bytes;
  if (lds > 65536) QPH_TRY(allow_full_lds((const void*)mask4_shared_kernel<E, W, NQ, EVEN>));
  const int64_t blocks = EVEN ? (waves > 4 ? 256 : 512)
                                : (int64_t)g.a.row_tiles * g.a.splits * g.a.heads * g.a.batch;
  hipLaunchKernelGGL((mask4_shared_kernel<E, W, NQ, EVEN>), dim3((unsigned)blocks), dim3(64 * waves), lds, s, g);
  return launch_check("mask4_shared_kernel");
}

template <typename E, int W>
static int launch_mask4_w(const Mask4& g, const Mask4Plan& p, hipStream_t s) {
  constexpr int NQ = mask4_nq(E::terms, W);
  if (p.even) return launch_mask4_shared<E, W, NQ, true>(g, p.waves, s);
  if (p.waves) return launch_mask4_shared<E, W, NQ, false>(g, p.waves, s);
  if constexpr (mask4_nq(E::terms, W) == 2) {
    if (p.nq == 2) return launch_mask4_few<E, W, 2>(g, p.few, s);
  }
  return launch_mask4_few<E, W, 1>(g, p.few, s);
}

template <typename E>
static int launch_mask4(const Mask4& g, const Mask4Plan& p, int dh, hipStream_t s) {
  switch (dh) {
    case 32: return launch_mask4_w<E, 1>(g, p, s);
    case 64: return launch_mask4_w<E, 2>(g, p, s);
    case 96: return launch_mask4_w<E, 3>(g, p, s);
    case 128: return launch_mask4_w<E, 4>(g, p, s);
    case 192: return launch_mask4_w<E, 6>(g, p, s);
    default: return launch_mask4_w<E, 8>(g, p, s);
  }
}

// One source file an element type.
int launch_mask4_f32(const Mask4& g, const Mask4Plan& p, int dh, hipStream_t s);
int launch_mask4_f16(const Mask4& g, const Mask4Plan& p, int dh, hipStream_t s);
int launch_mask4_bf16(const Mask4& g, const Mask4Plan& p, int dh, hipStream_t s);

}  // namespace qph
