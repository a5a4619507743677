// Attention over the 4-bit cache where a row sees more than a run of keys: a window
// and a sequence's first tokens beside it, or the context and the drafted tokens on
// its own path of a tree.
//
// For a new token and a query head, over the keys j that the row sees:
//   s_j = scale q . k_j,  m = max s_j,  o = sum exp(s_j - m) v_j / sum exp(s_j - m)
// with the products, the running maximum and the second walk of qph_attn4.hip.  Two
// forms:
//
// Few rows of a sequence and head (SH false): the waves of a workgroup share 16 NQ
// rows and take the tiles of 32 keys in turn, codes to registers to operands.
//
// Many (SH true): each wave has 16 NQ rows of its own, so every tile is needed by all
// four.  Turning codes into operands takes about as many vector instructions as the
// softmax of 32 rows, and is done once: wave w turns tile 4 i + w and leaves the
// operands in LDS as the lanes will read them (16 bytes a lane, lane after lane:
// no bank conflict either way), then all four compute the four tiles, while the
// codes of the next four are on their way.
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

// Rows of a workgroup of the two forms.
constexpr int mask4_rows(int nq, bool shared) { return 16 * nq * (shared ? 4 : 1); }

// The four bits of a tree's row from drafted token d on (none before the first).
__device__ __forceinline__ unsigned path_bits(const unsigned* row, int words, int d) {
  if (d <= -4) return 0;
  const int e = max(d, 0), w = e >> 5;
  const unsigned long long lo = w < words ? row[w] : 0u, hi = w + 1 < words ? row[w + 1] : 0u;
  const unsigned v = (unsigned)((hi << 32 | lo) >> (e & 31));
  return d < 0 ? v << -d : v;
}

template <typename E, int W, int NQ, bool SH>
__global__ __launch_bounds__(256, SH ? ((E::terms == 3 ? W <= 2 : W <= 4) ? 2 : 1)
                                     : (NQ == 1 && W <= 4 && E::terms < 3 ? 3 : 1)) void
mask4_kernel(Mask4 g) {
  const Attn4& a = g.a;
  // (terms of the probabilities: as in attn4_kernel)
  constexpr int T = E::terms, PT = T < 2 ? 2 : T;
  constexpr int DH = 32 * W, R = mask4_rows(NQ, SH);
  extern __shared__ u32x4 lds[];
  int* flags = (int*)(lds + 16 * W * 64);  // which halves of the staged tiles lie on pages
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
  const int first = len - news;          // position of the first new token; the context's keys
  const bool tree = g.tree != nullptr;
  // the first key inside the window of a token at position p
  auto window_from = [&](int64_t p) {
    return a.window > 0 ? (int)max((int64_t)0, p - a.window + 1) : 0;
  };
  // the key behind the last that a token at position p sees (a tree's: of the context)
  auto border = [&](int64_t p) {
    return tree ? max(first, 0) : a.causal ? (int)min((int64_t)len, max(p + 1, (int64_t)0)) : len;
  };

  // the two runs of keys of the whole sequence, [0, s32) and from `base` on, and of
  // this split: a run of both counted as one (a path has first - 1 or more as its
  // position: the window of none starts before that of first - 1)
  const int s32 = (min(g.sinks, len) + 31) & ~31;
  const int base = a.window > 0 ? max(s32, window_from((int64_t)first - tree) & ~31) : 0;
  const int64_t va = split * a.chunk, vb = split == a.splits - 1 ? INT64_MAX / 2 : va + a.chunk;
  const int a0 = (int)min(va, (int64_t)s32), a1 = (int)min(vb, (int64_t)s32);
  const int64_t bfrom = base + max(va - s32, (int64_t)0), bto = base + max(vb - s32, (int64_t)0);

  const Place<W> place(li, kg);
  const float c = fabsf(a.scale) * kLog2e;
  const float sign = a.scale < 0.0f ? -1.0f : 1.0f;
  // (the bound's distance as a score; it vanishes beside a far one)
  const float lazy = fminf(kLazy / c, FLT_MAX);

  for (int64_t tile = rt0; tile * R < rows; tile += a.row_tiles) {
    // keys that some row of the workgroup sees
    const int64_t r0 = tile * R, r1 = min(rows, r0 + R) - 1;
    const int ghi = tree ? len : border((int64_t)first + (int)(r1 / a.group));
    const int glo = window_from(tree ? (int64_t)first - 1 : (int64_t)first + (int)(r0 / a.group));
    const int n1 = (max(min(a1, ghi) - a0, 0) + 31) >> 5;
    const int b0 = (int)max(bfrom, (int64_t)(glo & ~31));
    const int n2 = bfrom >= ghi ? 0 : (max((int)min(bto, (int64_t)ghi) - b0, 0) + 31) >> 5;
    const int tiles = n1 + n2;
    auto key_of = [&](int t) { return t < n1 ? a0 + 32 * t : b0 + 32 * (t - n1); };

    // (a row has seen a key if and only if its sum is not 0: the largest score's
    // term is 1 or near it, and NaN is not 0 either)
    // rows of this wave: query fragments, what each sees
    const int64_t w0 = r0 + (SH ? 16 * NQ * wave : 0), w1 = min(rows, w0 + 16 * NQ) - 1;
    const bool idle = w0 >= rows;
    bf16x8 qf[NQ][T][W];
    int64_t tok[NQ];
    int lo[NQ], hi[NQ], head[NQ];
    bool live[NQ];
#pragma unroll
    for (int q = 0; q < NQ; q++) {
      const int64_t r = w0 + 16 * q + li;
      live[q] = r < rows;
      const int64_t rr = live[q] ? r : rows - 1;
      const int i = (int)(rr / a.group);
      head[q] = h * a.group + (int)(rr - (int64_t)i * a.group);
      tok[q] = t0 + i;
      int64_t pos = (int64_t)first + i;
      if (tree && a.window > 0) {
        // a path's end stands as many places behind the context as it has tokens
        const unsigned* path = g.tree + tok[q] * g.words;
        int depth = 0;
        for (int w = 0; w < g.words && 32 * w < news; w++) {
          const int left = news - 32 * w;
          depth += __popc(left < 32 ? path[w] & ((1u << left) - 1) : path[w]);
        }
        pos = (int64_t)first + depth - 1;
      }
      hi[q] = live[q] ? border(pos) : 0;
      lo[q] = window_from(pos);
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
    // tiles that need no masks: from all_lo, or before sure, up to all_hi
    const int sure = g.sinks;
    const int all_lo = window_from((int64_t)first + (tree ? news - 1 : (int)(max(w1, (int64_t)0) / a.group)));
    const int all_hi = min(ghi, border((int64_t)first + (int)(w0 / a.group)));

    f32x4 o[NQ][2 * W];
    float m[NQ], l[NQ], shift[NQ];     // shift: what a second walk takes off the scores
#pragma unroll
    for (int q = 0; q < NQ; q++) {
      m[q] = -INFINITY;
      shift[q] = 0.0f;
    }
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int q = 0; q < NQ; q++) {
        l[q] = 0.0f;
#pragma unroll
        for (int x = 0; x < 2 * W; x++) o[q][x] = f32x4{0, 0, 0, 0};
      }
    };

    // Scores of a tile from key j0 on, masked, and their terms; kop(u, n): operand n of
    // 16 keys.
    auto terms = [&](auto&& kop, bool there0, bool there1, int j0, bool all, f32x4 (&s)[2][NQ],
                     bf16x8 (&pf)[NQ][PT]) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < 2; u++) {
#pragma unroll
        for (int q = 0; q < NQ; q++) s[u][q] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int n = 0; n < W; n++) {
          const bf16x8 kf = kop(u, n);
#pragma unroll
          for (int q = 0; q < NQ; q++)
#pragma unroll
            for (int t = T - 1; t >= 0; t--) s[u][q] = mfma16(kf, qf[q][t][n], s[u][q]);
        }
      }
      if (!all) {
#pragma unroll
        for (int q = 0; q < NQ; q++)
#pragma unroll
          for (int u = 0; u < 2; u++) {
            const int j1 = j0 + 16 * u + 4 * kg;
            unsigned bits = 0;
            if (tree && j0 + 32 > first) bits = path_bits(g.tree + tok[q] * g.words, g.words, j1 - first);
#pragma unroll
            for (int r = 0; r < 4; r++) {
              const int j = j1 + r;
              const bool near = j < hi[q] && (j >= lo[q] || j < g.sinks);
              const bool see = (u ? there1 : there0) && j < len && (near || (live[q] && (bits >> r & 1)));
              s[u][q][r] = see ? s[u][q][r] - shift[q] : -INFINITY;
            }
          }
      }
      // running maximum, exponentials
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
    };
    auto add_values = [&](bf16x8 v, int x, bf16x8 (&pf)[NQ][PT]) __attribute__((always_inline)) {
#pragma unroll
      for (int q = 0; q < NQ; q++)
#pragma unroll
        for (int t = PT - 1; t >= 0; t--) o[q][x] = mfma16(v, pf[q][t], o[q][x]);
    };
    auto needs_no_masks = [&](int j0) {
      return (j0 >= all_lo || j0 + 32 <= sure) && j0 + 32 <= all_hi;
    };

    // A lane's operands out of the codes it has loaded.
    auto key_operand = [&](const KeyTile<W>& kt, int u, int n) __attribute__((always_inline)) {
      const float s0 = scale_of_byte(kt.s[u][0]);
      const float s1 = Lane<W>::kblocks > 1 ? scale_of_byte(kt.s[u][Lane<W>::kblocks - 1]) : s0;
      return fp4_word(kt.w[u][n], (W * kg + n) / 4 == W * kg / 4 ? s0 : s1);
    };
    // the values of keys that no row sees, whatever stands there, are zeros
    auto clear_unseen = [&](ValueTile<W>& vt, const Pages& pg, int j0) __attribute__((always_inline)) {
      if (j0 >= glo && j0 + 32 <= ghi && pg.there[0] && pg.there[1]) return;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int j = j0 + 16 * (e / 4) + 4 * kg + e % 4;
        if (!pg.there[e / 4] || j >= ghi || (j < glo && j >= g.sinks)) {
#pragma unroll
          for (int i = 0; i < Lane<W>::vblocks; i++) vt.s[e][i] = 127;
#pragma unroll
          for (int i = 0; i < Lane<W>::vwords; i++) vt.w[e][i] = 0;
        }
      }
    };
    auto value_operands = [&](ValueTile<W>& vt, auto&& take) __attribute__((always_inline)) {
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
    };

    // One tile from this wave's registers; the second walk is careful, see below.
    auto compute = [&](const KeyTile<W>& kt, ValueTile<W>& vt, const Pages& pg, int j0, auto second) __attribute__((always_inline)) {
      constexpr bool careful = decltype(second)::value;
      f32x4 s[2][NQ];
      bf16x8 pf[NQ][PT];
      terms([&](int u, int n) __attribute__((always_inline)) { return key_operand(kt, u, n); }, pg.there[0], pg.there[1], j0,
            !careful && needs_no_masks(j0) && pg.there[0] && pg.there[1], s, pf);
      clear_unseen(vt, pg, j0);
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
              if (hit[r] != 0.0f) o[q][x][r] = NAN;
          }
        }
#pragma unroll
        for (int e = 0; e < 8; e++)
#pragma unroll
          for (int i = 0; i < Lane<W>::vblocks; i++)
            if (vt.s[e][i] > 252) vt.s[e][i] = 0;
      }
      value_operands(vt, [&](int x, u32x4 v) __attribute__((always_inline)) {
        add_values(__builtin_bit_cast(bf16x8, v), x, pf);
      });
    };

    // This wave's tiles t, t + 4, ... from its registers; the next one's loads in flight
    // while one is computed (with more rows a wave the values' come late, behind the
    // keys' products).
    auto walk = [&](int t) __attribute__((always_inline)) {
      if (t >= tiles) return;
      constexpr bool late = NQ > 1;
      KeyTile<W> ka, kb;
      ValueTile<W> va, vb;
      int j0 = key_of(t);
      Pages pa = find_pages(a, page_ids(a, table, j0, ghi), j0, h), pb;
      load_keys<W>(a, pa, place, ka);
      if (!late) load_values<W>(a, pa, place, va);
      int j1 = key_of(min(t + 4, tiles - 1));
      PageIds ids = page_ids(a, table, j1, ghi);
      while (true) {
        if (late) load_values<W>(a, pa, place, va);
        pb = find_pages(a, ids, j1, h);
        load_keys<W>(a, pb, place, kb);
        if (!late) load_values<W>(a, pb, place, vb);
        const int j2 = key_of(min(t + 8, tiles - 1));
        ids = page_ids(a, table, j2, ghi);
        __builtin_amdgcn_sched_barrier(0);
        compute(ka, va, pa, j0, std::false_type());
        t += 4;
        if (t >= tiles) break;
        if (late) load_values<W>(a, pb, place, va);
        pa = find_pages(a, ids, j2, h);
        load_keys<W>(a, pa, place, ka);
        if (!late) load_values<W>(a, pa, place, va);
        j0 = key_of(min(t + 8, tiles - 1));
        ids = page_ids(a, table, j0, ghi);
        __builtin_amdgcn_sched_barrier(0);
        compute(kb, late ? va : vb, pb, j1, std::false_type());
        t += 4;
        if (t >= tiles) break;
        j1 = j0;
        j0 = j2;
      }
    };

    clear();
    if constexpr (!SH) {
      walk(wave);
    } else {
      // four tiles at a time by way of LDS: keys' operands (u, n) at 2 W items of
      // 64 x 16 bytes, values' after them
      KeyTile<W> kt;
      ValueTile<W> vt;
      Pages pg;
      int mine = wave, j = 0;
      if (tiles > 0) {
        j = key_of(min(mine, tiles - 1));
        pg = find_pages(a, page_ids(a, table, j, ghi), j, h);
        load_keys<W>(a, pg, place, kt);
        load_values<W>(a, pg, place, vt);
      }
      for (int t = 0; t < tiles; t += 4) {
        if (mine < tiles) {
          u32x4* to = lds + wave * (4 * W * 64) + lane;
          clear_unseen(vt, pg, j);
#pragma unroll
          for (int u = 0; u < 2; u++)
#pragma unroll
            for (int n = 0; n < W; n++)
              to[(u * W + n) * 64] = __builtin_bit_cast(u32x4, key_operand(kt, u, n));
          value_operands(vt, [&](int x, u32x4 v) __attribute__((always_inline)) { to[(2 * W + x) * 64] = v; });
          if (lane == 0) flags[wave] = pg.there[0] + 2 * pg.there[1];
        }
        mine += 4;
        if (mine < tiles) {
          j = key_of(mine);
          pg = find_pages(a, page_ids(a, table, j, ghi), j, h);
          load_keys<W>(a, pg, place, kt);
          load_values<W>(a, pg, place, vt);
        }
        __syncthreads();
        if (!idle) {
          const int n = min(4, tiles - t);
          for (int i = 0; i < n; i++) {
            const u32x4* from = lds + i * (4 * W * 64) + lane;
            const int there = __builtin_amdgcn_readfirstlane(flags[i]), j0 = key_of(t + i);
            f32x4 s[2][NQ];
            bf16x8 pf[NQ][PT];
            terms([&](int u, int n) __attribute__((always_inline)) { return __builtin_bit_cast(bf16x8, from[(u * W + n) * 64]); },
                  there & 1, there & 2, j0, needs_no_masks(j0) && there == 3, s, pf);
#pragma unroll
            for (int x = 0; x < 2 * W; x++)
              add_values(__builtin_bit_cast(bf16x8, from[(2 * W + x) * 64]), x, pf);
          }
        }
        __syncthreads();
      }
    }
    // Keys are walked a second time, for what would cost the first one more in every
    // tile (the reasons stand at attn4_kernel's): blocks of NaN in the values are
    // zeros the second time, and the rows that see them get their NaN from a product
    // of ones; a row whose maximum ended past kFar has it taken off its scores, one
    // whose sum overflowed on the way starts with its last maximum.  (Each wave
    // by itself, from its registers.)
    bool again = false;
#pragma unroll
    for (int q = 0; q < NQ; q++) {
      again |= m[q] != -INFINITY && is_far(m[q] * c);
#pragma unroll
      for (int x = 0; x < 2 * W; x++)
#pragma unroll
        for (int r = 0; r < 4; r++) again |= o[q][x][r] != o[q][x][r];
    }
    if (__any(again)) {
#pragma unroll
      for (int q = 0; q < NQ; q++) {
        const float sum = column_sum(l[q]);
        const bool far = m[q] != -INFINITY && is_far(m[q] * c);
        shift[q] = far ? m[q] : 0.0f;
        m[q] = far ? 0.0f : sum != sum ? m[q] : -INFINITY;
      }
      clear();
      for (int t = SH ? 0 : wave; t < tiles; t += SH ? 1 : 4) {
        KeyTile<W> kt;
        ValueTile<W> vt;
        const int j = key_of(t);
        const Pages pg = find_pages(a, page_ids(a, table, j, ghi), j, h);
        load_keys<W>(a, pg, place, kt);
        load_values<W>(a, pg, place, vt);
        compute(kt, vt, pg, j, std::true_type());
      }
    }
#pragma unroll
    for (int q = 0; q < NQ; q++) m[q] += shift[q];

    // the sums of a row: over the lanes of its column, then (waves that share their
    // rows) over the workgroup's waves, in their order
#pragma unroll
    for (int q = 0; q < NQ; q++) l[q] = column_sum(l[q]);
    if constexpr (!SH) {
      float* ml = (float*)lds;                  // [4][NQ * 16][2]
      float* ol = ml + 4 * NQ * 32;             // [4 waves][NQ * 2W * 4][64]
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
    constexpr int NR = SH ? 4 : 1;
#pragma unroll
    for (int q = 0; q < NQ; q++) {
      if (!live[q]) continue;
      const int64_t at = tok[q] * (a.heads * a.group) + head[q];
      if (a.splits > 1) {
        const int64_t part = (int64_t)split * a.tokens * (a.heads * a.group) + at;
        if (kg == 0 && (SH || wave == 0)) {
          a.part_ml[2 * part] = m[q];
          a.part_ml[2 * part + 1] = l[q];
        }
        if (l[q] == 0.0f) continue;
#pragma unroll
        for (int r = 0; r < NR; r++) {
          float* p = a.part_o + part * DH + 2 * W * (4 * kg + (SH ? r : wave));
#pragma unroll
          for (int x = 0; x < 2 * W; x++) p[x] = o[q][x][r];
        }
      } else {
        const float inv = l[q] == 0.0f ? 0.0f : 1.0f / l[q];
        if (a.lse && kg == 0 && (SH || wave == 0))
          a.lse[at] = l[q] == 0.0f ? -INFINITY : log_sum(m[q], l[q], fabsf(a.scale));
#pragma unroll
        for (int r = 0; r < NR; r++) {
          typename E::type* p = (typename E::type*)a.out + tok[q] * a.ot + head[q] * a.oh +
                                2 * W * (4 * kg + (SH ? r : wave));
          typename E::type t[2 * W];
#pragma unroll
          for (int x = 0; x < 2 * W; x++) t[x] = (typename E::type)(o[q][x][r] * inv);
          __builtin_memcpy(p, t, sizeof t);
        }
      }
    }
  }
}

// How a call is run.
struct Mask4Plan {
  int nq;
  bool shared;
  int row_tiles, splits;
  int64_t chunk;
  size_t workspace;
};

template <typename E, int W, int NQ, bool SH>
static int launch_mask4_one(const Mask4& g, hipStream_t s) {
  const size_t lds = SH ? (size_t)4 * 4 * W * 1024 + 16 : (size_t)4 * NQ * (32 + 2 * W * 4 * 64) * 4;
  if (lds > 65536) QPH_TRY(allow_full_lds((const void*)mask4_kernel<E, W, NQ, SH>));
  const int64_t blocks = (int64_t)g.a.row_tiles * g.a.splits * g.a.heads * g.a.batch;
  hipLaunchKernelGGL((mask4_kernel<E, W, NQ, SH>), dim3((unsigned)blocks), dim3(256), lds, s, g);
  return launch_check("mask4_kernel");
}

template <typename E, int W>
static int launch_mask4_w(const Mask4& g, const Mask4Plan& p, hipStream_t s) {
  if (p.shared) return launch_mask4_one<E, W, 2, true>(g, s);
  if (p.nq == 2) return launch_mask4_one<E, W, 2, false>(g, s);
  return launch_mask4_one<E, W, 1, false>(g, s);
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
