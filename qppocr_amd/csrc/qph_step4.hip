// What a decoder's step needs beside its products and its attention, when it
// checks a tree of drafted tokens over the paged 4-bit cache (qph_fp4.h):
// pages, slots, positions and masks of a batch from its lengths; the rotation
// of queries and keys by their positions; tokens moved inside the cache.
#include <algorithm>

#include "qph_fp4.h"

namespace qph {

typedef unsigned long long u64;

// ------------------------------------------------- pages, slots and masks

struct Extend4 {
  int32_t* table;
  int64_t table_stride;
  int max_pages, shift, batch;
  const int32_t *lens, *news;
  int32_t* ring;
  unsigned ring_n;
  const int64_t* ends;
  int tokens;
  const int32_t* parents;         // or NULL
  int words;
  int32_t *out_lens, *out_starts;
  int64_t *out_slots, *out_ends;
  int32_t* out_positions;
  u64* out_tree;
  int *rows, *takes, *gives;      // a batch of more than kExtendFew: [batch + 1] each
};

// Sequences whose sums every workgroup makes by itself.
constexpr int kExtendItems = 8, kExtendFew = 256 * kExtendItems;

constexpr int kMaxLen = 0x7fffff00;   // as the attention's: positions stay in 31 bits

// A sum that stays at 2^31 - 1 once it is there (terms 0 to 2^31 - 1): the order
// of its additions does not change it.
__device__ __forceinline__ int add_sat(int a, int b) {
  return (int)min((unsigned)a + (unsigned)b, 0x7fffffffu);
}

// The sum of v over the workgroup's earlier threads, and over all (*all).
template <int WAVES>
__device__ __forceinline__ int block_scan(int v, int* part, int* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x = add_sat(x, y);
  }
  int before = __shfl_up(x, 1);
  if (lane == 0) before = 0;
  __syncthreads();                       // (an earlier scan's reads)
  if (lane == 63) part[wave] = x;
  __syncthreads();
  int base = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < WAVES; w++) {
    if (w == wave) base = sum;
    sum = add_sat(sum, part[w]);
  }
  *all = sum;
  return add_sat(base, before);
}

// One sequence: its cached tokens inside what its row of the table can hold, the
// tokens after the step as if it were granted, and the pages of both.
struct Seq4 {
  int len, held, pages;
  int64_t after;
};

__device__ __forceinline__ Seq4 seq4(const Extend4& a, int len, int n) {
  const int64_t room = min((int64_t)a.max_pages << a.shift, (int64_t)kMaxLen);
  Seq4 s;
  s.len = (int)min((int64_t)max(len, 0), room);
  s.after = max((int64_t)s.len + n, (int64_t)0);
  const int round = (1 << a.shift) - 1;
  s.held = (int)(((int64_t)s.len + round) >> a.shift);
  s.pages = (int)((s.after + round) >> a.shift);
  return s;
}

// Sums before each of a thread's ITEMS sequences from `first` on: rows of earlier
// sequences, pages that they take and pages that they give back; from and to the
// sums of the tiles before (carry).
template <int WAVES, int ITEMS>
__device__ __forceinline__ void extend_sums(const Extend4& a, int first, int (&rows)[ITEMS + 1],
                                            int (&takes)[ITEMS + 1], int (&gives)[ITEMS + 1],
                                            int* part, int (&carry)[3]) {
  const int64_t room = min((int64_t)a.max_pages << a.shift, (int64_t)kMaxLen);
  int len[ITEMS], n[ITEMS], all;
#pragma unroll
  for (int i = 0; i < ITEMS; i++) {
    const bool there = first + i < a.batch;
    len[i] = there ? a.lens[first + i] : 0;
    n[i] = there ? a.news[first + i] : 0;
  }
  int sum = 0;
#pragma unroll
  for (int i = 0; i < ITEMS; i++) sum = add_sat(sum, max(n[i], 0));
  rows[0] = add_sat(carry[0], block_scan<WAVES>(sum, part, &all));
  carry[0] = add_sat(carry[0], all);
#pragma unroll
  for (int i = 0; i < ITEMS; i++) rows[i + 1] = add_sat(rows[i], max(n[i], 0));
  takes[0] = gives[0] = 0;
#pragma unroll
  for (int i = 0; i < ITEMS; i++) {
    const Seq4 s = seq4(a, len[i], n[i]);
    const bool fits = n[i] >= 0 && s.after <= room && rows[i + 1] <= a.tokens;
    takes[i + 1] = add_sat(takes[i], fits ? s.pages - s.held : 0);
    gives[i + 1] = add_sat(gives[i], n[i] < 0 ? s.held - s.pages : 0);
  }
  const int t = add_sat(carry[1], block_scan<WAVES>(takes[ITEMS], part, &all));
  carry[1] = add_sat(carry[1], all);
  const int g = add_sat(carry[2], block_scan<WAVES>(gives[ITEMS], part, &all));
  carry[2] = add_sat(carry[2], all);
#pragma unroll
  for (int i = 0; i <= ITEMS; i++) {
    takes[i] = add_sat(t, takes[i]);
    gives[i] = add_sat(g, gives[i]);
  }
}

// Many sequences: their sums by one workgroup, a tile of 1024 x kExtendItems at a
// time, for the launch after it.
__global__ __launch_bounds__(1024) void extend4_sums_kernel(Extend4 a) {
  __shared__ int part[16];
  int carry[3] = {0, 0, 0};
  for (int t0 = 0; t0 < a.batch; t0 += 1024 * kExtendItems) {
    const int first = t0 + threadIdx.x * kExtendItems;
    int r[kExtendItems + 1], t[kExtendItems + 1], g[kExtendItems + 1];
    extend_sums<16, kExtendItems>(a, first, r, t, g, part, carry);
#pragma unroll
    for (int i = 0; i < kExtendItems; i++)
      if (first + i < a.batch) {
        a.rows[first + i] = r[i];
        a.takes[first + i] = t[i];
        a.gives[first + i] = g[i];
      }
  }
  if (threadIdx.x == 0) {
    a.rows[a.batch] = carry[0];
    a.takes[a.batch] = carry[1];
    a.gives[a.batch] = carry[2];
  }
}

// The last i < n with at[i] <= v (at not decreasing, at[0] <= v).
__device__ __forceinline__ int last_at(const int* at, int n, int v) {
  int lo = 0;
  while (n > 1) {
    const int half = n / 2;
    if (at[lo + half] <= v) lo += half;
    n -= half;
  }
  return lo;
}

__device__ __forceinline__ unsigned ring_place(int64_t at, unsigned n) {
  const int64_t r = at % (int64_t)n;
  return (unsigned)(r < 0 ? r + n : r);
}

// Everything of the step but the sums.  A workgroup of a small batch makes the
// sums itself (in LDS): a second launch, or a wait for another workgroup, costs
// more than the few thousand additions.  A row's page comes from the table where
// its sequence had the page before, and else from the ring, not from the entry
// that another thread writes now.  Bound by trips to memory one after the other
// (lengths, sums, a page, its entry, a parent): 48 trees of up to 32 tokens 8.3
// us, 384 prompts of some 940000 tokens in all (11 MB) 12.6.  A path is such a row of
// trips as long as it is deep, 0.19 us each: 48 sequences of 32, 200 and 700 tokens 9,
// 38 and 134 us as chains, 6.5, 7.4 and 9.2 as binary trees; one chain of 16384 3.2 ms.
template <bool FEW>
__global__ __launch_bounds__(256) void extend4_kernel(Extend4 a) {
  __shared__ int lds[FEW ? 3 * (kExtendFew + 1) : 1];
  __shared__ int part[4];
  const int *rows, *takes, *gives;
  if constexpr (FEW) {
    int* w = lds;
    int r[kExtendItems + 1], t[kExtendItems + 1], g[kExtendItems + 1], carry[3] = {0, 0, 0};
    const int first = threadIdx.x * kExtendItems;
    extend_sums<4, kExtendItems>(a, first, r, t, g, part, carry);
#pragma unroll
    for (int i = 0; i < kExtendItems; i++)
      if (first + i < a.batch) {
        w[first + i] = r[i];
        w[kExtendFew + 1 + first + i] = t[i];
        w[2 * (kExtendFew + 1) + first + i] = g[i];
      }
    if (threadIdx.x < 3) w[threadIdx.x * (kExtendFew + 1) + a.batch] = carry[threadIdx.x];
    __syncthreads();
    rows = w; takes = w + kExtendFew + 1; gives = w + 2 * (kExtendFew + 1);
  } else {
    rows = a.rows; takes = a.takes; gives = a.gives;
  }
  const int64_t room = min((int64_t)a.max_pages << a.shift, (int64_t)kMaxLen);
  const int64_t head = a.ends[0], tail = a.ends[1];
  // (a difference that wraps is no count either)
  const int64_t left = (int64_t)((u64)tail - (u64)head);
  const int free = (int)min(max(left, (int64_t)0), (int64_t)a.ring_n);
  const unsigned head_at = ring_place(head, a.ring_n), tail_at = ring_place(tail, a.ring_n);
  const unsigned all = gridDim.x * 256, id = blockIdx.x * 256 + threadIdx.x;
  // (pages given back that the ring has no room for are dropped: none overwrites one
  // that is taken now)
  const int taken_most = takes[a.batch], given = min(gives[a.batch], (int)a.ring_n - free);
  auto ring_index = [&](unsigned at, unsigned i) {     // i < ring_n
    const unsigned p = at + i;
    return p >= a.ring_n ? p - a.ring_n : p;
  };
  // a sequence's pages are granted where all up to its last are there
  auto granted = [&](int b, int n, const Seq4& s) {
    const int take = takes[b + 1] - takes[b];
    return n >= 0 && s.after <= room && rows[b + 1] <= a.tokens &&
           (take == 0 || takes[b + 1] <= free);
  };

  // sequences: the starts of their rows, their lengths after the step
  for (unsigned b = id; b <= (unsigned)a.batch; b += all) {
    a.out_starts[b] = min(rows[b], a.tokens);
    if (b == (unsigned)a.batch) continue;
    const int n = a.news[b];
    const Seq4 s = seq4(a, a.lens[b], n);
    a.out_lens[b] = n < 0 || granted(b, n, s) ? (int)s.after : s.len;
  }
  if (id == 0) {
    // the pages taken: those of the sequences up to the last that is granted some
    int taken = taken_most;
    if (taken > free) taken = takes[last_at(takes, a.batch + 1, free)];
    a.out_ends[0] = (int64_t)((u64)head + (u64)taken);
    a.out_ends[1] = (int64_t)((u64)tail + (u64)given);
  }

  // pages taken, into the table; pages given back, into the ring
  for (unsigned t = id; t < (unsigned)min(taken_most, free); t += all) {
    const int b = last_at(takes, a.batch, (int)t);
    const Seq4 s = seq4(a, a.lens[b], a.news[b]);
    if (takes[b + 1] > free) continue;
    a.table[b * a.table_stride + s.held + ((int)t - takes[b])] = a.ring[ring_index(head_at, t)];
  }
  for (unsigned t = id; t < (unsigned)given; t += all) {
    const int b = last_at(gives, a.batch, (int)t);
    const Seq4 s = seq4(a, a.lens[b], a.news[b]);
    a.ring[ring_index(tail_at, t)] = a.table[b * a.table_stride + s.pages + ((int)t - gives[b])];
  }

  // rows
  const int mask = (1 << a.shift) - 1, last = min(rows[a.batch], a.tokens);
  for (unsigned r = id; r < (unsigned)a.tokens; r += all) {
    int64_t slot = -1;
    int position = 0, i = -1, b = 0;
    if ((int)r < last) {
      b = last_at(rows, a.batch, (int)r);
      i = (int)r - rows[b];
      const int n = a.news[b];
      const Seq4 s = seq4(a, a.lens[b], n);
      const int64_t at = (int64_t)s.len + i;
      position = (int)min(at, (int64_t)INT32_MAX);
      if (granted(b, n, s)) {
        const int column = (int)(at >> a.shift);
        const int page = column < s.held
                             ? a.table[b * a.table_stride + column]
                             : a.ring[ring_index(head_at, takes[b] + (column - s.held))];
        if (page >= 0) slot = ((int64_t)page << a.shift) + (at & mask);
      }
      if (a.parents) {
        // the path to the context, from the row up: each parent stands before its
        // child (else the child is a root), so the walk ends
        u64* out = a.out_tree + (int64_t)r * a.words;
        const int32_t* up = a.parents + rows[b];
        int at_word = a.words, depth = 0, k = i;
        u64 bits = 0;
        while (true) {
          if (k >> 6 != at_word) {
            if (at_word < a.words) out[at_word] = bits;
            for (int w = min(at_word, a.words) - 1; w > k >> 6; w--) out[w] = 0;
            at_word = k >> 6;
            bits = 0;
          }
          bits |= 1ull << (k & 63);
          depth++;
          const int p = up[k];
          if (p < 0 || p >= k) break;
          k = p;
        }
        if (at_word < a.words) out[at_word] = bits;
        for (int w = min(at_word, a.words) - 1; w >= 0; w--) out[w] = 0;
        position = (int)min((int64_t)s.len + depth - 1, (int64_t)INT32_MAX);
      }
    } else if (a.parents) {
      for (int w = 0; w < a.words; w++) a.out_tree[(int64_t)r * a.words + w] = 0;
    }
    a.out_slots[r] = slot;
    a.out_positions[r] = position;
  }
}

static int launch_extend4(const Extend4& a, hipStream_t s) {
  const bool few = a.batch <= kExtendFew;
  if (!few) {
    hipLaunchKernelGGL(extend4_sums_kernel, dim3(1), dim3(1024), 0, s, a);
    QPH_TRY(launch_check("extend4_sums_kernel"));
  }
  const int64_t items = std::max<int64_t>(a.tokens, a.batch + 1);
  const dim3 grid((unsigned)std::min<int64_t>((items + 255) / 256, 1024));
  if (few) hipLaunchKernelGGL(extend4_kernel<true>, grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(extend4_kernel<false>, grid, dim3(256), 0, s, a);
  return launch_check("extend4_kernel");
}

// ------------------------------------------------------------- rotation

struct Rotary {
  const void* x;
  void* out;
  int64_t xt, xh, ot, oh;         // strides of a token and a head
  int64_t tokens;
  int heads, dh;
  const void* pos;
  int pos64;
  int64_t pt, pa;                 // strides of a token and an axis
  int n_axes;
  const u64* turns;
  const int32_t* axes;
  int pairs, neighbours, inverse;
  int each, groups;               // heads a thread, threads along the heads
  int chunks, all_chunks;         // of V pairs; and of 2 V elements that stay
};

// cos and sin of the angle of `phase` 2^-64 turns.  The turn's quarter nearest to it
// is taken off in whole numbers, the rest (at most pi / 4) goes into the series of
// sine and cosine, whose first terms left out are below 2^-28.
__device__ __forceinline__ void cos_sin(u64 phase, float* c, float* s) {
  const unsigned quarter = (unsigned)((phase + (1ull << 61)) >> 62);
  const int64_t rest = (int64_t)(phase - ((u64)quarter << 62));
  // (two parts: the low one matters where the angle is small)
  const float t = __builtin_fmaf((float)(int)(rest >> 32), 0x1p-32f, (float)(unsigned)rest * 0x1p-64f);
  const float x = t * 6.283185307179586f, z = x * x;
  float p = 1.0f / 362880.0f;
  p = __builtin_fmaf(p, z, -1.0f / 5040.0f);
  p = __builtin_fmaf(p, z, 1.0f / 120.0f);
  p = __builtin_fmaf(p, z, -1.0f / 6.0f);
  const float sn = __builtin_fmaf(x * z, p, x);
  float q = -1.0f / 3628800.0f;
  q = __builtin_fmaf(q, z, 1.0f / 40320.0f);
  q = __builtin_fmaf(q, z, -1.0f / 720.0f);
  q = __builtin_fmaf(q, z, 1.0f / 24.0f);
  q = __builtin_fmaf(q, z, -0.5f);
  const float cs = __builtin_fmaf(q, z, 1.0f);
  const bool odd = quarter & 1;
  const float a = odd ? sn : cs, b = odd ? cs : sn;
  *c = (quarter + 1) & 2 ? -a : a;
  *s = quarter & 2 ? -b : b;
}

// A thread has V pairs of a token, computes their cosines and sines once and turns
// them in `each` heads.  The position times the turns a position, in 2^-64ths, is
// exact modulo a turn in 64 bits, however far the position.  Bound by memory: 20011
// tokens of 40 heads of 128 in bfloat16 (410 MB) 97 us, 4.2 TB/s where a large copy
// runs at 4.6; 32 tokens of them 5.0 us, a launch and two trips to memory.
template <typename E, int V, bool NB>
__global__ __launch_bounds__(256) void rotary_kernel(Rotary a) {
  typedef typename E::type T;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t rest = id / a.all_chunks;
  const int chunk = (int)(id - rest * a.all_chunks);
  const int64_t token = rest / a.groups;
  if (token >= a.tokens) return;
  const int h0 = (int)(rest - token * a.groups) * a.each, h1 = min(h0 + a.each, a.heads);
  const T* x = (const T*)a.x + token * a.xt;
  T* y = (T*)a.out + token * a.ot;
  if (chunk >= a.chunks) {
    // elements that are not turned
    const int d0 = 2 * a.pairs + (chunk - a.chunks) * 2 * V, n = min(2 * V, a.dh - d0);
    for (int h = h0; h < h1; h++) {
      if (n == 2 * V) {
        T t[2 * V];
        __builtin_memcpy(t, x + h * a.xh + d0, sizeof t);
        __builtin_memcpy(y + h * a.oh + d0, t, sizeof t);
      } else {
        for (int i = 0; i < n; i++) y[h * a.oh + d0 + i] = x[h * a.xh + d0 + i];
      }
    }
    return;
  }
  const int p0 = chunk * V, n = min(V, a.pairs - p0);
  float c[V], s[V];
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int p = min(p0 + i, a.pairs - 1);
    const int axis = min(max(a.axes[p], 0), a.n_axes - 1);
    const int64_t at = token * a.pt + axis * a.pa;
    const int64_t pos = a.pos64 ? ((const int64_t*)a.pos)[at] : ((const int32_t*)a.pos)[at];
    cos_sin((u64)pos * a.turns[p], &c[i], &s[i]);
    if (a.inverse) s[i] = -s[i];
  }
  if (n == V) {
#pragma unroll 2
    for (int h = h0; h < h1; h++) {
      const T* xa = x + h * a.xh + (NB ? 2 * p0 : p0);
      T* ya = y + h * a.oh + (NB ? 2 * p0 : p0);
      T in[2 * V], res[2 * V];
      __builtin_memcpy(in, xa, V * sizeof(T));
      __builtin_memcpy(in + V, xa + (NB ? V : a.pairs), V * sizeof(T));
#pragma unroll
      for (int i = 0; i < V; i++) {
        const float u = (float)in[NB ? 2 * i : i], v = (float)in[NB ? 2 * i + 1 : V + i];
        res[NB ? 2 * i : i] = (T)__builtin_fmaf(u, c[i], -(v * s[i]));
        res[NB ? 2 * i + 1 : V + i] = (T)__builtin_fmaf(u, s[i], v * c[i]);
      }
      __builtin_memcpy(ya, res, V * sizeof(T));
      __builtin_memcpy(ya + (NB ? V : a.pairs), res + V, V * sizeof(T));
    }
  } else {
    for (int h = h0; h < h1; h++)
#pragma unroll
      for (int i = 0; i < V; i++) {
        if (i >= n) break;
        const int da = NB ? 2 * (p0 + i) : p0 + i, db = NB ? da + 1 : da + a.pairs;
        const float u = (float)x[h * a.xh + da], v = (float)x[h * a.xh + db];
        y[h * a.oh + da] = (T)__builtin_fmaf(u, c[i], -(v * s[i]));
        y[h * a.oh + db] = (T)__builtin_fmaf(u, s[i], v * c[i]);
      }
  }
}

template <typename E>
static int launch_rotary(Rotary a, hipStream_t s) {
  constexpr int V = sizeof(typename E::type) == 2 ? 8 : 4;
  a.chunks = (a.pairs + V - 1) / V;
  // what is not turned is copied, unless it stands where it stays
  a.all_chunks = a.chunks + (a.out == a.x ? 0 : (a.dh - 2 * a.pairs + 2 * V - 1) / (2 * V));
  const int64_t waves = (a.tokens * a.all_chunks + 63) / 64;
  a.groups = (int)std::clamp<int64_t>(8192 / waves, 1, a.heads);
  a.each = (a.heads + a.groups - 1) / a.groups;
  a.groups = (a.heads + a.each - 1) / a.each;
  const int64_t blocks = (a.tokens * a.groups * a.all_chunks + 255) / 256;
  if (blocks > kMaxGroups) return fail(QPH_EUNSUPPORTED, "rotary: too many tokens for one call");
  const dim3 grid((unsigned)blocks);
  if (a.neighbours) hipLaunchKernelGGL((rotary_kernel<E, V, true>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((rotary_kernel<E, V, false>), grid, dim3(256), 0, s, a);
  return launch_check("rotary_kernel");
}

// ---------------------------------------------------------------- moves

struct Move4 {
  unsigned char *codes[2], *scales[2];
  int64_t slots_n;
  int shift;
  unsigned heads, blocks;         // blocks of a head: dh / 32
  const int64_t *src, *dst;
  int64_t tokens;
  u32x4* held_codes;              // of the two launches: [token][2][heads][blocks]
  unsigned char* held_scales;
};

__device__ __forceinline__ bool move_there(const Move4& a, int64_t src, int64_t dst) {
  return src >= 0 && src < a.slots_n && dst >= 0 && dst < a.slots_n;
}

// A token's block (16 bytes of codes and a scale) of the keys or values of a head.
__device__ __forceinline__ int64_t move_block(const Move4& a, int64_t slot, unsigned h, unsigned c) {
  const int64_t mask = ((int64_t)1 << a.shift) - 1;
  return ((((slot >> a.shift) * a.heads + h) << a.shift) + (slot & mask)) * a.blocks + c;
}

// A few tokens: a workgroup has all of them for its head's keys or values, reads
// all, then writes all, so that a place may be left and taken in one call.  (190
// tokens of 8 heads of 128: 2.8 us, a launch and three trips to memory.)
template <int U>
__global__ __launch_bounds__(1024) void move4_few_kernel(Move4 a) {
  const unsigned h = blockIdx.x >> 1, second = blockIdx.x & 1;
  const unsigned char *codes = a.codes[second], *scales = a.scales[second];
  const unsigned total = (unsigned)a.tokens * a.blocks;
  u32x4 code[U];
  unsigned char scale[U];
  int64_t to[U];
#pragma unroll
  for (int i = 0; i < U; i++) {
    const unsigned u = threadIdx.x + i * blockDim.x;
    to[i] = -1;
    if (u >= total) continue;
    const unsigned t = u / a.blocks, c = u % a.blocks;
    const int64_t src = a.src[t], dst = a.dst[t];
    if (!move_there(a, src, dst)) continue;
    const int64_t from = move_block(a, src, h, c);
    to[i] = move_block(a, dst, h, c);
    code[i] = ((const u32x4*)codes)[from];
    scale[i] = scales[from];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < U; i++)
    if (to[i] >= 0) {
      ((u32x4*)a.codes[second])[to[i]] = code[i];
      a.scales[second][to[i]] = scale[i];
    }
}

// Many tokens: out of the cache into the workspace, and in another launch back.
// (16001 tokens of 8 heads of 128, 35 MB read and written twice: 10.0 and 8.9 us.)
template <bool BACK>
__global__ __launch_bounds__(256) void move4_many_kernel(Move4 a) {
  const unsigned units = 2 * a.heads * a.blocks;
  const int64_t total = a.tokens * units;
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < total; u += (int64_t)gridDim.x * 256) {
    const int64_t t = u / units;
    unsigned w = (unsigned)(u - t * units);
    const unsigned second = w >= a.heads * a.blocks;
    if (second) w -= a.heads * a.blocks;
    const unsigned h = w / a.blocks, c = w % a.blocks;
    const int64_t src = a.src[t], dst = a.dst[t];
    if (!move_there(a, src, dst)) continue;
    const int64_t at = move_block(a, BACK ? dst : src, h, c);
    if (BACK) {
      ((u32x4*)a.codes[second])[at] = a.held_codes[u];
      a.scales[second][at] = a.held_scales[u];
    } else {
      a.held_codes[u] = ((const u32x4*)a.codes[second])[at];
      a.held_scales[u] = a.scales[second][at];
    }
  }
}

// Blocks of a head that a workgroup holds in its registers (4 each of 1024 threads).
static bool move4_few(const qph_cache4* c, int64_t tokens) {
  return tokens * (c->dh / 32) <= 4 * 1024;
}

static size_t move4_workspace(const qph_cache4* c, int64_t tokens) {
  if (move4_few(c, tokens)) return 0;
  return (size_t)tokens * 2 * c->heads * (c->dh / 32) * 17;
}

}  // namespace qph

using namespace qph;

extern "C" {

QPH_API int qph_cache4_extend_workspace(int64_t batch, size_t* bytes) {
  if (!bytes) return fail(QPH_EINVAL, "cache4_extend_workspace: NULL argument");
  *bytes = 0;
  if (batch < 0) return fail(QPH_EINVAL, "cache4_extend: negative size");
  if (batch > kExtendFew) *bytes = (size_t)(batch + 1) * 12;
  return QPH_OK;
}

QPH_API int qph_cache4_extend(qph_ctx* ctx, const qph_extend4* p) {
  if (!p) return fail(QPH_EINVAL, "cache4_extend: NULL arguments");
  if (p->batch < 0 || p->max_pages < 0 || p->tokens < 0 || p->ring_n < 0 || p->tree_words < 0)
    return fail(QPH_EINVAL, "cache4_extend: negative size");
  if (p->page_size < 16 || p->page_size > 32768 || (p->page_size & (p->page_size - 1)))
    return fail(QPH_EUNSUPPORTED, "cache4_extend: page size " + std::to_string(p->page_size) +
                                      " is no power of two from 16 to 32768");
  if (p->batch > (1 << 24) || p->tokens > (1 << 30) || p->ring_n > INT32_MAX || p->max_pages > INT32_MAX ||
      (p->batch && p->max_pages > INT32_MAX / p->batch))
    return fail(QPH_EUNSUPPORTED, "cache4_extend: more than 2^24 sequences, 2^30 rows or 2^31 - 1 pages");
  if (!p->out_starts || !p->out_ends || !p->ends || (p->batch && (!p->lens || !p->news || !p->out_lens)) ||
      (p->batch && p->max_pages && !p->page_table) || (p->ring_n && !p->ring) ||
      (p->tokens && (!p->out_slots || !p->out_positions)))
    return fail(QPH_EINVAL, "cache4_extend: NULL argument");
  if (p->ring_n == 0) return fail(QPH_EINVAL, "cache4_extend: empty ring");
  if (p->batch > 1 && p->table_stride < p->max_pages)
    return fail(QPH_EINVAL, "cache4_extend: rows of the page table overlap");
  if (p->parents && p->tokens && (!p->out_tree || p->tree_words == 0))
    return fail(QPH_EINVAL, "cache4_extend: parents without masks to write");
  if (p->tree_words > (1 << 20)) return fail(QPH_EUNSUPPORTED, "cache4_extend: masks of more than 2^20 words");
  size_t bytes = 0;
  QPH_TRY(qph_cache4_extend_workspace(p->batch, &bytes));
  if (bytes && (!p->workspace || p->workspace_bytes < bytes))
    return fail(QPH_EINVAL, "cache4_extend: workspace of " + std::to_string(p->workspace_bytes) +
                                " bytes, needs " + std::to_string(bytes));
  if (!ctx) return fail(QPH_EINVAL, "null context");
  Extend4 a{};
  a.table = p->page_table; a.table_stride = p->table_stride;
  a.max_pages = (int)p->max_pages;
  a.shift = __builtin_ctz((unsigned)p->page_size);
  a.batch = (int)p->batch;
  a.lens = p->lens; a.news = p->news;
  a.ring = p->ring; a.ring_n = (unsigned)p->ring_n;
  a.ends = p->ends;
  a.tokens = (int)p->tokens;
  a.parents = p->parents;
  a.words = (int)p->tree_words;
  a.out_lens = p->out_lens; a.out_starts = p->out_starts;
  a.out_slots = p->out_slots; a.out_ends = p->out_ends;
  a.out_positions = p->out_positions;
  a.out_tree = (u64*)p->out_tree;
  a.rows = (int*)p->workspace;
  a.takes = a.rows + p->batch + 1;
  a.gives = a.takes + p->batch + 1;
  OnDevice dev(ctx);
  QPH_TRY(dev.rc());
  return launch_extend4(a, ctx->stream);
}

QPH_API int qph_rotary(qph_ctx* ctx, const qph_rotary_args* p) {
  if (!p) return fail(QPH_EINVAL, "rotary: NULL arguments");
  if (!dtype_valid(p->dtype)) return fail(QPH_EINVAL, "rotary: unknown element type");
  if (p->tokens < 0 || p->heads < 0) return fail(QPH_EINVAL, "rotary: negative size");
  if (p->dh <= 0 || p->pairs <= 0 || p->pairs > p->dh / 2 || p->n_axes <= 0)
    return fail(QPH_EINVAL, "rotary: " + std::to_string(p->pairs) + " pairs of a head of " +
                                std::to_string(p->dh) + ", " + std::to_string(p->n_axes) + " axes");
  if (p->dh > (1 << 20) || p->heads > (1 << 20))
    return fail(QPH_EUNSUPPORTED, "rotary: more than 2^20 heads or elements of a head");
  const bool none = p->tokens == 0 || p->heads == 0;
  if (!none && (!p->x || !p->out || !p->positions || !p->turns || !p->axes))
    return fail(QPH_EINVAL, "rotary: NULL argument");
  if (!none && p->x == p->out && (p->x_strides[0] != p->out_strides[0] || p->x_strides[1] != p->out_strides[1]))
    return fail(QPH_EINVAL, "rotary: out is x with other strides");
  if (p->tokens > ((int64_t)1 << 40)) return fail(QPH_EUNSUPPORTED, "rotary: too many tokens for one call");
  if (!ctx) return fail(QPH_EINVAL, "null context");
  if (none) return QPH_OK;
  Rotary a{};
  a.x = p->x; a.out = p->out;
  a.xt = p->x_strides[0]; a.xh = p->x_strides[1];
  a.ot = p->out_strides[0]; a.oh = p->out_strides[1];
  a.tokens = p->tokens;
  a.heads = p->heads; a.dh = p->dh;
  a.pos = p->positions; a.pos64 = p->positions_64 != 0;
  a.pt = p->position_strides[1]; a.pa = p->position_strides[0];
  a.n_axes = p->n_axes;
  a.turns = (const u64*)p->turns; a.axes = p->axes;
  a.pairs = p->pairs; a.neighbours = p->neighbours != 0; a.inverse = p->inverse != 0;
  OnDevice dev(ctx);
  QPH_TRY(dev.rc());
  if (p->dtype == QPH_F32) return launch_rotary<F32>(a, ctx->stream);
  if (p->dtype == QPH_F16) return launch_rotary<F16>(a, ctx->stream);
  return launch_rotary<BF16>(a, ctx->stream);
}

QPH_API int qph_cache4_move_workspace(const qph_cache4* cache, int64_t tokens, size_t* bytes) {
  if (!bytes) return fail(QPH_EINVAL, "cache4_move_workspace: NULL argument");
  *bytes = 0;
  int shift = 0;
  QPH_TRY(cache4_check(cache, "cache4_move", &shift));
  if (tokens < 0) return fail(QPH_EINVAL, "cache4_move: negative token count");
  if (tokens > ((int64_t)1 << 31)) return fail(QPH_EUNSUPPORTED, "cache4_move: more than 2^31 tokens");
  *bytes = move4_workspace(cache, tokens);
  return QPH_OK;
}

QPH_API int qph_cache4_move(qph_ctx* ctx, const qph_cache4* cache, const int64_t* src,
                            const int64_t* dst, int64_t tokens, void* workspace,
                            size_t workspace_bytes) {
  size_t bytes = 0;
  QPH_TRY(qph_cache4_move_workspace(cache, tokens, &bytes));
  if (tokens && (!src || !dst)) return fail(QPH_EINVAL, "cache4_move: NULL argument");
  if (bytes && (!workspace || workspace_bytes < bytes))
    return fail(QPH_EINVAL, "cache4_move: workspace of " + std::to_string(workspace_bytes) +
                                " bytes, needs " + std::to_string(bytes));
  if ((uintptr_t)workspace % 16) return fail(QPH_EINVAL, "cache4_move: workspace is not 16-byte aligned");
  if (!ctx) return fail(QPH_EINVAL, "null context");
  if (tokens == 0) return QPH_OK;
  Move4 a{};
  a.codes[0] = (unsigned char*)cache->k_codes; a.scales[0] = (unsigned char*)cache->k_scales;
  a.codes[1] = (unsigned char*)cache->v_codes; a.scales[1] = (unsigned char*)cache->v_scales;
  a.shift = __builtin_ctz((unsigned)cache->page_size);
  a.slots_n = cache->n_pages << a.shift;
  a.heads = (unsigned)cache->heads;
  a.blocks = (unsigned)cache->dh / 32;
  a.src = src; a.dst = dst;
  a.tokens = tokens;
  OnDevice dev(ctx);
  QPH_TRY(dev.rc());
  if (move4_few(cache, tokens)) {
    const unsigned total = (unsigned)tokens * a.blocks;
    const dim3 grid(2 * a.heads);
    if (total <= 1024)
      hipLaunchKernelGGL(move4_few_kernel<1>, grid, dim3((total + 63) / 64 * 64), 0, ctx->stream, a);
    else hipLaunchKernelGGL(move4_few_kernel<4>, grid, dim3(1024), 0, ctx->stream, a);
    return launch_check("move4_few_kernel");
  }
  a.held_codes = (u32x4*)workspace;
  a.held_scales = (unsigned char*)workspace + (size_t)tokens * 2 * a.heads * a.blocks * 16;
  const int64_t blocks = (tokens * 2 * a.heads * a.blocks + 255) / 256;
  const dim3 grid((unsigned)std::min<int64_t>(blocks, kMaxGroups));
  hipLaunchKernelGGL(move4_many_kernel<false>, grid, dim3(256), 0, ctx->stream, a);
  QPH_TRY(launch_check("move4_many_kernel"));
  hipLaunchKernelGGL(move4_many_kernel<true>, grid, dim3(256), 0, ctx->stream, a);
  return launch_check("move4_many_kernel");
}

}  // extern "C"
