// 4-bit weights and caches: quantising, the cache's writes and reads, and the
// linear over 4-bit weights.  The format and its arithmetic: qph_fp4.h.
#include <algorithm>
#include <cmath>

#include "qph_fp4.h"

namespace qph {

// ---------------------------------------------------------------- quantise

struct Quant4 {
  const void* x;
  int64_t rows, k, rs, cs;    // element (r, i) at x[r * rs + i * cs]
  int64_t groups;             // blocks of 32 a row, those past k zero
  unsigned char* codes;
  unsigned char* scales;
};

// A block of 32 per thread.  Neighbouring threads take neighbouring blocks of
// a row, or (BYROW, elements of a row apart in memory) neighbouring rows, so
// that the loads of a wave touch whole lines.  Weights are packed once.
template <typename E, bool BYROW>
__global__ __launch_bounds__(256) void quantize4_kernel(Quant4 a) {
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (u >= a.rows * a.groups) return;
  const int64_t r = BYROW ? u % a.rows : u / a.groups;
  const int64_t g = BYROW ? u / a.rows : u % a.groups;
  const typename E::type* x = (const typename E::type*)a.x + r * a.rs;
  float v[32];
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 32; i++) {
    const int64_t k = g * 32 + i;
    v[i] = k < a.k ? (float)x[k * a.cs] : 0.0f;
    top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  }
  const int e = fp4_exponent(top);
  const bool bad = e == -1000;
  const float scale = scale_of_byte((unsigned)(bad ? 127 : e + 127));
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; i++) w[i] = bad ? 0u : fp4_encode8(v + 8 * i, scale);
  *(u32x4*)(a.codes + (r * a.groups + g) * 16) = w;
  a.scales[r * a.groups + g] = (unsigned char)(bad ? 255 : e + 127);
}

// ------------------------------------------------------------------- cache

struct Cache4Io {
  unsigned char *kc, *ks, *vc, *vs;
  int64_t slots_n;            // n_pages << shift
  int shift;
  unsigned heads, words;      // words of eight elements a head
  const int64_t* slots;
  int64_t tokens;
  void *k, *v;
  int64_t kt, kh, vt, vh;     // strides of a token and a head, in elements
  int per;                    // tokens a workgroup takes at once
};

// Where head h of a cached token starts, in heads' rows.
__device__ __forceinline__ int64_t cache4_row(int64_t slot, int shift, unsigned heads, unsigned h) {
  return ((((slot >> shift) * heads + h) << shift) + (slot & (((int64_t)1 << shift) - 1)));
}

// A word of codes (eight elements) per thread and token; the four threads of a
// block of 32 share its largest magnitude by two swaps inside a quad (a quad is
// of one token).  Bound by memory; more tokens in flight a thread gain nothing,
// the stores need no answer (four against one: 65521 tokens of 8 x 128 bfloat16
// 83 and 75 us, 262144 334 and 301, 300000 of 1 x 64 21.3 and 20.6).
template <typename E>
__global__ __launch_bounds__(256) void cache4_write_kernel(Cache4Io a) {
  const unsigned units = a.heads * a.words, total = units * (unsigned)a.per;
  const bool second = blockIdx.y != 0;
  const typename E::type* x = (const typename E::type*)(second ? a.v : a.k);
  const int64_t xt = second ? a.vt : a.kt, xh = second ? a.vh : a.kh;
  unsigned char* codes = second ? a.vc : a.kc;
  unsigned char* scales = second ? a.vs : a.ks;
  for (unsigned u = threadIdx.x; u < total; u += blockDim.x) {
    const unsigned lt = u / units, w = u % units, h = w / a.words, c = w % a.words;
    const int64_t t = (int64_t)blockIdx.x * a.per + lt;
    int64_t slot = -1;
    float v[8];
    if (t < a.tokens) {
      // (both at once: behind the slot's check the row would wait for it)
      slot = a.slots[t];
      load8<E>(x + t * xt + h * xh + c * 8, v);
    }
    if (slot < 0 || slot >= a.slots_n) continue;
    unsigned top = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
    top = max(top, (unsigned)__builtin_amdgcn_mov_dpp((int)top, 0xB1, 0xf, 0xf, true));  // lane ^ 1
    top = max(top, (unsigned)__builtin_amdgcn_mov_dpp((int)top, 0x4E, 0xf, 0xf, true));  // lane ^ 2
    const int e = fp4_exponent(top);
    const bool bad = e == -1000;
    const int64_t row = cache4_row(slot, a.shift, a.heads, h);
    ((unsigned*)codes)[row * a.words + c] =
        bad ? 0u : fp4_encode8(v, scale_of_byte((unsigned)(e + 127)));
    if (c % 4 == 0) scales[row * (a.words / 4) + c / 4] = (unsigned char)(bad ? 255 : e + 127);
  }
}

// A word of codes per thread and token, U tokens (per * U a workgroup) in
// flight: the slots, then the codes and scales, then the rows.
template <typename E, int U>
__global__ __launch_bounds__(256) void cache4_read_kernel(Cache4Io a) {
  const unsigned units = a.heads * a.words, total = units * (unsigned)a.per;
  const bool second = blockIdx.y != 0;
  typename E::type* y = (typename E::type*)(second ? a.v : a.k);
  const int64_t yt = second ? a.vt : a.kt, yh = second ? a.vh : a.kh;
  const unsigned char* codes = second ? a.vc : a.kc;
  const unsigned char* scales = second ? a.vs : a.ks;
  for (unsigned u = threadIdx.x; u < total; u += blockDim.x) {
    const unsigned lt = u / units, w = u % units, h = w / a.words, c = w % a.words;
    const int64_t t0 = (int64_t)blockIdx.x * (a.per * U) + lt;
    int64_t row[U];
#pragma unroll
    for (int i = 0; i < U; i++) {
      const int64_t slot = a.slots[min(t0 + i * a.per, a.tokens - 1)];
      row[i] = slot < 0 || slot >= a.slots_n ? -1 : cache4_row(slot, a.shift, a.heads, h);
    }
    unsigned code[U], scale[U];
#pragma unroll
    for (int i = 0; i < U; i++) {
      const int64_t r = max(row[i], (int64_t)0);
      code[i] = ((const unsigned*)codes)[r * a.words + c];
      scale[i] = scales[r * (a.words / 4) + c / 4];
    }
#pragma unroll
    for (int i = 0; i < U; i++) {
      const int64_t t = t0 + i * a.per;
      if (t >= a.tokens) break;
      const bf16x8 b = fp4_word(row[i] < 0 ? 0u : code[i], scale_of_byte(row[i] < 0 ? 127u : scale[i]));
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = (float)b[e];
      store8<E>(y + t * yt + h * yh + c * 8, v);
    }
  }
}

// ------------------------------------------------------------------ linear

struct Lin4 {
  const void* x; int64_t xs;            // row stride of x
  const unsigned char* codes;
  const unsigned char* scales;
  const void* bias;
  const void* res;
  void* y;
  int64_t rows, k, n;
  int64_t chunks;                       // k in chunks of 128
  Act act;
};

// GELU through erfc: (c3 v) (c2 + erf(v / c1)) without the cancellation of
// 1 + erf for negative v.
__device__ __forceinline__ float act4_apply(float v, const Act& a) {
  if (a.kind == 1) return a.c3 * v * ((a.c2 - 1.0f) + erfcf(-v * a.inv_c1));
  return act_apply(v, a);
}

// A block whose numbers are exact in float16: scale bytes 104 to 140 (6 2^13
// to half of 2^-23), or all codes zero.
__device__ __forceinline__ bool fits_f16(unsigned s, u32x4 w) {
  return s - 104u <= 36u || (s < 104u && ((w[0] | w[1] | w[2] | w[3]) & 0x77777777u) == 0);
}

// y[r][j] = act(sum_k x[r][k] W[j][k] + bias[j]) + res[r][j], on MFMAs whose
// rows are 16 columns j and whose columns are 16 rows r.  A lane holds 32
// neighbouring k of one column, one block: 16 bytes of codes and one scale, so
// it needs the 32 neighbouring elements of a row of x beside them.  x comes in
// whole lines and is turned in LDS; straight from memory each load would touch
// 64 lines (an early form, 32 rows of 4096 x 12288: 41 us so, 24 through LDS).  float16 x
// against weights that are exact in float16 (any of ordinary size) is one
// float16 product of full precision, otherwise x is split into bfloat16 terms.

// 16 bytes of a row of x from element k of it on; past the end of the row zeros.
template <typename E>
__device__ __forceinline__ u32x4 x_piece(const typename E::type* row, int64_t k, int64_t end) {
  constexpr int elems = 16 / sizeof(typename E::type);
  u32x4 v = {0, 0, 0, 0};
  if (k + elems <= end) {
    __builtin_memcpy(&v, row + k, 16);
  } else if (k < end) {
    typename E::type t[elems];
#pragma unroll
    for (int i = 0; i < elems; i++) t[i] = k + i < end ? row[k + i] : (typename E::type)0.0f;
    __builtin_memcpy(&v, t, 16);
  }
  return v;
}

// The lane's scale out of its column's four, into the exponent's place: the
// conversions read nothing else of that operand.
__device__ __forceinline__ float lane_scale(unsigned four, int kg) {
  return __uint_as_float(__builtin_amdgcn_alignbit(four, four, (8 * kg + 9) & 31));
}

// The products of a chunk: w and four a lane's 32 codes and its column's four
// scales for each of NT column tiles, part(m, xf) the lane's 32 elements of x,
// eight at a time, for each of NQ row tiles.  TS terms: the bfloat16 terms, or
// with float16 the elements themselves.
template <typename E, int NQ, int NT, int TS, typename Part>
__device__ __forceinline__ void chunk_products(const u32x4* w, const unsigned* four, int kg,
                                               Part part, f32x4 (&acc)[NT][NQ]) {
  float sc[NT];
#pragma unroll
  for (int i = 0; i < NT; i++) sc[i] = lane_scale(four[i], kg);
  bool f16 = false;
  if constexpr (E::terms == 2) {
    bool fits = true;
#pragma unroll
    for (int i = 0; i < NT; i++) fits &= fits_f16(four[i] >> (8 * kg) & 255, w[i]);
    f16 = __all(fits);
  }
  if (E::terms == 2 && f16) {
#pragma unroll
    for (int m = 0; m < 4; m++) {
      u32x4 x[NQ][TS];
      part(m, x);
#pragma unroll
      for (int i = 0; i < NT; i++) {
        const f16x8 wf = fp4_word_f16(w[i][m], sc[i]);
#pragma unroll
        for (int q = 0; q < NQ; q++)
          acc[i][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf, __builtin_bit_cast(f16x8, x[q][0]),
                                                             acc[i][q], 0, 0, 0);
      }
    }
  } else {
#pragma unroll
    for (int m = 0; m < 4; m++) {
      u32x4 x[NQ][TS];
      bf16x8 xf[NQ][E::terms];
      part(m, x);
#pragma unroll
      for (int q = 0; q < NQ; q++) {
        if constexpr (E::terms == 2) {
          const f16x8 h = __builtin_bit_cast(f16x8, x[q][0]);
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; e++) v[e] = (float)h[e];
          split8<2>(v, xf[q]);
        } else {
#pragma unroll
          for (int t = 0; t < TS; t++) xf[q][t] = __builtin_bit_cast(bf16x8, x[q][t]);
        }
      }
#pragma unroll
      for (int i = 0; i < NT; i++) {
        const bf16x8 wf = fp4_word(w[i][m], sc[i]);
#pragma unroll
        for (int t = E::terms - 1; t >= 0; t--)
#pragma unroll
          for (int q = 0; q < NQ; q++) acc[i][q] = mfma16(wf, xf[q][t], acc[i][q]);
      }
    }
  }
}

// Four neighbouring columns' results.
template <typename E>
__device__ __forceinline__ void linear4_store(const Lin4& a, int64_t r, int64_t j, f32x4 v) {
  typedef typename E::type T;
  if (r >= a.rows || j >= a.n) return;
  const T* bias = (const T*)a.bias + j;
  const T* res = (const T*)a.res + (r * a.n + j);
  T* y = (T*)a.y + (r * a.n + j);
  const bool whole = j + 4 <= a.n;
  T b[4] = {}, s[4] = {}, o[4];
  if (whole) {
    if (a.bias) __builtin_memcpy(b, bias, sizeof b);
    if (a.res) __builtin_memcpy(s, res, sizeof s);
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (a.bias && j + e < a.n) b[e] = bias[e];
      if (a.res && j + e < a.n) s[e] = res[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 4; e++) {
    if (a.bias) v[e] += (float)b[e];
    if (a.act.kind) v[e] = act4_apply(v[e], a.act);
    if (a.res) v[e] += (float)s[e];
    o[e] = (T)v[e];
  }
  if (whole) {
    __builtin_memcpy(y, o, sizeof o);
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (j + e < a.n) y[e] = o[e];
  }
}

// Few rows: bound by the weights' way from memory, each read once, and by the
// latencies before and after it, so everything is asked for at once.  The waves
// of a workgroup share 16 NT columns and take groups of U chunks of 128 k in
// turn: the group's x, then the codes and scales of all NT column tiles.  The
// waves' sums are added in LDS in their order.  The arguments that the loads
// need come first: they are in registers when the wave starts.
template <typename E, int NQ, int NT, int U>
__global__ __launch_bounds__(512) void linear4_few_kernel(const typename E::type* x,
                                                          const unsigned char* codes,
                                                          const unsigned char* scales, int64_t xs,
                                                          int rows, int k, int n, int chunks,
                                                          Lin4 a) {
  constexpr int size = sizeof(typename E::type);
  constexpr int TS = E::terms == 3 ? 3 : 1;
  constexpr int pieces = 8 * size, per = 2 * size;   // 16-byte pieces of 128 k; loads for 16 rows
  constexpr int elems = 16 / size, step = 64 / pieces;
  extern __shared__ __align__(16) char lds4[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int waves = blockDim.x >> 6;
  const int li = lane & 15, kg = lane >> 4;
  const int j0 = blockIdx.x * (16 * NT), r0 = blockIdx.y * (16 * NQ);
  char* part = lds4 + wave * (NQ * per * 1024);
  f32x4 acc[NT][NQ] = {};
  for (int c0 = wave * U; c0 < chunks; c0 += waves * U) {
    // x: piece lane % pieces of rows lane / pieces + step i
    u32x4 xv[U][NQ][per];
    const bool inside = (c0 + U) * 128 <= k;
#pragma unroll
    for (int q = 0; q < NQ; q++)
#pragma unroll
      for (int i = 0; i < per; i++) {
        if (r0 + 16 * q + step * i >= rows) continue;     // (the columns of no row hold anything)
        const int r = min(r0 + 16 * q + step * i + lane / pieces, rows - 1);
        const int at = c0 * 128 + (lane % pieces) * elems;
        const typename E::type* row = x + r * xs;
        if (inside) {
#pragma unroll
          for (int u = 0; u < U; u++) __builtin_memcpy(&xv[u][q][i], row + at + u * 128, 16);
        } else {
#pragma unroll
          for (int u = 0; u < U; u++) xv[u][q][i] = x_piece<E>(row, at + u * 128, k);
        }
      }
    // (a group that ends past the last chunk: that chunk again, against zeros)
    u32x4 w[NT][U];
    unsigned four[NT][U];
    const bool full = c0 + U <= chunks;
#pragma unroll
    for (int i = 0; i < NT; i++) {
      const int64_t at = (int64_t)min(j0 + 16 * i + li, n - 1) * chunks + c0;
      const unsigned char* cp = codes + at * 64 + kg * 16;
      const unsigned char* sp = scales + at * 4;
      if (full) {
#pragma unroll
        for (int u = 0; u < U; u++) w[i][u] = *(const u32x4*)(cp + u * 64);
        __builtin_memcpy(four[i], sp, 4 * U);
      } else {
#pragma unroll
        for (int u = 0; u < U; u++) {
          const int c = min(u, chunks - 1 - c0);
          w[i][u] = *(const u32x4*)(cp + c * 64);
          four[i][u] = *(const unsigned*)(sp + c * 4);
        }
      }
    }
    // piece p of row r at place p ^ r of the row: neither the rows' stores nor
    // the columns' loads meet in a bank
#pragma unroll
    for (int u = 0; u < U; u++) {
      wave_order();
#pragma unroll
      for (int q = 0; q < NQ; q++)
#pragma unroll
        for (int i = 0; i < per; i++) {
          if (r0 + 16 * q + step * i >= rows) continue;
          const int r = step * i + lane / pieces;
          *(u32x4*)(part + ((q * 16 + r) * pieces + ((lane % pieces) ^ r)) * 16) = xv[u][q][i];
        }
      wave_order();
      u32x4 wu[NT];
      unsigned fu[NT];
#pragma unroll
      for (int i = 0; i < NT; i++) { wu[i] = w[i][u]; fu[i] = four[i][u]; }
      chunk_products<E, NQ, NT, TS>(wu, fu, kg, [&](int m, u32x4 (&xf)[NQ][TS]) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < NQ; q++) {
          const char* row = part + (q * 16 + li) * pieces * 16;
          const int p = (4 * kg + m) * (size / 2);
          const u32x4 v0 = *(const u32x4*)(row + (p ^ li) * 16);
          if constexpr (E::terms == 3) {
            const u32x4 v1 = *(const u32x4*)(row + ((p + 1) ^ li) * 16);
            float v[8];
            bf16x8 t[3];
            __builtin_memcpy(v, &v0, 16);
            __builtin_memcpy(v + 4, &v1, 16);
            split8<3>(v, t);
#pragma unroll
            for (int i = 0; i < 3; i++) xf[q][i] = __builtin_bit_cast(u32x4, t[i]);
          } else {
            xf[q][0] = v0;
          }
        }
      }, acc);
    }
  }
  // (four columns' place in a row turns with the row where the rows would
  // otherwise start in a part of the banks only)
  constexpr int turn = NT % 2 ? 0 : 16 * NT - 4;
  float* red = (float*)lds4;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NT; i++)
#pragma unroll
    for (int q = 0; q < NQ; q++)
      *(f32x4*)&red[((wave * NQ + q) * 16 + li) * (16 * NT) + ((16 * i + 4 * kg) ^ (4 * li & turn))] = acc[i][q];
  __syncthreads();
  constexpr int tile = NQ * 16 * NT * 16;
  for (int i = 4 * threadIdx.x; i < tile; i += 4 * blockDim.x) {
    const int at = i ^ (4 * (i / (16 * NT)) & turn);
    f32x4 v = *(const f32x4*)&red[at];
    for (int w = 1; w < waves; w++) v += *(const f32x4*)&red[w * tile + at];
    linear4_store<E>(a, r0 + i / (16 * NT), j0 + i % (16 * NT), v);
  }
}

// More rows: a workgroup takes 16 NQ rows and 64 NT columns, its waves 16 NT
// columns of one half of every 256 k.  x is staged in LDS for all of them,
// split into its terms once, in the order of the MFMA's operand; two buffers,
// and the loads of the next D parts in flight.
template <typename E, int NQ, int NT, int D>
__global__ __launch_bounds__(512) void linear4_rows_kernel(const typename E::type* x,
                                                           const unsigned char* codes,
                                                           const unsigned char* scales, int64_t xs,
                                                           int rows, int k, int n, int chunks,
                                                           Lin4 a) {
  typedef typename E::type T;
  constexpr int TS = E::terms == 3 ? 3 : 1;
  constexpr int half = 4 * NQ * TS * 1024, buffer = 2 * half;
  extern __shared__ __align__(16) char lds4[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wave & 3, wk = wave >> 2;
  const int li = lane & 15, kg = lane >> 4;
  const int j0 = blockIdx.x * (64 * NT), r0 = blockIdx.y * (16 * NQ);
  const unsigned char *cp[NT], *sp[NT];
#pragma unroll
  for (int i = 0; i < NT; i++) {
    const int64_t at = (int64_t)min(j0 + 16 * (wn * NT + i) + li, n - 1) * chunks;
    cp[i] = codes + at * 64 + kg * 16;
    sp[i] = scales + at * 4;
  }
  // staged by this thread: eight elements, part p of 32, of row tid / 32 of each tile
  const int p = tid & 31, row = tid >> 5, ph = p >> 4, pk = p >> 2 & 3, pn = p & 3;
  const T* xr[NQ];
#pragma unroll
  for (int q = 0; q < NQ; q++) xr[q] = x + min(r0 + 16 * q + row, rows - 1) * xs;
  char* put = lds4 + ph * half + (pk * 16 + (row ^ (4 * pk + pn))) * 16;

  constexpr int XV = sizeof(T) / 2;     // 16-byte loads of eight elements
  struct Part {
    u32x4 x[NQ][XV], w[NT];
    unsigned four[NT];
  };
  const int parts = (chunks + 1) / 2;
  auto load = [&](int it, Part& s) __attribute__((always_inline)) {
    if (it >= parts) return;
    const int at = it * 256 + p * 8;
#pragma unroll
    for (int q = 0; q < NQ; q++)
#pragma unroll
      for (int i = 0; i < XV; i++) {
        if (it * 256 + 256 <= k) __builtin_memcpy(&s.x[q][i], xr[q] + at + i * (8 / XV), 16);
        else s.x[q][i] = x_piece<E>(xr[q], at + i * (8 / XV), k);
      }
    const int c = min(2 * it + wk, chunks - 1);     // (past the last: against zeros)
#pragma unroll
    for (int i = 0; i < NT; i++) {
      s.w[i] = *(const u32x4*)(cp[i] + (int64_t)c * 64);
      s.four[i] = *(const unsigned*)(sp[i] + (int64_t)c * 4);
    }
  };
  auto stage = [&](const Part& s, int b) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < NQ; q++) {
      if constexpr (TS == 3) {
        float v[8];
        bf16x8 t[3];
        __builtin_memcpy(v, &s.x[q][0], 32);
        split8<3>(v, t);
#pragma unroll
        for (int i = 0; i < 3; i++) *(bf16x8*)(put + b * buffer + ((pn * NQ + q) * 3 + i) * 1024) = t[i];
      } else {
        *(u32x4*)(put + b * buffer + (pn * NQ + q) * 1024) = s.x[q][0];
      }
    }
  };
  f32x4 acc[NT][NQ] = {};
  auto compute = [&](const Part& s, int b) __attribute__((always_inline)) {
    const char* from = lds4 + b * buffer + wk * half;
    chunk_products<E, NQ, NT, TS>(s.w, s.four, kg, [&](int m, u32x4 (&xf)[NQ][TS]) __attribute__((always_inline)) {
#pragma unroll
      for (int q = 0; q < NQ; q++)
#pragma unroll
        for (int t = 0; t < TS; t++)
          xf[q][t] = *(const u32x4*)(from + ((m * NQ + q) * TS + t) * 1024 +
                                     (kg * 16 + (li ^ (4 * kg + m))) * 16);
    }, acc);
  };
  // D is even, so that part it is in buffer it % 2: the one that a part is
  // staged into was read before the barrier that the part before it passed
  static_assert(D % 2 == 0, "two buffers");
  Part s[D];
#pragma unroll
  for (int d = 0; d < D; d++) load(d, s[d]);
  for (int it = 0; it < parts; it += D) {
#pragma unroll
    for (int d = 0; d < D; d++) {
      if (it + d >= parts) break;
      stage(s[d], d & 1);
      __syncthreads();
      compute(s[d], d & 1);
      load(it + d + D, s[d]);
    }
  }
  // the two halves' sums; four columns' place in a row turns with the row, or
  // all rows of a tile would be in the same banks
  float* red = (float*)lds4;
  __syncthreads();
  constexpr int cols = 64 * NT, tile = 16 * NQ * cols;
#pragma unroll
  for (int i = 0; i < NT; i++)
#pragma unroll
    for (int q = 0; q < NQ; q++)
      *(f32x4*)&red[wk * tile + (q * 16 + li) * cols + (((wn * NT + i) * 16 + 4 * kg) ^ (4 * li))] = acc[i][q];
  __syncthreads();
  for (int i = 4 * tid; i < tile; i += 2048) {
    const int at = i ^ (4 * (i / cols & 15));
    linear4_store<E>(a, r0 + i / cols, j0 + i % cols, *(f32x4*)&red[at] + *(f32x4*)&red[tile + at]);
  }
}

// HIP takes less than 2^32 threads along an axis of a launch.
static int linear4_fits(dim3 grid, int threads) {
  if ((uint64_t)grid.x * threads >> 32)
    return fail(QPH_EUNSUPPORTED, "linear4: too many columns for one call");
  return QPH_OK;
}

// (The launchers take the stream's context; without one they only check the launch.)
template <typename E, int NQ, int NT, int U>
static int launch_linear4_few(const Lin4& a, const qph_ctx* ctx) {
  // up to 8 waves along k, with a group of chunks each
  const int part = std::max(NQ * 16 * NT * 16 * 4, NQ * 2 * (int)sizeof(typename E::type) * 1024);
  int waves = 8;
  while (waves > 1 && (waves / 2) * U >= a.chunks) waves /= 2;
  const dim3 grid(ceil_div(a.n, 16 * NT), ceil_div(a.rows, 16 * NQ));
  QPH_TRY(linear4_fits(grid, 64 * waves));
  if (!ctx) return QPH_OK;
  if (waves * part > 65536) QPH_TRY(allow_full_lds((const void*)linear4_few_kernel<E, NQ, NT, U>));
  hipLaunchKernelGGL((linear4_few_kernel<E, NQ, NT, U>), grid, dim3(64 * waves), waves * part, ctx->stream,
                     (const typename E::type*)a.x, a.codes, a.scales, a.xs, (int)a.rows, (int)a.k,
                     (int)a.n, (int)a.chunks, a);
  return launch_check("linear4_few_kernel");
}

template <typename E, int NQ, int NT, int D>
static int launch_linear4_rows(const Lin4& a, const qph_ctx* ctx) {
  constexpr int TS = E::terms == 3 ? 3 : 1;
  const int lds = std::max(4 * 4 * NQ * TS * 1024, 2 * 16 * NQ * 64 * NT * 4);
  const dim3 grid(ceil_div(a.n, 64 * NT), ceil_div(a.rows, 16 * NQ));
  QPH_TRY(linear4_fits(grid, 512));
  if (!ctx) return QPH_OK;
  if (lds > 65536) QPH_TRY(allow_full_lds((const void*)linear4_rows_kernel<E, NQ, NT, D>));
  hipLaunchKernelGGL((linear4_rows_kernel<E, NQ, NT, D>), grid, dim3(512), lds, ctx->stream,
                     (const typename E::type*)a.x, a.codes, a.scales, a.xs, (int)a.rows, (int)a.k,
                     (int)a.n, (int)a.chunks, a);
  return launch_check("linear4_rows_kernel");
}

template <typename E, int NQ, int U>
static int launch_linear4_few_nt(const Lin4& a, const qph_ctx* ctx) {
  // Columns a workgroup: so many that one round of workgroups, one to each of
  // the 256 CUs, takes them, at most 64 (48 for two row tiles, whose registers
  // end there).  8 rows of 4096 x 12288 (768 column tiles) by one, two, three
  // and four tiles: 11.2, 11.4, 9.2 and 11.0 us; 16 of 4096 x 4096 (256): 5.9,
  // 7.5, 8.9 and 10.6.
  const int64_t tiles = (a.n + 15) / 16 * ((a.rows + 16 * NQ - 1) / (16 * NQ));
  if (tiles <= 256) return launch_linear4_few<E, NQ, 1, U>(a, ctx);
  if (tiles <= 512) return launch_linear4_few<E, NQ, 2, U>(a, ctx);
  if constexpr (NQ == 1) {
    // past 1024 tiles as many rounds as four tiles make, but even ones: 1 x 4096
    // x 20000 by three 15.1 us, by four 17.5, 16 x 256 x 18709 5.1 and 5.8
    const int64_t round = (tiles + 1023) / 1024 * 256;
    if (tiles > 3 * round) return launch_linear4_few<E, NQ, 4, U>(a, ctx);
  }
  return launch_linear4_few<E, NQ, 3, U>(a, ctx);
}

template <typename E>
static int launch_linear4(const Lin4& a, const qph_ctx* ctx) {
  constexpr bool f32 = E::terms == 3;
  // up to 16 rows: 16 x 4096 x 32768 22 us (float32 33), 33 (52) by more rows' kernel
  if (a.rows <= 16) return launch_linear4_few_nt<E, 1, 2>(a, ctx);
  // More rows cost their turning and, in float32, their split into terms in
  // every workgroup here; the other kernel shares them between more columns,
  // with less of the weights in flight.  So here while one round of workgroups
  // does: 64 x 4096 x 4096 10.7 us, 15.8 there, 32 x 4096 x 12288 in float32 25
  // and 34; past it 64 x 4096 x 8192 is 22.1 and 16.8, 64 x 4096 x 32768 60 and
  // 35, 32 x 4096 x 32768 in float32 67 and 53.
  const bool round = (a.n + 47) / 48 * ((a.rows + 31) / 32) <= 256;
  const bool round_32x64 = (a.n + 63) / 64 * ((a.rows + 31) / 32) <= 256;
  // (two-byte rows that 32 hold also where that one needs more than a round of
  // its smallest workgroups: 20 x 1024 x 18709 7.6 and 11.6 us, 32 x 4096 x 32768
  // 32.0 and 33.9, but 32 x 4096 x 16384 21.9 and 17.0)
  if (a.rows <= (f32 ? 32 : 64) && (round || (!f32 && a.rows <= 32 && !round_32x64)))
    return launch_linear4_few_nt<E, 2, f32 ? 1 : 2>(a, ctx);
  // Then the smallest workgroups that one round takes: 32 rows x 64 columns (128
  // x 4096 x 4096 16 us, 22 with 64 rows; in float32 35, 48 with 48 rows x 128
  // columns), 64 x 64 (256 x 4096 x 4096 23.4; 26.5 with 32 rows, 31.5 with 128
  // columns).  Past that the ones that do most with what they load: 64 x 128
  // (2048 x 4096 x 12288 343 us, 470 with 64 columns), in float32 48 x 128 (779
  // us, 1425 with 32 x 64).
  if (round_32x64) return launch_linear4_rows<E, 2, 1, 4>(a, ctx);
  if constexpr (f32) {
    return launch_linear4_rows<E, 3, 2, 2>(a, ctx);
  } else {
    if ((a.n + 63) / 64 * ((a.rows + 63) / 64) <= 256) return launch_linear4_rows<E, 4, 1, 4>(a, ctx);
    return launch_linear4_rows<E, 4, 2, 2>(a, ctx);
  }
}

// -------------------------------------------------------------- host checks

int cache4_check(const qph_cache4* c, const char* what, int* shift) {
  const std::string w(what);
  if (!c) return fail(QPH_EINVAL, w + ": NULL cache");
  if (!c->k_codes || !c->k_scales || !c->v_codes || !c->v_scales)
    return fail(QPH_EINVAL, w + ": NULL cache memory");
  if (c->n_pages <= 0 || c->heads <= 0) return fail(QPH_EINVAL, w + ": empty cache");
  if (c->page_size < 16 || c->page_size > 32768 || (c->page_size & (c->page_size - 1)))
    return fail(QPH_EUNSUPPORTED, w + ": page size " + std::to_string(c->page_size) +
                                      " is no power of two from 16 to 32768");
  switch (c->dh) {
    case 32: case 64: case 96: case 128: case 192: case 256: break;
    default:
      return fail(QPH_EUNSUPPORTED, w + ": head dimension " + std::to_string(c->dh) +
                                        " is not 32, 64, 96, 128, 192 or 256");
  }
  if (c->heads > 4096) return fail(QPH_EUNSUPPORTED, w + ": more than 4096 heads");
  // pages are numbered in 32 bits, and a token's place is held in 63
  if (c->n_pages > INT32_MAX) return fail(QPH_EUNSUPPORTED, w + ": more than 2^31 - 1 pages");
  if (((uintptr_t)c->k_codes | (uintptr_t)c->v_codes) % 16)
    return fail(QPH_EINVAL, w + ": codes are not 16-byte aligned");
  *shift = __builtin_ctz((unsigned)c->page_size);
  return QPH_OK;
}

static int cache4_io(qph_ctx* ctx, const qph_cache4* c, void* k, void* v, int32_t dtype,
                     int64_t tokens, const int64_t ks[2], const int64_t vs[2],
                     const int64_t* slots, bool write) {
  const char* what = write ? "cache4_write" : "cache4_read";
  const std::string w(what);
  int shift = 0;
  QPH_TRY(cache4_check(c, what, &shift));
  if (!dtype_valid(dtype)) return fail(QPH_EINVAL, w + ": unknown element type");
  if (tokens < 0) return fail(QPH_EINVAL, w + ": negative token count");
  if (tokens && (!k || !v || !slots || !ks || !vs)) return fail(QPH_EINVAL, w + ": NULL argument");
  if (!ctx) return fail(QPH_EINVAL, "null context");
  if (tokens == 0) return QPH_OK;
  Cache4Io a{};
  a.kc = (unsigned char*)c->k_codes; a.ks = (unsigned char*)c->k_scales;
  a.vc = (unsigned char*)c->v_codes; a.vs = (unsigned char*)c->v_scales;
  a.slots_n = c->n_pages << shift;
  a.shift = shift;
  a.heads = (unsigned)c->heads;
  a.words = (unsigned)c->dh / 8;
  a.kt = ks[0]; a.kh = ks[1]; a.vt = vs[0]; a.vh = vs[1];
  const unsigned units = a.heads * a.words;
  a.per = (int)std::max(1u, 256u / units);
  // Tokens that a thread reads at once: four where workgroups are many (65521
  // tokens of 8 x 128: 69 us, 88 with one and 67 with eight; 300000 of 1 x 64:
  // 18.5, 19.5 and 21), one where they are few.
  const int flight = !write && tokens / a.per >= 8192 ? 4 : 1;
  OnDevice dev(ctx);
  QPH_TRY(dev.rc());
  // (more tokens than one launch takes: in several)
  const int64_t most = kMaxGroups * a.per * flight, size = dtype == QPH_F32 ? 4 : 2;
  for (int64_t t = 0; t < tokens; t += most) {
    a.tokens = std::min(most, tokens - t);
    a.slots = slots + t;
    a.k = (char*)k + t * ks[0] * size;
    a.v = (char*)v + t * vs[0] * size;
    const dim3 grid(ceil_div(a.tokens, a.per * flight), 2);
#define QPH_LAUNCH(E)                                                                              \
  do {                                                                                             \
    auto fn = write ? cache4_write_kernel<E>                                                       \
                    : (flight == 4 ? cache4_read_kernel<E, 4> : cache4_read_kernel<E, 1>);         \
    hipLaunchKernelGGL(fn, grid, dim3(256), 0, ctx->stream, a);                                    \
  } while (0)
    if (dtype == QPH_F32) QPH_LAUNCH(F32);
    else if (dtype == QPH_F16) QPH_LAUNCH(F16);
    else QPH_LAUNCH(BF16);
#undef QPH_LAUNCH
    QPH_TRY(launch_check(what));
  }
  return QPH_OK;
}

template <typename E>
static void launch_quantize4(const Quant4& a, hipStream_t s) {
  const dim3 grid(ceil_div(a.rows * a.groups, 256));
  if (a.cs == 1) hipLaunchKernelGGL((quantize4_kernel<E, false>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((quantize4_kernel<E, true>), grid, dim3(256), 0, s, a);
}

}  // namespace qph

using namespace qph;

extern "C" {

QPH_API int qph_quantize4(qph_ctx* ctx, const void* x, int32_t dtype, int64_t rows, int64_t k,
                          int64_t row_stride, int64_t col_stride, void* codes, void* scales) {
  if (!dtype_valid(dtype)) return fail(QPH_EINVAL, "quantize4: unknown element type");
  if (rows < 0 || k <= 0) return fail(QPH_EINVAL, "quantize4: bad shape");
  if (k > (1 << 30)) return fail(QPH_EUNSUPPORTED, "quantize4: more than 2^30 columns");
  if (rows && (!x || !codes || !scales)) return fail(QPH_EINVAL, "quantize4: NULL argument");
  if ((uintptr_t)codes % 16) return fail(QPH_EINVAL, "quantize4: codes are not 16-byte aligned");
  if (rows > kMaxGroups * 256 / ((k + 127) / 128 * 4))
    return fail(QPH_EUNSUPPORTED, "quantize4: too many blocks for one call");
  if (!ctx) return fail(QPH_EINVAL, "null context");
  if (rows == 0) return QPH_OK;
  Quant4 a{};
  a.x = x; a.rows = rows; a.k = k; a.rs = row_stride; a.cs = col_stride;
  a.groups = (k + 127) / 128 * 4;
  a.codes = (unsigned char*)codes;
  a.scales = (unsigned char*)scales;
  OnDevice dev(ctx);
  QPH_TRY(dev.rc());
  if (dtype == QPH_F32) launch_quantize4<F32>(a, ctx->stream);
  else if (dtype == QPH_F16) launch_quantize4<F16>(a, ctx->stream);
  else launch_quantize4<BF16>(a, ctx->stream);
  return launch_check("quantize4_kernel");
}

QPH_API int qph_linear4(qph_ctx* ctx, const void* x, int32_t dtype, int64_t x_stride,
                        const void* codes, const void* scales, const void* bias, int64_t rows,
                        int64_t k, int64_t n, const qph_act* act, const void* residual, void* y) {
  if (!dtype_valid(dtype)) return fail(QPH_EINVAL, "linear4: unknown element type");
  if (rows < 0 || k <= 0 || n <= 0) return fail(QPH_EINVAL, "linear4: bad shape");
  if (!act_valid(act)) return fail(QPH_EINVAL, "linear4: unknown activation");
  if (rows && (!x || !codes || !scales || !y)) return fail(QPH_EINVAL, "linear4: NULL argument");
  if ((uintptr_t)codes % 16 || (uintptr_t)scales % 4)
    return fail(QPH_EINVAL, "linear4: codes are not 16-byte or scales not 4-byte aligned");
  // columns, rows and k are counted in 32 bits, row tiles by the grid's second axis
  if (n > (1 << 30) || k > (1 << 30) || rows > 65535 * 16)
    return fail(QPH_EUNSUPPORTED, "linear4: more than 2^30 columns or inputs, or 1048560 rows");
  Lin4 a{};
  a.x = x; a.xs = x_stride;
  a.codes = (const unsigned char*)codes;
  a.scales = (const unsigned char*)scales;
  a.bias = bias; a.res = residual; a.y = y;
  a.rows = rows; a.k = k; a.n = n;
  a.chunks = (k + 127) / 128;
  a.act = make_act(act);
  auto launch = [&](const qph_ctx* on) {
    if (rows == 0) return (int)QPH_OK;
    if (dtype == QPH_F32) return launch_linear4<F32>(a, on);
    if (dtype == QPH_F16) return launch_linear4<F16>(a, on);
    return launch_linear4<BF16>(a, on);
  };
  if (!ctx) {
    QPH_TRY(launch(nullptr));
    return fail(QPH_EINVAL, "null context");
  }
  if (rows == 0) return QPH_OK;
  OnDevice dev(ctx);
  QPH_TRY(dev.rc());
  return launch(ctx);
}

QPH_API int qph_cache4_write(qph_ctx* ctx, const qph_cache4* cache, const void* k, const void* v,
                             int32_t dtype, int64_t tokens, const int64_t k_strides[2],
                             const int64_t v_strides[2], const int64_t* slots) {
  return cache4_io(ctx, cache, (void*)k, (void*)v, dtype, tokens, k_strides, v_strides, slots, true);
}

QPH_API int qph_cache4_read(qph_ctx* ctx, const qph_cache4* cache, void* k, void* v, int32_t dtype,
                            int64_t tokens, const int64_t k_strides[2], const int64_t v_strides[2],
                            const int64_t* slots) {
  return cache4_io(ctx, cache, k, v, dtype, tokens, k_strides, v_strides, slots, false);
}

}  // extern "C"
