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
  int per;                    // tokens a workgroup
};

// Where head h of a cached token starts, in heads' rows.
__device__ __forceinline__ int64_t cache4_row(int64_t slot, int shift, unsigned heads, unsigned h) {
  return ((((slot >> shift) * heads + h) << shift) + (slot & (((int64_t)1 << shift) - 1)));
}

// A word of codes (eight elements) per thread; the four threads of a block of
// 32 share its largest magnitude by two swaps inside a quad.
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
    if (t >= a.tokens) break;                 // (a quad is of one token)
    const int64_t slot = a.slots[t];
    if (slot < 0 || slot >= a.slots_n) continue;
    float v[8];
    load8<E>(x + t * xt + h * xh + c * 8, v);
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
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

template <typename E>
__global__ __launch_bounds__(256) void cache4_read_kernel(Cache4Io a) {
  const unsigned units = a.heads * a.words, total = units * (unsigned)a.per;
  const bool second = blockIdx.y != 0;
  typename E::type* y = (typename E::type*)(second ? a.v : a.k);
  const int64_t yt = second ? a.vt : a.kt, yh = second ? a.vh : a.kh;
  const unsigned char* codes = second ? a.vc : a.kc;
  const unsigned char* scales = second ? a.vs : a.ks;
  for (unsigned u = threadIdx.x; u < total; u += blockDim.x) {
    const unsigned lt = u / units, w = u % units, h = w / a.words, c = w % a.words;
    const int64_t t = (int64_t)blockIdx.x * a.per + lt;
    if (t >= a.tokens) break;
    const int64_t slot = a.slots[t];
    float v[8];
    if (slot < 0 || slot >= a.slots_n) {
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = 0.0f;
    } else {
      const int64_t row = cache4_row(slot, a.shift, a.heads, h);
      const bf16x8 b = fp4_word(((const unsigned*)codes)[row * a.words + c],
                                scale_of_byte(scales[row * (a.words / 4) + c / 4]));
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = (float)b[i];
    }
    store8<E>(y + t * yt + h * yh + c * 8, v);
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

// y[r][j] = act(sum_k x[r][k] W[j][k] + bias[j]) + res[r][j].  A wave takes
// 16 NT columns j (MFMA rows) and 16 NQ rows r (MFMA columns); the waves of a
// workgroup take the chunks of k in turn and their sums are added in LDS in
// the waves' order.  A lane holds 32 neighbouring k of one column, one block:
// 16 bytes of codes and one scale.
template <typename E, int NQ, int NT>
__global__ __launch_bounds__(1024) void linear4_kernel(Lin4 a) {
  constexpr int T = E::terms;
  extern __shared__ float red[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int li = lane & 15, kg = lane >> 4;
  const int64_t j0 = (int64_t)blockIdx.x * (16 * NT), r0 = (int64_t)blockIdx.y * (16 * NQ);
  const unsigned char* wc[NT];
  const unsigned char* wsc[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const int64_t j = min(j0 + 16 * t + li, a.n - 1);
    wc[t] = a.codes + j * a.chunks * 64 + kg * 16;
    wsc[t] = a.scales + j * a.chunks * 4 + kg;
  }
  const typename E::type* xr[NQ];
#pragma unroll
  for (int q = 0; q < NQ; q++)
    xr[q] = (const typename E::type*)a.x + min(r0 + 16 * q + li, a.rows - 1) * a.xs;
  f32x4 acc[NT][NQ] = {};
  for (int64_t c = wave; c < a.chunks; c += waves) {
    u32x4 w[NT];
    float sc[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
      w[t] = *(const u32x4*)(wc[t] + c * 64);
      sc[t] = scale_of_byte(wsc[t][c * 4]);
    }
    const int64_t k0 = c * 128 + kg * 32;
    const bool whole = c * 128 + 128 <= a.k;
#pragma unroll
    for (int n = 0; n < 4; n++) {
      bf16x8 xf[NQ][T];
#pragma unroll
      for (int q = 0; q < NQ; q++) {
        float v[8];
        if (whole) load8<E>(xr[q] + k0 + 8 * n, v);
        else load8_upto<E>(xr[q] + k0 + 8 * n, (int)max((int64_t)0, min((int64_t)8, a.k - k0 - 8 * n)), v);
        split8<T>(v, xf[q]);
      }
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const bf16x8 wf = fp4_word(w[t][n], sc[t]);
#pragma unroll
        for (int q = 0; q < NQ; q++)
#pragma unroll
          for (int s = T - 1; s >= 0; s--) acc[t][q] = mfma16(wf, xf[q][s], acc[t][q]);
      }
    }
  }
  // sums of the waves, in their order
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int q = 0; q < NQ; q++)
#pragma unroll
      for (int r = 0; r < 4; r++)
        red[(((wave * NQ + q) * 16 + li) * NT + t) * 16 + 4 * kg + r] = acc[t][q][r];
  __syncthreads();
  constexpr int tile = NQ * 16 * NT * 16;
  for (int i = threadIdx.x; i < tile; i += blockDim.x) {
    const int64_t r = r0 + i / (16 * NT), j = j0 + i % (16 * NT);
    if (r >= a.rows || j >= a.n) continue;
    float v = 0.0f;
    for (int w = 0; w < waves; w++) v += red[w * tile + i];
    if (a.bias) v += (float)((const typename E::type*)a.bias)[j];
    v = act4_apply(v, a.act);
    if (a.res) v += (float)((const typename E::type*)a.res)[r * a.n + j];
    ((typename E::type*)a.y)[r * a.n + j] = (typename E::type)v;
  }
}

template <typename E, int NQ, int NT>
static int launch_linear4_tile(const Lin4& a, hipStream_t s) {
  // waves along k: a workgroup of up to 8, each with a chunk at least, and no
  // more than 64 KB of sums
  const int tile = NQ * 16 * NT * 16 * 4;
  int waves = 8;
  while (waves > 1 && (waves > a.chunks || waves * tile > 65536)) waves /= 2;
  const dim3 grid(ceil_div(a.n, 16 * NT), ceil_div(a.rows, 16 * NQ));
  hipLaunchKernelGGL((linear4_kernel<E, NQ, NT>), grid, dim3(64 * waves), waves * tile, s, a);
  return launch_check("linear4_kernel");
}

template <typename E>
static int launch_linear4(const Lin4& a, hipStream_t s) {
  if (a.rows <= 16) return launch_linear4_tile<E, 1, 1>(a, s);
  if (a.rows <= 32) return launch_linear4_tile<E, 2, 2>(a, s);
  return launch_linear4_tile<E, 4, 2>(a, s);
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
  a.slots = slots;
  a.tokens = tokens;
  a.k = k; a.v = v;
  a.kt = ks[0]; a.kh = ks[1]; a.vt = vs[0]; a.vh = vs[1];
  const unsigned units = a.heads * a.words;
  a.per = (int)std::max(1u, 256u / units);
  const int64_t groups = (tokens + a.per - 1) / a.per;
  if (groups > INT32_MAX) return fail(QPH_EUNSUPPORTED, w + ": too many tokens for one call");
  OnDevice dev(ctx);
  QPH_TRY(dev.rc());
  const dim3 grid((unsigned)groups, 2);
#define QPH_LAUNCH(E)                                                                     \
  do {                                                                                    \
    if (write) hipLaunchKernelGGL(cache4_write_kernel<E>, grid, dim3(256), 0, ctx->stream, a); \
    else hipLaunchKernelGGL(cache4_read_kernel<E>, grid, dim3(256), 0, ctx->stream, a);   \
  } while (0)
  if (dtype == QPH_F32) QPH_LAUNCH(F32);
  else if (dtype == QPH_F16) QPH_LAUNCH(F16);
  else QPH_LAUNCH(BF16);
#undef QPH_LAUNCH
  return launch_check(what);
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
  if (k > ((int64_t)1 << 31)) return fail(QPH_EUNSUPPORTED, "quantize4: more than 2^31 columns");
  if (rows && (!x || !codes || !scales)) return fail(QPH_EINVAL, "quantize4: NULL argument");
  if ((uintptr_t)codes % 16) return fail(QPH_EINVAL, "quantize4: codes are not 16-byte aligned");
  if (rows > ((int64_t)INT32_MAX * 256) / ((k + 127) / 128 * 4))
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
  // grid limits, and addresses that 63 bits hold
  if (n > ((int64_t)1 << 31) || k > ((int64_t)1 << 31) || rows > 65535 * (int64_t)16)
    return fail(QPH_EUNSUPPORTED, "linear4: shape past 2^31 columns or 1048560 rows");
  if (!ctx) return fail(QPH_EINVAL, "null context");
  if (rows == 0) return QPH_OK;
  Lin4 a{};
  a.x = x; a.xs = x_stride;
  a.codes = (const unsigned char*)codes;
  a.scales = (const unsigned char*)scales;
  a.bias = bias; a.res = residual; a.y = y;
  a.rows = rows; a.k = k; a.n = n;
  a.chunks = (k + 127) / 128;
  a.act = make_act(act);
  OnDevice dev(ctx);
  QPH_TRY(dev.rc());
  if (dtype == QPH_F32) return launch_linear4<F32>(a, ctx->stream);
  if (dtype == QPH_F16) return launch_linear4<F16>(a, ctx->stream);
  return launch_linear4<BF16>(a, ctx->stream);
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
