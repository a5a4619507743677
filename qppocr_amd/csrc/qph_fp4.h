// Device helpers of the 4-bit operators (qph_fp4.hip, qph_attn4.hip).
//
// The block format: 32 neighbouring elements share a scale byte s; an element
// is a code of a sign and three bits (0, 0.5, 1, 1.5, 2, 3, 4, 6) and stands
// for that number times 2^(s - 127); s = 255 marks a block that held a NaN or
// an infinity, all of whose elements read as NaN.  Two codes to a byte, the
// even element's in the low half.  Every number of the format is exact in
// bfloat16, and gfx950 converts two codes and a scale to two bfloat16 in one
// instruction of full rate (checked against ldexp for every scale byte and
// every pair of codes), so the products run on the bfloat16 MFMA with the
// stored numbers themselves.  The other operand is split into bfloat16 terms
// whose sum is the value: one for bfloat16, two for float16 (11 bits), three
// for float32 (24 bits); no rounding but that of the float32 accumulators.
#pragma once

#include "qph_internal.h"

namespace qph {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kFp4MinExp = -100, kFp4MaxExp = 125;

// Element types of the callers' tensors (qph_dtype) and their bfloat16 terms.
struct F32 { typedef float type; static constexpr int terms = 3; };
struct F16 { typedef _Float16 type; static constexpr int terms = 2; };
struct BF16 { typedef __bf16 type; static constexpr int terms = 1; };

// Workgroups of 256 threads along an axis of a launch, which HIP allows less
// than 2^32 threads.
constexpr int64_t kMaxGroups = (1 << 24) - 1;

inline bool dtype_valid(int32_t d) { return d == QPH_F32 || d == QPH_F16 || d == QPH_BF16; }

// Makes the context's device current for one call and puts the caller's back.
class OnDevice {
 public:
  explicit OnDevice(const qph_ctx* ctx) {
    rc_ = hip_check(hipGetDevice(&was_), "hipGetDevice");
    if (rc_ == QPH_OK && was_ != ctx->device) {
      rc_ = hip_check(hipSetDevice(ctx->device), "hipSetDevice");
      back_ = rc_ == QPH_OK;
    }
  }
  ~OnDevice() {
    if (back_) (void)hipSetDevice(was_);
  }
  int rc() const { return rc_; }

 private:
  int was_ = 0, rc_ = QPH_OK;
  bool back_ = false;
};

__device__ __forceinline__ float scale_of_byte(unsigned s) { return __uint_as_float(s << 23); }

// The codes of byte B of w as two bfloat16 (the low half's first).
template <int B>
__device__ __forceinline__ unsigned fp4_pair(unsigned w, float scale) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, B));
}

// The same in float16, exact for scale bytes 104 to 140 (6 2^13 to half of 2^-23).
template <int B>
__device__ __forceinline__ unsigned fp4_pair_f16(unsigned w, float scale) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, B));
}

// The eight numbers of a word of codes.
__device__ __forceinline__ bf16x8 fp4_word(unsigned w, float scale) {
  const u32x4 v = {fp4_pair<0>(w, scale), fp4_pair<1>(w, scale), fp4_pair<2>(w, scale),
                   fp4_pair<3>(w, scale)};
  return __builtin_bit_cast(bf16x8, v);
}

__device__ __forceinline__ f16x8 fp4_word_f16(unsigned w, float scale) {
  const u32x4 v = {fp4_pair_f16<0>(w, scale), fp4_pair_f16<1>(w, scale), fp4_pair_f16<2>(w, scale),
                   fp4_pair_f16<3>(w, scale)};
  return __builtin_bit_cast(f16x8, v);
}

// Eight neighbouring elements as float32; any alignment of the element's own.
template <typename E>
__device__ __forceinline__ void load8(const typename E::type* p, float v[8]) {
  typename E::type t[8];
  __builtin_memcpy(t, p, sizeof t);
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = (float)t[i];
}

template <typename E>
__device__ __forceinline__ void store8(typename E::type* p, const float v[8]) {
  typename E::type t[8];
#pragma unroll
  for (int i = 0; i < 8; i++) t[i] = (typename E::type)v[i];
  __builtin_memcpy(p, t, sizeof t);
}

// Eight float32 as T bfloat16 terms that sum to them: each but the last cut
// off (so that no term overflows, and the rest is exact), the last rounded to
// nearest (exact too where the terms hold all bits).  An infinity is its own
// first term and leaves nothing (INF false: there are none); a NaN stays one.
template <int T, bool INF = true>
__device__ __forceinline__ void split8(const float v[8], bf16x8 out[T]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; i++) r[i] = v[i];
#pragma unroll
  for (int t = 0; t < T; t++) {
    if (t == T - 1) {
#pragma unroll
      for (int i = 0; i < 8; i++) out[t][i] = (__bf16)r[i];
    } else {
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; i++)
        w[i] = __builtin_amdgcn_perm(__float_as_uint(r[2 * i + 1]), __float_as_uint(r[2 * i]),
                                     0x07060302u);
      out[t] = __builtin_bit_cast(bf16x8, w);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float c = __uint_as_float(__float_as_uint(r[i]) & 0xffff0000u);
        r[i] = INF && r[i] == c ? 0.0f : r[i] - c;
      }
    }
  }
}

// Between the stores and loads of a wave's own part of LDS that pass data between
// its lanes: they are carried out in order, and must stay in order.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// The scale exponent of a block whose largest magnitude has these bits: the
// smallest power of two that puts it at 6 or below.  -1000 for a block with
// an infinity or a NaN.
__device__ __forceinline__ int fp4_exponent(unsigned top) {
  if (top >= 0x7f800000u) return -1000;
  const int e = (int)(top >> 23) - 129 + ((top & 0x7fffffu) > 0x400000u ? 1 : 0);
  return e < kFp4MinExp ? kFp4MinExp : (e > kFp4MaxExp ? kFp4MaxExp : e);
}

// Eight elements to a word of codes: x / scale to the nearest number of the
// format, ties to the even code, past 6 to 6 (the instruction's own rounding,
// checked at and beside every border of the format).
__device__ __forceinline__ unsigned fp4_encode8(const float v[8], float scale) {
  unsigned w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
  return w;
}

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Checks a cache descriptor (host); sets *shift to log2 of its page size.
int cache4_check(const qph_cache4* c, const char* what, int* shift);

}  // namespace qph
