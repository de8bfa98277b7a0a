// cache8.hpp — the 8-bit cache format (FableCache8 in include/fable_attn_abi.h): e4m3 codes with an e8m0
// scale per block of tokens and head, and the conversions the kernels over it use.
//
// Scales are powers of two on purpose. A code times its scale is then exact in fp32 and bf16 (and in
// fp16 down to its subnormals), so nothing is rounded when a cache is read; the scale goes into the conversion
// instruction (v_cvt_scalef32_pk_*_fp8 takes it as an fp32 whose exponent it uses); and a block's scale can grow
// when a larger token arrives, with its older codes divided by a power of two: exact but for those that fall
// into e4m3's subnormals. With a floating code the finer steps of other scales would buy nothing: the relative error
// is 2^-4 at most either way.
#pragma once
#include <type_traits>

#include "attn_device.hpp"
#include "status.hpp"

namespace fa {

typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// the fp32 of an e8m0 byte (byte 0, below every scale an append stores, becomes 0)
__device__ __forceinline__ float e8_f32(unsigned byte) { return __uint_as_float(byte << 23); }
// 2^e for e in [-127, 127] (2^-127, the inverse of the largest scale, is subnormal)
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float(e > -127 ? (unsigned)(e + 127) << 23 : 0x400000u); }

// eight codes times `scale` (a power of two) in T
template <typename T>
__device__ __forceinline__ typename Dt<T>::V8 codes_to(u32x2 c, float scale) {
  typename Dt<T>::V8 r;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    if constexpr (std::is_same<T, __bf16>::value) {
      const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i], scale, false);
      const auto b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i], scale, true);
      r[4 * i] = a[0];
      r[4 * i + 1] = a[1];
      r[4 * i + 2] = b[0];
      r[4 * i + 3] = b[1];
    } else {
      const auto a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], scale, false);
      const auto b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], scale, true);
      r[4 * i] = a[0];
      r[4 * i + 1] = a[1];
      r[4 * i + 2] = b[0];
      r[4 * i + 3] = b[1];
    }
  }
  return r;
}

// codes of eight values times `inv` (a power of two; |x * inv| <= 448, or not finite: NaN codes), nearest even
__device__ __forceinline__ u32x2 to_codes(const float (&x)[8], float inv) {
  u32x2 r;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i] * inv, x[4 * i + 1] * inv, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2] * inv, x[4 * i + 3] * inv, w, true);
    r[i] = (unsigned)w;
  }
  return r;
}

// the least e with amax <= 448 * 2^e (448 = 0.875 * 2^9 is the largest code), in [-126, 119]; a block of
// zeros takes -126
__device__ __forceinline__ int code_exponent(float amax) {
  const unsigned u = __float_as_uint(amax);
  // amax = m * 2^x with m in [0.5, 1): x = exponent field - 126 (subnormals are below any bound of use)
  const int x = (int)(u >> 23) - 126;
  const int e = x - 9 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return amax > 0.0f ? max(min(e, 119), -126) : -126;
}

// whether the caches and scales have a form the kernels take (0: they do)
inline int cache8_check(const char* what, const FableCache8& c, int HD, int page) {
  if (HD <= 0 || HD > 256 || HD % 16) return fail(FA_ERR_HEADDIM, "%s: head_dim=%d (8-bit caches take multiples of 16 up to 256)", what, HD);
  if (page < 16 || (page & (page - 1))) return fail(FA_ERR_ARG, "%s: page=%d (a power of two of at least 16)", what, page);
  if (c.group < 1 || c.group > 256 || c.group > page || (c.group & (c.group - 1)))
    return fail(FA_ERR_ARG, "%s: group=%d (a power of two, at most 256 and the page)", what, c.group);
  if (c.num_blocks < 1) return fail(FA_ERR_ARG, "%s: num_blocks=%d", what, c.num_blocks);
  if (c.s.b < 0 || c.s.h < 0 || c.s.s < HD || c.s.s >= (1 << 26) || (c.s.b | c.s.h | c.s.s) % 16)
    return fail(FA_ERR_ARG, "%s: cache strides %lld, %lld, %lld", what, (long long)c.s.b, (long long)c.s.h, (long long)c.s.s);
  return FA_OK;
}

// fable_attn_append after the checks of a caller's own (append.hip); p.k null: only q is rotated
int append_rows(const FableAppendParams& p, int dtype, hipStream_t st);

}  // namespace fa
