// K/V rows in 8 bits: the code formats and the scale rule shared by the store's
// writer and reader (rows8.hip) and its attention kernels (rows8_attn.hip).
//
// A store holds, per (batch, KV head) row bh and for K and V apart, codes
// [BH, cap, D] of one byte and scales [BH, ceil(cap / 64)] of one float32 per
// 64-token block: value = code * scale.  Codes are e4m3 (the OCP format: 4
// exponent bits of bias 7, no infinity, NaN 0x7F / 0xFF, largest 448) or int8
// (-127 .. 127).
#pragma once

#include "common.hpp"

namespace fathom {
namespace rows8 {

// Smallest scale of a written block: its inverse and every product with it stay
// finite in float32 (a block of zeros holds this scale and codes 0).
constexpr float kMinScale = 7.888609052210118e-31f;  // 2^-100

typedef float f32x2 __attribute__((ext_vector_type(2)));

template <bool I8>
__host__ __device__ constexpr float code_max() {
  return I8 ? 127.0f : 448.0f;
}

// The four codes of a dword as floats (exact).
template <bool I8>
__device__ __forceinline__ void decode4(uint32_t w, float (&v)[4]) {
  if constexpr (I8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)(int8_t)(w >> (8 * i));
  } else {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    v[0] = a.x;
    v[1] = a.y;
    v[2] = b.x;
    v[3] = b.y;
  }
}

// Four floats, already divided by the scale, as a dword of codes: nearest code,
// ties to even; infinities saturate; NaN is NaN in e4m3 and 0 in int8.
template <bool I8>
__device__ __forceinline__ uint32_t encode4(const float (&y)[4]) {
  constexpr float kMax = code_max<I8>();
  float c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    c[i] = fminf(fmaxf(y[i], -kMax), kMax);
    if (y[i] != y[i]) c[i] = I8 ? 0.0f : y[i];
  }
  if constexpr (I8) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= ((uint32_t)(int)rintf(c[i]) & 0xFFu) << (8 * i);
    return w;
  } else {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], w, true);
  }
}

// Two 16-bit elements of a dword as floats.
template <int DT>
__device__ __forceinline__ void unpack2(uint32_t w, float &a, float &b) {
  if constexpr (DT == FATHOM_DT_BF16) {
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xFFFF0000u);
  } else {
    a = f16_bits_to_float((uint16_t)w);
    b = f16_bits_to_float((uint16_t)(w >> 16));
  }
}

// Two floats as 16-bit elements of a dword, rounded to nearest even.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == FATHOM_DT_BF16) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});  // one v_cvt_pk_bf16_f32
  } else {
    return float_to_f16_bits(a) | (uint32_t)float_to_f16_bits(b) << 16;
  }
}

// The scale s that a written block takes, and the factor f of its earlier codes: `was` its scale, `need` what its
// new tokens need, `earlier` the tokens that it holds already.
struct BlockScale {
  float s, f;
};
__device__ __forceinline__ BlockScale block_scale(float was, float need, int earlier) {
  const float size = fabsf(was);
  BlockScale to{need, 1.0f};
  if (earlier && size < INFINITY) {
    if (size == 0.0f) {
      to.f = 0.0f;
    } else {
      int by = 0;
      if (size < need) {
        int e0, e1;
        const float m0 = frexpf(size, &e0), m1 = frexpf(need, &e1);
        by = e1 - e0 + (m1 > m0 ? 1 : 0);
      }
      to.s = ldexpf(was, by);
      to.f = ldexpf(1.0f, -by);
    }
  }
  return to;
}
// `bytes` codes, times f, by a workgroup's threads.
template <bool I8>
__device__ __forceinline__ void rescale_codes(uint8_t *codes, int bytes, float f, int tid, int threads) {
  for (int o = 4 * tid; o < bytes; o += 4 * threads) {
    uint32_t *c = reinterpret_cast<uint32_t *>(codes + o);
    float y[4];
    decode4<I8>(*c, y);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] *= f;
    *c = encode4<I8>(y);
  }
}

// The length of row bh: the array's value, kept inside the store, or n.
__device__ __forceinline__ int64_t row_length(const int32_t *lens, int64_t n, int64_t cap, int64_t bh) {
  if (!lens) return n;
  const int64_t v = lens[bh];
  return v < 0 ? 0 : v < cap ? v : cap;
}

constexpr int64_t kMaxRows = 65535;           // of BH, and of heads G
constexpr int64_t kMaxCap = 0x7FFFFFFF - 64;  // tokens of a row

// Host checks common to the entry points: the store's shape, formats and alignment.
inline int check_store(const char *what, const void *k8, const void *v8, const float *ks, const float *vs, int code_dtype,
                       int64_t BH, int64_t cap, int64_t D) {
  if (!k8 || !v8 || !ks || !vs) return fail(FATHOM_ERR_INVALID, "%s: null store pointer", what);
  if (code_dtype != FATHOM_DT_E4M3 && code_dtype != FATHOM_DT_I8)
    return fail(FATHOM_ERR_INVALID, "%s: code_dtype %d is neither e4m3 nor int8", what, code_dtype);
  if (D != 64 && D != 128) return fail(FATHOM_ERR_INVALID, "%s: D=%lld, the store holds rows of 64 or 128", what, (long long)D);
  if (BH < 1 || BH > kMaxRows) return fail(FATHOM_ERR_INVALID, "%s: BH=%lld outside [1, 65535]", what, (long long)BH);
  if (cap < 1 || cap > kMaxCap) return fail(FATHOM_ERR_INVALID, "%s: cap=%lld", what, (long long)cap);
  if ((reinterpret_cast<uintptr_t>(k8) | reinterpret_cast<uintptr_t>(v8)) & 15)
    return fail(FATHOM_ERR_INVALID, "%s: the codes must be 16-byte aligned", what);
  if ((reinterpret_cast<uintptr_t>(ks) | reinterpret_cast<uintptr_t>(vs)) & 3)
    return fail(FATHOM_ERR_INVALID, "%s: the scales must be 4-byte aligned", what);
  return FATHOM_OK;
}

}  // namespace rows8
}  // namespace fathom
