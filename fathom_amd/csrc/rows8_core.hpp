// What the attention kernels of the 8-bit K/V row store share: lane exchanges, tanh, code
// conversions for the matrix cores, loads that end with a row, and the attention of single tokens
// as a part of another call.
#pragma once

#include <type_traits>

#include "rows8.hpp"

namespace fathom {
namespace rows8 {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLowest = -3.0e38f;  // below every score: the running maximum of no token
// A weight is 2^(x y - m), m the largest rounded x y: below kLarge with one rounding (a fused multiply-add), which leaves the
// maximum's own rounding in the weights, all alike, at most 2^(1/16) here.  Past it that would be 2 and more, up to
// infinity or 0, so there the product is rounded first and the largest weight is 1.
constexpr float kLarge = 1048576.0f;  // 2^20
// Eight consecutive elements of q from i (a multiple of eight).
__device__ __forceinline__ void load8_q(const void *q, int dt, int64_t i, float (&v)[8]) {
  if (dt == FATHOM_DT_F32) {
    const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(q) + i);
    const float4 x = p[0], y = p[1];
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
  } else {
    const uint4 x = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(q) + i);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (dt == FATHOM_DT_BF16) unpack2<FATHOM_DT_BF16>(w[e], v[2 * e], v[2 * e + 1]);
      else unpack2<FATHOM_DT_F16>(w[e], v[2 * e], v[2 * e + 1]);
    }
  }
}

// tanh to about a step of float32: below 1/2 u + u^3 P(u^2), P the least-squares fit of
// degree 4 to (tanh u - u) / u^3; from there (1 - t) / (1 + t), t = e^(-2 |u|), the quotient
// by the reciprocal and one correction.
__device__ __forceinline__ float tanh_small(float u) {
  const float w = u * u;
  float p = -0.006947011f;
  p = fmaf(p, w, 0.021472726f);
  p = fmaf(p, w, -0.05393379f);
  p = fmaf(p, w, 0.13333227f);
  p = fmaf(p, w, -0.3333333f);
  return fmaf(u * w, p, u);
}
__device__ __forceinline__ float tanh_any(float u) {
  const float x = fabsf(u);
  const float t = __builtin_amdgcn_exp2f(x * (-2.0f * kLog2e));
  const float n = 1.0f - t, d = 1.0f + t, r = __builtin_amdgcn_rcpf(d);
  float far = n * r;
  far = fmaf(fmaf(-far, d, n), r, far);
  return x < 0.5f ? tanh_small(u) : copysignf(far, u);
}

// Sum or maximum over the four lanes l, l ^ 16, l ^ 32, l ^ 48 (v_permlane32_swap
// and v_permlane16_swap give each lane its partner's value).
template <bool MAX>
__device__ __forceinline__ float across_groups(float v) {
  auto op = [](float x, float y) { return MAX ? fmaxf(x, y) : x + y; };
  const uint32_t x = __float_as_uint(v);
  const auto p32 = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  v = op(__uint_as_float(p32[0]), __uint_as_float(p32[1]));
  const uint32_t y = __float_as_uint(v);
  const auto p16 = __builtin_amdgcn_permlane16_swap(y, y, false, false);
  return op(__uint_as_float(p16[0]), __uint_as_float(p16[1]));
}

// v of another lane of the same row of 16, by a DPP control.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));  // folds into its use
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E;           // quad_perm [1,0,3,2], [2,3,0,1]
constexpr int kHalfMirror = 0x141;                  // row_half_mirror: lane 7 - l of a half row
constexpr int kRor4 = 0x124, kXor8 = 0x128;         // row_ror:4 and :8

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2v __attribute__((ext_vector_type(2)));

// Block b of a row's codes through a buffer descriptor that holds its tokens
// before `end`: loads behind that give zeros.  A single token's are streams (the nt bit): its
// step reads a row once, and other layers' rows come before its next step.  us with, without, rows
// that come from HBM: 8 x 1048576 tokens 345, 380; 32 x 32768 52, 57; 16 x 18432 21.6, 22.4 (while they fit the
// 256 MB cache and nothing else runs: 21.2, 19.9).
constexpr int kStream = 2;
template <int AUX>
struct RowsWith {
  __amdgpu_buffer_rsrc_t rsrc;
  __device__ __forceinline__ RowsWith(const uint8_t *codes, int64_t row0, int64_t b, int64_t end, int D) {
    const int64_t left = end - b * kBlk;
    const int tokens = left < 0 ? 0 : left < kBlk ? (int)left : kBlk;
    rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(codes) + (row0 + (tokens ? b * kBlk : 0)) * D, 0, tokens * D,
                                             0x00027000);
  }
  typedef u32x2v u32x2;
  __device__ __forceinline__ u32x4 load16(int off) const {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, 0, AUX));
  }
  __device__ __forceinline__ void load(int off, u32x2 &v) const {
    v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rsrc, off, 0, AUX));
  }
  __device__ __forceinline__ void load(int off, uint16_t &v) const { v = __builtin_amdgcn_raw_buffer_load_b16(rsrc, off, 0, AUX); }
  __device__ __forceinline__ void load(int off, uint32_t &v) const { v = __builtin_amdgcn_raw_buffer_load_b32(rsrc, off, 0, AUX); }
};
typedef RowsWith<kStream> RowsOf;

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Bytes 0, 1 (HI: 2, 3) of a dword of codes as two f16 values (exact: e4m3 and
// int8 both fit f16).  int8 codes come with their sign bit flipped (flip_sign),
// as c + 128 in 0 .. 255: under the exponent byte 0x64 that is the f16 number
// 1024 + (c + 128).
template <bool I8>
__device__ __forceinline__ uint32_t flip_sign(uint32_t w) {
  return I8 ? w ^ 0x80808080u : w;
}
template <bool I8, bool HI>
__device__ __forceinline__ f16x2 pair16(uint32_t w) {
  if constexpr (I8) {
    const uint32_t h = __builtin_amdgcn_perm(0x64646464u, w, HI ? 0x04030402u : 0x04010400u);
    const f16x2 b = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    return __builtin_bit_cast(f16x2, h) + b;
  } else {
    return __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, HI));
  }
}
__device__ __forceinline__ f16x8 join8(f16x2 a, f16x2 b, f16x2 c, f16x2 d) {
  return f16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// Two floats as f16 (keep = 0), or as the f16 of what those leave (keep = -1): to nearest both times.
__device__ __forceinline__ f16x2 split16(float x, float y, float keep) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f16x2 hi = __builtin_convertvector(f32x2{x, y}, f16x2);
  return __builtin_convertvector(f32x2{fmaf((float)hi.x, keep, x), fmaf((float)hi.y, keep, y)}, f16x2);
}

// Of a query channel x (the head's largest in [2^12, 2^14)): whether two f16 may hold fewer than 19 bits
// of it, and what they leave of such a one, times 2^38 (at most 2^13: they end at 2^-24).
__device__ __forceinline__ bool small_channel(float x) { return fabsf(x) < 0x1p-6f && x != 0.0f; }
__device__ __forceinline__ float rest_of(float x) {
  const float left = x - (float)(_Float16)x;
  return small_channel(x) ? ldexpf(left - (float)(_Float16)left, 38) : 0.0f;
}

// A caller's cap as the kernels take it, in a range where scale / softcap and its products stay normal: below
// 2^-64 every weight is 1 either way, and above 2^90 (0: none) scores below 2^78 do not notice a cap.
inline float kernel_cap(float softcap) {
  return softcap > 0x1p90f ? 0.0f : softcap > 0.0f && softcap < 0x1p-64f ? 0x1p-64f : softcap;
}

inline int check_query(const char *what, const void *q, int q_dtype, int64_t G, int64_t cap, const int32_t *lens, int64_t n,
                       float softcap, const void *out) {
  if (!q || !out) return fail(FATHOM_ERR_INVALID, "%s: null pointer", what);
  if (q_dtype < FATHOM_DT_F32 || q_dtype > FATHOM_DT_BF16) return fail(FATHOM_ERR_INVALID, "%s: q_dtype %d", what, q_dtype);
  if (G < 1 || G > kMaxRows) return fail(FATHOM_ERR_INVALID, "%s: G=%lld", what, (long long)G);
  if (!lens && (n < 0 || n > cap)) return fail(FATHOM_ERR_INVALID, "%s: length %lld outside [0, cap=%lld]", what, (long long)n, (long long)cap);
  if (!(softcap >= 0.0f && softcap < INFINITY)) return fail(FATHOM_ERR_INVALID, "%s: softcap must be 0 (none) or positive and finite", what);
  if (reinterpret_cast<uintptr_t>(q) & 15) return fail(FATHOM_ERR_INVALID, "%s: q must be 16-byte aligned", what);
  return FATHOM_OK;
}

// Whether the calls take this shape: the queries answer 0 for others, as their products could wrap.
inline bool shape_taken(int64_t BH, int64_t G, int64_t D) {
  return BH >= 1 && BH <= kMaxRows && G >= 1 && G <= kMaxRows && (D == 64 || D == 128);
}

// The attention of single tokens over whole rows of a store, left as partial results for the caller to join: row bh's
// are slots where[bh].x .. + where[bh].y - 1, or bh nsplit .. + nsplit - 1 where `where` is null.  Of slot s and head g,
// ml[s G + g] holds the largest score in log2 units and the sum of the weights 2^(score - it), part[(s G + g) D ..] the
// weighted rows.  workspace: tail_bytes for the longest row, 16-byte aligned.  The store, q and G are checked already.
struct Tail {
  const float *part;
  const float2 *ml;
  const int2 *where;
  int64_t nsplit;
};
size_t tail_bytes(int64_t BH, int64_t G, int64_t D, int64_t positions);
int tail_attention(Tail &t, const char *what, const void *q, int q_dtype, const void *k8, const void *v8, const float *k_scale,
                   const float *v_scale, bool i8, int64_t BH, int64_t G, int64_t D, int64_t cap, const int32_t *lens, int64_t n,
                   float scale, float softcap, const float *slopes, void *workspace, size_t workspace_bytes, hipStream_t st);

}  // namespace rows8
}  // namespace fathom
