// The 8-bit K/V row store's writer and reader.
//
// Write: tokens [p, p + T) of a row.  For each 64-token block they touch, with
// a = the largest finite |x| among the block's new tokens and kMax the format's
// largest code,
//   need = max(fl(a / kMax), 2^-100)
//   s'   = need               if the block holds no earlier token, or s is 0 or
//                             not finite
//        = s 2^j, the least j >= 0 with |s| 2^j >= need, otherwise
//   code = RN(fl(x fl(1 / s')))        of the new tokens
//        = RN(code 2^-j)               of the block's earlier ones (0 where s is 0, as their
//                                      values are; as they are where it is not finite)
// (fl: one float32 rounding; RN: nearest code, ties to even).  Scales grow by
// powers of two because a block that grows token by token is rounded anew each
// time: an e4m3 code then only changes its exponent (its value is rounded again
// only once it is a subnormal), and the roundings of an int8 code, half a step
// each, add up to less than one step of the last scale.
#include "rows8.hpp"

namespace fathom {
namespace rows8 {
namespace {

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kReadPieces = 4;
constexpr int64_t kMaxWrite = (1 << 30) - 128;  // tokens of a write: its grid stays below 2^32 threads

struct WriteArgs {
  const void *x[2];
  int64_t row_stride[2], tok_stride[2];  // in elements
  uint8_t *codes[2];
  float *scale[2];
  const int32_t *pos;
  int64_t pos_value, T, cap, nblk;
};

// One workgroup per (touched block, row, K or V): the block's new rows are read
// once into registers, their maximum is reduced, and the codes are written from
// the registers.  Rows and codes pass the caches as streams (nontemporal): nothing
// here reads them again.
//
// Bound: HBM.  8 x 131072 bf16 rows (805 MB in and out): 131 us back to back, 6.1 TB/s (143 us without
// the streams); a launch by itself 142, the median of twelve.  float32 rows of D = 128 take 230
// registers, which leaves two waves per SIMD: 8 x 65536 (671 MB) 253 us, 2.7 TB/s.
template <int D, int DT, bool I8>
__global__ __launch_bounds__(kThreads) void write_kernel(WriteArgs a) {
  constexpr int kElem = DT == FATHOM_DT_F32 ? 4 : 8;  // elements of a thread's 16-byte piece
  constexpr int kPieces = D / kElem;                  // pieces of a row
  constexpr int kRows = kThreads / kPieces;           // rows of a pass
  constexpr int kPasses = kBlk / kRows;
  __shared__ float wave_max[kThreads / kWave];
  const int tid = threadIdx.x;
  const int64_t bh = blockIdx.y;
  const int kv = blockIdx.z;
  const int64_t p = a.pos ? (int64_t)a.pos[bh] : a.pos_value;
  if (p < 0 || p + a.T > a.cap) return;  // the row's tokens do not all fit: it stays as it is
  const int64_t blk = p / kBlk + blockIdx.x;
  const int64_t t0 = blk * kBlk;
  if (t0 >= p + a.T) return;
  float *scale = a.scale[kv] + bh * a.nblk + blk;
  const float was = *scale;
  const int64_t row_bytes = (int64_t)D * (DT == FATHOM_DT_F32 ? 4 : 2);
  const char *src = static_cast<const char *>(a.x[kv]) + a.row_stride[kv] * bh * (row_bytes / D);
  const int64_t tok_bytes = a.tok_stride[kv] * (row_bytes / D);
  const int r0 = tid / kPieces, piece = tid % kPieces;
  u32x4 raw[kPasses];
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int64_t j = t0 + i * kRows + r0 - p;  // index among the new tokens
    raw[i] = u32x4{0u, 0u, 0u, 0u};
    if (j >= 0 && j < a.T) raw[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(src + j * tok_bytes + 16 * piece));
  }
  float x[kPasses][kElem];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (DT == FATHOM_DT_F32) x[i][e] = __uint_as_float(raw[i][e]);
      else unpack2<DT>(raw[i][e], x[i][2 * e], x[i][2 * e + 1]);
    }
#pragma unroll
    for (int e = 0; e < kElem; ++e) {
      const float v = fabsf(x[i][e]);
      if (v < INFINITY) amax = fmaxf(amax, v);  // NaN and infinities take no part
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
  if ((tid & 63) == 0) wave_max[tid >> 6] = amax;
  __syncthreads();
  amax = fmaxf(fmaxf(wave_max[0], wave_max[1]), fmaxf(wave_max[2], wave_max[3]));
  const float need = fmaxf(amax / code_max<I8>(), kMinScale);
  const int earlier = (int)(p > t0 ? p - t0 : 0);  // tokens that the block holds already
  const float size = fabsf(was);
  float s = need, f = 1.0f;  // f: what the earlier codes are multiplied by
  if (earlier && size < INFINITY) {
    if (size == 0.0f) {
      f = 0.0f;
    } else {
      int by = 0;
      if (size < need) {
        int e0, e1;
        const float m0 = frexpf(size, &e0), m1 = frexpf(need, &e1);
        by = e1 - e0 + (m1 > m0 ? 1 : 0);
      }
      s = ldexpf(was, by);
      f = ldexpf(1.0f, -by);
    }
  }
  const float inv = 1.0f / s;
  uint8_t *dst = a.codes[kv] + (bh * a.cap + t0) * D;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int r = i * kRows + r0;
    const int64_t j = t0 + r - p;
    if (j < 0 || j >= a.T) continue;
    uint32_t w[kElem / 4];
#pragma unroll
    for (int e = 0; e < kElem / 4; ++e) {
      const float y[4] = {x[i][4 * e] * inv, x[i][4 * e + 1] * inv, x[i][4 * e + 2] * inv, x[i][4 * e + 3] * inv};
      w[e] = encode4<I8>(y);
    }
    if constexpr (kElem == 8) __builtin_nontemporal_store(u32x2{w[0], w[1]}, reinterpret_cast<u32x2 *>(dst + r * D + 8 * piece));
    else __builtin_nontemporal_store(w[0], reinterpret_cast<uint32_t *>(dst + r * D + 4 * piece));
  }
  if (f != 1.0f) {
    for (int o = 4 * tid; o < earlier * D; o += 4 * kThreads) {
      uint32_t *c = reinterpret_cast<uint32_t *>(dst + o);
      float y[4];
      decode4<I8>(*c, y);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] *= f;
      *c = encode4<I8>(y);
    }
  }
  if (tid == 0) *scale = s;
}

struct ReadArgs {
  const uint8_t *codes[2];
  const float *scale[2];
  void *out[2];
  const int32_t *pos;
  const int64_t *idx;
  int64_t pos_value, R, cap, nblk;
};

// Row r of the output is token idx[bh, r], or pos + r; tokens outside the store give
// zeros.  A thread writes kReadPieces pieces of 16 bytes, kThreads pieces apart, with all of
// their codes requested first.
//
// Bound: HBM (D codes in, 2 D or 4 D bytes out per token).  8 x 131072 rows to bf16: 132 us,
// 6.1 TB/s, stores as streams (137 us without; one piece of four values per thread: 241 us).  8 x 16384 listed
// rows of 262144 tokens (104 MB): 17 us, 6.0 TB/s.
template <int D, int DT, bool I8>
__global__ __launch_bounds__(kThreads) void read_kernel(ReadArgs a) {
  constexpr int kElem = DT == FATHOM_DT_F32 ? 4 : 8;  // values of a piece
  constexpr int kRows = kReadPieces * kThreads * kElem / D;
  const int64_t bh = blockIdx.y, r0 = (int64_t)blockIdx.x * kRows;
  const int kv = blockIdx.z;
  const int64_t p = a.pos ? (int64_t)a.pos[bh] : a.pos_value;
  const uint8_t *codes = a.codes[kv] + bh * a.cap * D;
  const float *scale = a.scale[kv] + bh * a.nblk;
  uint32_t w[kReadPieces][kElem / 4];
  float s[kReadPieces];
#pragma unroll
  for (int i = 0; i < kReadPieces; ++i) {
    const int e = (i * kThreads + (int)threadIdx.x) * kElem;
    const int64_t r = r0 + e / D;
    int64_t tok = -1;
    if (r < a.R) tok = a.idx ? a.idx[bh * a.R + r] : p + r;
    s[i] = 0.0f;
#pragma unroll
    for (int x = 0; x < kElem / 4; ++x) w[i][x] = 0u;
    if (tok >= 0 && tok < a.cap) {
      const uint8_t *c = codes + tok * D + e % D;
      if constexpr (kElem == 8) {
        const uint2 v = *reinterpret_cast<const uint2 *>(c);
        w[i][0] = v.x;
        w[i][1] = v.y;
      } else {
        w[i][0] = *reinterpret_cast<const uint32_t *>(c);
      }
      s[i] = scale[(uint64_t)tok / kBlk];
    }
  }
#pragma unroll
  for (int i = 0; i < kReadPieces; ++i) {
    const int e = (i * kThreads + (int)threadIdx.x) * kElem;
    const int64_t r = r0 + e / D;
    if (r >= a.R) continue;
    float v[kElem];
#pragma unroll
    for (int x = 0; x < kElem / 4; ++x) {
      float c[4];
      decode4<I8>(w[i][x], c);
#pragma unroll
      for (int y = 0; y < 4; ++y) v[4 * x + y] = c[y] * s[i];
    }
    const int64_t o = (bh * a.R + r0) * D + e;
    if constexpr (DT == FATHOM_DT_F32) {
      typedef float f32x4 __attribute__((ext_vector_type(4)));
      __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4 *>(static_cast<float *>(a.out[kv]) + o));
    } else {
      const u32x4 h = {pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]), pack2<DT>(v[4], v[5]), pack2<DT>(v[6], v[7])};
      __builtin_nontemporal_store(h, reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(a.out[kv]) + o));
    }
  }
}

template <int D, int DT, bool I8>
void launch_write(const WriteArgs &a, int64_t BH, hipStream_t st) {
  // T tokens touch at most ceil((T + 63) / 64) blocks
  write_kernel<D, DT, I8><<<dim3((unsigned)cdiv(a.T + kBlk - 1, kBlk), (unsigned)BH, 2), kThreads, 0, st>>>(a);
}

template <int D, int DT, bool I8>
void launch_read(const ReadArgs &a, int64_t BH, hipStream_t st) {
  constexpr int64_t kRows = kReadPieces * kThreads * (DT == FATHOM_DT_F32 ? 4 : 8) / D;
  read_kernel<D, DT, I8><<<dim3((unsigned)cdiv(a.R, kRows), (unsigned)BH, 2), kThreads, 0, st>>>(a);
}

#define FATHOM_ROWS8_DISPATCH(fn, ...)                                         \
  do {                                                                         \
    const int sel = (D == 128 ? 6 : 0) + dt * 2 + (code_dtype == FATHOM_DT_I8); \
    switch (sel) {                                                             \
      case 0: fn<64, FATHOM_DT_F32, false>(__VA_ARGS__); break;                \
      case 1: fn<64, FATHOM_DT_F32, true>(__VA_ARGS__); break;                 \
      case 2: fn<64, FATHOM_DT_F16, false>(__VA_ARGS__); break;                \
      case 3: fn<64, FATHOM_DT_F16, true>(__VA_ARGS__); break;                 \
      case 4: fn<64, FATHOM_DT_BF16, false>(__VA_ARGS__); break;               \
      case 5: fn<64, FATHOM_DT_BF16, true>(__VA_ARGS__); break;                \
      case 6: fn<128, FATHOM_DT_F32, false>(__VA_ARGS__); break;               \
      case 7: fn<128, FATHOM_DT_F32, true>(__VA_ARGS__); break;                \
      case 8: fn<128, FATHOM_DT_F16, false>(__VA_ARGS__); break;               \
      case 9: fn<128, FATHOM_DT_F16, true>(__VA_ARGS__); break;                \
      case 10: fn<128, FATHOM_DT_BF16, false>(__VA_ARGS__); break;             \
      default: fn<128, FATHOM_DT_BF16, true>(__VA_ARGS__); break;              \
    }                                                                          \
  } while (0)

}  // namespace
}  // namespace rows8
}  // namespace fathom

using namespace fathom;
using namespace fathom::rows8;

extern "C" int fathom_rows8_write(const void *K, const void *V, int dtype, int64_t k_row_stride, int64_t k_tok_stride,
                                  int64_t v_row_stride, int64_t v_tok_stride, const int32_t *pos, int64_t pos_value,
                                  int64_t BH, int64_t T, int64_t D, int64_t cap, int code_dtype, void *k8, void *v8,
                                  float *k_scale, float *v_scale, void *stream) {
  int rc = check_store("rows8_write", k8, v8, k_scale, v_scale, code_dtype, BH, cap, D);
  if (rc) return rc;
  if (dtype < FATHOM_DT_F32 || dtype > FATHOM_DT_BF16) return fail(FATHOM_ERR_INVALID, "rows8_write: dtype %d", dtype);
  if (T < 0 || T > cap) return fail(FATHOM_ERR_INVALID, "rows8_write: T=%lld outside [0, cap=%lld]", (long long)T, (long long)cap);
  if (T > kMaxWrite) return fail(FATHOM_ERR_INVALID, "rows8_write: T=%lld, at most %lld at a time", (long long)T, (long long)kMaxWrite);
  if (!pos && (pos_value < 0 || pos_value > cap - T))  // in this form, as a sum could wrap
    return fail(FATHOM_ERR_INVALID, "rows8_write: %lld tokens from %lld outside [0, cap=%lld)", (long long)T,
                (long long)pos_value, (long long)cap);
  if (T == 0) return FATHOM_OK;
  if (!K || !V) return fail(FATHOM_ERR_INVALID, "rows8_write: null pointer");
  const int64_t size = dtype == FATHOM_DT_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(K) | reinterpret_cast<uintptr_t>(V)) & 15 ||
      ((k_row_stride | k_tok_stride | v_row_stride | v_tok_stride) * size) & 15)
    return fail(FATHOM_ERR_INVALID, "rows8_write: K and V and their strides must be multiples of 16 bytes");
  const WriteArgs a{{K, V},          {k_row_stride, v_row_stride}, {k_tok_stride, v_tok_stride}, {(uint8_t *)k8, (uint8_t *)v8},
                    {k_scale, v_scale}, pos, pos_value, T, cap, cdiv(cap, kBlk)};
  const int dt = dtype;
  FATHOM_ROWS8_DISPATCH(launch_write, a, BH, (hipStream_t)stream);
  return launch_status("rows8 write_kernel");
}

extern "C" int fathom_rows8_read(const void *k8, const void *v8, const float *k_scale, const float *v_scale,
                                 int code_dtype, int64_t BH, int64_t cap, int64_t D, const int64_t *idx, const int32_t *pos,
                                 int64_t pos_value, int64_t R, int dtype, void *K, void *V, void *stream) {
  int rc = check_store("rows8_read", k8, v8, k_scale, v_scale, code_dtype, BH, cap, D);
  if (rc) return rc;
  if (dtype < FATHOM_DT_F32 || dtype > FATHOM_DT_BF16) return fail(FATHOM_ERR_INVALID, "rows8_read: dtype %d", dtype);
  if (R < 0 || R > 0x7FFFFFFF) return fail(FATHOM_ERR_INVALID, "rows8_read: %lld rows", (long long)R);
  if (R == 0) return FATHOM_OK;
  if (!K || !V) return fail(FATHOM_ERR_INVALID, "rows8_read: null pointer");
  if ((reinterpret_cast<uintptr_t>(K) | reinterpret_cast<uintptr_t>(V)) & 15)
    return fail(FATHOM_ERR_INVALID, "rows8_read: the outputs must be 16-byte aligned");
  // wholly outside the store from there on: the kernel's sums do not wrap
  pos_value = pos_value > cap ? cap : pos_value < -R ? -R : pos_value;
  const ReadArgs a{{(const uint8_t *)k8, (const uint8_t *)v8}, {k_scale, v_scale}, {K, V}, pos, idx, pos_value, R, cap,
                   cdiv(cap, kBlk)};
  const int dt = dtype;
  FATHOM_ROWS8_DISPATCH(launch_read, a, BH, (hipStream_t)stream);
  return launch_status("rows8 read_kernel");
}
