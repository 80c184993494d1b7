// Queries and keys on their way from a layer's projections into the 8-bit K/V row
// store: a norm over each head's channels, the position rotation, and the write.
//
// Token i of row bh, at place p = pos + i of the store and position t = p + offset:
//   x' = x / sqrt(mean(x^2) + eps) * weight            where weights are given
//   (y_c, y_{c + r/2}) = (a cos - b sin, b cos + a sin), a = x'_c, b = x'_{c + r/2}, angle t inv_freq[c], c < r / 2
//   y_c = x'_c                                          for c >= r
// for each query head and for K (the rotate-half convention of scripts/common.py:44-47); K's y and V
// are quantised as rows8_write does.  All in float32 but the angle, which is formed and reduced in
// fixed point (see turn_of).
#include "rows8.hpp"

namespace fathom {
namespace rows8 {
namespace {

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kHeads = 4;           // of a workgroup of queries, which turn by the same angles
constexpr int64_t kFill = 2048;     // workgroups of queries: fewer heads each where there would not be as many
constexpr int64_t kMaxRotate = 1 << 27;  // tokens of a call: its grid stays below 2^32 threads

struct RotateArgs {
  const void *q, *x[2];  // x: K, V
  int64_t q_row, q_head, q_tok, row_stride[2], tok_stride[2];  // in elements
  uint8_t *codes[2];
  float *scale[2];
  const int32_t *pos, *offset;
  int64_t pos_value, offset_value;
  const float *inv_freq;
  int turn;  // r
  const void *weight[2];  // of queries and of keys
  int weight_dtype;
  float eps;
  int64_t G, T, cap, nblk;
  void *q_out, *k_out;
  int kv_blocks;  // workgroups of K, and of V, per row; the others take queries
  int q_tokens;   // tokens of a workgroup of queries, a power of two
  int q_heads;    // and its heads, of consecutive workgroups
  int q_parts;    // workgroups that share its tokens
};

// A thread holds sixteen channels of a row, as eight pairs that turn together: channels a .. a + 7 and b .. b + 7.
template <int D>
struct Lane {
  static constexpr int kLanes = D / 16;             // lanes of a row
  static constexpr int kSlots = kThreads / kLanes;  // rows that a workgroup holds at a time
  static constexpr int kPasses = kBlk / kSlots;     // of a block
};
struct Pairs {
  int a, b;
  bool turned;
};
template <int D>
__device__ __forceinline__ Pairs pairs_of(int turn) {
  const int c = 8 * (threadIdx.x % Lane<D>::kLanes);
  if (2 * c < turn) return Pairs{c, c + turn / 2, true};
  return Pairs{turn / 2 + c, D / 2 + c, false};  // of the channels behind r, which stay
}

template <int DT>
struct Raw {
  u32x4 w[DT == FATHOM_DT_F32 ? 4 : 2];
};
template <int DT>
__device__ __forceinline__ Raw<DT> load_pairs(const void *x, int64_t at, Pairs c) {
  Raw<DT> r;
  if constexpr (DT == FATHOM_DT_F32) {
    const float *p = static_cast<const float *>(x) + at;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      r.w[h] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p + c.a + 4 * h));
      r.w[2 + h] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p + c.b + 4 * h));
    }
  } else {
    const uint16_t *p = static_cast<const uint16_t *>(x) + at;
    r.w[0] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p + c.a));
    r.w[1] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p + c.b));
  }
  return r;
}
template <int DT>
__device__ __forceinline__ void unpack_pairs(const Raw<DT> &r, float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 4 * (int)(sizeof(r.w) / 16); ++i) {
    const uint32_t w = r.w[i / 4][i % 4];
    if constexpr (DT == FATHOM_DT_F32) x[i] = __uint_as_float(w);
    else unpack2<DT>(w, x[2 * i], x[2 * i + 1]);
  }
}
template <int DT>
__device__ __forceinline__ void store_pairs(void *out, int64_t at, Pairs c, const float (&x)[16]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t o = at + (h ? c.b : c.a);
    if constexpr (DT == FATHOM_DT_F32) {
      typedef float f32x4 __attribute__((ext_vector_type(4)));
      f32x4 *p = reinterpret_cast<f32x4 *>(static_cast<float *>(out) + o);
      __builtin_nontemporal_store(f32x4{x[8 * h], x[8 * h + 1], x[8 * h + 2], x[8 * h + 3]}, p);
      __builtin_nontemporal_store(f32x4{x[8 * h + 4], x[8 * h + 5], x[8 * h + 6], x[8 * h + 7]}, p + 1);
    } else {
      const u32x4 w = {pack2<DT>(x[8 * h], x[8 * h + 1]), pack2<DT>(x[8 * h + 2], x[8 * h + 3]),
                       pack2<DT>(x[8 * h + 4], x[8 * h + 5]), pack2<DT>(x[8 * h + 6], x[8 * h + 7])};
      __builtin_nontemporal_store(w, reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(out) + o));
    }
  }
}

// The thread's sixteen weights, or ones.
__device__ __forceinline__ void load_weights(const void *w, int dt, Pairs c, float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int at = (i < 8 ? c.a : c.b) + i % 8;
    v[i] = !w ? 1.0f
           : dt == FATHOM_DT_F32 ? load_elem<FATHOM_DT_F32>(w, at)
           : dt == FATHOM_DT_F16 ? load_elem<FATHOM_DT_F16>(w, at)
                                 : load_elem<FATHOM_DT_BF16>(w, at);
  }
}

// A frequency as turns per token, in fractions of 2^-64 of a turn: inv / (2 pi) in two float64, whole turns dropped.
__device__ __forceinline__ uint64_t turns_of(float inv) {
  constexpr double kTurn = 0.15915494309189534561, kRest = -9.8393383659123640e-18;  // 1 / (2 pi) in two parts
  const double hi = (double)inv * kTurn, lo = fma((double)inv, kTurn, -hi) + (double)inv * kRest;
  const double part = (hi - floor(hi)) * 0x1p32, whole = floor(part);
  return ((uint64_t)(uint32_t)whole << 32) + (uint64_t)(int64_t)rint((part - whole) * 0x1p32 + lo * 0x1p64);
}

// cos and sin of position t for the thread's pairs.  The angle is the product of t and the pair's turns, modulo whole turns by
// itself: its upper word is exact to 2^-31 of a turn whatever t.  In quarter turns n + f, |f| <= 1/2, x = f pi / 2: sin x = x + x^3
// P(x^2), cos x = 1 - x^2 / 2 + x^4 Q(x^2), P and Q least-squares fits of degree 2 on |x| <= pi / 4, off by less than a step of
// float32 each.  (Angles in float64, half as fast: 8 x 32768 tokens of 4 heads 176 us; 163.)
__device__ __forceinline__ void turn_of(const uint64_t (&turns)[8], int64_t t, float (&cs)[8], float (&sn)[8]) {
  const uint32_t lo = (uint32_t)t, hi = (uint32_t)((uint64_t)t >> 32);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t f0 = (uint32_t)turns[i], f1 = (uint32_t)(turns[i] >> 32);
    const uint32_t phase = __umulhi(lo, f0) + lo * f1 + hi * f0;  // 2^-32 of a turn
    const uint32_t n = (phase + 0x20000000u) >> 30;
    const float x = (float)(int32_t)(phase - (n << 30)) * 1.4629180792671596e-9f, w = x * x;  // 2 pi / 2^32
    float p = fmaf(w, -0.00019515919848345220f, 0.00833216588944196700f);
    p = fmaf(p, w, -0.16666655242443085f);
    const float s = fmaf(x * w, p, x);
    float k = fmaf(w, 2.4435816158074886e-5f, -0.0013887340901419520f);
    k = fmaf(k, w, 0.04166664555668831f);
    k = fmaf(fmaf(k, w, -0.5f), w, 1.0f);
    sn[i] = __uint_as_float(__float_as_uint(n & 1 ? k : s) ^ (n & 2) << 30);
    cs[i] = __uint_as_float(__float_as_uint(n & 1 ? s : k) ^ ((n + 1) & 2) << 30);
  }
}

template <int D>
__device__ __forceinline__ void norm(float (&x)[16], const float (&w)[16], float eps) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) s = fmaf(x[i], x[i], s);
#pragma unroll
  for (int o = 1; o < Lane<D>::kLanes; o *= 2) s += __shfl_xor(s, o);
  const float by = 1.0f / sqrtf(s / D + eps);
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = x[i] * by * w[i];
}
// Channels that stay are not turned by 0, which would make NaN of a finite one beside an infinite one.
__device__ __forceinline__ void turn(float (&x)[16], Pairs c, const float (&cs)[8], const float (&sn)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = x[i], b = x[8 + i];
    x[i] = c.turned ? a * cs[i] - b * sn[i] : a;
    x[8 + i] = c.turned ? b * cs[i] + a * sn[i] : b;
  }
}

// Workgroups of three kinds, per row: a block of K, a block of V, queries.  A row of D channels is D / 16 lanes', so that a
// pair's channels are in one thread and a head's norm is a sum over 4 or 8 lanes; a block's rows stay in registers between its
// largest value and its codes.  A workgroup's query tokens are as many as there are, up to its rows, and its heads the rest, so that
// a token's angles are formed once for up to four heads (fewer where the call would not fill the device).
//
// Bound: HBM.  8 x 32768 tokens of 4 heads in bf16, D = 128, keys returned (0.81 GB in and out) 163 us at the least of 20 under
// a trace, 4.9 TB/s, what a copy reaches (4.97), 175 in the median; norms and angles by themselves take less.  16 x 1777 of 7
// heads, D = 64 (77 MB, much of it from L2) 19 us.  One token of 32 rows 8 us: the launch, the frequencies on their way to LDS and
// the barrier, then the weights and the row.
template <int D, int DT, bool I8>
__global__ __launch_bounds__(kThreads) void rotate_kernel(RotateArgs a) {
  typedef Lane<D> L;
  const int tid = threadIdx.x, slot = tid / L::kLanes;
  const int64_t bh = blockIdx.y;
  const int64_t p = a.pos ? (int64_t)a.pos[bh] : a.pos_value;
  const int64_t shift = a.offset ? (int64_t)a.offset[bh] : a.offset_value;
  const Pairs c = pairs_of<D>(a.turn);
  __shared__ uint64_t shared_turns[D / 2];
  if (2 * tid < a.turn) shared_turns[tid] = turns_of(a.inv_freq[tid]);
  __syncthreads();
  uint64_t turns[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) turns[i] = c.turned ? shared_turns[c.a + i] : 0;
  float w[16];
  if ((int)blockIdx.x >= 2 * a.kv_blocks) {  // ---- queries: a token's heads share its angles
    load_weights(a.weight[0], a.weight_dtype, c, w);
    const int unit = (int)blockIdx.x - 2 * a.kv_blocks, part = unit % a.q_parts;
    const int64_t i = (int64_t)(unit / a.q_parts) * a.q_tokens + slot % a.q_tokens;
    if (i >= a.T) return;  // whole rows' lanes
    const int64_t step = L::kSlots / a.q_tokens, at = bh * a.q_row + i * a.q_tok;
    const int64_t last = (int64_t)(part + 1) * a.q_heads, end = last < a.G ? last : a.G;
    int64_t g = (int64_t)part * a.q_heads + slot / a.q_tokens;
    Raw<DT> next{};
    if (g < end) next = load_pairs<DT>(a.q, at + g * a.q_head, c);
    float cs[8], sn[8];
    turn_of(turns, p + i + shift, cs, sn);
    for (; g < end; g += step) {  // the next head is requested first
      const Raw<DT> now = next;
      if (g + step < end) next = load_pairs<DT>(a.q, at + (g + step) * a.q_head, c);
      float x[16];
      unpack_pairs<DT>(now, x);
      if (a.weight[0]) norm<D>(x, w, a.eps);
      turn(x, c, cs, sn);
      store_pairs<DT>(a.q_out, ((bh * a.G + g) * a.T + i) * D, c, x);
    }
    return;
  }
  const int kv = (int)blockIdx.x >= a.kv_blocks;
  const bool fits = p >= 0 && p + a.T <= a.cap;  // else the row's tokens are not written
  // a row that does not fit is still turned, in blocks that begin with its first token
  const int64_t blk = (fits ? p / kBlk : 0) + ((int)blockIdx.x - (kv ? a.kv_blocks : 0));
  const int64_t t0 = blk * kBlk, lead = fits ? p : 0;
  if (t0 >= lead + a.T || (!fits && (kv || !a.k_out))) return;
  float *scale = a.scale[kv] + bh * a.nblk + blk;
  const float was = fits ? *scale : 0.0f;
  __shared__ float wave_max[kThreads / kWave];
  Raw<DT> raw[L::kPasses];
#pragma unroll
  for (int i = 0; i < L::kPasses; ++i) {
    const int64_t j = t0 + i * L::kSlots + slot - lead;  // index among the new tokens
    raw[i] = Raw<DT>{};
    if (j >= 0 && j < a.T) raw[i] = load_pairs<DT>(a.x[kv], bh * a.row_stride[kv] + j * a.tok_stride[kv], c);
  }
  if (!kv) load_weights(a.weight[1], a.weight_dtype, c, w);
  float x[L::kPasses][16], amax = 0.0f;
#pragma unroll
  for (int i = 0; i < L::kPasses; ++i) {
    const int64_t j = t0 + i * L::kSlots + slot - lead;
    unpack_pairs<DT>(raw[i], x[i]);
    if (!kv) {
      if (a.weight[1]) norm<D>(x[i], w, a.eps);
      float cs[8], sn[8];
      turn_of(turns, p + j + shift, cs, sn);
      turn(x[i], c, cs, sn);
      if (a.k_out && j >= 0 && j < a.T) store_pairs<DT>(a.k_out, (bh * a.T + j) * D, c, x[i]);
    }
    if (j >= 0 && j < a.T) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float v = fabsf(x[i][e]);
        if (v < INFINITY) amax = fmaxf(amax, v);  // NaN and infinities take no part
      }
    }
  }
  if (!fits) return;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
  if ((tid & 63) == 0) wave_max[tid >> 6] = amax;
  __syncthreads();
  amax = fmaxf(fmaxf(wave_max[0], wave_max[1]), fmaxf(wave_max[2], wave_max[3]));
  const float need = fmaxf(amax / code_max<I8>(), kMinScale);
  const int earlier = (int)(p > t0 ? p - t0 : 0);  // tokens that the block holds already
  const BlockScale to = block_scale(was, need, earlier);
  const float inv = 1.0f / to.s;
  uint8_t *dst = a.codes[kv] + (bh * a.cap + t0) * D;
#pragma unroll
  for (int i = 0; i < L::kPasses; ++i) {
    const int r = i * L::kSlots + slot;
    const int64_t j = t0 + r - p;
    if (j < 0 || j >= a.T) continue;
    uint32_t code[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float y[4] = {x[i][4 * e] * inv, x[i][4 * e + 1] * inv, x[i][4 * e + 2] * inv, x[i][4 * e + 3] * inv};
      code[e] = encode4<I8>(y);
    }
    __builtin_nontemporal_store(u32x2{code[0], code[1]}, reinterpret_cast<u32x2 *>(dst + r * D + c.a));
    __builtin_nontemporal_store(u32x2{code[2], code[3]}, reinterpret_cast<u32x2 *>(dst + r * D + c.b));
  }
  if (to.f != 1.0f) rescale_codes<I8>(dst, earlier * D, to.f, tid, kThreads);
  if (tid == 0) *scale = to.s;
}

template <int D, int DT, bool I8>
void launch_rotate(RotateArgs a, int64_t BH, hipStream_t st) {
  a.kv_blocks = (int)cdiv(a.T + kBlk - 1, kBlk);  // T tokens touch at most so many
  a.q_tokens = 1;
  while (a.q_tokens < a.T && a.q_tokens < Lane<D>::kSlots) a.q_tokens *= 2;
  const int64_t units = cdiv(a.T, a.q_tokens), slots = Lane<D>::kSlots / a.q_tokens;  // heads of a pass
  int64_t heads = kHeads;
  while (heads > 1 && units * BH * cdiv(a.G, heads) < kFill) heads /= 2;
  a.q_heads = (int)(heads > slots ? heads : slots);
  a.q_parts = (int)cdiv(a.G, (int64_t)a.q_heads);
  const int64_t all = 2 * (int64_t)a.kv_blocks + units * a.q_parts;
  rotate_kernel<D, DT, I8><<<dim3((unsigned)all, (unsigned)BH), kThreads, 0, st>>>(a);
}

template <int D, int DT>
void launch_rotate(const RotateArgs &a, int64_t BH, bool i8, hipStream_t st) {
  if (i8) launch_rotate<D, DT, true>(a, BH, st);
  else launch_rotate<D, DT, false>(a, BH, st);
}

template <int D>
void launch_rotate(const RotateArgs &a, int64_t BH, int dtype, bool i8, hipStream_t st) {
  if (dtype == FATHOM_DT_F32) launch_rotate<D, FATHOM_DT_F32>(a, BH, i8, st);
  else if (dtype == FATHOM_DT_F16) launch_rotate<D, FATHOM_DT_F16>(a, BH, i8, st);
  else launch_rotate<D, FATHOM_DT_BF16>(a, BH, i8, st);
}

}  // namespace
}  // namespace rows8
}  // namespace fathom

using namespace fathom;
using namespace fathom::rows8;

extern "C" int fathom_rows8_write_rotated(const void *q, const void *K, const void *V, int dtype, int64_t q_row_stride,
                                          int64_t q_head_stride, int64_t q_tok_stride, int64_t k_row_stride,
                                          int64_t k_tok_stride, int64_t v_row_stride, int64_t v_tok_stride, const int32_t *pos,
                                          int64_t pos_value, const int32_t *offset, int64_t offset_value,
                                          const float *inv_freq, int64_t rotated, const void *q_weight, const void *k_weight,
                                          int weight_dtype, float eps, int64_t BH, int64_t G, int64_t T, int64_t D,
                                          int64_t cap, int code_dtype, void *k8, void *v8, float *k_scale, float *v_scale,
                                          void *q_out, void *k_out, void *stream) {
  const char *what = "rows8_write_rotated";
  int rc = check_store(what, k8, v8, k_scale, v_scale, code_dtype, BH, cap, D);
  if (rc) return rc;
  if (dtype < FATHOM_DT_F32 || dtype > FATHOM_DT_BF16) return fail(FATHOM_ERR_INVALID, "%s: dtype %d", what, dtype);
  if ((q_weight || k_weight) && (weight_dtype < FATHOM_DT_F32 || weight_dtype > FATHOM_DT_BF16))
    return fail(FATHOM_ERR_INVALID, "%s: weight_dtype %d", what, weight_dtype);
  if (G < 1 || G > kMaxRows) return fail(FATHOM_ERR_INVALID, "%s: G=%lld", what, (long long)G);
  if (T < 0 || T > cap) return fail(FATHOM_ERR_INVALID, "%s: T=%lld outside [0, cap=%lld]", what, (long long)T, (long long)cap);
  if (T > kMaxRotate) return fail(FATHOM_ERR_INVALID, "%s: T=%lld, at most %lld at a time", what, (long long)T, (long long)kMaxRotate);
  if (!pos && (pos_value < 0 || pos_value > cap - T))  // in this form, as a sum could wrap
    return fail(FATHOM_ERR_INVALID, "%s: %lld tokens from %lld outside [0, cap=%lld)", what, (long long)T, (long long)pos_value,
                (long long)cap);
  if (!offset && (offset_value < -0x80000000LL || offset_value > 0x7FFFFFFFLL))
    return fail(FATHOM_ERR_INVALID, "%s: offset %lld", what, (long long)offset_value);
  if (rotated < 0 || rotated > D || rotated % 16)
    return fail(FATHOM_ERR_INVALID, "%s: %lld rotated channels, not a multiple of 16 up to %lld", what, (long long)rotated, (long long)D);
  if (!(eps >= 0.0f && eps < INFINITY)) return fail(FATHOM_ERR_INVALID, "%s: eps must be finite and not negative", what);
  if (T == 0) return FATHOM_OK;
  if (!q || !K || !V || !q_out || (rotated && !inv_freq)) return fail(FATHOM_ERR_INVALID, "%s: null pointer", what);
  const int64_t size = dtype == FATHOM_DT_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(K) | reinterpret_cast<uintptr_t>(V) |
       reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(k_out)) & 15 ||
      ((q_row_stride | q_head_stride | q_tok_stride | k_row_stride | k_tok_stride | v_row_stride | v_tok_stride) * size) & 15)
    return fail(FATHOM_ERR_INVALID, "%s: q, K, V, the outputs and the strides must be multiples of 16 bytes", what);
  RotateArgs a{q, {K, V}, q_row_stride, q_head_stride, q_tok_stride, {k_row_stride, v_row_stride}, {k_tok_stride, v_tok_stride},
               {(uint8_t *)k8, (uint8_t *)v8}, {k_scale, v_scale}, pos, offset, pos_value, offset_value, inv_freq, (int)rotated,
               {q_weight, k_weight}, weight_dtype, eps, G, T, cap, cdiv(cap, kBlk), q_out, k_out, 0, 0};
  if (D == 128) launch_rotate<128>(a, BH, dtype, code_dtype == FATHOM_DT_I8, (hipStream_t)stream);
  else launch_rotate<64>(a, BH, dtype, code_dtype == FATHOM_DT_I8, (hipStream_t)stream);
  return launch_status("rows8 rotate_kernel");
}
