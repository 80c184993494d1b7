// Attention of many queries over one K/V row of the 8-bit store, on the matrix
// cores: the kernel of chunk attention (a row's last T tokens, each over what it
// sees) and of a shared prefix (a batch's single tokens over the row that they share).
//
// For a query at place p of its row, with c the codes:
//   u_t = scale s_K(t) (q . cK_t)
//   z_t = softcap tanh(u_t / softcap) (u_t without a cap) + slope (t - p)
//   out = sum_t e^(z_t - m) s_V(t) cV_t / sum_t e^(z_t - m)
// over the tokens t < end, end = p + 1 (the prefix's length where it is shared), without those of
// [sinks, p + 1 - window).
#pragma once

#include "rows8_core.hpp"

namespace fathom {
namespace rows8 {

struct MultiArgs {
  const void *q;  // query (o, g) of row r at r q_row + g q_head + o q_out, in elements: o a token, or a sequence of the batch
  int64_t q_row, q_head, q_out;
  const uint8_t *k8, *v8;
  const float *ks, *vs;
  int64_t cap, nblk;
  const int32_t *lens;  // of the store's rows, or n
  int64_t n;
  int G, O, window, sinks;  // M = G O queries of a row
  bool shared;
  const int32_t *tails;  // shared: tokens of sequence (o, r) behind the prefix, [O, BH], or tail_n
  int64_t tail_n, tail_cap;
  int64_t BH;
  float scale, softcap;
  const float *slopes;  // [BH, G]; shared: [O, BH, G]
  void *out;            // [BH, G, O, D] of the queries' type; shared: written by the join, [O, BH, G, D] float32
  float2 *ml;           // [slots, rows of a tile] a split's (m, l)
  float *part;          // [slots, rows, D] its weighted rows
  int2 *where;          // [BH, tiles] a tile's first slot and its splits, where they are shared out on the device; else null
  int shares, tiles, rows;
  int splits;  // of every tile, where that is the same for all: tile t's slots begin at t splits; 0: see `where`
  bool parts;  // partial results are written, for the join
};

// What a tile of `rows` queries from the first one m0 of row r sees: blocks [0, sink) and, `skip` blocks further, up to
// nb in all; `end` the last token's successor, len the row's length.
struct TileSpan {
  int len, end, sink, skip, nb;
  __device__ __forceinline__ int block(int i) const { return i < sink ? i : i + skip; }
};
__device__ __forceinline__ TileSpan tile_span(const MultiArgs &a, int64_t r, int m0) {
  TileSpan s;
  s.len = (int)row_length(a.lens, a.n, a.cap, r);
  int first = 0;  // the first token of the tile's windows
  s.end = s.len;
  if (!a.shared) {
    const int M = a.G * a.O, last = m0 + a.rows < M ? m0 + a.rows : M;
    const int64_t place = (int64_t)s.len - a.O + 1;
    const int64_t lo = place + (int)((unsigned)m0 / (unsigned)a.G) - a.window;
    const int64_t end = place + (int)((unsigned)(last - 1) / (unsigned)a.G);
    s.end = end < 0 ? 0 : (int)end;
    first = a.window > 0 && lo > 0 ? (int)lo : 0;
  }
  const int sinks = a.sinks < first ? a.sinks : first, from = first / kBlk;
  s.sink = (sinks + kBlk - 1) / kBlk;
  s.sink = s.sink < from ? s.sink : from;
  s.skip = from - s.sink;
  s.nb = (s.end + kBlk - 1) / kBlk - s.skip;
  if (s.nb < 0) s.nb = 0;
  return s;
}

// Four floats at element `at` of an output of type DT.
template <int DT>
__device__ __forceinline__ void store4(void *out, int64_t at, const float (&v)[4]) {
  if constexpr (DT == FATHOM_DT_F32) {
    *reinterpret_cast<float4 *>(static_cast<float *>(out) + at) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    const u32x2v w = {pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3])};
    *reinterpret_cast<u32x2v *>(static_cast<uint16_t *>(out) + at) = w;
  }
}

#ifdef FATHOM_ROWS8_MULTI_KERNEL
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// A weight is 2^(z - base), the base a whole number that is raised where a score passes it by kMost, to kStart below
// the score, so that the rows' sums are scaled anew only where a score has grown by 2^3 (a row's first blocks).
// The largest weight times scale is held between 2^10 and 2^15, so f16 (to 2^-24) ends at 2^-34 of it.
constexpr uint32_t kLeastBlocks = 4;  // of a workgroup's share
constexpr float kMost = 15.0f, kStart = 12.0f;
// Bases from which 11-bit weights take scores relative to them first: below, V's factor joins the base in the exponent, where it is
// rounded with it, by 2^-16 at most here.  (Bases of 2^17 would leave weights 2^-7 off, of 2^26 a factor of 8.)
constexpr float kNear = 256.0f;
constexpr float kLeastWeight = -112.0f;  // a block counts with that weight at least in the choice of its values' scale: it stays finite

__device__ __forceinline__ float power(float e) { return ldexpf(1.0f, (int)__builtin_amdgcn_fmed3f(e, -300.0f, 300.0f)); }

// Bytes 0, 1 (HI: 2, 3) of a dword of codes as two bf16 values (exact); int8 codes as pair16 takes them.
template <bool I8, bool HI>
__device__ __forceinline__ uint32_t pair_bf16(uint32_t w) {
  if constexpr (I8) {  // under 0x4B0000 a byte u is the float 2^23 + u
    const float x = __uint_as_float(__builtin_amdgcn_perm(0x4B000000u, w, HI ? 0x070C0C02u : 0x070C0C00u)) - 8388736.0f;
    const float y = __uint_as_float(__builtin_amdgcn_perm(0x4B000000u, w, HI ? 0x070C0C03u : 0x070C0C01u)) - 8388736.0f;
    return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)x, (__bf16)y});
  } else {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.0f, HI));
  }
}

__device__ __forceinline__ uint32_t dword_of(uint32_t v, int) { return v; }
__device__ __forceinline__ uint32_t dword_of(uint16_t v, int) { return v; }
__device__ __forceinline__ uint32_t dword_of(u32x2v v, int d) { return v[d]; }
// The top bits of a dword's bytes that hold an e4m3 NaN (0x7F, 0xFF).
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ void clear_nans(uint32_t &w) { w &= ~((nan_bytes(w) >> 7) * 0xFFu); }
__device__ __forceinline__ void clear_nans(uint16_t &w) {
  uint32_t x = w;
  clear_nans(x);
  w = (uint16_t)x;
}
__device__ __forceinline__ void clear_nans(u32x2v &w) {
  w[0] &= ~((nan_bytes(w[0]) >> 7) * 0xFFu);
  w[1] &= ~((nan_bytes(w[1]) >> 7) * 0xFFu);
}

// tanh of |u| < 1/2, a fit of u + u^3 P(u^2): P of degree 3 is off by 2^-26, of degree 2 by 2^-20.5, which is below what a chain of 64
// products may be off by, and far below a weight of 11 bits.
template <bool PREC>
__device__ __forceinline__ float tanh_near(float u) {
  const float w = u * u;
  float p;
  if constexpr (PREC) {
    p = fmaf(0.01724146865f, w, -0.05304548144f);
    p = fmaf(p, w, 0.13325878978f);
    p = fmaf(p, w, -0.33333143592f);
  } else {
    p = fmaf(-0.0447505787f, w, 0.13205356896f);
    p = fmaf(p, w, -0.33328157663f);
  }
  return fmaf(u * w, p, u);
}
// tanh without a branch: the compiler would make one of its select, for every score by itself.
template <bool PREC>
__device__ __forceinline__ float tanh_both(float u) {
  const float t = __builtin_amdgcn_exp2f(fabsf(u) * (-2.0f * kLog2e));
  const float n = 1.0f - t, d = 1.0f + t, r = __builtin_amdgcn_rcpf(d);
  float far = n * r;
  far = fmaf(fmaf(-far, d, n), r, far);
  const uint32_t near = fabsf(u) < 0.5f ? 0xFFFFFFFFu : 0u;
  return __uint_as_float((__float_as_uint(tanh_near<PREC>(u)) & near) | (__float_as_uint(copysignf(far, u)) & ~near));
}

// Two floats as f16, to nearest, and what that leaves of them.
__device__ __forceinline__ f16x2 round16(float x, float y) {
  typedef float f32x2v __attribute__((ext_vector_type(2)));
  return __builtin_convertvector(f32x2v{x, y}, f16x2);
}

__device__ __forceinline__ void barrier_lds() {  // waits for LDS only: loads of the next tile stay on their way
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

__device__ __forceinline__ float other_half(float v) {  // of lane l ^ 32
  const uint32_t x = __float_as_uint(v);
  const auto p = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return __uint_as_float((threadIdx.x & 32) ? p[0] : p[1]);
}

// The part of a workgroup where tiles are shared out: its tile (of all rows'), split, the tile's splits (0: the call needs
// no such workgroup) and blocks per split.
struct Share {
  int tile, split, active, per;
};
struct FindTile {
  uint64_t total[8];
  uint32_t wave[8];
  int share[4];
};
// Every workgroup takes `per` blocks, so that the tile that sees most does not hold the call up: each sums all tiles'
// blocks, which gives `per`, and finds its tile in the prefix sums of ceil(blocks / per).  Those are at most
// `shares` + tiles, the grid.  A thread takes some tiles in a row; workgroup 0 writes down where all begin.
template <int WAVES>
__device__ __forceinline__ Share find_tile(const MultiArgs &a, int w, FindTile &sh) {
  const int tid = threadIdx.x, wave = tid >> 6, n = (int)a.BH * a.tiles;
  const int c = (n + WAVES * kWave - 1) / (WAVES * kWave), i0 = tid * c;
  auto blocks = [&](int i) {
    const int r = i / a.tiles;
    return i < n ? (uint32_t)tile_span(a, r, (i - r * a.tiles) * a.rows).nb : 0u;
  };
  uint64_t sum = 0;  // tiles of one row count its blocks each
  for (int i = 0; i < c; ++i) sum += blocks(i0 + i);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if ((tid & 63) == 0) sh.total[wave] = sum;
  if (tid == 0) sh.share[2] = 0;
  __syncthreads();
  uint64_t total = 0;
#pragma unroll
  for (int v = 0; v < WAVES; ++v) total += sh.total[v];
  const uint64_t even = (total + a.shares - 1) / a.shares;
  const uint32_t per = even > kLeastBlocks ? (uint32_t)even : kLeastBlocks;
  uint32_t own = 0;
  for (int i = 0; i < c; ++i) own += (blocks(i0 + i) + per - 1) / per;
  uint32_t upto = wave_incl_scan_u32(own);
  if ((tid & 63) == 63) sh.wave[wave] = upto;
  __syncthreads();
  for (int v = 0; v < wave; ++v) upto += sh.wave[v];
  uint32_t at = upto - own;
  if (w == 0 || ((uint32_t)w >= at && (uint32_t)w < upto))
    for (int i = 0; i < c; ++i) {
      const uint32_t act = (blocks(i0 + i) + per - 1) / per;
      if ((uint32_t)w >= at && (uint32_t)w < at + act) {
        sh.share[0] = i0 + i;
        sh.share[1] = w - (int)at;
        sh.share[2] = (int)act;
      }
      if (w == 0 && i0 + i < n) a.where[i0 + i] = make_int2((int)at, (int)act);
      at += act;
    }
  __syncthreads();
  return Share{__builtin_amdgcn_readfirstlane(sh.share[0]), __builtin_amdgcn_readfirstlane(sh.share[1]),
               __builtin_amdgcn_readfirstlane(sh.share[2]), __builtin_amdgcn_readfirstlane((int)per)};
}

// Whether a wave has a SIMD's registers to itself: by itself it holds both operands of a block of 128 channels, to which float32
// queries, a cap or a bias add more than half of the registers take (4 x 4 capped queries of 8 rows of 262144 tokens 135 us
// with 73 registers spilled; 97).  Waves that share a block do better by twos (float32, capped, 8 x 4 x 1024 over 16384 tokens
// 888 us with 32 spilled outside the loop; 1199).
template <int D, int QT, bool EXTRA, int RW>
constexpr bool kWide = RW == 1 && D == 128 && (EXTRA || QT == FATHOM_DT_F32);

// A workgroup takes a tile of queries of one row, or one share of what they see; each wave has 32 of them.  A tile's queries
// are consecutive in (o, g), so that a chunk's tile is a few tokens of all heads.  RW waves share a block of the row, for 32 RW
// queries: four, or eight (one workgroup per CU).  Where a row has no more than 32, RW is one: all four waves of a workgroup
// have them all, and take blocks in turn.  Per 64-token block:
//   the codes are requested a block ahead.  Several waves convert them once and keep them in LDS as 16-bit numbers (exact): K
//     by tokens, V transposed, both with their 16-byte pieces in an order that spreads the lanes' reads over the banks (cycles lost
//     to conflicts per LDS instruction: 0.84 in 8 x 4 x 2048 queries over 65536 tokens, 2.2 at D = 64 with a cap and a bias).
//     A wave by itself takes its operands straight from the codes: the order of the channels inside K's contraction is
//     free, and so is that of V's channels over the tiles of the result, lane c's being kTiles c ..
//   S^T = K q^T (v_mfma_f32_32x32x16): lane l holds query l & 31 and 32 of the block's scores, so that maximum and sum
//     need one exchange, between l and l ^ 32.  bf16 and f16 queries are operands as they are; float32 ones are two f16, 22
//     bits, and where a wave has channels below 2^-18 of their query's largest that could move a score by 2^-25,
//     what is left of those, to 2^-76 of that largest, takes two more products, times 2^38.
//   O^T += V^T p^T with the weights in the layout that the scores come in, which fixes the order of the tokens in V's
//     operand.  A weight is one f16 (PREC: two, 22 bits) of p s_V 2^-E, E the exponent of the largest p s_V so far, so
//     that blocks of small values with large weights count fully.
//
// Bound: for many queries the matrix cores and the vector instructions between them, which the two waves of a SIMD overlap
// in part.  8 x 4 x 2048 queries over 65536 tokens (2.16 TFLOP): 2.22 ms, 970 TFLOP/s, 80 % of what an 8192^3 bf16 product
// reaches (1200); tiles of four waves 2.44 ms, and eight with the last four half a block behind the others 2.28.  For up to 32
// queries HBM: 8 rows of 262144 tokens (0.54 GB) 89 us, 6.0 TB/s.
template <int D, bool I8, int QT, bool PREC, bool EXTRA, int RW>
__global__ __launch_bounds__((RW == 8 ? 8 : 4) * kWave, (kWide<D, QT, EXTRA, RW>) ? 1 : 2) void multi_kernel(MultiArgs a) {
  constexpr bool kBf16 = QT == FATHOM_DT_BF16;
  constexpr int kParts = QT == FATHOM_DT_F32 ? 2 : 1, kSteps = D / 16, kTiles = D / 32;
  constexpr bool kDirect = RW == 1;  // operands straight from the codes, without LDS
  constexpr int kThreads = RW * kWave, kBufs = 2, kRows = 32 * RW;  // threads that share a block
  // Operands read ahead.  Fewer where registers are short (float32 queries take twice as many, caps and biases some), as
  // a spilled register's way back waits for all loads on theirs: 32 x 8 x 4 queries over 32768 tokens 121 us; 84.
  constexpr bool kLean = kDirect || (D == 128 && (kParts == 2 || EXTRA));
  constexpr int kAhead = kLean ? 2 : 4, kVBufs = kLean ? 1 : 2;
  constexpr int kWaves = RW == 8 ? 8 : 4, kGroups = kWaves / RW;  // of a workgroup
  constexpr bool kHalves = RW == 8 && D == 64;  // half of the threads stage K, the others V
  constexpr int kKeys = kHalves ? 1 : kBlk * D / 16 / kThreads;    // 16-byte pieces of K per thread
  constexpr int kCh = kDirect ? D / 32 : D == 64 || RW == 8 ? 4 : 8;        // channels of V per thread and item of four tokens
  constexpr int kItems = kHalves ? 1 : kBlk / 4 * D / kCh / kThreads;  // items per thread
  typedef typename std::conditional<kBf16, bf16x8, f16x8>::type frag;
  constexpr int kPitch = D + 4, kCodes = 2 * kBlk * D;  // of a row of sums; bytes of a block's K, or V, as 16-bit numbers
  __shared__ __attribute__((aligned(16))) char lds[kGroups][kDirect ? 32 * kPitch * 4 : 2 * kBufs * kCodes];
  __shared__ int odd[kGroups][2];  // the first and the last block that hold a NaN in V
  __shared__ FindTile find;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = wave / RW, tid = threadIdx.x % kThreads;
  const int col = lane & 31, half = lane >> 5;
  Share share{(int)(gridDim.y - 1 - blockIdx.y), 0, 1, 0};  // the tiles that see most come first
  int64_t r = blockIdx.x;
  if (a.parts) {  // uniform over the workgroup
    if (a.splits) share = Share{(int)blockIdx.x / a.splits, (int)blockIdx.x % a.splits, a.splits, 0};
    else share = find_tile<kWaves>(a, (int)blockIdx.x, find);
    if (share.active == 0) return;
    r = share.tile / a.tiles;
    share.tile %= a.tiles;
  }
  const int m0 = share.tile * kRows, M = a.G * a.O;
  const TileSpan span = tile_span(a, r, m0);
  if (a.splits) share.per = (span.nb + a.splits - 1) / a.splits;
  const int first = share.split * share.per;
  const int end_of = first + share.per, last = share.split + 1 < share.active && end_of < span.nb ? end_of : span.nb;

  // ---- the lane's query
  const int mine = m0 + 32 * (wave % RW) + col, m = mine < M ? mine : M - 1;
  const int64_t o_at = (unsigned)m / (unsigned)a.G, g = m - (int)o_at * a.G;
  int end = span.len, lo = 0;
  float back = 0.0f;  // the bias takes t - (end - 1) - back
  if (a.shared) {
    back = (float)(int)row_length(a.tails, a.tail_n, a.tail_cap, o_at * a.BH + r);
  } else {
    const int64_t e = (int64_t)span.len - a.O + 1 + o_at;
    end = e < 0 ? 0 : (int)e;
    lo = a.window > 0 && end > a.window ? end - a.window : 0;
  }
  const int from = a.sinks < lo ? a.sinks : lo;  // tokens of [from, lo) take no part
  const float slope = !EXTRA || !a.slopes ? 0.0f : a.slopes[a.shared ? (o_at * a.BH + r) * a.G + g : r * a.G + g] * kLog2e;
  frag qf[kParts][kSteps];
  int ex = 0;
  const int64_t q_at = r * a.q_row + g * a.q_head + o_at * a.q_out;
  auto channel = [&](int s) { return kDirect ? 32 * (s / 2) + 16 * half + 8 * (s % 2) : 16 * s + 8 * half; };  // of step s, eight of them
  // float32: times a block's scale of K, a bound of what two f16 of the wave's queries lack of their small channels, in scores times
  // 2^25; 0 without such channels
  float far = 0.0f;
  if constexpr (QT != FATHOM_DT_F32) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) qf[0][s] = *reinterpret_cast<const frag *>(static_cast<const uint16_t *>(a.q) + q_at + channel(s));
    if constexpr (kBf16) {  // times a power of two where products could pass float32's range: the largest |q| at 2^100 or more
      uint32_t big = 0;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const u32x4 w = __builtin_bit_cast(u32x4, qf[0][s]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t x = w[e] << 16 & 0x7FFF0000u, y = w[e] & 0x7FFF0000u;
          big = big > x ? big : x;
          big = big > y ? big : y;
        }
      }
      if (__builtin_expect(__any(big >= 0x71800000u), 0)) {
        ex = 60;
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int e = 0; e < 8; ++e) qf[0][s][e] = (__bf16)ldexpf((float)qf[0][s][e], -60);
      }
    }
  } else {
    float x[kSteps][8], big = 0.0f;
    int few = 0;  // small channels of the query
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      load8_q(a.q, QT, q_at + channel(s), x[s]);
#pragma unroll
      for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(x[s][e]));
    }
    big = fmaxf(big, other_half(big));
    if (big > 0.0f && big < INFINITY) {
      frexpf(big, &ex);
      ex -= 14;  // the largest |q| of the query in [2^13, 2^14)
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = ldexpf(x[s][e], -ex);
        qf[0][s][e] = (_Float16)v;
        qf[1][s][e] = (_Float16)(v - (float)(_Float16)v);
        few += small_channel(v);
      }
    few += __shfl_xor(few, 32);
    if (few) far = ldexpf(fabsf(a.scale) * (kLog2e * (I8 ? 128.0f : 448.0f)) * (float)few, ex);  // each lacks 2^-25 at most
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) far = fmaxf(far, __shfl_xor(far, x));
    far = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(far)));
  }
  const int exq = ex;
  // the scores' factor, scale log2 e or scale / softcap, as a fraction and a power of two
  float cm = EXTRA && a.softcap > 0.0f ? __builtin_amdgcn_fmed3f(a.scale / a.softcap, -3.0e38f, 3.0e38f) : a.scale * kLog2e;
  if (cm != 0.0f && fabsf(cm) < INFINITY) {
    int e;
    cm = frexpf(cm, &e);
    ex += e;
  }

  // ---- staging
  const int mine_v = kHalves ? tid % (kThreads / 2) : tid;
  u32x4 kr[kKeys];
  typedef typename std::conditional<kCh == 8, u32x2v, typename std::conditional<kCh == 4, uint32_t, uint16_t>::type>::type vpiece;
  vpiece vr[kItems][4];
  typedef const __attribute__((address_space(4))) float *scalar_ptr;
  const scalar_ptr ksp = (scalar_ptr)(a.ks + r * a.nblk), vsp = (scalar_ptr)(a.vs + r * a.nblk);
  float ks_next = 0.0f, vs_next = 0.0f;
  auto load_keys = [&](int i) __attribute__((always_inline)) {
    const int b = i < last ? span.block(i) : 0;
    const RowsWith<0> k(a.k8, r * a.cap, b, i < last ? span.end : 0, D);
#pragma unroll
    for (int x = 0; x < kKeys; ++x)  // direct: every other piece of token 32 (x / (kSteps / 2)) + col
      kr[x] = k.load16(kDirect ? (32 * (x / (kSteps / 2)) + col) * D + 32 * (x % (kSteps / 2)) + 16 * half : 16 * (x * kThreads + tid));
    ks_next = ksp[b];
    vs_next = vsp[b];
  };
  auto load_values = [&](int i) __attribute__((always_inline)) {
    // A load of 128 channels' values covers two whole lines: as streams they leave the caches to K, whose lines take four loads
    // each (8 rows of 262144 tokens, 4 x 4 queries: 105 us; 89.  With K as streams too 118).
    const RowsWith<kDirect && D == 128 ? kStream : 0> v(a.v8, r * a.cap, i < last ? span.block(i) : 0, i < last ? span.end : 0, D);
#pragma unroll
    for (int x = 0; x < kItems; ++x) {  // direct: channels kCh col .. of tokens 8 x + 4 half ..
      const int item = x * kThreads + mine_v, at = kDirect ? (8 * x + 4 * half) * D + kCh * col : item / (D / kCh) * 4 * D + item % (D / kCh) * kCh;
#pragma unroll
      for (int j = 0; j < 4; ++j) v.load(at + j * D, vr[x][j]);
    }
  };
  auto load = [&](int i) __attribute__((always_inline)) {
    load_keys(i);
    load_values(i);
  };
  auto mark = [&](int i) __attribute__((always_inline)) {
    atomicMin(&odd[group][0], i);
    atomicMax(&odd[group][1], i);
  };
  // A NaN among the thread's codes of V counts as 0, and is counted behind the loop.
  auto clear_values = [&](int i) __attribute__((always_inline)) {
    if constexpr (!I8) {
      uint32_t nan = 0;
#pragma unroll
      for (int x = 0; x < 4 * kItems; ++x)
#pragma unroll
        for (int d = 0; d < (kCh + 3) / 4; ++d) nan |= nan_bytes(dword_of(vr[x / 4][x % 4], d));
      if (__builtin_expect(nan != 0, 0)) {
        mark(i);
#pragma unroll
        for (int x = 0; x < 4 * kItems; ++x) clear_nans(vr[x / 4][x % 4]);
      }
    }
  };
  auto stage = [&](int buf, int i) __attribute__((always_inline)) {
    if (i >= last) return;
    if (!kHalves || tid < kThreads / 2) {
#pragma unroll
      for (int x = 0; x < kKeys; ++x) {
        const int at = x * kThreads + tid, tok = at / (D / 16), piece = at % (D / 16);
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t c = flip_sign<I8>(kr[x][e]);
          if constexpr (kBf16) {
            w[2 * e] = pair_bf16<I8, false>(c);
            w[2 * e + 1] = pair_bf16<I8, true>(c);
          } else {
            w[2 * e] = __builtin_bit_cast(uint32_t, pair16<I8, false>(c));
            w[2 * e + 1] = __builtin_bit_cast(uint32_t, pair16<I8, true>(c));
          }
        }
        char *row = lds[group] + 2 * buf * kCodes + tok * 2 * D;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<u32x4 *>(row + 16 * ((2 * piece + h) ^ (tok & (D / 8 - 1)))) = u32x4{w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]};
      }
    }
    if (kHalves && tid < kThreads / 2) return;
    clear_values(i);
#pragma unroll
    for (int x = 0; x < kItems; ++x) {
      const int item = x * kThreads + mine_v, quad = item / (D / kCh), ch0 = item % (D / kCh) * kCh;
      // tokens 4 quad ..: half (quad >> 1 & 1) of the piece that lane half quad & 1 reads for 16 tokens
      const int piece = (quad >> 3) * 4 + (quad >> 2 & 1) * 2 + (quad & 1);
      char *base = lds[group] + (2 * buf + 1) * kCodes + 8 * (quad >> 1 & 1);
#pragma unroll
      for (int d = 0; d < kCh / 4; ++d) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = flip_sign<I8>(dword_of(vr[x][j], d));
#pragma unroll
        for (int p = 0; p < 2; ++p) {  // channels 4 d + 2 p, + 1
          const uint32_t ab = __builtin_amdgcn_perm(w[1], w[0], p ? 0x07030602u : 0x05010400u);
          const uint32_t cd = __builtin_amdgcn_perm(w[3], w[2], p ? 0x07030602u : 0x05010400u);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int ch = ch0 + 4 * d + 2 * p + h;
            const u32x2v v = {__builtin_bit_cast(uint32_t, h ? pair16<I8, true>(ab) : pair16<I8, false>(ab)),
                              __builtin_bit_cast(uint32_t, h ? pair16<I8, true>(cd) : pair16<I8, false>(cd))};
            *reinterpret_cast<u32x2v *>(base + ch * 2 * kBlk + 16 * (piece ^ ((ch ^ ch >> 3) & 7))) = v;
          }
        }
      }
    }
  };

  f32x16 o[kTiles];
#pragma unroll
  for (int d = 0; d < kTiles; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;
  float base = kLowest, l = 0.0f, E = -1000.0f;

  // Bit 16 x + e: whether the query sees token at + 32 x + 8 (e / 4) + e % 4.  Those places rise with the bit, so the bits
  // of tokens before t are the lowest ones, four for each eight tokens.
  auto seen_of = [&](int at) __attribute__((always_inline)) {
    auto before = [&](int t) {
      const int n = t - at, bits = n <= 0 ? 0 : 4 * (n >> 3) + ((n & 7) < 4 ? n & 7 : 4);
      return bits >= 32 ? 0xFFFFFFFFu : (1u << bits) - 1u;
    };
    return before(end) & ~(before(lo) & ~before(from));
  };
  // ---- scores; operands are read kAhead products ahead
  f32x16 s[2];
  auto scores = [&](int buf, float ks) __attribute__((always_inline)) {
    const char *kb = lds[group] + 2 * buf * kCodes + col * 2 * D;
    frag kf[2][kAhead];
    auto key = [&](int x, int c) __attribute__((always_inline)) {  // of tokens 32 x .., step c
      if constexpr (kDirect) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t code = flip_sign<I8>(kr[x * (kSteps / 2) + c / 2][2 * (c & 1) + e]);
          if constexpr (kBf16) {
            w[2 * e] = pair_bf16<I8, false>(code);
            w[2 * e + 1] = pair_bf16<I8, true>(code);
          } else {
            w[2 * e] = __builtin_bit_cast(uint32_t, pair16<I8, false>(code));
            w[2 * e + 1] = __builtin_bit_cast(uint32_t, pair16<I8, true>(code));
          }
        }
        return __builtin_bit_cast(frag, u32x4{w[0], w[1], w[2], w[3]});
      } else {
        return *reinterpret_cast<const frag *>(kb + 64 * D * x + 16 * ((2 * c + half) ^ (col & (D / 8 - 1))));
      }
    };
    auto keys = [&](int n) __attribute__((always_inline)) {  // of products kAhead n ..: the block's two halves in turn
#pragma unroll
      for (int c = 0; c < kAhead; ++c) kf[n & 1][c] = key((kAhead * n + c) % 2, (kAhead * n + c) / 2);
    };
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[x][e] = 0.0f;
    keys(0);
#pragma unroll
    for (int n = 0; n < 2 * kSteps / kAhead; ++n) {
      if (n + 1 < 2 * kSteps / kAhead) keys(n + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = 0; c < kAhead; ++c)
#pragma unroll
        for (int p = kParts - 1; p >= 0; --p) {
          const int x = (kAhead * n + c) % 2, step = (kAhead * n + c) / 2;
          if constexpr (kBf16) s[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[n & 1][c], qf[p][step], s[x], 0, 0, 0);
          else s[x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[n & 1][c], qf[p][step], s[x], 0, 0, 0);
        }
    }
    if constexpr (QT == FATHOM_DT_F32) {
      // What two f16 leave of small channels, as two more, formed anew from the queries where scores could be off by 2^-25.  (32 x
      // 8 x 4 queries over 131072 tokens, one in thirty waves with such a channel: in every block 246 us; 174.)  In sums of their
      // own: in the others' chain the matrix cores end them 2^-46 below the largest channel, also where that meets a zero of K.
      if (__builtin_expect(!(fabsf(ks) * far <= 1.0f), 0)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          f32x16 t;
#pragma unroll
          for (int e = 0; e < 16; ++e) t[e] = 0.0f;
          auto left = [&](int c) __attribute__((always_inline)) {
            float x[8];
            load8_q(a.q, QT, q_at + channel(c), x);
            f16x8 v[2];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float rest = rest_of(ldexpf(x[e], -exq));
              v[0][e] = (_Float16)rest;
              v[1][e] = (_Float16)(rest - (float)v[0][e]);
            }
#pragma unroll
            for (int p = 1; p >= 0; --p) t = __builtin_amdgcn_mfma_f32_32x32x16_f16(key(h, c), v[p], t, 0, 0, 0);
          };
          if constexpr (kDirect) {  // the registers of K need constant places
#pragma unroll
            for (int c = 0; c < kSteps; ++c) left(c);
          } else {
#pragma unroll 1
            for (int c = 0; c < kSteps; ++c) left(c);
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) s[h][e] = fmaf(t[e], 0x1p-38f, s[h][e]);
        }
      }
    }
  };
  // ---- their weights, and the values' products
  auto block = [&](int buf, int i, float ks, float vs) __attribute__((always_inline)) {
    const int t0 = span.block(i) * kBlk;
    const bool edge = !__all(t0 + kBlk <= end && (t0 >= lo || t0 + kBlk <= from));
    const char *vb = lds[group] + (2 * buf + 1) * kCodes;
    f16x8 vf[kVBufs][kTiles];
    auto values = [&](int n) __attribute__((always_inline)) {  // of tokens 16 n ..
      if constexpr (kDirect) {
        f16x2 v[2][2][kTiles];  // of tokens 8 x + 4 half + 2 y, + 1 and channel kTiles col + d
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = flip_sign<I8>(dword_of(vr[2 * n + x][j], 0));
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int d = 0; d < kTiles; d += 2) {
              const uint32_t ab = __builtin_amdgcn_perm(w[2 * y + 1], w[2 * y], d ? 0x07030602u : 0x05010400u);
              v[x][y][d] = pair16<I8, false>(ab);
              v[x][y][d + 1] = pair16<I8, true>(ab);
            }
        }
#pragma unroll
        for (int d = 0; d < kTiles; ++d) vf[n % kVBufs][d] = join8(v[0][0][d], v[0][1][d], v[1][0][d], v[1][1][d]);
      } else {
#pragma unroll
        for (int d = 0; d < kTiles; ++d) {
          const int ch = 32 * d + col, piece = 2 * n + half;
          vf[n % kVBufs][d] = *reinterpret_cast<const f16x8 *>(vb + ch * 2 * kBlk + 16 * (piece ^ ((ch ^ ch >> 3) & 7)));
        }
      }
    };
    if (kVBufs == 2) values(0);
    float f = ldexpf(fabsf(ks) * fabsf(cm), ex);
    // never infinite: a score of 0 has to stay one; nor 0 without a cap: a score of -inf has to stay one too
    f = fabsf(ks) < INFINITY ? __builtin_amdgcn_fmed3f(f, EXTRA && a.softcap > 0.0f ? 0.0f : 1.2e-38f, 3.0e38f) : f;
    if ((ks < 0.0f) != (cm < 0.0f)) {
      asm volatile("");  // a branch, not selects in every block
#pragma unroll
      for (int x = 0; x < 2; ++x) s[x] = -s[x];
    }
    const int at = t0 + 4 * half;  // register e of s[x] is token at + 32 x + 8 (e / 4) + e % 4
    if (EXTRA && a.softcap > 0.0f) {
      float big = 0.0f;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          s[x][e] *= f;
          big = __builtin_elementwise_maximum(big, fabsf(s[x][e]));
        }
      if (__all(big < 0.5f)) {  // most blocks: scores well below the cap
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[x][e] = tanh_near<PREC>(s[x][e]);
      } else {
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
#pragma unroll
          for (int k = e; k < e + 4; ++k) s[k / 16][k % 16] = tanh_both<PREC>(s[k / 16][k % 16]);
          if (e < 28)  // four after four: all at once would spill a hundred registers
            asm volatile("" : "+v"(s[e / 16][e % 16]), "+v"(s[e / 16][e % 16 + 1]), "+v"(s[e / 16][e % 16 + 2]), "+v"(s[e / 16][e % 16 + 3]),
                              "+v"(s[(e + 4) / 16][(e + 4) % 16]), "+v"(s[(e + 5) / 16][(e + 5) % 16]),
                              "+v"(s[(e + 6) / 16][(e + 6) % 16]), "+v"(s[(e + 7) / 16][(e + 7) % 16]));
        }
      }
      f = a.softcap * kLog2e;
    }
    if (EXTRA && a.slopes) {
      const float b = slope * ((float)(at - (end - 1)) - back);
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[x][e] = fmaf(s[x][e], f, fmaf((float)(32 * x + 8 * (e / 4) + e % 4), slope, b));
      f = 1.0f;
    }
    if (edge) {
      asm volatile("");  // a branch, not selects in every block
      if (!(fabsf(ks) < INFINITY)) {  // behind the masks a factor of NaN would reach tokens that a query does not see
#pragma unroll
        for (int x = 0; x < 2; ++x) s[x] *= f;
        f = 1.0f;
      }
      if constexpr (kDirect) clear_values(i);  // what all queries see makes NaN by itself
      const uint32_t seen = seen_of(at);
#pragma unroll
      for (int b = 0; b < 32; ++b) {
        const uint32_t keep = (uint32_t)((int32_t)(seen << (31 - b)) >> 31), x = __float_as_uint(s[b / 16][b % 16]);
        s[b / 16][b % 16] = __uint_as_float((x & keep) | (0xFF800000u & ~keep));  // else -infinity
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e)  // NaN stays: its weights are NaN anyhow (fmaxf would first quieten every operand)
      mx = __builtin_elementwise_maximum(__builtin_elementwise_maximum(mx, s[0][e]), s[1][e]);
    mx *= f;
    if (__any(fabsf(mx) >= kLarge && fabsf(mx) < INFINITY)) {
#pragma unroll
      for (int x = 0; x < 2; ++x) s[x] *= f;
      f = 1.0f;
    }
    const float ev = (float)((int)((__float_as_uint(vs) >> 23) & 0xFF) - 127);  // |s_V| < 2^(ev + 1)
    if (__any(mx - base > kMost || fmaxf(mx - base, kLeastWeight) + ev - (kMost - 1.0f) > E)) {
      mx = __builtin_elementwise_maximum(mx, other_half(mx));
      const float to = mx - base > kMost ? floorf(mx) - kStart : base, up = to - base;
      const float most = ceilf(fmaxf(mx - to, kLeastWeight) + ev) - (kStart - 1.0f);
      const float was = E;
      E = fmaxf(was - up, most);
      l *= power(-up);
      const float by = power(was - E - up);
#pragma unroll
      for (int d = 0; d < kTiles; ++d) o[d] *= by;
      base = to;
    }
    // ---- weights and products, 16 tokens at a time.  A block's weights are added together first: alone, most would be lost
    // beside a large sum.  The factor wv of V multiplies weights of 22 bits; for those of 11 it goes into the exponent, and out of
    // the sum again.
    const float wv = ldexpf(fabsf(vs), -(int)E);
    float off = base;
    if (!PREC && __any(fabsf(base) >= kNear)) {
      asm volatile("");  // a branch, not selects in every block
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[x][e] = fmaf(s[x][e], f, -base);
      f = 1.0f;
      off = 0.0f;
    }
    // Where that factor is so small that weights which count in the sum would be lost in the products' operands, 11-bit ones
    // are added apart; below 2^-64 all of those are 0: the block has no value to add.
    const bool none = !(wv >= 0x1p-64f), small = PREC ? none : !(wv >= 0x1p-6f);
    if (__builtin_expect(__any(small), 0)) {
      const bool all = __all(none);
      float sum = 0.0f;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) sum += __builtin_amdgcn_exp2f(fmaf(s[x][e], f, -off));
      l += small && (!PREC || all) ? sum : 0.0f;
      if (all) {
        if constexpr (kDirect) clear_values(i);  // no product will make a NaN count
        return;
      }
    }
    if (vs < 0.0f) {  // not written by this store's writer
      asm volatile("");
#pragma unroll
      for (int d = 0; d < kTiles; ++d) o[d] = -o[d];
    }
    const float zero = PREC ? off : none ? INFINITY : off - __builtin_amdgcn_logf(wv);
    const float back_by = PREC ? 1.0f : small ? 0.0f : __builtin_amdgcn_rcpf(wv);
    float sum = 0.0f;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if (kDirect) __builtin_amdgcn_sched_barrier(0);
      if (kVBufs == 1) values(n);
      else if (n < 3) values(n + 1);
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = __builtin_amdgcn_exp2f(fmaf(s[n / 2][8 * (n % 2) + e], f, -zero));
      if constexpr (PREC) {
        sum += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] *= wv;
      }
      f16x2 hi[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) hi[e] = round16(w[2 * e], w[2 * e + 1]);
      if constexpr (!PREC) {  // the weights as they are held, so that they divide out
#pragma unroll
        for (int e = 0; e < 4; ++e) sum = __builtin_amdgcn_fdot2(hi[e], f16x2{(_Float16)1.0f, (_Float16)1.0f}, sum, false);
      }
      const f16x8 p = join8(hi[0], hi[1], hi[2], hi[3]);
      f16x8 rest;
      if constexpr (PREC) {
        f16x2 lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) lo[e] = round16(w[2 * e] - (float)hi[e].x, w[2 * e + 1] - (float)hi[e].y);
        rest = join8(lo[0], lo[1], lo[2], lo[3]);
      }
#pragma unroll
      for (int d = 0; d < kTiles; ++d) {
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[n % kVBufs][d], p, o[d], 0, 0, 0);
        if constexpr (PREC) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[n % kVBufs][d], rest, o[d], 0, 0, 0);
      }
    }
    l = fmaf(sum, back_by, l);
    if (vs < 0.0f) {
      asm volatile("");
#pragma unroll
      for (int d = 0; d < kTiles; ++d) o[d] = -o[d];
    }
  };

  if (tid < 2) odd[group][tid] = tid ? -1 : 0x7FFFFFFF;
  load(first + group);
  __syncthreads();  // `odd` is set before a thread changes it
  // Of a block that none of the wave's queries sees, nothing is formed.
  auto seen = [&](int i) __attribute__((always_inline)) {
    const int t0 = span.block(i) * kBlk;
    return __any(t0 < end && (t0 + kBlk > lo || t0 < from)) != 0;
  };
  // A block's scale of V, and 0 for one that is not finite: that is counted behind the loop.
  auto scale_of = [&](int i, float vs) __attribute__((always_inline)) {
    if (fabsf(vs) < INFINITY) return vs;
    if (lane == 0) mark(i);
    return 0.0f;
  };
  if constexpr (kDirect) {  // the next block's K is requested once the scores are formed, its V once the products are
    for (int i = first + group; i < last; i += kGroups) {
      const float ks = ks_next, vs = scale_of(i, vs_next);
      const bool some = seen(i);
      if (some) scores(0, ks);
      __builtin_amdgcn_sched_barrier(0);
      load_keys(i + kGroups);
      __builtin_amdgcn_sched_barrier(0);
      if (some) block(0, i, ks, vs);
      __builtin_amdgcn_sched_barrier(0);
      load_values(i + kGroups);
    }
    __syncthreads();
  } else {
    float ks = ks_next, vs = vs_next;
    stage(0, first);
    load(first + 1);
    barrier_lds();
    for (int i = first; i < last; ++i) {
      const int buf = (i - first) & 1;
      vs = scale_of(i, vs);
      if (seen(i)) {
        scores(buf, ks);
        block(buf, i, ks, vs);
      }
      ks = ks_next;
      vs = vs_next;
      stage(buf ^ 1, i + 1);
      load(i + 2);
      barrier_lds();
    }
  }

  // A NaN in V makes the results of the queries that see its token NaN in its channel, and no others; a scale of V that is
  // not finite in every channel.  Of the blocks between the first and the last that hold such, the product of what is NaN and
  // what is seen says where.
  if (__builtin_expect(odd[group][1] >= 0, 0)) {
#pragma unroll 1
    for (int i = odd[group][0]; i <= odd[group][1]; i += kGroups) {
      const int at = span.block(i) * kBlk + 4 * half;
      const uint32_t seen = seen_of(at);
      const bool whole = !(fabsf(vsp[span.block(i)]) < INFINITY);
#pragma unroll
      for (int d = 0; d < kTiles; ++d) {
        f32x16 hits;
#pragma unroll
        for (int e = 0; e < 16; ++e) hits[e] = 0.0f;
#pragma unroll 1
        for (int b = 0; b < 32; b += 8) {
          f16x8 is, sees;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int t = at + 2 * b + 8 * (e / 4) + e % 4;
            const uint32_t c = t < span.end ? a.v8[(r * a.cap + t) * D + (kDirect ? kTiles * col + d : 32 * d + col)] : 0u;
            is[e] = whole || (!I8 && (c & 0x7F) == 0x7F) ? (_Float16)1.0f : (_Float16)0.0f;
            sees[e] = seen >> (b + e) & 1 ? (_Float16)1.0f : (_Float16)0.0f;
          }
          hits = __builtin_amdgcn_mfma_f32_32x32x16_f16(is, sees, hits, 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = hits[e] > 0.0f ? NAN : o[d][e];
      }
    }
  }

  l += other_half(l);
  // What leaves the wave is relative to base + kStart, so that it stays finite: to the step that this sum takes, which is another
  // one from 2^26 on.
  const float top = base + kStart;
  const int down = (int)(top - base);
  const bool parts = a.parts;
  const int64_t slot = parts ? ((int64_t)blockIdx.x * kRows) : 0;
  if constexpr (kDirect) {  // ---- the waves' sums over their blocks
    __shared__ float wm[kWaves][32], wl[kWaves][32];
    typedef float piece __attribute__((ext_vector_type(kTiles)));
    float *mine_at = reinterpret_cast<float *>(lds[group]) + col * kPitch;
#pragma unroll
    for (int e = 0; e < 16; ++e) {  // register e of o[d] is channel kTiles (8 (e / 4) + 4 half + e % 4) + d
      piece v;
#pragma unroll
      for (int d = 0; d < kTiles; ++d) v[d] = ldexpf(o[d][e], (int)E - down);
      *reinterpret_cast<piece *>(mine_at + kTiles * (8 * (e / 4) + 4 * half + e % 4)) = v;
    }
    if (half == 0) {
      wm[wave][col] = top;
      wl[wave][col] = ldexpf(l, -down);
    }
    __syncthreads();
#pragma unroll
    for (int x = threadIdx.x; x < 32 * D / 4; x += kWaves * kWave) {
      const int row = x / (D / 4), c = 4 * (x % (D / 4));
      if (m0 + row >= M) break;
      float big = wm[0][row];
#pragma unroll
      for (int v = 1; v < kWaves; ++v) big = fmaxf(big, wm[v][row]);
      float L = 0.0f, out[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int v = 0; v < kWaves; ++v) {
        const float f = __builtin_amdgcn_exp2f(wm[v][row] - big);
        const float4 u = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(lds[v]) + row * kPitch + c);
        L = fmaf(wl[v][row], f, L);
        out[0] = fmaf(u.x, f, out[0]);
        out[1] = fmaf(u.y, f, out[1]);
        out[2] = fmaf(u.z, f, out[2]);
        out[3] = fmaf(u.w, f, out[3]);
      }
      if (parts) {
        if (c == 0) a.ml[slot + row] = make_float2(big, L);
        *reinterpret_cast<float4 *>(a.part + (slot + row) * D + c) = make_float4(out[0], out[1], out[2], out[3]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) out[k] = L == 0.0f ? 0.0f : out[k] / L;
        const int at_o = (unsigned)(m0 + row) / (unsigned)a.G, at_g = m0 + row - at_o * a.G;
        store4<QT>(a.out, ((r * a.G + at_g) * a.O + at_o) * D + c, out);
      }
    }
    return;
  }
  if (mine >= M) return;
  const int row = 32 * wave + col;
  if (parts && half == 0) a.ml[slot + row] = make_float2(top, ldexpf(l, -down));
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t out_at = ((r * a.G + g) * a.O + o_at) * D + 4 * half;
#pragma unroll
  for (int d = 0; d < kTiles; ++d)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int c = 32 * d + 2 * e;
      float v[4];
      if (parts) {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = ldexpf(o[d][e + k], (int)E - down);
        *reinterpret_cast<float4 *>(a.part + (slot + row) * D + c + 4 * half) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = ldexpf(o[d][e + k] * inv, (int)E);
        store4<QT>(a.out, out_at + c, v);
      }
    }
}

template <int D, bool I8, int QT, bool PREC, bool EXTRA>
void launch_multi(const MultiArgs &a, hipStream_t st) {
  constexpr bool kFour = EXTRA || QT == FATHOM_DT_F32;  // the host gives such calls no tiles of 256
  const dim3 grid = a.splits  ? dim3((unsigned)(a.splits * a.BH * a.tiles))
                    : a.parts ? dim3((unsigned)(a.shares + a.BH * a.tiles))
                              : dim3((unsigned)a.BH, (unsigned)a.tiles);
  if (a.rows == 32) multi_kernel<D, I8, QT, PREC, EXTRA, 1><<<grid, 4 * kWave, 0, st>>>(a);
  else if (kFour || a.rows == 128) multi_kernel<D, I8, QT, PREC, EXTRA, 4><<<grid, 4 * kWave, 0, st>>>(a);
  else multi_kernel<D, I8, QT, PREC, EXTRA, kFour ? 4 : 8><<<grid, 8 * kWave, 0, st>>>(a);
}
template <int D, bool I8, int QT, bool PREC>
void launch_multi(const MultiArgs &a, hipStream_t st) {
  if (a.softcap > 0.0f || a.slopes) launch_multi<D, I8, QT, PREC, true>(a, st);
  else launch_multi<D, I8, QT, PREC, false>(a, st);
}
template <int D, bool I8>
void launch_multi(const MultiArgs &a, int q_dtype, hipStream_t st) {
  if (q_dtype == FATHOM_DT_F32) launch_multi<D, I8, FATHOM_DT_F32, true>(a, st);
  else if (q_dtype == FATHOM_DT_F16 && a.shared) launch_multi<D, I8, FATHOM_DT_F16, true>(a, st);
  else if (q_dtype == FATHOM_DT_F16) launch_multi<D, I8, FATHOM_DT_F16, false>(a, st);
  else if (a.shared) launch_multi<D, I8, FATHOM_DT_BF16, true>(a, st);
  else launch_multi<D, I8, FATHOM_DT_BF16, false>(a, st);
}

}  // namespace
#endif

// Launches multi_kernel; one for each head size and code type, as they take long to compile.
void launch_multi_d64_e4m3(const MultiArgs &a, int q_dtype, hipStream_t st);
void launch_multi_d64_int8(const MultiArgs &a, int q_dtype, hipStream_t st);
void launch_multi_d128_e4m3(const MultiArgs &a, int q_dtype, hipStream_t st);
void launch_multi_d128_int8(const MultiArgs &a, int q_dtype, hipStream_t st);

}  // namespace rows8
}  // namespace fathom
