// Attention of single tokens over the 8-bit K/V row store: over a whole row (or
// its last tokens), or over listed tokens.
//
// With len the row's length and c the codes, for query head g of row bh:
//   u_t = scale s_K(t) (q . cK_t)
//   z_t = softcap tanh(u_t / softcap) (u_t without a cap) + slope_g (t - (len - 1))
//   out = sum_t e^(z_t - m) s_V(t) cV_t / sum_t e^(z_t - m)
// over the tokens t of [max(0, len - window), len) and of [0, sinks), or the listed ones of [0, len).
// Scores, maxima, sums and the weighted rows are float32.
#include "rows8_core.hpp"

namespace fathom {
namespace rows8 {
namespace {

constexpr int kTile = 32;  // listed positions of a wave at a time
constexpr int kMergeThreads = 256;
constexpr int kDenseWaves = 4;     // of a workgroup that takes a split of a row
constexpr int kDenseTotal = 2048;  // waves of a dense call: eight per CU, all at work at once
constexpr int kMaxSplits = 512;  // of a query head
constexpr float kNoValue = -1000.0f;  // log2 of the largest weight times scale before any
constexpr float kLeast = -112.0f;     // a block counts there with that weight at least: 2^14 s_V / (weight s_V) is finite

struct AttnArgs {
  const void *q;
  int q_dtype;
  const uint8_t *k8, *v8;
  const float *ks, *vs;
  int64_t G, cap, nblk;
  const int32_t *lens;
  int64_t n, window, sinks;
  const int64_t *idx;
  int64_t k;
  float scale, softcap;
  const float *slopes;
  float *out;
  float2 *ml;   // [slots, G] a split's (m, l): slot bh nsplit + split, or where[bh].x + split
  float *part;  // [slots, G, D] its weighted rows
  int2 *where;  // [BH] a row's first slot and its splits, where lengths are on the device; else null
  int64_t nsplit, BH, groups;
  bool join;  // the caller joins the results with others: every row leaves partial ones
};

// The factor that the queries take before the product, (scale log2 e, or scale /
// softcap), as a fraction in [1/2, 1) that multiplies q and a power of two for the
// scale of K: a rounding there would shift all scores of a block alike, in q they average out.
__device__ __forceinline__ float query_factor(const AttnArgs &a, int &e) {
  const float c = a.softcap > 0.0f ? fminf(fmaxf(a.scale / a.softcap, -3.0e38f), 3.0e38f) : a.scale * kLog2e;
  e = 0;
  return c == 0.0f || !(fabsf(c) < INFINITY) ? c : frexpf(c, &e);
}

// Sum over the LANES lanes (4 or 8) that hold one row; row_half_mirror pairs quads
// whose lanes already agree.
template <int LANES>
__device__ __forceinline__ float sum_row(float v) {
  v += dpp<kXor1>(v);
  v += dpp<kXor2>(v);
  if constexpr (LANES == 8) v += dpp<kHalfMirror>(v);
  return v;
}
// Sum or maximum over the wave's groups of LANES lanes, lane by lane; first inside a row of 16.
template <int LANES, bool MAX>
__device__ __forceinline__ float over_row16(float v) {
  if constexpr (LANES == 4) v = MAX ? fmaxf(v, dpp<kRor4>(v)) : v + dpp<kRor4>(v);
  return MAX ? fmaxf(v, dpp<kXor8>(v)) : v + dpp<kXor8>(v);
}
template <int LANES, bool MAX>
__device__ __forceinline__ float over_rows(float v) {
  return across_groups<MAX>(over_row16<LANES, MAX>(v));
}

__device__ const u32x4 kNoRow[8] = {};  // the row of a token that takes no part

// Attention over listed tokens: one workgroup of NW waves per (split, query head,
// row); its waves take tiles of 32 positions in turn.  A row is 16 channels in
// each of D / 16 lanes, and those lanes keep a softmax of their own (maximum, sum,
// weighted rows) over the positions they see, so that nothing crosses lanes inside
// the loop but the score's sum.  All pieces of a tile, K's first, are requested before the
// first score.  The groups of lanes are joined at the end by row swaps that add two
// channels at once (16 channels over 64 lanes: 12 swaps and 4 or 8 rotations), the waves in
// LDS.
//
// Bound: latency (index, then row, then the joins).  32 x 4 heads of 512 positions (17.6 MB of rows):
// 7.3 us, of 8 x 7 of 2048 (30.5 MB) 10.0 and the join's 3.8.  With shuffles for the joins and
// four waves per workgroup throughout: 11.5 with its join, and 14.5.
template <int D, bool I8, int NW>
__global__ __launch_bounds__(NW *kWave) void list_kernel(AttnArgs a) {
  constexpr int kLanes = D / 16;         // lanes of a row
  constexpr int kRows = kWave / kLanes;  // rows of a load
  constexpr int kLoads = kTile / kRows;
  __shared__ float wm[NW], wl[NW], wo[NW][D];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t s = blockIdx.x, g = blockIdx.y, bh = blockIdx.z;
  const int d0 = 16 * (lane % kLanes), rg = lane / kLanes;
  const int64_t len = row_length(a.lens, a.n, a.cap, bh);
  const float slope = a.slopes ? a.slopes[bh * a.G + g] * kLog2e : 0.0f;
  const int64_t *idx = a.idx + (bh * a.G + g) * a.k;
  const uint8_t *kb = a.k8 + bh * a.cap * D + d0, *vb = a.v8 + bh * a.cap * D + d0;
  const float *ksb = a.ks + bh * a.nblk, *vsb = a.vs + bh * a.nblk;
  const uint8_t *none = reinterpret_cast<const uint8_t *>(kNoRow);
  float q[2][8];
  float m = kLowest, l = 0.0f, o[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) o[e] = 0.0f;
  int ce;
  const float cm = query_factor(a, ce);
  bool first = true;
  for (int64_t t0 = (s * NW + wave) * kTile; t0 < a.k; t0 += a.nsplit * NW * kTile) {
    int64_t tok[kLoads];
    bool in[kLoads];
    u32x4 kc[kLoads], vc[kLoads];
    float ks[kLoads], vs[kLoads], x[kLoads], y[kLoads], bias[kLoads], z[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int64_t j = t0 + i * kRows + rg;
      tok[i] = idx[j < a.k ? j : a.k - 1];
      in[i] = j < a.k && tok[i] >= 0 && tok[i] < len;
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      kc[i] = *reinterpret_cast<const u32x4 *>(in[i] ? kb + tok[i] * D : none);
      ks[i] = ksb[in[i] ? (uint64_t)tok[i] / kBlk : 0];
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      vc[i] = *reinterpret_cast<const u32x4 *>(in[i] ? vb + tok[i] * D : none);
      vs[i] = vsb[in[i] ? (uint64_t)tok[i] / kBlk : 0];
    }
    // the queries are requested with the first tile, behind its rows
    if (first) {
#pragma unroll
      for (int h = 0; h < 2; ++h) load8_q(a.q, a.q_dtype, (bh * a.G + g) * D + d0 + 8 * h, q[h]);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (first) {
      first = false;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 8; ++e) q[h][e] *= cm;
    }
    float mt = m;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      float dot = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float c[4];
        decode4<I8>(kc[i][e], c);
#pragma unroll
        for (int f = 0; f < 4; ++f) dot = fmaf(q[e / 2][4 * (e & 1) + f], c[f], dot);
      }
      // z = x y + bias: below kLarge the product is rounded only once it is relative to the maximum
      x[i] = sum_row<kLanes>(dot);
      y[i] = ldexpf(ks[i], ce);
      if (a.softcap > 0.0f) {
        // finite for a finite scale: a score of 0 has to stay one
        y[i] = fabsf(ks[i]) < INFINITY ? __builtin_amdgcn_fmed3f(y[i], -3.0e38f, 3.0e38f) : y[i];
        x[i] = tanh_any(x[i] * y[i]);
        y[i] = a.softcap * kLog2e;
      }
      bias[i] = slope * (float)(int)(tok[i] - (len - 1));
      z[i] = fmaf(x[i], y[i], bias[i]);
      mt = fmaxf(mt, in[i] ? z[i] : kLowest);
    }
    const float f = __builtin_amdgcn_exp2f(m - mt);
    l *= f;
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] *= f;
    m = mt;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const float d = fabsf(m) < kLarge ? fmaf(x[i], y[i], bias[i] - m) : z[i] - m;
      const float p = in[i] ? __builtin_amdgcn_exp2f(d) : 0.0f;
      l += p;
      const float pv = in[i] ? p * vs[i] : 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float c[4];
        decode4<I8>(vc[i][e], c);
#pragma unroll
        for (int f = 0; f < 4; ++f) o[4 * e + f] = fmaf(pv, c[f], o[4 * e + f]);
      }
    }
  }
  // ---- the wave's groups against its maximum
  const float M = over_rows<kLanes, true>(m);
  const float f = __builtin_amdgcn_exp2f(m - M);
  l = over_rows<kLanes, false>(l * f);
  float r[4];
  {
    float h[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {  // lanes 0 .. 31: channel e, lanes 32 .. 63: channel e + 8
      const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(o[e] * f), __float_as_uint(o[e + 8] * f), false, false);
      h[e] = __uint_as_float(x[0]) + __uint_as_float(x[1]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {  // odd rows of 16 lanes: channel e + 4
      const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(h[e]), __float_as_uint(h[e + 4]), false, false);
      r[e] = over_row16<kLanes, false>(__uint_as_float(x[0]) + __uint_as_float(x[1]));
    }
  }
  if ((lane & 15) < kLanes)
    *reinterpret_cast<float4 *>(&wo[wave][d0 + 8 * (lane >> 5) + 4 * (lane >> 4 & 1)]) = make_float4(r[0], r[1], r[2], r[3]);
  if (lane == 0) {
    wm[wave] = M;
    wl[wave] = l;
  }
  __syncthreads();
  if (tid < D) {
    float mx = wm[0];
#pragma unroll
    for (int v = 1; v < NW; ++v) mx = fmaxf(mx, wm[v]);
    float L = 0.0f, O = 0.0f;
#pragma unroll
    for (int v = 0; v < NW; ++v) {
      const float e = __builtin_amdgcn_exp2f(wm[v] - mx);
      L = fmaf(wl[v], e, L);
      O = fmaf(wo[v][tid], e, O);
    }
    if (a.nsplit == 1) {
      a.out[(bh * a.G + g) * D + tid] = L == 0.0f ? 0.0f : O / L;
    } else {
      const int64_t at = (bh * a.nsplit + s) * a.G + g;
      a.part[at * D + tid] = O;
      if (tid == 0) a.ml[at] = make_float2(mx, L);
    }
  }
}

template <int N>
struct VPiece {
  typedef uint32_t type;
};
template <>
struct VPiece<8> {
  typedef unsigned int type __attribute__((ext_vector_type(2)));
};
__device__ __forceinline__ uint32_t dword_of(uint32_t v, int) { return v; }
__device__ __forceinline__ uint32_t dword_of(VPiece<8>::type v, int d) { return v[d]; }

// v + the value of the lane 8 columns away in the same row of 16 lanes (row_ror:8).
__device__ __forceinline__ float add_other_half(float v) {
  return v + dpp<kXor8>(v);
}

// The blocks of a row that a call takes: the first `sink` ones and, `skip` blocks further, those of the window, nb in
// all.  Tokens of them that take no part: [from, lo), and from len on.  Without sinks, from = sink = 0.
template <bool SINKS>
struct Span {
  int len, lo, from, sink, skip, nb;
  __device__ __forceinline__ int block(int i) const { return SINKS && i < sink ? i : i + skip; }  // the i-th of them
};
template <bool SINKS>
__device__ __forceinline__ Span<SINKS> row_span(const AttnArgs &a, int64_t bh) {
  Span<SINKS> s;
  s.len = (int)row_length(a.lens, a.n, a.cap, bh);
  s.lo = a.window > 0 && s.len > a.window ? s.len - (int)a.window : 0;
  const int first = s.lo / kBlk;
  s.from = !SINKS ? 0 : a.sinks < s.lo ? (int)a.sinks : s.lo;
  const int sink = (s.from + kBlk - 1) / kBlk;
  s.sink = sink < first ? sink : first;  // the last sinks may be in the window's first block
  s.skip = first - s.sink;
  s.nb = (s.len + kBlk - 1) / kBlk - s.skip;
  return s;
}

// The part of a workgroup: row, split of the row, the row's splits, blocks per split.
struct Part {
  int64_t bh;
  int split, active, per;
};
// Rows of their own lengths (on the device): every workgroup takes `per` blocks, so
// that the longest row does not hold the call up.  Each workgroup sums the rows'
// blocks, which gives `per`, and finds its row in the prefix sums of ceil(blocks /
// per).  Those are at most kDenseTotal / kDenseWaves / head groups + BH, the grid.  (32
// bits hold the sums: 2^31 blocks of D = 64 are 17 TB.)
template <bool SINKS>
__device__ __forceinline__ uint32_t blocks_of(const AttnArgs &a, int r) {
  return r < (int)a.BH ? (uint32_t)row_span<SINKS>(a, r).nb : 0u;
}
// Blocks per workgroup.  A row's last workgroup may have less to do: with few rows the
// share leaves room for those, so that all of the call's workgroups are at work at once.
__device__ __forceinline__ uint32_t share_of(const AttnArgs &a, uint32_t total) {
  const int BH = (int)a.BH, fit = kDenseTotal / kDenseWaves / (int)a.groups;
  const uint32_t groups = fit > 2 * BH ? fit - BH : fit > 0 ? fit : 1, even = (total + groups - 1) / groups;
  return even > (uint32_t)kDenseWaves ? even : (uint32_t)kDenseWaves;
}
// Workgroups of row r of nb blocks; a row without tokens takes one too: it writes the row's zeros.
__device__ __forceinline__ uint32_t groups_of(const AttnArgs &a, int r, uint32_t nb, uint32_t per) {
  return r >= (int)a.BH ? 0u : nb <= per ? 1u : (nb + per - 1) / per;
}

// Up to 64 rows: a lane per row, each wave for itself.
template <bool SINKS>
__device__ __forceinline__ Part find_part(const AttnArgs &a, uint32_t w) {
  const int lane = threadIdx.x & 63;
  const uint32_t nb = blocks_of<SINKS>(a, lane), per = share_of(a, __builtin_amdgcn_readlane(wave_incl_scan_u32(nb), 63));
  const uint32_t act = groups_of(a, lane, nb, per), upto = wave_incl_scan_u32(act);
  const uint64_t past = __ballot(upto > w);
  if (!past) return Part{a.BH, 0, 0, 0};  // the call needs no such workgroup
  const int at = __builtin_ctzll(past);
  const int active = __builtin_amdgcn_readlane((int)act, at);
  return Part{at, (int)w - (__builtin_amdgcn_readlane((int)upto, at) - active), active, (int)per};
}

// More rows: a thread takes BH / 256 of them in a row.  (512 rows, eight of them of 20032
// tokens, the others of 700: 38 us, against 268 with a workgroup for every row; all of 2048 tokens 48.9, 44.8.)
struct FindShared {
  uint32_t wave[2][kDenseWaves];
  int part[4];
};
template <bool SINKS>
__device__ __forceinline__ Part find_part_wide(const AttnArgs &a, uint32_t w, FindShared &sh) {
  constexpr int kThreads = kDenseWaves * kWave;
  const int tid = threadIdx.x, wave = tid >> 6;
  const int c = ((int)a.BH + kThreads - 1) / kThreads, r0 = tid * c;
  uint32_t sum = 0;
  for (int i = 0; i < c; ++i) sum += blocks_of<SINKS>(a, r0 + i);
  sum = wave_incl_scan_u32(sum);
  if ((tid & 63) == 63) sh.wave[0][wave] = sum;
  if (tid == 0) sh.part[0] = (int)a.BH;
  __syncthreads();
  uint32_t total = 0;
#pragma unroll
  for (int v = 0; v < kDenseWaves; ++v) total += sh.wave[0][v];
  const uint32_t per = share_of(a, total);
  uint32_t mine = 0;
  for (int i = 0; i < c; ++i) mine += groups_of(a, r0 + i, blocks_of<SINKS>(a, r0 + i), per);
  uint32_t upto = wave_incl_scan_u32(mine);
  if ((tid & 63) == 63) sh.wave[1][wave] = upto;
  __syncthreads();
  for (int v = 0; v < wave; ++v) upto += sh.wave[1][v];
  uint32_t at = upto - mine;
  if (w >= at && w < upto)
    for (int i = 0; i < c; ++i) {
      const uint32_t act = groups_of(a, r0 + i, blocks_of<SINKS>(a, r0 + i), per);
      if (w < at + act) {
        sh.part[0] = r0 + i;
        sh.part[1] = (int)(w - at);
        sh.part[2] = (int)act;
        break;
      }
      at += act;
    }
  __syncthreads();
  return Part{__builtin_amdgcn_readfirstlane(sh.part[0]), __builtin_amdgcn_readfirstlane(sh.part[1]),
              __builtin_amdgcn_readfirstlane(sh.part[2]), __builtin_amdgcn_readfirstlane((int)per)};
}

// Attention over every token of [lo, len), in splits, on the matrix cores.
//
// A workgroup takes one split of a row for a group of 8 NG query heads; its waves
// take the split's 64-token blocks in turn.  Per block (v_mfma_f32_16x16x32_f16,
// lane l = column l & 15, group l >> 4):
//   S^T = K q^T: A holds 16 tokens' codes as f16 (exact), straight from the
//     16-byte pieces of the rows (the channel order inside the contraction is
//     free, so it is the order that the pieces arrive in); B holds the queries,
//     column c < 8 the f16 of head c's q 2^sigma (times query_factor), column c + 8 the
//     f16 of what that leaves: 22 bits of q, at no cost, as 8 heads fill half of
//     the 16 columns.  One row rotation adds the halves.  Channels far below their head's
//     largest would have fewer: where a group has one below 2^-18 (1 % of normal queries), what is
//     left of those takes a second product, times 2^38, before the first (8 x 1048576 tokens 310 us for
//     305).  So 19 bits and more down to 2^-56 of the largest channel, and none below 2^-76.
//   softmax: a lane holds 16 scores of its head, tokens 16 i + 4 (l >> 4) + j; the
//     running maximum m (in log2 units) is raised only in the blocks where some
//     score passes it.  A weight is 2^(S f - m) with one rounding (see kLarge), f = s_K times a power of two.
//   O^T += V^T p^T: the layout that the scores come in is the one that B takes the
//     weights in once the contraction's token order is (tile, j): they never leave their lane.
//     Columns c < 8 hold the f16 of w = p s_V 2^(14 - E), columns c + 8 the f16 of
//     the rest: 22 bits of p, down to 2^-38 of the largest p s_V.  E = ceil(R), R the running
//     largest log2(p s_V) of a head, taken block by block as the block's largest score and
//     the exponent of its scale, and relative to m (it falls as m rises).  So w < 2^15, and a block of
//     large values without weight takes no bits from the others.
//     A holds V's codes, transposed inside the lane: it reads 8 (D = 64: 4) channels of 8
//     tokens and pairs two tokens' bytes with one v_perm.
// Rows are read through buffer descriptors that end at the row's length: what lies
// behind it reads as zeros.
// SINKS is a parameter as its masks cost calls without sinks 1 to 6 % (1 x 1000 tokens 10.5 us; 11.2).
//
// Bound: HBM, 2 D bytes per token and group of 16 heads: more heads read the rows once for each (8 x 65536
// tokens of 32 heads 46 to 53 us, 1.4 times the rows' bytes from HBM; of 12 heads 34, with cap and bias 39).
// The next block's K rows are requested once the scores are formed, its V rows once the products are, so that a
// wave has 8 to 16 KB on the way all the time.  A block takes 364 VALU instructions and 32 matrix ones (D = 128,
// NG = 1), a third of the time that its rows take.  8 x 1048576 tokens of 4 heads (2.15 GB) 304 us, 7.1 TB/s; 32 x
// 32768 (0.27 GB) 46 us with the join of the splits; one dot product per lane group and no matrix
// cores: 917 and 127 us.  Short rows are bound by latency: the launch, the rows' way from HBM, one block's arithmetic.
template <int D, bool I8, int NG, bool EXTRA, int NW, bool SINKS>
__global__ __launch_bounds__(NW *kWave, 2) void dense_kernel(AttnArgs a) {
  constexpr int kHalves = D / 64;  // 16-byte pieces of a row per lane
  constexpr int kSteps = D / 32;   // matrix instructions along the channels
  constexpr int kCh = D / 16;      // channels of V per lane
  __shared__ float wm[NW][8 * NG], wl[NW][8 * NG], wo[NW][8 * NG][D + 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int64_t g0 = (int64_t)blockIdx.y * 8 * NG;
  Part part{(int64_t)blockIdx.z, (int)blockIdx.x, (int)a.nsplit, 0};
  int64_t slot = (int64_t)blockIdx.z * a.nsplit + blockIdx.x;  // of the partial results
  if (NW == kDenseWaves && a.where) {  // uniform over the workgroup
    if (a.BH <= kWave) {
      part = find_part<SINKS>(a, blockIdx.x);
    } else {
      __shared__ FindShared find;
      part = find_part_wide<SINKS>(a, blockIdx.x, find);
    }
    if (part.bh >= a.BH) return;
    slot = blockIdx.x;
    if (part.split == 0 && blockIdx.y == 0 && tid == 0) a.where[part.bh] = make_int2((int)blockIdx.x, part.active);
  }
  const int64_t bh = part.bh;
  const Span<SINKS> span = row_span<SINKS>(a, bh);
  const int lo = span.lo, len = span.len;
  if (!a.where) part.per = (span.nb + part.active - 1) / part.active;
  const int first = part.split * part.per;  // of the row's blocks in the order of span.block
  const int last = part.split + 1 < part.active ? first + part.per : span.nb;

  // the queries are requested first and made ready while the first block's rows come
  float q[NG][kSteps][8];
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    const int64_t g = g0 + 8 * n + (col & 7), row = (bh * a.G + (g < a.G ? g : a.G - 1)) * D;
#pragma unroll
    for (int h = 0; h < kSteps; ++h)  // step h = (piece, half): channels 64 (h / 2) + 16 grp + 8 (h & 1) + e
      load8_q(a.q, a.q_dtype, row + 64 * (h / 2) + 16 * grp + 8 * (h & 1), q[n][h]);
  }
  u32x4 kr[4][kHalves];
  typedef typename VPiece<kCh>::type vpiece;
  vpiece vr[4][4];
  const int koff = col * D + 16 * grp, voff = 4 * grp * D + kCh * col;
  auto load_k = [&](int b) {
    const RowsOf r(a.k8, bh * a.cap, span.block(b), b < last ? len : 0, D);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int h = 0; h < kHalves; ++h) kr[i][h] = r.load16(koff + 16 * i * D + 64 * h);
  };
  auto load_v = [&](int b) {
    const RowsOf r(a.v8, bh * a.cap, span.block(b), b < last ? len : 0, D);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) r.load(voff + (16 * i + j) * D, vr[i][j]);
  };
  load_k(first + wave);
  load_v(first + wave);
  const float keep = col < 8 ? 0.0f : -1.0f;  // columns 8 .. 15 hold what the f16 of columns 0 .. 7 leave
  f16x8 qf[NG][kSteps];
  __shared__ f16x8 rest[NG][kSteps][kWave];  // what qf leaves of small channels, 2^38
  bool far = false;  // some channel is that small
  int ce, ex[NG];   // per lane: the exponent that its head's scores take
  float slope[NG];  // its bias per token
  const float cm = query_factor(a, ce);
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    const int64_t g = g0 + 8 * n + (col & 7);
    float mx = 0.0f;
    float mn = INFINITY;
#pragma unroll
    for (int h = 0; h < kSteps; ++h)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        mx = fmaxf(mx, fabsf(q[n][h][e]));
        mn = fminf(mn, fabsf(q[n][h][e]));
      }
    mx = across_groups<true>(mx);
    far |= mn < mx * 0x1p-18f || mx < 0x1p-100f;
    int sigma = 0;  // the largest |q| of the head in [2^13, 2^14)
    if (mx > 0.0f && mx < INFINITY) {
      frexpf(mx, &sigma);
      sigma = 14 - sigma;
    }
#pragma unroll
    for (int h = 0; h < kSteps; ++h) {
      f16x2 part[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = ldexpf(q[n][h][2 * e], sigma) * cm, y = ldexpf(q[n][h][2 * e + 1], sigma) * cm;
        part[e] = split16(x, y, keep);
        q[n][h][2 * e] = x;
        q[n][h][2 * e + 1] = y;
      }
      qf[n][h] = join8(part[0], part[1], part[2], part[3]);
    }
    ex[n] = ce - sigma;
    slope[n] = EXTRA && a.slopes && g < a.G ? a.slopes[bh * a.G + g] * kLog2e : 0.0f;
  }

  far = __any(far);  // uniform over the workgroup: its waves hold the same queries
  if (far) {  // channels of 0 are no small ones
    far = false;
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int h = 0; h < kSteps; ++h)
#pragma unroll
        for (int e = 0; e < 8; ++e) far |= small_channel(q[n][h][e]);
    far = __any(far);
  }
  // Two groups of eight heads keep them in LDS: in registers, D = 128 with cap and bias spills (8 x 65536 tokens, 12 heads
  // 47 us; 40).
  constexpr bool kQueryLds = NG > 1;
  __shared__ f16x8 qs[kQueryLds ? NG : 1][kSteps][kWave];
  if constexpr (kQueryLds) {
    if (wave == 0) {
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int h = 0; h < kSteps; ++h) qs[n][h][lane] = qf[n][h];
    }
    __syncthreads();
  }
  if (__builtin_expect(far, 0)) {
    if (wave == 0) {
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int h = 0; h < kSteps; ++h) {
          f16x2 part[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) part[e] = split16(rest_of(q[n][h][2 * e]), rest_of(q[n][h][2 * e + 1]), keep);
          rest[n][h][lane] = join8(part[0], part[1], part[2], part[3]);
        }
    }
    __syncthreads();
  }

  f32x4 o[NG][kCh];
  float m[NG], l[NG], R[NG];
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    m[n] = kLowest;
    l[n] = 0.0f;
    R[n] = kNoValue;
#pragma unroll
    for (int e = 0; e < kCh; ++e) o[n][e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // the scales come through the scalar cache, a block ahead too
  typedef const __attribute__((address_space(4))) float *scalar_ptr;
  const scalar_ptr ksp = (scalar_ptr)(a.ks + bh * a.nblk), vsp = (scalar_ptr)(a.vs + bh * a.nblk);
  float ks_next = 0.0f, vs_next = 0.0f;
  if (first + wave < last) {
    ks_next = ksp[span.block(first + wave)];
    vs_next = vsp[span.block(first + wave)];
  }
  for (int b = first + wave; b < last; b += NW) {
    const float ks = ks_next, vs = vs_next;
    f32x4 s[NG][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int n = 0; n < NG; ++n) s[n][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    auto keys = [&](int i, int h) {
      const uint32_t w0 = flip_sign<I8>(kr[i][h / 2][2 * (h & 1)]), w1 = flip_sign<I8>(kr[i][h / 2][2 * (h & 1) + 1]);
      return join8(pair16<I8, false>(w0), pair16<I8, true>(w0), pair16<I8, false>(w1), pair16<I8, true>(w1));
    };
    if (__builtin_expect(far, 0)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int h = 0; h < kSteps; ++h) {
          const f16x8 k = keys(i, h);
#pragma unroll
          for (int n = 0; n < NG; ++n) s[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, rest[n][h][lane], s[n][i], 0, 0, 0);
        }
#pragma unroll
        for (int n = 0; n < NG; ++n) s[n][i] *= 0x1p-38f;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)  // the operands are made anew: kept, they would take 64 registers
#pragma unroll
      for (int h = 0; h < kHalves; ++h) asm volatile("" : "+v"(kr[i][h]));
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int h = 0; h < kSteps; ++h) {
        const f16x8 k = keys(i, h);
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          const f16x8 query = kQueryLds ? qs[n][h][lane] : qf[n][h];
          s[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, query, s[n][i], 0, 0, 0);
        }
      }
    load_k(b + NW);
    if (b + NW < last) {
      ks_next = ksp[span.block(b + NW)];
      vs_next = vsp[span.block(b + NW)];
    }
    // ---- scores, in log2 units; tokens of [from, lo) and from len on have none
    const int t0 = span.block(b) * kBlk, in_block = t0 + 4 * grp;
    const bool edge = (t0 < lo && t0 + kBlk > span.from) || t0 + kBlk > len;
    // Bit 4 i + j: a token that takes no part.  Made where it is used, and in a register of the lane: as masks for
    // every token the compiler fills the scalar registers with it (70 spilled at two groups of heads).
    auto left_out = [&]() {
      uint32_t none = 0;
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const int t = in_block + 16 * (x / 4) + x % 4;
        none |= ((t >= span.from && t < lo) || t >= len ? 1u : 0u) << x;
      }
      asm volatile("" : "+v"(none));
      return none;
    };
    const int ev = (int)((__float_as_uint(vs) >> 23) & 0xFF) - 127;
    float fz[NG];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      // z = s f; below kLarge not rounded itself, but relative to the maximum
      float f = ldexpf(fabsf(ks), ex[n]);
      // never infinite: a score of 0 has to stay one; nor 0 without a cap: a score of -inf has to stay one too
      // (an infinite or NaN scale stays what it is)
      f = fabsf(ks) < INFINITY ? __builtin_amdgcn_fmed3f(f, EXTRA && a.softcap > 0.0f ? 0.0f : 1.2e-38f, 3.0e38f) : f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][i][j] = add_other_half(s[n][i][j]);
      if (ks < 0.0f) {  // not written by this store's writer
        asm volatile("");
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] = -s[n][i];
      }
      if constexpr (EXTRA) {
        if (a.softcap > 0.0f) {
          float big = 0.0f;
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              s[n][i][j] *= f;
              big = fmaxf(big, fabsf(s[n][i][j]));
            }
          if (__any(big >= 0.5f)) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int j = 0; j < 4; ++j) s[n][i][j] = tanh_any(s[n][i][j]);
          } else {  // most blocks: scores well below the cap
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int j = 0; j < 4; ++j) s[n][i][j] = tanh_small(s[n][i][j]);
          }
          f = a.softcap * kLog2e;
        }
        const float back = (float)(in_block - (len - 1));
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[n][i][j] = fmaf(s[n][i][j], f, slope[n] * (back + (float)(16 * i + j)));
        f = 1.0f;
      }
      if (edge) {
        if constexpr (SINKS) {
          const uint32_t none = left_out();
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[n][i][j] = none >> (4 * i + j) & 1 ? -INFINITY : s[n][i][j];
        } else {
          asm volatile("");  // a branch, not selects in every block
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int t = in_block + 16 * i + j;
              s[n][i][j] = t >= lo && t < len ? s[n][i][j] : -INFINITY;
            }
        }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = fmaxf(mx, s[n][i][j]);
      mx *= f;
      if constexpr (!EXTRA) {
        if (__any(fabsf(mx) >= kLarge && fabsf(mx) < INFINITY)) {
          asm volatile("");  // a branch, not products in every block
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][i] *= f;
          f = 1.0f;
        }
      }
      fz[n] = f;
      float by = 1.0f;
      const float was = R[n];
      if (__any(fmaxf(mx - m[n], kLeast) > fminf(0.0f, was - (float)ev))) {  // a larger score, or weight times scale
        mx = across_groups<true>(mx);
        const float M = fmaxf(m[n], mx), down = __builtin_amdgcn_exp2f(m[n] - M);
        R[n] = fmaxf(was + (m[n] - M), (float)ev + fmaxf(mx - M, kLeast));
        m[n] = M;
        l[n] *= down;
        by = ldexpf(down, (int)ceilf(was) - (int)ceilf(R[n]));
      }
      if (__any(by != 1.0f)) {  // apart from the branch above, which would take more registers (8 x 65536, G = 12: 45 us for 35)
#pragma unroll
        for (int e = 0; e < kCh; ++e) o[n][e] *= by;
      }
    }
    float wv[NG];
#pragma unroll
    for (int n = 0; n < NG; ++n) wv[n] = ldexpf(vs, 14 - (int)ceilf(R[n]));
    if (edge) {  // a token outside has no value either (its codes may be NaN)
      const uint32_t none = SINKS ? left_out() : 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (SINKS ? none >> (4 * i + j) & 1 : in_block + 16 * i + j < lo) vr[i][j] = vpiece{};
    }
    // ---- weights and products, 32 tokens at a time
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      f16x8 p[NG];
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        f16x2 pp[4];
        float ps[4];  // added together first: alone, most weights would be lost beside a large sum
#pragma unroll
        for (int x = 0; x < 4; ++x) {  // tokens (tile 2 c + x / 2, j = 2 (x & 1), + 1)
          const float p0 = __builtin_amdgcn_exp2f(fmaf(s[n][2 * c + x / 2][2 * (x & 1)], fz[n], -m[n]));
          const float p1 = __builtin_amdgcn_exp2f(fmaf(s[n][2 * c + x / 2][2 * (x & 1) + 1], fz[n], -m[n]));
          ps[x] = p0 + p1;
          pp[x] = split16(p0 * wv[n], p1 * wv[n], keep);
        }
        l[n] += (ps[0] + ps[1]) + (ps[2] + ps[3]);
        p[n] = join8(pp[0], pp[1], pp[2], pp[3]);
      }
#pragma unroll
      for (int d = 0; d < kCh / 4; ++d) {  // dword d of the lane's channels
        uint32_t w[2][4];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int j = 0; j < 4; ++j) w[x][j] = flip_sign<I8>(dword_of(vr[2 * c + x][j], d));
#pragma unroll
        for (int y = 0; y < 2; ++y) {  // channels 4 d + 2 y, + 1
          uint32_t ab[2][2];
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              ab[x][j] = __builtin_amdgcn_perm(w[x][2 * j + 1], w[x][2 * j], y ? 0x07030602u : 0x05010400u);
          const f16x8 v0 = join8(pair16<I8, false>(ab[0][0]), pair16<I8, false>(ab[0][1]), pair16<I8, false>(ab[1][0]),
                                 pair16<I8, false>(ab[1][1]));
          const f16x8 v1 = join8(pair16<I8, true>(ab[0][0]), pair16<I8, true>(ab[0][1]), pair16<I8, true>(ab[1][0]),
                                 pair16<I8, true>(ab[1][1]));
#pragma unroll
          for (int n = 0; n < NG; ++n) {
            o[n][4 * d + 2 * y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, p[n], o[n][4 * d + 2 * y], 0, 0, 0);
            o[n][4 * d + 2 * y + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, p[n], o[n][4 * d + 2 * y + 1], 0, 0, 0);
          }
        }
      }
    }
    load_v(b + NW);
  }
  // ---- the workgroup's waves
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    const float L = across_groups<false>(l[n]);
    const float up = ldexpf(1.0f, (int)ceilf(R[n]) - 14);
    if (lane < 8) {
      wm[wave][8 * n + lane] = m[n];
      wl[wave][8 * n + lane] = L;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < kCh; e += 4) {
        float4 v;
        v.x = add_other_half(o[n][e][j]) * up;
        v.y = add_other_half(o[n][e + 1][j]) * up;
        v.z = add_other_half(o[n][e + 2][j]) * up;
        v.w = add_other_half(o[n][e + 3][j]) * up;
        if (col < 8) *reinterpret_cast<float4 *>(&wo[wave][8 * n + col][(4 * grp + j) * kCh + e]) = v;
      }
  }
  __syncthreads();
  for (int x = tid; x < 8 * NG * D; x += NW * kWave) {
    const int h = x / D, d = x % D;
    if (g0 + h >= a.G) break;
    float M = wm[0][h];
#pragma unroll
    for (int v = 1; v < NW; ++v) M = fmaxf(M, wm[v][h]);
    float L = 0.0f, O = 0.0f;
#pragma unroll
    for (int v = 0; v < NW; ++v) {
      const float e = __builtin_amdgcn_exp2f(wm[v][h] - M);
      L = fmaf(wl[v][h], e, L);
      O = fmaf(wo[v][h][d], e, O);
    }
    const int64_t r = bh * a.G + g0 + h;
    if (part.active <= 1 && !a.join) {
      a.out[r * D + d] = L == 0.0f ? 0.0f : O / L;
    } else {
      const int64_t at = slot * a.G + g0 + h;
      a.part[at * D + d] = O;
      if (d == 0) a.ml[at] = make_float2(M, L);
    }
  }
}

// Joins the splits of a query head, 32 channels per workgroup: a thread takes 16 bytes
// of every 32nd split, requested before the splits' factors are known; sums run in a fixed order.
// Bound: latency, 2.5 to 4.6 us (one thread per channel and splits in a row: 26 us for 64 splits).
template <int D>
__global__ __launch_bounds__(kMergeThreads) void merge_kernel(AttnArgs a) {
  constexpr int kLanes = 8, kGroups = kMergeThreads / kLanes, kBatch = 4;
  constexpr int kOwn = kMaxSplits / kMergeThreads;  // splits whose factor a thread computes
  __shared__ float fac[kMaxSplits], red[2][kMergeThreads / kWave];
  __shared__ float4 acc[kGroups][kLanes];
  const int64_t bh = blockIdx.y, r = bh * a.G + blockIdx.x;
  const int tid = threadIdx.x, lane = tid % kLanes, grp = tid / kLanes;
  const int2 w = a.where ? a.where[bh] : make_int2((int)(bh * a.nsplit), (int)a.nsplit);
  const int ns = w.y;
  if (ns <= 1) return;  // written already
  const int64_t at = (int64_t)w.x * a.G + blockIdx.x;  // split s at + s G
  const float4 *p = reinterpret_cast<const float4 *>(a.part + at * D + 32 * blockIdx.z) + lane;
  const int64_t step = a.G * (D / 4);
  float4 v[kBatch];
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    const int s = grp + i * kGroups;
    v[i] = p[(s < ns ? s : 0) * step];
  }
  float2 x[kOwn];
  float m = kLowest;
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const int s = i * kMergeThreads + tid;
    x[i] = s < ns ? a.ml[at + s * a.G] : make_float2(kLowest, 0.0f);
    m = fmaxf(m, x[i].x);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  if ((tid & 63) == 0) red[0][tid >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kMergeThreads / kWave; ++k) m = fmaxf(m, red[0][k]);
  float l = 0.0f;
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const float f = __builtin_amdgcn_exp2f(x[i].x - m);
    fac[i * kMergeThreads + tid] = f;
    l = fmaf(x[i].y, f, l);
  }
  l = wave_sum_f(l);
  if ((tid & 63) == 0) red[1][tid >> 6] = l;
  __syncthreads();
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int s0 = grp; s0 < ns; s0 += kBatch * kGroups) {
    if (s0 != grp) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int s = s0 + i * kGroups;
        v[i] = p[(s < ns ? s : 0) * step];
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int s = s0 + i * kGroups;
      if (s >= ns) break;
      const float f = fac[s];
      o.x = fmaf(v[i].x, f, o.x);
      o.y = fmaf(v[i].y, f, o.y);
      o.z = fmaf(v[i].z, f, o.z);
      o.w = fmaf(v[i].w, f, o.w);
    }
  }
  acc[grp][lane] = o;
  __syncthreads();
  if (tid < 32) {
    float u = 0.0f;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) u += reinterpret_cast<const float *>(acc[g])[tid];
    l = 0.0f;
#pragma unroll
    for (int k = 0; k < kMergeThreads / kWave; ++k) l += red[1][k];
    a.out[r * D + 32 * blockIdx.z + tid] = l == 0.0f ? 0.0f : u / l;
  }
}

// Waves of list_kernel's workgroups, by the same rule as gather_attention's: 16 (512
// positions) for heads of 129 to 512, which then need no join of splits, and
// for longer ones where that still gives about a workgroup to every other CU; else 4.
int list_waves(int64_t heads, int64_t k) {
  constexpr int64_t kOne = 16 * kTile;
  if (k <= kOne) return k > 4 * kTile ? 16 : 4;
  return heads * cdiv(k, kOne) >= 96 ? 16 : 4;
}
// Splits of a head's listed positions: a tile per wave, as long as the chip has room
// for all workgroups at once (kListTotal waves, 16 per CU).  With twice as many:
// 32 x 4 heads of 2048 positions 21.1 us, 17.4 so; 64 x 4 of 1024 21.2, 13.6; 32 x 8 of 4096 50.7, 45.2.
constexpr int64_t kListTotal = 4096;
int64_t list_room(int64_t heads, int waves) {
  const int64_t room = kListTotal / waves / heads;
  return room < 1 ? 1 : room < kMaxSplits ? room : kMaxSplits;
}
int64_t list_splits(int64_t heads, int64_t k) {
  const int waves = list_waves(heads, k);
  const int64_t most = cdiv(k, (int64_t)waves * kTile), room = list_room(heads, waves);
  return most < 1 ? 1 : most < room ? most : room;
}

// Head groups of a row and their size in eights: a workgroup holds up to 16 heads.
int64_t head_groups(int64_t G) { return cdiv(G, (int64_t)16); }

// Blocks of a row that one workgroup of eight waves takes: two per wave, and one
// more as a window of 1024 tokens may begin inside a block (its wave takes three then).
constexpr int64_t kOneGroup = 17;

// Whether rows of up to nb blocks go to workgroups of eight waves, one per row: one launch for two (the join)
// and no workspace, two or three blocks per wave.  A call of 1 x 1000 tokens takes 10.3 us from Python and 11.4 in a
// graph, with splits of four waves 14.5 and 8.4: the host's part of a call counts more often, though a graph of
// such rows loses by it.  Rows of up to four
// blocks need no split of four waves either, and split rows are no faster in eight (32 x 4096 tokens 14.6 us
// both ways, 8 x 8192 11.1 with four; 13.8, 8 x 1048576 326; 331).
bool one_group(int64_t nb) { return nb > kDenseWaves && nb <= kOneGroup; }

// Splits of a row of up to nb blocks in a call of `rows` rows (head groups counted):
// at least one block per wave, and no more than kDenseTotal waves in all, as
// workgroups that have to wait for a place cost their whole prologue: 24 rows of 32768
// tokens take 39.3 us in 21 splits, 47.8 in 22.  Two splits all the same where one
// would leave more than a quarter of the places empty: 300 rows of 4096 tokens 67.7 us, in one split 73.0.
int64_t dense_splits(int64_t rows, int64_t nb) {
  if (nb <= kOneGroup) return 1;
  constexpr int64_t kPlaces = kDenseTotal / kDenseWaves;
  const int64_t most = cdiv(nb, (int64_t)kDenseWaves);
  int64_t room = kPlaces / rows;
  if (room == 1 && rows < kPlaces * 3 / 4) room = 2;
  const int64_t ns = most < room ? most : room;
  return ns < 1 ? 1 : ns;
}

// Slots of partial results of a dense call; 0: every row fits one workgroup.  With
// lengths on the device: the bound of find_part.  Neither falls as nb grows.
int64_t dense_slots(int64_t BH, int64_t G, int64_t nb, bool lens) {
  if (nb <= kOneGroup) return 0;
  const int64_t groups = head_groups(G), ns = dense_splits(BH * groups, nb);
  if (!lens) return ns > 1 ? BH * ns : 0;
  const int64_t all = kDenseTotal / kDenseWaves / groups + BH, most = BH * cdiv(nb, (int64_t)kDenseWaves);
  return all < most ? all : most;
}

// Bytes of `slots` partial results: rows, (m, l), the rows' slots.
size_t part_bytes(int64_t BH, int64_t G, int64_t D, int64_t slots) {
  return slots < 1 ? 0 : (size_t)(slots * G * (D + 2) + 2 * BH) * sizeof(float);
}

void place(AttnArgs &a, void *workspace, int64_t D, int64_t slots, bool lens) {
  if (slots < 1) return;
  a.part = static_cast<float *>(workspace);
  a.ml = reinterpret_cast<float2 *>(a.part + slots * a.G * D);
  if (lens) a.where = reinterpret_cast<int2 *>(a.ml + slots * a.G);
}

int merge(const AttnArgs &a, int64_t BH, int64_t D, hipStream_t st) {
  const dim3 grid((unsigned)a.G, (unsigned)BH, (unsigned)D / 32);  // an axis of BH G workgroups could pass 2^32 threads
  if (D == 128) merge_kernel<128><<<grid, kMergeThreads, 0, st>>>(a);
  else merge_kernel<64><<<grid, kMergeThreads, 0, st>>>(a);
  return launch_status("rows8 merge_kernel");
}

template <int D, bool I8>
void launch_list(const AttnArgs &a, int64_t BH, hipStream_t st) {
  const dim3 grid((unsigned)a.nsplit, (unsigned)a.G, (unsigned)BH);
  if (list_waves(BH * a.G, a.k) == 16) list_kernel<D, I8, 16><<<grid, 16 * kWave, 0, st>>>(a);
  else list_kernel<D, I8, 4><<<grid, 4 * kWave, 0, st>>>(a);
}

int run_list(AttnArgs a, int64_t BH, int64_t D, bool i8, hipStream_t st) {
  if (D == 128 && i8) launch_list<128, true>(a, BH, st);
  else if (D == 128) launch_list<128, false>(a, BH, st);
  else if (i8) launch_list<64, true>(a, BH, st);
  else launch_list<64, false>(a, BH, st);
  const int rc = launch_status("rows8 list_kernel");
  return rc || a.nsplit == 1 ? rc : merge(a, BH, D, st);
}

template <int D, bool I8, int NG, int NW>
void launch_dense(const AttnArgs &a, int64_t BH, hipStream_t st) {
  const dim3 grid((unsigned)a.nsplit, (unsigned)head_groups(a.G), a.where ? 1u : (unsigned)BH);
  const bool extra = a.softcap > 0.0f || a.slopes, sinks = a.sinks > 0 && a.window > 0;
  if (extra && sinks) dense_kernel<D, I8, NG, true, NW, true><<<grid, NW * kWave, 0, st>>>(a);
  else if (extra) dense_kernel<D, I8, NG, true, NW, false><<<grid, NW * kWave, 0, st>>>(a);
  else if (sinks) dense_kernel<D, I8, NG, false, NW, true><<<grid, NW * kWave, 0, st>>>(a);
  else dense_kernel<D, I8, NG, false, NW, false><<<grid, NW * kWave, 0, st>>>(a);
}

template <int D, bool I8>
void launch_dense(const AttnArgs &a, int64_t BH, bool one, hipStream_t st) {
  if (a.G > 8 && one) launch_dense<D, I8, 2, 8>(a, BH, st);
  else if (a.G > 8) launch_dense<D, I8, 2, kDenseWaves>(a, BH, st);
  else if (one) launch_dense<D, I8, 1, 8>(a, BH, st);
  else launch_dense<D, I8, 1, kDenseWaves>(a, BH, st);
}

int run_dense(AttnArgs a, int64_t BH, int64_t D, bool i8, bool one, hipStream_t st) {
  if (D == 128 && i8) launch_dense<128, true>(a, BH, one, st);
  else if (D == 128) launch_dense<128, false>(a, BH, one, st);
  else if (i8) launch_dense<64, true>(a, BH, one, st);
  else launch_dense<64, false>(a, BH, one, st);
  const int rc = launch_status("rows8 dense_kernel");
  return rc || a.nsplit == 1 || a.join ? rc : merge(a, BH, D, st);
}

// Blocks of a row at most, from what the host knows: exact without lengths on the device.
int64_t dense_blocks(const int32_t *lens, int64_t n, int64_t cap, int64_t window, int64_t sinks) {
  const int64_t all = cdiv(lens ? cap : n, (int64_t)kBlk);
  if (window <= 0 || window >= (lens ? cap : n)) return lens && window > 0 ? all + 1 : all;
  if (lens) {
    const int64_t nb = cdiv(window, (int64_t)kBlk) + 1, some = nb + cdiv(sinks < cap ? sinks : cap, (int64_t)kBlk);
    return sinks > 0 && some > all ? all : some;
  }
  const int64_t lo = n - window, from = sinks < lo ? sinks : lo, first = lo / kBlk, sink = cdiv(from, (int64_t)kBlk);
  return all - first + (sink < first ? sink : first);
}

// Slots of partial results of a call, as dense_slots, but one per row at least where others join them.
int64_t part_slots(int64_t BH, int64_t G, int64_t nb, bool lens, bool join) {
  const int64_t slots = dense_slots(BH, G, nb, lens);
  return join && slots < BH ? BH : slots;
}

// Bytes for calls of up to so many positions.
size_t dense_bytes(int64_t BH, int64_t G, int64_t D, int64_t positions, bool join) {
  if (positions > kMaxCap) positions = kMaxCap;
  const int64_t nb = cdiv(positions, (int64_t)kBlk) + 1;  // a window may begin inside a block
  const int64_t one = part_slots(BH, G, nb, false, join), own = part_slots(BH, G, nb, true, join);
  return part_bytes(BH, G, D, one > own ? one : own);
}

// Sets up and launches the splits; their join only where the results are not the caller's to join.
int dense_call(AttnArgs &a, const char *what, int64_t D, bool i8, void *workspace, size_t workspace_bytes, hipStream_t st) {
  const bool lens = a.lens != nullptr;
  const int64_t nb = dense_blocks(a.lens, a.n, a.cap, a.window, a.sinks), all = dense_slots(a.BH, a.G, nb, lens);
  const int64_t slots = part_slots(a.BH, a.G, nb, lens, a.join);
  a.groups = head_groups(a.G);
  a.nsplit = all < 1 ? 1 : lens ? all : cdiv(nb, cdiv(nb, all / a.BH));  // as many as shares of that size fill
  const size_t need = part_bytes(a.BH, a.G, D, slots);
  if (need && (!workspace || workspace_bytes < need))
    return fail(FATHOM_ERR_WORKSPACE, "%s: workspace %zu bytes, need %zu", what, workspace_bytes, need);
  if (need && reinterpret_cast<uintptr_t>(workspace) & 15)
    return fail(FATHOM_ERR_INVALID, "%s: the workspace must be 16-byte aligned", what);
  place(a, workspace, D, slots, lens && all > 0);
  return run_dense(a, a.BH, D, i8, one_group(nb), st);
}

int attention(const char *what, const void *q, int q_dtype, const void *k8, const void *v8, const float *k_scale,
              const float *v_scale, int code_dtype, int64_t BH, int64_t G, int64_t D, int64_t cap, const int32_t *lens, int64_t n,
              int64_t window, int64_t sinks, float scale, float softcap, const float *slopes, float *out, void *workspace,
              size_t workspace_bytes, void *stream) {
  int rc = check_store(what, k8, v8, k_scale, v_scale, code_dtype, BH, cap, D);
  if (!rc) rc = check_query(what, q, q_dtype, G, cap, lens, n, softcap, out);
  if (rc) return rc;
  if (window < 0) return fail(FATHOM_ERR_INVALID, "%s: window %lld", what, (long long)window);
  if (sinks < 0) return fail(FATHOM_ERR_INVALID, "%s: sinks %lld", what, (long long)sinks);
  AttnArgs a{q, q_dtype, (const uint8_t *)k8, (const uint8_t *)v8, k_scale, v_scale, G, cap, cdiv(cap, kBlk), lens, n, window,
             sinks, nullptr, 0, scale, kernel_cap(softcap), slopes, out, nullptr, nullptr, nullptr, 1, BH, 1, false};
  return dense_call(a, what, D, code_dtype == FATHOM_DT_I8, workspace, workspace_bytes, (hipStream_t)stream);
}

}  // namespace

size_t tail_bytes(int64_t BH, int64_t G, int64_t D, int64_t positions) { return dense_bytes(BH, G, D, positions, true); }

int tail_attention(Tail &t, const char *what, const void *q, int q_dtype, const void *k8, const void *v8, const float *k_scale,
                   const float *v_scale, bool i8, int64_t BH, int64_t G, int64_t D, int64_t cap, const int32_t *lens, int64_t n,
                   float scale, float softcap, const float *slopes, void *workspace, size_t workspace_bytes, hipStream_t st) {
  AttnArgs a{q, q_dtype, (const uint8_t *)k8, (const uint8_t *)v8, k_scale, v_scale, G, cap, cdiv(cap, kBlk), lens, n, 0,
             0, nullptr, 0, scale, kernel_cap(softcap), slopes, nullptr, nullptr, nullptr, nullptr, 1, BH, 1, true};
  const int rc = dense_call(a, what, D, i8, workspace, workspace_bytes, st);
  t = Tail{a.part, a.ml, a.where, a.nsplit};
  return rc;
}

}  // namespace rows8
}  // namespace fathom

using namespace fathom;
using namespace fathom::rows8;

extern "C" size_t fathom_rows8_attention_workspace_bytes(int64_t BH, int64_t G, int64_t D, int64_t positions) {
  if (!shape_taken(BH, G, D) || positions < 1) return 0;
  return dense_bytes(BH, G, D, positions, false);
}

extern "C" int fathom_rows8_attention(const void *q, int q_dtype, const void *k8, const void *v8, const float *k_scale,
                                      const float *v_scale, int code_dtype, int64_t BH, int64_t G, int64_t D, int64_t cap,
                                      const int32_t *lens, int64_t n, int64_t window, float scale, float softcap,
                                      const float *slopes, float *out, void *workspace, size_t workspace_bytes,
                                      void *stream) {
  return attention("rows8_attention", q, q_dtype, k8, v8, k_scale, v_scale, code_dtype, BH, G, D, cap, lens, n, window, 0, scale,
                   softcap, slopes, out, workspace, workspace_bytes, stream);
}

extern "C" int fathom_rows8_sink_attention(const void *q, int q_dtype, const void *k8, const void *v8, const float *k_scale,
                                           const float *v_scale, int code_dtype, int64_t BH, int64_t G, int64_t D, int64_t cap,
                                           const int32_t *lens, int64_t n, int64_t window, int64_t sinks, float scale,
                                           float softcap, const float *slopes, float *out, void *workspace,
                                           size_t workspace_bytes, void *stream) {
  return attention("rows8_sink_attention", q, q_dtype, k8, v8, k_scale, v_scale, code_dtype, BH, G, D, cap, lens, n, window,
                   sinks, scale, softcap, slopes, out, workspace, workspace_bytes, stream);
}

extern "C" size_t fathom_rows8_gather_attention_workspace_bytes(int64_t BH, int64_t G, int64_t D, int64_t k) {
  if (!shape_taken(BH, G, D) || k <= 16 * kTile) return 0;
  if (k > 0x7FFFFFFF / G) k = 0x7FFFFFFF / G;
  // of the narrower workgroups, so that it never falls as k grows
  int64_t ns = cdiv(k, (int64_t)4 * kTile);
  if (ns > list_room(BH * G, 4)) ns = list_room(BH * G, 4);
  return part_bytes(BH, G, D, ns > 1 ? BH * ns : 0);
}

extern "C" int fathom_rows8_gather_attention(const void *q, int q_dtype, const int64_t *idx, const void *k8, const void *v8,
                                             const float *k_scale, const float *v_scale, int code_dtype, int64_t BH,
                                             int64_t G, int64_t k, int64_t D, int64_t cap, const int32_t *lens, int64_t n,
                                             float scale, float softcap, const float *slopes, float *out, void *workspace,
                                             size_t workspace_bytes, void *stream) {
  int rc = check_store("rows8_gather_attention", k8, v8, k_scale, v_scale, code_dtype, BH, cap, D);
  if (!rc) rc = check_query("rows8_gather_attention", q, q_dtype, G, cap, lens, n, softcap, out);
  if (rc) return rc;
  if (k < 0 || k > 0x7FFFFFFF / G) return fail(FATHOM_ERR_INVALID, "rows8_gather_attention: G=%lld k=%lld", (long long)G, (long long)k);
  if (k > 0 && !idx) return fail(FATHOM_ERR_INVALID, "rows8_gather_attention: null index pointer");
  AttnArgs a{q, q_dtype, (const uint8_t *)k8, (const uint8_t *)v8, k_scale, v_scale, G, cap, cdiv(cap, kBlk), lens, n, 0,
             0, idx, k, scale, kernel_cap(softcap), slopes, out, nullptr, nullptr, nullptr, 1, BH, 1, false};
  a.nsplit = list_splits(BH * G, k);
  const int64_t slots = a.nsplit > 1 ? BH * a.nsplit : 0;
  const size_t need = part_bytes(BH, G, D, slots);
  if (need && (!workspace || workspace_bytes < need))
    return fail(FATHOM_ERR_WORKSPACE, "rows8_gather_attention: workspace %zu bytes, need %zu", workspace_bytes, need);
  if (need && reinterpret_cast<uintptr_t>(workspace) & 15)
    return fail(FATHOM_ERR_INVALID, "rows8_gather_attention: the workspace must be 16-byte aligned");
  place(a, workspace, D, slots, false);
  return run_list(a, BH, D, code_dtype == FATHOM_DT_I8, (hipStream_t)stream);
}
