// Chunk attention and shared-prefix attention over the 8-bit K/V row store: entry
// points, shares of the work, and the join of partial results.
#include "rows8_multi.hpp"

namespace fathom {
namespace rows8 {
namespace {

constexpr int kJoinThreads = 256;
constexpr int64_t kMaxTiles = 65535;  // grid y
// Queries from which D / 4 lanes join each one's splits: they fill the device, and have few splits each (8 x 12 x 396 queries over 501
// tokens in two shares 78 us with a workgroup per query; 38).
constexpr int64_t kJoinMany = 4096;
// Below that D / 32 workgroups take a query's channels (8 queries of 320 splits 28 us with the call; 24.  512 of 16 ragged ones 27.5; 28.7).
constexpr int64_t kJoinWide = 512;

// Where the partial results of query m of row blockIdx.y lie: `own` splits of its tile and, behind a shared prefix, `more` of its
// sequence's own tokens; `to` is its place in the output, in rows.
struct JoinFrom {
  int own, more;
  int64_t at, slot, to;
  __device__ __forceinline__ float2 ml(const MultiArgs &a, const Tail &t, int s) const {
    return s < own ? a.ml[at + (int64_t)s * a.rows] : t.ml[slot + (int64_t)(s - own) * a.G];
  }
  __device__ __forceinline__ const float *part(const MultiArgs &a, const Tail &t, int s, int D) const {
    return s < own ? a.part + (at + (int64_t)s * a.rows) * D : t.part + (slot + (int64_t)(s - own) * a.G) * D;
  }
};
__device__ __forceinline__ JoinFrom join_from(const MultiArgs &a, const Tail &tail, int m) {
  const int64_t r = blockIdx.y, g = m % a.G, o = m / a.G;
  const int tile = (int)r * a.tiles + m / a.rows;
  const int2 from = a.splits ? make_int2(tile * a.splits, a.splits) : a.where[tile];
  JoinFrom f{from.y, 0, (int64_t)from.x * a.rows + m % a.rows, 0, a.shared ? (o * a.BH + r) * a.G + g : (r * a.G + g) * a.O + o};
  if (a.shared) {
    const int64_t row = o * a.BH + r;
    const int2 w = tail.where ? tail.where[row] : make_int2((int)(row * tail.nsplit), (int)tail.nsplit);
    f.slot = (int64_t)w.x * a.G + g;
    f.more = w.y;
  }
  return f;
}

// Splits first, first + step, .. of a query in channels c .. c + 3: their largest score and, relative to it, the sums.  Four are on
// their way at a time (8 x 4 x 140 queries over 8000 tokens 52 us one by one; 47.5).
struct Joined {
  float big, l;
  float4 v;
};
__device__ __forceinline__ Joined join_splits(const MultiArgs &a, const Tail &tail, const JoinFrom &from, int first, int step, int D, int c) {
  const int ns = from.own + from.more;
  float big = kLowest, l = 0.0f;
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int s0 = first; s0 < ns; s0 += 4 * step) {
    float2 x[4];
    float4 u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int s = s0 + j * step, at = s < ns ? s : s0;
      x[j] = from.ml(a, tail, at);
      u[j] = *reinterpret_cast<const float4 *>(from.part(a, tail, at, D) + c);
      if (s >= ns) x[j].y = 0.0f;
    }
    float top = big;
#pragma unroll
    for (int j = 0; j < 4; ++j) top = fmaxf(top, x[j].x);
    const float was = __builtin_amdgcn_exp2f(big - top);
    big = top;
    l *= was;
    v = make_float4(v.x * was, v.y * was, v.z * was, v.w * was);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (x[j].y == 0.0f) continue;  // no weight, and perhaps nothing written
      const float f = __builtin_amdgcn_exp2f(x[j].x - top);
      l = fmaf(x[j].y, f, l);
      v.x = fmaf(u[j].x, f, v.x);
      v.y = fmaf(u[j].y, f, v.y);
      v.z = fmaf(u[j].z, f, v.z);
      v.w = fmaf(u[j].w, f, v.w);
    }
  }
  return Joined{big, l, v};
}

// Joins a query's splits, and its sequence's own tokens behind a shared prefix: a workgroup per query and CH channels, of which
// CH / 4 lanes take every (1024 / CH)-th split.  Bound: latency, and L2 for many (1024 queries of 64 splits, 34 MB, 9 us).
template <int D, int CH, int OUT>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(MultiArgs a, Tail tail) {
  constexpr int kLanes = CH / 4, kGroups = kJoinThreads / kLanes;
  __shared__ float4 acc[kGroups][kLanes];
  __shared__ float2 sums[kGroups];
  const int tid = threadIdx.x, lane = tid % kLanes, grp = tid / kLanes, c0 = CH * (int)blockIdx.z;
  const JoinFrom from = join_from(a, tail, (int)blockIdx.x);
  const Joined mine = join_splits(a, tail, from, grp, kGroups, D, c0 + 4 * lane);
  acc[grp][lane] = mine.v;
  if (lane == 0) sums[grp] = make_float2(mine.big, mine.l);
  __syncthreads();
  if (tid >= CH) return;
  float big = kLowest, sum = 0.0f, l = 0.0f;
#pragma unroll
  for (int k = 0; k < kGroups; ++k) big = fmaxf(big, sums[k].x);
#pragma unroll
  for (int k = 0; k < kGroups; ++k) {
    const float f = __builtin_amdgcn_exp2f(sums[k].x - big);
    sum = fmaf(reinterpret_cast<const float *>(acc[k])[tid], f, sum);
    l = fmaf(sums[k].y, f, l);
  }
  const float out = l == 0.0f ? 0.0f : sum / l;
  const int64_t to = from.to * D + c0 + tid;
  if constexpr (OUT == FATHOM_DT_F32) static_cast<float *>(a.out)[to] = out;
  else if constexpr (OUT == FATHOM_DT_F16) static_cast<uint16_t *>(a.out)[to] = float_to_f16_bits(out);
  else static_cast<uint16_t *>(a.out)[to] = float_to_bf16_bits(out);
}

// The same for many queries: D / 4 lanes take all of a query's splits.
template <int D, int OUT>
__global__ __launch_bounds__(kJoinThreads) void join_many_kernel(MultiArgs a, Tail tail) {
  constexpr int kLanes = D / 4;
  const int lane = threadIdx.x % kLanes, m = (int)blockIdx.x * (kJoinThreads / kLanes) + threadIdx.x / kLanes;
  if (m >= a.G * a.O) return;
  const JoinFrom from = join_from(a, tail, m);
  const Joined all = join_splits(a, tail, from, 0, 1, D, 4 * lane);
  const float v[4] = {all.v.x, all.v.y, all.v.z, all.v.w};
  float out[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) out[k] = all.l == 0.0f ? 0.0f : v[k] / all.l;
  store4<OUT>(a.out, from.to * D + 4 * lane, out);
}

template <int D, int CH>
void launch_join(const MultiArgs &a, const Tail &t, int out, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.G * a.O), (unsigned)a.BH, D / CH);
  if (out == FATHOM_DT_F32) join_kernel<D, CH, FATHOM_DT_F32><<<grid, kJoinThreads, 0, st>>>(a, t);
  else if (out == FATHOM_DT_F16) join_kernel<D, CH, FATHOM_DT_F16><<<grid, kJoinThreads, 0, st>>>(a, t);
  else join_kernel<D, CH, FATHOM_DT_BF16><<<grid, kJoinThreads, 0, st>>>(a, t);
}
template <int D>
void launch_join(const MultiArgs &a, const Tail &t, int out, hipStream_t st) {
  const int64_t M = (int64_t)a.G * a.O;
  if (M * a.BH >= kJoinMany) {
    const dim3 grid((unsigned)cdiv(M, (int64_t)(1024 / D)), (unsigned)a.BH);
    if (out == FATHOM_DT_F32) join_many_kernel<D, FATHOM_DT_F32><<<grid, kJoinThreads, 0, st>>>(a, t);
    else if (out == FATHOM_DT_F16) join_many_kernel<D, FATHOM_DT_F16><<<grid, kJoinThreads, 0, st>>>(a, t);
    else join_many_kernel<D, FATHOM_DT_BF16><<<grid, kJoinThreads, 0, st>>>(a, t);
    return;
  }
  if (M * a.BH >= kJoinWide) launch_join<D, D>(a, t, out, st);
  else launch_join<D, 32>(a, t, out, st);
}

// The tiles of a call: queries of one, and workgroups that are at work at once.
struct Tiling {
  int rows;
  int64_t places;
};
constexpr Tiling kTilings[] = {{32, 512}, {32, 256}, {128, 512}, {256, 256}};

bool takes_four(const MultiArgs &a, int q_dtype) { return q_dtype == FATHOM_DT_F32 || a.softcap > 0.0f || a.slopes; }

// Queries of a tile of rows that see up to nb blocks: one wave's, where a row has no more; eight waves', which stage a block for
// twice the queries (8 x 4 x 2048 over 65536 tokens 2.22 ms; by fours 2.44), where that leaves no more of their places empty or the
// queries are many, and there is work for all CUs in shares of four blocks (512 queries of 4 rows over 4096 tokens 42 us; 38).
// `four`: float32 queries and calls with a cap or bias take four waves.  Their registers or a block's longer way leave eight
// to wait for the slowest (f32, 8 x 4 x 1024 over 16384 tokens 797 us; 728.  Capped and biased, 4 x 12 x 3001 behind a window of
// 4096: 535; 464).
// A wave by itself with float32 queries, a cap or a bias has a SIMD's registers at D = 128, so that half as many workgroups are
// at work (8 rows of 262144 tokens, 4 x 4 f32 queries 119 us in twice as many shares; 105).
Tiling tiling_of(int64_t BH, int64_t M, int64_t D, int64_t nb, bool four) {
  if (M <= 32) return kTilings[four && D == 128 ? 1 : 0];
  const int64_t eights = cdiv(M, (int64_t)256);
  return kTilings[!four && (M >= 2048 || eights * 2 == cdiv(M, (int64_t)128)) && BH * eights * cdiv(nb, (int64_t)4) >= 256 ? 3 : 2];
}

// Whether tiles of up to nb blocks, of rows of one length, are cut into shares: up to half as many tiles as places where more
// than the partial results' time is won, about four blocks and with more queries more (8 x 12 x 200 queries over 501 tokens 22 us
// a workgroup per tile, 32 cut; over 1000 tokens 45, 37); up to three quarters where rows are long (8 x 4 x 1100 over 20000 tokens 647
// us, 478; x 1500 over 32768 1053, 1008, over 8192 278, 290).  More even out by themselves, those that see most first.
bool shares_pay(int64_t tiles, int64_t places, int64_t nb) {
  const int64_t won = nb * (places - tiles);
  return 2 * tiles <= places ? won > 4 * places + 10 * tiles : 4 * tiles <= 3 * places && won > 64 * places;
}

// The same for tiles of 32 queries, whose four waves take blocks in turn, and for ragged rows of such (600 rows of up to 1500
// tokens 27 us a workgroup per row, 53 cut; of up to 16000 201, 180).  Rows of one length that keep 7 of 10 CUs busy reach HBM's
// rate by themselves (200 of 16000 tokens 131 us, 140 cut; 300, two on some CUs, 258, 220; 128 of 8000 60, 49).
bool shares_pay_32(int64_t tiles, int64_t places, int64_t nb, bool ragged) {
  if (ragged) return nb * places > 16 * places + 96 * tiles;
  const int64_t cus = 256 * cdiv(tiles, (int64_t)256);
  return 10 * tiles < 7 * cus && (tiles > 256 ? nb > 128 : 256 * nb > 12 * 256 + 40 * tiles);
}

// Shares that tiles of up to nb blocks are cut into (at most that many and one per tile more); 0: a workgroup takes each tile.
// Few tiles are cut so that all places have the same to do; more of them, as those of ragged rows up to twice the places, into a
// few rounds, as every tile's last share is shorter; of shares, a workgroup's partial results cost about four blocks.  (32 ragged
// rows of 572 tokens of 4 heads in up to 16000: 1114 us a workgroup per tile; 414.)
int64_t tile_shares(int64_t BH, int64_t M, Tiling t, int64_t nb) {
  const int64_t tiles = BH * cdiv(M, (int64_t)t.rows), places = t.places;
  if (nb <= (t.rows == 32 ? 16 : 4) || tiles >= 2 * places) return 0;
  const int64_t rounds = cdiv(3 * tiles, places), most = tiles * cdiv(nb, (int64_t)4);
  const int64_t shares = rounds == 1 ? places - tiles : places * rounds - tiles * 5 / 8;
  return most < shares ? most : shares;
}
// Splits of each of so many tiles that all have the same to do, of four blocks and more: as many as there are places, or, of tiles of
// 32 queries, no more than are at work at once (128 rows of 8000 tokens, f32 queries, in two rounds 66 us; 57).
int64_t tile_splits(int64_t tiles, Tiling t, int64_t shares, int64_t nb) {
  int64_t room = (shares + tiles) / tiles;
  if (t.rows == 32 && tiles <= t.places) room = std::min(room, t.places / tiles);
  const int64_t most = cdiv(nb, (int64_t)4);
  return most < 1 ? 1 : room < most ? room : most;
}
// The same for a prefix, whose tiles always leave partial results.
int64_t prefix_shares(int64_t BH, int64_t M, Tiling t, int64_t nb) {
  const int64_t tiles = BH * cdiv(M, (int64_t)t.rows);
  const int64_t shares = 2 * tiles <= t.places || shares_pay(tiles, t.places, nb) ? tile_shares(BH, M, t, nb) : 0;
  return shares > tiles ? shares : tiles;
}

// Blocks that a tile sees at most, of rows of up to n tokens.
int64_t tile_blocks(int64_t n, int64_t T, int64_t window, int64_t sinks) {
  const int64_t all = cdiv(n, (int64_t)kBlk);
  if (window <= 0 || window >= n) return all;
  const int64_t some = cdiv(window + T - 1, (int64_t)kBlk) + 1 + cdiv(sinks < n ? sinks : n, (int64_t)kBlk);
  return some < all ? some : all;
}

// Bytes of the partial results of so many shares and of the tiles' slots.
size_t multi_bytes(int64_t BH, int64_t M, int rows, int64_t D, int64_t shares) {
  const int64_t tiles = BH * cdiv(M, (int64_t)rows);
  return (size_t)((shares + tiles) * rows * (D + 2) + cdiv(2 * tiles, (int64_t)4) * 4) * sizeof(float);
}

// Whether a call takes so many queries: of a row at most 65535 tiles of 32, in all so many that a grid of two workgroups per
// tile stays below 2^32 threads.
bool queries_taken(int64_t BH, int64_t G, int64_t O) {
  return O >= 1 && O <= kMaxCap && G <= kMaxTiles * 32 / O && BH * G * O <= (int64_t)1 << 27;
}

// The kernel keeps its factors, scale log2 e among them, in float32's range, and would make finite ones of other scales.
int check_scale(const char *what, float scale) {
  return fabsf(scale) <= 0x1p127f ? FATHOM_OK : fail(FATHOM_ERR_INVALID, "%s: the scale must be finite, of at most 2^127", what);
}

void place(MultiArgs &a, void *workspace, int64_t D) {
  const int64_t rows = (a.shares + a.BH * a.tiles) * a.rows;
  a.part = static_cast<float *>(workspace);
  a.ml = reinterpret_cast<float2 *>(a.part + rows * D);
  a.where = reinterpret_cast<int2 *>(a.ml + rows);
  a.parts = true;
}

int run_multi(const MultiArgs &a, int q_dtype, int64_t D, bool i8, hipStream_t st) {
  if (D == 128 && i8) launch_multi_d128_int8(a, q_dtype, st);
  else if (D == 128) launch_multi_d128_e4m3(a, q_dtype, st);
  else if (i8) launch_multi_d64_int8(a, q_dtype, st);
  else launch_multi_d64_e4m3(a, q_dtype, st);
  return launch_status("rows8 multi_kernel");
}

int run_join(const MultiArgs &a, const Tail &t, int out, int64_t D, hipStream_t st) {
  if (D == 128) launch_join<128>(a, t, out, st);
  else launch_join<64>(a, t, out, st);
  return launch_status("rows8 join_kernel");
}

}  // namespace
}  // namespace rows8
}  // namespace fathom

using namespace fathom;
using namespace fathom::rows8;

extern "C" size_t fathom_rows8_chunk_attention_workspace_bytes(int64_t BH, int64_t G, int64_t T, int64_t D, int64_t positions) {
  if (!shape_taken(BH, G, D) || !queries_taken(BH, G, T) || positions < 1) return 0;
  if (positions > kMaxCap) positions = kMaxCap;
  size_t most = 0;  // of whichever tiles a call takes
  for (const Tiling t : kTilings) {
    if ((t.rows == 32) != (G * T <= 32)) continue;
    const int64_t shares = tile_shares(BH, G * T, t, cdiv(positions, (int64_t)kBlk) + 1);
    if (shares) most = std::max(most, multi_bytes(BH, G * T, t.rows, D, shares));
  }
  return most;
}

extern "C" int fathom_rows8_chunk_attention(const void *q, int q_dtype, int64_t q_row_stride, int64_t q_head_stride,
                                            int64_t q_tok_stride, const void *k8, const void *v8, const float *k_scale,
                                            const float *v_scale, int code_dtype, int64_t BH, int64_t G, int64_t T, int64_t D,
                                            int64_t cap, const int32_t *lens, int64_t n, int64_t window, int64_t sinks,
                                            float scale, float softcap, const float *slopes, void *out, void *workspace,
                                            size_t workspace_bytes, void *stream) {
  const char *what = "rows8_chunk_attention";
  int rc = check_store(what, k8, v8, k_scale, v_scale, code_dtype, BH, cap, D);
  if (rc) return rc;
  if (T < 0) return fail(FATHOM_ERR_INVALID, "%s: T=%lld", what, (long long)T);
  if (T == 0) return FATHOM_OK;
  rc = check_query(what, q, q_dtype, G, cap, lens, n, softcap, out);
  if (rc) return rc;
  rc = check_scale(what, scale);
  if (rc) return rc;
  if (!queries_taken(BH, G, T)) return fail(FATHOM_ERR_INVALID, "%s: G=%lld T=%lld, at most %lld queries per row and 2^27 in all", what, (long long)G, (long long)T, (long long)kMaxTiles * 32);
  if (window < 0) return fail(FATHOM_ERR_INVALID, "%s: window %lld", what, (long long)window);
  if (sinks < 0) return fail(FATHOM_ERR_INVALID, "%s: sinks %lld", what, (long long)sinks);
  const int64_t size = q_dtype == FATHOM_DT_F32 ? 4 : 2;
  if (((q_row_stride | q_head_stride | q_tok_stride) * size) & 15 || reinterpret_cast<uintptr_t>(out) & 15)
    return fail(FATHOM_ERR_INVALID, "%s: the strides of q and out must be multiples of 16 bytes", what);
  if (window >= cap) window = 0;
  if (sinks > cap) sinks = cap;
  MultiArgs a{q, q_row_stride, q_head_stride, q_tok_stride, (const uint8_t *)k8, (const uint8_t *)v8, k_scale, v_scale, cap,
              cdiv(cap, kBlk), lens, n, (int)G, (int)T, (int)window, (int)sinks, false, nullptr, 0, 0, BH, scale,
              kernel_cap(softcap), slopes, out, nullptr, nullptr, nullptr, 0, 1, 0, 0, false};
  const int64_t most = lens ? cap : n;
  const int64_t nb = tile_blocks(most, T, window, sinks);
  const Tiling t = tiling_of(BH, G * T, D, nb, takes_four(a, q_dtype));
  a.rows = t.rows;
  a.tiles = (int)cdiv(G * T, (int64_t)a.rows);
  const int64_t tiles = BH * a.tiles;
  const bool cut = a.rows == 32 ? shares_pay_32(tiles, t.places, nb, lens) : lens || shares_pay(tiles, t.places, nb);
  a.shares = cut ? (int)tile_shares(BH, G * T, t, nb) : 0;
  if (a.shares) {
    const size_t need = multi_bytes(BH, G * T, a.rows, D, a.shares);
    if (!workspace || workspace_bytes < need)
      return fail(FATHOM_ERR_WORKSPACE, "%s: workspace %zu bytes, need %zu", what, workspace_bytes, need);
    if (reinterpret_cast<uintptr_t>(workspace) & 15)
      return fail(FATHOM_ERR_INVALID, "%s: the workspace must be 16-byte aligned", what);
    place(a, workspace, D);
    // tiles that see nearly the same are cut equally, without a search
    if (!lens && (window > 0 || most >= 4 * T) && 2 * tiles <= t.places) a.splits = (int)tile_splits(tiles, t, a.shares, nb);
  }
  rc = run_multi(a, q_dtype, D, code_dtype == FATHOM_DT_I8, (hipStream_t)stream);
  return rc || !a.shares ? rc : run_join(a, Tail{}, q_dtype, D, (hipStream_t)stream);
}

extern "C" size_t fathom_rows8_shared_attention_workspace_bytes(int64_t prefix_BH, int64_t sequences, int64_t G, int64_t D,
                                                                int64_t prefix_positions, int64_t positions) {
  if (!shape_taken(prefix_BH, G, D) || !queries_taken(prefix_BH, G, sequences) || sequences > kMaxRows / prefix_BH) return 0;
  if (prefix_positions > kMaxCap) prefix_positions = kMaxCap;
  if (prefix_positions < 0) prefix_positions = 0;
  size_t most = 0;  // of whichever tiles a call takes
  for (const Tiling t : kTilings) {
    if ((t.rows == 32) != (G * sequences <= 32)) continue;
    const int64_t shares = prefix_shares(prefix_BH, G * sequences, t, cdiv(prefix_positions, (int64_t)kBlk));
    most = std::max(most, multi_bytes(prefix_BH, G * sequences, t.rows, D, shares));
  }
  return most + tail_bytes(prefix_BH * sequences, G, D, positions < 0 ? 0 : positions);
}

extern "C" int fathom_rows8_shared_attention(const void *q, int q_dtype, const void *prefix_k8, const void *prefix_v8,
                                             const float *prefix_k_scale, const float *prefix_v_scale, int64_t prefix_BH,
                                             int64_t prefix_cap, const int32_t *prefix_lens, int64_t prefix_n, const void *k8,
                                             const void *v8, const float *k_scale, const float *v_scale, int code_dtype,
                                             int64_t sequences, int64_t G, int64_t D, int64_t cap, const int32_t *lens, int64_t n,
                                             float scale, float softcap, const float *slopes, float *out, void *workspace,
                                             size_t workspace_bytes, void *stream) {
  const char *what = "rows8_shared_attention";
  int rc = check_store(what, prefix_k8, prefix_v8, prefix_k_scale, prefix_v_scale, code_dtype, prefix_BH, prefix_cap, D);
  if (rc) return rc;
  if (sequences < 1 || sequences > kMaxRows / prefix_BH)
    return fail(FATHOM_ERR_INVALID, "%s: %lld sequences of %lld rows, at most 65535 rows", what, (long long)sequences, (long long)prefix_BH);
  const int64_t BH = prefix_BH * sequences;
  rc = check_store(what, k8, v8, k_scale, v_scale, code_dtype, BH, cap, D);
  if (!rc) rc = check_query(what, q, q_dtype, G, cap, lens, n, softcap, out);
  if (rc) return rc;
  rc = check_scale(what, scale);
  if (rc) return rc;
  if (!prefix_lens && (prefix_n < 0 || prefix_n > prefix_cap))
    return fail(FATHOM_ERR_INVALID, "%s: prefix length %lld outside [0, cap=%lld]", what, (long long)prefix_n, (long long)prefix_cap);
  if (!queries_taken(prefix_BH, G, sequences))
    return fail(FATHOM_ERR_INVALID, "%s: %lld sequences, G=%lld, at most %lld queries per row and 2^27 in all", what, (long long)sequences, (long long)G, (long long)kMaxTiles * 32);
  MultiArgs a{q, G * D, D, prefix_BH * G * D, (const uint8_t *)prefix_k8, (const uint8_t *)prefix_v8, prefix_k_scale,
              prefix_v_scale, prefix_cap, cdiv(prefix_cap, kBlk), prefix_lens, prefix_n, (int)G, (int)sequences, 0, 0, true,
              lens, n, cap, prefix_BH, scale, kernel_cap(softcap), slopes, out, nullptr, nullptr, nullptr, 1, 1, 0, 0, false};
  const int64_t nb = cdiv(prefix_lens ? prefix_cap : prefix_n, (int64_t)kBlk);
  const Tiling by = tiling_of(prefix_BH, G * sequences, D, nb, takes_four(a, q_dtype));
  a.rows = by.rows;
  a.tiles = (int)cdiv(G * sequences, (int64_t)a.rows);
  a.shares = (int)prefix_shares(prefix_BH, G * sequences, by, nb);
  const size_t first = multi_bytes(prefix_BH, G * sequences, a.rows, D, a.shares);
  if (!workspace || workspace_bytes < first)
    return fail(FATHOM_ERR_WORKSPACE, "%s: workspace %zu bytes, need more than %zu", what, workspace_bytes, first);
  if (reinterpret_cast<uintptr_t>(workspace) & 15)
    return fail(FATHOM_ERR_INVALID, "%s: the workspace must be 16-byte aligned", what);
  place(a, workspace, D);
  const int64_t tiles = prefix_BH * a.tiles;
  if (!prefix_lens && (2 * tiles <= by.places || a.shares == tiles)) a.splits = (int)tile_splits(tiles, by, a.shares, nb);
  const bool i8 = code_dtype == FATHOM_DT_I8;
  const hipStream_t st = (hipStream_t)stream;
  Tail t;
  rc = tail_attention(t, what, q, q_dtype, k8, v8, k_scale, v_scale, i8, BH, G, D, cap, lens, n, scale, softcap, slopes,
                      static_cast<char *>(workspace) + first, workspace_bytes - first, st);
  if (!rc) rc = run_multi(a, q_dtype, D, i8, st);
  return rc ? rc : run_join(a, t, FATHOM_DT_F32, D, st);
}
