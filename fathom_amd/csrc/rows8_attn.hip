// Attention of single tokens over the 8-bit K/V row store: over a whole row (or
// its last tokens), or over listed tokens.
//
// With len the row's length and c the codes, for query head g of row bh:
//   u_t = scale s_K(t) (q . cK_t)
//   z_t = softcap tanh(u_t / softcap) (u_t without a cap) + slope_g (t - (len - 1))
//   out = sum_t e^(z_t - m) s_V(t) cV_t / sum_t e^(z_t - m)
// over the tokens t of [max(0, len - window), len), or the listed ones of [0, len).
// Scores, maxima, sums and the weighted rows are float32.
#include "rows8.hpp"

namespace fathom {
namespace rows8 {
namespace {

constexpr int kWaves = 4;  // of a workgroup
constexpr int kTile = 32;  // positions of a wave at a time

struct AttnArgs {
  const void *q;
  int q_dtype;
  const uint8_t *k8, *v8;
  const float *ks, *vs;
  int64_t G, cap, nblk;
  const int32_t *lens;
  int64_t n, window;
  const int64_t *idx;
  int64_t k;
  float scale, softcap;
  const float *slopes;
  float *out, *part;
  int64_t nsplit;
};

__device__ __forceinline__ float load_q(const void *q, int dt, int64_t i) {
  return dt == FATHOM_DT_F32   ? load_elem<FATHOM_DT_F32>(q, i)
         : dt == FATHOM_DT_F16 ? load_elem<FATHOM_DT_F16>(q, i)
                               : load_elem<FATHOM_DT_BF16>(q, i);
}

// Adds (m1, l1, o1) to the running (m, l, o) of a softmax.
template <int N>
__device__ __forceinline__ void join(float &m, float &l, float (&o)[N], float m1, float l1, const float (&o1)[N]) {
  const float M = fmaxf(m, m1);
  const float f = m == -INFINITY ? 0.0f : expf(m - M), f1 = m1 == -INFINITY ? 0.0f : expf(m1 - M);
  l = l * f + l1 * f1;
#pragma unroll
  for (int e = 0; e < N; ++e) o[e] = o[e] * f + o1[e] * f1;
  m = M;
}

// One workgroup per (split, query head, row); its waves take tiles of 32
// positions in turn.  16 channels of a row per lane.
template <int D, bool I8, bool LIST>
__global__ __launch_bounds__(kWaves *kWave) void attn_kernel(AttnArgs a) {
  constexpr int kLanes = D / 16;         // lanes of a row
  constexpr int kRows = kWave / kLanes;  // rows of a load
  constexpr int kLoads = kTile / kRows;
  __shared__ float wm[kWaves], wl[kWaves], wo[kWaves][D];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t s = blockIdx.x, g = blockIdx.y, bh = blockIdx.z;
  const int d0 = 16 * (lane % kLanes), rg = lane / kLanes;
  const int64_t len = row_length(a.lens, a.n, a.cap, bh);
  const int64_t lo = !LIST && a.window > 0 && len > a.window ? len - a.window : 0;
  const int64_t count = LIST ? a.k : len - lo;
  const float slope = a.slopes ? a.slopes[bh * a.G + g] : 0.0f;
  float q[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) q[e] = load_q(a.q, a.q_dtype, (bh * a.G + g) * D + d0 + e);
  float m = -INFINITY, l = 0.0f, o[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) o[e] = 0.0f;
  for (int64_t t0 = (s * kWaves + wave) * kTile; t0 < count; t0 += a.nsplit * kWaves * kTile) {
    int64_t tok[kLoads];
    bool in[kLoads];
    uint4 kc[kLoads], vc[kLoads];
    float ks[kLoads], vs[kLoads], z[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int64_t j = t0 + i * kRows + rg;
      tok[i] = j >= count ? -1 : LIST ? a.idx[(bh * a.G + g) * a.k + j] : lo + j;
      in[i] = tok[i] >= 0 && tok[i] < len;
      kc[i] = vc[i] = make_uint4(0u, 0u, 0u, 0u);
      ks[i] = vs[i] = 0.0f;
      if (in[i]) {
        const int64_t at = (bh * a.cap + tok[i]) * D + d0, b = bh * a.nblk + tok[i] / kBlk;
        kc[i] = *reinterpret_cast<const uint4 *>(a.k8 + at);
        vc[i] = *reinterpret_cast<const uint4 *>(a.v8 + at);
        ks[i] = a.ks[b];
        vs[i] = a.vs[b];
      }
    }
    float mt = m;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint32_t w[4] = {kc[i].x, kc[i].y, kc[i].z, kc[i].w};
      float dot = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float c[4];
        decode4<I8>(w[e], c);
#pragma unroll
        for (int f = 0; f < 4; ++f) dot = fmaf(q[4 * e + f], c[f], dot);
      }
#pragma unroll
      for (int x = 1; x < kLanes; x <<= 1) dot += __shfl_xor(dot, x);
      float u = dot * (ks[i] * a.scale);
      if (a.softcap > 0.0f) u = a.softcap * tanhf(u / a.softcap);
      z[i] = in[i] ? fmaf(slope, (float)(tok[i] - (len - 1)), u) : -INFINITY;
      mt = fmaxf(mt, z[i]);
    }
    const float f = m == -INFINITY ? 0.0f : expf(m - mt);
    l *= f;
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] *= f;
    m = mt;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const float p = z[i] == -INFINITY ? 0.0f : expf(z[i] - m);
      l += p;
      const float pv = p * vs[i];
      const uint32_t w[4] = {vc[i].x, vc[i].y, vc[i].z, vc[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float c[4];
        decode4<I8>(w[e], c);
#pragma unroll
        for (int x = 0; x < 4; ++x) o[4 * e + x] = fmaf(pv, c[x], o[4 * e + x]);
      }
    }
  }
  // the wave's row groups, then the workgroup's waves
#pragma unroll
  for (int x = kLanes; x < kWave; x <<= 1) {
    float o1[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) o1[e] = __shfl_xor(o[e], x);
    const float m1 = __shfl_xor(m, x), l1 = __shfl_xor(l, x);
    join<16>(m, l, o, m1, l1, o1);
  }
  if (rg == 0)
#pragma unroll
    for (int e = 0; e < 16; ++e) wo[wave][d0 + e] = o[e];
  if (lane == 0) {
    wm[wave] = m;
    wl[wave] = l;
  }
  __syncthreads();
  if (tid < D) {
    float M = wm[0], L = wl[0], O[1] = {wo[0][tid]};
    for (int v = 1; v < kWaves; ++v) {
      const float o1[1] = {wo[v][tid]};
      join<1>(M, L, O, wm[v], wl[v], o1);
    }
    const int64_t r = bh * a.G + g;
    if (a.nsplit == 1) {
      a.out[r * D + tid] = L == 0.0f ? 0.0f : O[0] / L;
    } else {
      float *pb = a.part + (r * a.nsplit + s) * (D + 2);
      pb[2 + tid] = O[0];
      if (tid == 0) {
        pb[0] = M;
        pb[1] = L;
      }
    }
  }
}

// Joins the splits of a query head, in their order.
template <int D>
__global__ __launch_bounds__(D) void merge_kernel(const float *__restrict__ part, int64_t nsplit, float *__restrict__ out) {
  const int64_t r = blockIdx.x;
  const int d = threadIdx.x;
  float m = -INFINITY, l = 0.0f, o[1] = {0.0f};
  for (int64_t s = 0; s < nsplit; ++s) {
    const float *pb = part + (r * nsplit + s) * (D + 2);
    const float o1[1] = {pb[2 + d]};
    join<1>(m, l, o, pb[0], pb[1], o1);
  }
  out[r * D + d] = l == 0.0f ? 0.0f : o[0] / l;
}

// Splits of a head's positions: enough workgroups for the chip, at least one tile each.
int64_t splits(int64_t heads, int64_t positions) {
  const int64_t most = cdiv(positions, (int64_t)kWaves * kTile), want = cdiv((int64_t)2048, heads);
  const int64_t s = most < want ? most : want;
  return s < 1 ? 1 : s;
}

size_t workspace(int64_t BH, int64_t G, int64_t D, int64_t positions) {
  if (BH < 1 || G < 1 || D < 1 || positions < 0) return 0;
  const int64_t ns = splits(BH * G, positions);
  return ns == 1 ? 0 : (size_t)(BH * G * ns * (D + 2)) * sizeof(float);
}

template <bool LIST>
int run(const char *what, AttnArgs a, int64_t BH, int64_t D, bool i8, int64_t positions, size_t workspace_bytes,
        hipStream_t st) {
  const size_t need = workspace(BH, a.G, D, positions);
  if (need && (!a.part || workspace_bytes < need))
    return fail(FATHOM_ERR_WORKSPACE, "%s: workspace %zu bytes, need %zu", what, workspace_bytes, need);
  a.nsplit = splits(BH * a.G, positions);
  const dim3 grid((unsigned)a.nsplit, (unsigned)a.G, (unsigned)BH);
  if (D == 128 && i8) attn_kernel<128, true, LIST><<<grid, kWaves * kWave, 0, st>>>(a);
  else if (D == 128) attn_kernel<128, false, LIST><<<grid, kWaves * kWave, 0, st>>>(a);
  else if (i8) attn_kernel<64, true, LIST><<<grid, kWaves * kWave, 0, st>>>(a);
  else attn_kernel<64, false, LIST><<<grid, kWaves * kWave, 0, st>>>(a);
  const int rc = launch_status(what);
  if (rc || a.nsplit == 1) return rc;
  if (D == 128) merge_kernel<128><<<(unsigned)(BH * a.G), 128, 0, st>>>(a.part, a.nsplit, a.out);
  else merge_kernel<64><<<(unsigned)(BH * a.G), 64, 0, st>>>(a.part, a.nsplit, a.out);
  return launch_status("rows8 merge_kernel");
}

int check_query(const char *what, const void *q, int q_dtype, int64_t BH, int64_t G, int64_t D, int64_t cap, const int32_t *lens,
                int64_t n, float softcap, const float *out) {
  if (!q || !out) return fail(FATHOM_ERR_INVALID, "%s: null pointer", what);
  if (q_dtype < FATHOM_DT_F32 || q_dtype > FATHOM_DT_BF16) return fail(FATHOM_ERR_INVALID, "%s: q_dtype %d", what, q_dtype);
  if (G < 1 || G > 65535) return fail(FATHOM_ERR_INVALID, "%s: G=%lld", what, (long long)G);
  if (!lens && (n < 0 || n > cap)) return fail(FATHOM_ERR_INVALID, "%s: length %lld outside [0, cap=%lld]", what, (long long)n, (long long)cap);
  if (!(softcap >= 0.0f)) return fail(FATHOM_ERR_INVALID, "%s: softcap must be 0 (none) or positive", what);
  if (reinterpret_cast<uintptr_t>(q) & 15) return fail(FATHOM_ERR_INVALID, "%s: q must be 16-byte aligned", what);
  (void)BH;
  (void)D;
  return FATHOM_OK;
}

// An upper bound of a row's positions that the host knows.
int64_t dense_positions(const int32_t *lens, int64_t n, int64_t cap, int64_t window) {
  const int64_t most = lens ? cap : n;
  return window > 0 && window < most ? window : most;
}

}  // namespace
}  // namespace rows8
}  // namespace fathom

using namespace fathom;
using namespace fathom::rows8;

extern "C" size_t fathom_rows8_attention_workspace_bytes(int64_t BH, int64_t G, int64_t D, int64_t positions) {
  return workspace(BH, G, D, positions);
}

extern "C" int fathom_rows8_attention(const void *q, int q_dtype, const void *k8, const void *v8, const float *k_scale,
                                      const float *v_scale, int code_dtype, int64_t BH, int64_t G, int64_t D, int64_t cap,
                                      const int32_t *lens, int64_t n, int64_t window, float scale, float softcap,
                                      const float *slopes, float *out, void *workspace, size_t workspace_bytes,
                                      void *stream) {
  int rc = check_store("rows8_attention", k8, v8, k_scale, v_scale, code_dtype, BH, cap, D);
  if (!rc) rc = check_query("rows8_attention", q, q_dtype, BH, G, D, cap, lens, n, softcap, out);
  if (rc) return rc;
  if (window < 0) return fail(FATHOM_ERR_INVALID, "rows8_attention: window %lld", (long long)window);
  AttnArgs a{q, q_dtype, (const uint8_t *)k8, (const uint8_t *)v8, k_scale, v_scale, G, cap, cdiv(cap, kBlk), lens, n, window,
             nullptr, 0, scale, softcap, slopes, out, (float *)workspace, 1};
  return run<false>("rows8_attention", a, BH, D, code_dtype == FATHOM_DT_I8, dense_positions(lens, n, cap, window),
                    workspace_bytes, (hipStream_t)stream);
}

extern "C" size_t fathom_rows8_gather_attention_workspace_bytes(int64_t BH, int64_t G, int64_t D, int64_t k) {
  return workspace(BH, G, D, k);
}

extern "C" int fathom_rows8_gather_attention(const void *q, int q_dtype, const int64_t *idx, const void *k8, const void *v8,
                                             const float *k_scale, const float *v_scale, int code_dtype, int64_t BH,
                                             int64_t G, int64_t k, int64_t D, int64_t cap, const int32_t *lens, int64_t n,
                                             float scale, float softcap, const float *slopes, float *out, void *workspace,
                                             size_t workspace_bytes, void *stream) {
  int rc = check_store("rows8_gather_attention", k8, v8, k_scale, v_scale, code_dtype, BH, cap, D);
  if (!rc) rc = check_query("rows8_gather_attention", q, q_dtype, BH, G, D, cap, lens, n, softcap, out);
  if (rc) return rc;
  if (k < 0 || G * k > 0x7FFFFFFF) return fail(FATHOM_ERR_INVALID, "rows8_gather_attention: G=%lld k=%lld", (long long)G, (long long)k);
  if (k > 0 && !idx) return fail(FATHOM_ERR_INVALID, "rows8_gather_attention: null index pointer");
  AttnArgs a{q, q_dtype, (const uint8_t *)k8, (const uint8_t *)v8, k_scale, v_scale, G, cap, cdiv(cap, kBlk), lens, n, 0,
             idx, k, scale, softcap, slopes, out, (float *)workspace, 1};
  return run<true>("rows8_gather_attention", a, BH, D, code_dtype == FATHOM_DT_I8, k, workspace_bytes, (hipStream_t)stream);
}
