// LayerNorm of rows of any width up to 16384, f32 / bf16 / fp16, forward and backward:
//   mu = mean(x), rstd = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) rstd, y = xh gamma + beta
//   dx = rstd (gamma dy - mean(gamma dy) - xh mean(gamma dy xh)),  dgamma = sum_t dy xh,  dbeta = sum_t dy
// (norm_embed.hip holds the form of the Performer's own residual stream: f32, D <= 256, D % 4 == 0, bf16 out.)
//
// Both directions are bound by HBM: a row is held in registers between its one read and its one write, L lanes per
// row with at most 16 elements each (L = 16, 64: several rows per workgroup, no barrier; L = 256, 512, 1024: one row
// per workgroup, one barrier per row and direction).  Statistics, sums and parameter gradients are f32.
#include "scm_chunk.hpp"

namespace scm {

// Threads of a workgroup and rows it holds at once, for L lanes per row.
constexpr int norm_threads(int L) { return L < 256 ? 256 : L; }

template <typename TX, typename TY, int L, int EPT>
__global__ __launch_bounds__(norm_threads(L)) void norm_fwd_kernel(const TX* __restrict__ x, long ldx,
                                                                   const float* __restrict__ gamma,
                                                                   const float* __restrict__ beta, long T, int D,
                                                                   float eps, TY* __restrict__ y,
                                                                   float* __restrict__ mean, float* __restrict__ rstd) {
  constexpr int E = 16 / sizeof(TX), CPT = EPT / E, RPB = norm_threads(L) / L, NW = L / 64;
  __shared__ f32x2 part[2][NW > 1 ? NW : 1];
  __shared__ float part_n[NW > 1 ? NW : 1];
  const int lane = threadIdx.x % L, grp = threadIdx.x / L;
  int col[CPT], n[CPT];
  float g[CPT][E], b[CPT][E], cnt = 0.f;
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    col[c] = (c * L + lane) * E;
    n[c] = D - col[c];
    cnt += (float)max(0, min(n[c], E));
#pragma unroll
    for (int j = 0; j < E; ++j) {
      g[c][j] = (gamma && j < n[c]) ? gamma[col[c] + j] : 1.f;
      b[c][j] = (beta && j < n[c]) ? beta[col[c] + j] : 0.f;
    }
  }
  float wave_n = 0.f;   // columns of this wave (L > 64)
  if constexpr (L > 64) {
    wave_n = wave_sum(cnt);
    if ((threadIdx.x & 63) == 0) part_n[threadIdx.x >> 6] = wave_n;
    wave_n = fmaxf(wave_n, 1.f);
  }
  const float inv_d = 1.f / (float)D;
  const long stride = (long)gridDim.x * RPB;
  long row = (long)blockIdx.x * RPB + grp;
  Chunk<TX, E> cur[CPT], nxt[CPT];
#pragma unroll
  for (int c = 0; c < CPT; ++c) cur[c] = load_chunk<TX, E>(x + row * ldx + col[c], row < T ? n[c] : 0);
  for (int par = 0; row < T; row += stride, par ^= 1) {
    const bool more = row + stride < T;
#pragma unroll
    for (int c = 0; c < CPT; ++c) nxt[c] = load_chunk<TX, E>(x + (row + stride) * ldx + col[c], more ? n[c] : 0);
    float v[CPT][E], s = 0.f, q = 0.f;
#pragma unroll
    for (int c = 0; c < CPT; ++c)
#pragma unroll
      for (int j = 0; j < E; ++j) { v[c][j] = (float)cur[c].e[j]; s += v[c][j]; }
    // the mean over this row (L <= 64) or over this wave's columns (L > 64), then the squares around it
    const float mu0 = L > 64 ? wave_sum(s) / wave_n : lanes_sum<L>(s) * inv_d;
#pragma unroll
    for (int c = 0; c < CPT; ++c)
#pragma unroll
      for (int j = 0; j < E; ++j) { const float d = j < n[c] ? v[c][j] - mu0 : 0.f; q += d * d; }
    float mu = mu0, m2;
    if constexpr (L > 64) {
      // the waves' (mean, sum of squares) join exactly: m2 = sum_w m2_w + n_w (mu_w - mu)^2
      q = wave_sum(q);
      if ((threadIdx.x & 63) == 0) part[par][threadIdx.x >> 6] = f32x2{mu0, q};
      __syncthreads();   // the other buffer is written next: no wave can be two rows ahead of another
      mu = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) mu += part_n[w] * part[par][w][0];
      mu *= inv_d;
      m2 = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) { const float d = part[par][w][0] - mu; m2 += part[par][w][1] + part_n[w] * d * d; }
    } else {
      m2 = lanes_sum<L>(q);
    }
    const float rs = 1.f / sqrtf(m2 * inv_d + eps);
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      float o[E];
#pragma unroll
      for (int j = 0; j < E; ++j) o[j] = (v[c][j] - mu) * rs * g[c][j] + b[c][j];
      store_chunk<TY, E>(y + row * D + col[c], o, n[c]);
      cur[c] = nxt[c];
    }
    if (mean && lane == 0) { mean[row] = mu; rstd[row] = rs; }
  }
}

// partial (may be null) [gridDim.x][2][D]: this workgroup's sums of dy xh and of dy.  dx may be null.
template <typename TX, typename TY, int L, int EPT>
__global__ __launch_bounds__(norm_threads(L)) void norm_bwd_kernel(const TY* __restrict__ dy, long lddy,
                                                                   const TX* __restrict__ x, long ldx,
                                                                   const float* __restrict__ mean,
                                                                   const float* __restrict__ rstd,
                                                                   const float* __restrict__ gamma, long T, int D,
                                                                   TX* __restrict__ dx, float* __restrict__ partial) {
  constexpr int E = 16 / sizeof(TX), CPT = EPT / E, RPB = norm_threads(L) / L, NW = L / 64;
  __shared__ f32x2 part[2][NW > 1 ? NW : 1];
  __shared__ float red[RPB > 1 ? RPB : 1][2][RPB > 1 ? L * EPT : 1];
  const int lane = threadIdx.x % L, grp = threadIdx.x / L;
  int col[CPT], n[CPT];
  float g[CPT][E], ag[CPT][E], ab[CPT][E];
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    col[c] = (c * L + lane) * E;
    n[c] = D - col[c];
#pragma unroll
    for (int j = 0; j < E; ++j) {
      g[c][j] = (gamma && j < n[c]) ? gamma[col[c] + j] : 1.f;
      ag[c][j] = ab[c][j] = 0.f;
    }
  }
  const float inv_d = 1.f / (float)D;
  const long stride = (long)gridDim.x * RPB;
  long row = (long)blockIdx.x * RPB + grp;
  Chunk<TX, E> cx[CPT], nx[CPT];
  Chunk<TY, E> cy[CPT], ny[CPT];
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    cx[c] = load_chunk<TX, E>(x + row * ldx + col[c], row < T ? n[c] : 0);
    cy[c] = load_chunk<TY, E>(dy + row * lddy + col[c], row < T ? n[c] : 0);
  }
  for (int par = 0; row < T; row += stride, par ^= 1) {
    const bool more = row + stride < T;
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      nx[c] = load_chunk<TX, E>(x + (row + stride) * ldx + col[c], more ? n[c] : 0);
      ny[c] = load_chunk<TY, E>(dy + (row + stride) * lddy + col[c], more ? n[c] : 0);
    }
    const float mu = mean[row], rs = rstd[row];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int c = 0; c < CPT; ++c)
#pragma unroll
      for (int j = 0; j < E; ++j) {   // a column past D has dy = 0 and adds nothing anywhere
        const float d = (float)cy[c].e[j], xh = ((float)cx[c].e[j] - mu) * rs, gd = d * g[c][j];
        s1 += gd;
        s2 += gd * xh;
        ag[c][j] += d * xh;
        ab[c][j] += d;
      }
    if constexpr (L > 64) {
      s1 = wave_sum(s1);
      s2 = wave_sum(s2);
      if ((threadIdx.x & 63) == 0) part[par][threadIdx.x >> 6] = f32x2{s1, s2};
      __syncthreads();
      s1 = s2 = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) { s1 += part[par][w][0]; s2 += part[par][w][1]; }
    } else {
      s1 = lanes_sum<L>(s1);
      s2 = lanes_sum<L>(s2);
    }
    s1 *= inv_d;
    s2 *= inv_d;
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      if (dx) {
        float o[E];
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const float xh = ((float)cx[c].e[j] - mu) * rs;
          o[j] = rs * ((float)cy[c].e[j] * g[c][j] - s1 - xh * s2);
        }
        store_chunk<TX, E>(dx + row * D + col[c], o, n[c]);
      }
      cx[c] = nx[c];
      cy[c] = ny[c];
    }
  }
  if (!partial) return;
  float* out = partial + (long)blockIdx.x * 2 * D;
  if constexpr (RPB > 1) {
#pragma unroll
    for (int c = 0; c < CPT; ++c)
#pragma unroll
      for (int j = 0; j < E; ++j) { red[grp][0][col[c] + j] = ag[c][j]; red[grp][1][col[c] + j] = ab[c][j]; }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += norm_threads(L)) {
      const int k = i >= D, d = i - k * D;
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < RPB; ++r) s += red[r][k][d];
      out[i] = s;
    }
  } else {
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      store_chunk<float, E>(out + col[c], ag[c], n[c]);
      store_chunk<float, E>(out + D + col[c], ab[c], n[c]);
    }
  }
}

// dgamma[i] = sum_b partial[b][i], dbeta[i] = sum_b partial[b][D + i]; 64 columns x 16 slices of the rows per
// workgroup, slices added in order (the result does not depend on which workgroup ends first).
__global__ __launch_bounds__(1024) void norm_reduce_kernel(const float* __restrict__ partial, int nb, int D,
                                                           float* __restrict__ dgamma, float* __restrict__ dbeta) {
  __shared__ float red[16][64];
  const int c = threadIdx.x & 63, sl = threadIdx.x >> 6;
  const int i = blockIdx.x * 64 + c;
  float s = 0.f;
  if (i < 2 * D) {
#pragma unroll 8
    for (int b = sl; b < nb; b += 16) s += partial[(long)b * 2 * D + i];
  }
  red[sl][c] = s;
  __syncthreads();
  if (sl == 0 && i < 2 * D) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) t += red[k][c];
    float* out = i < D ? dgamma : dbeta;
    if (out) out[i < D ? i : i - D] = t;
  }
}

// ---------------------------------------------------------------- host launchers
// Lanes per row and elements per lane: the fewest lanes that hold a row at 16 elements each, and 8 where half the
// registers do (more rows in flight).
struct NormShape { int L, ept; };
static NormShape norm_shape(int D) {
  if (D <= 128) return {16, 8};
  if (D <= 256) return {16, 16};
  if (D <= 512) return {64, 8};
  if (D <= 1024) return {64, 16};
  if (D <= 2048) return {256, 8};
  if (D <= 4096) return {256, 16};
  if (D <= 8192) return {512, 16};
  return {1024, 16};
}
static int norm_rows_per_block(int D) { const int L = norm_shape(D).L; return norm_threads(L) / L; }
// workgroups of the backward pass: every one leaves 2 D partial sums behind, so no more than fill the card
int norm_bwd_blocks(long T, int D) {
  const int rpb = norm_rows_per_block(D);
  const long b = (T + rpb - 1) / rpb;
  return (int)(b < 512 ? b : 512);
}

template <typename TX, typename TY, int L, int EPT>
static void launch_fwd(const NormArgs& a, hipStream_t s) {
  constexpr int RPB = norm_threads(L) / L;
  const long want = (a.T + RPB - 1) / RPB, cap = 256 * (2048 / norm_threads(L));
  hipLaunchKernelGGL((norm_fwd_kernel<TX, TY, L, EPT>), dim3((unsigned)(want < cap ? want : cap)), dim3(norm_threads(L)),
                     0, s, (const TX*)a.x, a.ldx, a.gamma, a.beta, a.T, a.D, a.eps, (TY*)a.y, a.mean, a.rstd);
}
template <typename TX, typename TY, int L, int EPT>
static void launch_bwd(const NormArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((norm_bwd_kernel<TX, TY, L, EPT>), dim3(norm_bwd_blocks(a.T, a.D)), dim3(norm_threads(L)), 0, s,
                     (const TY*)a.dy, a.lddy, (const TX*)a.x, a.ldx, a.mean, a.rstd, a.gamma, a.T, a.D, (TX*)a.dx, a.ws);
}
template <typename TX, typename TY>
static void launch_shape(bool fwd, const NormArgs& a, hipStream_t s) {
  const NormShape k = norm_shape(a.D);
#define SCM_NORM_CASE(L_, E_) \
  if (k.L == L_ && k.ept == E_) { if (fwd) launch_fwd<TX, TY, L_, E_>(a, s); else launch_bwd<TX, TY, L_, E_>(a, s); return; }
  SCM_NORM_CASE(16, 8) SCM_NORM_CASE(16, 16) SCM_NORM_CASE(64, 8) SCM_NORM_CASE(64, 16)
  SCM_NORM_CASE(256, 8) SCM_NORM_CASE(256, 16) SCM_NORM_CASE(512, 16) SCM_NORM_CASE(1024, 16)
#undef SCM_NORM_CASE
}
static void norm_launch(bool fwd, const NormArgs& a, hipStream_t s) {
  if (a.x_type == SCM_F32 && a.y_type == SCM_F32) launch_shape<float, float>(fwd, a, s);
  else if (a.x_type == SCM_F32) launch_shape<float, bf16>(fwd, a, s);
  else if (a.x_type == SCM_BF16) launch_shape<bf16, bf16>(fwd, a, s);
  else launch_shape<f16, f16>(fwd, a, s);
}
bool norm_types_ok(int x_type, int y_type) {
  return (x_type == SCM_F32 && (y_type == SCM_F32 || y_type == SCM_BF16)) ||
         (x_type == SCM_BF16 && y_type == SCM_BF16) || (x_type == SCM_F16 && y_type == SCM_F16);
}
hipError_t norm_fwd(const NormArgs& a, hipStream_t s) {
  Traced tr(K_NORM, 0, s);
  norm_launch(true, a, s);
  return hipGetLastError();
}
hipError_t norm_bwd(const NormArgs& a, float* dgamma, float* dbeta, hipStream_t s) {
  Traced tr(K_NORM, 0, s);
  norm_launch(false, a, s);
  if (a.ws)
    hipLaunchKernelGGL(norm_reduce_kernel, dim3((2 * a.D + 63) / 64), dim3(1024), 0, s, a.ws, norm_bwd_blocks(a.T, a.D),
                       a.D, dgamma, dbeta);
  return hipGetLastError();
}

}  // namespace scm
