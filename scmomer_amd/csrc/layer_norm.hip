// LayerNorm of rows of any width up to 16384, f32 / bf16 / fp16, forward and backward:
//   mu = mean(x), rstd = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) rstd, y = xh gamma + beta
//   dx = rstd (gamma dy - mean(gamma dy) - xh mean(gamma dy xh)),  dgamma = sum_t dy xh,  dbeta = sum_t dy
// (norm_embed.hip holds the form of the Performer's own residual stream: f32, D <= 256, D % 4 == 0, bf16 out.)
//
// Both directions are bound by HBM: a row is held in registers between its one read and its one write, L lanes per
// row with at most 16 elements each (L = 16, 32, 64: several rows per workgroup, no barrier; L = 128 to 1024: one row
// per workgroup, one barrier per row and direction).  Statistics, sums and parameter gradients are f32.  Above 8192
// columns 1024 threads leave a lane 128 registers for its 16 elements and their sums: f32 rows then keep 8 values a lane
// in scratch memory forward (to bf16 only) and 20 backward, and the backward has no row ahead.  2048 x 16384 forward / backward:
// f32 55 / 105 us, floor 50 / 75; f32 to bf16 46 / 96, floor 38 / 63; bf16 28 / 59, floor 25 / 38 (at 8192 columns f32 24 / 48,
// floor 25 / 38).
#include "scm_chunk.hpp"

namespace scm {

// Threads of a workgroup for L lanes per row: L <= 64 several rows at once, else one.
constexpr int norm_threads(int L) { return L <= 64 ? 256 : L; }

// Which columns a lane holds: CPT chunks of E, lane-interleaved over the L lanes of a group.  Chunk c is loaded from column
// at[c]; its elements from first[c] on are the lane's (the last chunk of a row that is no multiple of E begins E columns
// before the end, first[c] of them again; E: none are).  So every lane loads and stores whole chunks on one path, without
// a branch between a load and its use: branches there make the compiler wait for the loads ahead as well (8192 x 4096 bf16
// that way: forward 31 us instead of 29, backward 55 instead of 47).  WHOLE = D >= E; narrower rows go element by element.
template <int E, int L, int CPT, bool WHOLE>
struct Columns {
  int at[CPT], first[CPT];
  bool ragged;   // some lane of the wave has first != 0
  SCM_DEV Columns(int lane, int D) {
    bool r = false;
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      const int col = (c * L + lane) * E;
      at[c] = col + E <= D ? col : col < D ? D - E : 0;
      first[c] = col < D ? col - at[c] : E;
      r |= first[c] != 0;
    }
    ragged = __builtin_amdgcn_ballot_w64(r) != 0;
  }
  template <typename T>
  SCM_DEV Chunk<T, E> load(const T* row, int c) const {
    Chunk<T, E> v;
    if constexpr (WHOLE) {
      __builtin_memcpy(&v, row + at[c], sizeof(v));
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) v.e[j] = j >= first[c] ? row[at[c] + j] : (T)0.f;
    }
    return v;
  }
  // the repeated elements of a last chunk get the value that their own lane stores
  template <bool STREAM, typename T>
  SCM_DEV void store(T* row, int c, const float (&v)[E]) const {
    if (first[c] == E) return;
    if constexpr (WHOLE) store_chunk<T, E, STREAM>(row + at[c], v, E);
    else store_own(row, c, v);
  }
  template <typename T>
  SCM_DEV void store_own(T* row, int c, const float (&v)[E]) const {
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (j >= first[c]) row[at[c] + j] = (T)v[j];
  }
};

// A group's next row is on its way while one is worked on (past the last row: the last row again).
template <typename TX, typename TY, int L, int EPT, bool STREAM, bool WHOLE>
__global__ __launch_bounds__(norm_threads(L)) void norm_fwd_kernel(const TX* __restrict__ x, long ldx,
                                                                   const float* __restrict__ gamma,
                                                                   const float* __restrict__ beta, long T, int D,
                                                                   float eps, TY* __restrict__ y,
                                                                   float* __restrict__ mean, float* __restrict__ rstd) {
  constexpr int E = 16 / sizeof(TX), CPT = EPT / E, RPB = norm_threads(L) / L, NW = L / 64;
  // gamma, beta in registers; longer slices of 2-byte types read them (from the caches) row by row
  constexpr bool HOLD = EPT <= 8 || sizeof(TX) == 4;
  __shared__ f32x2 part[2][NW > 1 ? NW : 1];
  __shared__ float part_n[NW > 1 ? NW : 1];
  const int lane = threadIdx.x % L, grp = threadIdx.x / L;
  const long stride = (long)gridDim.x * RPB;
  long row = (long)blockIdx.x * RPB + grp;
  const Columns<E, L, CPT, WHOLE> cols(lane, D);
  Chunk<TX, E> cur[CPT], nxt[CPT];
#pragma unroll
  for (int c = 0; c < CPT; ++c) cur[c] = cols.load(x + min(row, T - 1) * ldx, c);
  Chunk<float, E> g[CPT], b[CPT];
  auto affine = [&](int c) {
    if (gamma) g[c] = cols.load(gamma, c);
    if (beta) b[c] = cols.load(beta, c);
  };
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
#pragma unroll
    for (int j = 0; j < E; ++j) { g[c].e[j] = 1.f; b[c].e[j] = 0.f; }
    if constexpr (HOLD) affine(c);
  }
  float wave_n = 1.f;   // columns of this wave (L > 64)
  if constexpr (L > 64) {
    float cnt = 0.f;
#pragma unroll
    for (int c = 0; c < CPT; ++c) cnt += (float)(E - cols.first[c]);
    wave_n = wave_sum(cnt);
    if ((threadIdx.x & 63) == 0) part_n[threadIdx.x >> 6] = wave_n;
    wave_n = fmaxf(wave_n, 1.f);
  }
  const float inv_d = 1.f / (float)D;
  for (int par = 0; row < T; row += stride, par ^= 1) {
#pragma unroll
    for (int c = 0; c < CPT; ++c) nxt[c] = cols.load(x + min(row + stride, T - 1) * ldx, c);
    float s = 0.f, q = 0.f;
    if (!cols.ragged) {
#pragma unroll
      for (int c = 0; c < CPT; ++c)
#pragma unroll
        for (int j = 0; j < E; ++j) s += (float)cur[c].e[j];
    } else {
#pragma unroll
      for (int c = 0; c < CPT; ++c)
#pragma unroll
        for (int j = 0; j < E; ++j) s += j >= cols.first[c] ? (float)cur[c].e[j] : 0.f;
    }
    // the mean over this row (L <= 64) or over this wave's columns (L > 64), then the squares around it
    const float mu0 = L > 64 ? wave_sum(s) / wave_n : lanes_sum<L>(s) * inv_d;
    if (!cols.ragged) {
#pragma unroll
      for (int c = 0; c < CPT; ++c)
#pragma unroll
        for (int j = 0; j < E; ++j) { const float d = (float)cur[c].e[j] - mu0; q += d * d; }
    } else {
#pragma unroll
      for (int c = 0; c < CPT; ++c)
#pragma unroll
        for (int j = 0; j < E; ++j) { const float d = j >= cols.first[c] ? (float)cur[c].e[j] - mu0 : 0.f; q += d * d; }
    }
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
      if constexpr (!HOLD) affine(c);
      float o[E];
#pragma unroll
      for (int j = 0; j < E; ++j) o[j] = ((float)cur[c].e[j] - mu) * rs * g[c].e[j] + b[c].e[j];
      cols.template store<STREAM>(y + row * D, c, o);
      cur[c] = nxt[c];
    }
    if (mean && lane == 0) { mean[row] = mu; rstd[row] = rs; }
  }
}

// partial (may be null) [gridDim.x][2][D]: this workgroup's sums of dy xh and of dy.  dx may be null.  AHEAD: rows of a
// group that are on their way while one is worked on.
template <typename TX, typename TY, int L, int EPT, int AHEAD, bool STREAM, bool WHOLE>
__global__ __launch_bounds__(norm_threads(L)) void norm_bwd_kernel(const TY* __restrict__ dy, long lddy,
                                                                   const TX* __restrict__ x, long ldx,
                                                                   const float* __restrict__ mean,
                                                                   const float* __restrict__ rstd,
                                                                   const float* __restrict__ gamma, long T, int D,
                                                                   TX* __restrict__ dx, float* __restrict__ partial) {
  constexpr int E = 16 / sizeof(TX), CPT = EPT / E, RPB = norm_threads(L) / L, NW = L / 64;
  constexpr bool HOLD = EPT <= 8;
  __shared__ f32x2 part[2][NW > 1 ? NW : 1];
  __shared__ float red[RPB > 1 ? RPB : 1][2][RPB > 1 ? L * EPT : 1];
  const int lane = threadIdx.x % L, grp = threadIdx.x / L;
  const long stride = (long)gridDim.x * RPB;
  long row = (long)blockIdx.x * RPB + grp;
  const Columns<E, L, CPT, WHOLE> cols(lane, D);
  struct Rows { Chunk<TX, E> x[CPT]; Chunk<TY, E> y[CPT]; float mu, rs; } buf[AHEAD + 1];
  auto fetch = [&](Rows& r, long at) {
    at = min(at, T - 1);
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      r.x[c] = cols.load(x + at * ldx, c);
      r.y[c] = cols.load(dy + at * lddy, c);
    }
    r.mu = mean[at];
    r.rs = rstd[at];
  };
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) fetch(buf[k], row + k * stride);
  Chunk<float, E> g[CPT];
  float ag[CPT][E], ab[CPT][E];
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
#pragma unroll
    for (int j = 0; j < E; ++j) { g[c].e[j] = 1.f; ag[c][j] = ab[c][j] = 0.f; }
    if (HOLD && gamma) g[c] = cols.load(gamma, c);
  }
  const float inv_d = 1.f / (float)D;
  for (int par = 0; row < T; row += stride, par ^= 1) {
    fetch(buf[AHEAD], row + AHEAD * stride);
    const float mu = buf[0].mu, rs = buf[0].rs;
    float s1 = 0.f, s2 = 0.f;
    auto add = [&](int c, int j, float d) {
      const float xh = ((float)buf[0].x[c].e[j] - mu) * rs, gd = d * g[c].e[j];
      s1 += gd;
      s2 += gd * xh;
      ag[c][j] += d * xh;
      ab[c][j] += d;
    };
    if (!HOLD && gamma) {
#pragma unroll
      for (int c = 0; c < CPT; ++c) g[c] = cols.load(gamma, c);
    }
    if (!cols.ragged) {
#pragma unroll
      for (int c = 0; c < CPT; ++c)
#pragma unroll
        for (int j = 0; j < E; ++j) add(c, j, (float)buf[0].y[c].e[j]);
    } else {
#pragma unroll
      for (int c = 0; c < CPT; ++c)
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (j >= cols.first[c]) add(c, j, (float)buf[0].y[c].e[j]);
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
    if (dx) {
#pragma unroll
      for (int c = 0; c < CPT; ++c) {
        float o[E];
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const float xh = ((float)buf[0].x[c].e[j] - mu) * rs;
          float gd;
          {
#pragma clang fp contract(off)   // the product rounded as it was summed: one column's gradient is 0, not its rounding
            gd = (float)buf[0].y[c].e[j] * g[c].e[j];
            gd = gd - s1;
          }
          o[j] = rs * (gd - xh * s2);
        }
        cols.template store<STREAM>(dx + row * D, c, o);
      }
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) buf[k] = buf[k + 1];
  }
  if (!partial) return;
  float* out = partial + (long)blockIdx.x * 2 * D;
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    if constexpr (RPB > 1) {
      cols.store_own(&red[grp][0][0], c, ag[c]);
      cols.store_own(&red[grp][1][0], c, ab[c]);
    } else if (cols.first[c] == 0) {
      store_chunk<float, E>(out + cols.at[c], ag[c], E);
      store_chunk<float, E>(out + D + cols.at[c], ab[c], E);
    } else {
      cols.store_own(out, c, ag[c]);
      cols.store_own(out + D, c, ab[c]);
    }
  }
  if constexpr (RPB > 1) {
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += norm_threads(L)) {
      const int k = i >= D, d = i - k * D;
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < RPB; ++r) s += red[r][k][d];
      out[i] = s;
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
// Lanes per row and elements per lane: 8 elements each as long as 1024 threads hold the row.  (16 elements on half the
// lanes: 8192 x 4096 bf16 backward 54 us, against 40: the registers of a longer slice cost waves; forward 26 either way.)
struct NormShape { int L, ept; };
static NormShape norm_shape(int D) {
  if (D <= 128) return {16, 8};
  if (D <= 256) return {32, 8};
  if (D <= 512) return {64, 8};
  if (D <= 1024) return {128, 8};
  if (D <= 2048) return {256, 8};
  if (D <= 4096) return {512, 8};
  if (D <= 8192) return {1024, 8};
  return {1024, 16};
}
// Workgroups: 1024 threads per CU in either direction, each group going on from row to row with its loads ahead.  8192 x 4096
// bf16 forward: 512 threads per CU 34 us, 1024: 26, 2048: 25; backward (partial sums per workgroup): 38, 36 and 42; f32
// 84530 x 200 backward 36.6, 34.5 and 38.
static long norm_blocks(long T, int D) {
  const int nt = norm_threads(norm_shape(D).L), rpb = nt / norm_shape(D).L;
  const long b = (T + rpb - 1) / rpb, cap = 256L * (1024 / nt);
  return b < cap ? b : cap;
}
int norm_bwd_blocks(long T, int D) { return (int)norm_blocks(T, D); }

template <typename TX, typename TY, int L, int EPT, bool STREAM, bool WHOLE = true>
static void launch_shape(bool fwd, const NormArgs& a, hipStream_t s) {
  constexpr int AHEAD_B = EPT <= 8 ? 1 : 0;   // 16 elements: two sums per column and one row are all the registers there are
  const dim3 g((unsigned)norm_blocks(a.T, a.D)), b(norm_threads(L));
  if (fwd)
    hipLaunchKernelGGL((norm_fwd_kernel<TX, TY, L, EPT, STREAM, WHOLE>), g, b, 0, s, (const TX*)a.x, a.ldx, a.gamma, a.beta,
                       a.T, a.D, a.eps, (TY*)a.y, a.mean, a.rstd);
  else
    hipLaunchKernelGGL((norm_bwd_kernel<TX, TY, L, EPT, AHEAD_B, STREAM, WHOLE>), g, b, 0, s, (const TY*)a.dy, a.lddy,
                       (const TX*)a.x, a.ldx, a.mean, a.rstd, a.gamma, a.T, a.D, (TX*)a.dx, a.ws);
}
template <typename TX, typename TY, bool STREAM>
static void launch_typed(bool fwd, const NormArgs& a, hipStream_t s) {
  switch (norm_shape(a.D).L) {
    case 16:
      if (a.D < 16 / (int)sizeof(TX)) return launch_shape<TX, TY, 16, 8, STREAM, false>(fwd, a, s);
      return launch_shape<TX, TY, 16, 8, STREAM>(fwd, a, s);
    case 32: return launch_shape<TX, TY, 32, 8, STREAM>(fwd, a, s);
    case 64: return launch_shape<TX, TY, 64, 8, STREAM>(fwd, a, s);
    case 128: return launch_shape<TX, TY, 128, 8, STREAM>(fwd, a, s);
    case 256: return launch_shape<TX, TY, 256, 8, STREAM>(fwd, a, s);
    case 512: return launch_shape<TX, TY, 512, 8, STREAM>(fwd, a, s);
    default:
      if (norm_shape(a.D).ept == 8) return launch_shape<TX, TY, 1024, 8, STREAM>(fwd, a, s);
      return launch_shape<TX, TY, 1024, 16, STREAM>(fwd, a, s);
  }
}
template <typename TX, typename TY>
static void launch_sized(bool fwd, const NormArgs& a, hipStream_t s) {
  if (a.T * a.D * (long)(fwd ? sizeof(TY) : sizeof(TX)) > STREAM_BYTES) launch_typed<TX, TY, true>(fwd, a, s);
  else launch_typed<TX, TY, false>(fwd, a, s);
}
static void norm_launch(bool fwd, const NormArgs& a, hipStream_t s) {
  if (a.x_type == SCM_F32 && a.y_type == SCM_F32) launch_sized<float, float>(fwd, a, s);
  else if (a.x_type == SCM_F32) launch_sized<float, bf16>(fwd, a, s);
  else if (a.x_type == SCM_BF16) launch_sized<bf16, bf16>(fwd, a, s);
  else launch_sized<f16, f16>(fwd, a, s);
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
