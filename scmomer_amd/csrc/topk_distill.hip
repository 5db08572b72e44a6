// Distillation from a teacher's k named log probabilities.  Per row, with z = x / temperature the student's logits,
// entries (i_j, l_j), q_j = exp l_j, R the vocabulary without the named tokens:
//   tail bucket:   r = max(0, 1 - sum q_j);     renormalised:  q_j /= sum q_j, r = 0
//   L    = sum_j q_j (l_j - z_{i_j} + lse) + r (ln r - lse_R + lse)          lse over all tokens, lse_R over R
//   dz_i = A p_i - [i named] sum_{i_j = i} q_j - [i in R] r exp(z_i - lse_R),   A = sum q_j + r
// The named tokens are left out of the running sum (a bit per token in LDS tells them apart) and join it afterwards, so
// lse_R is exact where the student is nearly sure of them: no difference of nearly equal sums is formed.  For i in R
// the gradient is one exponential times a factor of the row, cr = A p(R) / s_R - r / s_R:  dz_i = cr 2^((x_i - m_R) c).
// Conventions: i_j < 0 is an unused entry; an index named twice counts once in R's complement and with both its q; where
// the student has nothing in R (-inf throughout) r is left out; a row of -inf only and a row of weight 0 have loss and
// gradient 0; i_j >= V and NaN give NaN.
//
// Bound by HBM: the loss reads the logits once, the gradient reads them once more and writes once; the two in one pass
// (one workgroup per row) read a row the second time while it is still in the caches.
#include "scm_softmax.hpp"

#include <algorithm>

namespace scm {

constexpr int DISTILL_SEGMENT = 131072;   // tokens whose bits fit a workgroup's 16 KB

// ---------------------------------------------------------------- one row's end: lane j of a wave holds entry j
struct DistillRow {
  float loss, m, cr;   // the loss; reference maximum and factor of the gradient in R
  float g;             // lane j: gradient at its named token
};
template <int CTRL>
SCM_DEV double dpp_move_f64(double v) {
  return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xF, 0xF, true),
                          __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xF, 0xF, true));
}
SCM_DEV double wave_sum_f64(double v) {
  v += dpp_move_f64<0xB1>(v);
  v += dpp_move_f64<0x4E>(v);
  v += dpp_move_f64<0x141>(v);
  v += dpp_move_f64<0x140>(v);
  v += __shfl_xor(v, 16);
  v += __shfl_xor(v, 32);
  return v;
}
// Entries of less mass than this together are renormalised relative to the largest of them: their sum and its logarithm
// would leave the range of f32, and from exp(-745) on of f64.
constexpr double HARDLY_ANY_MASS = 0x1p-60;
// rest: statistics over R.  idx (-1: unused), lp, x (the student's logit there) of this lane's entry.  beyond: some index
// lies outside the vocabulary (such entries come as unused).  twice: some token may be named more than once.
SCM_DEV DistillRow distill_row(const DistillTopkArgs& a, const Stat& rest, int idx, float lp, float x, bool beyond, bool twice) {
  const int lane = threadIdx.x & 63;
  const bool used = idx >= 0;
  double q = used ? exp((double)lp) : 0.0;
  double total = wave_sum_f64(q);
  if (!a.tail && total < HARDLY_ANY_MASS) {   // the same in all lanes
    const float top = wave_max(used ? lp : -INFINITY);
    if (top > -INFINITY) {
      lp -= top;
      q = used ? exp((double)lp) : 0.0;
      total = wave_sum_f64(q);
    }
  }
  float r = 0.f, big_a;
  if (a.tail) {
    r = rest.s == 0.f ? 0.f : (float)fmax(0.0, 1.0 - total);
    big_a = (float)total + r;
  } else {
    big_a = total > 0.0 ? 1.f : 0.f;
    if (total > 0.0) { q *= 1.0 / total; lp -= logf((float)total); }
  }
  const float qf = (float)q;
  // the first of equal indices, and the sum of q over them
  float qsum = qf;
  bool first = used;
  if (twice) {
    qsum = 0.f;
    for (int j = 0; j < a.k; ++j) {
      const int ij = __builtin_amdgcn_readlane(idx, j);
      const float qj = __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(qf), j));
      if (used && ij == idx) {
        qsum += qj;
        if (j < lane) first = false;
      }
    }
  }
  // all tokens: R and the named ones
  const float m = wave_max(fmaxf(rest.m, used ? x : LOWEST));
  const float f = exp2_fast(fmaxf((rest.m - m) * a.c, -200.f));
  const float e = used ? exp2_fast((x - m) * a.c) : 0.f;
  const float z = rest.s * f + wave_sum(first ? e : 0.f);
  const float l2 = log2_fast(z);
  const float logp = (x - m) * a.inv_t - LN2 * l2;
  float loss = wave_sum(used && qf > 0.f ? qf * (lp - logp) : 0.f);
  if (r > 0.f) loss += r * (logf(r) - ((rest.m - m) * a.inv_t + LN2 * (log2_fast(rest.s) - l2)));
  DistillRow o;
  o.loss = loss;
  o.m = rest.m;
  o.cr = rest.s == 0.f ? 0.f : big_a * f / z - r / rest.s;
  o.g = big_a * e / z - qsum;
  if (z == 0.f) { o.loss = 0.f; o.cr = 0.f; o.g = 0.f; }   // nothing above -inf
  if (beyond || total != total || rest.s != rest.s || z != z) o.loss = o.cr = o.g = __uint_as_float(0x7FC00000u);
  return o;
}
// Entry j of a row, in lane j of a wave: index (-1 where it is not used or lies outside), log probability, logit.
struct Entry { int idx; float lp, x; bool beyond; };
template <typename T>
SCM_DEV Entry load_entry(const DistillTopkArgs& a, long row, const T* x) {
  const int j = threadIdx.x & 63;
  Entry e{-1, 0.f, 0.f, false};
  if (j < a.k) {
    const long long i = a.index[row * a.k + j];
    e.lp = a.lp[row * a.k + j];
    e.beyond = i >= a.V;
    if (i >= 0 && i < a.V) { e.idx = (int)i; e.x = (float)x[i]; }
  }
  return e;
}
SCM_DEV bool any_lane(bool b) { return __builtin_amdgcn_ballot_w64(b) != 0; }
// what the gradient of a row of weight w is scaled by; sum_weights only where whole waves call
SCM_DEV float row_scale(const DistillTopkArgs& a, long row, float w) {
  const float g = a.gloss ? a.gloss[a.gloss_rows ? row : 0] : a.scale;
  float div = 1.f;
  if (a.mean) {
    if (a.sum_weights) {
      double s = 0.0;
#pragma unroll 4
      for (long i = threadIdx.x & 63; i < a.rows; i += 64) s += (double)a.weights[i];
      div = (float)wave_sum_f64(s);
    } else {
      div = a.wsum ? a.wsum[0] : (float)a.rows;
    }
  }
  return g * w * a.inv_t / div;
}

// ---------------------------------------------------------------- statistics over R of a segment
// A bit per token of a segment of at most 32 WORDS tokens.
template <int WORDS>
struct NamedBits { uint32_t w[WORDS]; };
// Marks the entries (lane j of the first wave: entry j) that lie in [lo, lo + len).  -> in the first wave: some token is
// named twice.  Begins after and ends with a barrier.
template <int NT, int WORDS>
SCM_DEV bool mark_named(NamedBits<WORDS>& bits, const Entry& e, int lo, int len) {
  for (int i = threadIdx.x; i < (len + 31) / 32; i += NT) bits.w[i] = 0;
  __syncthreads();
  bool again = false;
  if (threadIdx.x < 64) {
    const int i = e.idx - lo;
    if (e.idx >= 0 && i >= 0 && i < len) again = (atomicOr(&bits.w[i >> 5], 1u << (i & 31)) >> (i & 31)) & 1;
    again = any_lane(again);
  }
  __syncthreads();
  return again;
}
template <typename W, int WORDS>
SCM_DEV Stat rest_of_segment(const W& w, const NamedBits<WORDS>& bits, float c) {
  Stat st = stat_none();
  w.run([&](int s, const typename W::Raw& raw) {
    float v[W::EL], bm = LOWEST;
    w.values(s, raw, v);
#pragma unroll
    for (int u = 0; u < W::U; ++u) {
      const int i0 = w.first(s, u);
      const uint32_t word = i0 < w.len ? bits.w[i0 >> 5] >> (i0 & 31) : 0u;   // this chunk's bits, lowest first
      const uint32_t named = word & ((1u << W::E) - 1u);
      if (named) {   // at most k chunks of a row
#pragma unroll
        for (int j = 0; j < W::E; ++j)
          if ((named >> j) & 1) v[u * W::E + j] = -INFINITY;
      }
    }
#pragma unroll
    for (int j = 0; j < W::EL; ++j) bm = fmaxf(bm, v[j]);
    stat_add<false>(st, v, bm, c);
  });
  return st;
}

// Gradient of a segment from (m, cr), then the named tokens over it.
template <typename T, bool STREAM, typename W>
SCM_DEV void distill_write(const W& w, T* dx, int lo, float m, float cr, float c) {
  w.run([&](int s, const typename W::Raw& raw) {
#pragma unroll
    for (int u = 0; u < W::U; ++u) {
      float o[W::E];
#pragma unroll
      for (int j = 0; j < W::E; ++j) o[j] = cr * exp2_fast(((float)raw[u].e[j] - m) * c);
      store_chunk<T, W::E, STREAM>(dx + lo + w.first(s, u), o, w.len - w.first(s, u));
    }
  });
}
template <typename T, int NT>
SCM_DEV void zero_write(T* dx, int len) {
  constexpr int E = 16 / sizeof(T);
  const float none[E] = {};
  for (int i = threadIdx.x * E; i < len; i += NT * E) store_chunk<T, E>(dx + i, none, len - i);
}

// ---------------------------------------------------------------- one to four waves per row, or per segment of one
SCM_DEV void write_tape(const DistillTopkArgs& a, long row, float m, float cr, float g) {   // by a wave
  if (!a.tape) return;
  const int j = threadIdx.x & 63;
  if (j == 0) { a.tape[2 * row] = m; a.tape[2 * row + 1] = cr; }
  if (j < a.k) a.g_top[row * a.k + j] = g;
}

// GRAD: loss and gradient in one launch (S = 1).  Otherwise the loss, and (tape, g_top given) what the backward reads;
// with S > 1 the segment's statistics go to part for distill_join_kernel.
template <typename T, int NT, int EL, int WORDS, bool GRAD, bool STREAM = false>
__global__ __launch_bounds__(NT) void distill_kernel(DistillTopkArgs a, int S, int seg_len) {
  __shared__ Stat red[NT / 64];
  __shared__ NamedBits<WORDS> bits;
  __shared__ float row_m, row_cr;
  const long row = blockIdx.x / S;
  const int seg = blockIdx.x % S, lo = seg * seg_len, tid = threadIdx.x;
  const T* x = (const T*)a.x + row * a.ldx;
  const Walk<T, NT, EL> w{x + lo, min(a.V - lo, seg_len)};
  T* dx = GRAD ? (T*)a.dx + row * a.V : nullptr;
  const float wt = a.weight ? a.weight[row] : 1.f;
  if (wt == 0.f) {
    if constexpr (GRAD) zero_write<T, NT>(dx, a.V);
    if (S == 1 && tid < 64) {
      if (tid == 0) a.row_loss[row] = 0.f;
      write_tape(a, row, 0.f, 0.f, 0.f);
    }
    return;
  }
  Entry en{-1, 0.f, 0.f, false};
  if (tid < 64) en = load_entry(a, row, x);
  const float sc = GRAD ? row_scale(a, row, wt) : 0.f;
  const bool twice = mark_named<NT>(bits, en, lo, w.len);
  const Stat st = stat_block<false, NT>(rest_of_segment(w, bits, a.c), a.c, red);
  if (S > 1) {
    if (tid == 0) { a.part[2 * (row * S + seg)] = st.m; a.part[2 * (row * S + seg) + 1] = st.s; }
    return;
  }
  float g = 0.f;
  if (tid < 64) {
    const DistillRow r = distill_row(a, st, en.idx, en.lp, en.x, any_lane(en.beyond), twice);
    g = r.g;
    if (tid == 0) { a.row_loss[row] = wt * r.loss; row_m = r.m; row_cr = r.cr; }
    write_tape(a, row, r.m, r.cr, g);
  }
  if constexpr (GRAD) {
    __syncthreads();
    distill_write<T, STREAM>(Walk<T, NT>{x, a.V}, dx, 0, row_m, row_cr * sc, a.c);
    __syncthreads();   // the last store to a named token is this one; equal indices hold equal values
    if (en.idx >= 0) dx[en.idx] = (T)(g * sc);
  }
}

// Loss and gradient of a row that stays in registers between its one read and its one write: STEPS x EL elements a thread
// (at most 64 registers).
template <typename T, int NT, int STEPS, bool STREAM, int EL = 32>
__global__ __launch_bounds__(NT) void distill_resident_kernel(DistillTopkArgs a) {
  __shared__ Stat red[NT / 64];
  __shared__ NamedBits<STEPS * NT * EL / 32> bits;
  __shared__ float row_m, row_cr;
  typedef Walk<T, NT, EL> W;
  constexpr int E = W::E, U = W::U;
  const long row = blockIdx.x;
  const int tid = threadIdx.x;
  T* dx = (T*)a.dx + row * a.V;
  const float wt = a.weight ? a.weight[row] : 1.f;
  if (wt == 0.f) {
    zero_write<T, NT>(dx, a.V);
    if (tid == 0) a.row_loss[row] = 0.f;
    return;
  }
  const W w{(const T*)a.x + row * a.ldx, a.V};
  typename W::Raw raw[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) w.load(s, raw[s]);
  Entry en{-1, 0.f, 0.f, false};
  if (tid < 64) en = load_entry(a, row, w.p);
  const float sc = row_scale(a, row, wt);
  const bool twice = mark_named<NT>(bits, en, 0, STEPS * NT * EL);
  // the maximum over R first, then one exponential per element around it; named tokens and what lies past the end
  // become -inf in the registers
  Stat st = stat_none();
#pragma unroll
  for (int s = 0; s < STEPS; ++s)
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i0 = w.first(s, u), n = a.V - i0;
      const uint32_t named = (bits.w[i0 >> 5] >> (i0 & 31)) & ((1u << E) - 1u);
      if (named || n < E) {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (((named >> j) & 1) || j >= n) raw[s][u].e[j] = (T)-INFINITY;
      }
#pragma unroll
      for (int j = 0; j < E; ++j) st.m = fmaxf(st.m, (float)raw[s][u].e[j]);
      stay_packed(raw[s][u]);
    }
#pragma unroll
  for (int s = 0; s < STEPS; ++s)
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int j = 0; j < E; ++j) st.s += exp2_fast(((float)raw[s][u].e[j] - st.m) * a.c);
      stay_packed(raw[s][u]);
    }
  st = stat_block<false, NT>(st, a.c, red);
  float g = 0.f;
  if (tid < 64) {
    const DistillRow r = distill_row(a, st, en.idx, en.lp, en.x, any_lane(en.beyond), twice);
    g = r.g;
    if (tid == 0) { a.row_loss[row] = wt * r.loss; row_m = r.m; row_cr = r.cr; }
  }
  __syncthreads();
  const float m = row_m, cr = row_cr * sc;
#pragma unroll
  for (int s = 0; s < STEPS; ++s)
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float o[E];
#pragma unroll
      for (int j = 0; j < E; ++j) o[j] = cr * exp2_fast(((float)raw[s][u].e[j] - m) * a.c);
      store_chunk<T, E, STREAM>(dx + w.first(s, u), o, a.V - w.first(s, u));
    }
  __syncthreads();   // the last store to a named token is this one; equal indices hold equal values
  if (en.idx >= 0) dx[en.idx] = (T)(g * sc);
}

template <typename T>
__global__ __launch_bounds__(64) void distill_join_kernel(DistillTopkArgs a, int S) {
  const long row = blockIdx.x;
  const int tid = threadIdx.x;
  const float wt = a.weight ? a.weight[row] : 1.f;
  if (wt == 0.f) {
    if (tid == 0) a.row_loss[row] = 0.f;
    write_tape(a, row, 0.f, 0.f, 0.f);
    return;
  }
  const Entry en = load_entry(a, row, (const T*)a.x + row * a.ldx);
  Stat st = stat_none();
  for (int i = tid; i < S; i += 64)
    st = stat_join<false>(st, Stat{a.part[2 * (row * S + i)], a.part[2 * (row * S + i) + 1], 0.f}, a.c);
  st = stat_wave<false>(st, a.c);
  const DistillRow r = distill_row(a, st, en.idx, en.lp, en.x, any_lane(en.beyond), true);
  if (tid == 0) a.row_loss[row] = wt * r.loss;
  write_tape(a, row, r.m, r.cr, r.g);
}

template <typename T, int NT, int EL, bool STREAM>
__global__ __launch_bounds__(NT) void distill_bwd_kernel(DistillTopkArgs a, int S, int seg_len) {
  const long row = blockIdx.x / S;
  const int lo = (int)(blockIdx.x % S) * seg_len, tid = threadIdx.x;
  const Walk<T, NT, EL> w{(const T*)a.x + row * a.ldx + lo, min(a.V - lo, seg_len)};
  T* dx = (T*)a.dx + row * a.V;
  const float wt = a.weight ? a.weight[row] : 1.f;
  if (wt == 0.f) { zero_write<T, NT>(dx + lo, w.len); return; }
  const float sc = row_scale(a, row, wt);
  distill_write<T, STREAM>(w, dx, lo, a.tape[2 * row], a.tape[2 * row + 1] * sc, a.c);
  __syncthreads();
  if (tid < a.k) {
    const long long i = a.index[row * a.k + tid];
    if (i >= lo && i < lo + w.len) dx[i] = (T)(a.g_top[row * a.k + tid] * sc);
  }
}

// ---------------------------------------------------------------- short rows: a thread per row, a bit per token
// f(j, index, log probability) for a row's entries, eight of them on their way at once.
template <typename F>
SCM_DEV void each_entry(const int64_t* index, const float* lp, int k, F f) {
  constexpr int B = 8;
  for (int j = 0; j < k; j += B) {
    long long i[B];
    float l[B];
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const int jj = min(j + b, k - 1);
      i[b] = index[jj];
      l[b] = lp[jj];
    }
#pragma unroll
    for (int b = 0; b < B; ++b)
      if (j + b < k && i[b] >= 0) f(j + b, i[b], l[b]);
  }
}
// LDS: the logits of 64 rows, then q of their entries in f64.
template <typename T, bool GRAD>
__global__ __launch_bounds__(64) void distill_small_kernel(DistillTopkArgs a) {
  extern __shared__ uint32_t lds[];
  const int V = a.V, pitch = V | 1, rows = (int)min((long)64, a.T - (long)blockIdx.x * 64);
  double* q_of = (double*)(lds + 64 * pitch) + threadIdx.x;   // entry j: q_of[64 j]
  const long row = (long)blockIdx.x * 64 + threadIdx.x;
  stage_rows<const T, false>((const T*)a.x + (long)blockIdx.x * 64 * a.ldx, a.ldx, rows, V, lds, pitch);
  __syncthreads();
  if ((int)threadIdx.x < rows) {
    uint32_t* o = lds + threadIdx.x * pitch;
    auto x = [&](int i) { return __uint_as_float(o[i]); };
    const float wt = a.weight ? a.weight[row] : 1.f;
    float loss = 0.f;
    if (wt != 0.f) {
      const int64_t* index = a.index + row * a.k;
      const float* lps = a.lp + row * a.k;
      unsigned long long named = 0;
      bool beyond = false;
      double total = 0.0;
      each_entry(index, lps, a.k, [&](int j, long long i, float lp) {
        if (i >= V) { beyond = true; return; }
        named |= 1ull << i;
        const double q = exp((double)lp);
        q_of[64 * j] = q;
        total += q;
      });
      float top = 0.f;   // what the log probabilities are relative to
      if (!a.tail && total < HARDLY_ANY_MASS) {
        float most = -INFINITY;
        each_entry(index, lps, a.k, [&](int, long long i, float lp) { if (i < V) most = fmaxf(most, lp); });
        if (most > -INFINITY) {
          top = most;
          total = 0.0;
          each_entry(index, lps, a.k, [&](int j, long long i, float lp) {
            if (i >= V) return;
            const double q = exp((double)(lp - top));
            q_of[64 * j] = q;
            total += q;
          });
        }
      }
      Stat all = stat_none(), rest = stat_none();
#pragma unroll 8
      for (int i = 0; i < V; ++i) {
        all.m = fmaxf(all.m, x(i));
        if (!((named >> i) & 1)) rest.m = fmaxf(rest.m, x(i));
      }
#pragma unroll 8
      for (int i = 0; i < V; ++i) {
        all.s += exp2_fast((x(i) - all.m) * a.c);
        if (!((named >> i) & 1)) rest.s += exp2_fast((x(i) - rest.m) * a.c);
      }
      const float l2 = log2_fast(all.s);
      float r = 0.f, log_total = 0.f;
      double per = 1.0;
      if (a.tail) r = rest.s == 0.f ? 0.f : (float)fmax(0.0, 1.0 - total);
      else if (total > 0.0) { per = 1.0 / total; log_total = logf((float)total); }
      const float big_a = (float)(total * per) + r;
      each_entry(index, lps, a.k, [&](int j, long long i, float lp) {
        if (i >= V) return;
        const float q = (float)(q_of[64 * j] * per);
        if (q > 0.f) loss += q * (lp - top - log_total - ((x((int)i) - all.m) * a.inv_t - LN2 * l2));
      });
      if (r > 0.f) loss += r * (logf(r) - ((rest.m - all.m) * a.inv_t + LN2 * (log2_fast(rest.s) - l2)));
      const bool empty = all.s == 0.f, broken = beyond || total != total || all.s != all.s;
      if (empty) loss = 0.f;
      if (broken) loss = __uint_as_float(0x7FC00000u);
      loss *= wt;
      if constexpr (GRAD) {
        const float sc = row_scale(a, row, wt);
        const float ca = big_a / all.s * sc, cr = rest.s == 0.f ? 0.f : r / rest.s * sc;
#pragma unroll 8
        for (int i = 0; i < V; ++i) {
          float g = ca * exp2_fast((x(i) - all.m) * a.c);
          if (!((named >> i) & 1) && cr != 0.f) g -= cr * exp2_fast((x(i) - rest.m) * a.c);
          o[i] = __float_as_uint(empty ? 0.f : broken ? __uint_as_float(0x7FC00000u) : g);
        }
        if (!empty && !broken)
          each_entry(index, lps, a.k, [&](int j, long long i, float) {
            o[i] = __float_as_uint(add_product(x((int)i), -(float)(q_of[64 * j] * per), sc));
          });
      }
    } else if constexpr (GRAD) {
      for (int i = 0; i < V; ++i) o[i] = 0u;
    }
    if (a.row_loss) a.row_loss[row] = loss;
  }
  if constexpr (GRAD) {
    __syncthreads();
    stage_rows<T, true>((T*)a.dx + (long)blockIdx.x * 64 * V, V, rows, V, lds, pitch);
  }
}

// ---------------------------------------------------------------- sums over the rows
// f64, in a fixed order: thread, wave, workgroup, workgroups.  part [gridDim.x][2]: this workgroup's sums of row_loss and of
// weight (either may be null: 0).
__global__ __launch_bounds__(1024) void distill_part_kernel(const float* __restrict__ row_loss,
                                                            const float* __restrict__ weight, long T, long per,
                                                            double* __restrict__ part) {
  __shared__ double red[2][16];
  const long lo = blockIdx.x * per, hi = min(T, lo + per);
  double s = 0.0, w = 0.0;
#pragma unroll 4
  for (long i = lo + threadIdx.x; i < hi; i += 1024) {
    if (row_loss) s += (double)row_loss[i];
    if (weight) w += (double)weight[i];
  }
  s = wave_sum_f64(s);
  w = wave_sum_f64(w);
  if ((threadIdx.x & 63) == 0) { red[0][threadIdx.x >> 6] = s; red[1][threadIdx.x >> 6] = w; }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = w = 0.0;
    for (int k = 0; k < 16; ++k) { s += red[0][k]; w += red[1][k]; }
    part[2 * blockIdx.x] = s;
    part[2 * blockIdx.x + 1] = w;
  }
}
// out[0] = sum row_loss (mean: / sum weight), wsum_out = sum weight, from n <= 256 pairs or (part null) from the rows.
__global__ __launch_bounds__(1024) void distill_sum_kernel(const float* __restrict__ row_loss,
                                                           const float* __restrict__ weight, long T,
                                                           const double* __restrict__ part, int n, int mean,
                                                           float* __restrict__ out, float* __restrict__ wsum_out) {
  __shared__ double red[2][16];
  double s = 0.0, w = 0.0;
  if (part) {
    if ((int)threadIdx.x < n) { s = part[2 * threadIdx.x]; w = part[2 * threadIdx.x + 1]; }
  } else {
#pragma unroll 8
    for (long i = threadIdx.x; i < T; i += 1024) {
      if (row_loss) s += (double)row_loss[i];
      if (weight) w += (double)weight[i];
    }
  }
  s = wave_sum_f64(s);
  w = wave_sum_f64(w);
  if ((threadIdx.x & 63) == 0) { red[0][threadIdx.x >> 6] = s; red[1][threadIdx.x >> 6] = w; }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = w = 0.0;
    for (int k = 0; k < 16; ++k) { s += red[0][k]; w += red[1][k]; }
    if (!weight) w = (double)T;
    if (out) out[0] = (float)(mean ? s / w : s);
    if (wsum_out) wsum_out[0] = (float)w;
  }
}

// ---------------------------------------------------------------- host launchers
// Segments per row: as for the scores but for rows that one workgroup holds, and never more tokens than the bits take.  Loss
// of 400 x 50000 bf16 17 us in one segment, 22 in three; loss and gradient 27 and 37; of 4 x 30000 fp16 11 and 13.
int distill_segments(long T, int V) {
  const long least = (V + DISTILL_SEGMENT - 1) / DISTILL_SEGMENT;
  if (V <= 32768 || logits_rows_fill(T, V, 64)) return (int)least;
  long s = (512 + T - 1) / T, most = (V + 2047) / 2048;
  if (s > most) s = most;
  if (s > LOGITS_MAX_SEGMENTS) s = LOGITS_MAX_SEGMENTS;
  return (int)(s > least ? s : least);
}
static int seg_len_of(int V, int S) { return ((V + S - 1) / S + 31) / 32 * 32; }

// Loss and gradient of rows that fit a workgroup's registers.  false: they do not, or (2-byte types above 32768) would
// leave one workgroup per CU, whose reading, reducing and writing then follow each other: 4096 x 65536 bf16 261 us,
// against 249 us for the kernel that reads the row again from the last-level cache; 8192 x 32768: 227 against 261 us.
template <typename T, bool STREAM>
static bool launch_resident(const DistillTopkArgs& a, hipStream_t s) {
  constexpr int MAX = 64 / (32 * (int)sizeof(T) / 4);   // steps in 64 registers: 4 for 2-byte types, 2 for f32
  const dim3 g((unsigned)a.T);
  // Few rows: a row in one step of a large workgroup.  fp16: 100 x 3000 7.2 us, on one wave 10.6; 1000 x 3000 10.5 and 12.8;
  // 100 x 17339 12.3, in two steps of 256 threads 16.9, but 1000 x 17339 41 and 35.  (Never more than STREAM_BYTES of results.)
  if (a.V > 1024 && (a.V <= 8192 ? a.T <= 1024 : a.V <= 32768 && a.T <= 256)) {
    if (a.V <= 256 * 8) hipLaunchKernelGGL((distill_resident_kernel<T, 256, 1, false, 8>), g, dim3(256), 0, s, a);
    else if (a.V <= 256 * 16) hipLaunchKernelGGL((distill_resident_kernel<T, 256, 1, false, 16>), g, dim3(256), 0, s, a);
    else if (a.V <= 256 * 32) hipLaunchKernelGGL((distill_resident_kernel<T, 256, 1, false>), g, dim3(256), 0, s, a);
    else if (a.V <= 512 * 32) hipLaunchKernelGGL((distill_resident_kernel<T, 512, 1, false>), g, dim3(512), 0, s, a);
    else hipLaunchKernelGGL((distill_resident_kernel<T, 1024, 1, false>), g, dim3(1024), 0, s, a);
    return true;
  }
  if (a.V <= 64 * 8) hipLaunchKernelGGL((distill_resident_kernel<T, 64, 1, STREAM, 8>), g, dim3(64), 0, s, a);
  else if (a.V <= 64 * 16) hipLaunchKernelGGL((distill_resident_kernel<T, 64, 1, STREAM, 16>), g, dim3(64), 0, s, a);
  else if (a.V <= 64 * 32) hipLaunchKernelGGL((distill_resident_kernel<T, 64, 1, STREAM>), g, dim3(64), 0, s, a);
  else if (a.V <= 64 * 64) hipLaunchKernelGGL((distill_resident_kernel<T, 64, 2, STREAM>), g, dim3(64), 0, s, a);
  else if (a.V <= 256 * 32) hipLaunchKernelGGL((distill_resident_kernel<T, 256, 1, STREAM>), g, dim3(256), 0, s, a);
  else if (a.V <= 256 * 64) hipLaunchKernelGGL((distill_resident_kernel<T, 256, 2, STREAM>), g, dim3(256), 0, s, a);
  else if (a.V <= 256 * 32 * MAX) hipLaunchKernelGGL((distill_resident_kernel<T, 256, MAX, STREAM>), g, dim3(256), 0, s, a);
  else if (sizeof(T) == 4 && a.V <= 512 * 64)
    hipLaunchKernelGGL((distill_resident_kernel<float, 512, 2, STREAM>), g, dim3(512), 0, s, a);
  else if (sizeof(T) == 4 && a.V <= 1024 * 64)
    hipLaunchKernelGGL((distill_resident_kernel<float, 1024, 2, STREAM>), g, dim3(1024), 0, s, a);
  else return false;
  return true;
}
template <typename T, bool STREAM>
static void distill_typed(DistillTopkArgs a, bool loss, bool grad, hipStream_t s) {
  if (a.by_thread) {
    const dim3 g((unsigned)((a.T + 63) / 64));
    const unsigned lds = small_lds(a.V) + 64 * a.k * sizeof(double);   // 49 KB at most
    if (grad) hipLaunchKernelGGL((distill_small_kernel<T, true>), g, dim3(64), lds, s, a);
    else hipLaunchKernelGGL((distill_small_kernel<T, false>), g, dim3(64), lds, s, a);
    return;
  }
  int S = a.S;
  if (S == 1 && loss && grad) {
    a.tape = a.g_top = nullptr;   // for a backward of its own only
    // (512 threads: two workgroups per CU, whose rows fit the last-level cache together; 256: 2048 x 131072 300 us, 512: 251 us)
    if (!launch_resident<T, STREAM>(a, s))
      hipLaunchKernelGGL((distill_kernel<T, 512, 32, DISTILL_SEGMENT / 32, true, STREAM>), dim3((unsigned)a.T), dim3(512), 0, s,
                         a, 1, a.V);
    return;
  }
  if (loss) {
    const dim3 g((unsigned)a.T);
    if (S > 1) {
      const int len = seg_len_of(a.V, S);
      S = (a.V + len - 1) / len;
      const dim3 gs((unsigned)(a.T * S));
      if (len <= 2048) hipLaunchKernelGGL((distill_kernel<T, 256, 8, 64, false>), gs, dim3(256), 0, s, a, S, len);
      else if (len <= 4096) hipLaunchKernelGGL((distill_kernel<T, 256, 16, 128, false>), gs, dim3(256), 0, s, a, S, len);
      else hipLaunchKernelGGL((distill_kernel<T, 256, 32, DISTILL_SEGMENT / 32, false>), gs, dim3(256), 0, s, a, S, len);
      hipLaunchKernelGGL((distill_join_kernel<T>), g, dim3(64), 0, s, a, S);
    } else if (a.T <= 1024 && a.V > 1024 && a.V <= 4096) {   // one step: 400 x 3000 fp16 6.8 us, on one wave 8.3
      if (a.V <= 2048) hipLaunchKernelGGL((distill_kernel<T, 256, 8, 64, false>), g, dim3(256), 0, s, a, 1, a.V);
      else hipLaunchKernelGGL((distill_kernel<T, 256, 16, 128, false>), g, dim3(256), 0, s, a, 1, a.V);
    } else if (a.V <= 512) {
      hipLaunchKernelGGL((distill_kernel<T, 64, 8, 16, false>), g, dim3(64), 0, s, a, 1, a.V);
    } else if (a.V <= 1024) {
      hipLaunchKernelGGL((distill_kernel<T, 64, 16, 32, false>), g, dim3(64), 0, s, a, 1, a.V);
    } else if (a.V <= 8192 && a.T > 1024) {   // one wave: 20000 x 4000 bf16 47 us, 256 threads 89 us; 10000 x 8000 42 and 48 us
      hipLaunchKernelGGL((distill_kernel<T, 64, 32, 256, false>), g, dim3(64), 0, s, a, 1, a.V);
    } else if (a.T <= 256 && a.V > 8192) {   // a workgroup per CU: 100 x 131072 bf16 14.7 us, on 256 threads 20.3
      hipLaunchKernelGGL((distill_kernel<T, 512, 32, DISTILL_SEGMENT / 32, false>), g, dim3(512), 0, s, a, 1, a.V);
    } else {
      hipLaunchKernelGGL((distill_kernel<T, 256, 32, DISTILL_SEGMENT / 32, false>), g, dim3(256), 0, s, a, 1, a.V);
    }
  }
  if (grad) {
    if (a.V <= 512) {
      hipLaunchKernelGGL((distill_bwd_kernel<T, 64, 8, STREAM>), dim3((unsigned)a.T), dim3(64), 0, s, a, 1, a.V);
    } else if (a.V <= 1024) {
      hipLaunchKernelGGL((distill_bwd_kernel<T, 64, 16, STREAM>), dim3((unsigned)a.T), dim3(64), 0, s, a, 1, a.V);
    } else if (a.V <= 2048) {
      hipLaunchKernelGGL((distill_bwd_kernel<T, 64, 32, STREAM>), dim3((unsigned)a.T), dim3(64), 0, s, a, 1, a.V);
    } else {
      const int len = logits_bwd_segment(a.T, a.V), sb = (a.V + len - 1) / len;
      hipLaunchKernelGGL((distill_bwd_kernel<T, 256, 32, STREAM>), dim3((unsigned)(a.T * sb)), dim3(256), 0, s, a, sb, len);
    }
  }
}
template <typename T>
static void distill_sized(const DistillTopkArgs& a, bool loss, bool grad, hipStream_t s) {
  if (grad && a.T * a.V * (long)sizeof(T) > STREAM_BYTES) distill_typed<T, true>(a, loss, grad, s);
  else distill_typed<T, false>(a, loss, grad, s);
}
static void distill_dispatch(const DistillTopkArgs& all, bool loss, bool grad, hipStream_t s) {
  const long size = all.type == SCM_F32 ? 4 : 2, most = std::max(LOGITS_LAUNCH_ROWS / all.S, 1L);
  for (long t = 0; t < all.T; t += most) {
    DistillTopkArgs a = all;   // n rows from row t on
    a.T = std::min(all.T - t, most);
    a.x = (const char*)a.x + t * a.ldx * size;
    a.index += t * a.k;
    a.lp += t * a.k;
    if (a.weight) a.weight += t;
    if (a.row_loss) a.row_loss += t;
    if (a.tape) { a.tape += 2 * t; a.g_top += t * a.k; }
    if (a.part) a.part += 2 * t * a.S;
    if (a.gloss_rows) a.gloss += t;
    if (a.dx) a.dx = (char*)a.dx + t * a.V * size;
    if (a.type == SCM_F32) distill_sized<float>(a, loss, grad, s);
    else if (a.type == SCM_BF16) distill_sized<bf16>(a, loss, grad, s);
    else distill_sized<f16>(a, loss, grad, s);
  }
}
// One workgroup adds up to 16384 rows; more of them (1,000,000 rows: 330 us) go through 4096-row parts at least.
static void distill_sum(const DistillTopkArgs& a, const float* row_loss, const float* weight, int mean, float* out,
                        float* wsum_out, hipStream_t s) {
  int n = 0;
  if (a.T > DISTILL_SUM_ROWS) {
    const long per = a.T > 256L * 4096 ? (a.T + 255) / 256 : 4096;
    n = (int)((a.T + per - 1) / per);
    hipLaunchKernelGGL(distill_part_kernel, dim3(n), dim3(1024), 0, s, row_loss, weight, a.T, per, a.sums);
  }
  hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, s, row_loss, weight, a.T, n ? a.sums : (double*)nullptr, n,
                     mean, out, wsum_out);
}
hipError_t topk_distill_fwd(const DistillTopkArgs& a, float* out, float* wsum_out, hipStream_t s) {
  Traced tr(K_TOPK_DISTILL, 0, s);
  distill_dispatch(a, true, false, s);
  if (out || wsum_out) distill_sum(a, out ? a.row_loss : nullptr, a.weight, a.mean, out, wsum_out, s);
  return hipGetLastError();
}
hipError_t topk_distill_bwd(const DistillTopkArgs& a, hipStream_t s) {
  Traced tr(K_TOPK_DISTILL, 0, s);
  distill_dispatch(a, false, true, s);
  return hipGetLastError();
}
hipError_t topk_distill_step(const DistillTopkArgs& all, float* out, float* wsum, hipStream_t s) {
  Traced tr(K_TOPK_DISTILL, 0, s);
  // the gradient of a mean needs the weights' sum first: few of them are added up by every wave, which saves a launch
  // (37 x 1000 fp16: 7.0 us, with a launch of its own 8.7)
  DistillTopkArgs a = all;
  a.sum_weights = a.weight && a.mean && !a.by_thread && a.rows <= 1024;
  a.weights = a.weight;
  const bool first = a.weight && a.mean && !a.sum_weights;
  if (a.sum_weights) a.wsum = nullptr;
  else if (first) distill_sum(a, nullptr, a.weight, 0, nullptr, wsum, s);
  distill_dispatch(a, true, true, s);
  distill_sum(a, a.row_loss, a.weight, a.mean, out, first ? nullptr : wsum, s);
  return hipGetLastError();
}

}  // namespace scm
