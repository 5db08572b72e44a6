// What is read off a row of logits x[0..V), z = x / temperature, f32 / bf16 / fp16, any V: lse = log sum exp z, the log
// probability of a given token, the entropy, the k <= 64 most likely tokens; and the gradient of all of them.
//
// The logits are read once, in 16-byte chunks; every thread keeps a running maximum m and s = sum 2^((x - m) c),
// c = log2(e) / temperature, in f32; threads, waves and workgroups join by rescaling to the larger maximum.  x - m is
// formed first: a row of the type's lowest value is an ordinary (uniform) row, and -inf weighs nothing.
//   V <= 16, and many rows of V <= 64   one thread per row, 64 rows staged through LDS per wave
//   else                   64 to 512 threads per row by its length; where long rows are too few to fill the card a row is split
//                          into segments of one workgroup each, whose partial results a second launch joins in segment order
// What bounds them is HBM, and for 2-byte types the vector ALU nearly as much (an exponential costs four issue slots).
#include "scm_softmax.hpp"

#include <algorithm>

namespace scm {

// ---------------------------------------------------------------- order of the alternatives
// Larger key = earlier: by value, equal values (-0 and +0 among them) by lower index, NaN before everything.
// 0 is no key of any element.
SCM_DEV uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);   // -0 + 0 = +0
  const uint32_t o = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return x != x ? 0xFFFFFFFEu : o;
}
SCM_DEV float unordered(uint32_t o) {
  if (o == 0xFFFFFFFEu) return __uint_as_float(0x7FC00000u);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
SCM_DEV uint64_t key_of(uint32_t o, int idx) { return ((uint64_t)o << 32) | (uint32_t)~idx; }
SCM_DEV int key_index(uint64_t k) { return (int)~(uint32_t)k; }
SCM_DEV float key_value(uint64_t k) { return unordered((uint32_t)(k >> 32)); }
SCM_DEV uint64_t shfl64(uint64_t v, int mask) {
  return ((uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), mask) << 32) | (uint32_t)__shfl_xor((int)v, mask);
}

// ---------------------------------------------------------------- score: the k largest elements of a segment
// A lower bound of the k-th largest element comes free with the statistics: the k-th largest of the threads' maxima
// (each thread's maximum is an element of its own).  Only the elements of threads whose maximum reaches it (k or a few
// more) are looked at again, by the whole workgroup; what reaches the bound goes to LDS and is ranked there by counting.
struct TopBound { uint32_t value; int chunk; };   // at least value, equal ones at chunks <= chunk
template <int NT>
struct TopLds {
  static constexpr int CAP = NT == 64 ? 512 : 1024;   // NT >= 2 k: about NT ln 2 + spread at most are expected
  uint64_t cand[CAP];
  uint32_t best[NT];
  int at[NT];
  int count, threads;
  TopBound bound;
  uint64_t red[NT / 64];
  uint64_t picked[LOGITS_MAX_K + LOGITS_MAX_K / 8];
};
// Low bits of ordered() that carry nothing: the same for all values of one sign of a 16-bit type.
template <typename T> constexpr int order_spare = 0;
template <> constexpr int order_spare<bf16> = 16;
template <> constexpr int order_spare<f16> = 13;
// Minimum and maximum over the 64 lanes, in every lane.
template <int CTRL>
SCM_DEV uint32_t dpp_move_u32(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true); }
SCM_DEV void wave_range(uint32_t& lo, uint32_t& hi) {
  auto with = [&](uint32_t a, uint32_t b) { lo = min(lo, a); hi = max(hi, b); };
  with(dpp_move_u32<0xB1>(lo), dpp_move_u32<0xB1>(hi));
  with(dpp_move_u32<0x4E>(lo), dpp_move_u32<0x4E>(hi));
  with(dpp_move_u32<0x141>(lo), dpp_move_u32<0x141>(hi));
  with(dpp_move_u32<0x140>(lo), dpp_move_u32<0x140>(hi));
  with((uint32_t)__shfl_xor((int)lo, 16), (uint32_t)__shfl_xor((int)hi, 16));
  with((uint32_t)__shfl_xor((int)lo, 32), (uint32_t)__shfl_xor((int)hi, 32));
}
// Threshold (value, chunk) over the NT maxima, by the first wave: a value that k to k + k / 8 of them reach, found bit by
// bit below the bits that they all share; among equal maxima (more than that reach the last value) the chunk up to which
// the k-th place goes.  Threads without elements hold value 0.
template <int R>
SCM_DEV TopBound top_threshold(const uint32_t (&b)[R], const int (&at)[R], int k, int chunks, int spare) {
  constexpr int NT = R * 64;
  uint32_t lo = 0xFFFFFFFFu, hi = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    lo = b[r] ? min(lo, b[r]) : lo;
    hi = max(hi, b[r]);
  }
  wave_range(lo, hi);
  lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)lo);
  hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)hi);
  // all maxima lie in [lo, hi]; t keeps the invariant: reach of them are >= t, reach >= k (0: fewer than k threads hold
  // elements, then every element is a candidate)
  const int holders = min(chunks, NT);
  const int shared = lo == hi ? 0 : 32 - __builtin_clz(lo ^ hi);   // bits that differ
  uint32_t t = shared >= 32 || holders < k ? 0u : (hi >> shared) << shared;
  int reach = holders, above = 0, bit = holders < k ? -1 : shared - 1;
  const int enough = k + k / 8;
  if (k == 1) {   // the maximum itself
    t = hi;
    reach = 0;
    bit = -1;
#pragma unroll
    for (int r = 0; r < R; ++r) reach += __builtin_popcountll(__builtin_amdgcn_ballot_w64(b[r] == hi));
  }
  for (; bit >= spare && reach > enough; --bit) {
    const uint32_t cand = t | (1u << bit);
    int n = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(b[r] >= cand));
    if (n >= k) { t = cand; reach = n; } else { above = n; }
  }
  // all bits used and still too many: the maxima from t to t + 2^spare - 1 are equal, `above` lie above them
  const uint32_t top = t | ((1u << spare) - 1u);
  int lim = 0x7FFFFFFF;
  if (t && reach > enough) {
    const int need = k - above;   // the smallest bound with enough equal maxima at chunks <= lim
    lim = 0;
    for (bit = 31 - __builtin_clz(chunks | 1); bit >= 0; --bit) {
      const int cand = lim | (1 << bit);
      int n = 0;
#pragma unroll
      for (int r = 0; r < R; ++r)
        n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(b[r] >= t && b[r] <= top && at[r] < cand));
      if (n < need) lim = cand;
    }
  }
  return {t, lim};
}

// Many more candidates than places (rows with fewer chunks than places, ties): the first wave raises the bound to a key
// that k to k + k / 8 of the n candidates reach (keys are distinct), and those go to picked.  -> how many.
template <int NT>
SCM_DEV int top_thin_out(TopLds<NT>& L, int n, int k) {
  constexpr int R = TopLds<NT>::CAP / 64;
  const int l = threadIdx.x & 63;
  __syncthreads();
  if (threadIdx.x == 0) L.count = 0;
  __syncthreads();
  if (threadIdx.x < 64) {
    uint64_t c[R], lo = ~0ull, hi = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      c[r] = r * 64 + l < n ? L.cand[r * 64 + l] : 0;
      if (c[r]) { lo = c[r] < lo ? c[r] : lo; hi = c[r] > hi ? c[r] : hi; }
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint64_t x = shfl64(lo, o), y = shfl64(hi, o);
      lo = x < lo ? x : lo;
      hi = y > hi ? y : hi;
    }
    int bit = 63 - __builtin_clzll((lo ^ hi) | 1), reach = n;
    uint64_t t = bit >= 63 ? 0 : (hi >> (bit + 1)) << (bit + 1);
    for (; bit >= 0 && reach > k + k / 8; --bit) {
      const uint64_t cand = t | (1ull << bit);
      int m = 0;
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (r * 64 < n) m += __builtin_popcountll(__builtin_amdgcn_ballot_w64(c[r] >= cand));
      if (m >= k) { t = cand; reach = m; }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (c[r] && c[r] >= t) L.picked[atomicAdd(&L.count, 1)] = c[r];   // reach of them: all bits used, it is k
  }
  __syncthreads();
  return L.count;
}

// Calls emit(rank, key) for the k largest keys of the segment, each from one thread.  best, at: the thread's maximum
// (0: no elements) and the first of its chunks that holds it.  odd: the segment holds NaN or +inf (or may: then the
// threads' maxima are not to be used).
template <typename W, typename T, int NT, typename Emit>
SCM_DEV void top_of_segment(const W& w, int lo, int k, uint32_t best, int at, bool odd, TopLds<NT>& L, Emit emit) {
  constexpr int E = W::E, U = W::U, SPARE = order_spare<T>;
  const int tid = threadIdx.x;
  const int chunks = (w.len + E - 1) / E;
  TopBound bound;
  if constexpr (NT == 64) {
    const uint32_t b[1] = {best};
    const int a[1] = {at};
    bound = top_threshold(b, a, k, chunks, SPARE);
    if (tid == 0) L.count = 0;
  } else {
    L.best[tid] = best;
    L.at[tid] = at;
    if (tid == 0) L.count = L.threads = 0;
    __syncthreads();
    if (tid < 64) {
      uint32_t b[NT / 64];
      int a[NT / 64];
#pragma unroll
      for (int r = 0; r < NT / 64; ++r) { b[r] = L.best[r * 64 + tid]; a[r] = L.at[r * 64 + tid]; }
      bound = top_threshold(b, a, k, chunks, SPARE);
      if (tid == 0) L.bound = bound;
    }
    __syncthreads();
    bound = L.bound;
  }
  const uint32_t thr = bound.value, thr_top = thr | ((1u << SPARE) - 1u);
  const int thr_at = bound.chunk;
  if (!odd) {
    // the threads that reach it, then their chunks (thread t: t, t + NT, ...) spread over the whole workgroup
    const bool reaches = best && (best > thr_top || (best >= thr && at <= thr_at));
    int threads;
    if constexpr (NT == 64) {
      const unsigned long mask = __builtin_amdgcn_ballot_w64(reaches);
      if (reaches) L.at[__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u))] = tid;
      threads = __builtin_popcountll(mask);
      __syncthreads();
    } else {
      if (reaches) L.at[atomicAdd(&L.threads, 1)] = tid;
      __syncthreads();
      threads = L.threads;
    }
    // the bounds as numbers (at or below the order of -inf: every element)
    const float from = thr <= 0x007FFFFFu ? -INFINITY : unordered(thr), above = unordered(thr_top + 1);
    const int per = W::EL < 32 ? U : (chunks + NT - 1) / NT, pairs = threads * per;
    const float per_inv = 1.f / (float)per;
    for (int i = tid; i < pairs; i += NT) {
      // i / per: (i + 1/2) / per lies 1 / (2 per) or more from a whole number, further than f32 rounds it for i < 2^20
      const int nth = W::EL < 32 ? i / U : chunks < 1 << 20 ? (int)(((float)i + 0.5f) * per_inv) : i / per;
      const int c = L.at[nth] + NT * (i - nth * per);
      const Chunk<T, E> raw = load_chunk<T, E>(w.p + (long)c * E, w.len - c * E);
      const float least = c <= thr_at ? from : above;
      uint32_t hits = 0;
#pragma unroll
      for (int j = 0; j < E; ++j) hits |= (uint32_t)((float)raw.e[j] >= least) << j;
      if (w.len - c * E < E) hits &= (1u << max(w.len - c * E, 0)) - 1u;
      while (hits) {   // few: one read again each
        const int at_hit = c * E + __builtin_ctz(hits);
        hits &= hits - 1;
        const int pos = atomicAdd(&L.count, 1);
        if (pos < TopLds<NT>::CAP) L.cand[pos] = key_of(ordered((float)w.p[at_hit]), lo + at_hit);
      }
    }
  }
  __syncthreads();
  int n = L.count;
  if (!odd && n <= TopLds<NT>::CAP) {
    const uint64_t* list = L.cand;
    if (n > 128 && n > k + k / 8) {   // ranking reads n keys per candidate
      n = top_thin_out<NT>(L, n, k);
      list = L.picked;
    }
    for (int i = tid; i < n; i += NT) {
      const uint64_t mine = list[i];
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) rank += list[j] > mine;
      if (rank < k) emit(rank, mine);
    }
    return;
  }
  // more candidates than places (all large values in few threads' chunks), or NaN: k passes, each finding the largest
  // key below the last one
  uint64_t last = ~0ull;
  const int found = k < w.len ? k : w.len;
  for (int r = 0; r < found; ++r) {
    uint64_t mine = 0;
    for (int s = 0; s < w.steps(); ++s) {
      typename W::Raw raw;
      w.load(s, raw);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const int i = w.first(s, u) + j;
          const uint64_t key = key_of(ordered((float)raw[u].e[j]), lo + i);
          if (i < w.len && key < last && key > mine) mine = key;
        }
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const uint64_t x = shfl64(mine, o); mine = x > mine ? x : mine; }
    if ((tid & 63) == 0) L.red[tid >> 6] = mine;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < NT / 64; ++v) mine = L.red[v] > mine ? L.red[v] : mine;
    __syncthreads();
    last = mine;
    if (tid == 0) emit(r, mine);
  }
}

// ---------------------------------------------------------------- score: what a row's statistics give
struct RowScore {
  float m, s, l2, inv_t;   // l2 = log2 s
  SCM_DEV RowScore(const Stat& st, float inv_t_) : m(st.m), s(st.s), l2(log2_fast(st.s)), inv_t(inv_t_) {}
  SCM_DEV float lse() const { return s == 0.f ? -INFINITY : m * inv_t + LN2 * l2; }
  SCM_DEV float logp(float x) const { return s == 0.f ? -INFINITY : (x - m) * inv_t - LN2 * l2; }
  SCM_DEV float entropy(float h) const { return s == 0.f ? 0.f : LN2 * (l2 - h / s); }
};

template <bool ENT>
SCM_DEV void write_row(const ScoreArgs& a, long row, const Stat& st, float x_target, long long target) {
  const RowScore r(st, a.inv_t);
  if (a.target) {
    float lp = __uint_as_float(0x7FC00000u);   // an index outside the vocabulary has no probability
    if (target == a.ignore) lp = 0.f;
    else if (target >= 0 && target < a.V) lp = r.logp(x_target);
    a.logprob[row] = lp;
  }
  if (a.lse) a.lse[row] = r.lse();
  if constexpr (ENT) a.entropy[row] = r.entropy(st.h);
  if (a.tape) { a.tape[2 * row] = st.m; a.tape[2 * row + 1] = st.s; }
}

template <typename T, int NT, int EL, bool ENT, bool TOP>
__global__ __launch_bounds__(NT) void score_kernel(ScoreArgs a, int S, int seg_len) {
  __shared__ Stat red[NT / 64];
  __shared__ TopLds<TOP ? NT : 64> top;
  typedef Walk<T, NT, EL> W;
  const long row = blockIdx.x / S;
  const int seg = blockIdx.x % S, lo = seg * seg_len;
  const W w{(const T*)a.x + row * a.ldx + lo, min(a.V - lo, seg_len)};
  // the last thread writes the row's numbers (the first wave is busy with the alternatives); its target is here by then
  const bool writer = S == 1 && threadIdx.x == NT - 1;
  long long target = -1;
  float x_target = 0.f;
  if (writer && a.target) {
    target = a.target[row];
    if (target >= 0 && target < a.V) x_target = (float)w.p[target];
  }
  Stat st = stat_none();
  float best = -INFINITY;
  int at = threadIdx.x;
  w.run([&](int s, const typename W::Raw& raw) {
    float v[EL], bm = LOWEST;
    w.values(s, raw, v);
#pragma unroll
    for (int u = 0; u < W::U; ++u) {
      float cm = v[u * W::E];
#pragma unroll
      for (int j = 1; j < W::E; ++j) cm = fmaxf(cm, v[u * W::E + j]);
      bm = fmaxf(bm, cm);
      if constexpr (TOP) {
        at = cm > best ? (s * W::U + u) * NT + (int)threadIdx.x : at;
        best = fmaxf(best, cm);
      }
    }
    stat_add<ENT>(st, v, bm, a.c);
  });
  st = stat_block<ENT, NT>(st, a.c, red);
  const bool odd = !(st.s <= 3e38f);   // NaN
  if (S > 1) {
    const long slot = row * S + seg;
    if (threadIdx.x == 0) { a.part[3 * slot] = st.m; a.part[3 * slot + 1] = st.s; a.part[3 * slot + 2] = st.h; }
    if constexpr (TOP) {
      uint64_t* out = a.part_top + slot * a.k;
      for (int i = w.len + threadIdx.x; i < a.k; i += NT) out[i] = 0;   // a segment shorter than k
      top_of_segment<W, T, NT>(w, lo, a.k, (int)threadIdx.x * W::E < w.len ? ordered(best) : 0u, at, odd, top,
                            [&](int rank, uint64_t key) { out[rank] = key; });
    }
    return;
  }
  if (writer) write_row<ENT>(a, row, st, x_target, target);
  if constexpr (TOP) {
    const RowScore r(st, a.inv_t);
    top_of_segment<W, T, NT>(w, 0, a.k, (int)threadIdx.x * W::E < w.len ? ordered(best) : 0u, at, odd, top,
                          [&](int rank, uint64_t key) {
                            a.top_index[row * a.k + rank] = key_index(key);
                            a.top_logprob[row * a.k + rank] = r.logp(key_value(key));
                          });
  }
}

// Joins the S segments of a row.  Their sorted lists: with p = ceil(k / S) and q = ceil(k / p), at least p q >= k
// keys reach the q-th largest of the lists' p-th keys; those are collected and ranked by counting.
template <typename T, bool ENT>
__global__ __launch_bounds__(256) void score_join_kernel(ScoreArgs a, int S) {
  __shared__ uint64_t keys[LOGITS_JOIN_KEYS], cand[LOGITS_JOIN_KEYS];   // S k keys at most
  __shared__ uint64_t thr;
  __shared__ int count;
  const long row = blockIdx.x;
  const int tid = threadIdx.x, l = tid & 63, n = S * a.k;
  // everything that is read, at once: the keys, the segments' statistics (every wave joins them all), the target
  for (int i = tid; i < n; i += 256) keys[i] = a.part_top[row * n + i];
  Stat st = stat_none();
  if (l < S) {   // S <= 64
    const float* p = a.part + 3 * (row * S + l);
    st = Stat{p[0], p[1], p[2]};
  }
  long long target = -1;
  float x_target = 0.f;
  if (tid == 255 && a.target) {
    target = a.target[row];
    if (target >= 0 && target < a.V) x_target = (float)((const T*)a.x)[row * a.ldx + target];
  }
  st = stat_wave<ENT>(st, a.c);
  if (tid == 255) write_row<ENT>(a, row, st, x_target, target);
  if (!a.k) return;
  if (tid == 0) { count = 0; thr = 1; }
  __syncthreads();
  const int p = (a.k + S - 1) / S, q = (a.k + p - 1) / p;
  if (tid < S) {
    const uint64_t mine = keys[tid * a.k + p - 1];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < S; ++j) rank += keys[j * a.k + p - 1] > mine;
    if (rank == q - 1 && mine) thr = mine;   // keys are distinct; an empty place (0) bounds nothing
  }
  __syncthreads();
  const uint64_t t = thr;
  for (int i = tid; i < n; i += 256)
    if (keys[i] >= t) cand[atomicAdd(&count, 1)] = keys[i];
  __syncthreads();
  const RowScore r(st, a.inv_t);
  const int found = count;
  for (int i = tid; i < found; i += 256) {
    const uint64_t mine = cand[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < found; ++j) rank += cand[j] > mine;
    if (rank < a.k) {
      a.top_index[row * a.k + rank] = key_index(mine);
      a.top_logprob[row * a.k + rank] = r.logp(key_value(mine));
    }
  }
}

// ---------------------------------------------------------------- short rows, one thread each
// N > 0: rows of at most N logits, which stay in registers between the passes; else they are read from LDS in each.
template <typename T, bool ENT, int N>
__global__ __launch_bounds__(64) void score_small_kernel(ScoreArgs a) {
  extern __shared__ uint32_t lds[];
  const int V = a.V, pitch = V | 1, rows = (int)min((long)64, a.T - (long)blockIdx.x * 64);
  const long row = (long)blockIdx.x * 64 + threadIdx.x;
  const long long t = a.target && (int)threadIdx.x < rows ? a.target[row] : 0;   // on its way meanwhile
  stage_rows<const T, false>((const T*)a.x + (long)blockIdx.x * 64 * a.ldx, a.ldx, rows, V, lds, pitch);
  __syncthreads();
  if ((int)threadIdx.x >= rows) return;
  uint32_t* o = lds + threadIdx.x * pitch;
  float held[N > 0 ? N : 1];
  if constexpr (N > 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) held[i] = i < V ? __uint_as_float(o[i]) : -INFINITY;
  }
  const float xt = a.target && t >= 0 && t < V ? __uint_as_float(o[(int)t]) : 0.f;
  auto each = [&](auto f) {   // f(i, x_i); past the end -inf, which adds nothing
    if constexpr (N > 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) f(i, held[i]);
    } else {
#pragma unroll 8
      for (int i = 0; i < V; ++i) f(i, __uint_as_float(o[i]));
    }
  };
  Stat st = stat_none();
  each([&](int, float x) { st.m = fmaxf(st.m, x); });
  each([&](int, float x) {
    const float d = (x - st.m) * a.c, e = exp2_fast(d);
    st.s += e;
    if constexpr (ENT) st.h += e * fmaxf(d, -200.f);
  });
  write_row<ENT>(a, row, st, xt, t);
  if (!a.k) return;
  const RowScore r(st, a.inv_t);
  uint32_t order[N > 0 ? N : 1];
  if constexpr (N > 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) order[i] = i < V ? ordered(held[i]) : 0u;
  } else {
#pragma unroll 8
    for (int i = 0; i < V; ++i) o[i] = ordered(__uint_as_float(o[i]));
  }
  for (int j = 0; j < a.k; ++j) {   // k <= V selections, each taken out
    uint32_t b = 0;
    int bi = 0;
    if constexpr (N > 0) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (order[i] > b) { b = order[i]; bi = i; }
#pragma unroll
      for (int i = 0; i < N; ++i) order[i] = i == bi ? 0u : order[i];
    } else {
#pragma unroll 8
      for (int i = 0; i < V; ++i)
        if (o[i] > b) { b = o[i]; bi = i; }
      o[bi] = 0;
    }
    a.top_index[row * a.k + j] = bi;
    a.top_logprob[row * a.k + j] = r.logp(unordered(b));
  }
}

// ---------------------------------------------------------------- score: gradient
// dz_i = sum_{named s} g_s [i == s] - p_i (sum g_s - g_lse) - g_H p_i (ln p_i + H)  =  .. + e_i (ca + cb d_i),
// e_i = 2^d_i, d_i = (x_i - m) c, with the two coefficients of the row:
struct ScoreGrad { float m, ca, cb, g_target; long long target; bool has_target; };
SCM_DEV ScoreGrad score_grad(const ScoreGradArgs& a, long row, float g_top_sum) {
  ScoreGrad r{};
  r.m = a.tape[2 * row];
  const float s = a.tape[2 * row + 1];
  r.target = a.target ? a.target[row] : a.ignore;
  const bool used = r.target != a.ignore && a.g_logprob;
  r.has_target = used && r.target >= 0 && r.target < a.V;
  r.g_target = r.has_target ? a.g_logprob[row] : 0.f;
  float g = r.g_target + g_top_sum - (a.g_lse ? a.g_lse[row] : 0.f);
  if (used && !r.has_target) g = __uint_as_float(0x7FC00000u);
  const float gh = a.g_entropy ? a.g_entropy[row] : 0.f;
  if (s != 0.f) {   // a row without anything above -inf has no gradient
    const float f = a.inv_t / s;
    r.ca = -(g + gh * (a.g_entropy ? a.entropy[row] - LN2 * log2_fast(s) : 0.f)) * f;
    r.cb = -gh * LN2 * f;
  } else {
    r.has_target = false;
  }
  return r;
}
SCM_DEV float score_dx(const ScoreGrad& r, float x, float c) {
  const float d = (x - r.m) * c;
  return exp2_fast(d) * (r.ca + r.cb * fmaxf(d, -200.f));
}

template <typename T, int NT, int EL, bool STREAM>
__global__ __launch_bounds__(NT) void score_bwd_kernel(ScoreGradArgs a, int S, int seg_len) {
  __shared__ int target_named;
  typedef Walk<T, NT, EL> W;
  const long row = blockIdx.x / S;
  const int lo = (int)(blockIdx.x % S) * seg_len, tid = threadIdx.x;
  const T* x = (const T*)a.x + row * a.ldx;
  T* dx = (T*)a.dx + row * a.V;
  const W w{x + lo, min(a.V - lo, seg_len)};
  const int k = a.g_top ? a.k : 0;
  // every wave adds the k <= 64 gradients of the alternatives up by itself
  const float gt = wave_sum((tid & 63) < k ? a.g_top[row * k + (tid & 63)] : 0.f);
  const ScoreGrad r = score_grad(a, row, gt);
  if (tid == 0) target_named = 0;
  w.run([&](int s, const typename W::Raw& raw) {
#pragma unroll
    for (int u = 0; u < W::U; ++u) {
      float o[W::E];
#pragma unroll
      for (int j = 0; j < W::E; ++j) o[j] = score_dx(r, (float)raw[u].e[j], a.c);
      store_chunk<T, W::E, STREAM>(dx + lo + w.first(s, u), o, w.len - w.first(s, u));
    }
  });
  // the named elements again, after the barrier: the last store to an address is theirs
  __syncthreads();
  const bool row_empty = a.tape[2 * row + 1] == 0.f;
  if (tid < k && !row_empty) {
    const long long i = a.top_index[row * k + tid];
    float g = a.g_top[row * k + tid];
    if (r.has_target && i == r.target) { g += r.g_target; target_named = 1; }
    if (i >= lo && i < lo + w.len) dx[i] = (T)add_product(score_dx(r, (float)x[i], a.c), g, a.inv_t);
  }
  __syncthreads();
  if (tid == 0 && r.has_target && !target_named && r.target >= lo && r.target < lo + w.len)
    dx[r.target] = (T)add_product(score_dx(r, (float)x[r.target], a.c), r.g_target, a.inv_t);
}

template <typename T>
__global__ __launch_bounds__(64) void score_bwd_small_kernel(ScoreGradArgs a) {
  extern __shared__ uint32_t lds[];
  const int V = a.V, pitch = V | 1, rows = (int)min((long)64, a.T - (long)blockIdx.x * 64);
  const long row = (long)blockIdx.x * 64 + threadIdx.x;
  stage_rows<const T, false>((const T*)a.x + (long)blockIdx.x * 64 * a.ldx, a.ldx, rows, V, lds, pitch);
  __syncthreads();
  if ((int)threadIdx.x < rows) {
    uint32_t* o = lds + threadIdx.x * pitch;
    auto add = [&](long long i, float g) {
      if (i >= 0 && i < V) o[i] = __float_as_uint(add_product(__uint_as_float(o[i]), g, a.inv_t));
    };
    const int k = a.g_top ? a.k : 0;
    float gt = 0.f;
    for (int j = 0; j < k; ++j) gt += a.g_top[row * k + j];
    const ScoreGrad r = score_grad(a, row, gt);
    for (int i = 0; i < V; ++i) o[i] = __float_as_uint(score_dx(r, __uint_as_float(o[i]), a.c));
    if (a.tape[2 * row + 1] != 0.f) {
      for (int j = 0; j < k; ++j) add(a.top_index[row * k + j], a.g_top[row * k + j]);
      if (r.has_target) add(r.target, r.g_target);
    }
  }
  __syncthreads();
  stage_rows<T, true>((T*)a.dx + (long)blockIdx.x * 64 * V, V, rows, V, lds, pitch);
}

// ---------------------------------------------------------------- host launchers
// Segments per row.  One where a row is short or the rows alone keep the card busy: one launch, no partial results (bf16,
// k = 20: 400 x 131072 32 us against 35 us in 800 segments, 400 x 50000 20 and 23; but 100 x 131072 19 and 18 in 600, 64 x
// 65536 13.7 and 11.5 in 512).  Else about 512 workgroups (twice as many: 30 x 131072 15.1 us, against 14.7), of at least
// 2048 elements, and no more than the join takes.
int score_segments(long T, int V, int k) {
  if (V <= 8192 || logits_rows_fill(T, V, 128)) return 1;
  long s = (512 + T - 1) / T, most = (V + 2047) / 2048;
  if (s > most) s = most;
  if (s > LOGITS_MAX_SEGMENTS) s = LOGITS_MAX_SEGMENTS;
  if (k && s * k > LOGITS_JOIN_KEYS) s = LOGITS_JOIN_KEYS / k;
  return (int)s;
}
static int segment_length(int V, int S) { return ((V + S - 1) / S + 31) / 32 * 32; }
// segments that really hold elements once the length is rounded
static int segments_used(int V, int len) { return (V + len - 1) / len; }

// TOP_ONLY: a shape that is chosen for its alternatives
template <typename T, int NT, int EL = 32, bool TOP_ONLY = false>
static void launch_score(const ScoreArgs& a, int S, int len, hipStream_t s) {
  const dim3 g((unsigned)(a.T * S)), b(NT);
  if (TOP_ONLY || a.k) {
    if (a.entropy) hipLaunchKernelGGL((score_kernel<T, NT, EL, true, true>), g, b, 0, s, a, S, len);
    else hipLaunchKernelGGL((score_kernel<T, NT, EL, false, true>), g, b, 0, s, a, S, len);
  } else if constexpr (!TOP_ONLY) {
    if (a.entropy) hipLaunchKernelGGL((score_kernel<T, NT, EL, true, false>), g, b, 0, s, a, S, len);
    else hipLaunchKernelGGL((score_kernel<T, NT, EL, false, false>), g, b, 0, s, a, S, len);
  }
}
template <typename T, int N>
static void launch_score_small(const ScoreArgs& a, dim3 g, hipStream_t s) {
  if (a.entropy) hipLaunchKernelGGL((score_small_kernel<T, true, N>), g, dim3(64), small_lds(a.V), s, a);
  else hipLaunchKernelGGL((score_small_kernel<T, false, N>), g, dim3(64), small_lds(a.V), s, a);
}
template <typename T>
static void score_typed(const ScoreArgs& a, hipStream_t s) {
  if (score_by_thread(a.T, a.V)) {
    const dim3 g((unsigned)((a.T + 63) / 64));
    if (a.V <= 8) return launch_score_small<T, 8>(a, g, s);
    if (a.V <= 16) return launch_score_small<T, 16>(a, g, s);
    return launch_score_small<T, 0>(a, g, s);
  }
  int S = a.S;
  if (S > 1) {
    const int len = segment_length(a.V, S);
    S = segments_used(a.V, len);
    // a thread's elements by the segment: 3 x 131072 bf16, k = 20 in segments of 2048 13.6 us with 32, 12.5 with 8
    if (len <= 2048) launch_score<T, 256, 8>(a, S, len, s);
    else if (len <= 4096) launch_score<T, 256, 16>(a, S, len, s);
    else launch_score<T, 256>(a, S, len, s);
    if (a.entropy) hipLaunchKernelGGL((score_join_kernel<T, true>), dim3((unsigned)a.T), dim3(256), 0, s, a, S);
    else hipLaunchKernelGGL((score_join_kernel<T, false>), dim3((unsigned)a.T), dim3(256), 0, s, a, S);
    return;
  }
  // Threads per row by the row's bytes: more of them shorten the walk, fewer the reductions and the search for the
  // alternatives behind it, and leave more rows in flight; and at least two threads per alternative, so that the threads'
  // maxima bound them well.  bf16, k = 8: 20000 x 4000 52 us on 64 threads, 63 on 128; 6000 x 16000 50 on 128, 57 on 64, 55
  // on 256; 2048 x 65536 54 on 256, 56 on 128, 59 on 512; 1200 x 131072 68 on 512, 72 on 256.
  const long bytes = (long)a.V * sizeof(T);
  // few rows: a row in one step of four waves.  bf16: 100 x 3000 k = 20 7.2 us, on 64 threads 8.3; 400 x 6613 k = 32 8.5 and
  // 15.0; 1000 x 8000 k = 20 10.1 and 13.7, k = 2 10.7 and 9.6
  if (a.T <= (a.k > 8 ? 1024 : 512) && a.V > 1024 && a.V <= 8192) {
    if (a.V <= 2048) return launch_score<T, 256, 8>(a, 1, a.V, s);
    if (a.V <= 4096) return launch_score<T, 256, 16>(a, 1, a.V, s);
    return launch_score<T, 256>(a, 1, a.V, s);
  }
  if (a.V <= 512) return a.k <= 32 ? launch_score<T, 64, 8>(a, 1, a.V, s) : launch_score<T, 128, 8, true>(a, 1, a.V, s);
  if (a.V <= 1024 && a.k <= 32) return launch_score<T, 64, 16>(a, 1, a.V, s);
  if (bytes <= 16384 && a.k <= 32) return launch_score<T, 64>(a, 1, a.V, s);
  // a workgroup per CU at most, and many alternatives: 150 x 60000 bf16, k = 64 18 us, on 256 threads 22 (k = 20: 15 and 16)
  if (a.T <= 256 && a.V > 8192 && a.k > 32) return launch_score<T, 512>(a, 1, a.V, s);
  if (bytes <= 49152) return launch_score<T, 128>(a, 1, a.V, s);
  if (bytes <= 196608) return launch_score<T, 256>(a, 1, a.V, s);
  launch_score<T, 512>(a, 1, a.V, s);
}
template <typename T, bool STREAM>
static void score_bwd_typed(const ScoreGradArgs& a, hipStream_t s) {
  if (logits_by_thread(a.T, a.V)) {
    hipLaunchKernelGGL((score_bwd_small_kernel<T>), dim3((unsigned)((a.T + 63) / 64)), dim3(64), small_lds(a.V), s, a);
  } else if (a.V <= 512) {   // one step of one wave
    hipLaunchKernelGGL((score_bwd_kernel<T, 64, 8, STREAM>), dim3((unsigned)a.T), dim3(64), 0, s, a, 1, a.V);
  } else if (a.V <= 1024) {
    hipLaunchKernelGGL((score_bwd_kernel<T, 64, 16, STREAM>), dim3((unsigned)a.T), dim3(64), 0, s, a, 1, a.V);
  } else if (a.V <= 2048) {
    hipLaunchKernelGGL((score_bwd_kernel<T, 64, 32, STREAM>), dim3((unsigned)a.T), dim3(64), 0, s, a, 1, a.V);
  } else {
    // the gradient of an element needs the row's two coefficients only: segments at will, 8192 elements are one step
    const int len = logits_bwd_segment(a.T, a.V), S = segments_used(a.V, len);
    hipLaunchKernelGGL((score_bwd_kernel<T, 256, 32, STREAM>), dim3((unsigned)(a.T * S)), dim3(256), 0, s, a, S, len);
  }
}
template <typename T>
static void score_bwd_sized(const ScoreGradArgs& a, hipStream_t s) {
  if (a.T * a.V * (long)sizeof(T) > STREAM_BYTES) score_bwd_typed<T, true>(a, s);
  else score_bwd_typed<T, false>(a, s);
}
// At least 8192 elements per workgroup; longer where that leaves more workgroups of 256 threads than a launch takes.
int logits_bwd_segment(long T, int V) {
  int len = 8192;
  while ((long)segments_used(V, len) * T >= 1L << 24) len *= 2;
  return len;
}
// n rows of a call from row t on.
static ScoreArgs rows_from(ScoreArgs a, long t, long n) {
  a.x = (const char*)a.x + t * a.ldx * (a.type == SCM_F32 ? 4 : 2);
  a.T = n;
  if (a.target) { a.target += t; a.logprob += t; }
  if (a.lse) a.lse += t;
  if (a.entropy) a.entropy += t;
  if (a.k) { a.top_logprob += t * a.k; a.top_index += t * a.k; }
  if (a.tape) a.tape += 2 * t;
  return a;   // the partial results stay: rows are split only where one launch takes them all
}
static ScoreGradArgs rows_from(ScoreGradArgs a, long t, long n) {
  const long size = a.type == SCM_F32 ? 4 : 2;
  a.x = (const char*)a.x + t * a.ldx * size;
  a.dx = (char*)a.dx + t * a.V * size;
  a.T = n;
  a.tape += 2 * t;
  if (a.target) a.target += t;
  if (a.entropy) a.entropy += t;
  if (a.top_index) a.top_index += t * a.k;
  if (a.g_logprob) a.g_logprob += t;
  if (a.g_lse) a.g_lse += t;
  if (a.g_entropy) a.g_entropy += t;
  if (a.g_top) a.g_top += t * a.k;
  return a;
}
hipError_t score_fwd(const ScoreArgs& all, hipStream_t s) {
  Traced tr(K_SCORE, 0, s);
  for (long t = 0; t < all.T; t += LOGITS_LAUNCH_ROWS) {
    const ScoreArgs a = rows_from(all, t, std::min(all.T - t, LOGITS_LAUNCH_ROWS));
    if (a.type == SCM_F32) score_typed<float>(a, s);
    else if (a.type == SCM_BF16) score_typed<bf16>(a, s);
    else score_typed<f16>(a, s);
  }
  return hipGetLastError();
}
hipError_t score_bwd(const ScoreGradArgs& all, hipStream_t s) {
  Traced tr(K_SCORE, 0, s);
  for (long t = 0; t < all.T; t += LOGITS_LAUNCH_ROWS) {
    const ScoreGradArgs a = rows_from(all, t, std::min(all.T - t, LOGITS_LAUNCH_ROWS));
    if (a.type == SCM_F32) score_bwd_sized<float>(a, s);
    else if (a.type == SCM_BF16) score_bwd_sized<bf16>(a, s);
    else score_bwd_sized<f16>(a, s);
  }
  return hipGetLastError();
}

}  // namespace scm
