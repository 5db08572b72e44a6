// What the kernels that read rows of logits share: running softmax statistics and their joins, the walk of a workgroup
// over a row (or a segment of one), and the staging of short rows.
#pragma once
#include "scm_chunk.hpp"

namespace scm {

constexpr float LOWEST = -3.402823466e38f;
constexpr float LN2 = 0.6931471805599453f;

SCM_DEV float log2_fast(float x) { return __builtin_amdgcn_logf(x); }
// a + b c with the product rounded, as the terms that may cancel it were: where one token has all the probability its
// gradient is 0, not the rounding of a product.
SCM_DEV float add_product(float a, float b, float c) {
#pragma clang fp contract(off)
  const float p = b * c;
  return a + p;
}

// ---------------------------------------------------------------- softmax statistics
// m: maximum of the elements (LOWEST where there are none above it), s = sum 2^((x-m)c), h = sum 2^((x-m)c) (x-m)c.
// s == 0: no element above -inf.  s is NaN where an element is NaN or +inf.
struct Stat { float m, s, h; };
SCM_DEV Stat stat_none() { return {LOWEST, 0.f, 0.f}; }
// The factor for a maximum that grew: 2^-200 is 0 in f32, and the bound keeps 0 * inf out of h.
SCM_DEV float grown(float from, float to, float c) { return fmaxf((from - to) * c, -200.f); }
template <bool ENT>
SCM_DEV Stat stat_join(const Stat& a, const Stat& b, float c) {
  const float m = fmaxf(a.m, b.m);
  const float da = grown(a.m, m, c), db = grown(b.m, m, c);
  const float fa = exp2_fast(da), fb = exp2_fast(db);
  Stat r{m, a.s * fa + b.s * fb, 0.f};
  if constexpr (ENT) r.h = fa * (a.h + da * a.s) + fb * (b.h + db * b.s);
  return r;
}
// Over the 64 lanes, in every lane: the common maximum first, then one rescaling and plain sums.
template <bool ENT>
SCM_DEV Stat stat_wave(const Stat& v, float c) {
  const float m = wave_max(v.m), d = grown(v.m, m, c), f = exp2_fast(d);
  return {m, wave_sum(v.s * f), ENT ? wave_sum(f * (v.h + d * v.s)) : 0.f};
}
// Over the NT threads of the workgroup, in every thread.  red: NT / 64 entries.
template <bool ENT, int NT>
SCM_DEV Stat stat_block(Stat v, float c, Stat* red) {
  v = stat_wave<ENT>(v, c);
  if constexpr (NT == 64) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  Stat r{LOWEST, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) r.m = fmaxf(r.m, red[w].m);
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    const float d = grown(red[w].m, r.m, c), f = exp2_fast(d);
    r.s += red[w].s * f;
    if constexpr (ENT) r.h += f * (red[w].h + d * red[w].s);
  }
  return r;
}

// Per-thread view of a segment [lo, lo + len) of a row, in steps of EL elements (U chunks) a thread: chunk u of step s is
// chunk (s U + u) NT + tid of the segment.
template <typename T, int NT, int EL_ = 32>
struct Walk {
  static constexpr int EL = EL_, E = 16 / sizeof(T), U = EL / E, STEP = NT * EL;
  typedef Chunk<T, E> Raw[U];
  const T* p;
  int len;
  SCM_DEV int steps() const { return (len + STEP - 1) / STEP; }
  SCM_DEV int first(int step, int u) const { return ((step * U + u) * NT + (int)threadIdx.x) * E; }
  SCM_DEV void load(int step, Raw& raw) const {
    if ((step + 1) * STEP <= len) {   // the same for all threads
#pragma unroll
      for (int u = 0; u < U; ++u) __builtin_memcpy(&raw[u], p + first(step, u), sizeof(raw[u]));
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = load_chunk<T, E>(p + first(step, u), len - first(step, u));
    }
  }
  // f(step, raw) for every step; the next step's loads are on their way meanwhile
  template <typename F>
  SCM_DEV void run(F f) const {
    const int n = steps();
    Raw a, b;
    load(0, a);
    for (int s = 0; s < n; s += 2) {
      if (s + 1 < n) load(s + 1, b);
      f(s, a);
      if (s + 1 < n) {
        if (s + 2 < n) load(s + 2, a);
        f(s + 1, b);
      }
    }
  }
  // the elements of a step as f32, -inf past the end
  SCM_DEV void values(int step, const Raw& raw, float (&v)[EL]) const {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < E; ++j) v[u * E + j] = (float)raw[u].e[j];
    if ((step + 1) * STEP > len) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (first(step, u) + j >= len) v[u * E + j] = -INFINITY;
    }
  }
};

// Between two uses of a chunk that stays in registers: keeps the compiler from holding on to its f32 values (twice the
// registers) instead of unpacking them again.
template <typename T, int E>
SCM_DEV void stay_packed(Chunk<T, E>& c) {
  if constexpr (sizeof(T) == 4) return;   // f32 is as it lies
  u32x4 w = __builtin_bit_cast(u32x4, c);
#pragma unroll
  for (int i = 0; i < 4; ++i) { uint32_t x = w[i]; asm volatile("" : "+v"(x)); w[i] = x; }
  c = __builtin_bit_cast(Chunk<T, E>, w);
}

// Adds EL elements, their maximum bm, to a thread's running statistics.
template <bool ENT, int EL>
SCM_DEV void stat_add(Stat& st, const float (&v)[EL], float bm, float c) {
  const float m = fmaxf(st.m, bm);
  const float d0 = grown(st.m, m, c), f = exp2_fast(d0);
  float s = st.s * f, h = ENT ? f * (st.h + d0 * st.s) : 0.f;
#pragma unroll
  for (int j = 0; j < EL; ++j) {
    const float d = (v[j] - m) * c, e = exp2_fast(d);
    s += e;
    if constexpr (ENT) h += e * fmaxf(d, -200.f);
  }
  st = {m, s, h};
}

// Short rows, one thread each: 64 rows go through LDS (row stride odd: no bank conflicts along a column) as f32 bits,
// read and written along memory, eight elements of a thread on their way at once.
constexpr unsigned small_lds(int V) { return 64 * (V | 1) * 4; }
template <typename T, bool STORE>
SCM_DEV void stage_rows(T* p, long ld, int rows, int V, uint32_t* lds, int pitch) {
  constexpr int B = 8;
  const int dr = 64 / V, dc = 64 % V;
  int r = threadIdx.x / V, c = threadIdx.x % V;
  while (r < rows) {
    int row[B], col[B];
    uint32_t v[B];
#pragma unroll
    for (int b = 0; b < B; ++b) {
      row[b] = r;
      col[b] = c;
      const int rr = min(r, rows - 1);   // past the end: some element, not used
      v[b] = STORE ? lds[rr * pitch + c] : __float_as_uint((float)p[rr * ld + c]);
      r += dr;
      c += dc;
      if (c >= V) { c -= V; ++r; }
    }
#pragma unroll
    for (int b = 0; b < B; ++b)
      if (row[b] < rows) {
        if constexpr (STORE) p[row[b] * ld + col[b]] = (T)__uint_as_float(v[b]);
        else lds[row[b] * pitch + col[b]] = v[b];
      }
  }
}

}  // namespace scm
