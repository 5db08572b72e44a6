// Rows of f32 / bf16 / fp16 read and written in 16-byte chunks, computed on in f32.
#pragma once
#include "scm_launch.hpp"

namespace scm {

typedef _Float16 f16;

// E consecutive elements as they lie in memory.  Rows of odd width start at any element: the copies below ask for
// element alignment only, which global loads and stores of every width accept on this hardware (one instruction per
// chunk; a chunk that crosses a cache line costs a second lookup, no second instruction).
template <typename T, int E>
struct Chunk { T e[E]; };

template <typename T, int E>
SCM_DEV Chunk<T, E> load_chunk(const T* p, int n) {   // n valid elements (<= 0: none); the others are 0
  Chunk<T, E> c;
  if (n >= E) {
    __builtin_memcpy(&c, p, sizeof(c));
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j) c.e[j] = j < n ? p[j] : (T)0.f;
  }
  return c;
}

// STREAM: a store that does not keep its line in the caches (results larger than those, next to inputs read twice).
template <typename T, int E, bool STREAM = false>
SCM_DEV void store_chunk(T* p, const float (&v)[E], int n) {   // rounds to nearest even
  Chunk<T, E> c;
#pragma unroll
  for (int j = 0; j < E; ++j) c.e[j] = (T)v[j];
  if (n >= E) {
    if constexpr (STREAM && sizeof(c) == 16) {
      typedef u32x4 __attribute__((aligned(2))) any_u32x4;
      __builtin_nontemporal_store(__builtin_bit_cast(u32x4, c), (any_u32x4*)p);
    } else {
      __builtin_memcpy(p, &c, sizeof(c));
    }
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (j < n) p[j] = c.e[j];
  }
}

// Sum over groups of L consecutive lanes (L = 16, 32 or 64), in every lane of the group.
template <int L>
SCM_DEV float lanes_sum(float v) {
  if constexpr (L == 64) return wave_sum(v);
  v += dpp_move<0xB1>(v);
  v += dpp_move<0x4E>(v);
  v += dpp_move<0x141>(v);
  v += dpp_move<0x140>(v);
  if constexpr (L == 32) v += __shfl_xor(v, 16);
  return v;
}

// Results of more bytes than the L2 caches hold (8 x 4 MB) are written with STREAM: they would push out what is still to be
// read (8192 x 4096 bf16 layer norm forward: 26 us, 27 without; gradient of 4096 x 65536 bf16 logits: 186 and 214; loss and
// gradient of 20000 x 4000: 65 and 91, of 2048 x 131072: 251 and 291, of 8192 x 32768: 227 and 222).
constexpr long STREAM_BYTES = 32L << 20;

}  // namespace scm
