// Rotation of query/key heads in either rotary layout, shared by the rotary kernel and the
// latent-cache store.  A pair (a, b) at angle t becomes (a cos t - b sin t, b cos t + a sin t);
// the pair is elements (2i, 2i + 1) in the interleaved layout and (i, i + rot/2) in the half
// layout.  Products and sums are fp32 and the result is rounded once: with the fp32 table of
// far positions the error of an element is half a step of its type, while rounding each
// product (what the in-place NeoX op does, to equal vLLM's torch path) would add two more.
#pragma once

#include "common.cuh"

namespace ntb200 {
namespace {

// Vectors a lane of a prefill-sized call takes, all loaded before the first is rotated.  Consecutive
// warps take consecutive vectors of a token, so that what is in flight lies close together in DRAM:
// a warp that walked a whole token with the same bytes in flight was slower (8191 tokens of 128
// heads in the store: 60 us so, 94 us walking; 78 us with 2 vectors, 68 with 6, 85 with 8).
constexpr int kRotItems = 4;

// N table entries as fp32, in 16-byte (or narrower) loads
template <typename C, int N>
__device__ __forceinline__ void load_table(const C* p, float (&out)[N]) {
  constexpr int kPiece = N * sizeof(C) > 16 ? 16 / sizeof(C) : N;
#pragma unroll
  for (int i = 0; i < N; i += kPiece) {
    float piece[kPiece];
    load_f<C, kPiece>(p + i, piece);
#pragma unroll
    for (int j = 0; j < kPiece; ++j) out[i + j] = piece[j];
  }
}

// An item is one vector of VEC elements (interleaved: VEC / 2 pairs) or the vector of first
// halves with its partner rot/2 further on (half layout: VEC pairs).
template <typename T, int VEC, bool INTERLEAVED>
struct RotItem {
  using V = Vec<T, VEC>;
  static constexpr int kPairs = INTERLEAVED ? VEC / 2 : VEC;
  V a, b;

  __device__ __forceinline__ void load(const T* p, int half) {
    a = *reinterpret_cast<const V*>(p);
    if constexpr (!INTERLEAVED) b = *reinterpret_cast<const V*>(p + half);
  }
  // Keeps the vectors as they were loaded until here: converted as soon as they arrive, four items
  // of bf16 held 116 registers where they need 60.
  __device__ __forceinline__ void pin() {
    pin(a);
    if constexpr (!INTERLEAVED) pin(b);
  }
  static __device__ __forceinline__ void pin(V& v) {
    if constexpr (sizeof(V) % 4 == 0) {
      uint32_t* const w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
      for (int i = 0; i < int(sizeof(V) / 4); ++i) asm volatile("" : "+r"(w[i]));
    }
  }
  __device__ __forceinline__ void rotate(const float (&c)[kPairs], const float (&s)[kPairs]) {
    float x[VEC], y[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = Elem<T>::to_f(a.v[i]);
    if constexpr (INTERLEAVED) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const float u = x[2 * i], v = x[2 * i + 1];
        y[2 * i] = u * c[i] - v * s[i];
        y[2 * i + 1] = v * c[i] + u * s[i];
      }
      a = pack_f<T, VEC>(y);
    } else {
      float z[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float v = Elem<T>::to_f(b.v[i]);
        y[i] = x[i] * c[i] - v * s[i];
        z[i] = v * c[i] + x[i] * s[i];
      }
      a = pack_f<T, VEC>(y);
      b = pack_f<T, VEC>(z);
    }
  }
  __device__ __forceinline__ void store(T* p, int half) const {
    *reinterpret_cast<V*>(p) = a;
    if constexpr (!INTERLEAVED) *reinterpret_cast<V*>(p + half) = b;
  }
};

// Vectors a head has to rotate, and where vector v starts in the head and in the table's halves.
template <int VEC, bool INTERLEAVED>
__host__ __device__ constexpr int rot_vectors(int rot) {
  return INTERLEAVED ? rot / VEC : rot / (2 * VEC);
}

// Heads of one token: q heads first, then k heads.
template <typename T>
struct TokenHeads {
  T* q;
  T* k;
  int num_q, num_k;
  int64_t q_head, k_head;
  __device__ __forceinline__ T* head(int h) const {
    return h < num_q ? q + int64_t(h) * q_head : k + int64_t(h - num_q) * k_head;
  }
};

// Rotates vectors first + lane + 32 j, j < ITEMS, of a token in place.  `row()` gives the token's
// table row after the loads have been issued, or null to leave the heads untouched.
template <typename T, typename C, int VEC, bool INTERLEAVED, int ITEMS, typename Row>
__device__ __forceinline__ void rotate_unit(const TokenHeads<T>& t, int first, int rot, Row row) {
  using Item = RotItem<T, VEC, INTERLEAVED>;
  const int half = rot / 2;
  const int per_head = rot_vectors<VEC, INTERLEAVED>(rot);
  const int total = (t.num_q + t.num_k) * per_head;
  // lane l's vectors all sit at one offset of their heads when the vectors a head divide 32: one
  // table entry serves them all, and no vector needs a division
  const bool shared = (per_head & (per_head - 1)) == 0 && per_head <= 32;
  const int shift = 31 - __clz(per_head);
  const int i = first + (threadIdx.x & 31);
  Item item[ITEMS];
  T* at[ITEMS];
  int off[ITEMS];
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const int v = i + 32 * j;
    const int h = shared ? v >> shift : v / per_head;
    off[j] = (v - h * per_head) * VEC;
    at[j] = t.head(h) + off[j];
    if (v < total) item[j].load(at[j], half);
  }
  const C* const cs = row();
  if (cs == nullptr) return;
  float c[Item::kPairs], s[Item::kPairs];
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    if (i + 32 * j >= total) break;
    if (j == 0 || !shared) {
      const int e = INTERLEAVED ? off[j] / 2 : off[j];
      load_table<C, Item::kPairs>(cs + e, c);
      load_table<C, Item::kPairs>(cs + half + e, s);
    }
    item[j].pin();
    item[j].rotate(c, s);
    item[j].store(at[j], half);
  }
}

}  // namespace
}  // namespace ntb200
