// Element types of the sequence operators (single, bfloat16 and half precision) and their vector loads and stores.
#pragma once
#include "common.h"

namespace atlhip {

enum DType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };
using bf16_t = __bf16;
using f16_t = _Float16;

inline int dtype_size(int t) { return t == kF32 ? 4 : 2; }
inline bool dtype_ok(int t) { return t == kF32 || t == kBF16 || t == kF16; }
inline bool aligned_to(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

// V elements that move as one access (2 to 32 bytes, aligned to their size up to 16).
template <typename T, int V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Pack {
  T e[V];
};

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  return *reinterpret_cast<const Pack<T, V>*>(p);
}

// The same where a piece is aligned to its elements only (global memory takes that), of its first n elements; the others
// read as zero and are not written.
template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) LoosePack {
  T e[V];
};
template <int V, typename T>
__device__ __forceinline__ void load_loose(const T* p, int64_t n, float (&v)[V]) {
  if (n >= V) {
    const LoosePack<T, V> r = *reinterpret_cast<const LoosePack<T, V>*>(p);
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = (float)r.e[k];
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = k < n ? (float)p[k] : 0.f;
  }
}
template <int V, typename T>
__device__ __forceinline__ void store_loose(T* p, int64_t n, const float (&v)[V]) {
  if (n >= V) {
    LoosePack<T, V> r;
#pragma unroll
    for (int k = 0; k < V; ++k) r.e[k] = (T)v[k];
    *reinterpret_cast<LoosePack<T, V>*>(p) = r;
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k < n) p[k] = (T)v[k];
  }
}

template <int V, typename T>
__device__ __forceinline__ void load_f(const T* p, float (&v)[V]) {
  const Pack<T, V> r = load_pack<T, V>(p);
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] = (float)r.e[k];
}

// Rounds to nearest, ties to even.
template <int V, typename T>
__device__ __forceinline__ void store_f(T* p, const float (&v)[V]) {
  Pack<T, V> r;
#pragma unroll
  for (int k = 0; k < V; ++k) r.e[k] = (T)v[k];
  *reinterpret_cast<Pack<T, V>*>(p) = r;
}

// f(first, n): n of a call's workgroups (of at most `threads` threads) from the first on.  A launch takes fewer than 2^32
// threads in a direction, so a call of more is several launches.
template <typename F>
void in_launches(int64_t blocks, F&& f, int threads = kBlock) {
  const int64_t most = ((int64_t)1 << 31) / threads;
  for (int64_t first = 0; first < blocks; first += most) f(first, (unsigned)(blocks - first < most ? blocks - first : most));
}

// Smallest power of two >= n (n >= 1).
inline int ceil_pow2(int64_t n) {
  int p = 1;
  while (p < n) p <<= 1;
  return p;
}

}  // namespace atlhip
