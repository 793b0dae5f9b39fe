// Element access of the sequence operators (recurrence.hip, rotary.hip): storage types and their conversions, runs of
// consecutive elements that need not be aligned to more than an element, argument checks of the C entry points.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstdio>

#include "../../include/thunderfft_c.h"

extern "C" int tfft_internal_fail(int code, const char* message);
extern "C" int tfft_internal_finish(void* stream);

namespace tfft_seq {

using f16 = _Float16;
using bf16 = __bf16;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(f16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(bf16 v) { return (float)v; }
template <class T>
__device__ __forceinline__ T from_f32(float v) {
  return (T)v;  // round to nearest even, the one rounding of an output
}

// exp of a log decay: one product and the chip's 2^x. Off by one unit in the last place of 2^x and by |x| 1.3 half units
// of the rounded product and factor, which a decay worth keeping (|x| below 20) does not notice; it takes 5 issue slots where expf takes
// more than 20, and the scan's vector units are as busy as its memory.
__device__ __forceinline__ float exp_decay(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f); }

// A pointer to device memory from an address of which the compiler no longer sees where it came from, else it takes the flat
// loads and stores that could reach LDS too: those wait for LDS and the other way round, and take 64-bit addresses in vector registers.
template <class T>
__device__ __forceinline__ T* device_pointer(uint64_t base, uint64_t off = 0) {
  using Bytes = __attribute__((address_space(1))) char*;
  return (T*)(char*)((Bytes)base + off);
}

// N consecutive elements, 16-bit ones two to a register. The copies go through memcpy: the elements' addresses are multiples
// of the element size only (a row of 770 halves, a slice at an odd offset), and gfx950 loads and stores dwords at any
// address.
template <class T, int N>
struct Run {
  static constexpr bool kHalf = sizeof(T) == 2;
  uint32_t w[kHalf ? (N + 1) / 2 : N];
  __device__ __forceinline__ float get(int i) const {
    if constexpr (!kHalf) {
      return __uint_as_float(w[i]);
    } else {
      const uint16_t bits = (uint16_t)(w[i / 2] >> (i % 2 * 16));
      T v;
      __builtin_memcpy(&v, &bits, 2);
      return (float)v;
    }
  }
  // element i of an array filled in ascending order, rounded to nearest even: the one rounding of an output
  __device__ __forceinline__ void set(int i, float f) {
    const T v = (T)f;
    if constexpr (!kHalf) {
      w[i] = __float_as_uint(v);
    } else {
      uint16_t bits;
      __builtin_memcpy(&bits, &v, 2);
      if (i % 2 == 0) w[i / 2] = bits;
      else w[i / 2] |= (uint32_t)bits << 16;
    }
  }
  // elements 2 i and 2 i + 1, in one conversion where the chip has one
  __device__ __forceinline__ void set_pair(int i, float f0, float f1) {
    if constexpr (!kHalf) {
      w[2 * i] = __float_as_uint(f0), w[2 * i + 1] = __float_as_uint(f1);
    } else {
      using Two = T __attribute__((ext_vector_type(2)));
      using Floats = float __attribute__((ext_vector_type(2)));
      const Two two = __builtin_convertvector((Floats){f0, f1}, Two);
      __builtin_memcpy(&w[i], &two, 4);
    }
  }
  // all elements
  __device__ __forceinline__ void set_all(const float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) set_pair(i, f[2 * i], f[2 * i + 1]);
    if constexpr (N % 2) set(N - 1, f[N - 1]);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (uint32_t& word : w) word = 0;
  }
};
// STREAM: data that passes through the chip once and in whole cache lines, at addresses that are multiples of the run's size.
// Such loads and stores do not push other data out of the L2 and are faster for it (figures at the kernels); where several
// waves share a line it costs a second fetch instead.
template <class T, int N, bool STREAM = false>
__device__ __forceinline__ Run<T, N> load_run(const T* p) {
  Run<T, N> r;
  if constexpr (STREAM) {
    using Words = uint32_t __attribute__((ext_vector_type(sizeof(r.w) / 4)));
    const Words w = __builtin_nontemporal_load((const Words*)p);
    __builtin_memcpy(r.w, &w, sizeof(r.w));
  } else {
    if constexpr (sizeof(r) != N * sizeof(T)) r.clear();
    __builtin_memcpy(r.w, p, N * sizeof(T));
  }
  return r;
}
template <class T, int N, bool STREAM = false>
__device__ __forceinline__ void store_run(T* p, const Run<T, N>& r) {
  if constexpr (STREAM) {
    using Words = uint32_t __attribute__((ext_vector_type(sizeof(r.w) / 4)));
    Words w;
    __builtin_memcpy(&w, r.w, sizeof(r.w));
    __builtin_nontemporal_store(w, (Words*)p);
  } else {
    __builtin_memcpy(p, r.w, N * sizeof(T));
  }
}
// Rows of whole cache lines: the address and every stride that is used are multiples of 128 bytes
template <int n>
bool whole_lines(const void* p, int dtype, const long long (&stride)[n], const long long (&extent)[n]) {
  const long long size = dtype == TFFT_F32 ? 4 : 2;
  bool whole = (reinterpret_cast<uintptr_t>(p) & 127u) == 0;
  for (int i = 0; i < n; ++i) whole = whole && (extent[i] <= 1 || stride[i] * size % 128 == 0);
  return whole;
}

// The first `valid` of N elements, zeros behind them
template <int N, class T>
__device__ __forceinline__ Run<T, N> load_some(const T* p, int valid) {
  if (valid == N) return load_run<T, N>(p);
  Run<T, N> r;
  r.clear();
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < valid) {
      const Run<T, 1> one = load_run<T, 1>(p + i);
      if constexpr (sizeof(T) == 4) r.w[i] = one.w[0];
      else r.w[i / 2] |= one.w[0] << (i % 2 * 16);
    }
  return r;
}
template <int N, class T>
__device__ __forceinline__ void store_some(T* p, const Run<T, N>& r, int valid) {
  if (valid == N) return store_run<T, N>(p, r);
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < valid) {
      Run<T, 1> one;
      if constexpr (sizeof(T) == 4) one.w[0] = r.w[i];
      else one.w[0] = r.w[i / 2] >> (i % 2 * 16);
      store_run<T, 1>(p + i, one);
    }
}

// Moves the elements of a run `by` places to its front
template <int E, class T>
__device__ __forceinline__ void move_down(Run<T, E>& r, int by) {
  if (__all(by == 0)) return;
  constexpr int kWords = sizeof(r.w) / 4, kElements = 4 / sizeof(T);
#pragma unroll
  for (int m = kWords; m >= 1; m /= 2) {
    const bool move = by / kElements & m;
#pragma unroll
    for (int i = 0; i < kWords; ++i) r.w[i] = move ? (i + m < kWords ? r.w[i + m] : 0u) : r.w[i];
  }
  if constexpr (kElements == 2) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) r.w[i] = by & 1 ? r.w[i] >> 16 | (i + 1 < kWords ? r.w[i + 1] << 16 : 0u) : r.w[i];
  }
}
// The first `valid` of E elements, fewer than E: halves, quarters and so on as the bits of `valid` say, what follows moved down
template <int N, class T, int E>
__device__ __forceinline__ void store_head(T* p, Run<T, E> r, int valid) {
  if constexpr (N > 1) {
    constexpr int kWords = N / 2 * sizeof(T) / 4;  // of the half; 0: half a word
    if (valid & (N / 2)) {
      if constexpr (kWords == 0) {
        Run<T, 1> one;
        one.w[0] = r.w[0];
        store_run<T, 1>(p, one);
      } else {
        __builtin_memcpy(p, r.w, 4 * kWords);
#pragma unroll
        for (int i = 0; i < kWords; ++i) r.w[i] = r.w[i + kWords];
      }
      p += N / 2;
    }
    store_head<N / 2>(p, r, valid);
  }
}
inline bool misaligned(const void* p, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & (dtype == TFFT_F32 ? 3u : 1u)) != 0;
}

// What is wrong with a tensor of n dimensions, if anything. An output's elements may not overlap: every dimension has
// to step over all that the ones with smaller strides reach.
template <int n>
const char* check_tensor(const void* data, int dtype, const long long (&stride_in)[n], const long long (&extent_in)[n], bool output) {
  long long stride[n], extent[n];
  for (int i = 0; i < n; ++i) {
    if (extent_in[i] == 0) return nullptr;
    stride[i] = stride_in[i], extent[i] = extent_in[i];
  }
  if (!data || misaligned(data, dtype)) return "null or misaligned pointer";
  __int128 reach = 0;
  for (int i = 0; i < n; ++i) {
    if (extent[i] > 1 && stride[i] < 0) return "negative stride";
    reach += (__int128)(extent[i] - 1) * stride[i];
  }
  if (reach >= ((__int128)1 << 60)) return "strides that leave the address space";
  if (!output) return nullptr;
  for (int i = 0; i < n; ++i)
    for (int j = i + 1; j < n; ++j)
      if (stride[j] < stride[i]) {
        const long long s = stride[i], e = extent[i];
        stride[i] = stride[j], extent[i] = extent[j], stride[j] = s, extent[j] = e;
      }
  reach = 0;
  for (int i = 0; i < n; ++i) {
    if (extent[i] == 1) continue;
    if (stride[i] <= reach) return "an output's elements overlap";
    reach += (__int128)(extent[i] - 1) * stride[i];
  }
  return nullptr;
}

}  // namespace tfft_seq
