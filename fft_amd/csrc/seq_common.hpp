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

// N consecutive elements. The copies go through memcpy: the elements' addresses are multiples of the element size
// only (a row of 770 halves, a slice at an odd offset), and gfx950 loads and stores dwords at any address.
template <class T, int N>
struct Run {
  T v[N];
};
template <class T, int N>
__device__ __forceinline__ Run<T, N> load_run(const T* p) {
  Run<T, N> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
template <class T, int N>
__device__ __forceinline__ void store_run(T* p, const Run<T, N>& r) {
  __builtin_memcpy(p, &r, sizeof(r));
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
