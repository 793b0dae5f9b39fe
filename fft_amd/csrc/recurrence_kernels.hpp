// What the kernels of the gated linear recurrence share (recurrence_rows.hip, recurrence_signals.hip) and their plans.
//
// A stretch of steps maps the state before it to the state behind it by h -> A h + B, A the product of its decays and B
// the state it reaches from zero; two stretches join to (A2 A1, A2 B1 + B2). A workgroup holds a chunk of the
// time axis in registers, reads every value once, forms (A, B) of its pieces, gets the state before its chunk from the
// workgroups of earlier chunks, and walks its steps once more from there to write the results. The second walk multiplies as
// the definition does; only the states between pieces come from joined maps.
//
// The state travels between workgroups in 64-bit words, the fp32 value below and 1 above, written and read by single
// relaxed device-scope atomics on words that a kernel of the same call has zeroed: a word with the upper half set is
// complete, so no fence (on this chip a write-back of the whole L2) is needed. Chunks are taken by a ticket in the order in
// which they depend on each other: whatever a workgroup waits for has been taken before it by a workgroup that is already
// running and waits for still earlier ones only, so every wait ends. The order of all sums is fixed by the sizes.
#pragma once
#include "seq_common.hpp"

namespace tfft_seq {

using word = unsigned long long;

struct Chunking {
  long long tiles = 0;   // rows: groups of channels; signals: groups of rows
  long long chunks = 0;  // of the time axis
  int waves = 0;         // of a workgroup
  int group = 1;         // chunks whose (A, B) are joined directly; the state behind each group is handed on
  int lanes = 64;        // signals: threads of a row, where a wave holds several rows
  long long state_words = 0;  // words of one chunk
  long long words() const {  // the ticket, two words a state and chunk where groups are used, one a state and group
    return chunks <= 1 ? 0 : 1 + state_words * ((group > 1 ? 2 * chunks : 0) + (chunks + group - 1) / group);
  }
};

__device__ __forceinline__ void publish(word* at, float v) {
  __hip_atomic_store(at, (1ull << 32) | __float_as_uint(v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ word peek(const word* at) {
  return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float await(const word* at) {
  word w = peek(at);
  while (!(w >> 32)) {
    __builtin_amdgcn_s_sleep(1);
    w = peek(at);
  }
  return __uint_as_float((unsigned)w);
}

// A h + B; a state of zero stays out of a product that may have overflowed
__device__ __forceinline__ float join(float A, float h, float B) { return h != 0.0f ? fmaf(A, h, B) : B; }

__device__ __forceinline__ int steps_of(const int* lengths, long long b, int length) {
  if (!lengths) return length;
  const int n = lengths[b];
  return n < 0 ? 0 : n < length ? n : length;
}

// launchers; the plans are made from the settled arguments (a stride of an extent of one is 0 or 1)
bool rows_vector(const tfft_scan_args& p);
bool rows_vector(const tfft_scan_grad_args& p);
Chunking plan_rows(const tfft_scan_args& p);
Chunking plan_rows(const tfft_scan_grad_args& p);
bool rows_sums_shares(const tfft_scan_grad_args& p);
void launch_rows(const tfft_scan_args& p, const Chunking& c, word* words, hipStream_t s);
void launch_rows(const tfft_scan_grad_args& p, const Chunking& c, word* words, float* parts, hipStream_t s);

bool signals_fit(const tfft_scan_args& p);
bool signals_fit(const tfft_scan_grad_args& p);
Chunking plan_signals(const tfft_scan_args& p);
Chunking plan_signals(const tfft_scan_grad_args& p);
void launch_signals(const tfft_scan_args& p, const Chunking& c, word* words, hipStream_t s);
void launch_signals(const tfft_scan_grad_args& p, const Chunking& c, word* words, hipStream_t s);

// f(T(), G()) for the element types of a call
template <class F>
void with_types(int dtype, int gate_dtype, F f) {
  if (dtype == TFFT_F32) f(float(), float());
  else if (dtype == TFFT_F16 && gate_dtype == TFFT_F32) f(f16(), float());
  else if (dtype == TFFT_F16) f(f16(), f16());
  else if (gate_dtype == TFFT_F32) f(bf16(), float());
  else f(bf16(), bf16());
}

}  // namespace tfft_seq
