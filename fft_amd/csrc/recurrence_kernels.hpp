// What the kernels of the gated linear recurrence share (recurrence_rows.hip, recurrence_signals.hip) and their plans.
//
// A stretch of steps maps the state before it to the state behind it by h -> A h + B, A the product of its decays and B
// the state it reaches from zero; two stretches join to (A2 A1, A2 B1 + B2). A workgroup holds a chunk of the
// time axis in registers, reads every value once, forms (A, B) of its pieces, gets the state before its chunk from the
// workgroups of earlier chunks, and walks its steps once more from there to write the results. The second walk multiplies as
// the definition does; only the states between pieces come from joined maps.
//
// States and maps travel between workgroups in single words that a kernel of the same call has zeroed, written and read by
// relaxed device-scope atomics: (A, B) as two fp32 in 64 bits, a state as one fp32 in 32 bits, a zero among them written as -0.0
// (in A, where the sign of a zero does not show), so that a word with a bit set is there and complete and no fence (on this chip
// a write-back of a whole L2) is needed. Workgroups take chunks by tickets, in the order in which chunks depend on each
// other: whoever holds the smallest ticket of a counter that is not done waits for nothing that is not there, so every wait
// ends. The order of all sums is fixed by the sizes.
//
// Each of the eight XCDs has a counter of its own, with all chunks of an eighth of the tiles, neighbours beside each other (workgroups
// go round the XCDs): an XCD then reads whole rows, and lines that two tiles share once. B = 8, L = 4096 with D = 2048: 103 us forward
// and 170 back, where the XCDs take every eighth tile 106 and 182; with D = 2050 125 and 222 against 142 and 258. With fewer than
// kManyTiles tiles an eighth is too narrow, and all take from one counter, chunk by chunk: 65537 x 1152 (9 tiles) 93 us against
// 134 with eight. In a padded batch an XCD has a strip of every entry instead, or the one with the longest sequences would be
// the last to end: 8 entries of 1024 channels, one of 16384 steps and seven of 1000, 114 us forward and 204 back against 170 and 291.
#pragma once
#include "seq_common.hpp"

namespace tfft_seq {

using word = unsigned long long;

constexpr int kManyTiles = 32, kCounterWords = 16;  // a counter has a cache line of its own

struct Chunking {
  long long tiles = 0;   // rows: groups of channels; signals: groups of rows
  long long chunks = 0;  // of the time axis
  int waves = 0;         // of a workgroup
  int group = 1;         // chunks whose (A, B) are joined directly
  int row = 1;           // groups whose (A, B) are joined directly; the state behind each row of groups is handed on
  int lanes = 64;        // rows: lanes that a tile fills; signals: threads of a row, where a wave holds several rows
  int each = 1;          // signals: rows of a gate that a workgroup takes one after the other
  int side_by_side = 1;  // tiles that a workgroup holds at once; more than one only where a tile is one chunk
  bool walks = false;    // a workgroup takes all chunks of its tile, one after the other
  long long state_words = 0;  // states of one chunk
  // 64-bit words: the counters, a map a state and chunk where groups are used and a group where rows of them are, half a word a
  // state and row
  long long words() const {
    if (apart() <= 1 || tiles == 0) return 0;
    const long long groups = (chunks + group - 1) / group, rows = (groups + row - 1) / row;
    return kCounterWords * counters() + state_words * ((group > 1 ? chunks : 0) + (row > 1 ? groups : 0)) + (state_words * rows + 1) / 2;
  }
  long long apart() const { return walks ? 1 : chunks; }  // chunks that workgroups of their own take
  long long strip = 0;  // neighbouring tiles of a counter, 0: an eighth of all
  int counters() const { return tiles >= kManyTiles ? 8 : 1; }
  long long width() const { return strip && counters() > 1 ? strip : (tiles + counters() - 1) / counters(); }
  // workgroups: as many for every counter as the first one has tickets; a few find none left
  long long blocks() const {
    if (apart() <= 1 || tiles == 0) return (tiles + side_by_side - 1) / side_by_side;
    const long long round = counters() * width(), rest = tiles % round;
    return counters() * (tiles / round * width() + (rest < width() ? rest : width())) * chunks;
  }
};

// Tile and chunk of this workgroup, the same for all threads; false where there is none left. `shared` lies in LDS.
struct Turns {
  unsigned tiles, counters, chunks, width;
};
inline Turns turns_of(const Chunking& c) {
  return Turns{(unsigned)c.tiles, (unsigned)c.counters(), (unsigned)c.apart(), (unsigned)c.width()};
}
__device__ __forceinline__ bool take_turn(const Turns& f, word* words, unsigned* shared, unsigned* tile, unsigned* chunk) {
  if (f.chunks <= 1) {
    *tile = blockIdx.x, *chunk = 0;
    return true;
  }
  const unsigned counter = blockIdx.x % f.counters;
  if (threadIdx.x == 0)
    *shared = (unsigned)__hip_atomic_fetch_add(words + kCounterWords * counter, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  const unsigned ticket = __builtin_amdgcn_readfirstlane(*shared);
  const unsigned round = f.counters * f.width, before = counter * f.width, rest = f.tiles % round;
  const unsigned mine = f.tiles / round * f.width + min(rest > before ? rest - before : 0u, f.width);
  if (mine == 0) return false;
  *chunk = __builtin_amdgcn_readfirstlane(ticket / mine);
  const unsigned i = ticket - *chunk * mine;
  *tile = i / f.width * round + before + i % f.width;
  return *chunk < f.chunks;
}

__device__ __forceinline__ void publish_map(word* at, float A, float B) {
  const unsigned a = __float_as_uint(A);
  __hip_atomic_store(at, (word)(a ? a : 0x80000000u) << 32 | __float_as_uint(B), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void publish_state(unsigned* at, float h) {
  const unsigned v = __float_as_uint(h);
  __hip_atomic_store(at, v ? v : 0x80000000u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <class W>
__device__ __forceinline__ W peek(const W* at) {
  return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <class W>
__device__ __forceinline__ W await(const W* at) {
  W w = peek(at);
  while (!w) {
    __builtin_amdgcn_s_sleep(1);
    w = peek(at);
  }
  return w;
}
__device__ __forceinline__ float map_a(word w) { return __uint_as_float((unsigned)(w >> 32)); }
__device__ __forceinline__ float map_b(word w) { return __uint_as_float((unsigned)w); }
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
unsigned long long rows_parts(const tfft_scan_grad_args& p);  // fp32 words behind the others, for gates that many channels share
void launch_rows(const tfft_scan_args& p, const Chunking& c, word* words, hipStream_t s);
void launch_rows(const tfft_scan_grad_args& p, const Chunking& c, word* words, float* parts, hipStream_t s);

bool signals_fit(const tfft_scan_args& p);
bool signals_fit(const tfft_scan_grad_args& p);
Chunking plan_signals(const tfft_scan_args& p);
Chunking plan_signals(const tfft_scan_grad_args& p);
void launch_signals(const tfft_scan_args& p, const Chunking& c, word* words, hipStream_t s);
unsigned long long signals_parts(const tfft_scan_grad_args& p);
void launch_signals(const tfft_scan_grad_args& p, const Chunking& c, word* words, float* parts, hipStream_t s);

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
