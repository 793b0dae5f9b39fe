// The gated linear recurrence where neighbouring steps lie side by side: the convolution's signals [batch][channel]
// [time].
#include <algorithm>
#include <type_traits>

#include "recurrence_kernels.hpp"

namespace tfft_seq {
namespace {

// A thread holds E consecutive steps of one row (batch entry, channel). Rows of up to 64 E steps: the next power of two
// of lanes, several rows a wave. Longer rows: one a workgroup, in chunks of up to kMaxWaves waves. Pieces are joined within a
// wave by exchanges over 1, 2, 4 ... lanes, then over the waves through LDS.
//
// What bounds it: HBM. B = 64, D = 768, L = 4096 in fp16 takes 200 us forward (1208 MB, 6.0 TB/s) and 340 back (5.9), the same
// in chunks of 1024, 128 steps; in fp32 32 bytes a thread are 5 % faster than 64 (four accesses to a line, not two). Few long
// rows do not fill the chip as evenly: 16 signals of 1048573 steps in fp32 back 82 us (335 MB, 4.1 TB/s). Rows at odd addresses
// cost up to a quarter (L = 4095 in bf16 123 us against 103).
constexpr int kMaxGroup = 64;
// Longer rows that are many are walked by a workgroup each, chunk after chunk, few rows are split: 256 x 20000 in bf16 takes 11 us
// walked against 13 split, 256 x 100000 in fp32 65 against 69, 16 x 2^20 47 split (16 workgroups would walk). Back in 16 bits
// a few hundred workgroups, two on some CUs and one on the others, last longer: 294 x 52347 in bf16 61 us walked against 39
// split, 500 x 60000 71 against 64 (in fp32 300 x 30000 43 against 46). From kShortChunks
// rows on the workgroups have 4 waves, and several of a CU load, wait and store at different times: 49152 x 8200 in bf16 449 us
// forward and 769 back against 657 and 1351 with 8 waves; with 256 rows they are too few, 96 and 125 us against 65 and 110.
constexpr int kManyRows = 256, kManyRowsBack = 512, kShortChunks = 1024, kWalkWaves = 4;
// Rows of a shared gate that a workgroup takes one after the other: up to kEach, or kEachOfFew where that leaves fewer than
// kFewGroups workgroups. [8, 2048, 4096] in bf16 with 64 channels a gate takes 110, 101, 99, 108 us back with 4, 8, 16, 64 rows (209 with
// every row's terms in memory), [2, 768, 4096] 19, 22, 33, 103.
constexpr int kEach = 8, kEachOfFew = 4, kFewGroups = 1024;
enum { ONE, WALK, SPLIT };  // one chunk, or chunks after one another, or apart
template <class T>
constexpr int kSteps = 32 / sizeof(T);
template <class T>
constexpr int kMaxWaves = 4 * sizeof(T);  // chunks of 8192 steps

struct Shape {
  long long rows;
  int length, channels, share, log_gate;
  int chunks, group, lanes, each;
  Turns turns;
  word* words;
};

// Asks for E steps from t0 on. A piece that reaches over the end of the row is asked for as the row's last E steps, so that all
// threads load whole runs on one path; line_up() then moves its steps to where they belong. Rows shorter than a piece are loaded
// step by step.
template <int E, class T>
__device__ __forceinline__ Run<T, E> ask(const T* p, int t0, int length) {
  if (length < E) return load_some<E>(p, t0 == 0 ? length : 0);
  return load_run<T, E>(p + max(min(t0, length - E), 0));
}
template <int E, class G>
__device__ __forceinline__ Run<G, E> one(const G* p) {
  const uint32_t v = load_run<G, 1>(p).w[0];
  Run<G, E> r;
#pragma unroll
  for (uint32_t& w : r.w) w = sizeof(G) == 4 ? v : v | v << 16;
  return r;
}
template <int E, class T>
__device__ __forceinline__ void line_up(Run<T, E>& r, int t0, int length) {
  const int by = length < E ? 0 : min(max(t0 - (length - E), 0), E);  // steps that the run starts too early
  move_down<E>(r, by);
}
// STREAM: as in load_run. Two stores share a line here, which costs a row in one workgroup 1 to 8 %, but where chunks are taken apart the
// states come through faster: two entries of 8 signals of 1048573 steps in fp32 take 47 us forward and 74 back against 53 and 90 (outputs in the last-level cache).
template <int E, bool STREAM, class T>
__device__ __forceinline__ void store_steps(T* p, int t0, int length, const Run<T, E>& r) {
  const int valid = min(max(length - t0, 0), E);
  if (valid == E) {
    using Words = uint32_t __attribute__((ext_vector_type(4), aligned(2)));  // 16 bytes, or the compiler cuts them up otherwise
#pragma unroll
    for (int i = 0; i < (int)sizeof(r.w) / 4; i += 4) {
      const Words w = {r.w[i], r.w[i + 1], r.w[i + 2], r.w[i + 3]};
      if (STREAM) __builtin_nontemporal_store(w, (Words*)(p + t0) + i / 4);
      else ((Words*)(p + t0))[i / 4] = w;
    }
  } else {
    store_head<E>(p + t0, r, valid);
  }
}

// Decays of E steps that were asked for; 1 behind the sequence. time is 1, or 0 for one decay throughout.
template <int E, class G>
__device__ __forceinline__ void take_decays(Run<G, E>& r, long long time, int t0, int len, int length, int log_gate, float (&a)[E]) {
  if (time) line_up<E>(r, t0, length);
#pragma unroll
  for (int i = 0; i < E; ++i) a[i] = r.get(i);
  if (log_gate) {
#pragma unroll
    for (int i = 0; i < E; ++i) a[i] = exp_decay(a[i]);
  }
  if (!__all(t0 + E <= len)) {
#pragma unroll
    for (int i = 0; i < E; ++i) a[i] = t0 + i < len ? a[i] : 1.0f;
  }
}
// Values of E steps that were asked for; 0 from step len - t0 on
template <int E, class T>
__device__ __forceinline__ void take(Run<T, E>& r, int t0, int len, int length) {
  line_up<E>(r, t0, length);
  if (__all(t0 + E <= len)) return;
  constexpr int kElements = 4 / sizeof(T);
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (t0 + i >= len) r.w[i / kElements] &= kElements == 1 ? 0u : i % 2 == 0 ? 0xffff0000u : 0x0000ffffu;
}

// (A, B) of all pieces up to and with this thread's, among `width` threads that follow one another (a power of two,
// or a whole wave), then those in front of it
__device__ __forceinline__ void scan_lanes(int lane, int width, float& A, float& B, float& front_a, float& front_b) {
  const int i = lane & (width - 1);
  for (int d = 1; d < width; d *= 2) {
    const float a = __shfl_up(A, d), b = __shfl_up(B, d);
    if (i >= d) {
      B = join(A, b, B);
      A *= a;
    }
  }
  front_a = __shfl_up(A, 1), front_b = __shfl_up(B, 1);
  if (i == 0) front_a = 1.0f, front_b = 0.0f;
}

struct Lds {
  float A[16], B[16], h;
  unsigned ticket;
};

// The state in front of this thread's piece from its (A, B) and `h`, the state in front of the chunk, or where chunks are taken
// apart of the first one. `order`: 0 for the thread that comes first.
template <int MODE>
__device__ __forceinline__ float state_in_front(const Shape& f, Lds& lds, unsigned chunk, long long row, int order, float A, float B, float h) {
  const int lane = order & 63, wave = order >> 6, waves = blockDim.x >> 6;
  float front_a, front_b;
  scan_lanes(lane, f.lanes, A, B, front_a, front_b);
  if (f.lanes < 64 || (MODE == ONE && waves == 1)) return join(front_a, h, front_b);
  if (lane == 63) lds.A[wave] = A, lds.B[wave] = B;
  __syncthreads();
  float wave_a = 1.0f, wave_b = 0.0f;
  for (int w = 0; w < wave; ++w) {
    wave_b = join(lds.A[w], wave_b, lds.B[w]);
    wave_a *= lds.A[w];
  }
  if constexpr (MODE == SPLIT) {
    if (wave == waves - 1) {
      const int r = chunk % f.group, q = chunk / f.group;
      const bool more = chunk + 1 < (unsigned)f.chunks;
      word* maps = f.words + kCounterWords * f.turns.counters;
      word* own = maps + row * f.chunks + chunk;
      unsigned* states = (unsigned*)(maps + f.rows * f.chunks) + row * ((f.chunks + f.group - 1) / f.group);
      const float chunk_a = wave_a * lds.A[wave], chunk_b = join(lds.A[wave], wave_b, lds.B[wave]);
      if (more && r != f.group - 1 && lane == 0) publish_map(own, chunk_a, chunk_b);
      // lane k joins the k-th chunk of the group, those of this one's past are read together
      float a = 1.0f, b = 0.0f, fa, fb;
      if (lane < r) {
        const word w = await(own - (r - lane));
        a = map_a(w), b = map_b(w);
      }
      scan_lanes(lane, 64, a, b, fa, fb);
      a = __shfl(a, 63), b = __shfl(b, 63);
      if (q > 0) h = __uint_as_float(await(states + q - 1));
      h = join(a, h, b);
      if (more && r == f.group - 1 && lane == 0) publish_state(states + q, join(chunk_a, h, chunk_b));
      if (lane == 0) lds.h = h;
    }
    __syncthreads();
    h = lds.h;
  }
  h = join(wave_a, h, wave_b);
  return join(front_a, h, front_b);
}

// Row of this thread, and its chunk where chunks are taken apart
template <int MODE>
__device__ __forceinline__ bool take(const Shape& f, Lds& lds, long long* row, unsigned* chunk) {
  *chunk = 0;
  if constexpr (MODE == SPLIT) {
    unsigned tile;
    const bool there = take_turn(f.turns, f.words, &lds.ticket, &tile, chunk);
    *row = tile;
    return there;
  } else {
    *row = f.lanes < 64 ? ((long long)blockIdx.x * blockDim.x + threadIdx.x) / f.lanes : (long long)blockIdx.x;
    return true;
  }
}

// The state behind the chunk, for all threads of a workgroup that walks on; it is the one of the thread that comes last
__device__ __forceinline__ float state_behind(Lds& lds, bool mine, float h) {
  if (mine) lds.h = h;
  __syncthreads();
  return lds.h;
}

template <class T, class G, int MODE>
__global__ __launch_bounds__(64 * kMaxWaves<T>) void scan_signals_fwd(tfft_scan_args p, Shape f) {
  constexpr int E = kSteps<T>;
  __shared__ Lds lds;
  long long row;
  unsigned chunk;
  if (!take<MODE>(f, lds, &row, &chunk)) return;
  const bool live = row < f.rows;
  if (!live) row = 0;
  const int b = (int)((unsigned)row / (unsigned)f.channels), c = (int)((unsigned)row - (unsigned)b * (unsigned)f.channels), len = live ? steps_of(p.lengths, b, f.length) : 0;
  const int order = threadIdx.x, piece = f.lanes < 64 ? order & (f.lanes - 1) : order;
  const int pieces = f.lanes < 64 ? f.lanes : (int)blockDim.x;
  const T* x = (const T*)p.x.data + b * p.x.batch + c * p.x.channel;
  const G* g = (const G*)p.gate.data + b * p.gate.batch + (c / f.share) * p.gate.channel;
  T* y = (T*)p.y.data + b * p.y.batch + c * p.y.channel;
  float start = p.initial ? p.initial[row] : 0.0f, h;
  while (true) {
    const int t0 = (int)(chunk * pieces + piece) * E;
    Run<T, E> xr;
    Run<G, E> gr;
    if (f.length > 0) {
      xr = ask<E>(x, t0, f.length);
      gr = p.gate.time ? ask<E>(g, t0, f.length) : one<E>(g);
    }
    take<E>(xr, t0, len, f.length);
    float a[E];
    take_decays<E>(gr, p.gate.time, t0, len, f.length, f.log_gate, a);
    float A = 1.0f, B = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      A *= a[i];
      B = fmaf(a[i], B, xr.get(i));
    }
    h = state_in_front<MODE>(f, lds, chunk, row, order, A, B, start);
    Run<T, E> r;
    float out[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      h = fmaf(a[i], h, xr.get(i));
      out[i] = t0 + i < len ? h : 0.0f;
    }
    r.set_all(out);
    if (live) store_steps<E, MODE == SPLIT>(y, t0, f.length, r);
    if (MODE != WALK || chunk + 1 == (unsigned)f.chunks) break;
    start = state_behind(lds, piece == pieces - 1, h);
    ++chunk;
  }
  if (p.last && live && chunk + 1 == (unsigned)f.chunks && piece == pieces - 1) p.last[row] = h;
}

// Backwards in time: the first thread has the latest steps, chunk 0 is the latest. SHARED: each channel's terms of dgate go to
// `parts` (fp32, [batch][channel] and rows of `pitch`), to be summed by a kernel behind. kWaves: of a SIMD; chunks taken apart wait
// for each other, and two workgroups a CU in fp32 (62 registers, where the compiler takes 74) hide that: 16 signals of 1048573 steps
// 86 -> 82 us, one of 2^24 83 -> 75; 5 waves in 16 bits 294 x 52347 52 -> 49. Whole rows lose 2 %, walked ones spill.
template <class T, int MODE>
constexpr int kWaves = MODE != SPLIT ? 1 : sizeof(T) == 4 ? 8 : 5;
template <class T, class G, int MODE, bool SHARED>
__global__ __launch_bounds__(64 * kMaxWaves<T>, (kWaves<T, MODE>)) void scan_signals_bwd(tfft_scan_grad_args p, Shape f, float* parts, long long pitch) {
  constexpr int E = kSteps<T>;
  __shared__ Lds lds;
  long long row;
  unsigned chunk;
  if (!take<MODE>(f, lds, &row, &chunk)) return;
  const bool live = row < f.rows;
  if (!live) row = 0;
  const int b = (int)((unsigned)row / (unsigned)f.channels), c = (int)((unsigned)row - (unsigned)b * (unsigned)f.channels), len = live ? steps_of(p.lengths, b, f.length) : 0;
  const int order = threadIdx.x, piece = f.lanes < 64 ? order & (f.lanes - 1) : order;
  const int pieces = f.lanes < 64 ? f.lanes : (int)blockDim.x;
  const T* dy = (const T*)p.dy.data + b * p.dy.batch + c * p.dy.channel;
  const T* y = (const T*)p.y.data + b * p.y.batch + c * p.y.channel;
  const G* g = (const G*)p.gate.data + b * p.gate.batch + (c / f.share) * p.gate.channel;
  const float initial = p.initial ? p.initial[row] : 0.0f;
  float start = p.dlast ? p.dlast[row] : 0.0f, k;
  while (true) {
    const int t0 = ((int)(f.chunks - 1 - chunk) * pieces + pieces - 1 - piece) * E;
    Run<T, E> d, own;
    Run<T, 1> before;
    Run<G, E> gr;
    if (f.length > 0) {
      d = ask<E>(dy, t0, f.length);
      gr = p.gate.time ? ask<E>(g, t0, f.length) : one<E>(g);
      own = ask<E>(y, t0, f.length);
      before = load_run<T, 1>(y + min(max(t0 - 1, 0), f.length - 1));
    }
    take<E>(d, t0, len, f.length);
    float a[E];
    take_decays<E>(gr, p.gate.time, t0, len, f.length, f.log_gate, a);
    float A = 1.0f, B = 0.0f;
#pragma unroll
    for (int i = E - 1; i >= 0; --i) {
      A *= a[i];
      B = a[i] * (B + d.get(i));
    }
    k = state_in_front<MODE>(f, lds, chunk, row, order, A, B, start);
    take<E>(own, t0, len, f.length);
    float dx[E], dgate[E];
#pragma unroll
    for (int i = E - 1; i >= 0; --i) {
      const float e = d.get(i) + k;
      const float state = i > 0 ? own.get(i > 0 ? i - 1 : 0) : t0 > 0 ? before.get(0) : initial;
      const bool inside = t0 + i < len;
      dgate[i] = inside ? e * state * (f.log_gate ? a[i] : 1.0f) : 0.0f;
      dx[i] = inside ? e : 0.0f;
      k = a[i] * e;
    }
    using Sum = std::conditional_t<SHARED, float, G>;
    Run<T, E> r;
    Run<Sum, E> q;
    r.set_all(dx), q.set_all(dgate);
    if (live) {
      store_steps<E, MODE == SPLIT>((T*)p.dx.data + b * p.dx.batch + c * p.dx.channel, t0, f.length, r);
      Sum* to;
      if constexpr (SHARED) to = parts + row * pitch;
      else to = (G*)p.dgate.data + b * p.dgate.batch + c * p.dgate.channel;
      store_steps<E, MODE == SPLIT && sizeof(Sum) == sizeof(T)>(to, t0, f.length, q);
    }
    if (MODE != WALK || chunk + 1 == (unsigned)f.chunks) break;
    start = state_behind(lds, piece == pieces - 1, k);
    ++chunk;
  }
  if (p.dinitial && live && chunk + 1 == (unsigned)f.chunks && piece == pieces - 1) p.dinitial[row] = k;
}

// The same for gates that several channels share and rows in one chunk: a workgroup (or a row's lanes) takes f.each rows of a gate
// one after the other, the next one's loads under way, with the decays and the sums of dgate in registers.
template <class T, class G>
__global__ __launch_bounds__(64 * kMaxWaves<T>, 4) void scan_signals_bwd_heads(tfft_scan_grad_args p, Shape f, float* parts, long long pitch) {
  constexpr int E = kSteps<T>;
  __shared__ Lds lds[2];  // of this row and the one before: no wave is further apart
  long long group;
  unsigned chunk;
  take<ONE>(f, lds[0], &group, &chunk);
  const bool live = group < f.rows / f.each;
  if (!live) group = 0;
  const unsigned row = (unsigned)group * f.each;
  const int b = (int)(row / (unsigned)f.channels), c = (int)(row - (unsigned)b * (unsigned)f.channels), len = live ? steps_of(p.lengths, b, f.length) : 0;
  const int order = threadIdx.x, piece = f.lanes < 64 ? order & (f.lanes - 1) : order;
  const int pieces = f.lanes < 64 ? f.lanes : (int)blockDim.x, t0 = (pieces - 1 - piece) * E;
  const T* dy = (const T*)p.dy.data + b * p.dy.batch + c * p.dy.channel;
  const T* y = (const T*)p.y.data + b * p.y.batch + c * p.y.channel;
  T* dx = (T*)p.dx.data + b * p.dx.batch + c * p.dx.channel;
  const G* g = (const G*)p.gate.data + b * p.gate.batch + (c / f.share) * p.gate.channel;
  const int t_before = min(max(t0 - 1, 0), f.length - 1);
  Run<G, E> gr = p.gate.time ? ask<E>(g, t0, f.length) : one<E>(g);
  Run<T, E> d = ask<E>(dy, t0, f.length), own = ask<E>(y, t0, f.length);
  Run<T, 1> before = load_run<T, 1>(y + t_before);
  float a[E], sums[E], A = 1.0f;
  take_decays<E>(gr, p.gate.time, t0, len, f.length, f.log_gate, a);
#pragma unroll
  for (int i = E - 1; i >= 0; --i) A *= a[i], sums[i] = 0.0f;
  for (int n = 0; n < f.each; ++n) {
    if (n + 1 < f.each) dy += p.dy.channel, y += p.y.channel;
    const Run<T, E> next_d = ask<E>(dy, t0, f.length), next_own = ask<E>(y, t0, f.length);
    const Run<T, 1> next_before = load_run<T, 1>(y + t_before);
    const float initial = p.initial ? p.initial[row + n] : 0.0f;
    take<E>(d, t0, len, f.length);
    take<E>(own, t0, len, f.length);
    float B = 0.0f;
#pragma unroll
    for (int i = E - 1; i >= 0; --i) B = a[i] * (B + d.get(i));
    float k = state_in_front<ONE>(f, lds[n & 1], chunk, row, order, A, B, p.dlast ? p.dlast[row + n] : 0.0f);
    Run<T, E> r;
    float e[E];
#pragma unroll
    for (int i = E - 1; i >= 0; --i) {
      e[i] = d.get(i) + k;
      k = a[i] * e[i];
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float state = i > 0 ? own.get(i > 0 ? i - 1 : 0) : t0 > 0 ? before.get(0) : initial;
      const bool inside = t0 + i < len;
      sums[i] += inside ? e[i] * state : 0.0f;
      e[i] = inside ? e[i] : 0.0f;
    }
    r.set_all(e);
    if (live) store_steps<E, false>(dx, t0, f.length, r);
    if (p.dinitial && live && piece == pieces - 1) p.dinitial[row + n] = k;
    dx += p.dx.channel;
    d = next_d, own = next_own, before = next_before;
  }
  if (!live) return;
  if (f.log_gate) {
#pragma unroll
    for (int i = 0; i < E; ++i) sums[i] *= a[i];
  }
  if (parts) {
    Run<float, E> q;
    q.set_all(sums);
    store_steps<E, false>(parts + group * pitch, t0, f.length, q);
  } else {
    Run<G, E> q;
    q.set_all(sums);
    store_steps<E, false>((G*)p.dgate.data + b * p.dgate.batch + (c / f.share) * p.dgate.channel, t0, f.length, q);
  }
}

// dgate of gates that several channels share, from `count` rows of parts each: 32 threads with kSum steps each side by side, 8 of
// them for each of those, which take every eighth row. What it reads was written just before, and comes from the last-level cache
// where it fits.
constexpr int kSum = 4;
template <class G>
__global__ __launch_bounds__(256) void sum_signals(tfft_scan_grad_args p, const float* parts, long long pitch, int count, long long tiles) {
  __shared__ float lds[8][32][kSum + 1];
  const int column = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const long long gates = p.channels / p.share, across = (p.length + 32 * kSum - 1) / (32 * kSum);
  for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const long long row = tile / across, t = (tile - row * across) * 32 * kSum + column * kSum, b = row / gates, g = row - b * gates;
    float sum[kSum] = {};
    if (t < p.length) {  // rows of the parts are whole multiples of kSum
      const float* from = parts + row * count * pitch + t;
#pragma unroll 4
      for (int i = slice; i < count; i += 8) {
        const Run<float, kSum> r = load_run<float, kSum>(from + i * pitch);
#pragma unroll
        for (int k = 0; k < kSum; ++k) sum[k] += r.get(k);
      }
    }
#pragma unroll
    for (int k = 0; k < kSum; ++k) lds[slice][column][k] = sum[k];
    __syncthreads();
    if (slice == 0 && t < p.length) {
      for (int i = 1; i < 8; ++i)
#pragma unroll
        for (int k = 0; k < kSum; ++k) sum[k] += lds[i][column][k];
      Run<G, kSum> q;
#pragma unroll
      for (int k = 0; k < kSum; ++k) q.set(k, sum[k]);
      store_some<kSum>((G*)p.dgate.data + b * p.dgate.batch + g * p.dgate.channel + t, q, (int)min((long long)kSum, p.length - t));
    }
    __syncthreads();
  }
}
long long pitch_of(long long length) { return (length + kSum - 1) / kSum * kSum; }

Chunking plan(long long batch, long long length, long long channels, int dtype, bool padded_batch, int many, long long share = 1) {
  const int steps = dtype == TFFT_F32 ? kSteps<float> : kSteps<f16>, most = dtype == TFFT_F32 ? kMaxWaves<float> : kMaxWaves<f16>;
  Chunking c;
  const long long rows = batch * channels, pieces = (length + steps - 1) / steps;
  c.tiles = rows;
  c.state_words = rows;
  c.strip = padded_batch;
  c.group = kMaxGroup;
  if (pieces <= 32) {
    c.lanes = 1;
    while (c.lanes < pieces) c.lanes *= 2;
    c.waves = 4;
    c.chunks = 1;
    c.side_by_side = 64 * c.waves / c.lanes;
  } else {
    c.walks = pieces > 64 * most && rows >= many;
    const int waves = c.walks && rows >= kShortChunks ? kWalkWaves : most;
    c.chunks = (pieces + 64 * waves - 1) / (64 * waves);
    c.waves = (int)((pieces + 64 * c.chunks - 1) / (64 * c.chunks));
    c.chunks = (pieces + 64 * c.waves - 1) / (64 * c.waves);
  }
  if (c.chunks == 1 && length > 0) {
    const long long groups = c.lanes < 64 ? rows * c.lanes / (64 * c.waves) : rows;
    c.each = groups >= kEach * kFewGroups ? kEach : kEachOfFew;
    while (share % c.each) --c.each;
    c.tiles /= c.each;
  }
  return c;
}

template <class P>
Shape shape_of(const P& p, const Chunking& c, word* words) {
  return Shape{p.batch * p.channels, (int)p.length, (int)p.channels, (int)p.share, p.gate_form == TFFT_GATE_LOG,
               (int)c.chunks, c.group, c.lanes, c.each, turns_of(c), words};
}

}  // namespace

bool signals_fit(const tfft_scan_args& p) {
  return p.x.time == 1 && p.y.time == 1 && p.gate.time <= 1;
}
bool signals_fit(const tfft_scan_grad_args& p) {
  return p.dy.time == 1 && p.y.time == 1 && p.dx.time == 1 && p.dgate.time == 1 && p.gate.time <= 1;
}
Chunking plan_signals(const tfft_scan_args& p) { return plan(p.batch, p.length, p.channels, p.dtype, p.lengths != nullptr, kManyRows); }
Chunking plan_signals(const tfft_scan_grad_args& p) {
  return plan(p.batch, p.length, p.channels, p.dtype, p.lengths != nullptr, p.dtype == TFFT_F32 ? kManyRows : kManyRowsBack, p.share);
}

void launch_signals(const tfft_scan_args& p, const Chunking& c, word* words, hipStream_t s) {
  const Shape f = shape_of(p, c, words);
  const dim3 grid((unsigned)c.blocks()), block(64 * c.waves);
  with_types(p.dtype, p.gate_dtype, [&](auto t, auto g) {
    using T = decltype(t);
    using G = decltype(g);
    if (c.chunks <= 1) scan_signals_fwd<T, G, ONE><<<grid, block, 0, s>>>(p, f);
    else if (c.walks) scan_signals_fwd<T, G, WALK><<<grid, block, 0, s>>>(p, f);
    else scan_signals_fwd<T, G, SPLIT><<<grid, block, 0, s>>>(p, f);
  });
}
// Rows of parts a gate; one: none
static long long parts_of_gate(const tfft_scan_grad_args& p) { return p.length > 0 ? p.share / plan_signals(p).each : 1; }
unsigned long long signals_parts(const tfft_scan_grad_args& p) {
  const long long count = parts_of_gate(p);
  return count > 1 ? (unsigned long long)p.batch * (p.channels / p.share) * count * pitch_of(p.length) : 0;
}
void launch_signals(const tfft_scan_grad_args& p, const Chunking& c, word* words, float* parts, hipStream_t s) {
  const Shape f = shape_of(p, c, words);
  const long long pitch = pitch_of(p.length), count = parts_of_gate(p);
  const dim3 grid((unsigned)c.blocks()), block(64 * c.waves);
  if (count == 1) parts = nullptr;
  with_types(p.dtype, p.gate_dtype, [&](auto t, auto g) {
    using T = decltype(t);
    using G = decltype(g);
    const bool shared = p.share > 1 && p.length > 0;
    if (c.chunks <= 1 && shared) scan_signals_bwd_heads<T, G><<<grid, block, 0, s>>>(p, f, parts, pitch);
    else if (c.chunks <= 1) scan_signals_bwd<T, G, ONE, false><<<grid, block, 0, s>>>(p, f, parts, pitch);
    else if (c.walks && shared) scan_signals_bwd<T, G, WALK, true><<<grid, block, 0, s>>>(p, f, parts, pitch);
    else if (c.walks) scan_signals_bwd<T, G, WALK, false><<<grid, block, 0, s>>>(p, f, parts, pitch);
    else if (shared) scan_signals_bwd<T, G, SPLIT, true><<<grid, block, 0, s>>>(p, f, parts, pitch);
    else scan_signals_bwd<T, G, SPLIT, false><<<grid, block, 0, s>>>(p, f, parts, pitch);
    if (parts) {
      const long long tiles = p.batch * (p.channels / p.share) * ((p.length + 32 * kSum - 1) / (32 * kSum));
      sum_signals<G><<<(unsigned)std::min(tiles, 1LL << 16), 256, 0, s>>>(p, parts, pitch, (int)count, tiles);
    }
  });
}

}  // namespace tfft_seq
