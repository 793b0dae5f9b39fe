// The gated linear recurrence where neighbouring channels lie side by side ([batch][time][channel]), and, one element
// at a time, for any other strides.
#include <algorithm>
#include <initializer_list>
#include <type_traits>
#include <utility>

#include "recurrence_kernels.hpp"

namespace tfft_seq {
namespace {

// A lane holds a run of V channels of one batch entry over S steps, a wave 64 runs, a workgroup `waves` pieces of S steps one
// behind the other. Channels are counted over the whole batch (each entry padded to whole runs), so few channels
// fill a wave too.
//
// What bounds it: HBM, at the rate that this pattern reaches. B = 8, L = 4096, D = 2048 in bf16 with fp32 log decays takes
// 103 us forward (537 MB, 5.2 TB/s) and 171 back (939 MB, 5.5); as much in chunks that do not depend on each other
// (B = 64, L = 128, D = 8192) 87 and 156 (6.2, 6.0). The look-back is hidden there but for 4 us of clearing its words; with few
// channels chunks wait for each other: 65537 x 1024 in bf16 85 us (403 MB, 4.7 TB/s).
//
// Why these sizes: 16 steps of two channels are 48 registers of values, 24 in 16 bits 72, which leaves two workgroups of 8 waves a
// CU that load, wait and store at different times. On those two shapes runs of 4 and 4, 6, 10, 12 or 16 waves took 0 ... 40 %
// longer, and a workgroup that takes chunk after chunk with the next one's loads under way 6 %.
constexpr int kMaxWaves = 8, kMaxGroup = 16, kResident = 512, kRun = 2;
// Steps of a piece, forward: kStepsLong of 16-bit values where pieces of kSteps would not fit one chunk, of shared gates (whose kernels
// have three workgroups a CU with kSteps) from kLongShared steps on. In bf16 with 24 and 16: B = 8, L = 4096, D = 2048 with fp32 log
// decays 103 and 106 us, one sequence of 65537 x 1024 85 and 94, x 128 20 and 24, [32, 300, 4096] 49 and 52, but [64, 128, 8192]
// 90 and 87; 64 channels a gate: 65537 x 1024 70 and 78, [16, 500, 1024] 14 and 13. In fp32 [4, 3000, 600] 27.5 and 25.
constexpr int kSteps = 16, kStepsLong = 24, kLongShared = 4096;
// Backward: where a run of channels has one gate, fewer decays leave registers for more steps: 4 entries of up to 8191 steps with heads of
// 64 in bf16 83 us against 87 with 16, [8, 4096, 2048] in fp32 145 against 154 with 8. With a gate a channel 20 take 175 us where 16 take 171.
template <class T, bool kOneGate>
constexpr int kStepsBackward = sizeof(T) == 4 ? (kOneGate ? 12 : 8) : kOneGate ? 20 : 16;

// Runs take 32-bit offsets, which the plan has checked; single elements may lie anywhere
template <int V>
using offset_of = std::conditional_t<V == 1, long long, uint32_t>;

struct Shape {
  int batch, length, channels, padded;  // padded: channels rounded up to whole runs
  int share, log_gate;
  int chunks, group, row, lanes;
  long long state_words;
  unsigned tiles_of_entry;  // 0: tiles run through the whole batch
  Turns turns;
  word* words;
};

// Lane's place: its first word n among those of a chunk's states, batch entry b, first channel c of its run and how many
// channels of it are the lane's own. The last run of a row that does not fill it lies over the run before, so that every lane can
// load whole runs: its own channels are the run's last ones, the others' results are dropped. Lanes behind the last channel have
// none and lie over the tile's first run. Lanes behind the f.lanes that a tile fills do what the tile's first lanes do, side by
// side with them. first: the batch entry that the tile's addresses start from, the same for all lanes.
struct Place {
  unsigned n;
  int b, c, own, first;
};
template <int V>
__device__ __forceinline__ Place place_of(const Shape& f, unsigned tile, int lane) {
  Place p;
  p.n = tile * (64u * V) + lane * V;
  const unsigned width = f.lanes * V;
  if (lane >= f.lanes) lane -= f.lanes;
  if (f.tiles_of_entry == 0) {
    p.first = 0;
    const unsigned m = tile * width + lane * V;
    p.b = m / (unsigned)f.padded;
    p.c = m - p.b * (unsigned)f.padded;
  } else {
    p.first = p.b = __builtin_amdgcn_readfirstlane(tile / f.tiles_of_entry);
    p.c = (tile - p.b * f.tiles_of_entry) * width + lane * V;
  }
  p.own = p.b >= f.batch || p.c >= f.channels ? 0 : min(V, f.channels - p.c);
  if (p.own == 0) p.b = p.first, p.c = 0;
  else p.c -= V - p.own;
  return p;
}

// One of the tensors at a lane's place: an address that the wave shares, in scalar registers, and the lane's offset in bytes.
// Vector kernels take 32-bit offsets, so that a load needs no vector register but those that it fills.
template <class T, class Off>
struct Lane {
  uint64_t base;
  Off off;
  long long step;  // bytes from one time step to the next
  __device__ __forceinline__ Lane(const tfft_seq_view& v, const Place& p, int c)
      : base((uint64_t)v.data + p.first * v.batch * (long long)sizeof(T)),
        off((Off)(((p.b - p.first) * v.batch + c * v.channel) * (long long)sizeof(T))),
        step(v.time * (long long)sizeof(T)) {}
  // the lane's address at step t (the same for the wave), and its move to the next or the previous step: an addition in scalar
  // registers, said so for the compiler, which otherwise holds an address a step
  __device__ __forceinline__ void go(int t) {
    const uint64_t b = base + t * step;
    base = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(b >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)b);
  }
  __device__ __forceinline__ void move(long long by) {
    base += by;
    asm("" : "+s"(base));
  }
  __device__ __forceinline__ T* at(int t) const { return device_pointer<T>(base + t * step, off); }
  __device__ __forceinline__ T* here() const { return device_pointer<T>(base, off); }
};

template <int V>
__device__ __forceinline__ void load_state(const float* from, const Place& p, int channels, float (&h)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = from && v >= V - p.own ? from[(long long)p.b * channels + p.c + v] : 0.0f;
}
template <int V>
__device__ __forceinline__ void store_state(float* to, const Place& p, int channels, const float (&h)[V]) {
  if (!to) return;
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (v >= V - p.own) to[(long long)p.b * channels + p.c + v] = h[v];
}

// The joint map of `count` maps that follow one another, `step` words apart, as soon as they are there
template <int V>
__device__ __forceinline__ void join_words(const word* from, long long step, int count, float (&a)[V], float (&b)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) a[v] = 1.0f, b[v] = 0.0f;
  constexpr int kAtOnce = 4;
#pragma unroll 1
  for (int k = 0; k < count; k += kAtOnce, from += kAtOnce * step) {
    word w[kAtOnce][V];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) w[i][v] = peek(from + (k + i < count ? step * i : 0) + v);
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (k + i >= count) break;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (!w[i][v]) w[i][v] = await(from + step * i + v);
        b[v] = join(map_a(w[i][v]), b[v], map_b(w[i][v]));
        a[v] *= map_a(w[i][v]);
      }
    }
  }
}

// The state in front of this chunk, for the wave that has the (A, B) of the whole chunk, from the words of earlier chunks (or
// `start`, in front of the first): the maps of its group's chunks before it, those of the groups before it in their row of
// groups, and the state in front of that row. Publishes this chunk's own words on the way, each as soon as it is known.
template <int V>
__device__ __forceinline__ void state_before(const Shape& f, const float* start, const Place& at, unsigned chunk, const float (&A)[V],
                                             const float (&B)[V], float (&h)[V]) {
  const int r = chunk % f.group, q = chunk / f.group, u = q % f.row, s = q / f.row;
  const bool more = chunk + 1 < (unsigned)f.chunks, last = r == f.group - 1;
  word* maps = f.words + kCounterWords * f.turns.counters + at.n;
  word* of_groups = maps + (f.group > 1 ? f.state_words * f.chunks : 0);
  unsigned* states = (unsigned*)(of_groups - at.n + (f.row > 1 ? f.state_words * ((f.chunks + f.group - 1) / f.group) : 0)) + at.n;
  if (more && !last) {
#pragma unroll
    for (int v = 0; v < V; ++v) publish_map(maps + f.state_words * chunk + v, A[v], B[v]);
  }
  float a[V], b[V];
  join_words<V>(maps + f.state_words * (chunk - r), f.state_words, r, a, b);
  if (f.row > 1) {
    if (more && last && u != f.row - 1) {
#pragma unroll
      for (int v = 0; v < V; ++v) publish_map(of_groups + f.state_words * q + v, A[v] * a[v], join(A[v], b[v], B[v]));
    }
    float ga[V], gb[V];
    join_words<V>(of_groups + f.state_words * (q - u), f.state_words, u, ga, gb);
#pragma unroll
    for (int v = 0; v < V; ++v) b[v] = join(a[v], gb[v], b[v]), a[v] *= ga[v];
  }
  if (s == 0) {
    load_state<V>(start, at, f.channels, h);
  } else {
    unsigned w[V];
    const unsigned* from = states + f.state_words * (s - 1);
#pragma unroll
    for (int v = 0; v < V; ++v) w[v] = peek(from + v);
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = __uint_as_float(w[v] ? w[v] : await(from + v));
  }
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = join(a[v], h[v], b[v]);
  if (more && last && u == f.row - 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) publish_state(states + f.state_words * s + v, join(A[v], h[v], B[v]));
  }
}

// The (A, B) of the waves' pieces, the state in front of the chunk, the ticket
template <int V>
struct Joint {
  float A[kMaxWaves][64 * V], B[kMaxWaves][64 * V], h[64 * V];
  unsigned ticket;
};
// those in front of this wave's piece
template <int V>
__device__ __forceinline__ void join_pieces(const Joint<V>& lds, int wave, int lane, float (&a)[V], float (&b)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) a[v] = 1.0f, b[v] = 0.0f;
#pragma unroll 2
  for (int w = 0; w < wave; ++w) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float A = lds.A[w][lane * V + v];
      b[v] = join(A, b[v], lds.B[w][lane * V + v]);
      a[v] *= A;
    }
  }
}

// Asks for V elements at each of S steps from t0 on. Steps in front of the first and behind the last are asked for there (what
// that gives is not used): one path for all, because a load whose register two paths could have filled is waited for where they meet.
template <int S, int V, bool STREAM, class T, class Off>
__device__ __forceinline__ void ask(Lane<T, Off> x, int t0, int last, Run<T, V> (&r)[S]) {
  x.go(min(max(t0, 0), last));
#pragma unroll
  for (int s = 0; s < S; ++s) {
    r[s] = load_run<T, V, STREAM>(x.here());
    if (s + 1 < S) x.move(t0 + s >= 0 && t0 + s < last ? x.step : 0);
  }
}
// The last step that a wave has use for: a step behind the longest of its sequences is of none
__device__ __forceinline__ int last_step(const Shape& f, const int* lengths, int len) {
  if (!lengths) return f.length - 1;
  for (int m = 1; m < 64; m *= 2) len = max(len, __shfl_xor(len, m));
  return max(__builtin_amdgcn_readfirstlane(len), 1) - 1;
}

// What was asked for, with zeros outside the sequence. The values stay two to a register between the two walks: without stay() the
// compiler holds the first walk's unpacked copies for the second, twice the registers.
template <int S, int V, class T>
__device__ __forceinline__ void stay(Run<T, V> (&x)[S]) {
#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (uint32_t& w : x[s].w) asm("" : "+v"(w));
}
template <int S, int V, class T>
__device__ __forceinline__ void take(Run<T, V> (&x)[S], int t0, int len, bool all) {
  if (!all) {
#pragma unroll
    for (int s = 0; s < S; ++s)
      if (t0 + s < 0 || t0 + s >= len) x[s].clear();
  }
  stay<S, V>(x);
}
template <int S, int V, class G>
__device__ __forceinline__ void take_decays(const Run<G, V> (&r)[S], int t0, int len, bool all, int log_gate, float (&a)[S][V]) {
#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int v = 0; v < V; ++v) a[s][v] = r[s].get(v);
  if (log_gate) {
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int v = 0; v < V; ++v) a[s][v] = exp_decay(a[s][v]);
  }
  if (!all) {
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int v = 0; v < V; ++v) a[s][v] = t0 + s < len ? a[s][v] : 1.0f;
  }
}
// The lane's own elements of a run
template <int V, bool STREAM, class T>
__device__ __forceinline__ void put(T* to, const Run<T, V>& r, int own) {
  if (own == V) return store_run<T, V, STREAM>(to, r);
#pragma unroll
  for (int v = 1; v < V; ++v)
    if (v >= V - own) {
      Run<T, 1> one;
      if constexpr (sizeof(T) == 4) one.w[0] = r.w[v];
      else one.w[0] = r.w[v / 2] >> (v % 2 * 16);
      store_run<T, 1>(to + v, one);
    }
}

// From the (A, B) of this wave's piece to the state in front of it
template <int V>
__device__ __forceinline__ void state_of_piece(const Shape& f, Joint<V>& lds, const float* start, const Place& at, unsigned chunk, int wave,
                                               int waves, int lane, const float (&A)[V], const float (&B)[V], float (&h)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) lds.A[wave][lane * V + v] = A[v], lds.B[wave][lane * V + v] = B[v];
  __syncthreads();
  float front_a[V], front_b[V];
  join_pieces<V>(lds, wave, lane, front_a, front_b);
  if (wave == waves - 1) {
    float chunk_a[V], chunk_b[V];
#pragma unroll
    for (int v = 0; v < V; ++v) chunk_a[v] = A[v] * front_a[v], chunk_b[v] = join(A[v], front_b[v], B[v]);
    state_before<V>(f, start, at, chunk, chunk_a, chunk_b, h);
#pragma unroll
    for (int v = 0; v < V; ++v) lds.h[lane * V + v] = h[v];
  }
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = join(front_a[v], lds.h[lane * V + v], front_b[v]);
}

template <class T, class G, int V, int VG, bool STREAM, int S>
__global__ __launch_bounds__(64 * kMaxWaves, 4) void scan_rows_fwd(tfft_scan_args p, Shape f) {
  using Off = offset_of<V>;
  __shared__ Joint<V> lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  unsigned tile, chunk;
  if (!take_turn(f.turns, f.words, &lds.ticket, &tile, &chunk)) return;
  const Place at = place_of<V>(f, tile, lane);
  const int len = steps_of(p.lengths, at.b, f.length), t0 = (int)(chunk * waves + wave) * S;
  const bool all = __all(t0 + S <= len && at.own == V), none = __all(t0 >= len);  // of the wave's steps lie inside
  Run<T, V> x[S];
  Run<G, VG> g[S];
  if (!none) {
    const int last = last_step(f, p.lengths, len);
    ask<S, V, STREAM>(Lane<T, Off>(p.x, at, at.c), t0, last, x);
    ask<S, VG, STREAM && VG == V>(Lane<G, Off>(p.gate, at, f.share == 1 ? at.c : at.c / f.share), t0, last, g);
  }
  float a[S][VG];
  take<S, V>(x, t0, len, all);
  take_decays<S, VG>(g, t0, len, all, f.log_gate, a);

  float A[V], B[V], h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) A[v] = 1.0f, B[v] = 0.0f;
#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      A[v] *= a[s][v % VG];
      B[v] = fmaf(a[s][v % VG], B[v], x[s].get(v));
    }
  stay<S, V>(x);
  state_of_piece<V>(f, lds, p.initial, at, chunk, wave, waves, lane, A, B, h);

  Lane<T, Off> y(p.y, at, at.c);
  y.go(t0);
  const auto walk = [&](auto whole) {
#pragma unroll
    for (int s = 0; s < S; ++s, y.move(y.step)) {
      Run<T, V> r;
      float out[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        h[v] = fmaf(a[s][v % VG], h[v], x[s].get(v));
        out[v] = whole.value || t0 + s < len ? h[v] : 0.0f;
      }
      r.set_all(out);
      if (whole.value || t0 + s < f.length) put<V, STREAM>(y.here(), r, whole.value ? V : at.own);
    }
  };
  if (all) walk(std::true_type());
  else walk(std::false_type());
  if (chunk + 1 == (unsigned)f.chunks && wave == waves - 1) store_state<V>(p.last, at, f.channels, h);
}

// Sums of N values over groups of `lanes` lanes (a power of two, at least N), one value a lane: every exchange halves the
// values that a lane still has, N - 1 exchanges where one sum after the other takes N times the logarithm. The lane
// ends with the sum of value `at`. M: how far apart the lanes of the next exchange lie.
template <int N, int M = 1>
__device__ __forceinline__ float sum_values(const float (&q)[N], int lane, int lanes, int& at) {
  if constexpr (N == 1) {
    float sum = q[0];
    for (int m = M; m < lanes; m *= 2) sum += __shfl_xor(sum, m);
    return sum;
  } else {
    const bool upper = lane & M;
    at = 2 * at + upper;
    float half[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float keep = upper ? q[i + N / 2] : q[i], give = upper ? q[i] : q[i + N / 2];
      half[i] = keep + __shfl_xor(give, M);
    }
    return sum_values<N / 2, 2 * M>(half, lane, lanes, at);
  }
}

// Backwards in time: chunk 0 is the latest, wave 0 has the latest piece. The terms of a gate that several channels share are summed
// over `lanes` lanes: EVEN by exchanges over a power of two, ODD through LDS, a lane for every gate and step. Where a gate has
// more lanes than a wave, their sums (ODD) go to `parts` (fp32, [batch][time] and the channels in groups of `lanes` runs) for a
// kernel behind. B = 8, L = 4096, D = 2048 in bf16 with fp32 gates takes 85 us with 64 channels a gate, D = 2016 with 48 110
// (1109 with every channel's term in memory), D = 2000 with 200 128 (1048).
enum { EVEN, ODD };
template <class T, class G, int V, int VG, bool STREAM, int SUMS = EVEN>
__global__ __launch_bounds__(64 * kMaxWaves, 4) void scan_rows_bwd(tfft_scan_grad_args p, Shape f, float* parts, int lanes) {
  constexpr int S = kStepsBackward<T, (VG < V)>;
  constexpr bool kShared = V == 1 || VG < V;  // a gate may have several channels
  using Off = offset_of<V>;
  __shared__ Joint<V> lds;
  __shared__ float terms[SUMS == ODD ? kMaxWaves : 1][SUMS == ODD ? S : 1][65];  // 65: lanes read the same place of all steps
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  unsigned tile, chunk;
  if (!take_turn(f.turns, f.words, &lds.ticket, &tile, &chunk)) return;
  const Place at = place_of<V>(f, tile, lane);
  const int len = steps_of(p.lengths, at.b, f.length);
  const int t0 = ((int)(f.chunks - 1 - chunk) * waves + (waves - 1 - wave)) * S;
  const bool all = __all(t0 + S <= len && at.own == V), none = __all(t0 >= len);  // of the wave's steps lie inside
  const int gate = f.share == 1 ? at.c : at.c / f.share;
  Run<T, V> d[S], before[S];
  Run<G, VG> g[S];
  if (!none) {
    const int last = last_step(f, p.lengths, len);
    ask<S, V, STREAM>(Lane<T, Off>(p.dy, at, at.c), t0, last, d);
    ask<S, VG, STREAM && VG == V>(Lane<G, Off>(p.gate, at, gate), t0, last, g);
    ask<S, V, STREAM>(Lane<T, Off>(p.y, at, at.c), t0 - 1, last, before);
  }
  float a[S][VG];
  take<S, V>(d, t0, len, all);
  take_decays<S, VG>(g, t0, len, all, f.log_gate, a);

  float A[V], B[V], c[V];
#pragma unroll
  for (int v = 0; v < V; ++v) A[v] = 1.0f, B[v] = 0.0f;
#pragma unroll
  for (int s = S - 1; s >= 0; --s)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      A[v] *= a[s][v % VG];
      B[v] = a[s][v % VG] * (B[v] + d[s].get(v));
    }
  stay<S, V>(d);
  state_of_piece<V>(f, lds, p.dlast, at, chunk, wave, waves, lane, A, B, c);

  take<S, V>(before, t0 - 1, len, all && t0 > 0);
  float start[V];
#pragma unroll
  for (int v = 0; v < V; ++v) start[v] = 0.0f;
  if (t0 == 0) load_state<V>(p.initial, at, f.channels, start);
  Lane<T, Off> dx(p.dx, at, at.c);
  Lane<G, Off> dg(p.dgate, at, gate);
  dx.go(t0 + S - 1), dg.go(t0 + S - 1);
  float sums[S];  // of the run, where a gate has one or more runs of channels
  const auto walk = [&](auto whole) {
#pragma unroll
    for (int s = S - 1; s >= 0; --s, dx.move(-dx.step), dg.move(-dg.step)) {
      const int t = t0 + s;
      Run<T, V> r;
      float da[V], out[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float e = d[s].get(v) + c[v], k = a[s][v % VG];
        float state = before[s].get(v);
        if (s == 0) state = t == 0 ? start[v] : state;
        out[v] = whole.value || t < len ? e : 0.0f;
        c[v] = k * e;
        // (a gate's own decay, where it counts, multiplies the sum of its channels)
        da[v] = VG < V || !f.log_gate ? e * state : c[v] * state;
        if (!whole.value) da[v] = t < len ? da[v] : 0.0f;
      }
      r.set_all(out);
      const bool in = whole.value || t < f.length;
      const int own = whole.value ? V : at.own;
      if (in) put<V, STREAM>(dx.here(), r, own);
      if (!kShared || (V == 1 && f.share == 1)) {
        Run<G, V> q;
        q.set_all(da);
        if (in) put<V, STREAM>(dg.here(), q, own);
      } else {
        float sum = da[0];
#pragma unroll
        for (int v = 1; v < V; ++v) sum += da[v];
        if (VG < V && f.log_gate) sum *= a[s][0];
        if constexpr (SUMS == ODD) terms[wave][s][lane] = sum;
        else sums[s] = sum;
      }
    }
  };
  if (all) walk(std::true_type());
  else walk(std::false_type());
  if constexpr (SUMS == ODD) {
    // a wave reads what it wrote itself; a barrier would wait for its stores as well
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int gates = f.lanes / lanes, group = lanes * V;
    for (int i = lane; i < S * gates; i += 64) {
      const int s = i / gates, first = (i - s * gates) * lanes, t = t0 + s;
      float sum = terms[wave][s][first];
#pragma unroll 4
      for (int k = 1; k < lanes; ++k) sum += terms[wave][s][first + k];
      const Place of = place_of<V>(f, tile, first);
      if (of.own == 0 || t >= f.length) continue;
      Run<G, 1> q;
      q.set(0, sum);
      if (parts) parts[((long long)of.b * f.length + t) * (f.channels / group) + of.c / group] = sum;
      else store_run<G, 1>(Lane<G, long long>(p.dgate, of, of.c / f.share).at(t), q);
    }
  } else if (kShared && f.share > 1) {
    constexpr int kFirst = S >= 16 ? 16 : 8, kRest = S - kFirst;  // powers of two
    if (lanes >= kFirst) {
      const auto give = [&](const auto& some, auto count, int first) {
        constexpr int kCount = decltype(count)::value;
        int s = 0;
        Run<G, 1> q;
        q.set(0, sum_values<kCount>(some, lane, lanes, s));
        s += first;
        if (at.own > 0 && (lane & (lanes - 1)) < kCount && t0 + s < f.length) store_run<G, 1>(Lane<G, long long>(p.dgate, at, gate).at(t0 + s), q);
      };
      float some[kFirst];
#pragma unroll
      for (int i = 0; i < kFirst; ++i) some[i] = sums[i];
      give(some, std::integral_constant<int, kFirst>(), 0);
      if constexpr (kRest > 0) {
        float rest[kRest];
#pragma unroll
        for (int i = 0; i < kRest; ++i) rest[i] = sums[kFirst + i];
        give(rest, std::integral_constant<int, kRest>(), kFirst);
      }
    } else {
#pragma unroll
      for (int s = 0; s < S; ++s) {
        for (int m = 1; m < lanes; m *= 2) sums[s] += __shfl_xor(sums[s], m);
        Run<G, 1> q;
        q.set(0, sums[s]);
        if (at.own > 0 && (lane & (lanes - 1)) == 0 && t0 + s < f.length) store_run<G, 1>(Lane<G, long long>(p.dgate, at, gate).at(t0 + s), q);
      }
    }
  }
  if (chunk + 1 == (unsigned)f.chunks && wave == waves - 1) store_state<V>(p.dinitial, at, f.channels, c);
}

// dgate of a gate that has more lanes than a wave, from the sums of its groups of lanes: 16 threads a gate
template <class G>
__global__ __launch_bounds__(256) void sum_parts(tfft_scan_grad_args p, const float* parts, int groups) {
  const long long gates = p.channels / p.share, all = p.batch * p.length * gates;
  const int i = threadIdx.x & 15;
  for (long long n = 16ll * blockIdx.x + (threadIdx.x >> 4); n < all; n += 16ll * gridDim.x) {
    float sum = 0.0f;
    for (int k = i; k < groups; k += 16) sum += parts[n * groups + k];
    for (int m = 1; m < 16; m *= 2) sum += __shfl_xor(sum, m);
    const long long g = n % gates, bt = n / gates, b = bt / p.length, t = bt % p.length;
    if (i == 0) ((G*)p.dgate.data)[b * p.dgate.batch + t * p.dgate.time + g * p.dgate.channel] = from_f32<G>(sum);
  }
}

int steps_backward(int dtype, bool one_gate) {
  if (one_gate) return dtype == TFFT_F32 ? kStepsBackward<float, true> : kStepsBackward<f16, true>;
  return dtype == TFFT_F32 ? kStepsBackward<float, false> : kStepsBackward<f16, false>;
}

// Tiles run through the whole batch where that keeps a lane's offsets within 32 bits, so that few channels fill a wave too; else
// each batch entry has tiles of its own.
bool through_batch(int run, long long batch, long long channels, std::initializer_list<const tfft_seq_view*> views) {
  if (run == 1) return true;
  for (const tfft_seq_view* v : views)
    if ((__int128)(batch - 1) * v->batch + (__int128)(channels - 1) * v->channel >= (1LL << 32) / 4 - run) return false;
  return true;
}

Chunking plan(long long batch, long long length, long long channels, int run, int lanes, bool through, int steps, bool padded_batch) {
  Chunking c;
  const long long padded = (channels + run - 1) / run * run, width = lanes * run;
  c.lanes = lanes;
  c.tiles = through ? (batch * padded + width - 1) / width : batch * ((channels + width - 1) / width);
  // as few chunks as the workgroup's waves allow, then as few waves as those need
  const long long pieces = length > 0 ? (length + steps - 1) / steps : 1;
  c.chunks = (pieces + kMaxWaves - 1) / kMaxWaves;
  c.waves = (int)((pieces + c.chunks - 1) / c.chunks);
  c.chunks = (pieces + c.waves - 1) / c.waves;
  c.state_words = c.tiles * 64 * run;
  if (padded_batch && batch > 0) c.strip = c.tiles / (8 * batch) > 1 ? c.tiles / (8 * batch) : 1;
  // About kResident workgroups run at once, kResident / tiles chunks of each tile. That many are joined directly, so that few
  // channels wait for one state in that many chunks, and many channels do not read what they need not: B = 8,
  // L = 4096, D = 2048 (128 tiles) takes 170, 170, 172 us back with groups of 4, 8, 16; one sequence of 65537 steps
  // and 1024 channels (8 tiles) 101, 86, 85 us forward.
  while (c.group < kMaxGroup && c.group * c.tiles < kResident) c.group *= 2;
  // With one or two tiles the states of one group after the other are what a call waits for: one sequence of 65537 steps in bf16 takes
  // 30, 39 us with 128, 256 channels so, 20, 35 in rows of groups; with 1024 channels rows of groups cost 6 %.
  if (c.tiles <= 2) c.row = kMaxGroup;
  return c;
}

template <class P>
Shape shape_of(const P& p, const Chunking& c, int run, bool through, word* words) {
  return Shape{(int)p.batch, (int)p.length, (int)p.channels, (int)((p.channels + run - 1) / run * run), (int)p.share,
               p.gate_form == TFFT_GATE_LOG, (int)c.chunks, c.group, c.row, c.lanes, c.state_words, through ? 0u : (unsigned)(c.tiles / p.batch), turns_of(c), words};
}

// Runs of neighbouring channels, all within 32 bits of the row's first one; a gate may be shared by whole runs
bool runs_fit(long long channels, long long share, const tfft_seq_view& gate) {
  return channels >= kRun && channels < (1LL << 28) &&
         (share == 1 ? gate.channel == 1 : share % kRun == 0 && (__int128)(channels / share) * gate.channel < (1LL << 28));
}

}  // namespace

bool rows_vector(const tfft_scan_args& p) {
  return runs_fit(p.channels, p.share, p.gate) && p.x.channel == 1 && p.y.channel == 1;
}
bool rows_vector(const tfft_scan_grad_args& p) {
  return runs_fit(p.channels, p.share, p.gate) && p.dy.channel == 1 && p.y.channel == 1 && p.dx.channel == 1 &&
         (p.share > 1 ? runs_fit(p.channels, p.share, p.dgate) : p.dgate.channel == 1);
}

static int run_of_call(const tfft_scan_args& p) { return rows_vector(p) ? kRun : 1; }
static int run_of_call(const tfft_scan_grad_args& p) { return rows_vector(p) ? kRun : 1; }
static bool through_batch(const tfft_scan_args& p) {
  return through_batch(run_of_call(p), p.batch, p.channels, {&p.x, &p.gate, &p.y});
}
static bool through_batch(const tfft_scan_grad_args& p) {
  return through_batch(run_of_call(p), p.batch, p.channels, {&p.dy, &p.y, &p.gate, &p.dx, &p.dgate});
}
static bool long_pieces(const tfft_scan_args& p) {
  return p.dtype != TFFT_F32 && rows_vector(p) && (p.share == 1 ? p.length > kMaxWaves * kSteps : p.length >= kLongShared);
}
Chunking plan_rows(const tfft_scan_args& p) {
  return plan(p.batch, p.length, p.channels, run_of_call(p), 64, through_batch(p), long_pieces(p) ? kStepsLong : kSteps, p.lengths != nullptr);
}

// Lanes whose terms a wave sums: all that share a gate, or where those are more than a wave, as large a part of them as divides them. A
// tile fills as many lanes as such groups do.
static int lanes_of(const tfft_scan_grad_args& p) {
  if (p.share == 1) return 1;
  int lanes = 64;
  while (p.share / run_of_call(p) % lanes) --lanes;
  return lanes;
}
static int groups_of(const tfft_scan_grad_args& p) { return p.share == 1 ? 1 : (int)(p.share / run_of_call(p) / lanes_of(p)); }
unsigned long long rows_parts(const tfft_scan_grad_args& p) {
  return groups_of(p) > 1 ? (unsigned long long)p.batch * p.length * (p.channels / p.share) * groups_of(p) : 0;
}
Chunking plan_rows(const tfft_scan_grad_args& p) {
  return plan(p.batch, p.length, p.channels, run_of_call(p), 64 / lanes_of(p) * lanes_of(p), through_batch(p), steps_backward(p.dtype, rows_vector(p) && p.share > 1), p.lengths != nullptr);
}
// Rows that pass through in whole lines (the gate's too, where every channel has one): B = 8, L = 4096, D = 2048 with fp32 gates
// takes 103 us forward and 170 back as a stream, 111 and 183 without; D = 2050, where tiles share lines, 142 and 265 against 125
// and 222.
static bool streams(std::initializer_list<std::pair<const tfft_seq_view*, int>> views, long long batch, long long length) {
  for (const auto& [v, dtype] : views) {
    const long long stride[2] = {v->batch, v->time}, extent[2] = {batch, length};
    if (!whole_lines(v->data, dtype, stride, extent)) return false;
  }
  return true;
}

void launch_rows(const tfft_scan_args& p, const Chunking& c, word* words, hipStream_t s) {
  const bool vector = rows_vector(p);
  const bool stream = p.channels % kRun == 0 && streams({{&p.x, p.dtype}, {&p.y, p.dtype}}, p.batch, p.length) &&
                      (p.share > 1 || streams({{&p.gate, p.gate_dtype}}, p.batch, p.length));
  const Shape f = shape_of(p, c, run_of_call(p), through_batch(p), words);
  const dim3 grid((unsigned)c.blocks()), block(64 * c.waves);
  with_types(p.dtype, p.gate_dtype, [&](auto t, auto g) {
    using T = decltype(t);
    using G = decltype(g);
    constexpr int V = kRun;
    const auto launch = [&](auto steps) {
      constexpr int S = decltype(steps)::value;
      if (p.share == 1 && stream) scan_rows_fwd<T, G, V, V, true, S><<<grid, block, 0, s>>>(p, f);
      else if (p.share == 1) scan_rows_fwd<T, G, V, V, false, S><<<grid, block, 0, s>>>(p, f);
      else if (stream) scan_rows_fwd<T, G, V, 1, true, S><<<grid, block, 0, s>>>(p, f);
      else scan_rows_fwd<T, G, V, 1, false, S><<<grid, block, 0, s>>>(p, f);
    };
    if (!vector) return scan_rows_fwd<T, G, 1, 1, false, kSteps><<<grid, block, 0, s>>>(p, f);
    if constexpr (sizeof(T) == 2)
      if (long_pieces(p)) return launch(std::integral_constant<int, kStepsLong>());
    launch(std::integral_constant<int, kSteps>());
  });
}

void launch_rows(const tfft_scan_grad_args& p, const Chunking& c, word* words, float* parts, hipStream_t s) {
  const bool vector = rows_vector(p);
  const bool stream = p.channels % kRun == 0 && c.lanes == 64 && streams({{&p.dy, p.dtype}, {&p.y, p.dtype}, {&p.dx, p.dtype}}, p.batch, p.length) &&
                      (p.share > 1 || streams({{&p.gate, p.gate_dtype}, {&p.dgate, p.gate_dtype}}, p.batch, p.length));
  const Shape f = shape_of(p, c, run_of_call(p), through_batch(p), words);
  const dim3 grid((unsigned)c.blocks()), block(64 * c.waves);
  const int lanes = lanes_of(p), groups = groups_of(p);
  const bool odd = lanes & (lanes - 1) || groups > 1;
  if (groups == 1) parts = nullptr;
  with_types(p.dtype, p.gate_dtype, [&](auto t, auto g) {
    using T = decltype(t);
    using G = decltype(g);
    constexpr int V = kRun;
    if (!vector && odd) scan_rows_bwd<T, G, 1, 1, false, ODD><<<grid, block, 0, s>>>(p, f, parts, lanes);
    else if (!vector) scan_rows_bwd<T, G, 1, 1, false><<<grid, block, 0, s>>>(p, f, parts, lanes);
    else if (odd) scan_rows_bwd<T, G, V, 1, false, ODD><<<grid, block, 0, s>>>(p, f, parts, lanes);
    else if (p.share == 1 && stream) scan_rows_bwd<T, G, V, V, true><<<grid, block, 0, s>>>(p, f, parts, lanes);
    else if (p.share == 1) scan_rows_bwd<T, G, V, V, false><<<grid, block, 0, s>>>(p, f, parts, lanes);
    else if (stream) scan_rows_bwd<T, G, V, 1, true><<<grid, block, 0, s>>>(p, f, parts, lanes);
    else scan_rows_bwd<T, G, V, 1, false><<<grid, block, 0, s>>>(p, f, parts, lanes);
    if (parts && p.length > 0) {
      const long long n = p.batch * p.length * (p.channels / p.share);
      sum_parts<G><<<(unsigned)std::min((n + 15) / 16, 1LL << 16), 256, 0, s>>>(p, parts, groups);
    }
  });
}

}  // namespace tfft_seq
