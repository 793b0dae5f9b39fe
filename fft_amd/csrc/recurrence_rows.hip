// The gated linear recurrence where neighbouring channels lie side by side ([batch][time][channel]), and, one element
// at a time, for any other strides.
#include <initializer_list>
#include <type_traits>

#include "recurrence_kernels.hpp"

namespace tfft_seq {
namespace {

// A lane holds a run of V channels of one batch entry over S steps, a wave 64 runs, a workgroup `waves` pieces of S steps one
// behind the other. Channels are counted over the whole batch (each entry padded to whole runs), so few channels
// fill a wave too.
#ifndef FS
#define FS 16
#define FW 8
#define FO 4
#endif
constexpr int kSteps = FS, kMaxWaves = FW, kMaxGroup = 16, kResident = 512;
template <class T>
constexpr int run_of = 2;

// Runs take 32-bit offsets, which the plan has checked; single elements may lie anywhere
template <int V>
using offset_of = std::conditional_t<V == 1, long long, uint32_t>;

struct Shape {
  int batch, length, channels, padded;  // padded: channels rounded up to whole runs
  int share, log_gate;
  int chunks, group;
  long long state_words;
  unsigned tiles, tiles_of_entry;  // 0 tiles of an entry: tiles run through the whole batch
  word* words;
};

// Lane's place: first channel n among the states, batch entry b, channel c, valid channels of the run. first: the batch entry
// that the tile's addresses start from, the same for all lanes.
struct Place {
  unsigned n;
  int b, c, valid, first;
};
template <int V>
__device__ __forceinline__ Place place_of(const Shape& f, unsigned tile, int lane) {
  Place p;
  p.n = tile * (64u * V) + lane * V;
  if (f.tiles_of_entry == 0) {
    p.first = 0;
    p.b = p.n / (unsigned)f.padded;
    p.c = p.n - p.b * (unsigned)f.padded;
  } else {
    p.first = p.b = tile / f.tiles_of_entry;
    p.c = (tile - p.b * f.tiles_of_entry) * (64 * V) + lane * V;
  }
  p.valid = p.b >= f.batch || p.c >= f.channels ? 0 : min(V, f.channels - p.c);
  if (p.valid == 0) p.b = p.first, p.c = 0;
  return p;
}

// One of the tensors at a lane's place: an address that the wave shares, in scalar registers, and the lane's offset in bytes.
// Vector kernels take 32-bit offsets, so that a load needs no vector register but those that it fills.
template <class T, class Off>
struct Lane {
  char* base;
  Off off;
  long long step;  // bytes from one time step to the next
  __device__ __forceinline__ Lane(const tfft_seq_view& v, const Place& p, int c)
      : base((char*)v.data + p.first * v.batch * (long long)sizeof(T)),
        off((Off)(((p.b - p.first) * v.batch + c * v.channel) * (long long)sizeof(T))),
        step(v.time * (long long)sizeof(T)) {}
  __device__ __forceinline__ T* at(int t) const { return (T*)(base + t * step + off); }
};

// What ran before this chunk: the state at its start, from the words of earlier chunks. Called by all threads of a workgroup
// with the (A, B) of its whole chunk in the last wave. Publishes this chunk's own words on the way.
template <int V>
struct Lookback {
  float A[kMaxGroup][64 * V], B[kMaxGroup][64 * V], h[64 * V];
};
template <int V>
__device__ __forceinline__ void state_before(const Shape& f, Lookback<V>& lds, unsigned chunk, long long n, int wave, int waves,
                                             int lane, const float (&A)[V], const float (&B)[V], float (&h)[V]) {
  // h comes in as the state before the first chunk
  if (f.chunks <= 1) return;
  word* parts = f.words + 1;
  word* states = parts + (f.group > 1 ? 2 * f.state_words * f.chunks : 0);
  const int r = chunk % f.group, q = chunk / f.group;
  const bool last = wave == waves - 1, more = chunk + 1 < (unsigned)f.chunks;
  if (f.group > 1) {
    if (last && more && r != f.group - 1) {
      word* own = parts + 2 * f.state_words * chunk + n;
#pragma unroll
      for (int v = 0; v < V; ++v) publish(own + v, A[v]), publish(own + f.state_words + v, B[v]);
    }
    for (int k = wave; k < r; k += waves) {
      const word* from = parts + 2 * f.state_words * (chunk - r + k) + n;
      float a[V], b[V];
#pragma unroll
      for (int v = 0; v < V; ++v) a[v] = await(from + v), b[v] = await(from + f.state_words + v);
#pragma unroll
      for (int v = 0; v < V; ++v) lds.A[k][lane * V + v] = a[v], lds.B[k][lane * V + v] = b[v];
    }
  }
  if (last) {
    if (q > 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = await(states + f.state_words * (q - 1) + n + v);
    }
    if (f.group == 1 && more) {
#pragma unroll
      for (int v = 0; v < V; ++v) publish(states + f.state_words * q + n + v, join(A[v], h[v], B[v]));
    }
#pragma unroll
    for (int v = 0; v < V; ++v) lds.h[lane * V + v] = h[v];
  }
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = lds.h[lane * V + v];
  for (int k = 0; k < r; ++k) {
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = join(lds.A[k][lane * V + v], h[v], lds.B[k][lane * V + v]);
  }
  if (f.group > 1 && last && more && r == f.group - 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) publish(states + f.state_words * q + n + v, join(A[v], h[v], B[v]));
  }
}

// Chunk and tile of this workgroup: a ticket where chunks depend on each other
__device__ __forceinline__ unsigned take(const Shape& f, unsigned* ticket) {
  if (f.chunks <= 1) return blockIdx.x;
  if (threadIdx.x == 0) *ticket = (unsigned)__hip_atomic_fetch_add(f.words, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(*ticket);
}

// The (A, B) in front of each wave's piece, and behind the last wave's the chunk's
template <int V>
struct Pieces {
  float A[kMaxWaves][64 * V], B[kMaxWaves][64 * V];
};
template <int V>
__device__ __forceinline__ void join_pieces(Pieces<V>& lds, int wave, int waves, int lane, const float (&A)[V], const float (&B)[V],
                                            float (&front_a)[V], float (&front_b)[V], float (&chunk_a)[V], float (&chunk_b)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) lds.A[wave][lane * V + v] = A[v], lds.B[wave][lane * V + v] = B[v];
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v) front_a[v] = 1.0f, front_b[v] = 0.0f;
  for (int w = 0; w < wave; ++w) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float a = lds.A[w][lane * V + v];
      front_b[v] = join(a, front_b[v], lds.B[w][lane * V + v]);
      front_a[v] *= a;
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) chunk_a[v] = front_a[v] * A[v], chunk_b[v] = join(A[v], front_b[v], B[v]);
}

// Decays of S steps of a lane, one for the run (VG = 1) or one a channel; 1 behind the sequence
template <int S, int VG, class G, class Off>
__device__ __forceinline__ void load_decays(const Lane<G, Off>& g, int t0, int len, int valid, int log_gate, float (&a)[S][VG]) {
  const int vg = min(valid, VG);
  if (__all(t0 + S <= len && vg == VG)) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const Run<G, VG> r = load_run<G, VG>(g.at(t0 + s));
#pragma unroll
      for (int v = 0; v < VG; ++v) a[s][v] = r.get(v);
    }
  } else {
#pragma unroll
    for (int s = 0; s < S; ++s) {
#pragma unroll
      for (int v = 0; v < VG; ++v) a[s][v] = log_gate ? 0.0f : 1.0f;
      if (t0 + s < len && vg > 0) {
        const Run<G, VG> r = load_some<VG>(g.at(t0 + s), vg);
#pragma unroll
        for (int v = 0; v < VG; ++v) a[s][v] = r.get(v);
      }
    }
  }
  if (log_gate) {
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int v = 0; v < VG; ++v) a[s][v] = exp_decay(a[s][v]);
  }
}

// Values of the same steps; 0 outside the sequence
template <int S, int V, class T, class Off>
__device__ __forceinline__ void load_values(const Lane<T, Off>& x, int t0, int len, int valid, Run<T, V> (&r)[S]) {
  if (__all(t0 >= 0 && t0 + S <= len && valid == V)) {
#pragma unroll
    for (int s = 0; s < S; ++s) r[s] = load_run<T, V>(x.at(t0 + s));
  } else {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      r[s].clear();
      if (t0 + s >= 0 && t0 + s < len && valid > 0) r[s] = load_some<V>(x.at(t0 + s), valid);
    }
  }
}

template <int V>
__device__ __forceinline__ void load_state(const float* from, const Place& p, int channels, float (&h)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = from && v < p.valid ? from[(long long)p.b * channels + p.c + v] : 0.0f;
}
template <int V>
__device__ __forceinline__ void store_state(float* to, const Place& p, int channels, const float (&h)[V]) {
  if (!to) return;
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (v < p.valid) to[(long long)p.b * channels + p.c + v] = h[v];
}

template <class T, class G, int V, int VG>
__global__ __launch_bounds__(64 * kMaxWaves, FO) void scan_rows_fwd(tfft_scan_args p, Shape f) {
  constexpr int S = kSteps;
  __shared__ Pieces<V> pieces;
  __shared__ Lookback<V> lookback;
  __shared__ unsigned ticket;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const unsigned turn = take(f, &ticket), chunk = turn / f.tiles, tile = turn - chunk * f.tiles;
  const Place at = place_of<V>(f, tile, lane);
  const int len = steps_of(p.lengths, at.b, f.length), t0 = (int)(chunk * waves + wave) * S;
  using Off = offset_of<V>;
  const Lane<T, Off> x(p.x, at, at.c), y(p.y, at, at.c);
  const Lane<G, Off> g(p.gate, at, f.share == 1 ? at.c : at.c / f.share);
  float a[S][VG];
  Run<T, V> xr[S];
  load_values<S, V>(x, t0, len, at.valid, xr);
  load_decays<S, VG>(g, t0, len, at.valid, f.log_gate, a);
  float h[V];
  load_state<V>(p.initial, at, f.channels, h);

  float A[V], B[V], front_a[V], front_b[V], chunk_a[V], chunk_b[V];
#pragma unroll
  for (int v = 0; v < V; ++v) A[v] = 1.0f, B[v] = 0.0f;
#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      A[v] *= a[s][v % VG];
      B[v] = fmaf(a[s][v % VG], B[v], xr[s].get(v));
    }
  join_pieces<V>(pieces, wave, waves, lane, A, B, front_a, front_b, chunk_a, chunk_b);
  state_before<V>(f, lookback, chunk, at.n, wave, waves, lane, chunk_a, chunk_b, h);
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = join(front_a[v], h[v], front_b[v]);

  if (__all(t0 + S <= len && at.valid == V)) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      Run<T, V> r;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        h[v] = fmaf(a[s][v % VG], h[v], xr[s].get(v));
        r.set(v, h[v]);
      }
      store_run<T, V>(y.at(t0 + s), r);
    }
  } else {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      Run<T, V> r;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        h[v] = fmaf(a[s][v % VG], h[v], xr[s].get(v));
        r.set(v, t0 + s < len ? h[v] : 0.0f);
      }
      if (t0 + s < f.length) store_some<V>(y.at(t0 + s), r, at.valid);
    }
  }
  if (chunk + 1 == (unsigned)f.chunks && wave == waves - 1) store_state<V>(p.last, at, f.channels, h);
}

// Backwards in time: chunk 0 is the latest, wave 0 has the latest piece. `lanes`: lanes that share a gate, 0 where each
// channel's term goes to `parts` (fp32 [batch][time][channel]) to be summed by a kernel behind.
template <class T, class G, int V, int VG>
__global__ __launch_bounds__(64 * kMaxWaves, FO) void scan_rows_bwd(tfft_scan_grad_args p, Shape f, float* parts, int lanes) {
  constexpr int S = kSteps;
  __shared__ Pieces<V> pieces;
  __shared__ Lookback<V> lookback;
  __shared__ unsigned ticket;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const unsigned turn = take(f, &ticket), chunk = turn / f.tiles, tile = turn - chunk * f.tiles;
  const Place at = place_of<V>(f, tile, lane);
  const int len = steps_of(p.lengths, at.b, f.length);
  const int t0 = ((int)(f.chunks - 1 - chunk) * waves + (waves - 1 - wave)) * S;
  using Off = offset_of<V>;
  const int gate = f.share == 1 ? at.c : at.c / f.share;
  const Lane<T, Off> dy(p.dy, at, at.c), y(p.y, at, at.c), dx(p.dx, at, at.c);
  const Lane<G, Off> g(p.gate, at, gate), dg(p.dgate, at, gate);
  float a[S][VG];
  Run<T, V> d[S], before[S];
  load_values<S, V>(dy, t0, len, at.valid, d);
  load_decays<S, VG>(g, t0, len, at.valid, f.log_gate, a);
  load_values<S, V>(y, t0 - 1, len, at.valid, before);
  float c[V];
  load_state<V>(p.dlast, at, f.channels, c);

  float A[V], B[V], front_a[V], front_b[V], chunk_a[V], chunk_b[V];
#pragma unroll
  for (int v = 0; v < V; ++v) A[v] = 1.0f, B[v] = 0.0f;
#pragma unroll
  for (int s = S - 1; s >= 0; --s)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      A[v] *= a[s][v % VG];
      B[v] = a[s][v % VG] * (B[v] + d[s].get(v));
    }
  join_pieces<V>(pieces, wave, waves, lane, A, B, front_a, front_b, chunk_a, chunk_b);
  state_before<V>(f, lookback, chunk, at.n, wave, waves, lane, chunk_a, chunk_b, c);
#pragma unroll
  for (int v = 0; v < V; ++v) c[v] = join(front_a[v], c[v], front_b[v]);

  float start[V];
  load_state<V>(p.initial, at, f.channels, start);
  const auto walk = [&](auto whole) {
#pragma unroll
    for (int s = S - 1; s >= 0; --s) {
      const int t = t0 + s;
      Run<T, V> r;
      float da[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float e = d[s].get(v) + c[v], k = a[s][v % VG];
        float state = before[s].get(v);
        if (s == 0) state = t == 0 ? start[v] : state;
        r.set(v, whole.value || t < len ? e : 0.0f);
        c[v] = k * e;
        da[v] = (f.log_gate ? c[v] : e) * state;
        if (!whole.value) da[v] = t < len ? da[v] : 0.0f;
      }
      const bool in = whole.value || t < f.length;
      const int valid = whole.value ? V : at.valid;
      if (in) store_some<V>(dx.at(t), r, valid);
      if (f.share == 1) {
        Run<G, V> q;
#pragma unroll
        for (int v = 0; v < V; ++v) q.set(v, da[v]);
        if (in) store_some<V>(dg.at(t), q, valid);
      } else if (lanes > 0) {
        float sum = da[0];
#pragma unroll
        for (int v = 1; v < V; ++v) sum += da[v];
        for (int m = 1; m < lanes; m *= 2) sum += __shfl_xor(sum, m);
        if (in && valid > 0 && (lane & (lanes - 1)) == 0) {
          Run<G, 1> q;
          q.set(0, sum);
          store_run<G, 1>(dg.at(t), q);
        }
      } else if (in) {
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (v < valid) parts[((long long)at.b * f.length + t) * f.channels + at.c + v] = da[v];
      }
    }
  };
  if (__all(t0 + S <= len && at.valid == V)) walk(std::true_type());
  else walk(std::false_type());
  if (chunk + 1 == (unsigned)f.chunks && wave == waves - 1) store_state<V>(p.dinitial, at, f.channels, c);
}

// dgate of a shared gate: its channels' terms summed in their order
template <class G>
__global__ __launch_bounds__(256) void sum_shares(tfft_scan_grad_args p, const float* parts) {
  const long long gates = p.channels / p.share, n = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (n >= p.batch * p.length * gates) return;
  const long long g = n % gates, bt = n / gates, b = bt / p.length, t = bt % p.length;
  const float* from = parts + bt * p.channels + g * p.share;
  float sum = 0.0f;
  for (long long i = 0; i < p.share; ++i) sum += from[i];
  ((G*)p.dgate.data)[b * p.dgate.batch + t * p.dgate.time + g * p.dgate.channel] = from_f32<G>(sum);
}

int run_length(int dtype) { return dtype == TFFT_F32 ? run_of<float> : run_of<f16>; }

// Tiles run through the whole batch where that keeps a lane's offsets within 32 bits, so that few channels fill a wave too; else
// each batch entry has tiles of its own.
bool through_batch(int run, long long batch, long long channels, std::initializer_list<const tfft_seq_view*> views) {
  if (run == 1) return true;
  for (const tfft_seq_view* v : views)
    if ((__int128)(batch - 1) * v->batch + (__int128)(channels - 1) * v->channel >= (1LL << 32) / 4 - run) return false;
  return true;
}

Chunking plan(long long batch, long long length, long long channels, int run, bool through) {
  constexpr int steps = kSteps;
  Chunking c;
  const long long padded = (channels + run - 1) / run * run, width = 64 * run;
  c.tiles = through ? (batch * padded + width - 1) / width : batch * ((channels + width - 1) / width);
  c.waves = (int)(length > (kMaxWaves - 1) * steps ? kMaxWaves : length < steps ? 1 : (length + steps - 1) / steps);
  c.chunks = (length + c.waves * steps - 1) / (c.waves * steps);
  if (c.chunks < 1) c.chunks = 1;
  c.state_words = c.tiles * width;
  // About kResident workgroups run at once, kResident / tiles chunks of each tile. That many are joined directly, so that few
  // channels wait for one state in that many chunks, and many channels do not read what they need not: B = 8,
  // L = 4096, D = 2048 (128 tiles) takes 118, 121, 129 us with groups of 4, 8, 16; one sequence of 65537 steps
  // and 1024 channels (8 tiles) 180, 129, 119 us.
  while (c.group < kMaxGroup && c.group * c.tiles < kResident) c.group *= 2;
  return c;
}

template <class P>
Shape shape_of(const P& p, const Chunking& c, int run, bool through, word* words) {
  return Shape{(int)p.batch, (int)p.length, (int)p.channels, (int)((p.channels + run - 1) / run * run), (int)p.share,
               p.gate_form == TFFT_GATE_LOG, (int)c.chunks, c.group, c.state_words, (unsigned)c.tiles,
               through ? 0u : (unsigned)(c.tiles / p.batch), words};
}

bool gate_fits(const tfft_seq_view& gate, long long share, int run) { return share == 1 ? gate.channel == 1 : share % run == 0; }

}  // namespace

bool rows_vector(const tfft_scan_args& p) {
  return p.x.channel == 1 && p.y.channel == 1 && gate_fits(p.gate, p.share, run_length(p.dtype));
}
bool rows_vector(const tfft_scan_grad_args& p) {
  return p.dy.channel == 1 && p.y.channel == 1 && p.dx.channel == 1 && gate_fits(p.gate, p.share, run_length(p.dtype)) &&
         (p.share > 1 || p.dgate.channel == 1);
}

static int run_of_call(const tfft_scan_args& p) { return rows_vector(p) ? run_length(p.dtype) : 1; }
static int run_of_call(const tfft_scan_grad_args& p) { return rows_vector(p) ? run_length(p.dtype) : 1; }
static bool through_batch(const tfft_scan_args& p) {
  return through_batch(run_of_call(p), p.batch, p.channels, {&p.x, &p.gate, &p.y});
}
static bool through_batch(const tfft_scan_grad_args& p) {
  return through_batch(run_of_call(p), p.batch, p.channels, {&p.dy, &p.y, &p.gate, &p.dx, &p.dgate});
}
Chunking plan_rows(const tfft_scan_args& p) { return plan(p.batch, p.length, p.channels, run_of_call(p), through_batch(p)); }
Chunking plan_rows(const tfft_scan_grad_args& p) { return plan(p.batch, p.length, p.channels, run_of_call(p), through_batch(p)); }

// Lanes that share a gate, where whole power-of-two groups of a wave's lanes do; 0: summed by a kernel of its own
static int lanes_of(const tfft_scan_grad_args& p) {
  const int run = run_of_call(p);
  if (p.share % run) return 0;
  const long long lanes = p.share / run;
  return lanes <= 64 && (lanes & (lanes - 1)) == 0 ? (int)lanes : 0;
}
bool rows_sums_shares(const tfft_scan_grad_args& p) { return p.share > 1 && lanes_of(p) == 0; }

void launch_rows(const tfft_scan_args& p, const Chunking& c, word* words, hipStream_t s) {
  const bool vector = rows_vector(p);
  const Shape f = shape_of(p, c, run_of_call(p), through_batch(p), words);
  const dim3 grid((unsigned)(c.tiles * c.chunks)), block(64 * c.waves);
  with_types(p.dtype, p.gate_dtype, [&](auto t, auto g) {
    using T = decltype(t);
    using G = decltype(g);
    constexpr int V = run_of<T>;
    if (!vector) scan_rows_fwd<T, G, 1, 1><<<grid, block, 0, s>>>(p, f);
    else if (p.share == 1) scan_rows_fwd<T, G, V, V><<<grid, block, 0, s>>>(p, f);
    else scan_rows_fwd<T, G, V, 1><<<grid, block, 0, s>>>(p, f);
  });
}

void launch_rows(const tfft_scan_grad_args& p, const Chunking& c, word* words, float* parts, hipStream_t s) {
  const bool vector = rows_vector(p);
  const Shape f = shape_of(p, c, run_of_call(p), through_batch(p), words);
  const dim3 grid((unsigned)(c.tiles * c.chunks)), block(64 * c.waves);
  const int lanes = lanes_of(p);
  with_types(p.dtype, p.gate_dtype, [&](auto t, auto g) {
    using T = decltype(t);
    using G = decltype(g);
    constexpr int V = run_of<T>;
    if (!vector) scan_rows_bwd<T, G, 1, 1><<<grid, block, 0, s>>>(p, f, parts, lanes);
    else if (p.share == 1) scan_rows_bwd<T, G, V, V><<<grid, block, 0, s>>>(p, f, parts, lanes);
    else scan_rows_bwd<T, G, V, 1><<<grid, block, 0, s>>>(p, f, parts, lanes);
    if (rows_sums_shares(p) && p.length > 0) {
      const long long n = p.batch * p.length * (p.channels / p.share);
      sum_shares<G><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(p, parts);
    }
  });
}

}  // namespace tfft_seq
