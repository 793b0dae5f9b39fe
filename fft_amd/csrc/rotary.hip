// Rotary positions: pairs of values times exp(2 pi i p F[i]) for 64-bit positions p and fixed-point frequencies F
// (tfft_rotary). No counterpart in the reference.
#include <type_traits>

#include "seq_common.hpp"

namespace {
using namespace tfft_seq;

// cos and sin of `phase` 2^-64 turns, rounded to 2^-32 turns. For 16-bit values the chip's own functions, which take turns:
// within 1.25e-7 of the fp64 values on such arguments (the rounded argument adds 0.9e-7), nothing beside the rounding of
// the result. For fp32 the quadrant is taken off in integers, so that what is left, |r| <= 1/8 turn, is off by 2^-24 of
// itself; the Taylor sums to r^9 and r^10 are within 2e-9 there.
template <class T>
__device__ __forceinline__ void turn(uint64_t phase, float* c, float* s) {
  if constexpr (sizeof(T) == 2) {
    const float turns = (float)(int)(uint32_t)((phase + 0x80000000ull) >> 32) * (1.0f / 4294967296.0f);
    *c = __builtin_amdgcn_cosf(turns);
    *s = __builtin_amdgcn_sinf(turns);
  } else {
    const uint32_t top = (uint32_t)((phase + 0x2000000080000000ull) >> 32);
    const int rest = (int)(top & 0x3fffffffu) - 0x20000000;
    const float r = (float)rest * (6.283185307179586f / 4294967296.0f), q = r * r;
    const float sn = r + r * q * (-1.0f / 6 + q * (1.0f / 120 + q * (-1.0f / 5040 + q * (1.0f / 362880))));
    const float cs = 1.0f + q * (-0.5f + q * (1.0f / 24 + q * (-1.0f / 720 + q * (1.0f / 40320 + q * (-1.0f / 3628800)))));
    const uint32_t quadrant = top >> 30;
    const float a = quadrant & 1 ? sn : cs, b = quadrant & 1 ? cs : sn;
    *c = (quadrant == 1 || quadrant == 2) ? -a : a;
    *s = quadrant >= 2 ? -b : b;
  }
}

// What bounds it: HBM. 8 x 4096 tokens with 32 + 8 heads of 128 in bf16 take 116 us (671 MB, 5.8 TB/s); the factors, evaluated in
// registers from 8 bytes a pair, hide behind it. One token each of 64 sequences takes 4 us, a launch and its latency.
//
// A unit is what a thread holds of one head: R values of each half (pairs i, i + rotary / 2), twice as many pairs, or R values
// with their R / 2 interleaved pairs; behind the rotated ones, R values to copy. R is kRun<T> (16 bytes), or kShortRun in heads
// that have fewer values. A unit that reaches over the end of the head is loaded as the head's last R values and moved to where it
// belongs: all loads are whole runs on one path, because one whose registers two paths could fill is waited for where they meet
// (5 x 2489 tokens with 21 heads of 174 in fp16 take 49 us, 76 when the last units are loaded value by value).
template <class T>
constexpr int kRun = 16 / sizeof(T);
constexpr int kShortRun = 2;

// A thread evaluates the factors of its unit once and turns it in the heads hl, hl + lanes, ... of its token, the second
// tensor's heads counted behind the first's. Neighbouring threads have neighbouring units, then neighbouring heads: a wave
// reads whole lines.
struct Grid {
  unsigned units, turned;  // of a head, and how many of them are rotated
  unsigned lanes;          // threads that share the heads of a token
  unsigned heads;          // of both tensors
  unsigned threads;
};

template <class T>
struct Token {
  const T* in;
  T* out;
  long long in_head, out_head;
  __device__ __forceinline__ Token(const tfft_rotary_view& v, long long b, long long t)
      : in((const T*)v.in + b * v.in_batch + t * v.in_time), out((T*)v.out + b * v.out_batch + t * v.out_time),
        in_head(v.in_head), out_head(v.out_head) {}
};

template <int R, bool STREAM, class T>
__device__ __forceinline__ void put(T* to, const Run<T, R>& r, int valid) {
  if constexpr (STREAM) store_run<T, R, true>(to, r);  // all units are whole
  else if (valid == R) store_run<T, R>(to, r);
  else store_head<R>(to, r, valid);
}

template <class T, bool HALF, int R, int NH, bool STREAM>
__global__ __launch_bounds__(256) void rotary_units(tfft_rotary_args p, Grid g) {
  constexpr int pairs = HALF ? R : R / 2;
  const unsigned n = blockIdx.x * 256u + threadIdx.x;
  if (n >= g.threads) return;
  const unsigned a_token = g.units * g.lanes, token = n / a_token, rest = n - token * a_token;
  const unsigned entry = token / (unsigned)p.length;
  const long long b = entry, t = token - entry * (unsigned)p.length;
  const unsigned hl = rest / g.units, u = rest - hl * g.units;
  const Token<T> first(p.tensor[0], b, t), second(p.tensor[1], b, t);
  const unsigned heads0 = (unsigned)p.tensor[0].heads;
  const int half = p.rotary / 2;
  const bool turned = u < g.turned;
  // where the unit's values lie in the head, and how many of them are there
  const int at = turned ? (int)u * R : p.rotary + (int)(u - g.turned) * R;
  const int valid = min(R, turned ? (HALF ? half - at : p.rotary - at) : p.head - at);

  // where the unit's runs are loaded, and how many values too early
  const int from_x = min(at, p.head - R), from_y = min(at + half, p.head - R);

  float c[pairs], s[pairs];
  if (turned) {
    long long pos = p.first + t;
    const long long i = b * p.position_batch + t * p.position_time;
    if (p.positions) pos = p.position_bytes == 8 ? ((const long long*)p.positions)[i] : ((const int*)p.positions)[i];
    const uint64_t* f = (const uint64_t*)p.turns + (HALF ? at : at / 2);
#pragma unroll
    for (int k = 0; k < pairs; ++k) {
      turn<T>((HALF ? k : 2 * k) < valid ? (uint64_t)pos * f[k] : 0, &c[k], &s[k]);
      c[k] *= p.magnitude;
      s[k] *= p.inverse ? -p.magnitude : p.magnitude;
    }
  }
  for (unsigned h0 = hl; h0 < g.heads; h0 += NH * g.lanes) {
    Run<T, R> x[NH], y[NH];
#pragma unroll
    for (int j = 0; j < NH; ++j) {
      const unsigned h = h0 + j * g.lanes;
      if (h < g.heads) {
        const bool one = h < heads0;
        const long long i = one ? h : h - heads0;
        const T* from = one ? first.in + i * first.in_head : second.in + i * second.in_head;
        x[j] = load_run<T, R>(from + from_x);
        if (HALF && turned) y[j] = load_run<T, R>(from + from_y);
      }
    }
#pragma unroll
    for (int j = 0; j < NH; ++j) {
      const unsigned h = h0 + j * g.lanes;
      if (h >= g.heads) continue;
      const bool one = h < heads0;
      const long long i = one ? h : h - heads0;
      T* to = (one ? first.out + i * first.out_head : second.out + i * second.out_head) + at;
      move_down<R>(x[j], at - from_x);
      if (turned) {
        if (HALF) move_down<R>(y[j], at + half - from_y);
        float re[R], im[R];
#pragma unroll
        for (int k = 0; k < pairs; ++k) {
          const float v = x[j].get(HALF ? k : 2 * k), w = HALF ? y[j].get(k) : x[j].get(HALF ? k : 2 * k + 1);
          const float a = v * c[k] - w * s[k], d = v * s[k] + w * c[k];
          if (HALF) re[k] = a, im[k] = d;
          else re[2 * k] = a, re[2 * k + 1] = d;
        }
        x[j].set_all(re);
        if (HALF) {
          y[j].set_all(im);
          put<R, STREAM>(to + half, y[j], valid);
        }
      }
      put<R, STREAM>(to, x[j], valid);
    }
  }
}

// Heads whose factors a thread shares: 8 x 4096 tokens with 32 + 8 heads of 128 in bf16 take 153, 119, 116, 121, 123 us with
// 1, 2, 4, 5, 8, 5 x 2489 with 21 heads of 174 in fp16 58, 51, 49, 49, 50. Calls that would be left with fewer than kEnough
// threads (256 CUs of 1024) give every head its own.
constexpr int kHeads = 4;
constexpr long long kEnough = 256 * 1024, kMost = 1LL << 30;

int refuse(const char* why, int code = TFFT_ERR_INVALID) {
  char text[256];
  snprintf(text, sizeof text, "tfft_rotary: %s", why);
  return tfft_internal_fail(code, text);
}

}  // namespace

extern "C" int tfft_rotary(const tfft_rotary_args* args, void* stream) {
  if (!args || args->struct_size != (int)sizeof *args) return refuse("null arguments, or struct_size is not theirs");
  tfft_rotary_args p = *args;
  if (p.dtype < TFFT_F32 || p.dtype > TFFT_BF16) return refuse("element types: fp32, fp16 or bf16", TFFT_ERR_UNSUPPORTED);
  if (p.pairs != TFFT_PAIRS_HALF && p.pairs != TFFT_PAIRS_INTERLEAVED) return refuse("unknown layout of pairs");
  if (p.batch < 0 || p.length < 0 || p.head < 0 || p.tensor[0].heads < 0 || p.tensor[1].heads < 0) return refuse("negative extent");
  if (p.rotary < 2 || p.rotary % 2 || p.rotary > p.head) return refuse("rotary is even and between 2 and head");
  if (p.positions && p.position_bytes != 4 && p.position_bytes != 8) return refuse("position_bytes is 4 or 8");
  if (!p.turns) return refuse("no frequencies");
  if (!p.tensor[1].in) p.tensor[1].heads = 0;
  if (p.batch > kMost || p.length > kMost || p.head > kMost || p.tensor[0].heads > kMost / 4 || p.tensor[1].heads > kMost / 4)
    return refuse("an extent is too large");
  // Results that leave in whole lines and whole units are streamed: 8 x 4096 tokens with 32 + 8 heads of 128 in bf16 116 us
  // against 126, 160000 tokens with 12 heads of 96 in fp32 269 against 288.
  const long long size = p.dtype == TFFT_F32 ? 4 : 2;
  bool in_place = true, stream_out = p.rotary / 2 * size % 16 == 0 && p.head * size % 16 == 0;
  for (const tfft_rotary_view& v : p.tensor) {
    const long long extent[4] = {p.batch, p.length, v.heads, p.head};
    const long long in[4] = {v.in_batch, v.in_time, v.in_head, 1}, out[4] = {v.out_batch, v.out_time, v.out_head, 1};
    if (const char* why = check_tensor(v.in, p.dtype, in, extent, false)) return refuse(why);
    if (const char* why = check_tensor(v.out, p.dtype, out, extent, true)) return refuse(why);
    if (v.heads == 0 || p.batch == 0 || p.length == 0) continue;
    const bool here = v.in == v.out;
    for (int i = 0; i < 3; ++i)
      if (here && extent[i] > 1 && in[i] != out[i]) return refuse("in place needs equal strides on both sides");
    in_place = in_place && here;
    const long long steps[3] = {v.out_batch, v.out_time, v.out_head}, counts[3] = {p.batch, p.length, v.heads};
    stream_out = stream_out && whole_lines(v.out, p.dtype, steps, counts);
  }
  const int whole = p.dtype == TFFT_F32 ? kRun<float> : kRun<f16>, run = p.head < whole ? kShortRun : whole;
  const tfft_rotary_view &q = p.tensor[0], &k = p.tensor[1];
  if (q.heads && k.heads && p.batch && p.length && (q.out == k.out || q.out == k.in || k.out == q.in))
    return refuse("a result may not take the other tensor's place");
  Grid g;
  g.turned = ((p.pairs == TFFT_PAIRS_HALF ? p.rotary / 2 : p.rotary) + run - 1) / run;
  g.units = g.turned + (in_place ? 0 : (p.head - p.rotary + run - 1) / run);
  g.heads = (unsigned)(p.tensor[0].heads + p.tensor[1].heads);
  if (p.batch == 0 || p.length == 0 || g.heads == 0) return TFFT_OK;
  // kHeads heads a thread share its factors where that leaves enough threads to fill the chip, else one
  const bool many = run != kShortRun && (__int128)p.batch * p.length * g.units * g.heads >= (__int128)kHeads * kEnough;
  g.lanes = many ? (g.heads + kHeads - 1) / kHeads : g.heads;
  const __int128 threads = (__int128)p.batch * p.length * g.units * g.lanes;
  if (threads > 0xffff0000LL) return refuse("more tokens and heads than one launch takes");
  g.threads = (unsigned)threads;  // a launch counts its threads in 32 bits
  const unsigned grid = (g.threads + 255) / 256;
  hipStream_t stream_ = static_cast<hipStream_t>(stream);
  const auto launch = [&](auto t) {
    using T = decltype(t);
    const auto pairs = [&](auto half) {
      if (run == kShortRun) rotary_units<T, half.value, kShortRun, 1, false><<<grid, 256, 0, stream_>>>(p, g);
      else if (!many) rotary_units<T, half.value, kRun<T>, 1, false><<<grid, 256, 0, stream_>>>(p, g);
      else if (stream_out) rotary_units<T, half.value, kRun<T>, kHeads, true><<<grid, 256, 0, stream_>>>(p, g);
      else rotary_units<T, half.value, kRun<T>, kHeads, false><<<grid, 256, 0, stream_>>>(p, g);
    };
    if (p.pairs == TFFT_PAIRS_HALF) pairs(std::true_type());
    else pairs(std::false_type());
  };
  if (p.dtype == TFFT_F32) launch(float());
  else if (p.dtype == TFFT_F16) launch(f16());
  else launch(bf16());
  return tfft_internal_finish(stream);
}
