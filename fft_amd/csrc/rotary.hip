// Rotary positions: pairs of values times exp(2 pi i p F[i]) for 64-bit positions p and fixed-point frequencies F
// (tfft_rotary). No counterpart in the reference.
#include "seq_common.hpp"

namespace {
using namespace tfft_seq;

// cos and sin of `phase` 2^-64 turns. The phase is rounded to 2^-32 turns and the quadrant is taken off in integers, so
// that what is left, |r| <= 1/8 turn, is off by 2^-24 of itself; the Taylor sums to r^9 and r^10 are within 2e-9 there.
__device__ __forceinline__ void turn(uint64_t phase, float* c, float* s) {
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

template <class T>
__global__ __launch_bounds__(256) void rotary_pairs(tfft_rotary_args p, int which) {
  const tfft_rotary_view v = p.tensor[which];
  const int half = p.rotary / 2, units = half + (p.head - p.rotary);
  const long long n = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (n >= p.batch * p.length * v.heads * units) return;
  const int u = (int)(n % units);
  const long long h = n / units % v.heads, token = n / units / v.heads, b = token / p.length, t = token % p.length;
  const T* in = (const T*)v.in + b * v.in_batch + t * v.in_time + h * v.in_head;
  T* out = (T*)v.out + b * v.out_batch + t * v.out_time + h * v.out_head;
  if (u >= half) {
    out[u + half] = in[u + half];
    return;
  }
  long long pos = p.first + t;
  const long long at = b * p.position_batch + t * p.position_time;
  if (p.positions) pos = p.position_bytes == 8 ? ((const long long*)p.positions)[at] : ((const int*)p.positions)[at];
  float c, s;
  turn((uint64_t)pos * ((const uint64_t*)p.turns)[u], &c, &s);
  c *= p.magnitude, s *= p.inverse ? -p.magnitude : p.magnitude;
  const int i = p.pairs == TFFT_PAIRS_HALF ? u : 2 * u, j = p.pairs == TFFT_PAIRS_HALF ? u + half : 2 * u + 1;
  const float re = to_f32(in[i]), im = to_f32(in[j]);
  out[i] = from_f32<T>(re * c - im * s);
  out[j] = from_f32<T>(re * s + im * c);
}

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
  hipStream_t s = static_cast<hipStream_t>(stream);
  for (int i = 0; i < 2; ++i) {
    const tfft_rotary_view& v = p.tensor[i];
    const long long n = p.batch * p.length * v.heads * (p.head - p.rotary / 2);
    if (n == 0) continue;
    const long long extent[4] = {p.batch, p.length, v.heads, p.head};
    const long long in[4] = {v.in_batch, v.in_time, v.in_head, 1}, out[4] = {v.out_batch, v.out_time, v.out_head, 1};
    if (const char* why = check_tensor(v.in, p.dtype, in, extent, false)) return refuse(why);
    if (const char* why = check_tensor(v.out, p.dtype, out, extent, true)) return refuse(why);
    const unsigned grid = (unsigned)((n + 255) / 256);
    if (p.dtype == TFFT_F32) rotary_pairs<float><<<grid, 256, 0, s>>>(p, i);
    else if (p.dtype == TFFT_F16) rotary_pairs<f16><<<grid, 256, 0, s>>>(p, i);
    else rotary_pairs<bf16><<<grid, 256, 0, s>>>(p, i);
  }
  return tfft_internal_finish(stream);
}
