// Gated linear recurrence h[t] = a[t] h[t-1] + x[t] along the time axis: tfft_scan_forward, tfft_scan_backward and
// tfft_scan_step. No counterpart in the reference.
#include "seq_common.hpp"

namespace {
using namespace tfft_seq;

template <class T, class G>
__global__ __launch_bounds__(256) void scan_walk_fwd(tfft_scan_args p) {
  const long long n = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (n >= p.batch * p.channels) return;
  const long long b = n / p.channels, c = n % p.channels;
  const T* x = (const T*)p.x.data + b * p.x.batch + c * p.x.channel;
  const G* g = (const G*)p.gate.data + b * p.gate.batch + c / p.share * p.gate.channel;
  T* y = (T*)p.y.data + b * p.y.batch + c * p.y.channel;
  long long len = p.length;
  if (p.lengths) len = p.lengths[b] < 0 ? 0 : p.lengths[b] < len ? p.lengths[b] : len;
  float h = p.initial ? p.initial[n] : 0.0f;
  for (long long t = 0; t < p.length; ++t) {
    if (t < len) {
      float a = to_f32(g[t * p.gate.time]);
      if (p.gate_form == TFFT_GATE_LOG) a = expf(a);
      h = fmaf(a, h, to_f32(x[t * p.x.time]));
    }
    y[t * p.y.time] = t < len ? from_f32<T>(h) : from_f32<T>(0.0f);
  }
  if (p.last) p.last[n] = h;
}

template <class T, class G>
__global__ __launch_bounds__(256) void scan_walk_bwd(tfft_scan_grad_args p) {
  const long long n = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (n >= p.batch * p.channels) return;
  const long long b = n / p.channels, c = n % p.channels;
  const T* dy = (const T*)p.dy.data + b * p.dy.batch + c * p.dy.channel;
  const T* y = (const T*)p.y.data + b * p.y.batch + c * p.y.channel;
  const G* g = (const G*)p.gate.data + b * p.gate.batch + c / p.share * p.gate.channel;
  T* dx = (T*)p.dx.data + b * p.dx.batch + c * p.dx.channel;
  long long len = p.length;
  if (p.lengths) len = p.lengths[b] < 0 ? 0 : p.lengths[b] < len ? p.lengths[b] : len;
  float carry = p.dlast ? p.dlast[n] : 0.0f;
  for (long long t = p.length - 1; t >= 0; --t) {
    float e = 0.0f, da = 0.0f;
    if (t < len) {
      float a = to_f32(g[t * p.gate.time]);
      if (p.gate_form == TFFT_GATE_LOG) a = expf(a);
      e = to_f32(dy[t * p.dy.time]) + carry;
      const float before = t > 0 ? to_f32(y[(t - 1) * p.y.time]) : p.initial ? p.initial[n] : 0.0f;
      da = e * before;
      carry = a * e;
      if (p.gate_form == TFFT_GATE_LOG) da *= a;
    }
    dx[t * p.dx.time] = from_f32<T>(e);
    if (p.share == 1)
      ((G*)p.dgate.data)[b * p.dgate.batch + t * p.dgate.time + c * p.dgate.channel] = from_f32<G>(da);
    else
      ((float*)p.workspace)[(b * p.length + t) * p.channels + c] = da;
  }
  if (p.dinitial) p.dinitial[n] = carry;
}

// dgate of a shared gate: its channels' terms, which lie side by side in the workspace, summed in their order
template <class G>
__global__ __launch_bounds__(256) void sum_shares(tfft_scan_grad_args p) {
  const long long gates = p.channels / p.share;
  const long long n = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (n >= p.batch * p.length * gates) return;
  const long long g = n % gates, bt = n / gates, b = bt / p.length, t = bt % p.length;
  const float* part = (const float*)p.workspace + bt * p.channels + g * p.share;
  float sum = 0.0f;
  for (long long i = 0; i < p.share; ++i) sum += part[i];
  ((G*)p.dgate.data)[b * p.dgate.batch + t * p.dgate.time + g * p.dgate.channel] = from_f32<G>(sum);
}

template <class T, class G>
__global__ __launch_bounds__(256) void scan_step(tfft_scan_step_args p) {
  const long long n = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (n >= p.batch * p.channels) return;
  const long long b = n / p.channels, c = n % p.channels;
  float a = to_f32(((const G*)p.gate)[b * p.gate_batch + c / p.share]);
  if (p.gate_form == TFFT_GATE_LOG) a = expf(a);
  const float h = fmaf(a, p.state[b * p.state_batch + c], to_f32(((const T*)p.x)[b * p.x_batch + c]));
  p.new_state[b * p.new_state_batch + c] = h;
  if (p.y) ((T*)p.y)[b * p.y_batch + c] = from_f32<T>(h);
}

// ---- argument checks ----------------------------------------------------------------------------------------------

constexpr long long kMaxExtent = 0x7fffffffLL;

const char* check_sizes(int dtype, int gate_dtype, int gate_form, long long batch, long long length, long long channels,
                        long long share) {
  if (gate_form != TFFT_GATE_DECAY && gate_form != TFFT_GATE_LOG) return "gate_form is TFFT_GATE_DECAY or TFFT_GATE_LOG";
  if (batch < 0 || length < 0 || channels < 0) return "negative extent";
  if (batch > kMaxExtent || length > kMaxExtent || channels > kMaxExtent) return "an extent is 2^31 or more";
  if (share < 1 || channels % share) return "share does not divide the channels";
  return nullptr;
}

bool bad_types(int dtype, int gate_dtype) {
  return dtype < TFFT_F32 || dtype > TFFT_BF16 || (gate_dtype != TFFT_F32 && gate_dtype != dtype);
}

// A stride of an extent of one says nothing; the layout rules see it as the contiguous one.
void settle(tfft_seq_view* v, long long batch, long long length, long long channels) {
  if (batch <= 1) v->batch = 0;
  if (length <= 1) v->time = channels <= 1 ? 1 : 0;
  if (channels <= 1) v->channel = length <= 1 ? 1 : 0;
}

const char* check_view(const tfft_seq_view& v, int dtype, long long batch, long long length, long long channels,
                       bool output) {
  const long long stride[3] = {v.batch, v.time, v.channel}, extent[3] = {batch, length, channels};
  return check_tensor(v.data, dtype, stride, extent, output);
}

int refuse(const char* who, const char* why, int code = TFFT_ERR_INVALID) {
  char text[256];
  snprintf(text, sizeof text, "%s: %s", who, why);
  return tfft_internal_fail(code, text);
}

#define TFFT_SEQ_CHECK(expr)                               \
  do {                                                     \
    if (const char* why_ = (expr)) return refuse(who, why_); \
  } while (0)

int check(const char* who, tfft_scan_args* p) {
  if (bad_types(p->dtype, p->gate_dtype))
    return refuse(who, "element types: fp32, fp16 or bf16, and a gate of fp32 or the same type", TFFT_ERR_UNSUPPORTED);
  TFFT_SEQ_CHECK(check_sizes(p->dtype, p->gate_dtype, p->gate_form, p->batch, p->length, p->channels, p->share));
  settle(&p->x, p->batch, p->length, p->channels);
  settle(&p->y, p->batch, p->length, p->channels);
  settle(&p->gate, p->batch, p->length, p->channels / p->share);
  return TFFT_OK;
}

int check(const char* who, tfft_scan_grad_args* p) {
  if (bad_types(p->dtype, p->gate_dtype))
    return refuse(who, "element types: fp32, fp16 or bf16, and a gate of fp32 or the same type", TFFT_ERR_UNSUPPORTED);
  TFFT_SEQ_CHECK(check_sizes(p->dtype, p->gate_dtype, p->gate_form, p->batch, p->length, p->channels, p->share));
  for (tfft_seq_view* v : {&p->dy, &p->y, &p->dx}) settle(v, p->batch, p->length, p->channels);
  for (tfft_seq_view* v : {&p->gate, &p->dgate}) settle(v, p->batch, p->length, p->channels / p->share);
  return TFFT_OK;
}

const char* check_state(const void* p) { return misaligned(p, TFFT_F32) ? "misaligned pointer" : nullptr; }

const char* check_workspace(const void* p, unsigned long long bytes, unsigned long long need) {
  if (need == 0) return nullptr;
  if (!p || bytes < need) return "the workspace is smaller than tfft_scan_workspace_bytes";
  return (reinterpret_cast<uintptr_t>(p) & 7u) ? "the workspace is not aligned to 8 bytes" : nullptr;
}

unsigned long long workspace_of(const tfft_scan_args& p) { return 0; }
unsigned long long workspace_of(const tfft_scan_grad_args& p) {
  return p.share > 1 ? 4ull * p.batch * p.length * p.channels : 0;
}

unsigned blocks(long long threads) { return (unsigned)((threads + 255) / 256); }

// f(T(), G()) for the element types of a call
template <class F>
void with_types(int dtype, int gate_dtype, F f) {
  if (dtype == TFFT_F32) f(float(), float());
  else if (dtype == TFFT_F16 && gate_dtype == TFFT_F32) f(f16(), float());
  else if (dtype == TFFT_F16) f(f16(), f16());
  else if (gate_dtype == TFFT_F32) f(bf16(), float());
  else f(bf16(), bf16());
}

}  // namespace

extern "C" int tfft_scan_workspace_bytes(const tfft_scan_args* forward, const tfft_scan_grad_args* backward,
                                         unsigned long long* bytes) {
  const char* who = "tfft_scan_workspace_bytes";
  if (!bytes || !forward == !backward) return refuse(who, "one of forward and backward, and a result");
  if ((forward && forward->struct_size != (int)sizeof *forward) || (backward && backward->struct_size != (int)sizeof *backward))
    return refuse(who, "struct_size is not that of the argument structure");
  if (forward) {
    tfft_scan_args p = *forward;
    if (const int rc = check(who, &p)) return rc;
    *bytes = workspace_of(p);
  } else {
    tfft_scan_grad_args p = *backward;
    if (const int rc = check(who, &p)) return rc;
    *bytes = workspace_of(p);
  }
  return TFFT_OK;
}

extern "C" int tfft_scan_forward(const tfft_scan_args* args, void* stream) {
  const char* who = "tfft_scan_forward";
  if (!args || args->struct_size != (int)sizeof *args) return refuse(who, "null arguments, or struct_size is not theirs");
  tfft_scan_args p = *args;
  if (const int rc = check(who, &p)) return rc;
  if (p.batch == 0 || p.channels == 0) return TFFT_OK;
  TFFT_SEQ_CHECK(check_view(p.x, p.dtype, p.batch, p.length, p.channels, false));
  TFFT_SEQ_CHECK(check_view(p.gate, p.gate_dtype, p.batch, p.length, p.channels / p.share, false));
  TFFT_SEQ_CHECK(check_view(p.y, p.dtype, p.batch, p.length, p.channels, true));
  for (const void* s : {(const void*)p.lengths, (const void*)p.initial, (const void*)p.last}) TFFT_SEQ_CHECK(check_state(s));
  TFFT_SEQ_CHECK(check_workspace(p.workspace, p.workspace_bytes, workspace_of(p)));
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_types(p.dtype, p.gate_dtype, [&](auto t, auto g) {
    scan_walk_fwd<decltype(t), decltype(g)><<<blocks(p.batch * p.channels), 256, 0, s>>>(p);
  });
  return tfft_internal_finish(stream);
}

extern "C" int tfft_scan_backward(const tfft_scan_grad_args* args, void* stream) {
  const char* who = "tfft_scan_backward";
  if (!args || args->struct_size != (int)sizeof *args) return refuse(who, "null arguments, or struct_size is not theirs");
  tfft_scan_grad_args p = *args;
  if (const int rc = check(who, &p)) return rc;
  if (p.batch == 0 || p.channels == 0) return TFFT_OK;
  TFFT_SEQ_CHECK(check_view(p.dy, p.dtype, p.batch, p.length, p.channels, false));
  TFFT_SEQ_CHECK(check_view(p.y, p.dtype, p.batch, p.length, p.channels, false));
  TFFT_SEQ_CHECK(check_view(p.gate, p.gate_dtype, p.batch, p.length, p.channels / p.share, false));
  TFFT_SEQ_CHECK(check_view(p.dx, p.dtype, p.batch, p.length, p.channels, true));
  TFFT_SEQ_CHECK(check_view(p.dgate, p.gate_dtype, p.batch, p.length, p.channels / p.share, true));
  for (const void* s : {(const void*)p.lengths, (const void*)p.initial, (const void*)p.dlast, (const void*)p.dinitial})
    TFFT_SEQ_CHECK(check_state(s));
  TFFT_SEQ_CHECK(check_workspace(p.workspace, p.workspace_bytes, workspace_of(p)));
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_types(p.dtype, p.gate_dtype, [&](auto t, auto g) {
    scan_walk_bwd<decltype(t), decltype(g)><<<blocks(p.batch * p.channels), 256, 0, s>>>(p);
    if (p.share > 1 && p.length > 0)
      sum_shares<decltype(g)><<<blocks(p.batch * p.length * (p.channels / p.share)), 256, 0, s>>>(p);
  });
  return tfft_internal_finish(stream);
}

extern "C" int tfft_scan_step(const tfft_scan_step_args* args, void* stream) {
  const char* who = "tfft_scan_step";
  if (!args || args->struct_size != (int)sizeof *args) return refuse(who, "null arguments, or struct_size is not theirs");
  const tfft_scan_step_args& p = *args;
  if (bad_types(p.dtype, p.gate_dtype))
    return refuse(who, "element types: fp32, fp16 or bf16, and a gate of fp32 or the same type", TFFT_ERR_UNSUPPORTED);
  TFFT_SEQ_CHECK(check_sizes(p.dtype, p.gate_dtype, p.gate_form, p.batch, 1, p.channels, p.share));
  if (p.batch == 0 || p.channels == 0) return TFFT_OK;
  TFFT_SEQ_CHECK(check_view({(void*)p.x, p.x_batch, 0, 1}, p.dtype, p.batch, 1, p.channels, false));
  TFFT_SEQ_CHECK(check_view({(void*)p.gate, p.gate_batch, 0, 1}, p.gate_dtype, p.batch, 1, p.channels / p.share, false));
  TFFT_SEQ_CHECK(check_view({(void*)p.state, p.state_batch, 0, 1}, TFFT_F32, p.batch, 1, p.channels, false));
  TFFT_SEQ_CHECK(check_view({p.new_state, p.new_state_batch, 0, 1}, TFFT_F32, p.batch, 1, p.channels, true));
  if (p.y) TFFT_SEQ_CHECK(check_view({p.y, p.y_batch, 0, 1}, p.dtype, p.batch, 1, p.channels, true));
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_types(p.dtype, p.gate_dtype, [&](auto t, auto g) {
    scan_step<decltype(t), decltype(g)><<<blocks(p.batch * p.channels), 256, 0, s>>>(p);
  });
  return tfft_internal_finish(stream);
}
