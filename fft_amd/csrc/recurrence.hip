// Gated linear recurrence h[t] = a[t] h[t-1] + x[t] along the time axis: tfft_scan_forward, tfft_scan_backward and
// tfft_scan_step. No counterpart in the reference.
#include "recurrence_kernels.hpp"

namespace {
using namespace tfft_seq;

// The words that chunks hand their states on with, cleared by a kernel of the same call: it may be captured and
// replayed, and nothing of an earlier call is left in them.
__global__ __launch_bounds__(256) void clear_words(word* words, long long n) {
  const long long first = 1024ll * blockIdx.x + threadIdx.x;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (first + 256 * i < n) words[first + 256 * i] = 0;
}

// One token: a thread has kRun neighbouring channels of a row. What counts is latency (a full batch of 512 x 4096 channels is 29 MB,
// 5 us of HBM): one pass, 8- and 16-byte accesses, indexes in 32 bits.
constexpr int kRun = 4;
template <class T, class G>
__global__ __launch_bounds__(256) void scan_step(tfft_scan_step_args p, unsigned runs, unsigned threads) {
  const unsigned n = blockIdx.x * 256u + threadIdx.x;
  if (n >= threads) return;
  const unsigned b = n / runs, c = (n - b * runs) * kRun, share = (unsigned)p.share;
  const int valid = min(kRun, (int)(p.channels - c));
  const Run<T, kRun> x = load_some<kRun>((const T*)p.x + b * p.x_batch + c, valid);
  const Run<float, kRun> old = load_some<kRun>(p.state + b * p.state_batch + c, valid);
  const G* gate = (const G*)p.gate + b * p.gate_batch;
  float a[kRun];
  if (share == 1) {
    const Run<G, kRun> g = load_some<kRun>(gate + c, valid);
#pragma unroll
    for (int v = 0; v < kRun; ++v) a[v] = g.get(v);
  } else {
#pragma unroll
    for (int v = 0; v < kRun; ++v) a[v] = to_f32(gate[min(c + v, (unsigned)p.channels - 1) / share]);
  }
  Run<float, kRun> h;
  Run<T, kRun> y;
#pragma unroll
  for (int v = 0; v < kRun; ++v) {
    const float k = p.gate_form == TFFT_GATE_LOG ? exp_decay(a[v]) : a[v], next = fmaf(k, old.get(v), x.get(v));
    h.set(v, next), y.set(v, next);
  }
  store_some<kRun>(p.new_state + b * p.new_state_batch + c, h, valid);
  if (p.y) store_some<kRun>((T*)p.y + b * p.y_batch + c, y, valid);
}

// ---- argument checks ----------------------------------------------------------------------------------------------

constexpr long long kMaxExtent = 0x7fffffffLL, kMaxLength = 1LL << 30;

const char* check_sizes(int dtype, int gate_dtype, int gate_form, long long batch, long long length, long long channels,
                        long long share) {
  if (gate_form != TFFT_GATE_DECAY && gate_form != TFFT_GATE_LOG) return "gate_form is TFFT_GATE_DECAY or TFFT_GATE_LOG";
  if (batch < 0 || length < 0 || channels < 0) return "negative extent";
  if (batch > kMaxExtent || length > kMaxLength || channels > kMaxExtent - 3) return "an extent is too large";
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

// How a call runs. Steps side by side take the signals' kernels where channels do not lie side by side too; every other
// layout goes through the rows' kernels, which take any strides.
template <class P>
bool as_signals(const P& p) {
  return signals_fit(p) && !(rows_vector(p) && p.channels > 1);
}
template <class P>
Chunking plan_of(const P& p) {
  return as_signals(p) ? plan_signals(p) : plan_rows(p);
}
unsigned long long parts_of(const tfft_scan_args&) { return 0; }
unsigned long long parts_of(const tfft_scan_grad_args& p) {
  return 4 * (as_signals(p) ? signals_parts(p) : rows_parts(p));
}
template <class P>
unsigned long long workspace_of(const P& p) {
  return 8ull * plan_of(p).words() + parts_of(p);
}
// A launch counts its threads in 32 bits
template <class P>
const char* check_plan(const P& p) {
  const char* large = "more sequences or steps than one launch takes";
  constexpr long long most = 0xffff0000LL;
  if (p.batch * (p.channels + 3) > kMaxExtent) return large;
  const Chunking c = plan_of(p);
  return (__int128)c.blocks() * 64 * c.waves > most ? large : nullptr;
}

// Two tensors at one address: outputs take an input's place element for element, or none at all
bool same(const void* a, const void* b) { return a && a == b; }
bool alike(const tfft_seq_view& a, const tfft_seq_view& b) {
  return a.batch == b.batch && a.time == b.time && a.channel == b.channel;
}
const char* check_places(const tfft_scan_args& p) {
  if (same(p.y.data, p.gate.data)) return "y may not take the gate's place";
  return same(p.y.data, p.x.data) && !alike(p.x, p.y) ? "in place needs equal strides on both sides" : nullptr;
}
const char* check_places(const tfft_scan_grad_args& p) {
  for (const tfft_seq_view* v : {&p.dy, &p.y, &p.gate, &p.dx})
    if (same(p.dgate.data, v->data)) return "dgate may not take another tensor's place";
  if (same(p.dx.data, p.y.data) || same(p.dx.data, p.gate.data)) return "dx may not take y's or the gate's place";
  return same(p.dx.data, p.dy.data) && !alike(p.dx, p.dy) ? "in place needs equal strides on both sides" : nullptr;
}

template <class P>
void clear(const Chunking& c, const P& p, hipStream_t s) {
  const long long n = c.words();
  if (n) clear_words<<<(unsigned)((n + 1023) / 1024), 256, 0, s>>>((word*)p.workspace, n);
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
    TFFT_SEQ_CHECK(check_plan(p));
    *bytes = workspace_of(p);
  } else {
    tfft_scan_grad_args p = *backward;
    if (const int rc = check(who, &p)) return rc;
    TFFT_SEQ_CHECK(check_plan(p));
    *bytes = workspace_of(p);
  }
  return TFFT_OK;
}

extern "C" int tfft_scan_forward(const tfft_scan_args* args, void* stream) {
  const char* who = "tfft_scan_forward";
  if (!args || args->struct_size != (int)sizeof *args) return refuse(who, "null arguments, or struct_size is not theirs");
  tfft_scan_args p = *args;
  if (const int rc = check(who, &p)) return rc;
  TFFT_SEQ_CHECK(check_plan(p));
  if (p.batch == 0 || p.channels == 0) return TFFT_OK;
  TFFT_SEQ_CHECK(check_view(p.x, p.dtype, p.batch, p.length, p.channels, false));
  TFFT_SEQ_CHECK(check_view(p.gate, p.gate_dtype, p.batch, p.length, p.channels / p.share, false));
  TFFT_SEQ_CHECK(check_view(p.y, p.dtype, p.batch, p.length, p.channels, true));
  if (p.length > 0) TFFT_SEQ_CHECK(check_places(p));
  for (const void* s : {(const void*)p.lengths, (const void*)p.initial, (const void*)p.last}) TFFT_SEQ_CHECK(check_state(s));
  TFFT_SEQ_CHECK(check_workspace(p.workspace, p.workspace_bytes, workspace_of(p)));
  hipStream_t s = static_cast<hipStream_t>(stream);
  const Chunking c = plan_of(p);
  clear(c, p, s);
  if (as_signals(p)) launch_signals(p, c, (word*)p.workspace, s);
  else launch_rows(p, c, (word*)p.workspace, s);
  return tfft_internal_finish(stream);
}

extern "C" int tfft_scan_backward(const tfft_scan_grad_args* args, void* stream) {
  const char* who = "tfft_scan_backward";
  if (!args || args->struct_size != (int)sizeof *args) return refuse(who, "null arguments, or struct_size is not theirs");
  tfft_scan_grad_args p = *args;
  if (const int rc = check(who, &p)) return rc;
  TFFT_SEQ_CHECK(check_plan(p));
  if (p.batch == 0 || p.channels == 0) return TFFT_OK;
  TFFT_SEQ_CHECK(check_view(p.dy, p.dtype, p.batch, p.length, p.channels, false));
  TFFT_SEQ_CHECK(check_view(p.y, p.dtype, p.batch, p.length, p.channels, false));
  TFFT_SEQ_CHECK(check_view(p.gate, p.gate_dtype, p.batch, p.length, p.channels / p.share, false));
  TFFT_SEQ_CHECK(check_view(p.dx, p.dtype, p.batch, p.length, p.channels, true));
  TFFT_SEQ_CHECK(check_view(p.dgate, p.gate_dtype, p.batch, p.length, p.channels / p.share, true));
  if (p.length > 0) TFFT_SEQ_CHECK(check_places(p));
  for (const void* s : {(const void*)p.lengths, (const void*)p.initial, (const void*)p.dlast, (const void*)p.dinitial})
    TFFT_SEQ_CHECK(check_state(s));
  TFFT_SEQ_CHECK(check_workspace(p.workspace, p.workspace_bytes, workspace_of(p)));
  hipStream_t s = static_cast<hipStream_t>(stream);
  const Chunking c = plan_of(p);
  clear(c, p, s);
  float* parts = (float*)((word*)p.workspace + c.words());
  if (as_signals(p)) launch_signals(p, c, (word*)p.workspace, parts, s);
  else launch_rows(p, c, (word*)p.workspace, parts, s);
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
  if (same(p.new_state, p.x) || same(p.new_state, p.gate) || same(p.y, p.gate) || same(p.y, p.state) || same(p.y, p.new_state))
    return refuse(who, "an output may not take another tensor's place");
  if (p.batch > 1 && ((same(p.new_state, p.state) && p.new_state_batch != p.state_batch) || (same(p.y, p.x) && p.y_batch != p.x_batch)))
    return refuse(who, "in place needs equal strides on both sides");
  if (p.batch * (p.channels + kRun) > kMaxExtent) return refuse(who, "more sequences than one launch takes");
  const unsigned runs = (unsigned)((p.channels + kRun - 1) / kRun), threads = (unsigned)p.batch * runs;
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_types(p.dtype, p.gate_dtype, [&](auto t, auto g) {
    scan_step<decltype(t), decltype(g)><<<(threads + 255) / 256, 256, 0, s>>>(p, runs, threads);
  });
  return tfft_internal_finish(stream);
}
