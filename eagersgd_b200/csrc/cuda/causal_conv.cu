// The short causal convolution ahead of a scan: every channel by itself, over the last K inputs.
//
//   pre[t] = bias + sum_k w[k] x[t - K + 1 + k],   y[t] = act(pre[t])
//   dpre = dy act'(pre);  dx[t] = sum_j w[K - 1 - j] dpre[t + j];  dw[k] = sum dpre[t] x[t - K + 1 + k];  dbias = sum dpre
//
// Bound by memory.  A thread has a vector of channels and a run of steps, the window in registers: of every run only the K - 1
// inputs ahead of it are read twice (the backward pass makes the K - 1 dpre behind it again).
#include "launch.cuh"
#include "rows.cuh"

namespace {

using namespace esgd;

constexpr int kThreads = 256;

struct Conv {
  int64_t batch, length;
  int channels;
  int64_t xb, xt;              // strides of x, elements
  const int64_t* lengths;      // [batch], or null
  const float* weight;         // [channels][K]
  const float* bias;           // [channels], or null
  int lanes;                   // channel vectors of a block
  int runs;                    // of a block
  int steps;                   // of a run
  int vec_blocks, time_blocks;
};

__device__ __forceinline__ int64_t length_of(const Conv& c, int64_t b) {
  if (c.lengths == nullptr) return c.length;
  const int64_t n = c.lengths[b];
  return n < 0 ? 0 : n > c.length ? c.length : n;
}

// Where a thread works.
template <int kV> struct Spot {
  int64_t b, len, first, last;     // steps [first, last)
  int c, run;
  bool on;
  __device__ explicit Spot(const Conv& p) {
    int64_t i = blockIdx.x;
    const int64_t rest = i / p.vec_blocks;
    const int vb = (int)(i - rest * p.vec_blocks);
    b = rest / p.time_blocks;
    const int64_t tb = rest - b * p.time_blocks;
    run = threadIdx.x / p.lanes;
    c = (vb * p.lanes + threadIdx.x - run * p.lanes) * kV;
    len = length_of(p, b);
    first = (tb * p.runs + run) * p.steps;
    last = first + p.steps < p.length ? first + p.steps : p.length;
    on = run < p.runs && c < p.channels;
  }
};

template <class T, int kV> __device__ __forceinline__ void input(const T* x, const T* state, const Conv& p, int64_t b, int64_t t, int c,
                                                                 int taps, float (&f)[kV]) {
  if (t >= 0) {
    unpack<T, kV>(load<T, kV>(x + b * p.xb + t * p.xt + c), f);
  } else if (state != nullptr) {
    unpack<T, kV>(load<T, kV>(state + (b * (taps - 1) + t + taps - 1) * p.channels + c), f);
  } else {
#pragma unroll
    for (int q = 0; q < kV; ++q) f[q] = 0.0f;
  }
}

template <class T, int kV, int kTaps, int kAct>
__global__ void __launch_bounds__(kThreads) causal_conv_fwd_kernel(const T* __restrict__ x, const T* __restrict__ state, T* __restrict__ y,
                                                                   T* __restrict__ state_out, Conv p) {
  pdl_enter();
  const Spot<kV> s(p);
  if (!s.on) return;
  if (state_out != nullptr && s.first == (int64_t)s.run * p.steps)        // blocks of the first steps
    for (int i = s.run; i < kTaps - 1; i += p.runs) {
      float f[kV];
      input<T, kV>(x, state, p, s.b, s.len - (kTaps - 1) + i, s.c, kTaps, f);
      store<T, kV>(state_out + (s.b * (kTaps - 1) + i) * p.channels + s.c, f);
    }
  if (s.first >= p.length) return;
  float w[kTaps][kV], bias[kV], win[kTaps][kV];
#pragma unroll
  for (int q = 0; q < kV; ++q) {
    bias[q] = p.bias != nullptr ? p.bias[s.c + q] : 0.0f;
#pragma unroll
    for (int k = 0; k < kTaps; ++k) w[k][q] = p.weight[(s.c + q) * kTaps + k];
  }
#pragma unroll
  for (int k = 0; k < kTaps - 1; ++k) {
    if (s.first < s.len) {
      input<T, kV>(x, state, p, s.b, s.first - (kTaps - 1) + k, s.c, kTaps, win[k + 1]);
    } else {
#pragma unroll
      for (int q = 0; q < kV; ++q) win[k + 1][q] = 0.0f;
    }
  }
  const T* in = x + s.b * p.xb + s.c;
  T* out = y + s.b * p.length * p.channels + s.c;
  for (int64_t t = s.first; t < s.last; t += 4) {
    Pack<T, kV> raw[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (t + u < s.last && t + u < s.len) raw[u] = load<T, kV>(in + (t + u) * p.xt);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (t + u >= s.last) break;
      float f[kV];
#pragma unroll
      for (int q = 0; q < kV; ++q) f[q] = 0.0f;
      if (t + u < s.len) {
#pragma unroll
        for (int k = 0; k < kTaps - 1; ++k)
#pragma unroll
          for (int q = 0; q < kV; ++q) win[k][q] = win[k + 1][q];
        unpack<T, kV>(raw[u], win[kTaps - 1]);
#pragma unroll
        for (int q = 0; q < kV; ++q) {
          float pre = bias[q];
#pragma unroll
          for (int k = 0; k < kTaps; ++k) pre = fmaf(w[k][q], win[k][q], pre);
          f[q] = activate<kAct>(pre);
        }
      }
      store<T, kV>(out + (t + u) * p.channels, f);
    }
  }
}

// sums [blocks of a channel][channels * K + channels]: each block's share of dw and dbias.
template <class T, int kV, int kTaps, int kAct>
__global__ void __launch_bounds__(kThreads) causal_conv_bwd_kernel(const T* __restrict__ x, const T* __restrict__ state,
                                                                   const T* __restrict__ dy, T* __restrict__ dx, float* __restrict__ sums,
                                                                   Conv p) {
  pdl_enter();
  __shared__ float stage[kThreads * kV];
  const Spot<kV> s(p);
  float dw[kTaps + 1][kV];
#pragma unroll
  for (int k = 0; k <= kTaps; ++k)
#pragma unroll
    for (int q = 0; q < kV; ++q) dw[k][q] = 0.0f;
  if (s.on && s.first < p.length) {
    float w[kTaps][kV], bias[kV], win[kTaps][kV], dp[kTaps][kV];
#pragma unroll
    for (int q = 0; q < kV; ++q) {
      bias[q] = p.bias != nullptr ? p.bias[s.c + q] : 0.0f;
#pragma unroll
      for (int k = 0; k < kTaps; ++k) w[k][q] = p.weight[(s.c + q) * kTaps + k];
    }
#pragma unroll
    for (int k = 0; k < kTaps; ++k)
#pragma unroll
      for (int q = 0; q < kV; ++q) win[k][q] = dp[k][q] = 0.0f;
    if (s.first < s.len)
#pragma unroll
      for (int k = 0; k < kTaps - 1; ++k) input<T, kV>(x, state, p, s.b, s.first - (kTaps - 1) + k, s.c, kTaps, win[k + 1]);
    const T* in = x + s.b * p.xb + s.c;
    const T* up = dy + s.b * p.length * p.channels + s.c;
    T* out = dx + s.b * p.length * p.channels + s.c;
    for (int64_t t = s.first; t < s.last + kTaps - 1; t += 4) {
      Pack<T, kV> rx[4], rd[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (t + u < s.last + kTaps - 1 && t + u < s.len) {
          rx[u] = load<T, kV>(in + (t + u) * p.xt);
          rd[u] = load<T, kV>(up + (t + u) * p.channels);
        }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t now = t + u;
        if (now >= s.last + kTaps - 1) break;
#pragma unroll
        for (int k = 0; k < kTaps - 1; ++k)
#pragma unroll
          for (int q = 0; q < kV; ++q) { win[k][q] = win[k + 1][q]; dp[k][q] = dp[k + 1][q]; }
        if (now < s.len) {
          float d[kV];
          unpack<T, kV>(rx[u], win[kTaps - 1]);
          unpack<T, kV>(rd[u], d);
#pragma unroll
          for (int q = 0; q < kV; ++q) {
            if constexpr (kAct != kActNone) {
              float pre = bias[q];
#pragma unroll
              for (int k = 0; k < kTaps; ++k) pre = fmaf(w[k][q], win[k][q], pre);
              d[q] *= slope<kAct>(pre);
            }
            dp[kTaps - 1][q] = d[q];
            if (now < s.last) {
              dw[kTaps][q] += d[q];
#pragma unroll
              for (int k = 0; k < kTaps; ++k) dw[k][q] = fmaf(d[q], win[k][q], dw[k][q]);
            }
          }
        } else {
#pragma unroll
          for (int q = 0; q < kV; ++q) dp[kTaps - 1][q] = 0.0f;
        }
        const int64_t back = now - (kTaps - 1);
        if (back >= s.first && dx != nullptr) {
          float f[kV];
#pragma unroll
          for (int q = 0; q < kV; ++q) {
            f[q] = 0.0f;
#pragma unroll
            for (int j = 0; j < kTaps; ++j) f[q] = fmaf(w[kTaps - 1 - j][q], dp[j][q], f[q]);
          }
          store<T, kV>(out + back * p.channels, f);
        }
      }
    }
  }
  if (sums == nullptr) return;
  float* part = sums + (int64_t)(blockIdx.x / p.vec_blocks) * p.channels * (kTaps + 1);
#pragma unroll
  for (int k = 0; k <= kTaps; ++k) {
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kV; ++q) stage[threadIdx.x * kV + q] = dw[k][q];
    __syncthreads();
    const int vb = (int)(blockIdx.x % p.vec_blocks);
    for (int i = threadIdx.x; i < p.lanes * kV; i += kThreads) {
      const int c = vb * p.lanes * kV + i;
      if (c >= p.channels) break;
      float t = 0.0f;
      for (int r = 0; r < p.runs; ++r) t += stage[r * p.lanes * kV + i];
      part[k < kTaps ? c * kTaps + k : p.channels * kTaps + c] = t;
    }
  }
}

// One step: state [batch][K - 1][channels] moves on by one input; state_out may be state.
template <class T, int kV, int kTaps, int kAct>
__global__ void __launch_bounds__(128) causal_conv_step_kernel(const T* __restrict__ x, int64_t xb, const T* state, T* state_out,
                                                               T* __restrict__ y, const float* __restrict__ weight,
                                                               const float* __restrict__ bias, int64_t batch, int channels) {
  pdl_enter();
  const int vectors = channels / kV;
  const int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x;
  if (i >= batch * vectors) return;
  const int64_t b = i / vectors;
  const int c = (int)(i - b * vectors) * kV;
  float win[kTaps][kV], f[kV];
#pragma unroll
  for (int k = 0; k < kTaps - 1; ++k) unpack<T, kV>(load<T, kV>(state + (b * (kTaps - 1) + k) * channels + c), win[k]);
  unpack<T, kV>(load<T, kV>(x + b * xb + c), win[kTaps - 1]);
#pragma unroll
  for (int q = 0; q < kV; ++q) {
    float pre = bias != nullptr ? bias[c + q] : 0.0f;
#pragma unroll
    for (int k = 0; k < kTaps; ++k) pre = fmaf(weight[(c + q) * kTaps + k], win[k][q], pre);
    f[q] = activate<kAct>(pre);
  }
  store<T, kV>(y + b * channels + c, f);
#pragma unroll
  for (int k = 0; k < kTaps - 1; ++k) store<T, kV>(state_out + (b * (kTaps - 1) + k) * channels + c, win[k + 1]);
}

void plan(Conv* p, int v) {
  const int vectors = p->channels / v;
  p->lanes = 1;
  while (p->lanes < 32 && p->lanes < vectors) p->lanes *= 2;
  p->runs = kThreads / p->lanes;
  p->vec_blocks = (vectors + p->lanes - 1) / p->lanes;
  // long runs read least twice; short ones fill the GPU
  p->steps = 32;
  while (p->steps > 4 && p->batch * p->vec_blocks * ((p->length + (int64_t)p->runs * p->steps - 1) / (p->runs * p->steps)) < 4 * sm_count())
    p->steps /= 2;
  p->time_blocks = (int)((p->length + (int64_t)p->runs * p->steps - 1) / (p->runs * p->steps));
  if (p->time_blocks < 1) p->time_blocks = 1;
}
int64_t blocks_of(const Conv& p) { return p.batch * p.time_blocks * p.vec_blocks; }

template <class T, int kV, int kTaps, int kAct>
int forward(const void* x, const void* state, void* y, void* state_out, const Conv& p, void* stream) {
  return launch(causal_conv_fwd_kernel<T, kV, kTaps, kAct>, dim3((unsigned)blocks_of(p)), kThreads, 0, stream, (const T*)x, (const T*)state,
                (T*)y, (T*)state_out, p);
}
template <class T, int kV, int kTaps, int kAct>
int backward(const void* x, const void* state, const void* dy, void* dx, float* sums, const Conv& p, void* stream) {
  return launch(causal_conv_bwd_kernel<T, kV, kTaps, kAct>, dim3((unsigned)blocks_of(p)), kThreads, 0, stream, (const T*)x, (const T*)state,
                (const T*)dy, (T*)dx, sums, p);
}
template <class T, int kV, int kTaps, int kAct>
int step(const void* x, int64_t xb, const void* state, void* state_out, void* y, const float* weight, const float* bias, int64_t batch,
         int channels, void* stream) {
  const int64_t n = batch * (channels / kV);
  return launch(causal_conv_step_kernel<T, kV, kTaps, kAct>, dim3((unsigned)((n + 127) / 128)), 128, 0, stream, (const T*)x, xb,
                (const T*)state, (T*)state_out, (T*)y, weight, bias, batch, channels);
}

// F<T, kV, kTaps, kAct>(...)
#define ESGD_TAPS(T, V, F, ...)                                                                                        \
  (act == kActSilu ? (taps == 2 ? F<T, V, 2, kActSilu>(__VA_ARGS__) : taps == 3 ? F<T, V, 3, kActSilu>(__VA_ARGS__)    \
                                                                                : F<T, V, 4, kActSilu>(__VA_ARGS__))   \
                   : (taps == 2 ? F<T, V, 2, kActNone>(__VA_ARGS__) : taps == 3 ? F<T, V, 3, kActNone>(__VA_ARGS__)    \
                                                                                : F<T, V, 4, kActNone>(__VA_ARGS__)))
#define ESGD_TYPE(F, ...)                                                                                             \
  (is_bf16 ? (v == 8 ? ESGD_TAPS(__nv_bfloat16, 8, F, __VA_ARGS__) : ESGD_TAPS(__nv_bfloat16, 1, F, __VA_ARGS__))     \
           : (v == 4 ? ESGD_TAPS(float, 4, F, __VA_ARGS__) : ESGD_TAPS(float, 1, F, __VA_ARGS__)))

bool taken(int taps, int act) { return taps >= 2 && taps <= 4 && (act == kActSilu || act == kActNone); }
int width(int is_bf16, int channels, int64_t xb, int64_t xt, const void* a, const void* b, const void* c, const void* d) {
  const int v = is_bf16 ? 8 : 4;
  return channels % v || xb % v || xt % v || !aligned16(a) || !aligned16(b) || !aligned16(c) || !aligned16(d) ? 1 : v;
}

}  // namespace

extern "C" {

// x [batch][length][channels] with strides xb, xt; y dense; state, state_out [batch][taps - 1][channels] or null.
int esgd_causal_conv_fwd(const void* x, int64_t xb, int64_t xt, const void* state, const float* weight, const float* bias,
                         const int64_t* lengths, void* y, void* state_out, int is_bf16, int64_t batch, int64_t length, int channels, int taps,
                         int act, void* stream) {
  if (!taken(taps, act)) return (int)cudaErrorInvalidValue;
  if (batch == 0 || channels == 0) return 0;
  const int v = width(is_bf16, channels, xb, xt, x, state, y, state_out);
  Conv p = {batch, length, channels, xb, xt, lengths, weight, bias};
  plan(&p, v);
  return ESGD_TYPE(forward, x, state, y, state_out, p, stream);
}

// The parts that esgd_causal_conv_bwd leaves in sums, each [channels * taps + channels].
int64_t esgd_causal_conv_parts(int is_bf16, int64_t batch, int64_t length, int channels) {
  // the narrowest vector has the most blocks of steps or fewer runs: room for either
  int64_t most = 0;
  for (int v : {1, is_bf16 ? 8 : 4}) {
    if (channels % v) continue;
    Conv p = {batch, length, channels};
    plan(&p, v);
    if (p.batch * p.time_blocks > most) most = p.batch * p.time_blocks;
  }
  return most;
}

// dx dense, or null; sums null: only dx.  parts: how many there are in sums.
int esgd_causal_conv_bwd(const void* x, int64_t xb, int64_t xt, const void* state, const float* weight, const float* bias,
                         const int64_t* lengths, const void* dy, void* dx, float* sums, int64_t* parts, int is_bf16, int64_t batch,
                         int64_t length, int channels, int taps, int act, void* stream) {
  if (!taken(taps, act)) return (int)cudaErrorInvalidValue;
  *parts = 0;
  if (batch == 0 || channels == 0 || length == 0) return 0;
  const int v = width(is_bf16, channels, xb, xt, x, state, dy, dx);
  Conv p = {batch, length, channels, xb, xt, lengths, weight, bias};
  plan(&p, v);
  *parts = p.batch * p.time_blocks;
  return ESGD_TYPE(backward, x, state, dy, dx, sums, p, stream);
}

int esgd_causal_conv_step(const void* x, int64_t xb, const void* state, void* state_out, const float* weight, const float* bias, void* y,
                          int is_bf16, int64_t batch, int channels, int taps, int act, void* stream) {
  if (!taken(taps, act)) return (int)cudaErrorInvalidValue;
  if (batch == 0 || channels == 0) return 0;
  const int v = width(is_bf16, channels, xb, 0, x, state, state_out, y);
  return ESGD_TYPE(step, x, xb, state, state_out, y, weight, bias, batch, channels, stream);
}

}  // extern "C"
