// The short causal convolution ahead of a scan: every channel by itself, over the last K inputs.
//
//   pre[t] = bias + sum_k w[k] x[t - K + 1 + k],   y[t] = act(pre[t])
//   dpre = dy act'(pre);  dx[t] = sum_j w[K - 1 - j] dpre[t + j];  dw[k] = sum dpre[t] x[t - K + 1 + k];  dbias = sum dpre
//
// Bound by memory.  A thread has four channels and a run of steps, the window in registers: of every run only the K - 1 inputs ahead
// of it are read twice (the backward pass makes the K - 1 dpre behind it again).  Eight channels a thread took twice the registers,
// and half the warps were not enough loads in flight; two channels a thread, backward, took 263 us for 235: its instructions count.
//
// 64 x 1000 steps of 2048 channels, four taps, bf16: forward 112 us (4.7 TB/s of 6.5), backward 235 us (3.3); 16 x 331 steps, which L2
// holds: 13.7 and 26 us.
#include "launch.cuh"
#include "rows.cuh"

namespace {

using namespace esgd;

constexpr int kThreads = 256;
// steps that are loaded at a time, while those ahead of them are at work; backward 4 do not fit into the registers (261 -> 235 us with 2;
// 1: 310 us, though 26 -> 23 us where all comes out of L2)
constexpr int kAhead = 4, kBack = 2;

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

template <class T, int kV>
__device__ __forceinline__ void input(const T* x, const T* state, const Conv& p, int64_t b, int64_t t, int c, int taps, f2 (&f)[PairsOf<kV>::n]) {
  if (t >= 0) {
    unpack2<T, kV>(load<T, kV>(x + b * p.xb + t * p.xt + c), f);
  } else if (state != nullptr) {
    unpack2<T, kV>(load<T, kV>(state + (b * (taps - 1) + t + taps - 1) * p.channels + c), f);
  } else {
#pragma unroll
    for (int q = 0; q < PairsOf<kV>::n; ++q) f[q] = 0;
  }
}
template <int kV, int kTaps> struct Filter {
  static constexpr int kP = PairsOf<kV>::n;
  f2 w[kTaps][kP], bias[kP];
  // c: the first of the channels, whose taps lie in a row.
  __device__ Filter(const float* weight, const float* bias_of, int c) {
    float taps[kV * kTaps], b[kV];
    const float* from = weight + (int64_t)c * kTaps;
    if (kV == 4 && ((uintptr_t)from & 15) == 0) {
#pragma unroll
      for (int k = 0; k < kTaps * kV / 4; ++k) {
        const float4 v = reinterpret_cast<const float4*>(from)[k];
        taps[4 * k % (kV * kTaps)] = v.x;
        taps[(4 * k + 1) % (kV * kTaps)] = v.y;
        taps[(4 * k + 2) % (kV * kTaps)] = v.z;
        taps[(4 * k + 3) % (kV * kTaps)] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kV * kTaps; ++i) taps[i] = from[i];
    }
#pragma unroll
    for (int q = 0; q < kV; ++q) b[q] = bias_of != nullptr ? bias_of[c + q] : 0.0f;
#pragma unroll
    for (int q = 0; q < kP; ++q) {
      bias[q] = pair(b[2 * q], kV > 1 ? b[(2 * q + 1) % kV] : 0.0f);
#pragma unroll
      for (int k = 0; k < kTaps; ++k) w[k][q] = pair(taps[2 * q * kTaps + k], kV > 1 ? taps[((2 * q + 1) * kTaps + k) % (kV * kTaps)] : 0.0f);
    }
  }
  __device__ __forceinline__ f2 at(const f2 (&win)[kTaps][kP], int q) const {
    f2 pre = bias[q];
#pragma unroll
    for (int k = 0; k < kTaps; ++k) pre = fma2(w[k][q], win[k][q], pre);
    return pre;
  }
};

template <class T, int kV, int kTaps, int kAct>
__global__ void __launch_bounds__(kThreads) causal_conv_fwd_kernel(const T* __restrict__ x, const T* __restrict__ state, T* __restrict__ y,
                                                                   T* __restrict__ state_out, Conv p) {
  pdl_enter();
  constexpr int kP = PairsOf<kV>::n;
  const Spot<kV> s(p);
  if (!s.on) return;
  if (state_out != nullptr && s.first == (int64_t)s.run * p.steps)        // blocks of the first steps
    for (int i = s.run; i < kTaps - 1; i += p.runs) {
      f2 f[kP];
      input<T, kV>(x, state, p, s.b, s.len - (kTaps - 1) + i, s.c, kTaps, f);
      store2<T, kV>(state_out + (s.b * (kTaps - 1) + i) * p.channels + s.c, f);
    }
  if (s.first >= p.length) return;
  const int steps = (int)(s.last - s.first), live = (int)(s.len - s.first < 0 ? 0 : s.len - s.first < steps ? s.len - s.first : steps);
  const T* in = x + s.b * p.xb + s.first * p.xt + s.c;
  T* out = y + (s.b * p.length + s.first) * p.channels + s.c;
  if (live > 0) {
    const Filter<kV, kTaps> filter(p.weight, p.bias, s.c);
    f2 win[kTaps][kP];
#pragma unroll
    for (int k = 0; k < kTaps - 1; ++k) input<T, kV>(x, state, p, s.b, s.first - (kTaps - 1) + k, s.c, kTaps, win[k + 1]);
    Pack<T, kV> next[kAhead];
    auto fetch = [&](int n) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (u < n) next[u] = load<T, kV>(in + u * p.xt);
      in += kAhead * p.xt;
    };
    fetch(live);
    for (int t = 0; t < live; t += kAhead) {
      Pack<T, kV> raw[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) raw[u] = next[u];
      fetch(live - t - kAhead);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (t + u >= live) break;
        f2 f[kP];
#pragma unroll
        for (int q = 0; q < kP; ++q)
#pragma unroll
          for (int k = 0; k < kTaps - 1; ++k) win[k][q] = win[k + 1][q];
        unpack2<T, kV>(raw[u], win[kTaps - 1]);
#pragma unroll
        for (int q = 0; q < kP; ++q) f[q] = activate2<kAct>(filter.at(win, q));
        store2<T, kV>(out + (int64_t)u * p.channels, f);
      }
      out += (int64_t)kAhead * p.channels;
    }
  }
  const f2 zero[kP] = {};
  for (int t = live; t < steps; ++t) store2<T, kV>(y + (s.b * p.length + s.first + t) * p.channels + s.c, zero);
}

// sums [blocks of a channel][channels * K + channels]: each block's share of dw and dbias.
template <class T, int kV, int kTaps, int kAct>
__global__ void __launch_bounds__(kThreads, 2) causal_conv_bwd_kernel(const T* __restrict__ x, const T* __restrict__ state,
                                                                      const T* __restrict__ dy, T* __restrict__ dx, float* __restrict__ sums,
                                                                      Conv p) {
  pdl_enter();
  constexpr int kP = PairsOf<kV>::n;
  __shared__ __align__(16) float stage[(kTaps + 1) * kThreads * kV];
  const Spot<kV> s(p);
  f2 dw[kTaps + 1][kP];
#pragma unroll
  for (int k = 0; k <= kTaps; ++k)
#pragma unroll
    for (int q = 0; q < kP; ++q) dw[k][q] = 0;
  if (s.on && s.first < p.length) {
    // steps of the run, and up to K - 1 behind it for the gradients of its last inputs
    const int steps = (int)(s.last - s.first), ahead = (int)(s.len - s.first < 0 ? 0 : s.len - s.first < steps + kTaps - 1 ? s.len - s.first : steps + kTaps - 1);
    const T* in = x + s.b * p.xb + s.first * p.xt + s.c;
    const int64_t row = (s.b * p.length + s.first) * p.channels + s.c;
    const T* up = dy + row;
    T* out = dx + row - (int64_t)(kTaps - 1) * p.channels;
    int t = 0;
    if (ahead > 0) {
      const Filter<kV, kTaps> filter(p.weight, p.bias, s.c);
      f2 win[kTaps][kP], dp[kTaps][kP];
#pragma unroll
      for (int q = 0; q < kP; ++q)
#pragma unroll
        for (int k = 0; k < kTaps; ++k) win[k][q] = dp[k][q] = 0;
#pragma unroll
      for (int k = 0; k < kTaps - 1; ++k) input<T, kV>(x, state, p, s.b, s.first - (kTaps - 1) + k, s.c, kTaps, win[k + 1]);
      Pack<T, kV> next_x[kBack], next_d[kBack];
      auto fetch = [&](int n) {
#pragma unroll
        for (int u = 0; u < kBack; ++u)
          if (u < n) {
            next_x[u] = load<T, kV>(in + u * p.xt);
            next_d[u] = load<T, kV>(up + (int64_t)u * p.channels);
          }
        in += kBack * p.xt;
        up += (int64_t)kBack * p.channels;
      };
      fetch(ahead);
      for (; t < steps + kTaps - 1; t += kBack) {
        Pack<T, kV> rx[kBack], rd[kBack];
#pragma unroll
        for (int u = 0; u < kBack; ++u) {
          rx[u] = next_x[u];
          rd[u] = next_d[u];
        }
        fetch(ahead - t - kBack);
#pragma unroll
        for (int u = 0; u < kBack; ++u) {
          if (t + u >= steps + kTaps - 1) break;
#pragma unroll
          for (int q = 0; q < kP; ++q)
#pragma unroll
            for (int k = 0; k < kTaps - 1; ++k) { win[k][q] = win[k + 1][q]; dp[k][q] = dp[k + 1][q]; }
          if (t + u < ahead) {
            f2 d[kP];
            unpack2<T, kV>(rx[u], win[kTaps - 1]);
            unpack2<T, kV>(rd[u], d);
#pragma unroll
            for (int q = 0; q < kP; ++q) {
              if constexpr (kAct != kActNone) d[q] = mul2(d[q], slope2<kAct>(filter.at(win, q)));
              dp[kTaps - 1][q] = d[q];
              if (t + u < steps) {
                dw[kTaps][q] = add2(dw[kTaps][q], d[q]);
#pragma unroll
                for (int k = 0; k < kTaps; ++k) dw[k][q] = fma2(d[q], win[k][q], dw[k][q]);
              }
            }
          } else {
#pragma unroll
            for (int q = 0; q < kP; ++q) dp[kTaps - 1][q] = 0;
          }
          if (t + u >= kTaps - 1 && dx != nullptr) {
            f2 f[kP];
#pragma unroll
            for (int q = 0; q < kP; ++q) {
              f[q] = mul2(filter.w[kTaps - 1][q], dp[0][q]);
#pragma unroll
              for (int j = 1; j < kTaps; ++j) f[q] = fma2(filter.w[kTaps - 1 - j][q], dp[j][q], f[q]);
            }
            store2<T, kV>(out + (int64_t)u * p.channels, f);
          }
        }
        out += (int64_t)kBack * p.channels;
      }
    } else if (dx != nullptr) {
      const f2 zero[kP] = {};
      for (; t < steps; ++t) store2<T, kV>(dx + row + (int64_t)t * p.channels, zero);
    }
  }
  if (sums == nullptr) return;
  float* part = sums + (int64_t)(blockIdx.x / p.vec_blocks) * p.channels * (kTaps + 1);
#pragma unroll
  for (int k = 0; k <= kTaps; ++k) store2<float, kV>(stage + (k * kThreads + threadIdx.x) * kV, dw[k]);
  __syncthreads();
  const int wide = p.lanes * kV, c0 = (int)(blockIdx.x % p.vec_blocks) * wide;
  for (int i = threadIdx.x; i < (kTaps + 1) * wide; i += kThreads) {
    const int k = i / wide, c = i - k * wide;
    if (c0 + c >= p.channels) continue;
    float t = 0.0f;
    for (int r = 0; r < p.runs; ++r) t += stage[(k * kThreads + r * p.lanes) * kV + c];
    part[k < kTaps ? (c0 + c) * kTaps + k : p.channels * kTaps + c0 + c] = t;
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
  constexpr int kP = PairsOf<kV>::n;
  f2 win[kTaps][kP], f[kP];
#pragma unroll
  for (int k = 0; k < kTaps - 1; ++k) unpack2<T, kV>(load<T, kV>(state + (b * (kTaps - 1) + k) * channels + c), win[k]);
  unpack2<T, kV>(load<T, kV>(x + b * xb + c), win[kTaps - 1]);
  const Filter<kV, kTaps> filter(weight, bias, c);
#pragma unroll
  for (int q = 0; q < kP; ++q) f[q] = activate2<kAct>(filter.at(win, q));
  store2<T, kV>(y + b * channels + c, f);
#pragma unroll
  for (int k = 0; k < kTaps - 1; ++k) store2<T, kV>(state_out + (b * (kTaps - 1) + k) * channels + c, win[k + 1]);
}

// Blocks of an SM at a time.
constexpr int kForwardFull = 4, kBackwardFull = 2;
void plan(Conv* p, int v, int full) {
  const int vectors = p->channels / v;
  p->lanes = 1;
  while (p->lanes < 32 && p->lanes < vectors) p->lanes *= 2;
  p->runs = kThreads / p->lanes;
  p->vec_blocks = (vectors + p->lanes - 1) / p->lanes;
  // The number of steps that is estimated to take least: a run begins with what takes as long as 12 steps, an SM has `full` blocks at a
  // time, and a wave of few blocks takes as long as a full one (16 x 331 steps of 2048 channels, backward: 16 steps and three waves
  // 33 us, 44 steps and one wave 26 us).
  p->steps = 64;
  int64_t best = -1;
  for (int steps = 64; steps >= 4; steps -= 4) {
    const int64_t blocks = p->batch * p->vec_blocks * ((p->length + (int64_t)p->runs * steps - 1) / (p->runs * steps));
    const int64_t cost = (blocks + full * sm_count() - 1) / (full * sm_count()) * (steps + 12);
    if (best >= 0 && cost >= best) continue;
    best = cost;
    p->steps = steps;
  }
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
  (is_bf16 ? (v == 4 ? ESGD_TAPS(__nv_bfloat16, 4, F, __VA_ARGS__) : ESGD_TAPS(__nv_bfloat16, 1, F, __VA_ARGS__))     \
           : (v == 4 ? ESGD_TAPS(float, 4, F, __VA_ARGS__) : ESGD_TAPS(float, 1, F, __VA_ARGS__)))

bool taken(int taps, int act) { return taps >= 2 && taps <= 4 && (act == kActSilu || act == kActNone); }
// Channels of a thread: four where all rows begin on a multiple of four.
int width(int is_bf16, int channels, int64_t xb, int64_t xt, const void* a, const void* b, const void* c, const void* d) {
  const uintptr_t bytes = is_bf16 ? 8 : 16;
  return channels % 4 || xb % 4 || xt % 4 || ((uintptr_t)a | (uintptr_t)b | (uintptr_t)c | (uintptr_t)d) % bytes ? 1 : 4;
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
  plan(&p, v, kForwardFull);
  return ESGD_TYPE(forward, x, state, y, state_out, p, stream);
}

// The parts that esgd_causal_conv_bwd leaves in sums, each [channels * taps + channels].
int64_t esgd_causal_conv_parts(int64_t batch, int64_t length, int channels) {
  // the narrowest vector has the most blocks of steps or fewer runs: room for either
  int64_t most = 0;
  for (int v : {1, 4}) {
    if (channels % v) continue;
    Conv p = {batch, length, channels};
    plan(&p, v, kBackwardFull);
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
  plan(&p, v, kBackwardFull);
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
