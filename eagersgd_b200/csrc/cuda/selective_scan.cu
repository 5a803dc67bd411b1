// The selective state-space scan: a recurrence with N states a channel whose decay and input depend on the step.
//
//   dt[t] = softplus(delta[t] + delta_bias)                          (or delta + bias as it is)
//   h[t]  = exp(dt[t] A) h[t - 1] + dt[t] u[t] B[t]                  A [D][N], B and C [T][N] shared by all channels
//   y[t]  = sum_n C[t] h[t] + D u[t],   out[t] = y[t] silu(z[t])
//
// backward, with dy = dout silu(z), a = exp(dt A) and dh[t] = C[t] dy[t] + a[t + 1] dh[t + 1] from the last step back:
//
//   dC = sum_d dy h,  dB = sum_d dh dt u,  dA = sum_t dt a h[t - 1] dh,
//   ddt = sum_n A a h[t - 1] dh + u sum_n B dh,  du = dt sum_n B dh + D dy
//
// One exponential a state and step, against some 8 bytes a channel and step: bound by the special function units, not by memory.
// A channel's states lie in kLanes threads, four in each, all of them in registers over the whole sequence; a tile of steps is
// prepared (dt, B and C in fp32) and finished (sums over the threads, gate) elementwise by way of shared memory.
#include "selective_scan.h"
#include "launch.cuh"
#include "rows.cuh"

namespace {

using namespace esgd;

constexpr int kThreads = 128;
constexpr int kStates = 4;           // of a thread
constexpr int kTile = 32;            // steps of a tile, forward
constexpr int kKeep = 8;             // steps between kept states, and of a tile of the backward pass

// [batch][length][width]: strides in elements, the last one is 1.
struct Seq {
  const void* p;
  int64_t b, t;
};
struct Scan {
  Seq u, delta, z, B, C;             // z.p null: no gate
  const float *A, *D, *bias;         // D, bias: or null
  const int64_t* lengths;            // [batch], or null
  const float* state;                // [batch][channels][states], or null: zero
  int64_t batch, length;
  int channels, states, softplus;
};

__device__ __forceinline__ int64_t length_of(const Scan& s, int64_t b) {
  if (s.lengths == nullptr) return s.length;
  const int64_t n = s.lengths[b];
  return n < 0 ? 0 : n > s.length ? s.length : n;
}
template <class T> __device__ __forceinline__ float at(const Seq& q, int64_t b, int64_t t, int c) {
  return as_float(reinterpret_cast<const T*>(q.p)[b * q.b + t * q.t + c]);
}
__device__ __forceinline__ float softplus(float x) { return x > 20.0f ? x : log1pf(exp_fine(x)); }
__device__ __forceinline__ float time_step(const Scan& s, float delta, int c) {
  const float raw = delta + (s.bias != nullptr ? s.bias[c] : 0.0f);
  return s.softplus ? softplus(raw) : raw;
}

// A block's channels [c0, c0 + kWide), and the states of a thread of them.
template <int kLanes> struct Spot {
  static constexpr int kWide = kThreads / kLanes;
  int64_t b;
  int block, c0, c, lane;      // c: the thread's channel within the block
  __device__ explicit Spot(const Scan& s) {
    const int blocks = (s.channels + kWide - 1) / kWide;
    b = blockIdx.x / blocks;
    block = (int)(blockIdx.x - b * blocks);
    c0 = block * kWide;
    c = threadIdx.x / kLanes;
    lane = threadIdx.x % kLanes;
  }
};

// keep: [tiles of kKeep steps][batch][channels][kLanes * 4], the state ahead of every eighth step; or null.
template <class T, int kLanes>
__global__ void __launch_bounds__(kThreads) selective_scan_fwd_kernel(Scan s, T* __restrict__ out, float* __restrict__ state_out,
                                                                      float* __restrict__ keep) {
  pdl_enter();
  constexpr int kWide = Spot<kLanes>::kWide;
  extern __shared__ float4 smem4[];
  float4* s_bc = smem4;                                               // [kTile][2][kLanes]
  float2* s_dt = reinterpret_cast<float2*>(s_bc + kTile * 2 * kLanes);   // [kTile][kWide]: dt, dt * u
  float* s_y = reinterpret_cast<float*>(s_dt + kTile * kWide);        // [kTile][kWide][kLanes]
  const Spot<kLanes> p(s);
  const int64_t len = length_of(s, p.b);
  const int channel = p.c0 + p.c;
  const bool on = channel < s.channels;
  float a[kStates], h[kStates];
#pragma unroll
  for (int j = 0; j < kStates; ++j) {
    const int n = p.lane * kStates + j;
    const bool is = on && n < s.states;
    a[j] = is ? s.A[(int64_t)channel * s.states + n] * kLog2e : 0.0f;
    h[j] = is && s.state != nullptr ? s.state[(p.b * s.channels + channel) * s.states + n] : 0.0f;
  }
  T* y = out + p.b * s.length * s.channels;
  for (int64_t t0 = 0; t0 < len; t0 += kTile) {
    const int steps = (int)(len - t0 < kTile ? len - t0 : kTile);
    for (int i = threadIdx.x; i < steps * kWide; i += kThreads) {
      const int t = i / kWide, c = p.c0 + i % kWide;
      float2 v = make_float2(0.0f, 0.0f);
      if (c < s.channels) {
        v.x = time_step(s, at<T>(s.delta, p.b, t0 + t, c), c);
        v.y = v.x * at<T>(s.u, p.b, t0 + t, c);
      }
      s_dt[i] = v;
    }
    float* bc = reinterpret_cast<float*>(s_bc);
    for (int i = threadIdx.x; i < steps * 2 * kLanes * kStates; i += kThreads) {
      const int t = i / (2 * kLanes * kStates), k = i / (kLanes * kStates) % 2, n = i % (kLanes * kStates);
      bc[i] = n < s.states ? at<T>(k == 0 ? s.B : s.C, p.b, t0 + t, n) : 0.0f;
    }
    __syncthreads();
#pragma unroll 4
    for (int t = 0; t < steps; ++t) {
      if (keep != nullptr && t % kKeep == 0 && on)
        reinterpret_cast<float4*>(keep)[(((t0 + t) / kKeep * s.batch + p.b) * s.channels + channel) * kLanes + p.lane] =
            make_float4(h[0], h[1], h[2], h[3]);
      const float2 dt = s_dt[t * kWide + p.c];
      const float4 b4 = s_bc[(t * 2) * kLanes + p.lane], c4 = s_bc[(t * 2 + 1) * kLanes + p.lane];
      const float b[4] = {b4.x, b4.y, b4.z, b4.w}, c[4] = {c4.x, c4.y, c4.z, c4.w};
      float part = 0.0f;
#pragma unroll
      for (int j = 0; j < kStates; ++j) {
        h[j] = fmaf(exp2_approx(dt.x * a[j]), h[j], dt.y * b[j]);
        part = fmaf(c[j], h[j], part);
      }
      s_y[t * kThreads + threadIdx.x] = part;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < steps * kWide; i += kThreads) {
      const int t = i / kWide, c = p.c0 + i % kWide;
      if (c >= s.channels) continue;
      float v = 0.0f;
#pragma unroll
      for (int l = 0; l < kLanes; ++l) v += s_y[i * kLanes + l];
      if (s.D != nullptr) v = fmaf(s.D[c], at<T>(s.u, p.b, t0 + t, c), v);
      if (s.z.p != nullptr) v *= activate<kActSilu>(at<T>(s.z, p.b, t0 + t, c));
      y[(t0 + t) * s.channels + c] = as_type<T>(v);
    }
  }
  for (int64_t i = threadIdx.x; i < (s.length - len) * kWide; i += kThreads) {
    const int c = p.c0 + (int)(i % kWide);
    if (c < s.channels) y[(len + i / kWide) * s.channels + c] = as_type<T>(0.0f);
  }
  if (state_out != nullptr && on)
#pragma unroll
    for (int j = 0; j < kStates; ++j) {
      const int n = p.lane * kStates + j;
      if (n < s.states) state_out[(p.b * s.channels + channel) * s.states + n] = h[j];
    }
}

struct Grads {
  const void* dout;            // [batch][length][channels]
  const float* keep;
  void *du, *ddelta, *dz;      // like dout; dz null without a gate
  float* narrow;               // [blocks of channels][batch][length][2][kLanes * 4]: shares of dB, dC
  float* sums;                 // [batch][channels * states + channels + channels]: dA, dD, ddelta_bias of a sequence
};

template <class T, int kLanes>
__global__ void __launch_bounds__(kThreads) selective_scan_bwd_kernel(Scan s, Grads g) {
  pdl_enter();
  constexpr int kWide = Spot<kLanes>::kWide, kPadded = kLanes * kStates, kWarps = kThreads / 32;
  __shared__ float4 s_bc[kKeep * 2 * kLanes];
  __shared__ float2 s_dt[kKeep * kWide];
  __shared__ float s_dy[kKeep * kWide];
  __shared__ float s_part[3][kKeep * kThreads];          // over a thread's states: C h, B dh, A a h[t - 1] dh
  __shared__ float s_narrow[kWarps][kKeep][2][kPadded];  // over a warp's channels: dh dt u, dy h
  const Spot<kLanes> p(s);
  const int64_t len = length_of(s, p.b);
  const int channel = p.c0 + p.c, warp = threadIdx.x / 32;
  const bool on = channel < s.channels;
  float A[kStates], carry[kStates], dA[kStates];
#pragma unroll
  for (int j = 0; j < kStates; ++j) {
    const int n = p.lane * kStates + j;
    A[j] = on && n < s.states ? s.A[(int64_t)channel * s.states + n] : 0.0f;
    carry[j] = dA[j] = 0.0f;
  }
  float dD = 0.0f, dbias = 0.0f;                         // of channel p.c0 + threadIdx.x % kWide, every kThreads / kWide-th step
  const T* dout = reinterpret_cast<const T*>(g.dout) + p.b * s.length * s.channels;
  T* du = reinterpret_cast<T*>(g.du) + p.b * s.length * s.channels;
  T* ddelta = reinterpret_cast<T*>(g.ddelta) + p.b * s.length * s.channels;
  T* dz = g.dz != nullptr ? reinterpret_cast<T*>(g.dz) + p.b * s.length * s.channels : nullptr;
  for (int64_t tile = (len + kKeep - 1) / kKeep - 1; tile >= 0; --tile) {
    const int64_t t0 = tile * kKeep;
    const int steps = (int)(len - t0 < kKeep ? len - t0 : kKeep);
    for (int i = threadIdx.x; i < kKeep * kWide; i += kThreads) {
      const int t = i / kWide, c = p.c0 + i % kWide;
      float2 v = make_float2(0.0f, 0.0f);
      float d = 0.0f;
      if (c < s.channels && t < steps) {
        v.x = time_step(s, at<T>(s.delta, p.b, t0 + t, c), c);
        v.y = v.x * at<T>(s.u, p.b, t0 + t, c);
        d = as_float(dout[(t0 + t) * s.channels + c]);
        if (s.z.p != nullptr) d *= activate<kActSilu>(at<T>(s.z, p.b, t0 + t, c));
      }
      s_dt[i] = v;
      s_dy[i] = d;
    }
    float* bc = reinterpret_cast<float*>(s_bc);
    for (int i = threadIdx.x; i < kKeep * 2 * kPadded; i += kThreads) {
      const int t = i / (2 * kPadded), k = i / kPadded % 2, n = i % kPadded;
      bc[i] = n < s.states && t < steps ? at<T>(k == 0 ? s.B : s.C, p.b, t0 + t, n) : 0.0f;
    }
    __syncthreads();
    float4 first = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (on) first = reinterpret_cast<const float4*>(g.keep)[((tile * s.batch + p.b) * s.channels + channel) * kLanes + p.lane];
    float h[kKeep + 1][kStates], a[kKeep][kStates];
    h[0][0] = first.x; h[0][1] = first.y; h[0][2] = first.z; h[0][3] = first.w;
#pragma unroll
    for (int t = 0; t < kKeep; ++t) {
      const float2 dt = s_dt[t * kWide + p.c];
      const float4 b4 = s_bc[(t * 2) * kLanes + p.lane];
      const float b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
      for (int j = 0; j < kStates; ++j) {
        a[t][j] = exp2_approx(dt.x * (A[j] * kLog2e));
        h[t + 1][j] = fmaf(a[t][j], h[t][j], dt.y * b[j]);
      }
    }
#pragma unroll
    for (int t = kKeep - 1; t >= 0; --t) {
      const float2 dt = s_dt[t * kWide + p.c];
      const float dy = s_dy[t * kWide + p.c];
      const float4 b4 = s_bc[(t * 2) * kLanes + p.lane], c4 = s_bc[(t * 2 + 1) * kLanes + p.lane];
      const float b[4] = {b4.x, b4.y, b4.z, b4.w}, c[4] = {c4.x, c4.y, c4.z, c4.w};
      float ch = 0.0f, bdh = 0.0f, ada = 0.0f, share[8];
#pragma unroll
      for (int j = 0; j < kStates; ++j) {
        const float dh = fmaf(c[j], dy, carry[j]);
        carry[j] = a[t][j] * dh;
        const float da = carry[j] * h[t][j];
        dA[j] = fmaf(da, dt.x, dA[j]);
        ada = fmaf(da, A[j], ada);
        bdh = fmaf(b[j], dh, bdh);
        ch = fmaf(c[j], h[t + 1][j], ch);
        share[j] = dh * dt.y;
        share[4 + j] = dy * h[t + 1][j];
      }
      s_part[0][t * kThreads + threadIdx.x] = ch;
      s_part[1][t * kThreads + threadIdx.x] = bdh;
      s_part[2][t * kThreads + threadIdx.x] = ada;
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int o = 16; o >= kLanes; o >>= 1) share[j] += __shfl_xor_sync(0xffffffffu, share[j], o);
      if ((threadIdx.x & 31) < kLanes)
#pragma unroll
        for (int j = 0; j < 8; ++j) s_narrow[warp][t][j / 4][p.lane * kStates + j % 4] = share[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < steps * 2 * kPadded; i += kThreads) {
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v += (&s_narrow[w][0][0][0])[i];
      g.narrow[(((int64_t)p.block * s.batch + p.b) * s.length + t0) * 2 * kPadded + i] = v;
    }
    for (int i = threadIdx.x; i < steps * kWide; i += kThreads) {
      const int t = i / kWide, c = p.c0 + i % kWide;
      if (c >= s.channels) continue;
      float y = 0.0f, bdh = 0.0f, ddt = 0.0f;
#pragma unroll
      for (int l = 0; l < kLanes; ++l) {
        y += s_part[0][i * kLanes + l];
        bdh += s_part[1][i * kLanes + l];
        ddt += s_part[2][i * kLanes + l];
      }
      const int64_t o = (t0 + t) * s.channels + c;
      const float u = at<T>(s.u, p.b, t0 + t, c), raw = at<T>(s.delta, p.b, t0 + t, c) + (s.bias != nullptr ? s.bias[c] : 0.0f);
      const float skip = s.D != nullptr ? s.D[c] : 0.0f, dy = s_dy[i];
      if (dz != nullptr) {
        const float z = at<T>(s.z, p.b, t0 + t, c);
        dz[o] = as_type<T>(as_float(dout[o]) * fmaf(skip, u, y) * slope<kActSilu>(z));
      }
      ddt = fmaf(bdh, u, ddt);
      if (s.softplus) ddt *= sigmoid(raw);
      du[o] = as_type<T>(fmaf(bdh, s_dt[i].x, skip * dy));
      ddelta[o] = as_type<T>(ddt);
      dD = fmaf(dy, u, dD);
      dbias += ddt;
    }
    __syncthreads();
  }
  for (int64_t i = threadIdx.x; i < (s.length - len) * kWide; i += kThreads) {
    const int c = p.c0 + (int)(i % kWide);
    if (c >= s.channels) continue;
    const int64_t o = (len + i / kWide) * s.channels + c;
    du[o] = ddelta[o] = as_type<T>(0.0f);
    if (dz != nullptr) dz[o] = as_type<T>(0.0f);
  }
  float* sums = g.sums + p.b * (int64_t)s.channels * (s.states + 2);
  if (on)
#pragma unroll
    for (int j = 0; j < kStates; ++j) {
      const int n = p.lane * kStates + j;
      if (n < s.states) sums[(int64_t)channel * s.states + n] = dA[j];
    }
  s_part[0][threadIdx.x] = dD;
  s_part[1][threadIdx.x] = dbias;
  __syncthreads();
  for (int i = threadIdx.x; i < kWide; i += kThreads) {
    if (p.c0 + i >= s.channels) break;
    float v = 0.0f, w = 0.0f;
    for (int k = i; k < kThreads; k += kWide) { v += s_part[0][k]; w += s_part[1][k]; }
    sums[(int64_t)s.channels * s.states + p.c0 + i] = v;
    sums[(int64_t)s.channels * (s.states + 1) + p.c0 + i] = w;
  }
}

// dB, dC [batch][length][states] out of the shares of the blocks; nothing behind a sequence's end.
template <class T>
__global__ void __launch_bounds__(256) selective_scan_narrow_kernel(const float* __restrict__ narrow, int blocks, Scan s, int padded,
                                                                    T* __restrict__ dB, T* __restrict__ dC) {
  pdl_enter();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, n = s.batch * s.length * 2 * padded;
  if (i >= n) return;
  const int64_t row = i / (2 * padded);
  const int k = (int)(i - row * 2 * padded) / padded, j = (int)(i % padded);
  if (j >= s.states) return;
  const int64_t b = row / s.length;
  float v = 0.0f;
  if (row - b * s.length < length_of(s, b))
    for (int q = 0; q < blocks; ++q) v += narrow[q * n + i];
  (k == 0 ? dB : dC)[row * s.states + j] = as_type<T>(v);
}

// One step of every sequence: the state moves on; state_out may be s.state.
template <class T, int kLanes>
__global__ void __launch_bounds__(kThreads) selective_scan_step_kernel(Scan s, float* state_out, T* __restrict__ out) {
  pdl_enter();
  constexpr int kWide = Spot<kLanes>::kWide;
  const int blocks = (s.channels + kWide - 1) / kWide;
  const int64_t b = blockIdx.x / blocks;
  const int c = (int)(blockIdx.x - b * blocks) * kWide + threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  const bool on = c < s.channels;
  float part = 0.0f, u = 0.0f;
  if (on) {
    u = at<T>(s.u, b, 0, c);
    const float dt = time_step(s, at<T>(s.delta, b, 0, c), c);
#pragma unroll
    for (int j = 0; j < kStates; ++j) {
      const int n = lane * kStates + j;
      if (n >= s.states) break;
      const int64_t i = (b * s.channels + c) * s.states + n;
      const float h = fmaf(exp2_approx(dt * (s.A[(int64_t)c * s.states + n] * kLog2e)), s.state[i], dt * u * at<T>(s.B, b, 0, n));
      state_out[i] = h;
      part = fmaf(at<T>(s.C, b, 0, n), h, part);
    }
  }
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
  if (on && lane == 0) {
    if (s.D != nullptr) part = fmaf(s.D[c], u, part);
    if (s.z.p != nullptr) part *= activate<kActSilu>(at<T>(s.z, b, 0, c));
    out[b * s.channels + c] = as_type<T>(part);
  }
}

int lanes_of(int states) {
  int l = 1;
  while (l * kStates < states) l *= 2;
  return l;
}
int blocks_of(int channels, int lanes) { return (channels + kThreads / lanes - 1) / (kThreads / lanes); }

template <class T, int kLanes> int forward(const Scan& s, void* out, float* state_out, float* keep, void* stream) {
  static SmemAllowed allowed{0};
  constexpr int kWide = kThreads / kLanes;
  constexpr size_t kSmem = kTile * (2 * kLanes * 16 + kWide * 8 + kThreads * 4);
  if (kSmem > 48 * 1024) {
    const int rc = allow_smem(selective_scan_fwd_kernel<T, kLanes>, kSmem, allowed);
    if (rc != 0) return rc;
  }
  return launch(selective_scan_fwd_kernel<T, kLanes>, dim3((unsigned)(s.batch * blocks_of(s.channels, kLanes))), kThreads, kSmem, stream, s,
                (T*)out, state_out, keep);
}
template <class T, int kLanes> int backward(const Scan& s, const Grads& g, void* dB, void* dC, void* stream) {
  const int blocks = blocks_of(s.channels, kLanes);
  const int rc = launch(selective_scan_bwd_kernel<T, kLanes>, dim3((unsigned)(s.batch * blocks)), kThreads, 0, stream, s, g);
  if (rc != 0) return rc;
  const int64_t n = s.batch * s.length * 2 * kLanes * kStates;
  return launch(selective_scan_narrow_kernel<T>, dim3((unsigned)((n + 255) / 256)), 256, 0, stream, g.narrow, blocks, s, kLanes * kStates,
                (T*)dB, (T*)dC);
}
template <class T, int kLanes> int step(const Scan& s, float* state_out, void* out, void* stream) {
  return launch(selective_scan_step_kernel<T, kLanes>, dim3((unsigned)(s.batch * blocks_of(s.channels, kLanes))), kThreads, 0, stream, s,
                state_out, (T*)out);
}

// F<T, kLanes>(...)
#define ESGD_LANES(T, F, ...)                                                                                   \
  (lanes == 1 ? F<T, 1>(__VA_ARGS__) : lanes == 2 ? F<T, 2>(__VA_ARGS__) : lanes == 4 ? F<T, 4>(__VA_ARGS__)    \
   : lanes == 8 ? F<T, 8>(__VA_ARGS__) : F<T, 16>(__VA_ARGS__))
#define ESGD_TYPE(F, ...) (is_bf16 ? ESGD_LANES(__nv_bfloat16, F, __VA_ARGS__) : ESGD_LANES(float, F, __VA_ARGS__))

bool taken(const Scan& s) { return s.states >= 1 && s.states <= 64 && s.channels >= 1 && s.batch >= 0 && s.length >= 0; }

}  // namespace

extern "C" {

static Scan scan_of(const esgd_scan* e) {
  Scan s;
  Seq* q[5] = {&s.u, &s.delta, &s.z, &s.B, &s.C};
  for (int i = 0; i < 5; ++i) *q[i] = {e->p[i], e->b[i], e->t[i]};
  s.A = e->A; s.D = e->D; s.bias = e->bias;
  s.lengths = e->lengths;
  s.state = e->state;
  s.batch = e->batch; s.length = e->length;
  s.channels = e->channels; s.states = e->states; s.softplus = e->softplus;
  return s;
}

// Floats that the forward pass keeps for the backward pass, and that the backward pass needs beside it.
int64_t esgd_selective_scan_keep(int64_t batch, int64_t length, int channels, int states) {
  return (length + kKeep - 1) / kKeep * batch * channels * lanes_of(states) * kStates;
}
int64_t esgd_selective_scan_narrow(int64_t batch, int64_t length, int channels, int states) {
  const int lanes = lanes_of(states);
  return blocks_of(channels, lanes) * batch * length * 2 * lanes * kStates;
}

int esgd_selective_scan_fwd(const esgd_scan* e, void* out, float* state_out, float* keep, void* stream) {
  const Scan s = scan_of(e);
  if (!taken(s)) return (int)cudaErrorInvalidValue;
  if (s.batch == 0) return 0;
  const int is_bf16 = e->is_bf16, lanes = lanes_of(s.states);
  return ESGD_TYPE(forward, s, out, state_out, keep, stream);
}

int esgd_selective_scan_bwd(const esgd_scan* e, const void* dout, const float* keep, void* du, void* ddelta, void* dz, void* dB, void* dC,
                            float* narrow, float* sums, void* stream) {
  const Scan s = scan_of(e);
  if (!taken(s)) return (int)cudaErrorInvalidValue;
  if (s.batch == 0 || s.length == 0) return 0;
  const int is_bf16 = e->is_bf16, lanes = lanes_of(s.states);
  const Grads g = {dout, keep, du, ddelta, dz, narrow, sums};
  return ESGD_TYPE(backward, s, g, dB, dC, stream);
}

int esgd_selective_scan_step(const esgd_scan* e, float* state_out, void* out, void* stream) {
  const Scan s = scan_of(e);
  if (!taken(s) || s.state == nullptr) return (int)cudaErrorInvalidValue;
  if (s.batch == 0) return 0;
  const int is_bf16 = e->is_bf16, lanes = lanes_of(s.states);
  return ESGD_TYPE(step, s, state_out, out, stream);
}

}  // extern "C"
