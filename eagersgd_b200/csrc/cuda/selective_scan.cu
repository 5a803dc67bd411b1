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
// One exponential a state and step, against some 8 bytes a channel and step: bound by the special function units and the issue of
// instructions, not by memory.  States stay in registers over the whole sequence, two to a 64-bit register for the paired fp32
// instructions.  A tile of steps is prepared elementwise (a thread: two neighbouring channels of a step; their operands are fetched
// a tile ahead), goes through shared memory to the threads that have the states, and comes back for the sums over the states and
// the gates.
//
// Forward: a channel's states lie in kLanes threads, four in each.  Backward: a warp has eight channels and sixteen states, a
// thread two by two of them as the tensor cores' m16n8k8 fragments want them: the sums over the channels that dB and dC are, eight
// values a thread and step, are two matrix instructions instead of some forty shuffles and additions.  The states ahead of every
// eighth step are kept by the forward pass, so that the backward pass needs one exponential a state and step as well.
//
// Few sequences of few channels: the steps are split into chunks that run at the same time.  A first pass scans every chunk from a
// state of zero; what a chunk begins with is then the chunks ahead of it joined, h = exp(A sum dt) h + (its own scan).
#include "selective_scan.h"
#include "launch.cuh"
#include "rows.cuh"

namespace {

using namespace esgd;

constexpr int kThreads = 128;
constexpr int kStates = 4;           // of a thread
constexpr int kTile = 16;            // steps of a tile, forward
constexpr int kKeep = 8;             // steps between kept states, and of a tile of the backward pass
constexpr int kMaxChunks = 64;

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
  int even, even_narrow;             // neighbouring channels (states) are one load: even counts, strides and beginnings
  int chunks;
  int64_t chunk;                     // steps of a chunk, a multiple of kTile
  float *local, *span;               // [chunks][batch][channels][kLanes * 4] and [chunks][batch][channels], with more than one chunk
};

__device__ __forceinline__ int64_t length_of(const Scan& s, int64_t b) {
  if (s.lengths == nullptr) return s.length;
  const int64_t n = s.lengths[b];
  return n < 0 ? 0 : n > s.length ? s.length : n;
}

// log(1 + e^x) = max(x, 0) + log(1 + v) with v = e^-|x|, and log(1 + v) = 2 artanh(v / (2 + v)): an odd function whose argument
// is at most 1/3, so five terms, fitted to the relative error, are right to 4e-9.  slope: 1 / (1 + e^-x).
__device__ __forceinline__ float softplus(float x, float* slope = nullptr) {
  const float v = exp2_approx(fminf(fabsf(x), 120.0f) * -kLog2e);
  const float r = v * reciprocal(2.0f + v), q = r * r;
  const float log = fmaf(fmaf(fmaf(fmaf(0.281614542f, q, 0.279643446f), q, 0.400246501f), q, 0.666663229f), q, 2.0f);
  float top;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(top) : "f"(x), "f"(0.0f));
  if (slope != nullptr) *slope = reciprocal(1.0f + v) * (x < 0.0f ? v : 1.0f);
  return fmaf(r, log, top);
}

// Two neighbouring values as they lie in memory.
template <class T> struct Two;
template <> struct Two<float> {
  float a, b;
  __device__ __forceinline__ void load(const float* p) { const float2 v = *reinterpret_cast<const float2*>(p); a = v.x; b = v.y; }
  __device__ __forceinline__ void set(float x, float y) { a = x; b = y; }
  __device__ __forceinline__ float2 get() const { return make_float2(a, b); }
};
template <> struct Two<__nv_bfloat16> {
  uint32_t w;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { w = *reinterpret_cast<const uint32_t*>(p); }
  __device__ __forceinline__ void set(__nv_bfloat16 x, __nv_bfloat16 y) {
    w = (uint32_t)__bfloat16_as_ushort(x) | (uint32_t)__bfloat16_as_ushort(y) << 16;
  }
  __device__ __forceinline__ float2 get() const { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
};
// Values c and c + 1 of a row of `width`, zero beyond it.
template <class T> __device__ __forceinline__ Two<T> fetch(const T* row, int c, int width, int even) {
  Two<T> r;
  if (even && c < width) r.load(row + c);
  else r.set(c < width ? row[c] : as_type<T>(0.0f), c + 1 < width ? row[c + 1] : as_type<T>(0.0f));
  return r;
}
template <class T> __device__ __forceinline__ Two<T> fetch(const Seq& q, int64_t b, int64_t t, int c, int width, int even) {
  return fetch<T>(reinterpret_cast<const T*>(q.p) + b * q.b + t * q.t, c, width, even);
}
template <class T> __device__ __forceinline__ void put(T* row, int c, int width, int even, float x, float y) {
  if (even && c < width) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(row + c) = make_float2(x, y);
    else *reinterpret_cast<__nv_bfloat162*>(row + c) = __floats2bfloat162_rn(x, y);
  } else {
    if (c < width) row[c] = as_type<T>(x);
    if (c + 1 < width) row[c + 1] = as_type<T>(y);
  }
}
__device__ __forceinline__ float2 two_of(const float* p, int c, int width) {
  return make_float2(p != nullptr && c < width ? p[c] : 0.0f, p != nullptr && c + 1 < width ? p[c + 1] : 0.0f);
}

// Paired fp32 arithmetic.
using f2 = unsigned long long;
__device__ __forceinline__ f2 pair(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 halves(f2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 exp2_2(f2 x) {
  const float2 v = halves(x);
  return pair(exp2_approx(v.x), exp2_approx(v.y));
}
__device__ __forceinline__ float sum_of(f2 v) {
  const float2 h = halves(v);
  return h.x + h.y;
}

// A block: a sequence's channels [c0, c0 + kWide) and steps [first, last) of a chunk, as far as the sequence goes.
template <int kWide_> struct Block {
  static constexpr int kWide = kWide_;
  int64_t b, len, first, last, end;      // end: of the chunk, where the sequence is shorter
  int block, c0, chunk;
  __device__ explicit Block(const Scan& s) {
    const int blocks = (s.channels + kWide - 1) / kWide;
    const int64_t rest = blockIdx.x / blocks;
    block = (int)(blockIdx.x - rest * blocks);
    b = rest / s.chunks;
    chunk = (int)(rest - b * s.chunks);
    c0 = block * kWide;
    len = length_of(s, b);
    first = chunk * s.chunk;
    end = chunk + 1 < s.chunks ? first + s.chunk : s.length;
    last = end < len ? end : len;
  }
};

// The steps' operands of a thread, fetched a tile ahead: kPairs pairs of channels and kNarrow pairs of states.
template <class T, int kLanes> struct Ahead {
  static constexpr int kWide = kThreads / kLanes, kPadded = kLanes * kStates;
  static constexpr int kPairs = kTile * kWide / 2 <= kThreads ? 1 : kTile * kWide / 2 / kThreads;
  // a row of partial sums: a warp's channels of every lane fall into banks of their own
  static constexpr int kRow = kWide + (32 / kLanes - kWide % 32 + 32) % 32;
  static constexpr int kNarrow = kTile * kPadded / 2 <= kThreads ? 1 : kTile * kPadded / 2 / kThreads;
  __device__ static __forceinline__ int step(int k) { return (threadIdx.x + k * kThreads) / (kWide / 2); }
  __device__ static __forceinline__ int channel(int k) { return (threadIdx.x + k * kThreads) % (kWide / 2) * 2; }
  __device__ static __forceinline__ int narrow_step(int k) { return (threadIdx.x + k * kThreads) / (kPadded / 2); }
  __device__ static __forceinline__ int state(int k) { return (threadIdx.x + k * kThreads) % (kPadded / 2) * 2; }
};

// The states that a block begins with: the given one (forward) or none (backward), and the other chunks' joined to it.
template <int kLanes, bool kReverse>
__device__ __forceinline__ void joined(const Scan& s, int64_t b, int chunk, int channel, int lane, const float (&a)[kStates], float (&h)[kStates]) {
  if (s.chunks <= 1) return;
  for (int i = kReverse ? s.chunks - 1 : 0; i != chunk; kReverse ? --i : ++i) {
    const int64_t at = (i * s.batch + b) * s.channels + channel;
    const float span = s.span[at];
    const float4 l = reinterpret_cast<const float4*>(s.local)[at * kLanes + lane];
    const float own[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
    for (int j = 0; j < kStates; ++j) h[j] = fmaf(exp2_approx(span * a[j]), h[j], own[j]);
  }
}

// keep: [tiles of kKeep steps][batch][channels][kLanes * 4], the state ahead of every eighth step; or null.
template <class T, int kLanes>
__global__ void __launch_bounds__(kThreads) selective_scan_fwd_kernel(Scan s, T* __restrict__ out, float* __restrict__ state_out,
                                                                      float* __restrict__ keep) {
  pdl_enter();
  using In = Ahead<T, kLanes>;
  constexpr int kWide = In::kWide, kPadded = In::kPadded;
  extern __shared__ float4 smem4[];
  float4* s_bc = smem4;                                                   // [kTile][kLanes][2]: four of B, four of C
  float4* s_dt = s_bc + kTile * 2 * kLanes;                               // [kTile][kWide]: dt twice, dt * u twice
  float* s_y = reinterpret_cast<float*>(s_dt + kTile * kWide);            // [kTile][kLanes][In::kRow]
  const Block<kWide> p(s);
  const int c = threadIdx.x / kLanes, lane = threadIdx.x % kLanes, channel = p.c0 + c;
  const bool on = channel < s.channels;
  float a[kStates], start[kStates];
#pragma unroll
  for (int j = 0; j < kStates; ++j) {
    const int n = lane * kStates + j;
    const bool is = on && n < s.states;
    a[j] = is ? s.A[(int64_t)channel * s.states + n] * kLog2e : 0.0f;
    start[j] = is && s.state != nullptr ? s.state[(p.b * s.channels + channel) * s.states + n] : 0.0f;
  }
  if (on) joined<kLanes, false>(s, p.b, p.chunk, channel, lane, a, start);
  const f2 a0 = pair(a[0], a[1]), a1 = pair(a[2], a[3]);
  f2 h0 = pair(start[0], start[1]), h1 = pair(start[2], start[3]);
  T* y = out + p.b * s.length * s.channels;

  Two<T> u[In::kPairs], delta[In::kPairs], z[In::kPairs], bb[In::kNarrow], cc[In::kNarrow];
  auto prefetch = [&](int64_t t0) {
#pragma unroll
    for (int k = 0; k < In::kPairs; ++k) {
      const int64_t t = t0 + In::step(k);
      if (In::step(k) < kTile && t < p.last) {
        u[k] = fetch<T>(s.u, p.b, t, p.c0 + In::channel(k), s.channels, s.even);
        delta[k] = fetch<T>(s.delta, p.b, t, p.c0 + In::channel(k), s.channels, s.even);
        if (s.z.p != nullptr) z[k] = fetch<T>(s.z, p.b, t, p.c0 + In::channel(k), s.channels, s.even);
      }
    }
#pragma unroll
    for (int k = 0; k < In::kNarrow; ++k) {
      const int64_t t = t0 + In::narrow_step(k);
      if (In::narrow_step(k) < kTile && t < p.last) {
        bb[k] = fetch<T>(s.B, p.b, t, In::state(k), s.states, s.even_narrow);
        cc[k] = fetch<T>(s.C, p.b, t, In::state(k), s.states, s.even_narrow);
      }
    }
  };
  float2 skip[In::kPairs], bias[In::kPairs];
#pragma unroll
  for (int k = 0; k < In::kPairs; ++k) {
    skip[k] = two_of(s.D, p.c0 + In::channel(k), s.channels);
    bias[k] = two_of(s.bias, p.c0 + In::channel(k), s.channels);
  }
  if (p.first < p.last) prefetch(p.first);
  for (int64_t t0 = p.first; t0 < p.last; t0 += kTile) {
    const int steps = (int)(p.last - t0 < kTile ? p.last - t0 : kTile);
    float2 du[In::kPairs], gate[In::kPairs];             // D u and silu(z) of the tile, for its end
#pragma unroll
    for (int k = 0; k < In::kPairs; ++k) {
      if (In::step(k) >= steps) continue;
      const float2 uv = u[k].get(), dv = delta[k].get();
      const float x = dv.x + bias[k].x, w = dv.y + bias[k].y;
      const float tx = s.softplus ? softplus(x) : x, tw = s.softplus ? softplus(w) : w;
      float4* to = s_dt + In::step(k) * kWide + In::channel(k);
      to[0] = make_float4(tx, tx, tx * uv.x, tx * uv.x);
      to[1] = make_float4(tw, tw, tw * uv.y, tw * uv.y);
      du[k] = make_float2(skip[k].x * uv.x, skip[k].y * uv.y);
      gate[k] = make_float2(1.0f, 1.0f);
      if (s.z.p != nullptr) {
        const float2 zv = z[k].get();
        gate[k] = make_float2(activate<kActSilu>(zv.x), activate<kActSilu>(zv.y));
      }
    }
    float* bc = reinterpret_cast<float*>(s_bc);
#pragma unroll
    for (int k = 0; k < In::kNarrow; ++k) {
      if (In::narrow_step(k) >= steps) continue;
      const int n = In::state(k);
      float* to = bc + In::narrow_step(k) * 2 * kPadded + n / kStates * 2 * kStates + n % kStates;
      *reinterpret_cast<float2*>(to) = bb[k].get();
      *reinterpret_cast<float2*>(to + kStates) = cc[k].get();
    }
    __syncthreads();
    if (t0 + kTile < p.last) prefetch(t0 + kTile);
    const ulonglong2* bc2 = reinterpret_cast<const ulonglong2*>(s_bc) + lane * 2;
    const ulonglong2* dt2 = reinterpret_cast<const ulonglong2*>(s_dt) + c;
#pragma unroll 8
    for (int t = 0; t < steps; ++t) {
      if (keep != nullptr && t % kKeep == 0 && on) {
        const float2 x = halves(h0), w = halves(h1);
        reinterpret_cast<float4*>(keep)[(((t0 + t) / kKeep * s.batch + p.b) * s.channels + channel) * kLanes + lane] =
            make_float4(x.x, x.y, w.x, w.y);
      }
      const ulonglong2 dt = dt2[t * kWide], b2 = bc2[t * 2 * kLanes], c2 = bc2[t * 2 * kLanes + 1];
      h0 = fma2(exp2_2(mul2(dt.x, a0)), h0, mul2(dt.y, b2.x));
      h1 = fma2(exp2_2(mul2(dt.x, a1)), h1, mul2(dt.y, b2.y));
      s_y[(t * kLanes + lane) * In::kRow + c] = sum_of(fma2(c2.y, h1, mul2(c2.x, h0)));
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < In::kPairs; ++k) {
      if (In::step(k) >= steps) continue;
      const float* from = s_y + In::step(k) * kLanes * In::kRow + In::channel(k);
      float v = 0.0f, w = 0.0f;
#pragma unroll
      for (int l = 0; l < kLanes; ++l) {
        const float2 part = *reinterpret_cast<const float2*>(from + l * In::kRow);
        v += part.x;
        w += part.y;
      }
      put<T>(y + (t0 + In::step(k)) * s.channels, p.c0 + In::channel(k), s.channels, s.channels % 2 == 0, (v + du[k].x) * gate[k].x,
             (w + du[k].y) * gate[k].y);
    }
  }
  for (int64_t t = (p.first > p.len ? p.first : p.len) + threadIdx.x / (kWide / 2); t < p.end; t += kThreads / (kWide / 2))
    put<T>(y + t * s.channels, p.c0 + threadIdx.x % (kWide / 2) * 2, s.channels, s.channels % 2 == 0, 0.0f, 0.0f);
  // the chunk that the sequence ends in
  if (state_out != nullptr && on && (p.first < p.len || p.chunk == 0) && p.end >= p.len) {
    const float2 x = halves(h0), w = halves(h1);
    const float h[kStates] = {x.x, x.y, w.x, w.y};
#pragma unroll
    for (int j = 0; j < kStates; ++j) {
      const int n = lane * kStates + j;
      if (n < s.states) state_out[(p.b * s.channels + channel) * s.states + n] = h[j];
    }
  }
}

// A chunk by itself, from a state of zero: forward h, or backward the carry a dh that leaves its first step; and the sum of its dt.
template <class T, int kLanes, bool kReverse>
__global__ void __launch_bounds__(kThreads) selective_scan_chunk_kernel(Scan s, const T* __restrict__ dout) {
  pdl_enter();
  using In = Ahead<T, kLanes>;
  constexpr int kWide = In::kWide, kPadded = In::kPadded;
  __shared__ float4 s_bc[kTile * kLanes];                  // B, or C
  __shared__ float4 s_dt[kTile * kWide];                   // dt twice, dt * u (or dy) twice
  const Block<kWide> p(s);
  const int c = threadIdx.x / kLanes, lane = threadIdx.x % kLanes, channel = p.c0 + c;
  const bool on = channel < s.channels;
  float a[kStates], span = 0.0f;
#pragma unroll
  for (int j = 0; j < kStates; ++j) {
    const int n = lane * kStates + j;
    a[j] = on && n < s.states ? s.A[(int64_t)channel * s.states + n] * kLog2e : 0.0f;
  }
  const f2 a0 = pair(a[0], a[1]), a1 = pair(a[2], a[3]);
  f2 h0 = 0, h1 = 0;
  Two<T> x[In::kPairs], delta[In::kPairs], z[In::kPairs], bc[In::kNarrow];
  auto prefetch = [&](int64_t t0) {
#pragma unroll
    for (int k = 0; k < In::kPairs; ++k) {
      const int64_t t = t0 + In::step(k);
      const int ch = p.c0 + In::channel(k);
      if (In::step(k) < kTile && t < p.last) {
        delta[k] = fetch<T>(s.delta, p.b, t, ch, s.channels, s.even);
        if constexpr (kReverse) {
          x[k] = fetch<T>(dout + (p.b * s.length + t) * s.channels, ch, s.channels, s.channels % 2 == 0);
          if (s.z.p != nullptr) z[k] = fetch<T>(s.z, p.b, t, ch, s.channels, s.even);
        } else {
          x[k] = fetch<T>(s.u, p.b, t, ch, s.channels, s.even);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < In::kNarrow; ++k) {
      const int64_t t = t0 + In::narrow_step(k);
      if (In::narrow_step(k) < kTile && t < p.last) bc[k] = fetch<T>(kReverse ? s.C : s.B, p.b, t, In::state(k), s.states, s.even_narrow);
    }
  };
  float2 bias[In::kPairs];
#pragma unroll
  for (int k = 0; k < In::kPairs; ++k) bias[k] = two_of(s.bias, p.c0 + In::channel(k), s.channels);
  const int64_t tiles = p.first < p.last ? (p.last - p.first + kTile - 1) / kTile : 0;
  if (tiles > 0) prefetch(p.first + (kReverse ? tiles - 1 : 0) * kTile);
  for (int64_t i = 0; i < tiles; ++i) {
    const int64_t t0 = p.first + (kReverse ? tiles - 1 - i : i) * kTile;
    const int steps = (int)(p.last - t0 < kTile ? p.last - t0 : kTile);
    if (i > 0) __syncthreads();
#pragma unroll
    for (int k = 0; k < In::kPairs; ++k) {
      if (In::step(k) >= steps) continue;
      float2 v = x[k].get();
      const float2 dv = delta[k].get();
      const float e = dv.x + bias[k].x, w = dv.y + bias[k].y;
      const float te = s.softplus ? softplus(e) : e, tw = s.softplus ? softplus(w) : w;
      if constexpr (kReverse) {
        if (s.z.p != nullptr) {
          const float2 zv = z[k].get();
          v.x *= activate<kActSilu>(zv.x);
          v.y *= activate<kActSilu>(zv.y);
        }
      } else {
        v.x *= te;
        v.y *= tw;
      }
      float4* to = s_dt + In::step(k) * kWide + In::channel(k);
      to[0] = make_float4(te, te, v.x, v.x);
      to[1] = make_float4(tw, tw, v.y, v.y);
    }
#pragma unroll
    for (int k = 0; k < In::kNarrow; ++k)
      if (In::narrow_step(k) < steps)
        *reinterpret_cast<float2*>(reinterpret_cast<float*>(s_bc) + In::narrow_step(k) * kPadded + In::state(k)) = bc[k].get();
    __syncthreads();
    if (i + 1 < tiles) prefetch(kReverse ? t0 - kTile : t0 + kTile);
    const ulonglong2* bc2 = reinterpret_cast<const ulonglong2*>(s_bc) + lane;
    const ulonglong2* dt2 = reinterpret_cast<const ulonglong2*>(s_dt) + c;
#pragma unroll 4
    for (int k = 0; k < steps; ++k) {
      const int t = kReverse ? steps - 1 - k : k;
      const ulonglong2 dt = dt2[t * kWide], b2 = bc2[t * kLanes];
      const f2 e0 = exp2_2(mul2(dt.x, a0)), e1 = exp2_2(mul2(dt.x, a1));
      if constexpr (kReverse) {
        h0 = mul2(e0, fma2(dt.y, b2.x, h0));
        h1 = mul2(e1, fma2(dt.y, b2.y, h1));
      } else {
        h0 = fma2(e0, h0, mul2(dt.y, b2.x));
        h1 = fma2(e1, h1, mul2(dt.y, b2.y));
      }
      span += halves(dt.x).x;
    }
  }
  if (!on) return;
  const int64_t at = (p.chunk * s.batch + p.b) * s.channels + channel;
  const float2 v = halves(h0), w = halves(h1);
  reinterpret_cast<float4*>(s.local)[at * kLanes + lane] = make_float4(v.x, v.y, w.x, w.y);
  if (lane == 0) s.span[at] = span;
}

struct Grads {
  const void* dout;            // [batch][length][channels]
  const float* keep;
  int kept;                    // states of a channel there
  void *du, *ddelta, *dz;      // like dout; dz null without a gate
  float* narrow;               // [blocks of channels][batch][length][2][16 * kBlocks]: shares of dB, dC
  float* sums;                 // [batch][chunks][channels * states + channels + channels]: dA, dD, ddelta_bias
};

__device__ __forceinline__ uint32_t tf32(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// d += a b with eleven bits of each factor, or (fp32 gradients) with the next eleven as well.
template <bool kFine> __device__ __forceinline__ void product(float (&d)[4], const float (&a)[4], const float (&b)[2]) {
  uint32_t ah[4], bh[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) ah[i] = tf32(a[i]);
#pragma unroll
  for (int i = 0; i < 2; ++i) bh[i] = tf32(b[i]);
  mma(d, ah, bh);
  if constexpr (kFine) {
    uint32_t al[4], bl[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) al[i] = tf32(a[i] - __uint_as_float(ah[i]));
#pragma unroll
    for (int i = 0; i < 2; ++i) bl[i] = tf32(b[i] - __uint_as_float(bh[i]));
    mma(d, ah, bl);
    mma(d, al, bh);
  }
}

// A warp: eight channels and sixteen states.  Thread: channels c and c + 4 (c = lane % 4), states n and n + 8 (n = lane / 4).
// kBlocks warps side by side have the states of wider layers.
template <class T, int kBlocks>
__global__ void __launch_bounds__(kThreads, 3) selective_scan_bwd_kernel(Scan s, Grads g) {
  pdl_enter();
  constexpr int kWarps = kThreads / 32, kWide = 8 * kWarps / kBlocks, kPadded = 16 * kBlocks, kSlots = 8 * kBlocks;
  constexpr int kRow = kWide + 4;                            // a warp's eight slots of four channels fall into banks of their own
  constexpr bool kFine = sizeof(T) == 4;
  __shared__ float4 s_bc[kKeep][kSlots];                     // B of states n and n + 8, C of them
  __shared__ float4 s_dt[kKeep][kWide];                      // dt twice, dt u twice
  __shared__ __align__(16) float2 s_dy[kKeep][kWide];                      // dy twice
  __shared__ __align__(16) float s_part[3][kKeep][kSlots][kRow];           // C h, B dh, A a h[t - 1] dh of a thread's two states
  __shared__ float s_narrow[kWarps / kBlocks][2][kKeep][kPadded + 4];   // dB, dC over a warp's channels
  const Block<kWide> p(s);
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, part = warp % kBlocks, group = warp / kBlocks;
  const int slot = part * 8 + lane / 4, n0 = part * 16 + lane / 4, w0 = group * 8 + lane % 4;     // state, channel in the block
  const int ch[2] = {p.c0 + w0, p.c0 + w0 + 4};
  f2 A[2], A2[2], carry[2], dA[2];                           // of a channel: its two states
  float dA_sum[2][2], dA_low[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float v[2], c[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = n0 + 8 * j;
      const bool is = ch[i] < s.channels && n < s.states;
      v[j] = is ? s.A[(int64_t)ch[i] * s.states + n] : 0.0f;
      dA_sum[i][j] = dA_low[i][j] = 0.0f;
      if (is && s.chunks > 1)
        for (int q = s.chunks - 1; q > p.chunk; --q) {
          const int64_t at = (q * s.batch + p.b) * s.channels + ch[i];
          c[j] = fmaf(exp2_approx(s.span[at] * (v[j] * kLog2e)), c[j], s.local[at * g.kept + n]);
        }
    }
    A[i] = pair(v[0], v[1]);
    A2[i] = pair(v[0] * kLog2e, v[1] * kLog2e);
    carry[i] = pair(c[0], c[1]);
  }
  // what a thread prepares and finishes: two channels of a step
  constexpr int kPairs = kWide / 2;
  const int pt = threadIdx.x / kPairs, pc = threadIdx.x % kPairs * 2, channel = p.c0 + pc;
  const bool mine = pt < kKeep;
  // ... and what it prepares of B (the first half of the threads' turns) and C
  constexpr int kNarrow = kKeep * kPadded / 2 <= kThreads ? 1 : kKeep * kPadded / 2 / kThreads;
  const float2 skip = two_of(s.D, channel, s.channels), bias = two_of(s.bias, channel, s.channels);
  float2 dD = make_float2(0.0f, 0.0f), dbias = dD;
  const int even = s.channels % 2 == 0;
  const int64_t base = p.b * s.length;
  Two<T> u, delta, z, up, bb[kNarrow], cc[kNarrow];
  float kept[2][2];
  auto prefetch = [&](int64_t t0) {
    if (mine && t0 + pt < p.last) {
      u = fetch<T>(s.u, p.b, t0 + pt, channel, s.channels, s.even);
      delta = fetch<T>(s.delta, p.b, t0 + pt, channel, s.channels, s.even);
      if (s.z.p != nullptr) z = fetch<T>(s.z, p.b, t0 + pt, channel, s.channels, s.even);
      up = fetch<T>(reinterpret_cast<const T*>(g.dout) + (base + t0 + pt) * s.channels, channel, s.channels, even);
    }
#pragma unroll
    for (int k = 0; k < kNarrow; ++k) {
      const int i = threadIdx.x + k * kThreads, t = i / (kPadded / 2), n = i % (kPadded / 2) * 2;
      if (t < kKeep && t0 + t < p.last) {
        bb[k] = fetch<T>(s.B, p.b, t0 + t, n, s.states, s.even_narrow);
        cc[k] = fetch<T>(s.C, p.b, t0 + t, n, s.states, s.even_narrow);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int n = n0 + 8 * j;
        kept[i][j] = ch[i] < s.channels && n < s.states ? g.keep[((t0 / kKeep * s.batch + p.b) * s.channels + ch[i]) * g.kept + n] : 0.0f;
      }
  };
  const int64_t tiles = p.first < p.last ? (p.last - p.first + kKeep - 1) / kKeep : 0;
  if (tiles > 0) prefetch(p.first + (tiles - 1) * kKeep);
  for (int64_t tile = tiles - 1; tile >= 0; --tile) {
    const int64_t t0 = p.first + tile * kKeep;
    const int steps = (int)(p.last - t0 < kKeep ? p.last - t0 : kKeep);
    // prepare; steps behind the end do nothing: dt = 0 and dy = 0
    float2 uv = make_float2(0.0f, 0.0f), dt = uv, slope_dt = uv, dz = uv, dy = uv;
    if (mine) {
      if (pt < steps) {
        const float2 dv = delta.get(), ov = up.get();
        uv = u.get();
        const float x = dv.x + bias.x, w = dv.y + bias.y;
        dt = make_float2(x, w);
        slope_dt = make_float2(1.0f, 1.0f);
        if (s.softplus) dt = make_float2(softplus(x, &slope_dt.x), softplus(w, &slope_dt.y));
        dy = ov;
        if (s.z.p != nullptr) {
          const float2 zv = z.get();
          const float gx = sigmoid(zv.x), gw = sigmoid(zv.y);
          dy = make_float2(ov.x * zv.x * gx, ov.y * zv.y * gw);
          dz = make_float2(ov.x * gx * (1.0f + zv.x * (1.0f - gx)), ov.y * gw * (1.0f + zv.y * (1.0f - gw)));
        }
      }
      s_dt[pt][pc] = make_float4(dt.x, dt.x, dt.x * uv.x, dt.x * uv.x);
      s_dt[pt][pc + 1] = make_float4(dt.y, dt.y, dt.y * uv.y, dt.y * uv.y);
      *reinterpret_cast<float4*>(&s_dy[pt][pc]) = make_float4(dy.x, dy.x, dy.y, dy.y);
    }
#pragma unroll
    for (int k = 0; k < kNarrow; ++k) {
      const int i = threadIdx.x + k * kThreads, t = i / (kPadded / 2), n = i % (kPadded / 2) * 2;
      if (t >= kKeep) continue;
      const float2 zero = make_float2(0.0f, 0.0f), bv = t < steps ? bb[k].get() : zero, cv = t < steps ? cc[k].get() : zero;
      // states n, n + 1 of sixteen: slots n % 8 and the next, the first or second of each
      float* to = reinterpret_cast<float*>(&s_bc[t][n / 16 * 8 + n % 8]) + n % 16 / 8;
      to[0] = bv.x;
      to[2] = cv.x;
      to[4] = bv.y;
      to[6] = cv.y;
    }
    f2 h[kKeep + 1][2], a[kKeep][2];
    h[0][0] = pair(kept[0][0], kept[0][1]);
    h[0][1] = pair(kept[1][0], kept[1][1]);
    __syncthreads();
    if (tile > 0) prefetch(t0 - kKeep);
#pragma unroll
    for (int t = 0; t < kKeep; ++t) {
      const f2 b = *reinterpret_cast<const f2*>(&s_bc[t][slot]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const ulonglong2 d = *reinterpret_cast<const ulonglong2*>(&s_dt[t][w0 + 4 * i]);
        a[t][i] = exp2_2(mul2(d.x, A2[i]));
        h[t + 1][i] = fma2(a[t][i], h[t][i], mul2(d.y, b));
      }
    }
    float dB[4] = {0, 0, 0, 0}, dC[4] = {0, 0, 0, 0};        // state n (n + 8), steps 2 (lane % 4) and the next
    dA[0] = dA[1] = 0;
#pragma unroll
    for (int t = kKeep - 1; t >= 0; --t) {
      const ulonglong2 bc = *reinterpret_cast<const ulonglong2*>(&s_bc[t][slot]);
      f2 dh[2];
      float by[2], bu[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const ulonglong2 d = *reinterpret_cast<const ulonglong2*>(&s_dt[t][w0 + 4 * i]);
        const f2 y2 = *reinterpret_cast<const f2*>(&s_dy[t][w0 + 4 * i]);
        dh[i] = fma2(bc.y, y2, carry[i]);
        carry[i] = mul2(a[t][i], dh[i]);
        const f2 da = mul2(carry[i], h[t][i]);
        dA[i] = fma2(da, d.x, dA[i]);
        s_part[0][t][slot][w0 + 4 * i] = sum_of(mul2(bc.y, h[t + 1][i]));
        s_part[1][t][slot][w0 + 4 * i] = sum_of(mul2(bc.x, dh[i]));
        s_part[2][t][slot][w0 + 4 * i] = sum_of(mul2(da, A[i]));
        const bool column = lane / 4 == t;
        by[i] = column ? halves(y2).x : 0.0f;
        bu[i] = column ? halves(d.y).x : 0.0f;
      }
      const float2 h0 = halves(h[t + 1][0]), h1 = halves(h[t + 1][1]), d0 = halves(dh[0]), d1 = halves(dh[1]);
      const float ha[4] = {h0.x, h0.y, h1.x, h1.y}, da4[4] = {d0.x, d0.y, d1.x, d1.y};
      product<kFine>(dC, ha, by);
      product<kFine>(dB, da4, bu);
    }
    // into the running sum with its rounding errors beside it: a sequence has thousands of terms
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 v = halves(dA[i]);
      const float add[2] = {v.x, v.y};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float y = add[j] - dA_low[i][j], t = dA_sum[i][j] + y;
        dA_low[i][j] = (t - dA_sum[i][j]) - y;
        dA_sum[i][j] = t;
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      s_narrow[group][0][2 * (lane % 4) + q % 2][n0 + q / 2 * 8] = dB[q];
      s_narrow[group][1][2 * (lane % 4) + q % 2][n0 + q / 2 * 8] = dC[q];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < steps * 2 * kPadded; i += kThreads) {
      const int t = i / (2 * kPadded), k = i / kPadded % 2, n = i % kPadded;
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps / kBlocks; ++w) v += s_narrow[w][k][t][n];
      g.narrow[((p.block * s.batch + p.b) * s.length + t0) * 2 * kPadded + i] = v;
    }
    if (mine && pt < steps) {
      float2 v[3];
#pragma unroll
      for (int q = 0; q < 3; ++q) {
        float x = 0.0f, w = 0.0f;
#pragma unroll
        for (int l = 0; l < kSlots; ++l) {
          const float2 o = *reinterpret_cast<const float2*>(&s_part[q][pt][l][pc]);
          x += o.x;
          w += o.y;
        }
        v[q] = make_float2(x, w);
      }
      const int64_t row = (base + t0 + pt) * s.channels;
      if (g.dz != nullptr)
        put<T>(reinterpret_cast<T*>(g.dz) + row, channel, s.channels, even, dz.x * fmaf(skip.x, uv.x, v[0].x), dz.y * fmaf(skip.y, uv.y, v[0].y));
      put<T>(reinterpret_cast<T*>(g.du) + row, channel, s.channels, even, fmaf(v[1].x, dt.x, skip.x * dy.x), fmaf(v[1].y, dt.y, skip.y * dy.y));
      const float ex = fmaf(v[1].x, uv.x, v[2].x) * slope_dt.x, ew = fmaf(v[1].y, uv.y, v[2].y) * slope_dt.y;
      put<T>(reinterpret_cast<T*>(g.ddelta) + row, channel, s.channels, even, ex, ew);
      dD.x = fmaf(dy.x, uv.x, dD.x);
      dD.y = fmaf(dy.y, uv.y, dD.y);
      dbias.x += ex;
      dbias.y += ew;
    }
  }
  for (int64_t t = (p.first > p.len ? p.first : p.len) + pt; t < p.end; t += kThreads / kPairs) {
    const int64_t row = (base + t) * s.channels;
    put<T>(reinterpret_cast<T*>(g.du) + row, channel, s.channels, even, 0.0f, 0.0f);
    put<T>(reinterpret_cast<T*>(g.ddelta) + row, channel, s.channels, even, 0.0f, 0.0f);
    if (g.dz != nullptr) put<T>(reinterpret_cast<T*>(g.dz) + row, channel, s.channels, even, 0.0f, 0.0f);
  }
  float* sums = g.sums + (p.b * s.chunks + p.chunk) * (int64_t)s.channels * (s.states + 2);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (ch[i] < s.channels && n0 + 8 * j < s.states) sums[(int64_t)ch[i] * s.states + n0 + 8 * j] = dA_sum[i][j];
  __syncthreads();
  float4* stage = reinterpret_cast<float4*>(&s_part[0][0][0][0]);      // room for one of each thread
  stage[threadIdx.x] = make_float4(dD.x, dD.y, dbias.x, dbias.y);
  __syncthreads();
  if (threadIdx.x < kPairs) {
    float4 v = stage[threadIdx.x];
    for (int k = threadIdx.x + kPairs; k < kThreads; k += kPairs) {
      const float4 w = stage[k];
      v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
    }
    float* to = sums + (int64_t)s.channels * s.states;
    put<float>(to, channel, s.channels, 0, v.x, v.y);
    put<float>(to + s.channels, channel, s.channels, 0, v.z, v.w);
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
#pragma unroll 8
    for (int q = 0; q < blocks; ++q) v += narrow[q * n + i];
  (k == 0 ? dB : dC)[row * s.states + j] = as_type<T>(v);
}

template <class T> __device__ __forceinline__ float at(const Seq& q, int64_t b, int c) {
  return as_float(reinterpret_cast<const T*>(q.p)[b * q.b + c]);
}

// One step of every sequence: the state moves on; state_out may be s.state.
template <class T, int kLanes>
__global__ void __launch_bounds__(kThreads) selective_scan_step_kernel(Scan s, float* state_out, T* __restrict__ out) {
  pdl_enter();
  constexpr int kWide = kThreads / kLanes;
  const int blocks = (s.channels + kWide - 1) / kWide;
  const int64_t b = blockIdx.x / blocks;
  const int c = (int)(blockIdx.x - b * blocks) * kWide + threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  const bool on = c < s.channels;
  float part = 0.0f, u = 0.0f;
  if (on) {
    u = at<T>(s.u, b, c);
    const float raw = at<T>(s.delta, b, c) + (s.bias != nullptr ? s.bias[c] : 0.0f);
    const float dt = s.softplus ? softplus(raw) : raw;
#pragma unroll
    for (int j = 0; j < kStates; ++j) {
      const int n = lane * kStates + j;
      if (n >= s.states) break;
      const int64_t i = (b * s.channels + c) * s.states + n;
      const float h = fmaf(exp2_approx(dt * (s.A[(int64_t)c * s.states + n] * kLog2e)), s.state[i], dt * u * at<T>(s.B, b, n));
      state_out[i] = h;
      part = fmaf(at<T>(s.C, b, n), h, part);
    }
  }
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
  if (on && lane == 0) {
    if (s.D != nullptr) part = fmaf(s.D[c], u, part);
    if (s.z.p != nullptr) part *= activate<kActSilu>(at<T>(s.z, b, c));
    out[b * s.channels + c] = as_type<T>(part);
  }
}

int lanes_of(int states) {
  int l = 1;
  while (l * kStates < states) l *= 2;
  return l;
}
int state_blocks(int states) { return states <= 16 ? 1 : states <= 32 ? 2 : 4; }
int blocks_of(int channels, int wide) { return (channels + wide - 1) / wide; }

// Chunks of a pass over `blocks` blocks.  CHUNK_RULE
void split(Scan* s, int64_t blocks, int64_t shortest) {
  int64_t n = 1;
  while (n < kMaxChunks && blocks * n < 2 * sm_count() && s->length / (2 * n) >= shortest) n *= 2;
  s->chunk = ((s->length + n - 1) / n + kTile - 1) / kTile * kTile;
  s->chunks = s->chunk > 0 ? (int)((s->length + s->chunk - 1) / s->chunk) : 1;
}
constexpr int64_t kShortest = 128;

template <class T, int kLanes> int forward(const Scan& s, void* out, float* state_out, float* keep, void* stream) {
  static SmemAllowed allowed{0};
  constexpr int kWide = kThreads / kLanes;
  constexpr size_t kSmem = kTile * (2 * kLanes * 16 + kWide * 16 + kLanes * Ahead<T, kLanes>::kRow * 4);
  if (kSmem > 48 * 1024) {
    const int rc = allow_smem(selective_scan_fwd_kernel<T, kLanes>, kSmem, allowed);
    if (rc != 0) return rc;
  }
  const dim3 grid((unsigned)(s.batch * s.chunks * blocks_of(s.channels, kWide)));
  if (s.chunks > 1) {
    const int rc = launch(selective_scan_chunk_kernel<T, kLanes, false>, grid, kThreads, 0, stream, s, (const T*)nullptr);
    if (rc != 0) return rc;
  }
  return launch(selective_scan_fwd_kernel<T, kLanes>, grid, kThreads, kSmem, stream, s, (T*)out, state_out, keep);
}
template <class T, int kLanes> int carries(const Scan& s, const void* dout, void* stream) {
  const dim3 grid((unsigned)(s.batch * s.chunks * blocks_of(s.channels, kThreads / kLanes)));
  return launch(selective_scan_chunk_kernel<T, kLanes, true>, grid, kThreads, 0, stream, s, (const T*)dout);
}
template <class T, int kBlocks> int backward_blocks(const Scan& s, const Grads& g, void* dB, void* dC, void* stream) {
  const int blocks = blocks_of(s.channels, 32 / kBlocks), padded = 16 * kBlocks;
  const int rc = launch(selective_scan_bwd_kernel<T, kBlocks>, dim3((unsigned)(s.batch * s.chunks * blocks)), kThreads, 0, stream, s, g);
  if (rc != 0) return rc;
  const int64_t n = s.batch * s.length * 2 * padded;
  return launch(selective_scan_narrow_kernel<T>, dim3((unsigned)((n + 255) / 256)), 256, 0, stream, g.narrow, blocks, s, padded, (T*)dB, (T*)dC);
}
template <class T> int backward(const Scan& s, const Grads& g, void* dB, void* dC, void* stream) {
  switch (state_blocks(s.states)) {
    case 1: return backward_blocks<T, 1>(s, g, dB, dC, stream);
    case 2: return backward_blocks<T, 2>(s, g, dB, dC, stream);
    default: return backward_blocks<T, 4>(s, g, dB, dC, stream);
  }
}
template <class T, int kLanes> int step(const Scan& s, float* state_out, void* out, void* stream) {
  return launch(selective_scan_step_kernel<T, kLanes>, dim3((unsigned)(s.batch * blocks_of(s.channels, kThreads / kLanes))), kThreads, 0, stream, s,
                state_out, (T*)out);
}

// F<T, kLanes>(...)
#define ESGD_LANES(T, F, ...)                                                                                   \
  (lanes == 1 ? F<T, 1>(__VA_ARGS__) : lanes == 2 ? F<T, 2>(__VA_ARGS__) : lanes == 4 ? F<T, 4>(__VA_ARGS__)    \
   : lanes == 8 ? F<T, 8>(__VA_ARGS__) : F<T, 16>(__VA_ARGS__))
#define ESGD_TYPE(F, ...) (is_bf16 ? ESGD_LANES(__nv_bfloat16, F, __VA_ARGS__) : ESGD_LANES(float, F, __VA_ARGS__))

bool taken(const Scan& s) { return s.states >= 1 && s.states <= 64 && s.channels >= 1 && s.batch >= 0 && s.length >= 0; }

Scan scan_of(const esgd_scan* e) {
  Scan s = {};
  Seq* q[5] = {&s.u, &s.delta, &s.z, &s.B, &s.C};
  const uintptr_t size = e->is_bf16 ? 2 : 4;
  s.even = e->channels % 2 == 0;
  s.even_narrow = e->states % 2 == 0;
  for (int i = 0; i < 5; ++i) {
    *q[i] = {e->p[i], e->b[i], e->t[i]};
    if (e->p[i] != nullptr && ((uintptr_t)e->p[i] % (2 * size) || e->b[i] % 2 || e->t[i] % 2)) (i < 3 ? s.even : s.even_narrow) = 0;
  }
  s.A = e->A; s.D = e->D; s.bias = e->bias;
  s.lengths = e->lengths;
  s.state = e->state;
  s.batch = e->batch; s.length = e->length;
  s.channels = e->channels; s.states = e->states; s.softplus = e->softplus;
  split(&s, s.batch * blocks_of(s.channels, kThreads / lanes_of(s.states)), kShortest);
  return s;
}
int64_t local_floats(const Scan& s) { return s.chunks <= 1 ? 0 : s.chunks * s.batch * s.channels * (lanes_of(s.states) * kStates + 1); }
// The chunks' room: their states, and behind these the sums of their time steps.
void place(Scan* s, float* local) {
  s->local = local;
  s->span = local + s->chunks * s->batch * s->channels * lanes_of(s->states) * kStates;
}

}  // namespace

extern "C" {

// Floats of room for a pass in either direction (the chunks'; none for many sequences or short ones), for what the forward pass
// keeps for the backward pass, and for the shares of dB, dC and of the parameters' gradients.
int64_t esgd_selective_scan_local(const esgd_scan* e) { return local_floats(scan_of(e)); }
int64_t esgd_selective_scan_keep(const esgd_scan* e) {
  return (e->length + kKeep - 1) / kKeep * e->batch * e->channels * lanes_of(e->states) * kStates;
}
int64_t esgd_selective_scan_narrow(const esgd_scan* e) {
  const int side = state_blocks(e->states);
  return blocks_of(e->channels, 32 / side) * e->batch * e->length * 2 * 16 * side;
}
int64_t esgd_selective_scan_parts(const esgd_scan* e) { return e->length > 0 ? e->batch * scan_of(e).chunks : 0; }

int esgd_selective_scan_fwd(const esgd_scan* e, void* out, float* state_out, float* keep, float* local, void* stream) {
  Scan s = scan_of(e);
  if (!taken(s)) return (int)cudaErrorInvalidValue;
  if (s.batch == 0) return 0;
  place(&s, local);
  const int is_bf16 = e->is_bf16, lanes = lanes_of(s.states);
  return ESGD_TYPE(forward, s, out, state_out, keep, stream);
}

// sums [parts][channels * states + 2 * channels].
int esgd_selective_scan_bwd(const esgd_scan* e, const void* dout, const float* keep, void* du, void* ddelta, void* dz, void* dB, void* dC,
                            float* narrow, float* sums, float* local, void* stream) {
  Scan s = scan_of(e);
  if (!taken(s)) return (int)cudaErrorInvalidValue;
  if (s.batch == 0 || s.length == 0) return 0;
  place(&s, local);
  const int is_bf16 = e->is_bf16, lanes = lanes_of(s.states);
  if (s.chunks > 1) {
    const int rc = ESGD_TYPE(carries, s, dout, stream);
    if (rc != 0) return rc;
  }
  const Grads g = {dout, keep, lanes * kStates, du, ddelta, dz, narrow, sums};
  return is_bf16 ? backward<__nv_bfloat16>(s, g, dB, dC, stream) : backward<float>(s, g, dB, dC, stream);
}

int esgd_selective_scan_step(const esgd_scan* e, float* state_out, void* out, void* stream) {
  const Scan s = scan_of(e);
  if (!taken(s) || s.state == nullptr) return (int)cudaErrorInvalidValue;
  if (s.batch == 0) return 0;
  const int is_bf16 = e->is_bf16, lanes = lanes_of(s.states);
  return ESGD_TYPE(step, s, state_out, out, stream);
}

}  // extern "C"
