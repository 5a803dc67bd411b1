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
// instructions, not by memory.  States stay in registers over the whole sequence, those of two neighbouring channels in a 64-bit
// register for the paired fp32 instructions.  A tile of steps is prepared elementwise (a thread: two neighbouring channels of a
// step; their operands are fetched a tile ahead), goes through shared memory to the threads that have the states, and comes back
// for the sums over the states and the gates.
//
// Forward: two channels' states lie in kLanes threads, two by four in each: with one channel to a thread the reads of B and C out
// of shared memory (32 bytes a thread and step) took longer than the exponentials.  Backward: a warp has eight channels and sixteen
// states, a thread two by two of them as the tensor cores' m16n8k8 fragments want them: the sums over the channels that dB and dC
// are, eight values a thread and step, are four matrix instructions instead of some forty shuffles and additions.  The states ahead
// of every eighth step are kept by the forward pass, so that the backward pass needs one exponential a state and step as well.
//
// 64 x 331 steps of 2048 channels, 16 states, bf16: forward 279 us (694 M exponentials, 154 us at 16 a clock and SM), backward 1230 us:
// the partial sums' way through shared memory takes half of its time there.  (The exponentials made again, instead of kept in
// registers from the first half of a tile to the second, and four blocks an SM: 1061 us for 1035; arithmetic without pairs: 1125 for
// 1072.)
//
// The exponentials are those of the special function units, of dt A log2 e as fp32 rounds it, some 2e-7 off.  dA of fp32 sequences is 4.6e-7
// off in all (3 x 77 steps of 500 channels; the plain formula in fp32: 2.4e-7).  Putting the argument's rounding right left that as it was
// and took 143 us for 90 forward (16 x 331 x 2048).
//
// Kept for the backward pass are 4 bytes a state, every eighth step: 8 bytes a step and channel with 16 states (16 with 17 to 32, and so on by
// powers of two), four times a bf16 u.  That pass has shares of dB and dC, 128 bytes a step and 32 channels of up to 16 states.
//
// Few sequences of few channels: the steps are split into chunks that run at the same time.  A first pass scans every chunk from a
// state of zero; what a chunk begins with is then the chunks ahead of it joined, h = exp(A sum dt) h + (its own scan).
#include "selective_scan.h"
#include "launch.cuh"
#include "rows.cuh"

namespace {

using namespace esgd;

constexpr int kThreads = 128;
constexpr int kStates = 4;           // of a thread and channel, forward
constexpr int kTile = 16;            // steps of a tile, forward
constexpr int kKeep = 8;             // steps between kept states, and of a tile of the backward pass
constexpr int kHalf = kKeep / 2;     // steps that a matrix product's columns hold
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
  int even;                          // neighbouring channels and states are one load: even counts, strides and beginnings
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
// is at most 1/3, so five terms, fitted to the relative error, are right to 8e-9.  slope: 1 / (1 + e^-x).
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
// Two neighbouring values of a row, or as many as there are.
template <class T, bool kEven> __device__ __forceinline__ void put(T* to, int in, float x, float y) {
  if constexpr (!kEven) {
    if (in > 0) to[0] = as_type<T>(x);
    if (in > 1) to[1] = as_type<T>(y);
  } else if (in > 0) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(to) = make_float2(x, y);
    else *reinterpret_cast<__nv_bfloat162*>(to) = __floats2bfloat162_rn(x, y);
  }
}
__device__ __forceinline__ float2 two_of(const float* p, int c, int width) {
  return make_float2(p != nullptr && c < width ? p[c] : 0.0f, p != nullptr && c + 1 < width ? p[c + 1] : 0.0f);
}

// The i-th longest sequence: the blocks of long ones begin first, so that none of them is left for the end (16 of 110 to 331 steps,
// backward: 245 -> 223 us).
__device__ __forceinline__ int64_t by_length(const Scan& s, int64_t i) {
  if (s.lengths == nullptr || s.batch > kThreads) return i;
  __shared__ int64_t length[kThreads];
  __shared__ int found;
  const int t = threadIdx.x;
  const int64_t own = t < s.batch ? length_of(s, t) : -1;
  length[t] = own;
  __syncthreads();
  int longer = 0;
  for (int j = 0; j < (int)s.batch; ++j) longer += length[j] > own || (length[j] == own && j < t);
  if (t < s.batch && longer == (int)i) found = t;
  __syncthreads();
  return found;
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
    const int64_t i = rest / s.chunks;
    chunk = (int)(rest - i * s.chunks);
    b = by_length(s, i);
    c0 = block * kWide;
    len = length_of(s, b);
    first = chunk * s.chunk;
    end = chunk + 1 < s.chunks ? first + s.chunk : s.length;
    last = end < len ? end : len;
  }
};

// What a thread fetches of a tile of kSteps steps: kPairs pairs of channels, always the same two and kPitch steps apart, and kNarrow
// pairs of states.
template <int kSteps, int kWide_, int kPadded_> struct Share {
  static constexpr int kWide = kWide_, kPadded = kPadded_;
  static constexpr int kPitch = kThreads / (kWide / 2), kPairs = kSteps <= kPitch ? 1 : kSteps / kPitch;
  static constexpr int kNarrowPitch = kThreads / (kPadded / 2), kNarrow = kSteps <= kNarrowPitch ? 1 : kSteps / kNarrowPitch;
  int channel, step, state, narrow_step;
  __device__ Share() {
    channel = threadIdx.x % (kWide / 2) * 2;
    step = threadIdx.x / (kWide / 2);
    state = threadIdx.x % (kPadded / 2) * 2;
    narrow_step = threadIdx.x / (kPadded / 2);
  }
};

// A thread's pairs of one operand: where the next tile's are.
template <class T> struct Cursor {
  const T* p;
  int64_t pitch, tile;       // elements between a thread's pairs, and to the next tile
  __device__ __forceinline__ void set(const Seq& q, int64_t b, int64_t t, int c, int pitch_, int tile_) {
    p = reinterpret_cast<const T*>(q.p) + (b * q.b + t * q.t + c);
    pitch = pitch_ * q.t;
    tile = tile_ * q.t;
  }
  // `n` steps are left from the thread's first on; `in`: how many of the two values there are.
  template <bool kEven, int kPairs> __device__ __forceinline__ void fetch(Two<T> (&to)[kPairs], int n, int between, int in) {
    if constexpr (kEven) {
#pragma unroll
      for (int k = 0; k < kPairs; ++k)
        if (k * between < n && in > 0) to[k].load(p + k * pitch);
    } else {
#pragma unroll
      for (int k = 0; k < kPairs; ++k)
        if (k * between < n) to[k].set(in > 0 ? p[k * pitch] : as_type<T>(0.0f), in > 1 ? p[k * pitch + 1] : as_type<T>(0.0f));
    }
    p += tile;
  }
};
__device__ __forceinline__ int left_of(int width, int c) { return width - c < 0 ? 0 : width - c > 2 ? 2 : width - c; }

// Forward passes.  A row of partial sums: a warp's channels of every lane fall into banks of their own.
template <int kLanes> struct Lanes : Share<kTile, 2 * kThreads / kLanes, kLanes * kStates> {
  static_assert(kLanes <= kTile, "every thread's pairs are steps of the tile");
  static constexpr int kRow = 2 * kThreads / kLanes + (32 / kLanes - 2 * kThreads / kLanes % 32 + 32) % 32;
};

// h e^(x ln 2), by way of a chunk.  In two halves, of which neither is infinite before the result is, nor zero; and a state of zero stays
// zero, whatever the chunk would have made of another.
__device__ __forceinline__ float across(float h, float x) {
  const float half = exp2_approx(0.5f * x);
  return h == 0.0f ? 0.0f : h * half * half;
}
__device__ __forceinline__ f2 across(f2 h, f2 x) {
  const float2 v = halves(h), w = halves(x);
  return pair(across(v.x, w.x), across(v.y, w.y));
}

// The states that a thread begins with: those given, and the other chunks' joined to them; of two channels, four states each.
template <int kLanes, bool kReverse>
__device__ __forceinline__ void joined(const Scan& s, int64_t b, int chunk, int channel, int two, int lane, const f2 (&a)[kStates], f2 (&h)[kStates]) {
  for (int i = kReverse ? s.chunks - 1 : 0; i != chunk; kReverse ? --i : ++i) {
    const int64_t at = (i * s.batch + b) * s.channels + channel;
    const f2 span = pair(s.span[at], two > 1 ? s.span[at + 1] : 0.0f);
    const float4* local = reinterpret_cast<const float4*>(s.local) + at * kLanes + lane;
    const float4 l = local[0], r = two > 1 ? local[kLanes] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const float own[2][4] = {{l.x, l.y, l.z, l.w}, {r.x, r.y, r.z, r.w}};
#pragma unroll
    for (int j = 0; j < kStates; ++j) h[j] = add2(across(h[j], mul2(span, a[j])), pair(own[0][j], own[1][j]));
  }
}
// A value of two channels' four states each, zero where there is none.
template <int kLanes> __device__ __forceinline__ void states_of(const float* p, int64_t row, int states, int two, int lane, float factor, f2 (&to)[kStates]) {
#pragma unroll
  for (int j = 0; j < kStates; ++j) {
    const int n = lane * kStates + j;
    const bool is = p != nullptr && n < states;
    to[j] = pair(is && two > 0 ? p[row * states + n] * factor : 0.0f, is && two > 1 ? p[(row + 1) * states + n] * factor : 0.0f);
  }
}

// keep: [tiles of kKeep steps][batch][channels][kLanes * 4], the state ahead of every eighth step; or null.
template <class T, int kLanes, bool kEven>
__global__ void __launch_bounds__(kThreads) selective_scan_fwd_kernel(Scan s, T* __restrict__ out, float* __restrict__ state_out,
                                                                      float* __restrict__ keep) {
  pdl_enter();
  using In = Lanes<kLanes>;
  constexpr int kWide = In::kWide, kPadded = In::kPadded;
  extern __shared__ float4 smem4[];
  float4* s_bc = smem4;                                                   // [kTile][kLanes][2]: four of B, four of C
  float4* s_dt = s_bc + kTile * 2 * kLanes;                               // [kTile][kWide / 2]: dt of two channels, dt * u of them
  float* s_y = reinterpret_cast<float*>(s_dt + kTile * kWide / 2);        // [kTile][kLanes][In::kRow]
  const Block<kWide> p(s);
  const In in;
  const int c = threadIdx.x / kLanes * 2, lane = threadIdx.x % kLanes, channel = p.c0 + c, on = left_of(s.channels, channel);
  const int two = left_of(s.channels, p.c0 + in.channel), narrow_two = left_of(s.states, in.state);
  Cursor<T> at_u, at_delta, at_z, at_b, at_c;
  Two<T> u[In::kPairs], delta[In::kPairs], z[In::kPairs], bb[In::kNarrow], cc[In::kNarrow];
  at_u.set(s.u, p.b, p.first + in.step, p.c0 + in.channel, In::kPitch, kTile);
  at_delta.set(s.delta, p.b, p.first + in.step, p.c0 + in.channel, In::kPitch, kTile);
  at_z.set(s.z, p.b, p.first + in.step, p.c0 + in.channel, In::kPitch, kTile);
  at_b.set(s.B, p.b, p.first + in.narrow_step, in.state, In::kNarrowPitch, kTile);
  at_c.set(s.C, p.b, p.first + in.narrow_step, in.state, In::kNarrowPitch, kTile);
  const bool gated = s.z.p != nullptr;
  auto prefetch = [&](int steps) {
    const int n = steps - in.step, m = steps - in.narrow_step;
    at_u.template fetch<kEven, In::kPairs>(u, n, In::kPitch, two);
    at_delta.template fetch<kEven, In::kPairs>(delta, n, In::kPitch, two);
    if (gated) at_z.template fetch<kEven, In::kPairs>(z, n, In::kPitch, two);
    at_b.template fetch<kEven, In::kNarrow>(bb, m, In::kNarrowPitch, narrow_two);
    at_c.template fetch<kEven, In::kNarrow>(cc, m, In::kNarrowPitch, narrow_two);
  };
#pragma unroll
  for (int k = 0; k < In::kPairs; ++k) u[k] = delta[k] = z[k] = Two<T>{};
#pragma unroll
  for (int k = 0; k < In::kNarrow; ++k) bb[k] = cc[k] = Two<T>{};
  int steps = (int)(p.last - p.first < kTile ? p.last - p.first : kTile);
  prefetch(steps);
  f2 a[kStates], h[kStates];
  states_of<kLanes>(s.A, channel, s.states, on, lane, kLog2e, a);
  states_of<kLanes>(s.state, p.b * s.channels + channel, s.states, on, lane, 1.0f, h);
  if (s.chunks > 1 && on) joined<kLanes, false>(s, p.b, p.chunk, channel, on, lane, a, h);
  T* y = out + (p.b * s.length + p.first + in.step) * s.channels + p.c0 + in.channel;
  const int64_t y_pitch = (int64_t)In::kPitch * s.channels, kept_tile = s.batch * s.channels * kLanes;
  float4* kept = keep != nullptr && on > 0
      ? reinterpret_cast<float4*>(keep) + ((p.first / kKeep * s.batch + p.b) * s.channels + channel) * kLanes + lane : nullptr;
  const float2 skip = two_of(s.D, p.c0 + in.channel, s.channels), bias = two_of(s.bias, p.c0 + in.channel, s.channels);
  float4* put_dt = s_dt + (in.step * kWide + in.channel) / 2;
  float* put_bc = reinterpret_cast<float*>(s_bc) + in.narrow_step * 2 * kPadded + in.state / kStates * 2 * kStates + in.state % kStates;
  const float* from_y = s_y + in.step * kLanes * In::kRow + in.channel;
  const float4* bc = s_bc + lane * 2;
  const ulonglong2* dt2 = reinterpret_cast<const ulonglong2*>(s_dt) + c / 2;
  float* put_y = s_y + lane * In::kRow + c;
  for (int64_t t0 = p.first; t0 < p.last; t0 += kTile) {
    // Steps behind the end are prepared as well, out of whatever is there, and not used: without branches the pairs' chains overlap.
    float2 du[In::kPairs], gate[In::kPairs];             // D u and silu(z) of the tile, for its end
#pragma unroll
    for (int k = 0; k < In::kPairs; ++k) {
      const float2 uv = u[k].get(), dv = delta[k].get();
      const float x = dv.x + bias.x, w = dv.y + bias.y;
      const float px = softplus(x), pw = softplus(w), tx = s.softplus ? px : x, tw = s.softplus ? pw : w;
      put_dt[k * In::kPitch * kWide / 2] = make_float4(tx, tw, tx * uv.x, tw * uv.y);
      du[k] = make_float2(skip.x * uv.x, skip.y * uv.y);
      const float2 zv = z[k].get(), silu = make_float2(activate<kActSilu>(zv.x), activate<kActSilu>(zv.y));
      gate[k] = make_float2(gated ? silu.x : 1.0f, gated ? silu.y : 1.0f);
    }
#pragma unroll
    for (int k = 0; k < In::kNarrow; ++k) {
      if (In::kNarrowPitch > kTile && in.narrow_step >= kTile) continue;
      *reinterpret_cast<float2*>(put_bc + k * In::kNarrowPitch * 2 * kPadded) = bb[k].get();
      *reinterpret_cast<float2*>(put_bc + k * In::kNarrowPitch * 2 * kPadded + kStates) = cc[k].get();
    }
    __syncthreads();
    const int now = steps;
    steps = (int)(p.last - t0 - kTile < kTile ? p.last - t0 - kTile : kTile);
    if (steps > 0) prefetch(steps);
    auto step = [&](int t) {
      if (t % kKeep == 0 && kept != nullptr) {
        float2 v[kStates];
#pragma unroll
        for (int j = 0; j < kStates; ++j) v[j] = halves(h[j]);
        kept[0] = make_float4(v[0].x, v[1].x, v[2].x, v[3].x);
        if (on > 1) kept[kLanes] = make_float4(v[0].y, v[1].y, v[2].y, v[3].y);
        kept += kept_tile;
      }
      const ulonglong2 dt = dt2[t * kWide / 2];
      const float4 b4 = bc[t * 2 * kLanes], c4 = bc[t * 2 * kLanes + 1];
      const float b[kStates] = {b4.x, b4.y, b4.z, b4.w}, c[kStates] = {c4.x, c4.y, c4.z, c4.w};
      f2 sum = 0;
#pragma unroll
      for (int j = 0; j < kStates; ++j) {
        h[j] = fma2(exp2_2(mul2(dt.x, a[j])), h[j], mul2(dt.y, b[j]));
        sum = j == 0 ? mul2(h[j], c[j]) : fma2(h[j], c[j], sum);
      }
      *reinterpret_cast<f2*>(put_y + t * kLanes * In::kRow) = sum;
    };
    if (now == kTile) {
#pragma unroll
      for (int t = 0; t < kTile; ++t) step(t);
    } else {
      for (int t = 0; t < now; ++t) step(t);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < In::kPairs; ++k) {
      float v = 0.0f, w = 0.0f;
#pragma unroll
      for (int l = 0; l < kLanes; ++l) {
        const float2 part = *reinterpret_cast<const float2*>(from_y + (k * In::kPitch * kLanes + l) * In::kRow);
        v += part.x;
        w += part.y;
      }
      put<T, kEven>(y + k * y_pitch, in.step + k * In::kPitch < now ? two : 0, (v + du[k].x) * gate[k].x, (w + du[k].y) * gate[k].y);
    }
    y += (int64_t)kTile * s.channels;
  }
  // behind the end: the rows of the chunk that are left
  T* rest = out + p.b * s.length * s.channels + p.c0 + in.channel;
  for (int64_t t = (p.first > p.len ? p.first : p.len) + in.step; t < p.end; t += In::kPitch)
    put<T, kEven>(rest + t * s.channels, two, 0.0f, 0.0f);
  // the chunk that the sequence ends in
  if (state_out != nullptr && (p.first < p.len || p.chunk == 0) && p.end >= p.len)
#pragma unroll
    for (int j = 0; j < kStates; ++j) {
      const int n = lane * kStates + j;
      float* to = state_out + (p.b * s.channels + channel) * s.states + n;
      if (n < s.states && on > 0) to[0] = halves(h[j]).x;
      if (n < s.states && on > 1) to[s.states] = halves(h[j]).y;
    }
}

// A chunk by itself, from a state of zero: forward h, or backward the carry a dh that leaves its first step; and the sum of its dt.
template <class T, int kLanes, bool kReverse, bool kEven>
__global__ void __launch_bounds__(kThreads) selective_scan_chunk_kernel(Scan s, const T* __restrict__ dout) {
  pdl_enter();
  using In = Lanes<kLanes>;
  constexpr int kWide = In::kWide, kPadded = In::kPadded;
  // what leaves the last chunk goes nowhere
  if ((int)(blockIdx.x / ((s.channels + kWide - 1) / kWide) % s.chunks) == (kReverse ? 0 : s.chunks - 1)) return;
  __shared__ float4 s_bc[kTile * kLanes];                  // B, or C
  __shared__ float4 s_dt[kTile * kWide / 2];               // of two channels: dt, and dt * u (or dy)
  const Block<kWide> p(s);
  const In in;
  const int c = threadIdx.x / kLanes * 2, lane = threadIdx.x % kLanes, channel = p.c0 + c, on = left_of(s.channels, channel);
  const bool gated = kReverse && s.z.p != nullptr;
  const int two = left_of(s.channels, p.c0 + in.channel), narrow_two = left_of(s.states, in.state);
  const int64_t tiles = p.first < p.last ? (p.last - p.first + kTile - 1) / kTile : 0;
  const int64_t t1 = p.first + (kReverse && tiles > 0 ? tiles - 1 : 0) * kTile;        // the first tile to do
  constexpr int kStep = kReverse ? -kTile : kTile;
  Cursor<T> at_x, at_delta, at_z, at_bc;
  const Seq x_of = kReverse ? Seq{dout, s.length * s.channels, s.channels} : s.u;
  at_x.set(x_of, p.b, t1 + in.step, p.c0 + in.channel, In::kPitch, kStep);
  at_delta.set(s.delta, p.b, t1 + in.step, p.c0 + in.channel, In::kPitch, kStep);
  at_z.set(s.z, p.b, t1 + in.step, p.c0 + in.channel, In::kPitch, kStep);
  at_bc.set(kReverse ? s.C : s.B, p.b, t1 + in.narrow_step, in.state, In::kNarrowPitch, kStep);
  Two<T> x[In::kPairs], delta[In::kPairs], z[In::kPairs], bc[In::kNarrow];
#pragma unroll
  for (int k = 0; k < In::kPairs; ++k) x[k] = delta[k] = z[k] = Two<T>{};
#pragma unroll
  for (int k = 0; k < In::kNarrow; ++k) bc[k] = Two<T>{};
  auto prefetch = [&](int steps) {
    const int n = steps - in.step, m = steps - in.narrow_step;
    at_x.template fetch<kEven, In::kPairs>(x, n, In::kPitch, two);
    at_delta.template fetch<kEven, In::kPairs>(delta, n, In::kPitch, two);
    if (gated) at_z.template fetch<kEven, In::kPairs>(z, n, In::kPitch, two);
    at_bc.template fetch<kEven, In::kNarrow>(bc, m, In::kNarrowPitch, narrow_two);
  };
  int steps = (int)(p.last - t1 < kTile ? p.last - t1 : kTile);
  if (tiles > 0) prefetch(steps);
  f2 a[kStates], h[kStates] = {0, 0, 0, 0};
  float2 span = make_float2(0.0f, 0.0f);
  states_of<kLanes>(s.A, channel, s.states, on, lane, kLog2e, a);
  const float2 bias = two_of(s.bias, p.c0 + in.channel, s.channels);
  float4* put_dt = s_dt + (in.step * kWide + in.channel) / 2;
  float* put_bc = reinterpret_cast<float*>(s_bc) + in.narrow_step * kPadded + in.state;
  const float4* in_bc = s_bc + lane;
  const ulonglong2* dt2 = reinterpret_cast<const ulonglong2*>(s_dt) + c / 2;
  for (int64_t i = 0; i < tiles; ++i) {
    if (i > 0) __syncthreads();
#pragma unroll
    for (int k = 0; k < In::kPairs; ++k) {
      float2 v = x[k].get();
      const float2 dv = delta[k].get();
      const float e = dv.x + bias.x, w = dv.y + bias.y;
      const float pe = softplus(e), pw = softplus(w), te = s.softplus ? pe : e, tw = s.softplus ? pw : w;
      if constexpr (kReverse) {
        const float2 zv = z[k].get(), silu = make_float2(activate<kActSilu>(zv.x), activate<kActSilu>(zv.y));
        v.x *= gated ? silu.x : 1.0f;
        v.y *= gated ? silu.y : 1.0f;
      } else {
        v.x *= te;
        v.y *= tw;
      }
      put_dt[k * In::kPitch * kWide / 2] = make_float4(te, tw, v.x, v.y);
    }
#pragma unroll
    for (int k = 0; k < In::kNarrow; ++k)
      if (In::kNarrowPitch <= kTile || in.narrow_step < kTile)
        *reinterpret_cast<float2*>(put_bc + k * In::kNarrowPitch * kPadded) = bc[k].get();
    __syncthreads();
    const int now = steps;
    const int64_t after = p.first + (kReverse ? tiles - 2 - i : i + 1) * kTile;
    steps = (int)(p.last - after < kTile ? p.last - after : kTile);
    if (i + 1 < tiles) prefetch(steps);
    float2 sum = make_float2(0.0f, 0.0f);
    auto step = [&](int t) {
      const ulonglong2 dt = dt2[t * kWide / 2];
      const float4 b4 = in_bc[t * kLanes];
      const float b[kStates] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
      for (int j = 0; j < kStates; ++j) {
        const f2 e = exp2_2(mul2(dt.x, a[j]));
        if constexpr (kReverse) h[j] = mul2(e, fma2(dt.y, b[j], h[j]));
        else h[j] = fma2(e, h[j], mul2(dt.y, b[j]));
      }
      sum.x += halves(dt.x).x;
      sum.y += halves(dt.x).y;
    };
    if (now == kTile) {
#pragma unroll
      for (int t = 0; t < kTile; ++t) step(kReverse ? kTile - 1 - t : t);
    } else {
      for (int t = 0; t < now; ++t) step(kReverse ? now - 1 - t : t);
    }
    span.x += sum.x;
    span.y += sum.y;
  }
  const int64_t at = (p.chunk * s.batch + p.b) * s.channels + channel;
  float2 v[kStates];
#pragma unroll
  for (int j = 0; j < kStates; ++j) v[j] = halves(h[j]);
  float4* local = reinterpret_cast<float4*>(s.local) + at * kLanes + lane;
  if (on > 0) local[0] = make_float4(v[0].x, v[1].x, v[2].x, v[3].x);
  if (on > 1) local[kLanes] = make_float4(v[0].y, v[1].y, v[2].y, v[3].y);
  if (on > 0 && lane == 0) s.span[at] = span.x;
  if (on > 1 && lane == 0) s.span[at + 1] = span.y;
}

struct Grads {
  const void* dout;            // [batch][length][channels]
  const float* keep;
  int kept;                    // states of a channel there
  void *du, *ddelta, *dz;      // like dout; dz null without a gate
  float* narrow;               // [blocks of channels][batch][length][2][16 * kBlocks]: shares of dB, dC
  float* sums;                 // [batch][chunks][channels * states + channels + channels]: dA, dD, ddelta_bias
};

// The matrix instruction reads the upper eleven bits of a factor and leaves out the others: what that is, and (fp32 gradients) half a step
// more of it, which rounds it to the nearest.  What is no number stays none: its bits may be all set, and a carry out of them is zero.
__device__ __forceinline__ float left_out(float x) { return x - __uint_as_float(__float_as_uint(x) & ~0x1fffu); }
template <class T> __device__ __forceinline__ uint32_t low_part(float x) {
  const int bits = __float_as_int(left_out(x));
  return (uint32_t)(sizeof(T) == 4 ? min(bits, 0x7fffefff) + 0x1000 : bits);
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// d += a b, 22 bits of each factor: a's two parts after one another, b's in columns of their own.  A step has two of the eight columns, the
// others of its product are times zero: a state that is no number, or infinite, makes dB and dC of the four steps that share the
// columns no numbers.  Eleven bits of each would leave dB and dC 1e-3 off in all (bf16, 16 x 331 steps of 2048 channels; so they are
// 3e-5 off) in 294 us for 345; high and low parts in three products without columns of their own: 361 us.  The low parts of fp32 are
// rounded: 2.6e-7 off, unrounded 4.2e-7 (the plain formula in fp32: 1.9e-7), 383 us for 365.
template <class T> __device__ __forceinline__ void product(float (&d)[4], const float (&a)[4], const uint32_t (&b)[2]) {
  uint32_t high[4], low[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    high[i] = __float_as_uint(a[i]);
    low[i] = low_part<T>(a[i]);
  }
  mma(d, high, b);
  mma(d, low, b);
}

// A warp: eight channels and sixteen states.  Thread: channels 2 c and 2 c + 1 (c = lane % 4, the fragments' columns c and c + 4),
// states n and n + 8 (n = lane / 4, their rows).
// kBlocks warps side by side have the states of wider layers.
template <class T, int kBlocks, bool kEven>
__global__ void __launch_bounds__(kThreads, 3) selective_scan_bwd_kernel(Scan s, Grads g) {
  pdl_enter();
  constexpr int kWarps = kThreads / 32, kWide = 8 * kWarps / kBlocks, kPadded = 16 * kBlocks, kSlots = 8 * kBlocks;
  constexpr int kRow = kWide == 8 ? 8 : kWide + 8;           // four slots of eight channels fall into banks of their own
  using In = Share<kKeep, kWide, kPadded>;
  static_assert(In::kPairs == 1, "a thread finishes what it has prepared, out of registers");
  __shared__ float4 s_bc[kKeep][kSlots];                     // B of states n and n + 8, C of them
  __shared__ float4 s_dt[kKeep][kWide / 2];                  // of two channels: dt, and dt u
  __shared__ f2 s_dy[kKeep][kWide / 2];                      // dy of them
  __shared__ __align__(16) float s_part[3][kKeep][kSlots][kRow];           // C h, B dh, A a h[t - 1] dh of a thread's two states
  __shared__ float s_narrow[kWarps / kBlocks][2][kKeep][kPadded + 8];   // dB, dC over a warp's channels; written without bank conflicts
  const Block<kWide> p(s);
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, part = warp % kBlocks, group = warp / kBlocks;
  const int slot = part * 8 + lane / 4, n0 = part * 16 + lane / 4, w0 = group * 8 + lane % 4 * 2;     // state, channel in the block
  const int channel = p.c0 + w0, on = left_of(s.channels, channel);
  f2 A[2], carry[2], dA[2];                                  // of a state: its two channels
  float dA_sum[2][2], dA_low[2][2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int n = n0 + 8 * j;
    float v[2], c[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool is = i < on && n < s.states;
      v[i] = is ? s.A[(int64_t)(channel + i) * s.states + n] : 0.0f;
      dA_sum[j][i] = dA_low[j][i] = 0.0f;
      if (is && s.chunks > 1)
        for (int q = s.chunks - 1; q > p.chunk; --q) {
          const int64_t at = (q * s.batch + p.b) * s.channels + channel + i;
          c[i] = across(c[i], s.span[at] * (v[i] * kLog2e)) + s.local[at * g.kept + n];
        }
    }
    A[j] = pair(v[0], v[1]);
    carry[j] = pair(c[0], c[1]);
  }
  const f2 A2[2] = {mul2(A[0], kLog2e), mul2(A[1], kLog2e)};
  // a thread prepares and finishes two channels of a step, and prepares some of B and C
  const In in;
  const int two = left_of(s.channels, p.c0 + in.channel), narrow_two = left_of(s.states, in.state);
  const bool mine = in.step < kKeep, gated = s.z.p != nullptr;
  const float2 skip = two_of(s.D, p.c0 + in.channel, s.channels), bias = two_of(s.bias, p.c0 + in.channel, s.channels);
  float2 dD = make_float2(0.0f, 0.0f), dbias = dD;
  const int64_t tiles = p.first < p.last ? (p.last - p.first + kKeep - 1) / kKeep : 0;
  const int64_t t1 = p.first + (tiles > 0 ? tiles - 1 : 0) * kKeep;
  Cursor<T> at_u, at_delta, at_z, at_up, at_b, at_c;
  at_u.set(s.u, p.b, t1 + in.step, p.c0 + in.channel, 0, -kKeep);
  at_delta.set(s.delta, p.b, t1 + in.step, p.c0 + in.channel, 0, -kKeep);
  at_z.set(s.z, p.b, t1 + in.step, p.c0 + in.channel, 0, -kKeep);
  at_up.set({g.dout, s.length * s.channels, s.channels}, p.b, t1 + in.step, p.c0 + in.channel, 0, -kKeep);
  at_b.set(s.B, p.b, t1 + in.narrow_step, in.state, In::kNarrowPitch, -kKeep);
  at_c.set(s.C, p.b, t1 + in.narrow_step, in.state, In::kNarrowPitch, -kKeep);
  const float* at_kept = g.keep + ((t1 / kKeep * s.batch + p.b) * s.channels + channel) * g.kept + n0;
  const int64_t kept_tile = s.batch * s.channels * g.kept;
  Two<T> u[1] = {}, delta[1] = {}, z[1] = {}, up[1] = {}, bb[In::kNarrow] = {}, cc[In::kNarrow] = {};
  float kept[2][2];
  auto prefetch = [&](int steps) {
    const int n = mine ? steps - in.step : 0, m = steps - in.narrow_step;
    at_u.template fetch<kEven, 1>(u, n, 0, two);
    at_delta.template fetch<kEven, 1>(delta, n, 0, two);
    if (gated) at_z.template fetch<kEven, 1>(z, n, 0, two);
    at_up.template fetch<kEven, 1>(up, n, 0, two);
    at_b.template fetch<kEven, In::kNarrow>(bb, m, In::kNarrowPitch, narrow_two);
    at_c.template fetch<kEven, In::kNarrow>(cc, m, In::kNarrowPitch, narrow_two);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) kept[j][i] = i < on && n0 + 8 * j < s.states ? at_kept[i * g.kept + 8 * j] : 0.0f;
    at_kept -= kept_tile;
  };
  int steps = (int)(p.last - t1 < kKeep ? p.last - t1 : kKeep);
  if (tiles > 0) prefetch(steps);
  const int64_t first_row = (p.b * s.length + t1 + in.step) * s.channels + p.c0 + in.channel, rows = (int64_t)kKeep * s.channels;
  T *to_du = reinterpret_cast<T*>(g.du) + first_row, *to_ddelta = reinterpret_cast<T*>(g.ddelta) + first_row;
  T* to_dz = g.dz != nullptr ? reinterpret_cast<T*>(g.dz) + first_row : nullptr;
  float* to_narrow = g.narrow + ((p.block * s.batch + p.b) * s.length + t1) * 2 * kPadded + threadIdx.x;
  for (int64_t tile = tiles - 1; tile >= 0; --tile) {
    const int now = steps;
    steps = kKeep;                 // of the tiles ahead of the last one
    // prepare; steps behind the end do nothing: dt = 0 and dy = 0
    float2 uv = make_float2(0.0f, 0.0f), dt = uv, slope_dt = uv, dz = uv, dy = uv;
    if (mine) {
      if (in.step < now) {
        const float2 dv = delta[0].get(), ov = up[0].get();
        uv = u[0].get();
        const float x = dv.x + bias.x, w = dv.y + bias.y;
        const float px = softplus(x, &slope_dt.x), pw = softplus(w, &slope_dt.y);
        dt = make_float2(s.softplus ? px : x, s.softplus ? pw : w);
        slope_dt = make_float2(s.softplus ? slope_dt.x : 1.0f, s.softplus ? slope_dt.y : 1.0f);
        const float2 zv = z[0].get();
        const float gx = sigmoid(zv.x), gw = sigmoid(zv.y);
        dy = make_float2(gated ? ov.x * zv.x * gx : ov.x, gated ? ov.y * zv.y * gw : ov.y);
        dz = make_float2(ov.x * gx * (1.0f + zv.x * (1.0f - gx)), ov.y * gw * (1.0f + zv.y * (1.0f - gw)));
      }
      s_dt[in.step][in.channel / 2] = make_float4(dt.x, dt.y, dt.x * uv.x, dt.y * uv.y);
      s_dy[in.step][in.channel / 2] = pair(dy);
    }
#pragma unroll
    for (int k = 0; k < In::kNarrow; ++k) {
      const int t = in.narrow_step + k * In::kNarrowPitch;
      if (t >= kKeep) continue;
      const float2 zero = make_float2(0.0f, 0.0f), bv = t < now ? bb[k].get() : zero, cv = t < now ? cc[k].get() : zero;
      // states n, n + 1 of sixteen: slots n % 8 and the next, the first or second of each
      float* to = reinterpret_cast<float*>(&s_bc[t][in.state / 16 * 8 + in.state % 8]) + in.state % 16 / 8;
      to[0] = bv.x;
      to[2] = cv.x;
      to[4] = bv.y;
      to[6] = cv.y;
    }
    f2 h[kKeep + 1][2], a[kKeep][2];
    h[0][0] = pair(kept[0][0], kept[0][1]);
    h[0][1] = pair(kept[1][0], kept[1][1]);
    __syncthreads();
    if (tile > 0) prefetch(kKeep);
#pragma unroll
    for (int t = 0; t < kKeep; ++t) {
      const float2 b = *reinterpret_cast<const float2*>(&s_bc[t][slot]);
      const ulonglong2 d = *reinterpret_cast<const ulonglong2*>(&s_dt[t][w0 / 2]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        a[t][j] = exp2_2(mul2(d.x, A2[j]));
        h[t + 1][j] = fma2(a[t][j], h[t][j], mul2(d.y, j == 0 ? b.x : b.y));
      }
    }
    uint32_t own_dy[2], own_du[2];       // of the step whose column this lane has: columns 0 to 3 high parts, 4 to 7 low parts of these
    float dB[4], dC[4];                  // state n (n + 8), columns 2 (lane % 4) and the next
    dA[0] = dA[1] = 0;
#pragma unroll
    for (int t = kKeep - 1; t >= 0; --t) {
      if (t % kHalf == kHalf - 1) {
        const int own = t / kHalf * kHalf + lane / 4 % kHalf;
        const float2 y2 = halves(s_dy[own][w0 / 2]), u2 = halves(reinterpret_cast<const ulonglong2*>(&s_dt[own][w0 / 2])->y);
        const float y[2] = {y2.x, y2.y}, u[2] = {u2.x, u2.y};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          own_dy[i] = lane < 16 ? __float_as_uint(y[i]) : low_part<T>(y[i]);
          own_du[i] = lane < 16 ? __float_as_uint(u[i]) : low_part<T>(u[i]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) dB[q] = dC[q] = 0.0f;
      }
      const float4 bc = s_bc[t][slot];
      const f2 d = *reinterpret_cast<const f2*>(&s_dt[t][w0 / 2]), y2 = s_dy[t][w0 / 2];
      f2 dh[2], da[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        dh[j] = fma2(y2, j == 0 ? bc.z : bc.w, carry[j]);
        carry[j] = mul2(a[t][j], dh[j]);
        da[j] = mul2(carry[j], h[t][j]);
        dA[j] = fma2(da[j], d, dA[j]);
      }
      *reinterpret_cast<f2*>(&s_part[0][t][slot][w0]) = fma2(h[t + 1][1], bc.w, mul2(h[t + 1][0], bc.z));
      *reinterpret_cast<f2*>(&s_part[1][t][slot][w0]) = fma2(dh[1], bc.y, mul2(dh[0], bc.x));
      *reinterpret_cast<f2*>(&s_part[2][t][slot][w0]) = fma2(da[1], A[1], mul2(da[0], A[0]));
      const bool column = lane / 4 % kHalf == t % kHalf;
      const uint32_t by[2] = {column ? own_dy[0] : 0u, column ? own_dy[1] : 0u}, bu[2] = {column ? own_du[0] : 0u, column ? own_du[1] : 0u};
      const float2 h0 = halves(h[t + 1][0]), h1 = halves(h[t + 1][1]), d0 = halves(dh[0]), d1 = halves(dh[1]);
      const float ha[4] = {h0.x, h1.x, h0.y, h1.y}, da4[4] = {d0.x, d1.x, d0.y, d1.y};
      product<T>(dC, ha, by);
      product<T>(dB, da4, bu);
      if (t % kHalf == 0) {
        // columns j and j + 4 belong together, in the lanes c and c + 2: each of the two goes on with one state
        const bool second = lane % 4 >= 2;
        const int n = n0 + (second ? 8 : 0), to = t + 2 * (lane % 2);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          s_narrow[group][0][to + q][n] = (second ? dB[2 + q] : dB[q]) + __shfl_xor_sync(0xffffffffu, second ? dB[q] : dB[2 + q], 2);
          s_narrow[group][1][to + q][n] = (second ? dC[2 + q] : dC[q]) + __shfl_xor_sync(0xffffffffu, second ? dC[q] : dC[2 + q], 2);
        }
      }
    }
    // into the running sum with its rounding errors beside it: a sequence has thousands of terms
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float2 v = halves(dA[j]);
      const float add[2] = {v.x, v.y};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float y = add[i] - dA_low[j][i], t = dA_sum[j][i] + y;
        dA_low[j][i] = (t - dA_sum[j][i]) - y;
        dA_sum[j][i] = t;
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kKeep * 2 * kPadded / kThreads; ++j) {
      const unsigned i = threadIdx.x + j * kThreads, t = i / (2 * kPadded), k = i / kPadded % 2, n = i % kPadded;
      if ((int)t >= now) break;
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps / kBlocks; ++w) v += s_narrow[w][k][t][n];
      to_narrow[j * kThreads] = v;
    }
    to_narrow -= kKeep * 2 * kPadded;
    if (mine && in.step < now) {
      float2 v[3];
#pragma unroll
      for (int q = 0; q < 3; ++q) {
        float x = 0.0f, w = 0.0f;
#pragma unroll
        for (int l = 0; l < kSlots; ++l) {
          const float2 o = *reinterpret_cast<const float2*>(&s_part[q][in.step][l][in.channel]);
          x += o.x;
          w += o.y;
        }
        v[q] = make_float2(x, w);
      }
      if (to_dz != nullptr) put<T, kEven>(to_dz, two, dz.x * fmaf(skip.x, uv.x, v[0].x), dz.y * fmaf(skip.y, uv.y, v[0].y));
      put<T, kEven>(to_du, two, fmaf(v[1].x, dt.x, skip.x * dy.x), fmaf(v[1].y, dt.y, skip.y * dy.y));
      const float ex = fmaf(v[1].x, uv.x, v[2].x) * slope_dt.x, ew = fmaf(v[1].y, uv.y, v[2].y) * slope_dt.y;
      put<T, kEven>(to_ddelta, two, ex, ew);
      dD.x = fmaf(dy.x, uv.x, dD.x);
      dD.y = fmaf(dy.y, uv.y, dD.y);
      dbias.x += ex;
      dbias.y += ew;
    }
    to_du -= rows;
    to_ddelta -= rows;
    if (to_dz != nullptr) to_dz -= rows;
  }
  // behind the end: the rows of the chunk that are left
  const int64_t lead = p.b * s.length * s.channels + p.c0 + in.channel;
  for (int64_t t = (p.first > p.len ? p.first : p.len) + in.step; t < p.end; t += In::kPitch) {
    const int64_t row = lead + t * s.channels;
    put<T, kEven>(reinterpret_cast<T*>(g.du) + row, two, 0.0f, 0.0f);
    put<T, kEven>(reinterpret_cast<T*>(g.ddelta) + row, two, 0.0f, 0.0f);
    if (g.dz != nullptr) put<T, kEven>(reinterpret_cast<T*>(g.dz) + row, two, 0.0f, 0.0f);
  }
  float* sums = g.sums + (p.b * s.chunks + p.chunk) * (int64_t)s.channels * (s.states + 2);
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (i < on && n0 + 8 * j < s.states) sums[(int64_t)(channel + i) * s.states + n0 + 8 * j] = dA_sum[j][i];
  __syncthreads();
  float4* stage = reinterpret_cast<float4*>(&s_part[0][0][0][0]);      // room for one of each thread
  stage[threadIdx.x] = make_float4(dD.x, dD.y, dbias.x, dbias.y);
  __syncthreads();
  if (threadIdx.x < kWide / 2) {
    float4 v = stage[threadIdx.x];
    for (int k = threadIdx.x + kWide / 2; k < kThreads; k += kWide / 2) {
      const float4 w = stage[k];
      v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
    }
    float* to = sums + (int64_t)s.channels * s.states;
    put<float, false>(to + p.c0 + in.channel, two, v.x, v.y);
    put<float, false>(to + s.channels + p.c0 + in.channel, two, v.z, v.w);
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
// Four states from the n-th on, as many as there are; kWhole: always four, on a boundary.
template <class T, bool kWhole> __device__ __forceinline__ void four(const T* p, int n, int states, float (&to)[kStates]) {
  if constexpr (kWhole) {
    unpack<T, kStates>(load<T, kStates>(p + n), to);
  } else {
#pragma unroll
    for (int j = 0; j < kStates; ++j) to[j] = n + j < states ? as_float(p[n + j]) : 0.0f;
  }
}

// One step of every sequence: the state moves on; state_out may be s.state.  A block has kWide channels of `many` sequences, one
// after the other, each fetched while the one ahead is at work.  Bound by memory: 8 bytes a state (1000 sequences of 2048 channels with
// 16 states: 65 us, 4.0 TB/s of 6.5; four states fetched at once 71 us, without softplus and gate it would be 61).
template <class T, int kLanes, bool kWhole>
__global__ void __launch_bounds__(kThreads) selective_scan_step_kernel(Scan s, float* state_out, T* __restrict__ out, int many) {
  pdl_enter();
  constexpr int kWide = kThreads / kLanes;
  const int blocks = (s.channels + kWide - 1) / kWide;
  const int64_t rest = blockIdx.x / blocks, first = rest * many, last = first + many < s.batch ? first + many : s.batch;
  const int c = (int)(blockIdx.x - rest * blocks) * kWide + threadIdx.x / kLanes, lane = threadIdx.x % kLanes, n = lane * kStates;
  const bool on = c < s.channels && n < s.states;
  float a[kStates] = {}, bias = 0.0f, skip = 0.0f;
  if (on) {
    four<float, kWhole>(s.A + (int64_t)c * s.states, n, s.states, a);
#pragma unroll
    for (int j = 0; j < kStates; ++j) a[j] *= kLog2e;
    if (s.bias != nullptr) bias = s.bias[c];
    if (s.D != nullptr) skip = s.D[c];
  }
  float h[kStates] = {}, bb[kStates] = {}, cc[kStates] = {}, u = 0.0f, delta = 0.0f, z = 0.0f;
  auto fetch = [&](int64_t b) {
    four<float, kWhole>(s.state + (b * s.channels + c) * s.states, n, s.states, h);
    four<T, kWhole>(reinterpret_cast<const T*>(s.B.p) + b * s.B.b, n, s.states, bb);
    four<T, kWhole>(reinterpret_cast<const T*>(s.C.p) + b * s.C.b, n, s.states, cc);
    u = at<T>(s.u, b, c);
    delta = at<T>(s.delta, b, c);
    if (s.z.p != nullptr) z = at<T>(s.z, b, c);
  };
  if (on) fetch(first);
  for (int64_t b = first; b < last; ++b) {
    float part = 0.0f, x = 0.0f, gate = 0.0f, next[kStates];
    if (on) {
      const float raw = delta + bias, dt = s.softplus ? softplus(raw) : raw;
#pragma unroll
      for (int j = 0; j < kStates; ++j) {
        next[j] = fmaf(exp2_approx(dt * a[j]), h[j], dt * u * bb[j]);
        part = fmaf(cc[j], next[j], part);
      }
      x = u;
      gate = z;
      if (b + 1 < last) fetch(b + 1);
      float* to = state_out + (b * s.channels + c) * s.states + n;
      if constexpr (kWhole) {
        store<float, kStates>(to, next);
      } else {
#pragma unroll
        for (int j = 0; j < kStates; ++j)
          if (n + j < s.states) to[j] = next[j];
      }
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    if (on && lane == 0) {
      part = fmaf(skip, x, part);
      if (s.z.p != nullptr) part *= activate<kActSilu>(gate);
      out[b * s.channels + c] = as_type<T>(part);
    }
  }
}

int lanes_of(int states) {
  int l = 2;
  while (l * kStates < states) l *= 2;
  return l;
}
int state_blocks(int states) { return states <= 16 ? 1 : states <= 32 ? 2 : 4; }
int blocks_of(int channels, int wide) { return (channels + wide - 1) / wide; }

// Chunks of a pass over `blocks` blocks, the number that is estimated to take least.  A block takes as long as its steps, a start of
// some 24 steps, and the chunks ahead of it to join; an SM has `full` blocks at the pace of one, and takes longer with more, up to
// `most` at a time; with chunks there is a pass more, and all that is done `again` times.  Us without and with them, forward and
// backward: 1 x 4099 steps of 2048 channels 513 / 119 and 784 / 291, 1 x 2000 of 64 250 / 23 and 369 / 30, 4 x 1000 of 2048 128 / 102
// and 329 / 265; 16 x 200 of 1024 would take 35 / 61 forward and has none.
struct Pace {
  double full, again;
  int64_t most;
};
constexpr Pace kForward = {4.2, 1.9, 8}, kBackward = {3.0, 1.25, 3};
void split(Scan* s, int64_t blocks, const Pace& p) {
  double best = 0.0;
  for (int64_t n = 1; n <= kMaxChunks; n *= 2) {
    const int64_t chunk = ((s->length + n - 1) / n + kTile - 1) / kTile * kTile;
    if (n > 1 && chunk >= s->length) break;
    const int64_t chunks = chunk > 0 ? (s->length + chunk - 1) / chunk : 1;
    const int64_t here = (blocks * chunks + sm_count() - 1) / sm_count(), rest = here % p.most;
    const double pace = (double)(here / p.most) * (double)p.most / p.full + (rest == 0 ? 0.0 : rest < p.full ? 1.0 : (double)rest / p.full);
    const double cost = (chunks > 1 ? p.again : 1.0) * ((double)chunk + 24.0 + 0.25 * (double)chunks) * pace;
    if (n > 1 && cost >= best) continue;
    best = cost;
    s->chunk = chunk;
    s->chunks = (int)chunks;
  }
}

template <class T, int kLanes, bool kEven> int forward_even(const Scan& s, void* out, float* state_out, float* keep, void* stream) {
  static SmemAllowed allowed{0};
  constexpr int kWide = Lanes<kLanes>::kWide;
  constexpr size_t kSmem = kTile * (2 * kLanes * 16 + kWide * 8 + kLanes * Lanes<kLanes>::kRow * 4);
  if (kSmem > 48 * 1024) {
    const int rc = allow_smem(selective_scan_fwd_kernel<T, kLanes, kEven>, kSmem, allowed);
    if (rc != 0) return rc;
  }
  const dim3 grid((unsigned)(s.batch * s.chunks * blocks_of(s.channels, kWide)));
  if (s.chunks > 1) {
    const int rc = launch(selective_scan_chunk_kernel<T, kLanes, false, kEven>, grid, kThreads, 0, stream, s, (const T*)nullptr);
    if (rc != 0) return rc;
  }
  return launch(selective_scan_fwd_kernel<T, kLanes, kEven>, grid, kThreads, kSmem, stream, s, (T*)out, state_out, keep);
}
template <class T, int kLanes> int forward(const Scan& s, void* out, float* state_out, float* keep, void* stream) {
  return s.even ? forward_even<T, kLanes, true>(s, out, state_out, keep, stream) : forward_even<T, kLanes, false>(s, out, state_out, keep, stream);
}
template <class T, int kLanes> int carries(const Scan& s, const void* dout, void* stream) {
  const dim3 grid((unsigned)(s.batch * s.chunks * blocks_of(s.channels, Lanes<kLanes>::kWide)));
  return s.even ? launch(selective_scan_chunk_kernel<T, kLanes, true, true>, grid, kThreads, 0, stream, s, (const T*)dout)
                : launch(selective_scan_chunk_kernel<T, kLanes, true, false>, grid, kThreads, 0, stream, s, (const T*)dout);
}
template <class T, int kBlocks> int backward_blocks(const Scan& s, const Grads& g, void* dB, void* dC, void* stream) {
  const int blocks = blocks_of(s.channels, 32 / kBlocks), padded = 16 * kBlocks;
  const dim3 grid((unsigned)(s.batch * s.chunks * blocks));
  const int rc = s.even ? launch(selective_scan_bwd_kernel<T, kBlocks, true>, grid, kThreads, 0, stream, s, g)
                        : launch(selective_scan_bwd_kernel<T, kBlocks, false>, grid, kThreads, 0, stream, s, g);
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
  // as many sequences to a block as leave eight blocks to every SM, four at most: A, D and the bias are read once for them
  const int64_t blocks = blocks_of(s.channels, kThreads / kLanes);
  int many = 1;
  while (many < 4 && blocks * (s.batch / (2 * many)) >= 8 * sm_count()) many *= 2;
  const dim3 grid((unsigned)((s.batch + many - 1) / many * blocks));
  const uintptr_t bytes = 4 * sizeof(T);
  const bool whole = s.states % 4 == 0 && aligned16(s.A) && aligned16(s.state) && aligned16(state_out) && (uintptr_t)s.B.p % bytes == 0 &&
                     (uintptr_t)s.C.p % bytes == 0 && s.B.b % 4 == 0 && s.C.b % 4 == 0;
  return whole ? launch(selective_scan_step_kernel<T, kLanes, true>, grid, kThreads, 0, stream, s, state_out, (T*)out, many)
               : launch(selective_scan_step_kernel<T, kLanes, false>, grid, kThreads, 0, stream, s, state_out, (T*)out, many);
}

// F<T, kLanes>(...)
#define ESGD_LANES(T, F, ...)                                                                                   \
  (lanes == 2 ? F<T, 2>(__VA_ARGS__) : lanes == 4 ? F<T, 4>(__VA_ARGS__) : lanes == 8 ? F<T, 8>(__VA_ARGS__) : F<T, 16>(__VA_ARGS__))
#define ESGD_TYPE(F, ...) (is_bf16 ? ESGD_LANES(__nv_bfloat16, F, __VA_ARGS__) : ESGD_LANES(float, F, __VA_ARGS__))

bool taken(const Scan& s) { return s.states >= 1 && s.states <= 64 && s.channels >= 1 && s.batch >= 0 && s.length >= 0; }

Scan scan_of(const esgd_scan* e, bool backward) {
  Scan s = {};
  Seq* q[5] = {&s.u, &s.delta, &s.z, &s.B, &s.C};
  const uintptr_t size = e->is_bf16 ? 2 : 4;
  s.even = e->channels % 2 == 0 && e->states % 2 == 0;
  for (int i = 0; i < 5; ++i) {
    *q[i] = {e->p[i], e->b[i], e->t[i]};
    if (e->p[i] != nullptr && ((uintptr_t)e->p[i] % (2 * size) || e->b[i] % 2 || e->t[i] % 2)) s.even = 0;
  }
  s.A = e->A; s.D = e->D; s.bias = e->bias;
  s.lengths = e->lengths;
  s.state = e->state;
  s.batch = e->batch; s.length = e->length;
  s.channels = e->channels; s.states = e->states; s.softplus = e->softplus;
  if (backward) split(&s, s.batch * blocks_of(s.channels, 32 / state_blocks(s.states)), kBackward);
  else split(&s, s.batch * blocks_of(s.channels, 2 * kThreads / lanes_of(s.states)), kForward);
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

// Floats of room for a pass in a direction (the chunks'; none for many sequences or short ones), for what the forward pass
// keeps for the backward pass, and for the shares of dB, dC and of the parameters' gradients.
int64_t esgd_selective_scan_local(const esgd_scan* e, int backward) { return local_floats(scan_of(e, backward)); }
int64_t esgd_selective_scan_keep(const esgd_scan* e) {
  return (e->length + kKeep - 1) / kKeep * e->batch * e->channels * lanes_of(e->states) * kStates;
}
int64_t esgd_selective_scan_narrow(const esgd_scan* e) {
  const int side = state_blocks(e->states);
  return blocks_of(e->channels, 32 / side) * e->batch * e->length * 2 * 16 * side;
}
int64_t esgd_selective_scan_parts(const esgd_scan* e) { return e->length > 0 ? e->batch * scan_of(e, true).chunks : 0; }

int esgd_selective_scan_fwd(const esgd_scan* e, void* out, float* state_out, float* keep, float* local, void* stream) {
  Scan s = scan_of(e, false);
  if (!taken(s)) return (int)cudaErrorInvalidValue;
  if (s.batch == 0) return 0;
  place(&s, local);
  const int is_bf16 = e->is_bf16, lanes = lanes_of(s.states);
  return ESGD_TYPE(forward, s, out, state_out, keep, stream);
}

// sums [parts][channels * states + 2 * channels].
int esgd_selective_scan_bwd(const esgd_scan* e, const void* dout, const float* keep, void* du, void* ddelta, void* dz, void* dB, void* dC,
                            float* narrow, float* sums, float* local, void* stream) {
  Scan s = scan_of(e, true);
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
  const Scan s = scan_of(e, false);
  if (!taken(s)) return (int)cudaErrorInvalidValue;
  if (s.batch == 0) return 0;
  if (s.state == nullptr) return (int)cudaErrorInvalidValue;
  const int is_bf16 = e->is_bf16, lanes = lanes_of(s.states);
  return ESGD_TYPE(step, s, state_out, out, stream);
}

}  // extern "C"
