// Group norm (+ residual) (+ activation) of channels-last activations, forward and backward.
//
//   mean, var over a sample's pixels and a group's C / G channels;   n = (x - mean) / sqrt(var + eps)
//   z  = act(gamma n + beta [+ residual])
//   d  = dz act'(.);  dgamma = sum d n,  dbeta = sum d,  dresidual = d
//   dx = (gamma d - avg(gamma d) - n avg(gamma d n)) / sqrt(var + eps)      averages over the group
//
// Bound by memory: x (and residual) in, z out; x, dz (and residual) in, dx (and dresidual) out.  A cluster of CTAs has a sample's
// slice of whole groups, the rows (pixels) split among its CTAs; the sums of the CTAs meet in distributed shared memory, so that
// one launch does statistics and result.  A CTA asks for all of its rows at once (cp.async), and they stay in shared memory for the
// passes that follow; what does not fit there, and the residual, is read again and found in L2, of which what the resident
// clusters work on at a time is a fraction.
//
// Variances are squared deviations about a thread's, then a CTA's own mean of each channel, joined with the means: with sum and sum of
// squares a mean of 100 deviations would cost four digits.
//
// 128 x 256 x 56 x 56 bf16, SiLU and residual: 160 us forward (3.9 TB/s of 6.5), 273 us backward (3.8 TB/s); 64 x 512 x 14 x 14: 11.5 and
// 19 us.  The CTAs of a cluster wait for their slowest, and rows beyond the shared memory come out of L2 again.  Rows loaded at a time
// by a thread, forward statistics 4 or 2: 32 x 64 x 112 x 112 47 or 51 us; backward 4, 2 or 6: 286, 307 or 368 us, and where all rows
// are held 19.0, 18.2 or 19.2; forward results 2 or 4: 160 or 171 us (registers).
#include <cooperative_groups.h>
#include "launch.cuh"
#include "rows.cuh"

namespace {

namespace cg = cooperative_groups;
using namespace esgd;

constexpr int kThreads = 256;
constexpr int kMaxSlice = 4096;      // channels of a slice: two floats each in shared memory, beside the threads' sums

struct Shape {
  int64_t rows;        // pixels of a sample
  int channels, per;   // C, and channels of a group
  int slice;           // channels of a slice: whole groups
  int split;           // CTAs of a cluster
  int held;            // rows of a CTA that stay in shared memory
  int passing;         // nothing of a tensor is in L2 when the next operator reads it
  float eps;
};

// The backward pass' sums of two sets, and later three rows of coefficients.
__host__ __device__ constexpr int stage_floats(int v, int slice) { return 2 * kThreads * v > 3 * slice ? 2 * kThreads * v : (3 * slice + 3) / 4 * 4; }

// How L2 keeps what the backward pass fetches once or writes: as ever, or, of tensors that it cannot hold, less long than the rows that
// are fetched again (128 x 256 x 56 x 56 with residual: 286 -> 273 us, 885 -> 744 MB read for 616; forward the registers for it cost
// more than it brings, 32 x 64 x 112 x 112: 47 -> 51 us).
__device__ __forceinline__ uint64_t l2_policy(const Shape& s) {
  uint64_t first, normal;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(first));
  asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(normal));
  return s.passing ? first : normal;
}
template <class T, int kV> __device__ __forceinline__ void leave2(T* p, const f2 (&f)[PairsOf<kV>::n], uint64_t policy) {
  if constexpr (kV == 1) {
    store2<T, kV>(p, f);
  } else {
    uint4 w;
    store2<T, kV>(reinterpret_cast<T*>(&w), f);
    asm volatile("st.global.L2::cache_hint.v4.b32 [%0], {%1, %2, %3, %4}, %5;" ::"l"(p), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w), "l"(policy)
                 : "memory");
  }
}

// Where a thread works: a vector of kV channels, every `lanes`-th row of its CTA's.
template <int kV> struct Place {
  int vectors, wide, lanes, lane, vec;
  int rows;            // of the CTA
  bool fold;           // a warp has whole rows: its lanes are added up before they go to shared memory
  __device__ Place(const Shape& s, int rank) {
    vectors = s.slice / kV;
    wide = min(vectors, kThreads);
    lanes = kThreads / wide;
    lane = threadIdx.x / wide;
    vec = threadIdx.x - lane * wide;
    rows = (int)(s.rows * (rank + 1) / s.split - s.rows * rank / s.split);
    fold = wide <= 16 && (wide & (wide - 1)) == 0;
  }
  __device__ bool on(int v) const { return lane < lanes && v < vectors; }
};

// Sum over a warp.
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sums over the CTA's rows of the threads' channels (kSets of them at a time), into out[set * slice + channel] from channel v0 * kV
// on.  Every thread calls it.
template <int kSets, int kV>
__device__ __forceinline__ void channel_sums(const Place<kV>& p, const f2 (&sets)[kSets][PairsOf<kV>::n], int v0, float* stage, float* out, int slice) {
  int partial = p.lanes, row = p.lane;
  bool writes = p.lane < p.lanes;
  float a[kSets][kV];
#pragma unroll
  for (int i = 0; i < kSets; ++i)
#pragma unroll
    for (int q = 0; q < kV; ++q) a[i][q] = q % 2 == 0 ? halves(sets[i][q / 2]).x : halves(sets[i][q / 2]).y;
  if (p.fold) {
    partial = kThreads / 32;
    row = threadIdx.x / 32;
    writes = (threadIdx.x & 31) < p.wide;
    for (int o = p.wide; o < 32; o *= 2)
#pragma unroll
      for (int i = 0; i < kSets; ++i)
#pragma unroll
        for (int q = 0; q < kV; ++q) a[i][q] += __shfl_xor_sync(0xffffffffu, a[i][q], o);
  }
  const int pitch = p.wide * kV;
  if (writes)
#pragma unroll
    for (int i = 0; i < kSets; ++i)
#pragma unroll
      for (int q = 0; q < kV; ++q) stage[(i * partial + row) * pitch + p.vec * kV + q] = a[i][q];
  __syncthreads();
  const int here = min(p.wide, p.vectors - v0) * kV;
  for (int c = threadIdx.x; c < kSets * here; c += kThreads) {
    const int i = kSets > 1 && c >= here ? 1 : 0, ch = c - i * here;
    float t = 0.0f;
    for (int r = 0; r < partial; ++r) t += stage[(i * partial + r) * pitch + ch];
    out[i * slice + v0 * kV + ch] = t;
  }
  __syncthreads();
}
// A thread's channels of a row of shared memory.
template <int kV> __device__ __forceinline__ void channels_of(const float* p, f2 (&to)[PairsOf<kV>::n]) {
  if constexpr (kV == 1) {
    to[0] = pair(p[0], 0.0f);
  } else {
#pragma unroll
    for (int q = 0; q < kV / 4; ++q) {
      const float4 v = *reinterpret_cast<const float4*>(p + 4 * q);
      to[2 * q] = pair(v.x, v.y);
      to[2 * q + 1] = pair(v.z, v.w);
    }
  }
}

// Rows of kMany tensors from `base` on: the first `held` of a CTA in shared memory, each thread's own vectors, the others where they
// are.
template <class T, int kV, int kMany> struct Rows {
  const T* p[kMany];   // the CTA's first row and the slice's first channel
  T* in;               // [kMany][held][slice]
  int held, slice;
  int64_t pitch;
  __device__ Rows(T* in_, const Shape& s) : in(in_), held(s.held), slice(s.slice), pitch(s.channels) {}
  template <bool kPolicy> __device__ __forceinline__ void ask(const Place<kV>& pl, uint64_t policy = 0) const {
    if constexpr (kV > 1) {
      const int n = held < pl.rows ? held : pl.rows;
      for (int v = pl.vec; pl.on(v); v += pl.wide)
#pragma unroll
        for (int i = 0; i < kMany; ++i) {
          const T* from = p[i] + pl.lane * pitch + v * kV;
          uint32_t to = (uint32_t)__cvta_generic_to_shared(in + (i * held + pl.lane) * slice + v * kV);
          for (int r = pl.lane; r < n; r += pl.lanes) {
            if constexpr (kPolicy)
              asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "l"(policy) : "memory");
            else
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
            from += pl.lanes * pitch;
            to += pl.lanes * slice * (int)sizeof(T);
          }
        }
    }
  }
  // The vector of a thread's first row.
  __device__ __forceinline__ Pack<T, kV> first(const Place<kV>& pl, int v) const {
    return load<T, kV>(kV > 1 && pl.lane < held ? in + pl.lane * slice + v * kV : p[0] + pl.lane * pitch + v * kV);
  }
  // use(vectors, the vector of `more`, their offset from p[]) for a thread's rows; kAhead of them are loaded at a time, and then used()
  // is called (behind single rows it is not: those are fewer than kAhead, twice).
  template <int kAhead, bool kMore, class Use> __device__ __forceinline__ void each(const Place<kV>& pl, int v, const T* more, Use use) const {
    each<kAhead, kMore>(pl, v, more, use, [] {});
  }
  template <int kAhead, bool kMore, class Use, class Used>
  __device__ __forceinline__ void each(const Place<kV>& pl, int v, const T* more, Use use, Used used) const {
    const int lanes = pl.lanes, n = kV == 1 ? 0 : held < pl.rows ? held : pl.rows, next = lanes * slice;
    const int64_t down = lanes * pitch;
    const T* own = in + pl.lane * slice + v * kV;
    int64_t o = pl.lane * pitch + v * kV;
    int r = pl.lane;
    Pack<T, kV> x[kAhead][kMany], e[kAhead];
    for (; r + (kAhead - 1) * lanes < n; r += kAhead * lanes, o += kAhead * down, own += kAhead * next) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if constexpr (kMore) e[u] = load<T, kV>(more + o + u * down);
#pragma unroll
        for (int i = 0; i < kMany; ++i) x[u][i] = load<T, kV>(own + i * held * slice + u * next);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) use(x[u], e[u], o + u * down);
      used();
    }
    for (; r < n; r += lanes, o += down, own += next) {
      if constexpr (kMore) e[0] = load<T, kV>(more + o);
#pragma unroll
      for (int i = 0; i < kMany; ++i) x[0][i] = load<T, kV>(own + i * held * slice);
      use(x[0], e[0], o);
    }
    for (; r + (kAhead - 1) * lanes < pl.rows; r += kAhead * lanes, o += kAhead * down) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if constexpr (kMore) e[u] = load<T, kV>(more + o + u * down);
#pragma unroll
        for (int i = 0; i < kMany; ++i) x[u][i] = load<T, kV>(p[i] + o + u * down);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) use(x[u], e[u], o + u * down);
      used();
    }
    for (; r < pl.rows; r += lanes, o += down) {
      if constexpr (kMore) e[0] = load<T, kV>(more + o);
#pragma unroll
      for (int i = 0; i < kMany; ++i) x[0][i] = load<T, kV>(p[i] + o);
      use(x[0], e[0], o);
    }
  }
};
__device__ __forceinline__ void arrived() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// The unit that a cluster works on.
struct Unit {
  int rank, c0;
  int64_t sample, base;      // of its first row and channel
  __device__ Unit(const Shape& s, int rank_) : rank(rank_) {
    const int slices = s.channels / s.slice;
    const int64_t unit = blockIdx.x / s.split;
    sample = unit / slices;
    c0 = (int)(unit - sample * slices) * s.slice;
    base = (sample * s.rows + s.rows * rank / s.split) * s.channels + c0;
  }
};

template <class T, int kV, int kAct, bool kAdd>
__global__ void __launch_bounds__(kThreads, 4)
group_norm_fwd_kernel(const T* __restrict__ x, const T* __restrict__ residual, T* __restrict__ z, const float* __restrict__ gamma,
                      const float* __restrict__ beta, float* __restrict__ stats, Shape s) {
  pdl_enter();
  extern __shared__ float4 smem4[];
  const int groups = s.slice / s.per;
  T* held = reinterpret_cast<T*>(smem4);                   // [held][slice]
  float* stage = reinterpret_cast<float*>(held + s.held * s.slice);
  float* mean = stage + kThreads * kV;                     // [slice] the channels' sums, then -means
  float* m2 = mean + s.slice;                              // [slice], then what a deviation is multiplied with
  float* shift = m2 + s.slice;                             // [slice]
  float* gmean = shift + s.slice;                          // [groups] of this CTA's rows
  float* gm2 = gmean + groups;
  cg::cluster_group cluster = cg::this_cluster();
  const Unit unit(s, s.split > 1 ? (int)cluster.block_rank() : 0);
  const Place<kV> p(s, unit.rank);
  Rows<T, kV, 1> in(held, s);
  in.p[0] = x + unit.base;
  constexpr int kP = PairsOf<kV>::n;
  const int rows = p.rows;
  in.ask<false>(p);
  arrived();
  const float inv_rows = rows > 0 ? 1.0f / (float)rows : 0.0f;
  // A thread's rows about a centre: its first one, and after 4, 8, 16, ... of them the mean so far.  Up to the next of these the squares
  // about that centre are at most twice those about the mean, so that they lose no more than the roundings of a sum of so many terms.
  // (About the first row alone, were it an outlier, they would be as many times as large as there are rows: 1e-3 of the variance with
  // 1024 of them.)  Threads, channels and CTAs are then joined as means and squared deviations.
  const float own_rows = (float)(rows > p.lane ? (rows - p.lane + p.lanes - 1) / p.lanes : 0), inv_own = own_rows > 0.0f ? 1.0f / own_rows : 0.0f;
  for (int v0 = 0; v0 < p.vectors; v0 += p.wide) {
    const int v = v0 + p.vec;
    f2 a[1][kP] = {}, square[kP] = {}, first[kP] = {};
    if (p.on(v) && p.lane < rows) {
      unpack2<T, kV>(in.first(p, v), first);
#pragma unroll
      for (int q = 0; q < kP; ++q) first[q] = mul2(first[q], -1.0f);
      int seen = 0, next = 4;
      in.template each<4, false>(p, v, nullptr, [&](const Pack<T, kV>(&raw)[1], const Pack<T, kV>&, int64_t) {
        ++seen;
        f2 f[kP];
        unpack2<T, kV>(raw[0], f);
#pragma unroll
        for (int q = 0; q < kP; ++q) {
          const f2 d = add2(f[q], first[q]);
          a[0][q] = add2(a[0][q], d);
          square[q] = fma2(d, d, square[q]);
        }
      }, [&] {
        if (seen < next) return;
        next = 2 * seen;
        const float n = (float)seen, inv = 1.0f / n;
#pragma unroll
        for (int q = 0; q < kP; ++q) {
          const f2 to = fma2(a[0][q], -inv, first[q]), by = add2(first[q], mul2(to, -1.0f));       // -centre, and how far that moved
          square[q] = fma2(mul2(by, -1.0f), fma2(by, -n, mul2(a[0][q], 2.0f)), square[q]);
          a[0][q] = fma2(by, -n, a[0][q]);
          first[q] = to;
        }
      });
    }
    // from here: the thread's mean about -first, its squares about the mean, and its sum
    f2 off[kP];
#pragma unroll
    for (int q = 0; q < kP; ++q) {
      off[q] = mul2(a[0][q], inv_own);
      square[q] = fma2(mul2(a[0][q], -1.0f), off[q], square[q]);
      a[0][q] = fma2(first[q], -own_rows, a[0][q]);
    }
    channel_sums<1, kV>(p, a, v0, stage, mean, s.slice);
    if (p.on(v)) {
      f2 m[kP];
      channels_of<kV>(mean + v * kV, m);
#pragma unroll
      for (int q = 0; q < kP; ++q) {
        const f2 d = add2(off[q], mul2(add2(first[q], mul2(m[q], inv_rows)), -1.0f));
        a[0][q] = fma2(mul2(d, own_rows), d, square[q]);
      }
    } else {
#pragma unroll
      for (int q = 0; q < kP; ++q) a[0][q] = 0;
    }
    channel_sums<1, kV>(p, a, v0, stage, m2, s.slice);
  }
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  for (int g = warp; g < groups; g += kThreads / 32) {
    float m = 0.0f;
    for (int c = lane; c < s.per; c += 32) m += mean[g * s.per + c] * inv_rows;
    m = warp_sum(m) / (float)s.per;
    float q = 0.0f;
    for (int c = lane; c < s.per; c += 32) {
      const float d = mean[g * s.per + c] * inv_rows - m;
      q += m2[g * s.per + c] + (float)rows * d * d;
    }
    q = warp_sum(q);
    if (lane == 0) { gmean[g] = m; gm2[g] = q; }
  }
  if (s.split > 1) cluster.sync(); else __syncthreads();
  // every channel's thread joins its group's statistics of all CTAs
  for (int c = threadIdx.x; c < s.slice; c += kThreads) {
    const int g = c / s.per;
    float m = gmean[g], q = gm2[g];
    if (s.split > 1) {
      float part[8];
      m = q = 0.0f;
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < s.split) {
          part[r] = cluster.map_shared_rank(gmean, r)[g];
          m += part[r] * (float)(s.rows * (r + 1) / s.split - s.rows * r / s.split);
        }
      m /= (float)s.rows;
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < s.split) {
          const float n = (float)(s.rows * (r + 1) / s.split - s.rows * r / s.split) * (float)s.per, d = part[r] - m;
          q += cluster.map_shared_rank(gm2, r)[g] + n * d * d;
        }
    }
    const float rstd = rsqrtf(q / ((float)s.rows * (float)s.per) + s.eps);
    if (unit.rank == 0 && stats != nullptr && c == g * s.per) {
      const int64_t at = unit.sample * (s.channels / s.per) + unit.c0 / s.per + g;
      stats[2 * at] = m;
      stats[2 * at + 1] = rstd;
    }
    mean[c] = -m;
    m2[c] = rstd * gamma[unit.c0 + c];
    shift[c] = beta[unit.c0 + c];
  }
  if (s.split > 1) cluster.barrier_arrive();      // done with the others' sums
  __syncthreads();
  for (int v = p.vec; p.on(v); v += p.wide) {
    f2 m[kP], k[kP], b[kP];
    channels_of<kV>(mean + v * kV, m);
    channels_of<kV>(m2 + v * kV, k);
    channels_of<kV>(shift + v * kV, b);
    in.template each<2, kAdd>(p, v, residual + unit.base, [&](const Pack<T, kV>(&raw)[1], const Pack<T, kV>& more, int64_t o) {
      f2 f[kP], e[kP];
      unpack2<T, kV>(raw[0], f);
      if constexpr (kAdd) unpack2<T, kV>(more, e);
#pragma unroll
      for (int q = 0; q < kP; ++q) {
        f2 pre = fma2(add2(f[q], m[q]), k[q], b[q]);
        if constexpr (kAdd) pre = add2(pre, e[q]);
        f[q] = activate2<kAct>(pre);
      }
      store2<T, kV>(z + unit.base + o, f);
    });
  }
  if (s.split > 1) cluster.barrier_wait();        // nobody leaves while its sums are being read
}

// sums [samples][2][C]: what a sample adds to dbeta and dgamma.
template <class T, int kV, int kAct, bool kAdd>
__global__ void __launch_bounds__(kThreads, 2)
group_norm_bwd_kernel(const T* __restrict__ x, const T* __restrict__ residual, const T* __restrict__ dz, T* __restrict__ dx,
                      T* __restrict__ dres, const float* __restrict__ gamma, const float* __restrict__ beta,
                      const float* __restrict__ stats, float* __restrict__ sums, Shape s) {
  pdl_enter();
  extern __shared__ float4 smem4[];
  const int groups = s.slice / s.per;
  T* held = reinterpret_cast<T*>(smem4);                   // [2][held][slice]: x, dz
  float* stage = reinterpret_cast<float*>(held + 2 * s.held * s.slice);
  float* own = stage + stage_floats(kV, s.slice);          // [2][slice] over this CTA's rows: sum d, sum d n
  float* coef = own + 2 * s.slice;                         // [4][slice]: 1 / deviation, -mean, gamma, beta; then for dx
  float* avg = coef + 4 * s.slice;                         // [groups][2]
  cg::cluster_group cluster = cg::this_cluster();
  const Unit unit(s, s.split > 1 ? (int)cluster.block_rank() : 0);
  const Place<kV> p(s, unit.rank);
  Rows<T, kV, 2> in(held, s);
  in.p[0] = x + unit.base;
  in.p[1] = dz + unit.base;
  constexpr int kP = PairsOf<kV>::n;
  constexpr bool kRead = kAdd && kAct != kActNone;         // the residual moves the activation's slope
  const uint64_t policy = l2_policy(s);
  in.ask<true>(p, policy);
  const float* st = stats + 2 * (unit.sample * (s.channels / s.per) + unit.c0 / s.per);
  for (int c = threadIdx.x; c < s.slice; c += kThreads) {
    const int g = c / s.per;
    coef[c] = st[2 * g + 1];
    coef[s.slice + c] = -st[2 * g];
    coef[2 * s.slice + c] = gamma[unit.c0 + c];
    coef[3 * s.slice + c] = beta[unit.c0 + c];
  }
  __syncthreads();
  // n = (f + c) r, pre = n k + h (+ residual): of a thread's channels
  f2 r_[kP], c_[kP], k[kP], h[kP];
  auto coefficients = [&](int v) {
    channels_of<kV>(coef + v * kV, r_);
    channels_of<kV>(coef + s.slice + v * kV, c_);
    channels_of<kV>(coef + 2 * s.slice + v * kV, k);
    channels_of<kV>(coef + 3 * s.slice + v * kV, h);
  };
  // f: n; d: dz act'(.)
  auto derive = [&](const Pack<T, kV>(&raw)[2], const Pack<T, kV>& more, f2 (&f)[kP], f2 (&d)[kP]) {
    f2 e[kP];
    unpack2<T, kV>(raw[0], f);
    unpack2<T, kV>(raw[1], d);
    if constexpr (kRead) unpack2<T, kV>(more, e);
#pragma unroll
    for (int q = 0; q < kP; ++q) {
      f[q] = mul2(add2(f[q], c_[q]), r_[q]);
      if constexpr (kAct != kActNone) {
        f2 pre = fma2(f[q], k[q], h[q]);
        if constexpr (kRead) pre = add2(pre, e[q]);
        d[q] = mul2(d[q], slope2<kAct>(pre));
      }
    }
  };
  if (p.on(p.vec)) coefficients(p.vec);
  arrived();
  for (int v0 = 0; v0 < p.vectors; v0 += p.wide) {
    const int v = v0 + p.vec;
    f2 a[2][kP] = {};
    if (p.on(v)) {
      if (v0 > 0) coefficients(v);
      in.template each<4, kRead>(p, v, residual + unit.base, [&](const Pack<T, kV>(&raw)[2], const Pack<T, kV>& more, int64_t) {
        f2 f[kP], d[kP];
        derive(raw, more, f, d);
#pragma unroll
        for (int q = 0; q < kP; ++q) { a[0][q] = add2(a[0][q], d[q]); a[1][q] = fma2(d[q], f[q], a[1][q]); }
      });
    }
    channel_sums<2, kV>(p, a, v0, stage, own, s.slice);
  }
  if (s.split > 1) cluster.sync();
  float* sum = stage;                                      // [2][slice] over the sample's, times gamma
  for (int c = threadIdx.x; c < s.slice; c += kThreads) {
    float ta = 0.0f, tb = 0.0f;
    if (s.split > 1) {
      for (int r = 0; r < s.split; ++r) {
        const float* o = cluster.map_shared_rank(own, r);
        ta += o[c];
        tb += o[s.slice + c];
      }
    } else {
      ta = own[c];
      tb = own[s.slice + c];
    }
    if (unit.rank == 0) {
      sums[2 * unit.sample * s.channels + unit.c0 + c] = ta;
      sums[(2 * unit.sample + 1) * s.channels + unit.c0 + c] = tb;
    }
    const float w = coef[2 * s.slice + c];
    sum[c] = ta * w;
    sum[s.slice + c] = tb * w;
  }
  if (s.split > 1) cluster.barrier_arrive();      // done with the others' sums
  __syncthreads();
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const float inv = 1.0f / ((float)s.rows * (float)s.per);
  for (int g = warp; g < groups; g += kThreads / 32) {
    float ta = 0.0f, tb = 0.0f;
    for (int c = lane; c < s.per; c += 32) {
      ta += sum[g * s.per + c];
      tb += sum[s.slice + g * s.per + c];
    }
    ta = warp_sum(ta);
    tb = warp_sum(tb);
    if (lane == 0) { avg[2 * g] = ta * inv; avg[2 * g + 1] = tb * inv; }
  }
  __syncthreads();
  // dx = d gamma r - avg(gamma d) r - n avg(gamma d n) r
  float* last = stage;                                     // [3][slice]
  for (int c = threadIdx.x; c < s.slice; c += kThreads) {
    const int g = c / s.per;
    const float r = coef[c];
    last[c] = coef[2 * s.slice + c] * r;
    last[s.slice + c] = -avg[2 * g] * r;
    last[2 * s.slice + c] = -avg[2 * g + 1] * r;
  }
  __syncthreads();
  for (int v = p.vec; p.on(v); v += p.wide) {
    if (p.vectors > p.wide) coefficients(v);
    f2 kr[kP], a1[kP], a2[kP];
    channels_of<kV>(last + v * kV, kr);
    channels_of<kV>(last + s.slice + v * kV, a1);
    channels_of<kV>(last + 2 * s.slice + v * kV, a2);
    in.template each<4, kRead>(p, v, residual + unit.base, [&](const Pack<T, kV>(&raw)[2], const Pack<T, kV>& more, int64_t o) {
      f2 f[kP], d[kP];
      derive(raw, more, f, d);
#pragma unroll
      for (int q = 0; q < kP; ++q) f[q] = fma2(f[q], a2[q], fma2(d[q], kr[q], a1[q]));
      if (dx != nullptr) leave2<T, kV>(dx + unit.base + o, f, policy);
      if (dres != nullptr) leave2<T, kV>(dres + unit.base + o, d, policy);
    });
  }
  if (s.split > 1) cluster.barrier_wait();        // nobody leaves while its sums are being read
}

// A slice has whole groups and whole vectors, and 128 bytes or more of a row where it can, so that a warp reads whole lines; more where
// a slice of so few pixels is hardly worth a CTA, as long as all SMs have some (256x512x7x7: 27 -> 17 us forward).  A cluster has as
// many CTAs as give three to every two SMs, and up to four so that its rows stay in shared memory, `budget` bytes a CTA for
// `tensors` of them: 128x256x56x56 with residual forward / backward, two rows loaded at a time, 180 / 321 us with two, 161 / 308 with
// four, 181 / 320 with eight.
// False where a slice is too wide.
constexpr int kSmallUnit = 16 * 1024;
constexpr int64_t kPassing = 32 << 20;      // bytes; a backward pass has three to five such tensors, L2 room for four
bool plan(int64_t samples, int64_t rows, int channels, int groups, int v, int size, int tensors, int budget, Shape* s) {
  s->rows = rows;
  s->channels = channels;
  s->per = channels / groups;
  s->slice = 0;
  for (int n = 1; n <= groups && n * s->per <= kMaxSlice; ++n) {
    const int slice = n * s->per;
    if (groups % n || slice % v) continue;
    if (s->slice < 8 * v || (rows * s->slice * size < kSmallUnit && samples * (channels / slice) >= 3 * sm_count())) s->slice = slice;
  }
  if (s->slice == 0) return false;
  const int64_t units = samples * (channels / s->slice), row = (int64_t)s->slice * size * tensors;
  const int lanes = kThreads / (s->slice / v < kThreads ? s->slice / v : kThreads);
  s->split = 1;
  while (s->split < 8 && rows / s->split >= 8 * lanes &&
         (2 * units * s->split < 3 * sm_count() || (s->split < 4 && rows / s->split * row > budget)))
    s->split *= 2;
  const int64_t held = v > 1 ? budget / row : 0, most = (rows + s->split - 1) / s->split;
  s->held = (int)(held < most ? held : most);
  s->passing = (double)samples * (double)rows * channels * size > (double)kPassing;
  return true;
}
// CTAs of a pass; as many as a grid takes.
int64_t ctas(const Shape& s, int64_t samples) { return samples * (s.channels / s.slice) * s.split; }
constexpr int64_t kMostCtas = ((int64_t)1 << 31) - 1;

template <int kCluster, class... K, class... A>
int launch_cluster(void (*kernel)(K...), int64_t units, size_t smem, void* stream, A... args) {
  return launch<kCluster>(kernel, dim3((unsigned)(units * kCluster)), kThreads, smem, stream, args...);
}
template <class... K, class... A>
int launch_split(void (*kernel)(K...), int split, int64_t units, size_t smem, SmemAllowed& allowed, void* stream, A... args) {
  if (smem > 48 * 1024) {
    const int rc = allow_smem(kernel, 227 * 1024, allowed);
    if (rc != 0) return rc;
  }
  switch (split) {
    case 1: return launch_cluster<1>(kernel, units, smem, stream, args...);
    case 2: return launch_cluster<2>(kernel, units, smem, stream, args...);
    case 4: return launch_cluster<4>(kernel, units, smem, stream, args...);
    default: return launch_cluster<8>(kernel, units, smem, stream, args...);
  }
}
// Shared memory of a CTA; the widest slices leave less of it to the rows.
size_t fit(Shape* s, size_t row, size_t fixed) {
  constexpr size_t kMost = 224 * 1024;
  if (s->held * row + fixed > kMost) s->held = (int)((kMost - fixed) / row);
  return s->held * row + fixed;
}
constexpr int kForwardHeld = 45 * 1024, kBackwardHeld = 64 * 1024;
// The plan of a direction with vectors of v elements, or single ones where a slice of whole vectors is too wide.
bool plan_of(bool backward, int64_t samples, int64_t rows, int channels, int groups, int* v, int size, Shape* s) {
  const int tensors = backward ? 2 : 1, budget = backward ? kBackwardHeld : kForwardHeld;
  if (plan(samples, rows, channels, groups, *v, size, tensors, budget, s)) return true;
  *v = 1;
  return plan(samples, rows, channels, groups, *v, size, tensors, budget, s);
}

template <class T, int kV, int kAct, bool kAdd>
int forward(const void* x, const void* residual, void* z, const float* gamma, const float* beta, float* stats, int64_t samples,
            Shape s, void* stream) {
  static SmemAllowed allowed{0};
  const size_t smem = fit(&s, (size_t)s.slice * sizeof(T), sizeof(float) * (kThreads * kV + 3 * s.slice + 4 * (s.slice / s.per)));
  return launch_split(group_norm_fwd_kernel<T, kV, kAct, kAdd>, s.split, samples * (s.channels / s.slice), smem, allowed, stream, (const T*)x,
                      (const T*)residual, (T*)z, gamma, beta, stats, s);
}
template <class T, int kV, int kAct, bool kAdd>
int backward(const void* x, const void* residual, const void* dz, void* dx, void* dres, const float* gamma, const float* beta,
             const float* stats, float* sums, int64_t samples, Shape s, void* stream) {
  static SmemAllowed allowed{0};
  const size_t smem = fit(&s, (size_t)s.slice * sizeof(T) * 2, sizeof(float) * (stage_floats(kV, s.slice) + 6 * s.slice + 2 * (s.slice / s.per)));
  return launch_split(group_norm_bwd_kernel<T, kV, kAct, kAdd>, s.split, samples * (s.channels / s.slice), smem, allowed, stream, (const T*)x,
                      (const T*)residual, (const T*)dz, (T*)dx, (T*)dres, gamma, beta, stats, sums, s);
}

// F<T, kV, kAct, kAdd>(): kV whole vectors where rows and pointers allow them.
#define ESGD_ADD(T, V, ACT, F, ...) (residual != nullptr ? F<T, V, ACT, true>(__VA_ARGS__) : F<T, V, ACT, false>(__VA_ARGS__))
#define ESGD_ACT(T, V, F, ...)                                                                                      \
  (act == kActRelu ? ESGD_ADD(T, V, kActRelu, F, __VA_ARGS__) : act == kActSilu ? ESGD_ADD(T, V, kActSilu, F, __VA_ARGS__) \
                                                                                : ESGD_ADD(T, V, kActNone, F, __VA_ARGS__))
#define ESGD_TYPE(F, ...)                                                                                             \
  (is_bf16 ? (v == 8 ? ESGD_ACT(__nv_bfloat16, 8, F, __VA_ARGS__) : ESGD_ACT(__nv_bfloat16, 1, F, __VA_ARGS__))       \
           : (v == 4 ? ESGD_ACT(float, 4, F, __VA_ARGS__) : ESGD_ACT(float, 1, F, __VA_ARGS__)))

}  // namespace

extern "C" {

// Channels of a group at most: a slice holds a group, kMaxSlice channels.
int esgd_group_norm_max_group() { return kMaxSlice; }

// Whether grids hold so many samples, in both directions and however the tensors lie.
int esgd_group_norm_fits(int64_t samples, int64_t rows, int channels, int groups, int is_bf16) {
  if (samples > kMostCtas) return 0;
  for (int backward = 0; backward < 2; ++backward)
    for (int most : {1, is_bf16 ? 8 : 4}) {
      int v = channels % most ? 1 : most;
      Shape s;
      if (!plan_of(backward, samples, rows, channels, groups, &v, is_bf16 ? 2 : 4, &s) || ctas(s, samples) > kMostCtas) return 0;
    }
  return 1;
}

// x, residual, z [samples][rows][channels]; stats [samples][groups][2] (mean, 1 / deviation), or null.
int esgd_group_norm_fwd(const void* x, const void* residual, void* z, const float* gamma, const float* beta, float* stats, int is_bf16,
                        int64_t samples, int64_t rows, int channels, int groups, int act, float eps, void* stream) {
  if (samples == 0 || rows == 0) return 0;
  int v = is_bf16 ? 8 : 4;
  if (channels % v || !aligned16(x) || !aligned16(z) || !aligned16(residual)) v = 1;
  Shape s;
  if (!plan_of(false, samples, rows, channels, groups, &v, is_bf16 ? 2 : 4, &s) || ctas(s, samples) > kMostCtas) return (int)cudaErrorInvalidValue;
  s.eps = eps;
  return ESGD_TYPE(forward, x, residual, z, gamma, beta, stats, samples, s, stream);
}

// residual: as in the forward pass (it is read where there is an activation).  dx, dres: null where not wanted.
int esgd_group_norm_bwd(const void* x, const void* residual, const void* dz, void* dx, void* dres, const float* gamma, const float* beta,
                        const float* stats, float* sums, int is_bf16, int64_t samples, int64_t rows, int channels, int groups, int act,
                        void* stream) {
  if (samples == 0 || rows == 0) return 0;
  int v = is_bf16 ? 8 : 4;
  if (channels % v || !aligned16(x) || !aligned16(residual) || !aligned16(dz) || !aligned16(dx) || !aligned16(dres)) v = 1;
  Shape s;
  if (!plan_of(true, samples, rows, channels, groups, &v, is_bf16 ? 2 : 4, &s) || ctas(s, samples) > kMostCtas) return (int)cudaErrorInvalidValue;
  s.eps = 0.0f;
  return ESGD_TYPE(backward, x, residual, dz, dx, dres, gamma, beta, stats, sums, samples, s, stream);
}

}  // extern "C"
