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
// A CTA's variance is that about the CTA's own mean of each channel, and CTAs and channels are joined as means and squared
// deviations: with sum and sum of squares a mean of 100 deviations would cost four digits.
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
  float eps;
};

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

// Sums over the CTA's rows of the threads' channels, into out[channel * stride] from channel v0 * kV on.  Every thread calls it.
template <int kV>
__device__ __forceinline__ void channel_sums(const Place<kV>& p, const f2 (&pairs)[PairsOf<kV>::n], int v0, float* stage, float* out, int stride) {
  int partial = p.lanes;
  float a[kV];
#pragma unroll
  for (int q = 0; q < kV; ++q) a[q] = q % 2 == 0 ? halves(pairs[q / 2]).x : halves(pairs[q / 2]).y;
  if (p.fold) {
    partial = kThreads / 32;
    for (int o = p.wide; o < 32; o *= 2)
#pragma unroll
      for (int q = 0; q < kV; ++q) a[q] += __shfl_xor_sync(0xffffffffu, a[q], o);
    if ((threadIdx.x & 31) < p.wide)
#pragma unroll
      for (int q = 0; q < kV; ++q) stage[(threadIdx.x / 32 * p.wide + p.vec) * kV + q] = a[q];
  } else if (p.lane < p.lanes) {
#pragma unroll
    for (int q = 0; q < kV; ++q) stage[threadIdx.x * kV + q] = a[q];
  }
  __syncthreads();
  const int here = min(p.wide, p.vectors - v0) * kV;
  for (int c = threadIdx.x; c < here; c += kThreads) {
    float t = 0.0f;
    for (int r = 0; r < partial; ++r) t += stage[r * p.wide * kV + c];
    out[(v0 * kV + c) * stride] = t;
  }
  __syncthreads();
}

// Rows of one tensor: the first `held` of a CTA in shared memory, each thread's own vectors, the others where they are.
template <class T, int kV> struct Rows {
  const T* p;          // the CTA's first row and the slice's first channel
  T* in;               // [held][slice]
  int held, slice;
  int64_t pitch;
  __device__ Rows(const T* p_, T* in_, const Shape& s) : p(p_), in(in_), held(s.held), slice(s.slice), pitch(s.channels) {}
  __device__ __forceinline__ void ask(const Place<kV>& pl) const {
    if constexpr (kV > 1) {
      const int n = held < pl.rows ? held : pl.rows;
      for (int v = pl.vec; pl.on(v); v += pl.wide) {
        const T* from = p + pl.lane * pitch + v * kV;
        uint32_t to = (uint32_t)__cvta_generic_to_shared(in + pl.lane * slice + v * kV);
        for (int r = pl.lane; r < n; r += pl.lanes) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
          from += pl.lanes * pitch;
          to += pl.lanes * slice * (int)sizeof(T);
        }
      }
    }
  }
  __device__ __forceinline__ Pack<T, kV> row(int r, int v) const {
    if (kV > 1 && r < held) return load<T, kV>(in + r * slice + v * kV);
    return load<T, kV>(p + r * pitch + v * kV);
  }
};
// f(row, of which u-th of kMany at a time): loads first, then what is done with them.
template <int kMany, class Load, class Use> __device__ __forceinline__ void over_rows(int first, int step, int rows, Load load_row, Use use_row) {
  int r = first;
  for (; r + (kMany - 1) * step < rows; r += kMany * step) {
#pragma unroll
    for (int u = 0; u < kMany; ++u) load_row(r + u * step, u);
#pragma unroll
    for (int u = 0; u < kMany; ++u) use_row(r + u * step, u);
  }
  for (; r < rows; r += step) {
    load_row(r, 0);
    use_row(r, 0);
  }
}
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
__global__ void __launch_bounds__(kThreads, 3)
group_norm_fwd_kernel(const T* __restrict__ x, const T* __restrict__ residual, T* __restrict__ z, const float* __restrict__ gamma,
                      const float* __restrict__ beta, float* __restrict__ stats, Shape s) {
  pdl_enter();
  extern __shared__ float4 smem4[];
  const int groups = s.slice / s.per;
  T* held = reinterpret_cast<T*>(smem4);                   // [held][slice]
  float* stage = reinterpret_cast<float*>(held + s.held * s.slice);
  float* mean = stage + kThreads * kV;                     // [slice]
  float* m2 = mean + s.slice;
  float* gmean = m2 + s.slice;                             // [groups] of this CTA's rows
  float* gm2 = gmean + groups;
  float* scale = gm2 + groups;                             // [groups] of the sample: 1 / deviation, mean
  float* centre = scale + groups;
  cg::cluster_group cluster = cg::this_cluster();
  const Unit unit(s, s.split > 1 ? (int)cluster.block_rank() : 0);
  const Place<kV> p(s, unit.rank);
  const Rows<T, kV> in(x + unit.base, held, s);
  constexpr int kP = PairsOf<kV>::n;
  const int rows = p.rows;
  in.ask(p);
  arrived();
  const float inv_rows = rows > 0 ? 1.0f / (float)rows : 0.0f;
  for (int v0 = 0; v0 < p.vectors; v0 += p.wide) {
    const int v = v0 + p.vec;
    f2 a[kP] = {};
    Pack<T, kV> raw[4];
    if (p.on(v))
      over_rows<4>(p.lane, p.lanes, rows, [&](int r, int u) { raw[u] = in.row(r, v); }, [&](int, int u) {
        f2 f[kP];
        unpack2<T, kV>(raw[u], f);
#pragma unroll
        for (int q = 0; q < kP; ++q) a[q] = add2(a[q], f[q]);
      });
    channel_sums<kV>(p, a, v0, stage, mean, 1);
  }
  for (int v0 = 0; v0 < p.vectors; v0 += p.wide) {
    const int v = v0 + p.vec;
    f2 a[kP] = {}, m[kP];
    Pack<T, kV> raw[4];
    if (p.on(v)) {
#pragma unroll
      for (int q = 0; q < kP; ++q) m[q] = pair(-mean[v * kV + 2 * q] * inv_rows, kV > 1 ? -mean[v * kV + 2 * q + 1] * inv_rows : 0.0f);
      over_rows<4>(p.lane, p.lanes, rows, [&](int r, int u) { raw[u] = in.row(r, v); }, [&](int, int u) {
        f2 f[kP];
        unpack2<T, kV>(raw[u], f);
#pragma unroll
        for (int q = 0; q < kP; ++q) {
          const f2 d = add2(f[q], m[q]);
          a[q] = fma2(d, d, a[q]);
        }
      });
    }
    channel_sums<kV>(p, a, v0, stage, m2, 1);
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
  for (int g = threadIdx.x; g < groups; g += kThreads) {
    float m = 0.0f, q = 0.0f;
    if (s.split > 1) {
      float part[8];
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
    } else {
      m = gmean[g];
      q = gm2[g];
    }
    const float rstd = rsqrtf(q / ((float)s.rows * (float)s.per) + s.eps);
    scale[g] = rstd;
    centre[g] = m;
    if (unit.rank == 0 && stats != nullptr) {
      const int64_t at = unit.sample * (s.channels / s.per) + unit.c0 / s.per + g;
      stats[2 * at] = m;
      stats[2 * at + 1] = rstd;
    }
  }
  __syncthreads();
  for (int v = p.vec; p.on(v); v += p.wide) {
    f2 m[kP], k[kP], b[kP];
    float f[3][kV];
#pragma unroll
    for (int q = 0; q < kV; ++q) {
      const int c = v * kV + q, g = c / s.per;
      f[0][q] = -centre[g];
      f[1][q] = scale[g] * gamma[unit.c0 + c];
      f[2][q] = beta[unit.c0 + c];
    }
#pragma unroll
    for (int q = 0; q < kP; ++q) {
      m[q] = pair(f[0][2 * q], f[0][(2 * q + 1) % kV]);
      k[q] = pair(f[1][2 * q], f[1][(2 * q + 1) % kV]);
      b[q] = pair(f[2][2 * q], f[2][(2 * q + 1) % kV]);
    }
    const int64_t at = unit.base + v * kV;
    Pack<T, kV> raw[4], add[4];
    over_rows<4>(p.lane, p.lanes, rows, [&](int r, int u) {
      if constexpr (kAdd) add[u] = load<T, kV>(residual + at + r * in.pitch);
      raw[u] = in.row(r, v);
    }, [&](int r, int u) {
      f2 f[kP], e[kP];
      unpack2<T, kV>(raw[u], f);
      if constexpr (kAdd) unpack2<T, kV>(add[u], e);
#pragma unroll
      for (int q = 0; q < kP; ++q) {
        f2 pre = fma2(add2(f[q], m[q]), k[q], b[q]);
        if constexpr (kAdd) pre = add2(pre, e[q]);
        f[q] = activate2<kAct>(pre);
      }
      store2<T, kV>(z + at + r * in.pitch, f);
    });
  }
  if (s.split > 1) cluster.sync();       // nobody leaves while its sums are being read
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
  float* own = stage + kThreads * kV;                      // [slice][2] over this CTA's rows
  float* all = own + 2 * s.slice;                          // [slice][2] over the sample's
  float* avg = all + 2 * s.slice;                          // [groups][2]
  cg::cluster_group cluster = cg::this_cluster();
  const Unit unit(s, s.split > 1 ? (int)cluster.block_rank() : 0);
  const Place<kV> p(s, unit.rank);
  const Rows<T, kV> in(x + unit.base, held, s), up(dz + unit.base, held + s.held * s.slice, s);
  constexpr int kP = PairsOf<kV>::n;
  constexpr bool kRead = kAdd && kAct != kActNone;         // the residual moves the activation's slope
  const int rows = p.rows;
  in.ask(p);
  up.ask(p);
  const float* st = stats + 2 * (unit.sample * (s.channels / s.per) + unit.c0 / s.per);
  // n = (f + c) r, pre = n k + h (+ residual): of a thread's channels
  f2 r_[kP], c_[kP], k[kP], h[kP];
  auto coefficients = [&](int v) {
    float f[4][kV];
#pragma unroll
    for (int q = 0; q < kV; ++q) {
      const int c = v * kV + q, g = c / s.per;
      f[0][q] = st[2 * g + 1];
      f[1][q] = -st[2 * g];
      f[2][q] = gamma[unit.c0 + c];
      f[3][q] = beta[unit.c0 + c];
    }
#pragma unroll
    for (int q = 0; q < kP; ++q) {
      r_[q] = pair(f[0][2 * q], f[0][(2 * q + 1) % kV]);
      c_[q] = pair(f[1][2 * q], f[1][(2 * q + 1) % kV]);
      k[q] = pair(f[2][2 * q], f[2][(2 * q + 1) % kV]);
      h[q] = pair(f[3][2 * q], f[3][(2 * q + 1) % kV]);
    }
  };
  // f: n; d: dz act'(.)
  auto derive = [&](const Pack<T, kV>& rx, const Pack<T, kV>& rd, const Pack<T, kV>& rr, f2 (&f)[kP], f2 (&d)[kP]) {
    f2 e[kP];
    unpack2<T, kV>(rx, f);
    unpack2<T, kV>(rd, d);
    if constexpr (kRead) unpack2<T, kV>(rr, e);
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
  Pack<T, kV> rx[2], rd[2], rr[2];
  for (int v0 = 0; v0 < p.vectors; v0 += p.wide) {
    const int v = v0 + p.vec;
    f2 a[kP] = {}, b[kP] = {};
    if (p.on(v)) {
      if (v0 > 0) coefficients(v);
      const T* more = residual + unit.base + v * kV;
      over_rows<2>(p.lane, p.lanes, rows, [&](int r, int u) {
        if constexpr (kRead) rr[u] = load<T, kV>(more + r * in.pitch);
        rx[u] = in.row(r, v);
        rd[u] = up.row(r, v);
      }, [&](int, int u) {
        f2 f[kP], d[kP];
        derive(rx[u], rd[u], rr[u], f, d);
#pragma unroll
        for (int q = 0; q < kP; ++q) { a[q] = add2(a[q], d[q]); b[q] = fma2(d[q], f[q], b[q]); }
      });
    }
    channel_sums<kV>(p, a, v0, stage, own, 2);
    channel_sums<kV>(p, b, v0, stage, own + 1, 2);
  }
  if (s.split > 1) cluster.sync();
  for (int c = threadIdx.x; c < s.slice; c += kThreads) {
    float ta = 0.0f, tb = 0.0f;
    if (s.split > 1) {
      for (int r = 0; r < s.split; ++r) {
        const float2 o = reinterpret_cast<const float2*>(cluster.map_shared_rank(own, r))[c];
        ta += o.x;
        tb += o.y;
      }
    } else {
      ta = own[2 * c];
      tb = own[2 * c + 1];
    }
    if (unit.rank == 0) {
      sums[2 * unit.sample * s.channels + unit.c0 + c] = ta;
      sums[(2 * unit.sample + 1) * s.channels + unit.c0 + c] = tb;
    }
    all[2 * c] = ta * gamma[unit.c0 + c];
    all[2 * c + 1] = tb * gamma[unit.c0 + c];
  }
  __syncthreads();
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const float inv = 1.0f / ((float)s.rows * (float)s.per);
  for (int g = warp; g < groups; g += kThreads / 32) {
    float ta = 0.0f, tb = 0.0f;
    for (int c = lane; c < s.per; c += 32) {
      ta += all[2 * (g * s.per + c)];
      tb += all[2 * (g * s.per + c) + 1];
    }
    ta = warp_sum(ta);
    tb = warp_sum(tb);
    if (lane == 0) { avg[2 * g] = ta * inv; avg[2 * g + 1] = tb * inv; }
  }
  __syncthreads();
  for (int v = p.vec; p.on(v); v += p.wide) {
    if (p.vectors > p.wide) coefficients(v);
    // dx = d k r - avg(k d) r - n avg(k d n) r
    f2 kr[kP], a1[kP], a2[kP];
#pragma unroll
    for (int q = 0; q < kP; ++q) {
      const int g = (v * kV + 2 * q) / s.per, g2 = (v * kV + (2 * q + 1) % kV) / s.per;
      kr[q] = mul2(k[q], r_[q]);
      a1[q] = mul2(pair(-avg[2 * g], -avg[2 * g2]), r_[q]);
      a2[q] = mul2(pair(-avg[2 * g + 1], -avg[2 * g2 + 1]), r_[q]);
    }
    const int64_t at = unit.base + v * kV;
    over_rows<2>(p.lane, p.lanes, rows, [&](int r, int u) {
      if constexpr (kRead) rr[u] = load<T, kV>(residual + at + r * in.pitch);
      rx[u] = in.row(r, v);
      rd[u] = up.row(r, v);
    }, [&](int r, int u) {
      f2 f[kP], d[kP];
      derive(rx[u], rd[u], rr[u], f, d);
#pragma unroll
      for (int q = 0; q < kP; ++q) f[q] = fma2(f[q], a2[q], fma2(d[q], kr[q], a1[q]));
      if (dx != nullptr) store2<T, kV>(dx + at + r * in.pitch, f);
      if (dres != nullptr) store2<T, kV>(dres + at + r * in.pitch, d);
    });
  }
  if (s.split > 1) cluster.sync();
}

// A slice has whole groups and whole vectors, and 128 bytes or more of a row where it can, so that a warp reads whole lines (more where
// a slice of so few pixels is hardly worth a CTA, as long as all SMs have some); a cluster has as many CTAs as keep two of them busy on every SM with eight rows a thread or more, and its rows in shared memory:
// `budget` bytes a CTA for `tensors` of them.  False where a slice is too wide.
constexpr int kSmallUnit = 16 * 1024;
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
  while (s->split < 8 && rows / s->split >= 8 * lanes && (units * s->split < 2 * sm_count() || rows / s->split * row > budget)) s->split *= 2;
  const int64_t held = v > 1 ? budget / row : 0, most = (rows + s->split - 1) / s->split;
  s->held = (int)(held < most ? held : most);
  return true;
}

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
constexpr int kForwardHeld = 56 * 1024, kBackwardHeld = 100 * 1024;

template <class T, int kV, int kAct, bool kAdd>
int forward(const void* x, const void* residual, void* z, const float* gamma, const float* beta, float* stats, int64_t samples,
            const Shape& s, void* stream) {
  static SmemAllowed allowed{0};
  const size_t smem = (size_t)s.held * s.slice * sizeof(T) + sizeof(float) * (kThreads * kV + 2 * s.slice + 4 * (s.slice / s.per));
  return launch_split(group_norm_fwd_kernel<T, kV, kAct, kAdd>, s.split, samples * (s.channels / s.slice), smem, allowed, stream, (const T*)x,
                      (const T*)residual, (T*)z, gamma, beta, stats, s);
}
template <class T, int kV, int kAct, bool kAdd>
int backward(const void* x, const void* residual, const void* dz, void* dx, void* dres, const float* gamma, const float* beta,
             const float* stats, float* sums, int64_t samples, const Shape& s, void* stream) {
  static SmemAllowed allowed{0};
  const size_t smem = (size_t)s.held * s.slice * sizeof(T) * 2 + sizeof(float) * (kThreads * kV + 4 * s.slice + 2 * (s.slice / s.per));
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

// x, residual, z [samples][rows][channels]; stats [samples][groups][2] (mean, 1 / deviation), or null.
int esgd_group_norm_fwd(const void* x, const void* residual, void* z, const float* gamma, const float* beta, float* stats, int is_bf16,
                        int64_t samples, int64_t rows, int channels, int groups, int act, float eps, void* stream) {
  if (samples == 0 || rows == 0) return 0;
  int v = is_bf16 ? 8 : 4;
  if (channels % v || !aligned16(x) || !aligned16(z) || !aligned16(residual)) v = 1;
  Shape s;
  if (!plan(samples, rows, channels, groups, v, is_bf16 ? 2 : 4, 1, kForwardHeld, &s)) {
    v = 1;
    if (!plan(samples, rows, channels, groups, v, is_bf16 ? 2 : 4, 1, kForwardHeld, &s)) return (int)cudaErrorInvalidValue;
  }
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
  if (!plan(samples, rows, channels, groups, v, is_bf16 ? 2 : 4, 2, kBackwardHeld, &s)) {
    v = 1;
    if (!plan(samples, rows, channels, groups, v, is_bf16 ? 2 : 4, 2, kBackwardHeld, &s)) return (int)cudaErrorInvalidValue;
  }
  s.eps = 0.0f;
  return ESGD_TYPE(backward, x, residual, dz, dx, dres, gamma, beta, stats, sums, samples, s, stream);
}

}  // extern "C"
