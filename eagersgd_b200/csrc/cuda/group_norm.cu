// Group norm (+ residual) (+ activation) of channels-last activations, forward and backward.
//
//   mean, var over a sample's pixels and a group's C / G channels;   n = (x - mean) / sqrt(var + eps)
//   z  = act(gamma n + beta [+ residual])
//   d  = dz act'(.);  dgamma = sum d n,  dbeta = sum d,  dresidual = d
//   dx = (gamma d - avg(gamma d) - n avg(gamma d n)) / sqrt(var + eps)      averages over the group
//
// Bound by memory: x (and residual) in, z out; x, dz (and residual) in, dx (and dresidual) out.  A cluster of CTAs has a sample's
// slice of whole groups, the rows (pixels) split among its CTAs; the sums of the CTAs meet in distributed shared memory, so that
// one launch does statistics and result.  The second pass over the rows finds them in L2: what the resident clusters work on at a
// time is a fraction of it.
//
// The statistics are taken about a value of the data itself (a thread's first row), and thread, row and CTA statistics are joined
// as means and squared deviations: with sum and sum of squares a mean of 100 deviations would cost four digits.
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
  float eps;
};

// Where a thread works: a vector of kV channels, every `lanes`-th row of its CTA's.
template <int kV> struct Place {
  int wide, lanes, lane, vec;
  int64_t first, last;
  __device__ Place(const Shape& s, int rank) {
    const int vectors = s.slice / kV;
    wide = min(vectors, kThreads);
    lanes = kThreads / wide;
    lane = threadIdx.x / wide;
    vec = threadIdx.x - lane * wide;
    first = s.rows * rank / s.split;
    last = s.rows * (rank + 1) / s.split;
  }
};

// Sum over a warp.
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The CTA's statistics of each channel of the slice (over its rows) into mean[], m2[].
template <class T, int kV>
__device__ void channel_stats(const T* x, const Shape& s, const Place<kV>& p, float* stage, float* mean, float* m2) {
  const int vectors = s.slice / kV;
  const int64_t rows = p.last - p.first;
  for (int v0 = 0; v0 < vectors; v0 += p.wide) {
    const int v = v0 + p.vec;
    const bool on = p.lane < p.lanes && v < vectors;
    const int64_t n = on && rows > p.lane ? (rows - p.lane + p.lanes - 1) / p.lanes : 0;
    float shift[kV], a[kV], b[kV];
#pragma unroll
    for (int q = 0; q < kV; ++q) shift[q] = a[q] = b[q] = 0.0f;
    if (n > 0) {
      const T* at = x + (p.first + p.lane) * s.channels + v * kV;
      const int64_t step = (int64_t)p.lanes * s.channels;
      unpack<T, kV>(load<T, kV>(at), shift);
      for (int64_t i = 1; i < n; i += 4) {
        Pack<T, kV> raw[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (i + k < n) raw[k] = load<T, kV>(at + (i + k) * step);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (i + k >= n) break;
          float f[kV];
          unpack<T, kV>(raw[k], f);
#pragma unroll
          for (int q = 0; q < kV; ++q) {
            const float d = f[q] - shift[q];
            a[q] += d;
            b[q] = fmaf(d, d, b[q]);
          }
        }
      }
    }
    const float inv = n > 0 ? 1.0f / (float)n : 0.0f;
#pragma unroll
    for (int q = 0; q < kV; ++q) {
      stage[threadIdx.x * kV + q] = shift[q] + a[q] * inv;
      stage[kThreads * kV + threadIdx.x * kV + q] = fmaxf(b[q] - a[q] * a[q] * inv, 0.0f);
    }
    __syncthreads();
    const int here = min(p.wide, vectors - v0) * kV;
    for (int c = threadIdx.x; c < here; c += kThreads) {
      float m = 0.0f;
      for (int r = 0; r < p.lanes; ++r) {
        const int64_t k = rows > r ? (rows - r + p.lanes - 1) / p.lanes : 0;
        m += (float)k * stage[r * p.wide * kV + c];
      }
      m = rows > 0 ? m / (float)rows : 0.0f;
      float sq = 0.0f;
      for (int r = 0; r < p.lanes; ++r) {
        const int64_t k = rows > r ? (rows - r + p.lanes - 1) / p.lanes : 0;
        const float d = stage[r * p.wide * kV + c] - m;
        if (k > 0) sq += stage[kThreads * kV + r * p.wide * kV + c] + (float)k * d * d;
      }
      mean[v0 * kV + c] = m;
      m2[v0 * kV + c] = sq;
    }
    __syncthreads();
  }
}

template <class T, int kV, int kAct>
__global__ void __launch_bounds__(kThreads, 3)
group_norm_fwd_kernel(const T* __restrict__ x, const T* __restrict__ residual, T* __restrict__ z, const float* __restrict__ gamma,
                      const float* __restrict__ beta, float* __restrict__ stats, Shape s) {
  pdl_enter();
  extern __shared__ float smem[];
  float* stage = smem;                               // [2][kThreads * kV]
  float* mean = stage + 2 * kThreads * kV;           // [slice]
  float* m2 = mean + s.slice;
  const int groups = s.slice / s.per;
  float* gmean = m2 + s.slice;                       // [groups] of this CTA's rows
  float* gm2 = gmean + groups;
  float* scale = gm2 + groups;                       // [groups] of the sample: 1 / deviation, mean
  float* centre = scale + groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = s.split > 1 ? (int)cluster.block_rank() : 0;
  const int slices = s.channels / s.slice;
  const int64_t unit = blockIdx.x / s.split;
  const int64_t sample = unit / slices;
  const int c0 = (int)(unit - sample * slices) * s.slice;
  const int64_t base = sample * s.rows * s.channels + c0;
  const Place<kV> p(s, rank);
  channel_stats<T, kV>(x + base, s, p, stage, mean, m2);
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int64_t rows = p.last - p.first;
  for (int g = warp; g < groups; g += kThreads / 32) {
    float m = 0.0f;
    for (int c = lane; c < s.per; c += 32) m += mean[g * s.per + c];
    m = warp_sum(m) / (float)s.per;
    float q = 0.0f;
    for (int c = lane; c < s.per; c += 32) {
      const float d = mean[g * s.per + c] - m;
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
    if (rank == 0 && stats != nullptr) {
      const int64_t at = sample * (s.channels / s.per) + c0 / s.per + g;
      stats[2 * at] = m;
      stats[2 * at + 1] = rstd;
    }
  }
  __syncthreads();
  const int vectors = s.slice / kV;
  for (int v = p.vec; v < vectors && p.lane < p.lanes; v += p.wide) {
    float m[kV], k[kV], b[kV];
#pragma unroll
    for (int q = 0; q < kV; ++q) {
      const int c = v * kV + q, g = c / s.per;
      m[q] = centre[g];
      k[q] = scale[g] * gamma[c0 + c];
      b[q] = beta[c0 + c];
    }
    for (int64_t r = p.first + p.lane; r < p.last; r += 4 * p.lanes) {
      Pack<T, kV> raw[4], add[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (r + u * p.lanes < p.last) {
          const int64_t at = base + (r + u * p.lanes) * s.channels + v * kV;
          raw[u] = load<T, kV>(x + at);
          if (residual != nullptr) add[u] = load<T, kV>(residual + at);
        }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (r + u * p.lanes >= p.last) break;
        float f[kV], e[kV];
        unpack<T, kV>(raw[u], f);
        if (residual != nullptr) unpack<T, kV>(add[u], e);
#pragma unroll
        for (int q = 0; q < kV; ++q) {
          float pre = fmaf(f[q] - m[q], k[q], b[q]);
          if (residual != nullptr) pre += e[q];
          f[q] = activate<kAct>(pre);
        }
        store<T, kV>(z + base + (r + u * p.lanes) * s.channels + v * kV, f);
      }
    }
  }
  if (s.split > 1) cluster.sync();       // nobody leaves while its sums are being read
}

// sums [samples][2][C]: what a sample adds to dbeta and dgamma.
template <class T, int kV, int kAct>
__global__ void __launch_bounds__(kThreads, 2)
group_norm_bwd_kernel(const T* __restrict__ x, const T* __restrict__ residual, const T* __restrict__ dz, T* __restrict__ dx,
                      T* __restrict__ dres, const float* __restrict__ gamma, const float* __restrict__ beta,
                      const float* __restrict__ stats, float* __restrict__ sums, Shape s) {
  pdl_enter();
  extern __shared__ float smem[];
  float* stage = smem;                               // [2][kThreads * kV]
  float* own = stage + 2 * kThreads * kV;            // [slice][2] over this CTA's rows
  float* all = own + 2 * s.slice;                    // [slice][2] over the sample's
  const int groups = s.slice / s.per;
  float* avg = all + 2 * s.slice;                    // [groups][2]
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = s.split > 1 ? (int)cluster.block_rank() : 0;
  const int slices = s.channels / s.slice;
  const int64_t unit = blockIdx.x / s.split;
  const int64_t sample = unit / slices;
  const int c0 = (int)(unit - sample * slices) * s.slice;
  const int64_t base = sample * s.rows * s.channels + c0;
  const float* st = stats + 2 * (sample * (s.channels / s.per) + c0 / s.per);
  const Place<kV> p(s, rank);
  const int vectors = s.slice / kV;
  for (int v0 = 0; v0 < vectors; v0 += p.wide) {
    const int v = v0 + p.vec;
    float a[kV], b[kV];
#pragma unroll
    for (int q = 0; q < kV; ++q) a[q] = b[q] = 0.0f;
    if (p.lane < p.lanes && v < vectors) {
      float m[kV], r_[kV], k[kV], sh[kV];
#pragma unroll
      for (int q = 0; q < kV; ++q) {
        const int c = v * kV + q, g = c / s.per;
        m[q] = st[2 * g];
        r_[q] = st[2 * g + 1];
        k[q] = gamma[c0 + c];
        sh[q] = beta[c0 + c];
      }
      for (int64_t r = p.first + p.lane; r < p.last; r += 2 * p.lanes) {
        Pack<T, kV> rx[2], rd[2], rr[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (r + u * p.lanes < p.last) {
            const int64_t at = base + (r + u * p.lanes) * s.channels + v * kV;
            rx[u] = load<T, kV>(x + at);
            rd[u] = load<T, kV>(dz + at);
            if (kAct != kActNone && residual != nullptr) rr[u] = load<T, kV>(residual + at);
          }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (r + u * p.lanes >= p.last) break;
          float f[kV], d[kV], e[kV];
          unpack<T, kV>(rx[u], f);
          unpack<T, kV>(rd[u], d);
          if (kAct != kActNone && residual != nullptr) unpack<T, kV>(rr[u], e);
#pragma unroll
          for (int q = 0; q < kV; ++q) {
            const float n = (f[q] - m[q]) * r_[q];
            float g = d[q];
            if constexpr (kAct != kActNone) g *= slope<kAct>(fmaf(n, k[q], sh[q]) + (residual != nullptr ? e[q] : 0.0f));
            a[q] += g;
            b[q] = fmaf(g, n, b[q]);
          }
        }
      }
    }
#pragma unroll
    for (int q = 0; q < kV; ++q) {
      stage[threadIdx.x * kV + q] = a[q];
      stage[kThreads * kV + threadIdx.x * kV + q] = b[q];
    }
    __syncthreads();
    const int here = min(p.wide, vectors - v0) * kV;
    for (int c = threadIdx.x; c < here; c += kThreads) {
      float ta = 0.0f, tb = 0.0f;
      for (int r = 0; r < p.lanes; ++r) {
        ta += stage[r * p.wide * kV + c];
        tb += stage[kThreads * kV + r * p.wide * kV + c];
      }
      own[2 * (v0 * kV + c)] = ta;
      own[2 * (v0 * kV + c) + 1] = tb;
    }
    __syncthreads();
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
    if (rank == 0) {
      sums[2 * sample * s.channels + c0 + c] = ta;
      sums[(2 * sample + 1) * s.channels + c0 + c] = tb;
    }
    all[2 * c] = ta * gamma[c0 + c];
    all[2 * c + 1] = tb * gamma[c0 + c];
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
  for (int v = p.vec; v < vectors && p.lane < p.lanes; v += p.wide) {
    float m[kV], r_[kV], k[kV], sh[kV], a1[kV], a2[kV];
#pragma unroll
    for (int q = 0; q < kV; ++q) {
      const int c = v * kV + q, g = c / s.per;
      m[q] = st[2 * g];
      r_[q] = st[2 * g + 1];
      k[q] = gamma[c0 + c];
      sh[q] = beta[c0 + c];
      a1[q] = avg[2 * g];
      a2[q] = avg[2 * g + 1];
    }
    for (int64_t r = p.first + p.lane; r < p.last; r += 2 * p.lanes) {
      Pack<T, kV> rx[2], rd[2], rr[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (r + u * p.lanes < p.last) {
          const int64_t at = base + (r + u * p.lanes) * s.channels + v * kV;
          rx[u] = load<T, kV>(x + at);
          rd[u] = load<T, kV>(dz + at);
          if (kAct != kActNone && residual != nullptr) rr[u] = load<T, kV>(residual + at);
        }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (r + u * p.lanes >= p.last) break;
        const int64_t at = base + (r + u * p.lanes) * s.channels + v * kV;
        float f[kV], d[kV], e[kV];
        unpack<T, kV>(rx[u], f);
        unpack<T, kV>(rd[u], d);
        if (kAct != kActNone && residual != nullptr) unpack<T, kV>(rr[u], e);
#pragma unroll
        for (int q = 0; q < kV; ++q) {
          const float n = (f[q] - m[q]) * r_[q];
          float g = d[q];
          if constexpr (kAct != kActNone) g *= slope<kAct>(fmaf(n, k[q], sh[q]) + (residual != nullptr ? e[q] : 0.0f));
          d[q] = g;
          f[q] = (g * k[q] - a1[q] - n * a2[q]) * r_[q];
        }
        if (dx != nullptr) store<T, kV>(dx + at, f);
        if (dres != nullptr) store<T, kV>(dres + at, d);
      }
    }
  }
  if (s.split > 1) cluster.sync();
}

// A slice has whole groups and whole vectors, and 128 bytes or more of a row where it can, so that a warp reads whole lines; a
// cluster has as many CTAs as keep two of them busy on every SM with eight rows a thread or more.  False where a slice is too wide.
bool plan(int64_t samples, int64_t rows, int channels, int groups, int v, Shape* s) {
  s->rows = rows;
  s->channels = channels;
  s->per = channels / groups;
  s->slice = 0;
  for (int n = 1; n <= groups && n * s->per <= kMaxSlice; ++n) {
    if (groups % n || (n * s->per) % v) continue;
    s->slice = n * s->per;
    if (s->slice >= 8 * v) break;
  }
  if (s->slice == 0) return false;
  const int64_t units = samples * (channels / s->slice);
  const int lanes = kThreads / (s->slice / v < kThreads ? s->slice / v : kThreads);
  s->split = 1;
  while (s->split < 8 && rows / s->split >= 8 * lanes && (units * s->split < 2 * sm_count() || rows / s->split > 32 * lanes)) s->split *= 2;
  return true;
}

template <int kCluster, class... K, class... A>
int launch_cluster(void (*kernel)(K...), int64_t units, size_t smem, void* stream, A... args) {
  return launch<kCluster>(kernel, dim3((unsigned)(units * kCluster)), kThreads, smem, stream, args...);
}
template <class... K, class... A>
int launch_split(void (*kernel)(K...), int split, int64_t units, size_t smem, SmemAllowed& allowed, void* stream, A... args) {
  if (smem > 48 * 1024) {
    const int rc = allow_smem(kernel, 200 * 1024, allowed);
    if (rc != 0) return rc;
  }
  switch (split) {
    case 1: return launch_cluster<1>(kernel, units, smem, stream, args...);
    case 2: return launch_cluster<2>(kernel, units, smem, stream, args...);
    case 4: return launch_cluster<4>(kernel, units, smem, stream, args...);
    default: return launch_cluster<8>(kernel, units, smem, stream, args...);
  }
}

template <class T, int kV, int kAct>
int forward(const void* x, const void* residual, void* z, const float* gamma, const float* beta, float* stats, int64_t samples,
            const Shape& s, void* stream) {
  static SmemAllowed allowed{0};
  const size_t smem = sizeof(float) * (2 * kThreads * kV + 2 * s.slice + 4 * (s.slice / s.per));
  return launch_split(group_norm_fwd_kernel<T, kV, kAct>, s.split, samples * (s.channels / s.slice), smem, allowed, stream, (const T*)x,
                      (const T*)residual, (T*)z, gamma, beta, stats, s);
}
template <class T, int kV, int kAct>
int backward(const void* x, const void* residual, const void* dz, void* dx, void* dres, const float* gamma, const float* beta,
             const float* stats, float* sums, int64_t samples, const Shape& s, void* stream) {
  static SmemAllowed allowed{0};
  const size_t smem = sizeof(float) * (2 * kThreads * kV + 4 * s.slice + 2 * (s.slice / s.per));
  return launch_split(group_norm_bwd_kernel<T, kV, kAct>, s.split, samples * (s.channels / s.slice), smem, allowed, stream, (const T*)x,
                      (const T*)residual, (const T*)dz, (T*)dx, (T*)dres, gamma, beta, stats, sums, s);
}

// f<T, kV, kAct>(): kV whole vectors where rows and pointers allow them.
#define ESGD_ACT(T, V, F, ...)                                                          \
  (act == kActRelu ? F<T, V, kActRelu>(__VA_ARGS__) : act == kActSilu ? F<T, V, kActSilu>(__VA_ARGS__) : F<T, V, kActNone>(__VA_ARGS__))
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
  if (!plan(samples, rows, channels, groups, v, &s)) {
    v = 1;
    if (!plan(samples, rows, channels, groups, v, &s)) return (int)cudaErrorInvalidValue;
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
  if (!plan(samples, rows, channels, groups, v, &s)) {
    v = 1;
    if (!plan(samples, rows, channels, groups, v, &s)) return (int)cudaErrorInvalidValue;
  }
  s.eps = 0.0f;
  return ESGD_TYPE(backward, x, residual, dz, dx, dres, gamma, beta, stats, sums, samples, s, stream);
}

}  // extern "C"
