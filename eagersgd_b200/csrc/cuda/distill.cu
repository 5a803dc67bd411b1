// Distillation from a teacher's top logits, loss and gradient in one pass over the logits.
//
//   p = softmax(v / T) over the classes i_k that the teacher names;  q = softmax(z / T), r = softmax(z) over all classes
//   loss_row = (1 - w) T^2 sum_k p_k (log p_k - log q_{i_k})  -  w log r_label
//   dz_j     = ((1 - w) T (q_j - sum_{k: i_k = j} p_k) + w (r_j - [j = label])) / rows
//
// Bound by memory and, nearly as much, by the exponentials: a row is read from memory once (running maxima and sums), is found in L2
// the second time, and its gradient is written once.  (4096 x 32000 bf16, top 64: 121 us, 4.4 TB/s of 6.5; rows held in registers in
// between, 64 KB a block and a third of the warps: 119 -> 154 us.)  A block has a row, or a cluster of blocks has one where rows are fewer
// than SMs; their maxima and sums meet in distributed shared memory.  The few classes that the teacher or the label names are
// written again, from their own sums, after the others: a class that is named twice counts twice.  An index outside the classes is
// no class; a row without a teacher (or label) has no such term, whatever its logits are.
#include <cooperative_groups.h>
#include <float.h>
#include "launch.cuh"
#include "rows.cuh"

namespace {

using namespace esgd;

namespace cg = cooperative_groups;

constexpr int kMaxTop = 1024;
constexpr int kMaxThreads = 512;
constexpr int kThreadVectors = 8, kSplitVectors = 512;

struct Args {
  const int64_t* classes_of;   // [rows][top]
  const int64_t* labels;       // [rows], or null
  const void* values;          // [rows][top]
  int values_bf16, top, classes, ld;
  int split;                   // blocks of a row
  float inv_t, t, soft, hard;  // soft = (1 - w), hard = w
  float inv_rows;
  float* row_loss;             // [rows]
};

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The logarithm of a sum whose largest term is one: its approximation's error is 4e-7 however small the logarithm is, that of log1p half a
// step of it.  (Two or three a row.)
__device__ __forceinline__ float log_sum(float v) { return log1pf(v - 1.0f); }

// Two vectors' maximum; a bf16 pair at a time.
template <class T, int kV> __device__ __forceinline__ Pack<T, kV> larger(const Pack<T, kV>& a, const Pack<T, kV>& b) {
  Pack<T, kV> r;
  const uint32_t x[4] = {a.v.x, a.v.y, a.v.z, a.v.w}, y[4] = {b.v.x, b.v.y, b.v.z, b.v.w};
  uint32_t z[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if constexpr (sizeof(T) == 4) {
      z[q] = __float_as_uint(fmaxf(__uint_as_float(x[q]), __uint_as_float(y[q])));
    } else {
      const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&x[q]), *reinterpret_cast<const __nv_bfloat162*>(&y[q]));
      z[q] = *reinterpret_cast<const uint32_t*>(&m);
    }
  }
  r.v = make_uint4(z[0], z[1], z[2], z[3]);
  return r;
}

// The blocks' maxima (or sums) of kMany values; every thread gets them.  sh: [kMany][16], and own[kMany] for the cluster.
template <int kMany, bool kMax> __device__ __forceinline__ void meet(float (&v)[kMany], float* sh, float* own, int split, cg::cluster_group& cluster) {
  const int warps = blockDim.x / 32;
#pragma unroll
  for (int i = 0; i < kMany; ++i) {
    v[i] = kMax ? warp_max(v[i]) : warp_sum(v[i]);
    if ((threadIdx.x & 31) == 0) sh[i * 16 + threadIdx.x / 32] = v[i];
  }
  __syncthreads();
  const int w = threadIdx.x & 15;
#pragma unroll
  for (int i = 0; i < kMany; ++i) {
    float r = w < warps ? sh[i * 16 + w] : kMax ? -INFINITY : 0.0f;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      const float other = __shfl_xor_sync(0xffffffffu, r, o);
      r = kMax ? fmaxf(r, other) : r + other;
    }
    v[i] = r;
    if (split > 1 && threadIdx.x == 0) own[i] = r;
  }
  if (split > 1) {
    cluster.sync();
#pragma unroll
    for (int i = 0; i < kMany; ++i) {
      float r = cluster.map_shared_rank(own, 0)[i];
      for (int k = 1; k < split; ++k) {
        const float o = cluster.map_shared_rank(own, k)[i];
        r = kMax ? fmaxf(r, o) : r + o;
      }
      v[i] = r;
    }
  }
}

template <class T, bool kHard, bool kGrad>
__global__ void __launch_bounds__(kMaxThreads, 4) distill_kernel(const T* __restrict__ logits, T* __restrict__ grad, Args a) {
  pdl_enter();
  constexpr int kV = vector_of<T>(), kP = kV / 2;
  extern __shared__ int4 smem4[];
  const int fours = (a.top + 3) / 4;
  int* index = reinterpret_cast<int*>(smem4);               // [top], -1: none; -2 up to a multiple of four
  float* prob = reinterpret_cast<float*>(smem4 + fours);    // [top]
  __shared__ float sh[3][3 * 16], own[3][3];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = a.split > 1 ? (int)cluster.block_rank() : 0;
  const int row = blockIdx.x / a.split, tid = threadIdx.x, threads = blockDim.x;
  const T* x = logits + (int64_t)row * a.ld;
  const float cs = a.inv_t * kLog2e, ch = kLog2e;

  // vectors from the first 16-byte boundary on, this block's share of them, and the single elements at the ends (the first block's)
  const int head = min(a.classes, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T));
  const int vectors = (a.classes - head) / kV, tail = head + vectors * kV, ends = rank == 0 ? head + a.classes - tail : 0;
  const int from = (int)((int64_t)vectors * rank / a.split), to = (int)((int64_t)vectors * (rank + 1) / a.split);
  const T* base = x + head;

  // the teacher's logits
  float peaks[2] = {-FLT_MAX, -INFINITY};
  if (tid < 4 * fours - a.top) index[a.top + tid] = -2;
  for (int k = tid; k < a.top; k += threads) {
    const int64_t at = (int64_t)row * a.top + k, c = a.classes_of[at];
    const float v = a.values_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.values)[at])
                                  : reinterpret_cast<const float*>(a.values)[at];
    const bool is = c >= 0 && c < a.classes && v != -INFINITY;
    prob[k] = v;
    index[k] = is ? (int)c : -1;
    if (is) peaks[1] = fmaxf(peaks[1], v == v ? v : INFINITY);      // a row of NaN has a teacher: its loss is NaN
  }
  int64_t label = -1;
  if constexpr (kHard) {
    label = a.labels[row];
    if (label < 0 || label >= a.classes) label = -1;
  }
  // a thread's maximum so far, and its sums of e^((z - max) / T) and e^(z - max) about it
  const f2 cs2 = pair(cs, cs), ch2 = pair(ch, ch);
  f2 soft = 0, hard = 0;
  auto raise = [&](float m) {
    if (m > peaks[0]) {
      soft = mul2(soft, exp2_approx((peaks[0] - m) * cs));
      if constexpr (kHard) hard = mul2(hard, exp2_approx((peaks[0] - m) * ch));
      peaks[0] = m;
    }
  };
  auto add = [&](const f2 (&f)[kP]) {
    const f2 minus = pair(-peaks[0], -peaks[0]);
#pragma unroll
    for (int q = 0; q < kP; ++q) {
      const f2 d = add2(f[q], minus);
      soft = add2(soft, exp2_2(mul2(d, cs2)));
      if constexpr (kHard) hard = add2(hard, exp2_2(mul2(d, ch2)));
    }
  };
  auto largest = [&](const Pack<T, kV>& m) {
    f2 f[kP];
    unpack2<T, kV>(m, f);
    float r = -INFINITY;
#pragma unroll
    for (int q = 0; q < kP; ++q) r = fmaxf(r, fmaxf(halves(f[q]).x, halves(f[q]).y));
    return r;
  };
  int i = from + tid;
  for (; i + threads < to; i += 2 * threads) {
    const Pack<T, kV> r0 = load<T, kV>(base + (int64_t)i * kV), r1 = load<T, kV>(base + (int64_t)(i + threads) * kV);
    raise(largest(larger<T, kV>(r0, r1)));
    f2 f[kP];
    unpack2<T, kV>(r0, f);
    add(f);
    unpack2<T, kV>(r1, f);
    add(f);
  }
  if (i < to) {
    const Pack<T, kV> r = load<T, kV>(base + (int64_t)i * kV);
    raise(largest(r));
    f2 f[kP];
    unpack2<T, kV>(r, f);
    add(f);
  }
  float sums[3] = {halves(soft).x + halves(soft).y, halves(hard).x + halves(hard).y, 0.0f};
  float own_end = peaks[0];
  for (int e = tid; e < ends; e += threads) {
    const float z = as_float(x[e < head ? e : tail + e - head]);
    if (z > own_end) {
      sums[0] *= exp2_approx((own_end - z) * cs);
      sums[1] *= exp2_approx((own_end - z) * ch);
      own_end = z;
    }
    sums[0] += exp2_approx((z - own_end) * cs);
    if constexpr (kHard) sums[1] += exp2_approx((z - own_end) * ch);
  }
  peaks[0] = own_end;
  meet<2, true>(peaks, sh[0], own[0], a.split, cluster);
  const float peak = peaks[0], top_peak = peaks[1];
  const bool taught = a.soft != 0.0f && top_peak != -INFINITY, any = taught || label >= 0;
  const f2 minus = pair(-peak, -peak);
  sums[0] *= exp2_approx((own_end - peak) * cs);
  if constexpr (kHard) sums[1] *= exp2_approx((own_end - peak) * ch);
  if (rank == 0)
    for (int k = tid; k < a.top; k += threads)
      if (index[k] >= 0) sums[2] += exp_fine((prob[k] - top_peak) * a.inv_t);
  meet<3, false>(sums, sh[1], own[1], a.split, cluster);
  const float log_soft = log_sum(sums[0]);

  // loss: log p_k - log q_k = (v_k - v_max) / T - log(sum) - (z_k - z_max) / T + log(sum_z)
  float kl = 0.0f;
  const float log_top = taught ? log_sum(sums[2]) : 0.0f, inv_top = taught ? 1.0f / sums[2] : 0.0f;
  for (int k = tid; k < a.top; k += threads) {
    float p = 0.0f;
    if (taught && index[k] >= 0) {
      const float v = (prob[k] - top_peak) * a.inv_t;
      p = exp_fine(v) * inv_top;
      if (rank == 0 && p != 0.0f) kl += p * ((v - log_top) - ((as_float(x[index[k]]) - peak) * a.inv_t - log_soft));
    }
    prob[k] = p;
  }
  kl = warp_sum(kl);
  if ((tid & 31) == 0) sh[2][tid / 32] = kl;
  if (a.split > 1) cluster.barrier_arrive();                // done with the others' sums

  const float ks = taught ? a.soft * a.t * a.inv_rows : 0.0f, kh = kHard && label >= 0 ? a.hard * a.inv_rows : 0.0f;
  if constexpr (kGrad) {
    T* d = grad + (int64_t)row * a.ld;
    const float fs = ks != 0.0f ? ks / sums[0] : 0.0f, fh = kh != 0.0f ? kh / sums[1] : 0.0f;
    const f2 fs2 = pair(fs, fs), fh2 = pair(fh, fh);
    auto dense = [&](const Pack<T, kV>& r, T* at) {
      f2 f[kP];
      unpack2<T, kV>(r, f);
#pragma unroll
      for (int q = 0; q < kP; ++q) {
        const f2 e = add2(f[q], minus);
        f[q] = mul2(exp2_2(mul2(e, cs2)), fs2);
        if constexpr (kHard) f[q] = fma2(exp2_2(mul2(e, ch2)), fh2, f[q]);
        if (!any) f[q] = 0;
      }
      store2<T, kV>(at, f);
    };
    int i = from + tid;
    for (; i + threads < to; i += 2 * threads) {
      const Pack<T, kV> r0 = load<T, kV>(base + (int64_t)i * kV), r1 = load<T, kV>(base + (int64_t)(i + threads) * kV);
      dense(r0, d + head + (int64_t)i * kV);
      dense(r1, d + head + (int64_t)(i + threads) * kV);
    }
    if (i < to) dense(load<T, kV>(base + (int64_t)i * kV), d + head + (int64_t)i * kV);
    auto one = [&](float z) {
      float v = 0.0f;
      if (any) {
        v = exp2_approx((z - peak) * cs) * fs;
        if constexpr (kHard) v = fmaf(exp2_approx((z - peak) * ch), fh, v);
      }
      return v;
    };
    for (int i = tid; i < ends; i += threads) {
      const int c = i < head ? i : tail + i - head;
      d[c] = as_type<T>(one(as_float(x[c])));
    }
    __syncthreads();
    // the named classes among this block's
    auto mine = [&](int c) { return c < head || c >= tail ? rank == 0 : (c - head) / kV >= from && (c - head) / kV < to; };
    if (taught) {
      for (int k = tid; k < a.top; k += threads) {
        const int c = index[k];
        if (c < 0 || !mine(c)) continue;
        float p = prob[k];
        bool first = true;
        for (int j = 0; j < fours; ++j) {
          const int4 o = smem4[j];
          if (o.x != c && o.y != c && o.z != c && o.w != c) continue;
          const int same[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (same[i] != c || 4 * j + i == k) continue;
            if (4 * j + i < k) first = false;
            else p += prob[4 * j + i];
          }
        }
        if (first) d[c] = as_type<T>(one(as_float(x[c])) - ks * p - (c == label ? kh : 0.0f));
      }
    }
    if (kHard && label >= 0) {       // a label that the teacher does not name
      bool named = false;
      if (taught)
        for (int k = tid; k < a.top; k += threads) named = named || index[k] == (int)label;
      if (!__syncthreads_or(named) && tid == 0 && mine((int)label)) d[label] = as_type<T>(one(as_float(x[label])) - kh);
    }
  } else {
    __syncthreads();
  }
  if (tid == 0 && rank == 0) {
    for (int w = 1; w < threads / 32; ++w) kl += sh[2][w];
    float loss = taught ? a.soft * a.t * a.t * kl : 0.0f;
    if constexpr (kHard)
      if (label >= 0) loss += a.hard * (log_sum(sums[1]) - (as_float(x[label]) - peak));
    a.row_loss[row] = loss;
  }
  if (a.split > 1) cluster.barrier_wait();                  // nobody leaves while its sums are being read
}

// The rows' mean in a fixed order.
__global__ void __launch_bounds__(1024) distill_mean_kernel(const float* __restrict__ row_loss, int rows, float* __restrict__ loss) {
  pdl_enter();
  __shared__ double sh[32];
  double t = 0.0;
  for (int i = threadIdx.x; i < rows; i += 1024) t += (double)row_loss[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x / 32] = t;
  __syncthreads();
  if (threadIdx.x < 32) {
    t = sh[threadIdx.x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (threadIdx.x == 0) *loss = (float)(t / (double)rows);
  }
}

// out = in * *factor; nothing to do where the two are one buffer and the factor is one.
template <class T, int kV>
__global__ void __launch_bounds__(256) distill_scale_kernel(const T* in, T* out, const float* __restrict__ factor, int64_t n) {
  pdl_enter();
  const float f = *factor;
  if (f == 1.0f && in == out) return;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n / kV; i += (int64_t)gridDim.x * 256) {
    float v[kV];
    unpack<T, kV>(load<T, kV>(in + i * kV), v);
#pragma unroll
    for (int q = 0; q < kV; ++q) v[q] *= f;
    store<T, kV>(out + i * kV, v);
  }
  if (blockIdx.x == 0 && threadIdx.x < n % kV) {
    const int64_t i = n / kV * kV + threadIdx.x;
    out[i] = as_type<T>(as_float(in[i]) * f);
  }
}

// Eight vectors a thread or more; rows that are fewer than SMs are spread over more blocks as long as these have something to do.
template <class T, class... K> int launch_row(void (*kernel)(K...), const T* x, T* d, Args a, int rows, void* stream) {
  const int vectors = (a.classes + vector_of<T>() - 1) / vector_of<T>();
  a.split = 1;
  while (a.split < 8 && rows * a.split < 2 * sm_count() && vectors > a.split * kSplitVectors) a.split *= 2;
  int threads = 128;
  while (threads < kMaxThreads && vectors > a.split * threads * kThreadVectors) threads *= 2;
  const dim3 grid((unsigned)(rows * a.split));
  const size_t smem = (size_t)((a.top + 3) / 4 * 4) * 8;
  switch (a.split) {
    case 1: return launch<1>(kernel, grid, threads, smem, stream, x, d, a);
    case 2: return launch<2>(kernel, grid, threads, smem, stream, x, d, a);
    case 4: return launch<4>(kernel, grid, threads, smem, stream, x, d, a);
    default: return launch<8>(kernel, grid, threads, smem, stream, x, d, a);
  }
}
template <class T>
int launch_rows(const void* logits, void* grad, const Args& a, int rows, void* stream) {
  const bool hard = a.labels != nullptr && a.hard != 0.0f;
  const T* x = (const T*)logits;
  T* d = (T*)grad;
  if (grad != nullptr)
    return hard ? launch_row(distill_kernel<T, true, true>, x, d, a, rows, stream) : launch_row(distill_kernel<T, false, true>, x, d, a, rows, stream);
  return hard ? launch_row(distill_kernel<T, true, false>, x, d, a, rows, stream) : launch_row(distill_kernel<T, false, false>, x, d, a, rows, stream);
}

}  // namespace

extern "C" {

int esgd_distill_max_top() { return kMaxTop; }

// logits, grad [rows][ld] (grad null: loss only); they begin on 16 bytes.  row_loss [rows]: room for the rows' losses.
int esgd_distill(const void* logits, void* grad, int is_bf16, const void* values, int values_bf16, const int64_t* classes_of,
                 const int64_t* labels, int rows, int classes, int ld, int top, float temperature, float hard_weight, float* row_loss,
                 float* loss, void* stream) {
  if (rows <= 0 || classes <= 0 || top < 0 || top > kMaxTop || rows > (1 << 27)) return (int)cudaErrorInvalidValue;
  const Args a = {classes_of, labels, values, values_bf16, top, classes, ld, 1, 1.0f / temperature, temperature, 1.0f - hard_weight,
                  hard_weight, 1.0f / (float)rows, row_loss};
  int rc = is_bf16 ? launch_rows<__nv_bfloat16>(logits, grad, a, rows, stream) : launch_rows<float>(logits, grad, a, rows, stream);
  if (rc == 0) rc = launch(distill_mean_kernel, dim3(1), 1024, 0, stream, row_loss, rows, loss);
  return rc;
}

int esgd_distill_scale(const void* in, void* out, int is_bf16, const float* factor, int64_t n, void* stream) {
  const int64_t blocks = (n + 256 * 16 - 1) / (256 * 16);
  const dim3 grid((unsigned)(blocks < 1 ? 1 : blocks > 8 * sm_count() ? 8 * sm_count() : blocks));
  return is_bf16 ? launch(distill_scale_kernel<__nv_bfloat16, 8>, grid, 256, 0, stream, (const __nv_bfloat16*)in, (__nv_bfloat16*)out, factor, n)
                 : launch(distill_scale_kernel<float, 4>, grid, 256, 0, stream, (const float*)in, (float*)out, factor, n);
}

}  // extern "C"
