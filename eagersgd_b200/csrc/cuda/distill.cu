// Distillation from a teacher's top logits, loss and gradient in one pass over the logits.
//
//   p = softmax(v / T) over the classes i_k that the teacher names;  q = softmax(z / T), r = softmax(z) over all classes
//   loss_row = (1 - w) T^2 sum_k p_k (log p_k - log q_{i_k})  -  w log r_label
//   dz_j     = ((1 - w) T (q_j - sum_{k: i_k = j} p_k) + w (r_j - [j = label])) / rows
//
// Bound by memory: a row is read from memory once (running maximum and sums), is found in L2 the second time, and its gradient is
// written once.  The few classes that the teacher or the label names are written again, from their own sums, after the others: a
// class that is named twice counts twice.  An index outside the classes is no class; a row without a teacher (or label) has no
// such term, whatever its logits are.
#include <float.h>
#include "launch.cuh"
#include "rows.cuh"

namespace {

using namespace esgd;

constexpr int kMaxTop = 1024;

struct Args {
  const int64_t* classes_of;   // [rows][top]
  const int64_t* labels;       // [rows], or null
  const void* values;          // [rows][top]
  int values_bf16, top, classes, ld;
  float inv_t, t, soft, hard;  // soft = (1 - w), hard = w
  float inv_rows;
  float* row_loss;             // [rows]
};

struct MaxOp { __device__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct SumOp { __device__ float operator()(float a, float b) const { return a + b; } };
template <class Op> __device__ __forceinline__ float warp_all(float v, Op op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// Over the block, in a fixed order; sh: one float a warp, and its own for each call in a row.
template <class Op> __device__ __forceinline__ float block_all(float v, Op op, float* sh) {
  const int warps = blockDim.x / 32;
  v = warp_all(v, op);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x / 32] = v;
  __syncthreads();
  float r = sh[0];
  for (int w = 1; w < warps; ++w) r = op(r, sh[w]);
  return r;
}

// Maximum so far and the sums of e^(z - max) (kHard) and e^((z - max) / T) about it.
template <bool kHard> struct Running {
  float peak = -FLT_MAX, soft = 0.0f, hard = 0.0f;
  __device__ __forceinline__ void raise(float to, float cs, float ch) {
    if (to > peak) {
      soft *= exp2_approx((peak - to) * cs);
      if constexpr (kHard) hard *= exp2_approx((peak - to) * ch);
      peak = to;
    }
  }
  __device__ __forceinline__ void add(float x, float cs, float ch) {
    soft += exp2_approx((x - peak) * cs);
    if constexpr (kHard) hard += exp2_approx((x - peak) * ch);
  }
};

template <class T, bool kHard, bool kGrad>
__global__ void __launch_bounds__(512) distill_kernel(const T* __restrict__ logits, T* __restrict__ grad, Args a) {
  pdl_enter();
  constexpr int kV = vector_of<T>();
  extern __shared__ float smem[];
  float* prob = smem;                                       // [top]
  int* index = reinterpret_cast<int*>(smem + a.top);        // [top], -1: none
  __shared__ float sh[6][16];
  const int row = blockIdx.x, tid = threadIdx.x, threads = blockDim.x;
  const T* x = logits + (int64_t)row * a.ld;
  const float cs = a.inv_t * kLog2e, ch = kLog2e;

  // the teacher's distribution
  float top_peak = -INFINITY;
  for (int k = tid; k < a.top; k += threads) {
    const int64_t at = (int64_t)row * a.top + k, c = a.classes_of[at];
    const float v = a.values_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.values)[at])
                                  : reinterpret_cast<const float*>(a.values)[at];
    const bool is = c >= 0 && c < a.classes && v != -INFINITY;
    prob[k] = v;
    index[k] = is ? (int)c : -1;
    if (is) top_peak = fmaxf(top_peak, v);
  }
  top_peak = block_all(top_peak, MaxOp(), sh[0]);
  float top_sum = 0.0f;
  for (int k = tid; k < a.top; k += threads)
    if (index[k] >= 0) top_sum += exp_fine((prob[k] - top_peak) * a.inv_t);
  top_sum = block_all(top_sum, SumOp(), sh[1]);
  const bool taught = a.soft != 0.0f && top_peak != -INFINITY;
  int64_t label = -1;
  if constexpr (kHard) {
    label = a.labels[row];
    if (label < 0 || label >= a.classes) label = -1;
  }

  // the row's maximum and sums; vectors from the first 16-byte boundary on
  const int head = min(a.classes, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T));
  const int vectors = (a.classes - head) / kV, tail = head + vectors * kV;
  Running<kHard> run;
  if (taught || label >= 0) {
    for (int i = tid; i < vectors; i += 2 * threads) {
      const bool two = i + threads < vectors;
      const Pack<T, kV> r0 = load<T, kV>(x + head + i * kV);
      Pack<T, kV> r1 = r0;
      if (two) r1 = load<T, kV>(x + head + (i + threads) * kV);
      float f[kV], g[kV];
      unpack<T, kV>(r0, f);
      unpack<T, kV>(r1, g);
      float m = f[0];
#pragma unroll
      for (int q = 0; q < kV; ++q) m = fmaxf(m, fmaxf(f[q], g[q]));
      run.raise(m, cs, ch);
#pragma unroll
      for (int q = 0; q < kV; ++q) run.add(f[q], cs, ch);
      if (two) {
#pragma unroll
        for (int q = 0; q < kV; ++q) run.add(g[q], cs, ch);
      }
    }
    for (int i = tid; i < head + a.classes - tail; i += threads) {
      const float f = as_float(x[i < head ? i : tail + i - head]);
      run.raise(f, cs, ch);
      run.add(f, cs, ch);
    }
  }
  const float peak = block_all(run.peak, MaxOp(), sh[2]);
  run.raise(peak, cs, ch);
  const float soft_sum = block_all(run.soft, SumOp(), sh[3]);
  float hard_sum = 1.0f;
  if constexpr (kHard) hard_sum = block_all(run.hard, SumOp(), sh[4]);
  const float log_soft = __logf(soft_sum);

  // loss: log p_k - log q_k = (v_k - v_max) / T - log(sum) - (z_k - z_max) / T + log(sum_z)
  float kl = 0.0f;
  const float log_top = taught ? __logf(top_sum) : 0.0f, inv_top = taught ? 1.0f / top_sum : 0.0f;
  for (int k = tid; k < a.top; k += threads) {
    float p = 0.0f;
    if (taught && index[k] >= 0) {
      const float v = (prob[k] - top_peak) * a.inv_t;
      p = exp_fine(v) * inv_top;
      if (p != 0.0f) kl += p * ((v - log_top) - ((as_float(x[index[k]]) - peak) * a.inv_t - log_soft));
    }
    prob[k] = p;
  }
  kl = block_all(kl, SumOp(), sh[5]);        // prob[] is whole behind its barrier
  if (tid == 0) {
    float loss = taught ? a.soft * a.t * a.t * kl : 0.0f;
    if constexpr (kHard)
      if (label >= 0) loss += a.hard * (__logf(hard_sum) - (as_float(x[label]) - peak));
    a.row_loss[row] = loss;
  }
  if constexpr (kGrad) {
    T* d = grad + (int64_t)row * a.ld;
    const float ks = taught ? a.soft * a.t * a.inv_rows : 0.0f, kh = kHard && label >= 0 ? a.hard * a.inv_rows : 0.0f;
    const float fs = ks != 0.0f ? ks / soft_sum : 0.0f, fh = kh != 0.0f ? kh / hard_sum : 0.0f;
    const bool any = ks != 0.0f || kh != 0.0f;
    auto dense = [&](float z) {
      float v = 0.0f;
      if (any) {
        v = exp2_approx((z - peak) * cs) * fs;
        if constexpr (kHard) v = fmaf(exp2_approx((z - peak) * ch), fh, v);
      }
      return v;
    };
    for (int i = tid; i < vectors; i += threads) {
      float f[kV];
      unpack<T, kV>(load<T, kV>(x + head + i * kV), f);
#pragma unroll
      for (int q = 0; q < kV; ++q) f[q] = dense(f[q]);
      store<T, kV>(d + head + i * kV, f);
    }
    for (int i = tid; i < head + a.classes - tail; i += threads) {
      const int c = i < head ? i : tail + i - head;
      d[c] = as_type<T>(dense(as_float(x[c])));
    }
    __syncthreads();
    if (taught) {
      for (int k = tid; k < a.top; k += threads) {
        const int c = index[k];
        if (c < 0) continue;
        float p = 0.0f;
        bool first = true;
        for (int j = 0; j < a.top; ++j)
          if (index[j] == c) {
            if (j < k) { first = false; break; }
            p += prob[j];
          }
        if (first) d[c] = as_type<T>(dense(as_float(x[c])) - ks * p - (c == label ? kh : 0.0f));
      }
    }
    if (kHard && label >= 0) {       // a label that the teacher does not name
      bool named = false;
      if (taught)
        for (int k = tid; k < a.top; k += threads) named = named || index[k] == (int)label;
      if (!__syncthreads_or(named) && tid == 0) d[label] = as_type<T>(dense(as_float(x[label])) - kh);
    }
  }
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

template <class T>
int launch_rows(const void* logits, void* grad, const Args& a, int rows, void* stream) {
  const int threads = a.classes <= 1024 * vector_of<T>() / 4 ? 128 : 512;
  const size_t smem = (size_t)a.top * 8;
  const bool hard = a.labels != nullptr && a.hard != 0.0f;
  const T* x = (const T*)logits;
  T* d = (T*)grad;
  if (grad != nullptr)
    return hard ? launch(distill_kernel<T, true, true>, dim3(rows), threads, smem, stream, x, d, a)
                : launch(distill_kernel<T, false, true>, dim3(rows), threads, smem, stream, x, d, a);
  return hard ? launch(distill_kernel<T, true, false>, dim3(rows), threads, smem, stream, x, d, a)
              : launch(distill_kernel<T, false, false>, dim3(rows), threads, smem, stream, x, d, a);
}

}  // namespace

extern "C" {

int esgd_distill_max_top() { return kMaxTop; }

// logits, grad [rows][ld] (grad null: loss only); they begin on 16 bytes.  row_loss [rows]: room for the rows' losses.
int esgd_distill(const void* logits, void* grad, int is_bf16, const void* values, int values_bf16, const int64_t* classes_of,
                 const int64_t* labels, int rows, int classes, int ld, int top, float temperature, float hard_weight, float* row_loss,
                 float* loss, void* stream) {
  if (rows <= 0 || classes <= 0 || top < 0 || top > kMaxTop) return (int)cudaErrorInvalidValue;
  const Args a = {classes_of, labels, values, values_bf16, top, classes, ld, 1.0f / temperature, temperature, 1.0f - hard_weight,
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
