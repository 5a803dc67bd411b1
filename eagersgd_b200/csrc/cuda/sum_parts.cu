// Sums over the first dimension of a workspace [parts][n], in a fixed order: the gradients of parameters that many blocks have
// a share of.  Up to three parameters lie one after the other in a part.
#include "launch.cuh"

namespace {

struct Segment {
  float* out;        // null: not wanted
  int64_t n;
  int add;           // to what is there
};

__global__ void __launch_bounds__(256) sum_parts_kernel(const float* __restrict__ ws, int64_t parts, int64_t n, Segment a, Segment b,
                                                        Segment c) {
  esgd::pdl_enter();
  __shared__ float sh[8][32];
  const int64_t i = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
  const int lane = threadIdx.x / 32;
  float t = 0.0f;
  if (i < n)
    for (int64_t p = lane; p < parts; p += 8) t += ws[p * n + i];
  sh[lane][threadIdx.x & 31] = t;
  __syncthreads();
  if (lane == 0 && i < n) {
    for (int k = 1; k < 8; ++k) t += sh[k][threadIdx.x];
    int64_t j = i;
    const Segment& s = j < a.n ? a : (j -= a.n) < b.n ? b : (j -= b.n, c);
    if (s.out != nullptr) s.out[j] = t + (s.add ? s.out[j] : 0.0f);
  }
}

}  // namespace

extern "C" int esgd_sum_parts(const float* ws, int64_t parts, float* a, int64_t na, int add_a, float* b, int64_t nb, int add_b, float* c,
                              int64_t nc, int add_c, void* stream) {
  const int64_t n = na + nb + nc;
  if (n == 0 || (a == nullptr && b == nullptr && c == nullptr)) return 0;
  return esgd::launch(sum_parts_kernel, dim3((unsigned)((n + 31) / 32)), 256, 0, stream, ws, parts, n, Segment{a, na, add_a},
                      Segment{b, nb, add_b}, Segment{c, nc, add_c});
}
