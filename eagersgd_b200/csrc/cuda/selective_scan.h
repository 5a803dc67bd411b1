// What a selective scan reads, as its launchers take it.
#pragma once
#include <stdint.h>

struct esgd_scan {
  const void* p[5];            // u, delta, z (or null), B, C: [batch][length][channels or states], the last dimension dense
  int64_t b[5], t[5];          // their strides, in elements
  const float *A, *D, *bias;   // [channels][states]; [channels] or null
  const int64_t* lengths;      // [batch], or null
  const float* state;          // [batch][channels][states], or null: zero
  int64_t batch, length;
  int channels, states, softplus, is_bf16;
};
