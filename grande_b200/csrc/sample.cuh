// Sampling from logits rows on the device: temperature, top-k, top-p, min-p
// and a draw with a given uniform number per row.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "paged.cuh"  // OpType

namespace omg {

struct SampleArgs {
  const void* logits;  // [rows] rows of vocab values
  int64_t stride;      // elements between rows
  int rows, vocab;
  const int* row_of;   // [rows] the logits row of each sampled row; null: in order
  int dtype;           // OpType
  const float* u;      // [rows] in [0, 1)
  // Per-row settings, or null and the one value for all rows.
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature1, top_p1, min_p1;
  int top_k1;
  int* tokens;         // [rows]
  float* probs;        // [rows] or null
};

// The largest vocabulary that a call takes.
int sample_max_vocab();
void launch_sample(const SampleArgs& a, int num_sms, cudaStream_t s);
void sample_setup_device();

}  // namespace omg
