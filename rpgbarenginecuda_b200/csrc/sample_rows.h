// sample_rows.h -- host-side launcher of the sampling of a batch (k_sample_rows.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "kv.h"

namespace rpgb {

struct SampleRowsParams {
  ElemType type = ElemType::kF32;
  const void* logits = nullptr;
  int64_t stride = 0;  // elements
  int32_t n_rows = 0, vocab = 0;
  // [n_rows] each; null: the option is off (temperature 1)
  const float* temperature = nullptr;
  const int32_t* top_k = nullptr;
  const float *top_p = nullptr, *min_p = nullptr, *u = nullptr;
  int32_t* tok = nullptr;
  float* prob = nullptr;  // null: not wanted
};
void LaunchSampleRows(const SampleRowsParams& p, cudaStream_t s);

}  // namespace rpgb
