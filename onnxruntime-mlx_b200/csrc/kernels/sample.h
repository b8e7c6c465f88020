// Internal launcher of token sampling (sample.cu); csrc/capi_sample.cu validates and calls it.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace b200ep {

constexpr int64_t kMaxVocab = 262144;  // 8 CTAs of 32768 tokens each

struct SampleArgs {
  const void* logits;         // [rows, vocab], row stride in elements
  const float* noise;         // [rows, vocab], row stride in elements
  const float* temperature;   // [rows] or null (1)
  const int32_t* top_k;       // [rows] or null (off)
  const float* top_p;         // [rows] or null (off)
  const float* min_p;         // [rows] or null (off)
  int64_t* tokens;            // [rows]
  float* logprobs;            // [rows] or null
  int64_t logits_stride, noise_stride;
  int rows, vocab, dtype;
};
cudaError_t launch_sample(const SampleArgs& a, cudaStream_t st);

}  // namespace b200ep
