// extern "C" entry point of token sampling (include/b200ep.h).  No counterpart in the reference, which hands
// the logits back to the host.
#include <string>

#include "common.cuh"
#include "kernels/sample.h"

using namespace b200ep;

extern "C" B200EP_API int b200ep_sample(const void* logits, const float* noise, const float* temperature,
                                        const int32_t* top_k, const float* top_p, const float* min_p,
                                        int64_t* tokens, float* logprobs, int64_t rows, int64_t vocab,
                                        int64_t logits_stride, int64_t noise_stride, int dtype, void* stream) {
  try {
    B200EP_CHECK_ARG(is_float_dtype(dtype), "Sample: dtype must be float32, float16 or bfloat16");
    B200EP_CHECK_ARG(vocab > 0 && vocab <= kMaxVocab, "Sample: vocab must lie in [1, 262144]");
    B200EP_CHECK_ARG(rows >= 0 && rows < (1ll << 27), "Sample: rows must lie in [0, 2^27)");
    B200EP_CHECK_ARG((!logits_stride || logits_stride >= vocab) && (!noise_stride || noise_stride >= vocab),
                     "Sample: row strides must be at least vocab");
    if (rows == 0) return B200EP_OK;
    B200EP_CHECK_ARG(logits && noise && tokens, "Sample: null pointer");
    SampleArgs a{};
    a.logits = logits, a.noise = noise, a.temperature = temperature, a.top_k = top_k, a.top_p = top_p;
    a.min_p = min_p, a.tokens = tokens, a.logprobs = logprobs;
    a.logits_stride = logits_stride ? logits_stride : vocab;
    a.noise_stride = noise_stride ? noise_stride : vocab;
    a.rows = (int)rows, a.vocab = (int)vocab, a.dtype = dtype;
    return cuda_status(launch_sample(a, static_cast<cudaStream_t>(stream)), "Sample launch");
  } catch (const std::exception& e) {
    return set_error(B200EP_EINTERNAL, std::string("exception: ") + e.what());
  }
}
