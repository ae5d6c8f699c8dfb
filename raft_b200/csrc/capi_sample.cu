// b2r_sample_tokens: one token per row of logits by temperature, top-k, top-p and min-p.
#include "capi_internal.cuh"

#include <raft_b200/detail/sample_tokens.cuh>

namespace raft_b200 {
namespace capi {

template <typename T>
static int sample(const b2r_sample_desc& d, void* tokens, float* logprobs, const void* logits, const float* uniform,
                  cudaStream_t s)
{
  detail::sample::Args<T> a = {};
  a.logits          = static_cast<const T*>(logits);
  a.ldl             = d.ld;
  a.uniform         = uniform;
  a.temperature     = d.temperature;
  a.top_k           = d.top_k;
  a.top_p           = d.top_p;
  a.min_p           = d.min_p;
  a.temperature_all = d.temperature_all;
  a.top_k_all       = d.top_k_all;
  a.top_p_all       = d.top_p_all;
  a.min_p_all       = d.min_p_all;
  a.out             = tokens;
  a.out64           = d.out_dtype == B2R_I64 ? 1 : 0;
  a.logprobs        = logprobs;
  a.n_rows          = d.n_rows;
  a.vocab           = int(d.vocab);
  return set_cuda_error(detail::sample::launch_sample<T>(a, s));
}

}  // namespace capi
}  // namespace raft_b200

using namespace raft_b200;
using namespace raft_b200::capi;

extern "C" int b2r_sample_tokens(const b2r_sample_desc* desc, void* tokens, float* logprobs, const void* logits,
                                 const float* uniform, b2r_stream_t stream)
{
  if (desc == nullptr) return B2R_ERR_BAD_ARG;
  const b2r_sample_desc& d = *desc;
  if (d.n_rows < 0 || d.vocab < 0 || d.ld < d.vocab) return B2R_ERR_BAD_ARG;
  if (d.n_rows > 0x7fffffff || d.vocab > detail::sample::kMaxVocab) return B2R_ERR_TOO_LARGE;
  if (d.n_rows > 0 && (tokens == nullptr || uniform == nullptr || (d.vocab > 0 && logits == nullptr)))
    return B2R_ERR_BAD_ARG;
  if (d.out_dtype != B2R_I32 && d.out_dtype != B2R_I64) return B2R_ERR_UNSUPPORTED;
  if (d.dtype != B2R_F32 && d.dtype != B2R_F16 && d.dtype != B2R_BF16) return B2R_ERR_UNSUPPORTED;
  if (d.n_rows == 0) return B2R_OK;
  cudaStream_t s = to_stream(stream);
  if (d.dtype == B2R_F32) return sample<float>(d, tokens, logprobs, logits, uniform, s);
  if (d.dtype == B2R_F16) return sample<__half>(d, tokens, logprobs, logits, uniform, s);
  return sample<__nv_bfloat16>(d, tokens, logprobs, logits, uniform, s);
}
