// b2r_embedding_lookup / b2r_embedding_grad: rows of a table by token, and the sums of rows by token.
#include "capi_internal.cuh"

#include <raft_b200/detail/embedding.cuh>

namespace raft_b200 {
namespace capi {

constexpr int64_t kMaxExtent = 0x7fffffff;

template <typename T, typename TokT>
static int lookup(void* out, int64_t ldo, const void* table, int64_t ldt, const void* tokens, int64_t n, int64_t c,
                  int64_t vocab, double scale, cudaStream_t s)
{
  return set_cuda_error(detail::emb::launch_lookup<T, TokT>(static_cast<T*>(out), ldo, static_cast<const T*>(table),
                                                            ldt, static_cast<const TokT*>(tokens), n, c, vocab,
                                                            float(scale), s));
}

template <typename InT, typename OutT, typename TokT>
static int grad(void* out, int64_t ldg, const void* g, int64_t ldo, const void* tokens, int64_t n, int64_t c,
                int64_t vocab, double scale, bool accumulate, detail::Workspace ws, cudaStream_t s)
{
  return set_cuda_error(detail::emb::launch_grad<InT, OutT, TokT>(
    static_cast<OutT*>(out), ldg, static_cast<const InT*>(g), ldo, static_cast<const TokT*>(tokens), n, c, vocab,
    float(scale), accumulate, s, ws));
}

}  // namespace capi
}  // namespace raft_b200

using namespace raft_b200;
using namespace raft_b200::capi;

extern "C" int b2r_embedding_lookup(void* out, int64_t ldo, const void* table, int64_t ldt, const void* tokens,
                                    int32_t dtype, int32_t token_dtype, int64_t n_tokens, int64_t n_cols,
                                    int64_t vocab, double scale, b2r_stream_t stream)
{
  if (n_tokens < 0 || n_cols < 0 || vocab < 0 || ldo < n_cols || ldt < n_cols) return B2R_ERR_BAD_ARG;
  if (n_tokens > kMaxExtent || n_cols > kMaxExtent || vocab > kMaxExtent) return B2R_ERR_TOO_LARGE;
  if (n_tokens > 0 && n_cols > 0 && (out == nullptr || tokens == nullptr || (vocab > 0 && table == nullptr)))
    return B2R_ERR_BAD_ARG;
  cudaStream_t s = to_stream(stream);
#define B2R_LOOKUP(T)                                                                                          \
  do {                                                                                                         \
    if (token_dtype == B2R_I32)                                                                                \
      return lookup<T, int>(out, ldo, table, ldt, tokens, n_tokens, n_cols, vocab, scale, s);                  \
    if (token_dtype == B2R_I64)                                                                                \
      return lookup<T, long long>(out, ldo, table, ldt, tokens, n_tokens, n_cols, vocab, scale, s);            \
  } while (0)
  if (dtype == B2R_F32) B2R_LOOKUP(float);
  if (dtype == B2R_F16) B2R_LOOKUP(__half);
  if (dtype == B2R_BF16) B2R_LOOKUP(__nv_bfloat16);
#undef B2R_LOOKUP
  return B2R_ERR_UNSUPPORTED;
}

extern "C" int b2r_embedding_grad(void* grad_table, int64_t ldg, int32_t table_dtype, const void* grad_out,
                                  int64_t ldo, int32_t dtype, const void* tokens, int32_t token_dtype,
                                  int64_t n_tokens, int64_t n_cols, int64_t vocab, double scale, int32_t accumulate,
                                  void* workspace, size_t workspace_bytes, b2r_stream_t stream)
{
  if (n_tokens < 0 || n_cols < 0 || vocab < 0 || ldo < n_cols || ldg < n_cols) return B2R_ERR_BAD_ARG;
  if (n_tokens > kMaxExtent || n_cols > kMaxExtent || vocab > kMaxExtent) return B2R_ERR_TOO_LARGE;
  if (vocab > 0 && n_cols > 0 && grad_table == nullptr) return B2R_ERR_BAD_ARG;
  if (n_tokens > 0 && n_cols > 0 && (grad_out == nullptr || tokens == nullptr)) return B2R_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return B2R_ERR_BAD_ARG;
  const detail::Workspace ws = make_workspace(workspace, workspace_bytes);
  cudaStream_t s             = to_stream(stream);
  const bool acc             = accumulate != 0;
#define B2R_GRAD(IN, OUT)                                                                                       \
  do {                                                                                                          \
    if (token_dtype == B2R_I32)                                                                                 \
      return grad<IN, OUT, int>(grad_table, ldg, grad_out, ldo, tokens, n_tokens, n_cols, vocab, scale, acc, ws, s); \
    if (token_dtype == B2R_I64)                                                                                 \
      return grad<IN, OUT, long long>(grad_table, ldg, grad_out, ldo, tokens, n_tokens, n_cols, vocab, scale, acc, ws, \
                                      s);                                                                       \
  } while (0)
  if (dtype == B2R_F32 && table_dtype == B2R_F32) B2R_GRAD(float, float);
  if (dtype == B2R_F16 && table_dtype == B2R_F16) B2R_GRAD(__half, __half);
  if (dtype == B2R_F16 && table_dtype == B2R_F32) B2R_GRAD(__half, float);
  if (dtype == B2R_BF16 && table_dtype == B2R_BF16) B2R_GRAD(__nv_bfloat16, __nv_bfloat16);
  if (dtype == B2R_BF16 && table_dtype == B2R_F32) B2R_GRAD(__nv_bfloat16, float);
#undef B2R_GRAD
  return B2R_ERR_UNSUPPORTED;
}

extern "C" size_t b2r_embedding_grad_workspace_bytes(int64_t n_tokens, int64_t n_cols, int64_t vocab)
{
  if (n_tokens > kMaxExtent || n_cols > kMaxExtent || vocab > kMaxExtent) return 0;
  return detail::emb::grad_scratch_bytes(n_tokens, n_cols, vocab);
}
