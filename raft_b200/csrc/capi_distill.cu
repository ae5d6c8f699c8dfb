// b2r_topk_distill / b2r_topk_distill_grad: distillation loss from a teacher's top logits, and its gradient.
#include "capi_internal.cuh"

#include <raft_b200/detail/topk_distill.cuh>

namespace raft_b200 {
namespace capi {

constexpr int64_t kMaxExtent = 0x7fffffff;

// what both entry points share; B2R_OK: go on
static int check_distill(const void* logits, int64_t ldl, const void* grad, int64_t ldg, const void* ids, int64_t ldi,
                         int32_t id_dtype, const void* teacher, int64_t ldt, int32_t teacher_dtype, int64_t n_rows,
                         int64_t vocab, int64_t k, double temperature)
{
  if (n_rows < 0 || vocab < 0 || k < 0 || ldl < vocab || ldi < k || ldt < k) return B2R_ERR_BAD_ARG;
  if (grad != nullptr && ldg < vocab) return B2R_ERR_BAD_ARG;
  if (!(temperature >= 1e-30 && temperature <= 1e30)) return B2R_ERR_BAD_ARG;  // 1 / T in fp32
  if (n_rows > kMaxExtent || vocab > kMaxExtent - 64 || k > detail::distill::kMaxK) return B2R_ERR_TOO_LARGE;
  if (n_rows > 0 && vocab > 0 && logits == nullptr) return B2R_ERR_BAD_ARG;
  if (n_rows > 0 && k > 0 && (ids == nullptr || teacher == nullptr)) return B2R_ERR_BAD_ARG;
  if (id_dtype != B2R_I32 && id_dtype != B2R_I64) return B2R_ERR_UNSUPPORTED;
  if (teacher_dtype != B2R_F32 && teacher_dtype != B2R_F16 && teacher_dtype != B2R_BF16) return B2R_ERR_UNSUPPORTED;
  return B2R_OK;
}

template <typename T>
static detail::distill::Args<T> distill_args(const void* logits, int64_t ldl, void* grad, int64_t ldg, const void* ids,
                                             int64_t ldi, int32_t id_dtype, const void* teacher, int64_t ldt,
                                             int32_t teacher_dtype, int64_t n_rows, int64_t vocab, int64_t k,
                                             double temperature)
{
  detail::distill::Args<T> a = {};
  a.logits      = static_cast<const T*>(logits);
  a.ldl         = ldl;
  a.grad        = static_cast<T*>(grad);
  a.ldg         = ldg;
  a.list        = {ids, ldi, teacher, ldt, id_dtype == B2R_I64 ? 1 : 0, teacher_dtype, int(k)};
  a.n_rows      = n_rows;
  a.vocab       = int(vocab);
  a.temperature = temperature;
  a.ctl         = detail::ring_ctl(kernel_status_word());
  a.late_warp   = detail::tuning().test_late_warp - 1;
  return a;
}

}  // namespace capi
}  // namespace raft_b200

using namespace raft_b200;
using namespace raft_b200::capi;

extern "C" int b2r_topk_distill(float* loss, float* lse, void* grad, int64_t ldg, const float* grad_loss,
                                const void* logits, int64_t ldl, int32_t dtype, const void* ids, int64_t ldi,
                                int32_t id_dtype, const void* teacher, int64_t ldt, int32_t teacher_dtype,
                                int64_t n_rows, int64_t vocab, int64_t k, double temperature, b2r_stream_t stream)
{
  const int chk = check_distill(logits, ldl, grad, ldg, ids, ldi, id_dtype, teacher, ldt, teacher_dtype, n_rows,
                                vocab, k, temperature);
  if (chk != B2R_OK) return chk;
  if (n_rows > 0 && grad != nullptr && grad_loss == nullptr) return B2R_ERR_BAD_ARG;
  if (dtype != B2R_F32 && dtype != B2R_F16 && dtype != B2R_BF16) return B2R_ERR_UNSUPPORTED;
  if (n_rows == 0) return B2R_OK;
  cudaStream_t s = to_stream(stream);
#define B2R_DISTILL(T)                                                                                            \
  do {                                                                                                            \
    auto a = distill_args<T>(logits, ldl, grad, ldg, ids, ldi, id_dtype, teacher, ldt, teacher_dtype, n_rows,     \
                             vocab, k, temperature);                                                              \
    a.loss      = loss;                                                                                           \
    a.lse       = lse;                                                                                            \
    a.grad_loss = grad_loss;                                                                                      \
    return set_cuda_error(grad != nullptr ? detail::distill::launch_loss_and_grad<T>(a, s)                        \
                                          : detail::distill::launch_loss<T>(a, s));                               \
  } while (0)
  if (dtype == B2R_F32) B2R_DISTILL(float);
  if (dtype == B2R_F16) B2R_DISTILL(__half);
  B2R_DISTILL(__nv_bfloat16);
#undef B2R_DISTILL
}

extern "C" int b2r_topk_distill_grad(void* grad, int64_t ldg, const float* lse, const float* grad_loss,
                                     const void* logits, int64_t ldl, int32_t dtype, const void* ids, int64_t ldi,
                                     int32_t id_dtype, const void* teacher, int64_t ldt, int32_t teacher_dtype,
                                     int64_t n_rows, int64_t vocab, int64_t k, double temperature,
                                     b2r_stream_t stream)
{
  const int chk = check_distill(logits, ldl, grad, ldg, ids, ldi, id_dtype, teacher, ldt, teacher_dtype, n_rows,
                                vocab, k, temperature);
  if (chk != B2R_OK) return chk;
  if (n_rows > 0 && vocab > 0 && (grad == nullptr || lse == nullptr || grad_loss == nullptr)) return B2R_ERR_BAD_ARG;
  if (dtype != B2R_F32 && dtype != B2R_F16 && dtype != B2R_BF16) return B2R_ERR_UNSUPPORTED;
  if (n_rows == 0 || vocab == 0) return B2R_OK;
  cudaStream_t s = to_stream(stream);
#define B2R_DISTILL(T)                                                                                            \
  do {                                                                                                            \
    auto a = distill_args<T>(logits, ldl, grad, ldg, ids, ldi, id_dtype, teacher, ldt, teacher_dtype, n_rows,     \
                             vocab, k, temperature);                                                              \
    a.lse_in    = lse;                                                                                            \
    a.grad_loss = grad_loss;                                                                                      \
    return set_cuda_error(detail::distill::launch_grad_only<T>(a, s));                                            \
  } while (0)
  if (dtype == B2R_F32) B2R_DISTILL(float);
  if (dtype == B2R_F16) B2R_DISTILL(__half);
  B2R_DISTILL(__nv_bfloat16);
#undef B2R_DISTILL
}
