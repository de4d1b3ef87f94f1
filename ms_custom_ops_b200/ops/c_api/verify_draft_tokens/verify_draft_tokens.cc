// verify_draft_tokens: operator glue.  An extension of the plugin (no reference counterpart): what follows the
// multi-token attention of a speculative step.  The device work is msco_verify_draft_tokens (libmsco_b200.so).
#include "ms_custom_ops_c.h"
#include "ops/framework/checks.h"
#include "ops/framework/module.h"
#include "ops/framework/tensor.h"

namespace ms_custom_ops {
namespace {

constexpr const char *kOpName = "VerifyDraftTokens";

struct Sizes {
  int64_t batch = 0, drafts = 0, vocab = 0;
};

Sizes Check(const Tensor &target, const Tensor &draft, const Tensor &draft_tokens, const Tensor &uniform,
            const Tensor &draft_lens) {
  Sizes s;
  CheckProvided(target, kOpName, "target_probs");
  CheckProvided(draft_tokens, kOpName, "draft_tokens");
  CheckProvided(uniform, kOpName, "uniform");
  CheckRank(target, kOpName, "target_probs", 3);
  CheckRank(draft, kOpName, "draft_probs", 3);
  CheckRank(draft_tokens, kOpName, "draft_tokens", 2);
  CheckRank(uniform, kOpName, "uniform", 2);
  CheckRank(draft_lens, kOpName, "draft_lens", 1);
  s.batch = draft_tokens.dim(0);
  s.drafts = draft_tokens.dim(1);
  s.vocab = target.dim(2);
  if (target.dtype() != MSCO_DTYPE_F32 && target.dtype() != MSCO_DTYPE_F16 && target.dtype() != MSCO_DTYPE_BF16)
    MS_TYPE_ERROR << "For " << kOpName << ", target_probs must be Float32/Float16/BFloat16, but got "
                  << DTypeName(target.dtype()) << ".";
  CheckDType(draft, kOpName, "draft_probs", target.dtype());
  CheckDType(draft_tokens, kOpName, "draft_tokens", MSCO_DTYPE_I32);
  CheckDType(uniform, kOpName, "uniform", MSCO_DTYPE_F32);
  CheckDType(draft_lens, kOpName, "draft_lens", MSCO_DTYPE_I32);
  if (s.vocab <= 0 || s.vocab > (1 << 30) || s.batch > (1 << 24) || s.drafts > (1 << 20))
    MS_VALUE_ERROR << "For " << kOpName << ", bad sizes: batch " << s.batch << ", drafts " << s.drafts << ", vocab " << s.vocab
                   << ".";
  if (target.dim(0) != s.batch || target.dim(1) != s.drafts + 1)
    MS_VALUE_ERROR << "For " << kOpName << ", target_probs must be (" << s.batch << ", " << s.drafts + 1 << ", vocab).";
  if (draft.defined() && (draft.dim(0) != s.batch || draft.dim(1) != s.drafts || draft.dim(2) != s.vocab))
    MS_VALUE_ERROR << "For " << kOpName << ", draft_probs must be (" << s.batch << ", " << s.drafts << ", " << s.vocab << ").";
  if (uniform.dim(0) != s.batch || uniform.dim(1) != s.drafts + 1)
    MS_VALUE_ERROR << "For " << kOpName << ", uniform must be (" << s.batch << ", " << s.drafts + 1 << ").";
  CheckNumel(draft_lens, kOpName, "draft_lens", s.batch);
  const struct { const Tensor *t; const char *name; } all[] = {{&target, "target_probs"}, {&draft, "draft_probs"},
                                                              {&draft_tokens, "draft_tokens"}, {&uniform, "uniform"},
                                                              {&draft_lens, "draft_lens"}};
  for (const auto &v : all) CheckContiguous(*v.t, kOpName, v.name);
  return s;
}

int Launch(const Tensor &target, const Tensor &draft, const Tensor &draft_tokens, const Tensor &uniform,
           const Tensor &draft_lens, const Tensor &tokens, const Tensor &accepted, void *stream) {
  const Sizes s = Check(target, draft, draft_tokens, uniform, draft_lens);
  CheckProvided(tokens, kOpName, "tokens");
  CheckProvided(accepted, kOpName, "accepted");
  CheckDType(tokens, kOpName, "tokens", MSCO_DTYPE_I32);
  CheckDType(accepted, kOpName, "accepted", MSCO_DTYPE_I32);
  CheckNumel(tokens, kOpName, "tokens", s.batch * (s.drafts + 1));
  CheckNumel(accepted, kOpName, "accepted", s.batch);
  const struct { const Tensor *t; const char *name; } all[] = {
      {&target, "target_probs"}, {&draft, "draft_probs"}, {&draft_tokens, "draft_tokens"}, {&uniform, "uniform"},
      {&draft_lens, "draft_lens"}, {&tokens, "tokens"}, {&accepted, "accepted"}};
  for (const auto &v : all) {
    CheckContiguous(*v.t, kOpName, v.name);
    CheckOnDevice(*v.t, kOpName, v.name);
  }
  return msco_verify_draft_tokens(
      target.data(), draft.data(), target.dtype(), static_cast<const int32_t *>(draft_tokens.data()),
      static_cast<const int32_t *>(draft_lens.data()), static_cast<const float *>(uniform.data()),
      static_cast<int32_t *>(tokens.data()), static_cast<int32_t *>(accepted.data()), static_cast<int32_t>(s.batch),
      static_cast<int32_t>(s.drafts), static_cast<int32_t>(s.vocab), stream);
}

}  // namespace
}  // namespace ms_custom_ops

MS_CUSTOM_OPS_REGISTER_OP(verify_draft_tokens,
                          "verify_draft_tokens(target_probs, draft_probs, draft_tokens, uniform, draft_lens=None)")

extern "C" int ms_custom_ops_verify_draft_tokens_infer(const MsTensorDesc *target_probs, const MsTensorDesc *draft_probs,
                                                       const MsTensorDesc *draft_tokens, const MsTensorDesc *uniform,
                                                       const MsTensorDesc *draft_lens, int32_t *out_dtype,
                                                       int32_t *out_ndim, int64_t *out_shape) {
  using namespace ms_custom_ops;
  return GuardedCall(kOpName, [&] {
    const Sizes s = Check(Tensor(target_probs), Tensor(draft_probs), Tensor(draft_tokens), Tensor(uniform),
                          Tensor(draft_lens));
    if (out_dtype != nullptr) *out_dtype = MSCO_DTYPE_I32;
    if (out_ndim != nullptr) *out_ndim = 2;
    if (out_shape != nullptr) {
      out_shape[0] = s.batch;
      out_shape[1] = s.drafts + 1;
    }
    return MSCO_OK;
  });
}

extern "C" int ms_custom_ops_verify_draft_tokens(const MsTensorDesc *target_probs, const MsTensorDesc *draft_probs,
                                                 const MsTensorDesc *draft_tokens, const MsTensorDesc *uniform,
                                                 const MsTensorDesc *draft_lens, const MsTensorDesc *tokens,
                                                 const MsTensorDesc *accepted, void *stream) {
  using namespace ms_custom_ops;
  return GuardedCall(kOpName, [&] {
    return Launch(Tensor(target_probs), Tensor(draft_probs), Tensor(draft_tokens), Tensor(uniform), Tensor(draft_lens),
                  Tensor(tokens), Tensor(accepted), stream);
  });
}
