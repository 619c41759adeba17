// Loss operators over rows of logits and their gradients: names, operand checks, launch plans.
//
// The reference's decomposer and op registry stop at softmax and the norms; these operators are what a training step
// puts behind them.  Every op has ONE result, as all ops here; the forward pass and the gradient over the same logits
// meet in one kernel when a program holds both (FusePasses merges them, MatchLossGroup takes the merged group).
#pragma once

#include <map>
#include <memory>
#include <string>
#include <vector>

#include "group_desc.h"

namespace cinn_b200 {

// token_logprob, token_logprob_grad, policy_loss, policy_loss_grad, distill_loss, distill_loss_grad, expert_counts,
// balance_part, balance_loss_grad.  (balance_loss is balance_part, followed by reduce_sum where the tokens make more than
// one part.)
bool IsLossOp(const std::string& op_type);

// Checks the operands and attributes of one loss op, fills in default attributes and the result's type and shape.
// False with *err set when something does not fit.
bool InferLossOp(const std::string& op_type, const std::vector<TensorDesc>& in,
                 std::map<std::string, std::string>* attrs, TensorDesc* out, std::string* err);

// The launch plan of a group that consists of loss ops; nullptr with *err set when no kernel takes it.
std::unique_ptr<CompiledGroup> MatchLossGroup(const GroupDesc& g, const DeviceInfo& dev, std::string* err);

}  // namespace cinn_b200
