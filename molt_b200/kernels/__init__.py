from molt_b200.kernels.gated_activation import enable_fused_silu_mlp, fused_silu_multiply
from molt_b200.kernels.grad_norm import clip_grad_norm, global_grad_norm
from molt_b200.kernels.policy_loss import PolicyLoss, PreferenceLoss, clipped_policy_loss, preference_loss
from molt_b200.kernels.token_logprobs import token_logprobs, token_logprobs_with_grad

__all__ = ["PolicyLoss", "PreferenceLoss", "clip_grad_norm", "clipped_policy_loss", "enable_fused_silu_mlp",
           "fused_silu_multiply", "global_grad_norm", "preference_loss", "token_logprobs", "token_logprobs_with_grad"]
