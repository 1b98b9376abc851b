"""B200 (sm_100a) build of the Mamba-3 selective-scan hot path.

Drop-in for the scan path of the reference package ``mamba3_ssm`` (v0.2.1): the same
module and class names (ops.ssm_scan_siso / ssm_scan_mimo, Mamba3, MambaLMHeadModel,
MambaBlock, RMSNorm, apply_rope, MambaConfig, SSMConfig), with the scans, their backward
and the decode step running as hand-written CUDA kernels behind the C ABI of
libmamba3_b200.so. There is no CPU path.

For fine-tuning, on the same terms: losses over the model's logits (token_logprobs,
policy_loss, preference_loss) and the gradients' global norm and clipping (clip_grads_,
clip_grad_norm_).
"""

from .config import MambaConfig, SSMConfig
from .layer import Mamba3
from .block import MambaLMHeadModel, MambaBlock, DecodeGraph
from .ops import RMSNorm, apply_rope, ssm_scan_siso, ssm_scan_mimo
from .losses import PolicyLoss, PreferenceLoss, policy_loss, preference_loss, token_logprobs
from .grads import clip_grad_norm_, clip_grads_

__all__ = [
    "MambaConfig",
    "SSMConfig",
    "Mamba3",
    "MambaLMHeadModel",
    "MambaBlock",
    "DecodeGraph",
    "RMSNorm",
    "apply_rope",
    "ssm_scan_siso",
    "ssm_scan_mimo",
    "PolicyLoss",
    "PreferenceLoss",
    "policy_loss",
    "preference_loss",
    "token_logprobs",
    "clip_grad_norm_",
    "clip_grads_",
]
