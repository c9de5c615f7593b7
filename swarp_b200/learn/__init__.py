"""Policy training on the simulator's rollouts: advantages, the clipped policy loss and AdamW.

    advantages, returns = gae(rewards, values, None, terminated, truncated,
                              next_values=next_values)   # of info["final_obs"]
    out = policy_loss(logits, tokens, old_logp, advantages, mask=mask)
    out.loss.backward()
    optimizer.step()                                     # AdamW

Each is one or a few hand-written kernels behind the C ABI (include/swarp_b200.h); like the
step, they run on a CUDA device only, on torch's current stream, and are deterministic.
"""

from swarp_b200.learn.adamw import AdamW, Moment8, adamw_step
from swarp_b200.learn.advantage import gae
from swarp_b200.learn.policy import PolicyLoss, policy_loss, policy_loss_and_grad, token_logp

__all__ = ["AdamW", "Moment8", "PolicyLoss", "adamw_step", "gae", "policy_loss",
           "policy_loss_and_grad", "token_logp"]
