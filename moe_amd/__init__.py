"""moe_amd — MI355X (gfx950) HIP implementation of the Qwen3-MoE expert layer.

Public API:
  experts_forward(hidden_states, top_k_index, top_k_weights, gate_up_proj, down_proj)
  mi355x_experts_forward(self, hidden_states, top_k_index, top_k_weights)   # ExpertsInterface
  few.moe_layer_few / few.experts_forward_few                                 # a few tokens, forward
  ops.pack4 / hf.pack_experts: expert banks in 4 bits, which the three above take, forward
  MI355XTopKRouter / MI355XDeepSeekRouter                                     # router modules
  hf.register() / hf.install(model)                                           # transformers hook
  ops.*                                                                       # one wrapper per C entry
  torch.ops.moe_amd.*                                                         # custom ops (library.py)
"""
from . import few, library, ops
from .experts import experts_forward, mi355x_experts_forward
from .router import MI355XDeepSeekRouter, MI355XTopKRouter

__all__ = [
    "few",
    "ops",
    "library",
    "experts_forward",
    "mi355x_experts_forward",
    "MI355XTopKRouter",
    "MI355XDeepSeekRouter",
]
