"""transformers integration: the "mi355x" ExpertsInterface key and install().

``register()`` adds ``"mi355x"`` to transformers' ExpertsInterface
(transformers/integrations/moe.py:481-506; class-wide registry of
utils/generic.py GeneralInterface).  ``install(model)`` then swaps every
Qwen3MoeTopKRouter-derived gate for its HIP counterpart in place (as
src/models/standard_moe.py:72-78 swaps in DeepSeekRouter) and selects the
experts implementation with ``model.set_experts_implementation("mi355x")``
(the call train.py:239-245 makes with "grouped_mm").  Both the per-layer
banks (Qwen3MoeSparseMoeBlock.experts) and the global shared bank
(GlobalMoEModel.global_experts) dispatch through that key unchanged.
"""
from __future__ import annotations

from torch import nn

from .experts import mi355x_experts_forward
from .library import KEEPS
from .router import MI355XDeepSeekRouter, MI355XTopKRouter, _RouterBase

EXPERTS_KEY = "mi355x"


def register() -> None:
    from transformers.integrations.moe import ExpertsInterface
    ExpertsInterface.register(EXPERTS_KEY, mi355x_experts_forward)


def swap_routers(model: nn.Module) -> int:
    """Replaces each router (a Qwen3MoeTopKRouter or subclass) by the HIP one.
    Routers carrying an ``expert_bias`` buffer become MI355XDeepSeekRouter.
    Parameters and buffers are shared, so state_dict keys are unchanged.
    Returns the number of routers swapped."""
    n = 0
    for parent in list(model.modules()):
        for name, child in list(parent.named_children()):
            if isinstance(child, (MI355XTopKRouter, MI355XDeepSeekRouter)):
                continue
            if not isinstance(child, _RouterBase):
                continue
            cls = MI355XDeepSeekRouter if hasattr(child, "expert_bias") else MI355XTopKRouter
            new = cls.from_router(child)
            new.train(child.training)
            setattr(parent, name, new)
            n += 1
    return n


def expert_banks(model: nn.Module) -> list[nn.Module]:
    """The modules that hold an expert bank (gate_up_proj and down_proj)."""
    return [m for m in model.modules()
            if hasattr(m, "gate_up_proj") and hasattr(m, "down_proj")
            and getattr(m.gate_up_proj, "ndim", 0) == 3]


def install(model: nn.Module, routers: bool = True, experts: bool = True,
            few_tokens: int = 0, saved_activations: str = "exact") -> nn.Module:
    """Swaps the routers and selects the "mi355x" experts.  ``few_tokens``
    (with ``experts``): calls of at most that many tokens (up to
    ``moe_amd.few.MAX_TOKENS``) that want no gradient run the few-token
    experts.  ``saved_activations`` (with ``experts``): what the experts keep
    for their backward, as ``experts_forward`` takes it: other than "exact", calls
    that want a gradient take bf16 experts only."""
    if saved_activations not in KEEPS:
        raise ValueError(f"unknown saved_activations {saved_activations!r} (expected one of "
                         f"{KEEPS})")
    register()
    if routers:
        swap_routers(model)
    if experts:
        model.set_experts_implementation(EXPERTS_KEY)
        for bank in expert_banks(model):
            bank.few_tokens = int(few_tokens)
            bank.saved_activations = saved_activations
    return model
