"""The expert layer for a few tokens (a served model's decode step), forward
only: the experts with a caller's routing (``experts_forward_few``) and the
whole layer with its router (``moe_layer_few``), at most ``MAX_TOKENS`` tokens
a call.

Same functions of the same inputs as ``experts_forward`` and ``moe_layer``,
with fewer roundings on the way: gate, up and y stay fp32 and so do the routing
weights, where those round them to the layer's type.  Their kernels stream each
routed expert's weights once; ``SparseMoeBlock.few_tokens`` and
``hf.install(model, few_tokens=...)`` choose them by the number of tokens.
They may be captured in a HIP graph.

A bank in 4 bits (``ops.Packed4`` for both of gate_up_proj and down_proj; bf16 hidden
states) is streamed as it is, 0.27 of the bytes.
"""
from __future__ import annotations

import torch

from . import library, ops  # noqa: F401  (library registers the moe_amd:: ops)

MAX_TOKENS = ops.FEW_MAX_TOKENS


def wanted(few_tokens: int, top_k: int, num_experts: int, *tensors: torch.Tensor) -> bool:
    """Whether a layer that takes the few-token form up to ``few_tokens``
    tokens takes it for ``tensors``, its hidden states [T, H] and what else goes
    into it, the weights' last dimensions being H or I: it has the shape, and no
    gradient is wanted of any of them."""
    # (the number of tokens last, so that a trace in which it is data-dependent
    # is asked for it only where the answer depends on it)
    return (few_tokens > 0 and top_k <= ops.FEW_MAX_TOP_K and num_experts <= ops.FEW_MAX_EXPERTS
            and all(t.shape[-1] <= ops.FEW_MAX_FEATURES for t in tensors)
            and not _grad(*tensors) and 0 < tensors[0].shape[0] <= min(few_tokens, MAX_TOKENS))


def _grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _refuse_grad(name: str, *tensors) -> None:
    if _grad(*tensors):
        raise RuntimeError(f"{name} is forward only: call it under torch.no_grad(), or "
                           "experts_forward / moe_layer where a gradient is wanted")


# What the dispatcher adds to every tensor's own keys while no mode, tracer or
# function transform is active, in inference mode and outside of it.
_included = getattr(torch._C, "_dispatch_tls_local_include_set", None)


def _at_rest() -> tuple[int, ...]:
    if _included is None:
        return ()
    key = torch._C.DispatchKey
    inference = torch._C.DispatchKeySet(key.BackendSelect)
    return inference.raw_repr(), inference.add(key.ADInplaceOrView).raw_repr()


_AT_REST = _at_rest()
_PLAIN = (torch.Tensor, torch.nn.Parameter, type(None))


def _unseen(*tensors) -> bool:
    """Whether nothing but the kernels takes part in a call on ``tensors``: they
    are torch's own, and no fake or other dispatch mode, tracer or transform is
    active.  Such a call goes to the C entry at once, every other one through the
    dispatcher as the moe_amd:: op, which all of those see (20.5 us for one token
    of the experts where the direct call takes 16, the host bounding both; 1 us of
    it is this check)."""
    if torch.compiler.is_compiling() or _included is None \
            or _included().raw_repr() not in _AT_REST:
        return False
    for t in tensors:
        if type(t) not in _PLAIN or (t is not None and t.is_neg()):
            return False
    return True


def _tensors4(*weights):
    """The tensors of weights of which one at least is in 4 bits (both, else the
    call is refused)."""
    return [t for w in weights for t in ((w.q, w.scale) if type(w) is ops.Packed4 else (w,))]


def experts_forward_few(hidden_states: torch.Tensor, top_k_index: torch.Tensor,
                        top_k_weights: torch.Tensor, gate_up_proj: torch.Tensor | ops.Packed4,
                        down_proj: torch.Tensor | ops.Packed4) -> torch.Tensor:
    """``experts_forward`` for at most MAX_TOKENS tokens.  hidden_states are
    cast to the weights' dtype and the result back to theirs; ids outside
    [0, E) contribute nothing."""
    _refuse_grad("experts_forward_few", hidden_states, top_k_weights, gate_up_proj, down_proj)
    if isinstance(gate_up_proj, ops.Packed4) or isinstance(down_proj, ops.Packed4):
        dtype = hidden_states.dtype
        x = hidden_states if dtype == torch.bfloat16 else hidden_states.to(torch.bfloat16)
        if _unseen(x, top_k_index, top_k_weights, *_tensors4(gate_up_proj, down_proj)):
            out = ops.experts_few4(x, top_k_index, top_k_weights, gate_up_proj, down_proj)
        else:
            bank, *_ = ops.packed_bank("experts_forward_few", x, gate_up_proj, down_proj)
            out = torch.ops.moe_amd.experts_few4(x, top_k_index, top_k_weights, *bank)
        return out if dtype == torch.bfloat16 else out.to(dtype)
    op = (ops.experts_few if _unseen(hidden_states, top_k_index, top_k_weights, gate_up_proj,
                                     down_proj) else torch.ops.moe_amd.experts_few)
    dtype = hidden_states.dtype
    if dtype == gate_up_proj.dtype:
        return op(hidden_states, top_k_index, top_k_weights, gate_up_proj, down_proj)
    return op(hidden_states.to(gate_up_proj.dtype), top_k_index, top_k_weights, gate_up_proj,
              down_proj).to(dtype)


def moe_layer_few(x: torch.Tensor, w_router: torch.Tensor,
                  gate_up_proj: torch.Tensor | ops.Packed4,
                  down_proj: torch.Tensor | ops.Packed4, top_k: int, router: str = "softmax",
                  renormalize: bool = True, logit_offset: torch.Tensor | None = None,
                  expert_bias: torch.Tensor | None = None, scaling_factor: float | None = None,
                  num_groups: int | None = None, group_topk: int | None = None,
                  return_routing: bool = False):
    """``moe_layer`` for at most MAX_TOKENS tokens: out [T,H], or with
    ``return_routing`` (out, weights fp32 [T,K], index int64 [T,K]).  The
    softmax router decides on logits of x's dtype, the sigmoid router on fp32
    logits, as there, but on its own sums: where two logits lie within their
    roundings, another expert may be selected than there."""
    _refuse_grad("moe_layer_few", x, w_router, gate_up_proj, down_proj)
    rest = (int(top_k), router, bool(renormalize), logit_offset, expert_bias, scaling_factor,
            num_groups, group_topk)
    if isinstance(gate_up_proj, ops.Packed4) or isinstance(down_proj, ops.Packed4):
        if _unseen(x, w_router, logit_offset, expert_bias, *_tensors4(gate_up_proj, down_proj)):
            return ops.moe_layer_few4(x, w_router, gate_up_proj, down_proj, *rest,
                                      return_routing=return_routing)
        bank, *_ = ops.packed_bank("moe_layer_few", x, gate_up_proj, down_proj)
        res = torch.ops.moe_amd.moe_layer_few4(x, w_router, *bank, *rest)
        return res if return_routing else res[0]
    args = (x, w_router, gate_up_proj, down_proj, *rest)
    if _unseen(x, w_router, gate_up_proj, down_proj, logit_offset, expert_bias):
        return ops.moe_layer_few(*args, return_routing=return_routing)
    res = torch.ops.moe_amd.moe_layer_few(*args)
    return res if return_routing else res[0]
