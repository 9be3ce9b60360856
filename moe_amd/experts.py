"""The expert layer: permute -> grouped GEMM-1 + SwiGLU -> grouped GEMM-2 ->
combine, with a hand-written backward, all on the HIP kernels.

``experts_forward`` is the functional form, a call of the differentiable
custom op ``moe_amd::experts_fwd`` (fake and autograd registered, so
torch.compile traces it without a graph break, as the reference's backend
registers its grouped GEMM, integrations/moe.py:245-257; backward op
``moe_amd::experts_bwd``, formulas :226-242, the combine's backward fused
into GEMM-2's).  ``mi355x_experts_forward`` has the transformers
ExpertsInterface signature
``fn(self, hidden_states [T,H], top_k_index [T,K], top_k_weights [T,K])``
(transformers/integrations/moe.py:377-382) and reads the bank's
``gate_up_proj [E,2I,H]`` / ``down_proj [E,H,I]`` from ``self``.
"""
from __future__ import annotations

import functools
import inspect

import torch

from torch import nn

from . import few, library, ops  # library registers the moe_amd:: ops


def traced_with_defaults(fn):
    """torch.fx's tracers (make_fx) want a value for each parameter that a
    function declares, those with a default too; of one that takes any arguments
    they take as many as they are given.  So a new option with a default does not
    refuse the traces that do without it."""
    @functools.wraps(fn)
    def call(*args, **kwargs):
        return fn(*args, **kwargs)
    del call.__wrapped__  # the tracers count the innermost function's parameters
    call.__signature__ = inspect.signature(fn)
    return call


@traced_with_defaults
def experts_forward(hidden_states: torch.Tensor, top_k_index: torch.Tensor,
                    top_k_weights: torch.Tensor, gate_up_proj: torch.Tensor | ops.Packed4,
                    down_proj: torch.Tensor | ops.Packed4,
                    saved_activations: str = "exact") -> torch.Tensor:
    """out[t] = sum_k w[t,k] * down_e(silu(gate_e(x_t)) * up_e(x_t)), e = idx[t,k].

    ``saved_activations`` (bf16 layers): what the backward finds of the
    activations.  "exact": gate_up [S,2I] and the hidden states as they are.
    "int8": gate_up in 8 bits (half the memory; ``ops.pack8``'s values), packed
    where GEMM-1 leaves it and read so by the backward: the gradients are those
    of the restored gate_up, the output is the same.  "int8_all": the hidden
    states too, for d_gate_up_proj; worth it where nothing else keeps them.

    A bank in 4 bits (``ops.Packed4`` for both weights; bf16 layers) is forward
    only: calls that want a gradient are refused.

    hidden_states is cast to the weights' dtype (as transformers' _grouped_mm
    does, integrations/moe.py:330-335) and the result is returned in
    hidden_states' dtype (:478)."""
    if hidden_states.dim() != 2:
        raise ValueError("hidden_states must be [T, H]")
    if isinstance(gate_up_proj, ops.Packed4) or isinstance(down_proj, ops.Packed4):
        return _experts_forward4(hidden_states, top_k_index, top_k_weights, gate_up_proj,
                                 down_proj, saved_activations)
    if gate_up_proj.dim() != 3 or down_proj.dim() != 3:
        raise ValueError("gate_up_proj must be [E, 2I, H] and down_proj [E, H, I]")
    E, I2, H = gate_up_proj.shape
    if down_proj.shape != (E, H, I2 // 2) or hidden_states.shape[1] != H:
        raise ValueError(
            f"shape mismatch: hidden {tuple(hidden_states.shape)}, gate_up_proj "
            f"{tuple(gate_up_proj.shape)}, down_proj {tuple(down_proj.shape)}")
    if top_k_index.shape != top_k_weights.shape or top_k_index.shape[0] != hidden_states.shape[0]:
        raise ValueError("top_k_index / top_k_weights must both be [T, K]")
    library.check_keep(saved_activations, gate_up_proj.dtype)
    out_dtype = hidden_states.dtype
    x = hidden_states.to(gate_up_proj.dtype).contiguous()
    w = top_k_weights.contiguous()
    save = torch.is_grad_enabled() and any(t.requires_grad
                                           for t in (x, w, gate_up_proj, down_proj))
    out = torch.ops.moe_amd.experts_fwd(x, top_k_index, w, gate_up_proj.contiguous(),
                                        down_proj.contiguous(), save, saved_activations)[0]
    return out.to(out_dtype)


def _experts_forward4(hidden_states, top_k_index, top_k_weights, gate_up_proj, down_proj,
                      saved_activations):
    library.check_keep(saved_activations, gate_up_proj.dtype)
    refuse_grad4("experts_forward", hidden_states, top_k_weights, gate_up_proj, down_proj)
    x = hidden_states.to(torch.bfloat16)
    if few._unseen(x, top_k_index, top_k_weights, *few._tensors4(gate_up_proj, down_proj)):
        out = ops.experts4(x, top_k_index, top_k_weights, gate_up_proj, down_proj)
    else:
        bank, *_ = ops.packed_bank("experts_forward", x, gate_up_proj, down_proj)
        if top_k_index.dim() != 2 or top_k_index.shape != top_k_weights.shape \
                or top_k_index.shape[0] != x.shape[0]:
            raise ValueError("top_k_index / top_k_weights must both be [T, K]")
        out = torch.ops.moe_amd.experts_fwd4(x, top_k_index, top_k_weights, *bank)
    return out.to(hidden_states.dtype)


def refuse_grad4(name: str, *tensors: torch.Tensor) -> None:
    """A bank in 4 bits has no backward."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f"{name}: a bank in 4 bits is forward only: call it under "
                           "torch.no_grad()")


def _check_module(self) -> None:
    if not getattr(self, "has_gate", True):
        raise NotImplementedError("mi355x experts: only gated (gate_up_proj) experts are supported")
    if getattr(self, "has_bias", False):
        raise NotImplementedError("mi355x experts: expert biases are not supported")
    if getattr(self, "is_transposed", False):
        raise NotImplementedError("mi355x experts: transposed expert weights are not supported")
    if not getattr(self, "is_concatenated", True):
        raise NotImplementedError("mi355x experts: interleaved gate/up layout is not supported")
    act = getattr(self, "act_fn", None)
    name = type(act).__name__.lower() if act is not None else "silu"
    if "silu" not in name and "swish" not in name:
        raise NotImplementedError(f"mi355x experts: activation {type(act).__name__} is not SiLU")


_BANK = ("gate_up_proj", "down_proj")


def is_packed_bank(bank: nn.Module) -> bool:
    return hasattr(bank, "packed_shapes")


def check_packable(bank: nn.Module) -> None:
    """Raises unless the experts take the bank in 4 bits."""
    _check_module(bank)
    weights = [getattr(bank, name) for name in _BANK]
    for name, w in zip(_BANK, weights):
        if w.dtype != torch.bfloat16:
            raise NotImplementedError(f"pack_bank: {name} of {w.dtype}; banks in 4 bits take bf16 "
                                      "layers")
        if w.dim() != 3 or w.shape[1] % 64 or w.shape[2] % 64:
            raise ValueError(f"pack_bank: {name} {tuple(w.shape)}: both of its dimensions must be "
                             "multiples of 64")
    shape1, shape2 = (tuple(w.shape) for w in weights)
    E, I2, H = shape1
    if shape2 != (E, H, I2 // 2):
        raise ValueError(f"pack_bank: gate_up_proj {shape1} and down_proj {shape2}, expected "
                         "[E, 2I, H] and [E, H, I]")
    ops.check_bank4_size("pack_bank", E, H, I2 // 2)


def pack_bank(bank: nn.Module) -> nn.Module:
    """Replaces a bank's parameters gate_up_proj and down_proj (bf16, on the GPU) by
    their 4 bits, in place: buffers gate_up_proj_q, gate_up_proj_scale and down_proj's,
    which state_dict holds and ``to`` moves.  The bank is forward only from then on."""
    if is_packed_bank(bank):
        return bank
    check_packable(bank)
    packed = [ops.pack4(getattr(bank, name).detach()) for name in _BANK]
    for name, p in zip(_BANK, packed):
        delattr(bank, name)
        bank.register_buffer(f"{name}_q", p.q)
        bank.register_buffer(f"{name}_scale", p.scale)
    bank.packed_shapes = tuple(p.shape for p in packed)
    return bank


def bank_weights(bank: nn.Module):
    """(gate_up_proj, down_proj) of a bank: its parameters, or its weights in 4
    bits."""
    if not is_packed_bank(bank):
        return bank.gate_up_proj, bank.down_proj
    return tuple(ops.Packed4(getattr(bank, f"{name}_q"), getattr(bank, f"{name}_scale"), shape,
                             torch.bfloat16) for name, shape in zip(_BANK, bank.packed_shapes))


def mi355x_experts_forward(self, hidden_states: torch.Tensor, top_k_index: torch.Tensor,
                           top_k_weights: torch.Tensor) -> torch.Tensor:
    """ExpertsInterface entry ("mi355x"), drop-in for grouped_mm_experts_forward
    (transformers/integrations/moe.py:377-478).  A bank with a ``few_tokens``
    attribute runs the few-token experts up to that many tokens where no
    gradient is wanted, and a ``saved_activations`` attribute is
    experts_forward's (``hf.install`` sets both).  A bank that ``pack_bank`` packed
    runs on its weights in 4 bits."""
    _check_module(self)
    w1, w2 = bank_weights(self)
    if few.wanted(getattr(self, "few_tokens", 0), top_k_index.shape[-1], w1.shape[0],
                  hidden_states, top_k_weights, w1, w2):
        return few.experts_forward_few(hidden_states, top_k_index, top_k_weights, w1, w2)
    keep = library.keep_of_call(getattr(self, "saved_activations", "exact"), hidden_states,
                                top_k_weights, w1, w2)
    return experts_forward(hidden_states, top_k_index, top_k_weights, w1, w2, keep)
