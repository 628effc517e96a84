"""A causal spiking attention block over token streams.

Spikformer's spiking self-attention (``patterns.FusedSSA``) attends without a
softmax and sees all tokens of an image at once.  ``DecayAttentionLIF`` is the form
for streams: one fused q/k/v projection, a norm and rotation of queries and keys
(``ops.qk_norm_rope``), attention through a state per head that leaks from token to
token (``ops.decay_attention`` for prompts, ``ops.decay_attention_step`` for single
tokens), an output projection, and a LIF neuron whose time axis is the token axis
(``ops.lif_fwd``).  The attention states and the membrane are carried from call to
call until ``reset()``, so a prompt may come whole, in pieces, or token by token;
another number of streams needs a ``reset()``.

    python -m catfuse_b200.decay_block      # a prompt, then tokens, timed
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from . import ops
from .state import StateBuffer

__all__ = ["DecayAttentionLIF"]


class DecayAttentionLIF(nn.Module):
    """x [B, L, dim] -> spikes [B, L, dim] (``forward``), x [B, dim] -> [B, dim] (``step``).

    ``heads`` query heads of ``head_dim`` share ``kv_heads`` states.  ``sections``
    gives the rotated pairs of each position axis (one axis: text; three: time,
    height and width of a patch stream); positions are [B, L] or [axes, B, L].
    The decays run from e^-1 to e^-1/512 over the states.  ``dtype`` (fp16 or bf16, also
    by ``.half()`` or ``.to(dtype)``) is that of the projections and what lies between."""

    def __init__(self, dim: int, heads: int, kv_heads: Optional[int] = None,
                 head_dim: Optional[int] = None, sections=None, axis_order: str = "blocks",
                 lif: ops.LIFConfig = ops.LIFConfig(), dtype=torch.bfloat16):
        super().__init__()
        self.heads, self.kv_heads = heads, kv_heads or heads
        self.head_dim = head_dim or dim // heads
        self.sections, self.axis_order, self.lif = sections, axis_order, lif
        width = self.heads * self.head_dim
        self.qkv = nn.Linear(dim, width + 2 * self.kv_heads * self.head_dim, bias=False, dtype=dtype)
        self.proj = nn.Linear(width, dim, bias=False, dtype=dtype)
        pairs = sum(sections) if sections else self.head_dim // 2
        self.register_buffer("inv_freq", 10000.0 ** (-torch.arange(pairs, dtype=torch.float32) / pairs))
        self.register_buffer("log_decay", -torch.exp2(torch.linspace(0.0, -9.0, self.kv_heads)))
        self.q_weight = nn.Parameter(torch.ones(self.head_dim))
        self.k_weight = nn.Parameter(torch.ones(self.head_dim))
        self.state, self.membrane = StateBuffer(), StateBuffer()

    def _apply(self, fn, recurse=True):
        # what the operators take in fp32 stays in fp32 under .half() and .to(dtype)
        names = ("inv_freq", "log_decay", "q_weight", "k_weight")
        kept = {n: getattr(self, n).data for n in names}
        super()._apply(fn, recurse)
        for n in names:
            t = getattr(self, n)
            if t.dtype != torch.float32:
                t.data = kept[n].to(t.device)
        return self

    def reset(self) -> None:
        self.state.reset()
        self.membrane.reset()

    def _check_streams(self, x) -> int:
        """The batch, which must be that of the carried states."""
        B, held = x.shape[0], self.state.tensor
        if held is not None and (held.shape[0] != B or held.device != x.device):
            raise ValueError(f"the block carries the states of {held.shape[0]} streams on {held.device}, got "
                             f"{B} on {x.device}: call reset() first")
        return B

    def _project(self, x, positions):
        h, hk, d = self.heads, self.kv_heads, self.head_dim
        qkv = self.qkv(x.to(self.qkv.weight.dtype))
        q, k, v = (t.unflatten(-1, (-1, d)) for t in qkv.split((h * d, hk * d, hk * d), -1))
        q, k = ops.qk_norm_rope(q, k, positions, self.inv_freq, q_weight=self.q_weight,
                                k_weight=self.k_weight, sections=self.sections, axis_order=self.axis_order)
        return q, k, v

    def _fire(self, y):
        """LIF over the tokens of y [L, B, dim]."""
        z = self.proj(y).float().contiguous()
        v0 = self.membrane.tensor
        spikes, v = ops.lif_fwd(z, v0, self.lif)
        self.membrane.set(v)
        return spikes

    @torch.no_grad()
    def forward(self, x: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        B = self._check_streams(x)
        if x.shape[1] == 0:  # nothing to attend to: states and membrane stay as they are
            return x.new_zeros(x.shape, dtype=torch.float32)
        q, k, v = self._project(x, positions)
        s = self.state.get((B, self.kv_heads, self.head_dim, self.head_dim), x.device)
        y = ops.decay_attention(q, k, v, self.log_decay, s_in=s, s_out=s)
        return self._fire(y.flatten(-2).transpose(0, 1)).transpose(0, 1)

    @torch.no_grad()
    def step(self, x: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        B = self._check_streams(x)
        q, k, v = self._project(x, positions)
        s = self.state.get((B, self.kv_heads, self.head_dim, self.head_dim), x.device)
        y = ops.decay_attention_step(q, k, v, self.log_decay, s)
        return self._fire(y.flatten(-2)[None])[0]


def main() -> int:
    torch.manual_seed(0)
    B, L, dim, tokens = 4, 2048, 1024, 64
    block = DecayAttentionLIF(dim, heads=8, lif=ops.LIFConfig(v_threshold=0.5)).cuda()
    x = torch.randn(B, L + tokens, dim, device="cuda")
    pos = torch.arange(L + tokens, device="cuda", dtype=torch.int32).repeat(B, 1)
    whole = block(x, pos)
    for _ in range(3):  # the last one counts
        block.reset()
        marks = [torch.cuda.Event(enable_timing=True) for _ in range(3)]
        marks[0].record()
        parts = [block(x[:, :L], pos[:, :L].contiguous())]
        marks[1].record()
        for t in range(L, L + tokens):
            parts.append(block.step(x[:, t], pos[:, t].contiguous())[:, None])
        marks[2].record()
        torch.cuda.synchronize()
    same = (torch.cat(parts, 1) == whole).float().mean().item()
    print(f"prompt of {B} x {L} tokens: {marks[0].elapsed_time(marks[1]):.3f} ms, "
          f"{marks[1].elapsed_time(marks[2]) / tokens * 1e3:.0f} us a token after it; spike rate "
          f"{whole.mean().item():.3f}, {same:.6f} of the spikes as in one prompt")
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
