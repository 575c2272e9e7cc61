"""What stands between the input and the output projection of a state-space layer (Mamba2 and the layers of that kind in Bamba and Nemotron-H):
causal convolution, linear attention with a decay for each head, gated norm.  (The reference calls third-party kernels there,
modeling/mamba/mamba2_qblocks.py.)

    mixer = StateSpaceMixer.from_block(block)                    # the reference's block: conv1d, dt_bias, A_log, D, norm
    states = StateSpaceStates.like(mixer, max_requests, device="cuda")
    ...
    h = block.in_proj(x)                                         # rows in the order of the requests
    h = mixer(h, states, cu=step.cu, starts=lengths_before)      # prompts, pieces of prompts and single tokens in one batch
    x = block.out_proj(h, residual=x)

With attention layers in the model, `cu` is KVStep.cu, and `starts` a copy of what KVPages.lengths held before the step.  Requests that KVPages
refused keep their rows there, and are left out with
    places = torch.where(step.refused > 0, -1, torch.arange(max_requests, dtype=torch.int32, device="cuda"))
All of it runs from what is on the device and can be
recorded into a graph.  Nothing is recorded for autograd."""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _capi, ops


class StateSpaceStates(nn.Module):
    """The states of one layer, a place for each request: `conv` fp16 [places, conv_width - 1, channels], the last inputs of the convolution, and
    `ssm` float [places, heads, head_dim, states]."""

    def __init__(self, places, num_heads, head_dim, n_groups, state_size, conv_width=4, device=None):
        super().__init__()
        if places < 1:
            raise ValueError("there must be at least one place")
        channels = num_heads * head_dim + 2 * n_groups * state_size
        self.register_buffer("conv", torch.zeros(places, conv_width - 1, channels, dtype=torch.float16, device=device), persistent=False)
        self.register_buffer("ssm", torch.zeros(places, num_heads, head_dim, state_size, dtype=torch.float32, device=device), persistent=False)

    def _apply(self, fn, recurse=True):
        # .half() and .to(dtype) are for what a layer multiplies with; sums stay in 32 bits
        ssm = self.ssm
        super()._apply(fn, recurse)
        if self.ssm.dtype != ssm.dtype:
            self.ssm = ssm.to(self.ssm.device)
        return self

    @classmethod
    def like(cls, mixer: "StateSpaceMixer", places: int, device=None) -> "StateSpaceStates":
        return cls(places, mixer.num_heads, mixer.head_dim, mixer.n_groups, mixer.state_size, mixer.conv_width,
                   mixer.weight.device if device is None else device)

    def __repr__(self):
        return f"StateSpaceStates(places={self.ssm.shape[0]}, ssm={tuple(self.ssm.shape[1:])}, conv={tuple(self.conv.shape[1:])})"


class StateSpaceMixer(nn.Module):
    """From in_proj's output z | x | b | c | dt to out_proj's input.  Sizes may be pruned: head_dim 1 to 128, state_size 1 to 256.

    conv_weight [channels, 2 to 4] (or as nn.Conv1d has it, [channels, 1, width]), conv_bias [channels] or None, over x | b | c;
    a_log, d, dt_bias [heads]; norm_weight [heads * head_dim], norm_groups: ranges of channels that are normalised apart."""

    def __init__(self, num_heads, head_dim, n_groups, state_size, conv_weight, conv_bias, a_log, d, dt_bias, norm_weight, norm_groups=1, eps=1e-5,
                 dt_limit=(0.0, float("inf"))):
        super().__init__()
        self.num_heads, self.head_dim, self.n_groups, self.state_size = num_heads, head_dim, n_groups, state_size
        self.inner = num_heads * head_dim
        self.channels = self.inner + 2 * n_groups * state_size
        if not (1 <= head_dim <= 128 and 1 <= state_size <= 256):
            raise ValueError("heads must be 1 to 128 wide, with 1 to 256 states")
        if n_groups < 1 or num_heads % n_groups:
            raise ValueError("the heads must be a multiple of the groups")
        if norm_groups < 1 or self.inner % norm_groups:
            raise ValueError("norm_groups must divide the channels of all heads")
        weight = conv_weight.detach().reshape(conv_weight.shape[0], -1)
        if weight.shape[0] != self.channels or not 2 <= weight.shape[1] <= 4:
            raise ValueError(f"the convolution must have {self.channels} channels and a width of 2 to 4")
        for name, t, size in (("conv_bias", conv_bias, self.channels), ("a_log", a_log, num_heads), ("d", d, num_heads), ("dt_bias", dt_bias, num_heads),
                              ("norm_weight", norm_weight, self.inner)):
            if t is not None and t.numel() != size:
                raise ValueError(f"{name} must have {size} entries")
        if not eps >= 0.0:
            raise ValueError("eps must not be negative")
        if len(dt_limit) != 2 or not 0.0 <= dt_limit[0] <= dt_limit[1]:
            raise ValueError("dt_limit must be two numbers from 0 on, the smaller one first")
        self.conv_width, self.norm_groups, self.eps, self.dt_limit = weight.shape[1], norm_groups, eps, tuple(dt_limit)
        conv_bias, a_log, d, dt_bias, norm_weight = (None if t is None else t.detach().reshape(-1) for t in (conv_bias, a_log, d, dt_bias, norm_weight))
        half = dict(dtype=torch.float16)
        self.register_buffer("weight", weight.to(**half).contiguous())
        self.register_buffer("bias", None if conv_bias is None else conv_bias.to(**half).contiguous())
        self.register_buffer("a", -torch.exp(a_log.float()).contiguous())
        self.register_buffer("d", None if d is None else d.float().contiguous())
        self.register_buffer("dt_bias", None if dt_bias is None else dt_bias.float().contiguous())
        self.register_buffer("norm_weight", norm_weight.to(**half).contiguous())

    def _apply(self, fn, recurse=True):
        # .half() and .to(dtype) leave rates, skips and biases of the time step in 32 bits
        held = {name: self._buffers[name] for name in ("a", "d", "dt_bias") if self._buffers[name] is not None}
        super()._apply(fn, recurse)
        for name, t in held.items():
            if self._buffers[name].dtype != t.dtype:
                self._buffers[name] = t.to(self._buffers[name].device)
        return self

    @classmethod
    def from_block(cls, block, norm_groups=None) -> "StateSpaceMixer":
        """Of a block with the reference's attributes (num_heads, head_dim, n_groups, ssm_state_size, conv1d, A_log, D, dt_bias, norm), whole
        or cut (slicing.slice_conv1d, slice_norm).  norm_groups: the norm's own when None (group_size or n_groups of it), or one.  Refused are
        blocks that compute something else - another activation, the norm in front of the gate - and, without norm_groups, a norm whose
        group_size gives neither one group nor the block's n_groups, as that of a cut block does which kept the size of before."""
        inner = block.num_heads * block.head_dim
        for part in (block, block.norm):
            if getattr(part, "norm_before_gate", False):
                raise ValueError("the gate comes in front of the norm here, not behind it")
            activation = getattr(part, "activation", None)
            if isinstance(activation, str) and activation not in ("silu", "swish"):
                raise ValueError(f"the activation must be silu, not {activation}")
        if norm_groups is None:
            size = getattr(block.norm, "group_size", None)
            norm_groups = inner / size if size else getattr(block.norm, "n_groups", None) or 1
            if norm_groups not in (1, block.n_groups):
                raise ValueError(f"the norm's groups ({norm_groups:g} over {inner} channels) are neither one nor the block's {block.n_groups}: give norm_groups")
            norm_groups = int(norm_groups)
        eps = getattr(block.norm, "variance_epsilon", getattr(block.norm, "eps", 1e-5))
        return cls(block.num_heads, block.head_dim, block.n_groups, block.ssm_state_size, block.conv1d.weight, block.conv1d.bias, block.A_log, block.D,
                   block.dt_bias, block.norm.weight, norm_groups, eps, getattr(block, "time_step_limit", (0.0, float("inf"))))

    def forward(self, projected: torch.Tensor, states: StateSpaceStates | None = None, cu: torch.Tensor | None = None,
                places: torch.Tensor | None = None, starts: torch.Tensor | None = None) -> torch.Tensor:
        """projected fp16 [..., inner + channels + heads], in_proj's output (rows may be longer).  cu, places and starts: as for ops.causal_conv;
        without cu every row is one more token of a request, without states every sequence begins and ends in the call.
        Returns fp16 [..., inner]; rows in no sequence hold nothing of meaning.  A refused call leaves all states as they were."""
        width = self.inner + self.channels + self.num_heads
        if projected.shape[-1] < width:
            raise RuntimeError(f"projected has {projected.shape[-1]} columns, z | x | b | c | dt take {width}")
        rows = projected.reshape(-1, projected.shape[-1])
        z, mixed, dt = rows[:, :self.inner], rows[:, self.inner:self.inner + self.channels], rows[:, self.inner + self.channels:width]
        conv, ssm = (None, None) if states is None else (states.conv, states.ssm)
        if states is not None:
            _capi.host().check_state_space_layer(rows, self.a, self.d, self.dt_bias, *self.dt_limit, ssm, cu, places, starts, self.norm_weight,
                                                 self.norm_groups, self.eps, self.num_heads, self.head_dim, self.n_groups, self.state_size)
        mixed = ops.causal_conv(mixed, self.weight, self.bias, state=conv, cu=cu, places=places, starts=starts)
        x, b, c = mixed.split((self.inner, self.n_groups * self.state_size, self.n_groups * self.state_size), dim=1)
        y = ops.state_space_scan(x.unflatten(1, (self.num_heads, self.head_dim)), dt, self.a, b.unflatten(1, (self.n_groups, self.state_size)),
                                 c.unflatten(1, (self.n_groups, self.state_size)), d=self.d, dt_bias=self.dt_bias, dt_limit=self.dt_limit, state=ssm,
                                 cu=cu, places=places, starts=starts)
        y = y.flatten(1)
        return ops.gated_group_norm(y, z, self.norm_weight, self.norm_groups, self.eps, out=y).view(*projected.shape[:-1], self.inner)

    def __repr__(self):
        return (f"StateSpaceMixer(num_heads={self.num_heads}, head_dim={self.head_dim}, n_groups={self.n_groups}, state_size={self.state_size}, "
                f"conv_width={self.conv_width}, norm_groups={self.norm_groups})")
