"""StateSpaceMixer.from_block takes a block for what it is, or refuses it."""
from types import SimpleNamespace as NS

import pytest
import torch

from tests.test_state_space_module import parts
from uniql_amd.state_space import StateSpaceMixer


def block(heads=8, p=54, groups=8, norm=None, **more):
    args = parts(heads, p, groups, 16)
    return NS(**{**dict(num_heads=heads, head_dim=p, n_groups=groups, ssm_state_size=16, conv1d=NS(weight=args["conv_weight"], bias=args["conv_bias"]),
                        A_log=args["a_log"], D=args["d"], dt_bias=args["dt_bias"],
                        norm=NS(**{**dict(weight=args["norm_weight"], eps=1e-5), **(norm or {})})), **more})


def test_cut_blocks_that_kept_their_norms_group_size():
    """heads of 64 cut to 54 and 56, groups of 64 and 512: the norm's groups are still the block's eight (or one), not what the old size divides into"""
    for p, size in ((54, 64), (56, 64), (54, 512), (32, 64)):
        cut = block(p=p, norm=dict(group_size=size))
        with pytest.raises(ValueError, match="norm_groups"):
            StateSpaceMixer.from_block(cut)
        assert StateSpaceMixer.from_block(cut, norm_groups=8).norm_groups == 8
    with pytest.raises(ValueError, match="norm_groups"):
        StateSpaceMixer.from_block(block(norm=dict(n_groups=4)))


@pytest.mark.parametrize("norm,groups", [(dict(group_size=54), 8), (dict(group_size=432), 1), (dict(group_size=None), 1), (dict(n_groups=8), 8), (dict(n_groups=1), 1),
                                         (dict(n_groups=None), 1), (dict(), 1)])
def test_norm_groups(norm, groups):
    m = StateSpaceMixer.from_block(block(norm=norm))
    assert m.norm_groups == groups and isinstance(m.norm_groups, int)


@pytest.mark.parametrize("more", [dict(norm_before_gate=True), dict(norm=dict(norm_before_gate=True)), dict(activation="gelu"), dict(activation="relu"),
                                  dict(norm=dict(activation="sigmoid"))])
def test_blocks_that_compute_something_else(more):
    with pytest.raises(ValueError):
        StateSpaceMixer.from_block(block(**more))
    with pytest.raises(ValueError):
        StateSpaceMixer.from_block(block(**more), norm_groups=8)


def test_blocks_that_say_what_they_compute():
    for more in (dict(activation="silu"), dict(activation="swish"), dict(activation=torch.nn.SiLU()), dict(norm_before_gate=False),
                 dict(norm=dict(norm_before_gate=False, activation="swish"))):
        StateSpaceMixer.from_block(block(**more))
