"""StateSpaceMixer and StateSpaceStates as far as they need no GPU."""
import copy
import pickle
from types import SimpleNamespace as NS

import pytest
import torch

from uniql_amd.state_space import StateSpaceMixer, StateSpaceStates


def parts(heads=4, p=6, groups=2, n=8, width=4):
    channels = heads * p + 2 * groups * n
    return dict(num_heads=heads, head_dim=p, n_groups=groups, state_size=n, conv_weight=torch.randn(channels, 1, width), conv_bias=torch.randn(channels),
                a_log=torch.randn(heads), d=torch.randn(heads), dt_bias=torch.randn(heads), norm_weight=torch.randn(heads * p), norm_groups=2)


def test_sizes_and_types():
    args = parts()
    m = StateSpaceMixer(**args)
    assert m.weight.shape == (56, 4) and m.weight.dtype == torch.float16
    assert torch.equal(m.a, -torch.exp(args["a_log"]))
    s = StateSpaceStates.like(m, 5)
    assert s.conv.shape == (5, 3, 56) and s.ssm.shape == (5, 4, 6, 8) and s.ssm.dtype == torch.float32


@pytest.mark.parametrize("change", [dict(head_dim=5), dict(n_groups=3), dict(state_size=257), dict(head_dim=129), dict(norm_groups=5), dict(norm_groups=0),
                                    dict(conv_weight=torch.zeros(56, 5)), dict(conv_weight=torch.zeros(55, 4)), dict(a_log=torch.zeros(3)),
                                    dict(dt_bias=torch.zeros(5)), dict(norm_weight=torch.zeros(23)), dict(conv_bias=torch.zeros(1))])
def test_refusals(change):
    with pytest.raises(ValueError):
        StateSpaceMixer(**{**parts(), **change})
    with pytest.raises(ValueError):
        StateSpaceStates(0, 4, 6, 2, 8)


def test_other_types_leave_the_sums_in_32_bits():
    m = StateSpaceMixer(**parts())
    rates, states = m.a.clone(), StateSpaceStates.like(m, 2)
    m.half(), states.half()
    assert m.a.dtype == m.d.dtype == m.dt_bias.dtype == states.ssm.dtype == torch.float32
    assert torch.equal(m.a, rates) and states.conv.dtype == torch.float16
    for other in (copy.deepcopy(m), pickle.loads(pickle.dumps(m))):
        assert torch.equal(other.a, rates) and other.dt_limit == m.dt_limit


def test_from_a_block():
    args = parts()
    block = NS(num_heads=4, head_dim=6, n_groups=2, ssm_state_size=8, conv1d=NS(weight=args["conv_weight"], bias=args["conv_bias"]), A_log=args["a_log"],
               D=args["d"], dt_bias=args["dt_bias"], norm=NS(weight=args["norm_weight"], variance_epsilon=1e-6, group_size=12), time_step_limit=(0.0, 0.5))
    m = StateSpaceMixer.from_block(block)
    assert m.norm_groups == 2 and m.eps == 1e-6 and m.dt_limit == (0.0, 0.5)
    block.norm = NS(weight=args["norm_weight"], eps=1e-5)
    assert StateSpaceMixer.from_block(block).norm_groups == 1
    assert StateSpaceMixer.from_block(block, norm_groups=4).norm_groups == 4


def test_no_gpu_no_result():
    m = StateSpaceMixer(**parts())
    with pytest.raises(RuntimeError, match="columns"):
        m(torch.zeros(3, 50, dtype=torch.float16))
    with pytest.raises(RuntimeError, match="GPU"):
        m(torch.zeros(3, 84, dtype=torch.float16))
