"""What StateSpaceMixer refuses: at once where it is built, and in a call before any state is replaced."""
import pytest
import torch

from tests.test_state_space_module import parts
from uniql_amd.state_space import StateSpaceMixer, StateSpaceStates

NAN = float("nan")


@pytest.mark.parametrize("change", [dict(dt_limit=(-0.1, 1.0)), dict(dt_limit=(1.0, 0.5)), dict(dt_limit=(NAN, 1.0)), dict(dt_limit=(0.0, NAN)),
                                    dict(dt_limit=(0.0,)), dict(eps=-1e-5), dict(eps=NAN)])
def test_limits(change):
    with pytest.raises(ValueError):
        StateSpaceMixer(**{**parts(), **change})


def test_parameters_of_more_axes_are_flat():
    args = parts()
    flat = StateSpaceMixer(**args)
    for name in ("conv_bias", "a_log", "d", "dt_bias", "norm_weight"):
        args[name] = args[name].view(-1, 1)
    other = StateSpaceMixer(**args)
    for name, t in flat.named_buffers():
        assert torch.equal(t, dict(other.named_buffers())[name]), name


def set_to(name, value):
    return lambda m, s: setattr(m, name, value)


def other_states(**kw):
    def change(m, s):
        s.ssm = torch.zeros(3, *{**dict(heads=4, p=6, n=8), **kw}.values(), device=s.ssm.device)
    return change


CHANGES = {"limits": set_to("dt_limit", (-0.1, 1.0)), "swapped limits": set_to("dt_limit", (1.0, 0.5)), "eps": set_to("eps", -1.0), "norm groups": set_to("norm_groups", 5),
           "norm weight": lambda m, s: setattr(m, "norm_weight", m.norm_weight.float()), "rates": lambda m, s: setattr(m, "a", m.a.half()),
           "skips": lambda m, s: setattr(m, "d", m.d[:3].contiguous()), "bias": lambda m, s: setattr(m, "dt_bias", m.dt_bias.view(2, 2)),
           "heads": other_states(heads=8, p=3), "width": other_states(p=5), "states": other_states(n=16),
           "type": lambda m, s: setattr(s, "ssm", s.ssm.double()), "places": lambda m, s: setattr(s, "ssm", s.ssm[:1].clone()),
           "device": lambda m, s: setattr(s, "ssm", s.ssm.cpu()), "alignment": lambda m, s: setattr(s, "ssm", torch.zeros(577, device=s.ssm.device)[1:].view(3, 4, 6, 8))}


@pytest.mark.gpu
@pytest.mark.parametrize("change", CHANGES)
@pytest.mark.parametrize("cu", [True, False])
def test_a_refused_call_leaves_the_states(gpu, change, cu):
    """and the next one, with what was wrong put right, is as if there had been none"""
    gen = torch.Generator().manual_seed(1)
    m = StateSpaceMixer(**parts()).to(gpu)
    h = torch.randn(3, 84, generator=gen).half().to(gpu)
    offsets = torch.tensor([0, 1, 3, 3] if cu else [0, 1, 2, 3], dtype=torch.int32, device=gpu)
    kw = dict(cu=offsets) if cu else {}
    states, mirror = StateSpaceStates.like(m, 3), StateSpaceStates.like(m, 3)
    want = m(h, mirror, **kw)
    own, ssm = (m.a, m.d, m.dt_bias, m.norm_weight, m.dt_limit, m.eps, m.norm_groups), states.ssm
    CHANGES[change](m, states)
    with pytest.raises(RuntimeError):
        m(h, states, **kw)
    assert not states.conv.any() and not states.ssm.any()
    (m.a, m.d, m.dt_bias, m.norm_weight, m.dt_limit, m.eps, m.norm_groups), states.ssm = own, ssm
    assert torch.equal(m(h, states, **kw), want)
    assert torch.equal(states.conv, mirror.conv) and torch.equal(states.ssm, mirror.ssm)
