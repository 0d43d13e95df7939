"""CPU tests of the optimizer's own arithmetic: what needs no kernel."""
import math

import pytest
import torch

from fusiongpu_b200.adapter import Muon


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d", [0.02 * 0.05, 0.02 * 0.1, 1e-4, 3e-8, 0.01])
def test_small_decay_is_not_lost(dtype, d):
    """(1 - d)^n of every element.  Each factor of 1 - `due` is off by eps / 2 of the value
    at most, where at least `due` (4 eps, or d if that is eps or more) is taken at a time;
    less than 4 eps + d is still held back."""
    eps = torch.finfo(dtype).eps
    p = torch.nn.Parameter((torch.rand(60, 40, generator=torch.Generator().manual_seed(1)) + 0.5).to(dtype))
    start, opt = p.detach().double(), Muon([p])
    n = min(3000, math.ceil(1.0 / d))
    with torch.no_grad():
        for _ in range(n):
            opt._decay(p, d)
    want = n * math.log1p(-d)
    got = torch.log(p.detach().double() / start)
    due = d if d >= eps else 4 * eps
    assert float((got - want).abs().max()) <= 1.02 * eps / 2 / due * abs(want) + 4 * eps + d


def test_decay_that_is_resolved_is_taken_at_once():
    for dtype, d in ((torch.bfloat16, 0.01), (torch.float16, 0.002), (torch.float32, 1e-6)):
        p = torch.nn.Parameter(torch.randn(30, 20, generator=torch.Generator().manual_seed(2)).to(dtype))
        want = p.detach().clone().mul_(1 - d)
        opt = Muon([p])
        with torch.no_grad():
            opt._decay(p, d)
        assert torch.equal(p, want) and "decay" not in opt.state[p]


def test_decay_held_back_is_saved_with_the_state():
    p = torch.nn.Parameter(torch.ones(4, 8, dtype=torch.bfloat16))
    opt = Muon([p])
    with torch.no_grad():
        opt._decay(p, 1e-3)
    again = Muon([p])
    again.load_state_dict(opt.state_dict())
    assert again.state[p]["decay"] == opt.state[p]["decay"] == 1 - 1e-3


def _matrix(*shape, **kw):
    p = torch.nn.Parameter(torch.ones(*shape, **kw))
    p.grad = torch.ones_like(p)
    return p


def test_added_groups_are_checked():
    from fusiongpu_b200._lib import FgError
    opt = Muon([_matrix(4, 8)])
    for bad in (_matrix(8), _matrix(2, 3, 4), _matrix(4, 8, dtype=torch.float64)):
        with pytest.raises(ValueError):
            opt.add_param_group(dict(params=[bad]))
        with pytest.raises(ValueError):
            Muon([dict(params=[_matrix(4, 8)]), dict(params=[bad])])
    for kw in (dict(lr=-1.0), dict(lr=math.nan), dict(momentum=1.0), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            opt.add_param_group(dict(params=[_matrix(4, 8)], **kw))
        with pytest.raises(ValueError):
            Muon([dict(params=[_matrix(4, 8)], **kw)])
    for kw in (dict(steps=101), dict(eps=-1.0), dict(coefficients=(17.0, 0.0, 0.0))):
        with pytest.raises(FgError):
            opt.add_param_group(dict(params=[_matrix(4, 8)], **kw))
    for shape in ((0, 8), (1, 32769)):
        with pytest.raises(FgError):
            opt.add_param_group(dict(params=[_matrix(*shape)]))
    assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=[_matrix(4, 8)], lr=0.1))
    assert len(opt.param_groups) == 2 and opt.param_groups[1]["lr"] == 0.1


def test_a_refused_step_moves_nothing():
    """Parameters that are not on the GPU, and settings changed since."""
    p = _matrix(4, 8)
    opt = Muon([p], weight_decay=0.1)
    with pytest.raises(ValueError, match="GPU"):
        opt.step()
    opt.param_groups[0]["momentum"] = 1.5
    with pytest.raises(ValueError, match="momentum"):
        opt.step()
    assert (p == 1).all() and not opt.state[p]
