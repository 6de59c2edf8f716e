"""What the mixers' constructors draw: each parameter once, in the order of the layers."""
import pytest
import torch
import torch.nn as nn

from mamba_amd.modules import DeltaRule, LinearAttn


@pytest.mark.parametrize("Mixer,factors", [(LinearAttn, 1), (DeltaRule, 2)])
@pytest.mark.parametrize("groups,key_dim", [(None, None), (2, 24)])
def test_parameters_are_drawn_once(Mixer, factors, groups, key_dim, monkeypatch):
    torch.manual_seed(3)
    qk, heads = (groups or 4) * (key_dim or 32), 4
    first = nn.Linear(64, 2 * qk + 2 * 128 + factors * heads, bias=False)
    second = nn.Linear(128, 64, bias=False)
    torch.rand(heads)
    log_A = torch.log(1 + 15 * torch.rand(heads))
    after = torch.rand(1)

    built = []
    init = nn.Linear.__init__
    monkeypatch.setattr(nn.Linear, "__init__", lambda self, *a, **k: (built.append(a), init(self, *a, **k))[1])
    torch.manual_seed(3)
    m = Mixer(64, 32, key_dim=key_dim, n_groups=groups)
    assert len(built) == 2 and torch.equal(torch.rand(1), after)
    assert sum(m.sizes) == m.input_proj.out_features
    assert torch.equal(m.input_proj.weight, first.weight) and torch.equal(m.output_proj.weight, second.weight) and torch.equal(m.log_A, log_A)
    assert [n for n, _ in m.named_parameters()] == ["norm", "dt_bias", "log_A", "input_proj.weight", "output_proj.weight"]
