"""FusedAdam's refusals, without a GPU."""
import pytest
import torch

from nerf_amd.optim import FusedAdam


def test_a_refused_step_updates_nothing(monkeypatch):
    """A 16-bit parameter behind a float32 one: the step is refused before the first is touched, wherever it stands."""
    launched = []
    monkeypatch.setattr(FusedAdam, '_adam', lambda self, *a, **k: launched.append(a))
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda *a: type('S', (), {'synchronize': lambda self: None})())
    good, bad = torch.nn.Parameter(torch.ones(8)), torch.nn.Parameter(torch.ones(8, dtype=torch.bfloat16))
    for p in (good, bad):
        p.grad = torch.ones_like(p)
    for groups in ([good, bad], [bad, good], [{'params': [good]}, {'params': [bad], 'lr': 1e-2}]):
        opt = FusedAdam(groups, lr=1e-3)
        for _ in range(2):
            with pytest.raises(TypeError, match='float32 parameters'):
                opt.step()
        assert not launched and not opt.state
    bad.grad = None     # (it takes no part then)
    opt = FusedAdam([good, bad], lr=1e-3)
    opt.step()
    assert len(launched) == 1 and opt.state[good]['step'] == 1
