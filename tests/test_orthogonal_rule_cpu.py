"""Host side of the orthogonalising rule: what its kernels are given."""

import pytest
import torch
from torch import nn


def rules(monkeypatch, model, **kw):
    """The optimizer with an orthogonalising rule for every parameter, and the
    gradients that its updates are made of."""
    import chainerkfac_b200 as ck
    from chainerkfac_b200 import ops
    seen = []
    monkeypatch.setattr(ops, 'axpby_group', lambda a, xs, b, ys, outs:
                        seen.append([x.clone() for x in xs]))
    monkeypatch.setattr(ops, 'orthogonalize', lambda *a, **k: None)
    opt = ck.KFAC(constructor=lambda n, l, **k: None, **kw).setup(model)
    for p in opt.target.params():
        p.update_rule = ck.OrthogonalUpdateRule(opt.hyperparam,
                                                nesterov=False)
        p.grad = torch.full_like(p.data, 6.0)
    return opt, seen


@pytest.mark.parametrize('together', [True, False])
def test_a_blocks_gradient_is_taken_without_the_loss_scale(monkeypatch,
                                                           together):
    """As the momentum rule takes it: a scale that changes leaves the momentum
    of one size."""
    opt, seen = rules(monkeypatch, nn.Linear(3, 4, bias=False))
    p = next(opt.target.params())
    if not together:
        p.update_rule.add_hook(lambda rule, param: None, name='h')
    for scale in (2.0, 16.0, None):
        p.grad = torch.full_like(p.data, 6.0 * (scale or 1.0))
        p.kfgrad = torch.full_like(p.data, 3.0 * (scale or 1.0))
        p._loss_scale = scale
        opt.update()
        assert seen.pop()[0].unique().tolist() == [3.0] and not seen
        assert p.grad.unique().tolist() == [6.0]
