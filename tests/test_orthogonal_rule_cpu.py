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


@pytest.mark.parametrize('model,error,match', [
    (lambda: nn.Linear(3, 4, bias=False).half(), TypeError, 'float16'),
    (lambda: nn.Linear(3, 4, bias=False).bfloat16(), TypeError,
     'bfloat16'),
    (lambda: nn.Linear(3, 4), ValueError, 'only matrices'),
    (lambda: nn.Conv2d(3, 4, 3, bias=False).to(
        memory_format=torch.channels_last), ValueError, 'contiguous')])
def test_weights_it_cannot_take_are_refused_before_anything_changes(
        monkeypatch, model, error, match):
    opt, seen = rules(monkeypatch, model())
    params = list(opt.target.params())
    with pytest.raises(error, match=match):
        opt.update()
    assert opt.t == 0 and not seen
    bad = params[-1]
    with pytest.raises(error, match=match):
        bad.update()
    assert all(p.update_rule.t == 0 for p in params)
    # unless the rule is switched off
    for p in params:
        p.update_rule.enabled = False
    opt.update()
    assert opt.t == 1 and not seen
