"""``DistributedKFAC`` exchanges gradients and weights of blocks only: an
orthogonalised weight without one would stay as it is, or part from its copies
on the other ranks, and is refused."""

import pytest
import torch
from torch import nn


class Comm(object):
    """One of two ranks; nothing is exchanged."""
    rank, size = 0, 2

    def bcast_data(self, model):
        pass

    def reduce_scatter_v_arrays(self, arrays, stream=None):
        pass

    def all_gather_v_arrays(self, arrays, stream=None):
        pass


def optimizer(monkeypatch, blocks, **kw):
    import chainerkfac_b200 as ck
    from chainerkfac_b200 import ops
    from chainerkfac_b200.optimizers.kfac import KFAC, fblock_constructor
    for name in ('momentum_update', 'axpby_group', 'orthogonalize'):
        monkeypatch.setattr(ops, name, lambda *a, **k: None)
    monkeypatch.setattr(KFAC, 'update_kfgrads', lambda self, fblocks: None)
    m = nn.Sequential(nn.Linear(4, 4, bias=False), nn.Linear(4, 4, bias=False))
    opt = ck.DistributedKFAC(
        Comm(), constructor=lambda n, l, **k: fblock_constructor(n, l, **k)
        if n in blocks else None, **kw).setup(m)
    for fb in opt.fblocks:
        fb.covs = [torch.eye(4), torch.eye(4)]
    for p in opt.target.params():
        p.grad = torch.ones_like(p.data)
    return opt, dict(opt.target.namedparams())


@pytest.mark.parametrize('pic', [True, False])
def test_a_weight_without_a_block_is_refused(monkeypatch, pic):
    import chainerkfac_b200 as ck
    opt, params = optimizer(monkeypatch, ('/0',), only_pic_update_weight=pic)
    rule = params['/1/W'].update_rule = ck.OrthogonalUpdateRule(opt.hyperparam)
    for _ in range(2):
        with pytest.raises(ValueError, match='/1/W .*no block'):
            opt.update()
    assert opt.t == 0 and rule.t == 0
    with pytest.raises(ValueError, match='/1/W .*no block'):
        opt.update(lambda: 1 / 0)        # before anything is computed
    rule.enabled = False
    opt.update()                         # (the first one hands weights out)
    opt.update()
    assert opt.t == 1 and rule.t == 0


@pytest.mark.parametrize('pic', [True, False])
def test_a_weight_with_a_block_is_updated(monkeypatch, pic):
    import chainerkfac_b200 as ck
    opt, params = optimizer(monkeypatch, ('/0', '/1'),
                            only_pic_update_weight=pic)
    rules = []
    for p in params.values():
        p.update_rule = ck.OrthogonalUpdateRule(opt.hyperparam)
        rules.append(p.update_rule)
    for _ in range(3):
        opt.update()
    # the owner's, or everybody's
    assert [r.t for r in rules] == ([2, 0] if pic else [2, 2])
