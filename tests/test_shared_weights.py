"""A weight that is in a model under several names (an output layer that shares
the token embedding, a module in two places) is updated once a step."""

import pytest
import torch
from torch import nn
import torch.nn.functional as F


def only(*names):
    """Constructor that gives blocks to the links of these names."""
    from chainerkfac_b200.optimizers.kfac import fblock_constructor
    return lambda n, l, **k: fblock_constructor(n, l, **k) \
        if n in names else None


def tied(**kw):
    import chainerkfac_b200 as ck
    m = nn.Sequential(ck.EmbedID(7, 4, **kw), nn.Linear(4, 7, bias=False, **kw))
    m[1].weight = m[0].weight
    return m


class Twice(nn.Module):
    """One module below two parents."""

    def __init__(self, shared):
        super().__init__()
        self.a, self.b = nn.Sequential(shared), nn.Sequential(shared)


def steps_of(opt, monkeypatch):
    """Updates of each weight in one ``update``: by the fused K-FAC step, by
    the momentum kernel, by the orthogonalising one."""
    from chainerkfac_b200 import ops
    seen = []
    monkeypatch.setattr(
        ops, 'momentum_update',
        lambda g, p, *a: seen.append(('momentum', p.data_ptr())))
    monkeypatch.setattr(ops, 'axpby_group', lambda *a: None)
    monkeypatch.setattr(
        ops, 'orthogonalize', lambda xs, params, **k: seen.extend(
            ('orthogonal', p.data_ptr()) for p in params))

    def step(fblocks):
        for fb in fblocks:
            for p in fb.link.params():
                p.kfgrad = torch.zeros_like(p.data)
                if opt._can_fuse(p):
                    seen.append(('block', p.data.data_ptr()))
                    p._kfac_applied = True
    monkeypatch.setattr(opt, 'update_kfgrads', step)
    for p in opt.target.params():
        p.grad = torch.ones_like(p.data)
    opt.update()
    return seen


@pytest.mark.parametrize('block', ['/0', '/1'])
@pytest.mark.parametrize('fused', [True, False])
def test_a_tied_embedding_takes_one_step(monkeypatch, block, fused):
    import chainerkfac_b200 as ck
    m = tied()
    opt = ck.KFAC(constructor=only(block)).setup(m)
    opt.fuse_update = fused
    at = m[0].weight.data_ptr()
    for _ in range(2):
        assert steps_of(opt, monkeypatch) == \
            [('block' if fused else 'momentum', at)]


def test_a_tied_embedding_without_blocks_takes_one_step(monkeypatch):
    import chainerkfac_b200 as ck
    m = tied()
    opt = ck.KFAC(constructor=only()).setup(m)
    assert steps_of(opt, monkeypatch) == [('momentum', m[0].weight.data_ptr())]


def test_a_scaled_loss_is_divided_out_once(monkeypatch):
    import chainerkfac_b200 as ck
    m = tied()
    opt = ck.KFAC(constructor=only('/0'), loss_scale=8.0).setup(m)
    for p in opt.target.params():
        p._loss_scale = 8.0
    steps_of(opt, monkeypatch)
    assert m[0].weight.grad[0, 0] == 1 / 8


def test_an_embedding_in_two_places_takes_one_step(monkeypatch):
    import chainerkfac_b200 as ck
    e = ck.EmbedID(7, 4)
    opt = ck.KFAC(constructor=only('/a/0')).setup(Twice(e))
    assert len(opt.fblocks) == 1 and len(list(opt.target.params())) == 2
    assert steps_of(opt, monkeypatch) == [('block', e.weight.data_ptr())]


def test_an_orthogonalised_weight_takes_one_step(monkeypatch):
    import chainerkfac_b200 as ck
    # a layer in two places
    layer = nn.Linear(4, 4, bias=False)
    opt = ck.KFAC(constructor=only()).setup(Twice(layer))
    for p in opt.target.params():
        p.update_rule = ck.OrthogonalUpdateRule(opt.hyperparam)
    assert steps_of(opt, monkeypatch) == \
        [('orthogonal', layer.weight.data_ptr())]
    # the embedding's own name
    m = tied()
    opt = ck.KFAC(constructor=only()).setup(m)
    p = next(opt.target.params())
    p.update_rule = ck.OrthogonalUpdateRule(opt.hyperparam)
    assert steps_of(opt, monkeypatch) == \
        [('orthogonal', m[0].weight.data_ptr())]


@pytest.mark.parametrize('names', [('/0/W', '/1/W'), ('/1/W',)])
def test_rules_under_two_names_are_refused(monkeypatch, names):
    """Which of them is meant is not ours to say; nothing has changed by
    then."""
    import chainerkfac_b200 as ck
    for m, block in ((tied(), ()), (tied(), ('/0',)),
                     (nn.Sequential(nn.Linear(4, 4, bias=False),
                                    nn.Linear(4, 4, bias=False)), ())):
        m[1].weight = m[0].weight
        opt = ck.KFAC(constructor=only(*block)).setup(m)
        for n, p in opt.target.namedparams():
            if n in names:
                p.update_rule = ck.OrthogonalUpdateRule(opt.hyperparam)
        with pytest.raises(ValueError, match='/0/W and /1/W are one weight'):
            steps_of(opt, monkeypatch)
        assert opt.t == 0
        # one of them may be switched off, or taken away
        views = dict(opt.target.namedparams())
        views['/0/W'].update_rule.enabled = False
        assert steps_of(opt, monkeypatch)[-1] == \
            ('orthogonal', m[0].weight.data_ptr())
        views['/0/W'].update_rule = None
        assert steps_of(opt, monkeypatch)[-1] == \
            ('orthogonal', m[0].weight.data_ptr())


def test_layers_that_share_a_weight_are_as_before(monkeypatch):
    """Without embeddings or orthogonalised weights every name has its rule."""
    import chainerkfac_b200 as ck
    m = nn.Sequential(nn.Linear(4, 4, bias=False), nn.Linear(4, 4, bias=False))
    m[1].weight = m[0].weight
    opt = ck.KFAC().setup(m)
    assert all(p.update_rule is not None for p in opt.target.params())
    assert len(steps_of(opt, monkeypatch)) == 2


@pytest.mark.gpu
@pytest.mark.parametrize('block', ['/0', '/1'])
@pytest.mark.parametrize('fused', [True, False])
def test_the_weight_after_a_step(block, fused):
    """v = -lr kf and W + v, each rounded once; nothing else is added."""
    import chainerkfac_b200 as ck
    if not torch.cuda.is_available():
        pytest.skip('no CUDA device')
    torch.manual_seed(0)
    m = tied(device='cuda')
    opt = ck.KFAC(lr=0.1, damping=1e-2, constructor=only(block)).setup(m)
    opt.fuse_update = fused
    ids = torch.arange(12, device='cuda') % 7
    old = m[0].weight.detach().clone()
    opt.update(lambda x, t: F.cross_entropy(m(x), t), ids, (ids + 1) % 7)
    owner = [p for n, p in opt.target.namedparams() if n == block + '/W'][0]
    want = old.double() - 0.1 * owner.kfgrad.double()
    off = (m[0].weight.detach().double() - want).abs()
    half = 2.0 ** -24
    assert bool((off <= 3 * half * (old.abs() + want.abs())).all())
    assert not torch.equal(old, m[0].weight.detach())


def test_gradients_of_a_module_in_two_places_are_accumulated_once(monkeypatch):
    """acc += grad / 2 in each of two micro-steps."""
    import chainerkfac_b200 as ck
    from chainerkfac_b200 import ops

    def axpby(a, xs, b, ys, outs):
        for x, y, o in zip(xs, ys, outs):
            o.copy_(a * x + (b * y if b else 0.0))
    monkeypatch.setattr(ops, 'axpby_group', axpby)
    e = ck.EmbedID(7, 4)
    opt = ck.KFAC(constructor=only(), acc_iters=2).setup(Twice(e))
    for value in (1.0, 3.0):
        for p in opt.target.params():
            p.grad = torch.full_like(p.data, value)
        opt.accumulate()
    assert torch.equal(e.weight.grad, torch.full((7, 4), 2.0))


def test_every_name_keeps_a_rule(monkeypatch):
    """Programs go through all parameters' rules (hooks, settings); that of
    the further name is switched off."""
    import chainerkfac_b200 as ck
    m = tied()
    opt = ck.KFAC(constructor=only('/1')).setup(m)
    called = []
    for n, p in opt.target.namedparams():
        p.update_rule.add_hook(lambda rule, param, n=n: called.append(n),
                               name='h')
    assert [p.update_rule.enabled for p in opt.target.params()] == [False, True]
    assert steps_of(opt, monkeypatch) == [('momentum', m[0].weight.data_ptr())]
    assert called == ['/1/W']
    # both switched on: as rules under two names
    for p in opt.target.params():
        p.update_rule.enabled = True
    with pytest.raises(ValueError, match='/0/W and /1/W are one weight'):
        steps_of(opt, monkeypatch)


def test_a_tied_layer_waits_for_a_deferred_update(monkeypatch):
    """With ``defer_join`` a weight may still be being written on a side stream
    when either of its layers is called."""
    import chainerkfac_b200 as ck
    waited = []

    class Stream(object):
        def wait_event(self, event):
            waited.append(event)
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda *a: Stream())
    for block, at in (('/0', 1), ('/1', 1)):
        m = tied()
        opt = ck.KFAC(constructor=only(block)).setup(m)
        opt.defer_join = True
        opt._pending_classes = {0: block}
        opt._block_class = {id(opt.fblocks[0]): 0}
        m[at](torch.zeros(2, 4))
        assert waited.pop() == block and not opt._pending_classes
        m[at](torch.zeros(2, 4))
        assert not waited
