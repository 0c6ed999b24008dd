"""Host side of the embedding's block and of the orthogonalising rule: no
GPU."""

import numpy as np
import pytest
import torch
from torch import nn


def model():
    import chainerkfac_b200 as ck
    return nn.Sequential(ck.EmbedID(7, 4, ignore_label=-1, scale=2.0),
                         nn.Linear(4, 3))


def test_public_names_and_links():
    import chainerkfac_b200 as ck
    from chainerkfac_b200 import links
    from chainerkfac_b200.optimizers import fisher_blocks as FB
    opt = ck.KFAC().setup(model())
    assert [type(fb) for fb in opt.fblocks] == [FB.FisherBlockEmbedID,
                                                FB.FisherBlockLinear]
    link = opt.fblocks[0].link
    assert isinstance(link, links.EmbedID)
    assert link.ignore_label == -1 and link.scale == 2.0 and link.b is None
    assert [n for n, _ in opt.target.namedparams()] == ['/0/W', '/1/W', '/1/b']
    # torch's own embedding has no block, as before
    assert ck.KFAC().setup(nn.Sequential(nn.Embedding(7, 4))).fblocks == []


def test_embedding_on_the_host_is_refused():
    import chainerkfac_b200 as ck
    from chainerkfac_b200 import _lib
    m = ck.EmbedID(5, 3)
    with pytest.raises(_lib.KfacLibraryError, match='CUDA tensor'):
        m(torch.zeros(2, dtype=torch.int64))
    assert 'ignore_label=None, scale=1.0' in repr(m)
    assert list(m.state_dict()) == ['weight']


def test_a_weight_of_two_blocks_is_refused():
    import chainerkfac_b200 as ck
    from chainerkfac_b200.optimizers.kfac import fblock_constructor
    m = nn.Sequential(ck.EmbedID(7, 4), nn.Linear(4, 7, bias=False))
    m[1].weight = m[0].weight
    with pytest.raises(ValueError, match='share a weight'):
        ck.KFAC().setup(m)
    opt = ck.KFAC(constructor=lambda n, l, **k: None if n == '/1' else
                  fblock_constructor(n, l, **k)).setup(m)
    assert len(opt.fblocks) == 1


def fill(opt):
    fb = opt.fblocks[0]
    fb.covs = [torch.rand(7), torch.eye(4), torch.rand(1, 1)]
    for f in opt.fblocks:
        for p in f.link.params():
            p.grad = torch.zeros_like(p.data)
    return fb


def test_what_the_collectives_move():
    import chainerkfac_b200 as ck
    from chainerkfac_b200.optimizers.kfac import block_cost
    fb = fill(ck.KFAC().setup(model()))
    arrays = fb.extract_for_reduce_scatter_v()
    assert [(tuple(a.shape), tri) for a, tri in arrays] == \
        [((7, 4), False), ((7,), False), ((1, 1), False), ((4, 4), True)]
    assert fb.extract_for_reduce_scatter_v_after_forward() == []
    fb._communicate_after_forward = True
    assert [tuple(a.shape) for a, _ in
            fb.extract_for_reduce_scatter_v_after_forward()] == [(7,), (1, 1)]
    assert [tuple(a.shape) for a, _ in fb.extract_for_reduce_scatter_v()] == \
        [(7, 4), (4, 4)]
    # the owner inverts G alone, however large the vocabulary
    assert block_cost(fb) == 4.0 ** 3
    assert fb.max_side() == 4 and tuple(fb.dims()) == (7, 4)


def test_what_the_inverse_plan_gets():
    import chainerkfac_b200 as ck
    fb = fill(ck.KFAC().setup(model()))
    assert fb.plan_factors() == [] and not fb.has_state()
    fb.cov_emas = [c.clone() for c in fb.covs]
    mean, G = fb.plan_factors()
    assert mean is fb.cov_emas[2] and G is fb.cov_emas[1]
    assert [e[0] for e in fb.plan_entries()] == [0, 1]
    assert [tuple(i.shape) for i in fb.ensure_invs()] == [(1, 1), (4, 4)]
    fb.set_diag_vals(torch.tensor([0.5, 0.25]))
    fb._plan = object()
    a, g = fb.get_diagvals()
    assert a.tolist() == [0.5] * 7 and g.tolist() == [0.25] * 4


def test_hooks_remember_tokens_and_gradients():
    import chainerkfac_b200 as ck
    from chainerkfac_b200 import embed_id
    m = model()
    opt = ck.KFAC().setup(m)
    ids = torch.tensor([[1, 2], [3, -1]])

    class Lookup(nn.Module):      # the same call without the library
        def forward(self, ids):
            return m[0].weight[ids.clamp(min=0)]
    for fb in opt.fblocks:
        fb.deferred = True
    old = m[0].forward
    m[0].forward = Lookup().forward
    try:
        with opt.kfhook:
            m(ids).sum().backward()
    finally:
        m[0].forward = old
    fb = opt.fblocks[0]
    assert torch.equal(fb._pending_A[0], ids)
    assert fb._pending_G[1][0].shape == (2, 2, 4)
    assert embed_id.EmbedID is ck.EmbedID


def test_rule_settings_and_scales():
    import chainerkfac_b200 as ck
    opt = ck.KFAC(lr=0.3, momentum=0.7)
    rule = ck.OrthogonalUpdateRule(opt.hyperparam)
    assert rule._settings()[:2] == (0.3, 0.7)
    opt.lr = 0.1
    assert rule._settings()[0] == 0.1
    per_step = ck.OrthogonalUpdateRule(
        opt.hyperparam, steps=2, coefficients=[[1.5, -0.5, 0.0]] * 2)
    hash(per_step._settings())
    assert rule._scale_of(torch.zeros(8, 2)) == 2.0
    assert rule._scale_of(torch.zeros(2, 8)) == 1.0
    assert rule._scale_of(torch.zeros(16, 2, 1, 2)) == 2.0
    assert ck.OrthogonalUpdateRule(scale=0.25)._scale_of(torch.zeros(9, 1)) \
        == 0.25
    assert np.isclose(ck.OrthogonalUpdateRule().hyperparam.lr, 0.001)


def test_rules_without_gradients_and_disabled_ones_are_left_alone():
    import chainerkfac_b200 as ck
    from chainerkfac_b200.optimizers import orthogonal
    opt = ck.KFAC(constructor=lambda n, l, **k: None).setup(
        nn.Linear(3, 4, bias=False))
    p = next(opt.target.params())
    p.update_rule = rule = ck.OrthogonalUpdateRule(opt.hyperparam)
    assert orthogonal.update_together([p]) == [] and rule.t == 1
    rule.enabled = False
    assert orthogonal.update_together([p]) == [p] and rule.t == 1
    rule.enabled = True
    rule.add_hook(lambda rule, param: None, name='h')
    assert orthogonal.update_together([p]) == [p] and rule.t == 1
