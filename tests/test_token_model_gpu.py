"""Token models through the public interface: the embedding's block beside the
block of the fully connected layer that it is, orthogonalised updates under
``KFAC``, and both together."""

import copy

import numpy as np
import pytest
import torch
from torch import nn
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

COEF = (3.4445, -4.7750, 2.0315)


@pytest.fixture(autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip('no CUDA device')


def gen(seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    return g


def randint(high, shape, seed):
    return torch.randint(high, shape, device='cuda', generator=gen(seed))


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


# ------------------------------------------------------------------ the module

@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_module_and_its_gradient(dtype):
    import chainerkfac_b200 as ck
    torch.manual_seed(0)
    m = ck.EmbedID(50, 24, ignore_label=-1, scale=3.0, device='cuda',
                   dtype=dtype)
    ids = randint(50, (6, 7), 1)
    ids[0, :3] = -1
    y = m(ids)
    assert y.shape == (6, 7, 24) and y.dtype == dtype and y.requires_grad
    assert not y[0, :3].any()
    gy = torch.randn(y.shape, device='cuda', generator=gen(2)).to(dtype)
    y.backward(gy)
    live = ids >= 0
    want = torch.zeros((50, 24), dtype=torch.float64, device='cuda')
    want.index_add_(0, ids[live], 3.0 * gy[live].double())
    # at most 42 terms: 42 * 2^-24 of the sum of their sizes, and the rounding
    size = torch.zeros_like(want).index_add_(0, ids[live],
                                             3.0 * gy[live].double().abs())
    off = (m.weight.grad.double() - want).abs()
    assert bool((off <= 44 * 2.0 ** -24 * size +
                 torch.finfo(dtype).eps / 2 * want.abs()).all())
    # a second backward adds up; an expanded gradient is taken as it is
    m.weight.grad = None
    m(ids).sum().backward()
    count = torch.bincount(ids[live], minlength=50)
    assert torch.equal(m.weight.grad[:, 3].float(), 3.0 * count.float())
    with torch.no_grad():
        assert not m(ids).requires_grad


def test_gradient_against_differences():
    """A quadratic of the rows: its central difference is exact but for
    rounding, 2^-23 of the values over the step."""
    import chainerkfac_b200 as ck
    torch.manual_seed(1)
    m = ck.EmbedID(9, 5, scale=0.5, device='cuda')
    ids = randint(9, (4, 3), 3)
    c = torch.randn((4, 3, 5), device='cuda', generator=gen(4))

    def loss():
        y = m(ids)
        return (c.double() * y.double() ** 2).sum()
    loss().backward()
    grad = m.weight.grad.clone()
    step = 0.25
    with torch.no_grad():
        for v, k in ((0, 0), (int(ids[0, 0]), 2), (int(ids[3, 2]), 4)):
            w = float(m.weight[v, k])
            up, down = [], []
            for sign, out in ((1, up), (-1, down)):
                m.weight[v, k] = w + sign * step
                out.append(float(m.weight[v, k]))
                out.append(float(loss()))
            m.weight[v, k] = w
            diff = (up[1] - down[1]) / (up[0] - down[0])
            assert abs(diff - float(grad[v, k])) <= \
                2.0 ** -20 * (abs(up[1]) + abs(diff) + 1)


def test_module_is_saved_copied_and_captured():
    import chainerkfac_b200 as ck
    m = ck.EmbedID(40, 12, ignore_label=0, scale=2.0, device='cuda')
    other = ck.EmbedID(40, 12, ignore_label=0, scale=2.0, device='cuda')
    other.load_state_dict(m.state_dict())
    ids = randint(40, (30,), 5)
    gy = torch.randn((30, 12), device='cuda', generator=gen(6))
    want_y = m(ids).detach().clone()
    assert torch.equal(other(ids), want_y)
    assert torch.equal(copy.deepcopy(m)(ids), want_y)
    m(ids).backward(gy)
    want = m.weight.grad.clone()
    m.weight.grad = None
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):            # warm-up away from the main stream
        m(ids).backward(gy)
    torch.cuda.current_stream().wait_stream(side)
    m.weight.grad = None
    graph, x = torch.cuda.CUDAGraph(), ids.clone()
    with torch.cuda.graph(graph):
        y = m(x)
        y.backward(gy)
    for batch in (randint(40, (30,), 9), ids):
        x.copy_(batch)
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want_y) and torch.equal(m.weight.grad, want)


# ------------------------------------------------------------------- the block

class OneHot(nn.Module):
    """The layer that an embedding is: no bias, rows with a single entry."""

    def __init__(self, embed):
        super().__init__()
        vocab, width = embed.weight.shape
        self.linear = nn.Linear(vocab, width, bias=False, device='cuda')
        self.linear.weight.data.copy_(embed.weight.data.T)
        self.vocab, self.scale = vocab, embed.scale
        self.ignore_label = embed.ignore_label

    def forward(self, ids):
        x = F.one_hot(ids.clamp(min=0), self.vocab).float() * self.scale
        if self.ignore_label is not None:
            x = x * (ids != self.ignore_label)[..., None]
        return self.linear(x)


class Model(nn.Module):

    def __init__(self, embed, width, classes):
        super().__init__()
        self.embed = embed
        self.body = nn.Linear(width, 20, device='cuda')
        self.head = nn.Linear(20, classes, device='cuda')

    def forward(self, ids):
        return self.head(torch.tanh(self.body(self.embed(ids))))


def lossfun(model):
    def f(ids, t):
        return F.cross_entropy(model(ids).flatten(0, -2), t.flatten())
    return f


def pair(vocab=33, width=14, classes=11, scale=1.5, ignore_label=None):
    import chainerkfac_b200 as ck
    torch.manual_seed(3)
    a = Model(ck.EmbedID(vocab, width, ignore_label, scale, device='cuda'),
              width, classes)
    b = copy.deepcopy(a)
    b.embed = OneHot(a.embed)
    return a, b


def batches(vocab, classes, steps, ignore=False):
    out = []
    for k in range(steps):
        ids = randint(vocab, (8, 6), 100 + k)
        if ignore:
            ids[:, 4:] = -1
        out.append((ids, randint(classes, (8, 6), 200 + k)))
    return out


@pytest.mark.parametrize('kwargs,switches', [
    (dict(), {}), (dict(cov_ema_decay=0.5, momentum=0.5), {}),
    (dict(cov_ema_decay=1.0), dict(fuse_update=False)),
    (dict(acc_iters=2), {}), (dict(loss_scale=64.0), {}),
    (dict(), dict(group_factors=False)), (dict(), dict(defer_join=True)),
    (dict(), dict(eager_inverses=True)), (dict(pi_type='none'), {})])
@pytest.mark.parametrize('ignore', [False, True])
def test_block_is_that_of_the_layer_on_one_hot_rows(kwargs, switches, ignore):
    """Factors agree to 1e-4 and updates to 1e-3, what the framework holds its
    blocks to."""
    import chainerkfac_b200 as ck
    from chainerkfac_b200.optimizers import fisher_blocks as FB
    a, b = pair(ignore_label=-1 if ignore else None)
    opts = []
    for model in (a, b):
        opt = ck.KFAC(lr=0.05, **{**dict(damping=1e-2, cov_ema_decay=0.9),
                                  **kwargs}).setup(model)
        for k, v in switches.items():
            setattr(opt, k, v)
        opts.append(opt)
    start = a.embed.weight.detach().clone()
    steps = 6 if kwargs.get('acc_iters') else 4
    for ids, t in batches(33, 11, steps, ignore):
        for opt, model in zip(opts, (a, b)):
            opt.update(lossfun(model), ids, t)
    for opt in opts:
        opt.join()
    fa, fb = [[f for f in opt.fblocks if 'embed' in f.linkname][0]
              for opt in opts]
    assert isinstance(fa, FB.FisherBlockEmbedID)
    for x, y in ((fa.cov_emas[0].diag(), fb.cov_emas[0]),
                 (fa.cov_emas[1], fb.cov_emas[1])):
        assert rel(x, y) <= 1e-4
    assert rel(fa.cov_emas[2][0, 0], fb.cov_emas[0].diagonal().mean()) <= 1e-5
    assert rel(fa.invs[1], fb.invs[1]) <= 1e-3
    if not switches.get('defer_join'):
        assert rel(fa.diag_val_forward, fb.diag_val_forward) <= 1e-4
    step_a = a.embed.weight.detach() - start
    step_b = b.embed.linear.weight.detach().T - start
    assert rel(step_a, step_b) <= 1e-3
    assert rel(a.head.weight.detach(), b.head.weight.detach()) <= 1e-3


def test_blocks_own_interface():
    """Hooks, running averages, inverses and update called block by block."""
    import chainerkfac_b200 as ck
    a, b = pair()
    opts = [ck.KFAC(damping=1e-2).setup(m) for m in (a, b)]
    ids, t = batches(33, 11, 1)[0]
    for opt, model in zip(opts, (a, b)):
        with opt.kfhook:
            lossfun(model)(ids, t).backward()
        for fb in opt.fblocks:
            fb.update_cov_emas()
            fb.update_invs()
            fb.update_kfgrads()
    fa, fb = [[f for f in opt.fblocks if 'embed' in f.linkname][0]
              for opt in opts]
    assert rel(fa.link.W.kfgrad, fb.link.W.kfgrad.T) <= 1e-3
    for x, y in zip(fa.get_diagvals(), fb.get_diagvals()):
        assert x.shape == y.shape and rel(x, y) <= 1e-4


# ----------------------------------------------------------------- update rule

def newton_schulz(x, steps=5):
    x = x.double().reshape(x.shape[0], -1)
    x = x / (x.norm() + 1e-7)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    for _ in range(steps):
        A = x @ x.T
        x = COEF[0] * x + (COEF[1] * A + COEF[2] * (A @ A)) @ x
    return x.T if tall else x


@pytest.mark.parametrize('nesterov', [True, False])
@pytest.mark.parametrize('scale', [None, 0.3])
def test_rule(nesterov, scale):
    import chainerkfac_b200 as ck
    torch.manual_seed(4)
    model = nn.Sequential(nn.Linear(40, 70, device='cuda'), nn.Tanh(),
                          nn.Linear(70, 30, device='cuda'),
                          nn.Unflatten(1, (30, 1, 1)),
                          nn.Conv2d(30, 12, 1, device='cuda'), nn.Flatten())
    opt = ck.KFAC(lr=0.02, momentum=0.8,
                  constructor=lambda name, link, **k: None).setup(model)
    rule_of = {}
    for _, p in opt.target.namedparams():
        if len(p.shape) > 1:
            p.update_rule = rule_of[id(p._p)] = ck.OrthogonalUpdateRule(
                opt.hyperparam, nesterov=nesterov, scale=scale, decay=0.1)
    want = {n: p.detach().double() for n, p in model.named_parameters()}
    vel = {n: torch.zeros_like(w) for n, w in want.items()}
    for k in range(3):
        if k == 2:
            opt.lr = 0.01                 # rules see the optimizer's values
        x = torch.randn((16, 40), device='cuda', generator=gen(k))
        opt.update(lambda x: model(x).square().mean(), x)
        for n, p in model.named_parameters():
            g = p.grad.double()
            if id(p) not in rule_of:      # plain momentum
                vel[n] = 0.8 * vel[n] - opt.lr * g
                want[n] = want[n] + vel[n]
                continue
            vel[n] = 0.8 * vel[n] + g
            u = g + 0.8 * vel[n] if nesterov else vel[n]
            s = scale or max(1.0, u.shape[0] / (u.numel() / u.shape[0])) ** .5
            want[n] = (1 - 0.1 * opt.lr) * want[n] - \
                opt.lr * s * newton_schulz(u).reshape(u.shape)
    for n, p in model.named_parameters():
        # each step's part is within 4e-5 of its size, the weight rounded
        assert rel(p.detach(), want[n]) <= 2e-6, n
    assert all(r.t == 3 for r in rule_of.values())


def test_rule_with_hooks_loss_scale_and_one_by_one():
    import chainerkfac_b200 as ck
    torch.manual_seed(5)
    start = nn.Linear(33, 21, bias=False, device='cuda')
    weights = []
    for case in range(4):
        m = copy.deepcopy(start)
        opt = ck.KFAC(lr=0.02, momentum=0.8,
                      loss_scale=32.0 if case == 1 else None,
                      constructor=lambda name, link, **k: None).setup(m)
        p = next(opt.target.params())
        p.update_rule = ck.OrthogonalUpdateRule(opt.hyperparam)
        seen = []
        if case == 2:
            p.update_rule.add_hook(lambda rule, q: seen.append(rule.t),
                                   name='seen', timing='post')
        for k in range(2):
            x = torch.randn((16, 33), device='cuda', generator=gen(k))
            if case == 3:
                p.update_rule.enabled = k == 0
            opt.update(lambda x: m(x).square().mean(), x)
        weights.append(m.weight.detach())
        assert seen == ([1, 2] if case == 2 else [])
    assert rel(weights[1], weights[0]) <= 1e-6
    assert torch.equal(weights[2], weights[0])
    assert rel(weights[3], weights[0]) > 1e-4
    with pytest.raises(ValueError, match='matrices'):
        opt = ck.KFAC(constructor=lambda n, l, **k: None).setup(
            nn.Linear(3, 4, device='cuda'))
        for p in opt.target.params():
            p.update_rule = ck.OrthogonalUpdateRule(opt.hyperparam)
        opt.update(lambda x: opt.target(x).sum(), torch.ones(2, 3, device='cuda'))


def test_rule_takes_a_blocks_gradient():
    """On a layer with a block the preconditioned gradient is what is
    orthogonalised."""
    import chainerkfac_b200 as ck
    torch.manual_seed(6)
    m = nn.Linear(12, 9, bias=False, device='cuda')
    opt = ck.KFAC(lr=0.1, momentum=0.0, damping=1e-2).setup(m)
    p = next(opt.target.params())
    p.update_rule = ck.OrthogonalUpdateRule(opt.hyperparam, scale=1.0)
    old = m.weight.detach().clone()
    opt.update(lambda x: m(x).square().mean(),
               torch.randn((30, 12), device='cuda', generator=gen(1)))
    step = (old - m.weight.detach()).double() / 0.1
    assert rel(step, newton_schulz(p.kfgrad)) <= 1e-4
    assert rel(step, newton_schulz(m.weight.grad)) > 1e-2


# -------------------------------------------------------------------- together

def test_a_token_model_trains():
    """An embedding with its block, a layer with an orthogonalised update and a
    head with a block, in one ``update``."""
    import chainerkfac_b200 as ck
    from chainerkfac_b200.optimizers.kfac import fblock_constructor
    torch.manual_seed(7)
    model = Model(ck.EmbedID(300, 48, -1, 48 ** 0.5, device='cuda'), 48, 17)
    model.embed.weight.data.mul_(0.1)
    opt = ck.KFAC(lr=0.02, momentum=0.9, cov_ema_decay=0.9, damping=1e-2,
                  constructor=lambda name, link, **k: None if 'body' in name
                  else fblock_constructor(name, link, **k)).setup(model)
    assert [fb.linkname for fb in opt.fblocks] == ['/embed', '/head']
    body = [p for n, p in opt.target.namedparams() if n == '/body/W'][0]
    body.update_rule = ck.OrthogonalUpdateRule(opt.hyperparam)
    ids = randint(300, (16, 10), 1)
    ids[:, 8:] = -1
    t = randint(17, (16, 10), 2)
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    for _ in range(5):
        opt.update(lossfun(model), ids, t)
    assert np.isfinite(float(opt.loss))
    for n, p in model.named_parameters():
        assert torch.isfinite(p).all(), n
        assert not torch.equal(p, before[n]), n
    # tokens that never occurred have not moved
    absent = torch.ones(300, dtype=torch.bool, device='cuda')
    absent[ids[:, :8]] = False
    assert torch.equal(model.embed.weight[absent], before['embed.weight'][absent])
