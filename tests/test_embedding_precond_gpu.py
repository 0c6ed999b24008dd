"""K-FAC step of an embedding's gradient on the device against fp64.

Bound of an element: the terms hold each operand to 2^-22 of itself, so a
product to 2^-21; a sum of 128 products meets 20 additions that cut off up to a
last place, 2^-23, and the K / 128 partial sums, the scaling and the division
2^-24 each, all relative to the sum of the products' sizes.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip('no CUDA device')


def gen(seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    return g


def randn(shape, seed):
    return torch.randn(shape, device='cuda', generator=gen(seed))


def problem(vocab, width, reach, seed=1):
    """Gradient with about `reach` of its rows, factors of some spread."""
    grad = randn((vocab, width), seed)
    grad *= torch.exp(3 * randn((vocab, 1), seed + 1))
    grad[torch.rand(vocab, device='cuda', generator=gen(seed + 2)) >= reach] = 0
    x = randn((2 * width + 3, width), seed + 3)
    G = (x.T @ x).double() / len(x) + 1e-2 * torch.eye(width, device='cuda')
    G_inv = torch.linalg.inv(G).float()
    G_inv = 0.5 * (G_inv + G_inv.T)
    A = torch.rand(vocab, device='cuda', generator=gen(seed + 4)) / vocab
    return G_inv.contiguous(), A, torch.full((1,), 1e-3, device='cuda'), grad


def want_kf(G_inv, A, damping, grad):
    f = 1 / (A.double() + damping.double())[:, None]
    kf = (grad.double() @ G_inv.double()) * f
    size = (grad.double().abs() @ G_inv.double().abs()) * f
    width = G_inv.shape[0]
    bound = size * (2.0 ** -21 + 20 * 2.0 ** -23 + (width / 128 + 4) * 2.0 ** -24)
    return kf, bound


SHAPES = [(1, 1, 1.0), (5, 3, 1.0), (300, 64, 0.5), (1000, 257, 0.1),
          (513, 130, 1.0), (4000, 512, 0.02), (257, 1000, 0.7),
          (20000, 96, 0.3), (700, 33, 0.0)]


@pytest.mark.parametrize('vocab,width,reach', SHAPES)
def test_step(vocab, width, reach):
    from chainerkfac_b200 import ops
    args = problem(vocab, width, reach)
    kf, bound = want_kf(*args)
    got = ops.precondition_embedding(*args)
    assert bool(((got.double() - kf).abs() <= bound).all())
    assert not got[(args[3] == 0).all(1)].any()
    assert torch.equal(got, ops.precondition_embedding(*args))
    # with the update
    param, mom = randn((vocab, width), 8), randn((vocab, width), 9)
    p0, m0 = param.double(), mom.double()
    again = ops.precondition_embedding(*args, param=param, mom=mom, lr=0.1,
                                       momentum=0.9)
    assert torch.equal(again, got)
    v = 0.9 * m0 - 0.1 * got.double()
    tol = 2.0 ** -22 * (m0.abs() + got.double().abs())
    assert bool(((mom.double() - v).abs() <= tol).all())
    assert bool(((param.double() - p0 - mom.double()).abs() <=
                 2.0 ** -23 * (p0.abs() + mom.double().abs())).all())


def test_outputs_and_layouts():
    from chainerkfac_b200 import ops
    args = problem(200, 40, 0.4)
    kf = ops.precondition_embedding(*args)
    G_inv, grad = args[0], args[3]
    assert torch.equal(ops.precondition_embedding(*args, kf=torch.full_like(
        grad, 7.0)), kf)
    assert torch.equal(ops.precondition_embedding(G_inv.t(), *args[1:]), kf)
    with pytest.raises(ValueError, match='contiguous'):
        ops.precondition_embedding(torch.cat((G_inv, G_inv), 1)[:, :40],
                                   *args[1:])
    # the gradient itself may take kf
    assert torch.equal(ops.precondition_embedding(*args, kf=grad), kf)


def test_rows_of_any_size_and_not_finite():
    from chainerkfac_b200 import ops
    G_inv, A, damping, grad = problem(300, 130, 1.0)
    size = torch.logspace(-36, 30, 300, device='cuda')[:, None]
    grad = (grad / grad.abs().amax(1, keepdim=True) * size).contiguous()
    kf, bound = want_kf(G_inv, A, damping, grad)
    got = ops.precondition_embedding(G_inv, A, damping, grad)
    fine = kf.abs().amax(1) < 1e37
    assert int(fine.sum()) > 250
    assert bool(((got.double() - kf).abs() <= bound + 1e-44)[fine].all())
    grad = grad.clamp(-1e3, 1e3)
    base = ops.precondition_embedding(G_inv, A, damping, grad)
    for bad in (float('nan'), float('inf')):
        g = grad.clone()
        g[17, 100] = bad
        got = ops.precondition_embedding(G_inv, A, damping, g)
        assert got[17].isnan().all()
        keep = torch.arange(300, device='cuda') != 17
        assert torch.equal(got[keep], base[keep])


@pytest.mark.parametrize('width', [33, 96])
def test_zeros_stay_beside_results_out_of_range(width):
    """Factors of a row and of a column that fit, with a product that does not:
    a zero stays a zero, whatever the rows next to it are like."""
    from chainerkfac_b200 import ops
    G_inv = torch.eye(width, device='cuda') * 2.0 ** 60
    A = torch.zeros(64, device='cuda')
    damping = torch.full((1,), 2.0 ** -55, device='cuda')
    grad = torch.zeros((64, width), device='cuda')
    grad[::2, 5] = 2.0 ** 60
    grad[1::4, 7] = 2.0 ** -100
    kf, bound = want_kf(G_inv, A, damping, grad)
    got = ops.precondition_embedding(G_inv, A, damping, grad)
    # (what makes up for truncation, at most (6 * 2 - 3.5) 0.72 2^-24 < 2^-21 of a
    # value, is in the bound: finite values are not exact powers of two)
    want = kf.float()
    assert torch.equal(got.isinf(), want.isinf()) and int(got.isinf().sum()) == 32
    assert torch.equal(got == 0, want == 0) and not got.isnan().any()
    fine = want.isfinite()
    assert bool(((got.double() - kf).abs() <= bound)[fine].all())


def test_columns_of_different_sizes():
    """Features that never saw a gradient have large entries in G_inv."""
    from chainerkfac_b200 import ops
    G_inv, A, damping, grad = problem(400, 96, 0.6)
    s = torch.logspace(-4, 4, 96, device='cuda')
    G_inv = (G_inv * s * s[:, None]).contiguous()
    grad = (grad / s).contiguous()
    kf, bound = want_kf(G_inv, A, damping, grad)
    got = ops.precondition_embedding(G_inv, A, damping, grad)
    # (an operand's value is held to 2^-39 of its row's largest at least)
    f = 1 / (A.double() + damping.double())[:, None]
    top = (grad.double().abs().amax(1, keepdim=True) @
           G_inv.double().abs().sum(0, keepdim=True)) + \
        grad.double().abs().sum(1, keepdim=True) @ \
        G_inv.double().abs().amax(1)[None]
    assert bool(((got.double() - kf).abs() <= bound + 2.0 ** -39 * top * f).all())


def test_unaligned_rows_and_what_is_around_them():
    from chainerkfac_b200 import ops
    G_inv, A, damping, grad = problem(150, 64, 0.5)
    want = ops.precondition_embedding(G_inv, A, damping, grad)

    def shifted(x):
        buf = torch.full((x.numel() + 5,), 9.0, device='cuda')
        view = buf[1:1 + x.numel()].view(x.shape)
        view.copy_(x)
        return buf, view
    bufs = [shifted(x) for x in (G_inv, grad, torch.zeros_like(grad))]
    ops.precondition_embedding(bufs[0][1], A, damping, bufs[1][1],
                               kf=bufs[2][1])
    assert torch.equal(bufs[2][1], want)
    for buf, _ in bufs:
        assert buf[0] == 9 and (buf[-4:] == 9).all()


def test_offsets_beyond_32_bits():
    from chainerkfac_b200 import ops
    vocab, width = 2 ** 21 + 5, 1028
    grad = torch.zeros((vocab, width), device='cuda')
    rows = torch.tensor([0, 3, vocab - 2, vocab - 1], device='cuda')
    small = randn((4, width), 3)
    grad[rows] = small
    G_inv, _, damping, _ = problem(4, width, 1.0)
    A = torch.rand(vocab, device='cuda', generator=gen(1))
    got = ops.precondition_embedding(G_inv, A, damping, grad)
    kf, bound = want_kf(G_inv, A[rows], damping, small)
    assert bool(((got[rows].double() - kf).abs() <= bound).all())
    assert float(got.sum()) == pytest.approx(float(got[rows].sum()), abs=1e-3 *
                                             float(got[rows].abs().sum()))
    assert not got[4:vocab - 2].any()


def test_replayed_with_another_gradient():
    from chainerkfac_b200 import _lib, ops
    G_inv, A, damping, grad = problem(3000, 260, 0.3)
    other = problem(3000, 260, 0.9, seed=50)[3]
    want = [ops.precondition_embedding(G_inv, A, damping, g)
            for g in (grad, other, grad * 0)]
    x = grad.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.precondition_embedding(G_inv, A, damping, x)
    for g, w in zip((other, grad * 0, grad), (want[1], want[2], want[0])):
        x.copy_(g)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)
    status = _lib.ctypes.c_int(7)
    _lib.check(_lib.load().kfac_tc_status(_lib.ctypes.byref(status)), 'status')
    assert status.value == 0
