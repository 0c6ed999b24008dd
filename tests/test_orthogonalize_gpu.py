"""Orthogonalised updates on the device against the same products in fp64.

Tolerances (relative Frobenius error).  fp32: every operand of a product is
held to 2^-22 of its row's or matrix's size and every sum to a few 2^-23, 15
products deep, and an error of X, relative to its largest singular value, grows
with the smallest ones by up to |a|^5 = 485 while it is spread over all of the
result's sqrt(min side) of norm: 485 * 2^-22 = 1.2e-4 / sqrt(min side) in the
worst case, 2e-5 being for min side >= 33 and twice that below.  16 bits: the
result is rounded to eps / 2, and A and B to 2^-11 of their entries at most and
2^-12 in the mean, where these are of order one and up to |b| = 4.8 times that;
the last two steps' roundings are not damped: 2 * 4.8 * 2^-12 = 2.4e-3 and
eps / 2.  (Small matrices round neither so far.)
"""

import pytest
import torch

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


def reference(x, steps=5, coefficients=COEF, eps=1e-7):
    x = x.double().reshape(x.shape[0], -1)
    x = x / (x.norm() + eps)
    rows = [coefficients] * steps if not hasattr(coefficients[0], '__len__') \
        else coefficients
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    for a, b, c in rows:
        A = x @ x.T
        x = a * x + (b * A + c * (A @ A)) @ x
    return x.T if tall else x


def tolerance(x):
    if x.dtype == torch.float32:
        small = min(x.shape[0], x.numel() // x.shape[0])
        return 2e-5 if small >= 33 else 4e-5
    return 2.4e-3 + torch.finfo(x.dtype).eps / 2


def check(got, x, want=None, **kw):
    want = reference(x, **kw) if want is None else want
    got = got.double().reshape(want.shape)
    rel = float((got - want).norm() / want.norm())
    assert rel <= tolerance(x), (tuple(x.shape), x.dtype, rel)


SHAPES = [(1, 1), (1, 9), (7, 1), (2, 3), (16, 16), (31, 200), (64, 147),
          (127, 129), (128, 128), (129, 128), (255, 130), (300, 77),
          (513, 512), (64, 1500), (1500, 200), (700, 1100),
          # what a block does by itself, turned and not, up to its sides
          (147, 64), (256, 128), (128, 256), (256, 33), (33, 255), (257, 128),
          (128, 257), (129, 129), (48, 49), (90, 17),
          # and the blocks of a cluster, from two to sixteen
          (100, 384), (385, 33), (64, 576), (769, 128), (128, 1152), (1, 1537),
          (2999, 65), (128, 3000), (127, 3100)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16,
                                   torch.float16])
@pytest.mark.parametrize('shape', SHAPES)
def test_one_matrix(shape, dtype):
    from chainerkfac_b200 import ops
    x = torch.randn(shape, device='cuda', generator=gen(1)).to(dtype)
    keep = x.clone()
    got = ops.orthogonalize(x)
    assert got.dtype == dtype and got.shape == x.shape
    assert torch.equal(x, keep)
    check(got, x)
    assert torch.equal(got, ops.orthogonalize(x))


def test_singular_values_come_near_one():
    from chainerkfac_b200 import ops
    u, _, v = torch.linalg.svd(torch.randn((200, 333), device='cuda',
                                           generator=gen(2)),
                               full_matrices=False)
    s = torch.logspace(0, -2, 200, device='cuda')
    got = ops.orthogonalize((u * s) @ v)
    t = torch.linalg.svdvals(got.double())
    assert 0.6 < float(t.min()) and float(t.max()) < 1.25


@pytest.mark.parametrize('count', [2, 5, 41, 90])
def test_many_matrices_at_once(count):
    from chainerkfac_b200 import ops
    g = gen(count)
    xs = []
    for i in range(count):
        shape = SHAPES[(3 * i + 1) % len(SHAPES)]
        dtype = (torch.float32, torch.bfloat16)[i % 3 == 1]
        xs.append(torch.randn(shape, device='cuda', generator=g).to(dtype))
    scales = [1.0 + i for i in range(count)]
    got = ops.orthogonalize(xs, scale=scales)
    again = ops.orthogonalize(xs, scale=scales)
    for x, y, z, s in zip(xs, got, again, scales):
        check(y.float() / s, x)
        # (alone a long sum may be cut elsewhere: near, not the same bits)
        assert torch.equal(y, z)


def test_matrices_of_a_cluster_in_one_launch(dtype=torch.float32):
    """Short ones beside long ones: some blocks of their clusters have no
    columns."""
    from chainerkfac_b200 import ops
    g = gen(12)
    xs = [torch.randn(s, device='cuda', generator=g).to(dtype) for s in
          ((3, 2), (128, 2000), (1500, 40), (33, 33), (5, 900), (257, 128))]
    got = ops.orthogonalize(xs)
    again = ops.orthogonalize(xs)
    for x, y, z in zip(xs, got, again):
        check(y, x)
        assert torch.equal(y, z)
    # values that are not finite stay in their matrix
    xs[1][7, 1999] = float('inf')
    bad = ops.orthogonalize(xs)
    assert bad[1].isnan().all()
    for k in (0, 2, 3, 4, 5):
        assert torch.equal(bad[k], got[k])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('count', [3, 70])
def test_many_small_matrices(count, dtype):
    """As many blocks as matrices; alone each gives the same bits."""
    from chainerkfac_b200 import ops
    g = gen(count)
    xs = [torch.randn((1 + 37 * i % 128, 1 + 91 * i % 256)[::1 - 2 * (i % 2)],
                      device='cuda', generator=g).to(dtype)
          for i in range(count)]
    got = ops.orthogonalize(xs, scale=[0.5 + i for i in range(count)])
    for i, (x, y) in enumerate(zip(xs, got)):
        check(y.float() / (0.5 + i), x)
        assert torch.equal(y, ops.orthogonalize(x, scale=0.5 + i))


@pytest.mark.parametrize('shape', [(60, 200), (200, 60)])
def test_small_weights_are_updated_in_either_direction(shape):
    from chainerkfac_b200 import ops
    x = torch.randn(shape, device='cuda', generator=gen(1))
    w = torch.randn(shape, device='cuda', generator=gen(2))
    old, out = w.double(), torch.empty_like(x)
    ops.orthogonalize(x, outs=out, params=w, lr=0.1, decay=0.3, scale=2.0)
    step = 0.1 * 2.0 * reference(x)
    off = float((w.double() - (1 - 0.03) * old + step).norm())
    assert off <= tolerance(x) * float(step.norm()) + \
        2.0 ** -23 * float(old.norm())
    check(out / 2.0, x)


def test_steps_coefficients_and_eps():
    from chainerkfac_b200 import ops
    x = torch.randn((90, 140), device='cuda', generator=gen(4))
    rows = [(4.0, -6.0, 3.0), (2.0, -1.5, 0.5), (1.5, -0.5, 0.0)]
    check(ops.orthogonalize(x, steps=3, coefficients=rows), x, steps=3,
          coefficients=rows)
    check(ops.orthogonalize(x, steps=1), x, steps=1)
    check(ops.orthogonalize(x, steps=12, coefficients=(1.5, -0.5, 0.0)), x,
          steps=12, coefficients=(1.5, -0.5, 0.0))
    check(ops.orthogonalize(x, steps=4, coefficients=(1.5, 0.0, -0.5)), x,
          steps=4, coefficients=(1.5, 0.0, -0.5))
    check(ops.orthogonalize(x, eps=100.0), x, eps=100.0)


@pytest.mark.parametrize('size', [1e-38, 1e-30, 1e-7, 1e18, 1e37])
def test_sizes_of_the_elements(size):
    """Norms whose squares leave fp32 (eps is 1e-7: of the smallest updates
    nothing is left)."""
    from chainerkfac_b200 import ops
    x = torch.randn((70, 90), device='cuda', generator=gen(5))
    x = (x.double() * size).float()
    got = ops.orthogonalize(x)
    want = reference(x)
    assert float((got.double() - want).norm()) <= \
        2e-5 * float(want.norm()) + 1e-9
    check(ops.orthogonalize(x, eps=0.0), x, eps=0.0)


def test_zeros_and_values_that_are_not_finite():
    from chainerkfac_b200 import ops
    x = torch.zeros((40, 50), device='cuda')
    assert not ops.orthogonalize(x).any()
    x = torch.randn((200, 300), device='cuda', generator=gen(6))
    for bad in (float('nan'), float('inf'), -float('inf')):
        y = x.clone()
        y[150, 250] = bad
        assert ops.orthogonalize(y).isnan().all()
    # one matrix of a group does not touch the others
    got = ops.orthogonalize([y, x])
    assert got[0].isnan().all()
    check(got[1], x)


def test_low_rank_and_one_sided():
    from chainerkfac_b200 import ops
    g = gen(7)
    u = torch.randn((300, 4), device='cuda', generator=g)
    v = torch.randn((4, 150), device='cuda', generator=g)
    x = u @ v
    # an error of the zero singular directions grows 485 times: 2^-22 * 485
    # of the normalised matrix's norm of one, against a result's of two
    want = reference(x)
    got = ops.orthogonalize(x)
    assert float((got.double() - want).norm()) <= 485 * 2.0 ** -22 * 2
    x = torch.zeros((64, 64), device='cuda')
    x[3, 5] = -2.0
    check(ops.orthogonalize(x), x)


def test_convolution_weights_and_outputs_in_place():
    from chainerkfac_b200 import ops
    x = torch.randn((40, 6, 3, 3), device='cuda', generator=gen(8))
    want = reference(x)
    check(ops.orthogonalize(x), x, want)
    y = x.clone()
    assert ops.orthogonalize(y, outs=y) is y
    check(y, x, want)
    # rows that begin anywhere, and what stands around them
    buf = torch.full((35 * 33 + 2,), 9.0, device='cuda')
    z = buf[1:1 + 35 * 33].view(35, 33)
    z.copy_(torch.randn((35, 33), device='cuda', generator=gen(9)))
    want = reference(z)
    ops.orthogonalize(z, outs=z)
    check(z, z, want)
    assert buf[0] == 9 and buf[-1] == 9


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_weights_are_updated(dtype):
    from chainerkfac_b200 import ops
    g = gen(10)
    xs = [torch.randn(s, device='cuda', generator=g).to(dtype)
          for s in ((130, 70), (60, 200))]
    ws = [torch.randn(x.shape, device='cuda', generator=g).to(dtype)
          for x in xs]
    old = [w.clone() for w in ws]
    outs = [None, torch.empty_like(xs[1])]
    got = ops.orthogonalize(xs, outs=outs, scale=[0.5, 2.0], params=ws, lr=0.1,
                            decay=0.3)
    assert got[0] is None
    half = torch.finfo(dtype).eps / 2
    for x, w, o, s in zip(xs, ws, old, (0.5, 2.0)):
        step = 0.1 * s * reference(x)
        want = (1 - 0.03) * o.double() - step
        off = float((w.double() - want).norm())
        assert off <= tolerance(x) * float(step.norm()) + \
            2 * half * float(want.norm())
    check(got[1].float() / 2.0, xs[1])


def test_replayed_and_on_two_streams():
    from chainerkfac_b200 import _lib, ops
    xs = [torch.randn((200, 150), device='cuda', generator=gen(k))
          for k in range(3)]
    want = [ops.orthogonalize(x) for x in xs]
    x = xs[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.orthogonalize(x)
    for y, w in zip(xs, want):
        x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    torch.cuda.synchronize()
    for _ in range(5):
        for y, s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append(ops.orthogonalize(y))
    torch.cuda.synchronize()
    for k, y in enumerate(got):
        assert torch.equal(y, want[k % 3])
    status = _lib.ctypes.c_int(7)
    _lib.check(_lib.load().kfac_tc_status(_lib.ctypes.byref(status)), 'status')
    assert status.value == 0


def test_the_same_matrix_twice_and_a_weight_twice():
    from chainerkfac_b200 import _lib, ops
    x = torch.randn((300, 140), device='cuda', generator=gen(1))
    a, b = ops.orthogonalize([x, x], scale=[1.0, 2.0])
    check(a, x)
    assert torch.equal(2 * a, b)
    w = torch.zeros_like(x)
    for call in (lambda: ops.orthogonalize([x, x], params=[w, w], lr=0.1),
                 lambda: ops.orthogonalize([x, a], outs=[a, b]),
                 lambda: ops.orthogonalize([x, x[:64]], outs=[x, b[:64]])):
        with pytest.raises(_lib.KfacLibraryError, match='overlaps'):
            call()
    assert not w.any()


def test_calls_from_threads():
    """Several threads at once, a stream each, small and large matrices and an
    embedding's step in between."""
    import threading
    from chainerkfac_b200 import ops
    xs = [torch.randn(s, device='cuda', generator=gen(k)) for k, s in
          enumerate([(64, 147), (100, 900), (300, 260), (520, 390)])]
    G_inv = torch.eye(130, device='cuda')
    A, damping = torch.ones(700, device='cuda'), torch.ones(1, device='cuda')
    grad = torch.randn((700, 130), device='cuda', generator=gen(9))

    def work(x):
        return (ops.orthogonalize(x),
                ops.precondition_embedding(G_inv, A, damping, grad))
    want = [work(x) for x in xs]
    torch.cuda.synchronize()
    got, errors = {}, []

    def run(k):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                got[k] = [work(xs[k]) for _ in range(10)]
            stream.synchronize()
        except Exception as e:                     # shown below
            errors.append(e)
    threads = [threading.Thread(target=run, args=(k,)) for k in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for k, w in enumerate(want):
        for g in got[k]:
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('shape', [(256, 2304), (300, 1000), (512, 4608),
                                   (150, 160), (700, 600)])
def test_no_less_precise_than_products_in_fp32(shape, dtype):
    """Sums cut in parts of any length, and spectra where a step's rounding
    counts most: not over 1.25 times the error of the same steps in fp32."""
    from chainerkfac_b200 import ops
    here = plain = 0.0
    for seed in range(3):
        x = torch.randn(shape, device='cuda', generator=gen(seed)).to(dtype)
        want = reference(x)
        X = x.float() / x.float().norm()
        X = X.T if shape[0] > shape[1] else X
        for _ in range(5):
            A = X @ X.T
            X = 3.4445 * X + (-4.7750 * A + 2.0315 * (A @ A)) @ X
        X = (X.T if shape[0] > shape[1] else X).to(dtype)
        here += float((ops.orthogonalize(x).double() - want).norm())
        plain += float((X.double() - want).norm())
    assert here <= 1.25 * plain
