"""Token embeddings on the device: lookup, sorted tokens, gradient and counts
against plain fp64 arithmetic.

Tolerances are bounds, not measurements: a lookup rounds one fp32 product
(2^-24) and its result once more to the output's type (eps / 2); a sum of k
terms in fp32, in any order, is within (k - 1) 2^-24 of the sum of its terms'
sizes, and the scaling, the addition onto `out` and the rounding add 2^-24 and
eps / 2 of what they give.  Doubled where second-order terms could matter.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip('no CUDA device')


def half(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    return g


def tokens(n, vocab, seed, skew=True):
    u = torch.rand(n, device='cuda', generator=gen(seed), dtype=torch.float64)
    ids = (vocab * (u ** 4 if skew else u)).long().clamp_(max=vocab - 1)
    return ids


def grad_reference(gy, ids, vocab, scale):
    """fp64 gradient, the sum of its terms' sizes and the terms per token."""
    ids = ids.reshape(-1)
    gy = gy.reshape(ids.numel(), -1).double()
    live = (ids >= 0) & (ids < vocab)
    ids, gy = ids[live].long(), gy[live]
    want = torch.zeros((vocab, gy.shape[1]), dtype=torch.float64, device='cuda')
    size = torch.zeros_like(want)
    want.index_add_(0, ids, gy)
    size.index_add_(0, ids, gy.abs())
    return want * scale, size * abs(scale), \
        torch.bincount(ids, minlength=vocab).double()


def check_grad(got, gy, ids, vocab, scale, old=None):
    want, size, k = grad_reference(gy, ids, vocab, scale)
    if old is not None:
        want = want + old.double()
        size = size + old.double().abs()
        k = k + 1
    bound = 2 * (k[:, None] + 2) * U * size + half(got.dtype) * want.abs() * 1.01
    if got.dtype == torch.float16:
        bound = bound + 2.0 ** -25           # below its normal numbers
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off - bound).max())


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n,vocab,width', [
    (1, 7, 1), (1, 50, 1024), (3, 50, 8), (257, 1000, 513), (64, 5, 130),
    (1000, 333, 66), (4099, 4000, 260), (20000, 77, 4)])
def test_lookup(n, vocab, width, dtype):
    from chainerkfac_b200 import ops
    w = torch.randn((vocab, width), device='cuda', generator=gen(1)).to(dtype)
    ids = tokens(n, vocab, 2)
    ids[::5] = vocab - 1
    ids[-1] = 0
    got = ops.embedding(w, ids, scale=1.7)
    want = w.double()[ids] * float(torch.tensor(1.7, dtype=torch.float32))
    assert got.dtype == dtype and got.shape == (n, width)
    assert bool(((got.double() - want).abs() <=
                 (half(dtype) + 2 * U) * want.abs() + 2.0 ** -25).all())
    assert torch.equal(got, ops.embedding(w, ids.int(), scale=1.7))
    if dtype != torch.float16:
        assert torch.equal(ops.embedding(w, ids), w[ids])


def test_lookup_of_ignored_and_outside_tokens():
    from chainerkfac_b200 import ops
    w = torch.randn((10, 12), device='cuda', generator=gen(1))
    ids = torch.tensor([[3, -1, 10], [9, 2 ** 40, 4]], device='cuda')
    got = ops.embedding(w, ids, ignore_label=-1)
    assert got.shape == (2, 3, 12)
    assert torch.equal(got[0, 0], w[3]) and torch.equal(got[1, 0], w[9])
    assert not got[0, 1].any()
    assert got[0, 2].isnan().all() and got[1, 1].isnan().all()
    assert ops.embedding(w, ids)[0, 1].isnan().all()
    # a label inside the vocabulary
    got = ops.embedding(w, ids, ignore_label=4)
    assert not got[1, 2].any() and got[0, 1].isnan().all()
    # values that are not finite go through
    w[3, 0], w[3, 1] = float('inf'), float('nan')
    got = ops.embedding(w, ids[0, :1])
    assert torch.isinf(got[0, 0]) and torch.isnan(got[0, 1])
    assert ops.embedding(w, ids[:0]).shape == (0, 3, 12)


def test_lookup_leaves_what_is_behind_its_rows():
    from chainerkfac_b200 import ops
    for width, offset in ((6, 3), (64, 0), (33, 1)):
        buf = torch.full((offset + 5 * width + 7,), 9.0, device='cuda')
        w = torch.randn(4 * width + 1, device='cuda', generator=gen(1))
        w = w[1:].view(4, width)             # 4-byte aligned only
        out = buf[offset:offset + 5 * width].view(5, width)
        ids = torch.tensor([0, 3, 1, 2, 3], device='cuda')
        ops.embedding(w, ids, out=out)
        assert torch.equal(out, w[ids])
        assert (buf[:offset] == 9).all() and (buf[offset + 5 * width:] == 9).all()


@pytest.mark.parametrize('n', [1, 2, 31, 33, 512, 1025, 2049, 4097, 9000, 20000,
                               65537, 131072, 131073, 300001])
@pytest.mark.parametrize('vocab', [1, 2, 511, 512, 50021, 300000])
def test_order_is_a_stable_sort(n, vocab):
    from chainerkfac_b200 import ops
    ids = tokens(n, vocab, n + vocab)
    ids[n // 2::7] = -1
    order = ops.TokenOrder(ids, vocab, ignore_label=-1)
    keys = torch.where((ids < 0) | (ids >= vocab), vocab, ids)
    want, at = torch.sort(keys, stable=True)
    assert torch.equal(order.keys.long(), want)
    assert torch.equal(order.positions.long(), at)


def test_order_of_wide_vocabulary_and_of_narrow_tokens():
    from chainerkfac_b200 import ops
    for vocab in (2 ** 18 - 1, 2 ** 18, 2 ** 27 + 11, 2 ** 31 - 2):
        ids = tokens(6000, vocab, 5, skew=False)
        ids[17], ids[18], ids[19] = vocab - 1, vocab, 0
        order = ops.TokenOrder(ids, vocab)
        want, at = torch.sort(ids, stable=True)
        assert torch.equal(order.keys.long(), want)
        assert torch.equal(order.positions.long(), at)
        small = ops.TokenOrder(ids[:100].int(), vocab)
        assert torch.equal(small.positions.long(),
                           torch.sort(ids[:100], stable=True)[1])


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n,vocab,width', [
    (1, 3, 1), (1, 40, 1024), (7, 3, 5), (64, 1, 33), (100, 4000, 64),
    (513, 37, 771), (4097, 500, 130), (9001, 3, 40), (30000, 20011, 516),
    (70000, 100, 24)])
def test_gradient(n, vocab, width, dtype):
    from chainerkfac_b200 import ops
    ids = tokens(n, vocab, n)
    gy = torch.randn((n, width), device='cuda', generator=gen(3)).to(dtype)
    order = ops.TokenOrder(ids, vocab)
    scale = 0.5 if n > 60 else 3.0
    got = ops.embedding_grad(gy, order, scale=scale)
    check_grad(got, gy, ids, vocab, scale)
    assert torch.equal(got, ops.embedding_grad(gy, order, scale=scale))
    # onto rows that are there; the others stay as they are
    old = torch.randn((vocab, width), device='cuda', generator=gen(4)).to(dtype)
    out = old.clone()
    ops.embedding_grad(gy, order, scale=scale, out=out, accumulate=True)
    check_grad(out, gy, ids, vocab, scale, old=old)
    absent = torch.ones(vocab, dtype=torch.bool, device='cuda')
    absent[ids] = False
    assert torch.equal(out[absent], old[absent])


@pytest.mark.parametrize('ids', [
    [-1] * 100,                                # nothing at all
    [5] * 1000,                                # one token in every chunk
    [0] * 500 + [9] * 500, [9] * 8 + [-1] * 92,
    list(range(10)) * 50, [3] * 7 + [4] * 9 + [10, 11, 2 ** 40]])
def test_gradient_where_chunks_begin_and_end(ids):
    from chainerkfac_b200 import ops
    ids = torch.tensor(ids, device='cuda')
    gy = torch.randn((ids.numel(), 36), device='cuda', generator=gen(8))
    gy[ids < 0] = float('nan')                 # nobody reads these
    out = torch.full((10, 36), float('nan'), device='cuda')
    ops.embedding_grad(gy, ops.TokenOrder(ids, 10, ignore_label=-1), out=out)
    check_grad(out, torch.nan_to_num(gy), ids, 10, 1.0)


def test_gradient_of_no_tokens_clears_or_leaves():
    from chainerkfac_b200 import ops
    order = ops.TokenOrder(torch.empty(0, dtype=torch.int64, device='cuda'), 50)
    gy = torch.empty((0, 17), device='cuda')
    assert not ops.embedding_grad(gy, order).any()
    out = torch.ones((50, 17), device='cuda')
    ops.embedding_grad(gy, order, out=out, accumulate=True)
    assert (out == 1).all()


def test_gradient_of_unaligned_rows():
    from chainerkfac_b200 import ops
    for width, dtype in ((64, torch.float32), (64, torch.bfloat16),
                         (33, torch.bfloat16), (34, torch.float16)):
        ids = tokens(300, 20, 1)
        gy = torch.randn(300 * width + 1, device='cuda',
                         generator=gen(2)).to(dtype)[1:].view(300, width)
        buf = torch.full((20 * width + 3,), 9.0, dtype=dtype, device='cuda')
        out = buf[1:1 + 20 * width].view(20, width)
        ops.embedding_grad(gy, ops.TokenOrder(ids, 20), out=out)
        check_grad(out, gy, ids, 20, 1.0)
        assert buf[0] == 9 and (buf[1 + 20 * width:] == 9).all()


def test_offsets_beyond_32_bits():
    """Rows whose elements lie past 2^31 in the weight and the gradient."""
    from chainerkfac_b200 import ops
    vocab, width = 2 ** 21 + 5, 1040
    w = torch.zeros((vocab, width), dtype=torch.bfloat16, device='cuda')
    w[-1], w[-3] = 2.0, 5.0
    ids = torch.tensor([vocab - 1, 0, vocab - 3], device='cuda')
    got = ops.embedding(w, ids, scale=2.0)
    assert (got[0] == 4).all() and not got[1].any() and (got[2] == 10).all()
    gy = torch.ones((3, width), dtype=torch.bfloat16, device='cuda')
    w.fill_(7.0)
    ops.embedding_grad(gy, ops.TokenOrder(ids, vocab), scale=3.0, out=w)
    assert (w[vocab - 1] == 3).all() and (w[vocab - 3] == 3).all()
    assert (w[0] == 3).all() and not w[1:vocab - 3].any()


@pytest.mark.parametrize('n,vocab', [(0, 9), (1, 1), (1000, 7), (70000, 40000)])
def test_counts(n, vocab):
    from chainerkfac_b200 import ops
    ids = tokens(n, vocab, 6)
    ids[::3] = -1
    count = torch.bincount(ids[ids >= 0], minlength=vocab).double()
    old = torch.rand(vocab, device='cuda', generator=gen(1))
    out, mean = old.clone(), torch.full((1, 1), 2.0, device='cuda')
    ops.token_counts(ids, vocab, -1, alpha=0.25, beta=0.5, out=out, mean=mean)
    want = 0.25 * count + 0.5 * old.double()
    assert bool(((out.double() - want).abs() <= 2 * U * want).all())
    m = 0.25 * float(count.sum()) / vocab + 1.0
    assert abs(float(mean) - m) <= 3 * U * m
    assert torch.equal(ops.token_counts(ids, vocab, -1).double(), count)


def test_replayed_with_new_tokens_and_on_two_streams():
    from chainerkfac_b200 import ops
    vocab, width, n = 900, 96, 5000
    ids, gy = tokens(n, vocab, 1), torch.randn((n, width), device='cuda')

    def step(ids, gy):
        return ops.embedding_grad(gy, ops.TokenOrder(ids, vocab))
    graphs = []
    for _ in range(2):                        # two graphs, replayed at once
        a, b = ids.clone(), gy.clone()
        step(a, b)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(a, b)
        graphs.append((g, a, b, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for k, (g, a, b, out) in enumerate(graphs):
        a.copy_(tokens(n, vocab, 10 + k))
        b.copy_(torch.randn((n, width), device='cuda', generator=gen(k)))
    torch.cuda.synchronize()
    for _ in range(20):
        for (g, a, b, out), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for g, a, b, out in graphs:
        assert torch.equal(out, step(a, b))
        check_grad(out, b, a, vocab, 1.0)
    # sorted on one stream, walked on another
    order = ops.TokenOrder(ids, vocab)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.embedding_grad(gy, order)
    del order
    junk = [torch.full((n,), -1, dtype=torch.int32, device='cuda')
            for _ in range(8)]
    torch.cuda.synchronize()
    assert torch.equal(got, step(ids, gy)) and len(junk) == 8
