"""What the operators for token models refuse, and their host arithmetic (no
GPU needed: every refusal is raised before anything is launched)."""

import ctypes

import pytest
import torch


@pytest.fixture(scope='module')
def lib():
    from chainerkfac_b200 import _build, _lib
    _build.build()
    return _lib.load()


def message(lib):
    return lib.kfac_last_error().decode()


FAKE = ctypes.c_void_p(4096)      # an address that nothing may read


def test_cpu_tensors_are_refused():
    from chainerkfac_b200 import _lib, ops
    w, ids = torch.zeros(4, 3), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: ops.embedding(w, ids),
                 lambda: ops.TokenOrder(ids, 4),
                 lambda: ops.token_counts(ids, 4)):
        with pytest.raises(_lib.KfacLibraryError, match='CUDA tensor'):
            call()


def test_embedding_calls_are_checked(lib):
    look = lambda **k: lib.kfac_embedding(*({**dict(
        dtype=0, weight=FAKE, vocab=10, width=4, ids=FAKE, id_bytes=8, n=5,
        has=0, ignore=0, scale=1.0, out=FAKE, stream=None), **k}).values())
    for bad in (dict(dtype=3), dict(width=0), dict(vocab=0), dict(id_bytes=2),
                dict(n=-1), dict(n=2 ** 31), dict(vocab=2 ** 31),
                dict(weight=None), dict(out=None), dict(ids=None)):
        assert look(**bad) == 1, bad
        assert 'embedding' in message(lib)
    assert look(n=0, weight=None, out=None, ids=None) == 0


def test_token_orders_and_gradients_are_checked(lib):
    order = lambda **k: lib.kfac_token_order(*({**dict(
        ids=FAKE, id_bytes=4, n=500000, vocab=10, has=0, ignore=0, keys=FAKE,
        positions=FAKE, ws=FAKE, nbytes=1 << 30, stream=None), **k}).values())
    assert order(id_bytes=3) == 1 and order(keys=None) == 1
    assert order(ws=None) == 3 and order(nbytes=100) == 3
    assert order(ws=ctypes.c_void_p(4097)) == 1
    assert order(n=0) == 0
    grad = lambda **k: lib.kfac_embedding_grad(*({**dict(
        dtype=0, gy=FAKE, width=8, keys=FAKE, positions=FAKE, n=100, vocab=10,
        scale=1.0, accumulate=0, out=FAKE, ws=FAKE, nbytes=1 << 30,
        stream=None), **k}).values())
    assert grad(dtype=-1) == 1 and grad(width=0) == 1 and grad(gy=None) == 1
    assert grad(out=None) == 1 and grad(nbytes=8) == 3 and grad(ws=None) == 3
    assert grad(n=0, accumulate=1) == 0       # nothing to add
    counts = lambda **k: lib.kfac_token_counts(*({**dict(
        ids=FAKE, id_bytes=8, n=100, vocab=10, has=0, ignore=0, alpha=1.0,
        beta=0.0, out=FAKE, mean=None, ws=FAKE, nbytes=40, stream=None),
        **k}).values())
    assert counts(out=None) == 1 and counts(nbytes=39) == 3
    assert counts(vocab=-4) == 1


def test_workspaces_of_the_sort_and_the_gradient(lib):
    # one launch sorts up to 131072 tokens without any
    assert lib.kfac_token_order_workspace_bytes(131072, 50000) == 0
    assert lib.kfac_token_order_workspace_bytes(131073, 50000) >= 2 * 4 * 131073
    assert lib.kfac_token_order_workspace_bytes(-1, 5) == 0
    # two partial rows a chunk of at least eight positions
    for n, width in ((1, 1), (100, 33), (70000, 2048), (2 ** 31 - 5000, 8)):
        need = lib.kfac_embedding_grad_workspace_bytes(n, width)
        assert 8 * width <= need <= 2 * 4 * (width + 3) * (n // 8 + 1)


def ortho(lib, **k):
    import numpy as np
    from chainerkfac_b200 import _lib
    a = {**dict(dtype=0, rows=[4], cols=[6], x=[4096], out=[8192], param=None,
                scale=[1.0], steps=2, coef=[3.0, -4.0, 2.0] * 2, eps=1e-7,
                lr=0.0, decay=0.0, ws=4096, nbytes=1 << 40), **k}
    ptrs = lambda v: None if v is None else _lib.ptr_array(v)
    return lib.kfac_orthogonalize(
        a['dtype'], a.get('count', len(a['rows'])), _lib.int_array(a['rows']),
        _lib.int_array(a['cols']), ptrs(a['x']), ptrs(a['out']),
        ptrs(a['param']), _lib.float_array(a['scale']), a['steps'],
        _lib.float_array(a['coef']), a['eps'], a['lr'], a['decay'],
        ctypes.c_void_p(a['ws']), a['nbytes'], None)


def test_orthogonalize_calls_are_checked(lib):
    for bad in (dict(dtype=5), dict(rows=[0]), dict(cols=[-1]),
                dict(rows=[2 ** 20 + 1]), dict(steps=0), dict(steps=65),
                dict(eps=-1.0), dict(eps=float('nan')), dict(x=None),
                dict(x=[None]), dict(out=None), dict(out=[None]),
                dict(out=[None], param=[None]), dict(count=-1)):
        assert ortho(lib, **bad) == 1, bad
        assert 'orthogonalize' in message(lib)
    big = dict(rows=[300], cols=[200])
    assert ortho(lib, nbytes=64, **big) == 3 and ortho(lib, ws=None, **big) == 3
    assert ortho(lib, rows=[], cols=[], x=[], out=[], scale=[]) == 0


def test_workspace_of_an_orthogonalisation(lib):
    """Two places of X, A and the polynomial, four bytes an element, rows of
    whole 16-byte words."""
    from chainerkfac_b200 import _lib

    def need(*shapes):
        return lib.kfac_orthogonalize_workspace_bytes(
            len(shapes), _lib.int_array([s[0] for s in shapes]),
            _lib.int_array([s[1] for s in shapes]))
    for r, c in ((129, 130), (64, 3500), (1000, 240), (4096, 4096)):
        small = min(r, c)
        least = 4 * (2 * r * c + 2 * small * small)
        assert least <= need((r, c)) <= \
            least + 4 * (2 * r * 8 + 2 * small * 8) + 8192
    assert need((300, 300), (300, 20)) >= \
        need((300, 300)) + need((300, 20)) - 512
    # small ones stay in shared memory, unless they ride along with others
    assert need((1, 1), (64, 147), (256, 128), (100, 2000)) == 0
    assert need((64, 147), (300, 300)) > need((300, 300)) + 8 * 64 * 147
    assert need() == 0 and need((0, 4)) == 0


def test_orthogonalize_refuses_what_is_not_a_matrix():
    from chainerkfac_b200 import _lib, ops
    x = torch.zeros(3, 4)
    with pytest.raises(_lib.KfacLibraryError, match='CUDA tensor'):
        ops.orthogonalize(x)
    for bad in (dict(steps=0), dict(steps=65), dict(coefficients=(1.0, 2.0)),
                dict(coefficients=[(1.0, 2.0, 3.0)] * 4), dict(scale=[1.0] * 2)):
        with pytest.raises(ValueError):
            ops.orthogonalize([x], **bad)
    assert ops.orthogonalize([]) == []


def test_precondition_embedding_calls_are_checked(lib):
    step = lambda **k: lib.kfac_precondition_embedding(*({**dict(
        vocab=100, width=12, G=FAKE, A=FAKE, damping=FAKE, grad=FAKE, kf=FAKE,
        param=None, mom=None, lr=0.1, momentum=0.9, ws=FAKE, nbytes=1 << 30,
        stream=None), **k}).values())
    for bad in (dict(vocab=0), dict(width=0), dict(vocab=2 ** 31),
                dict(width=2 ** 20 + 1), dict(G=None), dict(A=None),
                dict(damping=None), dict(grad=None), dict(kf=None),
                dict(param=FAKE), dict(mom=FAKE)):
        assert step(**bad) == 1, bad
        assert 'precondition_embedding' in message(lib)
    assert step(ws=None) == 3 and step(nbytes=1000) == 3
    need = lib.kfac_precondition_embedding_workspace_bytes
    assert need(0, 5) == 0 and need(5, 0) == 0
    for v, d in ((1, 1), (1000, 100), (32000, 1024)):
        assert 4 * (v + d) * d <= need(v, d) <= \
            4 * (v + d) * (d + 7) + 8 * v + 4 * d + 4096
    from chainerkfac_b200 import _lib, ops
    x = torch.zeros(3, 3)
    with pytest.raises(_lib.KfacLibraryError, match='CUDA tensor'):
        ops.precondition_embedding(x, x[0], x[0, :1], x)


def test_results_do_not_overlap_what_is_read(lib):
    at = ctypes.c_void_p
    far = [at((k + 1) << 40) for k in range(9)]
    look = lambda **k: lib.kfac_embedding(*({**dict(
        dtype=0, weight=far[0], vocab=10, width=4, ids=far[1], id_bytes=8, n=5,
        has=0, ignore=0, scale=1.0, out=far[2], stream=None), **k}).values())
    for bad in (dict(out=far[0]), dict(out=at((1 << 40) + 156)),
                dict(out=at((1 << 40) - 76)), dict(out=at((2 << 40) + 36))):
        assert look(**bad) == 1, bad
        assert 'overlaps' in message(lib)
    order = lambda **k: lib.kfac_token_order(*({**dict(
        ids=far[0], id_bytes=4, n=50, vocab=10, has=0, ignore=0, keys=far[1],
        positions=far[2], ws=None, nbytes=0, stream=None), **k}).values())
    for bad in (dict(keys=far[0]), dict(positions=far[0]),
                dict(positions=at((2 << 40) + 196))):
        assert order(**bad) == 1 and 'overlaps' in message(lib), bad
    grad = lambda **k: lib.kfac_embedding_grad(*({**dict(
        dtype=1, gy=far[0], width=8, keys=far[1], positions=far[2], n=100,
        vocab=10, scale=1.0, accumulate=0, out=far[3], ws=far[4],
        nbytes=1 << 30, stream=None), **k}).values())
    for bad in (far[0], far[1], far[2], far[4], at((1 << 40) - 158)):
        assert grad(out=bad) == 1 and 'overlaps' in message(lib), bad
    counts = lambda **k: lib.kfac_token_counts(*({**dict(
        ids=far[0], id_bytes=8, n=100, vocab=10, has=0, ignore=0, alpha=1.0,
        beta=0.0, out=far[1], mean=far[2], ws=far[3], nbytes=40, stream=None),
        **k}).values())
    for bad in (dict(out=far[0]), dict(out=far[3]), dict(mean=far[1]),
                dict(mean=far[0]), dict(mean=far[3])):
        assert counts(**bad) == 1 and 'overlaps' in message(lib), bad
    step = lambda **k: lib.kfac_precondition_embedding(*({**dict(
        vocab=100, width=12, G=far[0], A=far[1], damping=far[2], grad=far[3],
        kf=far[4], param=far[5], mom=far[6], lr=0.1, momentum=0.9, ws=far[7],
        nbytes=1 << 30, stream=None), **k}).values())
    for bad in (dict(kf=far[0]), dict(kf=far[1]), dict(kf=far[2]),
                dict(kf=far[5]), dict(kf=at((4 << 40) + 4)), dict(mom=far[5]),
                dict(mom=far[3]), dict(param=far[3]), dict(param=far[7])):
        assert step(**bad) == 1 and 'overlaps' in message(lib), bad
    big = 1 << 30
    for bad in (dict(out=[8192, 8192]), dict(out=[8192, 4096]),
                dict(out=[4100, big]), dict(out=None, param=[8192, 8192]),
                dict(out=[8192, big], param=[8192, 2 * big]),
                dict(out=[16384 + 4, big]), dict(out=[8192, 8192 + 92])):
        got = ortho(lib, **{**dict(rows=[4, 4], cols=[6, 6], x=[4096, 16384],
                                   scale=[1.0, 1.0]), **bad})
        assert got == 1 and 'overlaps' in message(lib), bad


def test_arrays_are_aligned_and_rows_have_a_size(lib):
    at = ctypes.c_void_p
    far = [at((k + 1) << 40) for k in range(9)]
    odd = at((20 << 40) + 2)
    for k in (dict(ids=at(4100)), dict(weight=odd), dict(out=odd),
              dict(width=(1 << 28) + 1)):
        assert lib.kfac_embedding(*({**dict(
            dtype=0, weight=far[0], vocab=10, width=4, ids=far[1], id_bytes=8,
            n=5, has=0, ignore=0, scale=1.0, out=far[2], stream=None),
            **k}).values()) == 1, k
        assert 'aligned' in message(lib) or '2^28' in message(lib)
    assert ortho(lib, x=[4098]) == 1 and 'aligned' in message(lib)
    assert ortho(lib, out=[4099], dtype=1) == 1 and 'aligned' in message(lib)
    for name in ('G', 'A', 'damping', 'grad', 'kf'):
        assert lib.kfac_precondition_embedding(*({**dict(
            vocab=100, width=12, G=far[0], A=far[1], damping=far[2],
            grad=far[3], kf=far[4], param=None, mom=None, lr=0.1, momentum=0.9,
            ws=far[7], nbytes=1 << 30, stream=None), name: odd}).values()) == 1
        assert 'aligned' in message(lib)
    from chainerkfac_b200 import ops
    assert ops._c_int(7) == 7
    assert ctypes.c_int(ops._c_int(2 ** 32 + 5)).value == 2 ** 31 - 1
