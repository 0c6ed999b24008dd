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
        ids=FAKE, id_bytes=4, n=5000, vocab=10, has=0, ignore=0, keys=FAKE,
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
    # one block sorts up to 4096 tokens without any
    assert lib.kfac_token_order_workspace_bytes(4096, 50000) == 0
    assert lib.kfac_token_order_workspace_bytes(4097, 50000) >= 2 * 4 * 4097
    assert lib.kfac_token_order_workspace_bytes(-1, 5) == 0
    # two partial rows a chunk of at least eight positions
    for n, width in ((1, 1), (100, 33), (70000, 2048), (2 ** 31 - 5000, 8)):
        need = lib.kfac_embedding_grad_workspace_bytes(n, width)
        assert 8 * width <= need <= 2 * 4 * (width + 3) * (n // 8 + 1)
