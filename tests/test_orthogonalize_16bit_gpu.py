"""Orthogonalised updates of 16-bit matrices: the products of their values in
fp32, rounded once, whatever stands beside a matrix in the call.

Against the same products in fp64 the result is off by its rounding, at most
eps / 2 of each value, and by what fp32 matrices are: 2^-22 of every operand and
a few 2^-23 of every sum, grown by up to |a|^5 = 485 along the smallest
singular values, 2e-5 of the result for shorter sides of 33 and more, 4e-5
below.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]


@pytest.fixture(autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip('no CUDA device')


def draw(shape, seed, dtype):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    return torch.randn(shape, device='cuda', generator=g).to(dtype)


def reference(x):
    x = x.double().reshape(x.shape[0], -1)
    x = x / (x.norm() + 1e-7)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    for _ in range(5):
        A = x @ x.T
        x = 3.4445 * x + (-4.7750 * A + 2.0315 * (A @ A)) @ x
    return x.T if tall else x


def check(got, x):
    want = reference(x)
    rel = float((got.double() - want).norm() / want.norm())
    sums = 2e-5 if min(want.shape) >= 33 else 4e-5
    assert rel <= torch.finfo(x.dtype).eps / 2 + sums, (x.shape, x.dtype, rel)


SHAPES = [(2, 3), (33, 385), (64, 147), (127, 3100), (100, 5000), (129, 130),
          (300, 1000), (1000, 300), (512, 4608), (700, 1100), (1024, 1024),
          (8191, 515)]


@pytest.mark.parametrize('dtype', HALVES)
@pytest.mark.parametrize('shape', SHAPES)
def test_as_in_fp32_and_rounded_once(shape, dtype):
    from chainerkfac_b200 import ops
    x = draw(shape, 1, dtype)
    got = ops.orthogonalize(x)
    check(got, x)
    assert torch.equal(got, ops.orthogonalize(x.float()).to(dtype))


@pytest.mark.parametrize('dtype', HALVES)
def test_narrow_matrices_beside_a_larger_one(dtype):
    from chainerkfac_b200 import ops
    shapes = [(2, 3), (33, 385), (300, 1000), (127, 3100), (64, 64),
              (1500, 40)]
    xs = [draw(s, k, dtype) for k, s in enumerate(shapes)]
    got = ops.orthogonalize(xs)
    floats = ops.orthogonalize([x.float() for x in xs])
    for x, y, f in zip(xs, got, floats):
        check(y, x)
        assert torch.equal(y, f.to(dtype))


@pytest.mark.parametrize('dtype', HALVES)
def test_weights_of_sixteen_bits(dtype):
    """W = W - lr X in the last product's epilogue, rounded once: the values
    of an fp32 weight."""
    from chainerkfac_b200 import ops
    for shape in ((300, 1000), (60, 200)):
        x, w = draw(shape, 1, dtype), draw(shape, 2, dtype)
        wide = w.float()
        ops.orthogonalize(x.float(), params=wide, lr=0.25, decay=0.5)
        ops.orthogonalize(x, params=w, lr=0.25, decay=0.5)
        assert torch.equal(w, wide.to(dtype))
