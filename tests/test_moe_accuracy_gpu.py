"""Accuracy of the quantized products where values of x differ much in size, or
are near the ends of fp32's range: elementwise against 64 bits, with bounds of the
weights as they are (no allowance for codes that are summed apart from their offset)."""
from __future__ import annotations

import numpy as np
import pytest

import moe_reference as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
EPS = ref.EPS


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def check(got, want, bound, pkg):
    assert pkg.mlq.device_error(0) == 0
    got = got.cpu().numpy().astype(np.float64)
    assert np.isfinite(got).all()
    worst = (np.abs(got - want) / bound).max()
    assert worst <= 1.0, f"{worst} times the bound"


@pytest.mark.parametrize("fmt", ["q8_0", "q4_0", "q4_1"])
@pytest.mark.parametrize("rows", [1, 2, 4, 5, 12, 13])
def test_largest_finite_values(pkg, fmt, rows):
    """Every finite x is a value, up to fp32's largest, at any place of a block
    and in both forms (up to 12 rows, and more)."""
    rng = np.random.default_rng(rows)
    cin, out = 256, 128
    blocks = ref.random_blocks(rng, fmt, out, cin)
    x = rng.standard_normal((rows, cin)).astype(np.float32)
    x[:, ::3] *= np.float32(3e37) / 4
    x[0, 1], x[0, 17], x[-1, 40] = np.finfo(np.float32).max, 3e37, -np.finfo(np.float32).max
    y = pkg.mlq.linear_epilogue(fmt, dev(blocks), out, cin, dev(x))
    want, bound = ref.product(x.astype(np.float64), fmt, blocks, out)
    assert np.abs(want).max() < 3e38
    check(y, want, bound, pkg)


@pytest.mark.parametrize("fmt", ["q8_0", "q4_0", "q4_1"])
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_largest_finite_hidden_values(pkg, fmt, rows):
    """The hidden vector too may come near fp32's largest value."""
    rng = np.random.default_rng(rows)
    cin, hid, out = 128, 96, 64
    gate, up = (ref.random_blocks(rng, fmt, 2 * hid, cin) for _ in range(2))
    down = ref.random_blocks(rng, fmt, 2 * out, hid)
    x = rng.standard_normal((rows, cin)) * 1e19
    ids = np.tile(np.array([[1, 0]], np.int32), (rows, 1))
    w = np.full((rows, 2), 0.5, np.float32)
    with np.errstate(over="ignore"):
        # silu(g) = g or 0 at such sizes: the hidden values grow with the square of x
        hidden = lambda x: max(np.abs(np.maximum(g, 0) * u).max() for g, u in (  # noqa: E731
            [ref.product(x, fmt, b[e * b.size // 2:(e + 1) * b.size // 2], hid)[0] for b in (gate, up)] for e in (0, 1)))
        x = (x * np.sqrt(1e38 / hidden(x))).astype(np.float32)
        want, bound = ref.experts(x, ids, w, None, fmt, fmt, gate, up, down, 2, hid, out)
    assert 2.0 ** 124 < hidden(x.astype(np.float64)) < 3e38 and np.abs(want).max() < 3e38
    m = pkg.mlq.Experts(fmt, dev(gate), dev(up), dev(down), 2, cin, hid, out_features=out)
    check(pkg.mlq.moe_experts(m, dev(x), dev(ids), dev(w)), want, bound, pkg)
