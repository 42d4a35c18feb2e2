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


def with_codes(fmt, blocks, rows, cols, channels, code, m_of_d=None):
    """`blocks` with `code` at these columns of every row; m_of_d: q4_1's m as that
    multiple of d (exact in fp16: d gets 7 bits first)."""
    nb = (cols + 31) // 32
    raw = blocks.reshape(rows, nb, ref.BLOCK[fmt]).copy()
    if fmt == "q8_0":
        for c in channels:
            raw[:, c // 32, 2 + c % 32] = code & 255
        return raw.reshape(-1)
    if m_of_d is not None:
        d = raw[:, :, 0:2].copy().view(np.uint16) & 0xfff0
        raw[:, :, 0:2] = d.view(np.uint8)
        raw[:, :, 2:4] = (d.view(np.float16) * np.float16(m_of_d)).view(np.uint8)
    at = ref.BLOCK[fmt] - 16
    for c in channels:
        b, i = c // 32, c % 32
        old = raw[:, b, at + i % 16]
        raw[:, b, at + i % 16] = (old & 0xf0) | code if i < 16 else (old & 0x0f) | (code << 4)
    return raw.reshape(-1)


def tight(x, fmt, blocks, out):
    """x W^T and the bound of the form of few rows as the header states it:
    * a value is off by half a step, 1.01 * 2^-31 of its block's largest;
    * it goes in two parts of 16 bits, together at most |x| + 2^-15 of the block's largest
      (twice the second part); a block's sum of a part is rounded as it becomes fp32, in the product with
      the block's scale and in the sum over blocks, and with the parts of the K axis and the store there are at most
      blocks + 68 roundings of the sum of magnitudes;
    * q4_1: d times the codes' sum and m times the higher digits' sum of x meet in one rounding of what
      they leave, and the lower digits' share joins in the next.  Until then the first lacks that share, |m| times at
      most 2^-7 of the block's largest per value (and no more than the value has): a magnitude too, at most twice."""
    w, _ = ref.dequantize64(fmt, blocks, out, x.shape[1])
    x = x.astype(np.float64)
    most = ref.block_max(x)
    parts = np.abs(x) + 2.0 ** -15 * most
    nb = (x.shape[1] + 31) // 32
    bound = 1.01 * 2.0 ** -31 * (most @ np.abs(w).T) + (nb + 68) * EPS * (parts @ np.abs(w).T)
    if fmt == "q4_1":
        raw = np.ascontiguousarray(blocks).reshape(out, nb, 20)
        m = np.abs(raw[:, :, 2:4].copy().view(np.float16).astype(np.float64)).reshape(out, nb)
        m = np.repeat(m, 32, 1)[:, :x.shape[1]]
        bound += 2 * EPS * (np.minimum(parts, 2.0 ** -7 * most) @ m.T)
    return x @ w.T, bound + 1e-37


# (format, the code of a strong channel, q4_1's m as a multiple of d)
ZEROS = [("q8_0", 0, None), ("q4_0", 8, None), ("q4_1", 8, -8), ("q4_1", 3, -3), ("q4_1", 15, -15), ("q4_1", 0, 0)]



@pytest.mark.parametrize("strong", [1.0, 1e3, 1e4, 1e5, 1e7])
@pytest.mark.parametrize("fmt,code,m_of_d", ZEROS)
def test_a_strong_channel_with_weights_of_zero(pkg, fmt, code, m_of_d, strong):
    """A channel whose weights are all exactly 0 costs the others only what the
    fixed point of its own block cannot hold: any place of a block, one row to 12."""
    rng = np.random.default_rng(int(strong))
    cin, out = 2048, 256
    for rows in (1, 2, 4, 7, 12):
        for channel in (5, 640 + 21, 2047):
            blocks = with_codes(fmt, ref.random_blocks(rng, fmt, out, cin), out, cin, [channel], code, m_of_d)
            x = rng.standard_normal((rows, cin)).astype(np.float32)
            x[:, channel] = strong * rng.choice([-1, 1], rows) * rng.uniform(0.5, 1, rows)
            want, bound = tight(x, fmt, blocks, out)
            y = pkg.mlq.linear_epilogue(fmt, dev(blocks), out, cin, dev(x))
            check(y, want, bound, pkg)
            if strong <= 1e4:  # half a step of the strong channel's block: below 2e-6 of an ordinary value
                err = np.linalg.norm(y.cpu().numpy() - want, axis=1) / np.linalg.norm(want, axis=1)
                assert err.max() <= 1e-6


@pytest.mark.parametrize("rows", [13, 40, 130])
@pytest.mark.parametrize("fmt,code,m_of_d", ZEROS)
def test_a_strong_channel_among_many_rows(pkg, fmt, code, m_of_d, rows):
    """The form of many rows, to the header's 1e-6 (its terms: 2^-22 of x, of w and of
    their second values' product, the sums 1e-7 as in test_moe_gpu.py)."""
    rng = np.random.default_rng(rows)
    cin, out = 2048, 256
    for strong in (1.0, 1e3, 1e4):
        blocks = with_codes(fmt, ref.random_blocks(rng, fmt, out, cin), out, cin, [700], code, m_of_d)
        x = rng.standard_normal((rows, cin)).astype(np.float32)
        x[:, 700] = strong
        want, bound = ref.product(x.astype(np.float64), fmt, blocks, out)
        y = pkg.mlq.linear_epilogue(fmt, dev(blocks), out, cin, dev(x))
        check(y, want, bound, pkg)
        err = np.linalg.norm(y.cpu().numpy() - want, axis=1) / np.linalg.norm(want, axis=1)
        assert err.max() <= 1e-6


@pytest.mark.parametrize("fmt", ["q8_0", "q4_0", "q4_1"])
@pytest.mark.parametrize("cin", [1, 31, 33, 96, 257, 300])
def test_padding_blocks_of_a_row_and_of_the_hidden_vector(pkg, fmt, cin):
    """Rows that end inside a step of 8 blocks, aligned and not, in a workspace full
    of NaN bits: what lies behind the last block reaches no sum."""
    rng = np.random.default_rng(cin)
    hid, out, n = cin + 5, 48, 3
    gate, up = (ref.random_blocks(rng, fmt, n * hid, cin) for _ in range(2))
    down = ref.random_blocks(rng, fmt, n * out, hid)
    for rows, offset in ((1, 0), (4, 0), (5, 2)):
        x = rng.standard_normal((rows, cin)).astype(np.float32)
        ids = rng.integers(0, n, (rows, 2)).astype(np.int32)
        w = rng.uniform(0.1, 1, (rows, 2)).astype(np.float32)
        on = []
        for b in (gate, up, down):
            buf = torch.zeros(b.size + 64, dtype=torch.uint8, device="cuda")
            buf[offset:offset + b.size].copy_(dev(b))
            on.append(buf[offset:offset + b.size])
        m = pkg.mlq.Experts(fmt, *on, n, cin, hid, out_features=out)
        ws = torch.full((pkg.mlq.experts_workspace_bytes(m, rows, 2),), 255, dtype=torch.uint8, device="cuda")
        want, bound = ref.experts(x, ids, w, None, fmt, fmt, gate, up, down, n, hid, out)
        check(pkg.mlq.moe_experts(m, dev(x), dev(ids), dev(w), workspace=ws), want, bound, pkg)
        ws = torch.full((pkg.mlq.epilogue_workspace_bytes(fmt, hid, cin, rows),), 255, dtype=torch.uint8, device="cuda")
        y = pkg.mlq.linear_epilogue(fmt, on[0][:gate.size // n], hid, cin, dev(x), workspace=ws)
        check(y, *ref.product(x.astype(np.float64), fmt, gate[:gate.size // n], hid), pkg)
