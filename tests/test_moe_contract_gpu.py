"""Promises in the header about the mixture-of-experts entry points, on the GPU."""
from __future__ import annotations

import numpy as np
import pytest

import moe_reference as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


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


# experts, in, hidden, out, top_k, rows, rows of the first pass: the last pass has one row less than the first and more
# segments, or is a few rows in the other form
@pytest.mark.parametrize("c", [(468, 31744, 32, 64, 6, 2651, 1326), (60, 96, 64, 64, 6, 1365 + 5, 1365)],
                         ids=lambda c: "-".join(map(str, c)))
def test_two_passes_stay_in_their_workspace(pkg, c):
    """A workspace of exactly the stated size with guards around it."""
    n, cin, hid, out, k, rows, first = c
    mlq = pkg.mlq
    rng = np.random.default_rng(rows)
    # the stack repeats four experts
    gate, up = (ref.random_blocks(rng, "q4_0", 4 * hid, cin) for _ in range(2))
    down = ref.random_blocks(rng, "q4_0", 4 * out, hid)
    m = mlq.Experts("q4_0", *(dev(b).repeat(n // 4) for b in (gate, up, down)), n, cin, hid, out_features=out)
    x = rng.standard_normal((rows, cin), dtype=np.float32)
    ids = rng.integers(0, n, (rows, k), dtype=np.int32)
    w = rng.uniform(0.1, 1, (rows, k)).astype(np.float32)
    size = mlq.experts_workspace_bytes(m, rows, k)
    buf = torch.full((size + 8192,), 0xA5, dtype=torch.uint8, device="cuda")
    y = mlq.moe_experts(m, dev(x), dev(ids), dev(w), workspace=buf[4096:4096 + size])
    torch.cuda.synchronize()
    assert (buf[:4096] == 0xA5).all() and (buf[4096 + size:] == 0xA5).all()
    some = [0, first - 1, first, rows - 1]
    want, bound = ref.experts(x[some], ids[some] % 4, w[some], None, "q4_0", "q4_0", gate, up, down, 4, hid, out)
    check(y[some], want, bound, pkg)
