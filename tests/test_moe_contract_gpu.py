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


def test_stream_given_and_nothing_else(pkg):
    """Outputs and workspace that a call on another stream allocates are not what
    the current stream has just let go of and still writes, and what that stream is
    given next is not the call's workspace."""
    mlq = pkg.mlq
    rng = np.random.default_rng(4)
    rows, cin, hid, n, k = 40, 512, 256, 8, 2
    m = mlq.Experts("q4_0", *(dev(ref.random_blocks(rng, "q4_0", n * r, c)) for r, c in ((hid, cin), (hid, cin), (cin, hid))),
                    n, cin, hid)
    router = mlq.Router(dev(rng.standard_normal((n, cin)).astype(np.float32) / 23), k)
    x = dev(rng.standard_normal((rows, cin)).astype(np.float32))
    want = [t.clone() for t in mlq.moe_layer(router, m, x)]
    size = mlq.layer_workspace_bytes(router, m, rows)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for stream in (side, side.cuda_stream):
        # blocks of the sizes that the call needs, let go with a write of theirs still to come
        left = [torch.empty(size, dtype=torch.uint8, device="cuda"), torch.empty(rows, cin, device="cuda"),
                torch.empty(rows, k, dtype=torch.int32, device="cuda"), torch.empty(rows, k, device="cuda")]
        torch.cuda._sleep(100_000_000)
        for t in left:
            t.view(torch.uint8).fill_(255)
        gone = {t.data_ptr() for t in left}
        del left, t
        got = mlq.moe_layer(router, m, x, stream=stream)
        assert not gone & {t.data_ptr() for t in got}
        after = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        assert mlq.device_error(0) == 0
        for a, b in zip(want, (got[0], got[1], got[2])):
            assert torch.equal(a, b)
        del got, after
    # the default stream by its handle, while another one is current
    with torch.cuda.stream(side):
        got = mlq.moe_layer(router, m, x, stream=0)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_stream_given_under_capture(pkg):
    """A captured fork: the call runs on a second stream that joins the capture by
    events, and takes its workspace from the graph's pool."""
    mlq = pkg.mlq
    rng = np.random.default_rng(5)
    w = dev(ref.random_blocks(rng, "q4_0", 256, 512))
    x = dev(rng.standard_normal((3, 512)).astype(np.float32))
    want = mlq.linear_epilogue("q4_0", w, 256, 512, x).clone()
    torch.cuda.synchronize()
    side, z = torch.cuda.Stream(), torch.empty(3, 256, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        side.wait_stream(torch.cuda.current_stream())
        y = mlq.linear_epilogue("q4_0", w, 256, 512, x, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        z.copy_(y)
    for _ in range(2):
        z.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(z, want)
    assert mlq.device_error(0) == 0


@pytest.mark.parametrize("rows", [300, 3000])
def test_layer_of_a_prompt(pkg, rows):
    """More rows than a pass of either half holds (2048 of the router, 2730 of the
    experts with 3 slots): the bits of the halves, also written over x and over the residual."""
    mlq = pkg.mlq
    rng = np.random.default_rng(rows)
    n, cin, hid, k = 16, 256, 96, 3
    stacks = [ref.random_blocks(rng, f, n * r, c) for f, r, c in (("q4_0", hid, cin), ("q4_0", hid, cin), ("q4_1", cin, hid))]
    m = mlq.Experts("q4_0", *(dev(b) for b in stacks), n, cin, hid, fmt_down="q4_1")
    w = (rng.standard_normal((n, cin)) / 16).astype(np.float32)
    router = mlq.Router(dev(w), k)
    host = rng.standard_normal((rows, cin)).astype(np.float32)
    x = dev(host)
    y, ids, wt = mlq.moe_layer(router, m, x, residual=x)
    want_ids, _, _ = ref.route(host, w, k)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    ids2, wt2 = mlq.moe_route(router, x)
    assert torch.equal(ids, ids2) and torch.equal(wt, wt2)
    assert torch.equal(y, mlq.moe_experts(m, x, ids, wt, residual=x))
    into = x.clone()
    mlq.moe_layer(router, m, into, residual=into, y=into)
    assert torch.equal(y, into)
    some = [0, 1, rows // 2, 2047 % rows, 2048 % rows, 2729 % rows, 2730 % rows, rows - 1]
    want, bound = ref.experts(host[some], want_ids[some], wt.cpu().numpy()[some], host[some], "q4_0", "q4_1", *stacks, n,
                              hid, cin)
    check(y[some], want, bound, pkg)
