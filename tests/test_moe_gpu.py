"""The mixture-of-experts layer and the linear with an epilogue on the GPU,
elementwise against 64-bit references with derived bounds (moe_reference.py)."""
from __future__ import annotations

import numpy as np
import pytest

import gguf_writer as gw
import moe_reference as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def at_offset(a, offset):
    """`a` (uint8) on the device, starting `offset` bytes after an aligned address."""
    buf = torch.zeros(a.size + offset + 64, dtype=torch.uint8, device="cuda")
    v = buf[offset:offset + a.size]
    v.copy_(dev(a))
    return v


def check(got, want, bound, pkg):
    assert pkg.mlq.device_error(0) == 0
    got = got.cpu().numpy().astype(np.float64)
    assert np.isfinite(got).all()
    worst = (np.abs(got - want) / bound).max()
    assert worst <= 1.0, f"{worst} times the bound"


class Case:
    """A layer's inputs on the host, and on the device."""

    def __init__(self, pkg, fmt, fmt_down, rows, cin, hid, out, n, k, seed=0, residual=True, ids=None, offset=0):
        rng = np.random.default_rng(seed + 1000 * rows + cin)
        self.shape = (fmt, fmt_down, n, cin, hid, out)
        self.gate = ref.random_blocks(rng, fmt, n * hid, cin)
        self.up = ref.random_blocks(rng, fmt, n * hid, cin)
        self.down = ref.random_blocks(rng, fmt_down, n * out, hid)
        self.x = rng.standard_normal((rows, cin)).astype(np.float32)
        self.x[:, rng.integers(0, cin)] *= 30  # an outlier channel
        self.ids = np.stack([rng.permutation(n)[:k] for _ in range(rows)]).astype(np.int32) if ids is None else ids
        self.w = rng.uniform(0.01, 1, self.ids.shape).astype(np.float32)
        self.res = rng.standard_normal((rows, out)).astype(np.float32) if residual else None
        on = at_offset if offset else (lambda a, _: dev(a))
        self.experts = pkg.mlq.Experts(fmt, on(self.gate, offset), on(self.up, offset), on(self.down, offset), n, cin,
                                       hid, out_features=out, fmt_down=fmt_down)
        self.mlq = pkg.mlq

    def run(self, **kw):
        res = None if self.res is None else dev(self.res)
        return self.mlq.moe_experts(self.experts, dev(self.x), dev(self.ids), dev(self.w), residual=res, **kw)

    def want(self):
        fmt, fmt_down, n, _, hid, out = self.shape
        return ref.experts(self.x, self.ids, self.w, self.res, fmt, fmt_down, self.gate, self.up, self.down, n, hid, out)


# (gate/up format, down format, rows, in, hidden, out, experts, top_k): one row up to several segments of an expert (more
# than 32 rows), widths that are no multiple of 32 or of a step of 8 blocks, rows whose pitch is a multiple of 16 bytes and
# rows whose pitch is not, one of everything
CASES = [
    ("q8_0", "q8_0", 1, 256, 256, 256, 8, 2), ("q4_0", "q4_0", 1, 256, 256, 256, 8, 2),
    ("q4_1", "q4_1", 1, 256, 256, 256, 8, 2), ("q4_0", "q8_0", 2, 512, 128, 512, 4, 4),
    ("q8_0", "q4_1", 3, 1024, 352, 128, 16, 3), ("q4_1", "q4_0", 4, 2048, 96, 300, 4, 1),
    ("q4_0", "q4_0", 5, 768, 1024, 256, 2, 2), ("q8_0", "q8_0", 8, 256, 512, 1030, 3, 1),
    ("q4_1", "q8_0", 9, 512, 256, 512, 2, 1), ("q4_0", "q4_1", 17, 256, 288, 256, 3, 2),
    ("q8_0", "q4_0", 33, 256, 256, 256, 4, 2), ("q4_1", "q4_1", 70, 512, 64, 160, 2, 2),
    ("q4_0", "q8_0", 131, 288, 320, 96, 5, 3),
    ("q8_0", "q8_0", 1, 1, 1, 1, 1, 1), ("q4_0", "q4_0", 3, 33, 31, 17, 5, 2), ("q4_1", "q4_1", 2, 95, 100, 65, 7, 3),
    ("q8_0", "q4_1", 12, 96, 160, 96, 6, 2), ("q4_0", "q8_0", 40, 608, 36, 50, 9, 8),
    ("q8_0", "q8_0", 7, 2048, 1408, 256, 12, 6), ("q4_0", "q4_0", 1, 4096, 2048, 64, 3, 3),
]


# more rows per expert: mostly the form of many rows.  Segments of up to 128 rows and experts with more,
# hidden widths and outputs that end inside a tile of 64 and of 128, an odd number of blocks, rows that are not aligned, K
# axes that several CTAs share, one row above and exactly at the border to the form of few rows, two passes
CASES += [
    ("q8_0", "q8_0", 70, 256, 192, 384, 2, 1), ("q4_0", "q4_0", 300, 512, 96, 130, 2, 2),
    ("q4_1", "q8_0", 129, 2080, 65, 256, 1, 1), ("q8_0", "q4_1", 64, 3104, 128, 129, 4, 2),
    ("q4_0", "q8_0", 25, 4096, 64, 64, 4, 1), ("q8_0", "q4_0", 513, 64, 2048, 1024, 3, 1),
    ("q4_1", "q4_1", 1000, 96, 33, 40, 16, 3), ("q4_0", "q4_1", 25, 288, 160, 96, 5, 1),
    ("q4_0", "q4_1", 26, 288, 160, 96, 5, 1), ("q4_0", "q8_0", 3000, 64, 64, 32, 8, 3),
    ("q8_0", "q8_0", 128, 1024, 64, 1, 1, 1), ("q4_0", "q4_0", 2000, 1, 1, 1, 2, 1),
]


# the border itself: 11 rows per expert, and one more
CASES += [("q4_0", "q4_1", 55, 288, 160, 96, 5, 1), ("q4_0", "q4_1", 56, 288, 160, 96, 5, 1),
          ("q8_0", "q8_0", 44, 1024, 96, 200, 8, 2), ("q4_1", "q4_0", 45, 1024, 96, 200, 8, 2)]


@pytest.mark.parametrize("c", CASES, ids=lambda c: "-".join(map(str, c)))
def test_experts(pkg, c):
    t = Case(pkg, *c, residual=c[2] % 2 == 1)
    check(t.run(), *t.want(), pkg)


@pytest.mark.parametrize("fmt", ["q8_0", "q4_0", "q4_1"])
@pytest.mark.parametrize("offset", [2, 1, 16, 30])
def test_experts_at_any_address(pkg, fmt, offset):
    """Stacks that start inside a 16-byte window, at even and odd addresses."""
    for rows, n in ((3, 4), (48, 2)):
        t = Case(pkg, fmt, fmt, rows, 256, 288, 256, n, 2, offset=offset)
        check(t.run(), *t.want(), pkg)


def test_many_rows_guarded_replayed_and_not_finite(pkg):
    """A workspace of the stated size, full of NaN bits, with nothing written
    behind it; the same bits from a replayed graph; a NaN and an infinity stay
    in their rows."""
    t = Case(pkg, "q4_0", "q8_0", 150, 544, 224, 200, 3, 2)
    size = t.mlq.experts_workspace_bytes(t.experts, 150, 2)
    ws = torch.full((size + 512,), 255, dtype=torch.uint8, device="cuda")
    x, ids, w, res = dev(t.x), dev(t.ids), dev(t.w), dev(t.res)
    y = t.mlq.moe_experts(t.experts, x, ids, w, residual=res, workspace=ws[:size])
    check(y, *t.want(), pkg)
    assert (ws[size:] == 255).all()
    z = torch.empty_like(y)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        t.mlq.moe_experts(t.experts, x, ids, w, residual=res, y=z, workspace=ws[:size])
    for _ in range(2):
        z.fill_(float("nan"))
        g.replay()
        assert torch.equal(y, z)
    x[17, 3], x[90, 500] = float("nan"), float("inf")
    g.replay()
    rest = [i for i in range(150) if i not in (17, 90)]
    assert torch.equal(y[rest], z[rest]) and z[17].isnan().all() and z[90].isnan().all()
    assert pkg.mlq.device_error(0) == 0


def test_forms_side_by_side_on_streams(pkg):
    """Routers, experts and linears of both forms at once on three streams, each
    with a workspace of its own, while the next one's launches already wait
    for the last: the bits of every call are those of the call alone."""
    mlq = pkg.mlq
    rng = np.random.default_rng(21)
    few = Case(pkg, "q4_0", "q8_0", 6, 1024, 512, 768, 8, 2)
    many = Case(pkg, "q8_0", "q4_1", 200, 512, 320, 256, 4, 2)
    router = mlq.Router(dev(rng.standard_normal((64, 2048)).astype(np.float32) / 45), 4)
    xr = dev(rng.standard_normal((1024, 2048)).astype(np.float32))
    blocks = dev(ref.random_blocks(rng, "q4_0", 2048, 2048))
    xl = dev(rng.standard_normal((100, 2048)).astype(np.float32))
    on = {k: (dev(t.x), dev(t.ids), dev(t.w)) for k, t in (("few", few), ("many", many))}
    calls = [
        lambda ws: mlq.moe_experts(few.experts, *on["few"], workspace=ws),
        lambda ws: mlq.moe_experts(many.experts, *on["many"], workspace=ws),
        lambda ws: mlq.moe_route(router, xr, workspace=ws)[1],
        lambda ws: mlq.linear_epilogue("q4_0", blocks, 2048, 2048, xl, workspace=ws),
        lambda ws: mlq.linear_epilogue("q4_0", blocks, 2048, 2048, xl[:4], workspace=ws),
    ]
    size = max(mlq.experts_workspace_bytes(few.experts, 6, 2), mlq.experts_workspace_bytes(many.experts, 200, 2),
               mlq.route_workspace_bytes(router, 1024), mlq.epilogue_workspace_bytes("q4_0", 2048, 2048, 100))
    spaces = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(3)]
    want = [c(spaces[0]) for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for turn in range(12):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                n = (turn * (k + 1) + 2 * k) % len(calls)
                got.append((n, calls[n](spaces[k])))
    torch.cuda.synchronize()
    assert mlq.device_error(0) == 0
    for n, y in got:
        assert torch.equal(y, want[n])


@pytest.mark.parametrize("rows", [5, 40])
def test_slots_without_an_expert(pkg, rows):
    """-1 and ids past the stack add nothing; a row of only such slots is its
    residual, or zero; an expert named twice by a row counts twice."""
    rng = np.random.default_rng(rows)
    ids = rng.integers(0, 6, (rows, 3)).astype(np.int32)
    ids[0] = -1
    ids[1] = [2, 2, 2]
    ids[2] = [6, 1, 2 ** 31 - 1]
    ids[3] = [-2 ** 31, -7, 5]
    for residual in (True, False):
        t = Case(pkg, "q4_0", "q8_0", rows, 256, 64, 256, 6, 3, ids=ids, residual=residual)
        y = t.run()
        check(y, *t.want(), pkg)
        first = y[0].cpu().numpy()
        assert np.array_equal(first, t.res[0] if residual else np.zeros_like(first))


@pytest.mark.parametrize("rows", [3, 50])
def test_no_slot_has_an_expert(pkg, rows):
    ids = np.full((rows, 2), -1, np.int32)
    for residual in (True, False):
        t = Case(pkg, "q8_0", "q8_0", rows, 128, 64, 96, 6, 2, ids=ids, residual=residual)
        y = torch.full((rows, 96), 7.0, device="cuda")
        t.run(y=y)
        assert np.array_equal(y.cpu().numpy(), t.res if residual else np.zeros((rows, 96), np.float32))


def test_many_experts_and_skewed_load(pkg):
    """1024 experts (the most), half of all rows on one of them."""
    rng = np.random.default_rng(8)
    ids = rng.integers(0, 1024, (90, 4)).astype(np.int32)
    ids[::2, 1] = 1023
    t = Case(pkg, "q4_0", "q4_0", 90, 64, 32, 64, 1024, 4, ids=ids)
    check(t.run(), *t.want(), pkg)


def test_weights_of_zero_and_negative(pkg):
    t = Case(pkg, "q4_1", "q4_0", 6, 256, 64, 256, 6, 3)
    t.w[0] = 0
    t.w[1] *= -1
    check(t.run(), *t.want(), pkg)


def test_tiny_and_huge_activations(pkg):
    """Block scales over the fp32 range: 1e-30 next to 1e4, zeros, a subnormal."""
    t = Case(pkg, "q8_0", "q8_0", 4, 256, 64, 64, 4, 2)
    t.x[0] *= 1e-30
    t.x[1, :128] *= 1e4
    t.x[1, 128:] *= 1e-20
    t.x[2] = 0
    t.x[3, :32] = 1e-41
    y = t.run()
    want, bound = t.want()
    check(y, want, bound + 1e-36, pkg)  # below fp32's normal range the step is absolute


def test_values_that_are_not_finite_stay_in_their_row(pkg):
    """NaN and inf in x reach the outputs of their own row only; in a row
    without experts they reach nothing."""
    ids = np.array([[0, 1], [1, 2], [-1, -1], [2, 0]], np.int32)
    t = Case(pkg, "q4_0", "q4_0", 4, 256, 64, 256, 3, 2, ids=ids)
    t.x[1, 40] = np.nan
    t.x[2, :] = np.inf
    t.x[3, 7] = -np.inf
    y = t.run().cpu().numpy()
    assert np.isnan(y[1]).all() and np.isnan(y[3]).all()
    assert np.array_equal(y[2], t.res[2])
    t.x[[1, 2, 3]] = 0
    want, bound = t.want()
    assert (np.abs(y[0] - want[0]) <= bound[0]).all()


@pytest.mark.parametrize("rows", [1, 6, 48])
def test_same_bits_every_time_and_in_place(pkg, rows):
    """A repeated call gives the same bits; y may be the residual or x."""
    t = Case(pkg, "q4_0", "q8_0", rows, 256, 128, 256, 5, 3)
    first = t.run()
    x, ids, w, res = dev(t.x), dev(t.ids), dev(t.w), dev(t.res)
    ws = torch.full((pkg.mlq.experts_workspace_bytes(t.experts, rows, 3),), 255, dtype=torch.uint8, device="cuda")
    for _ in range(5):
        assert torch.equal(first, pkg.mlq.moe_experts(t.experts, x, ids, w, residual=res, workspace=ws))
    into = res.clone()
    pkg.mlq.moe_experts(t.experts, x, ids, w, residual=into, y=into, workspace=ws)
    assert torch.equal(first, into)
    into = x.clone()
    pkg.mlq.moe_experts(t.experts, into, ids, w, residual=res, y=into, workspace=ws)
    assert torch.equal(first, into)


def test_nothing_outside_the_outputs_is_written(pkg):
    """Guards around y, ids, weights, logits and the workspace (of exactly the
    size asked for) keep their bytes."""
    mlq = pkg.mlq

    def guarded(shape, dtype):
        n = int(np.prod(shape)) * torch.empty(0, dtype=dtype).element_size()
        buf = torch.full((n + 1024,), 0xA5, dtype=torch.uint8, device="cuda")
        return buf, buf[512:512 + n].view(dtype).view(shape)

    for rows in (1, 7, 45):
        t = Case(pkg, "q4_1", "q4_0", rows, 320, 100, 333, 9, 3)
        rng = np.random.default_rng(1)
        router = mlq.Router(dev(rng.standard_normal((9, 320)).astype(np.float32)), 3)
        bufs = {}
        bufs["y"], y = guarded((rows, 333), torch.float32)
        bufs["ids"], ids = guarded((rows, 3), torch.int32)
        bufs["w"], w = guarded((rows, 3), torch.float32)
        bufs["l"], logits = guarded((rows, 9), torch.float32)
        bufs["ws"], ws = guarded((mlq.layer_workspace_bytes(router, t.experts, rows),), torch.uint8)
        mlq.moe_layer(router, t.experts, dev(t.x), y=y, ids=ids, weights=w, workspace=ws)
        bufs["rws"], rws = guarded((mlq.route_workspace_bytes(router, rows),), torch.uint8)
        mlq.moe_route(router, dev(t.x), ids=ids, weights=w, logits=logits, workspace=rws)
        blocks = ref.random_blocks(rng, "q8_0", 333, 320)
        bufs["ews"], ews = guarded((mlq.epilogue_workspace_bytes("q8_0", 333, 320, rows),), torch.uint8)
        mlq.linear_epilogue("q8_0", dev(blocks), 333, 320, dev(t.x), residual=y, y=y, workspace=ews)
        torch.cuda.synchronize()
        for name, b in bufs.items():
            assert (b[:512] == 0xA5).all() and (b[-512:] == 0xA5).all(), name
    assert mlq.device_error(0) == 0


def test_two_streams_and_captured_graphs(pkg):
    """Calls on two streams with a workspace each, and two graphs captured on one stream and replayed on two, give
    the bits of the calls made alone."""
    mlq = pkg.mlq
    ts = [Case(pkg, "q4_0", "q4_0", 6, 512, 256, 512, 8, 2, seed=s) for s in (1, 2)]
    alone = [t.run() for t in ts]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ts]
    args, graphs = [], []
    for t in ts:
        args.append((dev(t.x), dev(t.ids), dev(t.w), dev(t.res), torch.empty(6, 512, device="cuda"),
                     torch.empty(mlq.experts_workspace_bytes(t.experts, 6, 2), dtype=torch.uint8, device="cuda")))
    torch.cuda.synchronize()

    def call(t, a, stream):
        mlq.moe_experts(t.experts, a[0], a[1], a[2], residual=a[3], y=a[4], workspace=a[5], stream=stream)

    for _ in range(20):
        for t, a, s in zip(ts, args, streams):
            call(t, a, s)
    torch.cuda.synchronize()
    for a, want in zip(args, alone):
        assert torch.equal(a[4], want)
    for t, a in zip(ts, args):
        a[4].zero_()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[0]):
            call(t, a, streams[0])
        graphs.append(g)
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for a, want in zip(args, alone):
        assert torch.equal(a[4], want)
    assert mlq.device_error(0) == 0


def test_graph_captures_its_own_workspace(pkg):
    """Without a workspace argument a captured call takes one from the graph's
    own pool: an eager call of another shape in between changes nothing."""
    mlq = pkg.mlq
    t, big = Case(pkg, "q4_0", "q4_0", 2, 256, 128, 256, 4, 2), Case(pkg, "q8_0", "q8_0", 64, 512, 256, 512, 4, 2)
    want = t.run()
    x, ids, w, res = dev(t.x), dev(t.ids), dev(t.w), dev(t.res)
    y = torch.empty(2, 256, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        mlq.moe_experts(t.experts, x, ids, w, residual=res, y=y)
    for _ in range(3):
        y.zero_()
        g.replay()
        big.run()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_stack_beyond_32_bit_offsets(pkg):
    """A stack of over 4 GB: the last expert's rows lie past 2^32 bytes."""
    mlq = pkg.mlq
    n, cin, hid = 70, 8192, 7424
    per = ref.bytes_of("q8_0", hid, cin)
    assert per * (n - 1) > 2 ** 32
    free, _ = torch.cuda.mem_get_info()
    if free < 4 * n * per:
        pytest.skip("not enough device memory")
    rng = np.random.default_rng(4)
    small = [ref.random_blocks(rng, "q8_0", hid, cin) for _ in range(2)]
    down = ref.random_blocks(rng, "q4_0", 64, hid)
    stack = [torch.zeros(n * per, dtype=torch.uint8, device="cuda") for _ in range(2)]
    for s, b in zip(stack, small):
        s[(n - 1) * per:].copy_(dev(b))
    downs = torch.zeros(n * down.size, dtype=torch.uint8, device="cuda")
    downs[(n - 1) * down.size:].copy_(dev(down))
    m = mlq.Experts("q8_0", stack[0], stack[1], downs, n, cin, hid, out_features=64, fmt_down="q4_0")
    x = rng.standard_normal((2, cin)).astype(np.float32)
    ids, w = np.array([[n - 1], [0]], np.int32), np.ones((2, 1), np.float32)
    y = mlq.moe_experts(m, dev(x), dev(ids), dev(w))
    want, bound = ref.experts(x[:1], np.zeros((1, 1), np.int32), w[:1], None, "q8_0", "q4_0", small[0], small[1], down, 1,
                              hid, 64)
    assert (y[1] == 0).all()  # expert 0: all zeros
    check(y[:1], want, bound, pkg)


# ---------------------------------------------------------------------------
# the router
# ---------------------------------------------------------------------------
# (rows, in, experts, top_k, scoring, bias, renormalize, scale)
ROUTES = [
    (1, 2048, 64, 6, "softmax", False, True, 1.0), (1, 1, 1, 1, "softmax", False, True, 1.0),
    (33, 896, 128, 8, "sigmoid", True, True, 2.5), (3, 100, 33, 33, "softmax", False, False, 1.0),
    (2, 4097, 1024, 64, "sigmoid", False, False, 1.0), (130, 257, 7, 2, "softmax", True, True, 1.0),
    (5, 3584, 256, 1, "sigmoid", True, False, 0.5), (64, 512, 160, 6, "softmax", False, True, 16.0),
    (4100, 64, 8, 2, "softmax", False, True, 1.0), (200, 1024, 70, 5, "sigmoid", True, True, 1.0),
]


@pytest.mark.parametrize("c", ROUTES, ids=lambda c: "-".join(map(str, c)))
def test_route(pkg, c):
    rows, cin, n, k, scoring, bias, renorm, scale = c
    rng = np.random.default_rng(rows + cin)
    x = rng.standard_normal((rows, cin)).astype(np.float32)
    w = (rng.standard_normal((n, cin)) / np.sqrt(cin)).astype(np.float32)
    b = (0.1 * rng.standard_normal(n)).astype(np.float32) if bias else None
    r = pkg.mlq.Router(dev(w), k, bias=None if b is None else dev(b), scoring=scoring, renormalize=renorm, scale=scale)
    logits = torch.empty(rows, n, device="cuda")
    ids, wt = pkg.mlq.moe_route(r, dev(x), logits=logits)
    want_ids, want_w, want_l = ref.route(x, w, k, b, scoring, renorm, scale)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    # 64-bit results rounded once
    assert (np.abs(wt.cpu().numpy() - want_w) <= 1.01 * ref.EPS * want_w).all()
    lbound = 1.01 * ref.EPS * np.abs(want_l) + 2.0 ** -50 * (np.abs(x).astype(np.float64) @ np.abs(w.T).astype(np.float64))
    assert (np.abs(logits.cpu().numpy() - want_l) <= lbound).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_ties_go_to_the_lowest_index(pkg, scoring):
    """Integer inputs: equal logits are equal in any order of summation."""
    rng = np.random.default_rng(2)
    x = rng.integers(-3, 4, (40, 64)).astype(np.float32)
    w = rng.integers(-1, 2, (5, 64)).astype(np.float32)[rng.integers(0, 5, 50)] / 8
    r = pkg.mlq.Router(dev(w), 7, scoring=scoring)
    ids, wt = pkg.mlq.moe_route(r, dev(x))
    want_ids, want_w, _ = ref.route(x, w, 7, None, scoring)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    assert (np.abs(wt.cpu().numpy() - want_w) <= 1.01 * ref.EPS * want_w).all()


def test_route_masked_experts(pkg):
    """A bias of -inf masks an expert; slots left over get -1 and weight 0."""
    rng = np.random.default_rng(6)
    x = rng.standard_normal((4, 128)).astype(np.float32)
    w = rng.standard_normal((10, 128)).astype(np.float32)
    for open_experts in ([1, 4, 9], [], list(range(10))):
        b = np.full(10, -np.inf, np.float32)
        b[open_experts] = 0
        for scoring in ("softmax", "sigmoid"):
            r = pkg.mlq.Router(dev(w), 5, bias=dev(b), scoring=scoring)
            ids, wt = pkg.mlq.moe_route(r, dev(x))
            want_ids, want_w, _ = ref.route(x, w, 5, b, scoring)
            assert np.array_equal(ids.cpu().numpy(), want_ids)
            assert np.allclose(wt.cpu().numpy(), want_w, rtol=2 * ref.EPS, atol=0)


def test_route_values_that_are_not_finite(pkg):
    """A NaN in x makes that row's logits NaN: the first experts, NaN weights;
    other rows keep their bits."""
    rng = np.random.default_rng(7)
    x = rng.standard_normal((3, 96)).astype(np.float32)
    w = rng.standard_normal((12, 96)).astype(np.float32)
    r = pkg.mlq.Router(dev(w), 4)
    ids, wt = pkg.mlq.moe_route(r, dev(x))
    x[1, 5] = np.nan
    ids2, wt2 = pkg.mlq.moe_route(r, dev(x))
    for k in (0, 2):
        assert torch.equal(ids[k], ids2[k]) and torch.equal(wt[k], wt2[k])
    assert ids2[1].tolist() == [0, 1, 2, 3] and torch.isnan(wt2[1]).all()
    # one expert's weights overflow: its logit is +inf or -inf
    x[1, 5] = 1
    big = w.copy()
    big[3] = np.float32(3e38) * np.sign(x[0])
    big[5] = -big[3]
    ids3, wt3 = pkg.mlq.moe_route(pkg.mlq.Router(dev(big), 4, scoring="sigmoid"), dev(x[:1]))
    assert ids3[0, 0] == 3 and wt3.isfinite().all() and 5 not in ids3[0].tolist()


# many rows: logits by digits, uncertain rows again in 64 bits.  From 64 Mi products
# (rows x in x experts) and 32 rows on
# (rows, in, experts, top_k, scoring, bias, renormalize, scale)
BIG_ROUTES = [
    (64, 4096, 256, 8, "softmax", False, False, 1.0), (33, 4097, 1024, 64, "sigmoid", True, True, 2.5),
    (300, 2049, 130, 6, "softmax", True, True, 1.0), (2100, 1024, 40, 2, "softmax", False, True, 1.0),
    (1025, 8192, 8, 8, "softmax", False, True, 1.0), (4096, 1030, 192, 4, "sigmoid", False, False, 1.0),
    (129, 17000, 33, 3, "sigmoid", True, True, 1.0), (2048, 36, 1000, 1, "softmax", True, True, 16.0), (1024, 4096, 16, 16, "sigmoid", False, True, 1.0),
]


def big_route(pkg, x, w, k, b, scoring, renorm, scale):
    """Runs the router and checks choice, weights and logits of finite rows."""
    r = pkg.mlq.Router(dev(w), k, bias=None if b is None else dev(b), scoring=scoring, renormalize=renorm, scale=scale)
    rows = x.shape[0]
    logits = torch.empty(rows, w.shape[0], device="cuda")
    ids, wt = pkg.mlq.moe_route(r, dev(x), logits=logits)
    want_ids, want_w, want_l = ref.route(x, w, k, b, scoring, renorm, scale)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    # a row whose bound is above 2^-15 is computed in 64 bits: then only the rounding to fp32 is left (half a step:
    # 2^-24 of the value, but 2^-150 where the value is below fp32's smallest normal one, 2^-126)
    bound = np.minimum(ref.digits_bound(x, w), 2.0 ** -15)
    assert (np.abs(logits.cpu().numpy() - want_l) <= bound + 1.01 * ref.EPS * np.abs(want_l) + 2.0 ** -150 + 2.0 ** -50 * (
        np.abs(x).astype(np.float64) @ np.abs(w.T).astype(np.float64))).all()
    # a score is off by a factor of at most exp(2 d) (softmax: its own logit and the sum), the sum of the chosen again
    rel = np.expm1(4 * bound.max(1))[:, None] + 1.01 * ref.EPS
    assert (np.abs(wt.cpu().numpy() - want_w) <= rel * want_w + 2.0 ** -150).all()
    return r, ids, wt


@pytest.mark.parametrize("c", BIG_ROUTES, ids=lambda c: "-".join(map(str, c)))
def test_route_many_rows(pkg, c):
    rows, cin, n, k, scoring, bias, renorm, scale = c
    rng = np.random.default_rng(rows + cin)
    x = rng.standard_normal((rows, cin)).astype(np.float32)
    w = (rng.standard_normal((n, cin)) / np.sqrt(cin)).astype(np.float32)
    b = (0.1 * rng.standard_normal(n)).astype(np.float32) if bias else None
    r, ids, wt = big_route(pkg, x, w, k, b, scoring, renorm, scale)
    # a workspace of exactly the stated size, filled with ones' bits; again from a graph: the same bits
    size = pkg.mlq.route_workspace_bytes(r, rows)
    ws = torch.full((size + 256,), 255, dtype=torch.uint8, device="cuda")
    xd = dev(x)
    ids2, wt2 = pkg.mlq.moe_route(r, xd, workspace=ws[:size])
    assert torch.equal(ids, ids2) and torch.equal(wt, wt2) and (ws[size:] == 255).all()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pkg.mlq.moe_route(r, xd, ids=ids2, weights=wt2, workspace=ws[:size])
    ids2.fill_(-7), wt2.fill_(-7)
    g.replay(), g.replay()
    assert torch.equal(ids, ids2) and torch.equal(wt, wt2)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_many_rows_ties_outliers_masks(pkg, scoring):
    """Equal experts (the lowest index), experts one fp32 step apart, rows of zeros, rows with
    an outlier of 1e5 and rows near the ends of fp32's range; then with masked experts."""
    rng = np.random.default_rng(12)
    rows, cin, n = 1100, 1000, 80
    x = rng.integers(-3, 4, (rows, cin)).astype(np.float32)
    w = (rng.integers(-1, 2, (11, cin)) / 64).astype(np.float32)[rng.integers(0, 11, n)]
    w[40:] = rng.standard_normal((n - 40, cin)).astype(np.float32) / 32
    w[50] = w[49]
    w[50, 3] = np.nextafter(w[50, 3], np.float32(9))
    x[5] = 0
    x[6, 10] = 1e5
    x[7] *= np.float32(1e-38)
    x[8] *= np.float32(1e30)
    x[8, 1:] = 0
    big_route(pkg, x, w, 9, None, scoring, True, 1.0)
    b = np.zeros(n, np.float32)
    b[5:] = -np.inf
    for open_experts in (3, 0):
        b[open_experts:] = -np.inf
        r = pkg.mlq.Router(dev(w), 4, bias=dev(b), scoring=scoring)
        ids, wt = pkg.mlq.moe_route(r, dev(x))
        want_ids, _, _ = ref.route(x, w, 4, b, scoring)
        assert np.array_equal(ids.cpu().numpy(), want_ids) and (wt[ids < 0] == 0).all()


@pytest.mark.parametrize("cin", [131072, 131104])
def test_route_many_rows_largest_sums(pkg, cin):
    """Every value near its row's largest, all products of one sign: the sums come
    as near to 64 bits as they can; from 131072 columns on the fp64 form takes over."""
    x = np.full((70, cin), 1.99 * 2.0 ** -10, np.float32) * np.linspace(0.9, 1, 70, dtype=np.float32)[:, None]
    w = np.full((8, cin), 1.99 * 2.0 ** -10, np.float32) * (1 - np.array([3, 1, 0, 2, 7, 5, 4, 6], np.float32) / 16)[:, None]
    _, ids, _ = big_route(pkg, x, w, 3, None, "softmax", True, 1.0)
    assert (ids.cpu().numpy() == [2, 1, 3]).all()


def test_route_many_rows_not_finite(pkg):
    """NaN or infinite rows of x take the first experts or infinite logits' order, as in
    few rows; the other rows keep their bits.  An infinite weight makes every row uncertain."""
    rng = np.random.default_rng(13)
    x = rng.standard_normal((720, 1536)).astype(np.float32)
    w = rng.standard_normal((66, 1536)).astype(np.float32)
    r = pkg.mlq.Router(dev(w), 4, scoring="sigmoid")
    ids, wt = pkg.mlq.moe_route(r, dev(x))
    y = x.copy()
    y[100, 5], y[300, 7], y[519, 0] = np.nan, np.inf, -np.inf
    ids2, wt2 = pkg.mlq.moe_route(r, dev(y))
    same = [k for k in range(720) if k not in (100, 300, 519)]
    assert torch.equal(ids[same], ids2[same]) and torch.equal(wt[same], wt2[same])
    for k in (100, 300, 519):  # one row alone is computed in 64 bits
        one, onew = pkg.mlq.moe_route(r, dev(y[k:k + 1]))
        assert torch.equal(one[0], ids2[k]) and torch.equal(onew[0].isnan(), wt2[k].isnan())
    assert ids2[100].tolist() == [0, 1, 2, 3] and wt2[100].isnan().all()
    big = w.copy()
    big[7, 3] = np.inf
    ids3, wt3 = pkg.mlq.moe_route(pkg.mlq.Router(dev(big), 4, scoring="sigmoid"), dev(x))
    want, want_w, _ = ref.route(x, big, 4, None, "sigmoid")  # a logit of inf scores 1, as any above 37 does in 64 bits
    assert np.array_equal(ids3.cpu().numpy(), want) and (np.abs(wt3.cpu().numpy() - want_w) <= 1.01 * ref.EPS * want_w).all()


# ---------------------------------------------------------------------------
# the whole layer, and a block of a model
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [1, 4, 19, 64])
def test_layer_is_route_then_experts(pkg, rows):
    mlq = pkg.mlq
    t = Case(pkg, "q4_0", "q8_0", rows, 512, 160, 512, 20, 3)
    rng = np.random.default_rng(rows)
    w = (rng.standard_normal((20, 512)) / 22).astype(np.float32)
    router = mlq.Router(dev(w), 3)
    y, ids, wt = mlq.moe_layer(router, t.experts, dev(t.x), residual=dev(t.res))
    ids2, wt2 = mlq.moe_route(router, dev(t.x))
    assert torch.equal(ids, ids2) and torch.equal(wt, wt2)
    assert torch.equal(y, mlq.moe_experts(t.experts, dev(t.x), ids, wt, residual=dev(t.res)))
    want_ids, _, _ = ref.route(t.x, w, 3)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    t.ids, t.w = ids.cpu().numpy(), wt.cpu().numpy()
    check(y, *t.want(), pkg)


def test_block_from_a_gguf_file(tmp_path, pkg):
    """A feed-forward block as a program runs it: the experts' stacks and a
    shared expert come from a GGUF file, the layer adds to the residual stream, and
    the shared expert (swiglu, then its gated down projection) adds to that."""
    mlq = pkg.mlq
    rows, cin, hid, n, k, shid = 5, 256, 96, 6, 2, 192
    rng = np.random.default_rng(12)
    gt = {"q8_0": 8, "q4_0": 2}
    made = {"ffn_gate_exps": ("q4_0", [cin, hid, n]), "ffn_up_exps": ("q4_0", [cin, hid, n]),
            "ffn_down_exps": ("q8_0", [hid, cin, n]), "ffn_gate_shexp": ("q4_0", [cin, shid]),
            "ffn_up_shexp": ("q4_0", [cin, shid]), "ffn_down_shexp": ("q8_0", [shid, cin])}
    host = {name: ref.random_blocks(rng, f, int(np.prod(dims[1:])), dims[0]) for name, (f, dims) in made.items()}
    wr = (rng.standard_normal((n, cin)) / 16).astype(np.float32)
    path = tmp_path / "moe.gguf"
    path.write_bytes(gw.build([], [(name, dims, gt[f], host[name].tobytes()) for name, (f, dims) in made.items()] +
                              [("ffn_gate_inp", [cin, n], 0, wr.tobytes())]))
    on = {}
    with mlq.GgufFile(path) as g:
        for name in list(made) + ["ffn_gate_inp"]:
            i = g.find(name)
            t = g.info(i)
            on[name] = torch.empty(t["nbytes"], dtype=torch.uint8, device="cuda")
            g.upload_rows(i, 0, t["rows"], on[name].data_ptr(), t["nbytes"])
    router = mlq.Router(on["ffn_gate_inp"].view(torch.float32).view(n, cin), k)
    ex = mlq.Experts("q4_0", on["ffn_gate_exps"], on["ffn_up_exps"], on["ffn_down_exps"], n, cin, hid, fmt_down="q8_0")
    x = rng.standard_normal((rows, cin)).astype(np.float32)
    stream = rng.standard_normal((rows, cin)).astype(np.float32)
    gate = rng.uniform(0, 1, rows).astype(np.float32)
    y, ids, wt = mlq.moe_layer(router, ex, dev(x), residual=dev(stream))
    h = mlq.linear_swiglu("q4_0", on["ffn_gate_shexp"], on["ffn_up_shexp"], shid, cin, dev(x))
    out = mlq.linear_epilogue("q8_0", on["ffn_down_shexp"], cin, shid, h, row_scale=dev(gate), residual=y)
    want, bound = ref.experts(x, ids.cpu().numpy(), wt.cpu().numpy(), stream, "q4_0", "q8_0", host["ffn_gate_exps"],
                              host["ffn_up_exps"], host["ffn_down_exps"], n, hid, cin)
    check(y, want, bound, pkg)
    # the shared expert's own step, on the h that the library gave
    w2, b2 = ref.epilogue(h.cpu().numpy(), "q8_0", host["ffn_down_shexp"], cin, None, "none", gate, y.cpu().numpy())
    check(out, w2, b2, pkg)


# ---------------------------------------------------------------------------
# the linear with an epilogue
# ---------------------------------------------------------------------------
# (format, rows, in, out, bias, activation, row_scale, residual)
LINEARS = [
    ("q8_0", 1, 4096, 256, False, "none", False, True), ("q4_0", 1, 2048, 1000, True, "silu", False, False),
    ("q4_1", 2, 1024, 520, True, "gelu", True, True), ("q8_0", 3, 100, 33, False, "gelu_tanh", False, False),
    ("q4_0", 4, 256, 4864, True, "relu", False, True), ("q4_1", 5, 896, 129, False, "sigmoid", True, False),
    ("q8_0", 8, 320, 64, True, "none", True, True), ("q4_0", 13, 96, 200, True, "gelu", False, True),
    ("q4_1", 31, 2560, 48, True, "silu", True, True), ("q8_0", 32, 256, 256, False, "gelu", False, False),
    ("q4_0", 33, 512, 1, True, "gelu_tanh", False, True), ("q4_1", 301, 64, 96, True, "sigmoid", False, True),
    ("q8_0", 65, 1, 5, True, "none", False, False), ("q4_0", 1, 32, 1, False, "none", False, False),
    ("q4_1", 1, 18944, 64, False, "none", False, True), ("q8_0", 17, 272, 77, False, "relu", True, True),
    # segments of 2 and of 4 rows, the borders between the forms and between one segment and two, K axes shared by CTAs
    ("q4_0", 3, 2048, 512, False, "none", False, True), ("q8_0", 4, 2048, 6000, True, "silu", True, False),
    ("q8_0", 12, 4096, 256, False, "none", True, True), ("q4_0", 12, 704, 300, True, "gelu", False, False),
    ("q4_1", 13, 4096, 130, False, "none", True, True), ("q8_0", 40, 18944, 64, False, "none", False, True),
    ("q4_0", 128, 1312, 256, True, "relu", False, False), ("q4_1", 129, 352, 200, False, "none", True, True),
    ("q8_0", 1000, 2080, 40, True, "sigmoid", False, False), ("q4_0", 257, 5000, 129, False, "none", False, False),
]


@pytest.mark.parametrize("c", LINEARS, ids=lambda c: "-".join(map(str, c)))
def test_linear_epilogue(pkg, c):
    fmt, rows, cin, out, bias, act, scale, residual = c
    rng = np.random.default_rng(rows * 7 + cin)
    blocks = ref.random_blocks(rng, fmt, out, cin)
    x = rng.standard_normal((rows, cin)).astype(np.float32)
    b = rng.standard_normal(out).astype(np.float32) if bias else None
    s = rng.uniform(-1, 1, rows).astype(np.float32) if scale else None
    r = rng.standard_normal((rows, out)).astype(np.float32) if residual else None
    on = lambda a: None if a is None else dev(a)  # noqa: E731
    for offset in (0, 6):
        y = pkg.mlq.linear_epilogue(fmt, at_offset(blocks, offset), out, cin, dev(x), bias=on(b), activation=act,
                                    row_scale=on(s), residual=on(r))
        check(y, *ref.epilogue(x, fmt, blocks, out, b, act, s, r), pkg)


def test_linear_epilogue_vector_and_in_place(pkg):
    """1-D x gives a 1-D y; y may be the residual, or x of the same width."""
    rng = np.random.default_rng(3)
    blocks = ref.random_blocks(rng, "q4_0", 256, 256)
    w, x = dev(blocks), dev(rng.standard_normal(256).astype(np.float32))
    res = dev(rng.standard_normal(256).astype(np.float32))
    y = pkg.mlq.linear_epilogue("q4_0", w, 256, 256, x, residual=res)
    assert tuple(y.shape) == (256,)
    into = res.clone()
    pkg.mlq.linear_epilogue("q4_0", w, 256, 256, x, residual=into, y=into)
    assert torch.equal(into, y)
    into = x.clone()
    pkg.mlq.linear_epilogue("q4_0", w, 256, 256, into, residual=res, y=into)
    assert torch.equal(into, y)


def test_linear_epilogue_activations_of_extreme_values(pkg):
    """Zero weights: y = act(bias), at values where naive forms overflow."""
    v = np.array([0, -0.0, 1e-38, -1e-3, 5, -5, 20, -20, 90, -90, 1e4, -1e4, 1e30, -1e30], np.float32)
    blocks = torch.zeros(v.size * 34, dtype=torch.uint8, device="cuda")
    x = torch.ones(1, 32, device="cuda")
    for act in ("none", "silu", "gelu", "gelu_tanh", "relu", "sigmoid"):
        y = pkg.mlq.linear_epilogue("q8_0", blocks, v.size, 32, x, bias=dev(v), activation=act).cpu().numpy()[0]
        with np.errstate(over="ignore"):
            want = ref.act64(v.astype(np.float64), act)
        assert np.isfinite(y).all()
        assert (np.abs(y - want) <= 16 * ref.EPS * (np.abs(want) + 1)).all(), act
