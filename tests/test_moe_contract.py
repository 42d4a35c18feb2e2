"""CPU tests of promises in the header about the mixture-of-experts entry
points: sizes of workspaces, and what the bindings refuse."""
from __future__ import annotations

import random

import pytest


def experts_struct(mlq, n, cin, hid, out, fmt=2, fmt_down=2):
    return mlq.ExpertsStruct(fmt, fmt_down, n, cin, hid, out, 0x1000, 0x2000, 0x3000,
                             n * hid * ((cin + 31) // 32), n * out * ((hid + 31) // 32))


def sizes(mlq, shape, k, rows):
    n, cin, hid, out = shape
    m = experts_struct(mlq, n, cin, hid, out)
    return [mlq._moe_lib().mlq_moe_experts_workspace_bytes(m, r, k) for r in rows]


# experts, in, hidden, out, top_k: few columns, or a narrow stack, so that the lists of segments weigh much; wide ones
# whose passes are shorter than the call
NARROW = [(256, 128, 64, 96, 1), (60, 96, 1, 1, 6), (400, 256, 128, 256, 1), (256, 64, 64, 64, 1), (1024, 1, 1, 1, 1),
          (1024, 33, 31, 17, 8), (481, 64, 64, 1, 1), (136, 32, 32, 32, 13), (3, 32, 32, 32, 1), (1, 1, 1, 1, 64),
          (468, 31744, 32, 64, 6), (468, 31744, 32, 1, 4), (1000, 64, 31744, 64, 8), (200, 1 << 20, 32, 32, 1)]


@pytest.mark.parametrize("c", NARROW, ids=lambda c: "-".join(map(str, c)))
def test_no_workspace_shrinks_with_more_rows(pkg, c):
    """Row by row around every border: rows per expert at which the longest
    segment steps (17, 38, 60) or the form changes (11), 32 rows, and the ends of passes.
    A call's last pass has fewer rows than the first, which its workspace is sized for."""
    n, k = c[0], c[4]
    around = {1, 32, 2 * 8192 // k, 8192 // k}
    for per_expert in (1, 2, 11, 12, 17, 38, 59, 60, 61):
        around.add(per_expert * n // k)
    rows = sorted({r for a in around for r in range(max(1, a - 40), a + 41)})
    got = sizes(pkg.mlq, c[:4], k, rows)
    assert got[0] > 0
    for r, a, b in zip(rows[1:], got, got[1:]):
        assert b >= a, (r, a, b)


def test_no_workspace_shrinks_over_random_shapes(pkg):
    rng = random.Random(5)
    log_int = lambda lo, hi: int(lo * (hi / lo) ** rng.random())  # noqa: E731
    for _ in range(300):
        c = (log_int(1, 1025), log_int(1, 40000), log_int(1, 40000), log_int(1, 40000))
        k = log_int(1, 65)
        at = log_int(1, max(2, 70 * c[0] // k))
        got = sizes(pkg.mlq, c, k, range(at, at + 60))
        assert got == sorted(got), (c, k, at)


def test_two_passes_of_unequal_length(pkg):
    """468 experts of 31744 columns, top_k 6: passes of 1326 rows, so 2651 rows
    are one of 1326 and one of 1325."""
    whole, first, last = sizes(pkg.mlq, (468, 31744, 32, 64), 6, [2651, 1326, 1325])
    assert whole == first >= last


def test_ids_of_one_row_serve_one_row_only(pkg):
    """The C call reads rows x top_k ids and weights: 1-D ones belong to a single
    row of x (CPU tensors: a call that passes the shapes is refused for its device)."""
    torch = pytest.importorskip("torch")
    mlq = pkg.mlq
    stack, down = (torch.zeros(4 * r * nb * 34, dtype=torch.uint8) for r, nb in ((32, 2), (64, 1)))
    m = mlq.Experts("q8_0", stack, stack, down, 4, 64, 32)
    ids, w = torch.zeros(2, dtype=torch.int32), torch.zeros(2)
    for x, i, v, text in [(torch.zeros(3, 64), ids, w, "ids: expected"), (torch.zeros(2, 64), ids, w, "ids: expected"),
                          (torch.zeros(3, 64), ids.expand(3, 2).contiguous(), w, "weights: expected"),
                          (torch.zeros(64), ids, w.view(1, 2), "weights: expected"),
                          (torch.zeros(64), ids[0], w, "ids: expected"),
                          (torch.zeros(64), ids, w, "CUDA"), (torch.zeros(1, 64), ids, w, "CUDA"),
                          (torch.zeros(64), ids.view(1, 2), w.view(1, 2), "CUDA"),
                          (torch.zeros(3, 64), ids.expand(3, 2).contiguous(), w.expand(3, 2).contiguous(), "CUDA")]:
        with pytest.raises(ValueError, match=text):
            mlq.moe_experts(m, x, i, v)
    # nothing to do is the library's to refuse
    for x, i, v in [(torch.zeros(0, 64), ids.view(1, 2)[:0], w.view(1, 2)[:0]), (torch.zeros(1, 64), ids[:0], w[:0])]:
        with pytest.raises(mlq.MLQError):
            mlq.moe_experts(m, x, i, v)


def test_a_refused_size_leaves_its_own_message(pkg):
    """Every size that is 0 says why, whatever failed before on this thread."""
    mlq, L = pkg.mlq, pkg.mlq._moe_lib()
    for args, text in [((7, 4, 64, 2), b"format"), ((8, 0, 64, 2), b"empty"), ((8, 4, 0, 2), b"empty"), ((8, 4, 64, 0), b"empty"),
                       ((8, 4, (1 << 20) + 1, 2), b"too large"), ((8, (1 << 24) + 1, 64, 2), b"too large")]:
        assert L.mlq_moe_route_workspace_bytes(None, 1) == 0 and b"null router" in L.mlq_last_error()
        assert L.mlq_linear_epilogue_workspace_bytes(*args) == 0
        assert b"mlq_linear_epilogue_workspace_bytes" in L.mlq_last_error() and text in L.mlq_last_error()
    m = experts_struct(mlq, 4, 64, 32, 64)
    r = mlq.RouterStruct(0x1000, None, 4, 64, 2, 0, 1, 1.0)
    for call in (lambda: L.mlq_moe_experts_workspace_bytes(m, 0, 2), lambda: L.mlq_moe_experts_workspace_bytes(m, 3, 0),
                 lambda: L.mlq_moe_experts_workspace_bytes(m, 3, 65), lambda: L.mlq_moe_route_workspace_bytes(r, 0),
                 lambda: L.mlq_moe_layer_workspace_bytes(r, m, -1)):
        assert L.mlq_linear_epilogue_workspace_bytes(7, 4, 64, 2) == 0
        assert call() == 0 and b"format" not in L.mlq_last_error()
    assert L.mlq_moe_layer_workspace_bytes(None, m, 3) == 0
    assert b"mlq_moe_layer_workspace_bytes: null router" in L.mlq_last_error()
