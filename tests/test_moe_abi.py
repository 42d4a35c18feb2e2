"""CPU tests of the mixture-of-experts entry points and of the linear with an
epilogue: structs match the header, every refusal happens on the host before any
CUDA call (the pointers are fake), and the 64-bit reference of the GPU tests
agrees with the oracle's decoding."""
from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

import moe_reference as ref

ROOT = Path(__file__).resolve().parents[1]


def test_structs_and_constants_match_header(pkg, tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not found")
    mlq = pkg.mlq
    checks = [("mlq_router", mlq.RouterStruct), ("mlq_experts", mlq.ExpertsStruct), ("mlq_epilogue", mlq.EpilogueStruct)]
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "mlq.h"', "int main(void) {"]
    want = []
    for cname, cls in checks:
        lines.append(f'  printf("%zu\\n", sizeof({cname}));')
        want.append(ctypes.sizeof(cls))
        for f, _ in cls._fields_:
            lines.append(f'  printf("%zu\\n", offsetof({cname}, {f}));')
            want.append(getattr(cls, f).offset)
    for c, v in [("MLQ_MOE_MAX_EXPERTS", mlq.MOE_MAX_EXPERTS), ("MLQ_MOE_MAX_TOP_K", mlq.MOE_MAX_TOP_K),
                 ("MLQ_SCORE_SOFTMAX", mlq.SCORINGS["softmax"]), ("MLQ_SCORE_SIGMOID", mlq.SCORINGS["sigmoid"]),
                 ("MLQ_ACT_NONE", mlq.ACTIVATIONS["none"]), ("MLQ_ACT_SILU", mlq.ACTIVATIONS["silu"]),
                 ("MLQ_ACT_GELU", mlq.ACTIVATIONS["gelu"]), ("MLQ_ACT_GELU_TANH", mlq.ACTIVATIONS["gelu_tanh"]),
                 ("MLQ_ACT_RELU", mlq.ACTIVATIONS["relu"]), ("MLQ_ACT_SIGMOID", mlq.ACTIVATIONS["sigmoid"])]:
        lines.append(f'  printf("%d\\n", (int){c});')
        want.append(v)
    lines.append("  return 0;\n}")
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines) + "\n")
    exe = tmp_path / "layout"
    subprocess.run([gcc, "-std=c99", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == want


def router(mlq, w=0x1000, bias=None, n=8, cin=64, k=2, scoring=0, renorm=1, scale=1.0):
    return mlq.RouterStruct(w, bias, n, cin, k, scoring, renorm, scale)


def experts(mlq, fmt=8, fmt_down=2, n=8, cin=64, hid=32, out=64, gate=0x1000, up=0x2000, down=0x3000, nb=None, nbd=None):
    return mlq.ExpertsStruct(fmt, fmt_down, n, cin, hid, out, gate, up, down,
                             n * hid * ((cin + 31) // 32) if nb is None else nb,
                             n * out * ((hid + 31) // 32) if nbd is None else nbd)


def test_workspace_of_more_rows_serves_fewer(pkg):
    mlq = pkg.mlq
    L = mlq._moe_lib()
    rows = sorted({*range(1, 140), *range(140, 9000, 61), 2047, 2048, 2049, 4096, 4097, 16384, 16385, 20000})
    for n, cin, hid, out, k in ((8, 64, 32, 64, 2), (60, 3584, 2560, 3584, 4), (128, 2048, 768, 2048, 8),
                                (1024, 7168, 96, 64, 64), (1, 1, 1, 1, 1), (3, 40000, 500, 100, 1)):
        r, m = router(mlq, n=n, cin=cin, k=k), experts(mlq, n=n, cin=cin, hid=hid, out=out)
        for size in (lambda i: L.mlq_moe_route_workspace_bytes(r, i), lambda i: L.mlq_moe_experts_workspace_bytes(m, i, k),
                     lambda i: L.mlq_moe_layer_workspace_bytes(r, m, i),
                     lambda i: L.mlq_linear_epilogue_workspace_bytes(8, out, cin, i)):
            sizes = [size(i) for i in rows]
            assert sizes[0] > 0 and sizes == sorted(sizes)


BIG = 1 << 40  # a workspace size that is never too small


@pytest.mark.parametrize("change,status,text", [
    ({"w": None}, 2, b"null router weights"), ({"n": 0}, 3, b"empty"), ({"cin": 0}, 3, b"empty"),
    ({"k": 0}, 3, b"empty"), ({"n": 1025}, 9, b"at most 1024 experts"), ({"k": 9}, 9, b"top_k"),
    ({"n": 128, "k": 65}, 9, b"top_k"), ({"scoring": 2}, 9, b"scoring"), ({"renorm": 2}, 9, b"renormalize"),
    ({"cin": (1 << 20) + 1}, 9, b"too large"),
])
def test_router_refusals(pkg, change, status, text):
    mlq, L = pkg.mlq, pkg.mlq._moe_lib()
    r = router(mlq, **change)
    assert L.mlq_moe_route(r, 0x5000, 1, 0x6000, 0x7000, None, 0x10000, BIG, None) == status
    assert text in L.mlq_last_error()
    assert L.mlq_moe_route_workspace_bytes(r, 1) == 0
    assert L.mlq_moe_layer(r, experts(mlq), 0x5000, 1, None, 0x6000, 0x7000, 0x8000, 0x10000, BIG, None) == status


def test_route_call_refusals(pkg):
    mlq, L = pkg.mlq, pkg.mlq._moe_lib()
    r = router(mlq)
    need = L.mlq_moe_route_workspace_bytes(r, 3)
    assert need > 0
    ok = [r, 0x5000, 3, 0x6000, 0x7000, None, 0x10000, need, None]
    for at, value, status, text in [(0, None, 2, b"null router"), (1, None, 2, b"null input"), (2, 0, 3, b"empty"),
                                    (2, 1 << 30, 9, b"too many rows"), (3, None, 2, b"null"), (4, None, 2, b"null"),
                                    (6, None, 2, b"null workspace"), (6, 0x10010, 9, b"256-byte aligned"),
                                    (7, need - 1, 9, b"needed")]:
        args = list(ok)
        args[at] = value
        assert L.mlq_moe_route(*args) == status, (at, value)
        assert text in L.mlq_last_error()


@pytest.mark.parametrize("change,status,text", [
    ({"fmt": 7}, 1, b"format"), ({"fmt_down": 0}, 1, b"format"), ({"gate": None}, 2, b"null weight"),
    ({"up": None}, 2, b"null weight"), ({"down": None}, 2, b"null weight"), ({"n": 0}, 3, b"empty"),
    ({"cin": -1}, 3, b"empty"), ({"hid": 0}, 3, b"empty"), ({"out": 0}, 3, b"empty"),
    ({"n": 1025}, 9, b"at most 1024 experts"), ({"nb": 5}, 5, b"gate/up block count mismatch: expected 512, got 5"),
    ({"nbd": 7}, 5, b"down block count mismatch: expected 512, got 7"),
    ({"n": 1024, "hid": 1 << 21}, 9, b"too large"), ({"n": 1024, "out": 1 << 22}, 9, b"too large"),
])
def test_experts_refusals(pkg, change, status, text):
    mlq, L = pkg.mlq, pkg.mlq._moe_lib()
    m = experts(mlq, **change)
    assert L.mlq_moe_experts(m, 0x5000, 1, 2, 0x6000, 0x7000, None, 0x8000, 0x10000, BIG, None) == status
    assert text in L.mlq_last_error()
    assert L.mlq_moe_experts_workspace_bytes(m, 1, 2) == 0
    assert L.mlq_moe_layer(router(mlq), m, 0x5000, 1, None, 0x6000, 0x7000, 0x8000, 0x10000, BIG, None) == status


def test_experts_call_refusals(pkg):
    mlq, L = pkg.mlq, pkg.mlq._moe_lib()
    m = experts(mlq)
    need = L.mlq_moe_experts_workspace_bytes(m, 3, 2)
    assert need > 0
    ok = [m, 0x5000, 3, 2, 0x6000, 0x7000, None, 0x8000, 0x10000, need, None]
    for at, value, status, text in [(0, None, 2, b"null experts"), (1, None, 2, b"null input"), (2, 0, 3, b"empty"),
                                    (2, -4, 3, b"empty"), (3, 0, 3, b"empty"), (3, 65, 9, b"top_k"),
                                    (2, 1 << 30, 9, b"too many rows"), (4, None, 2, b"null"), (5, None, 2, b"null"),
                                    (7, None, 2, b"null"), (8, None, 2, b"null workspace"),
                                    (8, 0x10080, 9, b"256-byte aligned"), (9, need - 1, 9, b"needed")]:
        args = list(ok)
        args[at] = value
        assert L.mlq_moe_experts(*args) == status, (at, value)
        assert text in L.mlq_last_error()


def test_layer_call_refusals(pkg):
    mlq, L = pkg.mlq, pkg.mlq._moe_lib()
    m, r = experts(mlq), router(mlq)
    need = L.mlq_moe_layer_workspace_bytes(r, m, 3)
    assert need >= L.mlq_moe_experts_workspace_bytes(m, 3, 2)
    ok = [r, m, 0x5000, 3, None, 0x6000, 0x7000, 0x8000, 0x10000, need, None]
    for at, value, status, text in [(0, router(mlq, n=16), 4, b"differ"), (0, router(mlq, cin=32), 4, b"differ"),
                                    (2, None, 2, b"null"), (3, 0, 3, b"empty"), (5, None, 2, b"null"),
                                    (6, None, 2, b"null"), (7, None, 2, b"null"), (8, None, 2, b"null workspace"),
                                    (9, need - 1, 9, b"needed")]:
        args = list(ok)
        args[at] = value
        assert L.mlq_moe_layer(*args) == status, (at, value)
        assert text in L.mlq_last_error()


def test_epilogue_refusals(pkg):
    mlq, L = pkg.mlq, pkg.mlq._moe_lib()
    ep = mlq.EpilogueStruct(None, 0, None, None)
    need = L.mlq_linear_epilogue_workspace_bytes(8, 4, 64, 2)
    assert need > 0 and L.mlq_linear_epilogue_workspace_bytes(7, 4, 64, 2) == 0
    ok = [8, 0x1000, 8, 4, 64, 0x5000, 2, ep, 0x6000, 0x10000, need, None]
    for at, value, status, text in [(0, 7, 1, b"format"), (1, None, 2, b"null weight"), (2, 7, 5, b"expected 8, got 7"),
                                    (3, 0, 3, b"empty"), (4, 0, 3, b"empty"), (6, 0, 3, b"empty"),
                                    (5, None, 2, b"null"), (7, None, 2, b"null"), (8, None, 2, b"null"),
                                    (7, mlq.EpilogueStruct(None, 6, None, None), 9, b"activation"),
                                    (7, mlq.EpilogueStruct(None, -1, None, None), 9, b"activation"),
                                    (9, None, 2, b"null workspace"), (9, 0x10008, 9, b"256-byte aligned"),
                                    (10, need - 1, 9, b"needed"), (4, (1 << 20) + 32, 9, b"too large")]:
        args = list(ok)
        args[at] = value
        assert L.mlq_linear_epilogue(*args) == status, (at, value)
        assert text in L.mlq_last_error()


def test_bindings_refuse_wrong_tensors(pkg):
    """The bindings pass bare pointers on, so they check type, shape,
    density and device first (CPU tensors: refused, nothing runs)."""
    torch = pytest.importorskip("torch")
    mlq = pkg.mlq
    w = torch.zeros(4, 64)
    r = mlq.Router(w, 2)
    with pytest.raises(ValueError, match="CUDA"):
        mlq.moe_route(r, torch.zeros(3, 64))
    with pytest.raises(ValueError, match="expected .rows, 64."):
        mlq.moe_route(r, torch.zeros(3, 32))
    with pytest.raises(ValueError, match="float32"):
        mlq.moe_route(r, torch.zeros(3, 64, dtype=torch.float64))
    with pytest.raises(ValueError, match="contiguous"):
        mlq.moe_route(r, torch.zeros(64, 3).t())
    with pytest.raises(ValueError, match="scoring"):
        mlq.Router(w, 2, scoring="top")
    with pytest.raises(mlq.MLQError, match="top_k"):
        mlq.route_workspace_bytes(mlq.Router(w, 5), 1)
    blocks = torch.zeros(4 * 32 * 2 * 34, dtype=torch.uint8)
    down = torch.zeros(4 * 64 * 34, dtype=torch.uint8)
    m = mlq.Experts("q8_0", blocks, blocks, down, 4, 64, 32)
    with pytest.raises(ValueError, match="w_down: expected"):
        mlq.Experts("q8_0", blocks, blocks, blocks[:-1], 4, 64, 32)
    ids, wt = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2)
    with pytest.raises(ValueError, match="CUDA"):
        mlq.moe_experts(m, torch.zeros(3, 64), ids, wt)
    with pytest.raises(ValueError, match="activation"):
        mlq.linear_epilogue("q8_0", blocks, 128, 64, torch.zeros(1, 64), activation="tanh")
    with pytest.raises(ValueError, match="w: expected"):
        mlq.linear_epilogue("q8_0", blocks, 127, 64, torch.zeros(1, 64))


@pytest.mark.parametrize("fmt", ["q8_0", "q4_0", "q4_1"])
def test_reference_decodes_like_the_oracle(oracle, fmt):
    rng = np.random.default_rng(3)
    blocks = ref.random_blocks(rng, fmt, 5, 70)
    w, mag = ref.dequantize64(fmt, blocks, 5, 70)
    got = oracle.dequantize(fmt, blocks, 5, 70).reshape(5, 70)
    # the oracle rounds d * c (+ m) to fp32, at most twice
    assert np.abs(got - w).max() <= 2 * ref.EPS * mag.max()
    assert (mag >= np.abs(w) * (1 - 1e-12)).all()
