"""The form that each size of a product with 4-bit weights takes, on the CPU: the sizes of the GPU tests
reach every one of them."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from semblend_amd import _lib

from . import quantized_forms as forms

HERE = Path(__file__).resolve().parent


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = tmp_path_factory.mktemp("w4") / "w4_plan"
    subprocess.run([gxx, "-O2", "-std=c++17", "-o", str(exe), str(HERE / "w4_plan.cpp")], check=True,
                   capture_output=True, text=True)

    def run(sizes):
        text = "\n".join(f"{m} {n} {k} {g} {int(dt is torch.bfloat16)}" for m, n, k, g, dt in sizes)
        r = subprocess.run([str(exe)], input=text, capture_output=True, text=True, timeout=60, check=True)
        return r.stdout.splitlines()

    return run


def test_sizes_take_their_forms(plan):
    both = (forms.BF16, forms.FP16)
    want = {(*s, dt): "rows " + f for d in (forms.ROWS, forms.ROWS_ONCE) for s, f in d.items() for dt in both}
    want.update({s: "tiles " + f for s, f in forms.TILES.items()})
    got = dict(zip(want, plan(want)))
    assert got == want
    assert all(f.startswith("tiles") for f in plan(forms.KINDS))


def test_every_form_is_there(plan):
    """Rows: R of 4 with one and two tiles of features, of 16, 32 and 64 with one to four, three kinds of
    groups, sixteen waves for one tile of up to 16 rows, codes read once for more. Tiles: both types, kinds of
    groups, whole and in slices, slices of sums alone, vectors and single features."""
    rows = set(forms.ROWS.values())
    for gpt in (1, 2, 4):
        for r, js in ((4, (1, 2)), (16, (1, 2, 3, 4)), (32, (1, 2, 3, 4)), (64, (1, 2, 3, 4))):
            for j in js:
                assert f"{r} {j} {gpt} {7 if (r, j) == (64, 4) else 8} 0" in rows
                if r <= 16:
                    assert (f"{r} {j} {gpt} 16 0" in rows) if j == 1 else (
                        f"{r} {j} {gpt} 8 1" in forms.ROWS_ONCE.values())
    kinds = set()
    for (m, n, k, g, dt), f in forms.TILES.items():
        gpt, splits, per, sums = map(int, f.split())
        kinds.add((dt, gpt, splits > 1, n % 8 == 0))
        if splits > 1 and dt is forms.BF16:
            codes = -(-k // 128)
            starts = [s * per for s in range(splits)]
            kinds.add((gpt, "sums alone" if any(b >= codes for b in starts) else "",
                       "both" if any(b < codes < b + per for b in starts) else ""))
    for dt in (forms.BF16, forms.FP16):
        for gpt in (1, 2, 4):
            assert {(dt, gpt, s, v) for s in (False, True) for v in (False, True)} <= kinds
    assert any(k[1] == "sums alone" for k in kinds if len(k) == 3)
    assert any(k[2] == "both" for k in kinds if len(k) == 3)


def test_plan_is_the_librarys(plan):
    """The library's workspaces are those of the plan compiled here: sums of 256 bytes a row and step, parts of
    four bytes an output and slice."""
    sizes = list(forms.TILES) + forms.KINDS + [(*s, dt) for s in forms.ROWS for dt in (forms.BF16, forms.FP16)]
    for (m, n, k, g, dt), line in zip(sizes, plan(sizes)):
        f = line.split()
        want = 0
        if f[0] == "tiles":
            splits, sums = int(f[2]), int(f[4])
            want = m * sums * 256 + (splits * m * n * 4 if splits > 1 else 0)
        assert _lib.size_query("sb_w4_linear_workspace_size", m, n, k, g, _lib.SB_DTYPE[dt]) == want
