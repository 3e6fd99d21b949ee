"""Edges of the scoring head on the GPU: non-finite weights, tiny rows, queries of wide range, weights of tokens without
loss, bounded waits that run out, calls that have to be refused.

Tolerances count roundings: fp32 2^-24 and bf16 2^-8 of the value each (half a unit in the last place).
"""

import pytest
import torch

import vectoraccelerate_b200 as va
from test_gpu_scoring import DT, SCALE_TOL, gen, norm_reference, randn, run_norm, tctx  # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------ norm
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [200, 300, 1024, 4095, 4096])  # one vector a thread, two, rows at any address
@pytest.mark.parametrize("group", [0, 32, 64, 128])
@pytest.mark.parametrize("kind", ["nan", "inf over zero"])
def test_norm_nan_products_at_every_position(tctx, dtype, dim, group, kind):  # noqa: F811
    # the rows are finite: only the products of one column are not
    g = gen(dim)
    x = (randn(g, 3, dim) * 2).to(DT[dtype])
    w = (1 + 0.3 * randn(g, dim)).to(DT[dtype])
    size = group or dim
    columns = sorted(set(range(min(dim, 136))) | set(range(max(0, 2040), min(dim, 2056))) | set(range(dim - 9, dim)))
    for j in columns:
        bad, rows = w.clone(), x.clone()
        bad[j] = float("nan") if kind == "nan" else float("inf")
        if kind != "nan":
            rows[:, j] = 0
        codes, scales, _ = run_norm(tctx, rows, bad, None, dtype, group)
        want_codes, want_scales = norm_reference(rows, torch.where(torch.arange(dim, device="cuda") == j, 0.0, bad.float()), 1e-6, group)
        g0 = j // size
        here = torch.arange(dim, device="cuda") // size == g0
        assert torch.isnan(scales[:, g0]).all() and (codes[:, here] == 0).all(), j
        others = torch.arange(scales.shape[1], device="cuda") != g0
        assert torch.equal(codes[:, ~here].double(), want_codes[:, ~here]), j
        assert ((scales[:, others].double() - want_scales[:, others]).abs() <= SCALE_TOL * want_scales[:, others]).all(), j
