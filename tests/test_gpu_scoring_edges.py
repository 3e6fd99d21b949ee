"""Edges of the scoring head on the GPU: non-finite weights, tiny rows, queries of wide range, weights of tokens without
loss, bounded waits that run out, calls that have to be refused.

Tolerances count roundings: fp32 2^-24 and bf16 2^-8 of the value each (half a unit in the last place).
"""

import time

import numpy as np
import pytest
import torch

import vectoraccelerate_b200 as va
from test_gpu_scoring import (DT, SCALE_TOL, U16, U32, check_loss, gen, loss_reference, make_loss,  # noqa: F401
                              make_queries, make_table, matvec_reference, matvec_tolerance, norm_reference, randn,
                              run_loss, run_matvec, run_norm, tctx, unpack)

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


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim, group", [(64, 0), (200, 32), (1000, 0), (4096, 128), (4095, 0)])
@pytest.mark.parametrize("eps", [0.0, 1e-30])
def test_norm_tiny_rows_without_epsilon(tctx, dtype, dim, group, eps):  # noqa: F811
    # the squares of these rows are below fp32's range, or so near its bottom that they keep few bits
    g = gen(dim)
    sizes = torch.tensor([2.0 ** -60, 2.0 ** -64, 2.0 ** -70, 2.0 ** -75, 2.0 ** -78, 2.0 ** -100, 2.0 ** -120, 0.0, 1.0], device="cuda")
    x = (randn(g, 9, dim).clamp(-4, 4) * sizes[:, None]).to(DT[dtype])
    for lift in (1.0, 2.0 ** 60):  # (the second lifts the rows of 2^-100 and 2^-120 above what counts as zero)
        w = ((1 + 0.3 * randn(g, dim)) * lift).to(DT[dtype])
        codes, scales, _ = run_norm(tctx, x, w, None, dtype, group, eps)
        want_codes, want_scales = norm_reference(x, w, eps, group)
        top = want_scales * 127 * torch.sqrt((x.double() ** 2).mean(1) + eps)[:, None]
        live = top >= 2.0 ** -80
        assert live[:5].all() and live[8].all() and not live[7].any() and live[5:7].all() == (lift > 1)
        size = group or dim
        at = torch.arange(dim, device="cuda") // size
        assert torch.equal(codes.double(), torch.where(live[:, at], want_codes, 0.0))
        # a scale near the bottom of fp32's range is off by up to half its last unit, 2^-150, besides
        want = torch.where(live, want_scales, 0.0)
        assert ((scales.double() - want).abs() <= SCALE_TOL * want + 2.0 ** -150).all()


# ------------------------------------------------------------------------------------------ 4-bit rows
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n, dim, group, nq, zeros", [(400, 512, 64, 1, False), (333, 520, 32, 2, True), (300, 4096, 32, 1, True), (200, 4096, 128, 2, False),
                                                     (300, 1544, 64, 3, False), (257, 2304, 32, 8, True), (300, 4090, 128, 17, False), (100, 512, 64, 9, True)])
@pytest.mark.parametrize("outlier", [2.0 ** 20, 2.0 ** 34])
def test_matvec_outliers_that_meet_zero(tctx, dtype, n, dim, group, nq, zeros, outlier):  # noqa: F811
    # the columns of the outliers hold what stands for zero: the answer is made of the other elements alone
    g = gen(dim + nq)
    codes, scales, zp = make_table(g, n, dim, group, "f32", zeros)
    x, _ = make_queries(g, nq, dim, dtype)
    x = (randn(g, nq, dim)).to(DT[dtype])
    for j in range(1, dim, 30):
        x[:, j] *= outlier
        nibble = (zp[:, j // group].to(torch.int32) & 15 if zeros else torch.zeros(n, dtype=torch.int32, device="cuda")).to(torch.uint8)
        byte = codes[:, j // 2]
        codes[:, j // 2] = (byte & 0xF0) | nibble if j % 2 == 0 else (byte & 0x0F) | (nibble << 4)
    out = run_matvec(tctx, x, None, codes, scales, zp, dim, group)
    want, size = matvec_reference(x, None, codes, scales, zp, dim, group)
    # one or two queries are multiples of 2^-62 of the power of two above their group's largest |x| (< 2 times that):
    # off by at most 2^-62 of it
    at = torch.arange(dim, device="cuda") // group
    groups = -(-dim // group)
    top = torch.nn.functional.pad(x.abs().double(), (0, -dim % group)).view(nq, groups, group).amax(2)[:, at]
    w = unpack(codes, dim) - (zp.to(torch.int32)[:, at] if zeros else 0)
    w = (w.double() * scales.double()[:, at]).abs()
    assert ((out.double() - want).abs() <= matvec_tolerance(dim, group) * size + 2.0 ** -62 * (top @ w.t())).all()


def test_matvec_wide_queries_in_strided_rows(tctx):  # noqa: F811
    # fp32 queries over more than 1536 columns are summed over ranges of columns: rows between the outputs are kept,
    # what was in the output before is not added
    g = gen(61)
    n, dim, nq = 77, 3333, 11
    codes, scales, zp = make_table(g, n, dim, 64, "bf16", True)
    x = randn(g, nq, dim)
    wide = torch.full((nq, 100), 5.0, device="cuda")
    wide[:, :n] = float("nan")
    run_matvec(tctx, x, None, codes, scales, zp, dim, 64, out=wide[:, :n])
    want, size = matvec_reference(x, None, codes, scales, zp, dim, 64)
    assert ((wide[:, :n].double() - want).abs() <= matvec_tolerance(dim, 64) * size).all()
    assert (wide[:, n:] == 5.0).all()


def test_quantizer_of_groups_wider_than_fp32(tctx):  # noqa: F811
    # finite rows whose largest and smallest elements are further apart than fp32's largest number
    g = gen(13)
    n, dim = 40, 256
    x = randn(g, n, dim).clamp(-3, 3) * 1e38
    x[::2] = x[::2].clamp(-0.5e38, 3e38)
    for scale in ("f32", "bf16"):
        codes = torch.empty((n, va.scoring.int4_row_bytes(dim)), dtype=torch.uint8, device="cuda")
        scales = torch.empty((n, 4), dtype=DT[scale], device="cuda")
        zp = torch.empty((n, 4), dtype=torch.int8, device="cuda")
        va.Int4GroupQuantizationKernel(tctx).encode(x, n, dim, 64, codes, scales, zp, va.DTYPE_F32, va.DTYPE_F32 if scale == "f32" else va.DTYPE_BF16)
        tctx.synchronize()
        z = x.double().view(n, 4, 64)
        lo, hi = z.amin(2).clamp(max=0), z.amax(2).clamp(min=0)
        s = ((hi.float() / 2 - lo.float() / 2).double() / 7.5).float().to(DT[scale])  # hi - lo rounded once, at half its size
        assert torch.isfinite(scales.float()).all() and torch.equal(scales, s)
        zero = torch.round(-8 - (lo.float() / s.float())).clamp(-8, 7)
        assert torch.equal(zp.float(), zero)
        want = torch.round(x.view(n, 4, 64) / s.float()[:, :, None] + zero[:, :, None]).clamp(-8, 7).view(n, dim)
        assert torch.equal(unpack(codes, dim).float(), want)


@pytest.mark.parametrize("kind", ["f32", "int8"])
def test_search_keeps_a_bounded_piece_of_the_scores(ctx, monkeypatch, kind):
    rng = np.random.default_rng(8)
    rows, q = rng.standard_normal((20000, 96)).astype(np.float32), rng.standard_normal((333, 96)).astype(np.float32)
    db = va.Int4Database(ctx, rows, group=32, type="asymmetric")
    scales = None
    if kind == "int8":
        q, scales, _ = va.RMSNormInt8Kernel(ctx).compute(q, np.ones(96, np.float32))
    want = db.search(q, 9, query_scales=scales)
    sizes = []
    get = ctx.get_buffer
    monkeypatch.setattr(ctx, "get_buffer", lambda size, *a: sizes.append(size) or get(size, *a))
    monkeypatch.setattr(va.Int4Database, "SCORE_BYTES", 4 * 20000 * 100)  # 96 queries
    vals, ids = db.search(q, 9, query_scales=scales)
    assert max(sizes) == 4 * 20000 * 96
    # whole passes: the same scores
    assert (ids == want[1]).all() and (vals == want[0]).all()
    monkeypatch.setattr(va.Int4Database, "SCORE_BYTES", 1)
    vals, ids = db.search(q, 9, query_scales=scales)
    assert (ids == want[1]).all() and (vals == want[0]).all()
    none, no_ids = db.search(q[:0], 9, query_scales=None if scales is None else scales[:0])
    assert none.shape == no_ids.shape == (0, 9)
    db.close()


# ------------------------------------------------------------------------------------------ loss
@pytest.mark.parametrize("t, v, d", [(1, 1, 64), (70, 900, 128), (333, 5003, 512), (600, 30001, 256)])
@pytest.mark.parametrize("scale", [1.0, 7.3])
def test_loss_of_confident_tokens(tctx, t, v, d, scale):  # noqa: F811
    # Labels that have nearly all of the probability, at logits of hundreds: the loss is a small difference of large
    # numbers and never below zero.
    g = gen(t + v)
    w = randn(g, v, d).bfloat16()
    labels = torch.randint(0, v, (t,), generator=g, device="cuda")
    h = (w[labels].float() * torch.linspace(0.02, 4.0, t, device="cuda")[:, None]).bfloat16()
    loss, lse, _, _ = run_loss(tctx, h, w, labels, scale, None)
    z = scale * (h.double() @ w.double().t())
    want = torch.logsumexp(z, 1)
    zl = z.gather(1, labels[:, None])[:, 0]
    assert (loss >= 0).all()
    # The logits come from one set of fp32 sums: D / 16 matrix steps of 18 roundings of the sum of magnitudes each, the
    # label's and the others'. Of the rest, exponents near 0 and a logarithm of a number above 1/2: 2^-20 in all (the
    # terms of v rows, 2^-24 each, add up in (v / 256 + 64) steps), and one rounding of the result.
    size = scale * (h.double().abs() @ w.double().abs().t()).amax(1)
    dz = 2 * 18 * d / 16 * U32 * size
    rest = (v / 256 + 64) * U32 + 2.0 ** -20
    exact = want - zl
    assert ((loss.double() - exact).abs() <= dz + rest + 2 * U32 * exact).all()
    # a token with nothing beside its label: the same logit in lse and in the loss, one exponential and one logarithm
    alone = exact < 1e-9
    assert (loss[alone] <= 2.0 ** -21).all()
    assert ((lse.double() - want).abs() <= dz + rest + 2 * U32 * want.abs()).all()


def test_loss_of_whole_numbers_is_exact_to_fp32(tctx):  # noqa: F811
    # small whole numbers: every logit is exact in fp32, so only the statistics can be off
    g = gen(44)
    t, v, d = 300, 4001, 64
    h = torch.randint(-6, 7, (t, d), generator=g, device="cuda").bfloat16()
    w = torch.randint(-6, 7, (v, d), generator=g, device="cuda").bfloat16()
    for scale in (1.0, 0.3, 1.7):
        c = float(torch.tensor(scale))  # as fp32
        z = c * (h.double() @ w.double().t())
        labels = z.topk(3, 1).indices[:, torch.randint(0, 3, (1,), generator=g, device="cuda").item()].contiguous()
        loss, lse, _, _ = run_loss(tctx, h, w, labels, scale, None)
        want = torch.logsumexp(z, 1)
        exact = want - z.gather(1, labels[:, None])[:, 0]
        # An exponent is a difference of logits, off by 3 roundings of its size, which is at most ln v on the average over
        # the softmax: 25 roundings. The sum of v terms in v / 256 steps and its joins: 39. The exponential and the
        # logarithm: 2^-21.
        rest = (v / 256 + 64) * U32 + 2.0 ** -21
        assert ((loss.double() - exact).abs() <= rest + 3 * U32 * exact.abs()).all()
        assert ((lse.double() - want).abs() <= rest + 1.01 * U32 * want.abs()).all()


@pytest.mark.parametrize("t, v, d", [(700, 500, 64), (3000, 900, 72), (2100, 20000, 136)])
@pytest.mark.parametrize("lead", [1, 257, 600])
def test_loss_equal_weights_wherever_ignored_tokens_lie(tctx, t, v, d, lead):  # noqa: F811
    # equal weights that are no powers of two: hidden rows enter the table's gradient as they are, so that ignored
    # tokens in front change nothing but the order of sums
    h, w, labels, _ = make_loss(t + lead, t, v, d, ignored=0.0)
    labels[:lead] = -100
    grad = torch.full((t,), 1.0 / 6553, device="cuda")
    _, _, _, dw = run_loss(tctx, h, w, labels, 1.0, grad)
    ones = run_loss(tctx, h, w, labels, 1.0, None)[3]
    # dw = rho * sum(G h) with the same G and h: the fp32 sums are those of weights of 1
    want = (ones.double() * float(grad[0])).float()
    # `ones` is rounded to bf16, and so is dw, the same sums times rho: two roundings of half a step each apart
    assert ((dw.double() - want.double()).abs() <= 2 * U16 * want.double().abs() * (1 + U16) + 1e-38).all()
    check_loss(run_loss(tctx, h, w, labels, 1.0, grad), loss_reference(h, w, labels, 1.0, grad))


def test_loss_weights_far_apart(tctx):  # noqa: F811
    # |c g| of 2^-59 first and 2^100 later: nothing overflows on the way to a gradient that fp32 holds
    h, w, labels, _ = make_loss(18, 300, 900, 64, ignored=0.0)
    for small, large in ((2.0 ** -59, 2.0 ** 100), (2.0 ** -100, 3.0 ** 60), (2.0 ** -120, 1.0), (1.0, 2.0 ** -120)):
        grad = torch.full((300,), small, device="cuda")
        grad[150:] = large
        check_loss(run_loss(tctx, h, w, labels, 1.0, grad), loss_reference(h, w, labels, 1.0, grad))


# ------------------------------------------------------------------------------------------ bounded waits
@pytest.fixture
def stalled(monkeypatch):
    """Issuers of the tile kernels stop after some tiles and waits expire after 50 ms, while the returned call runs."""
    def run(c, tiles, call):
        with monkeypatch.context() as m:
            m.setenv("VA_TC_TEST_STALL_TILES", str(tiles))
            m.setenv("VA_TC_WAIT_LIMIT_MS", "50")
            start = time.perf_counter()
            call()
            with pytest.raises(va.Timeout, match="bounded device-side wait expired"):
                c.synchronize()
            # far below the second that draining a copy which never was may take
            assert time.perf_counter() - start < 0.9
        c.synchronize()  # the error has been taken
    return run


@pytest.mark.parametrize("n, dim, nq, dtype, copies", [(200000, 512, 1, "f32", 0), (200000, 512, 1, "f32", 4), (200000, 1536, 16, "int8", 1),
                                                       (200000, 1536, 16, "int8", 8), (300, 4096, 4, "bf16", 0), (300, 4096, 4, "bf16", 1),
                                                       (40000, 4096, 5, "f32", 3)])
def test_matvec_wait_expires_and_the_context_recovers(tctx, stalled, n, dim, nq, dtype, copies):  # noqa: F811
    g = gen(n)
    codes, scales, zp = make_table(g, n, dim, 64, "bf16", False)
    x, xs = make_queries(g, nq, dim, dtype)
    k = va.Int4MatVecKernel(tctx)
    out = torch.empty(nq, n, device="cuda")
    dt = {"f32": va.DTYPE_F32, "bf16": va.DTYPE_BF16, "int8": va.DTYPE_INT8}[dtype]
    torch.cuda.synchronize()
    stalled(tctx, copies, lambda: k.encode(x, nq, codes, scales, n, dim, 64, out, zp, dt, xs))
    out = run_matvec(tctx, x, xs, codes, scales, zp, dim, 64)
    want, size = matvec_reference(x, xs, codes, scales, zp, dim, 64)
    assert ((out.double() - want).abs() <= matvec_tolerance(dim, 64) * size).all()


@pytest.mark.parametrize("t, v, d, tiles", [(120, 50000, 136, 0), (300, 5003, 320, 0), (513, 30000, 768, 0), (513, 30000, 768, 1),
                                            (2047, 9999, 1000, 2)])  # single CTAs, narrow tiles, pairs
def test_loss_wait_expires_and_the_context_recovers(tctx, stalled, t, v, d, tiles):  # noqa: F811
    h, w, labels, grad = make_loss(t + v, t, v, d)
    k = va.SoftmaxCrossEntropyKernel(tctx)
    loss, lse, dh, dw = torch.empty(t, device="cuda"), torch.empty(t, device="cuda"), torch.empty_like(h), torch.empty_like(w)
    want = loss_reference(h, w, labels, 1.0, grad)
    torch.cuda.synchronize()
    stalled(tctx, tiles, lambda: k.encode_forward(h, w, labels, t, v, d, loss, lse))
    check_loss(run_loss(tctx, h, w, labels, 1.0, grad), want)
    lse.copy_(want[1])
    torch.cuda.synchronize()
    stalled(tctx, tiles, lambda: k.encode_backward(h, w, labels, lse, grad, t, v, d, dh, dw))
    check_loss(run_loss(tctx, h, w, labels, 1.0, grad), want)


# ------------------------------------------------------------------------------------------ overlaps
def test_outputs_between_the_rows_of_an_input(tctx):  # noqa: F811
    # arrays that interleave without sharing a byte are not refused
    g = gen(70)
    buf = randn(g, 4, 128).bfloat16()
    x, w = buf[:, :64], torch.ones(64, dtype=torch.bfloat16, device="cuda")
    scales = buf[1, 64:72].view(torch.float32)
    codes = buf[2, 64:].view(torch.int8)
    codes4 = torch.empty(4, 64, dtype=torch.int8, device="cuda")
    want_codes, want_scales = norm_reference(x.contiguous(), w, 1e-6, 0)
    k = va.RMSNormInt8Kernel(tctx)
    k.encode(x, w, 4, 64, codes4, scales, x_stride=128)
    tctx.synchronize()
    assert torch.equal(codes4.double(), want_codes)
    assert ((scales.double() - want_scales[:, 0]).abs() <= SCALE_TOL * want_scales[:, 0]).all()
    k.encode(x[:2], w, 2, 64, codes, torch.empty(2, device="cuda"), x_stride=128)
    tctx.synchronize()
    assert torch.equal(codes.view(2, 64).double(), want_codes[:2])


def test_workspace_over_an_argument_is_refused(tctx):  # noqa: F811
    t, v, d = 40, 300, 64
    h, w, labels, grad = make_loss(71, t, v, d)
    k = va.SoftmaxCrossEntropyKernel(tctx)
    need = max(k.workspace_bytes(t, v, d, b) for b in (False, True))
    space = torch.empty(need + 4096, dtype=torch.uint8, device="cuda")
    loss, lse = space[:4 * t].view(torch.float32), torch.zeros(t, device="cuda")
    with pytest.raises(va.InvalidInput, match="workspace must not overlap loss"):
        k.encode_forward(h, w, labels, t, v, d, loss, lse, workspace=space)
    gh = space[1024:1024 + 2 * t * d].view(torch.bfloat16).view(t, d)
    with pytest.raises(va.InvalidInput, match="workspace must not overlap grad_hidden"):
        k.encode_backward(h, w, labels, lse, grad, t, v, d, gh, torch.empty_like(w), workspace=space)
