"""More refusals of the scoring head, decided on the host before anything is launched: outputs that overlap other
arrays of the call, addresses that do not suit their elements, buffers that have been freed, sizes past 32 bits,
arrays of another kind of number."""

import numpy as np
import pytest

import vectoraccelerate_b200 as va
from vectoraccelerate_b200 import scoring

from test_scoring_host import BF16, CTX, F32, INT8, _Context, refused

M = 1 << 20  # far apart: eight arrays of the calls below fit between multiples


def args(base, change):
    assert set(change) <= set(base), change
    return list({**base, **change}.values())


# ------------------------------------------------------------------------------------------ overlaps
NORM = dict(ctx=CTX, x=M, residual=2 * M, weight=3 * M, rows=4, dim=64, dtype=BF16, xs=64, rs=64, eps=1e-6, group=0, out=4 * M, codes=5 * M,
            scales=6 * M)


@pytest.mark.parametrize("change, word", [
    (dict(out=M + 16), "residual_out must not overlap x"), (dict(out=2 * M - 16), "residual_out must not overlap residual"),
    (dict(out=M - 510), "residual_out must not overlap x"), (dict(out=3 * M + 126), "residual_out must not overlap weight"),
    (dict(codes=M + 511), "codes must not overlap x"), (dict(codes=4 * M + 8), "residual_out must not overlap codes"),
    (dict(out=M, codes=M + 256), "residual_out must not overlap codes"), (dict(scales=5 * M + 252), "codes must not overlap scales"),
    (dict(scales=3 * M), "scales must not overlap weight"), (dict(scales=2 * M + 508), "scales must not overlap residual"),
    (dict(out=M + 300, xs=128), "residual_out must not overlap x"),  # longer than the gap between x's rows
    (dict(scales=M + 124, xs=128), "scales must not overlap x"), (dict(scales=M + 896 - 4, xs=128, codes=M + 512), "codes must not overlap x"),
    (dict(dtype=F32, out=M + 1020), "residual_out must not overlap x")])
def test_norm_overlaps(change, word):
    refused("va_rms_norm_int8", args(NORM, change), word)


QUANT = dict(ctx=CTX, x=M, dtype=F32, n=10, dim=64, xs=64, group=64, sd=BF16, codes=2 * M, scales=3 * M, zeros=4 * M)


@pytest.mark.parametrize("change, word", [
    (dict(codes=M + 2544), "codes must not overlap x"), (dict(scales=2 * M + 318), "codes must not overlap scales"),
    (dict(zeros=2 * M), "codes must not overlap zeros"), (dict(zeros=3 * M + 19), "scales must not overlap zeros"),
    (dict(scales=M), "scales must not overlap x"), (dict(zeros=M + 255), "zeros must not overlap x")])
def test_quantizer_overlaps(change, word):
    refused("va_sq_quantize_int4_groups", args(QUANT, change), word)


@pytest.mark.parametrize("change, word", [
    (dict(out=M + 300), "out must not overlap codes"), (dict(out=2 * M - 2556), "out must not overlap scales"),
    (dict(out=3 * M), "out must not overlap zeros")])
def test_dequantizer_overlaps(change, word):
    base = dict(ctx=CTX, codes=M, scales=2 * M, zeros=3 * M, n=10, dim=64, group=64, sd=BF16, out=4 * M)
    refused("va_sq_dequantize_int4_groups", args(base, change), word)


@pytest.mark.parametrize("change, word", [
    (dict(out=M + 508), "out must not overlap the queries"), (dict(out=2 * M + 4), "out must not overlap the query scales"),
    (dict(out=3 * M - 400), "out must not overlap codes"), (dict(out=4 * M + 196), "out must not overlap scales"),
    (dict(out=5 * M), "out must not overlap zeros"), (dict(out=2 * M - 4000, os=1000), "out must not overlap the query scales")])
def test_matvec_overlaps(change, word):
    base = dict(ctx=CTX, x=M, dtype=INT8, xs=2 * M, nq=8, codes=3 * M, scales=4 * M, zeros=5 * M, n=100, dim=64, group=64, sd=BF16, out=6 * M,
                os=100)
    refused("va_int4_matvec", args(base, change), word)


@pytest.mark.parametrize("change, word", [
    (dict(loss=M + 636), "loss must not overlap hidden"), (dict(lse=2 * M), "lse must not overlap table"),
    (dict(loss=3 * M), "loss must not overlap labels"), (dict(loss=4 * M + 16, lse=4 * M), "loss must not overlap lse"),
    (dict(lse=M + 256 - 4, hs=128), "lse must not overlap hidden")])  # the gap is 128 bytes long and starts 128 bytes on
def test_loss_forward_overlaps(change, word):
    base = dict(ctx=CTX, h=M, hs=64, w=2 * M, ws=64, labels=3 * M, tokens=5, rows=100, dim=64, scale=1.0, space=None, size=0, loss=4 * M,
                lse=5 * M)
    refused("va_softmax_xent_forward", args(base, change), word)


@pytest.mark.parametrize("change, word", [
    (dict(gh=M + 16), "grad_hidden must not overlap hidden"), (dict(gh=2 * M + 12784), "grad_hidden must not overlap table"),
    (dict(gw=2 * M - 16), "grad_table must not overlap table"), (dict(gw=3 * M), "grad_table must not overlap labels"),
    (dict(gh=4 * M), "grad_hidden must not overlap lse"), (dict(gw=5 * M), "grad_table must not overlap grad_loss"),
    (dict(gh=7 * M + 12784), "grad_hidden must not overlap grad_table")])
def test_loss_backward_overlaps(change, word):
    base = dict(ctx=CTX, h=M, hs=64, w=2 * M, ws=64, labels=3 * M, lse=4 * M, g=5 * M, tokens=5, rows=100, dim=64, scale=1.0, space=None, size=0,
                gh=6 * M, gw=7 * M)
    refused("va_softmax_xent_backward", args(base, change), word)


# ------------------------------------------------------------------------------------------ alignment
FORWARD = dict(ctx=CTX, h=M, hs=64, w=2 * M, ws=64, labels=3 * M, tokens=5, rows=100, dim=64, scale=1.0, space=None, size=0, loss=4 * M, lse=5 * M)
BACKWARD = dict(ctx=CTX, h=M, hs=64, w=2 * M, ws=64, labels=3 * M, lse=4 * M, g=5 * M, tokens=5, rows=100, dim=64, scale=1.0, space=None, size=0,
                gh=6 * M, gw=7 * M)


@pytest.mark.parametrize("change", [dict(labels=3 * M + 4), dict(loss=4 * M + 2), dict(lse=5 * M + 1)])
def test_loss_forward_alignment(change):
    refused("va_softmax_xent_forward", args(FORWARD, change), "aligned")


@pytest.mark.parametrize("change", [dict(labels=3 * M + 4), dict(lse=4 * M + 2), dict(g=5 * M + 2)])
def test_loss_backward_alignment(change):
    refused("va_softmax_xent_backward", args(BACKWARD, change), "aligned")


def test_loss_scale_beyond_powers_of_two():
    refused("va_softmax_xent_forward", args(FORWARD, dict(scale=3e38)), "logit_scale")
    refused("va_softmax_xent_backward", args(BACKWARD, dict(scale=3e38)), "logit_scale")


def test_dequantizer_alignment():
    base = dict(ctx=CTX, codes=M, scales=2 * M, zeros=3 * M, n=10, dim=64, group=64, sd=BF16, out=4 * M + 2)
    refused("va_sq_dequantize_int4_groups", list(base.values()), "aligned")


# ------------------------------------------------------------------------------------------ the classes
def freed():
    """A DeviceBuffer as free() leaves it, without a device."""
    b = va.DeviceBuffer.__new__(va.DeviceBuffer)
    b.context, b.nbytes, b.dtype, b.shape, b.ptr = _Context(), 1 << 30, np.dtype(np.uint8), (1 << 30,), None
    return b


def test_freed_buffers_are_refused():
    # (an optional argument that has been freed would pass for one that is not there)
    gone = freed()
    norm, matvec, xent = (k(_Context()) for k in (va.RMSNormInt8Kernel, va.Int4MatVecKernel, va.SoftmaxCrossEntropyKernel))
    quant = va.Int4GroupQuantizationKernel(_Context())
    calls = [("x", lambda: norm.encode(gone, P(3), 4, 64, P(5), P(6))),
             ("residual", lambda: norm.encode(P(1), P(3), 4, 64, P(5), P(6), residual=gone)),
             ("residual_out", lambda: norm.encode(P(1), P(3), 4, 64, P(5), P(6), residual=P(2), residual_out=gone)),
             ("zero_points", lambda: quant.encode(P(1), 10, 64, 64, P(2), P(3), gone)),
             ("zero_points", lambda: matvec.encode(P(1), 8, P(3), P(4), 100, 64, 64, P(6), zero_points=gone)),
             ("query_scales", lambda: matvec.encode(P(1), 8, P(3), P(4), 100, 64, 64, P(6), query_dtype=INT8, query_scales=gone)),
             ("workspace", lambda: xent.encode_forward(P(1), P(2), P(3), 5, 100, 64, P(4), P(5), workspace=gone)),
             ("grad_loss", lambda: xent.encode_backward(P(1), P(2), P(3), P(4), gone, 5, 100, 64, P(6), P(7)))]
    for name, call in calls:
        with pytest.raises(va.InvalidInput, match=f"{name} has been freed"):
            call()


def P(i):
    return i * M


def test_sizes_past_32_bits_are_refused():
    norm, matvec, xent = (k(_Context()) for k in (va.RMSNormInt8Kernel, va.Int4MatVecKernel, va.SoftmaxCrossEntropyKernel))
    quant = va.Int4GroupQuantizationKernel(_Context())
    big = (1 << 32) + 64  # 64 when cut to 32 bits
    calls = [("dimension", lambda: norm.encode(P(1), P(3), 4, big, P(5), P(6))),
             ("group", lambda: norm.encode(P(1), P(3), 4, 64, P(5), P(6), group=big)),
             ("dimension", lambda: quant.encode(P(1), 10, big, 64, P(2), P(3))),
             ("dimension", lambda: matvec.encode(P(1), 8, P(3), P(4), 100, big, 64, P(6))),
             ("num_queries", lambda: matvec.encode(P(1), big, P(3), P(4), 100, 64, 64, P(6))),
             ("num_queries", lambda: matvec.encode(P(1), -1, P(3), P(4), 100, 64, 64, P(6))),
             ("dimension", lambda: xent.workspace_bytes(5, 100, big, True)),
             ("dimension", lambda: xent.encode_forward(P(1), P(2), P(3), 5, 100, big, P(4), P(5))),
             ("dimension", lambda: xent.encode_backward(P(1), P(2), P(3), P(4), None, 5, 100, big, P(6), P(7)))]
    for name, call in calls:
        with pytest.raises(va.InvalidInput, match=f"{name} must be in"):
            call()


def test_arrays_of_another_kind_of_number_are_refused():
    # (they were cut to the type that the call takes)
    db = va.Int4Database.__new__(va.Int4Database)
    db.context, db.n, db.dim, db.table = _Context(), 10, 8, None
    for q in (np.full((2, 8), 0.7, np.float32), np.full((2, 8), 200), np.full((2, 8), 255, np.uint8), np.full((2, 8), -129)):
        with pytest.raises(va.InvalidInput, match="queries with query_scales"):
            db.search(q, 3, query_scales=np.ones(2, np.float32))
    xent = va.SoftmaxCrossEntropyKernel(_Context())
    for y in (np.array([1.5, 2.0]), np.array([1 << 63, 0], np.uint64), np.array(["1", "2"])):
        with pytest.raises(va.InvalidInput, match="labels"):
            xent.compute(np.zeros((2, 8), np.float32), np.zeros((3, 8), np.float32), y)
    assert scoring._whole([1, -128, 127], np.int8, "q").tolist() == [1, -128, 127]
    assert scoring._whole([], np.int64, "labels").shape == (0,)


def test_an_empty_workspace_is_not_the_contexts(monkeypatch):
    torch = pytest.importorskip("torch")
    xent = va.SoftmaxCrossEntropyKernel(_Context())
    monkeypatch.setattr(scoring, "_device_of", lambda *a: None)  # (a CPU tensor stands for one of the GPU)
    monkeypatch.setattr(xent, "workspace_bytes", lambda *a: 1000)
    for nothing in (torch.empty(0, dtype=torch.uint8), 0):
        with pytest.raises(va.InvalidInput, match="workspace of 0 bytes"):
            xent.encode_forward(P(1), P(2), P(3), 5, 100, 64, P(4), P(5), workspace=nothing)
        with pytest.raises(va.InvalidInput, match="workspace of 0 bytes"):
            xent.encode_backward(P(1), P(2), P(3), P(4), None, 5, 100, 64, P(6), P(7), workspace=nothing)
