"""The scoring head without a GPU: refusals of the C entry points (they are decided before anything is
launched) and of the classes, and the bf16 conversion of the host-array methods."""

import ctypes

import numpy as np
import pytest

import vectoraccelerate_b200 as va
from vectoraccelerate_b200 import _ffi, scoring

F32, BF16, INT8 = va.DTYPE_F32, va.DTYPE_BF16, va.DTYPE_INT8
CTX = ctypes.addressof(ctypes.create_string_buffer(1 << 14))  # never read by a refused call
P = 1 << 20  # a 16-byte aligned address, never read


def refused(name, args, word, status=-1):
    assert getattr(_ffi.load(), name)(*args) == status
    assert word in _ffi.last_error(), _ffi.last_error()


def norm_args(**k):
    a = dict(ctx=CTX, x=P, residual=P, weight=P, rows=4, dim=64, dtype=BF16, xs=64, rs=64, eps=1e-6, group=0, out=P, codes=P,
             scales=P)
    a.update(k)
    return [a[n] for n in ("ctx", "x", "residual", "weight", "rows", "dim", "dtype", "xs", "rs", "eps", "group", "out", "codes",
                           "scales")]


@pytest.mark.parametrize("change, word", [
    (dict(ctx=None), "NULL"), (dict(x=None), "NULL"), (dict(weight=None), "NULL"), (dict(codes=None), "NULL"),
    (dict(scales=None), "NULL"), (dict(rows=-1), "rows"), (dict(dim=0), "dimension"), (dict(dim=4097, xs=5000, rs=5000), "dimension"),
    (dict(dtype=INT8), "dtype"), (dict(xs=63), "x_stride"), (dict(rs=63), "residual_stride"),
    (dict(residual=None), "residual_out"), (dict(eps=-1.0), "epsilon"), (dict(eps=float("nan")), "epsilon"),
    (dict(group=48), "group"), (dict(x=P + 1), "aligned"), (dict(scales=P + 2), "aligned"),
    (dict(xs=72), "in place"), (dict(x=2 * P, rs=72), "in place")])
def test_norm_refusals(change, word):
    refused("va_rms_norm_int8", norm_args(**change), word)


def matvec_args(**k):
    a = dict(ctx=CTX, x=P, dtype=F32, xs=None, nq=2, codes=P, scales=P, zeros=None, n=100, dim=64, group=64, sd=BF16, out=P, os=100)
    a.update(k)
    return [a[n] for n in ("ctx", "x", "dtype", "xs", "nq", "codes", "scales", "zeros", "n", "dim", "group", "sd", "out", "os")]


@pytest.mark.parametrize("change, word", [
    (dict(ctx=None), "NULL"), (dict(x=None), "NULL"), (dict(codes=None), "NULL"), (dict(scales=None), "NULL"), (dict(out=None), "NULL"),
    (dict(dtype=3), "dtype"), (dict(xs=P), "INT8"), (dict(nq=-1), "numQueries"), (dict(n=-1), "rows"), (dict(dim=0), "dimension"),
    (dict(dim=4097), "dimension"), (dict(group=16), "group"), (dict(sd=INT8), "scale_dtype"), (dict(os=99), "out_stride"),
    (dict(codes=P + 8), "16 bytes"), (dict(scales=P + 1), "aligned"), (dict(x=P + 2), "aligned"), (dict(out=P + 2), "aligned")])
def test_matvec_refusals(change, word):
    refused("va_int4_matvec", matvec_args(**change), word)


@pytest.mark.parametrize("change, word", [
    (dict(x=None), "NULL"), (dict(dtype=INT8), "dtype"), (dict(n=-1), "rows"), (dict(group=0), "group"), (dict(xs=10), "x_stride"),
    (dict(codes=P + 1), "16 bytes")])
def test_quantizer_refusals(change, word):
    a = dict(ctx=CTX, x=P, dtype=F32, n=10, dim=64, xs=64, group=64, sd=BF16, codes=P, scales=P, zeros=None)
    a.update(change)
    refused("va_sq_quantize_int4_groups", list(a.values()), word)


def forward_args(**k):
    a = dict(ctx=CTX, h=P, hs=64, w=P, ws=64, labels=P, tokens=5, rows=100, dim=64, scale=1.0, space=None, size=0, loss=P, lse=P)
    a.update(k)
    return list(a.values())


LOSS = [
    (dict(h=None), "NULL"), (dict(labels=None), "NULL"), (dict(tokens=-1), "tokens"), (dict(rows=0), "rows"), (dict(dim=100), "multiple of 8"),
    (dict(dim=4104, hs=5000, ws=5000), "multiple of 8"), (dict(hs=60), "hidden_stride"), (dict(hs=68), "hidden_stride"),
    (dict(ws=56), "table_stride"), (dict(h=P + 2), "16 bytes"), (dict(w=P + 8), "16 bytes"), (dict(scale=0.0), "logit_scale"),
    (dict(scale=float("inf")), "logit_scale"), (dict(scale=float("nan")), "logit_scale"),
    (dict(tokens=1 << 24, rows=1 << 28), "too large")]


@pytest.mark.parametrize("change, word", LOSS)
def test_loss_forward_refusals(change, word):
    refused("va_softmax_xent_forward", forward_args(**change), word)


@pytest.mark.parametrize("change, word", LOSS + [(dict(gw=P), "must not be"), (dict(gh=P), "must not be"), (dict(gh=P + 2), "16 bytes"), (dict(gw=None), "NULL"), (dict(lse=None), "NULL")])
def test_loss_backward_refusals(change, word):
    a = dict(ctx=CTX, h=P, hs=64, w=P, ws=64, labels=P, lse=P, g=None, tokens=5, rows=100, dim=64, scale=1.0, space=None, size=0, gh=2 * P,
             gw=3 * P)
    a.update(change)
    refused("va_softmax_xent_backward", list(a.values()), word)


class _Context:
    """Stands for a context in checks that come before any call."""

    handle, device = CTX, 0


def test_class_refusals():
    quant, matvec = va.Int4GroupQuantizationKernel(_Context()), va.Int4MatVecKernel(_Context())
    with pytest.raises(va.InvalidInput, match="group"):
        quant.quantize(np.zeros((2, 8), np.float32), group=100)
    with pytest.raises(va.InvalidInput, match="type"):
        quant.quantize(np.zeros((2, 8), np.float32), type="other")
    with pytest.raises(va.InvalidInput, match="Empty"):
        quant.quantize(np.zeros((0, 8), np.float32))
    with pytest.raises(va.InvalidInput, match="dtype"):
        matvec.encode(P, 1, P, P, 1, 8, 64, P, query_dtype=7)
    with pytest.raises(va.InvalidInput, match="data_ptr"):
        matvec.encode("x", 1, P, P, 1, 8, 64, P)
    with pytest.raises(va.InvalidInput, match="dtype"):
        va.RMSNormInt8Kernel(_Context()).encode(P, P, 1, 8, P, P, dtype=INT8)


def test_tensor_arguments_are_checked():
    torch = pytest.importorskip("torch")
    norm = va.RMSNormInt8Kernel(_Context())
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(va.InvalidInput, match="cuda:0"):  # on another device than the context
        norm.encode(x, P, 4, 64, P, P)
    with pytest.raises(va.InvalidInput, match="elements of 2 bytes"):
        norm.encode(x, P, 4, 64, P, P, dtype=F32)
    with pytest.raises(va.InvalidInput, match="does not hold"):
        norm.encode(x, P, 5, 64, P, P)
    with pytest.raises(va.InvalidInput, match="does not hold"):
        norm.encode(x, P, 4, 64, P, P, x_stride=128)
    with pytest.raises(va.InvalidInput, match="contiguous"):
        norm.encode(P, P, 4, 64, torch.zeros(64, 4, dtype=torch.int8).t(), P)
    with pytest.raises(va.InvalidInput, match="bytes"):
        norm.encode(P, P, 4, 64, torch.zeros(4, 63, dtype=torch.int8), P)


def test_tensors_of_another_type_are_refused():
    torch = pytest.importorskip("torch")
    norm, matvec, loss = (k(_Context()) for k in (va.RMSNormInt8Kernel, va.Int4MatVecKernel, va.SoftmaxCrossEntropyKernel))
    half, table = torch.zeros(4, 64, dtype=torch.float16), torch.zeros(9, 64, dtype=torch.bfloat16)
    with pytest.raises(va.InvalidInput, match="x is torch.float16"):
        norm.encode(half, P, 4, 64, P, P)
    with pytest.raises(va.InvalidInput, match="weight has elements of 4 bytes"):  # fp32 weights of bf16 rows
        norm.encode(P, torch.zeros(64), 4, 64, P, P)
    with pytest.raises(va.InvalidInput, match="scales has elements of 4 bytes"):
        matvec.encode(P, 1, P, torch.zeros(4, 1), 4, 64, 64, P, scale_dtype=BF16)
    with pytest.raises(va.InvalidInput, match="queries is torch.int32"):
        matvec.encode(torch.zeros(1, 64, dtype=torch.int32), 1, P, P, 4, 64, 64, P, query_dtype=F32)
    with pytest.raises(va.InvalidInput, match="hidden is torch.float16"):
        loss.encode_forward(half, table, P, 4, 9, 64, P, P)
    with pytest.raises(va.InvalidInput, match="labels has elements of 4 bytes"):
        loss.encode_forward(P, P, torch.zeros(8, dtype=torch.int32), 4, 9, 64, P, P)
    with pytest.raises(va.InvalidInput, match="grad_table has elements of 4 bytes"):
        loss.encode_backward(P, P, P, P, None, 4, 9, 64, P, torch.zeros(9, 64))
    with pytest.raises(va.InvalidInput, match="workspace"):
        loss.encode_forward(P, P, P, 4, 9, 64, P, P, workspace=torch.zeros(64, dtype=torch.uint8))
    with pytest.raises(va.InvalidInput, match="hidden is on cpu"):  # bf16 bit patterns are taken
        loss.encode_forward(torch.zeros(4, 64, dtype=torch.int16), P, P, 4, 9, 64, P, P)


def test_bf16_conversion_rounds_to_even():
    x = np.array([1.0, 1.00390625, 1.01171875, -2.5, 3.0e38, np.inf, -np.inf, 1e-40], np.float32)
    assert scoring._to_bf16(x).tolist() == [0x3F80, 0x3F80, 0x3F82, 0xC020, 0x7F62, 0x7F80, 0xFF80, 0x0001]
    assert np.isnan(scoring._from_bf16(scoring._to_bf16(np.array([np.nan], np.float32))))[0]
    assert scoring.int4_row_bytes(1) == 16 and scoring.int4_row_bytes(33) == 32 and scoring.int4_row_bytes(768) == 384
