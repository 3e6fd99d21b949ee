"""The scoring head on the GPU against plain 64-bit implementations: int8 RMS norm, 4-bit rows and their
products with queries, softmax cross entropy with its gradients, and a run of them together.

Tolerances count roundings: fp32 2^-24 and bf16 2^-8 of the value each (half a unit in the last place).
"""

import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import vectoraccelerate_b200 as va

pytestmark = pytest.mark.gpu

U32, U16 = 2.0 ** -24, 2.0 ** -8
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
VA = {"f32": va.DTYPE_F32, "bf16": va.DTYPE_BF16, "int8": va.DTYPE_INT8}


@pytest.fixture(scope="module")
def tctx():
    """A context on torch's default stream."""
    torch.zeros(1, device="cuda")
    c = va.GPUContext(va.Metal4Configuration(device=0, stream=1))
    yield c
    c.close()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


# ------------------------------------------------------------------------------------------ norm
def norm_reference(h, weight, eps, group):
    """codes, scales, both in 64 bits, of rows h [rows, dim]."""
    h64 = h.double()
    z = h64 * weight.double()
    rows, dim = z.shape
    size = group or dim
    z = torch.nn.functional.pad(z, (0, -dim % size)).view(rows, -1, size)
    top = z.abs().amax(2)
    codes = torch.round(z * 127.0 / torch.where(top > 0, top, 1.0)[:, :, None])
    scales = top / (127.0 * torch.sqrt((h64 * h64).mean(1) + eps))[:, None]
    return codes.view(rows, -1)[:, :dim], scales


# The scale: the longest chain of the sum of squares is 16 fmas, 5 shuffles, 8 warps and the fp32 product
# (30 roundings, halved by the root), then the mean, the root (2 units), two divisions and a product.
SCALE_TOL = (30 / 2 + 8) * U32


def run_norm(c, x, weight, residual, dtype, group, eps=1e-6, inplace=False):
    rows, dim = x.shape
    groups = -(-dim // group) if group else 1
    codes = torch.full((rows, dim), 99, dtype=torch.int8, device="cuda")
    scales = torch.full((rows, groups), -1.0, device="cuda")
    out = None
    if residual is not None:
        out = residual if inplace else torch.empty((rows, dim), dtype=x.dtype, device="cuda")
    va.RMSNormInt8Kernel(c).encode(x, weight, rows, dim, codes, scales, residual, out, VA[dtype], eps, group,
                                   x.stride(0) if rows > 1 else dim,
                                   residual.stride(0) if residual is not None and rows > 1 else None)
    c.synchronize()
    return codes, scales, out


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows, dim, group, residual, pad", [
    (1, 1, 0, False, 0), (1, 7, 32, True, 0), (3, 33, 32, True, 0), (5, 64, 64, False, 0), (4, 512, 0, True, 0), (9, 511, 128, True, 1),
    (130, 520, 0, True, 0), (17, 1000, 64, False, 24), (2, 1536, 0, True, 0), (33, 2048, 128, True, 8), (6, 2049, 0, True, 0),
    (12, 4096, 0, True, 0), (3, 4096, 32, False, 0), (5, 4095, 128, True, 13)])
def test_norm_matches_64_bits(tctx, dtype, rows, dim, group, residual, pad):
    g = gen(rows * 10007 + dim)
    x = (randn(g, rows, dim + pad) * 2).to(DT[dtype])[:, :dim]
    w = (1 + 0.3 * randn(g, dim)).to(DT[dtype])
    r = (randn(g, rows, dim) * 3).to(DT[dtype]) if residual else None
    h = (x.float() + r.float()).to(DT[dtype]) if residual else x
    codes, scales, out = run_norm(tctx, x, w, r, dtype, group)
    want_codes, want_scales = norm_reference(h, w, 1e-6, group)
    assert torch.equal(codes.double(), want_codes)
    assert ((scales.double() - want_scales).abs() <= SCALE_TOL * want_scales).all()
    if residual:
        assert torch.equal(out, h)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_norm_in_place_and_untouched_neighbours(tctx, dtype):
    g = gen(3)
    x, w = randn(g, 37, 768).to(DT[dtype]), torch.ones(768, dtype=DT[dtype], device="cuda")
    buf = randn(g, 40, 768).to(DT[dtype])
    before = buf.clone()
    h = (x.float() + before[:37].float()).to(DT[dtype])
    codes, scales, out = run_norm(tctx, x, w, buf[:37], dtype, 0, inplace=True)
    assert torch.equal(out, h) and torch.equal(buf[37:], before[37:])
    assert torch.equal(codes.double(), norm_reference(h, w, 1e-6, 0)[0])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows, dim, pad, group, offsets, inplace", [
    (1, 1, 0, 0, (1, 2, 3, 5), None), (40, 3, 0, 0, (3, 0, 1, 2), None), (20000, 9, 2, 0, (0, 1, 0, 7), None),
    (9001, 17, 0, 32, (5, 5, 5, 5), "x"), (7000, 255, 0, 64, (7, 3, 2, 1), None), (6001, 256, 1, 0, (1, 0, 0, 3), None),
    (5000, 257, 0, 128, (0, 0, 0, 0), "residual"), (4000, 511, 3, 0, (2, 4, 6, 4), None), (3001, 513, 0, 32, (0, 6, 0, 0), "x"),
    (2000, 1023, 0, 0, (4, 4, 4, 0), "residual"), (1500, 1024, 0, 64, (1, 1, 1, 1), None), (1201, 2047, 0, 0, (6, 1, 7, 6), None),
    (1000, 2050, 0, 128, (0, 0, 0, 0), "x"), (900, 4095, 0, 0, (0, 0, 0, 0), None), (901, 4089, 2, 32, (7, 2, 5, 3), None),
    (700, 4096, 0, 0, (0, 1, 0, 1), None)])
def test_norm_rows_at_any_address(tctx, dtype, rows, dim, pad, group, offsets, inplace):
    # every array at its own offset from a 16-byte boundary, many rows per block, neighbours kept
    g = gen(dim)

    def at(offset, stride, t, fill):
        flat = torch.full((offset + rows * stride + 64,), fill, dtype=t, device="cuda")
        return flat, flat[offset:offset + rows * stride].view(rows, stride)[:, :dim]

    xs, rs, outs = dim + (0 if inplace == "x" else pad), dim, dim
    fx, x = at(offsets[0], xs, DT[dtype], float("nan"))
    fr, r = at(offsets[1], rs, DT[dtype], float("nan"))
    x.copy_((randn(g, rows, dim) * 2).to(DT[dtype]))
    r.copy_((randn(g, rows, dim) * 3).to(DT[dtype]))
    w = (1 + 0.3 * randn(g, dim + 1)).to(DT[dtype])[1:]
    h = (x.float() + r.float()).to(DT[dtype])
    flat, out = {"x": (fx, x), "residual": (fr, r), None: at(offsets[2], outs, DT[dtype], 55.0)}[inplace]
    first = offsets[{"x": 0, "residual": 1, None: 2}[inplace]]
    fc, codes = at(offsets[3], dim, torch.int8, 99)
    scales = torch.full((rows, -(-dim // group) if group else 1), -1.0, device="cuda")
    edges = [t.clone() for t in (flat[:first], flat[first + rows * dim:])]
    va.RMSNormInt8Kernel(tctx).encode(x, w, rows, dim, codes, scales, r, out, VA[dtype], 1e-6, group, xs, rs)
    tctx.synchronize()
    want_codes, want_scales = norm_reference(h, w, 1e-6, group)
    assert torch.equal(out, h)
    assert torch.equal(codes.double(), want_codes)
    assert ((scales.double() - want_scales).abs() <= SCALE_TOL * want_scales).all()
    assert all(torch.equal(torch.nan_to_num(a, 77.0), torch.nan_to_num(b, 77.0))
               for a, b in zip(edges, (flat[:first], flat[first + rows * dim:])))
    assert (fc[:offsets[3]] == 99).all() and (fc[offsets[3] + rows * dim:] == 99).all()
    if not inplace:
        bare = torch.empty_like(codes)
        va.RMSNormInt8Kernel(tctx).encode(h, w, rows, dim, bare, scales, dtype=VA[dtype], group=group)
        tctx.synchronize()
        assert torch.equal(bare, codes)


def test_norm_zero_and_non_finite_rows(tctx):
    x = torch.ones(6, 256, device="cuda")
    x[1] = 0
    x[2, 5] = float("nan")
    x[3, 200] = float("inf")
    x[4, :] = 1e30  # the sum of squares overflows
    x[5, 64:128] = 0
    w = torch.ones(256, device="cuda")
    for group in (0, 64):
        codes, scales, _ = run_norm(tctx, x, w, None, "f32", group)
        for r in (2, 3, 4):
            assert (codes[r] == 0).all() and torch.isnan(scales[r]).all()
        assert (codes[1] == 0).all() and (scales[1] == 0).all()
        assert (codes[0] == 127).all()
    assert (codes[5, 64:128] == 0).all() and scales[5, 1] == 0 and (codes[5, :64] == 127).all()
    w[3] = float("inf")  # one group of the weight
    codes, scales, _ = run_norm(tctx, x[:1], w, None, "f32", 64)
    assert torch.isnan(scales[0, 0]) and (codes[0, :64] == 0).all() and (codes[0, 64:] == 127).all()


def test_norm_codes_at_borders(tctx):
    # 127 z / a is a half for every odd entry: the exact quotient decides (to even)
    z = torch.arange(-127, 128, device="cuda", dtype=torch.float32) / 2
    x = torch.cat([torch.full((1,), 127.0, device="cuda"), z])[None, :].repeat(3, 1)
    x[1] *= 3.0
    x[2] = torch.nextafter(x[2], torch.tensor(0.0, device="cuda"))
    w = torch.ones(256, device="cuda")
    for row in range(3):
        codes, _, _ = run_norm(tctx, x[row:row + 1].contiguous(), w, None, "f32", 0)
        assert torch.equal(codes.double(), norm_reference(x[row:row + 1], w, 1e-6, 0)[0])
    tiny = torch.full((2, 64), 2.0 ** -81, device="cuda")  # below 2^-80: counts as zero
    tiny[1, 3] = 2.0 ** -80
    codes, scales, _ = run_norm(tctx, tiny, torch.ones(64, device="cuda"), None, "f32", 0)
    assert (codes[0] == 0).all() and scales[0, 0] == 0
    assert torch.equal(codes[1].double(), norm_reference(tiny[1:], torch.ones(64, device="cuda"), 1e-6, 0)[0][0]) and scales[1, 0] > 0


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_norm_many_borders(tctx, dtype):
    # few distinct values, so that quotients fall on and next to the borders between codes all the time
    g = gen(8)
    x = (torch.randint(-255, 256, (2000, 1024), generator=g, device="cuda") / 8).to(DT[dtype])
    w = (torch.randint(1, 5, (1024,), generator=g, device="cuda") * (1.0 if dtype == "bf16" else 1.0 / 3)).to(DT[dtype])
    for group in (0, 32):
        codes, _, _ = run_norm(tctx, x, w, None, dtype, group)
        assert torch.equal(codes.double(), norm_reference(x, w, 1e-6, group)[0])


def test_norm_no_rows(tctx):
    e = torch.empty(0, 64, device="cuda")
    va.RMSNormInt8Kernel(tctx).encode(e, torch.ones(64, device="cuda"), 0, 64, torch.empty(0, 64, dtype=torch.int8, device="cuda"),
                                      torch.empty(0, 1, device="cuda"), dtype=va.DTYPE_F32)
    tctx.synchronize()


# ------------------------------------------------------------------------------------------ 4-bit rows
def unpack(codes, dim):
    c = torch.stack((codes & 15, codes >> 4), 2).flatten(1)[:, :dim].to(torch.int32)
    return torch.where(c > 7, c - 16, c)


def quantize_reference(x, group, zeros, scale_dtype):
    """The documented formula with fp32 quotients (by 15 and 7 in 64 bits, rounded once: torch divides an fp32
    tensor by a Python number through its reciprocal)."""
    n, dim = x.shape
    z = torch.nn.functional.pad(x, (0, -dim % group)).view(n, -1, group)
    lo, hi = z.amin(2).clamp(max=0), z.amax(2).clamp(min=0)
    s = ((hi - lo).double() / 15 if zeros else torch.maximum(-lo, hi).double() / 7).float().clamp(min=1e-8)
    s = s.to(scale_dtype).float()
    zero = torch.round(-8 - lo / s).clamp(-8, 7) if zeros else torch.zeros_like(s)
    codes = torch.round(z / s[:, :, None] + zero[:, :, None]).clamp(-8, 7)
    return codes.view(n, -1)[:, :dim].to(torch.int32), s, zero.to(torch.int32)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("n, dim, dtype, scale, pad", [(1, 1, "f32", "bf16", 0), (7, 40, "bf16", "f32", 3), (50, 129, "f32", "f32", 0),
                                                      (33, 768, "f32", "bf16", 0), (5, 4096, "bf16", "bf16", 8)])
def test_quantizer(tctx, group, zeros, n, dim, dtype, scale, pad):
    g = gen(n + dim + group)
    x = (randn(g, n, dim + pad) * torch.exp(randn(g, dim + pad))).to(DT[dtype])[:, :dim]
    if n > 4:
        x[2] = 0
        x[3] = x[3].abs()
    groups, stride = -(-dim // group), va.scoring.int4_row_bytes(dim)
    codes = torch.full((n, stride), 0xAA, dtype=torch.uint8, device="cuda")
    scales = torch.empty((n, groups), dtype=DT[scale], device="cuda")
    zp = torch.full((n, groups), 77, dtype=torch.int8, device="cuda") if zeros else None
    k = va.Int4GroupQuantizationKernel(tctx)
    k.encode(x, n, dim, group, codes, scales, zp, VA[dtype], VA[scale], x_stride=dim + pad)
    tctx.synchronize()
    want, s, zero = quantize_reference(x.float(), group, zeros, DT[scale])
    assert torch.equal(scales.float(), s)
    assert torch.equal(unpack(codes, dim), want)
    if zeros:
        assert torch.equal(zp.to(torch.int32), zero)
    full = torch.stack((codes & 15, codes >> 4), 2).flatten(1)
    assert (full[:, dim:] == 0).all()
    out = torch.empty((n, dim), device="cuda")
    va._ffi.call("va_sq_dequantize_int4_groups", tctx.handle, codes.data_ptr(), scales.data_ptr(), zp.data_ptr() if zeros else None, n,
                 dim, group, VA[scale], out.data_ptr())
    tctx.synchronize()
    at = torch.arange(dim, device="cuda") // group
    assert torch.equal(out, (want - zero[:, at]).float() * s[:, at])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("zeros", [False, True])
def test_quantizer_at_borders(tctx, dtype, zeros):
    # few distinct values: quotients fall on and next to the borders between codes all the time
    g = gen(77)
    n, dim = 3000, 517
    x = (torch.randint(-30, 31, (n, dim), generator=g, device="cuda") / 4).to(DT[dtype])
    x[::3] *= 1 / 3
    if dtype == "f32":
        x[1::3] = torch.nextafter(x[1::3], torch.zeros((), device="cuda"))
    for scale in ("f32", "bf16"):
        codes = torch.empty((n, va.scoring.int4_row_bytes(dim)), dtype=torch.uint8, device="cuda")
        scales = torch.empty((n, 17), dtype=DT[scale], device="cuda")
        zp = torch.empty((n, 17), dtype=torch.int8, device="cuda") if zeros else None
        va.Int4GroupQuantizationKernel(tctx).encode(x, n, dim, 32, codes, scales, zp, VA[dtype], VA[scale])
        tctx.synchronize()
        want, s, zero = quantize_reference(x.float(), 32, zeros, DT[scale])
        assert torch.equal(scales.float(), s) and torch.equal(unpack(codes, dim), want)
        if zeros:
            assert torch.equal(zp.to(torch.int32), zero)


def make_table(g, n, dim, group, scale, zeros):
    stride, groups = va.scoring.int4_row_bytes(dim), -(-dim // group)
    codes = torch.randint(0, 256, (n, stride), generator=g, device="cuda", dtype=torch.uint8)  # padding holds anything
    scales = (0.01 * torch.exp(randn(g, n, groups))).to(DT[scale])
    zp = torch.randint(-8, 8, (n, groups), generator=g, device="cuda", dtype=torch.int8) if zeros else None
    return codes, scales, zp


def make_queries(g, nq, dim, dtype):
    if dtype == "int8":
        return torch.randint(-128, 128, (nq, dim), generator=g, device="cuda", dtype=torch.int8), torch.rand(nq, generator=g, device="cuda")
    return (randn(g, nq, dim) * torch.exp(2 * randn(g, nq, 1))).to(DT[dtype]), None


def matvec_reference(x, xs, codes, scales, zp, dim, group):
    """Products in 64 bits and the sums of their magnitudes."""
    at = torch.arange(dim, device="cuda") // group
    w = unpack(codes, dim).double()
    if zp is not None:
        w = w - zp.double()[:, at]
    w = w * scales.double()[:, at]
    q = x.double() * (xs.double()[:, None] if xs is not None else 1.0)
    return q @ w.t(), q.abs() @ w.abs().t()


def matvec_tolerance(dim, group):
    """Of the sum of magnitudes: each of the dim / 16 matrix steps of a piece aligns 17 addends to 24 bits and
    rounds once; then one fma per group, the pieces, partial sums of up to 8 warps and the query's scale."""
    return (18 * dim / 16 + 18 + dim / group + 1 + 8 + 4) * U32


def run_matvec(c, x, xs, codes, scales, zp, dim, group, out=None):
    n, nq = codes.shape[0], x.shape[0]
    out = torch.full((nq, n), float("nan"), device="cuda") if out is None else out
    dt = {torch.int8: va.DTYPE_INT8, torch.bfloat16: va.DTYPE_BF16, torch.float32: va.DTYPE_F32}[x.dtype]
    va.Int4MatVecKernel(c).encode(x, nq, codes, scales, n, dim, group, out, zp, dt, xs,
                                  va.DTYPE_BF16 if scales.dtype is torch.bfloat16 else va.DTYPE_F32,
                                  out.stride(0) if nq > 1 else None)
    c.synchronize()
    return out


@pytest.mark.parametrize("dtype", ["bf16", "f32", "int8"])
@pytest.mark.parametrize("n, dim, group, nq, scale, zeros", [
    (1, 1, 32, 1, "bf16", False), (31, 31, 32, 2, "f32", True), (33, 64, 64, 3, "bf16", True), (100, 100, 32, 8, "f32", False),
    (257, 129, 128, 9, "bf16", False), (1000, 768, 64, 1, "bf16", True), (999, 770, 64, 16, "f32", True), (64, 4096, 128, 5, "bf16", False),
    (500, 4095, 32, 16, "f32", True), (40, 2304, 64, 33, "bf16", True), (7001, 256, 32, 1, "bf16", False), (6000, 1536, 128, 4, "bf16", True)])
def test_matvec_matches_64_bits(tctx, dtype, n, dim, group, nq, scale, zeros):
    g = gen(n * 31 + dim + nq)
    codes, scales, zp = make_table(g, n, dim, group, scale, zeros)
    x, xs = make_queries(g, nq, dim, dtype)
    out = run_matvec(tctx, x, xs, codes, scales, zp, dim, group)
    want, size = matvec_reference(x, xs, codes, scales, zp, dim, group)
    assert ((out.double() - want).abs() <= matvec_tolerance(dim, group) * size).all()
    assert torch.equal(out, run_matvec(tctx, x, xs, codes, scales, zp, dim, group))  # a fixed order of sums


def test_matvec_large_table_of_many_tiles(tctx):
    g = gen(5)
    codes, scales, zp = make_table(g, 200003, 512, 64, "bf16", False)
    x, _ = make_queries(g, 3, 512, "f32")
    out = run_matvec(tctx, x, None, codes, scales, zp, 512, 64)
    want, size = matvec_reference(x, None, codes, scales, zp, 512, 64)
    assert ((out.double() - want).abs() <= matvec_tolerance(512, 64) * size).all()


def test_matvec_and_norm_past_32_bit_offsets(tctx):
    n, dim = 1100000, 4090  # 2.25e9 bytes of codes
    g = gen(9)
    codes = torch.randint(0, 256, (n, va.scoring.int4_row_bytes(dim)), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.rand(n, 32, generator=g, device="cuda")
    x = randn(g, 2, dim)
    out = run_matvec(tctx, x, None, codes, scales, None, dim, 128)
    for rows in (slice(0, 500), slice(n - 500, n)):
        want, size = matvec_reference(x, None, codes[rows], scales[rows], None, dim, 128)
        assert ((out[:, rows].double() - want).abs() <= matvec_tolerance(dim, 128) * size).all()
    del codes
    rows = 530000  # 2.17e9 elements
    x = torch.empty(rows, 4096, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    w = torch.ones(4096, dtype=torch.bfloat16, device="cuda")
    codes, scales, _ = run_norm(tctx, x, w, None, "bf16", 128)
    for part in (slice(0, 200), slice(rows - 200, rows)):
        want, ws = norm_reference(x[part], w, 1e-6, 128)
        assert torch.equal(codes[part].double(), want) and ((scales[part].double() - ws).abs() <= SCALE_TOL * ws).all()
    del x, codes
    torch.cuda.empty_cache()


def test_unaligned_norm_and_quantizer_past_32_bit_offsets(tctx):
    g = gen(10)
    rows, dim = 530000, 4093  # 2.17e9 elements
    x = torch.empty(rows, dim, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    w = torch.ones(dim, dtype=torch.bfloat16, device="cuda")
    parts = (slice(0, 200), slice(rows - 200, rows))
    r = x[:1].expand(rows, dim).contiguous()
    h = [(x[p].float() + r[p].float()).bfloat16() for p in parts]
    codes, scales, out = run_norm(tctx, x, w, r, "bf16", 0, inplace=True)
    for p, hp in zip(parts, h):
        want, ws = norm_reference(hp, w, 1e-6, 0)
        assert torch.equal(out[p], hp) and torch.equal(codes[p].double(), want)
        assert ((scales[p].double() - ws).abs() <= SCALE_TOL * ws).all()
    del r, out, codes
    q = va.Int4GroupQuantizationKernel(tctx)
    packed = torch.empty(rows, va.scoring.int4_row_bytes(dim), dtype=torch.uint8, device="cuda")
    s = torch.empty(rows, 32, device="cuda")
    q.encode(x, rows, dim, 128, packed, s, None, va.DTYPE_BF16, va.DTYPE_F32)
    tctx.synchronize()
    for p in parts:
        want, ws, _ = quantize_reference(x[p].float(), 128, False, torch.float32)
        assert torch.equal(unpack(packed[p], dim), want) and torch.equal(s[p], ws)
    del x, packed
    torch.cuda.empty_cache()


def test_matvec_strided_output_and_extreme_queries(tctx):
    g = gen(6)
    codes, scales, _ = make_table(g, 70, 96, 32, "f32", False)
    x = randn(g, 3, 96)
    x[0] *= 1e-36  # products near the bottom of fp32's range
    x[1] *= 1e36
    wide = torch.full((3, 128), 5.0, device="cuda")
    run_matvec(tctx, x, None, codes, scales, None, 96, 32, out=wide[:, :70])
    want, size = matvec_reference(x, None, codes, scales, None, 96, 32)
    assert ((wide[:, :70].double() - want).abs() <= matvec_tolerance(96, 32) * size + 1e-38).all()
    assert (wide[:, 70:] == 5.0).all()
    x[2, 7] = float("nan")
    x[0, 50] = float("inf")
    out = run_matvec(tctx, x, None, codes, scales, None, 96, 32)
    assert torch.isnan(out[2]).all() and not torch.isfinite(out[0]).any() and torch.isfinite(out[1]).all()


@pytest.mark.parametrize("nq", [1, 3])
def test_matvec_query_with_outliers(tctx, nq):
    # a few elements far above the rest: one or two queries are fixed-point numbers below their group's largest
    g = gen(10)
    codes, scales, zp = make_table(g, 400, 512, 64, "f32", True)
    x = randn(g, nq, 512)
    x[:, ::100] *= 3e4
    out = run_matvec(tctx, x, None, codes, scales, zp, 512, 64)
    want, size = matvec_reference(x, None, codes, scales, zp, 512, 64)
    at = torch.arange(512, device="cuda") // 64
    top = x.abs().double().view(nq, 8, 64).amax(2)[:, at]
    w = ((unpack(codes, 512) - zp.to(torch.int32)[:, at]).double() * scales.double()[:, at]).abs()
    assert ((out.double() - want).abs() <= matvec_tolerance(512, 64) * size + 2.0 ** -30 * (top @ w.t())).all()


def test_first_call_inside_a_capture():
    """In a process of its own: nothing has been loaded or set up before the capture."""
    code = """
import torch, vectoraccelerate_b200 as va
s = torch.cuda.Stream()
c = va.GPUContext(va.Metal4Configuration(device=0, stream=s.cuda_stream))
t, v, d = 40, 500, 64
h, w = torch.randn(t, d, device="cuda").bfloat16(), torch.randn(v, d, device="cuda").bfloat16()
y, one = torch.zeros(t, dtype=torch.int64, device="cuda"), torch.ones(d, dtype=torch.bfloat16, device="cuda")
q, qs, out = torch.empty(t, d, dtype=torch.int8, device="cuda"), torch.empty(t, 1, device="cuda"), torch.empty(t, v, device="cuda")
codes, sc = torch.zeros(v, 32, dtype=torch.uint8, device="cuda") + 0x11, torch.ones(v, 1, dtype=torch.bfloat16, device="cuda")
loss, lse, dh, dw = torch.empty(t, device="cuda"), torch.empty(t, device="cuda"), torch.empty_like(h), torch.empty_like(w)
k = va.SoftmaxCrossEntropyKernel(c)
ws = torch.empty(max(k.workspace_bytes(t, v, d, b) for b in (False, True)), dtype=torch.uint8, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=s):
    va.RMSNormInt8Kernel(c).encode(h, one, t, d, q, qs)
    va.Int4MatVecKernel(c).encode(q, t, codes, sc, v, d, 64, out, query_dtype=va.DTYPE_INT8, query_scales=qs)
    k.encode_forward(h, w, y, t, v, d, loss, lse, workspace=ws)
    k.encode_backward(h, w, y, lse, None, t, v, d, dh, dw, workspace=ws)
g.replay()
torch.cuda.synchronize()
assert torch.allclose(out, (q.float().sum(1, keepdim=True) * qs).expand(t, v), rtol=1e-5, atol=1e-5)
assert torch.allclose(lse, torch.logsumexp(h.float() @ w.float().t(), 1), rtol=1e-4)
assert torch.isfinite(dh.float()).all() and torch.isfinite(dw.float()).all()
del g
c.synchronize()
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert "captured" in r.stdout, r.stdout + r.stderr


def test_matvec_nothing_to_do(tctx):
    codes, scales, _ = make_table(gen(7), 4, 64, 64, "bf16", False)
    k = va.Int4MatVecKernel(tctx)
    out = torch.full((1, 4), 3.0, device="cuda")
    k.encode(torch.empty(0, 64, device="cuda"), 0, codes, scales, 4, 64, 64, out)
    k.encode(torch.zeros(1, 64, device="cuda"), 1, codes, scales, 0, 64, 64, out)
    tctx.synchronize()
    assert (out == 3.0).all()


def test_int4_database_search(ctx):
    rng = np.random.default_rng(1)
    rows, q = rng.standard_normal((3000, 200)).astype(np.float32), rng.standard_normal((5, 200)).astype(np.float32)
    for kind in ("symmetric", "asymmetric"):
        db = va.Int4Database(ctx, rows, group=32, type=kind)
        stored = va.Int4GroupQuantizationKernel(ctx).dequantize(db.table)
        step = np.abs(rows).reshape(3000, -1).max() / 7 * 2  # no value is off by more than its widest group's step
        assert np.abs(stored - rows).max() <= step
        exact = q.astype(np.float64) @ stored.astype(np.float64).T
        tol = matvec_tolerance(200, 32) * (np.abs(q).astype(np.float64) @ np.abs(stored).astype(np.float64).T)
        assert (np.abs(db.scores(q) - exact) <= tol).all()
        vals, ids = db.search(q, 7)
        order = np.argsort(-db.scores(q), axis=1, kind="stable")[:, :7]
        assert (ids == order).all() and (vals == np.take_along_axis(db.scores(q), order, 1)).all()
        codes, scales, _ = va.RMSNormInt8Kernel(ctx).compute(q, np.ones(200, np.float32))
        _, ids8 = db.search(codes, 7, query_scales=scales)
        want = np.argsort(-(codes.astype(np.float64) @ stored.astype(np.float64).T), axis=1, kind="stable")[:, :1]
        assert (ids8[:, :1] == want).all()
        db.close()


# ------------------------------------------------------------------------------------------ loss
def loss_reference(h, w, labels, c, grad):
    """loss, lse, dh, dw and the bounds of the two gradients' errors, in 64 bits."""
    h, w = h.double(), w.double()
    valid = (labels >= 0) & (labels < w.shape[0])
    at = torch.where(valid, labels, 0)
    hm = torch.where(valid[:, None], h, 0.0)
    z = c * (hm @ w.t())
    lse = torch.logsumexp(c * (h @ w.t()), 1)
    loss = torch.where(valid, lse - z.gather(1, at[:, None])[:, 0], 0.0)
    g = torch.where(valid, grad.double() * c, 0.0)
    p = torch.softmax(z, 1) * g[:, None]
    gz = p.clone()
    gz.scatter_add_(1, at[:, None], -g[:, None])
    dh, dw = gz @ w, gz.t() @ hm
    # Errors of a logit: D / 16 matrix steps of 18 roundings, relative to sum |h w|; of p: that of its exponent
    # (the logit, lse, the fp32 product with c log2 e) and 2^-21 of the exponential and two products.
    dim, rows = h.shape[1], w.shape[0]
    size = c * (hm.abs() @ w.abs().t()).amax(1) + lse.nan_to_num(0.0).abs()
    dz = (18 * dim / 16 + 24) * U32 * size
    dl = dz + (rows / 256 + 64) * U32 + 8 * U32 * lse.abs()
    dp = torch.expm1(dz + dl) + 2.0 ** -20
    # p - [label] is rounded once to bf16, the products are summed in fp32 (the same count of roundings), the result
    # rounded; for dw the weighted rows of h are rounded to bf16 too: (1 + U16)^2 - 1 <= 2 U16 + U16^2 of each product.
    dg = gz.abs() * U16 + (p.abs() + 2.0 ** -126) * dp[:, None] * (1 + U16) + 1e-40
    tokens = h.shape[0]
    bh = dg @ w.abs() + (18 * rows / 16 + 64) * U32 * (gz.abs() @ w.abs())
    bw = dg.t() @ hm.abs() * (1 + U16) + ((18 * tokens / 16 + 64) * U32 + U16) * (gz.abs().t() @ hm.abs())
    return loss, lse, dh, dw, dl, bh * (1 + U16) + dh.abs() * U16 + 1e-38, bw * (1 + U16) + dw.abs() * U16 + 1e-38


def run_loss(c, h, w, labels, scale, grad, workspace=None, hs=None, ws=None):
    t, v, d = h.shape[0], w.shape[0], h.shape[1]
    k = va.SoftmaxCrossEntropyKernel(c)
    loss, lse = torch.full((t,), 7.0, device="cuda"), torch.full((t,), 7.0, device="cuda")
    dh = torch.full((t, d), 7.0, device="cuda", dtype=torch.bfloat16)
    dw = torch.full((v, d), 7.0, device="cuda", dtype=torch.bfloat16)
    k.encode_forward(h, w, labels, t, v, d, loss, lse, scale, hs, ws, workspace)
    k.encode_backward(h, w, labels, lse, grad, t, v, d, dh, dw, scale, hs, ws, workspace)
    c.synchronize()
    return loss, lse, dh, dw


def make_loss(seed, t, v, d, ignored=0.2, spread=2.0):
    g = gen(seed)
    h, w = randn(g, t, d).bfloat16(), (randn(g, v, d) * spread / d ** 0.5).bfloat16()
    labels = torch.randint(0, v, (t,), generator=g, device="cuda")
    labels[torch.rand(t, generator=g, device="cuda") < ignored] = -100
    return h, w, labels, torch.rand(t, generator=g, device="cuda") * 2 - 0.5


def check_loss(got, want):
    loss, lse, dh, dw = got
    rloss, rlse, rdh, rdw, dl, bh, bw = want
    assert ((lse.double() - rlse).abs() <= dl).all()
    assert ((loss.double() - rloss).abs() <= 2 * dl).all()
    assert ((dh.double() - rdh).abs() <= bh).all()
    assert ((dw.double() - rdw).abs() <= bw).all()


@pytest.mark.parametrize("t, v, d", [(1, 1, 8), (1, 300, 64), (2, 257, 72), (127, 255, 64), (129, 256, 128), (130, 1000, 200),
                                     (64, 5003, 512), (333, 5003, 320), (1000, 777, 768), (257, 12345, 136), (2000, 130, 1024), (5, 40000, 1536),
                                     (8192, 1000, 64), (4000, 300, 200), (20001, 700, 72), (3, 515, 4096), (700, 600, 4088)])
def test_loss_matches_64_bits(tctx, t, v, d):
    h, w, labels, grad = make_loss(t * 7 + v + d, t, v, d)
    check_loss(run_loss(tctx, h, w, labels, 1.0, grad), loss_reference(h, w, labels, 1.0, grad))


@pytest.mark.parametrize("t, v, d", [(257, 38000, 72), (1300, 15001, 200), (513, 30000, 768), (2047, 9999, 1000)])
def test_loss_of_many_tiles(tctx, t, v, d):
    # enough tiles for pairs of CTAs, with ragged last tiles
    h, w, labels, grad = make_loss(t + v + d, t, v, d)
    got = run_loss(tctx, h, w, labels, 1.0, grad)
    check_loss(got, loss_reference(h, w, labels, 1.0, grad))
    assert all(torch.equal(a, b) for a, b in zip(got, run_loss(tctx, h, w, labels, 1.0, grad)))


def test_loss_weights_of_every_size(tctx):
    h, w, labels, grad = make_loss(17, 300, 900, 64)
    for g in (grad * 1e-30, torch.where(torch.arange(300, device="cuda") % 7 == 0, grad * 1e20, grad), torch.full_like(grad, 0.1),
              torch.cat([torch.zeros(299, device="cuda"), torch.ones(1, device="cuda")]), -grad.abs() - 0.1):
        check_loss(run_loss(tctx, h, w, labels, 1.0, g), loss_reference(h, w, labels, 1.0, g))


def test_loss_leaves_its_neighbours_alone(tctx):
    for t, v, d in ((70, 300, 72), (400, 20000, 136)):
        h, w, labels, grad = make_loss(18, t, v, d)
        k = va.SoftmaxCrossEntropyKernel(tctx)
        bufs = [torch.full((n,), 7.0, device="cuda", dtype=dt) for n, dt in ((t + 999, torch.float32), (t + 999, torch.float32),
                                                                           (t * d + 9999, torch.bfloat16), (v * d + 9999, torch.bfloat16))]
        need = max(k.workspace_bytes(t, v, d, b) for b in (False, True))
        space = torch.full((need + 4096,), 0x55, dtype=torch.uint8, device="cuda")
        ws = space.data_ptr()
        k.encode_forward(h, w, labels, t, v, d, bufs[0], bufs[1], workspace=ws)
        k.encode_backward(h, w, labels, bufs[1], grad, t, v, d, bufs[2], bufs[3], workspace=ws)
        tctx.synchronize()
        for b, n in zip(bufs, (t, t, t * d, v * d)):
            assert (b[n:] == 7.0).all()
        assert (space[need:] == 0x55).all()


def test_loss_past_32_bit_offsets(tctx):
    # a table of 2.2e9 elements: the last rows against the first
    t, v, d = 130, 1500000, 1472
    g = gen(19)
    w = torch.empty(v, d, dtype=torch.bfloat16, device="cuda").normal_(0, 0.02, generator=g)
    h = randn(g, t, d).bfloat16()
    labels = torch.randint(v - 1000, v, (t,), generator=g, device="cuda")
    loss, lse, dh, dw = run_loss(tctx, h, w, labels, 1.0, None)
    z = torch.cat([h.double() @ w[i:i + 100000].double().t() for i in range(0, v, 100000)], 1)
    want = torch.logsumexp(z, 1)
    assert ((lse.double() - want).abs() <= 1e-5 * want.abs()).all()
    p = torch.softmax(z, 1)
    p[torch.arange(t, device="cuda"), labels] -= 1
    for rows in (slice(0, 300), slice(v - 1000, v)):
        ref = p[:, rows].t() @ h.double()
        # two roundings before the product, one after, and the logits' errors (2^-14 of p)
        bound = (3 * U16 + 2.0 ** -12) * (p[:, rows].abs().t() @ h.double().abs()) + 1e-38
        assert ((dw[rows].double() - ref).abs() <= bound).all()
    del p, z, w, dw
    torch.cuda.empty_cache()


def test_loss_in_several_chunks(tctx):
    # more than 2^28 gradient entries: several pieces of the table, dh added up over them
    h, w, labels, grad = make_loss(11, 4099, 70001, 64)
    check_loss(run_loss(tctx, h, w, labels, 1.0, grad), loss_reference(h, w, labels, 1.0, grad))


def test_loss_strides_scale_and_repeats(tctx):
    g = gen(12)
    hb, wb = randn(g, 150, 136).bfloat16(), randn(g, 400, 160).bfloat16()
    h, w = hb[:, :96], wb[:, 8:104]
    h = h / h.float().norm(dim=1, keepdim=True).bfloat16()
    hb[:, :96] = h
    h = hb[:, :96]
    labels = torch.randint(0, 400, (150,), generator=g, device="cuda")
    labels[:50] = 17  # the same row again and again
    grad = torch.ones(150, device="cuda")
    got = run_loss(tctx, h, w, labels, 3.0, grad, hs=136, ws=160)
    check_loss(got, loss_reference(h, w, labels, 3.0, grad))
    again = run_loss(tctx, h, w, labels, 3.0, None, hs=136, ws=160)
    assert all(torch.equal(a, b) for a, b in zip(got, again))  # None stands for ones; the order of sums is fixed


def test_loss_tokens_without_loss(tctx):
    h, w, labels, grad = make_loss(13, 200, 600, 64, ignored=0.0)
    clean = run_loss(tctx, h, w, labels.clone().index_fill_(0, torch.arange(0, 200, 3, device="cuda"), -1), 1.0, grad)
    # whatever such a token's hidden row holds, and whichever label outside the table it has
    labels[::3] = torch.tensor([-1, -100, 600, 1 << 40, -(1 << 62)], device="cuda").repeat(14)[:67]
    h[::3] = torch.tensor([float("nan"), float("inf"), -3e38], device="cuda").bfloat16().repeat(23)[:67, None]
    loss, lse, dh, dw = run_loss(tctx, h, w, labels, 1.0, grad)
    assert (loss[::3] == 0).all() and (dh[::3] == 0).all()
    keep = torch.ones(200, dtype=torch.bool, device="cuda")
    keep[::3] = False
    assert torch.equal(loss[keep], clean[0][keep]) and torch.equal(dh[keep], clean[2][keep]) and torch.equal(dw, clean[3])
    labels[:] = -1
    loss, lse, dh, dw = run_loss(tctx, h, w, labels, 1.0, grad)
    assert (loss == 0).all() and (dh == 0).all() and (dw == 0).all()


def test_loss_large_logits_and_infinite_rows(tctx):
    h, w, labels, grad = make_loss(14, 96, 700, 64, ignored=0.0, spread=60.0)  # logits of hundreds: softmax near one-hot
    check_loss(run_loss(tctx, h, w, labels, 1.0, grad), loss_reference(h, w, labels, 1.0, grad))
    w[5] = float("-inf")
    h = h.abs() + 0.1
    loss, lse, _, _ = run_loss(tctx, h, w, torch.full_like(labels, 6), 1.0, grad)  # row 5 has logit -inf: no share
    z = h.double() @ w.double().t()
    assert ((lse.double() - torch.logsumexp(z, 1)).abs() <= 1e-5 * z.abs().nan_to_num(0, 0, 0).amax(1)).all()
    w[:] = float("-inf")
    _, lse, _, _ = run_loss(tctx, h, w, labels, 1.0, grad)
    assert (lse == float("-inf")).all()


def test_loss_gradient_against_differences(tctx):
    # hidden on a grid of 1/8, so that a step of 1/8 is exact; |logit change| <= 1/16 per step
    g = gen(15)
    t, v, d = 40, 300, 64
    h = (torch.randint(-8, 9, (t, d), generator=g, device="cuda") / 8).bfloat16()
    w = (torch.randint(-4, 5, (v, d), generator=g, device="cuda") / 8).bfloat16()
    labels = torch.randint(0, v, (t,), generator=g, device="cuda")
    loss, _, dh, _ = run_loss(tctx, h, w, labels, 1.0, None)
    for j in (0, 13, 63):
        up, down = h.clone(), h.clone()
        up[:, j] += 0.125
        down[:, j] -= 0.125
        diff = (run_loss(tctx, up, w, labels, 1.0, None)[0].double() - run_loss(tctx, down, w, labels, 1.0, None)[0].double()) / 0.25
        # third derivative of lse along w_j: a third cumulant of values within +-1/2, at most 1/8; error eps^2 / 6 of it;
        # loss errors of 2^-18 each over the step; the gradient's bf16 sums within 2^-7 of sum |G| |w| <= 1
        assert ((diff - dh[:, j].double()).abs() <= 0.125 ** 2 / 6 / 8 + 2 * 2.0 ** -18 / 0.25 + 2.0 ** -7).all()


def test_loss_no_tokens(tctx):
    w = torch.ones(20, 64, dtype=torch.bfloat16, device="cuda")
    empty = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    *_, dw = run_loss(tctx, empty, w, torch.empty(0, dtype=torch.int64, device="cuda"), 1.0, None)
    assert (dw == 0).all()


def test_loss_of_a_database_and_host_arrays(ctx):
    rng = np.random.default_rng(2)
    h, w = rng.standard_normal((30, 64)).astype(np.float32), rng.standard_normal((90, 64)).astype(np.float32) / 8
    y = rng.integers(0, 90, 30)
    k = va.SoftmaxCrossEntropyKernel(ctx)
    loss, lse, dh, dw = k.compute(h, w, y)
    h16, w16 = (torch.from_numpy(a).bfloat16() for a in (h, w))
    want = loss_reference(h16.cuda(), w16.cuda(), torch.from_numpy(y).cuda(), 1.0, torch.ones(30, device="cuda"))
    check_loss([torch.from_numpy(a).cuda() for a in (loss, lse, dh, dw)], want)
    db = va.Database(ctx, va.scoring._to_bf16(w), dtype=va.DTYPE_BF16)
    dh_, dy = ctx.get_buffer_for(va.scoring._to_bf16(h)), ctx.get_buffer_for(y.astype(np.int64))
    l2, e2 = ctx.get_buffer(120, np.float32), ctx.get_buffer(120, np.float32)
    k.encode_forward(dh_, db, dy, 30, 90, 64, l2, e2)
    assert (l2.download() == loss).all() and (e2.download() == lse).all()
    with pytest.raises(va.InvalidInput, match="bf16 database"):
        k.encode_forward(dh_, va.Database(ctx, w), dy, 30, 90, 64, l2, e2)
    db.close()


# ------------------------------------------------------------------------------------------ together
def test_streams_graphs_and_workspaces():
    """Captured on a side stream and replayed on other inputs, two graphs with a workspace each."""
    s = torch.cuda.Stream()
    c = va.GPUContext(va.Metal4Configuration(device=0, stream=s.cuda_stream))
    norm, matvec, xent = va.RMSNormInt8Kernel(c), va.Int4MatVecKernel(c), va.SoftmaxCrossEntropyKernel(c)
    t, v, d = 70, 900, 128
    h, w, labels, grad = make_loss(21, t, v, d)
    codes, scales, _ = make_table(gen(22), v, d, 64, "bf16", False)
    one = torch.ones(d, dtype=torch.bfloat16, device="cuda")
    q, qs, out = (torch.empty(t, d, dtype=torch.int8, device="cuda"), torch.empty(t, 1, device="cuda"), torch.empty(t, v, device="cuda"))
    size = max(xent.workspace_bytes(t, v, d, b) for b in (False, True))
    sets = []
    for _ in range(2):
        sets.append([torch.empty(size, dtype=torch.uint8, device="cuda"), torch.empty(t, device="cuda"), torch.empty(t, device="cuda"),
                     torch.empty_like(h), torch.empty_like(w)])

    def step(k):
        ws, loss, lse, dh, dw = sets[k]
        norm.encode(h, one, t, d, q, qs)
        matvec.encode(q, t, codes, scales, v, d, 64, out, query_dtype=va.DTYPE_INT8, query_scales=qs)
        xent.encode_forward(h, w, labels, t, v, d, loss, lse, workspace=ws)
        xent.encode_backward(h, w, labels, lse, grad, t, v, d, dh, dw, workspace=ws)

    torch.cuda.synchronize()
    step(0)
    c.synchronize()
    with pytest.raises(va.InvalidInput, match="too small"):
        xent.encode_forward(h, w, labels, t, v, d, sets[0][1], sets[0][2], workspace=torch.empty(128, dtype=torch.uint8, device="cuda"))
    graphs = []
    for k in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            step(k)
            with pytest.raises(va.Unsupported, match="workspace"):
                xent.encode_forward(h, w, labels, t, v, d, sets[k][1], sets[k][2])
        graphs.append(gr)
    h2, w2, labels2, grad2 = make_loss(23, t, v, d)
    h.copy_(h2), w.copy_(w2), labels.copy_(labels2), grad.copy_(grad2)
    torch.cuda.synchronize()
    for gr in graphs:
        gr.replay()
    torch.cuda.synchronize()
    want = loss_reference(h, w, labels, 1.0, grad)
    for k in range(2):
        check_loss(sets[k][1:], want)
    codes_want, _ = norm_reference(h, one, 1e-6, 0)
    assert torch.equal(q.double(), codes_want)
    ref, mag = matvec_reference(q, qs[:, 0], codes, scales, None, d, 64)
    assert ((out.double() - ref).abs() <= matvec_tolerance(d, 64) * mag).all()
    del graphs
    c.synchronize()
    c.close()


def test_two_contexts_at_once():
    """The same work on two streams, each context with its own scratch."""
    ss = [torch.cuda.Stream() for _ in range(2)]
    cs = [va.GPUContext(va.Metal4Configuration(device=0, stream=s.cuda_stream)) for s in ss]
    data = [make_loss(31 + i, 500, 3000 + 700 * i, 256) for i in range(2)]
    torch.cuda.synchronize()
    outs = []
    for c, (h, w, labels, grad) in zip(cs, data):
        k = va.SoftmaxCrossEntropyKernel(c)
        o = [torch.empty(500, device="cuda"), torch.empty(500, device="cuda"), torch.empty_like(h), torch.empty_like(w)]
        outs.append((k, o))
    torch.cuda.synchronize()
    for _ in range(3):
        for (k, o), (h, w, labels, grad) in zip(outs, data):
            k.encode_forward(h, w, labels, 500, w.shape[0], 256, o[0], o[1])
            k.encode_backward(h, w, labels, o[1], grad, 500, w.shape[0], 256, o[2], o[3])
    for c in cs:
        c.synchronize()
    for (k, o), (h, w, labels, grad) in zip(outs, data):
        check_loss(o, loss_reference(h, w, labels, 1.0, grad))
    for c in cs:
        c.close()


def test_train_quantize_and_score(tctx):
    """A step of training moves the table, the table goes to 4 bits, a normed token finds its label."""
    t, v, d = 64, 512, 128
    h, w, labels, _ = make_loss(41, t, v, d, ignored=0.0)
    w32 = w.float()
    losses = []
    for _ in range(3):
        loss, lse, dh, dw = run_loss(tctx, h, w32.bfloat16(), labels, 1.0, torch.full((t,), 1.0 / t, device="cuda"))
        losses.append(loss.mean())
        want = loss_reference(h, w32.bfloat16(), labels, 1.0, torch.full((t,), 1.0 / t, device="cuda"))
        check_loss((loss, lse, dh, dw), want)
        w32 -= 4.0 * dw.float()
    db = va.Int4Database(tctx, w32.cpu().numpy(), group=32)
    q = torch.empty(t, d, dtype=torch.int8, device="cuda")
    qs = torch.empty(t, 1, device="cuda")
    va.RMSNormInt8Kernel(tctx).encode(h, torch.ones(d, dtype=torch.bfloat16, device="cuda"), t, d, q, qs)
    tctx.synchronize()
    vals, ids = db.search(q.cpu().numpy(), 5, query_scales=qs.cpu().numpy())
    stored = torch.from_numpy(va.Int4GroupQuantizationKernel(tctx).dequantize(db.table)).double().cuda()
    exact = (q.double() * qs.double()) @ stored.t()
    tol = matvec_tolerance(d, 32) * ((q.double() * qs.double()).abs() @ stored.abs().t())
    picked = torch.from_numpy(ids.astype(np.int64)).cuda()
    assert ((torch.from_numpy(vals).cuda().double() - exact.gather(1, picked)).abs() <= tol.gather(1, picked)).all()
    kth = exact.topk(5, 1).values[:, -1]  # what is returned is among the five best, up to the tolerance
    assert (exact.gather(1, picked) >= (kth - 2 * tol.amax(1))[:, None]).all()
    db.close()
