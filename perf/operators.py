"""Cases of the scoring-head operators: what is timed, on which inputs, and their plain forms.

Three operators around a table of rows that queries are scored against:

``norm``    residual addition + root-mean-square norm + int8 codes with scales (one token to a long
            batch): h = x + residual, z = h * weight, code = rint(127 z / max|z|) over a row or a
            group, scale = max|z| / (127 rms(h)).
``matvec``  scores of 1..16 queries against rows held as 4-bit codes with a scale (and a zero point)
            per group: out[q, r] = sum_j x[q, j] * scale[r, g(j)] * (code[r, j] - zero[r, g(j)]).
``loss``    softmax cross entropy of tokens against all rows of a table (the vocabulary, or the
            documents of a retrieval model), its logits never kept, forward alone or with the
            gradients of both sides; tokens whose label lies outside the table carry no loss.

With ``own`` false ``run`` is the plain form in elementary torch operations; with ``own`` true it
makes the library's calls.
"""

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # One token through the last norm of an encoder, as in serving: latency.
        dict(name="norm 1 token", op="norm", rows=1, dim=1536, dtype="bf16", group=0, residual=True, pad=0),
        # A ragged batch of fp32 embeddings, scales per group of 64, rows inside a wider buffer.
        dict(name="norm batch f32 groups", op="norm", rows=10007, dim=1000, dtype="f32", group=64, residual=False, pad=24),
        # A long prefill batch.
        dict(name="norm long", op="norm", rows=65536, dim=4096, dtype="bf16", group=0, residual=True, pad=0),
        # A small table, one query: latency.
        dict(name="matvec small", op="matvec", rows=5003, dim=512, queries=1, dtype="bf16", scales="bf16", group=64, zeros=False),
        # One fp32 query over a large table of embeddings.
        dict(name="matvec 1 query", op="matvec", rows=2000000, dim=768, queries=1, dtype="f32", scales="bf16", group=64, zeros=False),
        # A batch of int8 queries (the norm's output) over an asymmetric table.
        dict(name="matvec 16 int8 queries", op="matvec", rows=300007, dim=1536, queries=16, dtype="int8", scales="f32", group=128, zeros=True),
        # A few queries over wide rows with fine groups.
        dict(name="matvec wide rows", op="matvec", rows=50000, dim=4096, queries=5, dtype="bf16", scales="bf16", group=32, zeros=False),
        # Evaluation of a handful of tokens over a small table: latency.
        dict(name="loss eval small", op="loss", tokens=16, rows=10000, dim=128, train=False, temperature=False, ignored=0.0),
        # Evaluation of a batch over a large ragged table.
        dict(name="loss eval", op="loss", tokens=1000, rows=100003, dim=768, train=False, temperature=False, ignored=0.1),
        # A training step of a small model: a short, ragged batch.
        dict(name="loss train small", op="loss", tokens=333, rows=5003, dim=512, train=True, temperature=False, ignored=0.1),
        # A contrastive training step over unit vectors with a temperature.
        dict(name="loss train contrastive", op="loss", tokens=4096, rows=65536, dim=768, train=True, temperature=True, ignored=0.0),
        # A training step over a long batch and a large vocabulary, some of the tokens padding.
        dict(name="loss train large", op="loss", tokens=8192, rows=131072, dim=1536, train=True, temperature=False, ignored=0.2),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["norm", "matvec", "loss"])
    if op == "norm":
        rows, dim = _log_int(rng, 1, 65536), _log_int(rng, 64, 4096)
        return dict(op=op, rows=rows, dim=dim, dtype=rng.choice(["bf16", "f32"]) if rows <= 32768 else "bf16",
                    group=rng.choice([0, 0, 32, 64, 128]), residual=rng.random() < 0.6, pad=rng.choice([0, 0, 8, 13]))
    if op == "matvec":
        dim = _log_int(rng, 64, 4096)
        rows = _log_int(rng, 1000, min(2000000, 1500000000 // dim))
        return dict(op=op, rows=rows, dim=dim, queries=rng.choice([1, 1, 1, 2, 3, 4, 5, 7, 8, 11, 16]),
                    dtype=rng.choice(["bf16", "f32", "int8"]), scales=rng.choice(["bf16", "f32"]),
                    group=rng.choice([32, 64, 128]), zeros=rng.random() < 0.4)
    dim = 8 * _log_int(rng, 8, 192)
    tokens = _log_int(rng, 1, 8192)
    rows = _log_int(rng, 1000, 131072)
    return dict(op=op, tokens=tokens, rows=rows, dim=dim, train=rng.random() < 0.6, temperature=rng.random() < 0.3,
                ignored=rng.choice([0.0, 0.1, 0.3]))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    s = dict(case)
    if case["op"] == "norm":
        dt, rows, dim = _DT[case["dtype"]], case["rows"], case["dim"]
        # Activations with a few channels far above the rest, as hidden states have.
        channel = torch.exp(0.5 * normal(dim))
        s["x"] = (normal(rows, dim + case["pad"])[:, :dim] * channel).to(dt) if not case["pad"] else \
            normal(rows, dim + case["pad"], dtype=dt)[:, :dim]
        s["residual"] = normal(rows, dim, dtype=dt, scale=2.0) if case["residual"] else None
        s["weight"] = (1.0 + 0.2 * normal(dim)).to(dt)
    elif case["op"] == "matvec":
        rows, dim, group, nq = case["rows"], case["dim"], case["group"], case["queries"]
        stride, groups = (dim + 31) // 32 * 16, (dim + group - 1) // group
        # Codes as a quantizer leaves them: most in the middle of the range, the padding zero.
        codes = torch.randint(0, 256, (rows, stride), generator=g, device="cuda", dtype=torch.uint8)
        codes[:, (dim + 1) // 2:] = 0
        if dim % 2:
            codes[:, dim // 2] &= 15
        s["codes"] = codes
        s["scales"] = (0.004 * torch.exp(0.3 * normal(rows, groups))).to(_DT[case["scales"]])
        s["zeros"] = torch.randint(-3, 4, (rows, groups), generator=g, device="cuda", dtype=torch.int8) if case["zeros"] else None
        if case["dtype"] == "int8":
            s["x"] = torch.clamp(torch.round(normal(nq, dim) * 36), -127, 127).to(torch.int8)
            s["x_scales"] = 0.02 * torch.exp(0.2 * normal(nq))
        else:
            s["x"] = normal(nq, dim, dtype=_DT[case["dtype"]])
            s["x_scales"] = None
    else:
        tokens, rows, dim = case["tokens"], case["rows"], case["dim"]
        h, w = normal(tokens, dim), normal(rows, dim)
        if case["temperature"]:
            h, w = h / h.norm(dim=1, keepdim=True), w / w.norm(dim=1, keepdim=True)
            s["scale"] = 20.0
        else:
            w *= 2.0 / math.sqrt(dim)
            s["scale"] = 1.0
        s["h"], s["w"] = h.to(torch.bfloat16), w.to(torch.bfloat16)
        # Labels are skewed, as tokens and popular documents are.
        u = torch.rand(tokens, generator=g, device="cuda")
        labels = (rows * u * u).long().clamp_(0, rows - 1)
        labels[torch.rand(tokens, generator=g, device="cuda") < case["ignored"]] = -100
        s["labels"] = labels
        # The gradient of the mean over the tokens that carry a loss.
        valid = labels >= 0
        s["grad_loss"] = valid.float() / valid.sum().clamp(min=1)
    return s


def work(case):
    if case["op"] == "norm":
        n, b = case["rows"] * case["dim"], 2 if case["dtype"] == "bf16" else 4
        scales = case["rows"] * (-(-case["dim"] // case["group"]) if case["group"] else 1)
        moved = n * (b + 1) + (2 * n * b if case["residual"] else 0) + 4 * scales + b * case["dim"]
        return {"bytes": moved, "flops": 6 * n}
    if case["op"] == "matvec":
        rows, dim, nq = case["rows"], case["dim"], case["queries"]
        groups = -(-dim // case["group"])
        moved = rows * dim / 2 + rows * groups * ((2 if case["scales"] == "bf16" else 4) + (1 if case["zeros"] else 0))
        moved += nq * dim * {"bf16": 2, "f32": 4, "int8": 1}[case["dtype"]] + 4 * nq * rows
        return {"bytes": moved, "flops": 2 * nq * rows * dim}
    t, v, d = case["tokens"], case["rows"], case["dim"]
    if case["train"]:
        return {"bytes": 4 * (t + v) * d + 20 * t, "flops": 6 * t * v * d}
    return {"bytes": 2 * (t + v) * d + 16 * t, "flops": 2 * t * v * d}


# ------------------------------------------------------------------------------------------ plain forms
def _grouped(z, group):
    rows, dim = z.shape
    size = group if group else dim
    return torch.nn.functional.pad(z, (0, -dim % size)).view(rows, -1, size)


def _norm_plain(s):
    h = s["x"]
    if s["residual"] is not None:
        h = (h.float() + s["residual"].float()).to(h.dtype)
    # 64 bits: a code is decided at the border between two whole numbers.
    h64 = h.double()
    z = _grouped(h64 * s["weight"].double(), s["group"])
    rms = torch.sqrt((h64 * h64).mean(dim=1) + 1e-6)
    top = z.abs().amax(dim=2)
    codes = torch.round(z * 127.0 / torch.where(top > 0, top, 1.0)[:, :, None])
    scales = (top / (127.0 * rms[:, None])).float()
    values = (codes.float() * scales[:, :, None]).reshape(h.shape[0], -1)[:, : h.shape[1]].to(h.dtype)
    return {"values": values, "scales": scales, "residual": h if s["residual"] is not None else None}


def _matvec_plain(s):
    dim, group = s["dim"], s["group"]
    w = torch.stack((s["codes"] & 15, s["codes"] >> 4), dim=2).flatten(1)[:, :dim]
    w = ((w ^ 8).to(torch.float32) - 8.0)
    index = torch.arange(dim, device=w.device) // group
    if s["zeros"] is not None:
        w -= s["zeros"].float()[:, index]
    w *= s["scales"].float()[:, index]
    out = s["x"].float() @ w.t()
    return out * s["x_scales"][:, None] if s["x_scales"] is not None else out


def _loss_plain(s):
    h, w, labels = s["h"].float(), s["w"].float(), s["labels"]
    valid = (labels >= 0) & (labels < w.shape[0])
    at = torch.where(valid, labels, 0)
    logits = (h @ w.t()) * s["scale"]
    top = logits.amax(dim=1)
    lse = torch.log(torch.exp(logits - top[:, None]).sum(dim=1)) + top
    loss = torch.where(valid, lse - logits.gather(1, at[:, None])[:, 0], 0.0)
    if not s["train"]:
        return {"loss": loss, "lse": lse}
    g = torch.where(valid, s["grad_loss"], 0.0)
    p = torch.exp(logits - lse[:, None]) * (g * s["scale"])[:, None]
    p.scatter_add_(1, at[:, None], -(g * s["scale"])[:, None])
    return {"loss": loss, "lse": lse, "grad_hidden": (p @ w).to(torch.bfloat16),
            "grad_table": (p.t() @ torch.where(valid[:, None], h, 0.0)).to(torch.bfloat16)}


# ------------------------------------------------------------------------------------------ the library's calls
_kept = {}


def _kernels():
    """The context and kernel objects a program keeps, one set per device and stream: the calls go to the stream
    that torch's own work around them is on."""
    device = torch.cuda.current_device()
    # Stream handle 1 is CUDA's name of the default stream (torch calls it 0).
    stream = torch.cuda.current_stream(device).cuda_stream or 1
    if (device, stream) not in _kept:
        import vectoraccelerate_b200 as va
        ctx = va.GPUContext(va.Metal4Configuration(device=device, stream=stream))
        _kept[device, stream] = (va, va.RMSNormInt8Kernel(ctx), va.Int4MatVecKernel(ctx), va.SoftmaxCrossEntropyKernel(ctx))
    return _kept[device, stream]


def _norm_own(s):
    va, kernel, _, _ = _kernels()
    x = s["x"]
    rows, dim = x.shape
    group = s["group"]
    codes = torch.empty((rows, dim), dtype=torch.int8, device=x.device)
    scales = torch.empty((rows, -(-dim // group) if group else 1), dtype=torch.float32, device=x.device)
    out = torch.empty((rows, dim), dtype=x.dtype, device=x.device) if s["residual"] is not None else None
    kernel.encode(x, s["weight"], rows, dim, codes, scales, residual=s["residual"], residual_out=out,
                  dtype=va.DTYPE_BF16 if x.dtype is torch.bfloat16 else va.DTYPE_F32, epsilon=1e-6, group=group,
                  x_stride=x.stride(0))
    # The values that the codes stand for, as the plain form gives them.
    values = torch.empty((rows, dim), dtype=x.dtype, device=x.device)
    if group and dim % group:
        full = dim // group * group
        torch.mul(codes[:, :full].unflatten(1, (-1, group)), scales[:, :-1, None], out=values[:, :full].unflatten(1, (-1, group)))
        torch.mul(codes[:, full:], scales[:, -1:], out=values[:, full:])
    elif group:
        torch.mul(codes.view(rows, -1, group), scales[:, :, None], out=values.view(rows, -1, group))
    else:
        torch.mul(codes, scales, out=values)
    return {"values": values, "scales": scales, "residual": out}


def _matvec_own(s):
    va, _, kernel, _ = _kernels()
    x, rows, nq = s["x"], s["rows"], s["queries"]
    out = torch.empty((nq, rows), dtype=torch.float32, device=x.device)
    kernel.encode(x, nq, s["codes"], s["scales"], rows, s["dim"], s["group"], out, zero_points=s["zeros"],
                  query_dtype={"bf16": va.DTYPE_BF16, "f32": va.DTYPE_F32, "int8": va.DTYPE_INT8}[s["dtype"]],
                  query_scales=s["x_scales"], scale_dtype=va.DTYPE_BF16 if s["scales"].dtype is torch.bfloat16 else va.DTYPE_F32)
    return out


def _loss_own(s):
    _, _, _, kernel = _kernels()
    h, w = s["h"], s["w"]
    tokens, rows, dim = h.shape[0], w.shape[0], h.shape[1]
    loss = torch.empty(tokens, dtype=torch.float32, device=h.device)
    lse = torch.empty(tokens, dtype=torch.float32, device=h.device)
    kernel.encode_forward(h, w, s["labels"], tokens, rows, dim, loss, lse, logit_scale=s["scale"])
    if not s["train"]:
        return {"loss": loss, "lse": lse}
    grad_h, grad_w = torch.empty_like(h), torch.empty_like(w)
    kernel.encode_backward(h, w, s["labels"], lse, s["grad_loss"], tokens, rows, dim, grad_h, grad_w, logit_scale=s["scale"])
    return {"loss": loss, "lse": lse, "grad_hidden": grad_h, "grad_table": grad_w}


def run(s):
    if own:
        return {"norm": _norm_own, "matvec": _matvec_own, "loss": _loss_own}[s["op"]](s)
    return {"norm": _norm_plain, "matvec": _matvec_plain, "loss": _loss_plain}[s["op"]](s)


# ------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)

    def norm():
        x = s["x"].double()
        if s["residual"] is not None:
            # Stored in the input's type: the norm is that of what is stored.
            x = (x + s["residual"].double()).to(s["x"].dtype).double()
        rows, dim = x.shape
        group = case["group"] or dim
        inverse = (x.pow(2).sum(1) / dim + 1e-6).rsqrt()
        values, scales = torch.zeros(rows, dim, dtype=torch.float64, device=x.device), []
        for j in range(0, dim, group):
            z = x[:, j:j + group] * s["weight"].double()[j:j + group]
            peak = z.abs().max(1).values
            step = peak * inverse / 127.0
            codes = torch.round(z * 127.0 / peak.clamp(min=1e-300)[:, None])
            values[:, j:j + group] = codes * step[:, None]
            scales.append(step)
        return {"values": values, "scales": torch.stack(scales, 1), "residual": x if s["residual"] is not None else None}

    def matvec():
        rows, dim, group = case["rows"], case["dim"], case["group"]
        x = s["x"].double()
        if s["x_scales"] is not None:
            x = x * s["x_scales"].double()[:, None]
        out = torch.empty(case["queries"], rows, dtype=torch.float64, device=x.device)
        for r in range(0, rows, 100000):
            c = s["codes"][r:r + 100000].to(torch.int32)
            total = torch.zeros(case["queries"], c.shape[0], dtype=torch.float64, device=x.device)
            for j in range(0, dim, group):
                k = torch.arange(j, min(j + group, dim), device=x.device)
                v = (c[:, k // 2] >> (4 * (k % 2)).to(torch.int32)) & 15
                v = torch.where(v > 7, v - 16, v).double()
                if s["zeros"] is not None:
                    v = v - s["zeros"][r:r + 100000, j // group, None].double()
                total += (x[:, k] @ v.t()) * s["scales"][r:r + 100000, j // group].double()
            out[:, r:r + 100000] = total
        return out

    def cross_entropy():
        h, w, scale, labels = s["h"].double(), s["w"].double(), s["scale"], s["labels"]
        tokens = case["tokens"]
        loss = torch.zeros(tokens, dtype=torch.float64, device=h.device)
        lse = torch.empty(tokens, dtype=torch.float64, device=h.device)
        grad_h, grad_w = torch.zeros_like(h), torch.zeros_like(w)
        for t in range(0, tokens, 1024):
            rows = slice(t, min(tokens, t + 1024))
            z = scale * (h[rows] @ w.t())
            lse[rows] = torch.logsumexp(z, 1)
            keep = ((labels[rows] >= 0) & (labels[rows] < case["rows"])).nonzero()[:, 0]
            at = labels[rows][keep]
            loss[rows][keep] = lse[rows][keep] - z[keep, at]
            if case["train"]:
                p = torch.exp(z[keep] - lse[rows][keep, None])
                p[torch.arange(len(keep), device=p.device), at] -= 1.0
                p *= scale * s["grad_loss"][rows][keep, None].double()
                grad_h[rows][keep] = p @ w
                grad_w += p.t() @ h[rows][keep]
            del z
        if not case["train"]:
            return {"loss": loss, "lse": lse}
        return {"loss": loss, "lse": lse, "grad_hidden": grad_h, "grad_table": grad_w}

    return {"norm": norm, "matvec": matvec, "loss": cross_entropy}[case["op"]]()
