"""Benchmark cases of the operators around a gated feed-forward layer: layer norm and
its gradient, the gated product (both projections, the activation and their product)
and its gradient, and 8-bit operands with a scale for each block of 128, made and
multiplied.

Every case can be run in two ways: in plain torch operations (own = False), and
through vcsr_b200.layers (own = True).
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16,
          "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1}
EPS = 1e-5
BLOCK = 128     # values of a row (and rows of a weight matrix) that share a scale
TOP = 448.0     # the largest e4m3 value


def layers():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "vcsr-spmm_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from vcsr_b200 import layers as module
    return module


# ---------------------------------------------------------------------- cases

def listed():
    return [
        # one token's row between two layers of a model that answers
        dict(name="layernorm_token", op="layernorm", rows=1, dim=4096, x="bf16", y="bf16",
             residual=True, bias=True, train=False),
        # the FP32 result of the FEM product (62,451 rows, O = 128) made the 16-bit operand
        # of a dense product, mean and rstd kept for the gradient
        dict(name="layernorm_fem", op="layernorm", rows=62451, dim=128, x="f32", y="bf16",
             residual=True, bias=True, train=True),
        # a training batch's gradient with the residual stream's own, odd row count
        dict(name="layernorm_back", op="layernorm_back", rows=8191, dim=5120, x="bf16", y="bf16",
             residual=True, bias=True),
        # a small ragged batch in FP32: rows off 16 bytes
        dict(name="layernorm_back_odd", op="layernorm_back", rows=2001, dim=1501, x="f32", y="f32",
             residual=False, bias=True),
        # one token through both projections: the weights are read once
        dict(name="gated_token", op="gated", m=1, n=8192, k=4096, x="bf16", y="bf16", act="silu",
             bias=False, pre=False),
        # the rows of a training batch, both projections kept for the gradient: the largest
        dict(name="gated_large", op="gated", m=8192, n=8192, k=4096, x="bf16", y="bf16",
             act="silu", bias=False, pre=True),
        # the gradient of half such a batch
        dict(name="gated_back", op="gated_back", m=4096, n=8192, k=4096, x="bf16", act="silu",
             bias=False),
        # a small ragged layer: no size is a multiple of eight
        dict(name="gated_back_odd", op="gated_back", m=1001, n=777, k=1501, x="f16", act="gelu",
             bias=True),
        # a prompt's rows made 8-bit operands, 128 values to a scale
        dict(name="block_quantize_rows", op="block_quantize", rows=16384, dim=4096, x="bf16",
             block_rows=1),
        # FP32 weights made 8-bit ones, 128 x 128 to a scale, odd sizes
        dict(name="block_quantize_weights", op="block_quantize", rows=4001, dim=2500, x="f32",
             block_rows=128),
        # one token against 8-bit weights
        dict(name="block_linear_token", op="block_linear", m=1, n=8192, k=4096, y="bf16", act="none",
             bias=False, residual=True),
        # a prompt's rows against them
        dict(name="block_linear_prompt", op="block_linear", m=8192, n=8192, k=4096, y="bf16",
             act="none", bias=False, residual=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layernorm", "layernorm_back", "gated", "gated", "gated_back",
                     "block_quantize", "block_linear", "block_linear"])
    if op in ("layernorm", "layernorm_back", "block_quantize"):
        dim = _log(rng, 16, 16384)
        if rng.random() < 0.6:
            dim = max(8, dim // 8 * 8)
        rows = _log(rng, 1, max(1, min(65536, 16384 * 4096 // dim)))
        x = rng.choice(["f32", "bf16", "f16"])
        if op == "block_quantize":
            return dict(op=op, rows=rows, dim=dim, x=x, block_rows=rng.choice([1, BLOCK]))
        case = dict(op=op, rows=rows, dim=dim, x=x, residual=rng.random() < 0.7,
                    bias=rng.random() < 0.7)
        if op == "layernorm":
            case["y"] = rng.choice(["f32", "bf16", "f16", "e4m3"])
            case["train"] = rng.random() < 0.5
        else:
            case["y"] = rng.choice(["f32", "bf16", "f16"])
        return case
    n, k = _log(rng, 64, 8192), _log(rng, 64, 4096)
    if rng.random() < 0.6:
        n, k = max(16, n // 16 * 16), max(16, k // 16 * 16)
    m = _log(rng, 1, 8192)
    act = rng.choice(["none", "relu", "gelu", "silu"])
    if op == "block_linear":
        return dict(op=op, m=m, n=n, k=k, y=rng.choice(["bf16", "f16", "f32"]), act=act,
                    bias=rng.random() < 0.5, residual=rng.random() < 0.5)
    x = rng.choice(["bf16", "f16", "f32"] + (["e4m3"] if op == "gated" else []))
    if op == "gated_back":
        m = min(m, 4096)
    if x == "f32":
        m = min(m, 2048)
    case = dict(op=op, m=m, n=n, k=k, x=x, act=act, bias=rng.random() < 0.5)
    if op == "gated":
        case.update(y=x if x != "e4m3" else rng.choice(["bf16", "f16", "f32"]),
                    pre=rng.random() < 0.5)
    return case


def _blocks(n):
    return -(-n // BLOCK)


# --------------------------------------------------------------------- inputs

def _spread(scale, rows, dim, block_rows):
    """The scale of every value of a (rows, dim) matrix."""
    full = scale.repeat_interleave(block_rows, 0)[:rows] if block_rows > 1 else scale
    return full.repeat_interleave(BLOCK, 1)[:, :dim]


def _block_tops(x, block_rows):
    """The largest magnitude of every block of block_rows x 128 values."""
    rows, dim = x.shape
    down, across = -(-rows // block_rows), _blocks(dim)
    padded = torch.zeros(down * block_rows, across * BLOCK, device=x.device, dtype=x.dtype)
    padded[:rows, :dim] = x.abs()
    return padded.view(down, block_rows, across, BLOCK).amax(3).amax(1)


def _block_codes(x, block_rows):
    scale = _block_tops(x, block_rows) / TOP
    divisor = torch.where(scale > 0, scale, torch.ones_like(scale))
    codes = (x / _spread(divisor, *x.shape, block_rows)).to(DTYPES["e4m3"])
    return codes, scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev = torch.device("cuda")

    def normal(*shape, scale=1.0, shift=0.0, dtype=torch.float32):
        t = torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32)
        return t.mul_(scale).add_(shift).to(dtype)

    def activations(rows, dim):
        t = normal(rows, dim)
        t[:, :: max(1, dim // 7)] *= 8  # a few columns are larger, as activations have them
        return t

    st = dict(case=case)
    if case["op"] in ("layernorm", "layernorm_back"):
        xt, rows, dim = DTYPES[case["x"]], case["rows"], case["dim"]
        x = activations(rows, dim).add_(0.25)
        st["weight"] = normal(dim, scale=0.1, shift=1.0, dtype=xt)
        if case["op"] == "layernorm":
            st["x"] = x.to(xt)
            st["bias"] = normal(dim, scale=0.1, dtype=xt) if case["bias"] else None
            st["residual"] = normal(rows, dim, dtype=xt) if case["residual"] else None
        else:
            st["s"] = x.to(xt)
            s = st["s"].float()
            st["mean"] = s.mean(1)
            st["rstd"] = torch.rsqrt((s - st["mean"][:, None]).square().mean(1) + EPS)
            st["dy"] = normal(rows, dim, scale=1e-2, dtype=DTYPES[case["y"]])
            st["dsum"] = normal(rows, dim, scale=1e-2, dtype=xt) if case["residual"] else None
    elif case["op"] in ("gated", "gated_back"):
        xt, m, n, k = DTYPES[case["x"]], case["m"], case["n"], case["k"]
        yt = DTYPES[case.get("y", case["x"])]
        x, w = normal(m, k), normal(2 * n, k, scale=k ** -0.5)
        if case["x"] == "e4m3":
            st["x_scale"] = x.abs().amax(1) / TOP
            st["w_scale"] = w.abs().amax(1) / TOP
            x, w = x / st["x_scale"][:, None], w / st["w_scale"][:, None]
        st["x"], st["w"] = x.to(xt), w.to(xt)
        st["bias"] = normal(2 * n, scale=0.1, dtype=yt) if case["bias"] else None
        if case["op"] == "gated_back":
            st["dy"] = normal(m, n, scale=1e-2, dtype=xt)
            st["pre"] = normal(m, 2 * n, dtype=xt)
    elif case["op"] == "block_quantize":
        rows, dim = case["rows"], case["dim"]
        x = activations(rows, dim) if case["block_rows"] == 1 else normal(rows, dim, scale=dim ** -0.5)
        st["x"] = x.to(DTYPES[case["x"]])
    else:
        m, n, k, yt = case["m"], case["n"], case["k"], DTYPES[case["y"]]
        st["x"], st["x_scale"] = _block_codes(activations(m, k), 1)
        st["w"], st["w_scale"] = _block_codes(normal(n, k, scale=k ** -0.5), BLOCK)
        st["bias"] = normal(n, scale=0.1, dtype=yt) if case["bias"] else None
        st["residual"] = normal(m, n, dtype=yt) if case["residual"] else None
    return st


# ----------------------------------------------------------------------- runs

def run(st):
    return (run_own if own else run_plain)(st)


def run_own(st):
    case, L = st["case"], layers()
    if case["op"] == "layernorm":
        out = L.layernorm(st["x"], st["weight"], st["bias"], residual=st["residual"], eps=EPS,
                          out_dtype=DTYPES[case["y"]], save_stats=case["train"])
        y = out.y
        if case["y"] == "e4m3":
            y = L.dequantize(y, out.scale, torch.bfloat16)
        return dict(y=y, s=out.sum if case["residual"] else None, mean=out.mean, rstd=out.rstd)
    if case["op"] == "layernorm_back":
        dx, dw, db = L.layernorm_backward(st["dy"], st["s"], st["weight"], st["mean"], st["rstd"],
                                          dsum=st["dsum"], need_dbias=case["bias"])
        return dict(dx=dx, dw=dw, db=db)
    if case["op"] == "gated":
        out = L.gated_linear(st["x"], st["w"], bias=st["bias"], act=case["act"],
                             x_scale=st.get("x_scale"), w_scale=st.get("w_scale"),
                             out_dtype=DTYPES[case["y"]], save_pre=case["pre"])
        return dict(y=out.y, pre=out.pre)
    if case["op"] == "gated_back":
        g = L.gated_linear_backward(st["dy"], st["x"], st["w"], st["pre"], act=case["act"],
                                    need_db=case["bias"])
        return dict(dx=g.dx, dw=g.dw, db=g.db)
    if case["op"] == "block_quantize":
        q = L.block_quantize(st["x"], block_rows=case["block_rows"])
        return dict(values=L.block_dequantize(q.codes, q.scale, block_rows=case["block_rows"],
                                              out_dtype=torch.bfloat16), scale=q.scale)
    return dict(y=L.block_linear(st["x"], st["w"], st["x_scale"], st["w_scale"], bias=st["bias"],
                                 residual=st["residual"], act=case["act"],
                                 out_dtype=DTYPES[case["y"]]))


def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "gelu":
        return (0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
                + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi))
    if act == "silu":
        sig = 1 / (1 + torch.exp(-z))
        return sig * (1 + z * (1 - sig))
    return torch.ones_like(z)


def run_plain(st):
    case = st["case"]
    if case["op"] == "layernorm":
        s = st["x"].float()
        if case["residual"]:
            s = s + st["residual"].float()
        mean = s.mean(1)
        centred = s - mean[:, None]
        rstd = 1 / torch.sqrt((centred * centred).mean(1) + EPS)
        y = centred * rstd[:, None] * st["weight"].float()
        if case["bias"]:
            y = y + st["bias"].float()
        if case["y"] == "e4m3":
            scale = y.abs().amax(1, keepdim=True) / TOP
            q = (y / torch.where(scale > 0, scale, torch.ones_like(scale))).to(DTYPES["e4m3"])
            y = (q.float() * scale).to(torch.bfloat16)
        else:
            y = y.to(DTYPES[case["y"]])
        return dict(y=y, s=s.to(DTYPES[case["x"]]) if case["residual"] else None,
                    mean=mean if case["train"] else None, rstd=rstd if case["train"] else None)
    if case["op"] == "layernorm_back":
        rstd, dy = st["rstd"][:, None], st["dy"].float()
        h = (st["s"].float() - st["mean"][:, None]) * rstd
        g = dy * st["weight"].float()
        dx = rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
        if case["residual"]:
            dx = dx + st["dsum"].float()
        wt = st["weight"].dtype
        return dict(dx=dx.to(st["s"].dtype), dw=(dy * h).sum(0).to(wt),
                    db=dy.sum(0).to(wt) if case["bias"] else None)
    if case["op"] == "gated":
        z = st["x"].float() @ st["w"].float().t()
        if case["x"] == "e4m3":
            z = z * st["x_scale"][:, None] * st["w_scale"]
        if case["bias"]:
            z = z + st["bias"].float()
        n, yt = case["n"], DTYPES[case["y"]]
        y = _act(z[:, :n], case["act"]) * z[:, n:]
        return dict(y=y.to(yt), pre=z.to(yt) if case["pre"] else None)
    if case["op"] == "gated_back":
        n, xt = case["n"], st["x"].dtype
        gate, up, dy = st["pre"][:, :n].float(), st["pre"][:, n:].float(), st["dy"].float()
        dz = torch.cat([dy * up * _act_grad(gate, case["act"]), dy * _act(gate, case["act"])], 1)
        return dict(dx=(dz @ st["w"].float()).to(xt), dw=(dz.t() @ st["x"].float()).to(xt),
                    db=dz.sum(0).to(xt) if case["bias"] else None)
    if case["op"] == "block_quantize":
        rows, dim, block_rows = case["rows"], case["dim"], case["block_rows"]
        codes, scale = _block_codes(st["x"].float(), block_rows)
        values = codes.float() * _spread(scale, rows, dim, block_rows)
        return dict(values=values.to(torch.bfloat16), scale=scale)
    m, n, k = case["m"], case["n"], case["k"]
    x = st["x"].float() * _spread(st["x_scale"], m, k, 1)
    w = st["w"].float() * _spread(st["w_scale"], n, k, BLOCK)
    z = x @ w.t()
    if case["bias"]:
        z = z + st["bias"].float()
    y = _act(z, case["act"])
    if case["residual"]:
        y = y + st["residual"].float()
    return dict(y=y.to(DTYPES[case["y"]]))


# ----------------------------------------------------------------------- work

def work(case):
    if case["op"] == "layernorm":
        n, xb = case["rows"] * case["dim"], SIZE[case["x"]]
        yb = 2 if case["y"] == "e4m3" else SIZE[case["y"]]  # returned as 16-bit values
        return dict(bytes=n * (xb + yb + (2 * xb if case["residual"] else 0))
                    + case["dim"] * xb * (1 + case["bias"])
                    + (8 * case["rows"] if case["train"] else 0), flops=9 * n)
    if case["op"] == "layernorm_back":
        n, xb = case["rows"] * case["dim"], SIZE[case["x"]]
        return dict(bytes=n * (SIZE[case["y"]] + 2 * xb + (xb if case["residual"] else 0))
                    + (2 + case["bias"]) * case["dim"] * xb + 8 * case["rows"], flops=13 * n)
    if case["op"] == "block_quantize":
        n = case["rows"] * case["dim"]
        scales = -(-case["rows"] // case["block_rows"]) * _blocks(case["dim"])
        return dict(bytes=n * (SIZE[case["x"]] + 2) + 4 * scales, flops=4 * n)
    m, n, k = case["m"], case["n"], case["k"]
    if case["op"] == "gated":
        xb, yb = SIZE[case["x"]], SIZE[case["y"]]
        return dict(bytes=(m + 2 * n) * k * xb + m * n * yb * (3 if case["pre"] else 1)
                    + 2 * n * yb * case["bias"], flops=4 * m * n * k)
    if case["op"] == "gated_back":
        xb = SIZE[case["x"]]
        return dict(bytes=2 * (m + 2 * n) * k * xb + 3 * m * n * xb + 2 * n * xb * case["bias"],
                    flops=8 * m * n * k)
    yb = SIZE[case["y"]]
    return dict(bytes=(m + n) * k + 4 * (m + _blocks(n)) * _blocks(k)
                + m * n * yb * (1 + case["residual"]) + n * yb * case["bias"], flops=2 * m * n * k)


# ---------------------------------------------------------------------- exact

def _e4m3_64(a):
    """Magnitudes a (64 bits) on the e4m3 grid, to nearest, ties to even."""
    e = torch.floor(torch.log2(a.clamp_min(1e-300))).clamp_min(-6.0)
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=a.device), e - 3)
    return (torch.round(a / step) * step).clamp_max(TOP)


def _blocks_of(x, block_rows):
    """x's values, zeros behind them, as (row block, row, column block, column)."""
    rows, dim = x.shape
    x = torch.nn.functional.pad(x, (0, -dim % BLOCK, 0, -rows % block_rows))
    return x.unflatten(1, (-1, BLOCK)).unflatten(0, (-1, block_rows))


def _whole(blocks, rows, dim):
    return blocks.flatten(2, 3).flatten(0, 1)[:rows, :dim]


def exact(case, seed):
    st = prepare(case, seed)
    d = {key: t.double() for key, t in st.items() if isinstance(t, torch.Tensor)}

    def cdf(z):
        return 0.5 * torch.special.erfc(-z / math.sqrt(2.0))

    def act(z):
        return dict(none=lambda: z, relu=lambda: z.clamp_min(0), gelu=lambda: z * cdf(z),
                    silu=lambda: z * torch.sigmoid(z))[case["act"]]()

    if case["op"] == "layernorm":
        s = d["x"] + d["residual"] if case["residual"] else d["x"]
        mean = s.sum(1) / case["dim"]
        var = (s - mean[:, None]).pow(2).sum(1) / case["dim"]
        rstd = (var + EPS).pow(-0.5)
        y = torch.einsum("rd,r,d->rd", s - mean[:, None], rstd, d["weight"])
        if case["bias"]:
            y += d["bias"]
        if case["y"] == "e4m3":
            top = y.abs().max(1).values[:, None]
            unit = torch.where(top > 0, top / TOP, torch.ones_like(top))
            y = torch.sign(y) * _e4m3_64(y.abs() / unit) * unit
        return dict(y=y, s=s if case["residual"] else None, mean=mean if case["train"] else None,
                    rstd=rstd if case["train"] else None)
    if case["op"] == "layernorm_back":
        n = (d["s"] - d["mean"][:, None]) * d["rstd"][:, None]
        a = d["dy"] * d["weight"]
        shift = a.sum(1) / case["dim"]
        dot = torch.einsum("rd,rd->r", a, n) / case["dim"]
        dx = (a - shift[:, None] - n * dot[:, None]) * d["rstd"][:, None]
        if case["residual"]:
            dx += d["dsum"]
        return dict(dx=dx, dw=torch.einsum("rd,rd->d", d["dy"], n),
                    db=d["dy"].sum(0) if case["bias"] else None)
    if case["op"] == "gated":
        x, w = d["x"], d["w"]
        if case["x"] == "e4m3":
            x, w = x * d["x_scale"][:, None], w * d["w_scale"][:, None]
        z = torch.einsum("mk,nk->mn", x, w)
        if case["bias"]:
            z += d["bias"]
        gate, up = z.split(case["n"], 1)
        return dict(y=act(gate) * up, pre=z if case["pre"] else None)
    if case["op"] == "gated_back":
        z, up = d["pre"].split(case["n"], 1)
        slope = dict(none=lambda: torch.ones_like(z), relu=lambda: (z > 0).double(),
                     gelu=lambda: cdf(z) + z * torch.exp(-z * z / 2) * (2 * math.pi) ** -0.5,
                     silu=lambda: torch.sigmoid(z) * (1 + z * torch.sigmoid(-z)))[case["act"]]()
        dz = torch.stack([up * slope, act(z)], 1).mul_(d["dy"][:, None]).flatten(1)
        return dict(dx=torch.einsum("mn,nk->mk", dz, d["w"]),
                    dw=torch.einsum("mn,mk->nk", dz, d["x"]),
                    db=dz.sum(0) if case["bias"] else None)
    if case["op"] == "block_quantize":
        x = _blocks_of(d["x"], case["block_rows"])
        top = x.abs().amax((1, 3))
        unit = torch.where(top > 0, top / TOP, torch.ones_like(top))[:, None, :, None]
        values = torch.sign(x) * _e4m3_64(x.abs() / unit) * unit
        return dict(values=_whole(values, case["rows"], case["dim"]), scale=top / TOP)
    m, n, k = case["m"], case["n"], case["k"]
    x = _whole(_blocks_of(d["x"], 1) * d["x_scale"][:, None, :, None], m, k)
    w = _whole(_blocks_of(d["w"], BLOCK) * d["w_scale"][:, None, :, None], n, k)
    z = torch.einsum("mk,nk->mn", x, w)
    if case["bias"]:
        z += d["bias"]
    y = act(z)
    if case["residual"]:
        y = y + d["residual"]
    return dict(y=y)
