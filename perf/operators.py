"""Benchmark cases of the dense layer operators: the norm (rmsnorm), the product
with its epilogue (linear) and the optimizer step (AdamW), forward and backward.

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
ADAM = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01)
STEP0 = 10      # steps done before the pass
BLOCK = 256     # values per scale of an 8-bit state
GRAD_SCALE = 0.5


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
        dict(name="norm_token", op="norm", rows=1, dim=4096, x="bf16", y="bf16", residual=True,
             train=False),
        # the FP32 result of the FEM product (62,451 rows, O = 128) made the 16-bit operand
        # of a dense product, rstd kept for the gradient
        dict(name="norm_fem", op="norm", rows=62451, dim=128, x="f32", y="bf16", residual=True,
             train=True),
        # the rows of a long prompt made 8-bit operands
        dict(name="norm_e4m3", op="norm", rows=16384, dim=4096, x="bf16", y="e4m3", residual=True,
             train=False),
        # the norm's gradient with the residual stream's own, odd row count
        dict(name="norm_back", op="norm_back", rows=8191, dim=5120, x="bf16", y="bf16",
             residual=True),
        # one token through a square layer: the weights are read once
        dict(name="linear_token", op="linear", m=1, n=4096, k=4096, x="bf16", y="bf16",
             act="silu", bias=True, residual=True, pre=False),
        # the rows of the FEM product through a layer of its width, in FP32, training
        dict(name="linear_fem", op="linear", m=62451, n=128, k=128, x="f32", y="f32",
             act="relu", bias=True, residual=True, pre=True),
        # the rows of a large training batch: the largest product
        dict(name="linear_large", op="linear", m=16384, n=8192, k=4096, x="bf16", y="bf16",
             act="gelu", bias=True, residual=True, pre=True),
        # a prompt's 8-bit rows against 8-bit weights
        dict(name="linear_e4m3", op="linear", m=4096, n=8192, k=4096, x="e4m3", y="bf16",
             act="gelu", bias=True, residual=False, pre=False),
        # the gradient of a training batch
        dict(name="linear_back", op="linear_back", m=8192, n=4096, k=4096, x="bf16",
             act="gelu", bias=True),
        # a small ragged layer: no size is a multiple of eight
        dict(name="linear_back_odd", op="linear_back", m=1001, n=777, k=1501, x="f16",
             act="silu", bias=True),
        # FP32 weights with a 16-bit copy for the products, states in 32 bits
        dict(name="adamw_32", op="adamw", tensors=290, largest=4194304, total=67108864, p="f32",
             g="bf16", bits=32, copy=True),
        # the same count of weights with 8-bit states and dithered rounding
        dict(name="adamw_8", op="adamw", tensors=290, largest=4194304, total=67108864, p="f32",
             g="f32", bits=8, copy=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm_back", "linear", "linear", "linear_back", "adamw"])
    if op in ("norm", "norm_back"):
        dim = _log(rng, 16, 16384)
        if rng.random() < 0.6:
            dim = max(8, dim // 8 * 8)
        rows = _log(rng, 1, max(1, min(65536, 16384 * 4096 // dim)))
        x = rng.choice(["f32", "bf16", "f16"])
        case = dict(op=op, rows=rows, dim=dim, x=x, residual=rng.random() < 0.7)
        if op == "norm":
            case["y"] = rng.choice(["f32", "bf16", "f16", "e4m3"])
            case["train"] = rng.random() < 0.5
        else:
            case["y"] = rng.choice(["f32", "bf16", "f16"])
        return case
    if op in ("linear", "linear_back"):
        n, k = _log(rng, 64, 8192), _log(rng, 64, 8192)
        if rng.random() < 0.6:
            n, k = max(16, n // 16 * 16), max(16, k // 16 * 16)
        m = _log(rng, 1, 16384)
        x = rng.choice(["bf16", "f16", "f32"] + (["e4m3"] if op == "linear" else []))
        if op == "linear_back":
            m = min(m, 8192)
        if x == "f32":
            m = min(m, 4096)
        case = dict(op=op, m=m, n=n, k=k, x=x, act=rng.choice(["none", "relu", "gelu", "silu"]),
                    bias=rng.random() < 0.7)
        if op == "linear":
            case.update(y=x if x != "e4m3" else rng.choice(["bf16", "f16", "f32"]),
                        residual=rng.random() < 0.5, pre=rng.random() < 0.5)
        return case
    tensors = _log(rng, 1, 400)
    largest = _log(rng, 64, 4194304)
    return dict(op="adamw", tensors=tensors, largest=largest,
                total=min(67108864, tensors * largest), p=rng.choice(["f32", "bf16", "f16"]),
                g=rng.choice(["f32", "bf16", "f16"]), bits=rng.choice([32, 8]),
                copy=rng.random() < 0.5)


def _numels(case):
    """Sizes of the tensors of an AdamW case: matrices near the largest size, biases and gains
    between them, odd ones among both, at most `total` values in all."""
    out, left = [], case["total"]
    for i in range(case["tensors"]):
        if i % 3 == 0:
            n = case["largest"] // (1 + (i // 3) % 4)
        else:
            n = max(1, int(math.sqrt(case["largest"])) * (1 + i % 2) - i % 7)
        n = max(1, min(n, left - (case["tensors"] - 1 - i)))
        out.append(n)
        left -= n
    return out


# --------------------------------------------------------------------- inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev = torch.device("cuda")

    def normal(*shape, scale=1.0, shift=0.0, dtype=torch.float32):
        t = torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32)
        return t.mul_(scale).add_(shift).to(dtype)

    st = dict(case=case)
    if case["op"] in ("norm", "norm_back"):
        xt, rows, dim = DTYPES[case["x"]], case["rows"], case["dim"]
        x = normal(rows, dim)
        x[:, :: max(1, dim // 7)] *= 8  # a few columns are larger, as activations have them
        st["weight"] = normal(dim, scale=0.1, shift=1.0, dtype=xt)
        if case["op"] == "norm":
            st["x"] = x.to(xt)
            st["residual"] = normal(rows, dim, dtype=xt) if case["residual"] else None
        else:
            st["s"] = x.to(xt)
            st["rstd"] = torch.rsqrt(st["s"].float().square().mean(1) + EPS)
            st["dy"] = normal(rows, dim, scale=1e-2, dtype=DTYPES[case["y"]])
            st["dsum"] = normal(rows, dim, scale=1e-2, dtype=xt) if case["residual"] else None
    elif case["op"] in ("linear", "linear_back"):
        xt, m, n, k = DTYPES[case["x"]], case["m"], case["n"], case["k"]
        yt = DTYPES[case.get("y", case["x"])]
        x, w = normal(m, k), normal(n, k, scale=k ** -0.5)
        if case["x"] == "e4m3":
            st["x_scale"] = x.abs().amax(1) / 448
            st["w_scale"] = w.abs().amax(1) / 448
            x, w = x / st["x_scale"][:, None], w / st["w_scale"][:, None]
        st["x"], st["w"] = x.to(xt), w.to(xt)
        st["bias"] = normal(n, scale=0.1, dtype=yt) if case["bias"] else None
        if case["op"] == "linear":
            st["residual"] = normal(m, n, dtype=yt) if case["residual"] else None
        else:
            st["dy"] = normal(m, n, scale=1e-2, dtype=xt)
            st["pre"] = normal(m, n, dtype=xt) if case["act"] != "none" else None
    else:
        numels = _numels(case)
        starts, at = [], 0
        for n in numels:
            starts.append(at)
            at += -(-n // BLOCK) * BLOCK
        inside = torch.zeros(at, device=dev, dtype=torch.bool)
        for a, n in zip(starts, numels):
            inside[a:a + n] = True
        pt, gt = DTYPES[case["p"]], DTYPES[case["g"]]

        def flat(scale):
            return normal(at, scale=scale).mul_(inside)

        st["p"] = flat(0.05).to(pt)
        st["g"] = flat(2e-3).to(gt)
        m, v = flat(3e-4), flat(1e-3).square_()
        views = [slice(a, a + n) for a, n in zip(starts, numels)]
        if case["bits"] == 8:
            m, u = m.view(-1, BLOCK), v.sqrt().view(-1, BLOCK)
            st["m_scale"], st["u_scale"] = m.abs().amax(1) / 448, u.amax(1) / 448
            st["m"] = (m / st["m_scale"].clamp_min(1e-30)[:, None]).to(torch.float8_e4m3fn)
            st["u"] = (u / st["u_scale"].clamp_min(1e-30)[:, None]).to(torch.float8_e4m3fn)
            st["dither"] = torch.rand(BLOCK, generator=gen, device=dev)
        else:
            st["m"], st["v"] = m, v
        st["copy"] = torch.zeros(at, device=dev, dtype=torch.bfloat16) if case["copy"] else None
        st["step"] = STEP0
        st["grads"] = [st["g"][s] for s in views]
        if own:
            opt = layers().AdamW([st["p"][s] for s in views], lr=ADAM["lr"],
                                 betas=(ADAM["beta1"], ADAM["beta2"]), eps=ADAM["eps"],
                                 weight_decay=ADAM["weight_decay"], state_bits=case["bits"],
                                 copies=[st["copy"][s] for s in views] if case["copy"] else None)
            opt.steps = STEP0
            if case["bits"] == 8:
                opt.m_flat.view(-1, BLOCK).copy_(st["m"])
                opt.u_flat.view(-1, BLOCK).copy_(st["u"])
                opt.m_scale.copy_(st["m_scale"])
                opt.u_scale.copy_(st["u_scale"])
            else:
                opt.m_flat.copy_(st["m"])
                opt.v_flat.copy_(st["v"])
            st["opt"] = opt
    return st


# ----------------------------------------------------------------------- runs

def run(st):
    return (run_own if own else run_plain)(st)


def run_own(st):
    case, L = st["case"], layers()
    if case["op"] == "norm":
        out = L.rmsnorm(st["x"], st["weight"], residual=st["residual"], eps=EPS,
                        out_dtype=DTYPES[case["y"]], save_rstd=case["train"])
        y = out.y
        if case["y"] == "e4m3":
            y = L.dequantize(y, out.scale, torch.bfloat16)
        return dict(y=y, s=out.sum if case["residual"] else None,
                    rstd=out.rstd if case["train"] else None)
    if case["op"] == "norm_back":
        dx, dw = L.rmsnorm_backward(st["dy"], st["s"], st["weight"], st["rstd"], dsum=st["dsum"])
        return dict(dx=dx, dw=dw)
    if case["op"] == "linear":
        out = L.linear(st["x"], st["w"], bias=st["bias"], residual=st["residual"], act=case["act"],
                       x_scale=st.get("x_scale"), w_scale=st.get("w_scale"),
                       out_dtype=DTYPES[case["y"]], save_pre=case["pre"])
        return dict(y=out.y, pre=out.pre)
    if case["op"] == "linear_back":
        g = L.linear_backward(st["dy"], st["x"], st["w"], pre=st["pre"], act=case["act"],
                              need_db=case["bias"])
        return dict(dx=g.dx, dw=g.dw, db=g.db)
    opt = st["opt"]
    opt.step(st["grads"], grad_scale=GRAD_SCALE, dither=st.get("dither"))
    if case["bits"] == 8:
        m, v = opt.state_values(torch.bfloat16)
    else:
        m, v = opt.m_flat, opt.v_flat
    return dict(p=st["p"], m=m, v=v, copy=st["copy"])


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
    sig = 1 / (1 + torch.exp(-z))
    return sig * (1 + z * (1 - sig))


def _dither8(x, dither):
    """x / scale rounded to e4m3 up or down as `dither` says, and the scales: rows of BLOCK."""
    scale = x.abs().amax(1, keepdim=True) / 448
    a = x.abs() / torch.where(scale > 0, scale, torch.ones_like(scale))
    _, e = torch.frexp(a)
    step = torch.exp2((e - 1).clamp_min(-6).float() - 3)
    q = (torch.floor(a / step + dither) * step).clamp_max(448)
    return torch.where(x < 0, -q, q), scale


def run_plain(st):
    case = st["case"]
    if case["op"] == "norm":
        s = st["x"].float()
        if case["residual"]:
            s = s + st["residual"].float()
        rstd = 1 / torch.sqrt((s * s).mean(1) + EPS)
        y = s * rstd[:, None] * st["weight"].float()
        if case["y"] == "e4m3":
            scale = y.abs().amax(1, keepdim=True) / 448
            q = (y / torch.where(scale > 0, scale, torch.ones_like(scale))).to(DTYPES["e4m3"])
            y = (q.float() * scale).to(torch.bfloat16)
        else:
            y = y.to(DTYPES[case["y"]])
        return dict(y=y, s=s.to(DTYPES[case["x"]]) if case["residual"] else None,
                    rstd=rstd if case["train"] else None)
    if case["op"] == "norm_back":
        rstd = st["rstd"][:, None]
        xh, dy = st["s"].float() * rstd, st["dy"].float()
        g = dy * st["weight"].float()
        dx = rstd * (g - xh * (g * xh).mean(1, keepdim=True))
        if case["residual"]:
            dx = dx + st["dsum"].float()
        return dict(dx=dx.to(st["s"].dtype), dw=(dy * xh).sum(0).to(st["weight"].dtype))
    if case["op"] == "linear":
        z = st["x"].float() @ st["w"].float().t()
        if case["x"] == "e4m3":
            z = z * st["x_scale"][:, None] * st["w_scale"]
        if case["bias"]:
            z = z + st["bias"].float()
        y = _act(z, case["act"])
        if case["residual"]:
            y = y + st["residual"].float()
        yt = DTYPES[case["y"]]
        return dict(y=y.to(yt), pre=z.to(yt) if case["pre"] else None)
    if case["op"] == "linear_back":
        dz, xt = st["dy"].float(), st["x"].dtype
        if case["act"] != "none":
            dz = dz * _act_grad(st["pre"].float(), case["act"])
        return dict(dx=(dz @ st["w"].float()).to(xt), dw=(dz.t() @ st["x"].float()).to(xt),
                    db=dz.sum(0).to(xt) if case["bias"] else None)
    st["step"] += 1
    c1, c2 = 1 - ADAM["beta1"] ** st["step"], 1 - ADAM["beta2"] ** st["step"]
    g, p = st["g"].float() * GRAD_SCALE, st["p"].float()
    if case["bits"] == 8:
        m = (st["m"].float() * st["m_scale"][:, None]).view(-1)
        v = (st["u"].float() * st["u_scale"][:, None]).square().view(-1)
    else:
        m, v = st["m"], st["v"]
    m = ADAM["beta1"] * m + (1 - ADAM["beta1"]) * g
    v = ADAM["beta2"] * v + (1 - ADAM["beta2"]) * g * g
    p = (p * (1 - ADAM["lr"] * ADAM["weight_decay"])
         - ADAM["lr"] * (m / c1) / (torch.sqrt(v / c2) + ADAM["eps"]))
    st["p"].copy_(p)
    if case["copy"]:
        st["copy"].copy_(p)
    if case["bits"] == 8:
        mq, ms = _dither8(m.view(-1, BLOCK), st["dither"])
        u = torch.sqrt(v).view(-1, BLOCK)
        uq, us = _dither8(u, st["dither"])
        uq = torch.where((u > 0) & (uq == 0), torch.full_like(uq, 2.0 ** -9), uq)
        st["m"].copy_(mq)
        st["u"].copy_(uq)
        st["m_scale"].copy_(ms[:, 0])
        st["u_scale"].copy_(us[:, 0])
        m = (mq * ms).to(torch.bfloat16).view(-1)
        v = (uq * us).square().to(torch.bfloat16).view(-1)
    else:
        st["m"].copy_(m)
        st["v"].copy_(v)
        m, v = st["m"], st["v"]
    return dict(p=st["p"], m=m, v=v, copy=st["copy"])


# ----------------------------------------------------------------------- work

def work(case):
    if case["op"] == "norm":
        n, xb = case["rows"] * case["dim"], SIZE[case["x"]]
        yb = 2 if case["y"] == "e4m3" else SIZE[case["y"]]  # returned as 16-bit values
        return dict(bytes=n * (xb + yb + (2 * xb if case["residual"] else 0)) + case["dim"] * xb
                    + (4 * case["rows"] if case["train"] else 0), flops=6 * n)
    if case["op"] == "norm_back":
        n, xb = case["rows"] * case["dim"], SIZE[case["x"]]
        return dict(bytes=n * (SIZE[case["y"]] + 2 * xb + (xb if case["residual"] else 0))
                    + 2 * case["dim"] * xb + 4 * case["rows"], flops=10 * n)
    if case["op"] in ("linear", "linear_back"):
        m, n, k, xb = case["m"], case["n"], case["k"], SIZE[case["x"]]
        if case["op"] == "linear":
            yb = SIZE[case["y"]]
            return dict(bytes=(m + n) * k * xb + m * n * yb * (1 + case["residual"] + case["pre"])
                        + n * yb * case["bias"], flops=2 * m * n * k)
        return dict(bytes=2 * (m + n) * k * xb + m * n * xb * (1 + (case["act"] != "none"))
                    + n * xb * case["bias"], flops=4 * m * n * k)
    n = sum(_numels(case))
    state = 16 if case["bits"] == 32 else 4
    return dict(bytes=n * (2 * SIZE[case["p"]] + SIZE[case["g"]] + state
                           + (2 if case["copy"] else 0)), flops=15 * n)


# ---------------------------------------------------------------------- exact

def _e4m3_64(a, dither=None):
    """Magnitudes a (64 bits) on the e4m3 grid: to nearest, ties to even, or as dither says."""
    e = torch.floor(torch.log2(a.clamp_min(1e-300))).clamp_min(-6.0)
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=a.device), e - 3)
    k = a / step
    k = torch.round(k) if dither is None else torch.floor(k + dither)
    return (k * step).clamp_max(448.0)


def exact(case, seed):
    st = prepare(case, seed)
    d = {key: t.double() for key, t in st.items() if isinstance(t, torch.Tensor)}
    if case["op"] == "norm":
        s = d["x"] + d["residual"] if case["residual"] else d["x"]
        rstd = (s.pow(2).sum(1) / case["dim"] + EPS).pow(-0.5)
        y = torch.einsum("rd,r,d->rd", s, rstd, d["weight"])
        if case["y"] == "e4m3":
            top = y.abs().max(1).values[:, None]
            unit = torch.where(top > 0, top / 448, torch.ones_like(top))
            y = torch.sign(y) * _e4m3_64(y.abs() / unit) * unit
        return dict(y=y, s=s if case["residual"] else None, rstd=rstd if case["train"] else None)
    if case["op"] == "norm_back":
        n = d["s"] * d["rstd"][:, None]
        a = d["dy"] * d["weight"]
        dot = torch.einsum("rd,rd->r", a, n) / case["dim"]
        dx = (a - n * dot[:, None]) * d["rstd"][:, None]
        if case["residual"]:
            dx += d["dsum"]
        return dict(dx=dx, dw=torch.einsum("rd,rd->d", d["dy"], n))
    if case["op"] in ("linear", "linear_back"):
        def cdf(z):
            return 0.5 * torch.special.erfc(-z / math.sqrt(2.0))

        if case["op"] == "linear":
            x, w = d["x"], d["w"]
            if case["x"] == "e4m3":
                x, w = x * d["x_scale"][:, None], w * d["w_scale"][:, None]
            z = torch.einsum("mk,nk->mn", x, w)
            if case["bias"]:
                z += d["bias"]
            y = dict(none=lambda: z, relu=lambda: z.clamp_min(0), gelu=lambda: z * cdf(z),
                     silu=lambda: z * torch.sigmoid(z))[case["act"]]()
            if case["residual"]:
                y = y + d["residual"]
            return dict(y=y, pre=z if case["pre"] else None)
        dz = d["dy"]
        if case["act"] != "none":
            z = d["pre"]
            slope = dict(relu=lambda: (z > 0).double(),
                         gelu=lambda: cdf(z) + z * torch.exp(-z * z / 2) * (2 * math.pi) ** -0.5,
                         silu=lambda: torch.sigmoid(z) * (1 + z * torch.sigmoid(-z)))
            dz = dz * slope[case["act"]]()
        return dict(dx=torch.einsum("mn,nk->mk", dz, d["w"]),
                    dw=torch.einsum("mn,mk->nk", dz, d["x"]),
                    db=dz.sum(0) if case["bias"] else None)
    t, b1, b2 = STEP0 + 1, ADAM["beta1"], ADAM["beta2"]
    g = d["g"] * GRAD_SCALE
    if case["bits"] == 8:
        m = (d["m"] * d["m_scale"][:, None]).flatten()
        v = (d["u"] * d["u_scale"][:, None]).pow(2).flatten()
    else:
        m, v = d["m"], d["v"]
    m = torch.lerp(g, m, b1)
    v = torch.lerp(g.pow(2), v, b2)
    rate = ADAM["lr"] * math.sqrt(1 - b2 ** t) / (1 - b1 ** t)
    p = d["p"] - ADAM["lr"] * ADAM["weight_decay"] * d["p"] \
        - rate * m / (v.sqrt() + ADAM["eps"] * math.sqrt(1 - b2 ** t))
    copy = p if case["copy"] else None
    if case["bits"] == 8:
        def stored(x, floor):
            x = x.view(-1, BLOCK)
            unit = x.abs().max(1).values[:, None] / 448
            q = _e4m3_64(x.abs() / torch.where(unit > 0, unit, torch.ones_like(unit)), d["dither"])
            if floor:
                q = torch.where((x > 0) & (q == 0), torch.full_like(q, 2.0 ** -9), q)
            return (torch.sign(x) * q * unit).flatten()

        m, v = stored(m, False), stored(v.sqrt(), True).pow(2)
    return dict(p=p, m=m, v=v, copy=copy)
