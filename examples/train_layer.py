"""Trains one residual layer that mixes rows by a sparse matrix, and serves it in 8 bits.

    s = x + A x                       sparse product and residual, FP32
    y = s + W2 gelu(W1 norm(s) + b1) + b2    dense products on 16-bit rows

A training step runs the sparse product (Plan; its gradient is the product of A's
transpose), the norm that adds the residual and makes the rows 16-bit (rmsnorm),
the two products with their epilogues (linear), their gradients, and AdamW with
8-bit states on FP32 weights that keeps the products' 16-bit copies.  The trained
layer then answers with 8-bit rows and weights.

    python examples/train_layer.py [--rows 6000] [--width 128] [--steps 30]
"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "vcsr-spmm_b200"))
import vcsr_b200 as V  # noqa: E402
from vcsr_b200 import layers, torch_ops  # noqa: E402


def transpose(csr):
    rows = np.repeat(np.arange(csr.M, dtype=np.int32), np.diff(csr.row_ptr))
    order = np.argsort(csr.col, kind="stable")
    ptr = np.concatenate([[0], np.cumsum(np.bincount(csr.col, minlength=csr.N))])
    return V.CSR(csr.N, csr.M, csr.nnz, ptr.astype(np.int32), rows[order], csr.val[order])


class Mix(torch.autograd.Function):
    """A x with the gradient A^T dy, both on plans."""

    @staticmethod
    def forward(ctx, x, plan, plan_t):
        ctx.plan_t = plan_t
        return plan.spmm(x, torch.empty(plan.M, x.shape[1], device=x.device))

    @staticmethod
    def backward(ctx, dy):
        dy = dy.contiguous()
        out = torch.empty(ctx.plan_t.M, dy.shape[1], device=dy.device)
        return ctx.plan_t.spmm(dy, out), None, None


def codes_of(w):
    """8-bit rows of a weight matrix and their scales, laid out once."""
    scale = w.abs().amax(1).clamp_min(1e-12) / 448
    return (w / scale[:, None]).to(torch.float8_e4m3fn), scale


def main(rows=6000, width=128, steps=30, seed=0, verbose=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device="cuda") * scale

    csr = V.gen_csr("fem", seed, rows)
    sums = np.add.reduceat(np.abs(csr.val), csr.row_ptr[:-1])
    csr.val = csr.val / np.repeat(sums, np.diff(csr.row_ptr)).astype(np.float32)
    plan, plan_t = V.Plan(csr, target_O=width), V.Plan(transpose(csr), target_O=width)

    # FP32 weights and the 16-bit copies that the products read
    master = [randn(2 * width, width, scale=width ** -0.5), torch.zeros(2 * width, device="cuda"),
              randn(width, 2 * width, scale=(2 * width) ** -0.5), torch.zeros(width, device="cuda")]
    copies = [t.to(torch.bfloat16).requires_grad_() for t in master]
    w1, b1, w2, b2 = copies
    gain = torch.ones(width, device="cuda", requires_grad=True)
    weights = layers.AdamW(master, lr=3e-3, state_bits=8, copies=[t.detach() for t in copies])
    gains = layers.AdamW([gain.detach()], lr=3e-3, weight_decay=0.0)

    x = randn(csr.N, width)
    target = torch.tanh(randn(csr.M, width) * 0.1 + x.roll(1, 1)) + x

    def layer(x):
        y, s = torch_ops.rmsnorm(Mix.apply(x, plan, plan_t), gain, residual=x,
                                 out_dtype=torch.bfloat16)
        h = torch_ops.linear(y, w1, bias=b1, act="gelu")
        return s + torch_ops.linear(h, w2, bias=b2).float()

    losses = []
    for step in range(steps):
        loss = (layer(x) - target).square().mean()
        for t in copies + [gain]:
            t.grad = None
        loss.backward()
        weights.step([t.grad for t in copies],
                     dither=torch.rand(layers.BLOCK, generator=gen, device="cuda"))
        gains.step([gain.grad])
        losses.append(loss.detach())
    losses = [float(v) for v in losses]
    layers.check()

    # 8-bit rows and weights: the norm writes the first product's operand
    with torch.no_grad():
        want = layer(x)
        (q1, k1), (q2, k2) = codes_of(master[0]), codes_of(master[2])
        n = layers.rmsnorm(Mix.apply(x, plan, plan_t), gain, residual=x,
                           out_dtype=torch.float8_e4m3fn)
        h = layers.linear(n.y, q1, bias=b1, act="gelu", x_scale=n.scale, w_scale=k1)
        ones = torch.ones(2 * width, device="cuda")
        g = layers.rmsnorm(h.y, ones, out_dtype=torch.float8_e4m3fn, save_rstd=True)
        # the second operand's scale without the norm it was made by
        got = n.sum + layers.linear(g.y, q2, bias=b2, x_scale=g.scale / g.rstd, w_scale=k2,
                                    out_dtype=torch.bfloat16).y.float()
        off = float((got - want).norm() / want.norm())
    if verbose:
        print(f"rows {csr.M}, width {width}: loss {losses[0]:.4f} -> {losses[-1]:.4f} in {steps} "
              f"steps; 8-bit answer {off:.4f} off the 16-bit one")
    return losses, off


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--rows", type=int, default=6000)
    ap.add_argument("--width", type=int, default=128)
    ap.add_argument("--steps", type=int, default=30)
    args = ap.parse_args()
    main(args.rows, args.width, args.steps)
