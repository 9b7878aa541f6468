"""One gated MLP layer with 2:4 weights: trained in 16 bits, served in 8.

Training keeps the weights dense and re-prunes them after every step
(ffn_gated and its backward pass; the pruned weights' gradient is dense, so a
pruned value can come back).  Serving compresses the pruned weights, quantises
the kept values with one scale per output channel, and runs the layer in four
launches a call:

    rmsnorm_quant   residual + norm -> 8-bit rows, a scale per token
    gemm_scaled     gate and up projections, stacked, in one 2:4 product
    swiglu_quant    silu(gate) * up -> 8-bit rows
    gemm_scaled     down projection, 16-bit rows for the next residual

    python examples/mlp_block.py [--qdtype int8|e4m3] [--tokens N]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "sparse-gemm-with-hopper-sptc_b200"))
import sp24  # noqa: E402


class ServedLinear:
    """8-bit 2:4 weights of one projection, laid out once."""

    def __init__(self, pruned, qdtype):
        m, k = pruned.shape
        a_c, meta = sp24.compress(pruned)                        # 16-bit kept values + codes
        self.a_c, self.scale = sp24.quantize_rows(a_c, qdtype=qdtype)
        self.meta = sp24.repack_meta(meta, m, k, qdtype)

    def __call__(self, q, scale):
        return sp24.gemm_scaled(self.a_c, self.meta, q, self.scale, scale)


class ServedMlp:
    def __init__(self, norm, w_gate, w_up, w_down, qdtype):
        self.norm, self.qdtype, self.f = norm, qdtype, w_gate.shape[0]
        self.gate_up = ServedLinear(torch.cat((w_gate, w_up)), qdtype)
        self.down = ServedLinear(w_down, qdtype)

    def __call__(self, x, residual):
        """(layer output, residual stream for the next layer)."""
        q, scale, residual = sp24.rmsnorm_quant(x, self.norm, residual, qdtype=self.qdtype)
        y = self.gate_up(q, scale)
        q, scale = sp24.swiglu_quant(y[:, :self.f], y[:, self.f:], qdtype=self.qdtype)
        return self.down(q, scale), residual


def train_step(x, target, w_gate, w_up, lr):
    """One step of 0.5 |h - target|^2 / tokens; the weights stay 2:4."""
    h, saved = sp24.ffn_gated(x, w_gate, w_up, save=True)
    diff = h.float() - target.float()
    d_h = (diff / x.shape[0]).to(x.dtype)
    _, d_gate, d_up = sp24.ffn_gated_backward(d_h, x, w_gate, w_up, saved, need_dx=False)
    loss = 0.5 * diff.square().sum() / x.shape[0]
    new = [sp24.prune_2of4((w.float() - lr * d.float()).to(w.dtype))
           for w, d in ((w_gate, d_gate), (w_up, d_up))]
    return loss, new[0], new[1]


def reference_layer(x, residual, norm, w_gate, w_up, w_down, eps=1e-6):
    s = x.float() + residual.float()
    y = s * torch.rsqrt(s.square().mean(dim=1, keepdim=True) + eps) * norm.float()
    g = y @ w_gate.float().t()
    return (g * torch.sigmoid(g) * (y @ w_up.float().t())) @ w_down.float().t()


def run(tokens=512, hidden=1024, inter=2816, steps=8, qdtype=sp24.I8, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * std).to(torch.bfloat16)

    dense_gate, dense_up = (normal(inter, hidden, std=hidden ** -0.5) for _ in range(2))
    w_down = sp24.prune_2of4(normal(hidden, inter, std=inter ** -0.5))
    norm = normal(hidden, std=0.1) + 1
    # Recover the dense block's output with pruned weights.
    x = normal(tokens, hidden)
    target = sp24.ffn_gated(x, dense_gate, dense_up)
    w_gate, w_up = sp24.prune_2of4(dense_gate), sp24.prune_2of4(dense_up)
    losses = []
    for _ in range(steps):
        loss, w_gate, w_up = train_step(x, target, w_gate, w_up, lr=0.05)
        losses.append(loss.item())
    # Serve the trained layer: a prompt, then single tokens.
    mlp = ServedMlp(norm, w_gate, w_up, w_down, qdtype)
    errors = {}
    for name, t in (("prompt", tokens), ("token", 1)):
        x, residual = normal(t, hidden), normal(t, hidden, std=2.0)
        y, _ = mlp(x, residual)
        want = reference_layer(x, residual, norm, w_gate, w_up, w_down)
        errors[name] = ((y.float() - want).norm() / want.norm()).item()
    return losses, errors


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--qdtype", choices=("int8", "e4m3"), default="int8")
    ap.add_argument("--tokens", type=int, default=512)
    a = ap.parse_args()
    losses, errors = run(tokens=a.tokens, qdtype=sp24.I8 if a.qdtype == "int8" else sp24.E4M3)
    print("training loss:", " ".join(f"{v:.3f}" for v in losses))
    print("served in %s, error against fp32:" % a.qdtype, errors)
