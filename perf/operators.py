"""Cases of the MLP-block operators: what each one computes, in plain torch
operations, and the framework's call for the same thing.

  norm    rmsnorm_quant   residual addition, root-mean-square norm, 8-bit rows
                          with one scale per token
  swiglu  swiglu_quant    silu(gate) * up, 8-bit rows with one scale per token
  prod    gemm_scaled     8-bit product of tokens with 2:4 weights, scales for
                          each token and each channel
  ffn     ffn_gated       silu(x Wg^T) * (x Wu^T) in one kernel; with
                          "train" also its backward pass

Sizes: hidden 4096, intermediate 14336 (the MLP layer of this repository's
benchmark), and generic ragged ones.  Activations are token-major.
"""
import os
import sys

import torch

own = False

HIDDEN, INTER = 4096, 14336
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
QMAX = {"i8": 127.0, "e4m3": 448.0}
EPS = 1e-6


def listed():
    return [
        # decoding: the norm before a layer's first product, one token
        {"name": "norm 1 token", "op": "norm", "t": 1, "h": HIDDEN, "dtype": "bf16", "q": "e4m3"},
        # a short prompt through a narrower model, int8 rows
        {"name": "norm ragged int8", "op": "norm", "t": 333, "h": 5000, "dtype": "f16", "q": "i8"},
        # a full prompt chunk
        {"name": "norm 8192 tokens", "op": "norm", "t": 8192, "h": HIDDEN, "dtype": "bf16", "q": "e4m3"},
        # between the two halves of a quantised MLP
        {"name": "swiglu 4096 tokens", "op": "swiglu", "t": 4096, "h": INTER, "dtype": "bf16", "q": "e4m3"},
        # decoding: one token through the up projection; bound by the weights
        {"name": "prod 1 token", "op": "prod", "t": 1, "m": INTER, "k": HIDDEN, "q": "i8", "out": "bf16", "bias": False},
        # a small batch of decoding sequences through the down projection
        {"name": "prod 32 tokens e4m3", "op": "prod", "t": 32, "m": HIDDEN, "k": INTER, "q": "e4m3", "out": "bf16", "bias": False},
        # a short prompt, odd sizes everywhere, with a bias
        {"name": "prod ragged", "op": "prod", "t": 333, "m": 5003, "k": 4160, "q": "i8", "out": "f16", "bias": True},
        # a prompt chunk through the up projection; bound by the tensor cores
        {"name": "prod 4096 tokens", "op": "prod", "t": 4096, "m": INTER, "k": HIDDEN, "q": "i8", "out": "bf16", "bias": False},
        # decoding without quantisation
        {"name": "ffn 1 token", "op": "ffn", "t": 1, "h": HIDDEN, "f": INTER, "dtype": "bf16", "train": False},
        # a prompt chunk
        {"name": "ffn 4096 tokens", "op": "ffn", "t": 4096, "h": HIDDEN, "f": INTER, "dtype": "bf16", "train": False},
        # fine-tuning a small model on a ragged batch
        {"name": "ffn train ragged", "op": "ffn", "t": 777, "h": 1000, "f": 2744, "dtype": "f16", "train": True},
        # fine-tuning: forward and backward of the layer
        {"name": "ffn train 4096 tokens", "op": "ffn", "t": 4096, "h": HIDDEN, "f": INTER, "dtype": "bf16", "train": True},
    ]


def draw(rng):
    def log(lo, hi, unit=1):
        n = unit * min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))
        return n + unit if n == 3 << 10 else n

    op = rng.choice(["norm", "swiglu", "prod", "prod", "ffn", "ffn"])
    if op in ("norm", "swiglu"):
        return {"op": op, "t": log(1, 8192), "h": log(64, 4096 if op == "norm" else 14336),
                "dtype": rng.choice(["bf16", "f16"]), "q": rng.choice(["i8", "e4m3"])}
    if op == "prod":
        return {"op": op, "t": log(1, 4096), "m": log(64, 14336), "k": log(1, 64, 64),
                "q": rng.choice(["i8", "e4m3"]), "out": rng.choice(["bf16", "f16", "f32"]), "bias": rng.random() < 0.5}
    # widths are whole 16-byte rows of 16-bit values; the token count is any
    return {"op": op, "t": log(1, 4096), "h": log(8, 512, 8), "f": log(8, 1792, 8),
            "dtype": rng.choice(["bf16", "f16"]), "train": rng.random() < 0.5}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=g) * std

    op, t = case["op"], case["t"]
    if op == "norm":
        d = DTYPES[case["dtype"]]
        return {**case, "x": normal(t, case["h"]).to(d), "residual": normal(t, case["h"], std=3.0).to(d),
                "weight": (1.0 + normal(case["h"], std=0.1)).to(d)}
    if op == "swiglu":
        d = DTYPES[case["dtype"]]
        gate_up = normal(t, 2 * case["h"], std=1.3).to(d)   # the output of a stacked gate and up projection
        return {**case, "gate": gate_up[:, :case["h"]], "up": gate_up[:, case["h"]:]}
    if op == "prod":
        m, k, q = case["m"], case["k"], case["q"]
        x, sx = _rows_to_8_bits(normal(t, k), q)
        # magnitude-pruned 2:4 weights: the two largest of every four along k
        w = normal(m, k // 4, 4, std=0.02)
        at = w.abs().topk(2, dim=2).indices.sort(dim=2).values
        a_c, sw = _rows_to_8_bits(w.gather(2, at).reshape(m, k // 2), q)
        code = (at[:, :, 0] | at[:, :, 1] << 2).to(torch.uint8)
        meta = code[:, 0::2] | code[:, 1::2] << 4            # m x k/8 bytes, the row-major nibble layout
        return {**case, "x": x, "scale_x": sx, "a_c": a_c, "scale_w": sw, "meta": meta, "image": _tensor_core_image(meta, m, k),
                "bias_w": normal(m) if case["bias"] else None}
    d, h, f = DTYPES[case["dtype"]], case["h"], case["f"]
    return {**case, "x": normal(t, h).to(d), "w_gate": normal(f, h, std=0.02).to(d), "w_up": normal(f, h, std=0.02).to(d),
            "dh": normal(t, f, std=0.1).to(d) if case["train"] else None}


def _rows_to_8_bits(v, q):
    scale = v.abs().amax(dim=1) / QMAX[q]
    v = v / scale[:, None]
    return (v.round().to(torch.int8) if q == "i8" else v.to(torch.float8_e4m3fn)), scale


def _tensor_core_image(meta, m, k):
    """The metadata as the framework's products take it: for every 128 of k and
    every 128 rows, each row's 16 bytes in turn; an even number of row blocks,
    padded with the valid code 4."""
    blocks, atoms = (m + 255) // 256 * 2, (k + 127) // 128
    image = torch.full((blocks * 128, atoms * 16), 0x44, dtype=torch.uint8, device=meta.device)
    image[:m, :k // 8] = meta
    return image.reshape(blocks, 128, atoms, 16).permute(2, 0, 1, 3).contiguous().reshape(-1)


def run(state):
    return (_own if own else _plain)(state)


def _plain(s):
    if s["op"] == "norm":
        total = s["x"].float() + s["residual"].float()
        y = total * torch.rsqrt(total.square().mean(dim=1, keepdim=True) + EPS) * s["weight"].float()
        return {**_plain_quantised(y, s), "residual": total.to(s["x"].dtype)}
    if s["op"] == "swiglu":
        gate = s["gate"].float()
        return _plain_quantised(gate / (1 + torch.exp(-gate)) * s["up"].float(), s)
    if s["op"] == "prod":
        m, k = s["m"], s["k"]
        code = torch.stack((s["meta"] & 15, s["meta"] >> 4), dim=2).reshape(m, k // 4)
        at = torch.stack((code & 3, code >> 2), dim=2).long()
        w = torch.zeros(m, k // 4, 4, device="cuda").scatter_(2, at, s["a_c"].float().reshape(m, k // 4, 2))
        y = (s["x"].float() @ w.reshape(m, k).t()) * s["scale_x"][:, None] * s["scale_w"]
        return (y if s["bias_w"] is None else y + s["bias_w"]).to(DTYPES[s["out"]])
    x, w_gate, w_up, d = s["x"].float(), s["w_gate"].float(), s["w_up"].float(), s["x"].dtype
    gate, up = x @ w_gate.t(), x @ w_up.t()
    sig = 1 / (1 + torch.exp(-gate))
    h = gate * sig * up
    if not s["train"]:
        return h.to(d)
    dh = s["dh"].float()
    d_gate = dh * up * sig * (1 + gate * (1 - sig))
    d_up = dh * gate * sig
    return {"h": h.to(d), "dx": (d_gate @ w_gate + d_up @ w_up).to(d), "dw_gate": (d_gate.t() @ x).to(d), "dw_up": (d_up.t() @ x).to(d)}


def _plain_quantised(y, s):
    amax = y.abs().amax(dim=1)
    q = y * (QMAX[s["q"]] / amax)[:, None]
    return {"q": q.round().to(s["x" if "x" in s else "gate"].dtype) if s["q"] == "i8" else q.to(torch.float8_e4m3fn),
            "scale": amax / QMAX[s["q"]]}


def _own(s):
    sp24 = _framework()
    if s["op"] in ("norm", "swiglu"):
        code = sp24.I8 if s["q"] == "i8" else sp24.E4M3
        if s["op"] == "norm":
            q, scale, residual = sp24.rmsnorm_quant(s["x"], s["weight"], residual=s["residual"], eps=EPS, qdtype=code)
        else:
            q, scale = sp24.swiglu_quant(s["gate"], s["up"], qdtype=code)
        if s["q"] == "i8":
            q = q.to(s["x" if "x" in s else "gate"].dtype)   # the whole numbers that the bytes stand for
        return {"q": q, "scale": scale, "residual": residual} if s["op"] == "norm" else {"q": q, "scale": scale}
    if s["op"] == "prod":
        return sp24.gemm_scaled(s["a_c"], s["image"], s["x"], s["scale_w"], s["scale_x"], bias=s["bias_w"], out_dtype=DTYPES[s["out"]])
    if not s["train"]:
        return sp24.ffn_gated(s["x"], s["w_gate"], s["w_up"])
    h, saved = sp24.ffn_gated(s["x"], s["w_gate"], s["w_up"], save=True)
    dx, dw_gate, dw_up = sp24.ffn_gated_backward(s["dh"], s["x"], s["w_gate"], s["w_up"], saved)
    return {"h": h, "dx": dx, "dw_gate": dw_gate, "dw_up": dw_up}


def _framework():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparse-gemm-with-hopper-sptc_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import sp24
    return sp24


def work(case):
    op, t = case["op"], case["t"]
    if op in ("norm", "swiglu"):
        # two 16-bit inputs, 8-bit rows and their scales; the norm also writes the sum and reads its weight
        n = t * case["h"]
        return {"bytes": n * 5 + t * 4 + (2 * n + 2 * case["h"] if op == "norm" else 0), "flops": 8 * n}
    if op == "prod":
        # half of the weights' values and a 4-bit code for each four; one multiplication for each kept value
        m, k = case["m"], case["k"]
        out = 4 if case["out"] == "f32" else 2
        return {"bytes": m * k // 2 + m * k // 8 + t * k + t * m * out + 4 * (t + m * (2 if case["bias"] else 1)), "flops": t * m * k}
    h, f = case["h"], case["f"]
    fwd = {"bytes": 2 * (t * h + 2 * f * h + t * f), "flops": 4 * t * h * f}
    if not case["train"]:
        return fwd
    # dh in, dx and both weights' gradients out; four more products
    return {"bytes": fwd["bytes"] + 2 * (t * f + t * h + 2 * f * h), "flops": 12 * t * h * f}


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "norm":
        total = s["x"].double() + s["residual"].double()
        rms = torch.sqrt((total * total).mean(dim=1, keepdim=True) + EPS)
        return {**_exact_quantised(s["weight"].double() * (total / rms), s), "residual": total}
    if s["op"] == "swiglu":
        return _exact_quantised(s["up"].double() * s["gate"].double() * torch.sigmoid(s["gate"].double()), s)
    if s["op"] == "prod":
        # both kept values of each four gathered against their own column of x, by position within the four
        w = torch.zeros(s["m"], s["k"], dtype=torch.float64, device="cuda")
        first = torch.arange(0, s["k"], 4, device="cuda")
        for which in range(2):
            for odd in range(2):
                nibble = (s["meta"] >> (4 * odd)) & 15
                column = first[odd::2] + ((nibble >> (2 * which)) & 3).long()
                w.scatter_(1, column, s["a_c"].double()[:, 2 * odd + which::4])
        y = torch.mm(w * s["scale_w"].double()[:, None], (s["x"].double() * s["scale_x"].double()[:, None]).t()).t()
        return y if s["bias_w"] is None else y + s["bias_w"].double()
    x, wg, wu = s["x"].double(), s["w_gate"].double(), s["w_up"].double()
    gate, up = torch.mm(x, wg.t()), torch.mm(x, wu.t())
    sig = torch.sigmoid(gate)
    act = gate * sig
    if not s["train"]:
        return act * up
    dh = s["dh"].double()
    d_up, d_gate = dh * act, dh * up * (sig + act * (1 - sig))
    return {"h": act * up, "dx": torch.mm(d_gate, wg) + torch.mm(d_up, wu), "dw_gate": torch.mm(d_gate.t(), x), "dw_up": torch.mm(d_up.t(), x)}


def _exact_quantised(y, s):
    scale = y.abs().amax(dim=1) / QMAX[s["q"]]
    return {"q": y / scale[:, None], "scale": scale}
