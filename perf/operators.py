"""Measured calls of the 4-bit linear layers and the fused residual / norm block.

Each case is one call of a public operator of the binding (sdb.py), with inputs
made on the GPU from a seed.  With `own` false, run() computes the operator in
elementary torch operations; with `own` true it makes the binding's call.

  linear    y = x W^T with W of 4-bit numbers and group scales, then bias (and SiLU):  sdb.mul_mat_q4
  gated     act(x V^T + c) * (x W^T + b), both matrices of 4-bit numbers:              sdb.mul_mat_q4_gated
  quantize  a matrix turned into 4-bit numbers with group scales:                      sdb.q4_quantize
  residual  h = keep x + scale gate post(y), out = pre(h) (1 + mul) + add:             sdb.residual_norm
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parent.parent
DTYPES = {"f32": torch.float32, "f16": torch.float16}


def _sdb():
    pkg = str(ROOT / "stable-diffusion.assembly_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import sdb

    return sdb


# ---------------------------------------------------------------- cases

def _linear(rows, k, n, group, minimum, act="none", x="f32", out="f32"):
    return {"op": "linear", "rows": rows, "k": k, "n": n, "group": group, "minimum": minimum, "act": act,
            "x": x, "out": out}


def _gated(rows, k, half, group, minimum, act, x="f32", out="f32"):
    return {"op": "gated", "rows": rows, "k": k, "half": half, "group": group, "minimum": minimum, "act": act,
            "x": x, "out": out}


def _quantize(n, k, group, minimum, w):
    return {"op": "quantize", "n": n, "k": k, "group": group, "minimum": minimum, "w": w}


def _residual(images, tokens, c, post, pre, gate, mod, affine, x="f32", y="f32"):
    return {"op": "residual", "images": images, "tokens": tokens, "c": c, "post": post, "pre": pre, "gate": gate,
            "mod": mod, "affine": affine, "x": x, "y": y}


def listed():
    return [
        # The UNet's time embedding for one image with guidance: two rows, the smallest layer.
        {"name": "time_embedding_2x320x1280", **_linear(2, 320, 1280, 32, False, "silu")},
        # One token through a square projection, the ordinary single-token call.
        {"name": "token_1x4096x4096", **_linear(1, 4096, 4096, 32, False)},
        # One token through a wide feed-forward matrix: the largest weights, streamed once.
        {"name": "token_1x8192x28672", **_linear(1, 8192, 28672, 128, True)},
        # Every ResBlock's time-embedding projection of SD 1.5 at once, eight images with guidance.
        {"name": "resblocks_16x1280x20160", **_linear(16, 1280, 20160, 64, True)},
        # A prompt's 77 tokens through a square projection, half precision: the most arithmetic.
        {"name": "prompt_77x4096x4096_f16", **_linear(77, 4096, 4096, 32, False, x="f16", out="f16")},
        # A gated feed-forward layer for one token.
        {"name": "gated_silu_1x4096x11008", **_gated(1, 4096, 11008, 128, False, "silu")},
        # SD 1.5's GEGLU width for a few rows, an odd number of them.
        {"name": "gated_gelu_5x1280x5120", **_gated(5, 1280, 5120, 32, True, "gelu")},
        # A GEGLU matrix of the UNet quantized as a checkpoint is loaded.
        {"name": "quantize_10240x1280_f16", **_quantize(10240, 1280, 64, False, "f16")},
        # A ragged matrix with minima, every row's last group short.
        {"name": "quantize_4097x4001_f32", **_quantize(4097, 4001, 32, True, "f32")},
        # A modulated block over two images' tokens at 64 x 64: gate, LayerNorm, scale and shift an image.
        {"name": "modulated_2x4096x1280", **_residual(2, 4096, 1280, "none", "layer", "image", "image", False)},
        # One token between two blocks normalised before and after (RMS norms with weights).
        {"name": "token_1x1x4096_rms", **_residual(1, 1, 4096, "rms", "rms", "channel", "none", True)},
        # A ragged half-precision batch of prompts.
        {"name": "prompts_7x77x2047_f16", **_residual(7, 77, 2047, "layer", "rms", "none", "image", True, "f16", "f16")},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "gated", "quantize", "residual", "residual"])
    group = rng.choice([32, 64, 128])
    minimum = rng.random() < 0.5
    kind = lambda: rng.choice(["f32", "f32", "f16"])
    if op in ("linear", "gated"):
        k = _log(rng, 64, 8192)
        n = _log(rng, 16, 28672)
        if rng.random() < 0.7:  # most layers are whole groups
            k = max(128, k // 128 * 128)
            n = max(16, n // 16 * 16)
        rows = _log(rng, 1, 96)
        while rows > 1 and rows * k * n > 77 * 4096 * 4096:  # no more arithmetic than the prompt's call
            rows //= 2
        if op == "linear":
            return _linear(rows, k, n, group, minimum, rng.choice(["none", "silu"]), kind(), kind())
        return _gated(rows, k, max(8, n // 2), group, minimum, rng.choice(["gelu", "silu"]), kind(), kind())
    if op == "quantize":
        return _quantize(_log(rng, 16, 8192), _log(rng, 33, 4096), group, minimum, rng.choice(["f32", "f16"]))
    c = _log(rng, 64, 8192)
    if rng.random() < 0.5:
        c = max(64, c // 64 * 64)
    images, tokens = rng.randint(1, 8), _log(rng, 1, 4096)
    norm = lambda: rng.choice(["none", "layer", "rms"])
    case = _residual(images, tokens, c, norm(), rng.choice(["layer", "rms"]),
                     rng.choice(["none", "image", "channel", "token"]), rng.choice(["none", "image", "token"]),
                     rng.random() < 0.5, kind(), kind())
    while work(case)["bytes"] > 165e6:
        case["tokens"] //= 2
    return case


# ---------------------------------------------------------------- inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) % (1 << 62))
    return g


def _normal(g, *shape, std=1.0, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").mul_(std).to(dtype)


def _activations(g, rows, k, dtype):
    """Normal numbers with a few channels far larger than the rest, as trained networks have them."""
    x = torch.randn(rows, k, generator=g, device="cuda")
    loud = torch.rand(k, generator=g, device="cuda") < 0.01
    x[:, loud] *= 20.0
    return x.to(dtype)


def _matrix(g, n, k, group, minimum):
    """4-bit numbers (two a byte, the even column low), FP16 scales and, with `minimum`, FP16 minima."""
    groups = -(-k // group)
    lo = torch.randn(n, (k + 1) // 2, generator=g, device="cuda").mul_(2.7).add_(8.0).round_().clamp_(0, 15)
    codes = lo.to(torch.uint8)
    del lo
    hi = torch.randn(n, (k + 1) // 2, generator=g, device="cuda").mul_(2.7).add_(8.0).round_().clamp_(0, 15)
    codes += hi.to(torch.uint8) * 16
    del hi
    scales = (torch.rand(n, groups, generator=g, device="cuda") + 0.5) * (0.37 / math.sqrt(k))
    m = {"codes": codes, "scales": scales.half(), "minima": None, "k": k, "group": group}
    if minimum:
        m["minima"] = (-scales * (7.0 + 2.0 * torch.rand(n, groups, generator=g, device="cuda"))).half()
    if own:
        m["q4"] = _sdb().q4_import(m["codes"], m["scales"], m["minima"], k=k, group=group)
    return m


def _norm(g, kind, c, affine):
    """(kind, eps, weight, bias); an RMS norm has a weight alone."""
    weight = _normal(g, c, std=0.2).add_(1.0) if affine and kind != "none" else None
    bias = _normal(g, c, std=0.2) if affine and kind == "layer" else None
    return {"kind": kind, "eps": 1e-5 if kind == "layer" else 1e-6, "weight": weight, "bias": bias}


def _modulation(g, where, images, tokens, c):
    if where == "none":
        return None
    shape = {"image": (images, 1, c), "channel": (1, 1, c), "token": (images, tokens, c)}[where]
    return _normal(g, *shape, std=0.5)


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    st = {"case": case}
    if op == "linear":
        st["w"] = _matrix(g, case["n"], case["k"], case["group"], case["minimum"])
        st["x"] = _activations(g, case["rows"], case["k"], DTYPES[case["x"]])
        st["bias"] = _normal(g, case["n"], std=0.5)
        st["out"] = torch.empty(case["rows"], case["n"], dtype=DTYPES[case["out"]], device="cuda")
        if own:
            chain = _sdb().Chain().add(st["bias"])
            st["chain"] = chain.silu() if case["act"] == "silu" else chain
    elif op == "gated":
        half = case["half"]
        st["w"] = _matrix(g, half, case["k"], case["group"], case["minimum"])
        st["v"] = _matrix(g, half, case["k"], case["group"], case["minimum"])
        st["x"] = _activations(g, case["rows"], case["k"], DTYPES[case["x"]])
        st["bias"] = _normal(g, 2 * half, std=0.5)
        st["out"] = torch.empty(case["rows"], half, dtype=DTYPES[case["out"]], device="cuda")
        if own:
            st["chain"] = _sdb().Chain().add(st["bias"])
    elif op == "quantize":
        w = torch.randn(case["n"], case["k"], generator=g, device="cuda")
        w *= torch.rand(case["n"], 1, generator=g, device="cuda") * (1.0 / math.sqrt(case["k"]))
        st["w"] = w.to(DTYPES[case["w"]])
    else:
        b, t, c = case["images"], case["tokens"], case["c"]
        st["x"] = _activations(g, b * t, c, DTYPES[case["x"]]).view(b, t, c)
        st["y"] = _normal(g, b, t, c, std=0.7, dtype=DTYPES[case["y"]])
        st["post"] = _norm(g, case["post"], c, case["affine"])
        st["pre"] = _norm(g, case["pre"], c, case["affine"])
        st["gate"] = _modulation(g, case["gate"], b, t, c)
        st["mul"] = _modulation(g, case["mod"], b, t, c)
        st["add"] = _modulation(g, case["mod"], b, t, c)
        st["h"] = torch.empty_like(st["x"])
        st["out"] = torch.empty_like(st["y"])
        if own:
            sdb = _sdb()
            for key in ("post", "pre"):
                n = st[key]
                st[key + "_norm"] = (sdb.Norm(n["kind"], n["eps"], n["weight"], n["bias"])
                                     if n["kind"] != "none" else None)
    return st


# ---------------------------------------------------------------- the calls and their plain forms

KEEP, SCALE = 1.0, 0.5  # of the residual block: h = KEEP x + SCALE gate post(y)


def _values(m, dtype=torch.float32):
    """The numbers that a matrix of 4-bit numbers stands for."""
    n = m["codes"].shape[0]
    q = torch.stack((m["codes"] & 15, m["codes"] >> 4), dim=2).view(n, -1)[:, :m["k"]].to(dtype)
    d = m["scales"].to(dtype).repeat_interleave(m["group"], dim=1)[:, :m["k"]]
    if m["minima"] is None:
        return d * (q - 8.0)
    return d * q + m["minima"].to(dtype).repeat_interleave(m["group"], dim=1)[:, :m["k"]]


def _silu(y):
    return y / (1.0 + torch.exp(-y))


def _gelu(y):
    """GELU's tanh form, the one ggml defines."""
    return 0.5 * y * (1.0 + torch.tanh(0.79788456080286535588 * (y + 0.044715 * y * y * y)))


def _quantized_values(w, group, minimum):
    n, k = w.shape
    groups = -(-k // group)
    full = groups * group
    w = w.to(torch.float32)
    if full != k:  # a short last group: repeat its last number, which changes neither extreme
        w = torch.cat((w, w[:, -1:].expand(n, full - k)), dim=1)
    w = w.reshape(n, groups, group)
    hi, lo = w.amax(dim=2, keepdim=True), w.amin(dim=2, keepdim=True)
    half = lambda v: v.clamp(-65504.0, 65504.0).half().float()
    if minimum:
        d, m = half((hi - lo) / torch.full_like(hi, 15.0)), half(lo)  # a tensor: a true division
        q = torch.where(d == 0, torch.zeros_like(w), torch.floor((w - m) / d + 0.5).clamp(0.0, 15.0))
        v = d * q + m
    else:
        d = half(torch.where(hi >= -lo, hi, lo) / -8.0)
        q = torch.where(d == 0, torch.full_like(w, 8.0), torch.floor(w / d + 8.5).clamp(0.0, 15.0))
        v = d * (q - 8.0)
    return v.reshape(n, full)[:, :k].contiguous()


def _normed(v, norm):
    if norm["kind"] == "none":
        return v
    if norm["kind"] == "layer":
        v = v - v.mean(dim=-1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(dim=-1, keepdim=True) + norm["eps"])
    if norm["weight"] is not None:
        v = v * norm["weight"].to(v.dtype)
    if norm["bias"] is not None:
        v = v + norm["bias"].to(v.dtype)
    return v


def _residual_block(st, dtype):
    cast = lambda t: t.to(dtype)
    u = _normed(cast(st["y"]), st["post"])
    if st["gate"] is not None:
        u = u * cast(st["gate"])
    h = KEEP * cast(st["x"]) + SCALE * u
    out = _normed(h, st["pre"])
    if st["mul"] is not None:
        out = out * (1.0 + cast(st["mul"])) + cast(st["add"])
    return h, out


def run(st):
    case = st["case"]
    op = case["op"]
    if own:
        sdb = _sdb()
        if op == "linear":
            return sdb.mul_mat_q4(st["w"]["q4"], st["x"], out=st["out"], chain=st["chain"])
        if op == "gated":
            return sdb.mul_mat_q4_gated(st["w"]["q4"], st["v"]["q4"], st["x"], act=case["act"], out=st["out"],
                                        chain=st["chain"])
        if op == "quantize":
            return sdb.q4_quantize(st["w"], group=case["group"], minimum=case["minimum"]).values()
        return sdb.residual_norm(st["x"], st["y"], post=st["post_norm"], gate=st["gate"], keep=KEEP, scale=SCALE,
                                 pre=st["pre_norm"], mul=st["mul"], add=st["add"], h=st["h"], out=st["out"])
    if op == "linear":
        y = torch.matmul(st["x"].float(), _values(st["w"]).t()) + st["bias"]
        return (_silu(y) if case["act"] == "silu" else y).to(DTYPES[case["out"]])
    if op == "gated":
        x, half = st["x"].float(), case["half"]
        a = torch.matmul(x, _values(st["w"]).t()) + st["bias"][:half]
        b = torch.matmul(x, _values(st["v"]).t()) + st["bias"][half:]
        return (a * (_silu(b) if case["act"] == "silu" else _gelu(b))).to(DTYPES[case["out"]])
    if op == "quantize":
        return _quantized_values(st["w"], case["group"], case["minimum"])
    h, out = _residual_block(st, torch.float32)
    return h.to(DTYPES[case["x"]]), out.to(DTYPES[case["y"]])


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return None  # the numbers chosen turn on FP32 roundings at ties: run()'s plain form defines them
    if op == "residual":
        b, t, c = case["images"], case["tokens"], case["c"]

        def norm64(v, n):
            if n["kind"] == "layer":
                mu = v.sum(-1, keepdim=True) / c
                r = v - mu
            else:
                r = v
            if n["kind"] != "none":
                r = r * torch.rsqrt((r ** 2).sum(-1, keepdim=True) / c + n["eps"])
            if n["weight"] is not None:
                r = r * n["weight"].double()
            return r if n["bias"] is None else r + n["bias"].double()

        u = norm64(st["y"].double(), st["post"])
        h = st["x"].double() * KEEP + (u if st["gate"] is None else u * st["gate"].double()) * SCALE
        out = norm64(h, st["pre"])
        if st["mul"] is not None:
            out = out + out * st["mul"].double() + st["add"].double()
        return h, out

    def product(m):
        """x W^T in double, some rows of W at a time."""
        x, k, g = st["x"].double(), case["k"], case["group"]
        parts = []
        step = max(1, (1 << 26) // k)
        at = torch.arange(k, device="cuda")
        for i in range(0, m["codes"].shape[0], step):
            c = m["codes"][i:i + step].int()
            q = torch.where(at % 2 == 0, c[:, at // 2] % 16, c[:, at // 2] // 16).double()
            d = m["scales"][i:i + step].double()[:, at // g]
            w = (q - 8) * d if m["minima"] is None else q * d + m["minima"][i:i + step].double()[:, at // g]
            parts.append(x @ w.T)
        return torch.cat(parts, dim=1)

    bias = st["bias"].double()
    if op == "linear":
        y = product(st["w"]) + bias
        return y * torch.sigmoid(y) if case["act"] == "silu" else y
    half = case["half"]
    a, b = product(st["w"]) + bias[:half], product(st["v"]) + bias[half:]
    if case["act"] == "silu":
        return a * b * torch.sigmoid(b)
    return a * b * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (b + 0.044715 * b ** 3))


def work(case):
    size = {"f32": 4, "f16": 2}
    op = case["op"]
    if op in ("linear", "gated"):
        rows, k = case["rows"], case["k"]
        n = case["n"] if op == "linear" else 2 * case["half"]
        cols = n if op == "linear" else case["half"]
        groups = -(-k // case["group"])
        weights = n * ((k + 1) // 2) + n * groups * (4 if case["minimum"] else 2)
        return {"bytes": weights + rows * k * size[case["x"]] + 4 * n + rows * cols * size[case["out"]],
                "flops": 2 * rows * k * n}
    if op == "quantize":
        n, k = case["n"], case["k"]
        return {"bytes": n * k * (size[case["w"]] + 4), "flops": 8 * n * k}
    b, t, c = case["images"], case["tokens"], case["c"]
    total = b * t * c
    mod = {"none": 0, "image": b * c, "channel": c, "token": total}
    bytes_ = 2 * total * (size[case["x"]] + size[case["y"]]) + 4 * (mod[case["gate"]] + 2 * mod[case["mod"]])
    return {"bytes": bytes_, "flops": 20 * total}
