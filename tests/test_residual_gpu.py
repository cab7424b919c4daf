"""The residual block (sdb_residual_norm) against float64.

    h = keep x + scale gate post(y);  out = pre(h) (1 + mul) + add

Bounds, in units of u = 2^-24, counted over the roundings of a number's way:
post(y): the subtraction of the mean and of its remainder, the product with
1 / sqrt (its own error: the sums' few u, halved by the root, and two more),
weight, bias, gate and the final sums -- at most 16 u of the magnitudes summed
into h.  out: what h is off by, taken through the norm (a number's own error and
the row's mean and root mean square of them, times 1 / sigma), and 16 u of the
normalised magnitudes.  Sums over a row are FP32, at most a few hundred numbers
a thread and a tree: the variance's error, random in sign, is far inside the 16.
A LayerNorm's mean is off by a number of its own, which counts where a number is
near the mean: a sum of c numbers d of depth s (c / 256 numbers a thread and the
tree over a CTA where a row is read again, at most 32 numbers and the tree over a
warp or a CTA where it is in registers) errs by at most
s u sum |d|, the mean so by s u mean |d| <= s u sigma: s u of the normalised
numbers, s = max(48, c / 256 + 16).  A half precision output adds 2^-11 of its
value (2^-25 below the normal numbers).
"""
from __future__ import annotations

import numpy as np
import pytest

from helpers import cuda_tensor, host, rng

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def normed(v, err, norm):
    """A row norm of v (float64) known to within err: the result, its error and its magnitude."""
    if norm is None:
        return v, err, np.abs(v)
    kind, eps, w, b = norm
    mean = v.mean(-1, keepdims=True) if kind == "layer" else 0.0
    d = v - mean
    rstd = 1.0 / np.sqrt((d * d).mean(-1, keepdims=True) + eps)
    r = d * rstd
    # A norm's derivative: 1 / sigma of a number's error, of the errors' mean, and of their part along r.
    through = rstd * (err + err.mean(-1, keepdims=True)) + np.abs(r) * rstd * np.sqrt((err * err).mean(-1, keepdims=True))
    if kind == "layer":
        through = through + max(48, v.shape[-1] // 256 + 16) * U
    mag = np.abs(r)
    if w is not None:
        r, through, mag = r * w, through * np.abs(w), mag * np.abs(w)
    if b is not None:
        r, mag = r + b, mag + np.abs(b)
    return r, through + 16 * U * mag, mag


def reference(x, y, post, gate, keep, scale, pre, mul, add):
    zero = np.zeros((x if x is not None else y).shape)
    h, err = zero, zero
    if x is not None:
        h = keep * x.astype(np.float64)
        err = 2 * U * np.abs(h)
    if y is not None:
        u, ue, um = normed(y.astype(np.float64), zero, post)
        f = scale * (gate.astype(np.float64) if gate is not None else 1.0)
        h, err = h + f * u, err + np.abs(f) * (ue + 4 * U * um)
    err = err + 2 * U * np.abs(h)
    out, oe, om = normed(h, err, pre)
    if mul is not None:
        f = 1.0 + mul.astype(np.float64)
        out, oe, om = out * f, oe * np.abs(f) + 2 * U * om * (np.abs(f) + np.abs(mul)), om * np.abs(f)
    if add is not None:
        out, om = out + add, om + np.abs(add)
    return h, err, out, oe + 2 * U * om


def check(got, want, err, what):
    half = got.dtype == np.float16
    got = got.astype(np.float64)
    tol = err + 1e-300 + (2.0 ** -11 * np.abs(want) + 2.0 ** -25 if half else 2.0 ** -140)
    assert np.isfinite(got).all(), f"{what}: not written"
    worst = (np.abs(got - want) / tol).max()
    assert worst <= 1.0, f"{what}: {worst:.3g} of the bound"


def inputs(g, shape, xt=np.float32, yt=np.float32, offset=0.0):
    x = (g.standard_normal(shape) * 2 + offset).astype(xt)
    y = (g.standard_normal(shape) * 0.7 + offset).astype(yt)
    return x, y


def norm_of(sdb, cuda, norm):
    if norm is None:
        return None
    kind, eps, w, b = norm
    t = lambda a: cuda_tensor(a, cuda) if a is not None else None
    return sdb.Norm(kind, eps, t(w), t(b))


def run(cuda, x, y, post=None, gate=None, keep=1.0, scale=1.0, pre=None, mul=None, add=None, **kw):
    import sdb

    t = lambda a: cuda_tensor(a, cuda) if a is not None else None
    h, out = sdb.residual_norm(t(x), t(y), post=norm_of(sdb, cuda, post), gate=t(gate), keep=keep, scale=scale,
                               pre=norm_of(sdb, cuda, pre), mul=t(mul), add=t(add), **kw)
    wh, eh, wo, eo = reference(x, y, post, gate, keep, scale, pre, mul, add)
    if h is not None:
        check(host(h), wh, eh, "h")
    if out is not None:
        check(host(out), wo, eo, "out")
    return h, out


def made_norm(g, kind, c, affine=True):
    if kind is None:
        return None
    w = (1 + 0.3 * g.standard_normal(c)).astype(np.float32) if affine else None
    b = (0.3 * g.standard_normal(c)).astype(np.float32) if affine and kind == "layer" else None
    return kind, 1e-5, w, b


@pytest.mark.parametrize("c", [1, 2, 3, 7, 31, 32, 33, 64, 100, 127, 128, 130, 255, 256, 320, 500, 511, 512, 516, 640,
                               1000, 1024, 1280, 1500, 2047, 2048, 2052, 4096, 4100, 5003, 8191, 8192, 8196, 11008,
                               16384, 16388, 20001, 40000])
def test_widths(cuda, c):
    """Every form of a row's width, whole vectors and ragged, few rows and (narrow rows) many."""
    g = rng(c)
    for tokens in (1, 5) if c > 2048 else (1, 3, 300):
        x, y = inputs(g, (2, tokens, c))
        gate, mul, add = (g.standard_normal((2, 1, c)).astype(np.float32) * 0.5 for _ in range(3))
        run(cuda, x, y, made_norm(g, "rms", c), gate, 1.0, 0.5, made_norm(g, "layer", c), mul, add)


@pytest.mark.parametrize("xt", [np.float32, np.float16])
@pytest.mark.parametrize("yt", [np.float32, np.float16])
@pytest.mark.parametrize("post", [None, "layer", "rms"])
@pytest.mark.parametrize("pre", [None, "layer", "rms"])
@pytest.mark.parametrize("c", [65, 320, 1284, 4096])
def test_forms_and_types(cuda, c, post, pre, xt, yt):
    g = rng(c)
    x, y = inputs(g, (3, 4, c), xt, yt)
    run(cuda, x, y, made_norm(g, post, c), None, 0.75, -1.5, made_norm(g, pre, c, affine=False))


@pytest.mark.parametrize("c", [48, 320, 2050])
@pytest.mark.parametrize("gs,ms,as_", [((1, 1, 1), (2, 1, 1), (1, 6, 1)), ((2, 6, 1), (1, 1, "c"), (2, 1, "c")),
                                       ((1, 6, "c"), (2, 6, "c"), ("c",)), (("c",), None, (2, 6, "c")),
                                       (None, (6, "c"), None)])
def test_broadcasts(cuda, c, gs, ms, as_):
    """Operands of any of the rows' extents: a channel's, an image's, a token's, one number."""
    g = rng(c)
    make = lambda s: g.standard_normal([c if e == "c" else e for e in s]).astype(np.float32) if s else None
    x, y = inputs(g, (2, 6, c))
    run(cuda, x, y, None, make(gs), 1.0, 1.0, made_norm(g, "layer", c), make(ms), make(as_))


@pytest.mark.parametrize("c", [320, 1280, 5000])
def test_rows_far_from_zero(cuda, c):
    """Numbers of mean 1000 and deviation 1: the variance keeps its digits."""
    g = rng(c)
    x, y = inputs(g, (2, 9, c), offset=1000.0)
    run(cuda, x, y, made_norm(g, "layer", c), pre=made_norm(g, "layer", c))
    run(cuda, None, y, pre=made_norm(g, "layer", c))


@pytest.mark.parametrize("c", [64, 320, 4096, 20000])
def test_parts(cuda, c):
    """No stream yet, no block yet, the stream alone, the norm alone."""
    g = rng(c)
    x, y = inputs(g, (7, c))
    assert run(cuda, x, y, made_norm(g, "rms", c), want_out=False)[1] is None
    assert run(cuda, x, y, pre=made_norm(g, "rms", c), want_h=False)[0] is None
    run(cuda, None, y, made_norm(g, "layer", c), scale=2.0, pre=made_norm(g, "rms", c))
    mul = g.standard_normal((c,)).astype(np.float32)
    run(cuda, x, None, keep=0.5, pre=made_norm(g, "layer", c), mul=mul)


@pytest.mark.parametrize("c", [96, 320, 1281, 4096, 20000])
@pytest.mark.parametrize("xt,yt", [(np.float32, np.float32), (np.float16, np.float16)])
def test_in_place(cuda, c, xt, yt):
    """h in x's memory and out in y's; h in y's and out in x's."""
    import sdb

    g = rng(c)
    x, y = inputs(g, (4, 3, c), xt, yt)
    post, pre = made_norm(g, "layer", c), made_norm(g, "rms", c)
    wh, eh, wo, eo = reference(x, y, post, None, 1.0, 1.0, pre, None, None)
    for swap in (False, True):
        tx, ty = cuda_tensor(x, cuda), cuda_tensor(y, cuda)
        h, out = (ty, tx) if swap else (tx, ty)
        sdb.residual_norm(tx, ty, post=norm_of(sdb, cuda, post), pre=norm_of(sdb, cuda, pre), h=h, out=out)
        check(host(h), wh, eh, "h")
        check(host(out), wo, eo, "out")


@pytest.mark.parametrize("c", [100, 320, 4096])
def test_strides(cuda, c):
    """Rows over three permuted dimensions, further apart and at odd elements; what lies between stays."""
    import sdb
    import torch

    g = rng(c)
    x, y = inputs(g, (2, 3, 4, c))
    gate = g.standard_normal((2, 1, 4, c)).astype(np.float32)

    def view(a, pad, at):
        base = torch.full((3, 2, 4, c + pad), 5.0, device=cuda)
        v = base.permute(1, 0, 2, 3)[..., at:at + c]
        if a is not None:
            v.copy_(cuda_tensor(a, cuda))
        return base, v

    _, tx = view(x, 8, 4)
    _, ty = view(y, 5, 3)
    hb, h = view(None, 4, 0)
    ob, out = view(None, 7, 1)
    wide = torch.zeros(2, 1, 4, 2 * c, device=cuda)
    wide[..., ::2] = cuda_tensor(gate, cuda)
    pre = made_norm(g, "layer", c)
    sdb.residual_norm(tx, ty, gate=wide[..., ::2], pre=norm_of(sdb, cuda, pre), h=h, out=out)
    wh, eh, wo, eo = reference(x, y, None, gate, 1.0, 1.0, pre, None, None)
    check(host(h), wh, eh, "h")
    check(host(out), wo, eo, "out")
    assert (host(hb)[..., c:] == 5).all()
    assert (host(ob)[..., :1] == 5).all() and (host(ob)[..., 1 + c:] == 5).all()


@pytest.mark.parametrize("c", [3, 320, 5000])
def test_constant_and_bad_rows(cuda, c):
    """A constant row becomes 0 (and bias); a row with a NaN or an infinity keeps it to itself."""
    g = rng(c)
    x = np.zeros((5, c), dtype=np.float32)
    y = np.full((5, c), 3.25, dtype=np.float32)
    y[1:] += g.standard_normal((4, c)).astype(np.float32)
    norm = made_norm(g, "layer", c)
    h, out = run(cuda, x, y, norm)
    np.testing.assert_array_equal(host(h)[0], norm[3])
    import sdb

    clean = host(out)
    y[2, c // 2], y[3, 0] = np.nan, np.inf
    h, out = sdb.residual_norm(cuda_tensor(x, cuda), cuda_tensor(y, cuda), post=norm_of(sdb, cuda, norm))
    got = host(out)
    assert not np.isfinite(got[2]).any() and not np.isfinite(got[3]).all()
    np.testing.assert_array_equal(got[[0, 1, 4]], clean[[0, 1, 4]])


def test_many_rows(cuda):
    """More rows than CTAs of any form."""
    g = rng(1)
    x, y = inputs(g, (2, 9001, 64))
    run(cuda, x, y, made_norm(g, "rms", 64), g.standard_normal((2, 1, 64)).astype(np.float32),
        pre=made_norm(g, "layer", 64))
    x, y = inputs(g, (1, 5001, 640), np.float16, np.float16)
    run(cuda, x, y, None, None, pre=made_norm(g, "layer", 640))


def test_no_rows(cuda):
    import sdb
    import torch

    before = sdb.launch_count()
    h, out = sdb.residual_norm(torch.empty(2, 0, 64, device=cuda), torch.empty(2, 0, 64, device=cuda))
    assert h.shape == (2, 0, 64) and out.shape == (2, 0, 64) and sdb.launch_count() == before


def test_refusals(cuda):
    import sdb
    import torch

    x, y = torch.zeros(2, 3, 64, device=cuda), torch.zeros(2, 3, 64, device=cuda)
    z = lambda *s, **kw: torch.zeros(*s, device=cuda, **kw)
    for call in (lambda: sdb.residual_norm(None, None),
                 lambda: sdb.residual_norm(x, z(2, 3, 63)),
                 lambda: sdb.residual_norm(x, z(2, 64, 3).transpose(1, 2)),
                 lambda: sdb.residual_norm(x, y, gate=z(2, 3, 63)),
                 lambda: sdb.residual_norm(x, y, gate=z(3, 1, 64)),
                 lambda: sdb.residual_norm(x, y, gate=z(1, 2, 3, 64)),
                 lambda: sdb.residual_norm(x, y, mul=z(64, dtype=torch.float16)),
                 lambda: sdb.residual_norm(x, y, pre=sdb.Norm("rms", 1e-6, z(32))),
                 lambda: sdb.residual_norm(x, y, pre=sdb.Norm("rms", -1.0)),
                 lambda: sdb.residual_norm(x, None, post=sdb.Norm("rms")),
                 lambda: sdb.residual_norm(x, y, pre=sdb.Norm("rms"), want_out=False),
                 lambda: sdb.residual_norm(x, y, h=z(2, 3, 64, dtype=torch.float16)),
                 lambda: sdb.residual_norm(x, y.cpu()),
                 lambda: sdb.residual_norm(x.double(), y),
                 lambda: sdb.residual_norm(x, y, h=z(1, 1, 64).expand(2, 3, 64))):
        with pytest.raises(sdb.SdbError) as e:
            call()
        assert e.value.status == sdb.INVALID


# ---------------------------------------------------------------- the operators together

def test_modulated_block(cuda):
    """A modulated transformer feed-forward block with 4-bit weights, as a user strings it together: the
    conditioning row's modulation, the norm and shift, the gated layer, the projection, the gated residual and
    the next block's norm -- eager, and captured and replayed -- against float64 and the numbers the weights
    stand for."""
    import sdb
    import torch

    g = rng(77)
    images, tokens, c, ff = 2, 5, 320, 640
    t = lambda a: cuda_tensor(a, cuda)
    weights = {name: sdb.q4_quantize(t((g.standard_normal(s) / np.sqrt(s[1])).astype(np.float32)), 32, name != "down")
               for name, s in (("mod", (3 * c, c)), ("up", (ff, c)), ("gate", (ff, c)), ("down", (c, ff)))}
    cond = t(g.standard_normal((images, c)).astype(np.float32))
    x = t(g.standard_normal((images, tokens, c)).astype(np.float32))
    pre = sdb.Norm("layer", 1e-6)
    rms = sdb.Norm("rms", 1e-6, t((1 + 0.1 * g.standard_normal(c)).astype(np.float32)))

    def block():
        m = sdb.mul_mat_q4(weights["mod"], cond).view(images, 1, 3 * c)
        shift, scale, gate = m[..., :c], m[..., c:2 * c], m[..., 2 * c:]
        _, n = sdb.residual_norm(x, None, pre=pre, mul=scale, add=shift, want_h=False)
        y = sdb.mul_mat_q4(weights["down"], sdb.mul_mat_q4_gated(weights["up"], weights["gate"], n, "silu"))
        return sdb.residual_norm(x, y, post=rms, gate=gate, pre=pre)

    def plain():
        w = {k: v.values().double() for k, v in weights.items()}
        m = (cond.double() @ w["mod"].t()).view(images, 1, 3 * c)
        shift, scale, gate = m[..., :c], m[..., c:2 * c], m[..., 2 * c:]
        layer = lambda v: torch.nn.functional.layer_norm(v, (c,), eps=1e-6)
        n = layer(x.double()) * (1 + scale) + shift
        y = (n @ w["up"].t() * torch.nn.functional.silu(n @ w["gate"].t())) @ w["down"].t()
        h = x.double() + gate * (y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * rms.weight.double())
        return h, layer(h)

    def close(got):
        # Four operators deep, each within some 20 u of numbers of order 1 and gains of a few: 2^-24 x 400.
        for a, b in zip(got, plain()):
            assert (a.double() - b).abs().max() <= 400 * U * b.abs().max()

    close(block())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block()
    for _ in range(2):
        x.copy_(t(g.standard_normal((images, tokens, c)).astype(np.float32)))
        cond.copy_(t(g.standard_normal((images, c)).astype(np.float32)))
        graph.replay()
        close(out)


@pytest.mark.parametrize("where", ["post", "pre"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("t", [np.float32, np.float16])
@pytest.mark.parametrize("c", [3, 256, 320, 513, 1280, 2047, 4096, 5003, 8192, 16384, 20001])
def test_a_nan_fills_its_row(cuda, c, t, kind, where):
    """A NaN makes a norm's statistics NaN and so every number of its row, in every form of a row's width; an
    infinity makes its own number NaN, and the others' sum of squares infinite: 0 in an RMS norm.  No other
    row knows of either."""
    import sdb

    g = rng(c)
    x, y = inputs(g, (4, c), t, t)
    norm = made_norm(g, kind, c)
    args = {where: norm_of(sdb, cuda, norm)}
    clean = host(sdb.residual_norm(cuda_tensor(x, cuda), cuda_tensor(y, cuda), **args)[1])
    y[1, c // 2], y[2, c - 1] = np.nan, np.inf
    got = host(sdb.residual_norm(cuda_tensor(x, cuda), cuda_tensor(y, cuda), **args)[1])
    assert np.isnan(got[1]).all()
    if kind == "layer":
        assert np.isnan(got[2]).all()
    else:
        assert np.isnan(got[2, c - 1])
        want = x[2] if where == "post" else np.zeros(c, t)
        np.testing.assert_array_equal(got[2, :c - 1], want[:c - 1])
    np.testing.assert_array_equal(got[[0, 3]], clean[[0, 3]])


def test_memory_made_for_another_stream(cuda):
    """What a call on another stream makes is not memory that the current stream still writes."""
    import sdb
    from test_q4_gpu import assert_apart

    x, y = inputs(rng(5), (64, 256))
    tx, ty = cuda_tensor(x, cuda), cuda_tensor(y, cuda)
    assert_apart(lambda s: sdb.residual_norm(tx, ty, pre=sdb.Norm("rms"), stream=s))
