"""4-bit matrices and their linear layers against float64.

The matrices: made numbers and scales have to be those of the formulas (restated
here in numpy, FP32 operation by FP32 operation), bit for bit.  The products:
sum_k x value in float64 from the numbers the matrix stands for, held to the
linear layers' bound, oracle.K_B200 of the summed magnitudes.  x enters whole.
One row's sums over a group are exact, so that its error is that of one rounding a
group and digit and the FP32 sum over the groups; with more rows a group's sum
takes at most 8 products of a row's first part one after another and 16 of the
others, 2^-8 of it.  A running sum of s terms errs by at most s 2^-23 of the
magnitudes with sums cut instead of rounded; for the random signs of real rows (an
error of sqrt(s) steps) that is under 1e-6, which the bound was set for.
An FP16 output adds its rounding, 2^-11 of the value (2^-25 below FP16's normal
numbers).
"""
from __future__ import annotations

import numpy as np
import pytest

import oracle
from helpers import cuda_tensor, host, rng

pytestmark = pytest.mark.gpu

GROUPS = (32, 64, 128)


def made(g, n, k, group, minimum):
    """4-bit numbers, FP16 scales and minima at random, and the numbers they stand for (float64)."""
    groups = -(-k // group)
    q = g.integers(0, 16, (n, k)).astype(np.uint8)
    scales = ((g.random((n, groups)) + 0.25) * 0.05 * g.choice([-1.0, 1.0], (n, groups))).astype(np.float16)
    minima = g.standard_normal((n, groups)).astype(np.float16) if minimum else None
    d = np.repeat(scales.astype(np.float64), group, axis=1)[:, :k]
    if minimum:
        values = d * q + np.repeat(minima.astype(np.float64), group, axis=1)[:, :k]
    else:
        values = d * (q.astype(np.float64) - 8)
    return q, scales, minima, values


def codes_of(q):
    n, k = q.shape
    padded = np.zeros((n, (k + 1) // 2 * 2), dtype=np.uint8)
    padded[:, :k] = q
    return padded[:, 0::2] | padded[:, 1::2] << 4


def on_device(cuda, q, scales, minima, group):
    import sdb

    return sdb.q4_import(cuda_tensor(codes_of(q), cuda), cuda_tensor(scales, cuda),
                         cuda_tensor(minima, cuda) if minima is not None else None, k=q.shape[1], group=group)


def quantized(w, group, minimum):
    """The formulas of sdb_q4_quantize in numpy: FP32 values."""
    n, k = w.shape
    w = w.astype(np.float32)
    out = np.empty((n, k), dtype=np.float32)
    sat = lambda v: np.clip(v, np.float32(-65504), np.float32(65504)).astype(np.float16).astype(np.float32)
    for at in range(0, k, group):
        x = w[:, at:at + group]
        hi, lo = x.max(axis=1, keepdims=True), x.min(axis=1, keepdims=True)
        with np.errstate(divide="ignore", invalid="ignore"):
            if minimum:
                d, m = sat((hi - lo) / np.float32(15)), sat(lo)
                q = np.where(d == 0, np.float32(0), np.clip(np.floor((x - m) / d + np.float32(0.5)), 0, 15))
                out[:, at:at + group] = d * q + m
            else:
                d = sat(np.where(hi >= -lo, hi, lo) / np.float32(-8))
                q = np.where(d == 0, np.float32(8), np.clip(np.floor(x / d + np.float32(8.5)), 0, 15))
                out[:, at:at + group] = d * (q - np.float32(8))
    return out


# ---------------------------------------------------------------- the matrices

@pytest.mark.parametrize("minimum", [False, True])
@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (3, 31, 32), (17, 33, 32), (16, 128, 64), (5, 200, 64),
                                       (40, 640, 128), (33, 1001, 128), (2, 4096, 32)])
def test_import_stands_for_its_numbers(cuda, n, k, group, minimum):
    q, scales, minima, values = made(rng(n * k), n, k, group, minimum)
    got = host(on_device(cuda, q, scales, minima, group).values())
    np.testing.assert_array_equal(got, values.astype(np.float32))


@pytest.mark.parametrize("minimum", [False, True])
@pytest.mark.parametrize("n,k", [(1, 32), (18, 96), (7, 320), (16, 128)])
def test_ggml_blocks(cuda, n, k, minimum):
    """Q4_0 and Q4_1 blocks, rows further apart than their blocks."""
    import sdb

    q, scales, minima, values = made(rng(n + k), n, k, 32, minimum)
    size = 20 if minimum else 18
    rows = np.full((n, k // 32 * size + 6), 0xA5, dtype=np.uint8)
    for b in range(k // 32):
        at = b * size
        rows[:, at:at + 2] = scales[:, b:b + 1].view(np.uint8)
        if minimum:
            rows[:, at + 2:at + 4] = minima[:, b:b + 1].view(np.uint8)
        nib = q[:, b * 32:b * 32 + 32]
        rows[:, at + size - 16:at + size] = nib[:, :16] | nib[:, 16:] << 4
    got = host(sdb.q4_from_blocks(cuda_tensor(rows, cuda), k, minimum).values())
    np.testing.assert_array_equal(got, values.astype(np.float32))


@pytest.mark.parametrize("minimum", [False, True])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (9, 37, 32), (16, 256, 128), (31, 129, 64), (64, 1280, 64),
                                       (130, 1000, 128)])
def test_quantize(cuda, n, k, group, dtype, minimum):
    import sdb

    g = rng(n + k + group)
    w = g.standard_normal((n, k)).astype(dtype)
    w[0, :] = 0  # a row of zeros, then one of a single number, then ties of magnitude
    if n > 2:
        w[1, :] = dtype(-0.75)
        w[2, :] = np.where(np.arange(k) % 2 == 0, dtype(0.5), dtype(-0.5))
    got = host(sdb.q4_quantize(cuda_tensor(w, cuda), group, minimum).values())
    np.testing.assert_array_equal(got, quantized(w, group, minimum))


def test_quantize_strided_rows_and_extremes(cuda):
    """A view with rows further apart (odd alignment), numbers past FP16's scales, tiny ones, non-finite groups."""
    import sdb

    g = rng(5)
    w = g.standard_normal((6, 101)).astype(np.float32)
    w[0] *= 1e30
    w[1] *= 1e-9
    base = np.zeros((6, 150), dtype=np.float32)
    base[:, 7:108] = w
    t = cuda_tensor(base, cuda)[:, 7:108]
    for minimum in (False, True):
        got = host(sdb.q4_quantize(t, 32, minimum).values())
        np.testing.assert_array_equal(got, quantized(w, 32, minimum))
    w[3, 40], w[4, 0], w[5, 100] = np.nan, np.inf, -np.inf
    bad = np.zeros((6, 101), dtype=bool)
    bad[3, 32:64], bad[4, :32], bad[5, 96:] = True, True, True
    for minimum in (False, True):
        got = host(sdb.q4_quantize(cuda_tensor(w, cuda), 32, minimum).values())
        assert np.array_equal(np.isnan(got), bad)
        clean = np.where(bad, np.float32(1), w)
        np.testing.assert_array_equal(got[~bad], quantized(clean, 32, minimum)[~bad])


def test_values_into_strided_rows(cuda):
    """Rows further apart than their numbers: what lies between them stays."""
    import torch

    q, scales, minima, values = made(rng(8), 20, 70, 32, True)
    out = torch.full((20, 93), 7.0, device=cuda)
    on_device(cuda, q, scales, minima, 32).values(out=out[:, 11:81])
    got = host(out)
    np.testing.assert_array_equal(got[:, 11:81], values.astype(np.float32))
    assert (got[:, :11] == 7).all() and (got[:, 81:] == 7).all()


# ---------------------------------------------------------------- products

def check(got, exact, magnitude, half_out=False):
    got = np.asarray(got, dtype=np.float64)
    tol = oracle.K_B200 * np.where(magnitude > 0, magnitude, 1.0)
    if half_out:
        tol = tol + 2.0 ** -11 * np.abs(exact) + 2.0 ** -25
    assert np.isfinite(got).all(), "an output was not written"
    worst = (np.abs(got - exact) / tol).max()
    assert worst <= 1.0, f"{worst:.3g} of the bound"


def run_linear(cuda, g, rows, k, n, group, minimum, xt=np.float32, ot=np.float32):
    import sdb
    import torch

    q, scales, minima, values = made(g, n, k, group, minimum)
    x = g.standard_normal((rows, k)).astype(xt)
    x[:, g.random(k) < 0.02] *= xt(20)
    out = torch.full((rows, n), float("nan"), device=cuda,
                     dtype=torch.float16 if ot == np.float16 else torch.float32)
    sdb.mul_mat_q4(on_device(cuda, q, scales, minima, group), cuda_tensor(x, cuda), out=out)
    exact, mag = oracle.mul_mat_exact(values, x)
    check(host(out), exact, mag, ot == np.float16)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 24, 31, 32, 33, 64, 65, 77, 129])
def test_rows(cuda, rows):
    run_linear(cuda, rng(rows), rows, 320, 130, 32, False)
    run_linear(cuda, rng(rows + 1), rows, 416, 48, 128, True)


@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("minimum", [False, True])
@pytest.mark.parametrize("rows", [1, 2, 6, 20])
@pytest.mark.parametrize("xt,ot", [(np.float32, np.float32), (np.float16, np.float16), (np.float16, np.float32),
                                   (np.float32, np.float16)])
def test_forms_and_types(cuda, group, minimum, rows, xt, ot):
    run_linear(cuda, rng(group + rows), rows, 1000, 72, group, minimum, xt, ot)


@pytest.mark.parametrize("rows", [1, 3, 12])
@pytest.mark.parametrize("k,n", [(1, 1), (2, 17), (31, 16), (33, 15), (127, 31), (128, 16), (129, 33), (255, 1),
                                 (320, 1280), (1280, 20), (4128, 100), (5000, 9), (11000, 40), (28672, 64),
                                 (64, 5000)])
def test_sizes(cuda, k, n, rows):
    run_linear(cuda, rng(k + n), rows, k, n, 32, True)
    run_linear(cuda, rng(k + n + 1), rows, k, n, 128, False)


def test_wide_and_tall(cuda):
    run_linear(cuda, rng(1), 1, 4096, 4096, 32, False)
    run_linear(cuda, rng(2), 2, 1280, 20160, 64, True)
    run_linear(cuda, rng(3), 40, 28672, 48, 64, True)


@pytest.mark.parametrize("rows", [1, 2, 5, 12, 20])
def test_magnitudes(cuda, rows):
    """Rows of x from 1e-36 (numbers below the normal ones among them) to 1e30 and of mixed magnitudes: the bound
    holds at every scale."""
    import sdb

    g = rng(31)
    q, scales, minima, values = made(g, 50, 300, 64, True)
    w = on_device(cuda, q, scales, minima, 64)
    for scale in (1e-36, 1e-30, 1e-6, 1e6, 1e30):
        x = (g.standard_normal((rows, 300)) * scale * 10.0 ** g.uniform(-3, 3, (rows, 300))).astype(np.float32)
        exact, mag = oracle.mul_mat_exact(values, x)
        check(host(sdb.mul_mat_q4(w, cuda_tensor(x, cuda))), exact, mag)


@pytest.mark.parametrize("rows", [2, 7])
def test_a_bad_row_stays_alone(cuda, rows):
    """Infinities and NaN in one row of x reach that row's outputs and no other."""
    import sdb

    g = rng(6)
    q, scales, minima, values = made(g, 40, 200, 32, True)
    w = on_device(cuda, q, scales, minima, 32)
    x = g.standard_normal((rows, 200)).astype(np.float32)
    exact, mag = oracle.mul_mat_exact(values, x)
    for bad in (np.nan, np.inf, -np.inf):
        y = x.copy()
        y[1, 77] = bad
        got = host(sdb.mul_mat_q4(w, cuda_tensor(y, cuda)))
        assert not np.isfinite(got[1]).any()
        keep = [r for r in range(rows) if r != 1]
        check(got[keep], exact[keep], mag[keep])


@pytest.mark.parametrize("rows", [1, 4, 40])
def test_chain(cuda, rows):
    """Bias, a scale a column, a residual of the output's shape and SiLU, in order."""
    import sdb

    g = rng(rows)
    n, k = 90, 257
    q, scales, minima, values = made(g, n, k, 32, False)
    x = g.standard_normal((rows, k)).astype(np.float32)
    b, s, r = (g.standard_normal(shape).astype(np.float32) for shape in ((n,), (n,), (rows, n)))
    t = lambda a: cuda_tensor(a, cuda)
    chain = sdb.Chain().add(t(b)).mul(t(s)).add(t(r)).silu()
    got = host(sdb.mul_mat_q4(on_device(cuda, q, scales, minima, 32), t(x), chain=chain))
    exact, mag = oracle.mul_mat_exact(values, x)
    v = (exact + b) * s.astype(np.float64) + r
    m = (mag + np.abs(b)) * np.abs(s) + np.abs(r)
    check(got, v / (1 + np.exp(-v)), 1.1 * m)  # SiLU's slope is at most 1.1


@pytest.mark.parametrize("from_redirect", [False, True])
def test_redirect(cuda, from_redirect):
    """A residual in its own memory: the sum begins from it, or it is written alone."""
    import sdb
    import torch

    g = rng(3)
    q, scales, minima, values = made(g, 70, 160, 32, False)
    x, b, r = (g.standard_normal(s).astype(np.float32) for s in ((3, 160), (70,), (3, 70)))
    out = torch.full((3, 70), 5.0, device=cuda)
    res = cuda_tensor(r, cuda)
    sdb.mul_mat_q4(on_device(cuda, q, scales, minima, 32), cuda_tensor(x, cuda), out=out,
                   chain=sdb.Chain().add(cuda_tensor(b, cuda)).redirect(res, from_redirect))
    exact, mag = oracle.mul_mat_exact(values, x)
    check(host(res), exact + b + (r if from_redirect else 0), mag + np.abs(b) + np.abs(r))
    assert (host(out) == 5).all()


@pytest.mark.parametrize("rows", [(2, 3, 1), (1, 5, 2), (2, 2, 9)])
def test_strides(cuda, rows):
    """Rows over three dimensions, permuted and further apart, x at an odd element; what lies between stays."""
    import sdb
    import torch

    g = rng(9)
    a, b, c = rows
    k, n = 200, 33
    q, scales, minima, values = made(g, n, k, 64, True)
    x = g.standard_normal((a, b, c, k)).astype(np.float32)
    base = torch.full((b, a, c, k + 9), 3.0, device=cuda)
    view = base.permute(1, 0, 2, 3)[..., 3:3 + k]
    view.copy_(cuda_tensor(x, cuda))
    whole = torch.full((c, b, a, n + 6), 9.0, device=cuda)
    out = whole.permute(2, 1, 0, 3)[..., 1:1 + n]
    bias = g.standard_normal((a, 1, c, n)).astype(np.float32)
    sdb.mul_mat_q4(on_device(cuda, q, scales, minima, 64), view, out=out, chain=sdb.Chain().add(cuda_tensor(bias, cuda)))
    exact, mag = oracle.mul_mat_exact(values, x)
    check(host(out), exact + bias, mag + np.abs(bias))
    w = host(whole)
    assert (w[..., :1] == 9).all() and (w[..., 1 + n:] == 9).all()


@pytest.mark.parametrize("xt", [np.float32, np.float16])
@pytest.mark.parametrize("rows", [1, 3, 6, 12, 20])
def test_alignments(cuda, rows, xt):
    """Rows that begin at every alignment and lie any number of elements apart, k a multiple of 4 and not."""
    import sdb

    g = rng(rows)
    for k, offset, apart in ((260, 0, 0), (260, 4, 4), (260, 2, 2), (260, 1, 3), (257, 0, 7), (130, 8, 6)):
        q, scales, minima, values = made(g, 40, k, 32, True)
        x = g.standard_normal((rows, k)).astype(xt)
        base = np.full((rows, offset + k + apart), 1e4, dtype=xt)
        base[:, offset:offset + k] = x
        view = cuda_tensor(base, cuda)[:, offset:offset + k]
        exact, mag = oracle.mul_mat_exact(values, x)
        got = sdb.mul_mat_q4(on_device(cuda, q, scales, minima, 32), view)
        check(host(got), exact, mag, xt == np.float16)


def test_one_dimension(cuda):
    """A single row as a vector, in and out; rows of one image each over the third dimension."""
    import sdb

    g = rng(4)
    q, scales, minima, values = made(g, 33, 96, 32, False)
    w = on_device(cuda, q, scales, minima, 32)
    x = g.standard_normal((96,)).astype(np.float32)
    exact, mag = oracle.mul_mat_exact(values, x)
    out = sdb.mul_mat_q4(w, cuda_tensor(x, cuda))
    assert out.shape == (33,)
    check(host(out), exact, mag)
    x = g.standard_normal((3, 1, 96)).astype(np.float32)
    exact, mag = oracle.mul_mat_exact(values, x)
    check(host(sdb.mul_mat_q4(w, cuda_tensor(x, cuda))), exact, mag)


def test_infinities_with_many_rows(cuda):
    """The halves' form too keeps a bad row alone: 12 and 40 rows, FP32 and FP16."""
    import sdb

    g = rng(16)
    q, scales, minima, values = made(g, 48, 300, 64, False)
    w = on_device(cuda, q, scales, minima, 64)
    for rows in (12, 40):
        for xt in (np.float32, np.float16):
            x = g.standard_normal((rows, 300)).astype(xt)
            exact, mag = oracle.mul_mat_exact(values, x)
            y = x.copy()
            y[3, 5], y[9, 299] = np.inf, np.nan
            got = host(sdb.mul_mat_q4(w, cuda_tensor(y, cuda)))
            keep = [r for r in range(rows) if r not in (3, 9)]
            assert not np.isfinite(got[[3, 9]]).any()
            check(got[keep], exact[keep], mag[keep], xt == np.float16)


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("rows,k,half,group,minimum", [(1, 320, 1280, 32, False), (2, 100, 17, 32, True),
                                                       (5, 1280, 640, 64, True), (9, 777, 50, 128, False),
                                                       (33, 256, 48, 128, True), (1, 9000, 40, 64, False)])
@pytest.mark.parametrize("xt,ot", [(np.float32, np.float32), (np.float16, np.float16)])
def test_gated(cuda, rows, k, half, group, minimum, act, xt, ot):
    import sdb
    import torch

    g = rng(rows + k)
    qa = made(g, half, k, group, minimum)
    qb = made(g, half, k, group, minimum)
    x = (g.standard_normal((rows, k)) / np.sqrt(k)).astype(xt)
    bias = g.standard_normal((2 * half,)).astype(np.float32)
    out = torch.full((rows, half), float("nan"), device=cuda,
                     dtype=torch.float16 if ot == np.float16 else torch.float32)
    sdb.mul_mat_q4_gated(on_device(cuda, *qa[:3], group), on_device(cuda, *qb[:3], group), cuda_tensor(x, cuda), act,
                         out=out, chain=sdb.Chain().add(cuda_tensor(bias, cuda)))
    a, ma = oracle.mul_mat_exact(qa[3], x)
    b, mb = oracle.mul_mat_exact(qb[3], x)
    a, b, ma, mb = a + bias[:half], b + bias[half:], ma + np.abs(bias[:half]), mb + np.abs(bias[half:])
    if act == "gelu":
        act_b = 0.5 * b * (1 + np.tanh(np.sqrt(2 / np.pi) * (b + 0.044715 * b ** 3)))
    else:
        act_b = b / (1 + np.exp(-b))
    # The gate's slope is at most 1.13 (GELU) and 1.1 (SiLU).
    check(host(out), a * act_b, ma * np.abs(act_b) + np.abs(a) * 1.13 * mb, ot == np.float16)


# ---------------------------------------------------------------- use

def test_no_rows(cuda):
    import sdb
    import torch

    q, scales, minima, _ = made(rng(1), 8, 64, 32, False)
    w = on_device(cuda, q, scales, minima, 32)
    before = sdb.launch_count()
    out = sdb.mul_mat_q4(w, torch.empty(0, 64, device=cuda))
    assert out.shape == (0, 8) and sdb.launch_count() == before


def test_same_numbers_whatever_the_company(cuda):
    """A call's result does not turn on chance: twice the same, and on two streams at once."""
    import sdb
    import torch

    g = rng(12)
    q, scales, minima, _ = made(g, 1000, 2048, 32, True)
    w = on_device(cuda, q, scales, minima, 32)
    x = [cuda_tensor(g.standard_normal((r, 2048)).astype(np.float32), cuda) for r in (1, 3)]
    want = [host(sdb.mul_mat_q4(w, v)) for v in x]
    streams = [torch.cuda.Stream() for _ in x]
    outs = [[torch.empty(v.shape[0], 1000, device=cuda) for _ in range(20)] for v in x]
    torch.cuda.synchronize()
    for i in range(20):
        for s, v, o in zip(streams, x, outs):
            sdb.mul_mat_q4(w, v, out=o[i], stream=s)
    torch.cuda.synchronize()
    for o, first in zip(outs, want):
        for t in o:
            np.testing.assert_array_equal(host(t), first)


def test_captured_and_replayed(cuda):
    """A graph of a gated layer and a projection: replayed on new numbers in the same memory, first call included."""
    import sdb
    import torch

    g = rng(13)
    up = [on_device(cuda, *made(g, 256, 192, 32, False)[:3], 32) for _ in range(2)]
    down = on_device(cuda, *made(g, 192, 256, 64, True)[:3], 64)
    x = torch.zeros(2, 192, device=cuda)
    mid, out = torch.empty(2, 256, device=cuda), torch.empty(2, 192, device=cuda)

    def call():
        sdb.mul_mat_q4_gated(up[0], up[1], x, out=mid)
        sdb.mul_mat_q4(down, mid, out=out, chain=sdb.Chain().add(x))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for _ in range(3):
        x.copy_(cuda_tensor(g.standard_normal((2, 192)).astype(np.float32), cuda))
        graph.replay()
        got = host(out)
        call()
        np.testing.assert_array_equal(got, host(out))


def test_a_chain_used_again_and_changed(cuda):
    """A chain's description follows what is done to it between calls."""
    import sdb

    g = rng(21)
    q, scales, minima, values = made(g, 24, 64, 32, False)
    w = on_device(cuda, q, scales, minima, 32)
    x = g.standard_normal((2, 64)).astype(np.float32)
    a, b = (g.standard_normal((24,)).astype(np.float32) for _ in range(2))
    exact, mag = oracle.mul_mat_exact(values, x)
    chain = sdb.Chain().add(cuda_tensor(a, cuda))
    t = cuda_tensor(x, cuda)
    for _ in range(2):
        check(host(sdb.mul_mat_q4(w, t, chain=chain)), exact + a, mag + np.abs(a))
    chain.mul(cuda_tensor(b, cuda))
    check(host(sdb.mul_mat_q4(w, t, chain=chain)), (exact + a) * b.astype(np.float64), (mag + np.abs(a)) * np.abs(b))
    chain.steps[0] = (sdb.STEP_MUL, *chain.steps[0][1:])
    want = exact * a.astype(np.float64) * b
    check(host(sdb.mul_mat_q4(w, t, chain=chain)), want, mag * np.abs(a.astype(np.float64) * b))


def test_refusals(cuda):
    import sdb
    import torch

    q, scales, minima, _ = made(rng(1), 8, 64, 32, False)
    w = on_device(cuda, q, scales, minima, 32)
    x = torch.zeros(2, 64, device=cuda)
    out = torch.empty(2, 8, device=cuda)

    def refused(status, call):
        with pytest.raises(sdb.SdbError) as e:
            call()
        assert e.value.status == status

    refused(sdb.NOT_SUPPORTED, lambda: sdb.mul_mat_q4(w, torch.zeros(2, 63, device=cuda), out=out))
    refused(sdb.NOT_SUPPORTED, lambda: sdb.mul_mat_q4(w, x, out=torch.empty(2, 9, device=cuda)))
    refused(sdb.NOT_SUPPORTED, lambda: sdb.mul_mat_q4(w, x, out=torch.empty(3, 8, device=cuda)))
    refused(sdb.NOT_SUPPORTED, lambda: sdb.mul_mat_q4(w, torch.zeros(64, 2, device=cuda).t(), out=out))
    refused(sdb.INVALID, lambda: sdb.mul_mat_q4(w, x.double(), out=out))
    refused(sdb.INVALID, lambda: sdb.mul_mat_q4(w, x.cpu(), out=out))
    refused(sdb.INVALID, lambda: sdb.mul_mat_q4(w, x, out=out, chain=sdb.Chain().add(torch.zeros(7, device=cuda))))
    refused(sdb.INVALID, lambda: sdb.mul_mat_q4(w, x.half(), out=out.half(),
                                                chain=sdb.Chain().redirect(torch.zeros(2, 8, device=cuda))))
    refused(sdb.INVALID, lambda: sdb.mul_mat_q4_gated(w, w, x, act="relu"))
    refused(sdb.INVALID, lambda: sdb.mul_mat_q4_gated(w, w, x, chain=sdb.Chain().add(torch.zeros(8, device=cuda))))
    refused(sdb.INVALID, lambda: sdb.mul_mat_q4_gated(w, w, x, out=out, chain=sdb.Chain().redirect(out)))
    other = on_device(cuda, *made(rng(2), 8, 64, 64, False)[:3], 64)
    refused(sdb.NOT_SUPPORTED, lambda: sdb.mul_mat_q4_gated(w, other, x))
    refused(sdb.INVALID, lambda: sdb.q4_quantize(torch.zeros(4, 4, 4, device=cuda)))
    refused(sdb.INVALID, lambda: sdb.q4_quantize(torch.zeros(4, 64, device=cuda), group=48))
    refused(sdb.INVALID, lambda: sdb.q4_quantize(torch.zeros(64, 4, device=cuda).t()))
    refused(sdb.INVALID, lambda: w.values(out=torch.empty(8, 64, device=cuda, dtype=torch.float16)))
    refused(sdb.INVALID, lambda: sdb.q4_import(torch.zeros(4, 16, device=cuda, dtype=torch.uint8),
                                               torch.zeros(4, 2, device=cuda, dtype=torch.float16)))
    refused(sdb.INVALID, lambda: sdb.q4_from_blocks(torch.zeros(4, 18, device=cuda, dtype=torch.uint8), 64))


# ---------------------------------------------------------------- groups that hold a NaN

@pytest.mark.parametrize("minimum", [False, True])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("k", [1, 33, 65, 129, 137, 300])
def test_a_short_last_group_of_nan(cuda, k, group, dtype, minimum):
    """Groups of nothing but NaN, short last ones and whole rows among them, stand for NaN; the others for what
    they stand for without them."""
    import sdb

    g = rng(k + group)
    w = g.standard_normal((20, k)).astype(dtype)
    bad = np.zeros(w.shape, dtype=bool)
    last = (k - 1) // group * group
    bad[3, last:], bad[17], bad[18, last:] = True, True, True
    w[3, last:], w[17], w[18, k - 1] = np.nan, np.nan, np.nan
    got = host(sdb.q4_quantize(cuda_tensor(w, cuda), group, minimum).values())
    np.testing.assert_array_equal(np.isnan(got), bad)
    np.testing.assert_array_equal(got[~bad], quantized(np.where(bad, dtype(1), w), group, minimum)[~bad])


# ---------------------------------------------------------------- what a call is described by

def test_copies_of_a_matrix(cuda):
    """A copied, pickled or saved matrix reads its own memory, and one whose memory is exchanged reads the new."""
    import copy
    import io
    import pickle

    import sdb
    import torch

    g = rng(41)
    q, scales, minima, values = made(g, 24, 96, 32, True)
    w = on_device(cuda, q, scales, minima, 32)
    x = cuda_tensor(g.standard_normal((3, 96)).astype(np.float32), cuda)
    want = host(sdb.mul_mat_q4(w, x))
    saved = io.BytesIO()
    torch.save(w, saved)
    saved.seek(0)
    for c in (copy.deepcopy(w), pickle.loads(pickle.dumps(w)), torch.load(saved, weights_only=False)):
        np.testing.assert_array_equal(host(c.values()), values.astype(np.float32))
        np.testing.assert_array_equal(host(sdb.mul_mat_q4(c, x)), want)
        c.data.zero_()
        assert (host(c.values()) == 0).all() and (host(sdb.mul_mat_q4(c, x)) == 0).all()
        np.testing.assert_array_equal(host(w.values()), values.astype(np.float32))
        c.data = w.data.clone()
        np.testing.assert_array_equal(host(sdb.mul_mat_q4(c, x)), want)
    for bad in (w.data[:-16], w.data.cpu(), w.data.view(torch.int8), w.data[::2], None):
        with pytest.raises(sdb.SdbError) as e:
            w.data = bad
        assert e.value.status == sdb.INVALID
    np.testing.assert_array_equal(host(sdb.mul_mat_q4(w, x)), want)


def test_a_redirect_exchanged(cuda):
    """A chain used again with a redirect of other strides, extents or type at the same address is refused."""
    import sdb
    import torch

    g = rng(42)
    q, scales, minima, values = made(g, 24, 64, 32, False)
    w = on_device(cuda, q, scales, minima, 32)
    x = g.standard_normal((24, 64)).astype(np.float32)
    t, r, out = cuda_tensor(x, cuda), torch.zeros(24, 24, device=cuda), torch.empty(24, 24, device=cuda)
    exact, mag = oracle.mul_mat_exact(values, x)
    chain = sdb.Chain().redirect(r)
    sdb.mul_mat_q4(w, t, out=out, chain=chain)
    check(host(r), exact, mag)
    r.fill_(7)
    for other in (r.t(), r.view(torch.int32), r.view(12, 48), r.view(1, 24, 24)):
        with pytest.raises(sdb.SdbError) as e:
            sdb.mul_mat_q4(w, t, out=out, chain=chain.redirect(other))
        assert e.value.status == sdb.INVALID
    assert (host(r) == 7).all()
    sdb.mul_mat_q4(w, t, out=out, chain=chain.redirect(r))
    check(host(r), exact, mag)


def test_operands_of_other_extents(cuda):
    """An operand whose extents are neither 1 nor the output's is refused, whatever lies behind it in its buffer;
    with strides of its own it has to lie within its buffer."""
    import sdb
    import torch

    g = rng(43)
    q, scales, minima, values = made(g, 8, 64, 32, False)
    w = on_device(cuda, q, scales, minima, 32)
    x = g.standard_normal((2, 64)).astype(np.float32)
    t = cuda_tensor(x, cuda)
    p = g.standard_normal((100,)).astype(np.float32)
    params = cuda_tensor(p, cuda)
    exact, mag = oracle.mul_mat_exact(values, x)
    for bad in (params[:7], params[:9], params[:21].view(3, 7), params[:24].view(3, 8), params[:14].view(2, 7),
                params[:3].view(3, 1), params[:32].view(2, 2, 8)):
        for chain in (sdb.Chain().add(bad), sdb.Chain().mul(bad)):
            with pytest.raises(sdb.SdbError) as e:
                sdb.mul_mat_q4(w, t, chain=chain)
            assert e.value.status == sdb.INVALID
    for bad in (params[:8], params[:15], params[:17]):  # the gated layer's chain has 2 N columns
        with pytest.raises(sdb.SdbError) as e:
            sdb.mul_mat_q4_gated(w, w, t, chain=sdb.Chain().add(bad))
        assert e.value.status == sdb.INVALID
    for good, b in ((params[:8], p[:8]), (params[:16].view(2, 8), p[:16].reshape(2, 8)), (params[4], p[4]),
                    (params[:2].view(2, 1), p[:2, None]), (params[:8].view(1, 1, 1, 8), p[:8]),
                    (params[:16:2], p[:16:2])):
        check(host(sdb.mul_mat_q4(w, t, chain=sdb.Chain().add(good))), exact + b, mag + np.abs(b))
    # Strides of its own: each column five apart, from any place that leaves room for them.
    b = p[60:100:5]
    check(host(sdb.mul_mat_q4(w, t, chain=sdb.Chain().add(params[60:61], [5, 0, 0, 0]))), exact + b, mag + np.abs(b))
    with pytest.raises(sdb.SdbError) as e:
        sdb.mul_mat_q4(w, t, chain=sdb.Chain().add(params[65:66], [5, 0, 0, 0]))
    assert e.value.status == sdb.INVALID


@pytest.mark.parametrize("call", ["quantize", "import", "blocks", "values", "linear", "gated"])
def test_memory_made_for_another_stream(cuda, call):
    """What a call on another stream makes is not memory that the current stream still writes."""
    import sdb
    import torch

    g = rng(44)
    w = cuda_tensor(g.standard_normal((256, 128)).astype(np.float32), cuda)
    x = cuda_tensor(g.standard_normal((64, 128)).astype(np.float32), cuda)
    q, scales, minima, _ = made(g, 256, 128, 32, False)
    codes, scales = cuda_tensor(codes_of(q), cuda), cuda_tensor(scales, cuda)
    blocks = cuda_tensor(g.integers(0, 60, (256, 72)).astype(np.uint8), cuda)
    m = sdb.q4_quantize(w)
    calls = {"quantize": lambda s: sdb.q4_quantize(w, stream=s).data,
             "import": lambda s: sdb.q4_import(codes, scales, stream=s).data,
             "blocks": lambda s: sdb.q4_from_blocks(blocks, 128, stream=s).data,
             "values": lambda s: m.values(stream=s),
             "linear": lambda s: sdb.mul_mat_q4(m, x, stream=s),
             "gated": lambda s: sdb.mul_mat_q4_gated(m, m, x, stream=s)}
    assert_apart(calls[call])


def assert_apart(call):
    """call(stream)'s tensors, made while the current stream still writes memory it has freed."""
    import torch

    tensors = lambda v: v if isinstance(v, tuple) else (v,)
    want = [t.clone() for t in tensors(call(None))]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)
    held = [torch.empty_like(t).fill_(1) for t in want]  # the blocks that the next such tensors would get
    del held
    got = tensors(call(side))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


# ---------------------------------------------------------------- every bit of x
#
# The bound here is the linear layers' own, 1e-6 of the magnitudes |x value| summed, with inputs whose sums hold
# nothing but what a wrong step would lose: numbers of x beside far greater ones whose weights are 0.  x enters
# the products whole, and a weight of 0 adds 0 whichever way it is 0, so the roundings left are those of sums of
# terms of the magnitudes counted, as in the tests above.

def beside_great_numbers(g, rows, k, n, group, kind, great, xt):
    """Rows of ordinary numbers with one great one in each 128 columns whose weight is 0: by code 8 of a symmetric
    matrix, by code 0 and no minimum, or by a code that the minimum meets (d q + m = 0)."""
    q, scales, minima, _ = made(g, n, k, group, kind != "code")
    scales = (g.integers(1, 128, scales.shape) * 2.0 ** -10 * g.choice([-1.0, 1.0], scales.shape)).astype(np.float16)
    at = np.arange(k) % 128 == 77 % min(k, 128)
    zero = {"code": 8, "least": 0}.get(kind)
    if kind == "least":
        minima = np.zeros_like(scales)
    if kind == "inside":
        z = g.integers(0, 16, scales.shape)
        minima = (-scales.astype(np.float64) * z).astype(np.float16)  # 7 bits by 4: exact
        zero = np.repeat(z, group, axis=1)[:, :k][:, at]
    q[:, at] = zero
    d = np.repeat(scales.astype(np.float64), group, axis=1)[:, :k]
    m = np.repeat(minima.astype(np.float64), group, axis=1)[:, :k] if minima is not None else -8 * d
    values = d * q + m
    assert (values[:, at] == 0).all()
    x = g.standard_normal((rows, k))
    x[:, at] *= great
    return q, scales, minima, values, x.astype(xt)


@pytest.mark.parametrize("kind", ["code", "least", "inside"])
@pytest.mark.parametrize("great", [300.0, 1e4, 1e6, 1e10, 1e20, 1e30])
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 7, 8, 9, 16, 17, 33])
def test_great_numbers_that_weigh_nothing(cuda, rows, great, kind):
    import sdb

    for group, k in ((32, 300), (64, 640), (128, 257)):
        q, scales, minima, values, x = beside_great_numbers(rng(rows + group), rows, k, 40, group, kind, great, np.float32)
        exact, mag = oracle.mul_mat_exact(values, x)
        check(host(sdb.mul_mat_q4(on_device(cuda, q, scales, minima, group), cuda_tensor(x, cuda))), exact, mag)


@pytest.mark.parametrize("kind", ["code", "least", "inside"])
@pytest.mark.parametrize("rows", [1, 2, 3, 8, 9, 17, 33])
def test_great_half_precision_numbers(cuda, rows, kind):
    import sdb
    import torch

    g = rng(rows)
    q, scales, minima, values, x = beside_great_numbers(g, rows, 400, 40, 32, kind, 1e4, np.float16)
    quiet = np.abs(x.astype(np.float64)) < 6
    x = np.where(quiet, x * np.float16(2.0 ** -10), x)
    exact, mag = oracle.mul_mat_exact(values, x)
    out = torch.empty(rows, 40, device=cuda)
    sdb.mul_mat_q4(on_device(cuda, q, scales, minima, 32), cuda_tensor(x, cuda), out=out)
    check(host(out), exact, mag)


@pytest.mark.parametrize("rows", [1, 2, 3, 5, 8, 9, 17, 33])
@pytest.mark.parametrize("gated", [False, True])
def test_one_number_a_column(cuda, rows, gated):
    """Each column of the output is one number of x, all other weights 0, the numbers of a row of any magnitudes."""
    import sdb

    g = rng(rows)
    k = 200
    q = np.full((k, k), 8, dtype=np.uint8)
    q[np.arange(k), np.arange(k)] = g.choice([0, 3, 7, 9, 15], k)
    scales = (1 + g.random((k, 7))).astype(np.float16)
    w = on_device(cuda, q, scales, None, 32)
    values = np.repeat(scales.astype(np.float64), 32, axis=1)[:, :k] * (q.astype(np.float64) - 8)
    x = (g.standard_normal((rows, k)) * 10.0 ** g.uniform(-15, 15, (rows, k))).astype(np.float32)
    exact, mag = oracle.mul_mat_exact(values, x)
    t = cuda_tensor(x, cuda)
    if gated:  # the gate's column: SiLU(40) = 40 to FP32's last bit
        got = host(sdb.mul_mat_q4_gated(w, on_device(cuda, q, np.zeros_like(scales), None, 32), t, "silu",
                                        chain=sdb.Chain().add(cuda_tensor(np.repeat(np.float32([0, 40]), k), cuda))))
        exact, mag = 40 * exact, 40 * mag
    else:
        got = host(sdb.mul_mat_q4(w, t))
    assert (np.abs(got - exact) <= oracle.K_B200 * mag).all()


@pytest.mark.parametrize("minimum", [False, True])
@pytest.mark.parametrize("rows", [1, 2, 3, 8, 9, 17, 33])
def test_the_smallest_numbers(cuda, rows, minimum):
    """Rows down to numbers below the normal ones, with scales that bring the sums back to normal numbers: the
    bound holds, and 2^-143 for some sixty sums rounded to 2^-149."""
    import sdb

    g = rng(rows)
    q, scales, minima, _ = made(g, 40, 300, 64, minimum)
    scales = (scales * np.float16(1000)).astype(np.float16)
    minima = (minima * np.float16(300)).astype(np.float16) if minimum else None
    d = np.repeat(scales.astype(np.float64), 64, axis=1)[:, :300]
    m = np.repeat(minima.astype(np.float64), 64, axis=1)[:, :300] if minimum else -8 * d
    w = on_device(cuda, q, scales, minima, 64)
    for scale in (1e-32, 1e-34, 3e-36, 1e-37, 1e-38, 1e-39, 1e-40):
        x = (g.standard_normal((rows, 300)) * scale).astype(np.float32)
        exact, mag = oracle.mul_mat_exact(d * q + m, x)
        got = host(sdb.mul_mat_q4(w, cuda_tensor(x, cuda)))
        worst = (np.abs(got - exact) / (oracle.K_B200 * mag + 2.0 ** -143)).max()
        assert worst <= 1, f"{scale}: {worst:.3g} of the bound"


@pytest.mark.parametrize("minimum", [False, True])
@pytest.mark.parametrize("rows", [1, 2, 3, 8, 9, 17, 33])
def test_sums_near_the_end_of_the_range(cuda, rows, minimum):
    """Great numbers and great scales: no sum on the way overflows where the output does not."""
    import sdb

    g = rng(rows)
    q, scales, minima, _ = made(g, 40, 256, 128, minimum)
    scales = (np.sign(scales) * g.uniform(20000, 60000, scales.shape)).astype(np.float16)
    d = np.repeat(scales.astype(np.float64), 128, axis=1)
    m = np.repeat(minima.astype(np.float64), 128, axis=1) if minimum else -8 * d
    w = on_device(cuda, q, scales, minima, 128)
    for exponent in (60, 70, 71, 72, 76, 84, 87, 88, 96):
        x = np.clip(g.standard_normal((rows, 256)), -1.9, 1.9).astype(np.float32) * np.float32(2.0 ** exponent)
        exact, mag = oracle.mul_mat_exact(d * q + m, x)
        check(host(sdb.mul_mat_q4(w, cuda_tensor(x, cuda))), exact, mag)


@pytest.mark.parametrize("kind", ["code", "inside", "below"])
@pytest.mark.parametrize("rows", [1, 2, 3, 8, 9, 17, 33])
def test_the_greatest_numbers(cuda, rows, kind):
    """Numbers up to FP32's greatest, with scales that bring the sums back: no sum of x alone overflows, whether its
    weight is 0 (no minimum or one that a code meets) or not."""
    import sdb

    g = rng(rows)
    n, k, group = 40, 300, 64
    q, scales, minima, _ = made(g, n, k, group, kind != "code")
    scales = (g.integers(1, 128, scales.shape) * 2.0 ** -20).astype(np.float16)
    if kind == "inside":
        minima = (-scales.astype(np.float64) * g.integers(0, 16, scales.shape)).astype(np.float16)
    elif kind == "below":
        minima = (-scales.astype(np.float64) * 24).astype(np.float16)
    d = np.repeat(scales.astype(np.float64), group, axis=1)[:, :k]
    m = np.repeat(minima.astype(np.float64), group, axis=1)[:, :k] if minima is not None else -8 * d
    w = on_device(cuda, q, scales, minima, group)
    for exponent in (112, 113, 114, 120, 126, 127):
        x = (g.uniform(1, 1.99, (rows, k)) * g.choice([1.0, 1.0, -1.0], (rows, k)) * 2.0 ** exponent).astype(np.float32)
        exact, mag = oracle.mul_mat_exact(d * q + m, x)
        assert mag.max() < 2.0 ** 127
        check(host(sdb.mul_mat_q4(w, cuda_tensor(x, cuda))), exact, mag)


# ---------------------------------------------------------------- rows that are held in parts

@pytest.mark.parametrize("minimum", [False, True])
@pytest.mark.parametrize("xt", [np.float32, np.float16])
@pytest.mark.parametrize("rows,k", [(1, 150001), (2, 90000), (2, 28672), (4, 60001), (7, 30000), (8, 28672)])
def test_long_rows(cuda, rows, k, xt, minimum):
    """Rows longer than the CTAs of a cluster hold at once, some k-blocks of one row with numbers of 1e-9 beside those
    of 1: digits and other k-blocks in one sum."""
    import sdb
    import torch

    g = rng(k)
    q, scales, minima, values = made(g, 20, k, 128, minimum)
    x = g.standard_normal((rows, k))
    x[:, ::1000] *= 1e-9 if xt == np.float32 else 1e-4
    x = x.astype(xt)
    out = torch.full((rows, 20), float("nan"), device=cuda)
    sdb.mul_mat_q4(on_device(cuda, q, scales, minima, 128), cuda_tensor(x, cuda), out=out)
    exact, mag = oracle.mul_mat_exact(values, x)
    check(host(out), exact, mag)


@pytest.mark.parametrize("minimum", [False, True])
@pytest.mark.parametrize("xt", [np.float32, np.float16])
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 6, 8, 9, 13, 16])
def test_gated_long_rows(cuda, rows, xt, minimum):
    """Two matrices of 16 k-blocks and more: the plan's other side for each form."""
    import sdb
    import torch

    g = rng(rows)
    k, half, group = 2100, 70, 64
    qa, qb = made(g, half, k, group, minimum), made(g, half, k, group, minimum)
    x = (g.standard_normal((rows, k)) / np.sqrt(k)).astype(xt)
    out = torch.full((rows, half), float("nan"), device=cuda)
    sdb.mul_mat_q4_gated(on_device(cuda, *qa[:3], group), on_device(cuda, *qb[:3], group), cuda_tensor(x, cuda), "silu",
                         out=out)
    a, ma = oracle.mul_mat_exact(qa[3], x)
    b, mb = oracle.mul_mat_exact(qb[3], x)
    act = b / (1 + np.exp(-b))
    check(host(out), a * act, ma * np.abs(act) + np.abs(a) * 1.13 * mb)
