"""What the 4-bit and residual entry points refuse before any memory is touched (no GPU needed)."""
from __future__ import annotations

import ctypes
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
LIB = ROOT / "stable-diffusion.assembly_b200" / "libsdb.so"


@pytest.fixture()
def sdb():
    if not LIB.exists():
        pytest.skip("libsdb.so not built")
    import sdb as binding

    binding.load()
    return binding


ADDRESS = 1 << 20  # never dereferenced


def tensor(sdb, ne, ty=0, nb=None, data=ADDRESS):
    es = 2 if ty else 4
    ne = list(ne) + [1] * (4 - len(ne))
    if nb is None:
        nb = [es]
        for d in range(3):
            nb.append(nb[-1] * ne[d])
    return sdb._TENSOR.pack(ty, *ne, *nb, data)


def q4(sdb, k, n, group=32, minimum=0, data=ADDRESS):
    return sdb._Q4.pack(data, k, n, group, minimum)


def test_struct_sizes(sdb):
    assert sdb._TENSOR.size == ctypes.sizeof(sdb.Tensor)
    assert sdb._STEP.size == ctypes.sizeof(sdb.Step)
    assert 8 + 6 * sdb._STEP.size + sdb._CHAIN_TAIL.size == ctypes.sizeof(sdb.ChainStruct)
    assert sdb._Q4.size == 32 and sdb._NORM_FORM.size == 24 and sdb._OPERAND.size == 40


def test_bytes(sdb):
    """Tiles of 16 rows x 128 columns: 1024 bytes of numbers and 32 a group of scales (and of minima)."""
    size = sdb.load().sdb_q4_bytes
    assert size(128, 16, 32, 0) == 1024 + 128
    assert size(128, 16, 64, 0) == 1024 + 64
    assert size(128, 16, 128, 1) == 1024 + 64
    assert size(129, 17, 32, 1) == 4 * (1024 + 256)
    assert size(8192, 28672, 128, 1) == 1792 * 64 * 1088
    for bad in ((0, 16, 32, 0), (128, 0, 32, 0), (128, 16, 48, 0), (128, 16, 256, 0), (128, 16, 32, 2),
                ((1 << 24) + 1, 1, 32, 0), (1, (1 << 30) + 1, 32, 0), (-1, 16, 32, 0)):
        assert size(*bad) == 0


def test_products_not_taken(sdb):
    lib = sdb.load()
    w, x, y = q4(sdb, 64, 8), tensor(sdb, [64, 3]), tensor(sdb, [8, 3])
    assert lib.sdb_mul_mat_q4_supported(w, x, y) == 1
    assert lib.sdb_mul_mat_q4_supported(w, tensor(sdb, [64, 3], 1), tensor(sdb, [8, 3], 1)) == 1
    assert lib.sdb_mul_mat_q4_gated_supported(w, w, x, y) == 1
    for bad in ((q4(sdb, 65, 8), x, y), (q4(sdb, 64, 9), x, y), (q4(sdb, 64, 8, data=0), x, y),
                (q4(sdb, 64, 8, data=ADDRESS + 8), x, y), (q4(sdb, 64, 8, 33), x, y), (None, x, y), (w, None, y),
                (w, x, None), (w, tensor(sdb, [64, 4]), y), (w, tensor(sdb, [64, 3], 7), y),
                (w, tensor(sdb, [64, 3], nb=[8, 512, 1536, 1536]), y),        # rows not contiguous
                (w, tensor(sdb, [64, 3], nb=[4, 258, 774, 774]), y),          # not whole elements
                (w, tensor(sdb, [64, 3], nb=[4, -256, 774, 774]), y),
                (w, x, tensor(sdb, [8, 3], nb=[4, 0, 96, 96])),               # rows written over one another
                (w, tensor(sdb, [64, 3], data=0), y), (w, tensor(sdb, [64, 3], data=ADDRESS + 2), y),
                (w, tensor(sdb, [64, 1 << 20, 1 << 20, 1]), tensor(sdb, [8, 1 << 20, 1 << 20, 1])),
                (w, tensor(sdb, [64, 1 << 62, 4, 1], nb=[4, 4, 4, 4]), tensor(sdb, [8, 1 << 62, 4, 1], nb=[4] * 4))):
        assert lib.sdb_mul_mat_q4_supported(*bad) == 0
        assert lib.sdb_mul_mat_q4(*bad, None, None) == sdb.NOT_SUPPORTED
    many = 1 << 20
    assert lib.sdb_mul_mat_q4_supported(w, tensor(sdb, [64, many]), tensor(sdb, [8, many])) == 1
    assert lib.sdb_mul_mat_q4_supported(w, tensor(sdb, [64, many + 1]), tensor(sdb, [8, many + 1])) == 0
    assert lib.sdb_mul_mat_q4_gated_supported(w, q4(sdb, 64, 8, 64), x, y) == 0
    assert lib.sdb_mul_mat_q4_gated_supported(w, q4(sdb, 64, 8, minimum=1), x, y) == 0
    assert lib.sdb_mul_mat_q4_gated_supported(w, q4(sdb, 64, 16), x, y) == 0
    assert lib.sdb_mul_mat_q4_gated_supported(w, None, x, y) == 0
    assert lib.sdb_mul_mat_q4_gated(w, w, x, y, 2, None, None) == sdb.INVALID
    # No rows: nothing is done.
    assert lib.sdb_mul_mat_q4(w, tensor(sdb, [64, 0], data=0), tensor(sdb, [8, 0], data=0), None, None) == sdb.OK


def test_chains_refused(sdb):
    lib = sdb.load()
    w, x, y = q4(sdb, 64, 8), tensor(sdb, [64, 3]), tensor(sdb, [8, 3])

    def chain(count=0, kind=0, operand=ADDRESS, redirect=0, from_redirect=0):
        c = sdb.ChainStruct()
        c.count, c.redirect, c.from_redirect = count, redirect or None, from_redirect
        c.steps[0].kind, c.steps[0].operand = kind, operand or None
        return ctypes.byref(c)

    for bad in (chain(7), chain(-1), chain(1, kind=3), chain(1, operand=0), chain(from_redirect=1),
                chain(1, kind=1, redirect=ADDRESS, from_redirect=1)):
        assert lib.sdb_mul_mat_q4(w, x, y, bad, None) == sdb.INVALID
    redirect = chain(redirect=ADDRESS)
    assert lib.sdb_mul_mat_q4(w, x, tensor(sdb, [8, 3], 1), redirect, None) == sdb.INVALID
    assert lib.sdb_mul_mat_q4_gated(w, w, x, y, 0, redirect, None) == sdb.INVALID


def test_matrices_refused(sdb):
    lib = sdb.load()
    q = q4(sdb, 64, 8)
    for bad in (tensor(sdb, [64, 9]), tensor(sdb, [63, 8]), tensor(sdb, [64, 8, 2]), tensor(sdb, [64, 8], data=0),
                tensor(sdb, [64, 8], nb=[4, 128, 128, 128]), tensor(sdb, [64, 8], nb=[8, 512, 512, 512]), None):
        assert lib.sdb_q4_quantize(bad, q, None) == sdb.INVALID
        assert lib.sdb_q4_dequantize(q, bad, None) == sdb.INVALID
    assert lib.sdb_q4_dequantize(q, tensor(sdb, [64, 8], 1), None) == sdb.INVALID
    assert lib.sdb_q4_import(None, ADDRESS, None, q, None) == sdb.INVALID
    assert lib.sdb_q4_import(ADDRESS, None, None, q, None) == sdb.INVALID
    assert lib.sdb_q4_import(ADDRESS, ADDRESS, ADDRESS, q, None) == sdb.INVALID
    assert lib.sdb_q4_import(ADDRESS, ADDRESS, None, q4(sdb, 64, 8, minimum=1), None) == sdb.INVALID
    assert lib.sdb_q4_import(ADDRESS, ADDRESS + 1, None, q, None) == sdb.INVALID
    assert lib.sdb_q4_from_blocks(ADDRESS, 35, q, None) == sdb.INVALID
    assert lib.sdb_q4_from_blocks(None, 36, q, None) == sdb.INVALID
    assert lib.sdb_q4_from_blocks(ADDRESS, 400, q4(sdb, 65, 8), None) == sdb.INVALID
    assert lib.sdb_q4_from_blocks(ADDRESS, 400, q4(sdb, 64, 8, 64), None) == sdb.INVALID


def residual(sdb, keep=1.0, scale=1.0, post=(0, 0.0), pre=(0, 0.0), gate=0, mul=0, add=0, nb=(0, 0, 0, 0)):
    form = lambda k, e: sdb._NORM_FORM.pack(k, e, 0, 0)
    return b"".join((sdb._KEEP_SCALE.pack(keep, scale), form(*post), form(*pre),
                     *(sdb._OPERAND.pack(a, *nb) for a in (gate, mul, add))))


def test_residual_refused(sdb):
    lib = sdb.load()
    t, t16, p = tensor(sdb, [64, 3]), tensor(sdb, [64, 3], 1), residual(sdb)
    call = lib.sdb_residual_norm
    for args in ((None, None, t, t, p), (t, t, None, None, p), (t, t, t, t, None), (t, tensor(sdb, [64, 4]), t, t, p),
                 (t, t, t, tensor(sdb, [65, 3]), p), (t, t, t16, t, p), (t, t, t, t16, p),
                 (tensor(sdb, [64, 3], 7), t, t, t, p), (tensor(sdb, [64, 3], data=0), t, t, t, p),
                 (t, tensor(sdb, [64, 3], nb=[8, 512, 1536, 1536]), t, t, p),
                 (t, t, tensor(sdb, [64, 3], nb=[4, 0, 0, 0]), t, p),
                 (t, t, t, t, residual(sdb, post=(3, 1e-5))), (t, t, t, t, residual(sdb, pre=(1, -1.0))),
                 (t, t, t, t, residual(sdb, pre=(1, float("nan")))),
                 (t, None, t, t, residual(sdb, post=(1, 1e-5))), (t, None, t, t, residual(sdb, gate=ADDRESS)),
                 (t, t, t, None, residual(sdb, pre=(2, 1e-5))), (t, t, t, None, residual(sdb, mul=ADDRESS)),
                 (t, t, t, t, residual(sdb, gate=ADDRESS, nb=(-1, 0, 0, 0))),
                 (t, t, t, t, residual(sdb, add=ADDRESS + 2)),
                 (*(tensor(sdb, [0, 3]),) * 4, p), (*(tensor(sdb, [64, 1 << 20, 1 << 20]),) * 4, p)):
        assert call(*args, None) == sdb.INVALID
    empty = tensor(sdb, [64, 0], data=0)
    assert call(empty, empty, empty, empty, p, None) == sdb.OK


def test_binding_refuses_host_tensors(sdb):
    import torch

    x = torch.zeros(2, 64)
    with pytest.raises(sdb.SdbError):
        sdb.residual_norm(x, x)
    with pytest.raises(sdb.SdbError):
        sdb.Norm("batch")
    with pytest.raises(sdb.SdbError):
        sdb.Norm("rms", weight=torch.zeros(4, 4))
    with pytest.raises(sdb.SdbError):
        sdb._packed_operand(torch.zeros(3, 1, 8), (2, 5, 8))
    with pytest.raises(sdb.SdbError):
        sdb.Norm("rms", weight=torch.zeros(4)).packed(5)




def test_operands_within_their_memory(sdb):
    """An operand with strides of its own is held to its memory, not to its count of numbers, and again on each use."""
    import numpy as np
    import torch

    out = torch.zeros(2, 8)
    numbers = np.zeros(40, dtype=np.float32)
    wide, short = torch.from_numpy(numbers)[:7], torch.from_numpy(numbers[:7])
    assert wide.data_ptr() == short.data_ptr() and wide.numel() == short.numel()

    def described(chain):
        return sdb._packed_chain(chain, sdb._chain_tensors(chain), out, 8)

    chain = sdb.Chain()
    chain.steps.append((sdb.STEP_ADD, wide, [1, 0, 0, 0]))
    assert len(described(chain)) == ctypes.sizeof(sdb.ChainStruct)
    chain.steps[0] = (sdb.STEP_ADD, short, [1, 0, 0, 0])
    # One number shown eight times, read as if there were eight of them.
    shown = sdb.Chain()
    shown.steps.append((sdb.STEP_ADD, torch.zeros(1).expand(8), [1, 0, 0, 0]))
    behind = sdb.Chain()
    behind.steps.append((sdb.STEP_ADD, wide, [-1, 0, 0, 0]))
    for bad in (chain, shown, behind):
        with pytest.raises(sdb.SdbError) as e:
            described(bad)
        assert e.value.status == sdb.INVALID
