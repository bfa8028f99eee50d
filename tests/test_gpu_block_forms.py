"""The block operators' larger forms on the device: attention in chunks (lists that cross blocks).  Each test first asserts that its
sizes take the form it is about, so that a changed rule cannot leave the form untested.  Tolerances as in
test_gpu_block_ops.py: the oracle's running error bounds."""
import ctypes
import math

import pytest
import torch

import nbody_amd._lib as lib
import nbody_amd.block_ops as B
from oracle import block_ops as O
from test_gpu_block_ops import (BF16, F16, F32, CALL, SEED, STEP, _attention_case, _lists, _rand,
                                rng)  # noqa: F401  (rng: a fixture)

import numpy as np

pytestmark = pytest.mark.gpu
CODE = {F32: lib.F32, BF16: lib.BF16, F16: lib.F16}

# borders at multiples of 64, a list over several chunks, single edges, empty nodes at the ends and in between
RAGGED = [0, 64, 0, 64, 1, 63, 0, 0, 128, 200, 65, 63, 500, 3, 0]          # 1151 edges, 15 nodes


# ------------------------------------------------------------------------------------------------ attention in chunks
def _chunked(V, E, K, H, D, vt=F32):
    """Whether the forward pass takes the chunk form: only that one needs a workspace."""
    a = lib.SegmentAttentionArgs(V=V, E=E, K=K, H=H, D=D, v_dtype=CODE[vt], l_dtype=lib.F32)
    n = lib.c_sz()
    lib.check(lib.lib().nbx_segment_attention_workspace_bytes(ctypes.byref(a), 0, ctypes.byref(n)), "workspace")
    return n.value > 0


@pytest.mark.parametrize("K,H,D,vt,lt", [
    (9, 4, 4, F32, F32), (1, 8, 64, BF16, F32), (1, 8, 64, F16, F16), (3, 4, 24, BF16, BF16), (2, 3, 5, F32, F32),
    (2, 3, 5, BF16, F32), (2, 3, 5, F16, F16), (2, 3, 4, F16, F32),
    (9, 7, 7, F32, F32), (49, 8, 16, F32, F32), (25, 8, 16, BF16, F32),     # rows of several slices, 1 / 4 / 8 wide
    (1, 64, 1, F32, F32), (3, 64, 16, F32, F32), (1, 64, 8, BF16, BF16), (1, 1, 1, F32, F32), (1, 1, 4096, BF16, F32)])
@pytest.mark.parametrize("p,masked", [(0.2, 0.0), (0.1, 0.3)])
def test_chunk_form(hip_device, rng, K, H, D, vt, lt, p, masked):            # noqa: F811
    assert _chunked(len(RAGGED), sum(RAGGED), K, H, D, vt)
    _attention_case(hip_device, rng, RAGGED, K, H, D, vt, lt, p, masked)


@pytest.mark.parametrize("lengths", [[1100, 0, 0], [1, 1088], [64] * 16 + [1], [0] * 70 + [1025] + [0] * 70, [2] * 600 + [1],
                                     [1024, 0, 64, 63, 1], [63] * 17, [5, 0] * 220 + [0], [1025, 1025]])
def test_chunk_borders(hip_device, rng, lengths):                            # noqa: F811
    """Lists that end on, before and after a chunk's border, one list over all chunks, runs of empty nodes."""
    lengths = lengths if sum(lengths) % len(lengths) else lengths + [1]
    assert _chunked(len(lengths), sum(lengths), 2, 4, 8)
    _attention_case(hip_device, rng, lengths, 2, 4, 8, F32, F32, 0.1, 0.1)
    _attention_case(hip_device, rng, lengths, 1, 2, 16, BF16, F32, 0.1, 0.1)


def test_chunk_form_rows_that_leave_nothing(hip_device, rng):                # noqa: F811
    """Whole lists at -inf or at the type's lowest value, within a chunk and over several."""
    ptr, eid = _lists(RAGGED, 2)
    lists = {v: eid[ptr[v]:ptr[v + 1]].long() for v in range(len(RAGGED))}
    gone, low = (4, 8, 12), (5, 9)                                           # 1, 128 and 500 edges; 63 and 200

    def logits(l):
        for v in gone:
            l[lists[v]] = -math.inf
        for v in low:
            l[lists[v]] = torch.finfo(F32).min
        return l
    out, dv, dl = _attention_case(hip_device, rng, RAGGED, 2, 3, 4, F32, F32, 0.0, logits=logits, seed=2)
    for v in gone:
        assert not out[v].any() and not dv[lists[v]].any() and not dl[lists[v]].any()
    for v, n in enumerate(RAGGED):
        assert n or not out[v].any()


def test_chunk_form_some_chunks_all_masked(hip_device, rng):                 # noqa: F811
    """A list whose first chunks are all -inf and whose last holds the only weights, and the other way round."""
    lengths = [300, 700, 101]
    assert _chunked(3, sum(lengths), 1, 2, 8)
    ptr, eid = _lists(lengths, 3)

    def logits(l):
        l[eid[ptr[0]:ptr[0] + 280].long()] = -math.inf
        l[eid[ptr[1] + 20:ptr[2]].long()] = -math.inf
        return l
    _attention_case(hip_device, rng, lengths, 1, 2, 8, F32, F32, 0.2, logits=logits, seed=3)


def test_chunk_form_large_logits(hip_device, rng):                           # noqa: F811
    _attention_case(hip_device, rng, RAGGED, 1, 2, 4, F32, F32, 0.0, logits=lambda l: 1e4 * l)


def test_chunk_form_nan_stays_in_its_list(hip_device):
    ptr, eid = _lists(RAGGED, 0)
    for v in (3, 9, 12):                                                     # 64, 200 and 500 edges
        l = torch.zeros(len(eid), 2)
        l[eid[int(ptr[v]) + 2], 0] = math.nan
        out = B.segment_attention(torch.ones(len(eid), 1, 2, 4, device=hip_device), l.to(hip_device), ptr.to(hip_device),
                                  eid.to(hip_device))
        want = torch.tensor([[1.0 if n else 0.0] * 2 for n in RAGGED])
        assert torch.isnan(out[v, 0, 0]).all()
        want[v, 0] = math.nan
        torch.testing.assert_close(out[:, 0, :, 0].cpu(), want, rtol=1e-6, atol=0, equal_nan=True)


def test_chunk_form_masked_values_hold_anything(hip_device, rng):            # noqa: F811
    ptr, eid = _lists(RAGGED, 3)
    E, V = len(eid), len(RAGGED)
    r = _rand(6)
    v, l, dout = r(E, 2, 2, 4), r(E, 2), r(V, 2, 2, 4)
    l[eid[::7].long()] = -math.inf
    k = O.keep(SEED, CALL, STEP, np.arange(E * 2).reshape(E, 2), 0.4)
    off = ~k | torch.isinf(l)
    bad = torch.where(off[:, None, :, None], torch.tensor([math.nan, math.inf, -math.inf, math.nan]), v)
    ref = O.segment_attention(v, l, ptr, eid, k, 0.4, dout)
    vd, ld = bad.to(hip_device).requires_grad_(), l.to(hip_device).requires_grad_()
    out = B.segment_attention(vd, ld, ptr.to(hip_device), eid.to(hip_device), p=0.4, rng=rng, call=CALL)
    for n, t in zip(("out", "dvalues", "dlogits"), (out, *torch.autograd.grad(out, (vd, ld), dout.to(hip_device)))):
        O.within(t, ref[n], n)


def test_chunk_form_edges_in_no_list(hip_device, rng):                       # noqa: F811
    """A tail of more than a chunk behind the last list."""
    assert _chunked(len(RAGGED), sum(RAGGED) + 131, 2, 2, 4)
    ptr, eid = _lists(RAGGED, 0, extra=131)
    _, dv, dl = _attention_case(hip_device, rng, RAGGED, 2, 2, 4, F32, F32, 0.2, extra=131)
    rest = eid[int(ptr[-1]):].long()
    assert not dv[rest].any() and not dl[rest].any()


def test_chunk_form_entries_out_of_range(hip_device):
    """eid entries outside [0, E) count as masked, lists are cut at E."""
    ptr, eid = _lists(RAGGED, 0)
    E, V = len(eid), len(RAGGED)
    r = _rand(3)
    v, l, dout = r(E, 1, 2, 4), r(E, 2), r(V, 1, 2, 4)
    at = [0, 64, 127, 128, 600, 900, E - 1]
    gone = eid[at].long()
    masked = l.clone()
    masked[gone] = -math.inf
    ref = O.segment_attention(v, masked, ptr, eid, torch.ones(E, 2, dtype=torch.bool), 0.0, dout)
    bad, long = eid.clone(), ptr.clone()
    bad[at] = torch.tensor([E, -1, -2 ** 31, 2 ** 31 - 1, E + 7, -3, E], dtype=torch.int32)
    long[-1] = E + 100
    vd, ld = v.to(hip_device).requires_grad_(), l.to(hip_device).requires_grad_()
    out = B.segment_attention(vd, ld, long.to(hip_device), bad.to(hip_device))
    O.within(out, ref["out"], "out")
    dv, dl = torch.autograd.grad(out, (vd, ld), dout.to(hip_device))
    rest = torch.ones(E, dtype=torch.bool)
    rest[gone] = False
    for t, n in ((dv, "dvalues"), (dl, "dlogits")):
        O.within(t[rest.to(hip_device)], O.B(ref[n].val[rest], ref[n].err[rest]), n)
