"""The block operators' larger forms on the device: attention in chunks (lists that cross blocks), residual rows
dealt to a block in turn, wide rows, many nodes of spherical-harmonics features.  Each test first asserts that its
sizes take the form it is about, so that a changed rule cannot leave the form untested.  Tolerances as in
test_gpu_block_ops.py: the oracle's running error bounds."""
import ctypes
import math

import pytest
import torch

import nbody_amd._lib as lib
import nbody_amd.block_ops as B
from oracle import block_ops as O
from test_gpu_block_ops import (BF16, F16, F32, CALL, SEED, STEP, _attention_case, _lists, _rand, _residual_case,
                                _sh_case, rng)  # noqa: F401  (rng: a fixture)

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


# ------------------------------------------------------------------------------------------------ rows in turn
def _rows_in_turn(R, C, gates, slots):
    """Whether a row slot of the backward pass has several rows, from its partial rows (four per block)."""
    a = lib.ResidualNormArgs(rows=R, C=C, ldx=C, ldy=C, gate=8 if gates else None, gate_groups=gates)
    n = lib.c_sz()
    lib.check(lib.lib().nbx_residual_norm_backward_workspace_bytes(ctypes.byref(a), ctypes.byref(n)), "workspace")
    return R > n.value // (16 * C) * slots


SIXTEEN, MIXED, ALL32 = (BF16, BF16, BF16), (F32, F16, F32), (F32, F32, F32)


# slots: row slots of a block (16 lanes a row up to 128 columns, a wave up to 512, then whole waves).  Gates: one
# for all rows, groups longer and shorter than a block's share (several whole groups a slot among them), a gate a row
@pytest.mark.parametrize("R,C,gates,slots", [
    (13001, 24, 1, 16), (13001, 24, 13001, 16), (13000, 24, 2, 16), (52000, 24, 26000, 16),
    (3500, 200, 1, 4), (3500, 200, 3500, 4), (3500, 200, 5, 4), (16000, 136, 8000, 4),
    (4001, 520, 0, 2), (4000, 520, 4, 2), (4000, 520, 1000, 2), (6400, 520, 3200, 2),
    (1700, 1100, 1, 1), (1700, 1100, 850, 1), (1700, 1100, 1700, 1), (3400, 1100, 1700, 1)])
@pytest.mark.parametrize("types", [ALL32, SIXTEEN, MIXED], ids=["f32", "bf16", "f16_in_f32"])
def test_residual_rows_in_turn(hip_device, rng, R, C, gates, slots, types):   # noqa: F811
    assert _rows_in_turn(R, C, gates, slots)
    _residual_case(hip_device, rng, R, C, "layer" if C % 8 else "rms", *types, gates, True, True, True, 0.1, 0)


@pytest.mark.parametrize("R,C,gates", [(600, 2100, 1), (600, 2100, 2), (600, 2100, 300), (600, 2100, 600), (520, 4096, 1),
                                       (600, 4200, 1), (600, 4200, 2), (600, 4200, 300), (600, 4200, 600), (300, 8191, 0),
                                       (300, 8192, 1)])
@pytest.mark.parametrize("types", [ALL32, SIXTEEN, MIXED], ids=["f32", "bf16", "f16_in_f32"])
def test_residual_wide_rows_in_turn(hip_device, rng, R, C, gates, types):     # noqa: F811
    """Rows of eight and of sixteen waves, several to a block."""
    assert _rows_in_turn(R, C, gates, 1)
    _residual_case(hip_device, rng, R, C, "layer", *types, gates, True, True, True, 0.1, 7 if C % 8 else 0)


@pytest.mark.parametrize("post,pre", [(False, True), (True, False), (False, False)])
@pytest.mark.parametrize("R,C,gates", [(3500, 200, 5), (1700, 1100, 850), (600, 2100, 600), (600, 4200, 2)])
def test_residual_rows_in_turn_parts(hip_device, rng, R, C, gates, post, pre):   # noqa: F811
    _residual_case(hip_device, rng, R, C, "rms", *SIXTEEN, gates, post, pre, False, 0.2, 0)


@pytest.mark.parametrize("R,C,gates,slots", [
    (13001, 32, 1, 16), (13000, 32, 26, 16), (13001, 32, 13001, 16), (52000, 32, 26000, 16), (3500, 256, 5, 4),
    (16000, 256, 8000, 4), (4000, 1024, 4, 2), (4000, 1024, 1000, 2), (600, 2048, 1, 0), (1700, 2048, 850, 1),
    (600, 4096, 2, 1), (600, 4096, 300, 1), (600, 8192, 2, 1), (600, 8192, 300, 1), (600, 8192, 600, 1)])
@pytest.mark.parametrize("xt,yt", [(F32, F32), (BF16, BF16), (F32, F16)])
def test_residual_sums_over_rows_are_exact(hip_device, R, C, gates, slots, xt, yt):
    """Inputs whose every intermediate is a multiple of 2^-2 / C: the normed rows are +-1 (RMS norm of +-1 and of
    +-2 gate, eps 0), gates 1 and 2, gradients -1, 0, 1.  Sums over the rows are below 2^10, so that float32
    holds them exactly in any order, and a row that is lost, doubled or in another group shows."""
    assert not slots or _rows_in_turn(R, C, gates, slots)
    g = torch.Generator().manual_seed(R + C)
    sign = lambda *s: 2.0 * torch.randint(0, 2, s, generator=g) - 1                              # noqa: E731
    unit = lambda *s: torch.randint(-1, 2, s, generator=g).float()                               # noqa: E731
    x, y, one = torch.zeros(R, C, dtype=xt), sign(R, C).to(yt), torch.ones(C)
    gate = (1.0 + torch.arange(gates) % 2)[:, None].expand(gates, C).contiguous()
    dh, dz = unit(R, C).to(xt), unit(R, C).to(yt)
    ref = O.residual_norm(x, y, gate, (one, one * 0), (one, one * 0), "rms", 0.0, 2.0, torch.ones(R, C, dtype=torch.bool),
                          0.0, dh, dz)
    ins = [t.to(hip_device).requires_grad_() for t in (gate, one, one * 0, one, one * 0)]
    h, z = B.residual_norm(x.to(hip_device), y.to(hip_device), gate=ins[0], scale=2.0, post=(ins[1], ins[2]),
                           pre=(ins[3], ins[4]), eps=0.0)
    got = torch.autograd.grad((h, z), ins, (dh.to(hip_device), dz.to(hip_device)))
    for n, t in zip(("dgate", "dpost_w", "dpost_b", "dpre_w", "dpre_b"), got):
        assert torch.equal(t.double().cpu(), ref[n].val), n


# ------------------------------------------------------------------------------------------------ many nodes
@pytest.mark.parametrize("V,lmax,C", [(2501, 2, 64), (2050, 1, 9), (4099, 0, 40), (2049, 3, 61)])
@pytest.mark.parametrize("dtype,pt", [(F32, F32), (BF16, BF16), (F16, F32)])
def test_sh_waves_per_node(hip_device, rng, V, lmax, C, dtype, pt):           # noqa: F811
    """A wave per node (one or two chunks a lane), nodes that are no multiple of a block's four, several a wave."""
    assert V >= 2048 and V % 4 and (lmax + 1) ** 2 * -(-C // 8) <= 128
    _sh_case(hip_device, rng, V, lmax, C, dtype, pt, 0.2, 5, 0.1)


@pytest.mark.parametrize("V,lmax,C", [(700, 3, 80), (1100, 2, 250)])
@pytest.mark.parametrize("dtype,pt", [(BF16, F32), (F16, F16)])
def test_sh_nodes_in_turn(hip_device, rng, V, lmax, C, dtype, pt):            # noqa: F811
    """A block per node, several nodes in turn, in 16 bits."""
    assert V > 512 and (lmax + 1) ** 2 * -(-C // 8) > 128
    _sh_case(hip_device, rng, V, lmax, C, dtype, pt, 0.2, 5, 0.1)


@pytest.mark.parametrize("V,lmax,C", [(2501, 2, 64), (4099, 0, 40), (2049, 3, 16), (700, 3, 80), (1100, 6, 128)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sh_sums_over_nodes(hip_device, V, lmax, C, dtype):
    """Normed features of +-1 (up to the rounding of the degrees' balance: 32 half steps at most) and gradients of -1,
    0, 1: the bias gradient is exact and a lost or doubled node is 1 in the weight's."""
    g = torch.Generator().manual_seed(V)
    S = (lmax + 1) ** 2
    y = 2.0 * torch.randint(0, 2, (V, S, C), generator=g) - 1
    half = 2.0 * (torch.arange(C) % 2) - 1                       # the l = 0 row has no mean
    y[:, 0] = torch.stack([half[torch.randperm(C, generator=g)] for _ in range(V)])
    dz = torch.randint(-1, 2, (V, S, C), generator=g).float()
    w, b = (t.to(hip_device).requires_grad_() for t in (torch.ones(lmax + 1, C), torch.zeros(C)))
    x, y, dz = (t.to(dtype) for t in (torch.zeros(V, S, C), y, dz))
    _, z = B.sh_residual_norm(x.to(hip_device), y.to(hip_device), w, b, eps=0.0)
    dw, db = torch.autograd.grad(z, (w, b), dz.to(hip_device))
    assert torch.equal(db.cpu(), dz[:, 0].float().sum(0))
    deg = torch.tensor([l for l in range(lmax + 1) for _ in range(2 * l + 1)])
    want = torch.zeros(lmax + 1, C, dtype=torch.float64).index_add_(0, deg, (dz.double() * y.double()).sum(0))
    # 32 half steps of each term, and one per addition (fewer than 128 deep: nodes in turn, slots, degree)
    off = (dw.double().cpu() - want).abs()
    assert float(off.max()) <= 160 * 2.0 ** -24 * V * (2 * lmax + 1) < 0.2, float(off.max())
