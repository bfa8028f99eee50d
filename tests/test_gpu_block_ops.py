"""Block operators on the device (block_ops.py) against their formulas in float64 (oracle/block_ops.py), whose
running error bounds are the tolerances: half a step of float32 per operation, n half steps for a sum of n
terms in any order, half a step of the storage type for each stored result."""
import math

import numpy as np
import pytest
import torch
import torch.utils.checkpoint

import nbody_amd.block_ops as B
from oracle import block_ops as O

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
SEED, STEP, CALL = -6148914691236517205, 4294967299, 17


@pytest.fixture
def rng(hip_device):
    return torch.tensor([SEED, STEP], dtype=torch.int64, device=hip_device)


def _rand(seed):
    g = torch.Generator().manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g)


def _bits(a, b):
    v = {4: torch.int32, 2: torch.int16}[a.element_size()]
    return torch.equal(a.contiguous().view(v), b.contiguous().view(v))


# ------------------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape,per,group", [
    ((1,), "element", 1), ((7, 3), "element", 1), ((33, 129), "element", 1), ((5, 4, 3, 8), "element", 1),
    ((1, 1), "group", 1), ((13, 9, 8), "group", 5), ((40, 7), "group", 3), ((6, 3000), "group", 2), ((9,), "group", 2),
    ((1, 1), "channel", 1), ((11, 9, 16), "channel", 1), ((7, 4, 61), "channel", 1), ((3, 700), "channel", 1),
    ((2, 3, 2, 5), "channel", 1), ((3, 5, 1000), "channel", 1), ((4, 300, 9), "channel", 1),
    ((2, 3, 2047), "channel", 1), ((2, 1, 2048), "channel", 1), ((1, 3, 2049), "channel", 1), ((2, 2, 5001), "channel", 1),
    ((1, 40, 2070), "channel", 1), ((1, 700000), "channel", 1)])
def test_dropout(rng, dtype, shape, per, group):
    r = _rand(1)
    x, dy = r(*shape).to(dtype), r(*shape).to(dtype)
    xd = x.to(rng.device).requires_grad_()
    y = B.dropout(xd, 0.3, rng, call=CALL, per=per, group=group)
    (dx,) = torch.autograd.grad(y, xd, dy.to(rng.device))
    k = O.dropout_keep(shape, per, group, SEED, CALL, STEP, 0.3)
    for got, src in ((y, x), (dx, dy)):
        O.within(got, O.dropout(src, k, 0.3), per)
        assert torch.equal(got.detach().cpu() != 0, k & (src != 0))
    with torch.no_grad():
        assert _bits(B.dropout(xd, 0.3, rng, call=CALL, per=per, group=group), y.detach())


def test_dropout_dropped_places_hold_anything(rng):
    """Infinities and NaN where the draw drops give 0, in the value and in the gradient."""
    k = O.dropout_keep((64, 16), "element", 1, SEED, CALL, STEP, 0.5)
    x = torch.where(k, torch.ones(64, 16), torch.tensor([math.inf, math.nan] * 8).expand(64, 16))
    xd = x.to(rng.device).requires_grad_()
    y = B.dropout(xd, 0.5, rng, call=CALL)
    (dx,) = torch.autograd.grad(y, xd, x.to(rng.device))
    assert torch.equal(y.detach().cpu(), k.float() * 2) and torch.equal(dx.cpu(), k.float() * 2)


def test_dropout_views_empties_and_no_rate(rng):
    x = torch.randn(12, 10, device=rng.device)
    t = x.t()                                        # a transposed view: draws follow the logical order
    assert _bits(B.dropout(t, 0.2, rng, call=1), B.dropout(t.contiguous(), 0.2, rng, call=1))
    for s in ((0,), (0, 4), (3, 0)):
        assert B.dropout(torch.empty(*s, device=rng.device), 0.2, rng, call=1).shape == s
    assert B.dropout(x, 0.0) is x
    with pytest.raises(TypeError, match="rng"):
        B.dropout(x, 0.1)


# ------------------------------------------------------------------------------------------------ residual + norms
def _residual_case(dev, rng, R, C, kind, xt, yt, pt, gates, post, pre, bias, p, group, scale=0.75, seed=0):
    r = _rand(seed)
    x, y = r(R, C).mul(2).to(xt), r(R, C).to(yt)
    gate = (0.5 + r(gates, C)).to(pt) if gates else None
    norm = lambda on: ((1 + 0.3 * r(C)).to(pt), (0.3 * r(C)).to(pt) if bias else None) if on else None   # noqa: E731
    post, pre = norm(post), norm(pre)
    dh, dz = r(R, C).to(xt), r(R, C).to(yt)
    k = torch.ones(R, C, dtype=torch.bool)
    if p:
        k = (O.keep(SEED, CALL, STEP, np.arange(R) // group, p)[:, None].expand(R, C) if group
             else O.keep(SEED, CALL, STEP, np.arange(R)[:, None] * O.pad8(C) + np.arange(C)[None], p))
    ref = O.residual_norm(x, y, gate, post, pre, kind, 1e-5, scale, k, p, dh, dz)
    d = lambda t: None if t is None else t.to(dev).requires_grad_()                                     # noqa: E731
    xd, yd, gd = d(x), d(y), d(gate)
    postd, pred = (None if n is None else tuple(d(t) for t in n) for n in (post, pre))
    call = lambda a, b: B.residual_norm(a, b, gate=gd, scale=scale, post=postd, pre=pred, norm=kind, p=p,  # noqa: E731
                                        group=group, rng=rng if p else None, call=CALL)
    h, z = call(xd, yd)
    assert h.dtype == xt and (z is None or z.dtype == yt) and (z is None) == (pre is None)
    ins = {"dx": xd, "dy": yd}
    for n, t in (("dgate", gd), ("dpost_w", postd and postd[0]), ("dpost_b", postd and postd[1]),
                 ("dpre_w", pred and pred[0]), ("dpre_b", pred and pred[1])):
        if t is not None:
            ins[n] = t
    outs, grads = ((h, z), (dh.to(dev), dz.to(dev))) if pre else ((h,), (dh.to(dev),))
    got = dict(zip(ins, torch.autograd.grad(outs, tuple(ins.values()), grads)))
    got["h"] = h.detach()
    if pre:
        got["z"] = z.detach()
    with torch.no_grad():            # the inference form gives the same bits
        h2, z2 = call(xd, yd)
        assert _bits(h2, got["h"]) and (z2 is None or _bits(z2, got["z"]))
    for n, t in got.items():
        O.within(t, ref[n], n)
    return got


@pytest.mark.parametrize("R,C", [(1, 1), (1, 8), (3, 5), (37, 128), (5, 129), (18, 255), (7, 512), (4, 513), (3, 1999),
                                 (2, 4104), (2, 8192), (2, 8191), (300, 64)])
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_residual_sizes(hip_device, rng, R, C, kind):
    _residual_case(hip_device, rng, R, C, kind, F32, F32, F32, 1, True, True, True, 0.2, 0)


@pytest.mark.parametrize("xt,yt,pt", [(F32, F32, F32), (BF16, BF16, BF16), (BF16, BF16, F32), (F16, F16, F16),
                                      (F32, BF16, F32), (F32, F16, F16)])
@pytest.mark.parametrize("C", [96, 333, 1100])
def test_residual_types(hip_device, rng, xt, yt, pt, C):
    _residual_case(hip_device, rng, 22, C, "rms", xt, yt, pt, 2, True, True, True, 0.1, 0)
    _residual_case(hip_device, rng, 22, C, "layer", xt, yt, pt, 22, True, True, False, 0.1, 4)


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("pre", [False, True])
@pytest.mark.parametrize("gates", [0, 1, 7, 84])
@pytest.mark.parametrize("p,group", [(0.0, 0), (0.4, 0), (0.4, 5)])
def test_residual_parts(hip_device, rng, post, pre, gates, p, group):
    _residual_case(hip_device, rng, 84, 72, "layer", F32, F32, F32, gates, post, pre, True, p, group)


@pytest.mark.parametrize("R,C,gates", [(2100, 40, 1), (2100, 40, 7), (2100, 40, 700), (2100, 40, 2100), (1300, 600, 2),
                                       (1300, 600, 260), (1200, 300, 1), (1200, 300, 400)])
def test_residual_many_rows(hip_device, rng, R, C, gates):
    """Several rows per block and slot, gate groups longer and shorter than a block's share."""
    _residual_case(hip_device, rng, R, C, "rms", F32, F32, F32, gates, True, True, False, 0.1, 0)


def test_residual_strided_rows_and_leading_axes(hip_device):
    r = _rand(3)
    big = r(20, 3, 50).to(hip_device)
    x, y = big[:, 0, :48], big[:, 2, 1:49]            # rows 150 apart, unaligned
    w = (torch.ones(48, device=hip_device), None)
    a = B.residual_norm(x, y, pre=w, norm="layer")
    b = B.residual_norm(x.contiguous(), y.contiguous(), pre=w, norm="layer")
    c = B.residual_norm(x.reshape(4, 5, 48), y.reshape(4, 5, 48), pre=w, norm="layer")
    t = B.residual_norm(x.t().contiguous().t(), y.expand(20, 48), pre=w, norm="layer")
    for q in (b, t):
        assert _bits(a[0], q[0]) and _bits(a[1], q[1])
    assert c[0].shape == (4, 5, 48) and _bits(a[1], c[1].reshape(20, 48))


def test_residual_partial_gradients(hip_device):
    """Any subset of inputs and of output gradients: the others' gradients keep their bits."""
    r = _rand(4)
    mk = lambda *s: r(*s).to(hip_device).requires_grad_()                                   # noqa: E731
    x, y, gate, w, b = mk(30, 40), mk(30, 40), mk(40), mk(40), mk(40)
    dh, dz = r(30, 40).to(hip_device), r(30, 40).to(hip_device)
    f = lambda x, y, gate, w, b: B.residual_norm(x, y, gate=gate, post=(w, b), pre=(b, w), norm="layer")   # noqa: E731
    full = torch.autograd.grad(f(x, y, gate, w, b), (x, y, gate), (dh, dz))
    for i, t in enumerate((x, y, gate)):
        args = [a.detach() for a in (x, y, gate, w, b)]
        args[i] = t
        (g,) = torch.autograd.grad(f(*args), t, (dh, dz))
        assert _bits(g, full[i])
    only_h = torch.autograd.grad(f(x, y, gate, w, b)[0], (x, w), dh)     # z unused: dx = dh
    assert _bits(only_h[0], dh)
    only_z = torch.autograd.grad(f(x, y, gate, w, b)[1], (x, y), dz)
    zero = torch.autograd.grad(f(x, y, gate, w, b), (x, y), (torch.zeros_like(dh), dz))
    assert all(_bits(a, c) for a, c in zip(only_z, zero))


def test_residual_dropped_places_hold_anything(hip_device, rng):
    k = O.keep(SEED, CALL, STEP, np.arange(32)[:, None] * 16 + np.arange(16)[None], 0.5)
    y = torch.where(k, torch.ones(32, 16), torch.tensor(math.nan)).to(hip_device).requires_grad_()
    gate = torch.ones(16, device=hip_device, requires_grad=True)
    x = torch.zeros(32, 16, device=hip_device)
    h, _ = B.residual_norm(x, y, gate=gate, p=0.5, rng=rng, call=CALL)
    dy, dg = torch.autograd.grad(h, (y, gate), torch.ones_like(h))
    assert torch.equal(h.detach().cpu(), 2 * k.float()) and torch.equal(dy.cpu(), 2 * k.float())
    assert torch.equal(dg.cpu(), 2 * k.float().sum(0))


@pytest.mark.parametrize("R,C,gates", [(50, 40, 5), (50, 40, 10), (21, 600, 3), (7, 2100, 7), (100, 300, 4)])
def test_residual_bad_row_stays_in_its_group(hip_device, R, C, gates):
    """A row of NaN reaches its own results and its gate group's gradient, no other's."""
    r = _rand(2)
    x, y = r(R, C), r(R, C)
    y[0, 0] = math.nan
    ins = [t.to(hip_device).requires_grad_() for t in (x, y, 1 + 0.1 * r(gates, C), 1 + 0.1 * r(C), 1 + 0.1 * r(C))]
    h, z = B.residual_norm(ins[0], ins[1], gate=ins[2], post=(ins[3], None), pre=(ins[4], None), norm="layer")
    dx, dy, dg = torch.autograd.grad((h, z), ins[:3], (torch.ones_like(h), r(R, C).to(hip_device)))
    for t in (h, z, dx, dy):
        assert torch.isnan(t[0]).any() and torch.isfinite(t[1:]).all()
    assert torch.isnan(dg[0]).all() and torch.isfinite(dg[1:]).all()


def test_residual_empty(hip_device):
    w = torch.ones(8, device=hip_device)
    h, z = B.residual_norm(torch.empty(0, 8, device=hip_device), torch.empty(0, 8, device=hip_device), pre=(w, None))
    assert h.shape == z.shape == (0, 8)
    ins = [torch.zeros(s, device=hip_device, dtype=d, requires_grad=True)
           for s, d in (((0, 8), F32), ((0, 8), BF16), ((3, 8), F32), *[((8,), F32)] * 4)]
    h, z = B.residual_norm(ins[0], ins[1], gate=ins[2], post=(ins[3], ins[4]), pre=(ins[5], ins[6]))
    assert h.dtype == F32 and z.dtype == BF16
    for g, t in zip(torch.autograd.grad((h, z), ins, (torch.empty_like(h), torch.empty_like(z))), ins):
        assert g.shape == t.shape and not g.any()


def test_residual_far_rows(hip_device):
    """Rows far from the origin: the mean is taken out before squares are formed."""
    r = _rand(9)
    x = (1000.0 + r(6, 300)).to(hip_device)
    w = torch.ones(300, device=hip_device)
    _, z = B.residual_norm(x, torch.zeros_like(x), pre=(w, None), norm="layer")
    ref = O.residual_norm(x.cpu(), torch.zeros(6, 300), None, None, (w.cpu(), None), "layer", 1e-5, 1.0,
                          torch.ones(6, 300, dtype=torch.bool), 0.0)
    O.within(z, ref["z"], "z")
    # one rounding of h at 1000 is 2^-14: the value itself is good to that share of the deviation
    assert float((z.double().cpu() - ref["z"].val).abs().max()) < 1e-3


# ------------------------------------------------------------------------------------------------ spherical harmonics
def _sh_case(dev, rng, V, lmax, C, dtype, pt, path_p, group, channel_p):
    r = _rand(V + lmax)
    S = (lmax + 1) ** 2
    x, y, dh, dz = (r(V, S, C).to(dtype) for _ in range(4))
    w, b = (1 + 0.3 * r(lmax + 1, C)).to(pt), (0.3 * r(C)).to(pt)
    k, f = torch.ones(V, S, C, dtype=torch.bool), 1.0
    if path_p:
        k = k & O.dropout_keep((V, S, C), "group", group, SEED, CALL, STEP, path_p)
        f *= O.keep_scale(path_p)
    if channel_p:
        k = k & O.dropout_keep((V, S, C), "channel", 1, SEED, CALL + 1, STEP, channel_p)
        f *= O.keep_scale(channel_p)
    ref = O.sh_residual_norm(x, y, w, b, 1e-5, k, f, dh, dz)
    ins = [t.to(dev).requires_grad_() for t in (x, y, w, b)]
    run = lambda: B.sh_residual_norm(*ins, path_p=path_p, path_group=group, channel_p=channel_p,          # noqa: E731
                                     rng=rng if path_p or channel_p else None, call=CALL)
    h, z = run()
    got = dict(zip(("dx", "dy", "dw", "db"), torch.autograd.grad((h, z), ins, (dh.to(dev), dz.to(dev)))))
    got["h"], got["z"] = h.detach(), z.detach()
    for n, t in got.items():
        O.within(t, ref[n], n)
    with torch.no_grad():
        h2, z2 = run()
        assert _bits(h2, got["h"]) and _bits(z2, got["z"])


@pytest.mark.parametrize("V,lmax,C", [(1, 0, 1), (5, 0, 512), (3, 1, 7), (20, 2, 64), (11, 2, 61), (9, 3, 128), (7, 6, 16),
                                      (4, 6, 128), (3, 6, 512), (2, 5, 333), (130, 1, 8), (40, 4, 24), (2, 6, 250)])
def test_sh_sizes(hip_device, rng, V, lmax, C):
    _sh_case(hip_device, rng, V, lmax, C, F32, F32, 0.3, 5, 0.2)


@pytest.mark.parametrize("dtype,pt", [(F32, F32), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("path_p,channel_p", [(0.0, 0.0), (0.4, 0.0), (0.0, 0.4)])
def test_sh_types_and_rates(hip_device, rng, dtype, pt, path_p, channel_p):
    _sh_case(hip_device, rng, 25, 2, 48, dtype, pt, path_p, 5, channel_p)
    _sh_case(hip_device, rng, 9, 6, 40, dtype, pt, path_p, 2, channel_p)


def test_sh_many_nodes(hip_device, rng):
    _sh_case(hip_device, rng, 2500, 1, 8, F32, F32, 0.1, 5, 0.1)
    _sh_case(hip_device, rng, 700, 3, 80, F32, F32, 0.1, 5, 0.1)


def test_sh_equals_the_separate_operators(hip_device):
    """Without dropout: the framework's own norm of x + y."""
    from nbody_amd.eqv2_train import _RMSNormGFn
    r = _rand(0)
    x, y, w, b = (r(*s).to(hip_device) for s in ((50, 49, 128), (50, 49, 128), (7, 128), (128,)))
    h, z = B.sh_residual_norm(x, y, w, b, eps=1e-12)
    ref = _RMSNormGFn.apply(x + y, w, b, 1e-12, 6)
    assert _bits(h, x + y)
    torch.testing.assert_close(z, ref, rtol=2e-5, atol=2e-6)


def test_sh_partial_gradients_and_empty(hip_device):
    r = _rand(5)
    x, y, w, b, dh, dz = (r(*s).to(hip_device) for s in ((6, 4, 9), (6, 4, 9), (2, 9), (9,), (6, 4, 9), (6, 4, 9)))
    ins = [t.clone().requires_grad_() for t in (x, y, w, b)]
    full = torch.autograd.grad(B.sh_residual_norm(*ins), ins, (dh, dz))
    for i in range(4):
        a = [t.detach() for t in ins]
        a[i] = ins[i]
        (g,) = torch.autograd.grad(B.sh_residual_norm(*a), ins[i], (dh, dz))
        assert _bits(g, full[i])
    assert _bits(torch.autograd.grad(B.sh_residual_norm(*ins)[0], ins[0], dh)[0], dh)
    h, z = B.sh_residual_norm(torch.empty(0, 4, 9, device=hip_device), torch.empty(0, 4, 9, device=hip_device), w, b)
    assert h.shape == z.shape == (0, 4, 9)
    ins = [torch.zeros(s, device=hip_device, requires_grad=True) for s in ((0, 4, 9), (0, 4, 9), (2, 9), (9,))]
    h, z = B.sh_residual_norm(*ins)
    for g, t in zip(torch.autograd.grad((h, z), ins, (torch.empty_like(h), torch.empty_like(z))), ins):
        assert g.shape == t.shape and not g.any()


# ------------------------------------------------------------------------------------------------ segment attention
def _lists(lengths, seed, extra=0):
    g = torch.Generator().manual_seed(seed)
    ptr = torch.tensor([0] + list(np.cumsum(lengths)), dtype=torch.int32)
    return ptr, torch.randperm(int(ptr[-1]) + extra, generator=g).to(torch.int32)


def _attention_case(dev, rng, lengths, K, H, D, vt, lt, p, masked=0.0, extra=0, logits=None, seed=0):
    ptr, eid = _lists(lengths, seed, extra)
    E = len(eid)
    r = _rand(seed + 1)
    v, l, dout = r(E, K, H, D).to(vt), 3 * r(E, H), r(len(lengths), K, H, D).to(vt)
    if masked:
        l = l.masked_fill(torch.rand(E, H, generator=torch.Generator().manual_seed(seed)) < masked, -math.inf)
    l = (l if logits is None else logits(l)).to(lt)
    k = O.keep(SEED, CALL, STEP, np.arange(E * H).reshape(E, H), p) if p else torch.ones(E, H, dtype=torch.bool)
    ref = O.segment_attention(v, l, ptr, eid, k, p, dout)
    vd, ld = v.to(dev).requires_grad_(), l.to(dev).requires_grad_()
    pd, ed = ptr.to(dev), eid.to(dev)
    run = lambda: B.segment_attention(vd, ld, pd, ed, p=p, rng=rng if p else None, call=CALL)     # noqa: E731
    out = run()
    dv, dl = torch.autograd.grad(out, (vd, ld), dout.to(dev))
    for n, t in (("out", out), ("dvalues", dv), ("dlogits", dl)):
        O.within(t, ref[n], n)
    with torch.no_grad():
        assert _bits(run(), out.detach())
    return out.detach(), dv, dl


@pytest.mark.parametrize("K,H,D", [(1, 1, 1), (1, 8, 64), (9, 4, 4), (49, 8, 16), (9, 2, 7), (1, 5, 7), (3, 64, 16),
                                   (1, 1, 4096), (2, 3, 24), (25, 8, 4), (1, 7, 146), (4, 16, 128), (1, 64, 1)])
@pytest.mark.parametrize("lengths", [[4] * 6, [0, 1, 70, 3, 0], [200, 64, 0, 130]])
def test_attention_sizes(hip_device, rng, K, H, D, lengths):
    if K * H * D > 3000:
        lengths = [min(n, 70) for n in lengths]
    _attention_case(hip_device, rng, lengths, K, H, D, F32, F32, 0.2)


@pytest.mark.parametrize("vt,lt", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("K,H,D", [(9, 4, 4), (1, 8, 64), (2, 3, 5), (3, 4, 24)])
@pytest.mark.parametrize("p,masked", [(0.0, 0.3), (0.3, 0.0)])
def test_attention_types(hip_device, rng, vt, lt, K, H, D, p, masked):
    _attention_case(hip_device, rng, [3, 0, 5, 9], K, H, D, vt, lt, p, masked)
    _attention_case(hip_device, rng, [70, 0, 129, 64], K, H, D, vt, lt, p, masked)


@pytest.mark.parametrize("lengths", [[64, 64], [63, 1, 65], [128], [1000, 0, 0, 24], [0, 0, 40], [1] * 130, [640]])
def test_attention_chunk_borders(hip_device, rng, lengths):
    """Lists that end on, before and after a chunk's border; one list over many chunks."""
    _attention_case(hip_device, rng, lengths, 2, 4, 8, F32, F32, 0.1, 0.1)


def test_attention_rows_that_leave_nothing(hip_device, rng):
    """All -inf: 0, with gradients of 0; all at the type's lowest value: the mean."""
    for lengths in ([5, 3, 0], [90, 70, 0]):
        n = lengths[0]
        ptr, eid = _lists(lengths, 2)

        def logits(l, ptr=ptr, eid=eid):
            l[eid[:ptr[1]].long()] = -math.inf
            l[eid[ptr[1]:].long()] = torch.finfo(F32).min
            return l
        out, dv, dl = _attention_case(hip_device, rng, lengths, 2, 3, 4, F32, F32, 0.0, logits=logits, seed=2)
        assert not out[0].any() and not out[2].any()
        assert not dv[eid[:n].long()].any() and not dl[eid[:n].long()].any()


@pytest.mark.parametrize("lengths", [[6, 4], [80, 90]])
def test_attention_masked_values_hold_anything(hip_device, rng, lengths):
    """The values of masked and of dropped edges may be infinite or NaN."""
    ptr, eid = _lists(lengths, 3)
    E = len(eid)
    r = _rand(6)
    v, l, dout = r(E, 2, 2, 4), r(E, 2), r(2, 2, 2, 4)
    l[eid[0]] = -math.inf
    k = O.keep(SEED, CALL, STEP, np.arange(E * 2).reshape(E, 2), 0.4)
    off = ~k | torch.isinf(l)
    bad = torch.where(off[:, None, :, None], torch.tensor([math.nan, math.inf, -math.inf, math.nan]), v)
    ref = O.segment_attention(v, l, ptr, eid, k, 0.4, dout)
    vd, ld = bad.to(hip_device).requires_grad_(), l.to(hip_device).requires_grad_()
    out = B.segment_attention(vd, ld, ptr.to(hip_device), eid.to(hip_device), p=0.4, rng=rng, call=CALL)
    for n, t in zip(("out", "dvalues", "dlogits"), (out, *torch.autograd.grad(out, (vd, ld), dout.to(hip_device)))):
        O.within(t, ref[n], n)


def test_attention_large_logits_and_nan(hip_device, rng):
    _attention_case(hip_device, rng, [9, 80, 70], 1, 2, 4, F32, F32, 0.0, logits=lambda l: 1e4 * l)
    ptr, eid = _lists([3, 3], 0)
    l = torch.zeros(6, 1)
    l[eid[0]] = math.nan
    out = B.segment_attention(torch.ones(6, 1, 1, 4, device=hip_device), l.to(hip_device), ptr.to(hip_device),
                              eid.to(hip_device))
    assert torch.isnan(out[0]).all() and torch.equal(out[1], torch.ones_like(out[1]))


@pytest.mark.parametrize("lengths", [[3, 2], [60, 50]])
def test_attention_edges_in_no_list(hip_device, rng, lengths):
    """Positions behind the last list: not read by any node, gradients of 0."""
    ptr, eid = _lists(lengths, 0, extra=17)
    _, dv, dl = _attention_case(hip_device, rng, lengths, 2, 2, 4, F32, F32, 0.2, extra=17)
    rest = eid[int(ptr[-1]):].long()
    assert not dv[rest].any() and not dl[rest].any()


@pytest.mark.parametrize("lengths", [[5, 3], [70, 60]])
def test_attention_entries_out_of_range(hip_device, lengths):
    """An eid entry outside [0, E) counts as masked; a list is cut at E."""
    ptr, eid = _lists(lengths, 0)
    E = len(eid)
    r = _rand(3)
    v, l, dout = r(E, 1, 2, 4), r(E, 2), r(2, 1, 2, 4)
    gone = eid[1].long().item()
    masked = l.clone()
    masked[gone] = -math.inf
    ref = O.segment_attention(v, masked, ptr, eid, torch.ones(E, 2, dtype=torch.bool), 0.0, dout)
    bad, long = eid.clone(), ptr.clone()
    bad[1] = E + 7 if lengths[0] == 5 else -3
    long[-1] = E + 100
    vd, ld = v.to(hip_device).requires_grad_(), l.to(hip_device).requires_grad_()
    out = B.segment_attention(vd, ld, long.to(hip_device), bad.to(hip_device))
    O.within(out, ref["out"], "out")
    dv, dl = torch.autograd.grad(out, (vd, ld), dout.to(hip_device))
    rest = torch.arange(E) != gone                    # the edge that no list names is not written
    for t, n in ((dv, "dvalues"), (dl, "dlogits")):
        O.within(t[rest.to(hip_device)], O.B(ref[n].val[rest], ref[n].err[rest]), n)


def test_library_refusals_reach_python(hip_device):
    from nbody_amd._lib import NbxError
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=hip_device)                # noqa: E731
    with pytest.raises(NbxError, match="H <= 64"):
        B.segment_attention(torch.zeros(1, 1, 65, 4, device=hip_device), torch.zeros(1, 65, device=hip_device), i32(0, 1), i32(0))
    with pytest.raises(NbxError, match="H D"):
        B.segment_attention(torch.zeros(1, 1, 2, 1001, device=hip_device), torch.zeros(1, 2, device=hip_device), i32(0, 1), i32(0))


def test_attention_empty(hip_device):
    dev = hip_device
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)                       # noqa: E731
    out = B.segment_attention(torch.empty(0, 2, 2, 4, device=dev), torch.empty(0, 2, device=dev), i32(0, 0, 0), i32())
    assert out.shape == (2, 2, 2, 4) and not out.any()
    out = B.segment_attention(torch.empty(0, 2, 2, 4, device=dev), torch.empty(0, 2, device=dev), i32(0), i32())
    assert out.shape == (0, 2, 2, 4)


@pytest.mark.parametrize("E", [1, 300])
def test_attention_without_nodes(hip_device, rng, E):
    """No node at all: every edge is in no list, its gradients are 0."""
    values = torch.ones(E, 2, 2, 4, device=hip_device, requires_grad=True)
    logits = torch.ones(E, 2, device=hip_device, requires_grad=True)
    eid = torch.arange(E, dtype=torch.int32, device=hip_device)
    del_me = [torch.full((E, 2, 2, 4), 7.0, device=hip_device), torch.full((E, 2), 7.0, device=hip_device)]
    del del_me   # what the gradients' memory may hold beforehand
    out = B.segment_attention(values, logits, torch.zeros(1, dtype=torch.int32, device=hip_device), eid, p=0.3, rng=rng, call=1)
    dv, dl = torch.autograd.grad(out, (values, logits), torch.empty_like(out))
    assert out.shape == (0, 2, 2, 4) and not dv.any() and not dl.any()


# ------------------------------------------------------------------------------------------------ across the operators
def _block(x, params, ptr, eid, rng, step_calls=True):
    """A block as the framework's training paths use the operators: attention over edges, gated residual with
    norms, spherical-harmonics residual, dropout."""
    V, E = ptr.numel() - 1, eid.numel()
    values = (x[eid.long()[torch.argsort(eid.long())] % V] * params["v"]).view(E, 4, 2, 4)
    logits = values.sum((1, 3)) * 0.3
    att = B.segment_attention(values, logits, ptr, eid, p=0.2, rng=rng).reshape(V, 32)
    h, z = B.residual_norm(x, att, gate=params["g"], post=(params["w"], None), pre=(params["w2"], params["b2"]),
                           norm="layer", p=0.1, rng=rng)
    y = B.dropout(torch.tanh(z), 0.1, rng)
    h2, z2 = B.sh_residual_norm(h.view(V, 4, 8), y.view(V, 4, 8), params["sw"], params["sb"], path_p=0.2, path_group=3,
                                channel_p=0.1, rng=rng)
    return (h2 * z2).sum()


def _block_inputs(dev):
    r = _rand(11)
    P = {n: r(*s).to(dev).requires_grad_() for n, s in (("v", (32,)), ("g", (32,)), ("w", (32,)), ("w2", (32,)), ("b2", (32,)),
                                                        ("sw", (2, 8)), ("sb", (8,)))}
    x = r(12, 32).to(dev).requires_grad_()
    ptr, eid = _lists([4, 0, 7, 1, 90, 3, 3, 3, 3, 3, 3, 3], 1)
    return x, P, ptr.to(dev), eid.to(dev)


def test_block_is_reproducible_and_moves_with_step_and_call(hip_device):
    x, P, ptr, eid = _block_inputs(hip_device)

    def run(step):
        rng = B.CounterRNG(5, hip_device, step)
        loss = _block(x, P, ptr, eid, rng)
        return [loss.detach(), *torch.autograd.grad(loss, [x, *P.values()])]
    a, b, c = run(3), run(3), run(4)
    assert all(_bits(u, v) for u, v in zip(a, b))
    assert not _bits(a[1], c[1])


def test_block_gradient_against_differences(hip_device):
    """Central difference of the whole block along a direction, in float32: rounding of the loss (a sum of
    about 400 terms of order one and their own chains, 2^-24 times a few hundred) over 2 h, and h^2 times third
    derivatives."""
    x, P, ptr, eid = _block_inputs(hip_device)
    r = _rand(13)
    with torch.no_grad():
        leaves = [x, *P.values()]
    dirs = [r(*t.shape).to(hip_device) / t.numel() ** 0.5 for t in leaves]

    def loss(s):
        rng = B.CounterRNG(5, hip_device, 3)
        q = [t + s * d for t, d in zip(leaves, dirs)]
        return _block(q[0], dict(zip(P, q[1:])), ptr, eid, rng)
    grads = torch.autograd.grad(loss(0.0), leaves)
    want = sum(float((g.double() * d.double()).sum()) for g, d in zip(grads, dirs))
    with torch.no_grad():
        diff = lambda h: (float(loss(h).double()) - float(loss(-h).double())) / (2 * h)      # noqa: E731
        d1, d2 = diff(0.02), diff(0.01)
        extrapolated, truncation = (4 * d2 - d1) / 3, abs(d1 - d2)
        noise = 2.0 ** -24 * 400 * float(loss(0.0).abs() + 100) / 0.01
    assert abs(extrapolated - want) <= noise + truncation, (extrapolated, want, noise, truncation)


def test_backward_draws_what_the_forward_drew(hip_device):
    """The state may move on between the passes: the backward pass keeps the pair the forward used."""
    rng = B.CounterRNG(1, hip_device)
    x = torch.ones(4096, device=hip_device, requires_grad=True)
    y = B.dropout(x, 0.5, rng)
    rng.advance()
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(dx, y.detach())


def test_recomputed_forward_draws_the_same(hip_device):
    """Activation checkpointing with explicit call numbers."""
    rng = B.CounterRNG(1, hip_device)
    r = _rand(3)
    x, w = (r(*s).to(hip_device).requires_grad_() for s in ((70, 33), (33,)))

    def body(x, w):
        y = B.dropout(x * x, 0.3, rng, call=4)
        return B.residual_norm(x, y, pre=(w, None), p=0.2, rng=rng, call=5)
    g = r(70, 33).to(hip_device)
    plain = torch.autograd.grad(body(x, w), (x, w), (g, g))
    again = torch.autograd.grad(torch.utils.checkpoint.checkpoint(body, x, w, use_reentrant=False), (x, w), (g, g))
    assert _bits(plain[0], again[0]) and _bits(plain[1], again[1])


def test_graph_capture_replays_new_draws(hip_device):
    """Forward, backward and the step's advance captured once; every replay equals the eager step, with eager
    work between the replays; a second graph of the same operators runs in between."""
    x, P, ptr, eid = _block_inputs(hip_device)
    leaves = [x, *P.values()]

    def step(rng):
        loss = _block(x, P, ptr, eid, rng)
        g = torch.autograd.grad(loss, leaves)
        rng.advance()
        return [loss.detach(), *g]
    eager = B.CounterRNG(9, hip_device, 100)
    want = [[t.clone() for t in step(eager)] for _ in range(4)]
    graphs = []
    for _ in range(2):
        rng = B.CounterRNG(9, hip_device, 100)
        side = torch.cuda.Stream(hip_device)
        side.wait_stream(torch.cuda.current_stream(hip_device))
        with torch.cuda.stream(side):
            step(rng)
        torch.cuda.current_stream(hip_device).wait_stream(side)
        rng.state[1] = 100
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(rng)
        rng.state[1] = 100
        graphs.append((g, out, rng))                       # the state is the caller's: it lives as long as the graph
    for i in range(4):
        for g, out, _ in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert all(_bits(a, b) for a, b in zip(out, want[i])), i
            step(B.CounterRNG(3, hip_device))              # eager work between


def test_other_stream(hip_device):
    """Work is queued on the caller's current stream."""
    x, P, ptr, eid = _block_inputs(hip_device)
    want = torch.autograd.grad(_block(x, P, ptr, eid, B.CounterRNG(2, hip_device)), x)[0]
    s = torch.cuda.Stream(hip_device)
    s.wait_stream(torch.cuda.current_stream(hip_device))
    with torch.cuda.stream(s):
        got = torch.autograd.grad(_block(x, P, ptr, eid, B.CounterRNG(2, hip_device)), x)[0]
    torch.cuda.current_stream(hip_device).wait_stream(s)
    assert _bits(got, want)


def test_no_second_derivatives(hip_device, rng):
    from nbody_amd._lib import NbxError
    x = torch.randn(8, 8, device=hip_device, requires_grad=True)
    with pytest.raises(NbxError, match="second derivatives"):
        torch.autograd.grad(B.dropout(x, 0.5, rng, call=1).square().sum(), x, create_graph=True)
