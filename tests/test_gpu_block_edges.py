"""Block operators on the device: calls at the edge of what their documentation allows."""
import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import nbody_amd.block_ops as B
from oracle import block_ops as O
from test_gpu_block_ops import BF16, F16, F32, _attention_case, _bits, _lists, _rand, rng  # noqa: F401

pytestmark = pytest.mark.gpu


def _operators(dev):
    """name -> (the operator as a function of its tensors, those tensors)."""
    r = _rand(0)
    t = lambda *s: r(*s).to(dev)                                                             # noqa: E731
    rng = torch.tensor([5, 1], dtype=torch.int64, device=dev)
    ptr, eid = (q.to(dev) for q in _lists([3, 0, 5], 1))
    return {
        "dropout": (lambda x: B.dropout(x, 0.3, rng, call=0), [t(6, 8)]),
        "residual_norm": (lambda x, y, g, w, b, w2, b2: B.residual_norm(x, y, gate=g, post=(w, b), pre=(w2, b2)),
                          [t(6, 8), t(6, 8), t(3, 8), t(8), t(8), t(8), t(8)]),
        "sh_residual_norm": (B.sh_residual_norm, [t(6, 4, 8), t(6, 4, 8), t(2, 8), t(8)]),
        "segment_attention": (lambda v, l: B.segment_attention(v, l, ptr, eid), [t(8, 3, 2, 4), t(8, 2)])}


OPERATORS = ("dropout", "residual_norm", "sh_residual_norm", "segment_attention")


# ------------------------------------------------------------------------------------------------ derivatives
@pytest.mark.parametrize("name", OPERATORS)
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(hip_device, name, grad):
    """A dual tensor in any place, recorded or not: its tangent would be lost."""
    from nbody_amd._lib import NbxError
    f, ins = _operators(hip_device)[name]
    for i, t in enumerate(ins):
        for mode in (torch.enable_grad, torch.no_grad):
            with forward_ad.dual_level(), mode():
                dual = forward_ad.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t))
                with pytest.raises(NbxError, match="forward-mode"):
                    f(*ins[:i], dual, *ins[i + 1:])
    f(*ins)                                            # plain tensors again


def _gradients(f, ins, seed=7):
    outs = f(*ins)
    outs = [o for o in (outs if isinstance(outs, tuple) else (outs,)) if o is not None]
    r = _rand(seed)
    return torch.autograd.grad(outs, ins, [r(*o.shape).to(o) for o in outs])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("name", OPERATORS)
def test_saved_tensors_with_other_strides(hip_device, name, dtype):
    """Hooks on saved tensors may give the values back in another order of memory."""
    f, ins = _operators(hip_device)[name]
    ins = [t.to(dtype).requires_grad_() for t in ins]
    want = _gradients(f, ins)
    turn = lambda t: t.transpose(0, -1).contiguous().transpose(0, -1) if t.dim() > 1 else t     # noqa: E731
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, turn):
        got = _gradients(f, ins)
    assert all(_bits(a, b) for a, b in zip(want, got))
    with torch.autograd.graph.save_on_cpu():
        got = _gradients(f, ins)
    assert all(_bits(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("name", OPERATORS)
def test_saved_tensors_of_another_kind_are_refused(hip_device, name):
    """One saved tensor after the other comes back with another type, another size or from another device."""
    from nbody_amd._lib import NbxError
    f, ins = _operators(hip_device)[name]
    ins = [t.requires_grad_() for t in ins]
    for change in (lambda t: t.to(torch.float16), lambda t: t.flatten()[:-1], lambda t: t.cpu()):
        seen = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: (seen.append(0), t)[1]):
            _gradients(f, ins)
        assert seen
        for i in range(len(seen)):
            at = []

            def unpack(t, i=i, at=at, change=change):
                at.append(0)
                return change(t) if len(at) == i + 1 else t
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
                with pytest.raises(NbxError, match="saved tensor"):
                    _gradients(f, ins)


# ------------------------------------------------------------------------------------------------ residual + norms
@pytest.mark.parametrize("C", [40, 300, 600, 2100, 4200])
@pytest.mark.parametrize("types", [(F32, F32, F32), (BF16, BF16, BF16), (F32, F16, F32)], ids=["f32", "bf16", "f16_in_f32"])
@pytest.mark.parametrize("norm,gates", [("rms", 0), ("layer", 1), ("layer", 4), ("rms", 24)])
@pytest.mark.parametrize("pre", [False, True])
def test_residual_dropped_rows_hold_anything(hip_device, C, types, norm, gates, pre):
    """Rows of a dropped group may hold infinities and NaN before their norm: results and every gradient are those
    of rows of zeros there."""
    xt, yt, pt = types
    r, dev, R = _rand(C), hip_device, 24
    rng = torch.tensor([11, 2], dtype=torch.int64, device=dev)
    kept = O.keep(11, 3, 2, torch.arange(R).numpy() // 2, 0.5)
    assert 4 < int(kept.sum()) < 20
    x, y, dh, dz = (r(R, C).to(dev, t) for t in (xt, yt, xt, yt))
    gate = (1 + 0.3 * r(gates, C)).to(dev, pt) if gates else None
    w, b, w2 = ((1 + 0.3 * r(C)).to(dev, pt) for _ in range(3))

    def run(fill):
        held = torch.where(kept.to(dev)[:, None], y, fill.to(dev, yt))
        ins = [t.clone().requires_grad_() for t in (x, held, w, b) + ((w2,) if pre else ()) + ((gate,) if gates else ())]
        h, z = B.residual_norm(ins[0], ins[1], gate=ins[-1] if gates else None, post=(ins[2], ins[3]),
                               pre=(ins[4], None) if pre else None, norm=norm, p=0.5, group=2, rng=rng, call=3)
        outs, grads = ((h, z), (dh, dz)) if pre else ((h,), (dh,))
        return [t.detach() for t in outs] + list(torch.autograd.grad(outs, ins, grads))
    want = run(torch.zeros(()))
    for fill in (torch.tensor(math.inf), torch.tensor(math.nan), torch.tensor([math.inf, -math.inf, 1.0, math.nan] * (C // 4))):
        for a, c in zip(want, run(fill)):
            assert torch.isfinite(c).all() and torch.equal(a, c)


# ------------------------------------------------------------------------------------------------ segment attention
@pytest.mark.parametrize("lengths", [[5, 3], [70, 0, 60], [0, 64, 1, 63, 200, 500, 3, 270, 0]])
@pytest.mark.parametrize("K,H,D,dtype", [(1, 2, 4, F32), (2, 3, 5, BF16), (1, 4, 64, F16), (49, 8, 16, F32)])
@pytest.mark.parametrize("needs", ["both", "values", "logits"])
def test_attention_edges_that_no_entry_names(hip_device, lengths, K, H, D, dtype, needs):
    """Where entries of eid lie outside [0, E), the edges that are missing get gradients of 0, whatever their memory
    held; the others' are those of a list without the entry."""
    ptr, eid = _lists(lengths, 0)
    E, V = len(eid), len(lengths)
    r = _rand(3)
    v, l, dout = r(E, K, H, D).to(dtype), r(E, H), r(V, K, H, D).to(dtype)
    at = sorted({0, 3, E // 2, E // 2 + 1, E - 1})
    gone, bad = eid[at].long(), eid.clone()
    bad[at] = torch.tensor([E, -1, 2 ** 31 - 1, -2 ** 31, -7][:len(at)], dtype=torch.int32)
    dev = hip_device
    vd, ld = v.to(dev).requires_grad_(needs != "logits"), l.to(dev).requires_grad_(needs != "values")
    out = B.segment_attention(vd, ld, ptr.to(dev), bad.to(dev))
    before = [torch.full((E, K, H, D), math.nan, device=dev, dtype=dtype), torch.full((E, H), math.nan, device=dev)]
    dout = dout.to(dev)
    del before   # what the gradients' memory may hold
    got = torch.autograd.grad(out, [t for t in (vd, ld) if t.requires_grad], dout)
    masked = l.clone()
    masked[gone] = -math.inf
    ref = O.segment_attention(v, masked, ptr, eid, torch.ones(E, H, dtype=torch.bool), 0.0, dout.cpu())
    for n, t in zip({"both": ("dvalues", "dlogits"), "values": ("dvalues",), "logits": ("dlogits",)}[needs], got):
        assert not t[gone.to(dev)].any(), n
        O.within(t, ref[n], n)


@pytest.mark.parametrize("runs", [(62,), (63,), (64,), (65,), (127,), (128,), (129, 62, 190), (4000,), (63, 64, 65, 700)])
@pytest.mark.parametrize("n", [3, 31, 300])
def test_attention_runs_of_empty_nodes(hip_device, rng, runs, n):             # noqa: F811
    """Many nodes that start at one position, inside a block of positions, at its ends and on either side."""
    lengths = [n]
    for i, k in enumerate(runs):
        lengths += [0] * k + [n + i]
    _attention_case(hip_device, rng, lengths, 1, 2, 4, F32, F32, 0.1)
    _attention_case(hip_device, rng, [0] * runs[0] + lengths + [0] * runs[-1], 1, 2, 4, F32, F32, 0.1, extra=5)
    if n == 300:   # in chunks
        _attention_case(hip_device, rng, lengths + [700, 5] + [0] * runs[0] + [60], 1, 2, 4, F32, F32, 0.1)


def test_attention_does_not_walk_empty_nodes(hip_device):
    """2^22 empty nodes between two lists of one block: 65536 dependent loads if they were walked 64 at a time (tens of
    milliseconds), a few if searched.  The best of five passes counts."""
    V, E, dev = 1 << 22, 61, hip_device
    ptr = torch.full((V + 1,), 30, dtype=torch.int32)
    ptr[0], ptr[-1] = 0, E
    r = _rand(1)
    v, l = r(E, 1, 2, 4).to(dev).requires_grad_(), r(E, 2).to(dev).requires_grad_()
    out = B.segment_attention(v, l, ptr.to(dev), torch.arange(E, dtype=torch.int32, device=dev))
    assert not out[1:-1].any()
    dout, times = torch.ones_like(out), []
    for _ in range(5):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        got = torch.autograd.grad(out, (v, l), dout, retain_graph=True)
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
    ref = B.segment_attention(v, l, torch.tensor([0, 30, E], dtype=torch.int32, device=dev),
                              torch.arange(E, dtype=torch.int32, device=dev))
    want = torch.autograd.grad(ref, (v, l), torch.ones_like(ref))
    assert all(_bits(p, q) for p, q in zip(got, want))
    assert min(times) < 4.0, times
