"""Block operators, host side (block_ops.py, include/nbx.h "Block operators"): the generator's known answers,
the oracle's gradients against differences, every refusal, the argument structs."""
import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch
import torch.utils.checkpoint

import nbody_amd._lib as lib
import nbody_amd.block_ops as B
from oracle import block_ops as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ------------------------------------------------------------------------------------------------ the generator
@pytest.mark.parametrize("ctr,key,words", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))])
def test_generator_known_answers(ctr, key, words):
    """The published test vectors of Philox4x32-10 (zeros, ones, digits of pi)."""
    got = O.philox_words([np.array([c], np.uint64) for c in ctr], *key)
    assert tuple(int(w) for w in got[0]) == words


def test_draws_have_their_rate():
    n, p = 1 << 20, 0.1
    k = O.keep(1234567, 5, 9, np.arange(n), p)
    rate = 1 - O.threshold(p) / 65536
    assert abs(float(k.double().mean()) - rate) < 6 * (rate * (1 - rate) / n) ** 0.5
    other = O.keep(1234567, 6, 9, np.arange(n), p)
    both = float((k & other).double().mean())
    assert abs(both - rate ** 2) < 6 * (rate ** 2 * (1 - rate ** 2) / n) ** 0.5     # calls are independent


# ------------------------------------------------------------------------------------------------ oracle gradients
def _directional(f, tensors, grads, outs_grad, h=1e-5):
    """Central difference of <outs, outs_grad> along a random direction against <grads, direction> (float64)."""
    g = torch.Generator().manual_seed(1)
    dirs = [torch.randn(t.shape, generator=g, dtype=torch.float64) for t in tensors]
    val = lambda s: sum(float((o.val * d.double()).sum()) for o, d in zip(                    # noqa: E731
        f(*[t + s * h * d for t, d in zip(tensors, dirs)]), outs_grad))
    diff = (val(1.0) - val(-1.0)) / (2 * h)
    want = sum(float((g_.val * d).sum()) for g_, d in zip(grads, dirs))
    # truncation h^2 times a third derivative of order one per term, rounding 2^-52 / h of the summed terms
    size = sum(float((g_.val.abs() * d.abs()).sum()) for g_, d in zip(grads, dirs)) + 1.0
    assert abs(diff - want) < 1e-7 * size, (diff, want)


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_residual_oracle_gradients(kind):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)                          # noqa: E731
    R, C = 6, 11
    x, y, gate = r(R, C), r(R, C), r(3, C)
    pw, pb, qw, qb, dh, dz = r(C), r(C), r(C), r(C), r(R, C), r(R, C)
    k = O.keep(3, 1, 0, np.arange(R * C).reshape(R, C), 0.3)
    f = lambda *t: list(O.residual_norm(t[0], t[1], t[2], (t[3], t[4]), (t[5], t[6]), kind, 1e-5, 0.7, k,   # noqa: E731
                                        0.3).values())
    args = (x, y, gate, pw, pb, qw, qb)
    o = O.residual_norm(x, y, gate, (pw, pb), (qw, qb), kind, 1e-5, 0.7, k, 0.3, dh, dz)
    _directional(f, args, [o[n] for n in ("dx", "dy", "dgate", "dpost_w", "dpost_b", "dpre_w", "dpre_b")], (dh, dz))


def test_sh_oracle_gradients():
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)                          # noqa: E731
    x, y, w, b, dh, dz = r(4, 9, 5), r(4, 9, 5), r(3, 5), r(5), r(4, 9, 5), r(4, 9, 5)
    k = O.dropout_keep((4, 9, 5), "channel", 1, 3, 1, 0, 0.3)
    f = lambda *t: list(O.sh_residual_norm(*t, 1e-5, k, 1.4).values())                        # noqa: E731
    o = O.sh_residual_norm(x, y, w, b, 1e-5, k, 1.4, dh, dz)
    _directional(f, (x, y, w, b), [o[n] for n in ("dx", "dy", "dw", "db")], (dh, dz))


def test_attention_oracle_gradients():
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)                          # noqa: E731
    v, l, dout = r(12, 2, 3, 4), r(12, 3), r(4, 2, 3, 4)
    ptr, eid = torch.tensor([0, 5, 5, 6, 12]), torch.randperm(12, generator=g)
    k = O.keep(3, 1, 0, np.arange(36).reshape(12, 3), 0.3)
    f = lambda *t: [O.segment_attention(*t, ptr, eid, k, 0.3)["out"]]                         # noqa: E731
    o = O.segment_attention(v, l, ptr, eid, k, 0.3, dout)
    _directional(f, (v, l), [o["dvalues"], o["dlogits"]], (dout,))


# ------------------------------------------------------------------------------------------------ refusals
def _t(*s, dtype=torch.float32):
    return torch.zeros(*s, dtype=dtype)


RNG = torch.zeros(2, dtype=torch.int64)


@pytest.mark.parametrize("p", [-0.1, 1.0, 1.5, 1e-6, 1 - 1e-6, float("nan")])
def test_rates_that_cannot_be_drawn(p):
    with pytest.raises(ValueError):
        B.dropout(_t(4, 4), p, RNG, call=0)
    with pytest.raises(ValueError):
        B.residual_norm(_t(4, 4), _t(4, 4), p=p, rng=RNG, call=0)
    with pytest.raises(ValueError):
        B.sh_residual_norm(_t(4, 4, 4), _t(4, 4, 4), _t(2, 4), _t(4), channel_p=p, rng=RNG, call=0)
    with pytest.raises(ValueError):
        B.segment_attention(_t(4, 1, 2, 4), _t(4, 2), _t(3, dtype=torch.int32), _t(4, dtype=torch.int32), p=p, rng=RNG, call=0)


@pytest.mark.parametrize("kw,err", [
    (dict(per="row"), ValueError), (dict(group=0, per="group"), ValueError),
    (dict(x=_t(5), per="channel"), ValueError), (dict(x=_t(()), per="group"), ValueError),
    (dict(x=_t(4, 4, dtype=torch.float64)), TypeError), (dict(x=_t(4, 4, dtype=torch.int32)), TypeError)])
def test_dropout_refusals(kw, err):
    x = kw.pop("x", _t(4, 4))
    with pytest.raises(err):
        B.dropout(x, 0.1, RNG, call=0, **kw)


@pytest.mark.parametrize("kw,err", [
    (dict(y=_t(4, 7)), ValueError), (dict(y=_t(4, 6, dtype=torch.float64)), TypeError),
    (dict(x=_t(4, 6, dtype=torch.bfloat16)), TypeError), (dict(norm="batch"), ValueError),
    (dict(x=_t(4, 6, dtype=torch.bfloat16), y=_t(4, 6, dtype=torch.float16)), TypeError),
    (dict(pre=(_t(7), None)), ValueError), (dict(pre=(None, _t(6))), ValueError), (dict(post=(_t(6), _t(5))), ValueError),
    (dict(gate=_t(3, 6)), ValueError), (dict(gate=_t(5)), ValueError), (dict(gate=_t(0, 6)), ValueError),
    (dict(gate=_t(())), ValueError), (dict(group=-1), ValueError),
    (dict(gate=_t(6), pre=(_t(6, dtype=torch.bfloat16), None)), TypeError),
    (dict(gate=_t(6, dtype=torch.bfloat16)), TypeError), (dict(gate=_t(6, dtype=torch.float64)), TypeError),
    (dict(x=_t(2, 8193), y=_t(2, 8193)), ValueError), (dict(x=_t(2, 0), y=_t(2, 0)), ValueError),
    (dict(x=_t(()), y=_t(())), ValueError)])
def test_residual_refusals(kw, err):
    kw = {"x": _t(4, 6), "y": _t(4, 6), **kw}
    with pytest.raises(err):
        B.residual_norm(kw.pop("x"), kw.pop("y"), **kw)


@pytest.mark.parametrize("shape,ok", [
    ((6,), True), ((2, 6), True), ((10, 6), True), ((2, 5, 6), True), ((2, 1, 6), True), ((1, 1, 6), True),
    ((1, 5, 6), False), ((1, 2, 6), False), ((5, 2, 6), False), ((1, 2, 1, 6), False)])
def test_residual_gate_shapes(shape, ok):
    """A gate whose rows broadcasting would repeat is refused: its rows are for consecutive rows of y.  What is
    allowed gets as far as the device check."""
    with pytest.raises(lib.NbxError if ok else ValueError, match="HIP device" if ok else "gate"):
        B.residual_norm(_t(2, 5, 6), _t(2, 5, 6), gate=_t(*shape))


@pytest.mark.parametrize("y,gates,ok", [
    ((2, 5, 6), 5, False), ((2, 5, 6), 1, True), ((2, 5, 6), 2, True), ((5, 5, 6), 5, True), ((1, 5, 6), 5, True),
    ((2, 1, 6), 1, True), ((2, 4, 6), 4, False), ((2, 4, 6), 8, True), ((4, 10, 6), 20, True), ((2, 3, 5, 6), 5, False),
    ((2, 3, 5, 6), 6, True), ((2, 3, 6, 6), 6, True), ((2, 3, 5, 6), 15, True), ((20, 6), 20, True), ((20, 6), 5, True)])
def test_residual_gate_rows_are_not_broadcast(y, gates, ok):
    """A gate [N, C] for y [B, N, C] reads as broadcasting, which is not what a [G, C] gate means: refused where the
    two differ."""
    with pytest.raises(lib.NbxError if ok else ValueError, match="HIP device" if ok else "broadcasting"):
        B.residual_norm(_t(*y), _t(*y), gate=_t(gates, 6))


@pytest.mark.parametrize("kw,err", [
    (dict(x=_t(3, 5, 8), y=_t(3, 5, 8)), ValueError), (dict(x=_t(3, 64, 8), y=_t(3, 64, 8)), ValueError),
    (dict(x=_t(3, 4, 513), y=_t(3, 4, 513)), ValueError), (dict(x=_t(3, 32), y=_t(3, 32)), ValueError),
    (dict(y=_t(3, 4, 7)), ValueError), (dict(y=_t(3, 4, 8, dtype=torch.float16)), ValueError),
    (dict(weight=_t(3, 8)), ValueError), (dict(bias=_t(7)), ValueError), (dict(path_group=0), ValueError),
    (dict(weight=_t(2, 8, dtype=torch.float16)), TypeError), (dict(x=_t(3, 0, 8), y=_t(3, 0, 8)), ValueError),
    (dict(x=_t(3, 4, 8, dtype=torch.float64), y=_t(3, 4, 8, dtype=torch.float64)), TypeError)])
def test_sh_refusals(kw, err):
    kw = {"x": _t(3, 4, 8), "y": _t(3, 4, 8), "weight": _t(2, 8), "bias": _t(8), **kw}
    with pytest.raises(err):
        B.sh_residual_norm(**kw)


@pytest.mark.parametrize("kw,err", [
    (dict(values=_t(4, 2, 4)), ValueError), (dict(logits=_t(4, 3)), ValueError),
    (dict(logits=_t(4, 2, dtype=torch.bfloat16)), TypeError), (dict(values=_t(4, 1, 2, 4, dtype=torch.float64)), TypeError),
    (dict(ptr=_t(3, dtype=torch.int64)), ValueError), (dict(ptr=_t(0, dtype=torch.int32)), ValueError),
    (dict(eid=_t(3, dtype=torch.int32)), ValueError), (dict(eid=_t(4, dtype=torch.int64)), ValueError)])
def test_attention_refusals(kw, err):
    kw = {"values": _t(4, 1, 2, 4), "logits": _t(4, 2), "ptr": _t(3, dtype=torch.int32), "eid": _t(4, dtype=torch.int32), **kw}
    with pytest.raises(err):
        B.segment_attention(**kw)


def test_cpu_tensors_are_refused():
    for f in (lambda: B.dropout(_t(4, 4), 0.1, RNG, call=0), lambda: B.dropout(_t(4, 4), 0.0),
              lambda: B.residual_norm(_t(4, 4), _t(4, 4)),
              lambda: B.sh_residual_norm(_t(4, 4, 4), _t(4, 4, 4), _t(2, 4), _t(4)),
              lambda: B.segment_attention(_t(4, 1, 2, 4), _t(4, 2), _t(3, dtype=torch.int32), _t(4, dtype=torch.int32))):
        with pytest.raises(lib.NbxError, match="HIP device only"):
            f()


def test_rng_state():
    r = B.CounterRNG(-1, device="cpu", step=7)
    assert r.state.tolist() == [-1, 7] and (r.take(), r.take(2), r.take()) == (0, 1, 3)
    d = r.state_dict()
    r.advance(3)
    assert r.state.tolist() == [-1, 10] and r.take() == 0
    r.load_state_dict(d)
    assert r.state.tolist() == [-1, 7] and r.take() == 4
    assert B.CounterRNG(2 ** 64 - 1, device="cpu").state.tolist() == [-1, 0]
    cpu = torch.device("cpu")
    with pytest.raises(TypeError):
        B._draws(None, 0, 1, cpu)
    with pytest.raises(ValueError, match="explicit call"):
        B._draws(RNG, None, 1, cpu)
    for bad in (torch.zeros(3, dtype=torch.int64), torch.zeros(2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="state"):
            B._draws(bad, 0, 1, cpu)
    for call in (-1, 2 ** 32):
        with pytest.raises(ValueError, match="call"):
            B._draws(RNG, call, 1, cpu)
    with pytest.raises(ValueError, match="call"):
        B._draws(RNG, 2 ** 32 - 1, 2, cpu)


# ------------------------------------------------------------------------------------------------ the C ABI
def _res(**kw):
    a = lib.ResidualNormArgs(rows=4, C=8, ldx=8, ldy=8, x=8, y=8, h=8)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,msg", [
    (dict(rows=-1), b"rows"), (dict(C=0), b"C <= 8192"), (dict(C=8200, ldx=8200, ldy=8200), b"C <= 8192"),
    (dict(x_dtype=1), b"x_dtype"), (dict(y_dtype=7), b"x_dtype"), (dict(param_dtype=2), b"param_dtype"),
    (dict(norm=2), b"norm"), (dict(threshold=65536), b"threshold"), (dict(threshold=1), b"rng"),
    (dict(gate=8, gate_groups=3), b"gate_groups"), (dict(gate=8), b"gate_groups"), (dict(ldx=7), b"strides"),
    (dict(pre_b=8), b"weight"), (dict(x=None), b"null operand"), (dict(pre_w=8), b"null operand")])
def test_residual_abi_refusals(kw, msg):
    L = lib.lib()
    assert L.nbx_residual_norm(ctypes.byref(_res(**kw)), None) == 1
    assert msg in L.nbx_last_error()


@pytest.mark.parametrize("kw,rc,msg", [
    (dict(rows=0), 1, b"row"), (dict(post_w=8, y=8), 1, b"stats"), (dict(pre_w=8, dz=8, h=None, stats=8), 1, b"null h"),
    (dict(dgate=8), 1, b"not there"), (dict(dpre_w=8), 1, b"not there"), (dict(), 4, b"workspace")])
def test_residual_backward_abi_refusals(kw, rc, msg):
    L = lib.lib()
    assert L.nbx_residual_norm_backward(ctypes.byref(_res(**kw)), None) == rc
    assert msg in L.nbx_last_error()


def test_other_abi_refusals():
    L = lib.lib()
    n = lib.c_sz()
    assert L.nbx_residual_norm(None, None) == 1
    drop = lambda **k: L.nbx_dropout(*{**dict(dtype=0, per=0, n=4, S=1, C=1, group=1, threshold=10, rng=8, call=0,   # noqa: E731
                                              used=None, X=8, Y=8, stream=None), **k}.values())
    for kw in (dict(dtype=3), dict(per=3), dict(n=-1), dict(group=0), dict(threshold=65536), dict(X=None), dict(rng=None),
               dict(n=2 ** 41), dict(n=2 ** 39)):
        assert drop(**kw) == 1, kw
    assert drop(n=0) == 0
    sh = lib.ShResidualNormArgs(V=3, path_group=1, lmax=7, C=8, weight=8)
    assert L.nbx_sh_residual_norm(ctypes.byref(sh), None) == 1 and b"lmax" in L.nbx_last_error()
    sh.lmax, sh.path_threshold = 2, 5
    assert L.nbx_sh_residual_norm(ctypes.byref(sh), None) == 1 and b"rng" in L.nbx_last_error()
    sh.path_threshold = 0
    assert L.nbx_sh_residual_norm(ctypes.byref(sh), None) == 1 and b"null operand" in L.nbx_last_error()
    sh.stats, sh.dweight = 8, 8
    assert L.nbx_sh_residual_norm_backward(ctypes.byref(sh), None) == 4
    at = lib.SegmentAttentionArgs(V=3, E=4, K=1, H=65, D=4)
    assert L.nbx_segment_attention(ctypes.byref(at), None) == 1 and b"H <= 64" in L.nbx_last_error()
    at.H, at.D = 5, 999
    assert L.nbx_segment_attention(ctypes.byref(at), None) == 1 and b"H D" in L.nbx_last_error()
    at.H, at.D, at.l_dtype = 2, 4, 1
    assert L.nbx_segment_attention(ctypes.byref(at), None) == 1 and b"l_dtype" in L.nbx_last_error()
    at.l_dtype = 0
    assert L.nbx_segment_attention(ctypes.byref(at), None) == 1 and b"null operand" in L.nbx_last_error()
    at.ptr = at.eid = at.values = at.logits = at.stats = at.dout = at.dlogits = 8
    assert L.nbx_segment_attention_backward(ctypes.byref(at), None) == 4 and b"workspace" in L.nbx_last_error()
    assert L.nbx_segment_attention_workspace_bytes(ctypes.byref(at), 1, ctypes.byref(n)) == 0 and n.value >= 4 * 2 * 4


@pytest.mark.parametrize("V,E,ok", [(2 ** 24 - 1, 2 ** 31 - 257, True), (2 ** 24 - 1, 2 ** 31 - 256, False),
                                    (2 ** 24 - 1, 128 * (2 ** 24 - 1), False), (1, 2 ** 31 - 65, False), (2 ** 24, 4, False)])
def test_attention_largest_sizes(V, E, ok):
    """The list form's steps of 256 positions are counted in 32 bits: the last one may not pass 2^31 (2^24 - 1 lists
    of 128 edges would have).  What is allowed gets as far as the operand check."""
    L = lib.lib()
    at = lib.SegmentAttentionArgs(V=V, E=E, K=1, H=1, D=4)
    assert L.nbx_segment_attention(ctypes.byref(at), None) == 1
    assert (b"null operand" in L.nbx_last_error()) == ok


@pytest.mark.parametrize("name,mirror", [("nbx_residual_norm_args", lib.ResidualNormArgs),
                                         ("nbx_sh_residual_norm_args", lib.ShResidualNormArgs),
                                         ("nbx_segment_attention_args", lib.SegmentAttentionArgs)])
def test_struct_layouts(tmp_path, name, mirror):
    """Size and offsets of the ctypes mirrors against the C compiler."""
    fields = [f[0] for f in mirror._fields_]
    src = tmp_path / "o.c"
    src.write_text('#include "nbx.h"\n#include <stdio.h>\nint main(){printf("%%zu\\n", sizeof(%s));\n%s return 0;}\n' % (
        name, "".join('printf("%%zu\\n", offsetof(%s, %s));\n' % (name, f) for f in fields)))
    exe = tmp_path / "o"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(mirror)] + [getattr(mirror, f).offset for f in fields]


def test_next_call_is_refused_in_a_backward_pass():
    """A forward that runs again in the backward pass (activation checkpointing) must not draw anew."""
    rng = B.CounterRNG(0, "cpu")
    taken = []

    def body(x):
        taken.append(rng.take())
        return x * x
    x = torch.ones(3, requires_grad=True)
    y = torch.utils.checkpoint.checkpoint(body, x, use_reentrant=False)
    with pytest.raises(RuntimeError, match="explicit call"):
        y.sum().backward()
    assert taken == [0] and rng.take() == 1
