"""Operators around a training block's products (include/nbx.h "Block operators", csrc/block_ops.hip and
csrc/segment_attention.hip), each an autograd operator (csrc/block_ops_torch.cpp) on the caller's stream:

* :func:`dropout` — dropout of elements, of whole groups of rows (stochastic depth) or of channels, whose
  mask is never stored: forward and backward draw it from a counter;
* :func:`residual_norm` — the residual add of a block's output with its gate (layer scale), dropout and the
  LayerNorm or RMS norm before and after it, in one pass;
* :func:`sh_residual_norm` — the same with EquiformerV2's norm over spherical-harmonics coefficients;
* :func:`segment_attention` — softmax over the edges into a node, dropout of the weights and the weighted sum
  of the edges' values in one pass.

Activations are float32, bfloat16 or float16; sums, statistics and draws' factors are float32 and each
result is rounded once.  Every reduction has a fixed order: the same call gives the same bits.

Random numbers: ``rng`` is a :class:`CounterRNG`, or its state tensor with an explicit ``call``.  A draw is a
function of (seed, step, call, index) alone (Philox4x32-10), so a step can be repeated, captured into a graph
(the step is read on the device: ``rng.advance()`` between or inside replays gives new draws) and its
backward pass needs no mask.  The drop rate is resolved to 2^-16 and the scale is that of the resolved rate,
so the mean is exact.  A dropped element is 0 whatever it held.

First derivatives by backward passes only: ``create_graph`` and forward-mode (dual) tensors are refused.

Like the framework's other operators these run on the HIP device only.
"""
from __future__ import annotations

import math

import torch

from . import _lib

_CODE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_PER = {"element": _lib.DROP_ELEMENT, "group": _lib.DROP_GROUP, "channel": _lib.DROP_CHANNEL}
_NORM = {"layer": 0, "rms": 1}


class CounterRNG:
    """The state of the counter-based draws: a device tensor ``state`` (seed, step) and the number of the next
    call of this step.  Call :meth:`advance` once per training step; ``seed`` is any 64-bit integer."""

    def __init__(self, seed=0, device="cuda", step=0):
        seed = int(seed) & (2 ** 64 - 1)
        self.state = torch.tensor([seed - 2 ** 64 if seed >= 2 ** 63 else seed, int(step)], dtype=torch.int64,
                                  device=device)
        self._next = 0

    def take(self, calls=1):
        """The number of the step's next call (of ``calls`` consecutive ones).  Refused inside a backward pass:
        a forward that is run again there (activation checkpointing) has to draw as it did, so give its operators
        ``call`` explicitly and advance after the backward pass."""
        if torch._C._current_graph_task_id() != -1:
            raise RuntimeError("the next call's number was asked for inside a backward pass: a recomputed forward "
                               "needs an explicit call")
        c = self._next
        self._next += calls
        return c

    def advance(self, steps=1):
        """The next step, on the device (may be captured), with its calls counted from 0 again."""
        self.state[1:].add_(steps)
        self._next = 0

    def state_dict(self):
        return {"state": self.state.clone(), "next": self._next}

    def load_state_dict(self, d):
        self.state.copy_(d["state"])
        self._next = int(d["next"])


def _threshold(p):
    """The 16-bit threshold of a drop rate."""
    p = float(p)
    if not 0.0 <= p < 1.0:
        raise ValueError(f"the drop rate must be in [0, 1), got {p}")
    t = int(65536 * p + 0.5)
    if (t == 0 and p > 0.0) or t >= 65536:
        raise ValueError(f"drop rates are resolved to 2^-16: {p} cannot be told from {0 if t == 0 else 1}")
    return t


def _draws(rng, call, calls, device):
    """(state tensor, number of the first of ``calls`` calls)."""
    if isinstance(rng, CounterRNG):
        state = rng.state
        call = rng.take(calls) if call is None else call
    elif isinstance(rng, torch.Tensor):
        state = rng
        if call is None:
            raise ValueError("a state tensor needs an explicit call")
    else:
        raise TypeError("a drop rate needs rng, a CounterRNG or its state tensor")
    if state.dtype != torch.int64 or state.shape != (2,) or state.device != device:
        raise ValueError(f"the state must be int64 [2] on {device}, got {state.dtype} {list(state.shape)} on {state.device}")
    call = int(call)
    if not 0 <= call <= 2 ** 32 - calls:
        raise ValueError(f"call must be in [0, 2^32), got {call}")
    return state.contiguous(), call


def _device(*tensors):
    """The HIP device of the tensors (None entries are skipped); raises unless all are on it."""
    dev = tensors[0].device
    for t in tensors:
        if t is not None:
            if not t.is_cuda:
                raise _lib.NbxError("nbx ops run on the HIP device only; got a CPU tensor")
            if t.device != dev:
                raise ValueError(f"tensors on {dev} and on {t.device}")
    return dev


def _with_parameters(t, *params):
    """An empty tensor with the parameters (None entries are skipped) in its graph."""
    for p in params:
        if p is not None:
            t = t + p.flatten()[:1].sum().to(t.dtype)
    return t


def _dtype(t, what):
    code = _CODE.get(t.dtype)
    if code is None:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


# ---------------------------------------------------------------------------------------------- dropout
def dropout(x, p, rng=None, *, call=None, per="element", group=1):
    """``x`` with a share ``p`` of it set to 0 and the rest scaled by 1 / (1 - p).

    per="element": every element on its own.  per="group": ``group`` consecutive entries of the first axis share
    a draw (stochastic depth of a system's nodes).  per="channel": x [n, ..., C], one draw for each (entry,
    channel), shared by the axes between.  p = 0 returns ``x``."""
    threshold = _threshold(p)
    if per not in _PER:
        raise ValueError(f'per must be "element", "group" or "channel", got {per!r}')
    if int(group) < 1:
        raise ValueError(f"group must be at least 1, got {group}")
    code = _dtype(x, "x")
    if per != "element" and x.dim() < (1 if per == "group" else 2):
        raise ValueError(f"per={per!r} needs more axes than {list(x.shape)} has")
    dev = _device(x)
    if threshold == 0:
        return x
    state, call = _draws(rng, call, 1, dev)
    n = x.shape[0] if x.dim() and per != "element" else 1
    C = x.shape[-1] if per == "channel" else 1
    return _lib.torch_ops().dropout(x, state, code, _PER[per], n, x.numel() // max(n * C, 1), C, int(group), threshold, call)


# ---------------------------------------------------------------------------------------------- residual + norms
def _consecutive(gate, y):
    """Whether a gate row belongs to consecutive rows of y: one or two axes, or y's axes from the front, then ones.
    Not [N, C] for y [B, N, C], which broadcasting would repeat over B (unless N is B, or 1)."""
    if gate.dim() <= 2:
        lead = y.shape[:-1]
        return (gate.dim() < 2 or len(lead) < 2 or gate.shape[0] != lead[-1]
                or any(gate.shape[0] == math.prod(lead[:k]) for k in range(len(lead) + 1)))
    same = 0
    while same < gate.dim() - 1 and gate.shape[:same + 1] == y.shape[:same + 1]:
        same += 1
    return gate.dim() == y.dim() and all(s == 1 for s in gate.shape[same:-1])


def residual_norm(x, y, *, gate=None, scale=1.0, post=None, pre=None, norm="rms", eps=1e-5, p=0.0, group=0, rng=None,
                  call=None):
    """The residual stream after a block: ``h = x + scale * dropout(gate * u)`` with ``u = y`` or, with ``post``
    (weight, bias or None), the norm of y; and with ``pre`` (weight, bias or None) the norm of h that the next
    block reads.  Returns (h, z); z is None without ``pre``.

    x (the stream) and y (the block's output) [..., C] of one shape, C <= 8192; y of x's type, or of 16 bits
    under a float32 stream.  norm = "rms" or "layer" (biased variance), for both places.  gate: [C] (layer
    scale), [G, C] (one row for each rows / G consecutive rows, whatever y's axes are; refused for y [.., N, C] with
    G = N, which reads as a row for each N, unless G is also the product of y's first axes), y's shape, or y's
    leading axes followed by ones ([B, 1, C] for y [B, N, C]).  gate and the norms' parameters are all float32 or
    all of y's type; their gradients are column sums in float32, rounded once.  p: drop rate of every element, or
    with group > 0 of whole groups of that many consecutive rows."""
    if norm not in _NORM:
        raise ValueError(f'norm must be "rms" or "layer", got {norm!r}')
    threshold = _threshold(p)
    post_w, post_b = post if post is not None else (None, None)
    pre_w, pre_b = pre if pre is not None else (None, None)
    if (post is not None and post_w is None) or (pre is not None and pre_w is None):
        raise ValueError("a norm needs its weight")
    params = [t for t in (gate, post_w, post_b, pre_w, pre_b) if t is not None]
    if x.shape != y.shape or x.dim() < 1:
        raise ValueError(f"x {list(x.shape)} and y {list(y.shape)} must have one shape [..., C]")
    cx, cy = _dtype(x, "x"), _dtype(y, "y")
    if cx != cy and cx != _lib.F32:
        raise TypeError(f"y must have x's type, or x be float32: got {x.dtype} and {y.dtype}")
    C = x.shape[-1]
    if not 1 <= C <= 8192:
        raise ValueError(f"need 1 <= C <= 8192, got {C}")
    rows = x.numel() // C
    cp = _dtype(params[0], "gate and norm parameters") if params else _lib.F32
    if any(t.dtype != params[0].dtype for t in params) or cp not in (_lib.F32, cy):
        raise TypeError(f"gate and norm parameters must all be float32 or all {y.dtype}")
    for t in (post_w, post_b, pre_w, pre_b):
        if t is not None and t.shape != (C,):
            raise ValueError(f"a norm's parameters must be [{C}], got {list(t.shape)}")
    if gate is not None and (gate.dim() < 1 or gate.shape[-1] != C or (rows and gate.numel() == 0)
                             or rows % max(gate.numel() // C, 1) or not _consecutive(gate, y)):
        raise ValueError(f"gate {list(gate.shape)} must be [C], [G, C] with G dividing the {rows} rows (a row for "
                         f"consecutive rows: broadcasting over y's first axes is not done), y's leading axes followed by "
                         f"ones, or y's shape {list(y.shape)}")
    if int(group) < 0:
        raise ValueError(f"group must be at least 0, got {group}")
    dev = _device(x, y, *params)
    state = None
    if threshold:
        state, call = _draws(rng, call, 1, dev)
    if rows == 0:   # empty results that know their parameters: gradients of 0
        h = x + _with_parameters(y, gate, post_w, post_b)
        return h, (_with_parameters(h.to(y.dtype), pre_w, pre_b) if pre_w is not None else None)
    return _lib.torch_ops().residual_norm(x, y, gate, post_w, post_b, pre_w, pre_b, state, cx, cy, cp, _NORM[norm], eps,
                                          scale, threshold, int(group), call or 0)


# ---------------------------------------------------------------------------------------------- spherical harmonics
def sh_residual_norm(x, y, weight, bias, *, eps=1e-5, path_p=0.0, path_group=1, channel_p=0.0, rng=None, call=None):
    """The residual add of an EquiformerV2 block with the norm behind it: ``h = x + dropout(y)`` and z, the
    equivariant RMS norm of h (degree-balanced mean square over coefficients and channels, the l = 0 row
    centred over the channels, ``weight`` [lmax + 1, C] per degree, ``bias`` [C] on l = 0).  Returns (h, z).

    x, y [V, (lmax + 1)^2, C] of one type, lmax <= 6, C <= 512.  path_p: one draw for each ``path_group``
    consecutive nodes (the nodes of a system); channel_p: one for each (node, channel), shared by the
    coefficients.  With a rate the call takes two call numbers, ``call`` and ``call`` + 1."""
    t1, t2 = _threshold(path_p), _threshold(channel_p)
    code = _dtype(x, "x")
    if x.dim() != 3 or x.shape != y.shape or x.dtype != y.dtype:
        raise ValueError(f"x {x.dtype} {list(x.shape)} and y {y.dtype} {list(y.shape)} must be one [V, (lmax + 1)^2, C]")
    V, S, C = x.shape
    lmax = round(max(S, 1) ** 0.5) - 1
    if (lmax + 1) ** 2 != S or lmax > 6 or not 1 <= C <= 512:
        raise ValueError(f"need (lmax + 1)^2 coefficients with lmax <= 6 and 1 <= C <= 512, got {S} and {C}")
    if weight.shape != (lmax + 1, C) or bias.shape != (C,):
        raise ValueError(f"weight must be [{lmax + 1}, {C}] and bias [{C}], got {list(weight.shape)} and {list(bias.shape)}")
    cp = _dtype(weight, "weight")
    if bias.dtype != weight.dtype or cp not in (_lib.F32, code):
        raise TypeError(f"weight and bias must both be float32 or both {x.dtype}")
    if int(path_group) < 1:
        raise ValueError(f"path_group must be at least 1, got {path_group}")
    dev = _device(x, y, weight, bias)
    state = None
    if t1 or t2:
        state, call = _draws(rng, call, 2, dev)
    if V == 0:
        h = x + y
        return h, _with_parameters(h, weight, bias)
    return _lib.torch_ops().sh_residual_norm(x, y, weight, bias, state, lmax, code, cp, eps, t1, int(path_group), t2,
                                             call or 0)


# ---------------------------------------------------------------------------------------------- segment attention
def segment_attention(values, logits, ptr, eid, *, p=0.0, rng=None, call=None):
    """Attention over the edges into each node: ``out[v] = sum over v's edges of dropout(a[e, h]) values[e, :, h]``
    with a the softmax of the edges' ``logits`` over v's list.  Returns [V, K, H, D].

    values [E, K, H, D] (K rows per edge that share the heads' weights), logits [E, H] float32 or of values'
    type; ptr int32 [V + 1] and eid int32 [E]: the edges by destination, eid a permutation of the edges
    (``segnn_train.Graph``'s dptr / deid).  A node without edges, or whose logits are all -inf, gets 0; edges
    in no list (positions from ptr[V] on, or named by no entry of eid) get gradients of 0.  A weight that is exactly
    0 reads nothing of its value.  H <= 64, H D <= 4096 (1024 if D is no multiple of 4), K H D < 2^20, V < 2^24 and
    E < 2^31 - 256."""
    threshold = _threshold(p)
    cv, cl = _dtype(values, "values"), _dtype(logits, "logits")
    if values.dim() != 4 or logits.shape != (values.shape[0], values.shape[2]):
        raise ValueError(f"values must be [E, K, H, D] and logits [E, H], got {list(values.shape)} and {list(logits.shape)}")
    E, K, H, D = values.shape
    if cl not in (_lib.F32, cv):
        raise TypeError(f"logits must be float32 or {values.dtype}, got {logits.dtype}")
    if ptr.dtype != torch.int32 or eid.dtype != torch.int32 or ptr.dim() != 1 or ptr.numel() < 1 or eid.shape != (E,):
        raise ValueError(f"ptr must be int32 [V + 1] and eid int32 [{E}], got {ptr.dtype} {list(ptr.shape)} and "
                         f"{eid.dtype} {list(eid.shape)}")
    dev = _device(values, logits, ptr, eid)
    state = None
    if threshold:
        state, call = _draws(rng, call, 1, dev)
    return _lib.torch_ops().segment_attention(values, logits, ptr, eid, state, cv, cl, threshold, call or 0)
