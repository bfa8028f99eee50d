"""The training compositions on block operators: EquiformerV2 with ``block_rng`` (residual adds, norms,
dropouts, attention), PONITA with ``fused_residual`` (layer scale + residual), against the default torch glue
with the same masks and against the fp64 oracles.  Tolerances are the training steps' own (fp32 device
arithmetic against fp64: predictions 1e-5 / 2e-5, gradients 2e-4 of a tensor's largest value); two fp32
computations are compared at twice that."""
import numpy as np
import pytest

import nbody_amd.eqv2_train as T
import test_gpu_ponita_train as PT
from oracle.graph import fc_edge_index
from test_gpu_eqv2_train import C4, SMALL, _check_grads, _inputs, _model, _oracle, _train_step

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ block operators
def _block_case(hip_device, cfg, rates, monkeypatch=None):
    """The composition with block operators against the default one given the same masks: (both runs)."""
    from nbody_amd.block_ops import CounterRNG
    from oracle import block_ops as O
    B, N = 4, 5
    loc, vel, mass, gauge, tgt = _inputs(B, N, seed=9)
    kw = dict(alpha_drop=rates[0], drop_path_rate=rates[1], proj_drop=rates[2])
    m = _model(cfg, hip_device, seed=3, **kw)
    m.block_rng = CounterRNG(77, hip_device, step=5)
    fused = _train_step(m, loc, vel, mass, gauge, tgt, hip_device)
    ref = _model(cfg, hip_device, seed=3, **kw)
    if monkeypatch is not None:
        # the same draws, in the order the operators take their calls: per block attention, residual (2), residual
        # (2); a rate of 0 takes none
        calls = iter(range(10 ** 6))
        held = {}

        def scaled(k, p):
            return k.to(hip_device).float() * O.keep_scale(p)

        def alpha(x, p, training=True, inplace=False):
            E, H = x.shape
            return x * scaled(O.keep(77, next(calls), 5, np.arange(E * H).reshape(E, H), p), p)

        def drop_path(self, x):
            held["call"] = next(calls) if rates[1] or rates[2] else None
            if rates[1] or rates[2]:
                next(calls)
            if not rates[1]:
                return x
            return x * scaled(O.dropout_keep(tuple(x.shape), "group", N, 77, held["call"], 5, rates[1]), rates[1])

        def proj_drop(self, x):
            if not rates[2]:
                return x
            return x * scaled(O.dropout_keep(tuple(x.shape), "channel", 1, 77, held["call"] + 1, 5, rates[2]), rates[2])
        monkeypatch.setattr(T.torch.nn.functional, "dropout", alpha)
        monkeypatch.setattr(T._Step, "drop_path", drop_path)
        monkeypatch.setattr(T._Step, "proj_drop", proj_drop)
    return fused, _train_step(ref, loc, vel, mass, gauge, tgt, hip_device)


@pytest.mark.parametrize("specialised", [False, True])
@pytest.mark.parametrize("rates", [(0.0, 0.0, 0.0), (0.1, 0.0, 0.0), (0.2, 0.3, 0.0), (0.1, 0.3, 0.2), (0.0, 0.0, 0.2)])
def test_block_operators_match_the_composition(hip_device, rates, specialised, monkeypatch):
    """model.block_rng: prediction and gradients equal the torch glue's with the same masks (both compute in
    fp32 in other orders: the training step's own tolerances)."""
    if specialised:
        monkeypatch.setenv("NBX_EQV2_SPECIALISED", "1")
    fused, ref = _block_case(hip_device, SMALL, rates, monkeypatch)
    scale = np.abs(ref[1]).max(0)
    assert (np.abs(fused[1] - ref[1]).max(0) <= 4e-5 * scale + 1e-7).all()
    _check_grads(fused[2], ref[2], rel=4e-4)


def test_block_operators_against_the_oracle(hip_device):
    """Without dropout: every gradient against the fp64 oracle."""
    from nbody_amd.block_ops import CounterRNG
    for cfg in (SMALL, C4):
        m = _model(cfg, hip_device)
        m.block_rng = CounterRNG(0, hip_device)
        loc, vel, mass, gauge, tgt = _inputs(3, 5, seed=35)
        rloss, rpred, rgrads = _oracle(m, cfg, loc, vel, mass, gauge, tgt)
        loss, pred, grads = _train_step(m, loc, vel, mass, gauge, tgt, hip_device)
        assert (np.abs(pred - rpred).max(0) <= 2e-5 * np.abs(rpred).max(0) + 1e-7).all()
        _check_grads(grads, rgrads)


def test_block_operators_draw_anew_and_repeat(hip_device):
    """Another step or call draws other masks; the same state repeats the step bit for bit."""
    from nbody_amd.block_ops import CounterRNG
    loc, vel, mass, gauge, tgt = _inputs(4, 5, seed=1)
    m = _model(SMALL, hip_device, seed=2, alpha_drop=0.1, drop_path_rate=0.2)

    def run(step):
        m.block_rng = CounterRNG(3, hip_device, step=step)
        return _train_step(m, loc, vel, mass, gauge, tgt, hip_device)
    a, b, c = run(1), run(1), run(2)
    for k in a[2]:
        np.testing.assert_array_equal(a[2][k], b[2][k])
    assert a[0] == b[0] and a[0] != c[0]
    m.eval()
    m.native_train = True
    e = [_train_step(m, loc, vel, mass, gauge, tgt, hip_device)[0] for _ in range(2)]
    assert e[0] == e[1]                       # no dropout in eval mode


@pytest.mark.parametrize("hidden,layers,num_ori,B,N,kw", [(32, 2, 10, 4, 5, dict(layer_scale=0.3)), (64, 2, 8, 3, 6, {}),
                                                          (32, 1, 6, 2, 3, dict(layer_scale=0.0))])
def test_ponita_fused_residual(hip_device, hidden, layers, num_ori, B, N, kw):
    """Every parameter gradient (the layer scale's among them) against the fp64 oracle, and the forward's bits
    against the two launches (one more rounding there: one unit at most)."""
    model = PT._model(hidden, layers, num_ori, hip_device, **kw)
    pos, vel, mass, tgt = PT._inputs(B, N, seed=hidden + layers)
    ei = fc_edge_index(B, N)
    PT._calibrate(model, pos, vel, mass, ei, hip_device, N)
    rloss, rpred, rgrads = PT._oracle(model, pos, vel, mass, ei, tgt)
    model.fused_residual = True
    loss, pred, grads = PT._train_step(model, pos, vel, mass, ei, tgt, hip_device, N)
    scale = np.abs(rpred).max(0)
    assert (np.abs(pred - rpred).max(0) <= 1e-5 * scale + 1e-7).all(), np.abs(pred - rpred).max(0) / scale
    assert abs(loss - rloss) <= 1e-5 * abs(rloss)
    PT._check_grads(grads, rgrads)


def test_defaults_are_the_reference_composition(hip_device):
    """Neither attribute is set by construction."""
    assert _model(SMALL, hip_device).block_rng is None
    assert PT._model(32, 1, 6, hip_device).fused_residual is False
