"""The row operators' refusals (no GPU needed: invalid arguments are refused before anything is launched), and their
64-bit definitions against differences."""
import ctypes

import pytest
import torch

import flyhigh_engine_b200 as fh
from flyhigh_engine_b200 import kernels as K
from row_ops_plain import ffn, ffn64

INVALID = 1  # cudaErrorInvalidValue
P = 1 << 20  # an aligned address that nothing reads


def ffn_params(**kw):
    d = dict(x=P, w_gate=P, w_up=P, w_down=P, y=P, a=P, x_pitch=48, wg_pitch=48, wu_pitch=48, wd_pitch=192, y_pitch=48,
             h_pitch=192, m=10, cin=48, hidden=192, cout=48, act=0, dtype=0, scratch=P, scratch_bytes=1 << 40)
    d.update(kw)
    return K.GatedFfnParams(**d)


def grad_params(**kw):
    d = dict(x=P, w_gate=P, w_up=P, w_down=P, g=P, u=P, a=P, dy=P, dx=P, dw_gate=P, dw_up=P, dw_down=P, db_gate=P,
             db_up=P, db_down=P, x_pitch=48, wg_pitch=48, wu_pitch=48, wd_pitch=192, h_pitch=192, dy_pitch=48, dx_pitch=48,
             dwg_pitch=48, dwu_pitch=48, dwd_pitch=192, m=10, cin=48, hidden=192, cout=48, act=0, dtype=0, scratch=P,
             scratch_bytes=1 << 40)
    d.update(kw)
    return K.GatedFfnGradParams(**d)


def norm_params(**kw):
    d = dict(x=P, f=P, gate=P, scale=P, w_post=P, b_post=P, w_pre=P, b_pre=P, y=P, h=P, x_pitch=48, f_pitch=48, y_pitch=48,
             h_pitch=48, gate_pitch=48, m=12, c=48, gates=3, pre=2, post=1, eps=1e-6, dtype=1)
    d.update(kw)
    return K.ResidualNormParams(**d)


def norm_grad_params(**kw):
    d = dict(dy=P, dh=P, y=P, f=P, gate=P, scale=P, w_post=P, b_post=P, w_pre=P, dx=P, df=P, dgate=P, dscale=P, dw_post=P,
             db_post=P, dw_pre=P, db_pre=P, dy_pitch=48, dh_pitch=48, y_pitch=48, f_pitch=48, gate_pitch=48, dx_pitch=48,
             df_pitch=48, dgate_pitch=48, m=12, c=48, gates=3, pre=2, post=1, eps=1e-6, dtype=1, scratch=P,
             scratch_bytes=1 << 40)
    d.update(kw)
    return K.ResidualNormGradParams(**d)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(w_gate=None), dict(w_up=None), dict(w_down=None), dict(y=None), dict(a=None, g=P, u=P), dict(g=P), dict(u=P),
    dict(x=P + 8), dict(w_down=P + 2), dict(y=P + 4), dict(b_gate=P + 2), dict(b_down=P + 8), dict(x_pitch=40),
    dict(x_pitch=52), dict(wd_pitch=184), dict(h_pitch=196), dict(h_pitch=1 << 25), dict(y_pitch=0), dict(m=-1), dict(m=1 << 31), dict(cin=0),
    dict(hidden=-4), dict(cout=0), dict(cin=(1 << 20) + 1), dict(act=5), dict(act=-1), dict(dtype=2), dict(dtype=-1),
    dict(wait_cycles=-1)], ids=str)
def test_gated_ffn_refusals(bad):
    assert fh.lib().fhk_gated_ffn(ctypes.byref(ffn_params(**bad)), None) == INVALID


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(g=None), dict(u=None), dict(a=None), dict(g=None, u=None), dict(b_gate=P + 2), dict(dy=None), dict(w_up=None), dict(dx=P + 8), dict(dw_up=P + 2),
    dict(db_up=P + 6), dict(dx_pitch=44), dict(dwg_pitch=40), dict(dwd_pitch=8), dict(h_pitch=100), dict(h_pitch=1 << 40), dict(m=-5), dict(cin=0),
    dict(act=9), dict(dtype=3), dict(scratch=None), dict(scratch=P + 4), dict(scratch_bytes=100)], ids=str)
def test_gated_ffn_gradient_refusals(bad):
    assert fh.lib().fhk_gated_ffn_grad(ctypes.byref(grad_params(**bad)), None) == INVALID


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(f=None), dict(y=None), dict(h=None), dict(pre=0), dict(pre=3), dict(post=-1), dict(c=0), dict(c=8193),
    dict(m=-1), dict(m=1 << 31), dict(gates=5), dict(gates=0), dict(gates=-1), dict(gate=None), dict(gate=P + 1),
    dict(x=P + 2), dict(h=P + 8), dict(w_pre=P + 2), dict(b_pre=P + 2), dict(scale=P + 8), dict(x_pitch=47),
    dict(f_pitch=40), dict(gate_pitch=12), dict(eps=-1.0), dict(eps=float("nan")), dict(dtype=7)], ids=str)
def test_residual_norm_refusals(bad):
    assert fh.lib().fhk_residual_norm(ctypes.byref(norm_params(**bad)), None) == INVALID


@pytest.mark.parametrize("bad", [
    dict(dy=None, dh=None), dict(y=None), dict(pre=0), dict(f=None), dict(gate=None), dict(gates=5), dict(c=8193), dict(m=-1),
    dict(scale=None), dict(w_post=None), dict(w_pre=None), dict(dx=P + 2), dict(df_pitch=52), dict(dscale=P + 8),
    dict(db_pre=P + 2), dict(scratch=None), dict(scratch_bytes=16), dict(eps=-0.5), dict(dtype=-2)], ids=str)
def test_residual_norm_gradient_refusals(bad):
    assert fh.lib().fhk_residual_norm_grad(ctypes.byref(norm_grad_params(**bad)), None) == INVALID


def test_null_params():
    L = fh.lib()
    for fn in (L.fhk_gated_ffn, L.fhk_gated_ffn_grad, L.fhk_residual_norm, L.fhk_residual_norm_grad):
        assert fn(None, None) == INVALID
    for fn in (L.fhk_gated_ffn_scratch_bytes, L.fhk_gated_ffn_grad_scratch_bytes, L.fhk_residual_norm_grad_scratch_bytes):
        assert fn(None) == 0


def test_python_refusals_without_a_gpu():
    w = torch.zeros(16, 8, dtype=torch.float16)
    with pytest.raises(fh.FlyHighError, match="CUDA"):
        K.GatedFFN(w, w, w.t())
    with pytest.raises(fh.FlyHighError, match="unknown activation"):
        K.GatedFFN(w, w, w, act="swish2")
    with pytest.raises(fh.FlyHighError, match="unknown norm"):
        K.ResidualNorm(8, torch.float16, pre="batch")
    with pytest.raises(fh.FlyHighError, match="float16 or bfloat16"):
        K.ResidualNorm(8, torch.float32)
    with pytest.raises(fh.FlyHighError, match="channels"):
        K.ResidualNorm(8193, torch.float16)
    with pytest.raises(fh.FlyHighError, match="eps"):
        K.ResidualNorm(8, torch.float16, eps=float("inf"))
    with pytest.raises(fh.FlyHighError, match="norm that is none"):
        K.ResidualNorm(8, torch.float16, pre="none", w_pre=torch.ones(8))
    t = torch.zeros(6, 16, dtype=torch.float16)
    dev = t.device
    assert K._rows("t", t, 16, t.dtype, dev)[1:] == (16, 6)
    assert K._rows("t", t.view(2, 3, 16)[..., 8:], 8, t.dtype, dev)[1:] == (16, 6)
    assert K._rows("t", t[:1, :5], 5, t.dtype, dev)[1:] == (8, 1)
    assert K._rows("t", t[:0], 16, t.dtype, dev)[2] == 0
    assert K._rows("t", t.view(1, 6, 1, 16), 16, t.dtype, dev)[1:] == (16, 6)
    for bad in (t[:, 1:9], t.t()[:8, :], t[:1].expand(4, 16), torch.zeros(6, 12, dtype=torch.float16),
                torch.zeros(2, 3, 24, dtype=torch.float16).transpose(0, 1), t[:, ::2]):
        with pytest.raises(fh.FlyHighError):
            K._rows("t", bad, bad.shape[-1], t.dtype, dev)
    with pytest.raises(fh.FlyHighError, match="expected"):
        K._rows("t", t, 15, t.dtype, dev)
    with pytest.raises(fh.FlyHighError, match="expected"):
        K._rows("t", t, 16, torch.bfloat16, dev)


@pytest.mark.parametrize("act", list(K.ACTIVATIONS))
def test_gradient_formulas_against_differences(act):
    """The gradients the kernels are held to, against central differences of the forward definition: the directional
    derivative of sum(y * dy), whose difference quotient is off by about step^2 and 64-bit rounding over the step."""
    gen = torch.Generator().manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64).to(torch.bfloat16)
    m, c, f, o = 9, 11, 13, 7
    args = {"x": rnd(m, c), "w_gate": rnd(f, c), "w_up": rnd(f, c), "w_down": rnd(o, f), "b_gate": rnd(f), "b_up": rnd(f),
            "b_down": rnd(o)}
    dy = rnd(m, o)
    grads = ffn(*args.values(), act=act, dy=dy)
    base = {k: v.double() for k, v in args.items()}
    step = 1e-6
    for k in args:
        d = torch.randn(args[k].shape, generator=gen, dtype=torch.float64)
        lo, hi = ({**base, k: base[k] + s * step * d} for s in (-1, 1))
        loss = lambda a: (ffn64(*a.values(), act) * dy.double()).sum()
        slope = (loss(hi) - loss(lo)) / (2 * step)
        want = (grads[k][0] * d).sum()
        assert abs(slope - want) <= 1e-5 * (grads[k][0] * d).abs().sum(), (k, slope, want)
