"""Gate values over the whole range of the type, seen one by one: a single row of x that is a unit vector hands every hidden
channel the gate that its weight holds, u = 1 and da = 1, so that y is act(g), w_up's gradient is act(g) and w_gate's is
act'(g), each behind one rounding to the type (or two of the same value)."""
import itertools
import math
import random

import pytest
import torch

from flyhigh_engine_b200.kernels import ACTIVATIONS, GatedFFN
from row_ops_plain import SUBNORMAL, act64, assert_within, half_step

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16

MAGNITUDES = [0.0, 1e-3, 0.3, 1.0, 2.5, 4.0, 6.0, 8.0, 10.0, 14.0, 20.0, 41.0, 42.0, 60.0, 100.0, 200.0, 300.0, 1000.0, 1e4, 6e4,
              1e5, 1e6, 1e10, 1e18, 3e19, 1e30]
# rows, channels in, copies of the gates (each in another order, so that gates meet other neighbours): the forms for few rows, for
# feature maps (forward), and tiles
FORMS = {"rows": (4, 8, 2), "map": (200, 16, 2), "tiles": (200, 16, 4)}


def exposed(form, dtype, seed=0):
    """(x, w_gate, w_up, w_down, dy, gates) of the block described above."""
    m, c, copies = FORMS[form]
    gates = [s * g for g in MAGNITUDES for s in (1, -1) if g <= torch.finfo(dtype).max]
    rng, order = random.Random(seed), []
    for _ in range(copies):
        rng.shuffle(gates)
        order += gates
    h = len(order)
    g = torch.tensor(order, dtype=torch.float64, device="cuda").to(dtype)
    zeros = lambda *s: torch.zeros(s, dtype=dtype, device="cuda")
    x, wg, wu, wd, dy = zeros(m, c), zeros(h, c), zeros(h, c), zeros(h, h), zeros(m, h)
    assert h % 8 == 0 and (h <= 128) == (form != "tiles")
    x[m // 2, 0], dy[m // 2] = 1, 1
    wg[:, 0], wu[:, 0] = g, 1
    wd.fill_diagonal_(1)
    return x, wg, wu, wd, dy, g


def evaluation(act, g):
    """How far act(g) and act'(g) may be off before they are rounded. The sigmoid's argument z is known to 5 2^-24 of itself
    (its products and constants in f32), |z| < 42 where its power counts, and the power and the reciprocal to 2^-21: s and
    1 - s to 2^-16 of themselves, and 0 in place of s below 2^-60. erfc by 7.1.26: to 1.5e-7, and never above
    exp(-g^2 / 2); the power there to 2^-19 of itself."""
    s, v = 1 / (1 + torch.exp(-g)), act64(act, g)[0].abs()
    if act == "relu":
        return torch.zeros_like(g), torch.zeros_like(g)
    if act == "gelu":
        e = torch.exp(-g * g / 2)
        return g.abs() * e.clamp(max=2.0 ** -22) + 2.0 ** -40, e.clamp(max=2.0 ** -22) + g.abs() * e * 2.0 ** -19 + 2.0 ** -24
    d = act64(act, g)[1].abs()
    if act == "silu":
        d = s + g.abs() * s * (1 - s)
    elif act == "gelu_tanh":
        k = 2 * math.sqrt(2 / math.pi)
        s = 1 / (1 + torch.exp(-k * (g + 0.044715 * g ** 3)))
        slope = k * (1 + 3 * 0.044715 * g * g)
        d = s + torch.where(s * (1 - s) > 0, g.abs() * s * (1 - s) * slope, 0.0)
    return 2.0 ** -16 * v + 2.0 ** -40, 2.0 ** -15 * d + 2.0 ** -40


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("act", list(ACTIVATIONS))
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_gates_of_every_size(dtype, act, form):
    x, wg, wu, wd, dy, g = exposed(form, dtype)
    row, e, tiny = x.shape[0] // 2, half_step(dtype), SUBNORMAL[dtype]
    (v, dv), (fv, fdv) = act64(act, g.double()), evaluation(act, g.double())
    bound = lambda v, fn: e * (v.abs() + fn) + tiny + fn
    y = GatedFFN(wg, wu, wd, act=act)(x)
    assert_within("y", y[row], v, bound(v, fv))
    for keep in (True, False):
        layer = GatedFFN(wg, wu, wd, act=act, keep=keep)
        y, saved = layer.forward(x)
        r = layer.backward(dy, x, saved)
        for name, got, want in (("y", y[row], (v, fv)), ("act", r["w_up"][:, 0], (v, fv)), ("act'", r["w_gate"][:, 0], (dv, fdv)),
                                ("a", r["w_down"].diagonal(), (v, fv))):
            assert_within(f"{name} (keep {keep})", got, want[0], bound(*want))
        assert not torch.isnan(r["x"]).any()


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("act", list(ACTIVATIONS))
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_hidden_values_between_the_types_steps(dtype, act, form):
    """g and u that 16 bits do not hold (sums of a weight and a small one, exact in 32): act(g) u, act'(g) u and act(g) are
    still one rounding away, so neither g nor u is rounded on the way, kept or formed again."""
    x, wg, wu, wd, dy, _ = exposed(form, dtype)
    h, row, e, tiny = wg.shape[0], x.shape[0] // 2, half_step(dtype), SUBNORMAL[dtype]
    gen = torch.Generator(device="cuda").manual_seed(7)
    rnd = lambda: torch.randn(h, generator=gen, device="cuda")
    x[row, 1] = 1
    for w, v in ((wg, 2 * rnd()), (wu, rnd())):
        w[:, 0], w[:, 1] = v.to(dtype), (v * rnd().clamp(-1, 1) * e).to(dtype)
    g, u = (w[:, 0].double() + w[:, 1].double() for w in (wg, wu))
    (v, dv), (fv, fdv) = act64(act, g), evaluation(act, g)
    # the evaluation's bound, and the products' roundings in 32 bits
    want = {"a": (v * u, fv * u.abs()), "act": (v, fv), "act'": (dv * u, fdv * u.abs())}
    bound = lambda v, fn: (e + 2.0 ** -22) * (v.abs() + fn) + tiny + fn
    for keep in (True, False):
        layer = GatedFFN(wg, wu, wd, act=act, keep=keep)
        y, saved = layer.forward(x)
        r = layer.backward(dy, x, saved)
        for name, got in (("a", y[row]), ("act", r["w_up"][:, 0]), ("act'", r["w_gate"][:, 1]), ("a", r["w_down"].diagonal())):
            assert_within(f"{name} (keep {keep})", got, want[name][0], bound(*want[name]))
    # the bound would tell: with g and u rounded to the type, some of these values are beyond it
    if act not in ("relu", "sigmoid"):
        g16, u16 = (t.to(dtype).double() for t in (g, u))
        rounded = act64(act, g16)[1] * u16
        assert ((rounded.to(dtype).double() - want["act'"][0]).abs() > bound(*want["act'"])).any()


@pytest.mark.parametrize("by", ["weight", "bias"])
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("act", list(ACTIVATIONS))
def test_a_gate_that_is_not_a_number_is_not_lost(act, form, by):
    """A NaN in one hidden channel's gate weight or gate bias alone: act(g) is NaN in every row, and so are the outputs and
    the gradients that it enters, and no others (its neighbour in a pair among them). relu's derivative there is 0, as
    that of g > 0 ? g : 0; the other activations' is NaN."""
    x, wg, wu, wd, dy, _ = exposed(form, BF16)
    h, row = wg.shape[0], x.shape[0] // 2
    wg = (torch.randn(wg.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) / 2).to(BF16)
    bias = torch.zeros(h, dtype=BF16, device="cuda")

    def step(wg, bias, keep):
        layer = GatedFFN(wg, wu, wd, bias, act=act, keep=keep)
        y, saved = layer.forward(x)
        return {"y": y, "inference": layer(x), **layer.backward(dy, x, saved)}

    for keep, j in itertools.product((True, False), (0, 33, h - 1)):
        clean = step(wg, bias, keep)
        wg2, bias2 = wg.clone(), bias.clone()
        (wg2 if by == "weight" else bias2)[j] = float("nan")
        got = step(wg2, bias2, keep)
        others = torch.arange(h, device="cuda") != j
        for k in ("y", "inference"):
            assert torch.isnan(got[k]).all(), (k, keep, j)
        for k in ("w_up", "w_gate", "b_gate"):
            if k == "w_up" or act != "relu":
                assert torch.isnan(got[k][j]).all(), (k, keep, j)
            assert torch.equal(got[k][others], clean[k][others]), (k, keep, j)
        assert torch.isnan(got["w_down"][:, j]).all() and torch.equal(got["w_down"][:, others], clean["w_down"][:, others])
        assert torch.isnan(got["x"][row]).all()
