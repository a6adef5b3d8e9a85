"""Calls of the row operators that their documentation allows beside the ordinary ones."""
import ctypes
import warnings

import pytest
import torch

import flyhigh_engine_b200 as fh
from flyhigh_engine_b200 import kernels as K
from flyhigh_engine_b200.kernels import GatedFFN, ResidualNorm
from row_ops_plain import act64, assert_within, ffn, half_step
from test_gpu_gated_ffn import block
from test_gpu_residual_norm import case

pytestmark = pytest.mark.gpu
F16 = torch.float16


@pytest.mark.parametrize("shape", [(6, 48, 192, 48), (200, 48, 192, 48), (20300, 64, 200, 64), (200, 136, 260, 72)], ids=str)
def test_the_activated_product_alone(shape):
    """fhk_gated_ffn with `a` but neither g nor u: a is written, in every form."""
    m, c, f, o = shape
    x, w, b, _ = block(m, c, f, o, F16)
    y, a = (torch.full((m, n), 7.0, dtype=F16, device="cuda") for n in (o, (f + 7) // 8 * 8))
    p = K.GatedFfnParams(x=x.data_ptr(), y=y.data_ptr(), a=a.data_ptr(), x_pitch=x.stride(0), y_pitch=o, h_pitch=a.shape[1], m=m, cin=c,
                         hidden=f, cout=o, act=K.ACTIVATIONS["silu"], dtype=0,
                         **{n: t.data_ptr() for n, t in zip(("w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down"), (*w, *b))},
                         **{n: t.stride(0) for n, t in zip(("wg_pitch", "wu_pitch", "wd_pitch"), w)})
    n = fh.lib().fhk_gated_ffn_scratch_bytes(ctypes.byref(p))
    scratch = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    p.scratch, p.scratch_bytes = scratch.data_ptr(), n
    assert fh.lib().fhk_gated_ffn(ctypes.byref(p), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert_within("y", y, *ffn(x, *w, *b, act="silu")["y"])
    (wg, wu), (bg, bu), x = (t.double() for t in w[:2]), (t.double() for t in b[:2]), x.double()
    g, u = x @ wg.t() + bg, x @ wu.t() + bu
    want = act64("silu", g)[0] * u
    # g and u are sums of c + 1 terms in 32 bits, |silu'| <= 1.1, silu itself to 2^-16 of itself (its argument's rounding)
    sums = lambda v, wt: 1.1 * (c + 1) * 2.0 ** -23 * (v.abs() + x.abs() @ wt.abs().t())
    off = sums(g, wg) * u.abs() + act64("silu", g)[0].abs() * sums(u, wu) + 2.0 ** -16 * want.abs()
    assert_within("a", a[:, :f], want, off + half_step(F16) * (want.abs() + off) + 2.0 ** -25)
    assert (a[:, f:] == 7).all()


@pytest.mark.parametrize("keep", [True, False])
@pytest.mark.parametrize("m", [5, 200])
def test_replaced_weights_are_used(m, keep):
    """A parameter whose .data is replaced lies elsewhere: calls use it there. What a layer cannot use it refuses, until it is
    put right."""
    x, w, b, dy = block(m, 48, 96, 40, F16)
    _, w2, b2, _ = block(m, 48, 96, 40, F16, seed=1)
    layer, other = GatedFFN(*w, *b, keep=keep), GatedFFN(*w2, *b2, keep=keep)

    def step(layer):
        y, saved = layer.forward(x)
        return {"y": y, "inference": layer(x), **layer.backward(dy, x, saved)}

    step(layer)
    old = [t.data for t in (*w, *b)]  # alive all along
    for t, new in zip((*w, *b), (*w2, *b2)):
        t.data = new
    got, want = step(layer), step(other)
    assert all(torch.equal(got[k], want[k]) for k in want)
    for i, bad in ((0, old[0][:, :40]), (0, old[0][:88]), (2, old[2].float()), (2, old[2].cpu()), (4, old[4][:90])):
        t = (*w, *b)[i]
        good, t.data = t.data, bad
        with pytest.raises(fh.FlyHighError):
            layer(x)
        with pytest.raises(fh.FlyHighError):
            layer.forward(x)
        t.data = good
        assert torch.equal(layer(x), want["inference"])


def test_replaced_vectors_of_a_norm_are_used():
    t, gate, p = case(40, 96, F16, "layer", "rms", gates=2)
    _, _, p2 = case(40, 96, F16, "layer", "rms", gates=2, seed=1)
    layer, other = (ResidualNorm(96, F16, pre="layer", post="rms", **v) for v in (p, p2))

    def step(layer):
        y, h = layer(t["x"], t["f"], gate)
        return {"y": y, "h": h, **layer.backward(t["dy"], t["dh"], y, t["f"], gate)}

    step(layer)
    old = {k: v.data for k, v in p.items()}  # alive all along
    for k, v in p.items():
        v.data = p2[k]
    got, want = step(layer), step(other)
    assert all(torch.equal(got[k], want[k]) for k in want)
    for bad in (old["scale"][:88], old["scale"].float(), old["scale"].cpu(), old["scale"][1:]):
        good, p["scale"].data = p["scale"].data, bad
        with pytest.raises(fh.FlyHighError, match="scale"):
            layer(t["x"], t["f"], gate)
        p["scale"].data = good
    assert torch.equal(layer(t["x"], t["f"], gate)[0], want["y"])


@pytest.mark.parametrize("lead", [(3, 0), (0, 3), (2, 0, 5)], ids=str)
def test_maps_without_pixels(lead):
    """No rows in any dimension: outputs of that shape, and parameters' gradients of 0."""
    x, w, b, _ = block(1, 48, 96, 40, F16)
    empty = lambda c: K.empty_rows((*lead, c), F16)
    layer = GatedFFN(*w, *b)
    y, saved = layer.forward(empty(48))
    assert y.shape == (*lead, 40) and layer(empty(48)).shape == y.shape
    g = layer.backward(empty(40), empty(48), saved)
    assert g["x"].shape == (*lead, 48) and all((v == 0).all() for v in g.values())
    _, gate, p = case(6, 48, F16, "rms", "rms", gates=2)
    norm = ResidualNorm(48, F16, pre="rms", post="rms", **p)
    y, h = norm(empty(48), empty(48), gate)
    assert y.shape == h.shape == (*lead, 48)
    assert all((v == 0).all() for v in norm.backward(empty(48), empty(48), y, empty(48), gate).values())


def test_a_call_that_autograd_cannot_see_says_so():
    x, w, b, _ = block(20, 48, 96, 48, F16)
    _, gate, p = case(20, 48, F16, "rms", "rms", gates=2)
    ffn_, norm = GatedFFN(*w, *b), ResidualNorm(48, F16, pre="rms", post="rms", **p)
    calls = [lambda: ffn_(x), lambda: ffn_.forward(x), lambda: norm(x, x, gate)]
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        quiet = [c() for c in calls]
    for t in (x, w[1], b[2], gate, p["w_post"]):
        t.requires_grad_(True)
        concerned = 0
        for call in calls:
            with warnings.catch_warnings(record=True) as seen:
                warnings.simplefilter("always")
                call()
            concerned += len(seen)
            assert all("not recorded by autograd" in str(v.message) and v.filename == __file__ for v in seen)
            with warnings.catch_warnings(), torch.no_grad():
                warnings.simplefilter("error")
                call()
        assert concerned == (3 if t is x else 2 if t is w[1] or t is b[2] else 1)
        t.requires_grad_(False)
    assert torch.equal(ffn_(x), quiet[0])
