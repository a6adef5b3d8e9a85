"""The residual norm on a B200 against its 64-bit definition and differentiation, and a run of it with the gated
feed-forward block as a network would use them."""
import itertools

import pytest
import torch

import flyhigh_engine_b200 as fh
from flyhigh_engine_b200.kernels import GatedFFN, ResidualNorm, empty_rows
from row_ops_plain import assert_within, ffn64, half_step, residual_norm64
from test_gpu_gated_ffn import rows

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
EPS = 1e-5


def case(m, c, dtype, pre, post, gates=0, affine=True, scale=True, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    vec = lambda mean, std: (mean + std * torch.randn(c, generator=gen, device="cuda")).to(dtype)
    p = {}
    for side, kind in (("pre", pre), ("post", post)):
        if affine and kind != "none":
            p["w_" + side], p["b_" + side] = vec(1.0, 0.2), vec(0.0, 0.2)
    if scale:
        p["scale"] = vec(0.5, 0.2)
    t = {n: rows(gen, m, c, dtype, s) for n, s in (("x", 1.0), ("f", 0.7), ("dy", 0.5), ("dh", 0.5))}
    gate = rows(gen, gates, c, dtype) if gates else None
    return t, gate, p


def reference(t, y, gate, p, pre, post):
    """Outputs and gradients in 64 bits with their bounds. The gradients are of the y that the kernel was given (rounded):
    norm_pre's part is differentiated at that y. A sum of n 32-bit terms is off by at most n 2^-24 of their magnitudes; the
    longest here (8192 channels over at least 64 threads, then a tree) stays under 2^-16 with the functions around it."""
    dt = t["x"].dtype
    e, tiny = half_step(dt), 2.0 ** -25 if dt == F16 else 0.0
    z = {k: v.double() for k, v in t.items()}
    pz = {k: v.double() for k, v in p.items()}
    gz = None if gate is None else gate.double()
    yv, hv = residual_norm64(z["x"], z["f"], gz, pre, post, EPS, **pz)
    slack = lambda v, mag: e * v.abs() + tiny + 2.0 ** -16 * mag
    r = {"y": (yv, slack(yv, 1 + yv.abs()))}
    if hv is not None:
        r["h"] = (hv, slack(hv, 1 + hv.abs()))
    # d: the gradient on y, at the rounded y
    yz = y.double().requires_grad_(True)
    pre_p = {k: v.clone().requires_grad_(True) for k, v in pz.items() if k.endswith("pre")}
    d = z["dy"]
    if pre != "none":
        hz = residual_norm64(yz, None, None, pre, "none", EPS, **pre_p)[1]
        names = list(pre_p)
        g = torch.autograd.grad((hz * z["dh"]).sum(), [yz] + [pre_p[k] for k in names])
        d = d + g[0]
        ny = residual_norm64(y.double(), None, None, pre, "none", EPS)[1]
        for k, v in zip(names, g[1:]):
            terms = z["dh"].abs() * (ny.abs() if k == "w_pre" else 1.0)
            r[k] = (v, slack(v, (terms.sum(0) if terms.dim() > 1 else terms)))
    dmax = d.abs().amax(1, keepdim=True)
    r["x"] = (d, slack(d, 1 + dmax))
    leaves = {"f": z["f"].clone().requires_grad_(True)}
    leaves.update({k: v.clone().requires_grad_(True) for k, v in pz.items() if not k.endswith("pre")})
    if gz is not None:
        leaves["gate"] = gz.clone().requires_grad_(True)
    out = residual_norm64(z["x"], leaves["f"], leaves.get("gate"), "none", post, EPS,
                          **{k: v for k, v in leaves.items() if k not in ("f", "gate")})[0]
    # magnitudes for the sums' bounds: every factor at its absolute value
    with torch.no_grad():
        c = z["x"].shape[1]
        nf = residual_norm64(z["f"], None, None, post, "none", EPS)[1] if post != "none" else z["f"]
        one = torch.ones(c, dtype=torch.float64, device="cuda")
        s, w, b = (pz.get(k, v).abs() for k, v in (("scale", one), ("w_post", one), ("b_post", 0 * one)))
        gr = one.expand_as(d) if gz is None else gz.abs().repeat_interleave(d.shape[0] // gz.shape[0], 0)
        pa = nf.abs() * w + b
        # d is a difference: r (dn - n mean(dn n) - mean(dn)) + dy. Each term is known to 2^-18 of itself (a product or two,
        # and a mean as above), so d to 2^-18 of the terms' magnitudes, which may be far more than 2^-16 |d|. The sums that
        # d enters are off by that much times d's factors; `da` is |d| with this error in units of the slack's 2^-16.
        da = d.abs() + z["dy"].abs() / 4
        if pre != "none":
            v = y.double()
            sp = torch.sqrt((v.var(1, unbiased=False, keepdim=True) if pre == "layer" else v.square().mean(1, keepdim=True)) + EPS)
            dn = z["dh"].abs() * pz.get("w_pre", one).abs()
            da = da + (dn + ny.abs() * (dn * ny.abs()).mean(1, keepdim=True) + dn.mean(1, keepdim=True)) / sp / 4
        mags = {"scale": (da * gr * pa).sum(0), "w_post": (da * gr * s * nf.abs()).sum(0),
                "b_post": (da * gr * s).sum(0)}
        if gz is not None:
            mags["gate"] = (da * s * pa).reshape(gz.shape[0], -1, c).sum(1)
        q = da * gr * s * w
        sd = torch.sqrt(z["f"].var(1, unbiased=False, keepdim=True) + EPS) if post == "layer" else \
            torch.sqrt(z["f"].square().mean(1, keepdim=True) + EPS)
        mags["f"] = q.amax(1, keepdim=True) * (1 + nf.abs()) * (1 + (1 / sd if post != "none" else 0))
    for k, v in zip(leaves, torch.autograd.grad((out * d).sum(), list(leaves.values()))):
        r[k] = (v, slack(v, mags[k]))
    return r


def check(m, c, dtype, pre, post, gates=0, affine=True, scale=True, seed=0, biases=True):
    t, gate, p = case(m, c, dtype, pre, post, gates, affine, scale, seed)
    if not biases:
        p = {k: v for k, v in p.items() if not k.startswith("b_")}
    layer = ResidualNorm(c, dtype, pre=pre, post=post, eps=EPS, **p)
    y, h = layer(t["x"], t["f"], gate)
    got = {"y": y}
    if h is not None:
        got["h"] = h
    got.update(layer.backward(t["dy"], t["dh"] if pre != "none" else None, y, t["f"], gate))
    want = reference(t, y, gate, p, pre, post)
    assert set(got) == set(want)
    for k in want:
        assert_within(k, got[k], *want[k])


@pytest.mark.parametrize("pre,post", list(itertools.product(["none", "rms", "layer"], repeat=2)))
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_kinds(pre, post, dtype):
    check(70, 48, dtype, pre, post, gates=5)
    check(33, 300, dtype, pre, post, gates=0, affine=False, scale=False)
    check(24, 1001, dtype, pre, post, gates=3, scale=False)


@pytest.mark.parametrize("c", [1, 7, 8, 9, 36, 63, 64, 65, 100, 255, 256, 257, 512, 513, 1000, 1024, 1025, 2048, 2050, 4096,
                               4097, 5000, 8191, 8192])
def test_channels(c):
    check(11, c, F16, "layer", "layer", gates=11)
    check(6, c, BF16, "rms", "rms", gates=2)


@pytest.mark.parametrize("m,gates", [(1, 1), (2, 1), (31, 0), (32, 32), (33, 3), (1000, 1), (1000, 1000), (3000, 600), (4000, 8),
                                     (20000, 4)])
def test_rows_and_gates(m, gates):
    check(m, 64, F16, "layer", "rms", gates=gates)
    check(m, 200, BF16, "rms", "layer", gates=gates)
    if m <= 4000:
        check(m, 1200, F16, "rms", "none", gates=gates)


@pytest.mark.parametrize("c", [60, 64, 120, 128, 250, 256, 500, 512, 1000, 1024, 2000, 2048, 4090, 4096, 5000, 8192])
def test_without_biases(c):
    """Several rows a CTA; without biases the gradient forms no sums of d and dh."""
    check(1501 if c <= 2048 else 333, c, BF16, "rms", "rms", gates=0, biases=False)
    check(300, c, F16, "layer", "none", gates=3, biases=False, scale=False)


@pytest.mark.parametrize("c", [40, 100, 128, 300, 512, 1000, 2056, 5000])
def test_many_gate_rows(c):
    """CTAs that finish whole runs of rows with one gate row, more than one run each."""
    check(2600, c, F16, "layer", "rms", gates=1300)
    check(1300, c, BF16, "rms", "none", gates=1300, biases=False)


def test_wide_many_rows():
    check(3000, 2048, BF16, "rms", "rms", gates=2)


def test_constant_rows_and_zero_rows():
    """A constant row has no variance and a zero row no square: eps carries both; eps 0 is NaN in that row alone."""
    x = empty_rows((4, 48), F16)
    x.copy_(torch.randn(4, 48, device="cuda"))
    x[1], x[2] = 2.5, 0.0
    for kind in ("rms", "layer"):
        _, h = ResidualNorm(48, F16, pre=kind, eps=EPS)(x)
        want = residual_norm64(x.double(), None, None, kind, "none", EPS)[1]
        assert torch.isfinite(h).all()
        assert_within(kind, h, want, 2.0 ** -11 * want.abs() + 1e-4)
        _, h0 = ResidualNorm(48, F16, pre=kind, eps=0.0)(x)
        assert torch.isfinite(h0[[0, 3]]).all() and torch.isnan(h0[2]).all()


def test_zero_eps_gradient_of_ragged_rows():
    """With eps 0 the threads without a row add nothing to the sums."""
    t, gate, p = case(37, 48, F16, "rms", "layer", gates=1)
    layer = ResidualNorm(48, F16, pre="rms", post="layer", eps=0.0, **p)
    y, _ = layer(t["x"], t["f"], gate)
    for k, v in layer.backward(t["dy"], t["dh"], y, t["f"], gate).items():
        assert torch.isfinite(v).all(), k


@pytest.mark.parametrize("c", [48, 300, 3000])
def test_non_finite_values_stay_in_their_rows(c):
    t, gate, p = case(40, c, F16, "layer", "rms", gates=1)
    layer = ResidualNorm(c, F16, pre="layer", post="rms", eps=EPS, **p)
    y, h = layer(t["x"], t["f"], gate)
    t["f"][7, 3] = float("nan")
    y2, h2 = layer(t["x"], t["f"], gate)
    assert torch.isnan(y2[7]).all() and torch.isnan(h2[7]).all()
    keep = torch.arange(40, device="cuda") != 7
    assert torch.equal(y2[keep], y[keep]) and torch.equal(h2[keep], h[keep])


def test_norm_before_a_first_block_and_partial_gradients():
    t, _, p = case(50, 96, BF16, "rms", "none", scale=False)
    layer = ResidualNorm(96, BF16, pre="rms", eps=EPS, **p)
    y, h = layer(t["x"])
    assert y is t["x"]
    want = residual_norm64(t["x"].double(), None, None, "rms", "none", EPS, **p)[1]
    assert_within("h", h, want, 2.0 ** -8 * want.abs() + 1e-4)
    g = layer.backward(t["dy"], t["dh"], y)
    assert set(g) == {"x", "w_pre", "b_pre"}
    a = layer.backward(None, t["dh"], y)
    b = layer.backward(t["dy"], None, y)
    assert torch.equal(b["x"], t["dy"]) and (b["w_pre"] == 0).all() and (b["b_pre"] == 0).all()
    assert torch.equal(a["w_pre"], g["w_pre"]) and not torch.equal(a["x"], g["x"])


def test_views_padding_and_no_rows():
    m, c = 30, 37
    t, gate, p = case(m, c, F16, "layer", "rms", gates=3)
    layer = ResidualNorm(c, F16, pre="layer", post="rms", eps=EPS, **p)
    y, h = layer(t["x"], t["f"], gate)
    wide = torch.full((3, 2, 5, 64), 5.0, dtype=F16, device="cuda")
    wide[..., 8:8 + c] = t["x"].reshape(3, 2, 5, c)
    y2, h2 = layer(wide[..., 8:8 + c], t["f"], gate)
    assert y2.shape == (3, 2, 5, c) and torch.equal(y2.reshape(m, c), y) and torch.equal(h2.reshape(m, c), h)
    z = empty_rows((0, c), F16)
    y0, h0 = layer(z, z, gate)
    assert y0.shape == h0.shape == (0, c)
    g = layer.backward(z, z, y0, z, gate)
    for k in ("gate", "scale", "w_pre", "b_pre", "w_post", "b_post"):
        assert (g[k] == 0).all(), k


def test_offsets_past_32_bits():
    m, c = 263000, 8192
    x = torch.ones((m, c), dtype=F16, device="cuda")
    x[-1] = torch.randn(c, device="cuda")
    x[0] = torch.randn(c, device="cuda")
    _, h = ResidualNorm(c, F16, pre="rms", eps=0.0)(x)
    for i in (0, m - 1):
        want = residual_norm64(x[i:i + 1].double(), None, None, "rms", "none", 0.0)[1]
        assert_within("h", h[i:i + 1], want, 2.0 ** -11 * want.abs() + 1e-5)
    assert (h[1:-1:1000] == 1).all()


def test_gates_of_any_alignment():
    t, gate, p = case(12, 37, F16, "rms", "layer", gates=4)
    layer = ResidualNorm(37, F16, pre="rms", post="layer", eps=EPS, **p)
    y, h = layer(t["x"], t["f"], gate)
    for other in (gate.contiguous(), torch.cat([gate[:, :1], gate], 1)[:, 1:]):
        assert torch.equal(layer(t["x"], t["f"], other)[1], h)
        g, g2 = (layer.backward(t["dy"], t["dh"], y, t["f"], v) for v in (gate, other))
        assert all(torch.equal(g[k], g2[k]) for k in g)


def test_refusals():
    t, gate, p = case(12, 48, F16, "rms", "rms", gates=3)
    layer = ResidualNorm(48, F16, pre="rms", post="rms", eps=EPS, **p)
    with pytest.raises(fh.FlyHighError, match="divide"):
        layer(t["x"], t["f"], torch.zeros(5, 48, dtype=F16, device="cuda"))
    with pytest.raises(fh.FlyHighError, match="without f"):
        layer(t["x"], None, gate)
    with pytest.raises(fh.FlyHighError, match="12 rows"):
        layer(t["x"], t["f"][:6])
    with pytest.raises(fh.FlyHighError, match="expected"):
        layer(t["x"].to(BF16), t["f"])
    with pytest.raises(fh.FlyHighError, match="dy or dh"):
        layer.backward(None, None, t["x"])
    with pytest.raises(fh.FlyHighError, match="w_pre"):
        ResidualNorm(48, F16, w_pre=torch.ones(47, dtype=F16, device="cuda"))


def _network(x, gate, norms, ffns):
    """Two pre/post-normed gated blocks over a residual stream; what the gradient needs is kept."""
    kept = []
    y, h = norms[0](x)
    for i, f in enumerate(ffns):
        o, saved = f.forward(h)
        y2, h2 = norms[i + 1](y, o, gate)
        kept.append((h, saved, o, y2))
        y, h = y2, h2
    return y, kept


def _network_grad(dy, x, gate, norms, ffns, kept):
    """The input's, the gate's and the first block's gate projection's gradients."""
    dh, dgate = None, 0.0
    for i in reversed(range(len(ffns))):
        h, saved, o, y2 = kept[i]
        g = norms[i + 1].backward(dy, dh, y2, o, gate)
        dgate = dgate + g["gate"].double()
        w = ffns[i].backward(g["f"], h, saved)
        dy, dh = g["x"], w["x"]
    return norms[0].backward(dy, dh, x)["x"], dgate, w["w_gate"]


def test_blocks_together_against_differentiation_in_64_bits():
    """The run as it would be used: norm, block, join + next norm, block, join; forward and gradient, eagerly and from a
    captured graph. Each of the about ten roundings on the way is off by at most 2^-8 (bf16), at random signs over the
    sums: the whole within 10 * 2^-8 of the result's 2-norm."""
    m, c, f, images = 3 * 40, 96, 256, 3
    gen = torch.Generator(device="cuda").manual_seed(11)
    mk = lambda *s, std: rows(gen, *s, BF16, std)
    vec = lambda mean: (mean + 0.1 * torch.randn(c, generator=gen, device="cuda")).to(BF16)
    x, dy, gate = mk(m, c, std=1.0), mk(m, c, std=1.0), mk(images, c, std=1.0)
    weights = [[mk(f, c, std=c ** -0.5), mk(f, c, std=c ** -0.5), mk(c, f, std=f ** -0.5)] for _ in range(2)]
    w1, w2, ws, wp = vec(1.0), vec(1.0), vec(0.5), vec(1.0)
    norms = [ResidualNorm(c, BF16, pre="rms", w_pre=w1, eps=EPS),
             ResidualNorm(c, BF16, pre="rms", w_pre=w2, post="layer", w_post=wp, scale=ws, eps=EPS),
             ResidualNorm(c, BF16, pre="none", post="layer", w_post=wp, scale=ws, eps=EPS)]
    ffns = [GatedFFN(*w) for w in weights]

    def step():
        y, kept = _network(x, gate, norms, ffns)
        return (y, *_network_grad(dy, x, gate, norms, ffns, kept))

    got = step()
    z = {k: v.double().requires_grad_(True) for k, v in (("x", x), ("gate", gate), ("w", weights[0][0]))}
    w64 = [[v.double() for v in w] for w in weights]
    w64[0][0] = z["w"]
    y, h = residual_norm64(z["x"], None, None, "rms", "none", EPS, w_pre=w1)
    for i, pre in enumerate(("rms", "none")):
        o = ffn64(h, *w64[i], None, None, None, "silu")
        y, h = residual_norm64(y, o, z["gate"], pre, "layer", EPS, w_pre=w2 if pre == "rms" else None, w_post=wp, scale=ws)
    want = (y.detach(), *torch.autograd.grad((y * dy.double()).sum(), [z["x"], z["gate"], z["w"]]))
    for name, a, b in zip(("y", "x", "gate", "w_gate"), got, want):
        rel = float((a.double() - b).norm() / b.norm())
        assert rel <= 10 * 2.0 ** -8, (name, rel)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, again))
