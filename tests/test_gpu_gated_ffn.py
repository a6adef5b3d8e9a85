"""The gated feed-forward block on a B200 against its 64-bit definition, elementwise within the bound its roundings
leave (row_ops_plain), at the sizes and layouts where tiles, tails and few-row paths begin and end."""
import pytest
import torch

import flyhigh_engine_b200 as fh
from flyhigh_engine_b200.kernels import GatedFFN, empty_rows
from row_ops_plain import assert_within, ffn

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def rows(gen, m, c, dtype, std=1.0, fill=float("nan")):
    """m rows of normal values at a 16-byte pitch, the padding NaN: it must never be read."""
    t = empty_rows((m, c), dtype)
    if t.stride(0) > c and m:
        torch.as_strided(t, (m, t.stride(0)), (t.stride(0), 1)).fill_(fill)
    t.copy_(torch.randn(m, c, generator=gen, device="cuda") * std)
    return t


def block(m, c, f, o, dtype, bias=True, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    vec = lambda n: (0.3 * torch.randn(n, generator=gen, device="cuda")).to(dtype) if bias else None
    w = (rows(gen, f, c, dtype, c ** -0.5), rows(gen, f, c, dtype, c ** -0.5), rows(gen, o, f, dtype, f ** -0.5))
    return rows(gen, m, c, dtype), w, (vec(f), vec(f), vec(o)), rows(gen, m, o, dtype, 0.5)


def check(m, c, f, o, dtype, act="silu", bias=True, seed=0, train=True):
    """Inference, and training with the hidden values kept and formed again."""
    x, w, b, dy = block(m, c, f, o, dtype, bias, seed)
    want = ffn(x, *w, *b, act=act, dy=dy if train else None)
    assert_within("y", GatedFFN(*w, *b, act=act)(x), *want["y"])
    for keep in (True, False) if train else ():
        layer = GatedFFN(*w, *b, act=act, keep=keep)
        y, saved = layer.forward(x)
        assert (saved.g is not None) == keep
        got = {"y": y, **layer.backward(dy, x, saved)}
        assert set(got) == set(want)
        for k in want:
            assert_within(f"{k} (keep {keep})", got[k], *want[k])
    assert fh.lib().fhk_gated_ffn_wait_timeouts(0) == 0


SHAPES = [(1, 1, 1, 1), (3, 3, 5, 7), (2, 36, 77, 36), (5, 48, 192, 48), (17, 16, 64, 16), (33, 64, 256, 64),
          (128, 64, 128, 64), (129, 72, 129, 80), (127, 63, 65, 127), (256, 128, 256, 128), (300, 96, 384, 96),
          (257, 100, 1000, 130), (513, 260, 300, 33), (1000, 48, 192, 48), (64, 520, 264, 776)]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_shapes(shape, dtype):
    check(*shape, dtype)


@pytest.mark.parametrize("m", [1, 2, 3, 4, 7, 8, 9, 15, 16, 17, 24, 25, 31, 32, 33, 40, 63, 64, 65, 96, 97])
def test_few_rows(m):
    """The forms for few rows, to either side of their borders, with ragged and with whole channel counts."""
    check(m, 200, 344, 152, F16, act="gelu", seed=m)
    check(m, 256, 1024, 256, BF16, bias=False, seed=m, train=m in (1, 8, 33))


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu", "sigmoid"])
@pytest.mark.parametrize("m", [4, 200])
def test_activations(act, m):
    check(m, 80, 160, 80, F16, act=act)
    check(m, 80, 160, 80, BF16, act=act, bias=False)


def test_larger():
    check(2000, 512, 1536, 512, BF16)
    check(1100, 1024, 2048, 640, F16, act="gelu_tanh", bias=False)
    check(4500, 64, 256, 64, F16)


@pytest.mark.parametrize("shape", [(20300, 64, 640, 64), (20300, 64, 256, 64), (19000, 128, 200, 128), (38100, 100, 333, 37),
                                   (18945, 16, 24, 96)], ids=str)
def test_maps(shape):
    """Maps of more than one 128-row tile per SM, where two tiles share a CTA and some have no second last one, with the
    weights resident and streamed."""
    check(*shape, F16, act="gelu_tanh", train=False)
    check(*shape, BF16, bias=False, train=False)


def test_long_sums():
    """Weight and bias gradients over many rows (K split over CTAs), and a long K in the down projection of few tiles."""
    check(20000, 160, 200, 136, BF16)
    check(20000, 48, 96, 48, F16, act="gelu")
    check(150, 64, 8000, 200, BF16, bias=False)


@pytest.mark.parametrize("m", [5, 70, 700])
def test_extreme_gates(m):
    """Gates far in both tails: act and act' reach their limits without NaN."""
    x, w, b, dy = block(m, 32, 64, 32, BF16)
    x = (x * 60).contiguous()
    for act in ("silu", "gelu", "gelu_tanh", "relu", "sigmoid"):
        layer = GatedFFN(*w, *b, act=act)
        want = ffn(x, *w, *b, act=act, dy=dy)
        y, saved = layer.forward(x)
        got = {"y": y, **layer.backward(dy, x, saved)}
        for k in want:
            assert_within(f"{act} {k}", got[k], *want[k])


@pytest.mark.parametrize("m", [1, 20, 300])
def test_non_finite_rows_stay_in_their_rows(m):
    x, w, b, _ = block(m, 48, 96, 48, F16)
    layer = GatedFFN(*w, *b)
    clean = layer(x)
    bad = m // 2
    x[bad, 5] = float("inf")
    got = layer(x)
    assert not torch.isfinite(got[bad]).any()
    keep = torch.arange(m, device="cuda") != bad
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("m", [3, 40, 400])
def test_views_and_padding(m):
    """Channel slices of a wider NHWC map in and out: the right values, nothing written beside them."""
    x, w, b, dy = block(m, 40, 72, 24, F16)
    layer = GatedFFN(*w, *b)
    wide = torch.full((m, 1, 64), 7.0, dtype=F16, device="cuda")
    wide[:, 0, 8:48] = x
    out = torch.full((m, 1, 48), 9.0, dtype=F16, device="cuda")
    layer(wide[..., 8:48], out=out[..., 16:40])
    assert torch.equal(out[:, 0, 16:40], layer(x))
    assert (out[..., :16] == 9).all() and (out[..., 40:] == 9).all()
    odd = torch.full((m + 2, 40), 3.0, dtype=F16, device="cuda")  # 37 of 40 channels, a row before and after
    x2, w2, _, _ = block(m, 33, 65, 37, F16)
    layer2 = GatedFFN(*w2)
    layer2(x2, out=odd[1:-1, :37])
    assert torch.equal(odd[1:-1, :37], layer2(x2))
    assert (odd[0] == 3).all() and (odd[-1] == 3).all() and (odd[:, 37:] == 3).all()


def test_no_rows():
    x, w, b, dy = block(0, 48, 96, 40, F16)
    layer = GatedFFN(*w, *b)
    assert layer(x).shape == (0, 40)
    y, saved = layer.forward(x)
    g = layer.backward(dy, x, saved)
    assert g["x"].shape == (0, 48)
    for k in ("w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down"):
        assert (g[k] == 0).all(), k


def test_wanted_gradients_only():
    x, w, b, dy = block(150, 48, 96, 48, F16)
    layer = GatedFFN(*w, *b)
    y, saved = layer.forward(x)
    every = layer.backward(dy, x, saved)
    for want in (("x",), ("w_down",), ("w_gate", "b_up"), ("b_down",), ()):
        some = layer.backward(dy, x, saved, want=want)
        assert set(some) == set(want)
        for k in want:
            assert torch.equal(some[k], every[k]), k
    with pytest.raises(fh.FlyHighError, match="not among"):
        layer.backward(dy, x, saved, want=("gate",))


@pytest.mark.parametrize("m", [1, 20, 600])
def test_repeatable_on_another_stream_and_in_a_graph(m):
    """The same bits twice, on a side stream, and from a replayed graph with new inputs; two captured graphs do not
    share anything."""
    x, w, b, dy = block(m, 96, 384, 96, F16, seed=1)
    x2, _, _, dy2 = block(m, 96, 384, 96, F16, seed=2)
    layer = GatedFFN(*w, *b)

    def step(x, dy):
        y, saved = layer.forward(x)
        return {"y": y, "inference": layer(x), **layer.backward(dy, x, saved)}

    first, second = step(x, dy), step(x2, dy2)
    again = step(x, dy)
    assert all(torch.equal(first[k], again[k]) for k in first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(x, dy)
    side.synchronize()
    assert all(torch.equal(first[k], other[k]) for k in first)
    graphs, ins, outs = [], [], []
    for _ in range(2):
        gx, gdy = x.clone(), dy.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = step(gx, gdy)
        graphs.append(g)
        ins.append((gx, gdy))
        outs.append(o)
    ins[1][0].copy_(x2)
    ins[1][1].copy_(dy2)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(first[k], outs[0][k]) for k in first)
    assert all(torch.equal(second[k], outs[1][k]) for k in second)


def test_overlapping_calls_on_two_streams():
    """Calls in flight at once share nothing: many of them on two streams, each result as alone."""
    cases = [block(m, c, f, c, F16, seed=m) for m, c, f in ((3, 256, 512), (700, 64, 192), (1500, 480, 640), (20, 96, 96))]
    layers = [GatedFFN(*w, *b) for _, w, b, _ in cases]

    def step(layer, x, dy):
        y, saved = layer.forward(x)
        return [y, *layer.backward(dy, x, saved).values()]

    alone = [step(layer, x, dy) for layer, (x, _, _, dy) in zip(layers, cases)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(24):
        with torch.cuda.stream(streams[i % 2]):
            k = (i // 2 + i) % len(cases)
            got.append((k, step(layers[k], cases[k][0], cases[k][3])))
    torch.cuda.synchronize()
    for k, r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, alone[k])), k


def test_weights_updated_in_place_are_used():
    x, w, b, _ = block(64, 48, 96, 48, F16)
    layer = GatedFFN(*w, *b)
    y = layer(x).clone()
    w[2].mul_(2)
    b[2].mul_(2)
    assert torch.equal(layer(x), (y * 2))


def test_offsets_past_32_bits():
    """Over 2^31 hidden elements: the last rows against the same rows alone."""
    m, f = 135000, 16384
    x, w, _, _ = block(m, 16, f, 16, BF16, bias=False)
    layer = GatedFFN(*w)
    y = layer(x)
    want = ffn(x[-300:], *w)["y"]
    assert_within("y", y[-300:], *want)
    want = ffn(x[:200], *w)["y"]
    assert_within("y", y[:200], *want)


def test_refusals():
    x, w, b, dy = block(8, 48, 96, 40, F16)
    with pytest.raises(fh.FlyHighError, match="do not match"):
        GatedFFN(w[0], w[1][:-1], w[2])
    with pytest.raises(fh.FlyHighError, match="w_down"):
        GatedFFN(w[0], w[1], w[2][:, :88])
    with pytest.raises(fh.FlyHighError, match="b_gate"):
        GatedFFN(*w, b_gate=b[2])
    with pytest.raises(fh.FlyHighError, match="expected"):
        GatedFFN(w[0], w[1].to(BF16), w[2])
    with pytest.raises(fh.FlyHighError, match="float16 or bfloat16"):
        GatedFFN(*(v.float() for v in w))
    layer = GatedFFN(*w, *b)
    with pytest.raises(fh.FlyHighError, match="rows of 48"):
        layer(x[:, :40])
    with pytest.raises(fh.FlyHighError, match="expected"):
        layer(x.to(BF16))
    with pytest.raises(fh.FlyHighError, match="expected"):
        layer(x.cpu())
    with pytest.raises(fh.FlyHighError, match="empty_rows"):
        layer(torch.zeros(9, 50, dtype=F16, device="cuda")[:, 1:49])
    with pytest.raises(fh.FlyHighError, match="8 rows"):
        layer(x, out=empty_rows((7, 40), F16))
    y, saved = layer.forward(x)
    with pytest.raises(fh.FlyHighError, match="not of one call"):
        layer.backward(dy[:4], x, saved)
    with pytest.raises(fh.FlyHighError, match="not of one call"):
        layer.backward(dy[:4], x[:4], saved)
    with pytest.raises(fh.FlyHighError, match="16-byte"):
        layer.backward(dy[:1].expand(8, 40), x, saved)
