"""Sums of the gated feed-forward block held to equality: with relu, rows of small whole numbers and weights of which few are
not 0, every product, hidden value and sum is a whole number that its type holds exactly (up to 2^11 in f16 and 2^8 in bf16
for what is rounded, 2^24 for the f32 sums), so nothing but the final rounding is left, and that is the same on both
sides. A K block, a slice or a tail that a sum leaves out shows in every element it belongs to."""
import pytest
import torch

from flyhigh_engine_b200.kernels import GatedFFN, empty_rows

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def whole(m, c, f, o, dtype, seed=0):
    """Rows of -1, 0, 1; two weights of +-1 a hidden channel (|g|, |u| <= 3 with a bias of +-1, a <= 9), and one hidden
    channel's way out to two outputs (|da| <= 2, |dg| <= 6, |du| <= 6)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    sign = lambda *s: torch.randint(0, 2, s, generator=gen, device="cuda") * 2 - 1

    def put(t):
        r = empty_rows(t.shape, dtype)
        r.copy_(t)
        return r

    def sparse(n, k):  # two +-1 in each of n rows of k (one, or their sum, where they meet)
        w = torch.zeros(n, k, dtype=torch.int64, device="cuda")
        at = torch.randint(0, k, (n, 2), generator=gen, device="cuda")
        return w.scatter_add_(1, at, sign(n, 2)).clamp_(-1, 1)

    x, dy = (torch.randint(-1, 2, (m, n), generator=gen, device="cuda") for n in (c, o))
    w = (put(sparse(f, c)), put(sparse(f, c)), put(sparse(f, o).t()))
    b = tuple(sign(n).to(dtype) for n in (f, f, o))
    return put(x), w, b, put(dy)


def exact(x, wg, wu, wd, bg, bu, bd, dy):
    x, wg, wu, wd, bg, bu, bd, dy = (t.double() for t in (x, wg, wu, wd, bg, bu, bd, dy))
    g, u = x @ wg.t() + bg, x @ wu.t() + bu
    a = g.clamp(min=0) * u
    da = dy @ wd
    dg, du = da * u * (g > 0), da * g.clamp(min=0)
    return {"y": a @ wd.t() + bd, "x": dg @ wg + du @ wu, "w_gate": dg.t() @ x, "w_up": du.t() @ x, "w_down": dy.t() @ a,
            "b_gate": dg.sum(0), "b_up": du.sum(0), "b_down": dy.sum(0)}


SHAPES = [(5, 40, 72, 24), (31, 1000, 2600, 1000), (37, 1000, 2600, 1000), (150, 64, 8000, 200), (200, 48, 192, 48),
          (1000, 130, 3000, 70), (3000, 512, 1536, 512), (8192, 640, 1024, 640), (20000, 48, 96, 48), (20000, 160, 200, 136),
          (25920, 96, 384, 96), (63, 33, 65, 127), (100000, 24, 40, 24)]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_whole_numbers(shape, dtype):
    x, w, b, dy = whole(*shape, dtype)
    want = exact(x, *w, *b, dy)
    short = exact(x[:-1], *w, *b, dy[:-1])
    for k in want:
        assert want[k].abs().max() < 2 ** 24
        if k[0] in "wb" and shape[0] > 64:  # the sums over rows would tell that one is missing
            assert not torch.equal(want[k].float(), short[k].float()), k
    assert torch.equal(GatedFFN(*w, *b, act="relu")(x), want["y"].to(dtype))
    for keep in (True, False):
        layer = GatedFFN(*w, *b, act="relu", keep=keep)
        y, saved = layer.forward(x)
        got = {"y": y, **layer.backward(dy, x, saved)}
        for k in want:
            assert torch.equal(got[k], want[k].to(dtype)), (k, keep)
