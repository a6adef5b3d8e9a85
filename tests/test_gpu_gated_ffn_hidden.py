"""The gated feed-forward block's hidden values in memory: more than 2^31 of them, and staged where memory is busy."""
import pytest
import torch

from flyhigh_engine_b200.kernels import GatedFFN, empty_rows
from row_ops_plain import assert_within, ffn

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("hidden", [16384, 16381])
@pytest.mark.parametrize("keep", [True, False])
def test_hidden_values_past_2_31_elements(keep, hidden):
    """135,000 rows of 16,384 (or 16,381, at the same pitch) hidden values in memory, forward and gradient, in tiles (more than 128
    channels). All rows but the first and last 300 are 0, and so are their hidden values: the weights' gradients are those
    of the 600 rows alone."""
    m, c, n = 135000, 136, 300
    gen = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda *s, std=1.0: (std * torch.randn(s, generator=gen, device="cuda")).to(BF16)
    ends = rnd(2 * n, c), rnd(2 * n, c, std=0.5)
    x, dy = (torch.zeros(m, c, dtype=BF16, device="cuda") for _ in range(2))
    for t, e in zip((x, dy), ends):
        t[:n], t[-n:] = e[:n], e[n:]
    down = empty_rows((c, hidden), BF16)
    down.copy_(rnd(c, hidden, std=hidden ** -0.5))
    w = rnd(hidden, c, std=c ** -0.5), rnd(hidden, c, std=c ** -0.5), down
    layer = GatedFFN(*w, keep=keep)
    y, saved = layer.forward(x)
    got = {"y": y, **layer.backward(dy, x, saved)}
    want = ffn(ends[0], *w, dy=ends[1])
    for k, (v, bound) in want.items():
        if k in ("y", "x"):
            assert (got[k][n:-n] == 0).all(), k
            got[k] = torch.cat([got[k][:n], got[k][-n:]])
        assert_within(k, got[k], v, bound)
    assert_within("inference", torch.cat([y[:n], y[-n:]]), *want["y"])
    y = layer(x)
    assert torch.equal(torch.cat([y[:n], y[-n:]]), got["y"])


def test_gradients_of_kept_values_where_memory_is_busy():
    """g and u pass through staging tiles that the next columns' copies take over once every lane has read them. Twelve calls
    with 17 GB of them, in fresh memory each time, have the same gradients to the bit: x's, which every dg and du enters,
    and w_gate's and w_up's, which are single dg and du: 136 rows of x are unit vectors, the others 0."""
    m, c, f = 135000, 136, 16384
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.zeros(m, c, dtype=BF16, device="cuda")
    at = torch.randint(0, m, (c,), generator=gen, device="cuda")
    x[at, torch.arange(c, device="cuda")] = 1
    dy = torch.randn(m, c, generator=gen, device="cuda").to(BF16)
    w = tuple((std * torch.randn(s, generator=gen, device="cuda")).to(BF16) for s, std in (((f, c), 1.0), ((f, c), 1.0), ((c, f), 0.1)))
    layer = GatedFFN(*w, act="relu", keep=True)
    first = None
    for _ in range(12):
        torch.cuda.empty_cache()
        _, saved = layer.forward(x)
        got = layer.backward(dy, x, saved, want=("x", "w_gate", "w_up"))
        del saved
        first = first or got
        for k in got:
            assert torch.equal(got[k], first[k]), k
    rows = torch.unique(at)
    want = ffn(x[rows], *w, act="relu", dy=dy[rows])
    got["x"] = got["x"][rows]
    for k in got:
        assert_within(k, got[k], *want[k])
