"""Waits that run out inside the gated feed-forward block's kernels. A barrier that expects 16 bytes more than its copies bring
never completes, so the waits for it, and those for what should follow, end at their bound: the call gives up, GatedFFN.check
raises, and the next call is right. Every role of the kernels has such a bound, so each launch ends."""
import ctypes

import pytest
import torch

import flyhigh_engine_b200 as fh
from flyhigh_engine_b200.kernels import GatedFFN
from test_gpu_gated_ffn import block
from test_row_ops import INVALID, ffn_params, grad_params

F16 = torch.float16
LIMIT = 2000000  # cycles: about a millisecond


@pytest.mark.parametrize("extra", [-16, 8, 65552])
def test_refusals(extra):
    assert fh.lib().fhk_gated_ffn(ctypes.byref(ffn_params(test_extra_tx=extra)), None) == INVALID
    assert fh.lib().fhk_gated_ffn_grad(ctypes.byref(grad_params(test_extra_tx=extra)), None) == INVALID


@pytest.mark.gpu
@pytest.mark.parametrize("shape,keep", [((200, 48, 192, 48), False), ((20300, 64, 640, 64), False), ((200, 136, 260, 72), True),
                                        ((200, 136, 260, 72), False), ((2000, 512, 1536, 512), True), ((2000, 512, 1536, 512), False)], ids=str)
def test_waits_that_run_out_are_reported(shape, keep):
    x, w, b, dy = block(*shape, F16)
    layer = GatedFFN(*w, *b, keep=keep, wait_cycles=LIMIT)

    def step():
        y, saved = layer.forward(x)
        return {"y": y, "inference": layer(x), **layer.backward(dy, x, saved)}

    want = step()
    layer.check()
    saved = layer.forward(x)[1]
    for params, call in ((layer._forward_params, lambda: layer(x)), (layer._forward_params, lambda: layer.forward(x)),
                         (layer._grad_params, lambda: layer.backward(dy, x, saved))):
        params.test_extra_tx = 16
        call()
        with pytest.raises(fh.FlyHighError, match="ran out"):
            layer.check()
        params.test_extra_tx = 0
        layer.check()  # reported once
        got = step()
        layer.check()
        assert all(torch.equal(got[k], want[k]) for k in want)


@pytest.mark.gpu
def test_a_side_stream_is_waited_for():
    """torch's side streams do not wait for the legacy stream that the count is read on."""
    x, w, b, _ = block(2000, 512, 1536, 512, F16)
    layer = GatedFFN(*w, *b, wait_cycles=LIMIT)
    layer._forward_params.test_extra_tx = 16
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x)
    with pytest.raises(fh.FlyHighError, match="ran out"):
        layer.check()
    with pytest.raises(fh.FlyHighError, match="wait_cycles"):
        GatedFFN(*w, *b, wait_cycles=-1)
