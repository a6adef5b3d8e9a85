"""The kernel-level C ABI (include/flyhigh_kernels.h) from Python: ctypes mirrors of its parameter structs, a 3x3
conv on NHWC f16 device tensors, for hosts that drive the conv kernels without the session layer (and for bench.py's
per-conv sweep), and the row operators beside it: the gated feed-forward block (GatedFFN) and the residual norm
(ResidualNorm), forward and gradient, on the rows of f16 or bf16 tensors. Device memory is torch's; the kernels run on
the caller's CUDA stream."""
from __future__ import annotations

import ctypes
import warnings
from ctypes import Structure, c_float, c_int, c_longlong, c_size_t, c_void_p
from typing import Optional

import numpy as np

from . import FlyHighError, lib

MAX_SRC = 6


class ConvSrc(Structure):  # FhConvSrc
    _fields_ = [("p", c_void_p), ("bs", c_longlong), ("cs", c_int), ("nc", c_int), ("scale", c_float), ("slot", c_int)]


class ConvParams(Structure):  # FhConvParams
    _fields_ = [("src", ConvSrc * MAX_SRC), ("nsrc", c_int), ("h", c_int), ("w", c_int), ("ho", c_int), ("wo", c_int),
                ("cp", c_int), ("cout", c_int), ("wpack", c_void_p), ("bias", c_void_p), ("slope", c_void_p),
                ("epi", c_int), ("out", c_void_p), ("out_cs", c_int), ("out_bs", c_longlong), ("res", c_void_p),
                ("res_cs", c_int), ("res_bs", c_longlong), ("n", c_int), ("wm", c_int), ("ngroups", c_int),
                ("wsmem", c_int), ("wait_cycles", c_longlong), ("test_extra_tx", c_int)]


def _up8(c: int) -> int:
    return (c + 7) // 8 * 8


class Conv3x3:
    """One 3x3 conv layer (pad 1, bias, optional PReLU slopes, optional residual) on NHWC f16 torch tensors.

    kernel "mma" (fhk_conv3x3: mma.sync, stride 1 or 2; wm = rows per CTA pair, 0 = by size) or "umma"
    (fhk_conv3x3_umma: tcgen05, stride 1 where fhk_conv_umma_fits; wm 1 = its persistent variant). weight: [cout][cin][3][3] (float values, rounded
    to f16); the input tensor is [n][h][w][cs] with cs = 4 for cin <= 4 else cin rounded up to 8."""

    def __init__(self, weight, bias, slope=None, stride: int = 1, kernel: str = "mma", wm: int = 0, device="cuda"):
        import torch
        L = lib()
        w = np.asarray(weight, np.float32)
        self.cout, self.cin = int(w.shape[0]), int(w.shape[1])
        self.stride, self.kernel, self.wm = int(stride), kernel, int(wm)
        self.cs = 4 if self.cin <= 4 else _up8(self.cin)
        self.cp = (_up8(self.cin) + 15) // 16 * 16
        umma = kernel == "umma"
        if umma and not (stride == 1 and L.fhk_conv_umma_fits(self.cp, self.cout, 1)):
            raise FlyHighError(f"conv {self.cin}->{self.cout} stride {stride}: the tcgen05 kernel does not take it")
        if umma and wm == 1 and not L.fhk_conv_umma_persistent_fits(self.cp, self.cout):
            raise FlyHighError(f"conv {self.cin}->{self.cout}: the persistent tcgen05 variant does not take it")
        cmap = np.full(self.cp, -1, np.int32)
        cmap[:self.cin] = np.arange(self.cin)
        n_pack = (L.fhk_conv_packed_elems_umma if umma else L.fhk_conv_packed_elems)(self.cout, self.cp)
        packed = np.zeros(n_pack, np.uint16)
        bits = np.ascontiguousarray(w.astype(np.float16)).view(np.uint16)
        pack = L.fhk_conv_pack_weights_umma if umma else L.fhk_conv_pack_weights
        if pack(bits.ctypes.data, self.cin, self.cout, cmap.ctypes.data, self.cp, packed.ctypes.data) != 0:
            raise FlyHighError("weight packing failed")
        self.wpack = torch.from_numpy(packed.view(np.int16)).to(device)
        self.bias = torch.from_numpy(np.asarray(bias, np.float32)).to(device)
        self.slope = None if slope is None else torch.from_numpy(np.asarray(slope, np.float32)).to(device)
        self.ocs = _up8(self.cout)

    def out_shape(self, n: int, h: int, w: int):
        return (n, (h - 1) // self.stride + 1, (w - 1) // self.stride + 1, self.ocs)

    def params(self, x, out, res=None) -> ConvParams:
        n, h, w, cs = x.shape
        assert cs == self.cs and tuple(out.shape) == self.out_shape(n, h, w)
        p = ConvParams()
        p.src[0] = ConvSrc(x.data_ptr(), h * w * cs, cs, self.cin, 1.0, 0)
        p.nsrc, p.h, p.w = 1, h, w
        p.ho, p.wo = out.shape[1], out.shape[2]
        p.cp, p.cout = self.cp, self.cout
        p.wpack, p.bias = self.wpack.data_ptr(), self.bias.data_ptr()
        p.slope = self.slope.data_ptr() if self.slope is not None else None
        p.out, p.out_cs, p.out_bs = out.data_ptr(), self.ocs, out.shape[1] * out.shape[2] * self.ocs
        if res is not None:
            assert tuple(res.shape) == tuple(out.shape)
            p.res, p.res_cs, p.res_bs = res.data_ptr(), self.ocs, p.out_bs
        p.n, p.wm = n, self.wm
        return p

    def launch(self, p: ConvParams, stream: int) -> None:
        L = lib()
        st = c_void_p(stream)
        rc = L.fhk_conv3x3_umma(ctypes.byref(p), st) if self.kernel == "umma" else \
            L.fhk_conv3x3(ctypes.byref(p), self.stride, st)
        if rc != 0:
            raise FlyHighError(f"conv launch failed: CUDA error {rc}")

    def __call__(self, x, res=None, out=None):
        import torch
        n, h, w, _ = x.shape
        if out is None:
            out = torch.zeros(self.out_shape(n, h, w), dtype=torch.float16, device=x.device)
        self.launch(self.params(x, out, res), torch.cuda.current_stream().cuda_stream)
        return out


# ---- row operators ----

ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3, "sigmoid": 4}
NORMS = {"none": 0, "rms": 1, "layer": 2}


class GatedFfnParams(Structure):  # FhGatedFfnParams
    _fields_ = [(n, c_void_p) for n in ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down", "y", "a", "g", "u")] + \
        [(n, c_longlong) for n in ("x_pitch", "wg_pitch", "wu_pitch", "wd_pitch", "y_pitch", "h_pitch", "m")] + \
        [(n, c_int) for n in ("cin", "hidden", "cout", "act", "dtype")] + \
        [("scratch", c_void_p), ("scratch_bytes", c_size_t), ("wait_cycles", c_longlong), ("test_extra_tx", c_int)]


class GatedFfnGradParams(Structure):  # FhGatedFfnGradParams
    _fields_ = [(n, c_void_p) for n in ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "g", "u", "a", "dy", "dx", "dw_gate", "dw_up",
                                        "dw_down", "db_gate", "db_up", "db_down")] + \
        [(n, c_longlong) for n in ("x_pitch", "wg_pitch", "wu_pitch", "wd_pitch", "h_pitch", "dy_pitch", "dx_pitch",
                                   "dwg_pitch", "dwu_pitch", "dwd_pitch", "m")] + \
        [(n, c_int) for n in ("cin", "hidden", "cout", "act", "dtype")] + \
        [("scratch", c_void_p), ("scratch_bytes", c_size_t), ("wait_cycles", c_longlong), ("test_extra_tx", c_int)]


class ResidualNormParams(Structure):  # FhResidualNormParams
    _fields_ = [(n, c_void_p) for n in ("x", "f", "gate", "scale", "w_post", "b_post", "w_pre", "b_pre", "y", "h")] + \
        [(n, c_longlong) for n in ("x_pitch", "f_pitch", "y_pitch", "h_pitch", "gate_pitch", "m")] + \
        [(n, c_int) for n in ("c", "gates", "pre", "post")] + [("eps", c_float), ("dtype", c_int)]


class ResidualNormGradParams(Structure):  # FhResidualNormGradParams
    _fields_ = [(n, c_void_p) for n in ("dy", "dh", "y", "f", "gate", "scale", "w_post", "b_post", "w_pre", "dx", "df",
                                        "dgate", "dscale", "dw_post", "db_post", "dw_pre", "db_pre")] + \
        [(n, c_longlong) for n in ("dy_pitch", "dh_pitch", "y_pitch", "f_pitch", "gate_pitch", "dx_pitch", "df_pitch",
                                   "dgate_pitch", "m")] + \
        [(n, c_int) for n in ("c", "gates", "pre", "post")] + [("eps", c_float), ("dtype", c_int)] + \
        [("scratch", c_void_p), ("scratch_bytes", c_size_t)]


def empty_rows(shape, dtype, device="cuda"):
    """An uninitialised tensor of rows for the row operators: shape (..., channels), each row beginning on a 16-byte
    boundary (a pitch of channels rounded up to 8, as the feature maps of the convs)."""
    import torch
    *lead, c = shape
    t = torch.empty((*lead, _up8(c)), dtype=dtype, device=device)
    return t if c % 8 == 0 else t[..., :c]


def _rows_like(t):
    """empty_rows of t's shape, type and device; t is a tensor of rows."""
    import torch
    c = t.shape[-1]
    if c % 8 == 0:
        return torch.empty_like(t)
    if t.dim() == 2:
        return torch.empty_strided(t.shape, (_up8(c), 1), dtype=t.dtype, device=t.device)
    return empty_rows(t.shape, t.dtype, t.device)


def _dtype_code(dtype) -> int:
    import torch
    if dtype == torch.float16:
        return 0
    if dtype == torch.bfloat16:
        return 1
    raise FlyHighError(f"row operators take float16 or bfloat16 tensors, not {dtype}")


def _rows(name: str, t, channels: int, dtype, device):
    """(pointer, pitch, rows) of a tensor of rows (..., channels); refuses what the kernels cannot address."""
    if t.dtype != dtype or t.device != device:
        raise FlyHighError(f"{name}: a {dtype} tensor on {device} is expected, got {t.dtype} on {t.device}")
    shape, stride = t.shape, t.stride()
    if len(shape) < 1 or shape[-1] != channels:
        raise FlyHighError(f"{name}: rows of {channels} channels are expected, got shape {tuple(shape)}")
    m, pitch = 1, 0
    if len(shape) == 2:
        m, pitch = shape[0], stride[0]
    else:
        for n, st in zip(reversed(shape[:-1]), reversed(stride[:-1])):  # the leading dimensions as one of constant pitch
            if n == 1:
                continue
            if m == 1:
                pitch = st
            elif st != pitch * m and 0 not in shape[:-1]:
                raise FlyHighError(f"{name}: its leading dimensions are not rows of one pitch (strides {stride})")
            m *= n
    ptr = t.data_ptr()
    if m <= 1:
        pitch = (channels + 7) // 8 * 8
    if (pitch < channels or pitch & 7 or ptr & 15 or (stride[-1] != 1 and channels > 1)) and m:
        raise FlyHighError(f"{name}: rows must be contiguous, begin on 16-byte boundaries and not overlap (strides "
                           f"{stride}, pointer {ptr:#x}); empty_rows allocates such tensors")
    return ptr, pitch, m


def _like(name: str, t, m: int, channels: int, dtype, device):
    """(pointer, pitch) of a tensor of m rows."""
    ptr, pitch, rows = _rows(name, t, channels, dtype, device)
    if rows != m:
        raise FlyHighError(f"{name}: {m} rows are expected, got {rows}")
    return ptr, pitch


def _vector(name: str, t, n: int, dtype, device) -> Optional[int]:
    if t is None:
        return None
    if t.dtype != dtype or t.device != device or tuple(t.shape) != (n,) or not t.is_contiguous() or t.data_ptr() & 15:
        raise FlyHighError(f"{name}: a contiguous, 16-byte aligned {dtype} vector of {n} on {device} is expected, got "
                           f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


class _Places:
    """Where a layer's parameters lie. A layer keeps its calls' parameter blocks with their pointers, and binds them anew
    where this has changed (a parameter's .data was replaced, a module was moved). Asked at every call, so it looks at what
    a replacement of the same shape and type may change: the addresses, and the pitches of matrices (0.8 us; all of
    shape, strides and type took 3)."""

    def __init__(self, tensors):
        given = [t for t in tensors if t is not None]
        self.ptr, self.stride = [t.data_ptr for t in given], [t.stride for t in given if t.dim() > 1]
        self.was = self.now()

    def now(self):
        return [f() for f in self.ptr], [f() for f in self.stride]

    def changed(self) -> bool:
        return self.now() != self.was


def _outside_autograd(layer: str, tensors, stacklevel: int) -> None:
    """Says so when autograd is on and would be expected to record a call that it cannot see."""
    import torch
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                warnings.warn(f"{layer} is not recorded by autograd, though one of its tensors requires a gradient: its outputs "
                              "are cut off from it. Call backward of the layer, and the layer under torch.no_grad()",
                              stacklevel=stacklevel)
                return


class _Call:
    """One entry point on the current stream of the tensors' device, and its scratch: the bytes by sizes are asked for
    once per layer (`sizes`, a dict of its own), the memory is torch's, for this call alone."""

    def __init__(self, what: str, name: str, scratch: Optional[str]):
        self.what, self.name, self.scratch_name, self.fn = what, name, scratch, None

    def __call__(self, p, device, sizes=None, key=None) -> None:
        import torch
        if self.fn is None:
            if self.scratch_name is not None:
                self.scratch_bytes = getattr(lib(), self.scratch_name)
            self.fn = getattr(lib(), self.name)
        ref, scratch = ctypes.byref(p), None
        if sizes is not None:
            n = sizes.get(key)
            if n is None:
                if len(sizes) >= 4096:
                    sizes.clear()
                n = sizes[key] = self.scratch_bytes(ref)
            if n:
                scratch = torch.empty(n, dtype=torch.uint8, device=device)
                p.scratch, p.scratch_bytes = scratch.data_ptr(), n
        stream = torch._C._cuda_getCurrentRawStream(device.index)  # torch.cuda.current_stream(device) without its object
        if torch.cuda.current_device() == device.index:
            rc = self.fn(ref, stream)
        else:
            with torch.cuda.device(device):
                rc = self.fn(ref, stream)
        if rc != 0:
            raise FlyHighError(f"{self.what} failed: CUDA error {rc}")


_gated_ffn = _Call("gated_ffn", "fhk_gated_ffn", "fhk_gated_ffn_scratch_bytes")
_gated_ffn_grad = _Call("gated_ffn gradient", "fhk_gated_ffn_grad", "fhk_gated_ffn_grad_scratch_bytes")
_residual_norm = _Call("residual_norm", "fhk_residual_norm", None)
_residual_norm_grad = _Call("residual_norm gradient", "fhk_residual_norm_grad", "fhk_residual_norm_grad_scratch_bytes")


class GatedFFNSaved:
    """What a training forward call keeps for the gradient: the activated product a, and the projections g and u in f32;
    nothing (None) where the gradient forms them again."""

    def __init__(self, rows: int, channels: int, a=None, gu=None):
        self.rows, self.channels, self._a, self._gu = rows, channels, a, gu  # (rows, pitch), (2, rows, pitch)

    @property
    def a(self):
        return None if self._a is None else self._a[:, :self.channels]

    @property
    def g(self):
        return None if self._gu is None else self._gu[0, :, :self.channels]

    @property
    def u(self):
        return None if self._gu is None else self._gu[1, :, :self.channels]


class GatedFFN:
    """Gated feed-forward block on rows (the pixels of an NHWC map, or tokens):
    y = (act(x w_gate^T + b_gate) * (x w_up^T + b_up)) w_down^T + b_down.

    w_gate, w_up: [hidden][cin], w_down: [cout][hidden], biases [hidden], [hidden], [cout] or None: CUDA tensors of one
    type (float16 or bfloat16), used where they lie at each call (no copy: an optimiser may update them in place, or their
    .data be replaced by a tensor of the same shape, type and device; a captured graph keeps the place of its capture).
    act: silu, gelu (erf), gelu_tanh, relu or sigmoid. x: (..., cin); every tensor's rows begin on 16-byte boundaries
    (empty_rows). keep: whether a training forward call keeps the hidden values for its gradient (10 bytes each), or the
    gradient forms them again, from the weights as they are when it is called; None: the faster, which is to form them
    again up to 448 channels in and out (bf16 step, keeping / forming again: 60,000 x 256 -> 1024 472 / 416 us, 16,000 x
    384 -> 1536 271 / 261, 16,000 x 512 -> 2048 335 / 348).
    wait_cycles: the bound of each wait inside the kernels, in SM clock cycles (0: about a second); a wait that runs out ends
    its call with unusable outputs, which `check` reports.
    No autograd: forward / backward are called by the training step, under torch.no_grad() where a tensor requires a
    gradient (else a warning says that nothing is recorded)."""

    def __init__(self, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, act: str = "silu", keep: Optional[bool] = None,
                 wait_cycles: int = 0):
        if not 0 <= wait_cycles < 2 ** 63:
            raise FlyHighError(f"wait_cycles {wait_cycles} is not a number of cycles")
        if act not in ACTIVATIONS:
            raise FlyHighError(f"unknown activation {act!r}: one of {', '.join(ACTIVATIONS)}")
        if w_gate.dim() != 2 or w_down.dim() != 2 or not w_gate.is_cuda:
            raise FlyHighError("the weights are CUDA matrices")
        self.dtype, self.device, self.act = w_gate.dtype, w_gate.device, act
        self.hidden, self.cin = w_gate.shape
        self.cout, self.wait_cycles = w_down.shape[0], int(wait_cycles)
        self.weights = (w_gate, w_up, w_down)
        self.biases = (b_gate, b_up, b_down)
        self._bind()
        self._sizes, self._grad_sizes = {}, {}
        self.keep = max(self.cin, self.cout) > 448 if keep is None else bool(keep)

    def _bind(self) -> None:
        """The calls' parameter blocks with all that does not change from call to call."""
        code, places = _dtype_code(self.dtype), _Places(self.weights + self.biases)
        (w_gate, w_up, w_down), (b_gate, b_up, b_down) = self.weights, self.biases
        wg, wgp, mg = _rows("w_gate", w_gate, self.cin, self.dtype, self.device)
        wu, wup, mu = _rows("w_up", w_up, self.cin, self.dtype, self.device)
        wd, wdp, md = _rows("w_down", w_down, self.hidden, self.dtype, self.device)
        if (mg, mu, md) != (self.hidden, self.hidden, self.cout) or w_up.dim() != 2 or min(self.hidden, self.cin, self.cout) < 1:
            raise FlyHighError(f"w_gate {tuple(w_gate.shape)}, w_up {tuple(w_up.shape)} and w_down {tuple(w_down.shape)} do not match")
        bias = [_vector(n, b, k, self.dtype, self.device) for n, b, k in
                (("b_gate", b_gate, self.hidden), ("b_up", b_up, self.hidden), ("b_down", b_down, self.cout))]
        common = dict(w_gate=wg, w_up=wu, w_down=wd, wg_pitch=wgp, wu_pitch=wup, wd_pitch=wdp, cin=self.cin,
                      hidden=self.hidden, cout=self.cout, act=ACTIVATIONS[self.act], dtype=code, h_pitch=_up8(self.hidden),
                      wait_cycles=self.wait_cycles)
        self._forward_params = GatedFfnParams(**common, b_gate=bias[0], b_up=bias[1], b_down=bias[2])
        self._grad_params = GatedFfnGradParams(**common, b_gate=bias[0], b_up=bias[1])
        self._places = places

    def _block(self, which: str):
        """A copy of a parameter block, bound to where the weights are now."""
        if self._places.changed():
            self._bind()
        p = getattr(self, which)
        return type(p).from_buffer_copy(p)

    def _forward(self, x, out, keep: bool):
        import torch
        _outside_autograd("GatedFFN", (x, *self.weights, *self.biases), 4)
        p = self._block("_forward_params")
        p.x, p.x_pitch, m = _rows("x", x, self.cin, self.dtype, self.device)
        if out is None:
            out = _rows_like(x) if self.cout == self.cin else empty_rows((*x.shape[:-1], self.cout), self.dtype, self.device)
            p.y, p.y_pitch = out.data_ptr(), _up8(self.cout)
        else:
            p.y, p.y_pitch = _like("out", out, m, self.cout, self.dtype, self.device)
        p.m = m
        if not keep:
            _gated_ffn(p, self.device, self._sizes, m)
            return out, m
        hp = p.h_pitch
        a = torch.empty((m, hp), dtype=self.dtype, device=self.device)
        gu = torch.empty((2, m, hp), dtype=torch.float32, device=self.device)
        p.a, p.g, p.u = a.data_ptr(), gu.data_ptr(), gu.data_ptr() + 4 * m * hp
        _gated_ffn(p, self.device, self._sizes, (m, True))
        return out, GatedFFNSaved(m, self.hidden, a, gu)

    def check(self) -> None:
        """Waits for the layer's device and raises if a wait inside the kernels of any gated feed-forward block there ran
        out since the last check: the outputs of the calls since then are not to be used. Not during a stream capture."""
        import torch
        with torch.cuda.device(self.device):
            torch.cuda.synchronize()
            n = lib().fhk_gated_ffn_wait_timeouts(1)
        if n:
            raise FlyHighError(f"gated_ffn: {n} waits inside its kernels ran out" if n > 0 else "gated_ffn: its count of waits cannot be read")

    def __call__(self, x, out=None):
        """y for x (inference: nothing is kept)."""
        return self._forward(x, out, False)[0]

    def forward(self, x, out=None):
        """(y, saved): y, and what `backward` needs beside x."""
        y, saved = self._forward(x, out, self.keep)
        return y, saved if self.keep else GatedFFNSaved(saved, self.hidden)

    def backward(self, dy, x, saved: GatedFFNSaved, want=None) -> dict:
        """The gradients for dy of the call that returned `saved`: "x", "w_gate", "w_up", "w_down" and the biases' there
        are, or those of them that `want` lists. They are new tensors, each written whole."""
        import torch
        names = ["x", "w_gate", "w_up", "w_down"] + [n for n, b in zip(("b_gate", "b_up", "b_down"), self.biases) if b is not None]
        if want is not None:
            if not set(want) <= set(names):
                raise FlyHighError(f"gradients of {sorted(set(want) - set(names))} are not among {names}")
            names = [n for n in names if n in set(want)]
        p = self._block("_grad_params")
        p.x, p.x_pitch, m = _rows("x", x, self.cin, self.dtype, self.device)
        p.dy, p.dy_pitch, mdy = _rows("dy", dy, self.cout, self.dtype, self.device)
        a = saved._a
        if mdy != m or saved.rows != m or saved.channels != self.hidden or \
                (a is not None and (a.dtype != self.dtype or a.device != self.device)):
            raise FlyHighError(f"x ({m} rows), dy ({mdy}) and saved ({saved.rows}) are not of one call")
        p.m = m
        if a is not None:
            at = saved._gu.data_ptr()
            p.a, p.g, p.u = a.data_ptr(), at, at + 4 * m * p.h_pitch
        r = {}
        if "x" in names:
            r["x"] = _rows_like(x)
            p.dx, p.dx_pitch = r["x"].data_ptr(), _up8(self.cin)
        if "w_gate" in names:
            r["w_gate"] = _rows_like(self.weights[0])
            p.dw_gate, p.dwg_pitch = r["w_gate"].data_ptr(), _up8(self.cin)
        if "w_up" in names:
            r["w_up"] = _rows_like(self.weights[1])
            p.dw_up, p.dwu_pitch = r["w_up"].data_ptr(), _up8(self.cin)
        if "w_down" in names:
            r["w_down"] = _rows_like(self.weights[2])
            p.dw_down, p.dwd_pitch = r["w_down"].data_ptr(), _up8(self.hidden)
        biases = [n for n in names if n[0] == "b"]
        if biases:
            for n, b in zip(("b_gate", "b_up", "b_down"), self.biases):
                if n in biases:
                    r[n] = torch.empty_like(b)
                    setattr(p, "d" + n, r[n].data_ptr())
        _gated_ffn_grad(p, self.device, self._grad_sizes, (m, a is None, *names))
        return r


class ResidualNorm:
    """The join of a block with its residual stream and the next block's norm, one pass over the rows:
    y = x + scale * gate * norm_post(f), h = norm_pre(y).

    pre, post: "rms", "layer" or "none"; w_pre, b_pre, w_post, b_post, scale: vectors of `channels` or None (a norm
    without them is only normalised). x, f: (..., channels); gate: (gates, channels) of any alignment, each of its rows
    for an equal run of rows (one per image of a batch, say), or None. f None: y is x (the norm before a first block). No
    autograd, as for GatedFFN."""

    def __init__(self, channels: int, dtype, pre: str = "rms", post: str = "none", w_pre=None, b_pre=None, w_post=None,
                 b_post=None, scale=None, eps: float = 1e-6):
        for kind in (pre, post):
            if kind not in NORMS:
                raise FlyHighError(f"unknown norm {kind!r}: one of {', '.join(NORMS)}")
        if not 1 <= channels <= 8192:
            raise FlyHighError(f"residual norms take 1 to 8192 channels, not {channels}")
        if not 0 <= eps < float("inf"):
            raise FlyHighError(f"eps {eps} is not a finite number >= 0")
        if (pre == "none" and (w_pre is not None or b_pre is not None)) or \
                (post == "none" and (w_post is not None or b_post is not None)):
            raise FlyHighError("a weight or bias was given for a norm that is none")
        self.channels, self.dtype, self.pre, self.post, self.eps = channels, dtype, pre, post, float(eps)
        self.params = {"w_pre": w_pre, "b_pre": b_pre, "w_post": w_post, "b_post": b_post, "scale": scale}
        _dtype_code(dtype)
        given = [t for t in self.params.values() if t is not None]
        if given and not given[0].is_cuda:
            raise FlyHighError("the norms' vectors are CUDA tensors")
        self.device = given[0].device if given else None
        self._bind()
        self._names = [n for n, t in self.params.items() if t is not None]
        self._sizes = {}

    def _bind(self) -> None:
        """The calls' parameter blocks with all that does not change from call to call."""
        places = _Places(self.params.values())
        ptrs = {n: _vector(n, t, self.channels, self.dtype, self.device) for n, t in self.params.items() if t is not None}
        common = dict(c=self.channels, pre=NORMS[self.pre], post=NORMS[self.post], eps=self.eps, dtype=_dtype_code(self.dtype))
        self._forward_params = ResidualNormParams(**common, **ptrs)
        ptrs.pop("b_pre", None)
        self._grad_params = ResidualNormGradParams(**common, **ptrs)
        self._places = places

    def _block(self, which: str):
        """A copy of a parameter block, bound to where the vectors are now."""
        if self._places.changed():
            self._bind()
        p = getattr(self, which)
        return type(p).from_buffer_copy(p)

    def _device(self, t):
        if not t.is_cuda or (self.device is not None and t.device != self.device):
            raise FlyHighError(f"a CUDA tensor on {self.device or 'a GPU'} is expected, got one on {t.device}")
        return t.device

    def _gate(self, p, gate, m, device):
        if gate.dim() != 2:
            raise FlyHighError(f"gate: (gates, {self.channels}) is expected, got {tuple(gate.shape)}")
        n, c = gate.shape
        if gate.dtype != self.dtype or gate.device != device or c != self.channels or \
                (n > 1 and gate.stride(0) < c) or (c > 1 and gate.stride(1) != 1):
            raise FlyHighError(f"gate: rows of {self.channels} {self.dtype} values on {device} are expected, got {gate.dtype} "
                               f"{tuple(gate.shape)} (strides {gate.stride()}) on {gate.device}")
        if n < 1 or m % n:
            raise FlyHighError(f"gate: {n} rows do not divide the {m} rows")
        p.gate, p.gate_pitch, p.gates = gate.data_ptr(), gate.stride(0) if n > 1 else c, n

    def __call__(self, x, f=None, gate=None):
        """(y, h); h is None where pre is "none", and y is x itself where f is None."""
        _outside_autograd("ResidualNorm", (x, f, gate, *self.params.values()), 3)
        dev, c, dt = self._device(x), self.channels, self.dtype
        p = self._block("_forward_params")
        p.x, p.x_pitch, m = _rows("x", x, c, dt, dev)
        p.m = m
        y, h = x, None
        if f is not None:
            p.f, p.f_pitch = _like("f", f, m, c, dt, dev)
            if gate is not None:
                self._gate(p, gate, m, dev)
            y = _rows_like(x)
            p.y, p.y_pitch = y.data_ptr(), _up8(c)
        else:
            if gate is not None or self.pre == "none":
                raise FlyHighError("without f there is no gate, and a norm before the block")
            p.post, p.scale, p.w_post, p.b_post = 0, None, None, None
        if self.pre != "none":
            h = _rows_like(x)
            p.h, p.h_pitch = h.data_ptr(), _up8(c)
        _residual_norm(p, dev)
        return y, h

    def backward(self, dy, dh, y, f=None, gate=None) -> dict:
        """The gradients for dy and dh (either may be None: zero) of the call that returned y: "x", and with f "f",
        "gate" where there is one, and those of the vectors there are. They are new tensors, each written whole."""
        import torch
        first = dy if dy is not None else dh
        if first is None or (dh is not None and self.pre == "none"):
            raise FlyHighError("dy or dh is needed, and dh only with a norm before the next block")
        dev, c, dt = self._device(first), self.channels, self.dtype
        p = self._block("_grad_params")
        ptr, pitch, m = _rows("dy" if dy is not None else "dh", first, c, dt, dev)
        p.m = m
        if dy is not None:
            p.dy, p.dy_pitch = ptr, pitch
        if dh is not None:
            p.dh, p.dh_pitch = (ptr, pitch) if dy is None else _like("dh", dh, m, c, dt, dev)
            p.y, p.y_pitch = _like("y", y, m, c, dt, dev)
        r = {"x": _rows_like(first)}
        p.dx, p.dx_pitch = r["x"].data_ptr(), _up8(c)
        if f is not None:
            p.f, p.f_pitch = _like("f", f, m, c, dt, dev)
            r["f"] = _rows_like(first)
            p.df, p.df_pitch = r["f"].data_ptr(), _up8(c)
            if gate is not None:
                self._gate(p, gate, m, dev)
                r["gate"] = gate.new_empty(gate.shape)
                p.dgate, p.dgate_pitch = r["gate"].data_ptr(), c
        else:
            if gate is not None:
                raise FlyHighError("without f there is no gate")
            p.post, p.scale, p.w_post, p.b_post = 0, None, None, None
        names = self._names if f is not None else [n for n in self._names if n in ("w_pre", "b_pre")]
        for n in names:
            r[n] = torch.empty_like(self.params[n])
            setattr(p, "d" + n, r[n].data_ptr())
        _residual_norm_grad(p, dev, self._sizes, (m, p.gates))
        return r
