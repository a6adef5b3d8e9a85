"""Timed cases of the row-wise operators of flyhigh_engine_b200.kernels: the gated feed-forward block (GatedFFN) and the
residual norm (ResidualNorm: norms before and after a block with its gate and residual scale), forward and training.

`run` computes them in their plain form (elementary torch operations in 32 bits, rounded once at the end), or, with
`own` set, by the package's kernels. `exact` gives the same outputs from the definitions in 64 bits."""
import math

import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-5


# ---- cases ----

def _ffn(name, rows, cin, hidden, cout, dtype, act, bias, train):
    return {"name": name, "op": "ffn", "rows": rows, "cin": cin, "hidden": hidden, "cout": cout, "dtype": dtype,
            "act": act, "bias": bias, "train": train}


def _norm(name, rows, channels, dtype, pre, post, affine, scale, gates, train):
    return {"name": name, "op": "norm", "rows": rows, "channels": channels, "dtype": dtype, "pre": pre, "post": post,
            "affine": affine, "scale": scale, "gates": gates, "train": train}


def listed():
    return [
        # one row through a wide block: a token, or a pooled descriptor; the launches and the weights' bytes count
        _ffn("ffn_one_row", 1, 1024, 4096, 1024, "bf16", "silu", False, False),
        # a ragged handful of rows, channel counts that fill no tile
        _ffn("ffn_few_rows_ragged", 37, 1000, 2600, 1000, "f16", "gelu", True, False),
        # the 1/8-resolution map of a 1080p frame (108 x 60) at the engine's recurrent width
        _ffn("ffn_e8_map", 6480, 48, 192, 48, "f16", "gelu", True, False),
        # a 480 x 270 map, the largest of the conv sweep's inputs at its widest: many rows, few channels
        _ffn("ffn_quarter_map", 129600, 64, 256, 64, "f16", "silu", True, False),
        # a long batch of rows through a wide block
        _ffn("ffn_wide", 8192, 2048, 8192, 2048, "bf16", "silu", False, False),
        # training on the 216 x 120 map of a 1080p frame, 96 channels (the engine's widest)
        _ffn("ffn_train_map", 25920, 96, 384, 96, "f16", "gelu_tanh", True, True),
        # training a wide block, the largest case
        _ffn("ffn_train_wide", 8192, 2048, 8192, 2048, "bf16", "silu", False, True),
        # one row between two blocks
        _norm("norm_one_row", 1, 2048, "bf16", "rms", "rms", True, True, 1, False),
        # the 480 x 270 map, one gate row per image of a batch of four (the place of a per-image modulation)
        _norm("norm_map_gated", 4 * 32400, 64, "f16", "layer", "none", True, True, 4, False),
        # a long batch of wide rows
        _norm("norm_wide", 16384, 4096, "bf16", "rms", "rms", True, False, 0, False),
        # training, odd channel count, three images
        _norm("norm_train_ragged", 3333, 1001, "f16", "layer", "layer", True, True, 3, True),
        # training a wide block's norms, a gate row per image of eight
        _norm("norm_train_wide", 16384, 2048, "bf16", "rms", "rms", True, True, 8, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    top = work(listed()[6])
    while True:
        train = rng.random() < 0.45
        dtype = rng.choice(["f16", "bf16"])
        if rng.random() < 0.6:
            cin, hidden = _log(rng, 16, 4096), _log(rng, 32, 16384)
            cout = cin if rng.random() < 0.7 else _log(rng, 16, 4096)
            if rng.random() < 0.5:  # whole tiles' worth of channels, as most blocks have
                cin, hidden, cout = (max(16, (v + 15) // 16 * 16) for v in (cin, hidden, cout))
            c = _ffn("", _log(rng, 1, 131072), cin, hidden, cout, dtype,
                     rng.choice(["silu", "gelu", "gelu_tanh", "relu", "sigmoid"]), rng.random() < 0.5, train)
        else:
            gates = rng.choice([0, 1, 2, 5, 8])
            rows = _log(rng, 1, 131072)
            if gates > 1:
                rows = max(1, rows // gates) * gates
            pre = rng.choice(["rms", "layer", "rms", "layer", "none"])
            post = rng.choice(["rms", "layer", "none"])
            c = _norm("", rows, _log(rng, 16, 8192), dtype, pre, post, rng.random() < 0.8, rng.random() < 0.5, gates, train)
        del c["name"]
        w = work(c)
        if w["flops"] <= top["flops"] and w["bytes"] <= top["bytes"]:
            return c


def work(case):
    if case["op"] == "ffn":
        m, c, f, o = case["rows"], case["cin"], case["hidden"], case["cout"]
        weights = f * (2 * c + o) + (2 * f + o if case["bias"] else 0)
        values, flops = m * (c + o) + weights, 2 * m * f * (2 * c + o)
        if case["train"]:
            return {"bytes": 2 * (2 * m * (c + o) + 2 * weights), "flops": 3 * flops}
        return {"bytes": 2 * values, "flops": flops}
    m, c = case["rows"], case["channels"]
    tensors = 4 if case["pre"] != "none" else 3  # x, f -> y, h
    params = c * ((2 * (case["pre"] != "none") + 2 * (case["post"] != "none")) * case["affine"] + case["scale"] + case["gates"])
    per_value = 6 + 5 * (case["pre"] != "none") + 5 * (case["post"] != "none")
    if case["train"]:  # and dy, dh -> dx, df
        return {"bytes": 2 * (2 * tensors * m * c + 2 * params), "flops": 3 * per_value * m * c}
    return {"bytes": 2 * (tensors * m * c + params), "flops": per_value * m * c}


# ---- inputs ----

def _rows(gen, rows, channels, dtype, std=1.0):
    """Normal values, each row beginning on a 16-byte boundary (the pitch of the package's feature maps)."""
    pitch = (channels + 7) // 8 * 8
    return (torch.randn(rows, pitch, generator=gen, device="cuda") * std).to(dtype)[:, :channels]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    t = _TYPES[case["dtype"]]
    s = dict(case)
    vec = lambda n, std, mean=0.0: (mean + std * torch.randn(n, generator=gen, device="cuda")).to(t)
    m = case["rows"]
    if case["op"] == "ffn":
        c, f, o = case["cin"], case["hidden"], case["cout"]
        s["x"] = _rows(gen, m, c, t)
        s["w_gate"], s["w_up"] = _rows(gen, f, c, t, c ** -0.5), _rows(gen, f, c, t, c ** -0.5)
        s["w_down"] = _rows(gen, o, f, t, f ** -0.5)
        s["b_gate"], s["b_up"], s["b_down"] = (vec(f, 0.1), vec(f, 0.1), vec(o, 0.1)) if case["bias"] else (None,) * 3
        if case["train"]:
            s["dy"] = _rows(gen, m, o, t, 0.1)
        return s
    c = case["channels"]
    s["x"], s["f"] = _rows(gen, m, c, t), _rows(gen, m, c, t, 0.7)
    for side in ("pre", "post"):
        on = case["affine"] and case[side] != "none"
        s["w_" + side] = vec(c, 0.1, 1.0) if on else None
        s["b_" + side] = vec(c, 0.1) if on and case[side] == "layer" else None
    s["scale_v"] = vec(c, 0.02, 0.1) if case["scale"] else None
    s["gate_v"] = vec((case["gates"], c), 0.3, 1.0) if case["gates"] else None
    if case["train"]:
        s["dy"] = _rows(gen, m, c, t, 0.1)
        s["dh"] = _rows(gen, m, c, t, 0.1) if case["pre"] != "none" else None
    return s


# ---- the plain forms: 32 bits, rounded once at the end ----

def _act(kind, g):
    """act(g) and its derivative."""
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if kind == "sigmoid":
        s = torch.sigmoid(g)
        return s, s * (1 - s)
    if kind == "relu":
        return g * (g > 0), (g > 0).to(g.dtype)
    if kind == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    k = math.sqrt(2 / math.pi)
    th = torch.tanh(k * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + th), 0.5 * (1 + th) + 0.5 * g * (1 - th * th) * k * (1 + 3 * 0.044715 * g * g)


def _ffn_plain(s):
    t = _TYPES[s["dtype"]]
    x, wg, wu, wd = (s[k].float() for k in ("x", "w_gate", "w_up", "w_down"))
    g, u = x @ wg.t(), x @ wu.t()
    if s["bias"]:
        g, u = g + s["b_gate"].float(), u + s["b_up"].float()
    v, dv = _act(s["act"], g)
    a = v * u
    y = a @ wd.t()
    if s["bias"]:
        y = y + s["b_down"].float()
    if not s["train"]:
        return {"y": y.to(t)}
    dy = s["dy"].float()
    da = dy @ wd
    dg, du = da * u * dv, da * v
    r = {"y": y, "x": dg @ wg + du @ wu, "w_gate": dg.t() @ x, "w_up": du.t() @ x, "w_down": dy.t() @ a}
    if s["bias"]:
        r.update(b_gate=dg.sum(0), b_up=du.sum(0), b_down=dy.sum(0))
    return {k: z.to(t) for k, z in r.items()}


def _normed(kind, v):
    """The normalised rows and what they were multiplied by."""
    if kind == "none":
        return v, None
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    r = torch.rsqrt((v * v).mean(1, keepdim=True) + _EPS)
    return v * r, r


def _affine(n, w, b):
    n = n if w is None else n * w.float()
    return n if b is None else n + b.float()


def _normed_back(kind, n, r, dn):
    if kind == "none":
        return dn
    d = dn - n * (dn * n).mean(1, keepdim=True)
    if kind == "layer":
        d = d - dn.mean(1, keepdim=True)
    return d * r


def _norm_plain(s):
    t = _TYPES[s["dtype"]]
    m, c = s["x"].shape
    x, f = s["x"].float(), s["f"].float()
    nf, rf = _normed(s["post"], f)
    p = _affine(nf, s["w_post"], s["b_post"])
    gate = torch.ones(1, c, device=x.device) if s["gate_v"] is None else s["gate_v"].float()
    gate = gate.repeat_interleave(m // gate.shape[0], 0)
    scale = torch.ones(c, device=x.device) if s["scale_v"] is None else s["scale_v"].float()
    y = x + scale * gate * p
    r = {"y": y}
    ny, ry = _normed(s["pre"], y)
    if s["pre"] != "none":
        r["h"] = _affine(ny, s["w_pre"], s["b_pre"])
    if not s["train"]:
        return {k: z.to(t) for k, z in r.items()}
    d = s["dy"].float()
    if s["pre"] != "none":
        dh = s["dh"].float()
        d = d + _normed_back(s["pre"], ny, ry, dh if s["w_pre"] is None else dh * s["w_pre"].float())
        if s["w_pre"] is not None:
            r["w_pre"] = (dh * ny).sum(0)
        if s["b_pre"] is not None:
            r["b_pre"] = dh.sum(0)
    q = d * scale * gate
    r["x"] = d
    r["f"] = _normed_back(s["post"], nf, rf, q if s["w_post"] is None else q * s["w_post"].float())
    if s["w_post"] is not None:
        r["w_post"] = (q * nf).sum(0)
    if s["b_post"] is not None:
        r["b_post"] = q.sum(0)
    if s["scale_v"] is not None:
        r["scale"] = (d * gate * p).sum(0)
    if s["gate_v"] is not None:
        r["gate"] = (d * scale * p).reshape(s["gates"], -1, c).sum(1)
    return {k: z.to(t) for k, z in r.items()}


# ---- the package's kernels ----

def _ffn_own(s):
    if "layer" not in s:  # the layer object a program makes once for its weights
        from flyhigh_engine_b200.kernels import GatedFFN
        s["layer"] = GatedFFN(s["w_gate"], s["w_up"], s["w_down"], s["b_gate"], s["b_up"], s["b_down"], act=s["act"])
    if not s["train"]:
        return {"y": s["layer"](s["x"])}
    y, saved = s["layer"].forward(s["x"])
    return {"y": y, **s["layer"].backward(s["dy"], s["x"], saved)}


def _norm_own(s):
    if "layer" not in s:
        from flyhigh_engine_b200.kernels import ResidualNorm
        s["layer"] = ResidualNorm(s["channels"], s["x"].dtype, pre=s["pre"], post=s["post"], w_pre=s["w_pre"],
                                  b_pre=s["b_pre"], w_post=s["w_post"], b_post=s["b_post"], scale=s["scale_v"], eps=_EPS)
    y, h = s["layer"](s["x"], s["f"], s["gate_v"])
    r = {"y": y} if h is None else {"y": y, "h": h}
    if s["train"]:
        r.update(s["layer"].backward(s["dy"], s["dh"], y, s["f"], s["gate_v"]))
    return r


def run(state):
    if own:
        return _ffn_own(state) if state["op"] == "ffn" else _norm_own(state)
    return _ffn_plain(state) if state["op"] == "ffn" else _norm_plain(state)


# ---- the definitions in 64 bits ----

def _exact_act(kind, g):
    """act(g), and its derivative from 64-bit differentiation."""
    g = g.clone().requires_grad_(True)
    if kind == "relu":
        v = torch.clamp(g, min=0)
    elif kind in ("silu", "sigmoid"):
        v = 1 / (1 + torch.exp(-g))
        v = v * g if kind == "silu" else v
    elif kind == "gelu":
        v = g * torch.erfc(-g / math.sqrt(2)) / 2
    else:
        v = g / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))
    d, = torch.autograd.grad(v.sum(), g)
    return v.detach(), d


def exact(case, seed):
    s = prepare(case, seed)
    z = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if case["op"] == "ffn":
        wb = torch.cat([z["w_gate"], z["w_up"]])
        gu = z["x"] @ wb.t()
        if case["bias"]:
            gu += torch.cat([z["b_gate"], z["b_up"]])
        g, u = gu.chunk(2, 1)
        v, dv = _exact_act(case["act"], g)
        a = v * u
        r = {"y": a @ z["w_down"].t() + (z["b_down"] if case["bias"] else 0)}
        if case["train"]:
            da = z["dy"] @ z["w_down"]
            dgu = torch.cat([da * u * dv, da * v], 1)
            dwb = dgu.t() @ z["x"]
            r["x"] = dgu @ wb
            r["w_gate"], r["w_up"] = dwb.chunk(2)
            r["w_down"] = z["dy"].t() @ a
            if case["bias"]:
                r["b_gate"], r["b_up"] = dgu.sum(0).chunk(2)
                r["b_down"] = z["dy"].sum(0)
        return r
    c, groups = case["channels"], max(1, case["gates"])
    leaf = {k: v.requires_grad_(case["train"]) for k, v in z.items() if k not in ("dy", "dh")}

    def norm(kind, v, w, b):
        if kind == "layer":
            v = (v - v.mean(1, keepdim=True)) / torch.sqrt(v.var(1, unbiased=False, keepdim=True) + _EPS)
        elif kind == "rms":
            v = v / torch.sqrt(v.square().mean(1, keepdim=True) + _EPS)
        v = v * w if w is not None else v
        return v + b if b is not None else v

    with torch.enable_grad():
        p = norm(case["post"], leaf["f"], leaf.get("w_post"), leaf.get("b_post"))
        if case["scale"]:
            p = p * leaf["scale_v"]
        if case["gates"]:
            p = (p.reshape(groups, -1, c) * leaf["gate_v"][:, None]).reshape(-1, c)
        y = leaf["x"] + p
        h = norm(case["pre"], y, leaf.get("w_pre"), leaf.get("b_pre")) if case["pre"] != "none" else None
        r = {"y": y.detach()}
        if h is not None:
            r["h"] = h.detach()
        if case["train"]:
            total = (y * z["dy"]).sum() + ((h * z["dh"]).sum() if h is not None else 0)
            names = sorted(leaf)
            for k, gr in zip(names, torch.autograd.grad(total, [leaf[n] for n in names])):
                r[{"scale_v": "scale", "gate_v": "gate"}.get(k, k)] = gr
    return r
