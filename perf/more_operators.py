"""What a training step of a layer with a norm on both sides of its block does between the FP8 products, over the sizes it does it at.

Four operators, each one call of `Lib` (include/cf_fp8.h) where `own` is true and elementary torch operations where it is not:

  gated_norm           the norm of a block's output, its gate, the scaled residual stream, the next norm and its 8-bit activations, in one pass
  gated_norm_backward  its gradient: the stream's, the block output's, both norm weights' and the gate's, from bf16 rows or from 8-bit checkpoints
  swiglu               SiLU(gate) * up with the 8-bit operand of the product behind it, and gate and up kept in 8 bits for the backward pass
  swiglu_backward      its gradient from those bytes: bf16, or the E5M2 and E4M3 operands of the three products that follow, transposed ones too
"""
import ctypes
import importlib
import math

import torch

own = False
DEV = torch.device("cuda:0")

E4M3_MAX, E5M2_MAX = 448.0, 57344.0
EPS = 1e-6
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
FMAX = {"e4m3": E4M3_MAX, "e5m2": E5M2_MAX}
STREAM = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    # gate: the rows that share a row of gates; 0 = the block has none.
    norm = {"kind": "gated_norm", "fmt": "e4m3", "normed": False}
    back = {"kind": "gated_norm_backward"}
    glu = {"kind": "swiglu", "fmt": "e4m3"}
    glu_back = {"kind": "swiglu_backward"}
    return [
        # Decode: one token between two blocks; nothing but latency, nothing kept.
        {"name": "gated_norm_token", **norm, "rows": 1, "h": 4096, "stream": "bf16", "form": "rows", "gate": 0, "res": 1.0, "kept": False},
        # Three sequences with gates of their own, the last one cut short, into a block-scaled layer.
        {"name": "gated_norm_prompt_1000", **norm, "rows": 1000, "h": 7168, "stream": "bf16", "form": "block", "gate": 400, "res": 1.0, "kept": True},
        # A training batch under delayed scaling: the stream in fp32, one learned gate a channel, the backward pass's inputs kept in 8 bits.
        {"name": "gated_norm_train_8192", **norm, "rows": 8192, "h": 4096, "stream": "f32", "form": "record", "gate": 8192, "res": 1.25, "kept": True},
        # Backward of a short, odd batch from the bf16 rows ...
        {"name": "gated_norm_backward_333", **back, "rows": 333, "h": 2048, "stream": "bf16", "gate": 0, "res": 1.0, "kept": False, "out": "bf16"},
        # ... of a wide layer with gates for each of three sequences, from 8-bit checkpoints ...
        {"name": "gated_norm_backward_2000", **back, "rows": 2000, "h": 7168, "stream": "f32", "gate": 667, "res": 1.0, "kept": True, "out": "both"},
        # ... and of a training batch, with the bytes for the product before the norm.
        {"name": "gated_norm_backward_8192", **back, "rows": 8192, "h": 4096, "stream": "bf16", "gate": 8192, "res": 1.25, "kept": True, "out": "e5m2"},
        # Decode of one token: gate and up as the two halves of one product's row.
        {"name": "swiglu_token", **glu, "rows": 1, "i": 14336, "form": "rows", "fused": True},
        # A prompt through a width that is a multiple of nothing.
        {"name": "swiglu_prompt_1000", **glu, "rows": 1000, "i": 5461, "form": "block", "fused": False},
        # A training batch under delayed scaling.
        {"name": "swiglu_train_8192", **glu, "rows": 8192, "i": 14336, "form": "record", "fused": True},
        # Backward of a short, odd batch into bf16 products.
        {"name": "swiglu_backward_333", **glu_back, "rows": 333, "i": 1408, "form": "bf16"},
        # Backward of a prompt-sized batch into FP8 products ...
        {"name": "swiglu_backward_2000", **glu_back, "rows": 2000, "i": 8192, "form": "e5m2"},
        # ... and of a training batch.
        {"name": "swiglu_backward_8192", **glu_back, "rows": 8192, "i": 14336, "form": "e5m2"},
    ]


def _log_size(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["gated_norm", "gated_norm_backward", "swiglu", "swiglu_backward"])
    if kind in ("gated_norm", "gated_norm_backward"):
        # widths of the library's own configurations, some in between, and some that are a multiple of nothing
        h = rng.choice([512, 1024, 2048, 4096, 7168, 8192, 8 * rng.randint(16, 2048), rng.randint(100, 9000)])
        rows = min(_log_size(rng, 1, 32768), 8192 * 4096 // h)
        # none, one for all, one for each sequence, one for each token
        gate = rng.choice([0, rows, rng.randint(1, rows), _log_size(rng, 1, rows), 1])
        c = {"kind": kind, "rows": rows, "h": h, "stream": rng.choice(["bf16", "f32"]), "gate": gate, "res": rng.choice([1.0, 1.0, 0.875, 1.5]),
             "kept": rng.random() < 0.5}
        if kind == "gated_norm_backward":
            return {**c, "out": rng.choice(["bf16", "e5m2", "both"])}
        form = rng.choice(["rows", "block", "record"])
        return {**c, "form": form, "fmt": "e4m3" if form == "block" else rng.choice(["e4m3", "e4m3", "e5m2"]), "normed": rng.random() < 0.5}
    i = rng.choice([1024, 1408, 2048, 4096, 8192, 14336, 16 * rng.randint(8, 1500), rng.randint(100, 20000)])
    c = {"kind": kind, "rows": min(_log_size(rng, 1, 32768), 8192 * 8192 // i), "i": i}
    if kind == "swiglu_backward":
        return {**c, "form": rng.choice(["bf16", "e5m2", "e5m2"])}
    form = rng.choice(["rows", "block", "record"])
    return {**c, "form": form, "fmt": "e4m3" if form == "block" else rng.choice(["e4m3", "e4m3", "e5m2"]), "fused": rng.random() < 0.5}


class State:
    pass


def _normal(g, *shape, sigma=1.0, dtype=torch.bfloat16):
    return torch.randn(*shape, device=DEV, generator=g).mul_(sigma).to(dtype)


def _empty(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device=DEV)


def _bytes(*shape):
    return torch.empty(*shape, dtype=torch.uint8, device=DEV)


def _one(value=0.0):
    return torch.full((1,), float(value), device=DEV)


def _lib():
    return importlib.import_module("__graft_entry__").load_package().lib()


def _groups(t):
    """[rows, cols] -> [rows, ceil(cols / 128), 128], zeros behind the last column."""
    cols = t.shape[1]
    return torch.nn.functional.pad(t, (0, -cols % 128)).unflatten(1, (-1, 128))


def _to8(v, fmt):
    return v.clamp(-FMAX[fmt], FMAX[fmt]).to(F8[fmt])


def _exact8(v, fmt):
    """What the bytes round, clipped to the format's range.  E5M2 steps are so wide that its distance from them says nothing."""
    return v.clamp(-FMAX[fmt], FMAX[fmt]) if fmt == "e4m3" else None


def _quantized(v, form, fmt, scale):
    """{"q", "scale", "descale"} or {"q", "amax"} of fp32 rows, as the library's quantizers give them."""
    if form == "record":
        return {"q": _to8(v * scale, fmt), "amax": v.abs().amax().reshape(1)}
    g = _groups(v) if form == "block" else v[:, None, :]
    a = g.abs().amax(2).clamp_min(1e-12)
    s, d = FMAX[fmt] / a, a / FMAX[fmt]
    q = _to8(g * s[:, :, None], fmt).flatten(1)[:, :v.shape[1]]
    return {"q": q, "scale": s if form == "block" else s[:, 0], "descale": d if form == "block" else d[:, 0]}


def _exact_quantized(y, form, fmt, scale):
    if form == "record":
        return {"q": _exact8(y * scale.double(), fmt), "amax": y.abs().max().view(1)}
    width = 128 if form == "block" else y.shape[1]
    a = torch.stack([part.abs().max(1).values for part in y.split(width, 1)], 1).clamp(min=1e-12)
    q = _exact8(y * (FMAX[fmt] / a).repeat_interleave(width, 1)[:, :y.shape[1]], fmt)
    a = a if form == "block" else a[:, 0]
    return {"q": q, "scale": FMAX[fmt] / a, "descale": a / FMAX[fmt]}


def prepare(case, seed):
    s = State()
    s.case = c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    {"gated_norm": _prepare_norm, "gated_norm_backward": _prepare_norm_backward, "swiglu": _prepare_swiglu,
     "swiglu_backward": _prepare_swiglu_backward}[c["kind"]](s, c, g)
    if own:
        s.cf = _lib()
        if c["kind"] == "gated_norm_backward":
            n = ctypes.c_size_t(0)
            s.cf.cf_gated_add_rmsnorm_backward_workspace_bytes(c["rows"], c["h"], c["gate"], ctypes.byref(n))
            s.ws, s.ws_bytes = _bytes(max(n.value, 1)), n.value
    return s


def run(state):
    s, c = state, state.case
    if own:
        return {"gated_norm": _own_norm, "gated_norm_backward": _own_norm_backward, "swiglu": _own_swiglu, "swiglu_backward": _own_swiglu_backward}[
            c["kind"]](s, c, s.cf, torch.cuda.current_stream().cuda_stream)
    return {"gated_norm": _plain_norm, "gated_norm_backward": _plain_norm_backward, "swiglu": _plain_swiglu,
            "swiglu_backward": _plain_swiglu_backward}[c["kind"]](s, c)


def exact(case, seed):
    s = prepare(case, seed)
    return {"gated_norm": _exact_norm, "gated_norm_backward": _exact_norm_backward, "swiglu": _exact_swiglu,
            "swiglu_backward": _exact_swiglu_backward}[s.case["kind"]](s, s.case)


# ---- norm, gate, residual, norm, 8 bits ---------------------------------------------------------------------------------

def _loud_rows(g, rows, h, dtype, sigma=1.0):
    """Rows of different loudness, with a few channels far above the others."""
    loud = torch.exp(0.3 * torch.randn(rows, 1, device=DEV, generator=g))
    channel = torch.where(torch.rand(h, device=DEV, generator=g) < 0.004, 20.0, 1.0)
    return (torch.randn(rows, h, device=DEV, generator=g) * loud * channel * sigma).to(dtype)


def _gamma(g, h):
    return (1.0 + 0.1 * torch.randn(h, device=DEV, generator=g)).to(torch.bfloat16)


def _gate(g, c):
    """Gates of the groups of rows that share them, the last group cut short where the rows end inside it."""
    return (0.5 + 0.2 * torch.randn(-(-c["rows"] // c["gate"]), c["h"], device=DEV, generator=g)).to(torch.bfloat16) if c["gate"] else None


def _gate_rows(gate, c):
    """The gate of each row, in fp32; 1 where there is none."""
    return gate.float().repeat_interleave(c["gate"], 0)[:c["rows"]] if c["gate"] else 1.0


def _kept_scale(h):
    """A normalised row has no element above sqrt(h), so one power of two serves all checkpoints of its width."""
    return 2.0 ** math.floor(math.log2(E4M3_MAX / math.sqrt(h)))


def _prepare_norm(s, c, g):
    R, H = c["rows"], c["h"]
    s.residual, s.x = _loud_rows(g, R, H, STREAM[c["stream"]]), _loud_rows(g, R, H, torch.bfloat16, 0.5)
    s.post_gamma, s.gamma, s.gate = _gamma(g, H), _gamma(g, H), _gate(g, c)
    s.sum, s.post_rms, s.rms, s.q = torch.empty_like(s.residual), _empty(R), _empty(R), _bytes(R, H)
    s.normed = _empty(R, H, dtype=torch.bfloat16) if c["normed"] else None
    s.x8, s.sum8 = (_bytes(R, H), _bytes(R, H)) if c["kept"] else (None, None)
    s.scale, s.descale, s.amax = None, None, None
    if c["form"] == "record":        # the scale that earlier batches left
        s.scale, s.amax = _one(FMAX[c["fmt"]] / 30.0), _one()
    else:
        groups = (R, (H + 127) // 128) if c["form"] == "block" else (R,)
        s.scale, s.descale = _empty(*groups), _empty(*groups)


def _own_norm(s, c, cf, st):
    R, H, e5m2 = c["rows"], c["h"], int(c["fmt"] == "e5m2")
    inputs = (s.residual, s.x, int(c["stream"] == "f32"), c["res"], s.gate, c["gate"], s.post_gamma, s.gamma, R, H, EPS)
    kept = (s.sum, s.normed, s.post_rms, s.rms, s.x8, s.sum8, s.q)
    f8 = lambda b, t: None if b is None else b.view(t)  # noqa: E731
    out = {"sum": s.sum, "normed": s.normed, "post_rms": s.post_rms, "rms": s.rms, "x8": f8(s.x8, F8["e4m3"]), "sum8": f8(s.sum8, F8["e4m3"]),
           "q": s.q.view(F8[c["fmt"]])}
    if c["form"] == "record":
        s.amax.zero_()
        cf.cf_gated_add_rmsnorm_quantize_record(*inputs, e5m2, *kept, s.scale, s.amax, st)
        return {**out, "amax": s.amax}
    if c["form"] == "block":
        cf.cf_gated_add_rmsnorm_quantize_block_1x128(*inputs, *kept, s.scale, s.descale, st)
    else:
        cf.cf_gated_add_rmsnorm_quantize_rows(*inputs, e5m2, *kept, s.scale, s.descale, st)
    return {**out, "scale": s.scale, "descale": s.descale}


def _plain_norm(s, c):
    x = s.x.float()
    post_rms = torch.sqrt((x * x).mean(1) + EPS)
    xhat = x / post_rms[:, None]
    total = (c["res"] * s.residual.float() + _gate_rows(s.gate, c) * (xhat * s.post_gamma.float())).to(s.residual.dtype)
    h = total.float()               # the second norm is of the stream as it is kept, which is what the backward pass has
    rms = torch.sqrt((h * h).mean(1) + EPS)
    hhat = h / rms[:, None]
    y = hhat * s.gamma.float()
    S = _kept_scale(c["h"])
    return {"sum": total, "normed": y.to(torch.bfloat16) if c["normed"] else None, "post_rms": post_rms, "rms": rms,
            "x8": _to8(xhat * S, "e4m3") if c["kept"] else None, "sum8": _to8(hhat * S, "e4m3") if c["kept"] else None,
            **_quantized(y, c["form"], c["fmt"], s.scale)}


def _exact_norm(s, c):
    H, S = c["h"], 2.0 ** int(math.log2(E4M3_MAX / c["h"] ** 0.5))
    x = s.x.double()
    post_rms = x.square().sum(1).div(H).add(EPS).sqrt()
    x = x / post_rms.unsqueeze(1)
    z = x * s.post_gamma.double()
    if c["gate"]:
        z = z * s.gate.double()[torch.div(torch.arange(c["rows"], device=DEV), c["gate"], rounding_mode="floor")]
    total = s.residual.double().mul(c["res"]).add(z)
    # the sum in fp32 or better, then rounded to the stream's type: a sum next to the border of two bf16 values may go to either
    h = total.to(s.residual.dtype).double()
    rms = h.square().sum(1).div(H).add(EPS).sqrt()
    hh = h / rms.unsqueeze(1)
    y = s.gamma.double() * hh
    kept = {"x8": x * S, "sum8": hh * S} if c["kept"] else {"x8": None, "sum8": None}
    return {"sum": total, "normed": y if c["normed"] else None, "post_rms": post_rms, "rms": rms, **kept,
            **_exact_quantized(y, c["form"], c["fmt"], s.scale)}


# ---- its gradient -----------------------------------------------------------------------------------------------------

def _prepare_norm_backward(s, c, g):
    R, H, T = c["rows"], c["h"], STREAM[c["stream"]]
    s.sum, s.x = _loud_rows(g, R, H, T), _loud_rows(g, R, H, torch.bfloat16, 0.5)
    s.post_gamma, s.gamma, s.gate = _gamma(g, H), _gamma(g, H), _gate(g, c)
    s.rms, s.post_rms = (torch.sqrt(t.float().square().mean(1) + EPS) for t in (s.sum, s.x))       # kept by the forward pass
    if c["kept"]:                    # and so are these, in place of the rows
        s.sum, s.x = (_to8(t.float() / r[:, None] * _kept_scale(H), "e4m3") for t, r in ((s.sum, s.rms), (s.x, s.post_rms)))
    s.grad_normed, s.grad_sum = _normal(g, R, H, sigma=1e-3), _normal(g, R, H, sigma=1e-3, dtype=T)
    s.grad_residual = _empty(R, H, dtype=T)
    s.grad_x = None if c["out"] == "e5m2" else _empty(R, H, dtype=torch.bfloat16)
    s.grad8, s.scale, s.amax = (None, None, None) if c["out"] == "bf16" else (_bytes(R, H), _one(E5M2_MAX / 0.1), _one())
    s.grad_gamma, s.grad_post_gamma = _empty(H), _empty(H)
    s.grad_gate = _empty(*s.gate.shape) if c["gate"] else None


def _own_norm_backward(s, c, cf, st):
    call = cf.cf_gated_add_rmsnorm_backward_ckpt8 if c["kept"] else cf.cf_gated_add_rmsnorm_backward
    if s.amax is not None:
        s.amax.zero_()
    call(s.grad_normed, s.sum, s.x, int(c["stream"] == "f32"), c["res"], s.gate, c["gate"], s.post_gamma, s.gamma, s.post_rms, s.rms, s.grad_sum,
         c["rows"], c["h"], s.grad_residual, s.grad_x, s.grad8, s.scale, s.amax, s.grad_post_gamma, s.grad_gamma, s.grad_gate, 0,
         s.ws, s.ws_bytes, st)
    return {"grad_residual": s.grad_residual, "grad_x": s.grad_x, "grad8": None if s.grad8 is None else s.grad8.view(F8["e5m2"]), "amax": s.amax,
            "grad_post_gamma": s.grad_post_gamma, "grad_gamma": s.grad_gamma, "grad_gate": s.grad_gate}


def _plain_norm_backward(s, c):
    R, H, gate = c["rows"], c["h"], c["gate"]
    inv, post_inv = 1.0 / s.rms[:, None], 1.0 / s.post_rms[:, None]
    if c["kept"]:
        hhat, xhat = s.sum.float() / _kept_scale(H), s.x.float() / _kept_scale(H)
    else:
        hhat, xhat = s.sum.float() * inv, s.x.float() * post_inv
    dy = s.grad_normed.float()
    g = dy * s.gamma.float()
    d = s.grad_sum.float() + (g - hhat * (g * hhat).mean(1, keepdim=True)) * inv
    e = d * _gate_rows(s.gate, c) * s.post_gamma.float()
    dx = (e - xhat * (e * xhat).mean(1, keepdim=True)) * post_inv
    per_gate = torch.nn.functional.pad(d * xhat, (0, 0, 0, -R % gate if gate else 0)).unflatten(0, (-1, gate or R)).sum(1, dtype=torch.float64)
    weighted = per_gate * s.gate.double() if gate else per_gate
    return {"grad_residual": (c["res"] * d).to(s.grad_sum.dtype), "grad_x": None if c["out"] == "e5m2" else dx.to(torch.bfloat16),
            "grad8": None if c["out"] == "bf16" else _to8(dx * s.scale, "e5m2"), "amax": None if c["out"] == "bf16" else dx.abs().amax().reshape(1),
            "grad_post_gamma": weighted.sum(0).float(), "grad_gamma": (dy * hhat).sum(0, dtype=torch.float64).float(),
            "grad_gate": (per_gate * s.post_gamma.double()).float() if gate else None}


def _exact_norm_backward(s, c):
    R, H = c["rows"], c["h"]
    r, pr = s.rms.double().unsqueeze(1), s.post_rms.double().unsqueeze(1)
    if c["kept"]:
        S = 2.0 ** int(math.log2(E4M3_MAX / H ** 0.5))
        hh, xh = s.sum.double() / S, s.x.double() / S
    else:
        hh, xh = s.sum.double() / r, s.x.double() / pr
    dy, w, pw = s.grad_normed.double(), s.gamma.double(), s.post_gamma.double()
    d = s.grad_sum.double() + dy * w / r - hh * (dy * w).mul(hh).sum(1, keepdim=True) / (H * r)
    e, grad_gate = d * pw, None
    grad_post = d * xh
    if c["gate"]:
        which = torch.div(torch.arange(R, device=DEV), c["gate"], rounding_mode="floor")
        gates = s.gate.double()[which]
        grad_gate = torch.zeros(s.gate.shape, dtype=torch.float64, device=DEV).index_add_(0, which, grad_post * pw)
        e, grad_post = e * gates, grad_post * gates
    dx = e / pr - xh * e.mul(xh).sum(1, keepdim=True) / (H * pr)
    return {"grad_residual": d * c["res"], "grad_x": None if c["out"] == "e5m2" else dx, "grad8": None,
            "amax": None if c["out"] == "bf16" else dx.abs().max().view(1), "grad_post_gamma": grad_post.sum(0),
            "grad_gamma": (dy * hh).sum(0), "grad_gate": grad_gate}


# ---- the gated activation, kept in 8 bits -------------------------------------------------------------------------------

def _prepare_swiglu(s, c, g):
    R, I = c["rows"], c["i"]
    if c["fused"]:                   # the two halves of a row of one product
        both = torch.cat([_loud_rows(g, R, I, torch.bfloat16), _loud_rows(g, R, I, torch.bfloat16)], 1)
        s.gate, s.up = both[:, :I], both[:, I:]
    else:
        s.gate, s.up = _loud_rows(g, R, I, torch.bfloat16), _loud_rows(g, R, I, torch.bfloat16)
    s.ld = s.gate.stride(0)
    groups = (R, (I + 127) // 128)
    s.gate8, s.up8, s.gate8_descale, s.up8_descale = _bytes(R, I), _bytes(R, I), _empty(*groups), _empty(*groups)
    s.q = _bytes(R, I)
    s.scale, s.descale, s.amax = None, None, None
    if c["form"] == "record":
        s.scale, s.amax = _one(FMAX[c["fmt"]] / 60.0), _one()
    else:
        shape = groups if c["form"] == "block" else (R,)
        s.scale, s.descale = _empty(*shape), _empty(*shape)


def _own_swiglu(s, c, cf, st):
    e5m2 = int(c["fmt"] == "e5m2")
    inputs = (s.gate, s.up, s.ld, c["rows"], c["i"])
    kept = (s.gate8, s.gate8_descale, s.up8, s.up8_descale, s.q)
    out = {"gate8": s.gate8.view(F8["e4m3"]), "gate8_descale": s.gate8_descale, "up8": s.up8.view(F8["e4m3"]), "up8_descale": s.up8_descale,
           "q": s.q.view(F8[c["fmt"]])}
    if c["form"] == "record":
        s.amax.zero_()
        cf.cf_swiglu_ckpt8_quantize_record(*inputs, e5m2, *kept, s.scale, s.amax, st)
        return {**out, "amax": s.amax}
    if c["form"] == "block":
        cf.cf_swiglu_ckpt8_quantize_block_1x128(*inputs, *kept, s.scale, s.descale, st)
    else:
        cf.cf_swiglu_ckpt8_quantize_rows(*inputs, e5m2, *kept, s.scale, s.descale, st)
    return {**out, "scale": s.scale, "descale": s.descale}


def _plain_swiglu(s, c):
    g, u = s.gate.float(), s.up.float()
    a = g / (1.0 + torch.exp(-g)) * u
    kg, ku = _quantized(g, "block", "e4m3", None), _quantized(u, "block", "e4m3", None)
    return {"gate8": kg["q"], "gate8_descale": kg["descale"], "up8": ku["q"], "up8_descale": ku["descale"], **_quantized(a, c["form"], c["fmt"], s.scale)}


def _exact_swiglu(s, c):
    g, u = s.gate.double(), s.up.double()
    kg, ku = _exact_quantized(g, "block", "e4m3", None), _exact_quantized(u, "block", "e4m3", None)
    a = torch.sigmoid(g) * g * u
    return {"gate8": kg["q"], "gate8_descale": kg["descale"], "up8": ku["q"], "up8_descale": ku["descale"],
            **_exact_quantized(a, c["form"], c["fmt"], s.scale)}


# ---- its gradient -----------------------------------------------------------------------------------------------------

def _prepare_swiglu_backward(s, c, g):
    R, I = c["rows"], c["i"]
    kg, ku = (_quantized(_loud_rows(g, R, I, torch.bfloat16).float(), "block", "e4m3", None) for _ in range(2))      # kept by the forward pass
    s.gate8, s.gate8_descale, s.up8, s.up8_descale = kg["q"].contiguous(), kg["descale"], ku["q"].contiguous(), ku["descale"]
    s.grad_out = _normal(g, R, I, sigma=1e-3)
    if c["form"] == "bf16":          # into the two halves of the fused product's gradient, and the activation for the weight gradient
        s.grad, s.act = _empty(R, 2 * I, dtype=torch.bfloat16), _empty(R, I, dtype=torch.bfloat16)
    else:
        s.grad8, s.grad8_t, s.act8_t = _bytes(R, 2 * I), _bytes(2 * I, R), _bytes(I, R)
        s.scale, s.amax, s.act_scale = _one(E5M2_MAX / 0.5), _one(), _one(E4M3_MAX / 60.0)


def _own_swiglu_backward(s, c, cf, st):
    R, I = c["rows"], c["i"]
    kept = (s.grad_out, s.gate8, s.gate8_descale, s.up8, s.up8_descale, R, I)
    if c["form"] == "bf16":
        cf.cf_swiglu_ckpt8_backward(*kept, s.grad, s.grad[:, I:], 2 * I, s.act, st)
        return {"grad": s.grad, "act": s.act}
    s.amax.zero_()
    cf.cf_swiglu_ckpt8_backward_quant_e5m2(*kept, s.grad8, s.grad8_t, s.scale, s.amax, s.act8_t, s.act_scale, st)
    return {"grad8": s.grad8.view(F8["e5m2"]), "grad8_t": s.grad8_t.view(F8["e5m2"]), "amax": s.amax, "act8_t": s.act8_t.view(F8["e4m3"])}


def _plain_swiglu_backward(s, c):
    I = c["i"]
    g, u = ((_groups(q.float()) * d[:, :, None]).flatten(1)[:, :I] for q, d in ((s.gate8, s.gate8_descale), (s.up8, s.up8_descale)))
    d, sig = s.grad_out.float(), 1.0 / (1.0 + torch.exp(-g))
    grad = torch.cat([d * u * (sig * (1.0 + g * (1.0 - sig))), d * (g * sig)], 1)
    act = g * sig * u
    if c["form"] == "bf16":
        return {"grad": grad.to(torch.bfloat16), "act": act.to(torch.bfloat16)}
    turn = lambda q: q.view(torch.uint8).t().contiguous().view(q.dtype)  # noqa: E731
    grad8 = _to8(grad * s.scale, "e5m2")
    return {"grad8": grad8, "grad8_t": turn(grad8), "amax": grad.abs().amax().reshape(1), "act8_t": turn(_to8(act * s.act_scale, "e4m3"))}


def _exact_swiglu_backward(s, c):
    I = c["i"]
    g, u = (q.double() * d.double().repeat_interleave(128, 1)[:, :I] for q, d in ((s.gate8, s.gate8_descale), (s.up8, s.up8_descale)))
    d = s.grad_out.double()
    silu, sig = torch.sigmoid(g) * g, torch.sigmoid(g)
    grad = torch.cat([d * u * (sig + silu - silu * sig), d * silu], 1)
    if c["form"] == "bf16":
        return {"grad": grad, "act": silu * u}
    return {"grad8": None, "grad8_t": None, "amax": grad.abs().max().view(1), "act8_t": _exact8((silu * u * s.act_scale.double()).t().contiguous(), "e4m3")}


# ---- what a pass cannot do without --------------------------------------------------------------------------------------

def work(case):
    c, kind, rows = case, case["kind"], case["rows"]
    if kind in ("gated_norm", "gated_norm_backward"):
        n, stream = rows * c["h"], 4 if c["stream"] == "f32" else 2
        gates = -(-rows // c["gate"]) * c["h"] if c["gate"] else 0
        if kind == "gated_norm":     # the stream and the block's output read, the new stream, the bytes and the checkpoints written
            per = 2 * stream + 2 + 1 + (2 if c["normed"] else 0) + (2 if c["kept"] else 0)
            scales = 8 * rows * {"rows": 1, "block": (c["h"] + 127) // 128, "record": 0}[c["form"]]
            return {"bytes": n * per + 4 * c["h"] + 8 * rows + scales + 2 * gates, "flops": 14 * n}
        # dy, the two saved tensors, the stream's gradient in and out, the block output's gradient
        per = 2 + (2 if c["kept"] else stream + 2) + 2 * stream + {"bf16": 2, "e5m2": 1, "both": 3}[c["out"]]
        return {"bytes": n * per + 12 * c["h"] + 8 * rows + 6 * gates, "flops": 26 * n}
    n, groups = rows * c["i"], rows * ((c["i"] + 127) // 128)
    if kind == "swiglu":             # gate and up read, their bytes and the product's operand written
        scales = {"rows": 8 * rows, "block": 8 * groups, "record": 0}[c["form"]]
        return {"bytes": 7 * n + 8 * groups + scales, "flops": 14 * n}
    # the output's gradient and the bytes read; bf16: two gradients and the activation; 8 bits: the gradients twice and the activation
    return {"bytes": n * (4 + (6 if c["form"] == "bf16" else 5)) + 8 * groups, "flops": 18 * n}
