"""What a training step of a pre-norm residual layer does around its FP8 products, over the sizes it does it at.

Four operators, each one call of `Lib` (include/cf_fp8.h) where `own` is true and elementary torch operations where it is not:

  norm           the residual addition, the RMS norm and the 8-bit activations with their scales, in one pass
  norm_backward  its gradient: the residual stream's, the norm weight's, and the E5M2 bytes for the product before it
  experts        the experts' product over rows gathered by routing, 1x128 activation scales and 128x128 weight scales
  grads          the global norm of a list of gradients, and the gradients clipped by it
"""
import ctypes
import importlib

import torch

own = False
DEV = torch.device("cuda:0")

E4M3_MAX, E5M2_MAX = 448.0, 57344.0
EPS = 1e-6
BLOCK_128, EPI_NONE = 2, 0
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
FMAX = {"e4m3": E4M3_MAX, "e5m2": E5M2_MAX}
STREAM = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # Decode: one token enters a layer; nothing but latency.
        {"name": "norm_token", "kind": "norm", "rows": 1, "h": 4096, "stream": "bf16", "form": "rows", "fmt": "e4m3", "normed": False},
        # A prompt whose length is a multiple of nothing, into a block-scaled layer.
        {"name": "norm_prompt_1000", "kind": "norm", "rows": 1000, "h": 7168, "stream": "bf16", "form": "block", "fmt": "e4m3", "normed": False},
        # A training batch under delayed scaling, the residual stream kept in fp32, the bf16 rows kept for the weight gradient.
        {"name": "norm_train_8192", "kind": "norm", "rows": 8192, "h": 4096, "stream": "f32", "form": "record", "fmt": "e4m3", "normed": True},
        # Backward of a short, odd batch at the first norm of the stack's top layer ...
        {"name": "norm_backward_333", "kind": "norm_backward", "rows": 333, "h": 2048, "stream": "bf16", "quant": False},
        # ... of a wide layer ...
        {"name": "norm_backward_2000", "kind": "norm_backward", "rows": 2000, "h": 7168, "stream": "f32", "quant": True},
        # ... and of a training batch, with the bytes for the projection before the norm.
        {"name": "norm_backward_8192", "kind": "norm_backward", "rows": 8192, "h": 4096, "stream": "bf16", "quant": True},
        # Decode of 16 sequences: a row or two for each expert, every selected expert's weights read.
        {"name": "experts_decode_16", "kind": "experts", "tokens": 16, "k": 2048, "n": 1408, "experts": 64, "top_k": 6, "gather": True, "even": True},
        # A prompt through few, larger experts whose popularity is uneven: the projection back, over rows already in expert order.
        {"name": "experts_prompt_1000", "kind": "experts", "tokens": 1000, "k": 2048, "n": 1024, "experts": 8, "top_k": 2, "gather": False, "even": False},
        # A training batch.
        {"name": "experts_train_16384", "kind": "experts", "tokens": 16384, "k": 2048, "n": 1408, "experts": 64, "top_k": 6, "gather": True, "even": True},
        # The gradients of a small network: some thirty tensors, half of them tiny, none but the first on a boundary.
        {"name": "grads_small", "kind": "grads", "layers": 4, "h": 256, "i": 683, "dtype": "f32", "max_norm": 0.1},
        # One layer's, in bf16, with norm weights and biases in fp32.
        {"name": "grads_layer", "kind": "grads", "layers": 1, "h": 4096, "i": 14336, "dtype": "mixed", "max_norm": 1.0},
        # A stack's, accumulated in fp32.
        {"name": "grads_stack", "kind": "grads", "layers": 4, "h": 4096, "i": 14336, "dtype": "f32", "max_norm": 1.0},
    ]


def _log_size(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm_backward", "norm_backward", "experts", "experts", "grads"])
    if kind in ("norm", "norm_backward"):
        # widths of the library's own configurations, some in between, and some that are a multiple of nothing
        h = rng.choice([512, 1024, 2048, 4096, 7168, 8192, 8 * rng.randint(16, 2048), rng.randint(100, 9000)])
        c = {"kind": kind, "rows": min(_log_size(rng, 1, 32768), 8192 * 4096 // h), "h": h, "stream": rng.choice(["bf16", "f32"])}
        if kind == "norm_backward":
            return {**c, "quant": rng.random() < 0.5}
        form = rng.choice(["rows", "block", "record"])
        return {**c, "form": form, "fmt": "e4m3" if form == "block" else rng.choice(["e4m3", "e4m3", "e5m2"]), "normed": rng.random() < 0.5}
    if kind == "experts":
        k, n, e, top = rng.choice([(2048, 1408, 64, 6), (1408, 2048, 64, 6), (2048, 1024, 8, 2), (1024, 2048, 8, 2), (4096, 1536, 16, 4),
                                   (7168, 2048, 16, 2), (512, 128 * rng.randint(1, 16), 32, 4), (1024, 8 * rng.randint(16, 200), 24, 3)])
        return {"kind": kind, "tokens": min(_log_size(rng, 1, 16384), int(2.5e11 / (k * n * top))), "k": k, "n": n, "experts": e, "top_k": top,
                "gather": rng.random() < 0.5, "even": rng.random() < 0.5}
    h = rng.choice([64, 256, 512, 1024, 2048, 4096])
    return {"kind": kind, "layers": _log_size(rng, 1, 48 if h < 1024 else 16 if h < 4096 else 4), "h": h, "i": rng.randint(2 * h, 7 * h // 2),
            "dtype": rng.choice(["bf16", "f32", "mixed"]), "max_norm": rng.choice([0.05, 1.0, 1.0, 1e4])}


class State:
    pass


def _normal(g, *shape, sigma=1.0, dtype=torch.bfloat16):
    return torch.randn(*shape, device=DEV, generator=g).mul_(sigma).to(dtype)


def _empty(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device=DEV)


def _one(value=0.0):
    return torch.full((1,), float(value), device=DEV)


def _lib():
    return importlib.import_module("__graft_entry__").load_package().lib()


def _workspace(size_fn, *args):
    n = ctypes.c_size_t(0)
    size_fn(*args, ctypes.byref(n))
    return _empty(max(n.value, 1), dtype=torch.uint8), n.value


def _groups(t):
    """[rows, cols] -> [rows, ceil(cols / 128), 128], zeros behind the last column."""
    cols = t.shape[1]
    return torch.nn.functional.pad(t, (0, -cols % 128)).unflatten(1, (-1, 128))


def _exact8(v, fmt):
    """What the bytes round, clipped to the format's range.  E5M2 steps are so wide that its distance from them says nothing."""
    return v.clamp(-FMAX[fmt], FMAX[fmt]) if fmt == "e4m3" else None


def _to8(v, fmt):
    return v.clamp(-FMAX[fmt], FMAX[fmt]).to(F8[fmt])


def prepare(case, seed):
    s = State()
    s.case = c = dict(case)
    s.g = torch.Generator(device=DEV).manual_seed(int(seed))
    {"norm": _prepare_norm, "norm_backward": _prepare_norm_backward, "experts": _prepare_experts, "grads": _prepare_grads}[c["kind"]](s, c, s.g)
    if own:
        s.cf = _lib()
        if c["kind"] == "norm_backward":
            s.ws, s.ws_bytes = _workspace(s.cf.cf_add_rmsnorm_backward_workspace_bytes, c["rows"], c["h"])
        elif c["kind"] == "experts":
            s.ws, s.ws_bytes = _workspace(s.cf.cf_fp8_grouped_gemm_workspace_bytes, s.total, c["experts"])
        elif c["kind"] == "grads":
            s.ws, s.ws_bytes = _workspace(s.cf.cf_grad_norm_workspace_bytes)
            s.list, s.list_bytes = _grad_list(s.cf, s.grads, s.clipped)
    return s


def run(state):
    s, c = state, state.case
    if own:
        return {"norm": _own_norm, "norm_backward": _own_norm_backward, "experts": _own_experts, "grads": _own_grads}[c["kind"]](
            s, c, s.cf, torch.cuda.current_stream().cuda_stream)
    return {"norm": _plain_norm, "norm_backward": _plain_norm_backward, "experts": _plain_experts, "grads": _plain_grads}[c["kind"]](s, c)


def exact(case, seed):
    s = prepare(case, seed)
    c = s.case
    return {"norm": _exact_norm, "norm_backward": _exact_norm_backward, "experts": _exact_experts, "grads": _exact_grads}[c["kind"]](s, c)


# ---- residual addition, RMS norm, 8-bit output ------------------------------------------------------------------------

def _stream_rows(g, rows, h, dtype, sigma=1.0):
    """A residual stream: rows of different loudness, with a few channels far above the others."""
    loud = torch.exp(0.3 * torch.randn(rows, 1, device=DEV, generator=g))
    channel = torch.where(torch.rand(h, device=DEV, generator=g) < 0.004, 20.0, 1.0)
    return (torch.randn(rows, h, device=DEV, generator=g) * loud * channel * sigma).to(dtype)


def _gamma(g, h):
    return (1.0 + 0.1 * torch.randn(h, device=DEV, generator=g)).to(torch.bfloat16)


def _prepare_norm(s, c, g):
    R, H = c["rows"], c["h"]
    s.residual, s.x = _stream_rows(g, R, H, STREAM[c["stream"]]), _normal(g, R, H, sigma=0.5)
    s.gamma = _gamma(g, H)
    s.sum, s.rms, s.q = torch.empty_like(s.residual), _empty(R), _empty(R, H, dtype=torch.uint8)
    s.normed = _empty(R, H, dtype=torch.bfloat16) if c["normed"] else None
    if c["form"] == "record":        # the scale that earlier batches left
        s.scale, s.amax = _one(FMAX[c["fmt"]] / 30.0), _one()
    else:
        groups = (R, (H + 127) // 128) if c["form"] == "block" else (R,)
        s.scale, s.descale = _empty(*groups), _empty(*groups)


def _own_norm(s, c, cf, st):
    R, H, f32, e5m2 = c["rows"], c["h"], int(c["stream"] == "f32"), int(c["fmt"] == "e5m2")
    out = {"sum": s.sum, "rms": s.rms, "q": s.q.view(F8[c["fmt"]]), "normed": s.normed}
    if c["form"] == "record":
        s.amax.zero_()
        cf.cf_add_rmsnorm_quantize_record(s.residual, s.x, f32, s.gamma, R, H, EPS, e5m2, s.sum, s.normed, s.rms, s.q, s.scale, s.amax, st)
        return {**out, "amax": s.amax}
    if c["form"] == "block":
        cf.cf_add_rmsnorm_quantize_block_1x128(s.residual, s.x, f32, s.gamma, R, H, EPS, s.sum, s.normed, s.rms, s.q, s.scale, s.descale, st)
    else:
        cf.cf_add_rmsnorm_quantize_rows(s.residual, s.x, f32, s.gamma, R, H, EPS, e5m2, s.sum, s.normed, s.rms, s.q, s.scale, s.descale, st)
    return {**out, "scale": s.scale, "descale": s.descale}


def _plain_norm(s, c):
    H, fmt = c["h"], c["fmt"]
    total = (s.residual.float() + s.x.float()).to(s.residual.dtype)
    h = total.float()               # the norm is of the stream as it is kept, which is what the backward pass has
    rms = torch.sqrt((h * h).mean(1) + EPS)
    y = h / rms[:, None] * s.gamma.float()
    out = {"sum": total, "rms": rms, "normed": y.to(torch.bfloat16) if c["normed"] else None}
    if c["form"] == "record":
        return {**out, "q": _to8(y * s.scale, fmt), "amax": y.abs().amax().reshape(1)}
    g = _groups(y) if c["form"] == "block" else y[:, None, :]
    a = g.abs().amax(2).clamp_min(1e-12)
    scale, descale = FMAX[fmt] / a, a / FMAX[fmt]
    q = _to8(g * scale[:, :, None], fmt).flatten(1)[:, :H]
    groups = scale.shape if c["form"] == "block" else (c["rows"],)
    return {**out, "q": q, "scale": scale.reshape(groups), "descale": descale.reshape(groups)}


def _exact_norm(s, c):
    H, F, fmt = c["h"], FMAX[c["fmt"]], c["fmt"]
    total = s.residual.double().add(s.x.double())
    h = total.to(s.residual.dtype).double()
    rms = h.square().sum(1).div(H).add(EPS).sqrt()
    y = s.gamma.double() * (h / rms.unsqueeze(1))
    out = {"sum": total, "rms": rms, "normed": y if c["normed"] else None}
    if c["form"] == "record":
        return {**out, "q": _exact8(y * s.scale.double(), fmt), "amax": y.abs().max().view(1)}
    width = 128 if c["form"] == "block" else H
    a = torch.stack([part.abs().max(1).values for part in y.split(width, 1)], 1).clamp(min=1e-12)
    q = y * (F / a).repeat_interleave(width, 1)[:, :H]
    a = a if c["form"] == "block" else a[:, 0]
    return {**out, "q": _exact8(q, fmt), "scale": F / a, "descale": a / F}


# ---- its gradient -----------------------------------------------------------------------------------------------------

def _prepare_norm_backward(s, c, g):
    R, H, T = c["rows"], c["h"], STREAM[c["stream"]]
    s.sum, s.gamma = _stream_rows(g, R, H, T), _gamma(g, H)
    s.rms = torch.sqrt(s.sum.float().square().mean(1) + EPS)       # kept by the forward pass
    s.grad_normed, s.grad_sum = _normal(g, R, H, sigma=1e-3), _normal(g, R, H, sigma=1e-3, dtype=T)
    s.grad_residual, s.grad_gamma = torch.empty_like(s.sum), _empty(H)
    s.grad8, s.scale, s.amax = _empty(R, H, dtype=torch.uint8), _one(E5M2_MAX / 0.05), _one()


def _own_norm_backward(s, c, cf, st):
    R, H, f32 = c["rows"], c["h"], int(c["stream"] == "f32")
    if not c["quant"]:
        cf.cf_add_rmsnorm_backward(s.grad_normed, s.sum, f32, s.gamma, s.rms, s.grad_sum, R, H, s.grad_residual, s.grad_gamma, 0,
                                   s.ws, s.ws_bytes, st)
        return {"grad_residual": s.grad_residual, "grad_gamma": s.grad_gamma}
    s.amax.zero_()
    cf.cf_add_rmsnorm_backward_quant_e5m2(s.grad_normed, s.sum, f32, s.gamma, s.rms, s.grad_sum, R, H, s.grad_residual, s.grad_gamma, 0,
                                          s.grad8, s.scale, s.amax, s.ws, s.ws_bytes, st)
    return {"grad_residual": s.grad_residual, "grad_gamma": s.grad_gamma, "grad8": s.grad8.view(torch.float8_e5m2), "amax": s.amax}


def _plain_norm_backward(s, c):
    inv = 1.0 / s.rms[:, None]
    dy, xhat = s.grad_normed.float(), s.sum.float() * inv
    g = dy * s.gamma.float()
    d = s.grad_sum.float() + (g - xhat * (g * xhat).mean(1, keepdim=True)) * inv
    out = {"grad_residual": d.to(s.sum.dtype), "grad_gamma": (dy * xhat).sum(0, dtype=torch.float64).float()}
    return {**out, "grad8": _to8(d * s.scale, "e5m2"), "amax": d.abs().amax().reshape(1)} if c["quant"] else out


def _exact_norm_backward(s, c):
    dy, h, r, w = s.grad_normed.double(), s.sum.double(), s.rms.double().unsqueeze(1), s.gamma.double()
    dot = (dy * w).mul(h).sum(1, keepdim=True)
    d = s.grad_sum.double() + dy * w / r - h * dot / (c["h"] * r ** 3)
    out = {"grad_residual": d, "grad_gamma": (dy / r * h).sum(0)}
    return {**out, "grad8": _exact8(d * s.scale.double(), "e5m2"), "amax": d.abs().max().view(1)} if c["quant"] else out


# ---- the experts' block-scaled product --------------------------------------------------------------------------------

def _prepare_experts(s, c, g):
    T, K, N, E, top = (c[n] for n in ("tokens", "k", "n", "experts", "top_k"))
    scores = torch.randn(T, E, device=DEV, generator=g)
    if not c["even"]:               # popularity falls with the expert's number
        scores += 1.5 * torch.log(1.0 / torch.arange(1, E + 1, device=DEV))
    chosen = torch.topk(scores, top, 1).indices
    s.total = T * top
    s.expert, order = torch.sort(chosen.flatten(), stable=True)       # rows by expert, tokens ascending within one
    s.index = (order // top).to(torch.int32)
    s.counts = torch.bincount(s.expert, minlength=E).to(torch.int32)
    s.offsets = (torch.cumsum(s.counts, 0) - s.counts).to(torch.int32)
    s.parts = s.counts.tolist()     # for the plain form, whose products are one for each expert
    s.rows = T if c["gather"] else s.total
    x = _groups(torch.randn(s.rows, K, device=DEV, generator=g) * torch.exp(0.5 * torch.randn(s.rows, 1, device=DEV, generator=g)))
    a = x.abs().amax(2)
    s.a, s.a_descale = _to8(x * (E4M3_MAX / a)[:, :, None], "e4m3").flatten(1), a / E4M3_MAX
    rows = -(-N // 128) * 128       # weight scales go by blocks of 128 x 128, the last one cut short where N ends inside it
    w = (0.02 * torch.randn(E, rows, K, device=DEV, generator=g)).view(E, rows // 128, 128, K // 128, 128)
    w[:, -1, N - (rows - 128):] = 0.0
    a = w.abs().amax((2, 4))
    w.mul_((E4M3_MAX / a)[:, :, None, :, None])
    s.w, s.w_descale = _to8(w, "e4m3").view(E, rows, K)[:, :N].contiguous(), a / E4M3_MAX
    s.c = torch.zeros(s.total, N, dtype=torch.bfloat16, device=DEV)


def _own_experts(s, c, cf, st):
    K, N, E = c["k"], c["n"], c["experts"]
    cf.cf_fp8_grouped_gemm_nt_bf16_ex(s.total, N, K, E, s.counts, s.offsets, s.a, s.rows, K, s.index if c["gather"] else None, s.a_descale,
                                      s.w, s.w_descale, BLOCK_128, EPI_NONE, None, None, s.c, N, s.ws, s.ws_bytes, st)
    return s.c


def _plain_experts(s, c):
    K, N = c["k"], c["n"]
    a = (s.a.float().unflatten(1, (K // 128, 128)) * s.a_descale[:, :, None]).flatten(1)
    a = a[s.index.long()] if c["gather"] else a
    spread = s.w_descale.repeat_interleave(128, 1)[:, :N, :, None]
    w = (s.w.float().unflatten(2, (K // 128, 128)) * spread).flatten(2)
    return torch.cat([x @ w[e].t() for e, x in enumerate(a.split(s.parts))]).to(torch.bfloat16)


def _exact_experts(s, c):
    N = c["n"]
    a = s.a.double() * s.a_descale.double().repeat_interleave(128, 1)
    out = torch.zeros(s.total, N, dtype=torch.float64, device=DEV)
    first = 0
    for e, rows in enumerate(s.parts):
        w = s.w[e].double() * s.w_descale[e].double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)
        x = a[s.index[first:first + rows].long()] if c["gather"] else a[first:first + rows]
        out[first:first + rows] = x.mm(w.t())
        first += rows
    return out


# ---- the gradients' norm and clipping -----------------------------------------------------------------------------------

def _prepare_grads(s, c, g):
    h, i = c["h"], c["i"]
    big = torch.float32 if c["dtype"] == "f32" else torch.bfloat16
    small = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32
    # two norm weights, q k v o, gate and up, their biases, down; back to back in one buffer for each type, as trainers keep them
    layer = [(h, small), (h, small), (4 * h * h, big), (h * i, big), (h * i, big), (i, small), (i, small), (h * i, big)]
    shapes = layer * c["layers"]
    s.flat = {t: _normal(g, sum(n for n, u in shapes if u == t), sigma=1e-3, dtype=t) for t in sorted({u for _, u in shapes}, key=str)}
    s.out = {t: torch.zeros_like(f) for t, f in s.flat.items()}
    at = {t: [n for n, u in shapes if u == t] for t in s.flat}
    s.grads = [v for t, f in s.flat.items() for v in f.split(at[t])]
    s.clipped = [v for t, f in s.out.items() for v in f.split(at[t])]
    s.norm, s.coef = _one(), _one()


def _grad_list(cf, tensors, out):
    """The device table of a list of gradients, made once: the buffers stay where they are from step to step."""
    ptrs, outs = (torch.tensor([t.data_ptr() for t in ts], dtype=torch.int64) for ts in (tensors, out))
    counts = torch.tensor([t.numel() for t in tensors], dtype=torch.int64)
    types = torch.tensor([int(t.dtype == torch.float32) for t in tensors], dtype=torch.int32)
    n = ctypes.c_size_t(0)
    cf.cf_grad_list_bytes(counts, len(tensors), ctypes.byref(n))
    table = torch.empty(n.value, dtype=torch.uint8)
    cf.cf_grad_list_fill(ptrs, outs, counts, types, len(tensors), table, n.value)
    return table.to(DEV), n.value


def _named(out):
    return {str(t).removeprefix("torch."): f for t, f in out.items()}


def _own_grads(s, c, cf, st):
    cf.cf_grad_norm_clip(s.list, s.list_bytes, float(c["max_norm"]), s.norm, s.coef, s.ws, s.ws_bytes, st)
    return {"norm": s.norm, "coef": s.coef, **_named(s.out)}


def _plain_grads(s, c):
    norm = sum(f.double().square().sum() for f in s.flat.values()).sqrt()
    coef = (c["max_norm"] / norm).clamp(max=1.0).float().reshape(1)
    return {"norm": norm.float().reshape(1), "coef": coef, **_named({t: (f.float() * coef).to(t) for t, f in s.flat.items()})}


def _exact_grads(s, c):
    norm = torch.stack([t.double().norm() for t in s.grads]).norm()
    coef = c["max_norm"] / norm if norm > c["max_norm"] else torch.ones_like(norm)
    return {"norm": norm.view(1), "coef": coef.view(1), **_named({t: f.double() * coef for t, f in s.flat.items()})}


# ---- what a pass cannot do without --------------------------------------------------------------------------------------

def work(case):
    c, kind = case, case["kind"]
    if kind in ("norm", "norm_backward"):
        n, stream = c["rows"] * c["h"], 4 if c["stream"] == "f32" else 2
        if kind == "norm":          # the stream and the layer's output read, the new stream and the bytes written
            per = 2 * stream + 2 + 1 + (2 if c["normed"] else 0)
            scales = 8 * c["rows"] * {"rows": 1, "block": (c["h"] + 127) // 128, "record": 0}[c["form"]]
            return {"bytes": n * per + 2 * c["h"] + 4 * c["rows"] + scales, "flops": 8 * n}
        per = 2 + 3 * stream + (1 if c["quant"] else 0)      # dy, the stream, its gradient in and out, the bytes
        return {"bytes": n * per + 6 * c["h"] + 4 * c["rows"], "flops": 14 * n}
    if kind == "experts":
        T, K, N, E, top = (c[n] for n in ("tokens", "k", "n", "experts", "top_k"))
        used = E * (1.0 - (1.0 - top / E) ** T)              # experts that some token selects, in expectation
        rows = T if c["gather"] else T * top
        return {"bytes": rows * K * (1 + 4 / 128) + used * N * K * (1 + 4 / 16384) + 2 * T * top * N, "flops": 2 * T * top * N * K}
    h, i, small = c["h"], c["i"], 2 if c["dtype"] == "bf16" else 4
    per_layer = (4 * h * h + 3 * h * i) * (4 if c["dtype"] == "f32" else 2) + (2 * h + 2 * i) * small
    return {"bytes": 2 * c["layers"] * per_layer, "flops": 3 * c["layers"] * (4 * h * h + 3 * h * i)}
