"""GPU: the sums over the rows in the gradient of the gated norm (both weights', the gates') are taken in 64 bits, but for one rounding of each worker's share.

rms are 1 and the second weight is 0, so that D = dh and every term dy * hh, D * xh is exact: c * 2^24 in one row of sixteen, c in the others, c a power of two by column; the first weight
and the gates are powers of two.  64 bits hold all sums exactly.  Rounding the shares loses at most 2^-24 of the sum of their sizes, which is the sum itself as all terms have one sign, and
the last rounding 2^-24 of it: 2^-23 in all.  Sums in 32 bits lose each small row behind a worker's first large one, as c is half a unit of c * 2^24 and the even neighbour takes the tie: some
fifteen 2^-24 of a worker's sum where it has tens of rows, more than half of that where its large rows lie anywhere among them."""
import ctypes

import pytest
import torch

from gpu_util import case, stream
from test_gpu_add_norm import STREAM, Out
from test_gpu_gated_norm import E4M3, kept_scale

pytestmark = pytest.mark.gpu

# rows, H: a wavefront a row, one chunk a thread, two, two of the wide kernel, the widest; multiples of eight and others; thirty rows a worker and more
SHAPES = [(70000, 64), (70000, 511), (33000, 1000), (8300, 2056), (8300, 4095), (8300, 4100), (8300, 7168), (8300, 8201), (8300, 12288), (8300, 16384)]
# none, one gate, some hundred rows that several workers have, a gate a row (whole groups: eight and more a worker)
GATE_ROWS = [0, None, 300, 1]


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("gate_rows", GATE_ROWS)
@pytest.mark.parametrize("rows,H", SHAPES)
def test_rows_are_summed_in_64_bits(cf, dev, rows, H, gate_rows, f32, kept):
    gate_rows = rows if gate_rows is None else gate_rows
    case(f"gated norm gradient sums rows={rows} H={H} gate_rows={gate_rows} f32={f32} kept={kept}")
    g = torch.Generator(device=dev).manual_seed(rows + H)
    power = torch.where(torch.rand(rows, 1, device=dev, generator=g) < 1 / 16, 2.0 ** 24, 1.0)
    column = 2.0 ** (torch.arange(H, device=dev) % 3).float()
    groups = -(-rows // gate_rows) if gate_rows else 0
    gate = 2.0 ** ((torch.arange(groups, device=dev)[:, None] + torch.arange(H, device=dev)) % 3 - 1).float() if gate_rows else None
    wp = 2.0 ** (torch.arange(H, device=dev) % 2).float()
    saved = lambda t: column.repeat(rows, 1).to(t).view(torch.uint8 if kept else t)  # noqa: E731
    S = kept_scale(H) if kept else 1.0
    h, x = saved(E4M3 if kept else STREAM[f32]), saved(E4M3 if kept else torch.bfloat16)
    dy, dh = power.to(torch.bfloat16).repeat(1, H), power.to(STREAM[f32]).repeat(1, H)
    one, zero = torch.ones(rows, device=dev), torch.zeros(H, dtype=torch.bfloat16, device=dev)
    bf = lambda t: t.to(torch.bfloat16) if t is not None else None  # noqa: E731
    n = ctypes.c_size_t(0)
    cf.cf_gated_add_rmsnorm_backward_workspace_bytes(rows, H, gate_rows, ctypes.byref(n))
    ws = torch.empty(n.value, dtype=torch.uint8, device=dev)
    dr, dx = torch.empty_like(dh), torch.empty_like(dy)
    gate16, wp16 = bf(gate), bf(wp)
    call = cf.cf_gated_add_rmsnorm_backward_ckpt8 if kept else cf.cf_gated_add_rmsnorm_backward

    def run(start=None):
        o = {"dw": Out(dev, (H,), torch.float32), "dwp": Out(dev, (H,), torch.float32), "dgate": Out(dev, (max(groups, 1), H), torch.float32)}
        if start is not None:
            for v in o.values():
                v.t.copy_(start)
        call(dy, h, x, f32, 1.0, gate16, gate_rows, wp16, zero, one, one, dh, rows, H, dr, dx, None, None, None, o["dwp"].t, o["dw"].t, o["dgate"].t, 0 if start is None else 3,
             ws, n.value, stream())
        torch.cuda.synchronize()
        assert all(v.unharmed() for v in o.values())
        return {k: v.t.double() for k, v in o.items()}

    # the sums of the rows' powers, exact in 64 bits, times the columns' factors
    p, c = power.double()[:, 0], column.double() / S
    exact = {"dw": p.sum() * c, "dwp": p.sum() * c}
    if gate_rows:
        per_group = torch.nn.functional.pad(p, (0, -rows % gate_rows)).view(groups, gate_rows).sum(1)[:, None] * c
        exact["dwp"], exact["dgate"] = (per_group * gate.double()).sum(0), per_group * wp.double()
    got = run()
    start = torch.linspace(0.0, 1e9, H, device=dev)
    added = run(start)
    for k, want in exact.items():
        assert torch.all((got[k] - want).abs() <= 2.0 ** -23 * want), k
        total = want + start.double()
        assert torch.all((added[k] - total).abs() <= 2.0 ** -24 * (want + total)), k
