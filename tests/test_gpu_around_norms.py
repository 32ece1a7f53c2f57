"""GPU tests of the norms around a block against bounds counted from the kernels' own sums, and at every width."""
import numpy as np
import pytest
import torch

import around_exact as exact
import test_gpu_around as base
from cases import bind

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import super_gemma_b200 as sg

    return sg.GpuContext(0)


def _check(got, y, h, w_post, gate, w_pre, kind, post, gates, plus_one, scale, eps, what):
    f = lambda t: t.float().cpu().numpy().astype(np.float64)  # noqa: E731
    g = (None, f(gate)[:h.shape[1]], f(gate)[:h.shape[0], None], f(gate)[:1])[gates]
    want, err, x, x_err = exact.block_norms(f(y), f(h), f(w_post) + plus_one, g, f(w_pre) + plus_one, post, float(np.float32(scale)), float(np.float32(eps)))
    if post != 2:
        base._within(f(got[0]), want, err + base.HALF_STEP[kind] * (np.abs(want) + err) + base.TINY[kind], f"{what}: h")
    base._within(f(got[1]), x, x_err + 2.0 ** -11 * (np.abs(x) + x_err) + 2.0 ** -25, f"{what}: x")


@pytest.mark.parametrize("kind", list(base.TYPES))
@pytest.mark.parametrize("rows,hidden", [(3, 8), (40, 72), (7, 512), (65, 1096), (20, 2048), (400, 5376), (9, 16384), (5000, 1096), (1500, 5376), (900, 16384), (40_001, 264)])
def test_norms_to_the_last_digits(ctx, kind, rows, hidden):
    some = torch.arange(rows) if rows <= 100 else torch.cat([torch.arange(40), torch.arange(rows - 60, rows)])
    some = some.cuda()
    for post, gates, plus_one, scale, eps in ((1, 1, 1, 0.75, 1e-6), (1, 2, 0, -1.5, 1e-5), (0, 3, 0, 1.0, 1e-6), (0, 0, 1, 0.5, 0.0), (2, 0, 1, 1.0, 1e-6)):
        y, h, w_post, gate, w_pre = base._norms_case(rows + hidden + post, kind, rows, hidden, gates)
        got = base._norms(ctx, kind, y, h, w_post, gate, w_pre, post, gates, plus_one, scale, eps)
        _check([t[some] for t in got], y[some], h[some], w_post, gate[some] if gates == 2 else gate, w_pre, kind, post, gates, plus_one, scale, eps, (post, gates))


@pytest.mark.parametrize("kind,step", [("f16", 8), ("bf16", 104), ("f32", 56)])
def test_norms_of_every_width(ctx, kind, step):
    """One row, rows that do not fit the GPU at once, and rows that come ahead or ask late: the first and the last of each."""
    most = 11_000_000 + 16384
    y, h, w_post, _, w_pre = base._norms_case(3, kind, 1, most, 0)
    h_out, x = torch.zeros_like(h), torch.zeros_like(y)
    torch.cuda.synchronize()
    kernel = ctx.load_kernel("block_norms_" + kind)
    buffers = bind(*(ctx.adopt(t.data_ptr(), t.numel() * t.element_size(), np.uint8, keep=t) for t in (y, h, w_post, w_post, w_pre, h_out, x)))
    for hidden in range(8, 16385, step):
        for total in (1, 9_900_000, 11_000_000):
            rows = max(1, total // hidden)
            ends = slice(0, hidden), slice((rows - 1) * hidden, rows * hidden)
            for e in ends:
                h_out[0, e], x[0, e] = 3, 3
            torch.cuda.synchronize()
            ctx.dispatch_blocking(kernel, buffers, (1, 0, 0, 0.5, 1e-6), [hidden, rows, 1])
            both = lambda t: torch.stack([t[0, e] for e in ends])  # noqa: E731
            _check((both(h_out), both(x)), both(y), both(h), w_post[:hidden], w_post[:1], w_pre[:hidden], kind, 1, 0, 0, 0.5, 1e-6, (rows, hidden))
