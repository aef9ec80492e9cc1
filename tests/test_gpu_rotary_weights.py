"""The norm weights' gradients over many rows against fp64, to the length of the sums that are taken in fp32: a
lane's share of its workgroup's rows, not all of them."""
import pytest
import torch

from pyasc_amd import kernels
from test_gpu_rotary import U, heads, turn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,hq,hk,s,d", [(4, 32, 8, 2047, 64), (2, 16, 16, 4096, 80), (1, 8, 1, 30000, 128)])
def test_many_rows(device, b, hq, hk, s, d, dtype):
    g = torch.Generator(device=device).manual_seed(s)
    x, dy = ([heads((b, h, s, d), dtype, g, "contiguous") for h in (hq, hk)] for _ in range(2))
    w = [1 + 0.3 * torch.randn(d, generator=g, device=device) for _ in range(2)]
    freqs, _ = kernels.rotary_frequencies(d)
    positions = torch.arange(s, device=device)
    dx = [torch.empty_like(t) for t in x]
    dw = [torch.empty_like(t) for t in w]
    kernels.qk_norm_rotary_bwd(*dy, *x, *w, positions, freqs, *dx, *dw, epsilon=1e-5)
    for i, h in enumerate((hq, hk)):
        r = 1 / torch.sqrt(x[i].double().pow(2).mean(-1, keepdim=True) + 1e-5)
        up, size = turn(dy[i].double(), positions, freqs, False, 1.0, -1.0)
        xr = x[i].double() * r
        want, terms = (up * xr).sum((0, 1, 2)), (size * xr.abs()).sum((0, 1, 2))
        # A workgroup's pass has at least 4 rows (a row has at most 64 lanes of 256), and up to 1024
        # workgroups share the tokens evenly, to a tile of at most 8: a lane adds up at most this many
        # rows, then at most 6 steps of a butterfly and 4 waves; what follows is fp64.  9 half steps for the
        # turned gradient, 30 for x r (as in the norm's own bound), one for their product.
        share = -(-b * s // 1024) + 8
        chain = -(-share * h // 4)
        bound = (chain + 6 + 4 + 9 + 30 + 1) * U * terms + U * want.abs()
        assert ((dw[i].double() - want).abs() <= bound).all(), float(((dw[i].double() - want).abs() / bound).max())
