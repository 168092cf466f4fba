"""Adapters whose inner sums are infinite: where the formula says infinity, infinity of its sign comes out, and NaN only where it says that."""
import pytest
import torch

from shiftaddllm_amd.lut_gemm.adapters import AdapterBank

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,rank", [(6, 8), (6, 40), (300, 16), (300, 128)])
def test_infinite_inner_sums(gpu_device, M, rank):
    gen = torch.Generator(device=gpu_device).manual_seed(M + rank)
    n = lambda *s: torch.randn(s, generator=gen, device=gpu_device)
    K, N, inf = 128, 68, float("inf")
    x, base = (n(M, K) * 100).half(), n(M, N).half()
    down, up, scale = (n(4, rank, K) * 100).half(), (n(4, N, rank) * 1e-4).half(), 0.5 + torch.rand(4, generator=gen, device=gpu_device)
    x[x == 0], down[down == 0], up[up == 0] = 1.0, 1.0, 1e-4
    down[0, 3, 5] = inf                                       # one infinite sum beside finite ones beyond fp16's range: its sign by the row's x
    down[1, 2, 9], down[1, rank - 1, 9] = inf, -inf           # two: NaN where they meet with unlike signs
    up[2, 7, 4] = 0.0
    down[2, 4, 0] = -inf                                      # 0 * infinity
    x[1, 3] = inf                                             # an input: all its sums, of the signs of down
    ids = torch.tensor([i % 4 for i in range(M)], dtype=torch.int32, device=gpu_device)
    ids[1] = 3
    up[3, :20] = up[3, :20].abs() * down[3, :, 3].sign()      # (all of one sign: infinity)
    got = AdapterBank.from_tensors(down, up, scale)(x, ids, base).double()
    want = base.double().cpu().clone()
    bound = torch.zeros_like(want)
    for m in range(M):
        a = int(ids[m])
        xr, d, w = x[m].double().cpu(), down[a].double().cpu(), up[a].double().cpu()
        h = (d * xr).sum(1)
        want[m] += float(scale[a]) * (w * h).sum(1)
        # exact products; sums in fp32, K and rank steps and four more of 2^-24 each
        bound[m] = float(scale[a]) * (w.abs() * (d * xr).abs().sum(1)).sum(1) * (K + rank + 4) * 2.0 ** -24
    bound += want.abs() * 2.0 ** -11 + 2.0 ** -24
    got = got.cpu()
    want = torch.where(want.abs() >= 65520, want.sign() * inf, want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ends = torch.isinf(want)
    assert bool(ends.any()) and bool(torch.isnan(want).any()) and bool(torch.isfinite(want).any())
    assert torch.equal(got[ends], want[ends])
    there = torch.isfinite(want)
    assert bool(((got[there] - want[there]).abs() <= bound[there]).all())
