"""Choosing tokens from logits at the ends of fp32's range."""
import math

import numpy as np
import pytest
import torch

from shiftaddllm_amd.sampling import sample

pytestmark = pytest.mark.gpu


def held(row, u, t, k, p, m):
    """(id, logprob) of a row whose largest logit is finite, with weights held as the header says: whole numbers of 2^-b, b = 63 - ceil(log2 vocab) but 51
    at most.  (Many equal weights, all rounded alike, move a sum by up to vocab * 2^-(b + 1): 2^-34 of 30000, more than a comparison with unrounded
    sums would leave room for.)"""
    x, V = row.double().cpu().numpy(), row.numel()
    one = 2 ** min(63 - (V - 1).bit_length(), 51)
    order = np.argsort(-x, kind="stable")
    w = [int(v) for v in np.rint(np.exp((x[order] - x[order[0]]) / t) * one)]
    n = k or V
    total = sum(w[:n])

    def first(target, at_most):
        s = 0
        for i in range(at_most):
            s += w[i]
            if s >= target:
                return i, s
    if p is not None:
        n, total = first(max(math.ceil(p * float(total)), 1), n)
        n += 1
    if m is not None:
        left = sum(v for v in w if v >= math.ceil(m * one))
        total = min(total, left)
    at, _ = first(min(math.floor(u * float(total)), total - 1) + 1, n)
    return int(order[at]), (x[order[at]] - x[order[0]]) / t - math.log(total / one)


@pytest.mark.parametrize("V", [40, 3000, 30000])
def test_logits_further_apart_than_the_largest_number(gpu_device, V):
    """Differences of finite logits beyond fp32's range, at temperatures that give both ends weight."""
    gen = torch.Generator(device=gpu_device).manual_seed(V)
    rows = torch.empty((4, V), device=gpu_device)
    rows[0] = -3e38
    rows[0, V // 2] = 3e38
    rows[1] = torch.where(torch.arange(V, device=gpu_device) % 2 == 0, 3.4e38, -3.4e38)
    rows[2] = (torch.rand(V, generator=gen, device=gpu_device) * 2 - 1) * 3.4e38
    rows[3] = -3e38
    rows[3, ::3] = float("-inf")
    rows[3, 1] = 2e38
    f32 = lambda v: float(np.float32(v)) if v is not None else None
    for t in (1e38, 3e37, 3e38):
        for u in (0.0, 0.3, 0.7, 0.95, 1 - 2.0 ** -24):
            for k, p, m in ((None, None, None), (V // 2, None, None), (None, 0.9, None), (V - 1, 0.99, 1e-4)):
                ids, lp = sample(rows, torch.full((4,), u, device=gpu_device), t, k, p, m)
                for r in range(4):
                    want, wlp = held(rows[r], f32(u), f32(t), k, f32(p), f32(m))
                    assert int(ids[r]) == want, (r, t, u, k, p, m)
                    # the sums are whole numbers, the logarithm rounds to fp32
                    assert abs(float(lp[r]) - wlp) <= abs(wlp) * 2.0 ** -24 + 2.0 ** -45, (r, t, u, k, p, m)
