"""Attention over a 4-bit cache with queries and keys of any size that fp16 and the cache hold: scores up to 2^36."""
import pytest
import torch

from shiftaddllm_amd.kv_cache import Q4Cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [100.0, 2000.0, 16000.0, 60000.0])
@pytest.mark.parametrize("B,H,KV,hd,P,T", [(1, 4, 1, 64, 200, 1), (2, 4, 2, 128, 3000, 1), (1, 8, 1, 96, 3000, 4), (1, 4, 2, 128, 500, 200), (1, 32, 4, 64, 1200, 700)])
def test_the_position_of_the_largest_score(gpu_device, B, H, KV, hd, P, T, size):
    """Scores so far apart that a row's softmax is one at its largest: the row comes out as that position's values, but for two roundings to
    fp16, of its weight and of the result, half a step (2^-11) each.

    Position j's key is a_j in every dimension (held as it is: a group of equal numbers is its minimum), a_j = size * (j's place in a shuffled order + 1) / P, a query +-size in
    every dimension.  Scores are size^2 * (place + 1) / P * sqrt(hd): neighbours lie size^2 sqrt(hd) / P apart, 2^-12 of the largest or more, where fp32 sums of
    hd products err by hd * 2^-24; at size 100 and 3000 positions that is 32 or more, e^-32 of the row's weight, far below half a step of fp16."""
    gen = torch.Generator(device=gpu_device).manual_seed(P + T)
    places = torch.stack([torch.randperm(P, generator=gen, device=gpu_device) for _ in range(B * KV)]).view(B, KV, P)
    a = ((places + 1).double() / P * size).half()
    k = a.transpose(1, 2).unsqueeze(-1).expand(B, P, KV, hd)
    sign = torch.randint(0, 2, (B, P, H, 1), generator=gen, device=gpu_device).mul(2).sub(1).half()
    q = (sign * size).expand(B, P, H, hd)
    v = torch.randn((B, P, KV, hd), generator=gen, device=gpu_device).half()
    q, k, v = (x.reshape(B, P, -1).contiguous() for x in (q, k, v))
    cos, sin = torch.ones((P, hd), dtype=torch.float16, device=gpu_device), torch.zeros((P, hd), dtype=torch.float16, device=gpu_device)
    cache = Q4Cache(B, KV, P, hd, gpu_device)
    zero = torch.zeros(B, dtype=torch.long, device=gpu_device)
    cache.attend(q[:, :P - T], k[:, :P - T], v[:, :P - T], cos, sin, zero)
    out = cache.attend(q[:, P - T:], k[:, P - T:], v[:, P - T:], cos, sin, zero + (P - T)).view(B, T, H, hd)
    looked = 0
    for b in range(B):
        _, values = cache.values(b, P)
        for t in sorted({0, T // 2, T - 1}):
            L = P - T + t + 1
            for h in range(H):
                own = a[b, h // (H // KV), :L].double() * float(sign[b, L - 1, h, 0])
                best = torch.topk(own, 2)
                if float(best.values[0] - best.values[1]) * size * hd ** 0.5 < 25:      # (keys that fp16 rounds to the same number)
                    continue
                looked += 1
                want = values[int(best.indices[0]), h // (H // KV)].double()
                assert bool(((out[b, t, h].double() - want).abs() <= want.abs() * 1.001 * 2.0 ** -10 + 2.0 ** -24).all()), (b, t, h)
    assert looked > 0
