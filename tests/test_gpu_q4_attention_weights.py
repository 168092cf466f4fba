"""Softmax weights of attention over a 4-bit cache where their range is what counts: a dominant position in front of a long tail."""
import math

import pytest
import torch

from shiftaddllm_amd.kv_cache import Q4Cache
from shiftaddllm_amd import native

pytestmark = pytest.mark.gpu


def plan(B, T, H, KV, hd, P):
    p = native.Q4AttentionPlan()
    assert native.cabi().lutgemm_describe_q4_attention_plan(B, T, H, KV, hd, P, p) == 0
    return p


def unturned(P, hd, device):
    """Angles of zero: keys and queries are cached and used as they are."""
    return torch.ones((P, hd), dtype=torch.float16, device=device), torch.zeros((P, hd), dtype=torch.float16, device=device)


# (batch, query heads, kv heads, head_dim, positions, tokens of the last call, workgroups that share positions): one token, a few, prompts
FORMS = [(1, 4, 1, 128, 320, 1, False), (1, 2, 1, 64, 8192, 1, True), (2, 8, 2, 128, 6000, 1, True), (1, 8, 1, 64, 4100, 4, True), (1, 4, 1, 128, 6000, 100, True),
         (1, 32, 4, 64, 8192, 2048, False), (1, 64, 8, 160, 1500, 400, False)]


@pytest.mark.parametrize("B,H,KV,hd,P,T,shared", FORMS)
@pytest.mark.parametrize("powers", [12, 17, 20, 23, 26, 29])
def test_a_long_tail_behind_one_dominant_position(gpu_device, B, H, KV, hd, P, T, shared, powers):
    """Position 0 has the largest score by 2^powers and values of 0: what comes out is the tail alone."""
    assert (plan(B, T, H, KV, hd, P).splits > 1) is shared
    gen = torch.Generator(device=gpu_device).manual_seed(P + powers)
    n = lambda *s: torch.randn(s, generator=gen, device=gpu_device)
    cos, sin = unturned(P, hd, gpu_device)
    k, v = n(B, P, KV, hd) * 0.2, 1000 + 300 * n(B, P, KV, hd)
    k[..., :32] = 0
    k[:, 0, :, :32] = 8.0
    v[:, 0] = 0
    q = n(B, P, H, hd) * 0.5
    q[..., :32] = powers * math.log(2) * math.sqrt(hd) / (32 * 8.0)
    q, k, v = (x.half().flatten(2) for x in (q, k, v))
    cache = Q4Cache(B, KV, P, hd, gpu_device)
    zero = torch.zeros(B, dtype=torch.long, device=gpu_device)
    cache.attend(q[:, :P - T], k[:, :P - T], v[:, :P - T], cos, sin, zero)
    out = cache.attend(q[:, P - T:], k[:, P - T:], v[:, P - T:], cos, sin, zero + (P - T)).view(B, T, H, hd)
    for b in range(B):
        kk, vv = (x.double() for x in cache.values(b, P))
        for t in sorted({0, T // 3, T - 1}):
            L = P - T + t + 1
            for h in range(H):
                keys, values, row = kk[:L, h // (H // KV)], vv[:L, h // (H // KV)], q[b, P - T + t].view(H, hd)[h].double()
                score = keys @ row / math.sqrt(hd)
                size = float((keys.abs() @ row.abs()).max()) / math.sqrt(hd)
                p = torch.softmax(score, 0)
                want, spread = p @ values, p @ values.abs()
                # A weight rounds to fp16, half a step of 2^-11, of itself where it is 2^-21 of the row's largest or more, of 2^-21 below; the result
                # rounds likewise.  Scores: at most hd steps of 2^-24 of what they are made of, the factor and the exponential 2^-22 each;
                # weights and their sum are off by as much.  Sums over positions: below 2^-13 at these lengths.
                bound = spread * (2.0 ** -11 + 2.0 ** -13 + 2 * size * (hd * 2.0 ** -24 + 2.0 ** -21)) + want.abs() * 2.0 ** -11 + \
                    L * 2.0 ** -32 * p.max() * values.abs().amax(0) + 2.0 ** -24
                off = (out[b, t, h].double() - want).abs()
                assert bool((off <= bound).all()), (b, t, h, float((off / bound).max()), float((off / want.abs()).max()))
