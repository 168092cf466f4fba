"""Prompts over a 4-bit cache in every head size, by four waves a workgroup and by eight, against the definition in 64 bits."""
import pytest
import torch

from shiftaddllm_amd.kv_cache import Q4Cache
from test_gpu_q4_attention import Model, check, make
from test_gpu_q4_attention_weights import plan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", range(32, 257, 32))
@pytest.mark.parametrize("B,H,KV,T,threads", [(2, 4, 2, 70, 256), (4, 32, 4, 515, 512)])
def test_prompts(gpu_device, hd, B, H, KV, T, threads):
    """Memory that held NaN, prompts of unlike lengths, then more tokens onto them from the middle of a block."""
    P = 2 * T + 7
    p = plan(B, T, H, KV, hd, P)
    assert p.rows_apart == 1 and p.threads == threads
    gen = torch.Generator(device=gpu_device).manual_seed(hd + T)
    cache = Q4Cache(B, KV, P, hd, gpu_device, torch.full((B, KV, -(-P // 32), 40 * hd), 255, dtype=torch.uint8, device=gpu_device))
    model = Model(B, KV, P, hd, gpu_device)
    counts = [T, T - 17, 1, T // 2 + 3][:B]
    check(cache, model, *make(gen, B, T, H, KV, hd, gpu_device), [0] * B, counts)
    check(cache, model, *make(gen, B, T, H, KV, hd, gpu_device), counts, [T - 1, T, T, 0][:B])
