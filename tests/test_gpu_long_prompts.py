"""Prompts of more tokens than a quantised product has rows."""
import pytest
import torch

from shiftaddllm_amd import decode
from test_gpu_served_decoder import CFG, fill_adapters

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [4, 21, 27])
def test_prompts_by_parts(gpu_device, monkeypatch, rows):
    """As calls of the parts one after the other, to the last bit; sequences that end in an earlier part or have no tokens among them."""
    B, T = 3, 20
    ids = torch.randint(0, CFG.vocab_size, (B, T), generator=torch.Generator().manual_seed(1))
    lengths, starts, most = [20, 0, 7], [3, -4, 0], rows // B
    results = []
    for parts in (False, True):
        m = decode.LutDecoder(CFG, None, batch=B, seed=1, device=gpu_device, kv_bits=4, adapters=(2, 8))
        fill_adapters(m, 2)
        m.adapter_ids.copy_(torch.tensor([0, 1, -1], dtype=torch.int32))
        m.logits.fill_(3.0)
        if parts:
            for t in range(0, T, most):
                m.prefill(ids[:, t:t + most], [min(max(n - t, 0), most) for n in lengths], [p + t if n > t else -1 for p, n in zip(starts, lengths)])
        else:
            with monkeypatch.context() as patch:
                patch.setattr(decode, "PREFILL_ROWS", rows)
                m.prefill(ids, lengths, starts)
        results.append([m.logits.clone(), *(c.data.clone() for c in m.q4)])
    assert all(torch.equal(a, b) for a, b in zip(*results)) and bool((results[0][0][1] == 3.0).all())


def test_more_tokens_than_a_product_has_rows(gpu_device):
    cfg = decode.DecoderConfig(vocab_size=64, hidden=128, intermediate=128, layers=1, heads=2, kv_heads=1, max_positions=34000, group_size=64)
    ids = torch.randint(0, 64, (2, 33000), generator=torch.Generator().manual_seed(2))
    results = []
    for whole in (True, False):
        m = decode.LutDecoder(cfg, None, batch=2, seed=1, device=gpu_device, kv_bits=4)
        if whole:
            m.prefill(ids, [33000, 32800])
        else:
            m.prefill(ids[:, :32767])
            m.prefill(ids[:, 32767:], [233, 33], [32767, 32767])
        results.append([m.logits.clone(), m.q4[0].data.clone()])
    assert bool(torch.isfinite(results[0][0]).all()) and all(torch.equal(a, b) for a, b in zip(*results))
