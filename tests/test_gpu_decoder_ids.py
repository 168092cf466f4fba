"""Ids that stand for no token: what sampling gives a row without weight, what a server leaves in an idle slot."""
import pytest
import torch

from shiftaddllm_amd import decode
from shiftaddllm_amd.sampling import SamplingOptions

pytestmark = pytest.mark.gpu
CFG = decode.DecoderConfig(vocab_size=320, hidden=256, intermediate=512, layers=2, heads=4, kv_heads=2, max_positions=64)


@pytest.mark.parametrize("kv_bits", [16, 4])
@pytest.mark.parametrize("capture", [False, True])
def test_a_row_without_weight_goes_on(gpu_device, kv_bits, capture):
    m = decode.LutDecoder(CFG, None, batch=2, seed=1, device=gpu_device, kv_bits=kv_bits, sampling=SamplingOptions(seed=1))
    head = m.lm_head.data.clone()
    if capture:
        m.capture()
    with torch.no_grad():
        m.lm_head.data.fill_(float("nan"))
        m.forward_token(torch.tensor([3, 4], device=gpu_device), 0)
        assert m.next_ids.tolist() == [-1, -1] and bool((m.next_logprob == float("-inf")).all())
        m.lm_head.data.copy_(head)
        got = m.forward_token(m.next_ids, 1).clone()
        assert torch.equal(got, m.forward_token(torch.zeros(2, dtype=torch.long), 1))
        assert bool((m.next_ids >= 0).all())
        m.lm_head.data.fill_(float("nan"))
        drawn = decode.benchmark(m, torch.tensor([[1, 2], [5, 6]]), generate=4, warmup=1)["generated"]
        assert bool((drawn == -1).all())


def test_an_idle_slot_holds_any_id(gpu_device):
    m = decode.LutDecoder(CFG, None, batch=4, seed=2, device=gpu_device, kv_bits=4)
    ids = torch.tensor([1, 2, 3, 4], device=gpu_device)
    with torch.no_grad():
        m.forward_token(ids, [0, 0, 0, 0])
        caches = [c.data.clone() for c in m.q4]
        want = m.forward_token(ids, [1, -1, 1, -7]).clone()
        after = [c.data.clone() for c in m.q4]
        for c, b in zip(m.q4, caches):
            c.data.copy_(b)
        got = m.forward_token(torch.tensor([1, -1, 3, 2 ** 40], device=gpu_device), [1, -1, 1, -7])
        assert torch.equal(got[[0, 2]], want[[0, 2]]) and all(torch.equal(c.data, a) for c, a in zip(m.q4, after))
