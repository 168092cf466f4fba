"""Capturing a decoder's step while it holds prompts and tokens: nothing that a caller can see changes."""
import pytest
import torch

from shiftaddllm_amd import decode
from shiftaddllm_amd.sampling import SamplingOptions

pytestmark = pytest.mark.gpu
CFG = decode.DecoderConfig(vocab_size=320, hidden=256, intermediate=512, layers=2, heads=4, kv_heads=2, max_positions=64)


def make(device, batch, sampling=True):
    return decode.LutDecoder(CFG, None, batch=batch, seed=1, device=device, kv_bits=4,
                             sampling=SamplingOptions(0.9, 20, 0.95, 0.0, 1) if sampling else None)


@pytest.mark.parametrize("batch,sampling", [(1, False), (3, True), (5, True)])
def test_prompt_capture_token(gpu_device, batch, sampling):
    """prefill, capture, forward_token: as the same calls without the capture, to the last bit."""
    gen = torch.Generator().manual_seed(batch)
    ids = torch.randint(0, CFG.vocab_size, (batch, 8), generator=gen)
    lengths = [8 - b for b in range(batch)]
    results = []
    for capture in (False, True):
        m = make(gpu_device, batch, sampling)
        with torch.no_grad():
            seen = [m.prefill(ids, lengths).clone()]
            if capture:
                m.capture()
            seen += [m.logits.clone(), *(c.data.clone() for c in m.q4)]
            if sampling:
                m.uniform.fill_(0.5)
            for t in range(3):
                seen.append(m.forward_token(ids[:, t].to(gpu_device), [n + t for n in lengths]).clone())
                if sampling:
                    seen += [m.next_ids.clone(), m.next_logprob.clone()]
            seen += [c.data.clone() for c in m.q4]
        results.append(seen)
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_a_slot_taken_over_between_a_token_and_a_capture(gpu_device):
    """A sequence that was at position 12 makes room for a new prompt; then the step is captured: the prompt stays, and so does what was drawn last."""
    gen = torch.Generator().manual_seed(4)
    ids = torch.randint(0, CFG.vocab_size, (2, 20), generator=gen)
    results = []
    for capture in (False, True):
        m = make(gpu_device, 2)
        with torch.no_grad():
            m.prefill(ids[:, :12])
            m.uniform.fill_(0.3)
            m.forward_token(ids[:, 12].to(gpu_device), [12, 12])
            drawn = [m.next_ids.clone(), m.next_logprob.clone()]
            m.prefill(ids, [20, 0], [0, 0])
            m.uniform.fill_(0.8)
            if capture:
                m.capture()
            assert torch.equal(m.next_ids, drawn[0]) and torch.equal(m.next_logprob, drawn[1])
            seen = [c.data.clone() for c in m.q4] + [m.logits.clone()]
            seen.append(m.forward_token(ids[:, 1].to(gpu_device), [20, 13]).clone())
        results.append(seen)
    assert all(torch.equal(a, b) for a, b in zip(*results))
