"""A decoder's caches and workspaces go where the decoder goes."""
import torch

from shiftaddllm_amd import decode
from shiftaddllm_amd.kv_cache import Q4Cache

CFG = decode.DecoderConfig(vocab_size=32, hidden=128, intermediate=128, layers=2, heads=2, kv_heads=1, max_positions=40)


def test_caches_of_four_bits_move_with_the_decoder():
    m = decode.LutDecoder(CFG, None, device="cpu", kv_bits=4, batch=2)
    for c in m.q4:
        c.data.fill_(7)
    before = set(m.state_dict())
    m.half()                                                         # (bytes stay bytes)
    assert all(c.data.dtype is torch.uint8 and bool((c.data == 7).all()) for c in m.q4)
    m.reset()
    assert all(bool((c.data == 0).all()) for c in m.q4)
    m.to("meta")
    assert m.logits.device.type == "meta" and all(c.data.device.type == "meta" for c in m.q4)
    assert not any("q4" in k for k in before)                        # caches are no state, as the fp16 ones


def test_a_cache_of_ones_own_is_the_memory_that_was_given():
    data = torch.zeros((1, 2, 2, 40 * 64), dtype=torch.uint8)
    cache = Q4Cache(1, 2, 40, 64, "cpu", data)
    assert cache.data is data and not cache.state_dict() and not list(cache.parameters())


def test_workspaces_are_where_the_decoder_is():
    m = decode.LutDecoder(CFG, None, device="cpu")
    a = m._workspace(100)
    assert m._workspace(50) == a
    m.to("meta")
    m._workspace(50)
    assert m._workspaces[-1].device.type == "meta" and m._workspaces[0].device.type == "cpu"
