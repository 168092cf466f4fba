"""Calls at the edge of what the served operators' documentation allows: positions given in other forms, prompts with anything at all
behind their ends, ids beyond 32 bits, outputs inside inputs, a row's share captured and replayed, two streams at once."""
import numpy as np
import pytest
import torch

from shiftaddllm_amd import decode
from shiftaddllm_amd.kv_cache import Q4Cache
from shiftaddllm_amd.lut_gemm.adapters import AdapterBank
from shiftaddllm_amd.sampling import sample

pytestmark = pytest.mark.gpu
CFG = decode.DecoderConfig(vocab_size=320, hidden=256, intermediate=512, layers=2, heads=4, kv_heads=2, max_positions=64)


@pytest.mark.parametrize("kv_bits", [16, 4])
def test_a_position_in_any_form_of_whole_number(gpu_device, kv_bits):
    model = decode.LutDecoder(CFG, None, batch=1, seed=1, device=gpu_device, kv_bits=kv_bits)
    ids = torch.tensor([5], device=gpu_device)
    with torch.no_grad():
        want = model.forward_token(ids, 0).clone()
        for position in (np.int64(0), np.int32(0), torch.tensor(0), torch.tensor(0, device=gpu_device)):
            model.reset()
            assert torch.equal(model.forward_token(ids, position), want)
        for position in (np.int64(64), torch.tensor(64), np.int64(-1)):
            with pytest.raises(ValueError):
                model.forward_token(ids, position)


def test_what_stands_behind_a_prompt_is_not_looked_at(gpu_device):
    model = decode.LutDecoder(CFG, None, batch=3, seed=2, device=gpu_device, kv_bits=4)
    ids = torch.randint(0, CFG.vocab_size, (3, 6), generator=torch.Generator().manual_seed(2))
    lengths = [2, 6, 0]
    with torch.no_grad():
        want = model.prefill(ids, lengths).clone()
        caches = [c.data.clone() for c in model.q4]
        padded = ids.clone()
        for b, n in enumerate(lengths):
            padded[b, n:] = torch.tensor([-100, 2 ** 40, CFG.vocab_size])[torch.arange(6 - n) % 3]
        model.reset()
        assert torch.equal(model.prefill(padded, lengths)[:2], want[:2])
        assert all(torch.equal(c.data, d) for c, d in zip(model.q4, caches))


def test_adapter_ids_beyond_32_bits_name_no_adapter(gpu_device):
    gen = torch.Generator(device=gpu_device).manual_seed(3)
    lin = decode.random_lut_linear(128, 64, 3, 128, gen, gpu_device)
    lin.adapters = AdapterBank(128, 64, 8, 2).to(gpu_device)
    lin.adapters.set(0, torch.randn((8, 128), generator=gen, device=gpu_device), torch.randn((64, 8), generator=gen, device=gpu_device))
    x = torch.randn((4, 128), generator=gen, device=gpu_device).half()
    ids = torch.tensor([2 ** 32, -2 ** 32, 2 ** 40, 2], device=gpu_device)
    assert torch.equal(lin(x, ids), lin(x))
    assert not torch.equal(lin(x, torch.zeros_like(ids)), lin(x))


def test_outputs_inside_inputs_are_refused(gpu_device):
    half = dict(device=gpu_device, dtype=torch.float16)
    cache = Q4Cache(2, 1, 32, 64, gpu_device)
    q, k, v = torch.randn((2, 64), **half), torch.randn((2, 64), **half), torch.randn((2, 64), **half)
    table, start = torch.ones((32, 64), **half), torch.zeros(2, dtype=torch.long, device=gpu_device)
    before = cache.data.clone()
    for out in (q, k, v, table[:2], cache.data.view(-1)[:256].view(torch.float16)):
        with pytest.raises((RuntimeError, ValueError)):
            cache.attend(q, k, v, table, table, start, out=out)
    assert torch.equal(cache.data, before)
    bank = AdapterBank(64, 64, 8, 1).to(gpu_device)
    x, ids = torch.randn((4, 64), **half), torch.zeros(4, dtype=torch.int32, device=gpu_device)
    base = torch.randn((8, 64), **half)
    for kw in (dict(base=base[:4], out=x), dict(base=base[:4], out=base[1:5]), dict(base=base[:4], out=base[:1].expand(4, 64))):
        with pytest.raises((RuntimeError, ValueError)):
            bank(x, ids, **kw)


def test_gradients_are_refused_where_there_are_none(gpu_device):
    half = dict(device=gpu_device, dtype=torch.float16)
    logits = torch.randn((2, 100), device=gpu_device, requires_grad=True)
    uniform = torch.rand(2, device=gpu_device)
    with pytest.raises(RuntimeError):
        sample(logits, uniform)
    with torch.no_grad():
        ids, _ = sample(logits, uniform)
    assert torch.equal(ids, sample(logits.detach(), uniform)[0])
    bank, x = AdapterBank(64, 64, 8, 1).to(gpu_device), torch.randn((1, 64), requires_grad=True, **half)
    with pytest.raises(RuntimeError):
        bank(x, torch.zeros(1, dtype=torch.int32, device=gpu_device), torch.zeros((1, 64), **half))
    cache = Q4Cache(1, 1, 32, 64, gpu_device)
    table = torch.ones((32, 64), **half)
    with pytest.raises(RuntimeError):
        cache.attend(x, x.detach(), x.detach(), table, table, torch.zeros(1, dtype=torch.long, device=gpu_device))


@pytest.mark.parametrize("rows,vocab", [(3, 30001), (40, 28000), (70, 40000), (130, 28003)])
def test_rows_that_workgroups_share_captured_and_replayed(gpu_device, rows, vocab):
    """Every replay is another draw from other logits, and the same as an eager call's; eager calls of other sizes lie between them."""
    gen = torch.Generator(device=gpu_device).manual_seed(rows)
    logits, uniform = torch.zeros((rows, vocab), device=gpu_device, dtype=torch.float16), torch.zeros(rows, device=gpu_device)
    options = dict(temperature=torch.full((rows,), 0.8, device=gpu_device), top_k=torch.full((rows,), 300, dtype=torch.int32, device=gpu_device),
                   top_p=torch.full((rows,), 0.9, device=gpu_device), min_p=torch.full((rows,), 1e-3, device=gpu_device))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        sample(logits, uniform, **options)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ids, logprob = sample(logits, uniform, **options)
    drawn = []
    for _ in range(4):
        logits.copy_(torch.randn((rows, vocab), generator=gen, device=gpu_device) * 3)
        uniform.copy_(torch.rand(rows, generator=gen, device=gpu_device))
        graph.replay()
        torch.cuda.synchronize()
        want = sample(logits, uniform, **options)
        sample(logits[:1, :200].contiguous(), uniform[:1])
        assert torch.equal(ids, want[0]) and torch.equal(logprob, want[1])
        drawn.append(ids.clone())
    assert not torch.equal(drawn[0], drawn[1])


def test_two_streams_at_once(gpu_device):
    """Two caches, two vocabularies, two banks, each on a stream of its own and all at once: as one after the other."""
    def work(seed):
        gen = torch.Generator(device=gpu_device).manual_seed(seed)
        normal = lambda *s: torch.randn(s, generator=gen, device=gpu_device).half()
        cache = Q4Cache(2, 2, 4096, 64, gpu_device)
        k, v = normal(2, 3000, 128), normal(2, 3000, 128)
        angle = torch.rand((4096, 64), generator=gen, device=gpu_device)
        cos, sin = angle.cos().half(), angle.sin().half()
        start = torch.zeros(2, dtype=torch.long, device=gpu_device)
        cache.attend(normal(2, 3000, 256), k, v, cos, sin, start)
        bank = AdapterBank.from_tensors(normal(5, 16, 256) / 16, normal(5, 64, 16))
        q, x, base, logits = normal(2, 256), normal(300, 256), normal(300, 64), normal(4, 30000)
        ids = torch.randint(-1, 5, (300,), generator=gen, device=gpu_device, dtype=torch.int32)
        uniform = torch.rand(4, generator=gen, device=gpu_device)
        return lambda: (cache.attend(q, k[:, 0], v[:, 0], cos, sin, start + 3000), bank(x, ids, base), *sample(logits, uniform, 0.7, 50, 0.95, 0.01))
    jobs = [work(1), work(2)]
    want = [job() for job in jobs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (job, stream) in enumerate(zip(jobs, streams)):
            with torch.cuda.stream(stream):
                got[i].append(job())
    torch.cuda.synchronize()
    for results, right in zip(got, want):
        for result in results:
            assert all(torch.equal(a, b) for a, b in zip(result, right))
