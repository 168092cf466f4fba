"""A decoder that serves: its cache in 4 bits, adapters beside its linears, tokens drawn from its logits, alone and together."""
import math

import pytest
import torch
import torch.nn.functional as F

import oracle as orc
from shiftaddllm_amd import decode
from shiftaddllm_amd.lut_gemm.adapters import AdapterBank
from shiftaddllm_amd.sampling import SamplingOptions, sample
from test_gpu_q4_attention import rotated

pytestmark = pytest.mark.gpu

CFG = decode.DecoderConfig(vocab_size=512, hidden=512, intermediate=1024, layers=3, heads=8, kv_heads=2, max_positions=96)


def fill_adapters(model, seed):
    gen = torch.Generator(device=model.logits.device).manual_seed(seed)
    for blk in model.blocks:
        for l in blk.linears():
            bank = l.adapters
            bank.down.copy_(torch.randn(bank.down.shape, generator=gen, device=bank.down.device) / math.sqrt(bank.K))
            bank.up.copy_(torch.randn(bank.up.shape, generator=gen, device=bank.up.device) * 0.02)
            bank.scale.copy_(0.5 + torch.rand(bank.count, generator=gen, device=bank.scale.device))


def close(a, b, rel=5e-3, mad=2e-2):
    """Two fp16 networks with differently rounded glue: the bar of the other decoder tests."""
    r, m = orc.error_metrics(a.float().cpu().numpy().reshape(-1, a.shape[-1]), b.float().cpu().numpy().reshape(-1, b.shape[-1]))
    assert r <= rel and m <= mad, (r, m)


def reference(m, ids, positions):
    """Logits of one token per sequence over the same LutLinear layers, attention in fp32 over what the model's caches hold after it took the
    token; sequences at negative positions get anything.

    The held values are taken from the cache because holding is not continuous: two networks whose keys differ in their last bits may choose
    neighbouring codes for a number halfway between, a step of a 15th of the group's range apart, which no bar for differently rounded
    networks counts.  That each value lies within half a step of the reference's own number is asserted here, that codes are the nearest
    ones exactly by the tests of the cache."""
    cfg = m.cfg
    hd, H, KV, B = cfg.head_dim, cfg.heads, cfg.kv_heads, m.batch
    adapters = m.adapter_ids if m.has_adapters else None
    x = m.embed[ids]
    at = torch.tensor([max(p, 0) for p in positions], device=x.device)
    for li, blk in enumerate(m.blocks):
        h = decode.rms_norm(x, blk.input_norm, cfg.rms_eps)
        q, k, v = (l(h, adapters) for l in (blk.q_proj, blk.k_proj, blk.v_proj))
        q, k = (rotated(t.view(B, -1, hd), m.cos[at], m.sin[at]) for t in (q, k))
        att = torch.zeros((B, H, hd), device=x.device)
        for b, p in enumerate(positions):
            if p < 0:
                continue
            kk, vv = m.q4[li].values(b, p + 1)                      # [p + 1, KV, hd]
            for cached, own in ((kk[p], k[b]), (vv[p], v[b].view(KV, hd))):
                own = own.float().unflatten(-1, (-1, 32))
                span = own.amax(-1, keepdim=True) - own.amin(-1, keepdim=True)
                # half a step, and the networks' difference: the bar below, of the group's largest number
                off = span / 30 * 1.01 + 2e-2 * own.abs().amax(-1, keepdim=True)
                assert bool(((cached.float().unflatten(-1, (-1, 32)) - own).abs() <= off).all())
            kk, vv = (t.float().repeat_interleave(H // KV, 1).transpose(0, 1).contiguous() for t in (kk, vv))
            w = torch.softmax(torch.matmul(kk, q[b].float().unsqueeze(-1)).squeeze(-1) / math.sqrt(hd), -1)
            att[b] = torch.matmul(w.unsqueeze(1), vv).squeeze(1)
        x = x + blk.o_proj(att.half().view(B, -1), adapters)
        h = decode.rms_norm(x, blk.post_norm, cfg.rms_eps)
        x = x + blk.down_proj(F.silu(blk.gate_proj(h, adapters)) * blk.up_proj(h, adapters), adapters)
    return decode.rms_norm(x, m.final_norm, cfg.rms_eps) @ m.lm_head.t()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_linear_with_adapters(gpu_device, dtype):
    gen = torch.Generator(device=gpu_device).manual_seed(1)
    lin = decode.random_lut_linear(256, 384, 3, 128, gen, gpu_device)
    bias = torch.randn(384, generator=gen, device=gpu_device)
    lin.bias = bias
    lin.adapters = AdapterBank(256, 384, 12, 3).to(gpu_device)
    for a in range(3):
        lin.adapters.set(a, torch.randn((12, 256), generator=gen, device=gpu_device) / 16, torch.randn((384, 12), generator=gen, device=gpu_device) / 4, 0.5 + a)
    for shape in ((5, 256), (2, 3, 256), (1, 256), (40, 256)):
        x = torch.randn(shape, generator=gen, device=gpu_device).to(dtype)
        rows = x.numel() // 256
        ids = torch.tensor([i % 4 - 1 for i in range(rows)], device=gpu_device)
        got = lin(x, ids.view(shape[:-1]))
        assert got.dtype is dtype and got.shape == (*shape[:-1], 384)
        plain, bank = lin(x.half()), lin.adapters
        want = plain.reshape(rows, 384).double()
        xs = x.half().reshape(rows, 256).double()
        for r, a in enumerate(ids.tolist()):
            if a >= 0:
                want[r] += bank.scale[a].double() * (bank.up[a].double() @ (bank.down[a].double() @ xs[r]))
        # the result rounds to fp16 (2^-11) and then to the caller's type; sums in fp32 are far below
        bound = want.abs() * (2.0 ** -10 + (2.0 ** -8 if dtype is torch.bfloat16 else 0)) + 1e-4
        assert bool(((got.reshape(rows, 384).double() - want).abs() <= bound).all())
        assert torch.equal(lin(x, torch.full_like(ids, -1)), plain.to(dtype))
    lin.adapters = None
    with pytest.raises(ValueError):
        lin(x, ids)
    lin.adapters = AdapterBank(256, 256, 8, 1).to(gpu_device)
    with pytest.raises(ValueError):
        lin(x, ids)


@pytest.mark.parametrize("batch", [1, 3])
def test_a_cache_of_four_bits(gpu_device, batch):
    """Captured steps, and a prompt at once, against the reference over what the caches hold."""
    model = decode.LutDecoder(CFG, None, batch=batch, seed=3, device=gpu_device, kv_bits=4)
    ids = torch.randint(0, CFG.vocab_size, (batch, 9), generator=torch.Generator().manual_seed(2)).to(gpu_device)
    model.capture()
    model.reset()
    with torch.no_grad():
        for t in range(9):
            logits = model.forward_token(ids[:, t], t)
            close(logits, reference(model, ids[:, t], [t] * batch))
        model.reset()
        logits = model.prefill(ids[:, :8])
        for t in range(7):                                            # (the keys and values of every token of the prompt)
            reference(model, ids[:, t], [t] * batch)
        close(logits, reference(model, ids[:, 7], [7] * batch))
        close(model.forward_token(ids[:, 8], 8), reference(model, ids[:, 8], [8] * batch))


def test_sequences_at_unlike_positions(gpu_device):
    """Four sequences that came at different times, one slot idle; chunks of prompts that follow one another."""
    B = 4
    model = decode.LutDecoder(CFG, None, batch=B, seed=4, device=gpu_device, kv_bits=4)
    ids = torch.randint(0, CFG.vocab_size, (B, 16), generator=torch.Generator().manual_seed(5)).to(gpu_device)
    lengths, live = [7, 0, 3, 11], [0, 2, 3]
    pick = lambda n: ids[torch.arange(B), torch.tensor(n)]
    with torch.no_grad():
        before = model.logits.fill_(3.0).clone()
        first = model.prefill(ids, lengths)
        close(first[live], reference(model, pick([6, 0, 2, 10]), [6, -1, 2, 10])[live])
        assert torch.equal(first[1], before[1])
        logits = model.forward_token(pick(lengths), [7, -1, 3, 11]).clone()
        close(logits[live], reference(model, pick(lengths), [7, -1, 3, 11])[live])
        assert bool((model.att[1] == 0).all())
        model.capture()
        again = model.forward_token(pick(lengths), torch.tensor([7, -1, 3, 11]))
        assert torch.equal(again[live], logits[live])
        more = model.prefill(ids[:, 12:], [2, 4, 3, 1], [8, 0, 4, 12])
        close(more, reference(model, pick([13, 15, 14, 12]), [9, 3, 6, 12]))
    for bad in ([0, 1, 2], [0, 1, 2, CFG.max_positions]):
        with pytest.raises(ValueError):
            model.forward_token(ids[:, 0], bad)


@pytest.mark.parametrize("batch,fuse", [(1, True), (5, True), (3, False)])
def test_adapters_beside_all_linears(gpu_device, batch, fuse):
    """The fused step with adapters against the step of framework operations; ids that change between replays."""
    ids = torch.randint(0, CFG.vocab_size, (batch, 6), generator=torch.Generator().manual_seed(7)).to(gpu_device)
    out = {}
    for glue in ("hip", "torch"):
        model = decode.LutDecoder(CFG, None, batch=batch, seed=6, device=gpu_device, glue=glue, adapters=(3, 12), fuse_launches=fuse)
        fill_adapters(model, 8)
        if glue == "hip":
            model.capture()
        model.reset()
        seq = []
        for t in range(6):
            model.adapter_ids.copy_(torch.tensor([(b + t // 2) % 4 - 1 for b in range(batch)], dtype=torch.int32))
            seq.append(model.forward_token(ids[:, t], t).clone())
        out[glue] = torch.stack(seq)
    close(out["hip"], out["torch"])
    plain = decode.LutDecoder(CFG, None, batch=batch, seed=6, device=gpu_device, fuse_launches=fuse)
    first = plain.forward_token(ids[:, 0], 0)
    none = decode.LutDecoder(CFG, None, batch=batch, seed=6, device=gpu_device, adapters=(3, 12), fuse_launches=fuse)
    close(none.forward_token(ids[:, 0], 0), first)


def test_drawn_tokens(gpu_device):
    """A captured step draws what sample() draws from its logits; temperature 0 is the argmax; a seed repeats its tokens."""
    B = 4
    model = decode.LutDecoder(CFG, None, batch=B, seed=9, device=gpu_device, sampling=SamplingOptions(0.9, 50, 0.95, 0.01))
    model.capture()
    gen = torch.Generator(device=gpu_device).manual_seed(1)
    ids = torch.randint(0, CFG.vocab_size, (B,), generator=gen, device=gpu_device)
    for t in range(5):
        if t == 3:
            model.sample_temperature.copy_(torch.tensor([0.0, 1.5, 0.7, 1.0]))
            model.sample_top_k.copy_(torch.tensor([0, 3, 0, 1], dtype=torch.int32))
        model.uniform.copy_(torch.rand(B, generator=gen, device=gpu_device))
        logits = model.forward_token(ids, t)
        want, lp = sample(logits, model.uniform, model.sample_temperature, model.sample_top_k, model.sample_top_p, model.sample_min_p)
        assert torch.equal(model.next_ids, want) and torch.equal(model.next_logprob, lp)
        if t >= 3:
            assert int(want[0]) == int(logits[0].argmax()) and int(want[3]) == int(logits[3].argmax())
        ids = want
    prompt = torch.randint(0, CFG.vocab_size, (B, 4), generator=torch.Generator().manual_seed(3))
    runs = []
    for seed in (1, 1, 2):
        m = decode.LutDecoder(CFG, None, batch=B, seed=9, device=gpu_device, sampling=SamplingOptions(seed=seed))
        m.capture()
        runs.append(decode.benchmark(m, prompt, generate=12, warmup=2)["generated"])
    assert torch.equal(runs[0], runs[1]) and not torch.equal(runs[0], runs[2])
    greedy = decode.LutDecoder(CFG, None, batch=B, seed=9, device=gpu_device)
    greedy.capture()
    cold = decode.LutDecoder(CFG, None, batch=B, seed=9, device=gpu_device, sampling=SamplingOptions(temperature=0.0))
    cold.capture()
    assert torch.equal(decode.benchmark(cold, prompt, generate=12, warmup=2)["generated"], decode.benchmark(greedy, prompt, generate=12, warmup=2)["generated"])


@pytest.mark.parametrize("batch", [2, 6])
def test_all_of_it_together(gpu_device, batch):
    """Requests with adapters of their own: prompts at once, then captured steps that draw their tokens from a cache of 4 bits; every step's
    logits against the reference fed with the same tokens, two captured decoders replayed in turn."""
    models = []
    for seed in (11, 12):
        m = decode.LutDecoder(CFG, None, batch=batch, seed=seed, device=gpu_device, kv_bits=4, adapters=(4, 8), sampling=SamplingOptions(0.8, 40, 0.95, 0.0, seed))
        fill_adapters(m, seed)
        m.adapter_ids.copy_(torch.tensor([b % 5 - 1 for b in range(batch)], dtype=torch.int32))
        m.capture()
        m.reset()
        models.append(m)
    gen = torch.Generator(device=gpu_device).manual_seed(13)
    prompt = torch.randint(0, CFG.vocab_size, (batch, 8), generator=gen, device=gpu_device)
    lengths = [8 - b for b in range(batch)]
    last = []
    with torch.no_grad():
        for m in models:
            logits = m.prefill(prompt, lengths)
            tokens = prompt[torch.arange(batch), torch.tensor(lengths) - 1]
            close(logits, reference(m, tokens, [n - 1 for n in lengths]))
            last.append(sample(logits, torch.rand(batch, generator=gen, device=gpu_device), 0.8, 40)[0])
        positions = list(lengths)
        for step in range(5):
            if step == 2:
                positions[1] = -1                                     # a request that has ended
            live = [b for b in range(batch) if positions[b] >= 0]
            for i, m in enumerate(models):
                m.uniform.copy_(torch.rand(batch, generator=gen, device=gpu_device))
                logits = m.forward_token(last[i], positions)
                close(logits[live], reference(m, last[i], positions)[live])
                want, lp = sample(logits, m.uniform, 0.8, 40, 0.95)
                assert torch.equal(m.next_ids, want) and torch.equal(m.next_logprob, lp)
                last[i] = m.next_ids.clone()
            positions = [p + 1 if p >= 0 else p for p in positions]
