"""What attention over a 4-bit cache, token sampling and adapters refuse, without a GPU: every call below fails on the host, before
anything is launched."""
import ctypes
import os

import pytest
import torch

E_INVAL, E_ALIGN = -1, -2
BASE = 0x100000


@pytest.fixture(scope="module")
def lib():
    from shiftaddllm_amd import native
    if not os.path.exists(native.KERNEL_LIB):
        from shiftaddllm_amd import build
        build.build_kernel_library()
    return native.cabi()


def attention(**kw):
    from shiftaddllm_amd import native
    f = dict(cache=BASE, q=BASE, k=BASE, v=BASE, cos_table=BASE, sin_table=BASE, start=BASE, counts=None, out=BASE, k_held=None, v_held=None,
             q_stride=(512, 512), k_stride=(256, 256), v_stride=(256, 256), batch=2, tokens=1, heads=4, kv_heads=2, head_dim=128, max_positions=64)
    f.update(kw)
    for n in ("q_stride", "k_stride", "v_stride"):
        f[n] = (ctypes.c_int64 * 2)(*f[n])
    return native.Q4Attention(**f)


def test_cache_sizes(lib):
    assert lib.lutgemm_q4_cache_bytes(2, 3, 64, 128) == 2 * 3 * 2 * 40 * 128
    assert lib.lutgemm_q4_cache_bytes(1, 1, 65, 32) == 3 * 40 * 32
    assert lib.lutgemm_q4_cache_bytes(64, 64, 1 << 20, 256) == 64 * 64 * 32768 * 40 * 256        # beyond 32 bits
    for bad in ((0, 1, 1, 32), (1, 0, 1, 32), (1, 1, 0, 32), (1, 1, 1, 48), (1, 1, 1, 288), (1, 1, 1, 0), (1, 1, (1 << 20) + 1, 32), (-1, 1, 1, 32),
                (65536, 1, 1, 32), (1, 4097, 1, 32)):
        assert lib.lutgemm_q4_cache_bytes(*bad) == 0


def test_attention_refuses(lib):
    call = lambda ws=None, size=0, **kw: lib.lutgemm_q4_attention_f16(ctypes.byref(attention(**kw)), ws, size, None)
    assert lib.lutgemm_q4_attention_f16(None, None, 0, None) == E_INVAL
    for name in ("cache", "q", "k", "v", "cos_table", "sin_table", "start", "out"):
        assert call(**{name: None}) == E_INVAL, name
    for kw in (dict(batch=0), dict(tokens=0), dict(tokens=65537), dict(heads=3), dict(heads=1), dict(kv_heads=0), dict(head_dim=100), dict(head_dim=264),
               dict(max_positions=0), dict(max_positions=(1 << 20) + 1), dict(heads=8192), dict(q_stride=(-8, 0)), dict(k_stride=(0, -8)),
               dict(batch=65535, heads=4096, kv_heads=4096, tokens=65536)):
        assert call(**kw) == E_INVAL, kw
    for name in ("cache", "q", "k", "v", "cos_table", "sin_table", "out", "k_held", "v_held"):
        assert call(**{name: BASE + 8}) == E_ALIGN, name
    assert call(start=BASE + 4) == E_ALIGN and call(counts=BASE + 2) == E_ALIGN
    for name in ("q_stride", "k_stride", "v_stride"):
        assert call(**{name: (4, 512)}) == E_ALIGN and call(**{name: (512, 12)}) == E_ALIGN


def test_attention_refuses_a_workspace_that_is_short(lib):
    sizes = dict(batch=1, tokens=1, heads=4, kv_heads=1, head_dim=128, max_positions=100000)
    need = lib.lutgemm_q4_attention_workspace(*sizes.values())
    assert need > 0
    for ws, size in ((None, 0), (BASE, need - 1), (None, need)):
        assert lib.lutgemm_q4_attention_f16(ctypes.byref(attention(**sizes)), ws, size, None) == E_INVAL
    assert lib.lutgemm_q4_attention_f16(ctypes.byref(attention(**sizes)), BASE + 8, need, None) == E_ALIGN
    assert lib.lutgemm_q4_attention_workspace(1, 1, 3, 2, 128, 100000) == 0


def test_attention_plans(lib):
    from shiftaddllm_amd import native
    plan = native.Q4AttentionPlan()
    describe = lambda *a: lib.lutgemm_describe_q4_attention_plan(*a, ctypes.byref(plan))
    assert lib.lutgemm_describe_q4_attention_plan(1, 1, 4, 2, 128, 64, None) == E_INVAL
    assert describe(1, 1, 4, 3, 128, 64) == E_INVAL and describe(1, 1, 4, 2, 120, 64) == E_INVAL
    for B, T, H, KV, hd, P in ((1, 1, 32, 32, 128, 256), (24, 1, 32, 8, 128, 4096), (2, 1, 64, 8, 128, 131072), (2, 2048, 32, 8, 128, 2048), (5, 37, 12, 2, 64, 8192),
                               (1, 1, 1, 1, 32, 1), (1, 65536, 8, 8, 64, 1 << 20), (300, 3, 71, 1, 256, 999)):
        assert describe(B, T, H, KV, hd, P) == 0
        rows = T * (H // KV)
        tile = plan.rows_per_wave * (plan.threads // 64 if plan.rows_apart else 1)
        assert plan.rows_per_wave % 16 == 0 and (plan.row_tiles - 1) * tile < rows <= plan.row_tiles * tile
        assert plan.workgroups == B * KV * plan.row_tiles * plan.splits
        need = lib.lutgemm_q4_attention_workspace(B, T, H, KV, hd, P)
        assert (need > 0) == (plan.splits > 1) and need >= (plan.splits * B * H * T * (hd + 2) * 4 if plan.splits > 1 else 0)


def sampling(**kw):
    from shiftaddllm_amd import native
    f = dict(logits=BASE, row_stride=1000, logits_type=0, rows=4, vocab=1000, temperature=None, top_k=None, top_p=None, min_p=None, uniform=BASE,
             ids=BASE, logprob=None)
    f.update(kw)
    return native.Sampling(**f)


def test_sampling_refuses(lib):
    need = lib.lutgemm_sampling_workspace(4, 1000)
    assert need > 0 and lib.lutgemm_sampling_workspace(0, 10) == 0 and lib.lutgemm_sampling_workspace(1, (1 << 20) + 1) == 0
    call = lambda ws=BASE, size=need, **kw: lib.lutgemm_sample_tokens(ctypes.byref(sampling(**kw)), ws, size, None)
    assert lib.lutgemm_sample_tokens(None, BASE, need, None) == E_INVAL
    for kw in (dict(logits=None), dict(uniform=None), dict(ids=None), dict(rows=0), dict(rows=65536), dict(vocab=0), dict(vocab=(1 << 20) + 1),
               dict(logits_type=3), dict(logits_type=-1), dict(row_stride=-1000), dict(ws=None), dict(size=need - 1)):
        assert call(**kw) == E_INVAL, kw
    for kw in (dict(logits=BASE + 1), dict(logits=BASE + 2, logits_type=2), dict(ids=BASE + 4), dict(logprob=BASE + 2), dict(uniform=BASE + 1),
               dict(temperature=BASE + 2), dict(top_k=BASE + 2), dict(top_p=BASE + 2), dict(min_p=BASE + 2), dict(ws=BASE + 8)):
        assert call(**kw) == E_ALIGN, kw


def adapters(**kw):
    from shiftaddllm_amd import native
    f = dict(x_f16=BASE, base_f16=BASE + 0x10000, out_f16=BASE + 0x20000, ids=BASE + 0x30000, down_f16=BASE + 0x40000, up_f16=BASE + 0x50000,
             scale=None, x_stride=64, base_stride=32, out_stride=32, M=3, N=32, K=64, rank=8, adapters=2)
    f.update(kw)
    return native.Adapters(**f)


def test_adapters_refuse(lib):
    from shiftaddllm_amd import native

    def call(*problems, ws=BASE + 0x60000, size=1 << 20):
        arr = (native.Adapters * max(len(problems), 1))(*problems)
        rc = lib.lutgemm_adapters_f16(len(problems), arr, ws, size, None)
        assert lib.lutgemm_adapters_workspace(len(problems), arr) == 0 or ws is None or size < 1 << 20 or ws % 16
        return rc
    one = lambda **kw: call(adapters(**kw))
    assert lib.lutgemm_adapters_f16(1, None, BASE, 1 << 20, None) == E_INVAL and call() == E_INVAL
    assert call(*[adapters(out_f16=BASE + 0x100000 + 0x1000 * i) for i in range(9)]) == E_INVAL
    for name in ("x_f16", "base_f16", "out_f16", "ids", "down_f16", "up_f16"):
        assert one(**{name: None}) == E_INVAL, name
    for kw in (dict(M=0), dict(M=65536), dict(N=0), dict(N=30), dict(K=48), dict(K=0), dict(rank=0), dict(rank=12), dict(rank=264), dict(adapters=0),
               dict(adapters=65536), dict(x_stride=-64), dict(base_stride=-32), dict(out_stride=28), dict(out_stride=0),
               dict(out_f16=BASE + 0x10000, out_stride=36)):
        assert one(**kw) == E_INVAL, kw
    for kw in (dict(x_f16=BASE + 8), dict(base_f16=BASE + 0x10004), dict(out_f16=BASE + 0x20004), dict(ids=BASE + 0x30002), dict(down_f16=BASE + 0x40008),
               dict(up_f16=BASE + 0x50008), dict(scale=BASE + 0x70002), dict(x_stride=68), dict(base_stride=34), dict(out_stride=34)):
        assert one(**kw) == E_ALIGN, kw
    # what is written overlaps what is read or written
    for kw in (dict(out_f16=BASE + 0x10000 + 8), dict(out_f16=BASE), dict(out_f16=BASE + 0x30000), dict(out_f16=BASE + 0x40000), dict(out_f16=BASE + 0x50000),
               dict(scale=BASE + 0x20000)):
        assert one(**kw) == E_INVAL, kw
    assert call(adapters(), adapters()) == E_INVAL                                                    # two write the same rows
    assert call(adapters(), adapters(x_f16=BASE + 0x20000, out_f16=BASE + 0x80000)) == E_INVAL         # one reads what the other writes
    assert call(adapters(), ws=None) == E_INVAL and call(adapters(), ws=BASE + 0x60008) == E_ALIGN
    need = lib.lutgemm_adapters_workspace(1, ctypes.byref(adapters()))
    assert need >= 3 * 8 * 4 and call(adapters(), size=need - 1) == E_INVAL


def test_python_checks():
    from shiftaddllm_amd import native
    from shiftaddllm_amd.kv_cache import Q4Cache
    from shiftaddllm_amd.lut_gemm.adapters import AdapterBank
    from shiftaddllm_amd.sampling import sample
    if not os.path.exists(native.TORCH_EXT):
        pytest.skip("torch extension not built (python -m shiftaddllm_amd.build)")
    with pytest.raises(ValueError):
        Q4Cache(1, 1, 10, 100, "cpu")
    with pytest.raises(ValueError):
        Q4Cache(1, 2, 10, 64, "cpu", torch.zeros((1, 2, 1, 40 * 32), dtype=torch.uint8))
    cache = Q4Cache(1, 2, 40, 64, "cpu")
    assert cache.data.shape == (1, 2, 2, 2560)
    with pytest.raises(ValueError):
        cache.values(0, 41)
    x = torch.zeros((1, 128), dtype=torch.float16)
    with pytest.raises(RuntimeError, match="GPU"):
        cache.attend(x, x, x, x, x, torch.zeros(1, dtype=torch.long))
    with pytest.raises(RuntimeError, match="GPU"):
        sample(torch.zeros((1, 8)), torch.zeros(1))
    bank = AdapterBank(64, 32, 5, 3)
    assert bank.down.shape == (3, 8, 64) and bank.up.shape == (3, 32, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        bank(torch.zeros((2, 64), dtype=torch.float16), torch.zeros(2, dtype=torch.int32), torch.zeros((2, 32), dtype=torch.float16))
    for bad in ((60, 32, 8, 1), (64, 30, 8, 1), (64, 32, 0, 1), (64, 32, 257, 1), (64, 32, 8, 0)):
        with pytest.raises(ValueError):
            AdapterBank(*bad)
    with pytest.raises(IndexError):
        bank.set(3, torch.zeros(8, 64), torch.zeros(32, 8))
    with pytest.raises(ValueError):
        bank.set(0, torch.zeros(9, 64), torch.zeros(32, 9))
    with pytest.raises(ValueError):
        AdapterBank.from_tensors(torch.zeros(2, 4, 64), torch.zeros(2, 32, 5))


def test_values_follow_the_stated_layout():
    """Codes and scales put where the layout says, read back as numbers."""
    from shiftaddllm_amd.kv_cache import Q4Cache
    hd, G, P = 96, 3, 70
    cache = Q4Cache(1, 1, P, hd, "cpu")
    gen = torch.Generator().manual_seed(1)
    cache.data.copy_(torch.randint(0, 256, cache.data.shape, generator=gen, dtype=torch.uint8))
    half = cache.data.view(torch.float16).view(3, -1)
    for first in (256 * G, 576 * G):
        half[:, first:first + 64 * G] = torch.randn((3, 64 * G), generator=gen).half()
    k, v = cache.values(0, P)
    words = cache.data.view(torch.int32).view(3, -1)
    bits = lambda w, e: int(w) >> (4 * (e // 2) + 16 * (e % 2)) & 15
    for p, d in ((0, 0), (5, 33), (31, 95), (32, 64), (50, 17), (69, 40), (63, 7)):
        b, i, g = p // 32, p % 32, d // 32
        code = bits(words[b, i * 4 * G + d % 32 // 8 * G + g], d % 8)
        scale, low = half[b, 256 * G + (i * G + g) * 2: 256 * G + (i * G + g) * 2 + 2].float()
        assert k[p, 0, d] == (low + scale * code).half()
        quad, e = i % 16 // 4, i % 4 + 4 * (i // 16)
        code = bits(words[b, 160 * G + (quad * 16 + d % 16) * 2 * G + d // 16], e)
        scale, low = half[b, 576 * G + g * 64 + quad * 8 + e].float(), half[b, 576 * G + g * 64 + 32 + quad * 8 + e].float()
        assert v[p, 0, d] == (low + scale * code).half()


def test_decoder_refuses():
    from shiftaddllm_amd import decode
    cfg = decode.DecoderConfig(vocab_size=32, hidden=128, intermediate=128, layers=1, heads=2, kv_heads=1, max_positions=8)
    make = lambda **kw: decode.LutDecoder(cfg, None, device="cpu", **kw)
    for kw in (dict(kv_bits=8), dict(kv_bits=4, glue="torch"), dict(kv_bits=4, chain=True), dict(adapters=(2, 8), chain=True), dict(adapters=(2, 0))):
        with pytest.raises(ValueError):
            make(**kw)
    with pytest.raises(ValueError):       # heads of 48 numbers
        decode.LutDecoder(decode.DecoderConfig(vocab_size=32, hidden=96, intermediate=128, layers=1, heads=2, kv_heads=1, max_positions=8, group_size=32),
                          None, device="cpu", kv_bits=4)
    plain, q4 = make(), make(kv_bits=4, batch=2)
    ids = torch.zeros((1, 2), dtype=torch.long)
    with pytest.raises(ValueError):
        plain.prefill(ids)
    with pytest.raises(ValueError):
        plain.forward_token(ids[:, 0], [0])
    for position in ([0], [0, 8], [0, 1, 2]):
        with pytest.raises(ValueError):
            q4.forward_token(torch.zeros(2, dtype=torch.long), position)
    two = torch.zeros((2, 4), dtype=torch.long)
    for kw in (dict(lengths=[4]), dict(lengths=[5, 1]), dict(lengths=[4, -1]), dict(starts=[5, 0]), dict(starts=[-1, 0]), dict(starts=[0])):
        with pytest.raises(ValueError):
            q4.prefill(two, **kw)
    with pytest.raises(ValueError):
        q4.prefill(ids)
    assert hasattr(plain, "k_cache") and not hasattr(q4, "k_cache") and q4.q4[0].data.shape == (2, 1, 1, 40 * 64)


def test_linear_layers_keep_their_state():
    """A layer without adapters has the state it had; with them, the bank's buffers beside its own."""
    from shiftaddllm_amd.lut_gemm.adapters import AdapterBank
    from shiftaddllm_amd.lut_gemm.quant import LutLinear
    lin = LutLinear(64, 32, group_size=32)
    assert sorted(lin.state_dict()) == ["alpha", "binaryWeight"] and lin.adapters is None
    with pytest.raises(ValueError):
        lin(torch.zeros((1, 64)), torch.zeros(1, dtype=torch.int32))
    lin.adapters = AdapterBank(64, 32, 8, 2)
    assert sorted(lin.state_dict()) == ["adapters.down", "adapters.scale", "adapters.up", "alpha", "binaryWeight"]


def test_attention_refuses_outputs_that_overlap(lib):
    """What a call writes may not lie in anything else that it is given, nor in what it writes besides."""
    place = {n: BASE + i * (1 << 20) for i, n in enumerate(("cache", "q", "k", "v", "cos_table", "sin_table", "start", "counts", "out", "k_held", "v_held"))}
    call = lambda **kw: lib.lutgemm_q4_attention_f16(ctypes.byref(attention(**{**place, **kw})), None, 0, None)
    size = dict(cache=2 * 2 * 2 * 40 * 128, out=2 * 512 * 2, k_held=2 * 256 * 2, v_held=2 * 256 * 2)
    for name, bytes_ in size.items():
        for other in place:
            if other == name:
                continue
            assert call(**{name: place[other]}) == E_INVAL, (name, other)
            assert call(**{other: place[name] + bytes_ - 16}) == E_INVAL, (name, other)
