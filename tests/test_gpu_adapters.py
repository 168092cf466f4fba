"""Low-rank adapters beside a shared projection against 64 bits: rows of one adapter, of many, of none, in any order."""
import ctypes
import math

import pytest
import torch

from shiftaddllm_amd import native
from shiftaddllm_amd.lut_gemm.adapters import AdapterBank

pytestmark = pytest.mark.gpu


def make(gen, M, K, N, rank, count, device):
    n = lambda *s: torch.randn(s, generator=gen, device=device)
    return n(M, K).half(), n(M, N).half(), (n(count, rank, K) / math.sqrt(K)).half(), (n(count, N, rank) * 0.3).half(), 0.25 + torch.rand((count,), generator=gen, device=device)


def expected(x, ids, base, down, up, scale):
    """(out, bound) in 64 bits."""
    out = base.double().clone()
    bound = torch.zeros_like(out)
    K, rank = x.shape[1], down.shape[1]
    for a in sorted(set(ids)):
        if not 0 <= a < down.shape[0]:
            continue
        at = torch.tensor([i for i, v in enumerate(ids) if v == a], device=x.device)
        h = x[at].double() @ down[a].double().t()
        size = x[at].double().abs() @ down[a].double().abs().t()
        out[at] += scale[a].double() * (h @ up[a].double().t())
        # h: exact products, sums in fp32 of at most K steps; up: its rows times h, rank steps more and the scale.  Each step 2^-24 of
        # what is summed.
        bound[at] = scale[a].double() * (size @ up[a].double().abs().t()) * (K + rank + 4) * 2.0 ** -24
    return out, bound + out.abs() * 2.0 ** -11 + base.double().abs() * 2.0 ** -24 + 2.0 ** -25


def check(bank, x, ids, base, down, up, scale, out=None):
    t = torch.tensor(ids, dtype=torch.int32, device=x.device)
    got = bank(x, t, base, out)
    want, bound = expected(x, ids, base, down, up, scale)
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"off by {float((off / bound).max()):.3g} of the bound"
    for i, a in enumerate(ids):
        if not 0 <= a < down.shape[0]:
            assert torch.equal(got[i], base[i])
    return got


@pytest.mark.parametrize("M,K,N,rank,count", [(1, 4096, 4096, 16, 3), (1, 32, 4, 8, 1), (2, 96, 20, 4, 2), (5, 11008, 512, 8, 4), (17, 256, 1028, 64, 6),
                                              (33, 4128, 260, 24, 33), (64, 512, 11008, 128, 5), (100, 1024, 1024, 256, 3), (300, 544, 772, 16, 7),
                                              (1000, 2048, 516, 32, 5), (3, 8192, 96, 1, 2)])
def test_rows_through_their_adapters(gpu_device, M, K, N, rank, count):
    gen = torch.Generator(device=gpu_device).manual_seed(M * 31 + K)
    x, base, down, up, scale = make(gen, M, K, N, rank, count, gpu_device)
    bank = AdapterBank.from_tensors(down, up, scale)
    rnd = torch.Generator().manual_seed(M)
    for ids in ([i % count for i in range(M)], torch.randint(-1, count, (M,), generator=rnd).tolist(), [i * count // M for i in range(M)],
                [count - 1] * M, [-1] * M, torch.randint(-3, 2 * count + 1, (M,), generator=rnd).tolist(), [-2 ** 31 if i % 2 else 2 ** 31 - 1 for i in range(M)]):
        check(bank, x, ids, base, down, up, scale)


def test_base_in_place_and_rows_apart(gpu_device):
    gen = torch.Generator(device=gpu_device).manual_seed(2)
    M, K, N, count = 7, 160, 52, 3
    x, base, down, up, scale = make(gen, M, K, N, 8, count, gpu_device)
    bank = AdapterBank.from_tensors(down, up, scale)
    ids = [0, 2, -1, 1, 1, 0, 2]
    want = check(bank, x, ids, base, down, up, scale)
    own = base.clone()
    assert check(bank, x, ids, base, down, up, scale, out=torch.empty_like(base)).equal(want)
    bank(x, torch.tensor(ids, dtype=torch.int32, device=gpu_device), own, own)
    assert torch.equal(own, want)
    wide_x = torch.randn((M, K + 24), generator=gen, device=gpu_device).half()
    wide_x[:, 8:8 + K] = x
    wide = torch.full((M, N + 12), 5.0, dtype=torch.float16, device=gpu_device)
    wide_base = wide.clone()
    wide_base[:, 4:4 + N] = base
    got = check(bank, wide_x[:, 8:8 + K], ids, wide_base[:, 4:4 + N], down, up, scale, out=wide[:, 4:4 + N])
    assert torch.equal(got, want) and bool((wide[:, :4] == 5).all()) and bool((wide[:, 4 + N:] == 5).all())
    assert torch.equal(check(bank, x, ids, base[:1].expand(M, N), down, up, scale)[0], want[0])         # one row of base for all
    odd = wide_x.flatten()[1:1 + M * K].view(M, K)                                                      # off alignment: copied
    check(bank, odd, ids, base, down, up, scale)
    deep = bank(x.view(7, 1, K), torch.tensor(ids, dtype=torch.int32, device=gpu_device), base.view(7, 1, N))
    assert deep.shape == (7, 1, N) and torch.equal(deep.view(M, N), want)


def test_values_that_are_not_finite_stay_in_their_rows(gpu_device):
    gen = torch.Generator(device=gpu_device).manual_seed(3)
    for M in (5, 200):
        x, base, down, up, scale = make(gen, M, 256, 128, 16, 4, gpu_device)
        bank = AdapterBank.from_tensors(down, up, scale)
        ids = torch.tensor([i % 4 - (i % 5 == 0) for i in range(M)], dtype=torch.int32, device=gpu_device)
        want = bank(x, ids, base)
        x2, b2 = x.clone(), base.clone()
        x2[1, 7], x2[3, 9], b2[4, 5] = float("nan"), float("inf"), float("inf")
        got = bank(x2, ids, b2)
        assert bool(torch.isnan(got[1]).all()) and not bool(torch.isfinite(got[3]).any()) and got[4, 5] == float("inf")
        keep = [i for i in range(M) if i not in (1, 3, 4)]
        assert torch.equal(got[keep], want[keep])
        # an adapter that is not finite: its rows only
        bad = AdapterBank.from_tensors(down, up, scale)
        bad.down[2, 3, 4] = float("nan")
        got = bad(x, ids, base)
        mine = ids == 2
        assert bool(torch.isnan(got[mine]).all()) and torch.equal(got[~mine], want[~mine])


def test_large_sums_stay_in_32_bits(gpu_device):
    """h far beyond fp16's range, brought back by small `up`."""
    gen = torch.Generator(device=gpu_device).manual_seed(4)
    for M in (2, 150):
        x, base, down, up, scale = make(gen, M, 1024, 64, 8, 2, gpu_device)
        x, down, up = x * 100, (down.float() * 900).half(), (up.float() * 2e-4).half()
        check(AdapterBank.from_tensors(down, up, scale), x, [i % 2 for i in range(M)], base, down, up, scale)


def test_adapters_set_one_by_one(gpu_device):
    gen = torch.Generator(device=gpu_device).manual_seed(5)
    x, base, down, up, scale = make(gen, 6, 128, 64, 12, 3, gpu_device)
    bank = AdapterBank(128, 64, 12, 3).to(gpu_device)
    ids = [0, 1, 2, 0, -1, 2]
    assert torch.equal(bank(x, torch.tensor(ids, dtype=torch.int32, device=gpu_device), base), base)
    for a in range(3):
        bank.set(a, down[a], up[a], float(scale[a]))
    check(bank, x, ids, base, down, up, scale)
    bank.set(1, down[0, :5], up[0, :, :5], 0.5)                      # a lower rank in the same place: nothing of the old one stays
    down[1], up[1] = 0, 0
    down[1, :5], up[1, :, :5], scale[1] = down[0, :5], up[0, :, :5], 0.5
    check(bank, x, ids, base, down, up, scale)


def _problem(x, ids, base, out, bank, M):
    return native.Adapters(x.data_ptr(), base.data_ptr(), out.data_ptr(), ids.data_ptr(), bank.down.data_ptr(), bank.up.data_ptr(),
                           bank.scale.data_ptr(), bank.K, bank.N, bank.N, M, bank.N, bank.K, bank.rank, bank.count)


@pytest.mark.parametrize("M", [1, 6, 90])
def test_projections_that_share_a_call(gpu_device, M):
    """q, k, v and another: unlike widths and ranks, the bits of calls of their own; captured and replayed for other rows."""
    lib = native.cabi()
    gen = torch.Generator(device=gpu_device).manual_seed(M)
    K = 512
    x = torch.randn((M, K), generator=gen, device=gpu_device).half()
    ids = torch.tensor([i % 4 - 1 for i in range(M)], dtype=torch.int32, device=gpu_device)
    banks, bases, outs = [], [], []
    for N, rank in ((512, 16), (128, 16), (132, 8), (1024, 40)):
        _, base, down, up, scale = make(gen, M, K, N, rank, 3, gpu_device)
        banks.append(AdapterBank.from_tensors(down, up, scale))
        bases.append(base)
        outs.append(torch.zeros_like(base))
    arr = (native.Adapters * 4)(*[_problem(x, ids, b, o, bank, M) for bank, b, o in zip(banks, bases, outs)])
    size = lib.lutgemm_adapters_workspace(4, arr)
    ws = torch.empty(size, dtype=torch.uint8, device=gpu_device)

    def call():
        sp = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        assert lib.lutgemm_adapters_f16(4, arr, ws.data_ptr(), size, sp) == 0
    call()
    for bank, b, o in zip(banks, bases, outs):
        assert torch.equal(o, bank(x, ids, b))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        call()
    for i in range(3):
        x.copy_(torch.randn((M, K), generator=gen, device=gpu_device))
        ids.copy_(torch.randint(-1, 3, (M,), generator=gen, device=gpu_device))
        ws.fill_(255)
        g.replay()
        torch.cuda.synchronize()
        for bank, b, o in zip(banks, bases, outs):
            assert torch.equal(o, bank(x, ids, b))
