"""Choosing tokens against the rules worked out in 64 bits: filters alone and together, ties, equal logits, infinities, empty rows."""
import math

import numpy as np
import pytest
import torch

from shiftaddllm_amd.sampling import sample

pytestmark = pytest.mark.gpu


def expected(logits, u, t=1.0, k=0, p=1.0, m=0.0):
    """(id, logprob) of one row by the definition, numpy float64."""
    x = logits.double().cpu().numpy()
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.argsort(-x, kind="stable")
    top = x[order[0]]
    if top == -np.inf:
        return -1, -math.inf
    if not t > 0:
        return int(order[0]), 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / t) if top < np.inf else 0.0)
    w = np.where(x[order] == -np.inf, 0.0, w)
    n = len(w)
    if k > 0:
        n = min(n, k)
    cum = np.cumsum(w[:n])
    if p < 1:
        n = min(n, int(np.searchsorted(cum, max(p, 0.0) * cum[-1], side="left")) + 1)
    if m > 0:
        n = min(n, int((w >= min(m, 1.0)).sum()))
    u = u if u > 0 else 0.0
    at = int(np.searchsorted(cum[:n], min(u, 1 - 2.0 ** -24) * cum[n - 1], side="right"))
    return int(order[at]), float(np.log(w[at] / cum[n - 1]))


def check(logits, u, t=None, k=None, p=None, m=None):
    R, dev = logits.shape[0], logits.device
    as_rows = lambda v, d: None if v is None else torch.tensor(v, dtype=d, device=dev) if isinstance(v, (list, tuple)) else torch.full((R,), v, dtype=d, device=dev)
    t, p, m, u = (as_rows(v, torch.float32) for v in (t, p, m, u))
    k = as_rows(k, torch.int32)
    ids, lp = sample(logits, u, t, k, p, m)
    assert ids.dtype is torch.int64 and lp.dtype is torch.float32
    pick = lambda v, r, off: off if v is None else float(v[r])
    for r in range(R):
        want, wlp = expected(logits[r], float(u[r]), pick(t, r, 1.0), int(pick(k, r, 0)), pick(p, r, 1.0), pick(m, r, 0.0))
        assert int(ids[r]) == want, f"row {r}: {int(ids[r])} for {want}"
        # the share is held to 2^-40 or so; its logarithm is rounded to fp32
        assert float(lp[r]) == wlp or abs(float(lp[r]) - wlp) <= abs(wlp) * 2.0 ** -24 + 2.0 ** -36, (r, float(lp[r]), wlp)
    return ids, lp


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,V", [(1, 1), (3, 7), (5, 1000), (4, 32000), (2, 50272), (9, 4097)])
def test_filters(gpu_device, R, V, dtype):
    gen = torch.Generator(device=gpu_device).manual_seed(R * 7 + V)
    logits = torch.randn((R, V), generator=gen, device=gpu_device) * 2.5
    logits[:, ::max(V // 50, 1)] += 5
    logits = logits.to(dtype)
    for i, (t, k, p, m) in enumerate([(None,) * 4, (0.7, None, None, None), (1.0, 40, None, None), (1.3, None, 0.9, None), (1.0, None, None, 0.05),
                                      (0.8, 50, 0.95, 0.02), (1.0, 1, None, None), (1.0, None, 0.0, None), (1.0, None, None, 1.0), (0.0, 5, 0.5, 0.1),
                                      (0.25, 3, 0.999, 0.0), (2.0, V, 1.0, 1e-9), (5.0, 0, 0.5, 0.0), (1.0, V - 1, 0.99999, None), (1e-30, None, None, None)]):
        check(logits, torch.rand(R, generator=gen, device=gpu_device).tolist(), t, k, p, m)
        check(logits, [(0.0, 1 - 2.0 ** -24, 0.5)[(r + i) % 3] for r in range(R)], t, k, p, m)


def test_rows_ask_for_unlike_things(gpu_device):
    gen = torch.Generator(device=gpu_device).manual_seed(3)
    R, V = 40, 3001
    logits = (torch.randn((R, V), generator=gen, device=gpu_device) * 3).half()
    cycle = lambda values: [values[r % len(values)] for r in range(R)]
    check(logits, torch.rand(R, generator=gen, device=gpu_device).tolist(), cycle([1.0, 0.0, 0.5, 1.7, float("nan"), -1.0, 1e9]),
          cycle([0, 1, 5, -3, 100, 4000]), cycle([1.0, 0.5, 0.9, 2.0, float("nan"), -1.0, 0.0]), cycle([0.0, 0.1, float("nan"), -2.0, 0.5, 7.0, 1e-5, 0.3, 0.01]))


@pytest.mark.parametrize("V", [64, 1500, 5000, 70000])
def test_equal_logits(gpu_device, V):
    """Ties go by index, in steps of any size: all equal, two values, a few values many times over, values of both signs of zero."""
    rows = [torch.full((V,), 2.5), torch.where(torch.arange(V) % 3 == 0, 1.0, 0.5), (torch.arange(V) * 7 % 5).float() / 4,
            torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0), torch.full((V,), -65504.0), (torch.arange(V) * 31 % 11).float() * 1e-6]
    for dtype in (torch.float16, torch.float32):
        logits = torch.stack(rows).to(dtype).to(gpu_device)
        for u in (0.0, 0.25, 0.5, 0.73, 1 - 2.0 ** -24):
            check(logits, u)
            check(logits, u, k=V // 2)
            check(logits, u, p=0.5)
            check(logits, u, 1.0, V // 3, 0.25, 0.5)
            check(logits, u, 0.0)


def test_infinities_and_empty_rows(gpu_device):
    inf, nan = float("inf"), float("nan")
    V = 300
    rows = torch.randn((9, V), generator=torch.Generator().manual_seed(4))
    rows[0] = -inf
    rows[1] = nan
    rows[2, 5:] = -inf
    rows[3, 17] = inf
    rows[4, 17] = rows[4, 200] = rows[4, 201] = inf
    rows[5, ::2] = nan
    rows[6] = -inf
    rows[6, 250] = -3e38
    rows[7, :-1] = -inf
    rows[8] = inf
    logits = rows.to(gpu_device)
    for u in (0.0, 0.4, 0.99):
        for t in (1.0, 0.0, 0.3, inf, 1e-38):
            for k, p, m in ((None, None, None), (2, None, None), (None, 0.6, None), (4, 0.9, 0.1)):
                check(logits, u, t, k, p, m)
    ids, lp = check(logits, 0.5)
    assert ids[0] == -1 and lp[0] == -inf and ids[1] == -1 and ids[3] == 17 and ids[7] == V - 1
    check(logits, [nan, -1.0, 1.0, 2.0, 0.3, nan, 1.0, 0.0, 1.0])


def test_an_endless_temperature_takes_all_logits_alike(gpu_device):
    gen = torch.Generator(device=gpu_device).manual_seed(5)
    logits = torch.randn((3, 9000), generator=gen, device=gpu_device)
    logits[1, ::3] = float("-inf")
    logits[2] = logits[2].round()
    for u in (0.0, 0.3, 0.9):
        for k, p in ((None, None), (5000, None), (None, 0.3), (1, None)):
            check(logits, u, float("inf"), k, p)


def test_rows_apart_and_room_around(gpu_device):
    """Rows of a larger tensor, starting off any alignment; a given row broadcast; a transposed tensor is copied."""
    gen = torch.Generator(device=gpu_device).manual_seed(6)
    for dtype in (torch.float16, torch.float32):
        big = (torch.randn((5, 3, 1013), generator=gen, device=gpu_device) * 3).to(dtype)
        view = big[:, -1, 3:1004]
        u = torch.rand(5, generator=gen, device=gpu_device).tolist()
        check(view, u, 0.9, 30, 0.9, 0.01)
        poisoned = big.clone()
        poisoned[:] = float("inf")
        poisoned[:, -1, 3:1004] = view
        a, b = sample(view, torch.tensor(u, device=gpu_device)), sample(poisoned[:, -1, 3:1004], torch.tensor(u, device=gpu_device))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        check(view[:1].expand(5, -1), u)
        check(view.t().contiguous().t(), u)


def test_numbers_for_all_rows(gpu_device):
    gen = torch.Generator(device=gpu_device).manual_seed(7)
    logits = torch.randn((4, 500), generator=gen, device=gpu_device).half()
    u = torch.rand(4, generator=gen, device=gpu_device)
    a = sample(logits, u, 0.8, 20, 0.9, 0.01)
    full = lambda v, d=torch.float32: torch.full((4,), v, dtype=d, device=gpu_device)
    b = sample(logits, u, full(0.8), full(20, torch.int32), full(0.9), full(0.01))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_shares_of_draws(gpu_device):
    """Numbers spread evenly over [0, 1) give every token its share of the draws, to one draw on either side."""
    V, R = 50, 20000
    logits = torch.randn((1, V), generator=torch.Generator().manual_seed(8)).to(gpu_device)
    u = ((torch.arange(R, device=gpu_device).double() + 0.5) / R).float()
    ids, _ = sample(logits.expand(R, V), u)
    share = torch.bincount(ids, minlength=V).double() / R
    assert float((share - torch.softmax(logits[0].double(), -1)).abs().max()) <= 1.5 / R


def test_captured_and_replayed(gpu_device):
    gen = torch.Generator(device=gpu_device).manual_seed(9)
    R, V = 3, 20000
    logits, u, t = torch.zeros((R, V), dtype=torch.float16, device=gpu_device), torch.zeros(R, device=gpu_device), torch.ones(R, device=gpu_device)
    k, p = torch.full((R,), 50, dtype=torch.int32, device=gpu_device), torch.full((R,), 0.9, device=gpu_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sample(logits, u, t, k, p)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            res = sample(logits, u, t, k, p)
        graphs.append((g, res))
    for i in range(4):
        logits.copy_(torch.randn((R, V), generator=gen, device=gpu_device) * 3)
        u.copy_(torch.rand(R, generator=gen, device=gpu_device))
        k.fill_((50, 0, 3, 1)[i])
        eager = sample(logits, u, t, k, p)
        for g, res in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, res in graphs:
            assert torch.equal(res[0], eager[0]) and torch.equal(res[1], eager[1])
        check(logits, u.tolist(), 1.0, int(k[0]), 0.9)


def test_many_rows_on_two_streams(gpu_device):
    gen = torch.Generator(device=gpu_device).manual_seed(10)
    logits = (torch.randn((300, 6000), generator=gen, device=gpu_device) * 3).half()
    u = torch.rand(300, generator=gen, device=gpu_device)
    want = sample(logits, u, 0.9, 100, 0.95)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            results.append(sample(logits, u, torch.full((300,), 0.9, device=gpu_device), torch.full((300,), 100, dtype=torch.int32, device=gpu_device),
                                  torch.full((300,), 0.95, device=gpu_device)))
    torch.cuda.synchronize()
    for ids, lp in results:
        assert torch.equal(ids, want[0]) and torch.equal(lp, want[1])
