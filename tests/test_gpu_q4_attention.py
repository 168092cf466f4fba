"""Attention over a cache held in 4 bits against its definition in 64 bits: appending, single tokens, several and prompts, sequences
that stand anywhere or are idle, and what lies in places that nobody attends to."""
import math

import pytest
import torch

from shiftaddllm_amd.kv_cache import Q4Cache

pytestmark = pytest.mark.gpu


def tables(P, hd, device):
    ang = torch.arange(P, device=device).double()[:, None] / 10000.0 ** (torch.arange(0, hd, 2, device=device).double() / hd)
    return tuple(torch.cat([f(ang)] * 2, -1).half() for f in (torch.cos, torch.sin))


def rotated(x, cos, sin):
    """x [T, heads, hd], rotated in fp32 (products of fp16 numbers are exact there) and rounded to fp16."""
    h = x.shape[-1] // 2
    x, c, s = x.float(), cos.float()[:, None], sin.float()[:, None]
    return (x * c + torch.cat([-x[..., h:], x[..., :h]], -1) * s).half()


def held(x):
    """What groups of 32 along the last dimension are held as, by the definition, in 64 bits."""
    x = torch.nan_to_num(x.double(), nan=0.0, posinf=60000.0, neginf=-60000.0).clamp(-60000, 60000).unflatten(-1, (-1, 32))
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((high - low) / 15).float().half().double()
    code = torch.where(scale > 0, torch.round((x - low) / torch.where(scale > 0, scale, 1.0)), 0.0).clamp(0, 15)
    return (low + scale * code).float().half().flatten(-2)


class Model:
    """The definition, kept as lists of held keys and values per sequence."""

    def __init__(self, B, KV, P, hd, device):
        self.k = torch.zeros((B, P, KV, hd), dtype=torch.float16, device=device)
        self.v = torch.zeros_like(self.k)
        self.cos, self.sin = tables(P, hd, device)

    def attend(self, q, k, v, starts, counts):
        """(out, error bound, k_held, v_held) in 64 bits."""
        B, T, KV, hd, P = q.shape[0], q.shape[1], self.k.shape[2], self.k.shape[3], self.k.shape[1]
        H = q.shape[2] // hd
        out = torch.zeros((B, T, H, hd), dtype=torch.float64, device=q.device)
        bound = torch.zeros_like(out)
        kh, vh = (torch.zeros((B, T, KV * hd), dtype=torch.float16, device=q.device) for _ in range(2))
        for b in range(B):
            start, n = starts[b], min(counts[b], T)
            if start < 0 or start >= P or n <= 0:
                continue
            n = min(n, P - start)
            at = slice(start, start + n)
            qr = rotated(q[b, :n].view(n, H, hd), self.cos[at], self.sin[at]).double()
            self.k[b, at] = held(rotated(k[b, :n].view(n, KV, hd), self.cos[at], self.sin[at]))
            self.v[b, at] = held(v[b, :n].view(n, KV, hd))
            kh[b, :n], vh[b, :n] = self.k[b, at].flatten(1), self.v[b, at].flatten(1)
            kk, vv = (x[b, :start + n].double().repeat_interleave(H // KV, 1).transpose(0, 1) for x in (self.k, self.v))   # [H, L, hd]
            s = qr.transpose(0, 1) @ kk.transpose(1, 2).contiguous() / math.sqrt(hd)
            size = (qr.transpose(0, 1).abs() @ kk.transpose(1, 2).abs().contiguous() / math.sqrt(hd)).amax(-1, keepdim=True)
            late = torch.arange(start + n, device=q.device)[None] > torch.arange(start, start + n, device=q.device)[:, None]
            p = torch.softmax(s.masked_fill(late, float("-inf")), -1)
            o, spread = p @ vv, p @ vv.abs()
            # weights and the result round to fp16: 2^-11 of |p v| and of the result.  Weights below 2^-14 of the largest: 2^-25 each.
            # Scores: sums of hd exact products in fp32 (2^-24 of what they are made of for each of at most hd steps), the scale's
            # factor and the exponential (another 2^-22 of the score each); a weight is off by as much, relatively, twice (its sum).
            # The sums over positions: 2^-24 a step and a joint, well below 2^-13 at these lengths; 2^-24: results near zero in fp16.
            off = spread * (2.0 ** -11 + 2.0 ** -13 + 2 * size * (hd * 2.0 ** -24 + 2.0 ** -21)) + o.abs() * 2.0 ** -11 + \
                (start + n) * 2.0 ** -25 * vv.abs().amax(1, keepdim=True) + 2.0 ** -24
            out[b, :n], bound[b, :n] = o.transpose(0, 1), off.transpose(0, 1)
        return out.flatten(2), bound.flatten(2), kh, vh


def make(gen, B, T, H, KV, hd, device):
    n = lambda *s: torch.randn(s, generator=gen, device=device)
    return (n(B, T, H * hd) * 1.5).half(), (n(B, T, KV * hd) * (0.3 + torch.rand((KV * hd,), generator=gen, device=device))).half(), n(B, T, KV * hd).half()


def check(cache, model, q, k, v, starts, counts=None, **kw):
    device = q.device
    start = torch.tensor(starts, device=device)
    count = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=device)
    out, kh, vh = cache.attend(q, k, v, model.cos, model.sin, start, count, held=True, **kw)
    want, bound, kw_, vw = model.attend(q, k, v, starts, counts or [q.shape[1]] * q.shape[0])
    assert torch.equal(kh, kw_) and torch.equal(vh, vw)
    off = (out.double() - want).abs()
    assert bool((off <= bound).all()), f"off by {float((off / bound.clamp_min(1e-30)).max()):.3g} of the bound"
    for b, s in enumerate(starts):
        if s >= 0:
            n = min(s + (counts[b] if counts else q.shape[1]), cache.max_positions)
            ck, cv = cache.values(b, n)
            assert torch.equal(ck, model.k[b, :n]) and torch.equal(cv, model.v[b, :n])
    return out


@pytest.mark.parametrize("B,H,KV,hd,P,steps", [
    (1, 32, 32, 128, 256, ((250,), (5, 1))),
    (2, 8, 2, 64, 100, ((31, 31), (1, 1), (1, 1), (32, 1))),            # either side of a block of 32
    (3, 6, 3, 96, 70, ((1, 40, 69), (1, 1, 1))),
    (2, 5, 1, 256, 90, ((64, 3), (2, 1))),
    (2, 16, 1, 32, 40, ((7, 8), (1, 1), (1, 1))),
    (1, 24, 1, 160, 130, ((128,), (1,))),                               # more query heads than one tile of rows
    (2, 3, 1, 224, 35, ((33, 2), (1, 1))),
    (2, 2, 2, 192, 35, ((33, 2), (1, 1))),
    (1, 1, 1, 128, 1, ((1,),)),                                         # a cache of one position
])
def test_prompts_and_tokens_that_follow(gpu_device, B, H, KV, hd, P, steps):
    """Prompts and single tokens one after another, counts differing, memory that held NaN everywhere before."""
    gen = torch.Generator(device=gpu_device).manual_seed(hd * 7 + P)
    data = torch.full((B, KV, -(-P // 32), 40 * hd), 255, dtype=torch.uint8, device=gpu_device)
    cache, model = Q4Cache(B, KV, P, hd, gpu_device, data), Model(B, KV, P, hd, gpu_device)
    at = [0] * B
    for counts in steps:
        counts = (list(counts) * B)[:B]
        T = max(counts)
        check(cache, model, *make(gen, B, T, H, KV, hd, gpu_device), at, counts)
        at = [a + c for a, c in zip(at, counts)]


@pytest.mark.parametrize("B,H,KV,hd,P,T", [(4, 8, 2, 128, 3000, 1), (3, 12, 2, 64, 2100, 5), (2, 8, 8, 128, 1500, 40), (2, 4, 2, 96, 700, 300),
                                           (1, 32, 1, 128, 600, 64), (1, 2, 1, 256, 9000, 1), (1, 7, 1, 128, 9000, 30)])
def test_sequences_anywhere(gpu_device, B, H, KV, hd, P, T):
    """Caches that hold earlier positions, sequences at unlike ones, one idle, one at the end, one with fewer tokens."""
    gen = torch.Generator(device=gpu_device).manual_seed(P + T)
    cache, model = Q4Cache(B, KV, P, hd, gpu_device), Model(B, KV, P, hd, gpu_device)
    fill = P - T
    check(cache, model, *make(gen, B, fill, H, KV, hd, gpu_device), [0] * B)
    for starts in ([fill] * B, [17] * B, [fill, -1, 0, fill // 2][:B], [-5, 31, 32, 64][:B], [fill // 3, P - 1, P, P + 7][:B]):
        check(cache, model, *make(gen, B, T, H, KV, hd, gpu_device), starts)
        check(cache, model, *make(gen, B, T, H, KV, hd, gpu_device), starts, [T, T // 2, 0, T + 3][:B])


def test_positions_nobody_attends_to(gpu_device):
    """NaN and infinities in scales behind the newest position, and in q, k, v, rows that are passed over."""
    B, H, KV, hd, P = 2, 4, 2, 64, 96
    gen = torch.Generator(device=gpu_device).manual_seed(5)
    cache, model = Q4Cache(B, KV, P, hd, gpu_device), Model(B, KV, P, hd, gpu_device)
    q, k, v = make(gen, B, 40, H, KV, hd, gpu_device)
    check(cache, model, q, k, v, [0, 0], [40, 37])
    half = cache.data.view(torch.float16).view(B, KV, 3, -1)
    G = hd // 32
    half[:, :, 2] = float("nan")                                                     # a block that no position is in
    half[0, :, 1, 256 * G:320 * G].view(KV, 32, G, 2)[:, 9:] = float("inf")          # keys of positions 41 ..
    half[0, :, 1, 576 * G:640 * G].view(KV, G, 2, 4, 2, 4)[:, :, :, 2:, 0, 1:] = float("nan")   # values of positions 32 + 9 .. 11, 13 .. 15
    half[0, :, 1, 576 * G:640 * G].view(KV, G, 2, 4, 2, 4)[:, :, :, 3, 0] = float("-inf")
    half[0, :, 1, 576 * G:640 * G].view(KV, G, 2, 4, 2, 4)[..., 1, :] = float("inf")  # ... and 48 ..
    q, k, v = make(gen, B, 3, H, KV, hd, gpu_device)
    q[0, 1:], k[0, 1:], v[0, 1:] = float("nan"), float("inf"), float("nan")
    check(cache, model, q, k, v, [40, 37], [1, 3])


def test_numbers_that_are_not_finite_are_held_as_finite_ones(gpu_device):
    B, H, KV, hd, P = 1, 2, 1, 64, 64
    cache, model = Q4Cache(B, KV, P, hd, gpu_device), Model(B, KV, P, hd, gpu_device)
    gen = torch.Generator(device=gpu_device).manual_seed(6)
    q, k, v = make(gen, B, 6, H, KV, hd, gpu_device)
    v[0, 0, 3], v[0, 1, 5], v[0, 2, 40], v[0, 3, :32] = float("nan"), float("inf"), float("-inf"), 65504.0
    v[0, 4], v[0, 5, ::2], v[0, 5, 1::2] = 0.25, 60000.0, -60000.0
    start = torch.zeros(1, dtype=torch.long, device=gpu_device)
    out, kh, vh = cache.attend(q, k, v, model.cos, model.sin, start, held=True)
    assert torch.equal(vh, held(v.view(1, 6, 1, hd)).flatten(2)) and bool(torch.isfinite(vh).all()) and bool((vh[0, 4] == 0.25).all())
    assert bool(torch.isfinite(out).all())
    # a query that is not finite spoils its own row and no other
    q[0, 2, :hd] = float("nan")
    again = cache.attend(q, k, v, model.cos, model.sin, start)
    assert bool(torch.isnan(again[0, 2, :hd]).all())
    again[0, 2, :hd] = out[0, 2, :hd]
    assert torch.equal(again, out)


def test_codes_next_to_halves(gpu_device):
    """Groups whose numbers lie halfway between codes, or a step beside: ties to even, and no error of a quotient decides."""
    B, KV, hd, P = 1, 4, 64, 320
    gen = torch.Generator(device=gpu_device).manual_seed(8)
    s = torch.randint(1, 200, (P, KV * hd // 32, 1), generator=gen, device=gpu_device).float() / 256
    x = torch.randint(0, 31, (P, KV * hd // 32, 32), generator=gen, device=gpu_device) / 2 * s
    x[..., 0], x[..., 1] = 0, 15 * s[..., 0]
    bits = x.half().view(torch.int16) + torch.randint(-1, 2, x.shape, generator=gen, device=gpu_device).short() * (x > 0) * (x < 15 * s)
    v = (bits.view(torch.float16).flatten(1) * torch.randint(0, 2, (P, 1), generator=gen, device=gpu_device).mul(2).sub(1).half()).view(1, P, KV * hd)
    cache = Q4Cache(B, KV, P, hd, gpu_device)
    cos, sin = tables(P, hd, gpu_device)
    _, _, vh = cache.attend(v, v, v, cos, sin, torch.zeros(1, dtype=torch.long, device=gpu_device), held=True)
    assert torch.equal(vh.view(P, KV, hd), held(v.view(P, KV, hd)))


def test_strided_operands_and_outputs_of_the_caller(gpu_device):
    """q, k, v as parts of one projection, rows apart; an output given; room behind output and cache stays as it was."""
    B, T, H, KV, hd, P = 3, 4, 6, 2, 64, 50
    gen = torch.Generator(device=gpu_device).manual_seed(9)
    both = torch.randn((B, T + 2, (H + 2 * KV) * hd + 8), generator=gen, device=gpu_device).half()
    q, k, v = both[:, 1:T + 1, :H * hd], both[:, 1:T + 1, H * hd:(H + KV) * hd], both[:, 1:T + 1, (H + KV) * hd:(H + 2 * KV) * hd]
    memory = torch.full((B * KV * 2 * 40 * hd + 256,), 77, dtype=torch.uint8, device=gpu_device)
    cache = Q4Cache(B, KV, P, hd, gpu_device, memory[:-256].view(B, KV, 2, 40 * hd))
    model = Model(B, KV, P, hd, gpu_device)
    room = torch.full((B * T * H * hd + 64,), 3.0, dtype=torch.float16, device=gpu_device)
    out = check(cache, model, q, k, v, [0, 0, 0], [4, 3, 2], out=room[:-64].view(B, T, H * hd))
    assert out.data_ptr() == room.data_ptr() and bool((room[-64:] == 3.0).all()) and bool((memory[-256:] == 77).all())
    odd = both.flatten()[1:1 + B * H * hd].view(B, H * hd)                      # off 16-byte alignment: copied
    single = cache.attend(odd, k[:, 0], v[:, 0], model.cos, model.sin, torch.tensor([4, 3, 2], device=gpu_device))
    assert single.shape == (B, H * hd)
    same = cache.attend(odd.clone().unsqueeze(1), k[:, :1], v[:, :1], model.cos, model.sin, torch.tensor([4, 3, 2], device=gpu_device))
    assert torch.equal(single, same[:, 0])


def test_only_the_new_positions_of_a_cache_are_written(gpu_device):
    B, H, KV, hd, P = 2, 4, 2, 128, 200
    gen = torch.Generator(device=gpu_device).manual_seed(10)
    cache, model = Q4Cache(B, KV, P, hd, gpu_device), Model(B, KV, P, hd, gpu_device)
    check(cache, model, *make(gen, B, P, H, KV, hd, gpu_device), [0, 0])
    before = [cache.values(b, P) for b in range(B)]
    check(cache, model, *make(gen, B, 3, H, KV, hd, gpu_device), [30, 95], [3, 2])
    for b, (lo, hi) in enumerate(((30, 33), (95, 97))):
        for x, y in zip(before[b], cache.values(b, P)):
            assert torch.equal(x[:lo], y[:lo]) and torch.equal(x[hi:], y[hi:])


@pytest.mark.parametrize("T", [1, 6])
def test_captured_and_replayed_at_other_positions(gpu_device, T):
    """Two captured steps share nothing; each is replayed at positions, counts and queries other than the captured ones, with eager
    work between."""
    B, H, KV, hd, P = 3, 8, 2, 128, 2100
    gen = torch.Generator(device=gpu_device).manual_seed(11)
    both = []
    for _ in range(2):
        cache, model = Q4Cache(B, KV, P, hd, gpu_device), Model(B, KV, P, hd, gpu_device)
        check(cache, model, *make(gen, B, P - T, H, KV, hd, gpu_device), [0] * B)
        q, k, v = make(gen, B, T, H, KV, hd, gpu_device)
        start, counts = torch.zeros(B, dtype=torch.long, device=gpu_device), torch.full((B,), T, dtype=torch.int32, device=gpu_device)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            cache.attend(q, k, v, model.cos, model.sin, start, counts)
        model.attend(q, k, v, [0] * B, [T] * B)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = cache.attend(q, k, v, model.cos, model.sin, start, counts)
        both.append((cache, model, q, k, v, start, counts, graph, out))
    for starts, n in (([5, 2000, 64], [T] * 3), ([P - T, -1, 0], [T, T, 1]), ([100, 200, P - 1], [1, T, T])):
        for cache, model, q, k, v, start, counts, graph, out in both:
            for x, fresh in zip((q, k, v), make(gen, B, T, H, KV, hd, gpu_device)):
                x.copy_(fresh)
            start.copy_(torch.tensor(starts))
            counts.copy_(torch.tensor(n, dtype=torch.int32))
        for _, _, _, _, _, _, _, graph, _ in both:
            graph.replay()
        torch.cuda.synchronize()
        for cache, model, q, k, v, start, counts, graph, out in both:
            want, bound, _, _ = model.attend(q, k, v, starts, n)
            assert bool(((out.double() - want).abs() <= bound).all())
            eager = cache.attend(q, k, v, model.cos, model.sin, start, counts)
            assert torch.equal(eager, out)


def test_results_do_not_change_from_run_to_run(gpu_device):
    B, H, KV, hd, P = 2, 8, 2, 128, 5000
    gen = torch.Generator(device=gpu_device).manual_seed(12)
    cache, model = Q4Cache(B, KV, P, hd, gpu_device), Model(B, KV, P, hd, gpu_device)
    q, k, v = make(gen, B, P, H, KV, hd, gpu_device)
    start = torch.zeros(B, dtype=torch.long, device=gpu_device)
    first = cache.attend(q, k, v, model.cos, model.sin, start)
    at = torch.full((B,), P - 1, device=gpu_device)
    one = cache.attend(q[:, -1], k[:, -1], v[:, -1], model.cos, model.sin, at)
    for _ in range(5):
        assert torch.equal(cache.attend(q, k, v, model.cos, model.sin, start), first)
        assert torch.equal(cache.attend(q[:, -1], k[:, -1], v[:, -1], model.cos, model.sin, at), one)


def test_offsets_beyond_32_bits(gpu_device):
    """A cache of more than 4 GB: its last sequence, at its end."""
    B, H, KV, hd, P = 14, 8, 8, 128, 1 << 18
    gen = torch.Generator(device=gpu_device).manual_seed(13)
    cache = Q4Cache(B, KV, P, hd, gpu_device)
    assert cache.data.numel() > 1 << 32
    cos, sin = tables(1 << 18, hd, gpu_device)
    q, k, v = make(gen, B, 20, H, KV, hd, gpu_device)
    start = torch.full((B,), P - 20, device=gpu_device)
    cache.attend(q, k, v, cos, sin, start)
    model = Model(1, KV, 64, hd, gpu_device)
    # earlier positions hold zeros: their scores are 0 and their values 0, P - 20 of them beside the new ones
    model.cos, model.sin = cos[P - 20:], sin[P - 20:]
    at = start + 19
    out = cache.attend(q[:, 19], k[:, 19], v[:, 19], cos, sin, at).double()
    kk, vv = held(rotated(k[-1].view(20, KV, hd), model.cos, model.sin)).double(), held(v[-1].view(20, KV, hd)).double()
    qr = rotated(q[-1, 19:].view(1, H, hd), cos[P - 1:], sin[P - 1:]).double()[0]
    w = torch.exp((qr[None] * kk).sum(-1) / math.sqrt(hd))                       # [20, H]
    total = w.sum(0) + (P - 20)
    want = (w[..., None] * vv).sum(0) / total[:, None]
    bound = (w[..., None] * vv.abs()).sum(0) / total[:, None] * (2.0 ** -10 + 2.0 ** -12) + 2.0 ** -24
    assert bool(((out[-1].view(H, hd) - want).abs() <= bound).all())
