"""What a decoded token goes through besides the quantised products, as cases that can be timed: attention over a
cache held in 4 bits, choosing the next token from its logits, and low-rank adapters beside a shared projection.

A case is a dict of plain values:
  op "attend":  one call for `batch` sequences of `tokens` new tokens each, `heads` query heads on `kv_heads`, over a
                cache of `max_positions` positions; `spread` draws where each sequence stands ("full": at the end of
                the cache, "ragged": anywhere, some sequences idle or with fewer new tokens than others).
  op "sample":  `rows` rows of `vocab` logits of `dtype`; `filters` says which of the filters are set.
  op "adapt":   `rows` rows through one of `count` adapters of `rank` each, beside a K -> N projection; `order` says
                how rows and adapters meet ("own": every request another, "runs": prompts one after another, "mixed").

`own` chooses between the plain form of each operator (elementary torch operations) and this package's kernels.

The cache: groups of 32 values along the head share a scale and a minimum in fp16, a value is fp16(minimum + scale *
code).  32 positions of a kv head lie together, 40 * head_dim bytes: the key codes, their scales, the value codes, their scales.
With G = head_dim / 32, a 32-bit word holds eight codes e = 0..7, the even ones in its low half from bit 0 up, the odd ones in
its high half:
  key codes     [32 positions][4 quads][G]      word: dimensions 32 t + 8 quad + e of group t
  key scales    [32 positions][G][scale, minimum]
  value codes   [4 quads][16][2 G]              word [quad][c][t]: dimension 16 t + c of positions 4 quad + e (e < 4), 16 + 4 quad + e - 4
  value scales  [G][scale, minimum][4 quads][8] in the same order of positions
"""
import math
import random

import torch

own = False
DEVICE = "cuda:0"
GROUP = 32
LARGEST = 60000.0


def _attend(name, batch, tokens, heads, kv_heads, head_dim, max_positions, spread, seed):
    return {"name": name, "op": "attend", "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "max_positions": max_positions, "spread": spread, "lengths": seed}


def _sample(name, rows, vocab, dtype, filters):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "filters": filters}


def _adapt(name, rows, K, N, rank, count, order, seed):
    return {"name": name, "op": "adapt", "rows": rows, "K": K, "N": N, "rank": rank, "count": count, "order": order, "ids": seed}


def listed():
    return [
        # the decode benchmark's geometry: one sequence at the end of its 256 positions
        _attend("attend, one sequence, 256 positions", 1, 1, 32, 32, 128, 256, "full", 1),
        # a server's step: sequences of all lengths, some slots idle
        _attend("attend, 24 sequences of mixed lengths", 24, 1, 32, 8, 128, 4096, "ragged", 2),
        # two long documents being answered
        _attend("attend, two sequences of 131072", 2, 1, 64, 8, 128, 131072, "full", 3),
        # prompts of up to 2048 tokens, from an empty cache
        _attend("attend, two prompts of 2048", 2, 2048, 32, 8, 128, 2048, "full", 4),
        # a few tokens at once onto caches in use (chunks of prompts, drafted tokens)
        _attend("attend, chunks of 37 onto 8192", 5, 37, 12, 2, 64, 8192, "ragged", 5),
        # one user's next token
        _sample("sample, one row of 32000", 1, 32000, "fp16", "all"),
        # a batch whose requests ask for different filters
        _sample("sample, 64 rows of 50272", 64, 50272, "fp16", "mixed"),
        # a large batch over a large vocabulary, logits kept in fp32, temperature only
        _sample("sample, 256 rows of 131072", 256, 131072, "fp32", "none"),
        # one request with its adapter
        _adapt("adapt, one row 4096 to 4096", 1, 4096, 4096, 16, 4, "own", 1),
        # nine requests, some without an adapter, down projection
        _adapt("adapt, 9 rows 11008 to 4096", 9, 11008, 4096, 8, 16, "mixed", 2),
        # a full batch, every request another adapter of higher rank, gate or up projection
        _adapt("adapt, 48 rows 4096 to 11008", 48, 4096, 11008, 64, 48, "own", 3),
        # prompts of six requests in one call
        _adapt("adapt, 4096 rows 4096 to 4096", 4096, 4096, 4096, 32, 6, "runs", 4),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))) - 0.5)))


def draw(rng):
    op = rng.choice(("attend", "attend", "sample", "adapt"))
    if op == "attend":
        while True:
            tokens = 1 if rng.random() < 0.5 else _log_int(rng, 2, 1500)
            kv_heads = rng.choice((1, 2, 3, 4, 8, 16))
            case = _attend(None, _log_int(rng, 1, 40), tokens, kv_heads * rng.choice((1, 1, 2, 3, 4, 5, 8)), kv_heads,
                           rng.choice((64, 128, 128, 96, 256, 32, 160)), _log_int(rng, max(tokens, 40), 60000),
                           rng.choice(("ragged", "full")), rng.randrange(1 << 20))
            scores = case["heads"] * tokens * case["max_positions"]
            w = work(case)
            if scores <= 1 << 28 and w["bytes"] <= 300e6 and w["flops"] <= 60e9:
                break
    elif op == "sample":
        case = _sample(None, _log_int(rng, 1, 200), _log_int(rng, 2000, 131072), rng.choice(("fp16", "bf16", "fp32")),
                       rng.choice(("all", "mixed", "none")))
    else:
        while True:
            case = _adapt(None, _log_int(rng, 1, 3000), 32 * _log_int(rng, 8, 350), 4 * _log_int(rng, 64, 2800),
                          rng.choice((4, 8, 16, 16, 24, 32, 64, 128)), _log_int(rng, 1, 64), rng.choice(("own", "mixed", "runs")),
                          rng.randrange(1 << 20))
            if work(case)["bytes"] <= 110e6 and case["count"] * case["rank"] * (case["K"] + case["N"]) <= 1 << 27:
                break
    del case["name"]
    return case


def _lengths(case):
    """For each sequence, the position of its first new token (-1: idle) and how many new tokens it has."""
    rng, B, T, P = random.Random(case["lengths"]), case["batch"], case["tokens"], case["max_positions"]
    if case["spread"] == "full":
        return [P - T] * B, [T] + [max(1, T - rng.randint(0, T // 5)) for _ in range(B - 1)]
    starts, counts = [], []
    for b in range(B):
        starts.append(-1 if b and rng.random() < 0.1 else _log_int(rng, 1, P - T + 1) - 1)
        counts.append(T if b == 0 else rng.randint(1, T))
    return starts, counts


def _ids(case):
    rng, M, count = random.Random(case["ids"]), case["rows"], case["count"]
    if case["order"] == "own":
        return [i % count for i in range(M)]
    if case["order"] == "mixed":
        return [rng.randint(-1, count - 1) for _ in range(M)]
    cuts = sorted(rng.randint(0, M) for _ in range(count - 1))
    return [sum(i >= c for c in cuts) for i in range(M)]


def work(case):
    if case["op"] == "attend":
        hd, KV, H = case["head_dim"], case["kv_heads"], case["heads"]
        nbytes = flops = 0
        for start, n in zip(*_lengths(case)):
            rows = case["tokens"] * hd * 2
            nbytes += rows * (H + 2 * KV)                     # out, what the cache holds of the new keys and values
            if start < 0:
                continue
            nbytes += n * hd * 2 * (H + 2 * KV) + n * hd * 4  # q, k, v, angles
            nbytes += (start + n) * KV * hd * 5 // 4          # 4 bits and a quarter of scales and minima, keys and values
            flops += 4 * hd * H * (n * start + n * (n + 1) // 2)
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * (4 if case["dtype"] == "fp32" else 2) + 32), "flops": 20 * case["rows"] * case["vocab"]}
    ids, K, N, r = _ids(case), case["K"], case["N"], case["rank"]
    used = len(set(i for i in ids if i >= 0))
    return {"bytes": case["rows"] * (2 * K + 4 * N + 4) + used * r * (K + N) * 2, "flops": 2 * r * (K + N) * sum(i >= 0 for i in ids)}


# ---- inputs ------------------------------------------------------------------------------------------
_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, device=DEVICE)
    uniform = lambda *shape: torch.rand(shape, generator=g, device=DEVICE)
    s = {"case": case}
    if case["op"] == "attend":
        B, T, H, KV, hd, P = (case[n] for n in ("batch", "tokens", "heads", "kv_heads", "head_dim", "max_positions"))
        G, blocks = hd // GROUP, -(-P // 32)
        s["starts"], s["counts"] = _lengths(case)
        s["start"] = torch.tensor(s["starts"], device=DEVICE)
        s["count"] = torch.tensor(s["counts"], dtype=torch.int32, device=DEVICE)
        # codes as earlier tokens left them: groups of values about zero, channels of unlike size
        cache = torch.empty((B, KV, blocks, 1280 * G), dtype=torch.uint8, device=DEVICE)
        words = cache.view(torch.int32)
        words.random_(-2 ** 31, 2 ** 31 - 1, generator=g)
        half = cache.view(torch.float16)
        for first, key in ((256 * G, True), (576 * G, False)):
            scale = (0.1 + 0.3 * uniform(B, KV, blocks, 32, G)).half()
            low = (-scale.float() * (6 + 3 * uniform(B, KV, blocks, 32, G))).half()
            pair = torch.stack([scale, low], -1)
            half[..., first:first + 64 * G] = (pair if key else pair.permute(0, 1, 2, 4, 5, 3)).reshape(B, KV, blocks, 64 * G)
        s["q"] = (normal(B, T, H * hd) * 1.5).half()
        s["k"] = (normal(B, T, KV * hd) * (0.5 + uniform(KV * hd))).half()
        s["v"] = normal(B, T, KV * hd).half()
        angle = torch.arange(P, device=DEVICE).double()[:, None] / 10000.0 ** (torch.arange(0, hd, 2, device=DEVICE).double() / hd)
        s["cos"], s["sin"] = (torch.cat([f(angle)] * 2, -1).half() for f in (torch.cos, torch.sin))
        s["cache"] = cache
        if own:
            from shiftaddllm_amd.kv_cache import Q4Cache
            s["handle"] = Q4Cache(B, KV, P, hd, device=DEVICE, data=cache)
    elif case["op"] == "sample":
        R, V = case["rows"], case["vocab"]
        logits = normal(R, V) * 2.2 - 3
        # what the context speaks for: one token from every fortieth of the vocabulary (a token twice would get either of two values)
        at = torch.randint(0, V // 40, (R, 40), generator=g, device=DEVICE) + torch.arange(40, device=DEVICE) * (V // 40)
        logits.scatter_(1, at, normal(R, 40) * 2.5 + 7)
        logits.masked_fill_(uniform(R, V) < 0.01, float("-inf"))                     # banned tokens
        s["logits"] = logits.to(_DTYPES[case["dtype"]])
        s["uniform"] = uniform(R)
        pick = lambda values, dtype=torch.float32: torch.tensor(values, dtype=dtype, device=DEVICE)[
            torch.randint(0, len(values), (R,), generator=g, device=DEVICE)]
        f = case["filters"]
        s["temperature"] = pick((0.6, 0.8, 1.0, 1.3) + ((0.0,) if f == "mixed" else ()))
        s["top_k"] = None if f == "none" else pick((20, 40, 200) + ((0, 1, 3000) if f == "mixed" else ()), torch.int32)
        s["top_p"] = None if f == "none" else pick((0.8, 0.9, 0.95) + ((1.0, 0.3, 0.999) if f == "mixed" else ()))
        s["min_p"] = None if f == "none" else pick((0.01, 0.05) + ((0.0, 0.2) if f == "mixed" else ()))
    else:
        M, K, N, r, count = (case[n] for n in ("rows", "K", "N", "rank", "count"))
        s["x"] = normal(M, K).half()
        s["base"] = normal(M, N).half()
        s["ids"] = torch.tensor(_ids(case), dtype=torch.int32, device=DEVICE)
        s["down"] = (normal(count, r, K) / math.sqrt(K)).half()
        s["up"] = (normal(count, N, r) * 0.3).half()
        s["scale"] = 0.25 + uniform(count)
        if own:
            from shiftaddllm_amd.lut_gemm.adapters import AdapterBank
            s["handle"] = AdapterBank.from_tensors(s["down"], s["up"], s["scale"])
    return s


# ---- the operators -----------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if op == "attend":
        if not own:
            return _plain_attend(s)
        return s["handle"].attend(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["start"], s["count"], held=True)
    if op == "sample":
        if not own:
            return _plain_sample(s)
        from shiftaddllm_amd.sampling import sample
        return sample(s["logits"], s["uniform"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    if not own:
        return _plain_adapt(s)
    return s["handle"](s["x"], s["ids"], s["base"])


def _turn(x, cos, sin):
    """Rotary embedding of x [T, heads, hd] at T rows of angles, rounded to fp16."""
    c, sn = cos.float()[:, None], sin.float()[:, None]
    h = x.shape[-1] // 2
    x = x.float()
    return (x * c + torch.cat([-x[..., h:], x[..., :h]], -1) * sn).half()


def _finite(x):
    return torch.nan_to_num(x.float(), nan=0.0, posinf=LARGEST, neginf=-LARGEST).clamp(-LARGEST, LARGEST)


def _quantise(x):
    """x [..., hd] -> codes, scales and minima, and the values that they stand for (fp16)."""
    x = _finite(x).double().unflatten(-1, (-1, GROUP))
    low, high = x.amin(-1), x.amax(-1)
    scale = ((high - low) / 15).float().half()
    d = scale.double()[..., None]
    code = torch.where(d > 0, ((x - low[..., None]) / torch.where(d > 0, d, 1.0)).round(), 0.0).clamp(0, 15)
    value = (low[..., None] + d * code).float().half()
    return code.to(torch.int32).flatten(-2), torch.stack([scale, low.half()], -1), value.flatten(-2)


_NIBBLE = [4 * (e // 2 + 4 * (e % 2)) for e in range(8)]


def _codes_of(words):
    return torch.stack([(words >> b) & 15 for b in _NIBBLE], -1)


def _words_of(codes):
    w = torch.zeros(codes.shape[:-1], dtype=torch.int64, device=codes.device)
    for e, b in enumerate(_NIBBLE):
        w |= codes[..., e].long() << b
    return torch.where(w >= 1 << 31, w - (1 << 32), w).int()


def _unpack(blocks):
    """Blocks [..., n, 1280 G] of a cache -> codes [..., 32 n, hd] and scales [..., 32 n, G, 2] of keys and values."""
    lead, n, G = blocks.shape[:-2], blocks.shape[-2], blocks.shape[-1] // 1280
    words, half = blocks.view(torch.int32), blocks.view(torch.float16)
    kc = _codes_of(words[..., :128 * G].unflatten(-1, (32, 4, G))).transpose(-3, -2)
    ks = half[..., 256 * G:320 * G].unflatten(-1, (32, G, 2))
    vc = _codes_of(words[..., 160 * G:288 * G].unflatten(-1, (4, 16, 2 * G))).unflatten(-1, (2, 4))   # quad, c, t, h, r
    d = vc.dim() - 5
    vc = vc.permute(*range(d), d + 3, d, d + 4, d + 2, d + 1)
    vs = half[..., 576 * G:640 * G].unflatten(-1, (G, 2, 4, 2, 4))                                     # group, part, quad, h, r
    vs = vs.permute(*range(d), d + 3, d + 2, d + 4, d, d + 1)
    hd = 32 * G
    return (kc.reshape(*lead, 32 * n, hd), ks.reshape(*lead, 32 * n, G, 2), vc.reshape(*lead, 32 * n, hd), vs.reshape(*lead, 32 * n, G, 2))


def _pack(kc, ks, vc, vs):
    """The inverse of _unpack."""
    lead, n, hd = kc.shape[:-2], kc.shape[-2] // 32, kc.shape[-1]
    G, d = hd // 32, len(lead) + 1
    out = torch.empty((*lead, n, 1280 * G), dtype=torch.uint8, device=kc.device)
    words, half = out.view(torch.int32), out.view(torch.float16)
    words[..., :128 * G] = _words_of(kc.reshape(*lead, n, 32, G, 4, 8).transpose(-3, -2)).flatten(-3)
    half[..., 256 * G:320 * G] = ks.reshape(*lead, n, 64 * G)
    v = vc.reshape(*lead, n, 2, 4, 4, 2 * G, 16).permute(*range(d), d + 1, d + 4, d + 3, d, d + 2)     # quad, c, t, h, r
    words[..., 160 * G:288 * G] = _words_of(v.flatten(-2)).flatten(-3)
    half[..., 576 * G:640 * G] = vs.reshape(*lead, n, 2, 4, 4, G, 2).permute(*range(d), d + 3, d + 4, d + 1, d, d + 2).flatten(-5)
    return out


def _values(codes, scales, dtype):
    """The values that codes stand for, fp16 numbers held in `dtype`."""
    s, low = scales[..., :1].double() if dtype is torch.float64 else scales[..., :1].float(), scales[..., 1:]
    return (low.to(s.dtype) + s * codes.unflatten(-1, (-1, GROUP))).half().to(dtype).flatten(-2)


def _plain_attend(s):
    c = s["case"]
    B, T, H, KV, hd = (c[n] for n in ("batch", "tokens", "heads", "kv_heads", "head_dim"))
    out = torch.zeros((B, T, H * hd), dtype=torch.float16, device=DEVICE)
    k_held, v_held = (torch.zeros((B, T, KV * hd), dtype=torch.float16, device=DEVICE) for _ in range(2))
    for b, (start, n) in enumerate(zip(s["starts"], s["counts"])):
        if start < 0:
            continue
        cos, sin = s["cos"][start:start + n], s["sin"][start:start + n]
        q = _turn(s["q"][b, :n].view(n, H, hd), cos, sin)
        k, v = _turn(s["k"][b, :n].view(n, KV, hd), cos, sin), s["v"][b, :n].view(n, KV, hd)
        first, last = start // 32, -(-(start + n) // 32)
        mine = s["cache"][b, :, first:last]
        parts = _unpack(mine)
        at = slice(start - 32 * first, start - 32 * first + n)
        for x, codes, scales, held in ((k, parts[0], parts[1], k_held), (v, parts[2], parts[3], v_held)):
            code, scale, value = _quantise(x)
            codes[:, at], scales[:, at] = code.transpose(0, 1), scale.transpose(0, 1)
            held[b, :n] = value.flatten(1)
        mine.copy_(_pack(*parts))
        kc, ks, vc, vs = (p[:, :start + n] for p in _unpack(s["cache"][b, :, :last]))
        kk, vv = _values(kc, ks, torch.float32), _values(vc, vs, torch.float32)
        rows = q.float().view(n, KV, H // KV, hd).permute(1, 2, 0, 3).reshape(KV, -1, hd)
        score = torch.matmul(rows, kk.transpose(1, 2).contiguous()).view(KV, H // KV, n, start + n) / math.sqrt(hd)
        late = torch.arange(start + n, device=DEVICE)[None] > torch.arange(start, start + n, device=DEVICE)[:, None]
        score.masked_fill_(late, float("-inf"))
        p = (score - score.amax(-1, keepdim=True)).exp()
        o = torch.matmul(p.view(KV, -1, start + n), vv).view(KV, H // KV, n, hd) / p.sum(-1, keepdim=True)
        out[b, :n] = o.permute(2, 0, 1, 3).reshape(n, H * hd).half()
    return out, k_held, v_held


def _plain_sample(s):
    x = s["logits"].double()
    R, V = x.shape
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    t = s["temperature"].double()
    greedy = ~(t > 0)
    w = ((x - x[:, :1]) / torch.where(greedy, 1.0, t)[:, None]).exp()
    rank = torch.arange(V, device=DEVICE)
    keep = torch.ones_like(w, dtype=torch.bool)
    if s["top_k"] is not None:
        k = s["top_k"].long()
        keep &= rank < torch.where(k > 0, k, V)[:, None]
    if s["top_p"] is not None:
        kept = torch.where(keep, w, 0.0)
        running = kept.cumsum(-1)
        p = s["top_p"].double()[:, None]
        keep &= ((running - kept) < p * running[:, -1:]) | (p >= 1)
    if s["min_p"] is not None:
        keep &= w >= s["min_p"].double()[:, None]
    keep &= ~greedy[:, None] | (rank == 0)
    running = torch.where(keep, w, 0.0).cumsum(-1)
    total = running[:, -1:]
    at = (running > s["uniform"].double()[:, None] * total).int().argmax(-1, keepdim=True)
    return order.gather(-1, at)[:, 0], (w.gather(-1, at) / total).log()[:, 0].float()


def _plain_adapt(s):
    out = s["base"].float()
    for a in range(s["case"]["count"]):
        at = torch.nonzero(s["ids"] == a)[:, 0]
        h = torch.matmul(s["x"][at].float(), s["down"][a].float().t().contiguous())
        out[at] += s["scale"][a] * torch.matmul(h, s["up"][a].float().t().contiguous())
    return out.half()


# ---- the definitions in 64 bits ----------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(s)
    return _exact_sample(s) if case["op"] == "sample" else _exact_adapt(s)


def _exact_group(x):
    """Held values of x [rows, hd] (float64, finite), one group of 32 at a time."""
    out = torch.empty_like(x)
    for d in range(0, x.shape[1], GROUP):
        g = x[:, d:d + GROUP]
        low, high = g.min(1, keepdim=True).values, g.max(1, keepdim=True).values
        step = ((high - low) / 15.0).float().half().double()
        code = torch.floor((g - low) / step.clamp_min(1e-30) + 0.5)
        tie = (g - low) == (code - 0.5) * step
        code = torch.where(tie & (code % 2 == 1), code - 1, code).clamp(0, 15)
        out[:, d:d + GROUP] = (low + step * code).float().half().double()
    return out


def _exact_attend(s):
    c = s["case"]
    B, T, H, KV, hd = (c[n] for n in ("batch", "tokens", "heads", "kv_heads", "head_dim"))
    G, f64 = hd // 32, torch.float64
    out = torch.zeros((B, T, H * hd), dtype=f64, device=DEVICE)
    k_held, v_held = (torch.zeros((B, T, KV * hd), dtype=f64, device=DEVICE) for _ in range(2))
    e, d, pos = torch.arange(8, device=DEVICE), torch.arange(hd, device=DEVICE), torch.arange(32, device=DEVICE)
    shift_of = 4 * (e // 2) + 16 * (e % 2)
    # where dimension d of position p of a block is kept: word and bits
    k_word = pos[:, None] * 4 * G + (d % 32 // 8) * G + d // 32
    k_bits = shift_of[d % 8].expand(32, hd)
    quad, slot = pos % 16 // 4, pos % 4 + 4 * (pos // 16)
    v_word = 160 * G + (quad[:, None] * 16 + d % 16) * 2 * G + d // 16
    v_bits = shift_of[slot][:, None].expand(32, hd)
    k_scale = 256 * G + (pos[:, None] * G + d // 32) * 2
    v_scale = 576 * G + (d // 32 * 2) * 32 + (quad * 8 + slot)[:, None]
    for b, (start, n) in enumerate(zip(s["starts"], s["counts"])):
        if start < 0:
            continue
        half = hd // 2
        cos, sin = (s[f][start:start + n].double()[:, None] for f in ("cos", "sin"))

        def turn(x):
            x = x.double()
            y = torch.empty_like(x)
            y[..., :half] = x[..., :half] * cos[..., :half] - x[..., half:] * sin[..., :half]
            y[..., half:] = x[..., half:] * cos[..., half:] + x[..., :half] * sin[..., half:]
            return y.float().half().double()
        q = turn(s["q"][b, :n].view(n, H, hd))
        new_k = _exact_group(turn(s["k"][b, :n].view(n, KV, hd)).reshape(n * KV, hd)).view(n, KV, hd)
        new_v = _exact_group(s["v"][b, :n].double().reshape(n * KV, hd)).view(n, KV, hd)
        k_held[b, :n], v_held[b, :n] = new_k.flatten(1), new_v.flatten(1)
        late = torch.arange(start + n, device=DEVICE)[None] > torch.arange(start, start + n, device=DEVICE)[:, None]
        used = -(-start // 32)
        for h in range(KV):
            block = s["cache"][b, h, :used]
            words, halves = block.view(torch.int32), block.view(torch.float16).double()

            def earlier(word, bits, scale, step):
                code = (words[:, word] >> bits) & 15
                return (halves[:, scale + step] + halves[:, scale] * code).float().half().double().reshape(-1, hd)[:start]
            kk = torch.cat([earlier(k_word, k_bits, k_scale, 1), new_k[:, h]])
            vv = torch.cat([earlier(v_word, v_bits, v_scale, 32), new_v[:, h]])
            for i in range(h * (H // KV), (h + 1) * (H // KV)):
                score = (q[:, i] @ kk.t()) / math.sqrt(hd)
                out[b, :n, i * hd:(i + 1) * hd] = torch.softmax(score.masked_fill(late, float("-inf")), -1) @ vv
    return out, k_held, v_held


def _exact_sample(s):
    import numpy as np
    x = s["logits"].double().cpu().numpy()
    host = {n: s[n].double().cpu().numpy() if s[n] is not None else None for n in ("temperature", "top_k", "top_p", "min_p", "uniform")}
    ids, logprob = [], []
    for r in range(x.shape[0]):
        order = np.argsort(-x[r], kind="stable")
        t = host["temperature"][r]
        if not t > 0:
            ids.append(int(order[0]))
            logprob.append(0.0)
            continue
        w = np.exp((x[r][order] - x[r][order[0]]) / t)
        n = len(w)
        if host["top_k"] is not None and host["top_k"][r] > 0:
            n = min(n, int(host["top_k"][r]))
        cum = np.cumsum(w[:n])
        if host["top_p"] is not None and host["top_p"][r] < 1:
            n = min(n, int(np.searchsorted(cum, host["top_p"][r] * cum[n - 1], side="left")) + 1)
        if host["min_p"] is not None:
            n = min(n, max(1, int((w >= host["min_p"][r]).sum())))
        at = int(np.searchsorted(cum[:n], host["uniform"][r] * cum[n - 1], side="right"))
        ids.append(int(order[at]))
        logprob.append(float(np.log(w[at] / cum[n - 1])))
    return torch.tensor(ids), torch.tensor(logprob, dtype=torch.float64)


def _exact_adapt(s):
    out = s["base"].double()
    ids = s["ids"].tolist()
    for a in sorted(set(ids) - {-1}):
        at = torch.tensor([i for i, v in enumerate(ids) if v == a], device=DEVICE)
        out[at] += s["scale"][a].double() * ((s["x"][at].double() @ s["down"][a].double().t()) @ s["up"][a].double().t())
    return out
