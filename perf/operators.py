"""Cases of the serving operators around the paged quantised cache: per-head
query/key norms with position rotation, the append of rotated keys and of
values to a paged cache, and decode attention for batches that share prefixes.

Each operator has a plain form in elementary torch operations (32 bits
throughout, rounded once at the end) and, where `own` is true, the call a user
makes of the package.  The caches are the package's plane layout: sign words,
INT4 residual codes (offset-binary, interleaved in blocks of 8 positions), and
fp16 scales, in pages of `page` positions of one (sequence, kv head).
"""
import math
import random
from functools import reduce

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # Queries and keys of one decode step of a 16-sequence grouped-query batch: latency.
        dict(name="rope_step", op="rope", tokens=16, q_heads=32, kv_heads=8, dim=128, dtype="fp16", rotary=128,
             interleaved=False, norm=True, positions=4096),
        # A chunk of prompts in a model's own type, per-head norms, straight from the packed projection.
        dict(name="rope_prompt", op="rope", tokens=16384, q_heads=32, kv_heads=8, dim=128, dtype="bf16", rotary=128,
             interleaved=False, norm=True, positions=32768),
        # An odd number of tokens, small heads, half of each head rotated in adjacent pairs, no norms, 32 bits.
        dict(name="rope_partial", op="rope", tokens=2999, q_heads=16, kv_heads=16, dim=64, dtype="fp32", rotary=32,
             interleaved=True, norm=False, positions=8192),
        # One new token for each of 16 sequences into the paged cache: latency.
        dict(name="append_step", op="append", seqs=16, fresh=1, start=900, q_heads=32, kv_heads=8, dim=128,
             dtype="fp16", rotary=128, interleaved=False, norm=False, residual=True, page=128, back=False, lens=1),
        # Ragged prompts written at once; the prompt's own attention is given the rows as the cache holds them.
        dict(name="append_prompts", op="append", seqs=24, fresh=1024, start=0, q_heads=32, kv_heads=8, dim=128,
             dtype="bf16", rotary=128, interleaved=False, norm=True, residual=True, page=256, back=True, lens=2),
        # Chunks appended to a binary-only cache with large heads, partly rotated.
        dict(name="append_binary_256", op="append", seqs=7, fresh=333, start=250, q_heads=16, kv_heads=4, dim=256,
             dtype="fp16", rotary=64, interleaved=True, norm=False, residual=False, page=128, back=False, lens=3),
        # Four short conversations behind one system prompt that ends inside a page: latency.
        dict(name="shared_small", op="shared", seqs=4, groups=1, prefix=1000, suffix=64, q_heads=32, kv_heads=8,
             dim=128, residual=True, page=128, lens=4),
        # The grouped-query batch of 16 sequences over a 32768-token document, each with its own turns.
        dict(name="shared_document", op="shared", seqs=16, groups=1, prefix=32768, suffix=2048, q_heads=32,
             kv_heads=8, dim=128, residual=True, page=256, lens=5),
        # A large batch behind a long system prompt: the prefix is matrix work.
        dict(name="shared_batch", op="shared", seqs=128, groups=1, prefix=8192, suffix=512, q_heads=32, kv_heads=8,
             dim=128, residual=True, page=128, lens=6),
        # Beams: 16 prompts of different lengths, 8 hypotheses each, one head per kv head.
        dict(name="shared_beams", op="shared", seqs=128, groups=16, prefix=4000, suffix=128, q_heads=16, kv_heads=16,
             dim=64, residual=True, page=128, lens=7),
        # No common prefix: ragged lengths from one token on, a binary-only cache with large heads.
        dict(name="ragged_binary_256", op="shared", seqs=48, groups=1, prefix=0, suffix=6000, q_heads=16, kv_heads=8,
             dim=256, residual=False, page=128, lens=8),
        # A few sequences over a very long context.
        dict(name="shared_long", op="shared", seqs=8, groups=1, prefix=200000, suffix=4096, q_heads=32, kv_heads=8,
             dim=128, residual=True, page=512, lens=9),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "shared", "shared"])
    dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    group = rng.choice([1, 2, 4, 8])
    heads = dict(q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim)
    rotated = dict(rotary=rng.choice([dim, dim, dim // 2]), interleaved=rng.random() < 0.3, norm=rng.random() < 0.5)
    if op == "rope":
        most = max(2, min(16384, 16384 * 40 * 128 // ((group + 1) * kv_heads * dim)))
        return dict(op=op, tokens=_spread(rng, 1, most), dtype=rng.choice(["fp16", "bf16", "fp32"]), positions=32768,
                    **heads, **rotated)
    if op == "append":
        seqs = _spread(rng, 1, 64)
        most = max(1, min(2048, 24 * 1024 * 8 * 128 // (seqs * kv_heads * dim)))
        return dict(op=op, seqs=seqs, fresh=_spread(rng, 1, most), start=rng.randrange(0, 600),
                    dtype=rng.choice(["fp16", "bf16", "fp32"]), residual=rng.random() < 0.7,
                    page=rng.choice([128, 256, 384]), back=rng.random() < 0.5, lens=rng.randrange(1 << 20),
                    **heads, **rotated)
    groups = rng.choice([1, 1, 1, 2, 4])
    seqs = groups * _spread(rng, 1, 128 // groups)
    prefix = rng.choice([0, 1]) and _spread(rng, 16, 131072 // groups // max(1, kv_heads * dim // 1024))
    suffix = _spread(rng, 1, 4096)
    rows = seqs * kv_heads * group * dim  # the plain form holds a score for each query head and key
    while seqs * kv_heads * group * (prefix + suffix) > 1 << 28 or rows * (prefix + suffix) > 1 << 35 or \
            seqs * kv_heads * dim * suffix > 1 << 29:
        prefix, suffix = prefix // 2, max(1, suffix // 2)
    return dict(op=op, seqs=seqs, groups=groups, prefix=prefix, suffix=suffix, residual=rng.random() < 0.7,
                page=rng.choice([128, 256, 512]), lens=rng.randrange(1 << 20), **heads)


# ---- lengths ---------------------------------------------------------------
def _append_lens(c):
    """New tokens and first position of each sequence."""
    r = random.Random(c["lens"])
    fresh = [c["fresh"] if c["fresh"] == 1 else r.randint(max(1, c["fresh"] // 2), c["fresh"]) for _ in range(c["seqs"])]
    start = [r.randint(0, c["start"]) for _ in range(c["seqs"])]
    return fresh, start


def _shared_lens(c):
    """Prefix length of each group and whole length of each sequence."""
    r = random.Random(c["lens"])
    prefix = [c["prefix"] if c["groups"] == 1 else r.randint(c["prefix"] // 2, c["prefix"]) for _ in range(c["groups"])]
    per = c["seqs"] // c["groups"]
    return prefix, [prefix[b // per] + r.randint(1, c["suffix"]) for b in range(c["seqs"])]


def work(c):
    d, hq, hkv = c["dim"], c["q_heads"], c["kv_heads"]
    if c["op"] == "rope":
        t, size = c["tokens"], 4 if c["dtype"] == "fp32" else 2
        return {"bytes": t * ((hq + hkv) * d * 2 * size + 4 * c["rotary"] + 4),
                "flops": t * (hq + hkv) * (3 * c["rotary"] + (4 * d if c["norm"] else 0))}
    vector = d // 8 + 2 + (d // 2 + 2 if c["residual"] else 0)
    if c["op"] == "append":
        t, size = sum(_append_lens(c)[0]), 4 if c["dtype"] == "fp32" else 2
        return {"bytes": t * ((hq + 2 * hkv) * d * size + hq * d * 2 + 2 * hkv * vector + 4 * c["rotary"] + 8
                              + (4 * hkv * d if c["back"] else 0)),
                "flops": t * ((hq + hkv) * (3 * c["rotary"] + (4 * d if c["norm"] else 0))
                              + 2 * hkv * d * (8 if c["residual"] else 2))}
    prefix, total = _shared_lens(c)
    per = c["seqs"] // c["groups"]
    keys = sum(prefix) + sum(n - prefix[b // per] for b, n in enumerate(total))
    return {"bytes": 2 * hkv * keys * vector + 2 * c["seqs"] * hq * d * 2, "flops": 4 * d * hq * sum(total)}


# ---- the plane layout ------------------------------------------------------
def _code_dims(d, device):
    """Dim held by each nibble of a row in chunk order: [d / 2 bytes, 2] (low, high)."""
    p = torch.arange(d // 2, device=device)
    c, j = p // 16, p % 16
    if d == 64:
        low, step = 8 * (j % 8) + 2 * c + j // 8, 4
    elif d == 128:
        low, step = 8 * j + c, 4
    elif d == 256:
        low, step = 128 * (c // 4) + 8 * j + c % 4, 4
    else:
        low, step = 32 * c + 2 * j, 1
    return torch.stack([low, low + step], -1)


def _halves(a):
    """Sum over the last axis by halves (stride d/2, ..., 2, 1): the order is part of the definition."""
    n = 1 << (a.shape[-1] - 1).bit_length()
    a = torch.nn.functional.pad(a, (0, n - a.shape[-1]))
    return reduce(lambda x, _: x[..., :x.shape[-1] // 2] + x[..., x.shape[-1] // 2:], range(n.bit_length() - 1), a)[..., 0]


def _by(a, value):
    """a / value, correctly rounded (a scalar divisor would become a product)."""
    return a / torch.full_like(a, value)


def _encode(x, residual):
    """fp32 vectors [..., d] -> sign words, fp16 scale, nibble bytes [..., d / 32, 16] in chunk order, fp16
    residual scale, and the values they stand for."""
    d = x.shape[-1]
    positive = x >= 0
    words = (positive.unflatten(-1, (d // 32, 32)).long() << torch.arange(32, device=x.device)).sum(-1)
    words = (words - ((words >> 31) << 32)).to(torch.int32)
    scale = _by(_halves(x.abs()), float(d))
    held = torch.where(positive, 1.0, -1.0) * scale.half().float()[..., None]
    if not residual:
        return words, scale.half(), None, None, held
    left = x - torch.where(positive, scale[..., None], -scale[..., None])
    most = left.abs().amax(-1)
    inverse = torch.where(most > 0, torch.full_like(most, 7.0) / most, torch.zeros_like(most))
    code = torch.round(left * inverse[..., None]).clamp(-7, 7)
    held = held + _by(code, 7.0) * most.half().float()[..., None]
    pair = (code + 8).to(torch.uint8)[..., _code_dims(d, x.device)]
    nib = (pair[..., 0] | (pair[..., 1] << 4)).unflatten(-1, (d // 32, 16))
    return words, scale.half(), nib, most.half(), held


def _rows_of(nib, rows, d):
    """A nibble pool as [pages, page / 8, d / 32, 8, 16]: chunk c of row 8i + r is [i, c, r]."""
    return nib.view(nib.shape[0], rows // 8, d // 32, 8, 16)


def _pool(pages, rows, d, residual, device):
    p = {"sign": torch.zeros(pages, rows, d // 32, dtype=torch.int32, device=device),
         "bscale": torch.zeros(pages, rows, dtype=torch.float16, device=device)}
    if residual:
        p["nib"] = torch.full((pages, rows, d // 2), 0x88, dtype=torch.uint8, device=device)
        p["rscale"] = torch.zeros(pages, rows, dtype=torch.float16, device=device)
    return p


def _filled_pool(pages, rows, d, residual, g, device):
    """Every row of the pool holds a vector of unit variance whose largest channels stand out (a few channels of
    keys and values do in language models)."""
    p = _pool(pages, rows, d, residual, device)
    step = max(1, (1 << 26) // (rows * d))
    loud = 1 + 3 * (torch.rand(d, generator=g, device=device) < 0.03).float()
    for at in range(0, pages, step):
        n = min(step, pages - at)
        words, scale, nib, most, _ = _encode(torch.randn(n, rows, d, generator=g, device=device) * loud, residual)
        p["sign"][at:at + n], p["bscale"][at:at + n] = words, scale
        if residual:
            _rows_of(p["nib"], rows, d)[at:at + n] = nib.unflatten(1, (rows // 8, 8)).transpose(2, 3)
            p["rscale"][at:at + n] = most
    return p


# ---- inputs ----------------------------------------------------------------
def _rotation(c, n, device):
    inverse = 10000.0 ** (-torch.arange(0, c["rotary"], 2, dtype=torch.float64, device=device) / c["rotary"])
    angle = torch.arange(n, dtype=torch.float64, device=device)[:, None] * inverse
    return angle.cos().float(), angle.sin().float()


def _packed(c, tokens, g, device):
    """q, k, v as views of one packed projection [tokens, (q_heads + 2 kv_heads) * dim]."""
    d, hq, hkv = c["dim"], c["q_heads"], c["kv_heads"]
    x = torch.randn(tokens, hq + 2 * hkv, d, generator=g, device=device)
    x = (x * (1 + 2 * (torch.rand(hq + 2 * hkv, d, generator=g, device=device) < 0.03).float())).to(DTYPES[c["dtype"]])
    return x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)
    c, d, hkv = case, case["dim"], case["kv_heads"]
    s = {"case": case}
    if c["op"] != "shared" and c["norm"]:
        s["q_weight"], s["k_weight"] = (1 + 0.2 * torch.randn(2, d, generator=g, device=device)).unbind(0)
    if c["op"] == "rope":
        s["cos"], s["sin"] = _rotation(c, c["positions"], device)
        s["q"], s["k"], _ = _packed(c, c["tokens"], g, device)
        s["positions"] = torch.randint(0, c["positions"], (c["tokens"],), generator=g, device=device, dtype=torch.int32)
        return s
    if c["op"] == "append":
        fresh, start = _append_lens(c)
        most = max(a + b for a, b in zip(fresh, start))
        pages = -(-most // c["page"])
        n = torch.tensor(fresh, device=device)
        s["seq_ids"] = torch.repeat_interleave(torch.arange(c["seqs"], device=device), n).int()
        first = (torch.cumsum(n, 0) - n)[s["seq_ids"].long()]
        s["positions"] = (torch.arange(sum(fresh), device=device) - first
                          + torch.tensor(start, device=device)[s["seq_ids"].long()]).int()
        s["cos"], s["sin"] = _rotation(c, most, device)
        s["q"], s["k"], s["v"] = _packed(c, sum(fresh), g, device)
        count = c["seqs"] * hkv * pages
        s["pages"] = torch.randperm(count, generator=g, device=device).int().view(c["seqs"] * hkv, pages)
        s["K"], s["V"] = (_pool(count, c["page"], d, c["residual"], device) for _ in range(2))
        return s
    prefix, total = _shared_lens(c)
    per, page = c["seqs"] // c["groups"], c["page"]
    most = -(-max(total) // page)
    # physical pages: the whole pages of a group's prefix once for all its sequences, every other one (and the
    # prefix page that a sequence goes on writing in) of its own
    r = random.Random(c["lens"] + 1)
    ids, table = 0, torch.zeros(c["seqs"], hkv, most, dtype=torch.int32)
    twins = []
    for grp, p in enumerate(prefix):
        whole = p // page
        common = ids + torch.arange(hkv * whole, dtype=torch.int32).view(hkv, whole)
        ids += hkv * whole
        for b in range(grp * per, (grp + 1) * per):
            mine = -(-total[b] // page) - whole
            table[b, :, :whole] = common
            table[b, :, whole:whole + mine] = ids + torch.arange(hkv * mine, dtype=torch.int32).view(hkv, mine)
            ids += hkv * mine
            if p % page and b > grp * per:
                twins += [(int(table[b, h, whole]), int(table[grp * per, h, whole]), p % page) for h in range(hkv)]
    order = torch.tensor(r.sample(range(ids), ids), dtype=torch.int32)
    s["pages"] = order[table.long()].view(c["seqs"] * hkv, most).to(device)
    s["K"], s["V"] = (_filled_pool(ids, page, d, c["residual"], g, device) for _ in range(2))
    if twins:  # the begun page of the prefix holds the same rows in every sequence's copy
        t = torch.tensor(twins)
        to, of = order[t[:, 0].long()].long().to(device), order[t[:, 1].long()].long().to(device)
        same = (torch.arange(page)[None, :] < t[:, 2:]).to(device)
        for pool in (s["K"], s["V"]):
            for name, x in pool.items():
                if name == "nib":
                    x = _rows_of(x, page, d).permute(0, 1, 3, 2, 4)
                    x[to] = torch.where(same.view(-1, page // 8, 8, 1, 1), x[of], x[to])
                else:
                    x[to] = torch.where(same.view(same.shape + (1,) * (x.dim() - 2)), x[of], x[to])
    s["prefix_lens"] = torch.tensor(prefix, dtype=torch.int32, device=device)
    s["seq_lens"] = torch.tensor(total, dtype=torch.int32, device=device)
    s["q"] = torch.randn(c["seqs"], c["q_heads"], d, generator=g, device=device).half()
    return s


# ---- plain forms -----------------------------------------------------------
def _normed(x, weight):
    x = x.float()
    if weight is None:
        return x
    mean = _by(_halves(x * x), float(x.shape[-1]))
    return x * (1 / torch.sqrt(mean + EPS))[..., None] * weight


def _rotated(x, cos, sin, rotary, interleaved):
    turned, kept = x[..., :rotary], x[..., rotary:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), kept], -1)
    a, b = turned[..., :rotary // 2], turned[..., rotary // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, kept], -1)


def _plain_rope(s, c):
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    q, k = (_rotated(_normed(s[n], s.get(n + "_weight")), cos, sin, c["rotary"], c["interleaved"]) for n in "qk")
    return q, k


def _plain_append(s, c):
    q, k = _plain_rope(s, c)
    page, hkv, d = c["page"], c["kv_heads"], c["dim"]
    at = s["positions"].long()[:, None]
    slot = s["seq_ids"].long()[:, None] * hkv + torch.arange(hkv, device=at.device)
    where, row = s["pages"].long()[slot, at // page], (at % page).expand(-1, hkv)

    def write(x, pool):
        words, scale, nib, most, held = _encode(x, c["residual"])
        pool["sign"][where, row] = words
        pool["bscale"][where, row] = scale
        if c["residual"]:
            _rows_of(pool["nib"], page, d)[where, row // 8, :, row % 8] = nib
            pool["rscale"][where, row] = most
        return held.half()

    out = {"q": q.half(), "K": s["K"], "V": s["V"]}
    k, v = write(k, s["K"]), write(s["v"].float(), s["V"])
    return {**out, "k_hat": k, "v_hat": v} if c["back"] else out


def _values(pool, ids, c):
    """Rows of the pages ids [...]: (sign part, residual part), each [..., pages * page, d]."""
    d, page = c["dim"], c["page"]
    sign = (pool["sign"][ids][..., None] >> torch.arange(32, device=ids.device, dtype=torch.int32)) & 1
    part = (2 * sign.flatten(-2).float() - 1) * pool["bscale"][ids].float()[..., None]
    if not c["residual"]:
        return part.flatten(-3, -2), None
    nib = _rows_of(pool["nib"], page, d)[ids].transpose(-3, -2).flatten(-2).flatten(-3, -2)
    code = torch.stack([nib & 15, nib >> 4], -1).flatten(-2).float() - 8
    code = code[..., torch.argsort(_code_dims(d, ids.device).flatten())]
    rest = _by(code, 7.0) * pool["rscale"][ids].float()[..., None]
    return part.flatten(-3, -2), rest.flatten(-3, -2)


def _scores(q, sign, rest):
    """(mean|q| sign(q)) . sign part + q . residual part, over sqrt(d)."""
    level = _by(q.abs().sum(-1, keepdim=True), float(q.shape[-1]))
    s = (torch.where(q >= 0, 1.0, -1.0) * level) @ sign.transpose(-1, -2)
    if rest is not None:
        s = s + q @ rest.transpose(-1, -2)
    return s * (1.0 / math.sqrt(q.shape[-1]))


def _plain_shared(s, c):
    n, groups, hkv, page, d = c["seqs"], c["groups"], c["kv_heads"], c["page"], c["dim"]
    per, group = n // groups, c["q_heads"] // hkv
    table = s["pages"].long().view(n, hkv, -1)
    q = s["q"].float().view(n, hkv, group, d)
    first = s["prefix_lens"].long().repeat_interleave(per) // page
    # the sequences' own pages, from the one that holds the end of the prefix
    mine = -(-c["suffix"] // page) + 1
    at = first[:, None] + torch.arange(mine, device=q.device)
    ids = table.gather(2, at.clamp(max=table.shape[2] - 1)[:, None].expand(-1, hkv, -1))
    key = (at[:, :, None] * page + torch.arange(page, device=q.device)).flatten(1)
    live = (key >= s["prefix_lens"].long().repeat_interleave(per)[:, None]) & (key < s["seq_lens"].long()[:, None])
    own_scores = _scores(q, *_values(s["K"], ids, c)).masked_fill(~live[:, None, None], -math.inf)
    peak = own_scores.amax(-1, keepdim=True)
    value, rest = _values(s["V"], ids, c)
    value = value if rest is None else value + rest
    if c["prefix"] == 0:
        e = torch.exp(own_scores - peak)
        return ((e @ value) / e.sum(-1, keepdim=True)).half().view(n, c["q_heads"], d)
    # the prefix of each group, for all of its query heads at once
    lead = table.view(groups, per, hkv, -1)[:, 0, :, :-(-c["prefix"] // page)]
    shown = torch.arange(lead.shape[2] * page, device=q.device) < s["prefix_lens"].long()[:, None]
    rows = q.view(groups, per, hkv, group, d).transpose(1, 2).reshape(groups, hkv, per * group, d)
    scores = _scores(rows, *_values(s["K"], lead, c)).masked_fill(~shown[:, None, None], -math.inf)
    lead_value, lead_rest = _values(s["V"], lead, c)
    lead_value = lead_value if lead_rest is None else lead_value + lead_rest

    def by_sequence(x):
        return x.view(groups, hkv, per, group, -1).transpose(1, 2).reshape(n, hkv, group, -1)

    def by_group(x):
        return x.view(groups, per, hkv, group, -1).transpose(1, 2).reshape(groups, hkv, per * group, -1)

    peak = torch.maximum(peak, by_sequence(scores.amax(-1, keepdim=True)))
    e = torch.exp(scores - by_group(peak))
    mine = torch.exp(own_scores - peak)
    total = mine.sum(-1, keepdim=True) + by_sequence(e.sum(-1, keepdim=True))
    return ((mine @ value + by_sequence(e @ lead_value)) / total).half().view(n, c["q_heads"], d)


# ---- the calls -------------------------------------------------------------
def _handle(s, c):
    """What a user's program keeps beside its tensors: the cache, the block table and the rotation."""
    from bitcache_b200 import planes

    h = {"planes": planes}
    if c["op"] != "shared":
        h["rope"] = planes.Rope(s["cos"], s["sin"], interleaved=c["interleaved"], q_weight=s.get("q_weight"),
                                k_weight=s.get("k_weight"), eps=EPS)
    if c["op"] != "rope":
        h["K"], h["V"] = (planes.Planes(p["sign"], p["bscale"], p.get("nib"), p.get("rscale"), c["dim"])
                          for p in (s["K"], s["V"]))
        h["table"] = planes.PageTable(s["pages"], c["page"], s["K"]["sign"].shape[0])
    return h


def run(state):
    s, c = state, state["case"]
    if not own:
        if c["op"] == "rope":
            return tuple(x.to(DTYPES[c["dtype"]]) for x in _plain_rope(s, c))
        return _plain_append(s, c) if c["op"] == "append" else _plain_shared(s, c)
    if "handle" not in s:
        s["handle"] = _handle(s, c)
    h = s["handle"]
    planes = h["planes"]
    if c["op"] == "rope":
        return planes.qk_norm_rope(s["q"], s["k"], s["positions"], h["rope"])
    if c["op"] == "append":
        got = planes.append_qkv_paged(s["q"], s["k"], s["v"], h["K"], h["V"], h["table"], s["seq_ids"], s["positions"],
                                      h["rope"], planes.RES_FP32_SCALE if c["residual"] else planes.RES_NONE,
                                      want_hat=c["back"])
        out = {"q": got[0] if c["back"] else got, "K": s["K"], "V": s["V"]}
        return {**out, "k_hat": got[1], "v_hat": got[2]} if c["back"] else out
    return planes.decode_attention_shared(s["q"], h["K"], h["V"], h["table"], s["seq_lens"], s["prefix_lens"],
                                          planes.MODE_COMPENSATED if c["residual"] else planes.MODE_BINARY)


# ---- the definitions in 64 bits --------------------------------------------
def _turn64(x, weight, cos, sin, c):
    """Norm and rotation of [tokens, heads, dim] in 64 bits, as complex products."""
    x = x.double()
    if weight is not None:
        x = x * weight.double() / (x.square().mean(-1, keepdim=True) + EPS).sqrt()
    half = c["rotary"] // 2
    i = torch.arange(half, device=x.device)
    re, im = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
    z = torch.complex(x[..., re], x[..., im]) * torch.complex(cos.double(), sin.double())[:, None]
    y = x.clone()
    y[..., re], y[..., im] = z.real, z.imag
    return y


def _hold64(x, residual):
    """Scale, residual scale and held values of vectors in 64 bits."""
    scale = x.abs().mean(-1)
    held = torch.where(x >= 0, scale[..., None], -scale[..., None])
    if not residual:
        return scale, None, held
    most = (x - held).abs().amax(-1)
    return scale, most, held + torch.round((x - held) * 7 / most[..., None]) * most[..., None] / 7


def _row64(pool, ids, count, c):
    """The first `count` rows of the pages ids [n] in 64 bits: sign part and residual part, [count, dim]."""
    d = c["dim"]
    words = pool["sign"][ids].flatten(0, 1)[:count].long()
    dim = torch.arange(d, device=ids.device)
    sign = (2 * ((words[:, dim // 32] >> (dim % 32)) & 1) - 1).double() * pool["bscale"][ids].flatten()[:count, None].double()
    if not c["residual"]:
        return sign, torch.zeros_like(sign)
    where = torch.empty(d, dtype=torch.long, device=ids.device)  # nibble of each dim
    where[_code_dims(d, ids.device).flatten()] = dim
    row = torch.arange(count, device=ids.device)
    flat = pool["nib"][ids].flatten(1)
    byte = where // 2
    at = (row % c["page"] // 8 * 4 * d + row % 8 * 16)[:, None] + (byte // 16 * 128 + byte % 16)[None]
    code = (flat[(row // c["page"])[:, None], at].long() >> (4 * (where % 2))) & 15
    return sign, (code - 8).double() / 7 * pool["rscale"][ids].flatten()[:count, None].double()


def exact(case, seed):
    c, s = case, prepare(case, seed)
    d = c["dim"]
    if c["op"] != "shared":
        at = s["positions"].long()
        q, k = (_turn64(s[n], s.get(n + "_weight"), s["cos"][at], s["sin"][at], c) for n in "qk")
        if c["op"] == "rope":
            return q, k
        out = {"q": q}
        slot = s["seq_ids"].long()[:, None] * c["kv_heads"] + torch.arange(c["kv_heads"], device=at.device)
        place = s["pages"].long()[slot, at[:, None] // c["page"]] * c["page"] + at[:, None] % c["page"]
        for name, x in (("K", k), ("V", s["v"].double())):
            scale, most, held = _hold64(x, c["residual"])
            out[name] = {"sign": None}
            for field, x in (("bscale", scale),) + ((("rscale", most),) if c["residual"] else ()):
                full = s[name][field].double()
                full.view(-1)[place] = x
                out[name][field] = full
            if c["residual"]:
                out[name]["nib"] = None
            if c["back"]:
                out[name.lower() + "_hat"] = held
        return out
    prefix, total = _shared_lens(c)
    per, hkv, group = c["seqs"] // c["groups"], c["kv_heads"], c["q_heads"] // c["kv_heads"]
    if c["seqs"] * hkv > 4096 or sum(total) * hkv * d > 5e9:
        return None  # a pass over every (sequence, kv head) would take too long
    out = torch.empty(c["seqs"], c["q_heads"], d, dtype=torch.float64, device=s["q"].device)
    table = s["pages"].long().view(c["seqs"], hkv, -1)
    for b in range(c["seqs"]):
        for h in range(hkv):
            ids = table[b, h, :-(-total[b] // c["page"])]
            (ks, kr), (vs, vr) = (_row64(s[n], ids, total[b], c) for n in "KV")
            q = s["q"][b, h * group:(h + 1) * group].double()
            mean = q.abs().mean(-1, keepdim=True)
            score = (torch.where(q >= 0, mean, -mean) @ ks.T + q @ kr.T) / math.sqrt(d)
            out[b, h * group:(h + 1) * group] = torch.softmax(score, -1) @ (vs + vr)
    return out
