"""The attention side of serving a model from a paged key-value cache, as cases that can be timed and compared.

Four operators, in the order in which a serving step calls them:

* ``slots``   the block tables, token positions and cache slots of a step, from the lengths of its requests;
* ``rope``    the norms of each head's queries and keys, the position rotation, and the new keys and values into the cache;
* ``decode``  attention of one new token of each request over its pages;
* ``prompt``  causal attention of the new tokens of ragged prompts (whole, or a chunk of a longer one) over the pages.

Both attentions take a sliding window and a few first tokens that stay visible (sinks).  ``run`` computes a case in plain
32-bit torch operations, or, where ``own`` is set, through ``boostr_b200.attention``.  Request lengths follow from the
case alone (their order, the pages they live in and all values follow from the seed), so the work of a case is known.

Head counts and widths are those of a Llama-3-8B-shaped decoder (32 query heads, 8 key-value heads of 128) or generic.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5
GOLDEN = 0.6180339887498949


def listed():
    return [
        # one decoding step of a batch: each request gets one token, now and then a page
        dict(name="slots_step_64", op="slots", requests=64, new_lo=1, new_hi=1, ctx_lo=0, ctx_hi=8191, page=16, pad=0, short=0),
        # prompts of many lengths admitted at once, some requests idle, the step padded to a captured size, the pool three pages short
        dict(name="slots_ragged_500", op="slots", requests=500, new_lo=0, new_hi=601, ctx_lo=0, ctx_hi=4000, page=64, pad=37, short=3),
        # the new token of a single sequence, straight from the 32-bit projections
        dict(name="rope_step_1", op="rope", tokens=1, q_heads=32, kv_heads=8, dim=128, rot=128, interleaved=False, norm=False, act="f32",
             out="f32", cache="bf16", page=16),
        # a long prompt, 16-bit projections, with the norms of each head
        dict(name="rope_norm_8192", op="rope", tokens=8192, q_heads=32, kv_heads=8, dim=128, rot=128, interleaved=False, norm=True, act="bf16",
             out="bf16", cache="bf16", page=16),
        # an odd number of tokens, part of each head rotated in the interleaved layout, heads of 80
        dict(name="rope_part_1031", op="rope", tokens=1031, q_heads=20, kv_heads=5, dim=80, rot=32, interleaved=True, norm=False, act="f16",
             out="f16", cache="f16", page=64),
        # one short conversation: latency
        dict(name="decode_1_short", op="decode", requests=1, empty=0, len_lo=517, len_hi=517, q_heads=32, kv_heads=8, dim=128, window=0, sinks=0,
             act="bf16", out="bf16", cache="bf16", page=16, heads_first=False, lse=False),
        # a batch at all stages of its conversations, padded to a captured size, 32-bit queries and results, log-sum-exp for a later join
        dict(name="decode_48_ragged", op="decode", requests=48, empty=3, len_lo=1, len_hi=8192, q_heads=32, kv_heads=8, dim=128, window=0, sinks=0,
             act="f32", out="f32", cache="bf16", page=16, heads_first=True, lse=True),
        # one very long document
        dict(name="decode_1_long", op="decode", requests=1, empty=0, len_lo=131085, len_hi=131085, q_heads=32, kv_heads=8, dim=128, window=0,
             sinks=0, act="bf16", out="bf16", cache="bf16", page=64, heads_first=False, lse=False),
        # long conversations under a window with sinks, heads of 64, one key-value head for 16 query heads
        dict(name="decode_96_window", op="decode", requests=96, empty=0, len_lo=100, len_hi=20000, q_heads=64, kv_heads=4, dim=64, window=1024,
             sinks=4, act="f16", out="f16", cache="f16", page=32, heads_first=False, lse=False),
        # one prompt of the usual length
        dict(name="prompt_1_512", op="prompt", requests=1, new_lo=512, new_hi=512, ctx_lo=0, ctx_hi=0, q_heads=32, kv_heads=8, dim=128, window=0,
             sinks=0, dtype="bf16", page=16, heads_first=False),
        # chunks of longer prompts, ragged, under a window with sinks
        dict(name="prompt_5_window", op="prompt", requests=5, new_lo=1, new_hi=1500, ctx_lo=0, ctx_hi=6000, q_heads=16, kv_heads=2, dim=64,
             window=1024, sinks=4, dtype="f16", page=32, heads_first=True),
        # a long prompt at once: the tensor cores' case
        dict(name="prompt_1_8192", op="prompt", requests=1, new_lo=8192, new_hi=8192, ctx_lo=0, ctx_hi=0, q_heads=32, kv_heads=8, dim=128, window=0,
             sinks=0, dtype="bf16", page=16, heads_first=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("slots", "rope", "decode", "decode", "prompt", "prompt"))
    page = rng.choice((16, 16, 32, 64, 128))
    kv_heads = rng.choice((1, 2, 4, 5, 8))
    group = rng.choice((1, 2, 3, 4, 6, 8, 16))
    while kv_heads * group > 64:
        group = rng.choice((1, 2, 3, 4, 6, 8))
    q_heads = kv_heads * group
    dim = rng.choice((64, 80, 96, 128, 128, 256))
    b16 = rng.choice(("bf16", "bf16", "f16"))
    if op == "slots":
        requests = _log(rng, 1, 1000)
        step = rng.random() < 0.5
        hi = 1 if step else _log(rng, 2, max(3, min(4096, 300000 // requests)))
        return dict(op=op, requests=requests, new_lo=1 if step else rng.choice((0, 1)), new_hi=hi, ctx_lo=0, ctx_hi=_log(rng, 1, 16384), page=page,
                    pad=rng.choice((0, 0, rng.randrange(1, 100))), short=rng.choice((0, 0, 0, rng.randrange(1, 8))))
    if op == "rope":
        return dict(op=op, tokens=_log(rng, 1, max(2, 8192 * 32 * 128 // max(32 * 128, q_heads * dim))), q_heads=q_heads, kv_heads=kv_heads, dim=dim,
                    rot=rng.choice((dim, dim, dim // 2, 32)), interleaved=rng.random() < 0.4, norm=rng.random() < 0.5,
                    act=rng.choice(("f32", b16)), out=rng.choice(("f32", b16)), cache=b16, page=page)
    window = rng.choice((0, 0, _log(rng, 64, 4096)))
    sinks = rng.choice((0, 4, rng.randrange(1, 64))) if window else 0
    if op == "decode":
        requests = _log(rng, 1, 256)
        # the plain form reads every page of a padded table: 2^28 elements of the cache at most
        most = min(131085, (1 << 28) // (requests * kv_heads * dim))
        hi = _log(rng, 16, max(17, most))
        act = rng.choice(("f32", b16, b16))
        return dict(op=op, requests=requests, empty=min(requests - 1, rng.choice((0, 0, 1, 3))), len_lo=rng.choice((1, hi, max(1, hi // 2))), len_hi=hi,
                    q_heads=q_heads, kv_heads=kv_heads, dim=dim, window=window, sinks=sinks, act=act, out=act, cache=b16, page=page,
                    heads_first=rng.random() < 0.5, lse=rng.random() < 0.5)
    requests = _log(rng, 1, 16)
    # the plain form keeps every score of a padded batch: 2^29 of them at most
    new_hi = _log(rng, 2, max(3, min(8192, int(math.sqrt((1 << 29) / (requests * q_heads))))))
    ctx_hi = rng.choice((0, 0, _log(rng, 1, max(2, min(32768, (1 << 29) // (requests * q_heads * new_hi))))))
    return dict(op=op, requests=requests, new_lo=rng.choice((1, new_hi, max(1, new_hi // 2))), new_hi=new_hi, ctx_lo=0, ctx_hi=ctx_hi, q_heads=q_heads,
                kv_heads=kv_heads, dim=dim, window=window, sinks=sinks, dtype=b16, page=page, heads_first=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------------------------ lengths


def _spread(n, lo, hi, offset=0.0):
    """n whole numbers that fill [lo, hi] evenly, in a fixed mixed order; the first is hi."""
    return [int(round(hi - (hi - lo) * ((i * GOLDEN + (offset if i else 0.0)) % 1.0))) for i in range(n)]


def _lengths(case):
    """[(tokens in the cache before the step, new tokens)] of a case's requests, before the seed puts them in order."""
    if case["op"] == "rope":
        return []
    if case["op"] == "decode":
        n = case["requests"] - case["empty"]
        return [(v - 1, 1) for v in _spread(n, case["len_lo"], case["len_hi"])] + [(0, 0)] * case["empty"]
    n = case["requests"]
    return list(zip(_spread(n, case["ctx_lo"], case["ctx_hi"], 0.37), _spread(n, case["new_lo"], case["new_hi"])))


def _visible(length, window, sinks):
    """Keys that the last of `length` tokens sees."""
    return length if not window or length <= window + sinks else window + sinks


def work(case):
    lens = _lengths(case)
    if case["op"] == "slots":
        b, p = len(lens), case["page"]
        added = sum(-(-(c + n) // p) + -c // p for c, n in lens)
        used = sum(-(-(c + n) // p) - c // p for c, n in lens if n)
        tokens = sum(n for _, n in lens) + case["pad"]
        # lengths in and out, their running sum, pages taken and entered, the pages of the new tokens, positions, slots
        return {"bytes": 4 * (4 * b + 1) + 8 * added + 4 * used + 12 * tokens, "flops": 0}
    d = case["dim"]
    if case["op"] == "rope":
        t, hq, hk = case["tokens"], case["q_heads"], case["kv_heads"]
        values = t * d * ((hq + 2 * hk) * SIZES[case["act"]] + hq * SIZES[case["out"]] + 2 * hk * SIZES[case["cache"]])
        flops = t * (hq + hk) * (3 * case["rot"] + (4 * d if case["norm"] else 0))
        return {"bytes": values + 12 * t + t * case["rot"] * 4 + (8 * d if case["norm"] else 0), "flops": flops}
    hq, hk = case["q_heads"], case["kv_heads"]
    if case["op"] == "decode":
        seen = sum(_visible(c + n, case["window"], case["sinks"]) for c, n in lens)
        rows = len(lens) * hq * (d * (SIZES[case["act"]] + SIZES[case["out"]]) + (4 if case["lse"] else 0))
        return {"bytes": seen * hk * d * 2 * SIZES[case["cache"]] + rows + 4 * len(lens), "flops": 4 * seen * hq * d}
    w, s = case["window"], case["sinks"]
    pairs = sum(sum(_visible(c + i + 1, w, s) for i in range(n)) for c, n in lens)
    keys = 0
    for c, n in lens:  # the keys that any new token sees
        first = max(0, c + 1 - w) if w else 0
        keys += (c + n - first + min(s, first)) if n else 0
    tokens = sum(n for _, n in lens)
    return {"bytes": 2 * (2 * keys * hk * d + 2 * tokens * hq * d), "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------------------------------------------------------------- inputs


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape, dtype=torch.float32, scale=1.0):
    return torch.empty(*shape, dtype=dtype, device="cuda").normal_(0.0, scale, generator=g)


def _tables(positions, rot, base=500000.0):
    """cos and sin of a rotation over positions 0 .. positions - 1, [positions, rot / 2] f32."""
    inv = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).cuda()


def _cache(case, g, pages):
    """Keys and values, [pages, page, kv_heads, dim]; heads_first: the heads of a page lie one after the other in memory."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"]) if case.get("heads_first") else (pages, case["page"], case["kv_heads"], case["dim"])
    k, v = (_normal(g, *shape, dtype=DTYPES[case.get("cache") or case["dtype"]]) for _ in range(2))
    return (k.transpose(1, 2), v.transpose(1, 2)) if case.get("heads_first") else (k, v)


def prepare(case, seed):
    g, rng = _generator(seed), random.Random(seed)
    s = dict(case)
    if case["op"] == "rope":
        t, page = case["tokens"], case["page"]
        a = DTYPES[case["act"]]
        pages = -(-t // page) + 16
        # the tokens of one step come from several requests: runs of consecutive positions, in slots all over the cache
        start = torch.randint(0, 8192, (-(-t // 64),), generator=g, device="cuda")
        s["positions"] = (start.repeat_interleave(64)[:t] + torch.arange(t, device="cuda") % 64).to(torch.int32)
        s["slots"] = torch.randperm(pages * page, generator=g, device="cuda")[:t].contiguous()
        # q, k and v as one projection leaves them: side by side in a row
        rows = _normal(g, t, (case["q_heads"] + 2 * case["kv_heads"]) * case["dim"], dtype=a, scale=1.5)
        nq, nk = case["q_heads"] * case["dim"], case["kv_heads"] * case["dim"]
        s["q"] = rows[:, :nq].view(t, case["q_heads"], case["dim"])
        s["k"] = rows[:, nq:nq + nk].view(t, case["kv_heads"], case["dim"])
        s["v"] = rows[:, nq + nk:].view(t, case["kv_heads"], case["dim"])
        s["cos"], s["sin"] = _tables(8192 + 64, case["rot"])
        s["qw"], s["kw"] = (1.0 + 0.1 * _normal(g, case["dim"]) for _ in range(2)) if case["norm"] else (None, None)
        s["k_cache"], s["v_cache"] = _cache(case, g, pages)
        return s
    lens = _lengths(case)
    rng.shuffle(lens)
    page = case["page"]
    ctx, new = [c for c, _ in lens], [n for _, n in lens]
    held = [-(-c // page) for c in ctx]
    full = [-(-(c + n) // page) for c, n in lens]
    width = max(1, max(full))
    if case["op"] == "slots":
        spare = max(0, sum(full) - sum(held) - case["short"]) + (0 if case["short"] else 100)
        order = torch.randperm(sum(held) + spare + 1, generator=g, device="cuda").to(torch.int32)
        s["ctx"], s["new"] = _ints(ctx), _ints(new)
        s["free"], s["free_count"] = order[sum(held):].contiguous(), _ints([spare])
        s["table"] = _fill_table(held, width, order)
        s["total"] = sum(new) + case["pad"]
        return s
    pages = sum(full) + 1
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    s["table"] = _fill_table(full, width, order)
    s["lens"] = _ints([c + n for c, n in lens])
    s["k_cache"], s["v_cache"] = _cache(case, g, pages)
    if case["op"] == "decode":
        s["q"] = _normal(g, len(lens), case["q_heads"], case["dim"], dtype=DTYPES[case["act"]], scale=1.5)
        return s
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    s["cu"] = _ints(cu)
    s["most"] = max(new)
    s["q"] = _normal(g, cu[-1], case["q_heads"], case["dim"], dtype=DTYPES[case["dtype"]], scale=1.5)
    return s


def _fill_table(held, width, order):
    """Block tables: row b has held[b] pages of `order`, one request after the other, and -1 behind them."""
    held = _ints(held, torch.int64)
    first = held.cumsum(0) - held
    col = torch.arange(width, device="cuda")
    return torch.where(col < held[:, None], order[(first[:, None] + col).clamp(max=order.numel() - 1)], -1).to(torch.int32)


# --------------------------------------------------------------------------------------------------------------- plain forms


def _plain_slots(s):
    ctx, new, page = s["ctx"].long(), s["new"].long(), s["page"]
    width, total = s["table"].shape[1], s["total"]
    held, want = (ctx + page - 1) // page, (ctx + new + page - 1) // page
    add = want.clamp(max=width) - held.clamp(max=width)
    taken = add.cumsum(0)
    col = torch.arange(width, device="cuda")
    at = (taken - add)[:, None] + col - held[:, None]
    fresh = (col >= held[:, None]) & (col < want[:, None])
    count = s["free_count"].long()
    page_at = s["free"][(count - 1 - at).clamp(0, s["free"].numel() - 1)]
    table = torch.where(fresh, torch.where(at < count, page_at, -1), s["table"])
    cu = torch.nn.functional.pad(new.cumsum(0), (1, 0))
    t = torch.arange(total, device="cuda")
    req = (torch.searchsorted(cu, t, right=True) - 1).clamp(max=new.numel() - 1)
    live = t < cu[-1]
    pos = torch.where(live, ctx[req] + t - cu[req], 0)
    held_page = table[req, (pos // page).clamp(max=width - 1)].long()
    slot = torch.where(live & (held_page >= 0) & (pos // page < width), held_page * page + pos % page, -1)
    wanted = (want - held).sum()
    got = torch.minimum(taken[-1], count[0])
    left = torch.stack((count[0] - got, wanted - got))
    return table, (ctx + new).int(), cu.int(), pos.int(), slot, left.int()


def _turn(x, cos, sin, interleaved):
    rot = 2 * cos.shape[-1]
    r, rest = x[..., :rot], x[..., rot:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., : rot // 2], r[..., rot // 2:])
    c, d = a * cos - b * sin, b * cos + a * sin
    r = torch.stack((c, d), -1).flatten(-2) if interleaved else torch.cat((c, d), -1)
    return torch.cat((r, rest), -1)


def _plain_rope(s):
    q, k = s["q"].float(), s["k"].float()
    if s["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * s["qw"]
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + EPS) * s["kw"]
    cos, sin = (s[n][s["positions"]][:, None] for n in ("cos", "sin"))
    q, k = (_turn(x, cos, sin, s["interleaved"]) for x in (q, k))
    kc, vc = s["k_cache"], s["v_cache"]
    at, off = s["slots"] // s["page"], s["slots"] % s["page"]
    kc[at, off] = k.to(kc.dtype)
    vc[at, off] = s["v"].float().to(vc.dtype)
    return q.to(DTYPES[s["out"]]), kc, vc


def _gathered(s):
    """The pages of each request in a row, [requests, kv_heads, tokens, dim] f32."""
    at = s["table"].clamp(min=0).long()
    return (c[at].flatten(1, 2).transpose(1, 2).float() for c in (s["k_cache"], s["v_cache"]))


def _seen(pos, key, window, sinks):
    m = key <= pos
    return m & ((pos - key < window) | (key < sinks)) if window else m


def _plain_decode(s):
    b, hq, d = s["q"].shape
    k, v = _gathered(s)
    q = s["q"].float().view(b, s["kv_heads"], -1, d) * d ** -0.5
    x = q @ k.transpose(2, 3)
    key = torch.arange(k.shape[2], device="cuda")
    seen = _seen(s["lens"].long()[:, None] - 1, key, s["window"], s["sinks"])[:, None, None]
    x = x.masked_fill_(~seen, -math.inf)
    most = x.amax(-1, keepdim=True)
    e = torch.exp_(x.sub_(most.clamp(min=-1e30)))
    total = e.sum(-1, keepdim=True)
    out = torch.where(total > 0, e @ v / total, 0.0).reshape(b, hq, d).to(DTYPES[s["out"]])
    return (out, (most + total.log()).reshape(b, hq)) if s["lse"] else out


def _plain_prompt(s):
    t, hq, d = s["q"].shape
    cu, lens, hk = s["cu"].long(), s["lens"].long(), s["kv_heads"]
    k, v = _gathered(s)
    i = torch.arange(s["most"], device="cuda")
    n = cu[1:] - cu[:-1]
    q = s["q"][(cu[:-1, None] + i).clamp(max=t - 1)].float()  # [requests, most, q_heads, dim]
    q = q.view(n.numel(), -1, hk, hq // hk, d).permute(0, 2, 3, 1, 4) * d ** -0.5
    x = q @ k.transpose(2, 3)[:, :, None]
    key = torch.arange(k.shape[2], device="cuda")
    pos = (lens - n)[:, None] + i
    x = x.masked_fill_(~_seen(pos[:, :, None], key, s["window"], s["sinks"])[:, None, None], -math.inf)
    e = torch.exp_(x.sub_(x.amax(-1, keepdim=True).clamp(min=-1e30)))
    total = e.sum(-1, keepdim=True)
    out = (e @ v[:, :, None] / total).permute(0, 3, 1, 2, 4)  # [requests, most, kv_heads, group, dim]
    j = torch.arange(t, device="cuda")
    req = torch.searchsorted(cu, j, right=True) - 1
    return out[req, j - cu[req]].reshape(t, hq, d).to(s["q"].dtype)


def run(s):
    if not own:
        return {"slots": _plain_slots, "rope": _plain_rope, "decode": _plain_decode, "prompt": _plain_prompt}[s["op"]](s)
    from boostr_b200 import attention

    if s["op"] == "slots":
        return tuple(attention.paged_slots(s["ctx"], s["new"], s["table"], s["page"], s["free"], s["free_count"], s["total"]))
    if s["op"] == "rope":
        q = attention.rope_append(s["q"], s["k"], s["v"], s["positions"], s["cos"], s["sin"], s["k_cache"], s["v_cache"], s["slots"],
                                  q_weight=s["qw"], k_weight=s["kw"], eps=EPS, interleaved=s["interleaved"], out_dtype=DTYPES[s["out"]])
        return q, s["k_cache"], s["v_cache"]
    if s["op"] == "decode":
        return attention.paged_decode(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], window=s["window"], sinks=s["sinks"],
                                      return_lse=s["lse"])
    return attention.paged_prompt(s["q"], s["cu"], s["k_cache"], s["v_cache"], s["table"], s["lens"], window=s["window"], sinks=s["sinks"])


# ------------------------------------------------------------------------------------------------------------ 64-bit results


def exact(case, seed):
    """The operators' definitions, a request and a head at a time in 64 bits; slots are whole numbers and need none."""
    if case["op"] == "slots":
        return None
    s = prepare(case, seed)
    f64 = dict(dtype=torch.float64, device="cuda")
    if case["op"] == "rope":
        half = s["rot"] // 2
        turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()][:, None]
        i = torch.arange(half, device="cuda")
        re, im = (2 * i, 2 * i + 1) if s["interleaved"] else (i, i + half)
        turned = []
        for x, w in ((s["q"].double(), s["qw"]), (s["k"].double(), s["kw"])):
            if s["norm"]:
                x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / s["dim"] + EPS) * w.double()
            z = torch.complex(x[..., re], x[..., im]) * turn
            x[..., re], x[..., im] = z.real, z.imag
            turned.append(x)
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        kc[s["slots"] // s["page"], s["slots"] % s["page"]] = turned[1]
        vc[s["slots"] // s["page"], s["slots"] % s["page"]] = s["v"].double()
        return turned[0], kc, vc
    rows, hq, d = s["q"].shape
    out = torch.zeros(rows, hq, d, **f64)
    lse = torch.full((rows, hq), -math.inf, **f64)
    lens = s["lens"].tolist()
    cu = s["cu"].tolist() if case["op"] == "prompt" else list(range(rows + 1))
    for r, length in enumerate(lens):
        n = min(length, cu[r + 1] - cu[r])  # a request of no tokens sees nothing
        if not n:
            continue
        mine = slice(cu[r], cu[r] + n)
        at = s["table"][r, : -(-length // s["page"])].long()
        k, v = (c[at].reshape(-1, s["kv_heads"], d)[:length].double() for c in (s["k_cache"], s["v_cache"]))
        key = torch.arange(length, device="cuda")
        gap = torch.arange(length - n, length, device="cuda")[:, None] - key
        hidden = gap < 0
        if s["window"]:
            hidden |= (gap >= s["window"]) & (key >= s["sinks"])
        for h in range(hq):
            kv = h // (hq // s["kv_heads"])
            x = torch.einsum("qd,kd->qk", s["q"][mine, h].double(), k[:, kv]) / math.sqrt(d)
            x[hidden] = -math.inf
            lse[mine, h] = torch.logsumexp(x, 1)
            out[mine, h] = torch.exp(x - lse[mine, h, None]) @ v[:, kv]
    return (out, lse) if s.get("lse") else out
