"""Workloads of the generation operators: appending keys and values to a paged cache with the position rotation, attention
over packed prompts, and attention of one new token per sequence over the paged cache.

`own` selects who computes a pass: False, elementary torch operations in 32 bits; True, the library's entry points.
`exact` states the same definitions once more in 64 bits."""
import math
import random

import torch

own = False

DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"bf16": 2, "f32": 4}


# ---- the cases ------------------------------------------------------------------------------------------------------
# op        "append", "prompt" or "decode"
# seqs      sequences; low, high: their lengths are spread over [low, high] (over the logarithm), mix: which lengths exactly
# past      append: tokens in the cache before the new ones; prompt: keys before the first query (a prompt taken in parts)
# heads, kv_heads, dim, page, type; rotary, pairs (append): rotated dimensions, and whether neighbours or halves are paired
# spare     rows of the token buffers behind the last sequence (a batch padded to a fixed size)
def listed():
    return [
        # one new token of one conversation on the encoder configuration's heads: what a call costs at least
        dict(name="append_one_token", op="append", seqs=1, low=1, high=1, mix=1, past=77, heads=8, kv_heads=8, dim=64, page=16, type="bf16",
             rotary=64, pairs=False, spare=0),
        # one decoding step of a batch, padded to a fixed number of rows as a captured step is
        dict(name="append_step_of_a_batch", op="append", seqs=120, low=1, high=1, mix=2, past=900, heads=32, kv_heads=8, dim=128, page=16,
             type="bf16", rotary=128, pairs=False, spare=8),
        # a large packed batch of prompts enters the cache
        dict(name="append_packed_prompts", op="append", seqs=24, low=16, high=2500, mix=3, past=0, heads=32, kv_heads=8, dim=128, page=64,
             type="bf16", rotary=128, pairs=False, spare=100),
        # fp32, neighbours paired, half of each head rotated, a head size that is no power of two
        dict(name="append_prompts_f32", op="append", seqs=3, low=200, high=900, mix=4, past=33, heads=8, kv_heads=2, dim=96, page=32,
             type="f32", rotary=48, pairs=True, spare=0),
        # a single short prompt: latency
        dict(name="prompt_one_short", op="prompt", seqs=1, low=40, high=40, mix=5, past=0, heads=8, kv_heads=8, dim=64, type="bf16", causal=True,
             spare=0),
        # the encoder configuration's batch (512 of up to 128 tokens, 8 heads of 64) with the lengths it really has, all keys visible
        dict(name="prompt_encoder_ragged", op="prompt", seqs=512, low=24, high=128, mix=6, past=0, heads=8, kv_heads=8, dim=64, type="bf16",
             causal=False, spare=0),
        # an ordinary packed batch of prompts, grouped heads
        dict(name="prompt_packed_causal", op="prompt", seqs=24, low=5, high=2500, mix=7, past=0, heads=32, kv_heads=8, dim=128, type="bf16",
             causal=True, spare=31),
        # one long prompt: tensor-core work
        dict(name="prompt_one_long", op="prompt", seqs=1, low=8192, high=8192, mix=8, past=0, heads=32, kv_heads=8, dim=128, type="bf16",
             causal=True, spare=0),
        # fp32: the second part of two prompts, whose first parts' keys come first
        dict(name="prompt_second_part_f32", op="prompt", seqs=2, low=250, high=700, mix=9, past=500, heads=8, kv_heads=2, dim=64, type="f32",
             causal=True, spare=0),
        # fp32, a few short conversations
        dict(name="decode_few_short_f32", op="decode", seqs=6, low=1, high=400, mix=10, heads=8, kv_heads=2, dim=64, page=16, type="f32", spare=0),
        # one long conversation: only a split over the cache's length fills the GPU
        dict(name="decode_one_long", op="decode", seqs=1, low=65543, high=65543, mix=11, heads=32, kv_heads=8, dim=128, page=16, type="bf16",
             spare=0),
        # a large serving batch of very different lengths
        dict(name="decode_large_batch", op="decode", seqs=160, low=100, high=8100, mix=12, heads=32, kv_heads=8, dim=128, page=64, type="bf16",
             spare=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.499))))))


MOST = {"append": 17000 * 48 * 128, "prompt": 32 * 8192 * 4097 * 128.0, "decode": 400000 * 8 * 128}


def _cost(c):
    n, f = lengths(c), 1 if c["type"] == "bf16" else 2
    if c["op"] == "append":
        return f * sum(n) * (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
    if c["op"] == "decode":
        return f * sum(n) * c["kv_heads"] * c["dim"]
    return 8 * (f - 1) * _pairs(c) * c["heads"] * c["dim"] + _pairs(c) * c["heads"] * c["dim"]


def draw(rng):
    while True:
        op = rng.choice(["append", "prompt", "decode"])
        group, kv = rng.choice([1, 1, 2, 3, 4, 4, 5, 7, 8, 16]), rng.choice([1, 2, 4, 8, 8, 16])
        c = dict(op=op, heads=group * kv, kv_heads=kv, dim=rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 192, 256]), mix=rng.randrange(1 << 20),
                 type=rng.choice(["bf16", "bf16", "bf16", "f32"]), spare=rng.choice([0, 0, 3, 64]))
        if op == "append":
            seqs, new = _log(rng, 1, 256), rng.choice([True, False])
            high = 1 if new else _log(rng, 1, 4096)
            c.update(seqs=seqs, low=1, high=high, past=rng.choice([0, 1, 500, 7000]), page=rng.choice([1, 8, 16, 32, 48, 64, 128, 256]),
                     rotary=rng.choice([c["dim"], c["dim"], c["dim"] // 2, 0]), pairs=rng.choice([True, False]))
        elif op == "prompt":
            high = _log(rng, 1, 8192)
            c.update(seqs=_log(rng, 1, 512), low=_log(rng, 1, high), high=high, past=rng.choice([0, 0, 0, 1, 100, 1111]), causal=rng.choice([True, True, False]))
        else:
            high = _log(rng, 1, 65536)
            c.update(seqs=_log(rng, 1, 256), low=_log(rng, 1, high), high=high, page=rng.choice([1, 8, 16, 32, 48, 64, 128, 256]))
        if c["heads"] > 64 or _cost(c) > MOST[op]:
            continue
        if op == "prompt" and c["heads"] * c["high"] * (c["high"] + c["past"]) > 32 * 8192 * 8192:
            continue
        if op == "prompt" and c["seqs"] > 64 and c["high"] > 512:   # the plain form goes sequence by sequence
            continue
        return c


def lengths(c):
    """Length of each sequence: new tokens (append), queries (prompt), tokens in the cache (decode)."""
    rng = random.Random(c["mix"])
    return [_log(rng, c["low"], c["high"]) for _ in range(c["seqs"])]


def _pairs(c):
    """(query, key) pairs that a prompt's mask leaves."""
    if c["causal"]:
        return sum(n * c["past"] + n * (n + 1) // 2 for n in lengths(c))
    return sum(n * (n + c["past"]) for n in lengths(c))


def work(case):
    c, n, es = case, lengths(case), SIZE[case["type"]]
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    if c["op"] == "append":      # q, k, v read; q, k, v written; one row of cosines and sines for each token
        t = sum(n)
        return {"bytes": 2.0 * t * (h + 2 * kv) * d * es + t * c["rotary"] * 4.0, "flops": 3.0 * t * (h + kv) * c["rotary"]}
    if c["op"] == "prompt":
        t = sum(n)
        return {"bytes": es * d * (2.0 * t * h + 2.0 * kv * (t + c["seqs"] * c["past"])), "flops": 4.0 * d * h * _pairs(c)}
    return {"bytes": es * d * (2.0 * kv * sum(n) + 2.0 * h * c["seqs"]) + 4.0 * sum(-(-x // c["page"]) for x in n), "flops": 4.0 * d * h * sum(n)}


# ---- what a program has in hand before the call -----------------------------------------------------------------------
def _normal(gen, shape, dtype, std=1.0):
    return torch.randn(shape, generator=gen, device=DEV, dtype=dtype).mul_(std)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _starts(n):
    s = [0]
    for x in n:
        s.append(s[-1] + x)
    return s


def _cache(c, gen, total):
    """A paged cache [pages, page, kv_heads, dim] for `total` tokens per sequence: pages in any order, a few that nobody owns."""
    per = [-(-x // c["page"]) for x in total]
    pages = sum(per) + 3
    order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    width = max(per)
    at = torch.arange(width, device=DEV)
    own_pages = at[None, :] < torch.tensor(per, device=DEV)[:, None]
    table = torch.zeros((c["seqs"], width), dtype=torch.int32, device=DEV)   # entries behind a sequence's last page stay 0
    table[own_pages] = order[: sum(per)]
    shape = (pages, c["page"], c["kv_heads"], c["dim"])
    return _normal(gen, shape, TYPES[c["type"]]), _normal(gen, shape, TYPES[c["type"]]), table


def prepare(case, seed):
    c, n, dt = case, lengths(case), TYPES[case["type"]]
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    h, kv, d, t = c["heads"], c["kv_heads"], c["dim"], sum(n) + c["spare"]
    s = {"case": c, "lengths": n}
    if c["op"] == "append":
        qkv = _normal(gen, (t, h + 2 * kv, d), dt)   # the output of one projection: q, k and v are column blocks of it
        s["q"], s["k"], s["v"] = qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:]
        past = [max(0, c["past"] - 13 * (i % 37)) for i in range(c["seqs"])]
        total = [p + x for p, x in zip(past, n)]
        s["cache_k"], s["cache_v"], s["table"] = _cache(c, gen, total)
        s["lens"], s["starts"] = _ints(total), _ints(_starts(n))
        s["new"] = sum(n)
        s["q_out"] = torch.zeros((t, h, d), dtype=dt, device=DEV)
        r = c["rotary"] // 2
        if r:
            angle = torch.arange(max(total), dtype=torch.float64, device=DEV)[:, None] * 10000.0 ** (-torch.arange(r, dtype=torch.float64, device=DEV) / r)[None]
            s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    elif c["op"] == "prompt":
        tk = sum(n) + c["seqs"] * c["past"] + c["spare"]
        s["q"] = _normal(gen, (t, h, d), dt, 1.5)
        s["k"], s["v"] = _normal(gen, (tk, kv, d), dt), _normal(gen, (tk, kv, d), dt)
        s["q_at"], s["k_at"] = _starts(n), _starts([x + c["past"] for x in n])
        s["starts"], s["starts_k"] = _ints(s["q_at"]), _ints(s["k_at"])
        s["y"] = torch.zeros((t, h, d), dtype=dt, device=DEV)
    else:
        s["cache_k"], s["cache_v"], s["table"] = _cache(c, gen, n)
        s["lens"] = _ints(n + [0] * c["spare"])
        s["table"] = torch.cat([s["table"], s["table"].new_zeros((c["spare"], s["table"].shape[1]))])
        s["q"] = _normal(gen, (c["seqs"] + c["spare"], h, d), dt, 1.5)
        s["y"] = torch.zeros_like(s["q"])
    if own:
        _handles(s)
    return s


_context = None


def _handles(s):
    """The context of the process, and the views and plans that a program makes once."""
    global _context
    from sofie_b200.ops import Context, PagedAttentionPlan, PagedKV, PromptAttentionPlan
    if _context is None:
        _context = Context(0)
    c, dt = s["case"], TYPES[s["case"]["type"]]
    s["ctx"] = _context
    if c["op"] == "prompt":
        s["plan"] = PromptAttentionPlan(_context, c["heads"], c["kv_heads"], c["dim"], dt, causal=c["causal"])
    else:
        s["kv"] = PagedKV(s["cache_k"], s["cache_v"], s["table"], s["lens"])
        if c["op"] == "decode":
            s["plan"] = PagedAttentionPlan(_context, c["heads"], c["kv_heads"], c["dim"], dt)


# ---- one pass ---------------------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        if op == "append":
            s["ctx"].kv_append(s["k"], s["v"], s["kv"], s["starts"], cos=s.get("cos"), sin=s.get("sin"), interleaved=s["case"]["pairs"], q=s["q"],
                               q_out=s["q_out"])
            return {"q": s["q_out"], "cache_k": s["cache_k"], "cache_v": s["cache_v"]}
        if op == "prompt":
            s["plan"].enqueue(s["q"], s["k"], s["v"], s["y"], s["starts"], s["starts_k"])
        else:
            s["plan"].enqueue(s["q"], s["kv"], s["y"])
        return s["y"]
    return {"append": _append, "prompt": _prompt, "decode": _decode}[op](s)


def _turn(x, cos, sin, rotary, pairs):
    """The first `rotary` dimensions of x [tokens, heads, dim] turned by the tokens' angles, in 32 bits."""
    if not rotary:
        return x
    a, rest = x[..., :rotary].float(), x[..., rotary:]
    c, sn = cos[:, None], sin[:, None]
    if pairs:
        u, w = a[..., 0::2], a[..., 1::2]
        a = torch.stack([u * c - w * sn, w * c + u * sn], dim=-1).flatten(-2)
    else:
        u, w = a[..., : rotary // 2], a[..., rotary // 2:]
        a = torch.cat([u * c - w * sn, w * c + u * sn], dim=-1)
    return torch.cat([a.to(x.dtype), rest], dim=-1)


def _append(s):
    c, new = s["case"], s["new"]
    n = s["starts"][1:] - s["starts"][:-1]
    seq = torch.repeat_interleave(torch.arange(c["seqs"], device=DEV), n, output_size=new)
    at = torch.arange(new, device=DEV) - s["starts"][seq] + (s["lens"] - n)[seq]
    page, slot = s["table"][seq, at // c["page"]].long(), at % c["page"]
    cos, sin = (s["cos"][at], s["sin"][at]) if c["rotary"] else (None, None)
    s["q_out"][:new] = _turn(s["q"][:new], cos, sin, c["rotary"], c["pairs"])
    s["cache_k"][page, slot] = _turn(s["k"][:new], cos, sin, c["rotary"], c["pairs"])
    s["cache_v"][page, slot] = s["v"][:new]
    return {"q": s["q_out"], "cache_k": s["cache_k"], "cache_v": s["cache_v"]}


def _weights(scores):
    """Softmax over the last axis, 0 where a row has nothing to look at (every score -inf)."""
    e = (scores - scores.amax(-1, keepdim=True).clamp(min=-1e30)).exp()
    return e / e.sum(-1, keepdim=True).clamp(min=1e-30)


def _prompt(s):
    c = s["case"]
    kv, g, d = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    for i in range(c["seqs"]):
        (a, b), (e, f) = s["q_at"][i:i + 2], s["k_at"][i:i + 2]
        q = s["q"][a:b].float().view(b - a, kv, g, d).permute(1, 2, 0, 3).reshape(kv, g * (b - a), d)
        k, v = s["k"][e:f].float().permute(1, 2, 0), s["v"][e:f].float().permute(1, 0, 2)
        scores = ((q @ k) * d ** -0.5).view(kv, g, b - a, f - e)
        if c["causal"]:
            scores.masked_fill_(torch.ones((b - a, f - e), dtype=torch.bool, device=DEV).triu(1 + (f - e) - (b - a)), -math.inf)
        y = _weights(scores).view(kv, g * (b - a), f - e) @ v
        s["y"][a:b] = y.view(kv, g, b - a, d).permute(2, 0, 1, 3).reshape(b - a, c["heads"], d).to(s["y"].dtype)
    return s["y"]


def _decode(s):
    c = s["case"]
    kv, g, d = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    n = s["q"].shape[0]
    table = s["table"].long()
    k = s["cache_k"][table].view(n, -1, kv, d).permute(0, 2, 3, 1).float()   # pages in the sequence's order, padded to the longest
    scores = (s["q"].float().view(n, kv, g, d) @ k) * d ** -0.5
    del k
    scores.masked_fill_((torch.arange(scores.shape[-1], device=DEV) >= s["lens"][:, None])[:, None, None], -math.inf)
    v = s["cache_v"][table].view(n, -1, kv, d).permute(0, 2, 1, 3).float()
    s["y"].copy_((_weights(scores) @ v).view(n, c["heads"], d))
    return s["y"]


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------
def exact(case, seed):
    c, s = case, prepare(case, seed)
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    if c["op"] == "append":
        out = {x: s[y].double() for x, y in (("q", "q_out"), ("cache_k", "cache_k"), ("cache_v", "cache_v"))}
        starts, lens, table, r = s["starts"].tolist(), s["lens"].tolist(), s["table"].tolist(), c["rotary"] // 2
        rows, where, slots = [], [], []
        for b in range(c["seqs"]):
            for i in range(starts[b], starts[b + 1]):
                p = lens[b] - (starts[b + 1] - i)
                rows.append(p), where.append(table[b][p // c["page"]]), slots.append(p % c["page"])
        rows, where, slots = (torch.tensor(v, device=DEV) for v in (rows, where, slots))

        def turned(x):
            x = x[: s["new"]].double()
            if r:
                first = torch.arange(r, device=DEV) * 2 if c["pairs"] else torch.arange(r, device=DEV)
                second = first + (1 if c["pairs"] else r)
                z = torch.complex(x[:, :, first], x[:, :, second]) * torch.complex(s["cos"].double(), s["sin"].double())[rows][:, None]
                x[:, :, first], x[:, :, second] = z.real, z.imag
            return x
        out["q"][: s["new"]] = turned(s["q"])
        out["cache_k"][where, slots] = turned(s["k"])
        out["cache_v"][where, slots] = s["v"][: s["new"]].double()
        return out
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b in range(c["seqs"]):
        if c["op"] == "prompt":
            (q0, q1), (k0, k1) = s["q_at"][b:b + 2], s["k_at"][b:b + 2]
            q, k, v = s["q"][q0:q1].double(), s["k"][k0:k1].double(), s["v"][k0:k1].double()
        else:
            q0, q1, n = b, b + 1, s["lengths"][b]
            pages = s["table"][b, : -(-n // c["page"])].long()
            q, k, v = s["q"][b:b + 1].double(), s["cache_k"][pages].flatten(0, 1)[:n].double(), s["cache_v"][pages].flatten(0, 1)[:n].double()
        for i in range(h):
            z = torch.einsum("qd,kd->qk", q[:, i], k[:, i * kv // h]) / math.sqrt(d)
            if c["op"] == "prompt" and c["causal"]:
                last = torch.arange(q1 - q0, device=DEV) + (k1 - k0) - (q1 - q0)
                z = torch.where(torch.arange(k1 - k0, device=DEV)[None] <= last[:, None], z, -math.inf)
            out[q0:q1, i] = torch.softmax(z, -1) @ v[:, i * kv // h]
    return out
