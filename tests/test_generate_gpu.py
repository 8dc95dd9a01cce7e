"""The generation operators on the GPU against their statement in 64 bits (tests/generate_ref.py): appending to a paged
cache with the rotation, attention over packed prompts, attention over the cache, and a run of the three together."""
import math

import pytest
import torch

import generate_ref as ref
from sofie_b200 import lib as L

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture()
def ctx(b200_lib):
    from sofie_b200.ops import Context
    c = Context(0)
    yield c
    c.close()


def gen_of(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def normal(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def tables(positions, rotary):
    r = rotary // 2
    ang = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * 10000.0 ** (-torch.arange(r, dtype=torch.float64, device=DEV) / max(r, 1))[None]
    return ang.cos().float(), ang.sin().float()


# ---- append ---------------------------------------------------------------------------------------------------------
APPEND = [
    # heads, kv_heads, dim, rotary, interleaved, page_size, [(past, new)], wide rows
    (8, 8, 64, 64, False, 16, [(77, 1)], False),
    (32, 8, 128, 128, False, 16, [(0, 5), (31, 1), (15, 17), (0, 0), (100, 33)], True),
    (6, 2, 96, 48, True, 32, [(0, 40), (7, 100)], False),
    (5, 1, 80, 40, False, 1, [(3, 9), (0, 1)], True),
    (4, 4, 256, 256, True, 48, [(47, 2), (48, 50)], False),
    (3, 3, 10, 6, False, 7, [(5, 20), (0, 3)], True),
    (2, 1, 9, 2, True, 5, [(0, 11)], False),
    (0, 4, 64, 0, False, 128, [(120, 20), (0, 256)], False),
    (64, 1, 192, 96, False, 256, [(255, 1), (256, 1), (0, 1)], True),
]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append(ctx, case, dtype):
    from sofie_b200.ops import PagedKV
    heads, kvh, dim, rotary, inter, size, seqs, wide = APPEND[case]
    g = gen_of(case)
    new, lens = [n for _, n in seqs], [p + n for p, n in seqs]
    cu = offsets(new)
    rows = cu[-1] + 3   # three rows that belong to nobody
    if wide:
        allq = normal(g, (rows, heads + 2 * kvh, dim), dtype)
        q, k, v = allq[:, :heads], allq[:, heads:heads + kvh], allq[:, heads + kvh:]
    else:
        q, k, v = normal(g, (rows, heads, dim), dtype), normal(g, (rows, kvh, dim), dtype), normal(g, (rows, kvh, dim), dtype)
    table, pages = ref.make_pages(lens, size, g)
    ck, cv = normal(g, (pages, size, kvh, dim), dtype), normal(g, (pages, size, kvh, dim), dtype)
    want_k, want_v = ck.double(), cv.double()
    tol_k = torch.zeros_like(want_k)
    cos, sin = tables(max(lens) + 1, rotary)
    pos = torch.tensor([p + i for p, n in seqs for i in range(n)], device=DEV, dtype=torch.long)
    seq = torch.tensor([b for b, n in enumerate(new) for _ in range(n)], device=DEV, dtype=torch.long)
    where, slot = table[seq, pos // size].long(), pos % size
    zk, tk = ref.turn(k[:cu[-1]], pos, cos, sin, rotary, inter)
    want_k[where, slot], tol_k[where, slot] = zk, tk
    want_v[where, slot] = v[:cu[-1]].double()
    q_out = torch.full((rows, heads, dim), 5.0, dtype=dtype, device=DEV) if heads else None
    k_out = torch.full((rows, kvh, dim), 6.0, dtype=dtype, device=DEV)
    kv = PagedKV(ck, cv, table, ints(lens))
    ctx.kv_append(k, v, kv, ints(cu), cos=cos if rotary else None, sin=sin if rotary else None, interleaved=inter, q=q if heads else None,
                  q_out=q_out, k_out=k_out)
    ctx.sync()
    ref.close(ck, want_k, tol_k, "cache k")
    ref.close(cv, want_v, torch.zeros_like(want_v), "cache v")
    ref.close(k_out[:cu[-1]], zk, tk, "k_out")
    assert (k_out[cu[-1]:] == 6.0).all()
    if heads:
        zq, tq = ref.turn(q[:cu[-1]], pos, cos, sin, rotary, inter)
        ref.close(q_out[:cu[-1]], zq, tq, "q_out")
        assert (q_out[cu[-1]:] == 5.0).all()
        # in place: the same bits
        before = q_out.clone()
        q2, k2 = q.contiguous().clone(), k.contiguous().clone()
        ctx.kv_append(k2, v, kv, ints(cu), cos=cos if rotary else None, sin=sin if rotary else None, interleaved=inter, q=q2, q_out=q2, k_out=k2)
        ctx.sync()
        assert torch.equal(q2[:cu[-1]], before[:cu[-1]]) and torch.equal(k2[:cu[-1]], k_out[:cu[-1]])
        assert torch.equal(q2[cu[-1]:], q[cu[-1]:]) and torch.equal(k2[cu[-1]:], k[cu[-1]:])


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_append_one_token_each_with_padding_rows(ctx, dtype):
    """No cu_seqlens: one token per sequence; rows of length 0 are padding and stay as they are.  Heads-first pages."""
    from sofie_b200.ops import PagedKV
    g = gen_of(3)
    lens, size, heads, kvh, dim = [17, 0, 1, 64, 0], 16, 4, 2, 64
    table, pages = ref.make_pages(lens, size, g)
    ck, cv = (normal(g, (pages, kvh, size, dim), dtype).transpose(1, 2) for _ in range(2))
    keep_k, keep_v = ck.clone(), cv.clone()
    q, k, v = normal(g, (5, heads, dim), dtype), normal(g, (5, kvh, dim), dtype), normal(g, (5, kvh, dim), dtype)
    cos, sin = tables(64, dim)
    q_out = torch.full_like(q, 9.0)
    ctx.kv_append(k, v, PagedKV(ck, cv, table, ints(lens)), cos=cos, sin=sin, q=q, q_out=q_out)
    ctx.sync()
    live = [0, 2, 3]
    pos = torch.tensor([lens[b] - 1 for b in live], device=DEV)
    zk, tk = ref.turn(k[live], pos, cos, sin, dim, False)
    zq, tq = ref.turn(q[live], pos, cos, sin, dim, False)
    ref.close(q_out[live], zq, tq)
    assert (q_out[[1, 4]] == 9.0).all()
    for i, b in enumerate(live):
        p, s = int(table[b, (lens[b] - 1) // size]), (lens[b] - 1) % size
        ref.close(ck[p, s], zk[i], tk[i])
        assert torch.equal(cv[p, s], v[b])
        ck[p, s], cv[p, s] = keep_k[p, s], keep_v[p, s]
    assert torch.equal(ck, keep_k) and torch.equal(cv, keep_v)


def test_append_leaves_out_bad_pages_and_positions(ctx):
    """A page that does not exist, a position without a page or without an angle, a length smaller than the new tokens: those
    tokens are left out, the others arrive, and the next sync says so once."""
    from sofie_b200.ops import PagedKV
    g = gen_of(4)
    size, kvh, dim, pages = 4, 2, 32, 6
    lens = [4, 8, 12, 1, 40, 4]
    table = ints([[0, 0], [1, 99], [2, 3], [4, 4], [5, 5], [-7, 0]])
    cu = offsets([1, 1, 1, 3, 1, 1])   # sequence 3 claims one token and brings three
    ck, cv = normal(g, (pages, size, kvh, dim), BF), normal(g, (pages, size, kvh, dim), BF)
    keep = ck.clone()
    k, v = normal(g, (cu[-1], kvh, dim), BF), normal(g, (cu[-1], kvh, dim), BF)
    cos, sin = tables(8, dim)   # sequence 2's token is at position 11
    ctx.kv_append(k, v, PagedKV(ck, cv, table, ints(lens)), ints(cu), cos=cos, sin=sin)
    with pytest.raises(L.SofieB200Error) as e:
        ctx.sync()
    assert e.value.status == L.ERR_DEVICE_INDEX
    ctx.sync()
    assert torch.equal(cv[0, 3], v[0]) and torch.equal(cv[4, 0], v[5])   # sequence 0, and the one token of sequence 3 that has a position
    ck[0, 3], ck[4, 0] = keep[0, 3], keep[4, 0]
    assert torch.equal(ck, keep)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_in_place(ctx, dtype, interleaved):
    """q_out = q and k_out = k, column blocks of one tensor: the bits of the call with outputs of their own, the values untouched."""
    from sofie_b200.ops import PagedKV
    g = gen_of(61)
    for heads, kvh, dim, rotary in ((6, 2, 64, 64), (3, 1, 40, 24), (2, 1, 9, 6)):
        lens, n = [30, 7], 37
        table, pages = ref.make_pages(lens, 16, g)
        cos, sin = tables(40, rotary)
        qkv = normal(g, (n, heads + 2 * kvh, dim), dtype)
        before = qkv.clone()
        caches = []
        for inplace in (False, True):
            ck, cv = (torch.zeros((pages, 16, kvh, dim), dtype=dtype, device=DEV) for _ in range(2))
            q, k, v = qkv[:, :heads], qkv[:, heads:heads + kvh], qkv[:, heads + kvh:]
            qo, ko = (q, k) if inplace else (torch.empty((n, heads, dim), dtype=dtype, device=DEV), torch.empty((n, kvh, dim), dtype=dtype, device=DEV))
            ctx.kv_append(k, v, PagedKV(ck, cv, table, ints(lens)), ints([0, 30, 37]), cos=cos, sin=sin, interleaved=interleaved, q=q, q_out=qo, k_out=ko)
            ctx.sync()
            caches.append((ck, cv, qo.clone(), ko.clone()))
            if not inplace:
                assert torch.equal(qkv, before)
        for a, b in zip(*caches):
            assert torch.equal(a, b)
        assert torch.equal(qkv[:, heads + kvh:], before[:, heads + kvh:])


def test_append_many_sequences(ctx):
    """More sequences than a warp looks at in one round or in two, many of them without a new token."""
    from sofie_b200.ops import PagedKV
    for batch in (33, 1025, 3000):
        g = gen_of(batch)
        new = torch.randint(0, 3, (batch,), generator=g, device=DEV).tolist()
        past = torch.randint(0, 20, (batch,), generator=g, device=DEV).tolist()
        total = [a + b for a, b in zip(past, new)]
        table, pages = ref.make_pages(total, 4, g, width=6)
        cu = offsets(new)
        k, v = normal(g, (cu[-1] + 3, 1, 8), BF), normal(g, (cu[-1] + 3, 1, 8), BF)
        ck, cv = (torch.zeros((pages, 4, 1, 8), dtype=BF, device=DEV) for _ in range(2))
        wk, wv = ck.clone(), cv.clone()
        rows = table.cpu()
        for b in range(batch):
            for i in range(new[b]):
                pos = past[b] + i
                wk[rows[b, pos // 4], pos % 4], wv[rows[b, pos // 4], pos % 4] = k[cu[b] + i], v[cu[b] + i]
        ctx.kv_append(k, v, PagedKV(ck, cv, table, ints(total)), ints(cu))
        ctx.sync()
        assert torch.equal(ck, wk) and torch.equal(cv, wv)


# ---- prompts --------------------------------------------------------------------------------------------------------
PROMPT = [
    # heads, kv_heads, dim, causal, query lengths, key lengths (None: the same)
    (8, 8, 64, True, [40], None),
    (8, 2, 64, True, [1, 127, 128, 129, 0, 255, 257, 2], None),
    (8, 8, 128, True, [300, 1, 64, 65], None),
    (32, 8, 128, True, [700, 33, 1], None),
    (8, 8, 64, False, [128, 100, 24, 1], None),
    (4, 4, 32, True, [200, 5], None),
    (6, 2, 80, True, [77, 130], [200, 131]),
    (7, 1, 96, False, [50, 19], [3, 400]),
    (10, 2, 128, True, [60, 20, 9], [20, 20, 0]),
    (16, 1, 64, True, [9, 300], [500, 300]),
    (64, 1, 128, True, [3, 130], None),
    (4, 1, 256, True, [150, 31], [300, 31]),
    (3, 3, 192, False, [140], [129]),
    (5, 1, 8, True, [13, 260], None),
    (2, 2, 104, True, [129], [513]),
    (12, 1, 128, True, [1] * 40, [5] * 40),
    (8, 2, 128, True, [1200], [2048]),
    (2, 1, 64, True, [21], [2100]),
    (3, 1, 128, False, [40, 9], [900, 1200]),
    (2, 2, 256, True, [33], [700]),
]


def prompt_case(heads, kvh, dim, lq, lk, dtype, seed, spare=5, wide=False):
    g = gen_of(seed)
    cq, ck = offsets(lq), offsets(lk or lq)
    n, m = cq[-1] + spare, ck[-1] + spare
    if wide and lk is None:
        allq = normal(g, (n, heads + 2 * kvh, dim), dtype)
        q, k, v = allq[:, :heads], allq[:, heads:heads + kvh], allq[:, heads + kvh:]
        q.mul_(1.5)
    else:
        q, k, v = normal(g, (n, heads, dim), dtype, 1.5), normal(g, (m, kvh, dim), dtype), normal(g, (m, kvh, dim), dtype)
    return q, k, v, cq, ck


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(PROMPT)))
def test_prompt(ctx, case, dtype):
    from sofie_b200.ops import PromptAttentionPlan
    heads, kvh, dim, causal, lq, lk = PROMPT[case]
    q, k, v, cq, ck = prompt_case(heads, kvh, dim, lq, lk, dtype, case, wide=case % 2 == 1)
    want, tol = ref.prompt(q, k, v, cq, ck, causal)
    for t, end in ((q, cq[-1]), (k, ck[-1]), (v, ck[-1])):
        t[end:] = float("nan")          # rows behind the last sequence hold anything
    y = torch.full((q.shape[0], heads, dim), 3.0, dtype=dtype, device=DEV)
    plan = PromptAttentionPlan(ctx, heads, kvh, dim, dtype, causal=causal)
    plan.enqueue(q, k, v, y, ints(cq), ints(ck) if lk else None)
    ctx.sync()
    ref.close(y[:cq[-1]], want[:cq[-1]], tol[:cq[-1]], plan.kernel)
    assert (y[cq[-1]:] == 3.0).all()
    again = torch.empty_like(y)
    plan.enqueue(q, k, v, again, ints(cq), ints(ck) if lk else None)
    ctx.sync()
    assert torch.equal(again[:cq[-1]], y[:cq[-1]])
    plan.close()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("heads,kvh,dim", [(4, 1, 64), (2, 2, 128)])
def test_prompt_hidden_keys_have_no_influence(ctx, dtype, heads, kvh, dim):
    """NaN and infinities in keys and values that a query does not see: the next sequence's, and later ones of its own."""
    from sofie_b200.ops import PromptAttentionPlan
    lens = [130, 70, 20]
    q, k, v, cq, _ = prompt_case(heads, kvh, dim, lens, None, dtype, 11)
    k[130:200] = float("nan")            # the whole second sequence
    v[130:200] = float("inf")
    k[100], v[90] = float("nan"), float("-inf")     # late tokens of the first
    v[215, :, 3] = float("nan")
    y = torch.zeros_like(q)
    PromptAttentionPlan(ctx, heads, kvh, dim, dtype).enqueue(q, k, v, y, ints(cq))
    ctx.sync()
    want, tol = ref.prompt(q, k, v, cq, cq, True)
    # the statement in 64 bits computes 0 * NaN; put those rows right: they see only what comes before
    for s, e, first in ((0, 130, 90), (200, 220, 215)):
        w2, t2 = ref.prompt(q[s:first], k[s:first], v[s:first], [0, first - s], [0, first - s], True)
        ref.close(y[s:first], w2, t2, f"rows {s}..{first}")
    assert torch.isnan(y[100:130]).all()
    late = v[90].double().sign() * math.inf
    assert (y[90:100].double() == late[0, 0]).all()
    assert torch.isnan(y[215:220, :, 3]).all() and torch.isfinite(y[215:220, :, :3]).all()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("heads,kvh,dim", [(3, 1, 64), (1, 1, 8), (4, 2, 128), (1, 1, 104), (2, 1, 256)])
def test_prompt_values_that_are_not_finite(ctx, dtype, heads, kvh, dim):
    """Single infinite and NaN values all along a prompt: the queries from them on have them in that dimension, everything else is what
    it is without them."""
    from sofie_b200.ops import PromptAttentionPlan
    lens = [9, 701]
    q, k, v, cq, _ = prompt_case(heads, kvh, dim, lens, None, dtype, 13)
    clean = v.clone()
    for at, d, value in ((3, 0, math.inf), (9 + 10, 7, -math.inf), (9 + 300, 2, math.inf), (9 + 305, 2, -math.inf), (9 + 500, 5, math.inf), (9 + 601, dim - 2, math.nan),
                         (9 + 700, 1, math.inf)):
        v[at, :, d], clean[at, :, d] = value, 0.0
    want, tol = ref.prompt(q, k, clean, cq, cq, True)
    y = torch.zeros_like(q)
    PromptAttentionPlan(ctx, heads, kvh, dim, dtype).enqueue(q, k, v, y, ints(cq))
    ctx.sync()
    for first, end, d, value in ((3, 9, 0, math.inf), (19, 710, 7, -math.inf), (309, 314, 2, math.inf), (314, 710, 2, math.nan), (509, 710, 5, math.inf),
                                 (610, 710, dim - 2, math.nan), (709, 710, 1, math.inf)):
        got = y[first:end, :, d].double()
        assert (got.isnan() if math.isnan(value) else got == value).all(), (first, d)
        want[first:end, :, d], y[first:end, :, d] = 0.0, 0.0
    ref.close(y[:710], want[:710], tol[:710])


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_prompt_many_sequences(ctx, dtype):
    """More sequences than the blocks' table has places, most of them a few tokens, some of them none."""
    from sofie_b200.ops import PromptAttentionPlan
    g = gen_of(17)
    lens = torch.randint(0, 9, (1000,), generator=g, device=DEV).tolist()
    lens[500], lens[999] = 400, 130
    q, k, v, cq, _ = prompt_case(4, 2, 64, lens, None, dtype, 17)
    want, tol = ref.prompt(q, k, v, cq, cq, True)
    y = torch.zeros_like(q)
    PromptAttentionPlan(ctx, 4, 2, 64, dtype).enqueue(q, k, v, y, ints(cq))
    ctx.sync()
    ref.close(y[:cq[-1]], want[:cq[-1]], tol[:cq[-1]])


@pytest.mark.parametrize("heads,kvh,dim", [(3, 1, 64), (5, 1, 40), (7, 1, 80), (3, 1, 128), (6, 2, 72), (5, 1, 192), (3, 3, 256)])
@pytest.mark.parametrize("gap", [0, 8])
def test_prompt_warps_that_hold_some_rows_only(ctx, heads, kvh, dim, gap):
    """Tiles that end inside a warp (groups that do not divide 32, sequences of every length up to a few), with rows of the result
    that are stored in 32-byte pieces and in 16-byte ones; what lies between the rows stays."""
    from sofie_b200.ops import PromptAttentionPlan
    lens = [1, 2, 3, 5, 7, 11, 13, 31, 33, 43, 64, 85, 129]
    q, k, v, cq, _ = prompt_case(heads, kvh, dim, lens, None, BF, dim + gap, spare=0)
    want, tol = ref.prompt(q, k, v, cq, cq, True)
    room = torch.full((cq[-1], heads * dim + gap), 3.0, dtype=BF, device=DEV)
    y = room[:, :heads * dim].view(cq[-1], heads, dim)
    PromptAttentionPlan(ctx, heads, kvh, dim, BF).enqueue(q, k, v, y, ints(cq))
    ctx.sync()
    ref.close(y, want, tol)
    assert (room[:, heads * dim:] == 3.0).all()


def test_prompt_rows_far_from_the_maximum(ctx):
    """Scores that grow along the keys by more than fp32's exponents hold: the running maximum has to follow."""
    from sofie_b200.ops import PromptAttentionPlan
    for dtype in (BF, F32):
        n, dim = 520, 64
        g = gen_of(5)
        q, k, v = normal(g, (n, 1, dim), dtype, 0.1), normal(g, (n, 1, dim), dtype, 0.1), normal(g, (n, 1, dim), dtype)
        q[:, 0, 0] = 8.0
        k[:, 0, 0] = (torch.arange(n, device=DEV) * 0.5).to(dtype)       # scores 0 .. 260
        k[300:, 0, 0] = -(torch.arange(n - 300, device=DEV) * 1.0).to(dtype)
        y = torch.zeros_like(q)
        for causal in (True, False):
            PromptAttentionPlan(ctx, 1, 1, dim, dtype, causal=causal).enqueue(q, k, v, y, ints([0, n]))
            ctx.sync()
            ref.close(y, *ref.prompt(q, k, v, [0, n], [0, n], causal))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("heads,kvh,dim,n,std", [(5, 1, 8, 260, 1.5), (1, 1, 64, 520, 6.0), (4, 1, 64, 300, 6.0), (1, 1, 128, 520, 6.0), (4, 1, 128, 520, 6.0),
                                                 (1, 1, 256, 520, 6.0), (3, 1, 80, 300, 5.0)])
def test_prompt_maximum_moves_late(ctx, heads, kvh, dim, n, std, dtype):
    """Peaked scores, and a last tile of keys of which a row sees few: the running maximum moves far in later tiles, in tiles of rows
    whose last warps hold no rows."""
    from sofie_b200.ops import PromptAttentionPlan
    for seed in range(4):
        g = gen_of(seed)
        q, k, v = normal(g, (n, heads, dim), dtype, std), normal(g, (n, kvh, dim), dtype), normal(g, (n, kvh, dim), dtype)
        for causal in (True, False):
            y = torch.zeros_like(q)
            PromptAttentionPlan(ctx, heads, kvh, dim, dtype, causal=causal).enqueue(q, k, v, y, ints([0, n]))
            ctx.sync()
            ref.close(y, *ref.prompt(q, k, v, [0, n], [0, n], causal), f"seed {seed}, causal {causal}")


def test_prompt_bad_offsets_are_left_out(ctx):
    from sofie_b200.ops import PromptAttentionPlan
    for dtype in (BF, F32):
        q, k, v, cq, _ = prompt_case(4, 2, 64, [20, 30], None, dtype, 6, spare=0)
        want, tol = ref.prompt(q, k, v, cq, cq, True)
        plan = PromptAttentionPlan(ctx, 4, 2, 64, dtype)
        y = torch.full_like(q, 3.0)
        plan.enqueue(q, k, v, y, ints(cq), ints([0, 20, 60]))      # ten keys too many for the second sequence
        with pytest.raises(L.SofieB200Error) as e:
            ctx.sync()
        assert e.value.status == L.ERR_DEVICE_INDEX
        ref.close(y[:20], want[:20], tol[:20])
        assert (y[20:] == 3.0).all()
        for cu in ([0, 30, 20], [-5, 20, 50], [0, 2000000000, 50], [0, 20, 51]):
            plan.enqueue(q, k, v, y, ints(cu))
            try:
                ctx.sync()
            except L.SofieB200Error as err:
                assert err.status == L.ERR_DEVICE_INDEX


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("cu,good", [([0, 30, 20], [(0, 30)]), ([-5, 20, 50], [(20, 50)]), ([0, 2000000000, 50], []), ([0, 20, 51], [(0, 20)]),
                                     ([0, 20, -1], [(0, 20)]), ([50, 0, 50], [(0, 50)])])
def test_prompt_refused_offsets_leave_the_others(ctx, dtype, cu, good):
    """Every list says so at the next sync; sequences whose offsets are in order come out, the rows of no such sequence stay."""
    from sofie_b200.ops import PromptAttentionPlan
    q, k, v, _, _ = prompt_case(4, 2, 64, [20, 30], None, dtype, 6, spare=0)
    y = torch.full_like(q, 3.0)
    PromptAttentionPlan(ctx, 4, 2, 64, dtype).enqueue(q, k, v, y, ints(cu))
    with pytest.raises(L.SofieB200Error) as e:
        ctx.sync()
    assert e.value.status == L.ERR_DEVICE_INDEX
    stays = torch.ones(50, dtype=torch.bool, device=DEV)
    for s, t in good:
        want, tol = ref.prompt(q[s:t], k[s:t], v[s:t], [0, t - s], [0, t - s], True)
        ref.close(y[s:t], want, tol)
        stays[s:t] = False
    assert (y[stays] == 3.0).all()


def test_prompt_far_rows(ctx):
    """Element offsets past 2^31: a token pitch of 2^23 elements."""
    from sofie_b200.ops import PromptAttentionPlan
    n, pitch = 280, 1 << 23
    buf = torch.empty(n * pitch, dtype=BF, device=DEV)
    rows = buf.view(n, pitch)
    g = gen_of(8)
    for dim, col in ((64, 0),):
        q, k, v, y = (rows[:, c:c + 2 * dim].view(n, 2, dim) for c in (0, 2 * dim, 4 * dim, 6 * dim))
        for t in (q, k, v):
            t.copy_(normal(g, t.shape, BF))
        PromptAttentionPlan(ctx, 2, 2, dim, BF).enqueue(q, k, v, y, ints([0, n]))
        ctx.sync()
        ref.close(y, *ref.prompt(q, k, v, [0, n], [0, n], True))


def test_prompt_of_more_keys_than_a_sequence_has(ctx):
    """2^27 keys in one bf16 sequence (19 GB): sums over so many would lose half of the result, and warps without a turn would wait for longer
    than a second.  The sequence is left out and reported, the one behind it is not."""
    from sofie_b200.ops import PromptAttentionPlan
    n, dim = 1 << 27, 72
    x = torch.ones((n, 1, dim), dtype=BF, device=DEV)   # keys and values
    x[n // 2:] = 3.0
    q, y = torch.zeros((2, 1, dim), dtype=BF, device=DEV), torch.full((2, 1, dim), 7.0, dtype=BF, device=DEV)
    plan = PromptAttentionPlan(ctx, 1, 1, dim, BF)
    for cu_k, left in (([0, n, n], (7.0, 0.0)), ([0, n - 4, n], (7.0, 3.0)), ([0, 4, (1 << 20) + 5], (1.0, 7.0))):
        y.fill_(7.0)
        plan.enqueue(q, x, x, y, ints([0, 1, 2]), ints(cu_k))
        with pytest.raises(L.SofieB200Error) as e:
            ctx.sync()
        assert e.value.status == L.ERR_DEVICE_INDEX
        assert (y[0] == left[0]).all() and (y[1] == left[1]).all()
    plan.enqueue(q, x, x, y, ints([0, 0, 1]), ints([0, n - 4, n]))    # no queries: nothing to leave out
    ctx.sync()
    assert (y[0] == 3.0).all()


@pytest.mark.parametrize("dtype,dim,most", [(BF, 64, 1 << 20), (BF, 128, 1 << 20), (BF, 256, 1 << 20), (F32, 8, 1 << 24)])
def test_prompt_of_the_most_keys(ctx, dtype, dim, most):
    """The longest sequence, equal weights, values of one sign: what sums over so many keys lose.  One key more is refused.
    Bounds, relative to the result.  bf16: the tensor cores cut each product and each sum of 16 products by less than 2^-23 of the running
    sum, which is half the result on average: n (17 / 16) 2^-24.  fp32: n / 2 sums in each of two teams of warps, each rounded by at
    most 2^-24 of the result, either way as the random values fall: 8 sqrt(n / 2) 2^-24, eight standard deviations.  Then the
    rounding of the result; the weights are 1."""
    from sofie_b200.ops import PromptAttentionPlan
    g = gen_of(3)
    k = torch.zeros((most + 1, 1, dim), dtype=dtype, device=DEV)
    v = (torch.rand((most + 1, 1, dim), generator=g, device=DEV) + 0.5).to(dtype)
    q, y = torch.zeros((1, 1, dim), dtype=dtype, device=DEV), torch.full((1, 1, dim), 7.0, dtype=dtype, device=DEV)
    plan = PromptAttentionPlan(ctx, 1, 1, dim, dtype)
    plan.enqueue(q, k, v, y, ints([0, 1]), ints([0, most + 1]))
    with pytest.raises(L.SofieB200Error) as e:
        ctx.sync()
    assert e.value.status == L.ERR_DEVICE_INDEX and (y == 7.0).all()
    plan.enqueue(q, k, v, y, ints([0, 1]), ints([0, most]))
    ctx.sync()
    want = v[:most].double().mean(0, keepdim=True)
    lost = most * 17 / 16 * 2.0 ** -24 if dtype is BF else 8 * math.sqrt(most / 2) * 2.0 ** -24
    ref.close(y, want, (lost + ref.HALF[dtype]) * want)


# ---- decode ---------------------------------------------------------------------------------------------------------
DECODE = [
    # heads, kv_heads, dim, page_size, lengths, pages heads first
    (8, 8, 64, 16, [5, 1, 0, 16, 17, 100], False),
    (32, 8, 128, 16, [1000, 3, 64, 63, 65], False),
    (32, 8, 128, 64, [5000], False),
    (8, 2, 64, 1, [300, 40], False),
    (6, 2, 80, 48, [500, 47, 48, 49], True),
    (7, 1, 96, 128, [1, 2, 127, 128, 129, 1000], False),
    (16, 1, 128, 32, [777, 31], True),
    (64, 1, 128, 16, [900, 1], False),
    (20, 1, 64, 16, [333, 2048], False),
    (4, 1, 256, 8, [600, 9], False),
    (5, 5, 32, 256, [1, 255, 256, 257, 2000], False),
    (3, 1, 8, 16, [100] * 70, False),
    (12, 4, 192, 16, [129] * 9 + [0] * 5, True),
    (1, 1, 128, 16, [40000], False),
    (8, 8, 64, 16, [13] * 300, False),
]


def decode_case(heads, kvh, dim, size, lens, first, dtype, seed):
    g = gen_of(seed)
    table, pages = ref.make_pages(lens, size, g)
    if first:
        ck, cv = (normal(g, (pages, kvh, size, dim), dtype).transpose(1, 2) for _ in range(2))
    else:
        both = normal(g, (pages, 2, size, kvh, dim), dtype)
        ck, cv = both[:, 0], both[:, 1]
    return normal(g, (len(lens), heads, dim), dtype, 1.5), ck, cv, table


def poison(cache, table, lens, size):
    """NaN in every slot that no sequence owns."""
    keep = torch.zeros(cache.shape[:2], dtype=torch.bool, device=DEV)
    for b, n in enumerate(lens):
        at = torch.arange(n, device=DEV)
        keep[table[b, at // size].long(), at % size] = True
    cache[~keep] = float("nan")


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(DECODE)))
def test_decode(ctx, case, dtype):
    from sofie_b200.ops import PagedAttentionPlan, PagedKV
    heads, kvh, dim, size, lens, first = DECODE[case]
    q, ck, cv, table = decode_case(heads, kvh, dim, size, lens, first, dtype, case)
    want, tol = ref.decode(q, ck, cv, table, lens)
    poison(ck, table, lens, size)
    poison(cv, table, lens, size)
    y = torch.full_like(q, 3.0)
    plan = PagedAttentionPlan(ctx, heads, kvh, dim, dtype)
    kv = PagedKV(ck, cv, table, ints(lens))
    plan.enqueue(q, kv, y)
    ctx.sync()
    ref.close(y, want, tol, plan.kernel)
    again = torch.empty_like(y)
    plan.enqueue(q, kv, again)
    ctx.sync()
    assert torch.equal(again, y)
    plan.close()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("heads,kvh,dim,lens", [(4, 1, 64, [1, 17, 300]), (8, 2, 128, [40, 3000]), (20, 1, 80, [500, 9]), (3, 1, 256, [33, 2000]), (1, 1, 8, [40000, 2])])
def test_decode_values_that_are_not_finite(ctx, dtype, heads, kvh, dim, lens):
    """Infinite and NaN values that a sequence sees come out in their dimension; everything else is what it is without them."""
    from sofie_b200.ops import PagedAttentionPlan, PagedKV
    q, ck, cv, table = decode_case(heads, kvh, dim, 16, lens, False, dtype, 91)
    clean = cv.clone()
    expect = []
    for b, n in enumerate(lens):
        for at, d, value in ((0, 0, math.inf), (n // 2, 3, -math.inf), (n - 1, 5, math.inf), (n // 3, 6, math.nan)):
            where = int(table[b, at // 16]), at % 16, slice(None), d
            cv[where], clean[where] = value, 0.0
            expect.append((b, d, value))
        if n > 1:
            for at, value in ((0, math.inf), (n - 1, -math.inf)):
                where = int(table[b, at // 16]), at % 16, slice(None), 7
                cv[where], clean[where] = value, 0.0
            expect.append((b, 7, math.nan))
    want, tol = ref.decode(q, ck, clean, table, lens)
    y = torch.empty_like(q)
    PagedAttentionPlan(ctx, heads, kvh, dim, dtype).enqueue(q, PagedKV(ck, cv, table, ints(lens)), y)
    ctx.sync()
    for b, d, value in expect:
        got = y[b, :, d].double()
        assert (got.isnan() if math.isnan(value) else got == value).all(), (b, d, value)
        want[b, :, d], y[b, :, d] = 0.0, 0.0
    ref.close(y, want, tol)


def test_decode_leaves_out_bad_pages(ctx):
    from sofie_b200.ops import PagedAttentionPlan, PagedKV
    for dtype in (BF, F32):
        lens, size = [40, 40, 40, 40], 16
        q, ck, cv, table = decode_case(4, 2, 64, size, lens, False, dtype, 21)
        want, tol = ref.decode(q, ck, cv, table, [40, 32, 40, 48])
        n_pages = ck.shape[0]
        table[1, 2] = n_pages                              # sequence 1 loses its last 8 tokens
        kv = PagedKV(ck, cv, table, ints([40, 40, -3, 4000]))   # sequence 2: a negative length; 3: more than its table holds
        y = torch.full_like(q, 3.0)
        plan = PagedAttentionPlan(ctx, 4, 2, 64, dtype)
        plan.enqueue(q, kv, y)
        with pytest.raises(L.SofieB200Error) as e:
            ctx.sync()
        assert e.value.status == L.ERR_DEVICE_INDEX
        ref.close(y[:2], want[:2], tol[:2])
        assert (y[2] == 0).all()
        ref.close(y[3], want[3], tol[3])
        table[0] = -1                                      # no page at all: nothing to attend to
        plan.enqueue(q, kv, y)
        with pytest.raises(L.SofieB200Error):
            ctx.sync()
        assert (y[0] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_decode_shared_pages(ctx, dtype):
    """A common prefix: sequences that share pages, one page twice in a sequence, a table with a pitch of its own."""
    from sofie_b200.ops import PagedAttentionPlan, PagedKV
    g = gen_of(23)
    ck, cv = normal(g, (12, 16, 2, 64), dtype), normal(g, (12, 16, 2, 64), dtype)
    wide = torch.full((3, 9), 99, dtype=torch.int32, device=DEV)
    table = wide[:, 2:7]
    table.copy_(ints([[3, 4, 5, 6, 0], [3, 4, 5, 7, 0], [8, 8, 3, 8, 1]]))
    lens = [61, 64, 80]
    q = normal(g, (3, 8, 64), dtype)
    y = torch.empty_like(q)
    PagedAttentionPlan(ctx, 8, 2, 64, dtype).enqueue(q, PagedKV(ck, cv, table, ints(lens)), y)
    ctx.sync()
    ref.close(y, *ref.decode(q, ck, cv, table, lens))


def test_far_pages(ctx):
    """Cache offsets past 2^31 elements: append there and read it back."""
    from sofie_b200.ops import PagedAttentionPlan, PagedKV
    kvh, dim, size = 2, 64, 16
    pages = (1 << 31) // (kvh * dim * size) + 40
    g = gen_of(9)
    ck, cv = (torch.empty((pages, size, kvh, dim), dtype=BF, device=DEV) for _ in range(2))
    table = ints([[pages - 1, pages - 3, 0], [pages - 2, 1, pages - 5]])
    lens = [40, 48]
    k, v, q = normal(g, (88, kvh, dim), BF), normal(g, (88, kvh, dim), BF), normal(g, (2, 4, dim), BF)
    kv = PagedKV(ck, cv, table, ints(lens))
    ctx.kv_append(k, v, kv, ints([0, 40, 88]))
    y = torch.zeros_like(q)
    PagedAttentionPlan(ctx, 4, kvh, dim, BF).enqueue(q, kv, y)
    ctx.sync()
    assert torch.equal(ref.gather(ck, table[0], 40), k[:40]) and torch.equal(ref.gather(cv, table[1], 48), v[40:])
    ref.close(y, *ref.decode(q, ck, cv, table, lens))


# ---- together -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,heads,kvh,dim", [(BF, 8, 2, 64), (F32, 4, 4, 32), (BF, 8, 8, 128)], ids=["bf16-grouped", "f32", "bf16-128"])
def test_generation_run(ctx, dtype, heads, kvh, dim):
    """Prompts enter the cache (append + prompt attention over the rotated keys), then tokens are generated one by one (append +
    attention over the cache).  Every step's result is the causal attention of the whole sequence so far, in 64 bits."""
    from sofie_b200.ops import PagedAttentionPlan, PagedKV, PromptAttentionPlan
    g = gen_of(31)
    prompts, steps, size = [70, 1, 133], 20, 16
    total = [n + steps for n in prompts]
    table, pages = ref.make_pages(total, size, g)
    ck, cv = (torch.full((pages, size, kvh, dim), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
    lens = ints(prompts)
    kv = PagedKV(ck, cv, table, lens)
    cos, sin = tables(max(total), dim)
    cu = offsets(prompts)
    qkv = normal(g, (cu[-1], heads + 2 * kvh, dim), dtype)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kvh], qkv[:, heads + kvh:]
    qr, kr, y = torch.empty((cu[-1], heads, dim), dtype=dtype, device=DEV), torch.empty((cu[-1], kvh, dim), dtype=dtype, device=DEV), torch.empty((cu[-1], heads, dim), dtype=dtype, device=DEV)
    prompt, step = PromptAttentionPlan(ctx, heads, kvh, dim, dtype), PagedAttentionPlan(ctx, heads, kvh, dim, dtype)
    ctx.kv_append(k, v, kv, ints(cu), cos=cos, sin=sin, q=q, q_out=qr, k_out=kr)
    prompt.enqueue(qr, kr, v, y, ints(cu))
    ctx.sync()
    ref.close(y, *ref.prompt(qr, kr, v, cu, cu, True), "prompts")
    for b, n in enumerate(prompts):
        assert torch.equal(ref.gather(ck, table[b], n), kr[cu[b]:cu[b + 1]])
    ys = torch.empty((3, heads, dim), dtype=dtype, device=DEV)
    for i in range(steps):
        lens += 1
        qkv = normal(g, (3, heads + 2 * kvh, dim), dtype)
        q1 = torch.empty((3, heads, dim), dtype=dtype, device=DEV)
        ctx.kv_append(qkv[:, heads:heads + kvh], qkv[:, heads + kvh:], kv, cos=cos, sin=sin, q=qkv[:, :heads], q_out=q1)
        step.enqueue(q1, kv, ys)
        ctx.sync()
        ref.close(ys, *ref.decode(q1, ck, cv, table, [n + i + 1 for n in prompts]), f"step {i}")
    # the last step once more as the last row of a causal prompt over the whole sequence
    full = [ref.gather(ck, table[b], n) for b, n in enumerate(total)], [ref.gather(cv, table[b], n) for b, n in enumerate(total)]
    y1 = torch.empty_like(ys)
    prompt.enqueue(q1, torch.cat(full[0]), torch.cat(full[1]), y1, ints([0, 1, 2, 3]), ints(offsets(total)))
    ctx.sync()
    w, t = ref.decode(q1, ck, cv, table, total)
    ref.close(y1, w, t + 2.0 ** -8 * (w.abs() + 4.0 * (dtype == BF)), "last step as a prompt")


def test_a_captured_step_is_replayed_for_other_lengths(b200_lib):
    """Append and attention of one step captured into a graph, replayed while the lengths and inputs change in place."""
    from sofie_b200.ops import Context, PagedAttentionPlan, PagedKV, PromptAttentionPlan
    side = torch.cuda.Stream(device=DEV)
    ctx = Context(0, stream=side)
    g = gen_of(41)
    heads, kvh, dim, size, room = 8, 2, 128, 16, 700
    table, pages = ref.make_pages([room] * 4, size, g)
    ck, cv = normal(g, (pages, size, kvh, dim), BF), normal(g, (pages, size, kvh, dim), BF)
    lens = ints([1, 1, 1, 1])
    kv = PagedKV(ck, cv, table, lens)
    cos, sin = tables(room, dim)
    q, k, v = normal(g, (4, heads, dim), BF), normal(g, (4, kvh, dim), BF), normal(g, (4, kvh, dim), BF)
    qr, y, yp = torch.empty_like(q), torch.empty_like(q), torch.zeros_like(q)
    plan, prompt = PagedAttentionPlan(ctx, heads, kvh, dim, BF), PromptAttentionPlan(ctx, heads, kvh, dim, BF)
    cu = ints([0, 2, 3, 4, 4])

    def step():
        ctx.kv_append(k, v, kv, cos=cos, sin=sin, q=q, q_out=qr)
        plan.enqueue(qr, kv, y)
        prompt.enqueue(q, k, v, yp, cu)

    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step()
    ctx.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for i, now in enumerate(([5, 700, 0, 64], [699, 1, 333, 2], [1, 2, 3, 4])):
        lens.copy_(ints(now))
        q.copy_(normal(g, q.shape, BF))
        k.copy_(normal(g, k.shape, BF))
        cu.copy_(ints([[0, 2, 3, 4, 4], [0, 4, 4, 4, 4], [0, 1, 2, 3, 4]][i]))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ctx.sync()
        w, t = ref.decode(qr, ck, cv, table, now)
        live = [b for b, n in enumerate(now) if n]
        ref.close(y[live], w[live], t[live], f"replay {i}")
        assert (y[[b for b, n in enumerate(now) if not n]] == 0).all()
        c = cu.tolist()
        ref.close(yp, *ref.prompt(q, k, v, c, c, True), f"replay {i}, prompt")
    del graph
    plan.close()
    prompt.close()
    ctx.close()


def test_two_streams_at_once(b200_lib):
    """Two contexts with plans of their own on two streams, their calls interleaved."""
    from sofie_b200.ops import Context, PagedAttentionPlan, PagedKV
    streams = [torch.cuda.Stream(device=DEV) for _ in range(2)]
    runs = []
    for i, s in enumerate(streams):
        c = Context(0, stream=s)
        lens = [3000 + i, 17, 900]
        q, ck, cv, table = decode_case(16, 4, 128, 16, lens, False, BF, 50 + i)
        runs.append((c, PagedAttentionPlan(c, 16, 4, 128, BF), q, PagedKV(ck, cv, table, ints(lens)), torch.empty_like(q), ref.decode(q, ck, cv, table, lens)))
    torch.cuda.synchronize()
    for _ in range(20):
        for c, plan, q, kv, y, _w in runs:
            plan.enqueue(q, kv, y)
    for c, plan, q, kv, y, (want, tol) in runs:
        c.sync()
        ref.close(y, want, tol)
        plan.close()
        c.close()


def test_two_graphs_replayed_side_by_side(b200_lib):
    """Two plans, each captured into a graph of its own, replayed on two streams at once."""
    from sofie_b200.ops import Context, PagedAttentionPlan, PagedKV, PromptAttentionPlan
    runs = []
    for i in range(2):
        s = torch.cuda.Stream(device=DEV)
        c = Context(0, stream=s)
        lens = [5000 - 700 * i, 3, 1200]
        q, ck, cv, table = decode_case(8, 2, 128, 16, lens, False, BF, 70 + i)
        qp, kp, vp, cq, _ = prompt_case(8, 2, 128, [300, 40 + i], None, BF, 80 + i, spare=0)
        kv, y, yp, cu = PagedKV(ck, cv, table, ints(lens)), torch.empty_like(q), torch.empty_like(qp), ints(cq)
        plan, prompt = PagedAttentionPlan(c, 8, 2, 128, BF), PromptAttentionPlan(c, 8, 2, 128, BF)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            for _ in range(3):
                plan.enqueue(q, kv, y)
                prompt.enqueue(qp, kp, vp, yp, cu)
        runs.append((s, c, graph, plan, prompt, y, yp, ref.decode(q, ck, cv, table, lens), ref.prompt(qp, kp, vp, cq, cq, True), (q, kv, qp, kp, vp, cu)))
    torch.cuda.synchronize()
    for _ in range(10):
        for s, c, graph, *_r in runs:
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for s, c, graph, plan, prompt, y, yp, d, pr, _keep in runs:
        c.sync()
        ref.close(y, *d)
        ref.close(yp, *pr)
    for r in runs:
        r[2].reset()
        r[3].close()
        r[4].close()
        r[1].close()


@pytest.mark.parametrize("wait_first", [True, False])
def test_a_wait_that_ran_out_is_reported_before_a_bad_index(ctx, wait_first):
    """Both in one step, in either order: the caller hears of the results that are unfinished."""
    from sofie_b200.ops import PagedKV
    ck, cv, k = (torch.zeros(s, dtype=BF, device=DEV) for s in ((2, 4, 1, 8), (2, 4, 1, 8), (1, 1, 8)))
    kv = PagedKV(ck, cv, ints([[9]]), ints([1]))

    def wait():
        assert L.load().sofie_b200_selftest_wait_timeout(ctx._h, 1000) == 0   # a bounded wait on a barrier that nothing signals

    for call in (wait, lambda: ctx.kv_append(k, k, kv))[::1 if wait_first else -1]:
        call()
    with pytest.raises(L.SofieB200Error) as e:
        ctx.sync()
    assert e.value.status == L.ERR_DEVICE_WAIT
    ctx.sync()
    ctx.kv_append(k, k, kv)
    with pytest.raises(L.SofieB200Error) as e:
        ctx.sync()
    assert e.value.status == L.ERR_DEVICE_INDEX


def test_workspace_belongs_to_the_contexts_stream(b200_lib):
    """Memory that was freed on the current stream, with a kernel there still to write it, is not the workspace of a plan on another stream."""
    from sofie_b200.ops import Context, PagedAttentionPlan
    for given in (True, False):   # the context's stream as an argument, and as the current one when the context was made
        side = torch.cuda.Stream(device=DEV)
        if given:
            ctx = Context(0, stream=side)
        else:
            with torch.cuda.stream(side):
                ctx = Context(0)
        first = PagedAttentionPlan(ctx, 8, 2, 128, BF)
        size = first._workspace.numel()
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        old = torch.empty(size, dtype=torch.uint8, device=DEV)
        begin, end = old.data_ptr(), old.data_ptr() + size
        torch.cuda._sleep(50_000_000)
        old.fill_(1)
        del old
        plan = PagedAttentionPlan(ctx, 8, 2, 128, BF)
        at = plan._workspace.data_ptr()
        assert at + size <= begin or at >= end
        torch.cuda.synchronize()
        for p in (first, plan):
            p.close()
        ctx.close()


def test_prompt_extents_that_are_refused(ctx):
    from sofie_b200.ops import PromptAttentionPlan
    q = torch.empty((8, 1, 8), dtype=BF, device=DEV)
    cu = ints([0, 8])
    plan = PromptAttentionPlan(ctx, 1, 1, 8, BF)
    for batch, n, m in ((-1, 8, 8), (1, -1, 8), (1, 8, -1), (1, (1 << 27) + 1, 8), (1, 8, (1 << 27) + 1), (1 << 30, 8, 8)):
        p = q.data_ptr()
        assert L.load().sofie_b200_prompt_attention_enqueue(plan._plan((0, 0, 0, 0)), p, p, p, p, cu.data_ptr(), cu.data_ptr(), batch, n, m) == L.ERR_INVALID
    ctx.sync()


def test_prompt_grids_that_are_refused(ctx):
    """More blocks than are asked for one by one in the limit of a wait."""
    from sofie_b200.ops import PromptAttentionPlan
    q = torch.empty((8, 16, 8), dtype=BF, device=DEV)
    cu, p = ints([0, 8]), q.data_ptr()
    plan = PromptAttentionPlan(ctx, 16, 16, 8, BF)
    assert L.load().sofie_b200_prompt_attention_enqueue(plan._plan((0, 0, 0, 0)), p, p, p, p, cu.data_ptr(), cu.data_ptr(), (1 << 23) + 1, 8, 8) == L.ERR_TOO_LARGE
    ctx.sync()


def test_refusals_with_a_context(ctx):
    from sofie_b200.ops import PagedAttentionPlan, PagedKV, PromptAttentionPlan
    q, ck, cv, table = decode_case(4, 2, 64, 16, [20, 20], False, BF, 1)
    kv = PagedKV(ck, cv, table, ints([20, 20]))
    plan = PagedAttentionPlan(ctx, 4, 2, 64, BF)
    with pytest.raises(ValueError):
        plan.enqueue(q[:1], kv, torch.empty_like(q[:1]))
    with pytest.raises(ValueError):
        plan.enqueue(q.float(), kv, torch.empty_like(q).float())
    odd = torch.empty(2 * 4 * 64 + 1, dtype=BF, device=DEV)[1:].view(2, 4, 64)
    with pytest.raises(L.SofieB200Error, match="aligned"):
        plan.enqueue(odd, kv, torch.empty_like(q))
    wide = torch.empty((2, 4 * 64 + 4), dtype=BF, device=DEV)[:, :256].view(2, 4, 64)
    with pytest.raises(L.SofieB200Error, match="multiples of 8"):
        plan.enqueue(wide, kv, torch.empty_like(q))
    prompt = PromptAttentionPlan(ctx, 4, 2, 64, BF)
    k = torch.empty((2, 2, 64), dtype=BF, device=DEV)
    with pytest.raises(L.SofieB200Error, match="aligned"):
        prompt.enqueue(odd, k, k, torch.empty_like(q), ints([0, 2]))
    with pytest.raises(ValueError):
        prompt.enqueue(q, k, k, q.float(), ints([0, 2]))
    with pytest.raises(ValueError):
        prompt.enqueue(q, k, k, q, ints([0, 2]).long())
    with pytest.raises(L.SofieB200Error, match="head size"):
        PromptAttentionPlan(ctx, 4, 2, 68, BF)
    prompt.enqueue(q[:0], k, k, q[:0], ints([0]))     # nothing to do is not an error
    for kw in (dict(q=q), dict(q_out=q), dict(q=q, q_out=q[:1]), dict(cos=torch.zeros(4, 8, device=DEV)), dict(k_out=q),
               dict(cos=torch.zeros(4, 8, device=DEV), sin=torch.zeros(4, 9, device=DEV))):
        with pytest.raises(ValueError):
            ctx.kv_append(k, k, kv, **kw)
    with pytest.raises(ValueError):
        ctx.kv_append(k, k[:1], kv)
    with pytest.raises(ValueError):
        ctx.kv_append(k, k, kv, ints([0, 2]))
    with pytest.raises(TypeError):
        ctx.kv_append(k, k, kv, cos=torch.zeros(40, 8, device=DEV, dtype=BF), sin=torch.zeros(40, 8, device=DEV, dtype=BF))
    ctx.sync()
