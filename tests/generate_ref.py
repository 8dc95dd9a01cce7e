"""Plain statements, in 64 bits, of the generation operators, with bounds on what a correct kernel may be off by.

Bounds.  u = 2^-24 is half a step of fp32, h the half step of the result's type (2^-8 bf16, 2^-24 fp32).
  rotation   two products and a sum in fp32: at most 2 u (|x| + |y|) as |cos|, |sin| <= 1; then one rounding, h |result|.
  attention  with A = max over the row's keys of scale * sum |q_d k_d|: a score of D products and D - 1 sums in fp32, scaled, minus a
             maximum, is off by at most e = a (D + 8) A, a = u (products and sums rounded) or, on the tensor cores, whose fp32
             sums truncate, a = 4 u.  Its exponential is off by the factor 1 + e + 2^-21 (the hardware exp2 keeps 2^-22).  Numerator and
             denominator each carry that and a sum over n keys (a n): together 2 (e + 2^-21 + a (n + 8)), relative to
             B = sum of weight * |v|.  Kernels that round the weights to bf16 for the second product add 2^-8 B.  The result is
             rounded once: h |y|."""
import torch

U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
DEV = "cuda:0"


def attend(q, k, v, limits, scale, weights_bf16, tensor_cores):
    """One sequence: q [n, heads, D], k and v [m, kv_heads, D]; query i sees the first limits[i] keys.  Returns (y, bound) in fp64."""
    n, heads, d = q.shape
    m, kv = k.shape[:2]
    dt = q.dtype
    y = torch.zeros((n, heads, d), dtype=torch.float64, device=q.device)
    tol = torch.full_like(y, 1e-300)
    if m == 0 or n == 0:
        return y, tol
    a = 4 * U if tensor_cores else U
    hidden = torch.arange(m, device=q.device)[None, :] >= limits[:, None]     # [n, m]
    empty = (limits <= 0)
    for h in range(heads):
        g = h * kv // heads
        qh, kh, vh = q[:, h].double(), k[:, g].double(), v[:, g].double()
        z = (qh @ kh.T * scale).masked_fill(hidden, float("-inf"))
        w = torch.softmax(z, -1).masked_fill(hidden | empty[:, None], 0.0)
        big = (qh.abs() @ kh.abs().T * scale).masked_fill(hidden, 0.0).amax(-1)
        out = w @ vh
        b = w @ vh.abs()
        e = a * (d + 8) * big
        rel = 2 * (e + 2.0 ** -21 + a * (m + 8)) + (2.0 ** -8 if weights_bf16 else 0.0)
        y[:, h] = out
        tol[:, h] = rel[:, None] * b * 1.01 + HALF[dt] * out.abs() + 1e-37
    return y, tol


def causal_limits(n, m, causal):
    i = torch.arange(n, device=DEV)
    return (i + 1 + m - n).clamp(0, m) if causal else torch.full((n,), m, device=DEV)


def prompt(q, k, v, cu_q, cu_k, causal, scale=None):
    """The packed form; rows that belong to nobody come back as NaN in y (nothing is said about them)."""
    scale = scale or q.shape[-1] ** -0.5
    bf = q.dtype == torch.bfloat16
    y = torch.full(q.shape, float("nan"), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(y)
    for b in range(len(cu_q) - 1):
        s, e, t, f = cu_q[b], cu_q[b + 1], cu_k[b], cu_k[b + 1]
        y[s:e], tol[s:e] = attend(q[s:e], k[t:f], v[t:f], causal_limits(e - s, f - t, causal), scale, bf, bf)
    return y, tol


def gather(cache, table_row, n):
    """The first n tokens of a sequence from a paged cache [pages, page_size, kv_heads, D]."""
    size = cache.shape[1]
    at = torch.arange(n, device=cache.device)
    return cache[table_row[at // size].long(), at % size]


def decode(q, cache_k, cache_v, table, lens, scale=None):
    scale = scale or q.shape[-1] ** -0.5
    bf = q.dtype == torch.bfloat16
    y = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(y)
    for b, n in enumerate(lens):
        k, v = gather(cache_k, table[b], n), gather(cache_v, table[b], n)
        y[b:b + 1], tol[b:b + 1] = attend(q[b:b + 1], k, v, torch.tensor([n], device=DEV), scale, False, bf)
    return y, tol


def turn(x, positions, cos, sin, rotary, interleaved):
    """Rotation of x [tokens, heads, D] at `positions`: (result, bound), both fp64."""
    z = x.double()
    tol = torch.zeros_like(z)
    if rotary:
        r = rotary // 2
        first = torch.arange(r, device=x.device) * (2 if interleaved else 1)
        second = first + (1 if interleaved else r)
        c, s = cos[positions].double()[:, None], sin[positions].double()[:, None]
        a, b = x[:, :, first].double(), x[:, :, second].double()
        z[:, :, first], z[:, :, second] = a * c - b * s, b * c + a * s
        lost = 2 * U * (a.abs() + b.abs())
        tol[:, :, first] = lost + HALF[x.dtype] * z[:, :, first].abs()
        tol[:, :, second] = lost + HALF[x.dtype] * z[:, :, second].abs()
        tol *= 1.01
    return z, tol


def close(got, want, tol, what=""):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound; first at {bad.nonzero()[0].tolist()}: "
                           f"{got[bad][0].item()} for {want[bad][0].item()} +- {tol[bad][0].item()}")


def make_pages(lens, page_size, gen, spare=2, width=None):
    """A block table over pages in random order: (table int32 [batch, width], pages)."""
    per = [-(-n // page_size) for n in lens]
    pages = sum(per) + spare
    order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    width = max(1, max(per, default=1)) if width is None else width
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages
