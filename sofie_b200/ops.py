"""Host-side handles over the C ABI: a Context (the Session's queue + blas object) and plans.

torch is used for device memory and streams only; every computation is a call into
libsofie_b200.so.  Tensors must live on the context's CUDA device.
"""
from __future__ import annotations

import contextlib
import ctypes as C

import numpy as np
from typing import Optional

import torch

from . import lib as L

_DT = {
    torch.float32: L.F32,
    torch.bfloat16: L.BF16,
    torch.int8: L.I8,
    torch.float8_e4m3fn: L.F8E4M3,
    torch.int32: L.I32,
    torch.uint8: L.U8,
}


def dtype_code(t: torch.dtype) -> int:
    try:
        return _DT[t]
    except KeyError:
        raise TypeError(f"dtype {t} is not part of the sofie_b200 ABI") from None


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("sofie_b200 operators take CUDA tensors; host data goes through run_host()")
    return t.data_ptr()


class Context:
    """One per Session / GPU / stream (sofie_b200_ctx)."""

    def __init__(self, device: int = 0, stream: Optional[torch.cuda.Stream] = None):
        self._lib = L.load()
        self.device = device
        self.stream = stream
        h = C.c_void_p()
        sp = C.c_void_p(stream.cuda_stream) if stream is not None else C.c_void_p(
            torch.cuda.current_stream(device).cuda_stream)
        L.check(self._lib.sofie_b200_ctx_create(C.byref(h), device, sp), "ctx_create")
        self._h = h
        self._torch_stream = stream if stream is not None else torch.cuda.current_stream(device)

    @contextlib.contextmanager
    def in_order(self):
        """What is enqueued inside runs behind the current stream's work so far and before what comes there later, as torch's own
        operators do.  Nothing to do where the context's stream is the current one (also under capture)."""
        current = torch.cuda.current_stream(self.device)
        apart = current != self._torch_stream and not torch.cuda.is_current_stream_capturing()
        if apart:
            self._torch_stream.wait_stream(current)
        yield
        if apart:
            current.wait_stream(self._torch_stream)

    def scratch(self, size: int) -> torch.Tensor:
        """Uninitialised device bytes that belong to the context's stream: of another stream's pool they could be a block that
        was just freed there and is still written, and after their release one that this stream still uses."""
        with torch.cuda.stream(self._torch_stream):
            return torch.empty(size, dtype=torch.uint8, device=f"cuda:{self.device}")

    def sync(self) -> None:
        L.check(self._lib.sofie_b200_ctx_sync(self._h), "ctx_sync")

    @property
    def launches(self) -> int:
        return int(self._lib.sofie_b200_ctx_launch_count(self._h))

    # another GPU's memory, for GemmPlan.enqueue_peers
    def enable_peer(self, peer_device: int) -> None:
        """One process driving several GPUs: this ctx's kernels may then store to `peer_device`'s memory."""
        L.check(self._lib.sofie_b200_ctx_enable_peer(self._h, int(peer_device)), "ctx_enable_peer")

    def peer_export(self, t: torch.Tensor) -> bytes:
        """The 72 bytes another process needs to open `t`'s first element (send them by any means)."""
        h = L.PeerHandle()
        L.check(self._lib.sofie_b200_peer_export(self._h, _ptr(t), C.byref(h)), "peer_export")
        return bytes(h)

    def peer_open(self, handle: bytes) -> int:
        """Device pointer, valid in this process, to the byte another process exported."""
        h = L.PeerHandle.from_buffer_copy(handle)
        p = C.c_void_p()
        L.check(self._lib.sofie_b200_peer_open(self._h, C.byref(h), C.byref(p)), "peer_open")
        return int(p.value)

    def peer_close(self, ptr: int) -> None:
        L.check(self._lib.sofie_b200_peer_close(self._h, C.c_void_p(ptr)), "peer_close")

    def close(self) -> None:
        if self._h:
            self._lib.sofie_b200_ctx_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ---- memory-bound operators -----------------------------------------------------
    def layernorm(self, x, y, scale=None, bias=None, eps=1e-5, mean_out=None, invstd_out=None):
        cols = x.shape[-1]
        rows = x.numel() // cols
        L.check(self._lib.sofie_b200_layernorm_enqueue(
            self._h, _ptr(x), _ptr(y), dtype_code(x.dtype), dtype_code(y.dtype), rows, cols, _ptr(scale),
            _ptr(bias), eps, _ptr(mean_out), _ptr(invstd_out)), "layernorm_enqueue")

    def softmax(self, x, y, log_softmax=False):
        cols = x.shape[-1]
        rows = x.numel() // cols if cols else 0
        L.check(self._lib.sofie_b200_softmax_enqueue(
            self._h, _ptr(x), _ptr(y), dtype_code(x.dtype), dtype_code(y.dtype), rows, cols, int(log_softmax)),
            "softmax_enqueue")

    def softmax_axis(self, x, y, axis, log_softmax=False):
        """Softmax over `axis` of a contiguous tensor (any axis)."""
        axis = axis + x.dim() if axis < 0 else axis
        outer = int(np.prod(x.shape[:axis])) if axis else 1
        inner = int(np.prod(x.shape[axis + 1:])) if axis + 1 < x.dim() else 1
        L.check(self._lib.sofie_b200_softmax_axis_enqueue(self._h, _ptr(x), _ptr(y), dtype_code(x.dtype), outer, x.shape[axis], inner,
                                                          int(log_softmax)), "softmax_axis_enqueue")

    def sdpa(self, q, k, v, y, mask=None, scale=0.0, heads=0, ldq=0, ldk=0, ldv=0):
        """Scaled dot-product attention through an SDPA plan made for this call.  Rank-4 tensors are [B,H,S,D]; rank-3
        tensors are folded [B,S,H*D] and need `heads` (ldq / ldk / ldv: row pitches when Q, K, V are column blocks of a
        wider tensor).  Returns the kernel family that ran ("attention" or "chain")."""
        import torch
        d = L.SdpaDesc()
        if q.dim() == 4:
            d.batch, d.heads, d.seq, d.head_dim = q.shape
            d.v_head_dim, d.folded = v.shape[3], 0
        else:
            d.batch, d.seq = q.shape[0], q.shape[1]
            d.heads, d.folded = heads, 1
            d.head_dim, d.v_head_dim = q.shape[2] // heads, y.shape[2] // heads
            d.ldq, d.ldk, d.ldv = ldq, ldk, ldv
        d.dtype, d.has_mask, d.scale = dtype_code(q.dtype), int(mask is not None), float(scale)
        h = C.c_void_p()
        L.check(self._lib.sofie_b200_sdpa_plan_create(self._h, C.byref(d), C.byref(h)), "sdpa_plan_create")
        try:
            ws = self.scratch(max(256, self._lib.sofie_b200_sdpa_workspace_bytes(h)))
            L.check(self._lib.sofie_b200_sdpa_enqueue(h, _ptr(q), _ptr(k), _ptr(v), _ptr(mask), _ptr(y), _ptr(ws)), "sdpa_enqueue")
            kernel = self._lib.sofie_b200_sdpa_plan_kernel(h).decode()
            self.sync()   # the workspace is released on return
        finally:
            self._lib.sofie_b200_sdpa_plan_destroy(h)
        return kernel

    def unary(self, x, y, act, act_alpha=0.0):
        L.check(self._lib.sofie_b200_unary_enqueue(self._h, _ptr(x), _ptr(y), dtype_code(x.dtype), x.numel(), act,
                                                   act_alpha), "unary_enqueue")

    def binary(self, a, b, y, op=0, act=L.ACT_NONE):
        L.check(self._lib.sofie_b200_binary_enqueue(self._h, _ptr(a), _ptr(b), _ptr(y), dtype_code(a.dtype),
                                                    a.numel(), b.numel(), op, act), "binary_enqueue")

    def batchnorm(self, x, y, fused_scale, bias, mean, act=L.ACT_NONE):
        outer, ch = x.shape[0], x.shape[1]
        inner = x.numel() // (outer * ch) if outer * ch else 0
        L.check(self._lib.sofie_b200_batchnorm_enqueue(self._h, _ptr(x), _ptr(y), outer, ch, inner,
                                                       _ptr(fused_scale), _ptr(bias), _ptr(mean), act),
                "batchnorm_enqueue")

    def global_avgpool(self, x, y):
        nc = x.shape[0] * x.shape[1]
        inner = x.numel() // nc if nc else 0
        L.check(self._lib.sofie_b200_global_avgpool_enqueue(self._h, _ptr(x), _ptr(y), dtype_code(x.dtype), nc,
                                                            inner), "global_avgpool_enqueue")

    def global_avgpool_nhwc(self, x, y):
        """x: channels-last [n, ..., c]; y: [n, c] fp32."""
        n, c = x.shape[0], x.shape[-1]
        pixels = x.numel() // (n * c) if n * c else 0
        L.check(self._lib.sofie_b200_global_avgpool_nhwc_enqueue(self._h, _ptr(x), _ptr(y), dtype_code(x.dtype), n, pixels, c),
                "global_avgpool_nhwc_enqueue")

    def quantize(self, x, q, scale, zero_point, channels=1, inner=1):
        L.check(self._lib.sofie_b200_quantize_enqueue(self._h, _ptr(x), _ptr(q), dtype_code(q.dtype), x.numel(),
                                                      _ptr(scale), _ptr(zero_point), channels, inner),
                "quantize_enqueue")

    def dequantize(self, q, x, scale, zero_point, channels=1, inner=1):
        L.check(self._lib.sofie_b200_dequantize_enqueue(self._h, _ptr(q), _ptr(x), dtype_code(q.dtype), q.numel(),
                                                        _ptr(scale), _ptr(zero_point), channels, inner),
                "dequantize_enqueue")

    def attention(self, qkv, out, batch, seq, heads, head_dim, scale):
        """qkv [batch, seq, 3, heads, head_dim] -> out [batch, seq, heads * head_dim] (fused Softmax(scale Q K^T) V)."""
        L.check(self._lib.sofie_b200_attention_enqueue(self._h, _ptr(qkv), _ptr(out), dtype_code(qkv.dtype), batch, seq, heads, head_dim,
                                                       float(scale)), "attention_enqueue")

    def kv_append(self, k, v, kv, cu_seqlens=None, cos=None, sin=None, interleaved=False, q=None, q_out=None, k_out=None):
        """Appends keys and values of new tokens to a paged cache (`kv`, a PagedKV), rotating keys and queries by their positions
        on the way.  k, v: [tokens, kv_heads, head_dim]; q, q_out: [tokens, heads, head_dim]; k_out: the rotated keys once more,
        packed, for PromptAttentionPlan.  cos, sin: fp32 [positions, rotary_dim / 2], absent = no rotation.  cu_seqlens: int32
        [batch + 1], the packed rows of each sequence; absent = one token per sequence.  Token rows may be column blocks of a
        wider tensor.  q_out may be q, k_out may be k."""
        dev = self.device
        tokens, kv_heads, dim, ldk, pk = _rows("k", k, dev)
        dtype = k.dtype
        if kv._device != dev:
            _wrong_device("kv_append: the cache", kv.k, dev)
        if kv_heads != kv.kv_heads or dim != kv.head_dim or dtype is not kv.dtype:
            raise ValueError(f"kv_append: keys of {kv_heads} heads of {dim} {dtype}, cache of {kv.kv_heads} of {kv.head_dim} {kv.dtype}")
        n, h, e, ldv, pv = _rows("v", v, dev)
        if n != tokens or h != kv_heads or e != dim or v.dtype is not dtype:
            raise ValueError(f"kv_append: values {tuple(v.shape)} {v.dtype} beside keys {tuple(k.shape)} {dtype}")
        ldko = heads = ldq = ldqo = rotary = positions = 0
        pko = pq = pqo = pcos = psin = pcu = None
        if k_out is not None:
            n, h, e, ldko, pko = _rows("k_out", k_out, dev)
            if n != tokens or h != kv_heads or e != dim or k_out.dtype is not dtype:
                raise ValueError(f"kv_append: k_out {tuple(k_out.shape)} {k_out.dtype} beside keys {tuple(k.shape)} {dtype}")
        if q is not None:
            if q_out is None:
                raise ValueError("kv_append: q needs q_out")
            n, heads, e, ldq, pq = _rows("q", q, dev)
            m, h, f, ldqo, pqo = _rows("q_out", q_out, dev)
            if n != tokens or e != dim or q.dtype is not dtype:
                raise ValueError("kv_append: q and k differ in tokens, head size or type")
            if m != tokens or h != heads or f != dim or q_out.dtype is not dtype:
                raise ValueError(f"kv_append: q_out {tuple(q_out.shape)} {q_out.dtype} beside queries {tuple(q.shape)} {dtype}")
        elif q_out is not None:
            raise ValueError("kv_append: q_out needs q")
        if cos is not None or sin is not None:
            if cos is None or sin is None or cos.dim() != 2 or cos.shape != sin.shape or not (cos.is_contiguous() and sin.is_contiguous()):
                raise ValueError("kv_append: cos and sin are two contiguous tensors of one shape [positions, rotary_dim / 2]")
            if cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
                raise TypeError("kv_append: cos and sin are fp32")
            positions, rotary = cos.shape
            rotary *= 2
            if rotary:
                if cos.get_device() != dev or sin.get_device() != dev:
                    _wrong_device("kv_append: cos and sin", cos if cos.get_device() != dev else sin, dev)
                pcos, psin = cos.data_ptr(), sin.data_ptr()
        if cu_seqlens is not None:
            pcu = _offsets("cu_seqlens", cu_seqlens, kv.batch, dev)
        d = L.KvAppendDesc(tokens, heads, kv_heads, dim, rotary, 1 if interleaved else 0, kv._dtype_code, positions, ldq, ldk, ldv, ldqo, ldko)
        status = self._lib.sofie_b200_kv_append_enqueue(self._h, C.byref(d), kv._ref, pcu, pq, pk, pv, pcos, psin, pqo, pko)
        if status:
            L.check(status, "kv_append_enqueue")

    def depth_unfold(self, x, y, taps, d_out, stride_d=1, pad_front=0, dil_d=1):
        """x [n, c, d, h, w] -> y [n * d_out, c * taps, h, w]: the depth taps of a 3-D convolution as channels."""
        n, c, d = x.shape[:3]
        hw = int(x[0, 0, 0].numel())
        L.check(self._lib.sofie_b200_depth_unfold_enqueue(self._h, _ptr(x), _ptr(y), dtype_code(x.dtype), n, c, d, hw, taps, d_out, stride_d, pad_front, dil_d),
                "depth_unfold_enqueue")

    def transpose(self, x, y, perm):
        shape = (C.c_int64 * x.dim())(*x.shape)
        pm = (C.c_int32 * x.dim())(*perm)
        L.check(self._lib.sofie_b200_transpose_enqueue(self._h, _ptr(x), _ptr(y), dtype_code(x.dtype), x.dim(), shape, pm),
                "transpose_enqueue")

    def convert(self, x, y, row_scale=None):
        cols = x.shape[-1]
        rows = x.numel() // cols if cols else 0
        L.check(self._lib.sofie_b200_convert_enqueue(self._h, _ptr(x), _ptr(y), dtype_code(x.dtype),
                                                     dtype_code(y.dtype), rows, cols, _ptr(row_scale)),
                "convert_enqueue")


def _rows(name, t, device):
    """(tokens, heads, head size, token pitch, address) of a [tokens, heads, head_dim] tensor on GPU `device` whose rows may be
    column blocks of wider ones."""
    shape = t.shape
    if len(shape) != 3:
        raise ValueError(f"{name}: [tokens, heads, head_dim] is expected, not {tuple(shape)}")
    n, h, d = shape
    sn, sh, sd = t.stride()
    if (sd != 1 and d > 1) or (sh != d and h > 1):
        raise ValueError(f"{name}: the heads of a token must lie one behind another (strides {t.stride()})")
    if n > 1 and sn < h * d:   # also a row expanded over all tokens: its stride, 0, is what the C side takes for "dense"
        raise ValueError(f"{name}: rows lie over one another (strides {t.stride()}); an expanded tensor needs contiguous()")
    if t.get_device() != device:
        _wrong_device(name, t, device)
    return n, h, d, sn if n > 1 else h * d, t.data_ptr()


def _wrong_device(name, t, device):
    if not t.is_cuda:
        raise ValueError("sofie_b200 operators take CUDA tensors; host data goes through run_host()")
    raise ValueError(f"{name}: on {t.device}, the context's device is cuda:{device}")


def _offsets(name, t, batch, device):
    """Address of an int32 tensor of batch + 1 row offsets on GPU `device`."""
    if t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] != batch + 1 or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous int32 tensor of batch + 1 = {batch + 1} row offsets is expected")
    if t.get_device() != device:
        _wrong_device(name, t, device)
    return t.data_ptr()


class PagedKV:
    """A paged key-value cache and the sequences in it (sofie_b200_paged_kv): k and v [pages, page_size, kv_heads, head_dim] of
    one shape and equal strides (innermost 1; a permuted or sliced view is fine), block_table int32 [batch, pages per sequence],
    seq_lens int32 [batch] (lengths after the tokens of a pending append).  The object keeps the tensors; their contents may
    change between calls (also under a captured graph), their places may not."""

    def __init__(self, k, v, block_table, seq_lens):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.stride() != v.stride():
            raise ValueError("PagedKV: k and v are [pages, page_size, kv_heads, head_dim] of one shape, type and strides")
        pages, page_size, kv_heads, dim = k.shape
        if page_size < 1 or kv_heads < 1 or dim < 1 or (dim > 1 and k.stride(3) != 1):
            raise ValueError("PagedKV: the head dimension must be the innermost, without gaps")
        for name, t, rank in (("block_table", block_table, 2), ("seq_lens", seq_lens, 1)):
            if t.dtype != torch.int32 or t.dim() != rank or (t.shape[-1] > 1 and t.stride(-1) != 1):
                raise ValueError(f"PagedKV: {name} is an int32 tensor of rank {rank}, contiguous along its last axis")
        if block_table.shape[0] != seq_lens.shape[0]:
            raise ValueError("PagedKV: one row of the block table per sequence")
        if block_table.shape[0] > 1 and block_table.stride(0) < block_table.shape[1]:   # 0, as expand leaves it, is "dense" to the C side
            raise ValueError(f"PagedKV: rows of block_table lie over one another (strides {block_table.stride()}); an expanded table needs contiguous()")
        if any(n > 1 and s == 0 for n, s in zip(k.shape[:3], k.stride())):
            raise ValueError(f"PagedKV: elements of k and v lie over one another (strides {k.stride()})")
        if len({t.device for t in (k, v, block_table, seq_lens)}) != 1:
            raise ValueError("PagedKV: all tensors live on one device")
        self.k, self.v, self.block_table, self.seq_lens = k, v, block_table, seq_lens
        self.kv_heads, self.head_dim, self.dtype, self.batch = kv_heads, dim, k.dtype, seq_lens.shape[0]
        self._dtype_code, self._device = dtype_code(k.dtype), k.get_device()
        width = block_table.shape[1]
        # the stride of an axis of one element says nothing: the dense one stands for it
        hs = k.stride(2) if kv_heads > 1 else dim
        ts = k.stride(1) if page_size > 1 else max(hs, dim) * kv_heads
        ps = k.stride(0) if pages > 1 else max(ts * page_size, hs * kv_heads)
        self._desc = L.PagedKv(_ptr(k), _ptr(v), _ptr(block_table), _ptr(seq_lens), self.batch, pages, width,
                               block_table.stride(0) if self.batch > 1 else width, ps, ts, hs, page_size)
        self._ref = C.byref(self._desc)


class PromptAttentionPlan:
    """Attention over packed prompts (sofie_b200_prompt_attention_plan): causal or full, heads / kv_heads query heads per key head."""

    def __init__(self, ctx: Context, heads, kv_heads, head_dim, dtype, causal=True, scale=0.0):
        self.ctx, self._lib, self._dtype = ctx, ctx._lib, dtype
        self._shape = (heads, kv_heads, head_dim)
        self._desc = (heads, kv_heads, head_dim, dtype_code(dtype), int(causal), float(scale))
        self._plans = {}
        self._plan((0, 0, 0, 0))   # refuses at once what no pitch could mend

    def _plan(self, pitches):
        h = self._plans.get(pitches)
        if h is None:
            h = C.c_void_p()
            d = L.PromptAttentionDesc(*self._desc, *pitches)
            L.check(self._lib.sofie_b200_prompt_attention_plan_create(self.ctx._h, C.byref(d), C.byref(h)), "prompt_attention_plan_create")
            self._plans[pitches] = h
        return h

    @property
    def kernel(self) -> str:
        return self._lib.sofie_b200_prompt_attention_plan_kernel(self._plan((0, 0, 0, 0))).decode()

    def enqueue(self, q, k, v, y, cu_seqlens, cu_seqlens_k=None) -> None:
        """q, y: [tokens, heads, head_dim]; k, v: [key tokens, kv_heads, head_dim], rows packed sequence behind sequence;
        cu_seqlens (and cu_seqlens_k, where keys have other lengths than queries): int32 [batch + 1] row offsets."""
        dtype, dev = self._dtype, self.ctx.device
        n, h, d, ldq, pq = _rows("q", q, dev)
        nk, hk, dk, ldk, pk = _rows("k", k, dev)
        nv, hv, dv, ldv, pv = _rows("v", v, dev)
        ny, hy, dy, ldy, py = _rows("y", y, dev)
        if (h, hk, d) != self._shape or dk != d or nv != nk or hv != hk or dv != d or ny != n or hy != h or dy != d:
            raise ValueError(f"prompt attention: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}, y {tuple(y.shape)} do not match the plan")
        if q.dtype is not dtype or k.dtype is not dtype or v.dtype is not dtype or y.dtype is not dtype:
            raise ValueError(f"prompt attention: {q.dtype}, {k.dtype}, {v.dtype}, {y.dtype} where the plan has {dtype}")
        batch = cu_seqlens.numel() - 1
        if batch < 0:
            raise ValueError("cu_seqlens: batch + 1 row offsets are expected")
        pcu = _offsets("cu_seqlens", cu_seqlens, batch, dev)
        pck = _offsets("cu_seqlens_k", cu_seqlens_k, batch, dev) if cu_seqlens_k is not None else None
        status = self._lib.sofie_b200_prompt_attention_enqueue(self._plan((ldq, ldk, ldv, ldy)), pq, pk, pv, py, pcu, pck, batch, n, nk)
        if status:
            L.check(status, "prompt_attention_enqueue")

    def close(self) -> None:
        for h in self._plans.values():
            self._lib.sofie_b200_prompt_attention_plan_destroy(h)
        self._plans = {}

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class PagedAttentionPlan:
    """Attention of one new token per sequence over a paged cache (sofie_b200_paged_attention_plan).  The plan owns the
    workspace in which the parts of split sequences meet, so its calls belong on one stream, the context's; graphs that are
    replayed side by side need a plan (and a context) each."""

    def __init__(self, ctx: Context, heads, kv_heads, head_dim, dtype, scale=0.0):
        self.ctx, self._lib, self._dtype = ctx, ctx._lib, dtype
        self._shape = (heads, kv_heads, head_dim)
        self._desc = (heads, kv_heads, head_dim, dtype_code(dtype), float(scale))
        self._plans = {}
        self._workspace = None
        h = self._plan((0, 0))
        size = int(self._lib.sofie_b200_paged_attention_workspace_bytes(h))
        if size:
            self._workspace = ctx.scratch(size)
        self._workspace_ptr = _ptr(self._workspace)

    def _plan(self, pitches):
        h = self._plans.get(pitches)
        if h is None:
            h = C.c_void_p()
            d = L.PagedAttentionDesc(*self._desc, *pitches)
            L.check(self._lib.sofie_b200_paged_attention_plan_create(self.ctx._h, C.byref(d), C.byref(h)), "paged_attention_plan_create")
            self._plans[pitches] = h
        return h

    @property
    def kernel(self) -> str:
        return self._lib.sofie_b200_paged_attention_plan_kernel(self._plan((0, 0))).decode()

    def enqueue(self, q, kv, y) -> None:
        """q, y: [batch, heads, head_dim]; kv: the PagedKV with the cache and its batch of sequences."""
        dtype, dev = self._dtype, self.ctx.device
        n, h, d, ldq, pq = _rows("q", q, dev)
        ny, hy, dy, ldy, py = _rows("y", y, dev)
        if (h, kv.kv_heads, d) != self._shape or kv.head_dim != d or n != kv.batch or q.dtype is not dtype or kv.dtype is not dtype:
            raise ValueError(f"paged attention: q {tuple(q.shape)} {q.dtype} over {kv.batch} sequences of {kv.kv_heads} heads of {kv.head_dim} "
                             f"{kv.dtype} does not match the plan")
        if kv._device != dev:
            _wrong_device("paged attention: the cache", kv.k, dev)
        if ny != n or hy != h or dy != d or y.dtype is not dtype:
            raise ValueError(f"paged attention: y {tuple(y.shape)} {y.dtype} beside q {tuple(q.shape)} {dtype}")
        status = self._lib.sofie_b200_paged_attention_enqueue(self._plan((ldq, ldy)), pq, kv._ref, py, self._workspace_ptr)
        if status:
            L.check(status, "paged_attention_enqueue")

    def close(self) -> None:
        for h in self._plans.values():
            self._lib.sofie_b200_paged_attention_plan_destroy(h)
        self._plans = {}
        self._workspace = self._workspace_ptr = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def make_epilogue(row_scale=None, col_scale=None, alpha=1.0, beta=1.0, bias=None, bias_mode=None, ldc=0,
                  residual=None, ldr=0, act=L.ACT_NONE, act_alpha=0.0, out_scale=1.0,
                  out_zero_point=0) -> tuple[L.Epilogue, list]:
    """Builds a sofie_b200_epilogue from torch tensors; returns it with the tensors to keep alive."""
    e = L.Epilogue()
    e.row_scale = _ptr(row_scale)
    e.col_scale = _ptr(col_scale)
    e.alpha = alpha
    e.beta = beta
    if bias is not None and bias_mode is None:
        bias_mode = L.BIAS_COL_I32 if bias.dtype == torch.int32 else L.BIAS_COL_F32
    e.bias_mode = bias_mode or L.BIAS_NONE
    e.bias = _ptr(bias)
    e.ldc = ldc
    e.residual = _ptr(residual)
    e.residual_dtype = dtype_code(residual.dtype) if residual is not None else L.F32
    e.ldr = ldr
    e.act = act
    e.act_alpha = act_alpha
    e.out_scale = out_scale
    e.out_zero_point = out_zero_point
    return e, [row_scale, col_scale, bias, residual]


class GemmPlan:
    """One registered contraction (sofie_b200_gemm_plan)."""

    def __init__(self, ctx: Context, M, N, K, ab_dtype, y_dtype, trans_a=False, trans_b=False, batch=1, lda=0,
                 ldb=0, ldy=0, stride_a=0, stride_b=0, stride_y=0, stride_c=0, stride_r=0, precise=True, flags=0):
        self.ctx = ctx
        self._lib = ctx._lib
        d = L.GemmDesc()
        d.M, d.N, d.K, d.batch = M, N, K, batch
        d.trans_a, d.trans_b = int(trans_a), int(trans_b)
        d.ab_dtype = dtype_code(ab_dtype)
        d.y_dtype = dtype_code(y_dtype)
        d.lda, d.ldb, d.ldy = lda, ldb, ldy
        d.stride_a, d.stride_b, d.stride_y = stride_a, stride_b, stride_y
        d.stride_c, d.stride_r = stride_c, stride_r
        d.precise = int(precise)
        d.flags = int(flags)
        self.desc = d
        h = C.c_void_p()
        L.check(self._lib.sofie_b200_gemm_plan_create(ctx._h, C.byref(d), C.byref(h)), "gemm_plan_create")
        self._h = h

    @property
    def kernel(self) -> str:
        return self._lib.sofie_b200_gemm_plan_kernel(self._h).decode()

    def enqueue(self, A, B, Y, epilogue: Optional[L.Epilogue] = None) -> None:
        ep = C.byref(epilogue) if epilogue is not None else None
        L.check(self._lib.sofie_b200_gemm_enqueue(self._h, _ptr(A), _ptr(B), _ptr(Y), ep), "gemm_enqueue")

    def enqueue_peers(self, A, B, y_ptr: int, peer_ptrs, epilogue: Optional[L.Epilogue] = None) -> None:
        """The contraction with every finished row segment stored to `y_ptr` and to each of `peer_ptrs` (raw device
        pointers: this rank's columns inside its own and inside the other ranks' full-width results)."""
        ep = C.byref(epilogue) if epilogue is not None else None
        n = len(peer_ptrs)
        arr = (C.c_void_p * max(n, 1))(*peer_ptrs)
        L.check(self._lib.sofie_b200_gemm_enqueue_peers(self._h, _ptr(A), _ptr(B), C.c_void_p(y_ptr), arr, n, ep), "gemm_enqueue_peers")

    def run_host(self, hostA, hostB, hostY, epilogue: Optional[L.Epilogue] = None) -> None:
        """Host operands (pinned or pageable CPU tensors): H2D, contraction, D2H, wait."""
        for t in (hostA, hostB, hostY):
            if t.is_cuda or not t.is_contiguous():
                raise ValueError("run_host takes contiguous CPU tensors")
        ep = C.byref(epilogue) if epilogue is not None else None
        L.check(self._lib.sofie_b200_gemm_run_host(self._h, hostA.data_ptr(), hostB.data_ptr(), hostY.data_ptr(), ep),
                "gemm_run_host")

    def run_host_many(self, hostA, hostB, hostY, epilogue: Optional[L.Epilogue] = None) -> None:
        """Lists of host operands, one entry per inference: copies and contractions of successive inferences overlap."""
        n = len(hostA)
        if len(hostB) != n or len(hostY) != n:
            raise ValueError("run_host_many takes three lists of the same length")
        for t in (*hostA, *hostB, *hostY):
            if t.is_cuda or not t.is_contiguous():
                raise ValueError("run_host_many takes contiguous CPU tensors")
        arr = lambda ts: (C.c_void_p * n)(*[t.data_ptr() for t in ts])
        ep = C.byref(epilogue) if epilogue is not None else None
        L.check(self._lib.sofie_b200_gemm_run_host_many(self._h, n, arr(hostA), arr(hostB), arr(hostY), ep), "gemm_run_host_many")

    def close(self) -> None:
        if self._h:
            self._lib.sofie_b200_gemm_plan_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
