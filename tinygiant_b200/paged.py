"""The paged 4-bit key/value cache of many sequences and the attention over it: the batched
form of the reference's norm, RoPE, append and attention steps (csrc/libtinygiant.c:380-445),
next to MoEModel.moe_batched, which is the batched form of its MoE block.

    batch = PagedBatch(q_start, kv_lens, page_table)   # int32 device tensors, see below
    cache = PagedKV4(n_kv_heads, head_dim, page_tokens=64, n_pages=4096)
    q = cache.append(batch, q, k, v, cos, sin, q_norm, k_norm)   # rotated q; k and v into the pages
    out = cache.attention(batch, q)

Everything runs on the current stream of the tensors' device (or `stream`), allocates from
torch's caching allocator only, and reads the batch's contents on the device: a captured graph
replays with whatever q_start, kv_lens and page_table hold by then."""
from __future__ import annotations

import ctypes

import torch

from ._lib import (TGX_BF16, TGX_F16, TGX_F32, TGX_KVQ_BAD_LENGTH, TGX_KVQ_BAD_NEW, TGX_KVQ_BAD_PAGE,
                   TGX_KVQ_BAD_POSITION, TgxKvqBatch, TgxKvqCache, check, get_lib)

DTYPES = {torch.float32: TGX_F32, torch.bfloat16: TGX_BF16, torch.float16: TGX_F16}


def dtype_code(t) -> int:
    code = DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"expected float32, bfloat16 or float16, got {t.dtype}")
    return code


# The cudaStream_t of a device's current stream, by the device's index; torch's own accessor
# without the Stream object around it, a tenth of current_stream()'s time.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def stream_handle(device) -> int:
    """The cudaStream_t of the device's current stream."""
    return _raw_stream(device.index)


def on_stream(stream, device):
    """A context in which `stream` (a torch stream or a cudaStream_t handle) is current: work goes
    there, and what is allocated belongs to it."""
    if not isinstance(stream, torch.cuda.Stream):
        stream = torch.cuda.ExternalStream(stream, device=device)
    if stream.device != device:
        raise ValueError(f"the stream is on {stream.device}, the call on {device}")
    return torch.cuda.stream(stream)


def rows_of(t, heads: int, head_dim: int, device, name: str):
    """(pointer, row stride) of token rows [T][heads][head_dim] or [T][heads * head_dim]: each
    row dense, rows any distance apart."""
    shape, stride = t.shape, t.stride()
    if len(shape) == 3:
        ok = shape[1] == heads and shape[2] == head_dim and stride[2] == 1 and (stride[1] == head_dim or heads == 1)
    else:
        ok = len(shape) == 2 and shape[1] == heads * head_dim and stride[1] == 1
    if not ok and t.numel():
        raise ValueError(f"{name}: expected rows of {heads} heads of {head_dim}, dense in a row, got {tuple(shape)} "
                         f"with strides {stride}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the cache on {device}")
    # the stride of a single row says nothing: any value may stand there
    return t.data_ptr(), stride[0] if shape[0] > 1 else heads * head_dim


def _f32(t, shape, device, name):
    if t is None:
        return None
    if t.shape != shape or t.dtype != torch.float32 or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name}: expected contiguous float32 {shape} on {device}")
    return t.data_ptr()


class PagedBatch:
    """The sequences of one step, as int32 device tensors that the caller owns and may refill:
    q_start[B + 1] (sequence b's new tokens are rows q_start[b] .. q_start[b + 1] - 1 of the
    step; rows behind q_start[B] are padding), kv_lens[B] (cached rows, the new ones included)
    and page_table[B][P] (the pages of a sequence in order; entries behind its last row are not
    read).  max_new: no sequence has more new tokens than this (1 for a decode step)."""

    def __init__(self, q_start, kv_lens, page_table, max_new: int):
        dev = q_start.device
        for t, name in ((q_start, "q_start"), (kv_lens, "kv_lens"), (page_table, "page_table")):
            if t.dtype != torch.int32 or not t.is_cuda or t.device != dev or not t.is_contiguous():
                raise ValueError(f"{name}: expected a contiguous int32 cuda tensor on {dev}")
        b = kv_lens.numel()
        if kv_lens.dim() != 1 or q_start.shape != (b + 1,) or page_table.dim() != 2 or page_table.shape[0] != b:
            raise ValueError("expected q_start[B + 1], kv_lens[B] and page_table[B][P]")
        if b < 1 or page_table.shape[1] < 1 or max_new < 1:
            raise ValueError("B, P and max_new must be positive")
        self.device, self.q_start, self.kv_lens, self.page_table, self.max_new = dev, q_start, kv_lens, page_table, max_new
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        self.c = TgxKvqBatch(b, page_table.shape[1], max_new, q_start.data_ptr(), kv_lens.data_ptr(),
                             page_table.data_ptr(), self.status.data_ptr())
        self.ref = ctypes.byref(self.c)

    def check(self):
        """Synchronise the device; raise if a call on this batch since the last check, on whichever
        stream, met contents that do not fit the cache (those tokens or rows were left out), and
        forget it."""
        torch.cuda.synchronize(self.device)   # the calls' streams, whichever they were
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            torch.cuda.synchronize(self.device)
            said = [text for bit, text in ((TGX_KVQ_BAD_PAGE, "a page id outside the cache"),
                                           (TGX_KVQ_BAD_LENGTH, "a length beyond the page table or fewer rows than new tokens"),
                                           (TGX_KVQ_BAD_POSITION, "a position outside the rope tables"),
                                           (TGX_KVQ_BAD_NEW, "more new tokens than max_new or the step's rows, or starts that go back")) if bits & bit]
            raise RuntimeError("paged cache: " + ", ".join(said))


class PagedKV4:
    """One layer's keys and values in 4 bits: pages[n_pages] of page_tokens tokens of every kv
    head (include/tinygiant.h has the layout)."""

    def __init__(self, n_kv_heads: int, head_dim: int, page_tokens: int = 64, n_pages: int | None = None, pages=None,
                 device=0):
        self.lib = get_lib()
        self.page_bytes = int(self.lib.tgx_kvq_page_bytes(n_kv_heads, head_dim, page_tokens))
        if not self.page_bytes:
            raise ValueError(f"no 4-bit pages of {page_tokens} tokens for {n_kv_heads} heads of {head_dim}: page_tokens a "
                             "multiple of 16 up to 1024, head_dim a multiple of 32 up to 256")
        if pages is None:
            if not n_pages or n_pages < 1:
                raise ValueError("n_pages must be positive")
            pages = torch.zeros((n_pages, self.page_bytes), dtype=torch.uint8, device=torch.device("cuda", device)
                                if isinstance(device, int) else device)
        if pages.dtype != torch.uint8 or not pages.is_cuda or not pages.is_contiguous() or pages.dim() != 2 or \
                pages.shape[1] != self.page_bytes:
            raise ValueError(f"pages: expected a contiguous uint8 cuda tensor [n_pages][{self.page_bytes}]")
        self.n_kv_heads, self.head_dim, self.page_tokens, self.pages = n_kv_heads, head_dim, page_tokens, pages
        self.device = pages.device
        self.c = TgxKvqCache(pages.data_ptr(), pages.shape[0], page_tokens, n_kv_heads, head_dim)
        self.ref = ctypes.byref(self.c)

    def _batch(self, batch: PagedBatch):
        if batch.device != self.device:
            raise ValueError(f"the batch is on {batch.device}, the cache on {self.device}")
        return batch.ref

    def append(self, batch: PagedBatch, q, k, v, cos=None, sin=None, q_norm=None, k_norm=None, eps: float = 1e-6,
               positions=None, q_out=None, stream=None):
        """Normalise and rotate the new tokens' heads, put k and v into the pages and return the
        rotated q [T][heads][head_dim] (None for q None).  q, k, v: token rows, views of a fused
        projection's output included; cos / sin: float32 [positions][head_dim / 2]; q_norm /
        k_norm: float32 [head_dim]; positions: int32 [T] when they are not the cache rows."""
        if stream is not None:
            with on_stream(stream, self.device):
                return self.append(batch, q, k, v, cos, sin, q_norm, k_norm, eps, positions, q_out)
        dev, hd = self.device, self.head_dim
        kp, ks = rows_of(k, self.n_kv_heads, hd, dev, "k")
        vp, vs = rows_of(v, self.n_kv_heads, hd, dev, "v")
        code, t = dtype_code(k), k.shape[0]
        if v.dtype != k.dtype or v.shape[0] != t:
            raise ValueError("k and v differ in type or rows")
        heads, qp, qs, op = 0, None, 0, None
        if q is not None:
            heads = q.shape[1] if q.dim() == 3 else q.shape[1] // hd
            qp, qs = rows_of(q, heads, hd, dev, "q")
            if q.dtype != k.dtype or q.shape[0] != t:
                raise ValueError("q and k differ in type or rows")
            if q_out is None:
                q_out = q.new_empty((t, heads, hd))
            elif q_out.dtype != q.dtype or q_out.device != dev or not q_out.is_contiguous() or \
                    q_out.numel() != t * heads * hd:
                raise ValueError("q_out: expected contiguous rows like q")
            op = q_out.data_ptr()
        if (cos is None) != (sin is None):
            raise ValueError("cos and sin go together")
        n_pos = cos.shape[0] if cos is not None else 0
        if positions is not None and (positions.dtype != torch.int32 or positions.device != dev or
                                      positions.shape != (t,) or not positions.is_contiguous()):
            raise ValueError("positions: expected contiguous int32 [T]")
        if not t:
            return q_out
        check(self.lib.tgx_kvq_append(
            self.ref, self._batch(batch), code, t, qp, qs, kp, ks, vp, vs, heads, _f32(q_norm, (hd,), dev, "q_norm"),
            _f32(k_norm, (hd,), dev, "k_norm"), eps, _f32(cos, (n_pos, hd // 2), dev, "cos"),
            _f32(sin, (n_pos, hd // 2), dev, "sin"), n_pos, None if positions is None else positions.data_ptr(), op,
            stream_handle(dev)), self.lib)
        return q_out

    def read(self, batch: PagedBatch, n_tokens: int, stream=None):
        """The held keys and values of the batch's new tokens, float32 [T][kv heads][head_dim]
        each.  A batch whose new tokens are all of a sequence's rows reads all of it."""
        if stream is not None:
            with on_stream(stream, self.device):
                return self.read(batch, n_tokens)
        shape = (n_tokens, self.n_kv_heads, self.head_dim)
        k = torch.empty(shape, dtype=torch.float32, device=self.device)
        v = torch.empty_like(k)
        if n_tokens:
            check(self.lib.tgx_kvq_read(self.ref, self._batch(batch), n_tokens, k.data_ptr(), v.data_ptr(),
                                        stream_handle(self.device)), self.lib)
        return k, v

    def attention(self, batch: PagedBatch, q, out=None, scale: float = 0.0, stream=None):
        """Causal attention of the new tokens' q [T][heads][head_dim] over their sequences' rows;
        scale 0: 1 / sqrt(head_dim).  out may be q."""
        if stream is not None:
            with on_stream(stream, self.device):
                return self.attention(batch, q, out, scale)
        dev, hd = self.device, self.head_dim
        heads = q.shape[1] if q.dim() == 3 else q.shape[1] // hd
        qp, qs = rows_of(q, heads, hd, dev, "q")
        t = q.shape[0]
        if out is None:
            out = q.new_empty((t, heads, hd))
            op, os = out.data_ptr(), heads * hd
        else:
            op, os = rows_of(out, heads, hd, dev, "out")
            if out.dtype != q.dtype or out.shape[0] != t:
                raise ValueError("out: expected rows like q")
        bref = self._batch(batch)
        if not t:
            return out
        n = self.lib.tgx_kvq_attention_scratch_bytes(self.ref, bref, t, heads)
        scratch = self.pages.new_empty(max(n, 256))
        check(self.lib.tgx_kvq_attention(self.ref, bref, dtype_code(q), t, qp, qs, heads, op, os, scale,
                                         scratch.data_ptr(), n, stream_handle(dev)), self.lib)
        return out
