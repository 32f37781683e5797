"""Decode layers of many sequences at once: AttentionModel's and DecodeEngine's batched forms
(the reference runs one token of one sequence, tinygiant/engine.py:188-266, 378-409).

BatchedAttention is the attention half of every layer for the T new tokens of a PagedBatch, next
to MoEModel.moe_batched: projections in 8-bit integers (tinygiant_b200/int8.py), keys and values
in paged 4-bit caches (tinygiant_b200/paged.py).  BatchedEngine puts embeddings, the layers and
the logits around it and generates for a list of prompts."""
from __future__ import annotations

import numpy as np
import torch

from . import _constants as C
from .engine import MoEModel, rope_cache, sample_token
from .int8 import Int8Linear
from .paged import DTYPES, PagedBatch, PagedKV4, on_stream, stream_handle


class BatchedAttention:
    """X += attention(RMSNorm(X) * attn_norm) for token rows X (cuda float32 [T][embed]); rows
    behind the batch's last token stay as they are (an MoE block knows no batch: forward's takes
    every row).

    One page table serves every layer: page p of a sequence is page p of each layer's cache.
    dtype is the type between the two projections of a layer: float32, or bfloat16 / float16,
    whose attention over long prompts runs on the 16-bit tensor cores.  X's elements count as
    rounded to it in front of the norm (those beyond its range stay as they are), and the output
    projection is rounded to it before it is added to X."""

    def __init__(self, embed=C.EMBED_DIM, n_heads=C.N_HEADS, n_kv_heads=C.N_KV_HEADS, head_dim=C.HEAD_DIM,
                 n_layers=C.N_LAYERS, n_pages=1024, page_tokens=64, max_pos=4096, dtype=torch.float32, device=0,
                 eps=C.RMS_EPS):
        if dtype not in DTYPES:
            raise TypeError(f"expected float32, bfloat16 or float16, got {dtype}")
        if n_heads % n_kv_heads or n_heads // n_kv_heads > 32:
            raise ValueError("n_heads must be a multiple of n_kv_heads, at most 32 per kv head")
        self.embed, self.n_heads, self.n_kv_heads, self.head_dim = embed, n_heads, n_kv_heads, head_dim
        self.n_layers, self.dtype, self.eps = n_layers, dtype, float(eps)
        self.device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.caches = [PagedKV4(n_kv_heads, head_dim, page_tokens, n_pages, device=self.device) for _ in range(n_layers)]
        self.layers = [None] * n_layers
        self.cos, self.sin = (torch.from_numpy(a).to(self.device) for a in rope_cache(max_pos, head_dim))

    def _tensor(self, a):
        return torch.as_tensor(a).to(self.device)

    def set_layer(self, layer: int, wq, wk, wv, wo, attn_norm, q_norm=None, k_norm=None):
        """Weights of one layer, [out][in] matrices of float32, bfloat16 or float16 (tensors or
        numpy arrays; quantised here) and float32 norm weights."""
        qd, kvd, parts = self.n_heads * self.head_dim, self.n_kv_heads * self.head_dim, []
        for name, a, shape in (("wq", wq, (qd, self.embed)), ("wk", wk, (kvd, self.embed)), ("wv", wv, (kvd, self.embed)),
                               ("wo", wo, (self.embed, qd))):
            a = self._tensor(a)
            if a.shape != shape:
                raise ValueError(f"{name}: expected {shape}, got {tuple(a.shape)}")
            parts.append(a)
        norms = [None if a is None else self._tensor(a).float().contiguous() for a in (attn_norm, q_norm, k_norm)]
        for name, a, n in zip(("attn_norm", "q_norm", "k_norm"), norms, (self.embed, self.head_dim, self.head_dim)):
            if a is not None and a.shape != (n,):
                raise ValueError(f"{name}: expected ({n},), got {tuple(a.shape)}")
        if norms[0] is None:
            raise ValueError("attn_norm is needed")
        self.layers[layer] = (Int8Linear.quantize(torch.cat(parts[:3])), Int8Linear.quantize(parts[3]), *norms)

    def fill_synthetic(self, seed: int):
        """Random weights N(0, 0.02), norm weights 1."""
        g = torch.Generator(device=self.device).manual_seed(seed)
        qd, kvd = self.n_heads * self.head_dim, self.n_kv_heads * self.head_dim
        one, head = torch.ones(self.embed, device=self.device), torch.ones(self.head_dim, device=self.device)
        for l in range(self.n_layers):
            w = [torch.randn(*s, device=self.device, generator=g) * 0.02
                 for s in ((qd, self.embed), (kvd, self.embed), (kvd, self.embed), (self.embed, qd))]
            self.set_layer(l, *w, one, head, head)

    def layer(self, layer: int, batch: PagedBatch, X, stream=None):
        """X += attention of `layer`: the batch's new tokens, rows of X, into its cache and over it."""
        if stream is not None:
            with on_stream(stream, self.device):
                return self.layer(layer, batch, X)
        if X.dtype != torch.float32 or X.dim() != 2 or X.shape[1] != self.embed or X.device != self.device:
            raise ValueError(f"X: expected float32 [T][{self.embed}] on {self.device}")
        if self.layers[layer] is None:
            raise ValueError(f"layer {layer} has no weights")
        wqkv, wo, attn_norm, q_norm, k_norm = self.layers[layer]
        cache, qd, kvd = self.caches[layer], self.n_heads * self.head_dim, self.n_kv_heads * self.head_dim
        q, k, v = wqkv(X, norm=attn_norm, eps=self.eps, dtype=self.dtype).split((qd, kvd, kvd), 1)
        # rows behind the batch's last token are in nobody's sequence: zeros there leave X's as they are
        o = X.new_zeros((X.shape[0], qd), dtype=self.dtype)
        cache.append(batch, q, k, v, self.cos, self.sin, q_norm, k_norm, self.eps, q_out=o)
        cache.attention(batch, o, out=o)
        if self.dtype == torch.float32:
            return wo(o, out=X, residual=X)
        return X.add_(wo(o))

    def check_moe(self, moe: MoEModel):
        """Raise unless moe's blocks go with these layers."""
        if moe.embed != self.embed or moe.n_layers < self.n_layers or moe.device != self.device.index:
            raise ValueError(f"moe: expected {self.n_layers} layers of width {self.embed} on device {self.device.index}, got "
                             f"{moe.n_layers} of {moe.embed} on device {moe.device}")

    def forward(self, batch: PagedBatch, X, moe: MoEModel | None = None, stream=None):
        """Every layer on X in place: attention, then moe's MoE block when given (X contiguous)."""
        if stream is not None:
            with on_stream(stream, self.device):
                return self.forward(batch, X, moe)
        if moe is not None:
            self.check_moe(moe)
            if not X.is_contiguous():
                raise ValueError("X: expected contiguous rows in front of an MoE block")
        for l in range(self.n_layers):
            self.layer(l, batch, X)
            if moe is not None:
                most = 65536 // moe.top_k   # tokens of one call
                for t in range(0, X.shape[0], most):
                    moe.moe_batched(l, X[t:t + most], stream_handle(self.device))
        return X


class BatchedEngine:
    """DecodeEngine for many sequences: embedding rows, every layer's attention and MoE block, then
    the final RMSNorm and the output projection of each sequence's last new token."""

    def __init__(self, moe: MoEModel | None, attn: BatchedAttention, token_embd, output_norm, output_weight):
        if moe is not None:
            attn.check_moe(moe)
            if moe.n_layers != attn.n_layers:
                raise ValueError("moe and attn differ in layers")
        if token_embd.dtype != torch.float32 or token_embd.dim() != 2 or token_embd.shape[1] != attn.embed:
            raise ValueError(f"token_embd: expected float32 [vocab][{attn.embed}]")
        self.moe, self.attn, self.embd = moe, attn, token_embd.to(attn.device)
        self.norm = output_norm.to(attn.device).float().contiguous()
        self.head = output_weight if isinstance(output_weight, Int8Linear) else \
            Int8Linear.quantize(output_weight.to(attn.device))
        self.vocab = self.head.out_features
        if self.embd.shape[0] != self.vocab or self.head.in_features != attn.embed or self.norm.shape != (attn.embed,):
            raise ValueError("embeddings, output norm and output weights differ in size")

    @classmethod
    def synthetic(cls, moe: MoEModel | None, attn: BatchedAttention, vocab: int, seed: int):
        """Random embeddings and output weights N(0, 0.02), output norm weights 1."""
        g = torch.Generator(device=attn.device).manual_seed(seed)
        embd, head = (torch.randn(vocab, attn.embed, generator=g, device=attn.device) * 0.02 for _ in range(2))
        return cls(moe, attn, embd, torch.ones(attn.embed), head)

    def step(self, batch: PagedBatch, tokens, stream=None):
        """Logits float32 [B][vocab] behind each sequence's last new token; tokens: int [T] on the
        device, the batch's new tokens in its rows' order (an id outside the vocabulary counts as
        the nearest in it).  The row of a sequence without new tokens says nothing."""
        if stream is not None:
            with on_stream(stream, self.attn.device):
                return self.step(batch, tokens)
        if tokens.dim() != 1 or not tokens.numel() or tokens.device != self.attn.device:
            raise ValueError(f"tokens: expected at least one, in a row on {self.attn.device}")
        X = self.attn.forward(batch, self.embd.index_select(0, tokens.clamp(0, self.vocab - 1)), self.moe)
        last = (batch.q_start[1:] - 1).clamp(0, X.shape[0] - 1)
        return self.head(X.index_select(0, last), norm=self.norm, eps=self.attn.eps)

    def generate(self, prompts, n_tokens: int = 128, temperature: float = 0.7, top_p: float = 0.9, rng=np.random):
        """Yield n_tokens lists, the next token of every prompt (lists of ids, none empty); the
        prompts are read in one step.  Greedy on the device when temperature is 0, else
        sample_token on the host.  Takes pages 0, 1, ... of the caches as it needs them."""
        dev, pt = self.attn.device, self.attn.caches[0].page_tokens
        lens = [len(p) for p in prompts]
        if not lens or min(lens) < 1 or n_tokens < 1:
            raise ValueError("expected prompts of at least one token, and tokens to generate")
        if any(not 0 <= t < self.vocab for p in prompts for t in p):
            raise ValueError(f"a token outside the vocabulary of {self.vocab}")
        if max(lens) + n_tokens - 1 > self.attn.cos.shape[0]:
            raise ValueError(f"positions up to {max(lens) + n_tokens - 1}: the rope tables end at {self.attn.cos.shape[0]}")
        need = [-(-(n + n_tokens - 1) // pt) for n in lens]
        if sum(need) > self.attn.caches[0].pages.shape[0]:
            raise ValueError(f"{sum(need)} pages needed, {self.attn.caches[0].pages.shape[0]} there")
        first = np.concatenate(([0], np.cumsum(need)))
        table = np.full((len(lens), max(need)), -1, np.int32)
        for b, n in enumerate(need):
            table[b, :n] = np.arange(first[b], first[b] + n)
        table, kv_lens = torch.from_numpy(table).to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)
        start = torch.from_numpy(np.concatenate(([0], np.cumsum(lens))).astype(np.int32)).to(dev)
        one = torch.arange(len(lens) + 1, dtype=torch.int32, device=dev)
        batch = PagedBatch(start, kv_lens, table, max(lens))
        tokens = torch.tensor([t for p in prompts for t in p], dtype=torch.int64, device=dev)
        for i in range(n_tokens):
            logits = self.step(batch, tokens)
            if temperature <= 0:
                tokens = logits.argmax(1)
                said = tokens.tolist()
            else:
                said = [sample_token(row, temperature, top_p, rng) for row in logits.cpu().numpy()]
                tokens = torch.tensor(said, dtype=torch.int64, device=dev)
            if i == 0:
                batch.check()
                batch = PagedBatch(one, kv_lens, table, 1)
            kv_lens += 1
            yield said
