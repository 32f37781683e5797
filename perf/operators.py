"""Measured cases of the operators of batched serving: the paged 4-bit key/value cache (appending
rotated keys and values to it, attention over it) and the 8-bit integer matrix product.

Head layouts, widths and the vocabulary are those of tinygiant_b200/_constants.py and of the
tests (32 query heads over 4 kv heads of 128, hidden size 2048, kv_max 4096, vocabulary 151936);
lengths and batches are generic.  `run` computes an operator with elementary torch operations, or,
where `own` is true, with the framework's kernels.

The cache: a page holds `page` tokens of every kv head; [kv head][page / 16] granules of 16 tokens,
each 18 * hd bytes: key codes, value codes (8 * hd bytes each), key scales, value scales (fp16, hd
bytes each).  Blocks of 32 along the head dimension have one scale d = m / -8 (m: the value of the
largest magnitude, the first of several) and codes min(15, floor(x / d + 8.5)); they stand for
fp16(d) * (code - 8), d held in 32 bits before it is cut to 16.  Token 8h + g, dimension 32b + 8i + 2c + e of a key is nibble i of halfword e
of word b in chunk (h, g, c); token 8h + 2c + e, dimension 32b + 8i + g of a value is there too;
key scales are at [token][b], value
scales at [h][c][b][e], token 8h + 2c + e."""
import random

import torch

own = False

F = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6
BASE = 1_000_000.0


def listed():
    heads = dict(nh=32, nkv=4, hd=128, page=64)
    return [
        # one stream's next token: latency of one small call
        dict(name="append 1 token", op="append", dtype="f32", batch=1, tokens=1, past=700, **heads),
        # a decode step of 96 streams of different ages
        dict(name="append 96 streams", op="append", dtype="bf16", batch=96, tokens=1, past=4000, **heads),
        # prompts read in: five ragged chunks of new and of running sequences
        dict(name="append prompts", op="append", dtype="bf16", batch=5, tokens=3600, past=900, **heads),
        # one stream, a short context
        dict(name="attend 1 stream", op="attend", dtype="f32", batch=1, tokens=1, past=611, **heads),
        # a decode step of 32 streams with caches of up to 4096 rows, the framework's own activation type
        dict(name="attend 32 streams", op="attend", dtype="f32", batch=32, tokens=1, past=4000, **heads),
        # one stream at a very long context: few rows of work, a long axis
        dict(name="attend long", op="attend", dtype="bf16", batch=1, tokens=1, past=200000, **heads),
        # a full server: 128 streams of up to 12000 rows
        dict(name="attend 128 streams", op="attend", dtype="bf16", batch=128, tokens=1, past=12000, **heads),
        # prompts read in by chunks of up to 1500 tokens behind what is cached
        dict(name="attend prompts", op="attend", dtype="bf16", batch=3, tokens=1500, past=2500, **heads),
        # the q, k and v projections of one token behind the attention norm
        dict(name="product 1 token", op="product", dtype="f32", m=1, n=5120, k=2048, norm=True, residual=False),
        # the output projection of 96 streams, added to the hidden state
        dict(name="product 96 streams", op="product", dtype="f32", m=96, n=2048, k=4096, norm=False, residual=True),
        # logits of 16 streams
        dict(name="product logits", op="product", dtype="bf16", m=16, n=151936, k=2048, norm=True, residual=False),
        # prompts read in: q, k and v of 8100 tokens
        dict(name="product prompts", op="product", dtype="bf16", m=8100, n=5120, k=2048, norm=True, residual=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    dtype = rng.choice(["f32", "bf16", "f16"])
    op = rng.choice(["append", "attend", "product"])
    if op == "product":
        while True:
            m, n, k = _log(rng, 1, 8000), _log(rng, 33, 60000), _log(rng, 40, 8000)
            if m * n * k <= 6e10 and m * n <= 5e7:
                return dict(op=op, dtype=dtype, m=m, n=n, k=k, norm=rng.random() < 0.5, residual=rng.random() < 0.5)
    hd = rng.choice([64, 96, 128, 128, 128, 256])
    nkv = rng.choice([1, 2, 4, 8])
    nh = nkv * rng.choice([1, 2, 3, 4, 5, 8, 8, 8, 16])
    page = rng.choice([16, 32, 64, 128])
    while True:
        batch, past = _log(rng, 1, 100), _log(rng, 1, 100000)
        tokens = 1 if rng.random() < 0.5 else _log(rng, 2, 2500)
        rows, new = batch * (past + tokens), batch * tokens
        if rows * nkv * hd <= 3e8 and new * nh * hd <= 6e7 and new * nh * hd * (past + tokens) <= 4e10:
            return dict(op=op, dtype=dtype, batch=batch, tokens=tokens, past=past, nh=nh, nkv=nkv, hd=hd, page=page)


def _lengths(case):
    """New tokens and rows cached before them, of each sequence: the first has the case's own numbers,
    the others a spread below them."""
    r = random.Random("%(batch)d %(tokens)d %(past)d" % case)
    new = [case["tokens"]] + [r.randint(max(1, case["tokens"] // 3), case["tokens"]) for _ in range(case["batch"] - 1)]
    past = [case["past"]] + [r.randint(case["past"] // 4, case["past"]) for _ in range(case["batch"] - 1)]
    return new, past


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        moved = m * k * e + n * k + 4 * n + m * n * e * (2 if case["residual"] else 1) + (4 * k if case["norm"] else 0)
        return {"bytes": moved, "flops": 2 * m * n * k}
    new, past = _lengths(case)
    t, nh, nkv, hd = sum(new), case["nh"], case["nkv"], case["hd"]
    row = nkv * hd * 2 * 9 // 16  # a token's codes and scales
    if case["op"] == "append":
        # q, k, v and the angles in, q and the rows out; then the new rows read back as f32
        return {"bytes": t * ((2 * nh + 2 * nkv) * hd * e + 4 * hd + row) + t * (row + 2 * nkv * hd * 4), "flops": 0}
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past))
    return {"bytes": sum(n + p for n, p in zip(new, past)) * row + 2 * t * nh * hd * e, "flops": 4 * pairs * nh * hd}


# ---------------------------------------------------------------- the 4-bit blocks and the pages


def _codes(x):
    """x [..., hd] in 64 bits -> codes (uint8) and scales (fp16) [..., hd / 32]."""
    b = x.unflatten(-1, (-1, 32))
    # the first element of the largest magnitude
    at = (b.abs() == b.abs().amax(-1, keepdim=True)).to(torch.uint8).argmax(-1, keepdim=True)
    m = b.gather(-1, at)
    q = torch.where(m == 0, torch.full_like(b, 8.5), 8.5 - 8.0 * b / m).floor().clamp(0, 15)
    return q.to(torch.uint8).flatten(-2), (m.float() * -0.125).squeeze(-1).half()


def _byte_of(nkv, hd, page, device):
    """Byte within a page of every (kind, kv head, token, dimension) code and (kind, kv head, token, block)
    scale; kind 0 keys, 1 values."""
    kind = torch.arange(2, device=device).view(2, 1, 1, 1)
    head = torch.arange(nkv, device=device).view(1, nkv, 1, 1)
    tok = torch.arange(page, device=device).view(1, 1, page, 1)
    d = torch.arange(hd, device=device).view(1, 1, 1, hd)
    base = (head * (page // 16) + tok // 16) * (18 * hd)
    t, b, i, w = tok % 16, d // 32, d % 32 // 8, d % 8
    g = torch.where(kind == 0, t % 8, w)
    c = torch.where(kind == 0, w // 2, t % 8 // 2)
    e = torch.where(kind == 0, w % 2, t % 2)
    code = base + kind * (8 * hd) + ((t // 8 * 8 + g) * 4 + c) * (hd // 8) + b * 4 + e * 2 + i // 2
    blk = torch.arange(hd // 32, device=device).view(1, 1, 1, -1)
    paired = ((t // 8 * 4 + t % 8 // 2) * (hd // 32) + blk) * 4 + t % 2 * 2
    scale = base + 16 * hd + torch.where(kind == 0, (t * (hd // 32) + blk) * 2, hd + paired)
    return code, scale


def _write(pages, page_of, tok_of, k, v, page):
    """Puts rows k, v [rows][nkv][hd] (64 bits) at (page, token) of `pages` [n][bytes]."""
    nkv, hd = k.shape[1:]
    code, scale = _byte_of(nkv, hd, page, k.device)
    flat, start = pages.view(-1), (page_of * pages.shape[1]).view(-1, 1, 1)
    low = torch.arange(hd, device=k.device) // 8 % 2 == 0  # nibbles 0 and 2, the low ones of their bytes
    for kind, x in ((0, k), (1, v)):
        q, d = _codes(x)
        flat[start + code[kind].permute(1, 0, 2)[tok_of][..., low]] = q[..., low] | (q[..., ~low] << 4)
        at = start + scale[kind].permute(1, 0, 2)[tok_of]
        pair = d.contiguous().view(torch.uint8).unflatten(-1, (-1, 2))
        flat[at] = pair[..., 0]
        flat[at + 1] = pair[..., 1]


def _read(pages, page_of, tok_of, nkv, hd, page):
    """Rows at (page, token) of `pages`: keys and values [rows][nkv][hd], f32."""
    code, scale = _byte_of(nkv, hd, page, pages.device)
    flat, start, out = pages.view(-1), (page_of * pages.shape[1]).view(-1, 1, 1), []
    high = torch.arange(hd, device=pages.device) // 8 % 2 == 1
    for kind in (0, 1):
        byte = flat[start + code[kind].permute(1, 0, 2)[tok_of]]
        at = start + scale[kind].permute(1, 0, 2)[tok_of]
        d = torch.stack((flat[at], flat[at + 1]), -1).view(torch.float16).squeeze(-1).float()
        out.append((torch.where(high, byte >> 4, byte & 15).float() - 8.0) * d.repeat_interleave(32, -1))
    return out


def _values(got, nkv, hd, page):
    """Whole pages' bytes [n][bytes] -> keys and values, each [n][page][nkv][hd] in f32."""
    nb, out = hd // 32, []
    gr = got.view(-1, nkv, page // 16, 18 * hd)
    # from n, head, granule, h, g, c, b, e, i to the token's axes, then the dimension's
    for kind, order in ((0, (0, 1, 2, 3, 4, 6, 8, 5, 7)), (1, (0, 1, 2, 3, 5, 7, 6, 8, 4))):
        y = gr[..., 8 * hd * kind:8 * hd * (kind + 1)].unflatten(-1, (2, 8, 4, nb, 2, 2))
        y = torch.stack((y & 15, y >> 4), -1).flatten(-2).permute(order).reshape(*gr.shape[:3], 16, nb, 32)
        d = gr[..., 16 * hd + hd * kind:16 * hd + hd * (kind + 1)].contiguous().view(torch.float16)
        d = d.unflatten(-1, (2, 4, nb, 2)).permute(0, 1, 2, 3, 4, 6, 5) if kind else d
        d = d.reshape(*gr.shape[:3], 16, nb, 1)
        out.append(((y.float() - 8.0) * d.float()).flatten(-2).flatten(2, 3).permute(0, 2, 1, 3))
    return out


# ---------------------------------------------------------------- inputs


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = F[case["dtype"]]
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        wide = 1.0 + 9.0 * (torch.rand(k, generator=gen, device="cuda") < 0.01)  # a few strong channels
        x = (_normal(gen, m, k) * wide).to(dtype)
        w = _normal(gen, n, k) * 0.02
        scales = w.abs().amax(1) / 127.0
        codes = torch.zeros(n, (k + 15) // 16 * 16, dtype=torch.int8, device="cuda")
        codes[:, :k] = (w / scales[:, None]).round().clamp(-127, 127)
        return {"case": case, "x": x, "codes": codes, "scales": scales,
                "norm": 1.0 + 0.1 * _normal(gen, k) if case["norm"] else None,
                "residual": _normal(gen, m, n).to(dtype) if case["residual"] else None}
    nh, nkv, hd, page = case["nh"], case["nkv"], case["hd"], case["page"]
    new, past = _lengths(case)
    lens = [n + p for n, p in zip(new, past)]
    need = [(n + page - 1) // page for n in lens]
    count, width, t = sum(need) + 3, max(need), sum(new)
    ids = torch.randperm(count, generator=gen, device="cuda")
    col = torch.arange(width, device="cuda")
    first = torch.tensor([0] + need, device="cuda").cumsum(0)
    table = torch.where(col < torch.tensor(need, device="cuda")[:, None],
                        ids[(first[:-1, None] + col).clamp(max=count - 1)], -1).int()
    start = torch.tensor([0] + new, device="cuda").cumsum(0)
    state = {"case": case, "table": table, "lens": torch.tensor(lens, device="cuda", dtype=torch.int32),
             "start": start.int()}
    size = nkv * (page // 16) * 18 * hd
    if case["op"] == "append":
        qkv = _normal(gen, t, (nh + 2 * nkv) * hd)
        angle = torch.arange(max(lens), device="cuda", dtype=torch.float64)[:, None] * BASE ** (
            -torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
        pages = torch.randint(0, 256, (count, size), generator=gen, device="cuda", dtype=torch.uint8)
        return state | {"qkv": qkv.to(dtype), "pages": pages, "cos": angle.cos().float(), "sin": angle.sin().float(),
                        "q_norm": 1.0 + 0.1 * _normal(gen, hd), "k_norm": 1.0 + 0.1 * _normal(gen, hd)}
    # a cache that was filled row by row; rows behind a sequence's last one hold what was there before
    pages = torch.empty(count, size, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 25) // (page * nkv * hd))
    for at in range(0, count, step):
        n = min(step, count - at)
        rows = torch.arange(n * page, device="cuda")
        k, v = _normal(gen, n * page, nkv, hd), _normal(gen, n * page, nkv, hd)
        _write(pages[at:at + n], rows // page, rows % page, k.double(), v.double(), page)
    return state | {"q": (1.5 * _normal(gen, t, nh, hd)).to(dtype), "pages": pages}


# ---------------------------------------------------------------- the operators


def _places(state):
    """Sequence, index in the sequence, cache row, page and token in the page of every new token."""
    start, page = state["start"].long(), state["case"]["page"]
    t = torch.arange(state["qkv"].shape[0] if "qkv" in state else state["q"].shape[0], device="cuda")
    seq = torch.searchsorted(start, t, right=True) - 1
    row = state["lens"].long()[seq] - start[seq + 1] + t
    return seq, t - start[seq], row, state["table"].long()[seq, row // page], row % page


def _rotate(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _append(state):
    case = state["case"]
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    _, _, row, page_of, tok_of = _places(state)
    q, k, v = state["qkv"].split([nh * hd, nkv * hd, nkv * hd], -1)
    q, k, v = q.unflatten(-1, (nh, hd)).float(), k.unflatten(-1, (nkv, hd)).double(), v.unflatten(-1, (nkv, hd)).double()
    cos, sin = state["cos"][row][:, None], state["sin"][row][:, None]
    q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * state["q_norm"]
    k = k / torch.sqrt(k.square().mean(-1, keepdim=True) + EPS) * state["k_norm"].double()  # codes are cut at borders
    q, k = _rotate(q, cos, sin), _rotate(k, cos.double(), sin.double())
    _write(state["pages"], page_of, tok_of, k, v, case["page"])
    keys, values = _read(state["pages"], page_of, tok_of, nkv, hd, case["page"])
    return {"q": q.to(state["qkv"].dtype), "k": keys, "v": values}


def _attend(state):
    case, q, lens, start = state["case"], state["q"], state["lens"].long(), state["start"].long()
    nkv, hd, t = case["nkv"], case["hd"], state["q"].shape[0]
    group, batch = case["nh"] // nkv, lens.numel()
    k, v = (x.reshape(batch, -1, nkv, hd) for x in _values(state["pages"][state["table"].clamp(min=0)], nkv, hd, case["page"]))
    seq, at, row, _, _ = _places(state)
    most = case["tokens"]
    qs = torch.zeros(batch, most, nkv, group, hd, device="cuda")
    qs[seq, at] = q.float().view(t, nkv, group, hd)
    last = (lens - (start[1:] - start[:-1]))[:, None] + torch.arange(most, device="cuda")  # a query's last row
    seen = torch.arange(k.shape[1], device="cuda") <= last[..., None]  # [batch][query][row]
    s = qs.permute(0, 2, 3, 1, 4).flatten(2, 3) @ k.permute(0, 2, 3, 1) * hd ** -0.5
    s = s.unflatten(2, (group, most)).masked_fill(~seen[:, None, None], float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    out = (p.flatten(2, 3) @ v.permute(0, 2, 1, 3)).unflatten(2, (group, most)) / p.sum(-1, keepdim=True)
    return out.permute(0, 3, 1, 2, 4)[seq, at].reshape(t, case["nh"], hd).to(q.dtype)


def _product(state):
    x, k = state["x"], state["x"].shape[1]
    y, r = x.double(), 1.0  # codes are cut at borders
    if state["norm"] is not None:
        r = torch.rsqrt(x.float().square().mean(1, keepdim=True) + EPS)
        y = y * state["norm"].double()
    top = y.abs().amax(1, keepdim=True)
    codes = (y * 127.0 / top.clamp(min=1e-300)).round().float()
    out = (codes @ state["codes"][:, :k].float().T) * (top.float() / 127.0 * r) * state["scales"]
    if state["residual"] is not None:
        out = out + state["residual"].float()
    return out.to(x.dtype)


def _own(state):
    case = state["case"]
    if case["op"] == "product":
        if "handle" not in state:
            from tinygiant_b200.int8 import Int8Linear
            state["handle"] = Int8Linear(state["codes"], state["scales"], state["x"].shape[1])
        return state["handle"](state["x"], norm=state["norm"], eps=EPS, residual=state["residual"])
    if "handle" not in state:
        from tinygiant_b200.paged import PagedBatch, PagedKV4
        state["handle"] = (PagedKV4(case["nkv"], case["hd"], case["page"], pages=state["pages"]),
                           PagedBatch(state["start"], state["lens"], state["table"], case["tokens"]))
    cache, batch = state["handle"]
    if case["op"] == "attend":
        return cache.attention(batch, state["q"])
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    q, k, v = state["qkv"].split([nh * hd, nkv * hd, nkv * hd], -1)
    q = cache.append(batch, q, k, v, state["cos"], state["sin"], state["q_norm"], state["k_norm"], eps=EPS)
    keys, values = cache.read(batch, q.shape[0])
    return {"q": q, "k": keys, "v": values}


def run(state):
    if own:
        return _own(state)
    return {"append": _append, "attend": _attend, "product": _product}[state["case"]["op"]](state)


# ---------------------------------------------------------------- the same from the definitions, in 64 bits


def _exact_rows(case, x, norm, cos, sin):
    x = x.double().view(x.shape[0], -1, case["hd"])
    if norm is None:
        return x
    x = x * norm.double() / (x.pow(2).sum(-1, keepdim=True) / case["hd"] + EPS).pow(0.5)
    half = case["hd"] // 2
    out = torch.empty_like(x)
    out[..., :half] = x[..., :half] * cos - x[..., half:] * sin
    out[..., half:] = x[..., half:] * cos + x[..., :half] * sin
    return out


def _exact_held(x):
    """What the 4-bit blocks of x stand for, by sorting each block's values against the code borders."""
    b = x.reshape(-1, 32)
    big, small = b.max(1).values, b.min(1).values
    # of a positive and a negative value of the same size the first counts
    first = (b == big[:, None]).int().argmax(1) < (b == small[:, None]).int().argmax(1)
    m = torch.where((big > -small) | ((big == -small) & first), big, small)
    scale = (m.float() / -8.0).half().double()
    border = torch.arange(1, 16, device=x.device, dtype=torch.float64) - 8.5  # code j starts at border j
    ratio = torch.where(m[:, None] == 0, torch.zeros_like(b), -8.0 * b / m[:, None])
    code = torch.bucketize(ratio, border, right=True)
    return (scale[:, None] * (code - 8)).view_as(x)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "product":
        x, w = state["x"].double(), state["codes"][:, :case["k"]].double() * state["scales"].double()[:, None]
        y = x if state["norm"] is None else x * state["norm"].double()
        step = y.abs().max(1, keepdim=True).values / 127
        held = torch.where(step > 0, torch.round(y / step), torch.zeros_like(y)) * step
        if state["norm"] is not None:
            held = held / torch.sqrt((x * x).sum(1, keepdim=True) / case["k"] + EPS)
        out = held @ w.T
        return out if state["residual"] is None else out + state["residual"].double()
    nh, nkv, hd, page = case["nh"], case["nkv"], case["hd"], case["page"]
    starts, lens = state["start"].tolist(), state["lens"].tolist()
    if case["op"] == "append":
        row = torch.cat([torch.arange(n - (b - a), n, device="cuda") for a, b, n in zip(starts, starts[1:], lens)])
        cos, sin = (state[s].double()[row][:, None] for s in ("cos", "sin"))
        q, k, v = state["qkv"].split([nh * hd, nkv * hd, nkv * hd], -1)
        return {"q": _exact_rows(case, q, state["q_norm"], cos, sin),
                "k": _exact_held(_exact_rows(case, k, state["k_norm"], cos, sin)),
                "v": _exact_held(_exact_rows(case, v, None, None, None))}
    out = torch.empty(starts[-1], nh, hd, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        a, z = starts[b], starts[b + 1]
        row = torch.arange(n, device="cuda")
        k, v = (x.double() for x in _read(state["pages"], state["table"][b].long()[row // page], row % page, nkv, hd, page))
        for lo in range(a, z, 512):  # queries in pieces
            hi = min(z, lo + 512)
            behind = row[None, :] > (n - (z - a) + torch.arange(lo - a, hi - a, device="cuda"))[:, None]
            for h in range(nh):
                s = state["q"][lo:hi, h].double() @ k[:, h // (nh // nkv)].T / hd ** 0.5
                s[behind] = -torch.inf
                out[lo:hi, h] = torch.softmax(s, 1) @ v[:, h // (nh // nkv)]
    return out
