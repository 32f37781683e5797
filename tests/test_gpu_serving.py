"""Decode layers of many sequences (tinygiant_b200/serving.py): the int8 projections, the 4-bit
cache's append and its attention as one layer runs them, stage by stage against plain 64-bit
forms; steps of prompts and single tokens, captured ones, and generation."""
from __future__ import annotations

import pytest

from tests import serve_ref as R

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
EMB, NH, NKV, HD, PAGE = 192, 6, 2, 64, 16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def build(dtype=F32, n_layers=1, n_pages=64, seed=1, max_pos=400):
    from tinygiant_b200.serving import BatchedAttention
    a = BatchedAttention(EMB, NH, NKV, HD, n_layers, n_pages, PAGE, max_pos, dtype)
    g = gen(seed)
    qd, kvd, w = NH * HD, NKV * HD, []
    for l in range(n_layers):
        m = [torch.randn(*s, generator=g, device="cuda") * s[1] ** -0.5 for s in ((qd, EMB), (kvd, EMB), (kvd, EMB), (EMB, qd))]
        n = [1 + 0.2 * torch.randn(s, generator=g, device="cuda") for s in (EMB, HD, HD)]
        a.set_layer(l, *m, *n)
        w.append((m, n))
    return a, w


def batch_of(seqs, width=12, max_new=None, ids=None):
    """seqs: (new tokens, rows with them)."""
    from tinygiant_b200.paged import PagedBatch
    start = [0]
    for n, _ in seqs:
        start.append(start[-1] + n)
    if ids is None:
        ids = torch.arange(len(seqs) * width, dtype=torch.int32).view(len(seqs), width).flip(1).contiguous()
    return PagedBatch(torch.tensor(start, dtype=torch.int32).cuda(),
                      torch.tensor([r for _, r in seqs], dtype=torch.int32).cuda(), ids.cuda(),
                      max_new or max(max(n for n, _ in seqs), 1))


def weights(lin):
    return lin.codes[:, :lin.in_features].double(), lin.scales.double()


def product_close(got, x, lin, norm, eps, residual, dtype):
    """The codes of x are integers that a product in 64 bits holds exactly; where y * 127 / top
    lies within the fp32 rounding of a half, either code is right: that moves a result by one
    step of x times a weight.  The rest: the scales (4 roundings of 2^-24), the product with
    them and the residual (3 more), and the type's own rounding.  Below 2^-14 fp16 has steps of
    2^-24 whatever the value, so its rounding is off by up to 2^-25 there, more than 2^-11 of it."""
    codes, s = R.i8_rows(x, norm, eps)
    w, sw = weights(lin)
    y = x.double() if norm is None else x.double() * norm.double()
    t = 127 * y / y.abs().amax(1, keepdim=True).clamp(min=1e-300)
    tie = ((t - torch.floor(t) - 0.5).abs() <= t.abs() * 4 * 2.0 ** -24 + 2.0 ** -40).double()
    ref = codes @ w.T * s * sw
    tol = (tie @ w.abs().T) * s * sw + 8 * 2.0 ** -24 * ref.abs()
    if residual is not None:
        ref = ref + residual.double()
        tol = tol + 2.0 ** -24 * (residual.double().abs() + ref.abs())
    tol = tol + 1.01 * R.EPS[dtype] * ref.abs() + (1.01 * 2.0 ** -25 if dtype == F16 else 1e-30)
    worst = ((got.double() - ref).abs() / tol).max().item()
    assert worst <= 1.0, worst


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("seqs", [[(5, 5), (1, 1), (33, 40)], [(1, 17), (1, 130), (1, 1), (1, 64)], [(0, 9), (150, 180)]])
def test_layer_is_its_stages(seqs, dtype):
    """Each stage on what the one in front has given, and the layer the same bits as its stages."""
    a, w = build(dtype)
    (lin, wo, an, qn, kn), cache = a.layers[0], a.caches[0]
    g = gen(7)
    past = [(r - n, r - n) for n, r in seqs]
    if sum(n for n, _ in past):   # what the caches hold before
        X = torch.randn(sum(n for n, _ in past), EMB, generator=g, device="cuda")
        b = batch_of(past)
        a.layer(0, b, X)
        b.check()
    T = sum(n for n, _ in seqs)
    X = torch.randn(T, EMB, generator=g, device="cuda")
    batch, before = batch_of(seqs), X.clone()
    got = a.layer(0, batch, X)
    assert got is X
    batch.check()
    # the stages by hand (the appended rows are the same, so appending again changes nothing)
    x = before.to(dtype)
    qkv = lin(x, norm=an, eps=a.eps)
    product_close(qkv, x, lin, an, a.eps, None, dtype)
    q, k, v = qkv.split((NH * HD, NKV * HD, NKV * HD), 1)
    pages = cache.pages.clone()
    rq = cache.append(batch, q, k, v, a.cos, a.sin, qn, kn, a.eps)
    assert torch.equal(cache.pages, pages)
    pos = torch.tensor([r - n + i for n, r in seqs for i in range(n)], device="cuda")
    cos, sin = a.cos[pos], a.sin[pos]
    # a rotated element: the norm's 4 roundings and its weight, two products and their sum
    for src, wt, out, heads in ((q, qn, rq, NH),):
        ref = R.norm_rope(src.double().view(T, heads, HD), wt, a.eps, cos, sin)
        n = R.norm_rope(src.double().view(T, heads, HD), wt, a.eps, None, None).abs()
        pair = torch.cat((n[..., HD // 2:], n[..., :HD // 2]), -1)
        tol = 16 * 2.0 ** -24 * (n + pair) + 1.01 * R.EPS[dtype] * ref.abs() + 1e-30
        assert ((out.double() - ref).abs() <= tol).all()
    # the new rows held: within half a step of the plain ones, a step being 1/8 of the block's
    # largest (its fp16 scale off by 2^-11; codes 0 .. 15 reach one side a step less far, where
    # half a step more is cut off)
    hk, hv = cache.read(batch, T)
    for src, wt, out, rope in ((k, kn, hk, True), (v, None, hv, False)):
        ref = R.norm_rope(src.double().view(T, NKV, HD), wt, a.eps, cos if rope else None, sin if rope else None)
        top = ref.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True).expand(-1, -1, -1, 32).flatten(-2)
        assert ((out.double() - ref).abs() <= top / 8 * 1.002 + 1e-6).all()
    # attention over what the cache holds, read as one batch of whole sequences
    whole = batch_of([(r, r) for _, r in seqs])
    kk, vv = cache.read(whole, sum(r for _, r in seqs))
    o = cache.attention(batch, rq)
    t0 = r0 = 0
    for n, r in seqs:
        ref, spread, size, top = R.attention(rq[t0:t0 + n].double(), kk[r0:r0 + r].double(), vv[r0:r0 + r].double(), HD ** -0.5)
        u = 2.0 ** -24   # as tests/test_gpu_kvq.py's close()
        tol = spread * (2 * (HD + 8) * u * size + (2 * r + 32) * u)
        if dtype != F32:
            tol = tol + spread * (4 * 2.0 ** -11 * size + 3 * 2.0 ** -11)
        tol = tol + r * 2.0 ** -31 * top
        tol = tol + 1.001 * R.EPS[dtype] * (ref.abs() + tol) + 1e-30
        assert ((o[t0:t0 + n].double() - ref).abs() <= tol).all()
        t0, r0 = t0 + n, r0 + r
    o = o.view(T, -1)
    if dtype == F32:
        y = wo(o, residual=before)
        product_close(y, o, wo, None, 0.0, before, dtype)
    else:
        y = wo(o)
        product_close(y, o, wo, None, 0.0, None, dtype)
        y = before + y
    assert torch.equal(got, y)


def test_padding_stays():
    a, _ = build(n_layers=2)
    X = torch.randn(12, EMB, generator=gen(3), device="cuda")
    before = X.clone()
    batch = batch_of([(4, 4), (3, 3)])
    a.forward(batch, X)
    batch.check()
    assert torch.equal(X[7:], before[7:]) and not torch.equal(X[:7], before[:7])
    Y = before[:7].clone()
    a.forward(batch, Y)   # the same rows again, without the padding
    assert torch.equal(X[:7], Y)


def test_one_step_or_many_fill_the_cache_alike():
    """Layer 0's rows depend on X alone, not on how the tokens come."""
    a, _ = build()
    b, _ = build()
    X = torch.randn(40, EMB, generator=gen(5), device="cuda")
    a.layer(0, batch_of([(40, 40)]), X.clone())
    for i in range(0, 40, 8):
        b.layer(0, batch_of([(8, i + 8)]), X[i:i + 8].clone())
    assert torch.equal(a.caches[0].pages, b.caches[0].pages)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured_step_follows_its_batch(dtype):
    """One captured step of 3 sequences, replayed as they grow: the same as steps that are not
    captured.  A second graph of another size shares nothing with it."""
    a, _ = build(dtype, n_layers=2)
    e, _ = build(dtype, n_layers=2)
    rows = [30, 1, 17]
    prompts = torch.randn(sum(r - 1 for r in rows), EMB, generator=gen(2), device="cuda")
    for m in (a, e):
        b = batch_of([(r - 1, r - 1) for r in rows])
        m.forward(b, prompts.clone())
        b.check()
    g = gen(9)
    x, x2 = torch.zeros(3, EMB, device="cuda"), torch.zeros(1, EMB, device="cuda")
    batch, batch2 = batch_of([(1, r) for r in rows]), batch_of([(1, 1)], ids=torch.full((1, 12), 60, dtype=torch.int32))
    graphs = []
    for bb, xx in ((batch, x), (batch2, x2)):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            a.forward(bb, xx.clone())
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a.forward(bb, xx)
        graphs.append(graph)
    lens = batch.kv_lens.clone()
    eager = batch_of([(1, r) for r in rows])
    for step in range(5):
        new = torch.randn(3, EMB, generator=g, device="cuda")
        x.copy_(new)
        batch.kv_lens.copy_(lens + step)
        eager.kv_lens.copy_(lens + step)
        graphs[0].replay()
        graphs[1].replay()
        want = e.forward(eager, new.clone())
        assert torch.equal(x, want), step
    batch.check()


def test_steps_with_experts_and_generation():
    """Prompts of several lengths with the MoE blocks between, greedy, against steps by hand; the
    host's sampling; and what does not fit is refused."""
    import numpy as np
    from tinygiant_b200.engine import MoEModel
    from tinygiant_b200.serving import BatchedAttention, BatchedEngine
    m = MoEModel(256, 256, 8, 2, 2)
    m.fill_synthetic(5)
    a = BatchedAttention(256, 4, 2, 64, 2, 24, 16, 64)
    a.fill_synthetic(6)
    eng = BatchedEngine.synthetic(m, a, 300, 7)
    prompts = [[3, 9, 200], [17], list(range(40, 57))]
    said = list(eng.generate(prompts, 6, temperature=0))
    assert len(said) == 6 and all(len(s) == 3 and all(0 <= t < 300 for t in s) for s in said)
    # by hand, on fresh caches, other pages
    for c in a.caches:
        c.pages.zero_()
    lens, toks = [len(p) for p in prompts], [t for p in prompts for t in p]
    ids = torch.arange(6).int().view(3, 2).flip(0).contiguous()
    for i in range(6):
        batch = batch_of([(n, n) for n in lens] if i == 0 else [(1, n + i) for n in lens], ids=ids)
        X = eng.embd[torch.tensor(toks, device="cuda")]
        for l in range(2):
            a.layer(l, batch, X)
            m.moe_batched(l, X)
        batch.check()
        last = (batch.q_start[1:] - 1).long()
        toks = eng.head(X[last], norm=eng.norm, eps=a.eps).argmax(1).tolist()
        assert toks == said[i], i
    assert len(list(eng.generate(prompts, 2, temperature=0.8, rng=np.random.RandomState(1)))) == 2
    for bad in (dict(prompts=[[1], []]), dict(prompts=[]), dict(n_tokens=0), dict(prompts=[[1] * 60], n_tokens=6),
                dict(prompts=[[1] * 40] * 9, n_tokens=6), dict(prompts=[[300]]), dict(prompts=[[-1]])):
        with pytest.raises(ValueError):
            next(eng.generate(**{**dict(prompts=prompts, n_tokens=4), **bad}))
    m.close()


def test_refusals():
    from tinygiant_b200.serving import BatchedAttention
    with pytest.raises(TypeError):
        BatchedAttention(64, 2, 1, 64, 1, 4, dtype=torch.float64)
    with pytest.raises(ValueError):
        BatchedAttention(64, 3, 2, 64, 1, 4)
    a = BatchedAttention(64, 2, 1, 64, 1, 4)
    batch, X = batch_of([(2, 2)], width=4), torch.zeros(2, 64, device="cuda")
    with pytest.raises(ValueError):
        a.layer(0, batch, X)   # no weights
    a.fill_synthetic(1)
    for bad in (X.half(), X[:, :32], X.cpu()):
        with pytest.raises(ValueError):
            a.layer(0, batch, bad)
    with pytest.raises(ValueError):
        a.set_layer(0, torch.zeros(64, 64), torch.zeros(64, 64), torch.zeros(64, 64), torch.zeros(64, 128), torch.ones(64))
    a.layer(0, batch, X)


def test_rows_that_are_not_finite_keep_to_themselves():
    """NaN in one row reaches that row's experts only: its logits all are NaN, and NaN too has a
    top-k of distinct experts."""
    from tinygiant_b200.engine import MoEModel
    m = MoEModel(256, 256, 8, 2, 1)
    m.fill_synthetic(5)
    for kernels in (1, 2):
        m.set_batched_kernels(kernels)
        X = torch.randn(9, 256, generator=gen(1), device="cuda")
        Y = X.clone()
        Y[4] = float("nan")
        m.moe_batched(0, X)
        m.moe_batched(0, Y)
        m.sync_status()
        keep = [i for i in range(9) if i != 4]
        assert torch.equal(X[keep], Y[keep]) and torch.isnan(Y[4]).any()
    m.close()


def test_step_with_tokens_and_starts_that_do_not_fit():
    """Ids outside the vocabulary and starts behind the last token reach no memory outside."""
    from tinygiant_b200.serving import BatchedAttention, BatchedEngine
    a = BatchedAttention(64, 2, 1, 64, 1, 8, 16, 64)
    a.fill_synthetic(1)
    eng = BatchedEngine.synthetic(None, a, 50, 2)
    want = eng.step(batch_of([(2, 2), (1, 1)], width=4), torch.tensor([49, 0, 7], device="cuda"))
    got = eng.step(batch_of([(2, 2), (1, 1)], width=4), torch.tensor([2 ** 40, -3, 7], device="cuda"))
    assert torch.equal(got, want)
    out = eng.step(batch_of([(2, 2), (9, 9)], width=4), torch.tensor([49, 0, 7], device="cuda"))
    assert out.shape == (2, 50) and torch.equal(out[0], want[0])
    for bad in (torch.zeros(0, dtype=torch.long, device="cuda"), torch.zeros(1, 1, dtype=torch.long, device="cuda"),
                torch.zeros(2, dtype=torch.long)):
        with pytest.raises(ValueError):
            eng.step(batch_of([(1, 1)], width=4), bad)
    with pytest.raises(ValueError):
        BatchedEngine(None, a, torch.zeros(49, 64), torch.ones(64), torch.zeros(50, 64))


def test_two_streams_at_once():
    """Prompts on one stream and single tokens on another, each on its own cache, over and over: the
    same bits as one after the other."""
    from tests.test_gpu_kvq import Setup
    from tinygiant_b200.int8 import Int8Linear
    p = Setup([(300, 900), (257, 257), (90, 1200)], 32, 4, 128, 64, BF16, seed=1)
    d = Setup([(1, 700 + 13 * i) for i in range(24)], 32, 4, 128, 64, BF16, seed=2)
    lin = Int8Linear.quantize(torch.randn(1000, 640, generator=gen(3), device="cuda"))
    x = torch.randn(700, 640, generator=gen(4), device="cuda")
    want = [p.cache.attention(p.batch, p.q), lin(x), d.cache.attention(d.batch, d.q), lin(x[:5])]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        got.append((p.cache.attention(p.batch, p.q, stream=streams[0]), lin(x, stream=streams[0]),
                    d.cache.attention(d.batch, d.q, stream=streams[1]), lin(x[:5], stream=streams[1])))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_experts_of_hidden_states_that_are_not_finite():
    """Infinities and NaN among the hidden values, and the largest finite ones: each token still
    goes to distinct experts, and its neighbours keep their values."""
    import numpy as np
    from tinygiant_b200.engine import MoEModel
    m = MoEModel(256, 256, 8, 3, 1)
    m.fill_synthetic(5)
    rows = torch.randn(6, 256, generator=gen(1), device="cuda")
    want = rows.clone()
    m.moe_batched(0, want)
    rows[0, 3], rows[0, 200] = float("inf"), float("inf")
    rows[1, 3], rows[1, 200] = float("inf"), -float("inf")
    rows[3, 7] = float("nan")
    rows[4] = 3.4e38
    got = rows.clone()
    m.moe_batched(0, got)
    assert torch.equal(got[[2, 5]], want[[2, 5]])
    for row in rows:
        m.moe_layer(0, row.clone())
        idx, _, logits = m.last_routing(0)
        order = sorted(range(8), key=lambda i: (np.where(np.isnan(logits), -np.inf, logits)[i], i), reverse=True)[:3]
        assert sorted(idx) == sorted(order)
    m.close()


def test_hidden_values_beyond_the_16_bit_types(dtype=F16):
    """A hidden state with values that fp16 does not reach: the norm brings them back."""
    a, _ = build(dtype)
    b, _ = build(F32)
    X = torch.randn(9, EMB, generator=gen(3), device="cuda")
    X[2, 5], X[4, 7], X[4, 100] = 1e5, -3e6, 2e6
    X[6] *= 1e5
    want = b.layer(0, batch_of([(9, 9)]), X.clone())
    got = a.layer(0, batch_of([(9, 9)]), X.clone())
    assert torch.isfinite(got).all()
    # the layer's own term, to what 8-bit codes and 4-bit rows that fall on the other side of a border may cost
    d, size = (got - want).norm(dim=1), (want - X).norm(dim=1)
    assert (d <= 0.2 * size).all(), (d / size).tolist()


def test_device_without_an_index():
    from tinygiant_b200.serving import BatchedAttention
    a = BatchedAttention(64, 2, 1, 64, 1, 4, device="cuda")
    a.fill_synthetic(1)
    X = torch.randn(2, 64, device="cuda")
    b = BatchedAttention(64, 2, 1, 64, 1, 4, device=0)
    b.fill_synthetic(1)
    assert torch.equal(a.layer(0, batch_of([(2, 2)], width=4), X.clone()), b.layer(0, batch_of([(2, 2)], width=4), X.clone()))


def test_experts_that_do_not_go_with_the_layers():
    """Another width, number of layers or device is refused before anything runs, as are rows that
    the MoE block cannot take."""
    from types import SimpleNamespace
    from tinygiant_b200.serving import BatchedAttention, BatchedEngine
    a = BatchedAttention(64, 2, 1, 64, 1, 8, 16, 64)
    a.fill_synthetic(1)
    X = torch.randn(3, 64, generator=gen(2), device="cuda")
    before, fits = X.clone(), dict(embed=64, n_layers=1, device=0, top_k=2)
    a.check_moe(SimpleNamespace(**fits))
    for bad in (dict(embed=128), dict(n_layers=0), dict(device=1), dict(n_layers=2)):
        moe = SimpleNamespace(**{**fits, **bad})
        if moe.n_layers < 2:
            with pytest.raises(ValueError, match="moe"):
                a.forward(batch_of([(3, 3)], width=4), X, moe)
        with pytest.raises(ValueError, match="moe"):
            BatchedEngine.synthetic(moe, a, 50, 2)
    wide = torch.randn(3, 128, generator=gen(2), device="cuda")
    kept = wide.clone()
    with pytest.raises(ValueError, match="contiguous"):
        a.forward(batch_of([(3, 3)], width=4), wide[:, :64], SimpleNamespace(**fits))
    assert torch.equal(X, before) and torch.equal(wide, kept)
