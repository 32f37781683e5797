"""Attention over the paged 4-bit cache for many query rows of 16-bit types (tcgen05): head counts
whose rows cut tiles anywhere, partial pages and tiles, scales that are not finite, values out of
the ordinary, and the batch's faults."""
from __future__ import annotations

import pytest

from tests import serve_ref as R
from tests.test_gpu_kvq import BF16, F16, F32, Setup, close

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

# several sequences each, so that there are tiles enough for the SMs
MANY = [(140, 300), (257, 257), (1, 90), (33, 900), (0, 40), (200, 201), (16, 2), (64, 1000)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("nh,nkv,hd,page", [(12, 4, 64, 48), (28, 4, 128, 16), (32, 1, 128, 1024), (8, 8, 128, 64),
                                            (160, 5, 64, 16), (10, 2, 128, 128)])
def test_heads_and_pages(nh, nkv, hd, page, dtype):
    s = Setup(MANY * (1 if nkv * nh > 60 else 2), nh, nkv, hd, page, dtype, seed=nh + page)
    close(s.cache.attention(s.batch, s.q), *s.expect(), hd, 1000, dtype)
    s.batch.check()


@pytest.mark.parametrize("n,r", [(128, 128), (256, 256), (32, 2048), (32, 2049), (33, 2111), (512, 513), (480, 3000)])
def test_even_tiles(n, r):
    """Rows and lengths at, before and behind the tiles' edges, alike in all sequences."""
    s = Setup([(n, r)] * 8, 32, 8, 64, 32, BF16, seed=n)
    close(s.cache.attention(s.batch, s.q), *s.expect(), 64, r, BF16)


def test_long_context():
    s = Setup([(300, 20011), (40, 9000), (500, 500)], 32, 4, 128, 64, BF16, seed=3)
    close(s.cache.attention(s.batch, s.q), *s.expect(), 128, 20011, BF16)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("values", [1e-6, 1e-3, 300.0])
def test_value_ranges(dtype, values):
    """V far from 1 (fp16 blocks that are nearly or wholly zero among them), scores far apart and
    all equal, q near its type's smallest and beyond what products in fp16 could hold."""
    s = Setup([(200, 700)] * 6, 16, 2, 128, 64, dtype, values=values, seed=9)
    s.q[0::5] *= 20
    s.q[1::5] = 0
    s.q[2::5] *= 1e-4
    s.q[3] = 3e4
    s.q[3, :, 1::2] = -3e4
    out = s.cache.attention(s.batch, s.q)
    ref = s.expect()
    keep = [t for t in range(s.T) if t != 3]   # one key takes all of row 3: finite is what is asked of it
    got, ref = out[keep], [x[keep] for x in ref]
    if dtype == F16:
        # Below 2^-14 fp16 has steps of 2^-24 whatever the value: rounding is off by up to 2^-25 (3% of
        # the mean output for values of 1e-6, so close()'s mean of relative errors does not apply).
        # The other terms are close()'s.
        want, spread, size, top = ref
        tol = spread * (2 * 136 * 2.0 ** -24 * size + 1432 * 2.0 ** -24 + 4 * 2.0 ** -11 * size + 3 * 2.0 ** -11)
        tol = tol + 700 * 2.0 ** -31 * top
        tol = tol + 1.001 * 2.0 ** -11 * (want.abs() + tol) + 1.001 * 2.0 ** -25
        assert ((got.double() - want).abs() <= tol).all()
    else:
        close(got, *ref, 128, 700, dtype)
    assert torch.isfinite(out[3].float()).all()


def test_garbage_behind_the_last_row():
    s = Setup([(200, 300), (200, 264), (150, 249)] * 3, 16, 2, 128, 64, BF16, seed=2, width=8)
    want = s.cache.attention(s.batch, s.q).clone()
    used = torch.zeros(s.pages.shape[0], s.page, dtype=torch.bool)
    for b, (_, r) in enumerate(s.seqs):
        for i, p in enumerate(s.ids[b]):
            used[p, :max(0, min(s.page, r - i * s.page))] = True
    k, v = s.k.clone(), s.v.clone()
    k[~used.cuda()], v[~used.cuda()] = float("nan"), float("nan")
    s.pages.copy_(R.Cache(1, s.nkv, s.hd, s.page).pages(k, v))
    for b in range(len(s.seqs)):
        s.batch.page_table[b, len(s.ids[b]):] = torch.tensor([10 ** 9, -5, 77777, 2 ** 31 - 1])[:8 - len(s.ids[b])]
    assert torch.equal(s.cache.attention(s.batch, s.q), want)
    s.batch.check()


@pytest.mark.parametrize("which", ["k", "v"])
def test_nan_rows_reach_the_rows_that_see_them(which):
    """A block held as NaN at row 250 of the second sequence: tokens in front of it and other
    sequences are as without it, those that see it are NaN (its 32 dimensions, for V)."""
    s = Setup([(200, 300), (200, 300), (100, 600)] * 3, 16, 2, 128, 64, BF16, seed=5)
    ref = s.expect()
    x = (s.k if which == "k" else s.v).clone()
    x[s.ids[1][250 // 64], 250 % 64, 1, 70] = float("nan")
    s.pages.copy_(R.Cache(1, 2, 128, 64).pages(*((x, s.v) if which == "k" else (s.k, x))))
    out = s.cache.attention(s.batch, s.q)
    first = s.start[1] + 150   # the token of row 250
    hit = torch.zeros(s.T, 16, 128, dtype=torch.bool, device="cuda")
    hit[first:s.start[2], 8:] = True
    if which == "v":
        hit[..., :64], hit[..., 96:] = False, False
    assert torch.isnan(out[hit]).all() and torch.isfinite(out[~hit].float()).all()
    rest = [t for t in range(s.T) if not first <= t < s.start[2]]
    close(out[rest], *[y[rest] for y in ref], 128, 600, BF16)
    s.batch.check()


@pytest.mark.parametrize("nh,nkv,hd", [(16, 4, 64), (12, 4, 128)])
def test_padding_strides_and_in_place(nh, nkv, hd):
    s = Setup([(300, 390), (129, 130)] * 4, nh, nkv, hd, 32, BF16, seed=4, pad=70)
    w, n = nh * hd, s.start[-1]
    want = s.cache.attention(s.batch, s.q)
    wide = torch.full((s.T, w + 260), 5.0, dtype=BF16, device="cuda")
    wide[:, 132:132 + w] = s.q.flatten(1)
    dst = torch.full((s.T, 3, w), 7.0, dtype=BF16, device="cuda")
    s.cache.attention(s.batch, wide[:, 132:132 + w], out=dst[:, 1])
    assert torch.equal(dst[:n, 1], want[:n].flatten(1))
    assert (dst[n:] == 7).all() and (dst[:, 0] == 7).all() and (dst[:, 2] == 7).all()
    s.cache.attention(s.batch, s.q, out=s.q)
    assert torch.equal(s.q[:n], want[:n])


def test_the_last_rows_of_the_last_page_of_memory():
    """q and out that end with their allocation's last row, at every number of rows of an item's
    second tile: what lies behind is neither read into results nor written."""
    for n in (129, 135, 255):
        s = Setup([(n, n)] * 16, 4, 4, 64, 16, BF16, seed=n)
        guard = torch.full((s.T + 300, 256), float("nan"), dtype=BF16, device="cuda")
        guard[:s.T] = s.q.flatten(1)
        out = torch.full((s.T + 300, 256), 9.0, dtype=BF16, device="cuda")
        s.cache.attention(s.batch, guard[:s.T], out=out[:s.T])
        close(out[:s.T].view(s.T, 4, 64), *s.expect(), 64, n, BF16)
        assert (out[s.T:] == 9).all()


def test_faults_are_reported():
    s = Setup([(150, 300), (150, 300), (130, 164)] * 3, 16, 2, 64, 16, BF16, seed=6)
    table = s.batch.page_table.clone()
    ref = s.expect()
    s.batch.page_table[0, 2] = 12345            # rows 32 .. 47 of sequence 0 are left out
    out = s.cache.attention(s.batch, s.q)
    keep = [r for r in range(300) if not 32 <= r < 48]
    one = R.attention(s.q[:150].double(), s.rows(0, s.hk)[keep], s.rows(0, s.hv)[keep], 0.125)
    close(out[:150], *one, 64, 300, BF16)
    close(out[150:], *[x[150:] for x in ref], 64, 300, BF16)
    with pytest.raises(RuntimeError, match="page id"):
        s.batch.check()
    s.batch.page_table.copy_(table)
    s.batch.kv_lens[1] = table.shape[1] * 16 + 50
    s.cache.attention(s.batch, s.q)
    with pytest.raises(RuntimeError, match="length"):
        s.batch.check()
    s.batch.kv_lens[1] = 300
    from tinygiant_b200.paged import PagedBatch
    few = PagedBatch(s.batch.q_start, s.batch.kv_lens, s.batch.page_table, 140)
    dst = torch.full_like(s.q, 3.0)
    s.cache.attention(few, s.q, out=dst)
    with pytest.raises(RuntimeError, match="max_new"):
        few.check()
    for b, (n, _) in enumerate(s.seqs):
        part = dst[s.start[b]:s.start[b + 1]]
        assert (part[140:] == 3).all() and (part[:140] != 3).any(-1).all()


def test_nonsense_starts_do_no_harm():
    s = Setup([(140, 150), (140, 160), (140, 170)] * 2, 32, 4, 64, 16, BF16, seed=8)
    for start in ([5, 0, 2 ** 31 - 1, 12, 700, 3, 800], [-2 ** 31, 2 ** 31 - 1, -1, 3, 0, 840, 0], [9] * 7,
                  [0, 840, 0, 840, 0, 840, 0], [840, 700, 500, 300, 200, 100, 0]):
        s.batch.q_start.copy_(torch.tensor(start, dtype=torch.int32))
        for lens in ([150, 160, 170] * 2, [-2 ** 31, 2 ** 31 - 1, -1] * 2, [0, 1, 16] * 2):
            s.batch.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
            s.cache.attention(s.batch, s.q)
    torch.cuda.synchronize()


def test_equal_results_every_time():
    s = Setup(MANY, 32, 4, 128, 64, F16, seed=11)
    want = s.cache.attention(s.batch, s.q).clone()
    for _ in range(200):
        assert torch.equal(s.cache.attention(s.batch, s.q), want)


def test_streams_and_two_graphs():
    """Captured twice and replayed with other lengths, starts and queries; a third graph of few
    tokens, on the same cache, in between."""
    s = Setup([(200, 700), (200, 290), (200, 1000)], 32, 4, 128, 64, BF16, seed=17)
    want = s.cache.attention(s.batch, s.q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = s.cache.attention(s.batch, s.q, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    outs, graphs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s.cache.attention(s.batch, s.q))
        graphs.append(g)
    q2 = torch.randn_like(s.q)
    for lens, start in (([200, 290, 264], [0, 200, 400, 600]), ([700, 264, 999], [0, 100, 101, 301]),
                        ([0, 233, 500], [0, 0, 200, 400]), ([700, 290, 1000], [600, 600, 600, 600])):
        s.batch.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        s.batch.q_start.copy_(torch.tensor(start, dtype=torch.int32))
        s.q.copy_(q2)
        for g, o in zip(graphs, outs):
            o.fill_(1)
            g.replay()
        ref = s.cache.attention(s.batch, s.q, out=torch.ones_like(s.q))
        torch.cuda.synchronize()
        assert torch.equal(outs[0], ref) and torch.equal(outs[1], ref)
    s.batch.check()


@pytest.mark.parametrize("seqs", [[(32, 3000)] * 40 + [(1000, 1000)], [(256, 256)] * 40, [(40, 64)] * 100])
def test_waits_end_whatever_the_warps_pace(seqs):
    """Thousands of items: a wait that misses its phase ends after a second with NaN."""
    s = Setup(seqs, 32, 4, 128, 64, BF16, seed=13)
    want = s.cache.attention(s.batch, s.q).clone()
    bad = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(1500):
        bad += (s.cache.attention(s.batch, s.q) != want).sum()
    assert torch.isfinite(want.float()).all() and int(bad) == 0


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_queries_that_are_not_finite(dtype):
    """An infinity or NaN in a query row makes its output NaN, whatever the scores' signs; a row
    without a token to attend to is 0 all the same, and its neighbours keep their values."""
    s = Setup([(200, 300), (200, 200), (200, 190), (200, 250)] * 2, 16, 2, 128, 64, dtype, seed=4)
    s.k[..., 3] = s.k[..., 3].abs() + 0.5      # one sign in the dimension of the infinity
    s.hk = R.held(s.k)
    s.pages.copy_(R.Cache(1, s.nkv, s.hd, s.page).pages(s.k, s.v))
    hit = torch.zeros(s.T, dtype=torch.bool)
    for t, x in ((5, -float("inf")), (17, float("inf")), (199, float("nan")), (640, -float("inf")), (403, -float("inf"))):
        s.q[t, :, 3] = x
        hit[t] = True
    got = s.cache.attention(s.batch, s.q)
    none = torch.zeros(s.T, dtype=torch.bool)   # tokens in front of their sequence's first row
    for b, (n, r) in enumerate(s.seqs):
        none[s.start[b]:s.start[b] + max(0, n - r)] = True
    assert hit[none].any() and (got[none.cuda()] == 0).all()
    assert torch.isnan(got[(hit & ~none).cuda()]).all()
    rest = ~(hit | none).cuda()
    close(got[rest], *[x[rest] for x in s.expect()], 128, 300, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("seqs,nh,nkv,hd", [([(1, 700), (3, 50), (1, 2900)], 8, 2, 128), ([(40, 300), (7, 40)], 16, 2, 64),
                                            ([(200, 300), (150, 700)] * 4, 16, 2, 128)])
def test_scores_beyond_the_exponent(seqs, nh, nkv, hd, dtype):
    """Queries so large that a softmax is one key's: scores of 1e4 to 1e13, where neighbouring fp32
    numbers are up to 2^20 apart.  The value of the largest score comes out."""
    s = Setup(seqs, nh, nkv, hd, 64, dtype, seed=21)
    g = torch.Generator().manual_seed(3)
    low, high = (3.0, 4.0) if dtype == F16 else (4.0, 12.0)
    size = 10.0 ** (low + (high - low) * torch.rand(s.T, 1, 1, generator=g)).cuda()
    s.q = (s.q.double() * size).clamp(-6e4 if dtype == F16 else -1e14, 6e4 if dtype == F16 else 1e14).to(dtype)
    out = s.cache.attention(s.batch, s.q).double()
    assert torch.isfinite(out).all()
    seen = 0
    for b, (n, r) in enumerate(s.seqs):
        q, k, v = s.q[s.start[b]:s.start[b + 1]].double(), s.rows(b, s.hk), s.rows(b, s.hv)
        sees = torch.arange(r, device="cuda")[None] <= (r - n + torch.arange(n, device="cuda"))[:, None]
        for h in range(nh):
            j = h // (nh // nkv)
            score = (q[:, h] @ k[:, j].T * hd ** -0.5).masked_fill(~sees, -float("inf"))
            size = (q[:, h].abs() @ k[:, j].abs().T * hd ** -0.5).amax(1)
            best = torch.topk(score, 2, 1)
            # 11 bits of q and of k, each off by 2^-12 of a product: what lies further apart than both scores'
            # errors, and 60 besides, decides alone
            clear = best.values[:, 0] - best.values[:, 1] > 2 * 2 * 2.0 ** -12 * size + 60
            want = v[best.indices[:, 0], j][clear]
            got = out[s.start[b]:s.start[b + 1], h][clear]
            # 11 bits each of p (which is a power of two at the reference only) and of v or p * d, 2^-11 at
            # most; the roundings of 1 / l and of the products; the type's
            tol = (2 * 2.0 ** -11 if dtype != F32 else 0) + 2.0 ** -20 + 1.001 * R.EPS[dtype]
            assert ((got - want).abs() <= tol * want.abs() + 2.0 ** -22).all(), (b, h)
            seen += int(clear.sum())
    assert seen > s.T * nh // 4


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_large_values_behind_the_last_row(dtype):
    """Finite values with the largest scales in rows that a sequence does not hold change no bit."""
    s = Setup([(200, 300), (200, 264), (150, 249)] * 3, 16, 2, 128, 64, dtype, seed=2, values=0.05)
    want = s.cache.attention(s.batch, s.q)
    used = torch.zeros(s.pages.shape[0], s.page, dtype=torch.bool)
    for b, (_, r) in enumerate(s.seqs):
        for i, p in enumerate(s.ids[b]):
            used[p, :max(0, min(s.page, r - i * s.page))] = True
    k, v = s.k.clone(), s.v.clone()
    k[~used.cuda()], v[~used.cuda()] = 5e5, -5e5
    s.pages.copy_(R.Cache(1, s.nkv, s.hd, s.page).pages(k, v))
    assert torch.equal(s.cache.attention(s.batch, s.q), want)
