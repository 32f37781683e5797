"""The paged 4-bit key/value cache on the GPU against plain 64-bit forms (tests/serve_ref.py):
appending (codes and scales byte for byte, rotated q), reading back, and attention over ragged
batches, with the lengths, pages and strides where it can go wrong."""
from __future__ import annotations

import math

import pytest

from tests import serve_ref as R

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


class Setup:
    """Sequences (new tokens, rows cached with them) over a cache of shuffled pages filled with
    random rows, as the operators and the plain form see it."""

    def __init__(self, seqs, nh, nkv, hd, page, dtype, seed=0, pad=0, extra_pages=2, width=None, values=1.0):
        from tinygiant_b200.paged import PagedBatch, PagedKV4
        g = gen(seed)
        self.seqs, self.nh, self.nkv, self.hd, self.page, self.dtype, self.g = seqs, nh, nkv, hd, page, dtype, g
        need = [-(-max(r, 0) // page) for _, r in seqs]
        n_pages = sum(need) + extra_pages
        ids = torch.randperm(n_pages, generator=g, device="cuda").tolist()
        width = width or max(max(need), 1)
        table = torch.full((len(seqs), width), -1, dtype=torch.int32)
        self.ids = []
        for b, n in enumerate(need):
            self.ids.append(ids[:n])
            table[b, :min(n, width)] = torch.tensor(ids[:min(n, width)], dtype=torch.int32)
            ids = ids[n:]
        self.k = torch.randn(n_pages, page, nkv, hd, generator=g, device="cuda", dtype=torch.float64)
        self.v = torch.randn(n_pages, page, nkv, hd, generator=g, device="cuda", dtype=torch.float64) * values
        self.pages = R.Cache(1, nkv, hd, page).pages(self.k, self.v)
        self.hk, self.hv = R.held(self.k), R.held(self.v)
        start = [0]
        for n, _ in seqs:
            start.append(start[-1] + n)
        self.start, self.T = start, start[-1] + pad
        self.q = (torch.randn(self.T, nh, hd, generator=g, device="cuda") * 1.5).to(dtype)
        self.cache = PagedKV4(nkv, hd, page, pages=self.pages)
        self.batch = PagedBatch(torch.tensor(start, dtype=torch.int32).cuda(),
                                torch.tensor([r for _, r in seqs], dtype=torch.int32).cuda(), table.cuda(),
                                max(max(n for n, _ in seqs), 1))

    def rows(self, b, held):
        n = self.seqs[b][1]
        x = held[self.ids[b]].flatten(0, 1)
        return x[:max(n, 0)]

    def expect(self, scale=None):
        scale = scale or self.hd ** -0.5
        parts = []
        for b, (n, r) in enumerate(self.seqs):
            q = self.q[self.start[b]:self.start[b + 1]].double()
            parts.append(R.attention(q, self.rows(b, self.hk), self.rows(b, self.hv), scale))
        return [torch.cat(x) for x in zip(*parts)]


def close(got, ref, spread, size, top, hd, rows, dtype):
    """fp32 path: a score sums hd products (each rounding 2^-24 of sum |q||k| = size) and is
    subtracted and scaled in fp32 (4 more of |s| <= size); p carries twice that and exp's 2 units;
    the sum over the rows and its norm `rows` roundings of sum p|v| each.  16-bit types: q, k, v
    and p may be held in 11 bits (2^-11 each at most) in front of the fp32 sums.  A probability is
    held in fp16 pieces, 2^6 at the largest one, whose last bit is 2^-24: each is off by up to
    2^-25 / 2^6 of the largest besides, whatever its own size, so an output by rows * 2^-31 * the
    largest |v| (seen where a peaked row's value is 0 and what is left is smaller still).  Then one
    rounding to the type."""
    u = 2.0 ** -24
    ds = (hd + 8) * u * size
    tol = spread * (2 * ds + (2 * rows + 32) * u)
    if dtype != F32:
        tol = tol + spread * (4 * 2.0 ** -11 * size + 3 * 2.0 ** -11)
    tol = tol + rows * 2.0 ** -31 * top
    tol = tol + 1.001 * R.EPS[dtype] * (ref.abs() + tol) + 1e-30
    d = (got.double() - ref).abs()
    assert torch.isfinite(got.float()).all()
    worst = (d / tol).max().item() if d.numel() else 0.0
    assert worst <= 1.0, worst
    # in the mean roundings add like their roots
    if ref.numel() and ref.norm() > 0:
        rel = ((got.double() - ref).norm() / ref.norm()).item()
        lim = 4 * u * math.sqrt(hd + rows) + (0 if dtype == F32 else 0.75 * R.EPS[dtype] + 2.0 ** -11)
        assert rel <= lim, (rel, lim)


DECODE = [(1, 1), (1, 15), (1, 16), (1, 17), (1, 63), (1, 64), (1, 65), (1, 0), (0, 30), (1, 333)]
HEADS = [(8, 1, 128, 64), (32, 4, 128, 64), (4, 4, 64, 16), (6, 2, 96, 32), (10, 2, 32, 128), (16, 1, 256, 16),
         (14, 2, 160, 48), (32, 1, 64, 64), (5, 1, 192, 64), (3, 1, 224, 1024)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("nh,nkv,hd,page", HEADS)
def test_decode_attention(nh, nkv, hd, page, dtype):
    s = Setup(DECODE, nh, nkv, hd, page, dtype, seed=nh * hd)
    out = s.cache.attention(s.batch, s.q)
    close(out, *s.expect(), hd, 333, dtype)
    assert (out[7] == 0).all()   # no rows to attend to
    s.batch.check()


CHUNKS = [(40, 40), (1, 70), (17, 200), (130, 131), (0, 5), (64, 64), (3, 2), (257, 300)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("nh,nkv,hd,page", [(8, 1, 128, 64), (32, 4, 128, 64), (4, 4, 64, 16), (6, 2, 96, 32),
                                            (16, 1, 256, 16), (10, 2, 32, 128), (32, 1, 160, 48)])
def test_chunk_attention(nh, nkv, hd, page, dtype):
    """Several new tokens per sequence, each seeing the rows up to its own; the first tokens of a
    sequence of fewer rows than new tokens see none."""
    s = Setup(CHUNKS, nh, nkv, hd, page, dtype, seed=hd + nh)
    out = s.cache.attention(s.batch, s.q)
    close(out, *s.expect(), hd, 300, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new", [1, 5])
def test_long_attention(dtype, new):
    s = Setup([(new, 20011), (new, 700)], 16, 2, 128, 64, dtype, seed=3)
    out = s.cache.attention(s.batch, s.q)
    close(out, *s.expect(), 128, 20011, dtype)


def test_many_sequences():
    """More sequences than a search step's 32 probes, empty ones among them."""
    seqs = [((b * 7) % 3, (b * 37) % 90 + 3) for b in range(1200)]
    s = Setup(seqs, 2, 1, 64, 16, F32, seed=5)
    close(s.cache.attention(s.batch, s.q), *s.expect(), 64, 93, F32)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("values", [1e-3, 300.0])
def test_value_ranges(dtype, values):
    """Values far from 1, scores far apart (a peaked softmax) and equal ones."""
    s = Setup([(1, 500), (2, 77)], 8, 1, 128, 64, dtype, values=values, seed=9)
    s.q[0] *= 20
    s.q[1] = 0
    close(s.cache.attention(s.batch, s.q), *s.expect(), 128, 500, dtype)


def test_equal_results_twice():
    s = Setup([(1, 3000)] * 5 + [(9, 900)], 8, 2, 128, 64, F32, seed=11)
    a, b = s.cache.attention(s.batch, s.q), s.cache.attention(s.batch, s.q)
    assert torch.equal(a, b)


@pytest.mark.parametrize("new", [1, 33])
def test_garbage_behind_the_last_row(new):
    """NaN scales and any codes in rows behind a sequence's last one, in pages it does not hold,
    and page ids outside the cache behind its last page change nothing."""
    s = Setup([(new, 100), (new, 64), (new, 49)], 8, 2, 128, 64, F32, seed=2, width=6)
    want = s.cache.attention(s.batch, s.q).clone()
    used = torch.zeros(s.pages.shape[0], s.page, dtype=torch.bool)
    for b, (_, r) in enumerate(s.seqs):
        for i, p in enumerate(s.ids[b]):
            used[p, :max(0, min(s.page, r - i * s.page))] = True
    k, v = s.k.clone(), s.v.clone()
    k[~used.cuda()], v[~used.cuda()] = float("nan"), float("nan")
    s.pages.copy_(R.Cache(1, s.nkv, s.hd, s.page).pages(k, v))
    for b in range(3):
        s.batch.page_table[b, len(s.ids[b]):] = torch.tensor([10 ** 9, -5, 77777, 2 ** 31 - 1, -1])[:6 - len(s.ids[b])]
    got = s.cache.attention(s.batch, s.q)
    assert torch.equal(got, want)
    s.batch.check()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new", [1, 20])
@pytest.mark.parametrize("nh,nkv,hd,page", [(8, 2, 128, 64), (6, 2, 96, 32), (32, 1, 64, 16)])
def test_large_values_behind_the_last_row(nh, nkv, hd, page, new, dtype):
    """What a page held before: finite values with the largest scales, behind a sequence's last row
    and in rows that it does not hold, change no bit of the outputs."""
    s = Setup([(new, 100), (new, 64), (new, 49), (new, 333)], nh, nkv, hd, page, dtype, seed=2, values=0.05)
    want = s.cache.attention(s.batch, s.q)
    used = torch.zeros(s.pages.shape[0], s.page, dtype=torch.bool)
    for b, (_, r) in enumerate(s.seqs):
        for i, p in enumerate(s.ids[b]):
            used[p, :max(0, min(s.page, r - i * s.page))] = True
    k, v = s.k.clone(), s.v.clone()
    k[~used.cuda()], v[~used.cuda()] = 5e5, -5e5   # scales of 62500
    s.pages.copy_(R.Cache(1, s.nkv, s.hd, s.page).pages(k, v))
    assert torch.equal(s.cache.attention(s.batch, s.q), want)
    close(want, *s.expect(), hd, 333, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_values_that_no_query_of_a_tile_sees(dtype):
    """Rows of a sequence behind all the queries of a tile are nothing to it, however large."""
    s = Setup([(64, 64), (64, 90)], 8, 2, 128, 64, dtype, seed=3, values=0.05)
    want = s.cache.attention(s.batch, s.q)
    v = s.v.clone()
    for b, (n, r) in enumerate(s.seqs):
        for row in range(r - 32, r):   # the second half of the new tokens
            v[s.ids[b][row // s.page], row % s.page] = -5e5
    s.pages.copy_(R.Cache(1, s.nkv, s.hd, s.page).pages(s.k, v))
    got = s.cache.attention(s.batch, s.q)
    for b in range(2):
        first = s.start[b]
        assert torch.equal(got[first:first + 32], want[first:first + 32])


def test_nan_rows_attended_give_nan():
    s = Setup([(1, 40)], 2, 1, 64, 16, F32)
    v = s.v.clone()
    v[s.ids[0][0], 3, 0, 40] = float("nan")
    s.pages.copy_(R.Cache(1, 1, 64, 16).pages(s.k, v))
    out = s.cache.attention(s.batch, s.q)
    assert torch.isnan(out[..., 32:]).all() and torch.isfinite(out[..., :32]).all()


@pytest.mark.parametrize("new", [1, 20])
def test_padding_strides_and_in_place(new):
    """Rows behind the last sequence stay as they were; q and out strided views; out over q."""
    seqs = [(new, 90), (new, 30)]
    s = Setup(seqs, 8, 2, 64, 32, BF16, seed=4, pad=7)
    want = s.cache.attention(s.batch, s.q)
    wide = torch.full((s.T, 8 * 64 + 256), 5.0, dtype=BF16, device="cuda")
    wide[:, 128:128 + 512] = s.q.flatten(1)
    dst = torch.full((s.T, 3, 512), 7.0, dtype=BF16, device="cuda")
    s.cache.attention(s.batch, wide[:, 128:640], out=dst[:, 1])
    n = 2 * new
    assert torch.equal(dst[:n, 1], want[:n].flatten(1))
    assert (dst[n:] == 7).all() and (dst[:, 0] == 7).all() and (dst[:, 2] == 7).all()
    s.cache.attention(s.batch, s.q, out=s.q)
    assert torch.equal(s.q[:n], want[:n])


def test_bad_pages_lengths_and_counts_are_reported():
    s = Setup([(1, 100), (1, 100), (3, 64)], 4, 2, 64, 16, F32, seed=6)
    table = s.batch.page_table.clone()
    s.batch.page_table[0, 2] = 12345            # rows 32 .. 47 of sequence 0 are left out
    out = s.cache.attention(s.batch, s.q)
    keep = [r for r in range(100) if not 32 <= r < 48]
    ref = R.attention(s.q[:1].double(), s.rows(0, s.hk)[keep], s.rows(0, s.hv)[keep], 0.125)
    close(out[:1], *ref, 64, 100, F32)
    with pytest.raises(RuntimeError, match="page id"):
        s.batch.check()
    s.batch.check()                              # forgotten
    s.batch.page_table.copy_(table)
    s.batch.kv_lens[1] = 7 * 16 + 50             # the table has 7 pages
    s.cache.attention(s.batch, s.q)
    with pytest.raises(RuntimeError, match="length"):
        s.batch.check()
    s.batch.kv_lens[1] = 100
    from tinygiant_b200.paged import PagedBatch
    few = PagedBatch(s.batch.q_start, s.batch.kv_lens, s.batch.page_table, 2)
    dst = torch.full_like(s.q, 3.0)
    s.cache.attention(few, s.q, out=dst)
    with pytest.raises(RuntimeError, match="max_new"):
        few.check()
    assert (dst[4] == 3).all() and (dst[:4] != 3).any(-1).all()


def test_nonsense_starts_do_no_harm():
    s = Setup([(4, 50), (4, 60), (4, 70)], 4, 2, 64, 16, F32, seed=8)
    for start in ([5, 0, 2 ** 31 - 1, 12], [-2 ** 31, 2 ** 31 - 1, -1, 3], [9, 9, 9, 9], [0, 2 ** 31 - 1, 5, -7]):
        s.batch.q_start.copy_(torch.tensor(start, dtype=torch.int32))
        for lens in ([50, 60, 70], [-2 ** 31, 2 ** 31 - 1, -1]):
            s.batch.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
            s.cache.attention(s.batch, s.q)
            s.cache.read(s.batch, s.T)
    torch.cuda.synchronize()


# ---------------------------------------------------------------- append and read


def append_case(s, n_pos=4096, norm=True, rotate=True):
    g, hd = s.g, s.hd
    qkv = torch.randn(s.T, (s.nh + 2 * s.nkv) * hd, generator=g, device="cuda").to(s.dtype)
    q, k, v = qkv.split([s.nh * hd, s.nkv * hd, s.nkv * hd], 1)
    ang = torch.arange(n_pos, device="cuda", dtype=torch.float64)[:, None] * 1e6 ** (
        -torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    cos, sin = (ang.cos().float(), ang.sin().float()) if rotate else (None, None)
    qn, kn = (1 + 0.1 * torch.randn(2, hd, generator=g, device="cuda")).unbind() if norm else (None, None)
    return q, k, v, cos, sin, qn, kn


def append_expect(s, q, k, v, cos, sin, qn, kn, eps, pages, positions=None):
    """q rotated, and the cache's bytes after the append."""
    hk, hv = s.k.clone(), s.v.clone()
    rq = torch.zeros(s.T, s.nh, s.hd, dtype=torch.float64, device="cuda")
    for b, (n, r) in enumerate(s.seqs):
        for i in range(n):
            t, row = s.start[b] + i, r - n + i
            if row < 0:
                continue
            pos = row if positions is None else int(positions[t])
            c, sn = (None, None) if cos is None else (cos[pos:pos + 1], sin[pos:pos + 1])
            rq[t] = R.norm_rope(q[t].view(1, s.nh, s.hd).double(), qn, eps, c, sn)[0]
            page = s.ids[b][row // s.page]
            hk[page, row % s.page] = R.norm_rope(k[t].view(1, s.nkv, s.hd).double(), kn, eps, c, sn)[0]
            hv[page, row % s.page] = v[t].view(s.nkv, s.hd).double()
    return rq, R.Cache(1, s.nkv, s.hd, s.page).pages(hk, hv), hk, hv


APPENDS = [(1, 1), (5, 5), (0, 12), (1, 65), (17, 40), (3, 2), (16, 64)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("nh,nkv,hd,page", HEADS)
def test_append(nh, nkv, hd, page, dtype):
    s = Setup(APPENDS, nh, nkv, hd, page, dtype, seed=hd, pad=2)
    args = append_case(s)
    rq, pages, hk, hv = append_expect(s, *args, 1e-6, s.pages)
    q_out = torch.full((s.T, nh, hd), 9.0, dtype=dtype, device="cuda")
    s.cache.append(s.batch, *args[:5], *args[5:], eps=1e-6, q_out=q_out)
    assert torch.equal(s.pages, pages)           # every byte, the untouched rows' too
    n = s.start[-1]
    assert (q_out[n:] == 9).all()
    # fp32: the sum of hd squares, its root and quotient, two products, the rotation's three
    # roundings, each relative to the rotated pair's size; then the type's rounding
    pair = rq.norm(dim=-1, keepdim=True)
    tol = (hd / 2 + 10) * 2.0 ** -24 * pair + R.EPS[dtype] * 1.001 * rq.abs() + (2.0 ** -25 if dtype == F16 else 0)
    assert ((q_out[:n].double() - rq[:n]).abs() <= tol[:n]).all()
    kv = s.cache.read(s.batch, s.T)
    for got, held in zip(kv, (R.held(hk), R.held(hv))):
        for b, (m, r) in enumerate(s.seqs):
            for i in range(m):
                row = r - m + i
                want = torch.zeros_like(got[0]).double() if row < 0 else held[s.ids[b][row // page], row % page]
                assert torch.equal(got[s.start[b] + i].double(), want)
    with pytest.raises(RuntimeError, match="length"):
        s.batch.check()                          # the sequence of two rows and three tokens


@pytest.mark.parametrize("norm,rotate", [(False, True), (True, False), (False, False)])
def test_append_without_norm_or_rotation(norm, rotate):
    s = Setup(APPENDS, 6, 2, 128, 32, F32, seed=1)
    args = append_case(s, norm=norm, rotate=rotate)
    rq, pages, _, _ = append_expect(s, *args, 1e-6, s.pages)
    got = s.cache.append(s.batch, *args)
    assert torch.equal(s.pages, pages)
    assert (got.double() - rq).abs().max() <= 100 * 2.0 ** -24 * rq.norm(dim=-1).max()


def test_append_positions_keys_only_and_in_place():
    s = Setup([(4, 9), (2, 20)], 4, 2, 64, 16, BF16, seed=13)
    args = append_case(s, n_pos=64)
    positions = torch.tensor([7, 0, 63, 5, 1, 33], dtype=torch.int32, device="cuda")
    rq, pages, _, _ = append_expect(s, *args, 1e-6, s.pages, positions)
    q = args[0].contiguous().view(s.T, 4, 64)
    s.cache.append(s.batch, q, *args[1:], positions=positions, q_out=q)
    assert torch.equal(s.pages, pages)
    assert ((q.double() - rq).abs() <= R.EPS[BF16] * 1.001 * rq.abs() + 50 * 2.0 ** -24 * rq.norm(dim=-1, keepdim=True)).all()
    s.pages.zero_()
    assert s.cache.append(s.batch, None, *args[1:], positions=positions) is None
    before = R.Cache(1, 2, 64, 16)
    again = s.pages.clone()
    s.pages.copy_(pages)
    s.cache.append(s.batch, None, *args[1:], positions=positions)
    assert torch.equal(s.pages, pages) and again.any() and before.hd == 64
    s.batch.check()


def test_append_bad_pages_and_positions_write_nothing():
    s = Setup([(2, 10), (2, 10)], 2, 1, 64, 16, F32, seed=14)
    args = append_case(s, n_pos=10)
    before = s.pages.clone()
    s.batch.page_table[:] = 999
    q = s.cache.append(s.batch, *args)
    assert torch.equal(s.pages, before) and (q == 0).all()
    with pytest.raises(RuntimeError, match="page id"):
        s.batch.check()
    for b in range(2):
        s.batch.page_table[b, 0] = s.ids[b][0]
    positions = torch.tensor([10, -1, 2 ** 31 - 1, 9], dtype=torch.int32, device="cuda")
    q = s.cache.append(s.batch, *args, positions=positions)
    with pytest.raises(RuntimeError, match="position"):
        s.batch.check()
    assert (q[:3] == 0).all() and (q[3] != 0).any()


def test_append_ties_zeros_and_values_out_of_range():
    """Blocks of equal magnitudes of both signs (the first counts), of zeros, with a value that is
    not finite or has no fp16 scale (held as NaN), and subnormal scales."""
    s = Setup([(12, 12)], 1, 1, 64, 16, F32, seed=15)
    v = torch.randn(12, 64, generator=s.g, device="cuda")
    v[0, :32] = 0
    v[1, 3], v[1, 9] = 4.0, -4.0
    v[2, 3], v[2, 9] = -4.0, 4.0
    v[3, 40] = float("inf")
    v[4, 10] = float("nan")
    v[5, 63] = 8 * 65536.0
    v[6] *= 1e-6
    v[7, :32] = torch.arange(-16, 16, device="cuda") / 4.0   # ratios on the borders
    v[8, :32] = 1.0
    v[9] *= 1e-30
    v[10, 32:] = -1.0
    v[11, 0] = -0.0
    k = v.flip(0).contiguous()
    pages = append_expect(s, v, k, v, None, None, None, None, 0.0, s.pages)[1]
    s.cache.append(s.batch, None, k, v)
    assert torch.equal(s.pages, pages)


@pytest.mark.parametrize("nh,nkv,hd,page", HEADS)
@pytest.mark.parametrize("off", [1, 2, 3])
def test_append_tables_at_any_element(nh, nkv, hd, page, off):
    """Norm weights and angles as views into packed vectors, wherever they begin."""
    s = Setup(APPENDS, nh, nkv, hd, page, BF16, seed=hd)
    args = append_case(s, n_pos=70)
    want = s.cache.append(s.batch, *args)
    pages = s.pages.clone()

    def packed(x):
        flat = torch.full((x.numel() + 8,), 7.0, device="cuda")
        view = flat[off:off + x.numel()].view(x.shape)
        view.copy_(x)
        assert view.data_ptr() % 16 == 4 * off
        return view

    s.pages.copy_(R.Cache(1, nkv, hd, page).pages(s.k, s.v))
    got = s.cache.append(s.batch, *args[:3], *map(packed, args[3:]))
    assert torch.equal(got, want) and torch.equal(s.pages, pages)

@pytest.mark.parametrize("hd,gap", [(64, 4), (128, 8), (256, 16), (32, 2), (96, 6)])
def test_append_keys_that_are_equal_in_32_bits_only(hd, gap):
    """Two rotated keys of one block that 32 bits round to the same magnitude: the larger of the
    exact ones gives the block its scale, whichever comes first."""
    s = Setup([(8, 8)], 1, 1, hd, 16, F32, seed=1)
    g, h = s.g, hd // 2
    cos, sin = torch.full((8, h), 0.50000006, device="cuda"), torch.zeros(8, h, device="cuda")
    lo, hi = 2 - 2.0 ** -22, 2 - 2.0 ** -23      # their products with the cosine: below and above 1
    k, v = torch.zeros(8, hd, device="cuda"), torch.randn(8, hd, generator=g, device="cuda")
    k[:, 32::32] = 2.0                           # blocks without a doubt
    for t, (a, b, at) in enumerate([(lo, -hi, 0), (hi, -lo, 0), (-lo, hi, 0), (lo, hi, 0), (-hi, lo, 0), (lo, -hi, 1),
                                    (-lo, hi, h % 32), (hi, -hi, 1)]):
        k[t, at], k[t, at + gap] = a, b
    pages = append_expect(s, v, k, v, cos, sin, None, None, 0.0, s.pages)[1]
    s.cache.append(s.batch, None, k, v, cos, sin)
    assert torch.equal(s.pages, pages)


@pytest.mark.parametrize("size", [1.0, 1.37, 40.0, 1000.0])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_append_keys_that_the_rotation_cancels(hd, size):
    """Blocks that come out of the rotation far smaller than they went in, whose roundings are those
    of the large products; tables with an attention factor folded in."""
    n, h = 512, hd // 2
    s = Setup([(n, n)], 1, 1, hd, 64, F32, seed=hd)
    turn = torch.rand(n, h, generator=s.g, device="cuda", dtype=torch.float64) * 1.2 + 0.2
    cos, sin = (size * turn.cos()).float(), (size * turn.sin()).float()
    depth = 10.0 ** (-6 * torch.rand(n, 1, generator=s.g, device="cuda", dtype=torch.float64) - 0.5)
    k = torch.cat((turn.sin() + depth * torch.randn(n, h, generator=s.g, device="cuda", dtype=torch.float64), turn.cos()),
                  1).float()
    v = torch.randn(n, hd, generator=s.g, device="cuda")
    pages = append_expect(s, v, k, v, cos, sin, None, None, 0.0, s.pages)[1]
    s.cache.append(s.batch, None, k, v, cos, sin)
    assert torch.equal(s.pages, pages)


def test_append_keys_whose_squares_vanish():
    """eps 0 and keys so small that fp32 squares are subnormal or 0: the norm is still the exact one's."""
    s = Setup([(96, 96)], 2, 2, 128, 64, F32, seed=5)
    q, k, v, cos, sin, qn, kn = append_case(s)
    k = k * 10.0 ** torch.linspace(-17, -37, 96, device="cuda")[:, None]
    pages = append_expect(s, q, k, v, cos, sin, qn, kn, 0.0, s.pages)[1]
    s.cache.append(s.batch, None, k, v, cos, sin, qn, kn, eps=0.0)
    assert torch.equal(s.pages, pages)


def test_offsets_beyond_32_bits():
    """Pages whose bytes lie behind the first 4 GB of the cache."""
    from tinygiant_b200.paged import PagedBatch, PagedKV4
    nkv, hd, page = 8, 256, 1024
    per = nkv * 64 * 18 * hd
    n = (2 ** 32 + 2 ** 31) // per + 2
    cache = PagedKV4(nkv, hd, page, pages=torch.zeros(n, per, dtype=torch.uint8, device="cuda"))
    start = torch.tensor([0, 40], dtype=torch.int32).cuda()
    batch = PagedBatch(start, torch.tensor([1060], dtype=torch.int32).cuda(),
                       torch.tensor([[n - 1, n - 2]], dtype=torch.int32).cuda(), 40)
    g = gen(16)
    k, v, q = (torch.randn(1060, h * hd, generator=g, device="cuda") for h in (nkv, nkv, 16))
    whole = PagedBatch(torch.tensor([0, 1060], dtype=torch.int32).cuda(), batch.kv_lens, batch.page_table, 1060)
    cache.append(whole, None, k, v)
    hk, hv = R.held(k.view(-1, nkv, hd).double()), R.held(v.view(-1, nkv, hd).double())
    got = cache.read(whole, 1060)
    assert torch.equal(got[0].double(), hk) and torch.equal(got[1].double(), hv)
    assert not cache.pages[:n - 2].any()
    out = cache.attention(batch, q[:40])
    close(out, *R.attention(q[:40].view(40, 16, hd).double(), hk, hv, hd ** -0.5), hd, 1060, F32)


# ---------------------------------------------------------------- streams and graphs


@pytest.mark.parametrize("new", [1, 24])
def test_streams_and_two_graphs(new):
    """The same call on another stream, and captured twice into graphs that replay with other
    lengths, pages and queries, one after the other."""
    s = Setup([(new, 200), (new, 90), (new, 1000)], 8, 2, 128, 64, F32, seed=17)
    want = s.cache.attention(s.batch, s.q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = s.cache.attention(s.batch, s.q, stream=side)
    got2 = s.cache.attention(s.batch, s.q, stream=side.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(got2, want)
    outs, graphs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s.cache.attention(s.batch, s.q))
        graphs.append(g)
    q2 = torch.randn_like(s.q)
    for lens in ([new, 90, 64], [200, 64, 999], [150, 33, 500]):
        s.batch.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        s.q.copy_(q2)
        for g, o in zip(graphs, outs):
            o.fill_(1)
            g.replay()
        ref = s.cache.attention(s.batch, s.q)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], ref) and torch.equal(outs[1], ref)
    s.batch.check()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("new", [1, 12])
def test_queries_that_are_not_finite(new, dtype):
    """As for prompts: NaN out, 0 where there is no token to attend to, nothing at the neighbours."""
    s = Setup([(new, 40 + new), (new, 300), (new, 0), (new, 90)], 8, 2, 64, 16, dtype, seed=12)
    s.k[..., 3] = s.k[..., 3].abs() + 0.5
    s.hk = R.held(s.k)
    s.pages.copy_(R.Cache(1, 2, 64, 16).pages(s.k, s.v))
    s.q[0, :, 3] = -float("inf")
    s.q[new, :, 3] = float("nan")
    s.q[2 * new, :, 3] = -float("inf")
    got = s.cache.attention(s.batch, s.q)
    assert torch.isnan(got[0]).all() and torch.isnan(got[new]).all() and (got[2 * new:3 * new] == 0).all()
    rest = [t for t in range(s.T) if t not in (0, new) and not 2 * new <= t < 3 * new]
    close(got[rest], *[x[rest] for x in s.expect()], 64, 300, dtype)


@pytest.mark.parametrize("start", [[0, 2, 9], [0, 5, 4], [-1, 2, 4], [0, 2, 2 ** 31 - 1]])
def test_starts_that_do_not_fit_are_reported(start):
    """A sequence whose new tokens are not the step's rows is left out, and check() says so."""
    s = Setup([(2, 50), (2, 60)], 4, 2, 64, 16, F32, seed=8)
    want = s.cache.attention(s.batch, s.q)
    s.batch.check()
    s.batch.q_start.copy_(torch.tensor(start, dtype=torch.int32))
    dst = torch.full_like(s.q, 3.0)
    s.cache.attention(s.batch, s.q, out=dst)
    if start[:2] == [0, 2]:
        assert torch.equal(dst[:2], want[:2]) and (dst[2:] == 3).all()
    with pytest.raises(RuntimeError, match="starts that go back"):
        s.batch.check()


def test_check_waits_for_every_stream():
    """A fault met on another stream than the current one, behind work that takes a while."""
    s = Setup([(1, 100), (1, 100)], 4, 2, 64, 16, F32, seed=6)
    a = torch.randn(4096, 4096, device="cuda")
    side = torch.cuda.Stream()
    s.cache.attention(s.batch, s.q, stream=side)   # everything is loaded
    a = a @ a * 1e-3
    s.batch.check()
    s.batch.page_table[0, 2] = 12345
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(40):
            a = a @ a * 1e-3
    s.cache.attention(s.batch, s.q, stream=side)
    with pytest.raises(RuntimeError, match="page id"):
        s.batch.check()
    s.batch.check()


@pytest.mark.parametrize("hd", [64, 96])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_append_leaves_q_alone_without_norm_or_rotation(hd, dtype):
    """Neither norm nor rope: q comes back as it is, its infinities and NaN in their places."""
    s = Setup([(3, 9), (2, 20)], 4, 2, hd, 16, dtype, seed=13)
    q, k, v = append_case(s)[:3]
    q = q.clone()
    q[0, 5], q[1, hd // 2 + 1], q[4, 3 * hd + 2] = float("inf"), float("nan"), -float("inf")
    got = s.cache.append(s.batch, q, k, v).flatten(1)
    assert torch.equal(torch.isnan(got), torch.isnan(q))
    assert torch.equal(torch.nan_to_num(got, 7.0), torch.nan_to_num(q, 7.0))


def test_streams_of_another_device_are_refused():
    from tinygiant_b200.paged import on_stream
    side = torch.cuda.Stream(device=0)
    with on_stream(side, torch.device("cuda", 0)), on_stream(side.cuda_stream, torch.device("cuda", 0)):
        assert torch.cuda.current_stream(0).cuda_stream == side.cuda_stream
    with pytest.raises(ValueError, match="stream"):
        on_stream(side, torch.device("cuda", 1))
