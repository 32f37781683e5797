"""Argument checks of the batched serving operators (no GPU calls), and the plain forms'
own consistency."""
import ctypes

import numpy as np
import pytest

from tinygiant_b200 import _lib as L

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def clib():
    return L.load_tinygiant_lib()


def test_sizes(clib):
    assert clib.tgx_kvq_page_bytes(4, 128, 64) == 4 * 4 * 18 * 128
    assert clib.tgx_kvq_page_bytes(1, 32, 16) == 18 * 32
    for bad in ((0, 128, 64), (4, 100, 64), (4, 288, 64), (4, 0, 64), (4, 128, 24), (4, 128, 0), (4, 128, 1040)):
        assert clib.tgx_kvq_page_bytes(*bad) == 0, bad
    assert clib.tgx_i8_row_bytes(1) == 16 and clib.tgx_i8_row_bytes(2048) == 2048
    assert clib.tgx_i8_row_bytes(0) == 0 and clib.tgx_i8_row_bytes(131073) == 0
    assert clib.tgx_i8_matmul_scratch_bytes(3, 10, 33) >= 3 * 48 + 12
    assert clib.tgx_i8_matmul_scratch_bytes(3, 0, 33) == 0


def refuse(clib, rc, text):
    assert rc == L.TG_EINVAL
    assert text in clib.tg_last_error().decode()


def test_cache_refusals(clib):
    buf = np.zeros(4096, np.uint8)
    p = (buf.ctypes.data + 255) // 256 * 256
    good_c = dict(pages=p, n_pages=2, page_tokens=16, n_kv_heads=2, head_dim=64)
    good_b = dict(n_seqs=1, max_pages=2, max_new=1, q_start=p, kv_lens=p, page_table=p, status=None)

    def append(c={}, b={}, dtype=0, t=1, q=p, qs=256, k=p, ks=128, v=p, vs=128, nh=4, cos=p, sin=p, n_pos=4, eps=1e-6, qo=p):
        return clib.tgx_kvq_append(ctypes.byref(L.TgxKvqCache(**{**good_c, **c})),
                                   ctypes.byref(L.TgxKvqBatch(**{**good_b, **b})), dtype, t, q, qs, k, ks, v, vs, nh, p,
                                   p, eps, cos, sin, n_pos, None, qo, None)

    def attend(c={}, b={}, dtype=0, t=1, q=p, qs=256, nh=4, o=p, os=256, scale=0.0, sc=p, size=None):
        C, B = L.TgxKvqCache(**{**good_c, **c}), L.TgxKvqBatch(**{**good_b, **b})
        n = clib.tgx_kvq_attention_scratch_bytes(ctypes.byref(C), ctypes.byref(B), t, nh) if size is None else size
        return clib.tgx_kvq_attention(ctypes.byref(C), ctypes.byref(B), dtype, t, q, qs, nh, o, os, scale, sc, n, None)

    for call in (append, attend):
        refuse(clib, call(c=dict(pages=None)), "null")
        refuse(clib, call(b=dict(q_start=None)), "null")
        refuse(clib, call(b=dict(page_table=None)), "null")
        refuse(clib, call(c=dict(head_dim=72)), "bad cache")
        refuse(clib, call(c=dict(page_tokens=20)), "bad cache")
        refuse(clib, call(c=dict(n_pages=0)), "bad cache")
        refuse(clib, call(c=dict(pages=p + 8)), "aligned")
        refuse(clib, call(b=dict(n_seqs=0)), "positive")
        refuse(clib, call(b=dict(max_pages=0)), "positive")
        refuse(clib, call(b=dict(max_new=0)), "positive")
        refuse(clib, call(b=dict(max_pages=1 << 30)), "32 bits")
        refuse(clib, call(dtype=3), "dtype")
        refuse(clib, call(t=-1), "n_tokens" if call is append else "n_heads")
        refuse(clib, call(q=None), "null")
        refuse(clib, call(qs=255), "stride")
        refuse(clib, call(qs=258), "stride")
        refuse(clib, call(q=p + 4), "aligned")
    refuse(clib, append(k=None), "null")
    refuse(clib, append(cos=None), "null")
    refuse(clib, append(n_pos=0), "n_pos")
    refuse(clib, append(ks=100), "stride")
    refuse(clib, append(eps=-1.0), "eps")
    refuse(clib, attend(nh=5), "multiple of n_kv_heads")
    refuse(clib, attend(nh=66, qs=66 * 64, os=66 * 64), "32 per kv head")
    refuse(clib, attend(scale=float("nan")), "scale")
    refuse(clib, attend(scale=-1.0), "scale")
    refuse(clib, attend(sc=None), "null")
    refuse(clib, attend(sc=p + 16), "scratch")
    refuse(clib, attend(size=0), "scratch")
    # everything in order but host memory, or no device at all
    for call in (append, attend):
        assert call() == (L.TG_ENODEV if clib.tg_device_count() == 0 else L.TG_EINVAL)



def test_append_refuses_tables_off_their_elements(clib):
    """Norm weights, angles and positions may begin at any element, but not inside one."""
    buf = np.zeros(4096, np.uint8)
    p = (buf.ctypes.data + 255) // 256 * 256
    cache = L.TgxKvqCache(pages=p, n_pages=2, page_tokens=16, n_kv_heads=2, head_dim=64)
    batch = L.TgxKvqBatch(n_seqs=1, max_pages=2, max_new=1, q_start=p, kv_lens=p, page_table=p, status=None)

    def append(qn=p, kn=p, cos=p, sin=p, pos=p):
        return clib.tgx_kvq_append(ctypes.byref(cache), ctypes.byref(batch), 0, 1, p, 256, p, 128, p, 128, 4, qn, kn, 1e-6,
                                   cos, sin, 4, pos, p, None)

    for name in ("qn", "kn", "cos", "sin", "pos"):
        for off in (1, 2, 3):
            refuse(clib, append(**{name: p + off}), "aligned to their elements")
        assert append(**{name: p + 4}) == (L.TG_ENODEV if clib.tg_device_count() == 0 else L.TG_EINVAL)
        assert "aligned" not in clib.tg_last_error().decode()

def test_product_refusals(clib):
    buf = np.zeros(8192, np.uint8)
    p = (buf.ctypes.data + 255) // 256 * 256

    def mat(dtype=0, x=p, xs=32, m=2, k=32, eps=0.0, w=p, ws=p, n=8, res=None, rs=0, out=p, os=8, sc=p, size=4096):
        return clib.tgx_i8_matmul(dtype, x, xs, m, k, None, eps, w, ws, n, res, rs, out, os, sc, size, None)

    for kw, text in ((dict(x=None), "null"), (dict(w=None), "null"), (dict(ws=None), "null"), (dict(out=None), "null"),
                     (dict(sc=None), "null"), (dict(dtype=7), "dtype"), (dict(m=-1), "bad m"), (dict(n=0), "bad m"),
                     (dict(k=0), "bad m"), (dict(k=131073, xs=131073), "bad m"), (dict(xs=31), "bad m"),
                     (dict(os=7), "bad m"), (dict(res=p, rs=7), "bad m"), (dict(eps=-1.0), "eps"),
                     (dict(w=p + 8), "aligned"), (dict(x=p + 2), "elements"), (dict(out=p + 1), "elements"),
                     (dict(sc=p + 128), "scratch"), (dict(size=64), "scratch")):
        refuse(clib, mat(**kw), text)
    assert mat() == (L.TG_ENODEV if clib.tg_device_count() == 0 else L.TG_EINVAL)

    def rows(x=p, xs=32, r=2, c=32, codes=p, scales=p):
        return clib.tgx_i8_quantize_rows(0, x, xs, r, c, None, 0.0, codes, scales, None)

    for kw, text in ((dict(x=None), "null"), (dict(codes=None), "null"), (dict(scales=None), "null"),
                     (dict(c=0), "bad rows"), (dict(r=-1), "bad rows"), (dict(xs=3), "bad rows"), (dict(codes=p + 8), "aligned")):
        refuse(clib, rows(**kw), text)



def test_types_of_fp32_rows(clib):
    """TGX_FROM_F32 goes with a 16-bit type, with x aligned as fp32 and out as the type."""
    buf = np.zeros(8192, np.uint8)
    p = (buf.ctypes.data + 255) // 256 * 256
    none = L.TG_ENODEV if clib.tg_device_count() == 0 else L.TG_EINVAL

    def mat(dtype, x=p, out=p):
        return clib.tgx_i8_matmul(dtype, x, 32, 2, 32, None, 0.0, p, p, 8, None, 0, out, 8, p, 4096, None)

    def rows(dtype, x=p):
        return clib.tgx_i8_quantize_rows(dtype, x, 32, 2, 32, None, 0.0, p, p, None)

    for call in (mat, rows):
        for bad in (L.TGX_FROM_F32 | L.TGX_F32, L.TGX_FROM_F32 | 3, 32 | L.TGX_BF16, -1):
            refuse(clib, call(bad), "dtype")
        for good in (L.TGX_BF16, L.TGX_F16):
            assert call(good | L.TGX_FROM_F32) == none and "dtype" not in clib.tg_last_error().decode()
            refuse(clib, call(good | L.TGX_FROM_F32, x=p + 2), "elements")
    assert mat(L.TGX_F16 | L.TGX_FROM_F32, out=p + 2) == none and "elements" not in clib.tg_last_error().decode()

def test_python_refusals():
    from tinygiant_b200.int8 import Int8Linear, quantize_rows
    from tinygiant_b200.paged import PagedBatch, PagedKV4, dtype_code
    with pytest.raises(ValueError, match="4-bit pages"):
        PagedKV4(4, 100)
    with pytest.raises(ValueError, match="n_pages"):
        PagedKV4(4, 128)
    with pytest.raises(ValueError, match="uint8 cuda"):
        PagedKV4(4, 128, pages=torch.zeros(2, 36864, dtype=torch.uint8))
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="int32 cuda"):
        PagedBatch(i, i[:1], i.view(1, 2), 1)
    with pytest.raises(TypeError):
        dtype_code(torch.zeros(1, dtype=torch.float64))
    with pytest.raises(ValueError, match="cuda matrix"):
        quantize_rows(torch.zeros(2, 2))
    with pytest.raises(ValueError, match="int8 cuda"):
        Int8Linear(torch.zeros(2, 16, dtype=torch.int8), torch.zeros(2), 16)


def test_plain_blocks_follow_the_q4_0_rule(oracle):
    """The 4-bit blocks' codes and scales are those of the library's Q4_0 quantiser."""
    from tests import serve_ref as R
    x = np.random.default_rng(3).standard_normal(4096).astype(np.float32)
    q, d = R.blocks(torch.from_numpy(x).double())
    raw = oracle.quantize_q4_0(x).reshape(-1, 18)
    assert np.array_equal(raw[:, :2].copy().view(np.uint16)[:, 0], d.view(torch.int16).numpy().view(np.uint16))
    lo, hi = raw[:, 2:] & 15, raw[:, 2:] >> 4
    assert np.array_equal(np.concatenate([lo, hi], 1), q.view(-1, 32).numpy())


@pytest.mark.parametrize("hd,page,nkv", [(32, 16, 1), (96, 32, 2), (128, 64, 4), (256, 16, 3)])
def test_plain_pages_cover_every_byte_once(hd, page, nkv):
    from tests import serve_ref as R
    size = nkv * (page // 16) * 18 * hd
    hits = torch.zeros(size, dtype=torch.int64)
    for kind in (0, 1):
        for j in range(nkv):
            tok, d, b = torch.arange(page).view(-1, 1), torch.arange(hd).view(1, -1), torch.arange(hd // 32).view(1, -1)
            at, shift = R.place(nkv, hd, page, kind, j, tok, d)
            hits.index_add_(0, at.expand(page, hd).reshape(-1), (1 + 3 * (shift > 0).long()).expand(page, hd).reshape(-1) * 1)
            s = R.scale_place(nkv, hd, page, kind, j, tok, b).expand(page, hd // 32).reshape(-1)
            hits.index_add_(0, s, torch.full_like(s, 5))
            hits.index_add_(0, s + 1, torch.full_like(s, 5))
    assert (hits == 5).all()   # a byte is a low (1) and a high (4) nibble, or half a scale
