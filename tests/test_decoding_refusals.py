"""What the operators over 8-bit pages, rotary positions, beam selection and pools of pages refuse before any GPU work:
through the C ABI, on any machine.  Pointers are made up; nothing reads them."""
import ctypes as C

import pytest

from rust_interference_engine_amd import _lib

P = 1 << 20  # an aligned address
V = P + (1 << 26)  # another, behind all that lies at P
G = C.c_void_p


def said(call):
    err = C.create_string_buffer(256)
    rc = call(err)
    return rc, err.value.decode()


def seqs(**kw):
    return _lib.Seqs(**{**dict(n_seq=2, n_rows=8, max_new=4, max_len=100, starts=P, lens=P), **kw})


def pages8(block=16, k_scale=P, v_scale=V, scale_page_stride=2, scale_block_stride=2, scale_head_stride=1, **kw):
    pg = _lib.Pages(**{**dict(ty=24, head_dim=64, n_kv=2, n_pages=9, page_size=16, table_cols=7, k=P, v=V, page_stride=2048, slot_stride=64,
                              head_stride=1024, table=P, table_stride=7), **kw})
    return _lib.Pages8(pages=pg, k_scale=k_scale, v_scale=v_scale, scale_page_stride=scale_page_stride, scale_block_stride=scale_block_stride,
                       scale_head_stride=scale_head_stride, block=block)


def attn(**kw):
    return _lib.Attn(**{**dict(n_head=4, window=0, scale=0.125, softcap=0.0, q=P, q_row_stride=256, q_head_stride=64, out=P, out_row_stride=256, out_head_stride=64), **kw})


def attend(pg=None, sq=None, at=None, ty=1, ws=P, n=1 << 40):
    L = _lib.lib()
    return said(lambda e: L.rie_hip_k_paged_attention8(C.byref(pg or pages8()), C.byref(sq or seqs()), ty, C.byref(at or attn()), ws, n, None, e, 256))


def append(pg=None, sq=None, ty=1, k=P, v=P, row=128, head=64):
    L = _lib.lib()
    return said(lambda e: L.rie_hip_k_paged_append8(C.byref(pg or pages8()), C.byref(sq or seqs()), ty, k, v, row, head, None, e, 256))


BAD_PAGES = [
    (dict(ty=1), -3, "int8"), (dict(ty=0), -3, "int8"), (dict(head_dim=80), -3, "head_dim"), (dict(head_dim=0), -3, "head_dim"), (dict(n_kv=0), -5, "n_kv"),
    (dict(page_size=24), -3, "page_size"), (dict(page_size=8), -3, "page_size"), (dict(page_size=8192), -3, "page_size"), (dict(n_pages=0), -5, "n_pages"),
    (dict(table_cols=0), -5, "table_cols"), (dict(block=8), -3, "block"), (dict(block=0), -3, "block"), (dict(block=-16), -3, "block"), (dict(block=32), -3, "block"),
    (dict(block=48, page_size=64), -3, "block"), (dict(scale_page_stride=-1), -5, "scales: strides"), (dict(scale_page_stride=1 << 31), -5, "scales: strides"),
    (dict(scale_head_stride=-1), -5, "scales: strides"), (dict(scale_block_stride=1 << 31, page_size=32), -5, "scales: strides"), (dict(k_scale=P + 2), -5, "scales have to be aligned"),
    (dict(v_scale=V + 1), -5, "scales have to be aligned"), (dict(k=P + 8), -5, "16-byte aligned"), (dict(slot_stride=72), -5, "16-byte aligned"),
    (dict(slot_stride=-64), -5, "strides"), (dict(page_stride=-16), -5, "page_stride"), (dict(page_stride=8), -5, "page_stride"),
]


@pytest.mark.parametrize("kw,code,text", BAD_PAGES)
def test_pages_in_8_bits(kw, code, text):
    for rc, m in (attend(pages8(**kw)), append(pages8(**kw))):
        assert rc == code and text in m, (rc, m)
    assert _lib.lib().rie_hip_k_paged_attention8_ws(C.byref(pages8(**{"table_cols": 10000, **kw})), C.byref(seqs(max_len=100000, max_new=1)), 1, C.byref(attn())) == 0


@pytest.mark.parametrize("kw,code,text", [
    (dict(pg=pages8(table=0)), -5, "table is NULL"), (dict(ty=0), -3, "f16 or bf16"), (dict(ty=24), -3, "f16 or bf16"), (dict(sq=seqs(n_seq=0)), -5, "n_seq"),
    (dict(sq=seqs(max_new=0)), -5, "max_new"), (dict(sq=seqs(max_len=-1)), -5, "max_len"), (dict(at=attn(n_head=3)), -5, "n_head"), (dict(at=attn(scale=float("nan"))), -5, "scale"),
    (dict(at=attn(scale=0.0)), -5, "scale"), (dict(at=attn(softcap=-1.0)), -5, "softcap"), (dict(at=attn(window=-1)), -5, "window"), (dict(at=attn(q=P + 2)), -5, "16-byte aligned"),
    (dict(at=attn(out_row_stride=64)), -5, "out: strides below"),
])
def test_attention(kw, code, text):
    rc, m = attend(**kw)
    assert rc == code and text in m, (rc, m)


def test_a_workspace_that_is_too_small_or_not_aligned():
    L = _lib.lib()
    for max_new in (1, 4000):  # both kernels
        sq, pg = seqs(max_len=100000, max_new=max_new, n_rows=8000), pages8(table_cols=10000)
        need = L.rie_hip_k_paged_attention8_ws(C.byref(pg), C.byref(sq), 1, C.byref(attn()))
        assert need > 0
        rc, m = attend(pg, sq, n=need - 1)
        assert rc == -5 and f"{need} needed" in m
        rc, m = attend(pg, sq, ws=P + 4, n=need)
        assert rc == -5 and "16-byte aligned" in m


def test_null_arguments():
    L = _lib.lib()
    assert L.rie_hip_k_paged_attention8(None, None, 1, None, None, 0, None, None, 0) == -5
    assert L.rie_hip_k_paged_attention8_ws(None, None, 1, None) == 0
    assert L.rie_hip_k_paged_append8(None, None, 1, None, None, 0, 0, None, None, 0) == -5
    assert said(lambda e: L.rie_hip_k_paged_append8(C.byref(pages8()), None, 1, P, P, 128, 64, None, e, 256)) == (-5, "seqs is NULL")
    assert L.rie_hip_k_rotary(None, None, None, None, 0) == -5
    assert L.rie_hip_k_page_ws(None) == 0
    for rc, m in (said(lambda e: L.rie_hip_k_page_reserve(None, P, 1 << 30, None, e, 256)), said(lambda e: L.rie_hip_k_page_fork(None, P, None, 0, P, 1 << 30, None, e, 256)),
                  said(lambda e: L.rie_hip_k_page_free(None, P, None, e, 256)), said(lambda e: L.rie_hip_k_page_compact(None, None, 0, P, 1 << 30, None, e, 256))):
        assert (rc, m) == (-5, "pool is NULL")


@pytest.mark.parametrize("kw,code,text", [
    (dict(ty=2), -3, "new rows"), (dict(ty=24), -3, "new rows"), (dict(k=P + 4), -5, "k: rows"), (dict(v=P + 8), -5, "v: rows"), (dict(row=132), -5, "aligned"), (dict(ty=0, row=130), -5, "aligned"),
    (dict(row=-128), -5, "strides"), (dict(head=1 << 40), -5, "strides"), (dict(sq=seqs(n_rows=0)), -5, "n_rows"), (dict(sq=seqs(n_seq=(1 << 24) - 1)), -5, "2^25"),
    # pages that are written and overlap: codes
    (dict(pg=pages8(slot_stride=0)), -5, "pages: strides below"), (dict(pg=pages8(head_stride=32)), -5, "pages: strides below"), (dict(pg=pages8(page_stride=0)), -5, "pages: strides below"),
    (dict(pg=pages8(page_stride=1984)), -5, "pages: strides below"), (dict(pg=pages8(v=P)), -5, "pages: strides below"), (dict(pg=pages8(v=P + 9 * 2048 - 16)), -5, "pages: strides below"),
    # and scales
    (dict(pg=pages8(scale_page_stride=0)), -5, "scales: strides below"), (dict(pg=pages8(scale_page_stride=1)), -5, "scales: strides below"),
    (dict(pg=pages8(scale_head_stride=0)), -5, "scales: strides below"), (dict(pg=pages8(v_scale=P)), -5, "scales: strides below"), (dict(pg=pages8(v_scale=P + 4)), -5, "scales: strides below"),
    (dict(pg=pages8(page_size=32, head_stride=2048, page_stride=4096, scale_page_stride=4, scale_block_stride=1)), -5, "scales: strides below"),
])
def test_append(kw, code, text):
    rc, m = append(**kw)
    assert rc == code and text in m, (rc, m)


@pytest.mark.parametrize("pg", [
    dict(), dict(v=P + 9 * 2048), dict(slot_stride=128, head_stride=64), dict(v_scale=P + 4 * 18),
    dict(scale_page_stride=4, v_scale=P + 8),                    # keys' and values' scales by the page
    dict(page_stride=4096, v=P + 2048), dict(page_size=64, head_stride=4096, page_stride=8192, block=32, scale_page_stride=4, scale_block_stride=2),
    dict(scale_page_stride=(1 << 31) - 1, v_scale=P + 8),
])
def test_pages_that_lie_apart_get_past_the_strides(pg):
    rc, m = append(pages8(**pg))
    assert rc == -5 and "overlap" not in m and "strides" not in m, (rc, m)  # made-up pointers, or no GPU at all


ROT = dict(n_rows=8, head_dim=64, dims=64, n_q=4, n_k=2, interleaved=0, src_ty=1, dst_ty=1, magnitude=1.0, freqs=P, positions=P, q=P, q_row_stride=256, q_head_stride=64,
           q_out=V, q_out_row_stride=256, q_out_head_stride=64, k=P, k_row_stride=128, k_head_stride=64, k_out=V, k_out_row_stride=128, k_out_head_stride=64)


def rotary(sq=None, **kw):
    x = _lib.Rotary(**{**ROT, **kw})
    return said(lambda e: _lib.lib().rie_hip_k_rotary(C.byref(x), C.byref(sq) if sq else None, None, e, 256))


@pytest.mark.parametrize("kw,code,text", [
    (dict(positions=0), -5, "positions or seqs"), (dict(sq=seqs()), -5, "positions or seqs"), (dict(src_ty=24), -3, "rows have to be"), (dict(dst_ty=8), -3, "rows have to be"),
    (dict(head_dim=0, dims=0), -3, "head_dim"), (dict(head_dim=1026), -3, "head_dim"), (dict(dims=0), -3, "dims"), (dict(dims=33), -3, "dims"), (dict(dims=66), -3, "dims"), (dict(dims=-2), -3, "dims"),
    (dict(n_q=-1), -5, "n_q"), (dict(n_q=0, n_k=0), -5, "n_q"), (dict(n_k=4097), -5, "n_q and n_k"), (dict(magnitude=float("inf")), -5, "magnitude"), (dict(magnitude=float("nan")), -5, "magnitude"),
    (dict(n_rows=0), -5, "n_rows"), (dict(n_rows=(1 << 26) - 3), -5, "n_rows"), (dict(freqs=P + 4), -5, "freqs"), (dict(positions=0, sq=seqs(n_rows=7)), -5, "differ"),
    (dict(q=P + 1), -5, "q has to be aligned"), (dict(src_ty=0, k=P + 2), -5, "k has to be aligned"), (dict(k_out=V + 1), -5, "k has to be aligned"), (dict(q_row_stride=-1), -5, "q: strides have"),
    (dict(k_out_head_stride=(1 << 40) + 1), -5, "k: strides have"), (dict(q_out_row_stride=0), -5, "q: strides below"), (dict(q_out_row_stride=64), -5, "q: strides below"),
    (dict(k_out_head_stride=32), -5, "k: strides below"), (dict(q_out=P, dst_ty=30), -5, "in place"), (dict(q_out=P, q_out_row_stride=512), -5, "in place"),
    (dict(k_out=P, k_out_row_stride=64, k_out_head_stride=512), -5, "in place"),
])
def test_rotary(kw, code, text):
    rc, m = rotary(**kw)
    assert rc == code and text in m, (rc, m)


@pytest.mark.parametrize("kw", [
    dict(), dict(n_q=0, q=0, q_out=0), dict(n_k=0, k=0, k_out=0), dict(q=P + 2, q_row_stride=257), dict(q_row_stride=0, q_head_stride=0), dict(n_rows=1, q_out_row_stride=-5),
    dict(q_out=P, k_out=P), dict(positions=0, sq=seqs()), dict(n_rows=(1 << 26) - 4), dict(head_dim=1024, dims=2, q_out_head_stride=1024, q_out_row_stride=4096, k_out_head_stride=1024, k_out_row_stride=2048),
])
def test_rotary_calls_that_get_past_the_checks(kw):
    rc, m = rotary(**kw)
    assert rc == -5 and not any(w in m for w in ("stride", "aligned", "has to", "have to", "place")), (rc, m)  # made-up pointers, or no GPU at all


@pytest.mark.parametrize("kw,code,text", [
    (dict(ty=24), -3, "logits have to be"), (dict(n=0), -5, "n_beams"), (dict(beams=0), -5, "n_beams"), (dict(beams=65), -5, "n_beams"), (dict(n=(1 << 20) + 1, beams=4), -5, "n_beams"), (dict(V=0), -5, "n_vocab"),
    (dict(V=(1 << 21) + 1), -5, "n_vocab"), (dict(out=0), -5, "n_out"), (dict(out=129), -5, "n_out"), (dict(V=2, beams=3, out=7), -5, "n_out"), (dict(n=1 << 20, beams=4, V=1 << 20), -5, "2^40"),
    (dict(x=P + 2), -5, "aligned"), (dict(x=P + 1, ty=1), -5, "aligned"), (dict(ld=-1), -5, "row_stride"), (dict(ld=(1 << 40) + 1), -5, "row_stride"), (dict(finished=P, pad=-1), -5, "pad"),
    (dict(finished=P, pad=1000), -5, "pad"), (dict(bytes=10), -5, "needed"), (dict(ws=P + 8), -5, "ws has"),
])
def test_beam_select(kw, code, text):
    d = {**dict(ty=0, x=P, n=3, beams=4, V=1000, ld=1000, finished=None, pad=0, out=8, ws=P, bytes=1 << 40), **kw}
    L = _lib.lib()
    rc, m = said(lambda e: L.rie_hip_k_beam_select(d["ty"], d["x"], d["n"], d["beams"], d["V"], d["ld"], P, d["finished"], d["pad"], d["out"], P, P, P, d["ws"], d["bytes"], None, e, 256))
    assert rc == code and text in m, (rc, m)


def test_the_beam_workspace():
    L = _lib.lib()
    assert L.rie_hip_k_beam_select_ws(0, 1, 5, 1) == L.rie_hip_k_beam_select_ws(1, 65, 500, 1) == L.rie_hip_k_beam_select_ws(1, 1, 5, 6) == L.rie_hip_k_beam_select_ws(1, 1, 1 << 22, 6) == 0
    need = L.rie_hip_k_beam_select_ws(3, 4, 1000, 8)
    rc, m = said(lambda e: L.rie_hip_k_beam_select(0, P, 3, 4, 1000, 1000, P, None, 0, 8, P, P, P, P, need - 1, None, e, 256))
    assert rc == -5 and f"{need} needed" in m
    assert 0 < need < 1 << 20 and L.rie_hip_k_beam_select_ws(1 << 16, 64, 1 << 18, 128) > 0


def pool(**kw):
    return _lib.Pool(**{**dict(n_seq=4, n_pages=100, table_cols=10, page_size=16, table=P, table_stride=10, lens=P, held=P, refs=P, counts=P), **kw})


def bufs(*kw):
    return (_lib.PageBuf * len(kw))(*(_lib.PageBuf(**{**dict(base=P, page_stride=4096, page_bytes=4096), **k}) for k in kw))


@pytest.mark.parametrize("kw,code,text", [
    (dict(n_seq=0), -5, "n_seq"), (dict(n_seq=4097), -5, "n_seq"), (dict(n_pages=0), -5, "n_pages"), (dict(n_pages=(1 << 24) + 1), -5, "n_pages"), (dict(table_cols=0), -5, "table_cols"),
    (dict(table_cols=(1 << 20) + 1, table_stride=1 << 21), -5, "table_cols"), (dict(page_size=0), -3, "page_size"), (dict(page_size=24), -3, "page_size"), (dict(page_size=8192), -3, "page_size"),
    (dict(page_size=-16), -3, "page_size"), (dict(table_stride=9), -5, "table_stride"), (dict(table_stride=-10), -5, "table_stride"), (dict(table_stride=(1 << 40) + 1), -5, "table_stride"),
])
def test_pools(kw, code, text):
    L, p = _lib.lib(), pool(**kw)
    for rc, m in (said(lambda e: L.rie_hip_k_page_reserve(C.byref(p), P, 1 << 40, None, e, 256)), said(lambda e: L.rie_hip_k_page_fork(C.byref(p), P, None, 0, P, 1 << 40, None, e, 256)),
                  said(lambda e: L.rie_hip_k_page_free(C.byref(p), P, None, e, 256)), said(lambda e: L.rie_hip_k_page_compact(C.byref(p), None, 0, P, 1 << 40, None, e, 256))):
        assert rc == code and text in m, (rc, m)
    assert L.rie_hip_k_page_ws(C.byref(p)) == 0


def with_bufs(b, n):
    L = _lib.lib()
    return (said(lambda e: L.rie_hip_k_page_fork(C.byref(pool()), P, b, n, P, 1 << 40, None, e, 256)), said(lambda e: L.rie_hip_k_page_compact(C.byref(pool()), b, n, P, 1 << 40, None, e, 256)),
            said(lambda e: L.rie_hip_k_page_copy(b, n, 100, P, P, 5, None, e, 256)))


@pytest.mark.parametrize("kw,text", [
    (dict(page_bytes=0), "page_bytes"), (dict(page_bytes=6), "page_bytes"), (dict(page_bytes=(1 << 30) + 4, page_stride=1 << 31), "page_bytes"), (dict(base=P + 2), "base"), (dict(page_stride=4098), "base"),
    (dict(page_stride=4092), "page_stride"), (dict(page_stride=0), "page_stride"), (dict(page_stride=-4096), "page_stride"), (dict(page_stride=(1 << 40) + 4), "page_stride"),
])
def test_caches_whose_pages_move(kw, text):
    for rc, m in with_bufs(bufs({}, kw), 2):
        assert rc == -5 and text in m, (rc, m)


def test_counts_of_caches_and_pages():
    for rc, m in with_bufs(None, 1):
        assert rc == -5 and "bufs is NULL" in m, (rc, m)
    for n in (-1, 4097):
        for rc, m in with_bufs(bufs({}), n):
            assert rc == -5 and "n_bufs" in m, (rc, m)
    L = _lib.lib()
    for n_pages, n in ((0, 5), (100, 0), (100, (1 << 24) + 1), ((1 << 24) + 1, 5)):
        rc, m = said(lambda e: L.rie_hip_k_page_copy(bufs({}), 1, n_pages, P, P, n, None, e, 256))
        assert rc == -5 and "2^24" in m, (rc, m)


def test_the_pools_workspace():
    L, p = _lib.lib(), pool(n_seq=4096, n_pages=1 << 24, table_cols=1 << 20, table_stride=1 << 20)
    assert L.rie_hip_k_page_ws(C.byref(p)) > 4096 << 20
    for n in (0, 15):
        for rc, m in (said(lambda e: L.rie_hip_k_page_reserve(C.byref(pool()), P, n, None, e, 256)), said(lambda e: L.rie_hip_k_page_fork(C.byref(pool()), P, None, 0, P, n, None, e, 256)),
                      said(lambda e: L.rie_hip_k_page_compact(C.byref(pool()), None, 0, P, n, None, e, 256))):
            assert rc == -5 and "needed" in m, (rc, m)
    rc, m = said(lambda e: L.rie_hip_k_page_reserve(C.byref(pool()), P + 8, 1 << 40, None, e, 256))
    assert rc == -5 and "16-byte aligned" in m


def test_the_python_layers_own_checks():
    torch = pytest.importorskip("torch")
    from rust_interference_engine_amd import RieError, ops

    z, i8, i32 = torch.zeros, torch.int8, torch.int32
    k, s, t = z(3, 32, 2, 64, dtype=i8), z(3, 2, 2), z(1, 3, dtype=i32)
    f, q, ids = z(32, dtype=torch.float64), z(5, 2, 64), z(5, dtype=i32)
    b = dict(logits=z(4, 10), scores=z(2, 2), next_scores=z(2, 3), parents=z(2, 3, dtype=i32), tokens=z(2, 3, dtype=i32))
    p = dict(table=z(2, 4, dtype=i32), lens=z(2, dtype=i32), held=z(2, dtype=i32), refs=z(9, dtype=i32), counts=z(2, dtype=i32), page_size=16)
    for make, text in [
        (lambda: ops.PagedKv(k, k.clone(), t), "k_scale and v_scale"),
        (lambda: ops.PagedKv(k, k.clone(), t, k_scale=s), "k_scale and v_scale"),
        (lambda: ops.PagedKv(k.half(), k.half(), t, k_scale=s, v_scale=s.clone()), "k_scale and v_scale"),
        (lambda: ops.PagedKv(k, k.clone(), t, k_scale=s, v_scale=z(3, 1, 2)), "scales have to be"),
        (lambda: ops.PagedKv(k, k.clone(), t, k_scale=z(2, 2, 2), v_scale=z(2, 2, 2)), "scales have to be"),
        (lambda: ops.PagedKv(k, k.clone(), t, k_scale=z(3, 3, 2), v_scale=z(3, 3, 2)), "scales have to be"),
        (lambda: ops.PagedKv(k, k.clone(), t, k_scale=z(3, 2), v_scale=z(3, 2)), "scales have to be"),
        (lambda: ops.PagedKv(k, k.clone(), t, k_scale=s.double(), v_scale=s.double()), "f32 is wanted"),
        (lambda: ops.PagedKv(k, k.clone(), t, k_scale=s, v_scale=z(3, 2, 4)[:, :, ::2]), "same strides"),
        (lambda: ops.PagedKv(k, k.clone(), t, k_scale=s, v_scale=s.clone()), "on one GPU"),
        (lambda: ops.Rotary(f.float(), q, None, q, None, positions=ids), "f64"),
        (lambda: ops.Rotary(z(33, dtype=torch.float64), q, None, q, None, positions=ids), "66 dims"),
        (lambda: ops.Rotary(f, q, None, q, None), "positions or seqs"),
        (lambda: ops.Rotary(f, q, q, q, None, positions=ids), "given together"),
        (lambda: ops.Rotary(f, q, None, q[:, :1], None, positions=ids), "one shape"),
        (lambda: ops.Rotary(f, q, q[:4], q, q[:4], positions=ids), "one shape"),
        (lambda: ops.Rotary(f, q, q.half(), q, q, positions=ids), "one type"),
        (lambda: ops.Rotary(f, q, None, q, None, positions=ids[:4]), "4 positions"),
        (lambda: ops.Rotary(f, q, None, q, None, positions=ids.long()), "positions"),
        (lambda: ops.Rotary(f, q, None, z(1, 2, 64).expand(5, 2, 64), None, positions=ids), "expanded"),
        (lambda: ops.Rotary(f, q, None, q, None, seqs=ops.Seqs(z(2, dtype=i32), max_new=5, max_len=5)), "no lens"),
        (lambda: ops.Rotary(f, q, None, q, None, positions=ids), "on one GPU"),
        (lambda: ops.BeamSelect(**{**b, "logits": z(4)}), "logits have to be"),
        (lambda: ops.BeamSelect(**{**b, "logits": z(10, 4).t()}), "consecutive"),
        (lambda: ops.BeamSelect(**{**b, "scores": z(3, 2)}), "scores have to be"),
        (lambda: ops.BeamSelect(**{**b, "scores": z(2, 2).double()}), "scores has to be"),
        (lambda: ops.BeamSelect(**{**b, "parents": z(2, 2, dtype=i32)}), "number wanted"),
        (lambda: ops.BeamSelect(**{**b, "tokens": z(2, 3)}), "tokens has to be"),
        (lambda: ops.BeamSelect(**{**b, "next_scores": z(3, 2).t()}), "next_scores has to be"),
        (lambda: ops.BeamSelect(**b, finished=z(4, dtype=i32)), "finished"),
        (lambda: ops.BeamSelect(**b), "on one GPU"),
        (lambda: ops.PagePool(**{**p, "lens": z(3, dtype=i32)}), "3 lens"),
        (lambda: ops.PagePool(**{**p, "held": z(2)}), "held"),
        (lambda: ops.PagePool(**{**p, "counts": z(1, dtype=i32)}), "two numbers"),
        (lambda: ops.PagePool(**{**p, "table": z(1, 4, dtype=i32).expand(2, 4)}), "table"),
        (lambda: ops.PagePool(**p), "on one GPU"),
        (lambda: ops.PageCopy([], ids, ids), "no caches"),
        (lambda: ops.PageCopy([k], ids, ids[:4]), "5 src and 4 dst"),
        (lambda: ops.PageCopy([k, k[:2]], ids, ids), "a cache has to be"),
        (lambda: ops.PageCopy([k[:, :, :, ::2]], ids, ids), "lie together"),
        (lambda: ops.PageCopy([k[:, :1].expand(3, 32, 2, 64)], ids, ids), "lie together"),
        (lambda: ops.PageCopy([k.transpose(1, 2)], ids, ids), "on one GPU"),
    ]:
        with pytest.raises(RieError, match=text):
            make()
