"""What the batched serving operators refuse before any GPU work: through the C ABI, on any machine.  Pointers are made
up; nothing reads them."""
import ctypes as C

import pytest

from rust_interference_engine_amd import _lib

P = 1 << 20  # an aligned address


def seqs(**kw):
    d = dict(n_seq=2, n_rows=8, max_new=4, max_len=100, starts=P, lens=P)
    d.update(kw)
    return _lib.Seqs(**d)


def pages(**kw):
    d = dict(ty=1, head_dim=64, n_kv=2, n_pages=9, page_size=16, table_cols=7, k=P, v=P, page_stride=2048, slot_stride=64,
             head_stride=1024, table=P, table_stride=7)
    d.update(kw)
    return _lib.Pages(**d)


def attn(**kw):
    d = dict(n_head=4, window=0, scale=0.125, softcap=0.0, q=P, q_row_stride=256, q_head_stride=64, out=P, out_row_stride=256, out_head_stride=64)
    d.update(kw)
    return _lib.Attn(**d)


def said(call):
    err = C.create_string_buffer(256)
    rc = call(err)
    return rc, err.value.decode()


def paged(pg=None, sq=None, at=None, ws=P, n=1 << 40):
    L = _lib.lib()
    return said(lambda e: L.rie_hip_k_paged_attention(C.byref(pg or pages()), C.byref(sq or seqs()), C.byref(at or attn()), ws, n, None, e, 256))


@pytest.mark.parametrize("kw,code,text", [
    (dict(pg=pages(ty=0)), -3, "f16 or bf16"), (dict(pg=pages(ty=8)), -3, "f16 or bf16"), (dict(pg=pages(head_dim=80)), -3, "head_dim"),
    (dict(pg=pages(head_dim=0)), -3, "head_dim"), (dict(pg=pages(page_size=24)), -3, "page_size"), (dict(pg=pages(page_size=8)), -3, "page_size"),
    (dict(pg=pages(page_size=0)), -3, "page_size"), (dict(pg=pages(page_size=8192)), -3, "page_size"), (dict(pg=pages(n_pages=0)), -5, "n_pages"),
    (dict(pg=pages(table_cols=0)), -5, "table_cols"), (dict(pg=pages(n_kv=0)), -5, "n_kv"), (dict(pg=pages(k=P + 8)), -5, "16-byte aligned"),
    (dict(pg=pages(slot_stride=68)), -5, "16-byte aligned"), (dict(pg=pages(slot_stride=-64)), -5, "strides"), (dict(pg=pages(slot_stride=1 << 40)), -5, "strides"),
    (dict(pg=pages(page_stride=-8)), -5, "page_stride"), (dict(pg=pages(page_stride=12)), -5, "page_stride"), (dict(pg=pages(table=0)), -5, "table is NULL"),
    (dict(sq=seqs(n_seq=0)), -5, "n_seq"), (dict(sq=seqs(n_rows=0)), -5, "n_rows"), (dict(sq=seqs(max_new=0)), -5, "max_new"), (dict(sq=seqs(max_len=-1)), -5, "max_len"),
    (dict(sq=seqs(n_rows=1 << 30)), -5, "2^26"), (dict(sq=seqs(n_rows=1 << 25)), -5, "2^26"), (dict(sq=seqs(n_seq=1 << 24)), -5, "2^24"),
    (dict(sq=seqs(n_seq=(1 << 23) + 1)), -5, "2^24"),
    (dict(at=attn(n_head=3)), -5, "n_head"), (dict(at=attn(n_head=0)), -5, "n_head"), (dict(at=attn(scale=0.0)), -5, "scale"), (dict(at=attn(scale=-1.0)), -5, "scale"),
    (dict(at=attn(scale=float("nan"))), -5, "scale"), (dict(at=attn(scale=float("inf"))), -5, "scale"), (dict(at=attn(softcap=-1.0)), -5, "softcap"),
    (dict(at=attn(softcap=float("nan"))), -5, "softcap"), (dict(at=attn(window=-1)), -5, "window"), (dict(at=attn(q=P + 2)), -5, "16-byte aligned"),
    (dict(at=attn(out_row_stride=250)), -5, "16-byte aligned"),
])
def test_paged_attention(kw, code, text):
    rc, m = paged(**kw)
    assert rc == code and text in m, (rc, m)


def test_a_workspace_that_is_too_small_or_not_aligned():
    L = _lib.lib()
    sq = seqs(max_len=100000, max_new=1)
    pg = pages(table_cols=10000)
    need = L.rie_hip_k_paged_attention_ws(C.byref(pg), C.byref(sq), C.byref(attn()))
    assert need > 0
    rc, m = paged(pg, sq, n=need - 1)
    assert rc == -5 and f"{need} needed" in m
    rc, m = paged(pg, sq, ws=P + 4, n=need)
    assert rc == -5 and "16-byte aligned" in m
    assert L.rie_hip_k_paged_attention_ws(C.byref(pages(head_dim=48)), C.byref(sq), C.byref(attn())) == 0


def test_null_arguments_and_error_buffers():
    L = _lib.lib()
    assert L.rie_hip_k_paged_attention(None, None, None, None, 0, None, None, 0) == -5
    assert L.rie_hip_k_paged_attention_ws(None, None, None) == 0
    assert L.rie_hip_k_packed_attention_ws(None, 1, 64, 1, None) == 0
    rc, m = said(lambda e: L.rie_hip_k_paged_attention(C.byref(pages()), None, C.byref(attn()), P, 1 << 30, None, e, 256))
    assert rc == -5 and "seqs is NULL" in m
    rc, m = said(lambda e: L.rie_hip_k_paged_attention(C.byref(pages()), C.byref(seqs()), None, P, 1 << 30, None, e, 256))
    assert rc == -5 and "attn is NULL" in m
    err = C.create_string_buffer(8)
    assert L.rie_hip_k_paged_attention(C.byref(pages(ty=0)), C.byref(seqs()), C.byref(attn()), None, 0, None, err, 8) == -3
    assert len(err.value) == 7  # cut, and ended


@pytest.mark.parametrize("args,code,text", [
    ((1, 80, 2, P, P, 256, 64, 256, 64), -3, "head_dim"), ((0, 64, 2, P, P, 256, 64, 256, 64), -3, "f16 or bf16"), ((1, 64, 3, P, P, 256, 64, 256, 64), -5, "n_head"),
    ((1, 64, 2, P + 2, P, 256, 64, 256, 64), -5, "k: rows"), ((1, 64, 2, P, P, 256, 64, 252, 64), -5, "v: rows"), ((1, 64, 2, P, P, -256, 64, 256, 64), -5, "k: strides"),
])
def test_packed_attention(args, code, text):
    L = _lib.lib()
    rc, m = said(lambda e: L.rie_hip_k_packed_attention(C.byref(seqs()), *args, C.byref(attn()), P, 1 << 40, None, e, 256))
    assert rc == code and text in m, (rc, m)


@pytest.mark.parametrize("ty,k,row,head,code,text", [
    (30, P, 128, 64, -3, "f32 or of the pages' type"), (2, P, 128, 64, -3, "f32 or"), (0, P + 4, 128, 64, -5, "aligned"), (0, P, 126, 64, -5, "aligned"), (1, P, 132, 64, -5, "aligned"),
])
def test_paged_append(ty, k, row, head, code, text):
    L = _lib.lib()
    rc, m = said(lambda e: L.rie_hip_k_paged_append(C.byref(pages()), C.byref(seqs()), ty, k, P, row, head, None, e, 256))
    assert rc == code and text in m, (rc, m)


@pytest.mark.parametrize("kw,code,text", [
    (dict(ty=2), -3, "logits have to be"), (dict(n=0), -5, "n has to"), (dict(V=0), -5, "n_vocab"), (dict(V=(1 << 21) + 1), -5, "n_vocab"), (dict(x=P + 2), -5, "aligned"),
    (dict(ld=-1), -5, "row_stride"), (dict(n=1 << 22, V=1 << 20, ld=0), -5, "2^40"), (dict(top=65), -5, "n_top"), (dict(top=-1), -5, "n_top"), (dict(V=10, top=11), -5, "n_top"), (dict(lp=None), -5, "together"),
    (dict(targets=None), -5, "together"), (dict(top=2, ids=None), -5, "top_ids"), (dict(top=2, tops=None), -5, "top_ids"), (dict(bytes=10), -5, "needed"), (dict(ws=P + 8), -5, "ws has"),
])
def test_token_logprobs(kw, code, text):
    d = dict(ty=0, x=P, n=3, V=1000, ld=1000, targets=P, lp=P, top=0, ids=P, tops=P, ws=P, bytes=1 << 30)
    d.update(kw)
    L = _lib.lib()
    rc, m = said(lambda e: L.rie_hip_k_token_logprobs(d["ty"], d["x"], d["n"], d["V"], d["ld"], d["targets"], d["lp"], P, d["top"], d["ids"], d["tops"], d["ws"], d["bytes"], None, e, 256))
    assert rc == code and text in m, (rc, m)
    assert L.rie_hip_k_token_logprobs_ws(0, 5) == 0 and L.rie_hip_k_token_logprobs_ws(5, 0) == 0


def test_the_python_layers_own_checks():
    torch = pytest.importorskip("torch")
    from rust_interference_engine_amd import RieError, ops

    z = torch.zeros
    i32 = torch.int32
    for make, text in [
        (lambda: ops.Seqs(z(1, dtype=i32), max_new=1, max_len=1), "starts"),
        (lambda: ops.Seqs(z(3), max_new=1, max_len=1), "int32"),
        (lambda: ops.Seqs(z(3, dtype=i32), z(3, dtype=i32), max_new=1, max_len=1), "lens for"),
        (lambda: ops.PagedKv(z(2, 16, 1, 64), z(2, 16, 1, 32), z(1, 1, dtype=i32)), "one shape"),
        (lambda: ops.PagedKv(z(2, 16, 64), z(2, 16, 64), z(1, 1, dtype=i32)), "pages have to be"),
        (lambda: ops.PagedKv(z(2, 16, 1, 64), z(2, 16, 1, 64), z(1, 1, dtype=i32)), "on one GPU"),
        (lambda: ops.TokenLogprobs(z(5)), "logits have to be"),
        (lambda: ops.TokenLogprobs(z(5, 4), targets=z(5, dtype=i32)), "together"),
        (lambda: ops.TokenLogprobs(z(5, 4), entropy=z(4)), "entropy has to be"),
        (lambda: ops.TokenLogprobs(z(4, 5).t()), "consecutive"),
        (lambda: ops.TokenLogprobs(z(5, 4)), "on one GPU"),
        (lambda: ops.TokenLogprobs(z(5, 4, requires_grad=True)), "no gradients"),
    ]:
        with pytest.raises(RieError, match=text):
            make()


@pytest.mark.parametrize("at,text", [
    (dict(out_row_stride=0), "out: strides below"), (dict(out_row_stride=32), "out: strides below"), (dict(out_head_stride=0), "out: strides below"),
])
def test_outputs_whose_rows_overlap(at, text):
    rc, m = paged(at=attn(**at))
    assert rc == -5 and text in m, (rc, m)


@pytest.mark.parametrize("pg", [dict(slot_stride=0), dict(head_stride=32), dict(page_stride=0)])
def test_pages_whose_rows_overlap_are_read_and_not_written(pg):
    L = _lib.lib()
    rc, m = said(lambda e: L.rie_hip_k_paged_append(C.byref(pages(**pg)), C.byref(seqs()), 1, P, P, 128, 64, None, e, 256))
    assert rc == -5 and "pages: strides below" in m, (rc, m)
    sq = seqs(max_len=100000, max_new=1)
    assert L.rie_hip_k_paged_attention_ws(C.byref(pages(table_cols=10000, **pg)), C.byref(sq), C.byref(attn())) > 0


def test_the_python_layers_numbers_and_dimensions():
    torch = pytest.importorskip("torch")
    from rust_interference_engine_amd import RieError, ops

    z, i32 = torch.zeros, torch.int32
    st = z(3, dtype=i32)
    sq = ops.Seqs(st, max_new=4, max_len=4)
    q = z(4, 2, 64, dtype=torch.float16)
    for make, text in [
        (lambda: ops.Seqs(st, max_new=(1 << 32) + 1, max_len=1), "max_new has to lie"),
        (lambda: ops.Seqs(st, max_new=1, max_len=(1 << 32) + 1), "max_len has to lie"),
        (lambda: ops.Seqs(st, max_new=0, max_len=1), "max_new has to lie"),
        (lambda: ops.Seqs(st, max_new=1.5, max_len=2), "max_new has to lie"),
        (lambda: ops.PackedAttention(sq, q, q, q, z(4, 2, 64, dtype=torch.float16), window=(1 << 32) + 1), "window has to lie"),
        (lambda: ops.PackedAttention(sq, q, q, q, q[:1].expand(4, 2, 64)), "out is expanded"),
        (lambda: ops.TokenLogprobs(z(5, 4), entropy=z(())), "entropy has 0"),
        (lambda: ops.TokenLogprobs(z(1, (1 << 21) + 1)), "vocabulary has to lie"),
    ]:
        with pytest.raises(RieError, match=text):
            make()


@pytest.mark.parametrize("at", [
    dict(out_row_stride=64),                                     # row r, head h + 1 is row r + 1, head h
    dict(out_row_stride=192),                                    # the last head is the next row's first
    dict(out_row_stride=64, out_head_stride=64 * 7),             # heads apart, by one row too little
])
def test_outputs_whose_rows_overlap_by_two_strides(at):
    rc, m = paged(at=attn(**at))
    assert rc == -5 and "out: strides below" in m, (rc, m)


def append_refusal(pg):
    L = _lib.lib()
    return said(lambda e: L.rie_hip_k_paged_append(C.byref(pg), C.byref(seqs()), 1, P, P, 128, 64, None, e, 256))


@pytest.mark.parametrize("pg", [
    dict(slot_stride=64, head_stride=64, page_stride=64), dict(page_stride=64), dict(page_stride=1984), dict(head_stride=960), dict(slot_stride=128, head_stride=64, page_stride=1984),
    dict(v=P), dict(v=P + 64), dict(v=P + 9 * 2048 * 2 - 16), dict(k=P + 2048, v=P),
])
def test_pages_whose_rows_overlap_by_two_strides(pg):
    rc, m = append_refusal(pages(**{"v": P + (1 << 20), **pg}))
    assert rc == -5 and "pages: strides below" in m, (rc, m)


@pytest.mark.parametrize("pg", [
    dict(), dict(v=P - 9 * 2048 * 2), dict(slot_stride=128, head_stride=64), dict(page_stride=4096, v=P + 2048 * 2),  # keys and values by the page
    dict(slot_stride=128, head_stride=2048, page_stride=4096, v=P + 128),                                             # by the slot
    dict(page_stride=1 << 40, n_pages=2 ** 31 - 1, v=P + (1 << 20)),
])
def test_pages_whose_rows_lie_apart_get_past_the_strides(pg):
    if "page_stride" in pg and pg["page_stride"] == 1 << 40:  # a span of 2^71 values
        rc, m = append_refusal(pages(**pg))
    else:
        rc, m = append_refusal(pages(**{"v": P + (1 << 20), **pg}))
    assert rc == -5 and "overlap" not in m, (rc, m)  # made-up pointers, or no GPU at all


def test_the_python_layers_written_tensors():
    torch = pytest.importorskip("torch")
    from rust_interference_engine_amd import RieError, ops

    z = torch.zeros(100000, dtype=torch.float16)
    q = z[:4 * 2 * 64].view(4, 2, 64)
    sq = ops.Seqs(torch.zeros(3, dtype=torch.int32), max_new=4, max_len=4)
    for stride in ((64, 64, 1), (96, 64, 1), (0, 64, 1), (64, 192, 1)):
        with pytest.raises(RieError, match="out is expanded or overlaps"):
            ops.PackedAttention(sq, q, q, q, z.as_strided((4, 2, 64), stride))
    for stride in ((128, 64, 1), (64, 256, 1), (200, 72, 1)):
        with pytest.raises(RieError, match="on one GPU"):  # past the strides
            ops.PackedAttention(sq, q, q, q, z.as_strided((4, 2, 64), stride))


@pytest.mark.parametrize("n,refused", [((1 << 26) - 4, False), ((1 << 26) - 3, True), ((1 << 26) - 1, True)])
def test_rows_that_a_launch_has_threads_for(n, refused):
    L = _lib.lib()
    pg = pages(v=P + (1 << 20))
    rc, m = said(lambda e: L.rie_hip_k_paged_append(C.byref(pg), C.byref(seqs(n_rows=n)), 1, P, P, 128, 64, None, e, 256))
    assert rc == -5 and ("1..2^26-4" in m) == refused, (rc, m)
    rc, m = paged(pages(n_kv=1), seqs(n_rows=n), attn(n_head=1))
    assert rc == -5 and ("1..2^26-4" in m) == refused, (rc, m)
    rc, m = paged(pages(n_kv=1), seqs(n_rows=n // 2), attn(n_head=2))  # pairs of rows and heads
    assert rc == -5 and ("1..2^26-4" in m) == (n // 2 * 2 > (1 << 26) - 4), (rc, m)
    torch = pytest.importorskip("torch")
    from rust_interference_engine_amd import RieError, ops

    sq = ops.Seqs(torch.zeros(3, dtype=torch.int32), max_new=4, max_len=4)
    if refused:
        with pytest.raises(RieError, match="rows has to lie"):
            sq._struct(n)
    else:
        assert sq._struct(n).n_rows == n


def test_strides_of_dimensions_with_one_entry_are_not_looked_at():
    L = _lib.lib()
    odd = 3
    one = pages(n_kv=1, n_pages=1, head_stride=odd, page_stride=-odd, v=P + (1 << 20))
    for call in (lambda e: L.rie_hip_k_paged_append(C.byref(one), C.byref(seqs(n_rows=1)), 1, P, P, odd, -odd, None, e, 256),
                 lambda e: L.rie_hip_k_paged_attention(C.byref(one), C.byref(seqs(n_rows=1)), C.byref(attn(
                     n_head=1, q_row_stride=odd, q_head_stride=1 << 50, out_row_stride=odd, out_head_stride=-1)), P, 1 << 40, None, e, 256),
                 lambda e: L.rie_hip_k_packed_attention(C.byref(seqs(n_rows=1)), 1, 64, 1, P, P, odd, odd, -odd, 1 << 50, C.byref(attn(n_head=1, out_row_stride=0)), P, 1 << 40, None, e, 256)):
        rc, m = said(call)
        assert rc == -5 and "stride" not in m and "aligned" not in m, (rc, m)  # made-up pointers, or no GPU at all
    torch = pytest.importorskip("torch")
    from rust_interference_engine_amd import RieError, ops

    z = torch.zeros(4096, dtype=torch.float16)
    with pytest.raises(RieError, match="on one GPU"):  # past the strides
        ops.PagedKv(z.as_strided((2, 16, 1, 64), (1024, 64, 5, 1)), z.as_strided((2, 16, 1, 64), (1024, 64, 64, 1)), torch.zeros(1, 1, dtype=torch.int32))
