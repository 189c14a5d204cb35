"""The mixed-serving-batch operators refuse on the host, before any device work, what they do not cover (no GPU)."""
import ctypes as C

import numpy as np
import pytest

from zeroplatform_b200 import _lib

BUF = np.zeros(4096 + 4, np.float64)  # never dereferenced: every call below is refused first
P = (BUF.ctypes.data + 15) // 16 * 16


def reserve(table=P, lens=P, free=P, count=P, max_rows=4, max_pages=8, num_pages=16, page=16, rows=None, new=P,
            batch=2, tokens=8, start=P, slots=P, pos=P, trow=P, ctx=P, granted=P):
    return _lib.lib().zcu_pages_reserve(table, lens, free, count, max_rows, max_pages, num_pages, page, rows, new,
                                        batch, tokens, start, slots, pos, trow, ctx, granted, None)


@pytest.mark.parametrize("bad", [dict(table=None), dict(lens=None), dict(free=None), dict(count=None), dict(new=None),
                                 dict(start=None), dict(slots=None), dict(pos=None), dict(trow=None), dict(ctx=None),
                                 dict(granted=None), dict(max_rows=0), dict(max_pages=0), dict(num_pages=0),
                                 dict(page=0), dict(page=-16), dict(batch=-1), dict(tokens=-1), dict(batch=5)])
def test_reserve_refuses(bad):
    assert reserve(**bad) == -2
    assert b"zcu_pages_reserve" in _lib.lib().zc_cuda_last_error()


def test_reserve_refuses_more_than_one_cta_holds():
    assert reserve(batch=20000, max_rows=20000) == -6
    assert reserve(batch=4, max_rows=60000, rows=P) == -6


def trim(table=P, lens=P, free=P, count=P, max_rows=4, max_pages=8, num_pages=16, page=16, rows=None, new=P, batch=2):
    return _lib.lib().zcu_pages_trim(table, lens, free, count, max_rows, max_pages, num_pages, page, rows, new, batch,
                                     None)


@pytest.mark.parametrize("bad", [dict(table=None), dict(lens=None), dict(free=None), dict(count=None), dict(new=None),
                                 dict(max_rows=0), dict(page=0), dict(batch=-1), dict(batch=5)])
def test_trim_refuses(bad):
    assert trim(**bad) == -2


def test_trim_of_nothing_is_nothing():
    assert trim(batch=0) == 0


def append(k=P, v=P, in_dtype=0, ks=256, vs=256, slots=P, tokens=2, kp=P, vp=P, kv_dtype=1, hkv=2, hd=128, page=16,
           pages=4, sp=4096, ss=128, sh=2048, bounds=P, scales=P):
    return _lib.lib().zcu_append_kv(k, v, in_dtype, ks, vs, slots, tokens, kp, vp, kv_dtype, hkv, hd, page, pages, sp,
                                    ss, sh, bounds, scales, None)


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(slots=None), dict(kp=None), dict(vp=None),
                                 dict(bounds=None), dict(scales=None), dict(in_dtype=2), dict(kv_dtype=-1),
                                 dict(hkv=0), dict(hd=0), dict(page=0), dict(pages=0), dict(tokens=-1), dict(ks=258),
                                 dict(ss=130), dict(k=P + 4), dict(kp=P + 4), dict(bounds=P + 1)])
def test_append_refuses(bad):
    assert append(**bad) == -2


def test_append_covers_four_head_sizes():
    assert append(hd=96) == -4 and append(hd=512) == -4 and append(hd=16) == -4
    assert append(tokens=0, k=None, v=None, slots=None) == 0


def test_append_refuses_more_tokens_than_it_indexes():
    assert append(tokens=2 ** 31 - 4096) == -6 and append(tokens=2 ** 31 - 1) == -6


def sparse(q=P, qs=1024, kp=P, vp=P, kv_dtype=1, bounds=P, scales=P, table=P, table_rows=2, rows=None, ctx=P, out=P,
           sel=P, batch=2, hq=8, hkv=2, hd=128, page=16, max_pages=64, pages=128, sp=4096, ss=128, sh=2048,
           max_ctx=1024, budget=8, sink=1, recent=1):
    return _lib.lib().zcu_sparse_paged_attention(q, qs, kp, vp, kv_dtype, bounds, scales, table, table_rows, rows, ctx,
                                                 out, sel, batch, hq, hkv, hd, page, max_pages, pages, sp, ss, sh,
                                                 0.125, max_ctx, budget, sink, recent, None)


@pytest.mark.parametrize("bad", [dict(q=None), dict(kp=None), dict(vp=None), dict(bounds=None), dict(scales=None),
                                 dict(table=None), dict(ctx=None), dict(out=None), dict(sel=None), dict(kv_dtype=2),
                                 dict(batch=-1), dict(hq=0), dict(hkv=0), dict(hq=7), dict(hd=0), dict(page=0),
                                 dict(max_pages=0), dict(pages=0), dict(table_rows=0), dict(table_rows=1),
                                 dict(max_ctx=-1), dict(budget=0), dict(sink=-1), dict(recent=-1),
                                 dict(sink=5, recent=4), dict(ss=132), dict(kp=P + 8), dict(bounds=P + 8),
                                 dict(sink=2 ** 31 - 1, recent=2 ** 31 - 1)])
def test_sparse_attention_refuses(bad):
    assert sparse(**bad) == -2


def test_sparse_attention_covers_three_head_sizes_and_pages_of_eights():
    assert sparse(hd=96, ss=96) == -4 and sparse(hd=32) == -4 and sparse(hd=512, ss=512) == -4
    assert sparse(page=20) == -4 and sparse(page=4) == -4
    assert sparse(max_pages=1 << 20, max_ctx=1 << 20) == -6
    assert sparse(batch=0) == 0


def lora(x=P, xs=64, y=P, ys=40, out=P, os=40, a=P, b=P, w=1, adapter=P, ranks=None, scales=None, rows=2, k=64, n=40,
         adapters=3, rank=8):
    return _lib.lib().zcu_lora_add(x, xs, y, ys, out, os, a, b, w, adapter, ranks, scales, rows, k, n, adapters, rank,
                                   None)


@pytest.mark.parametrize("bad", [dict(x=None), dict(y=None), dict(out=None), dict(a=None), dict(b=None),
                                 dict(adapter=None), dict(w=3), dict(w=-1), dict(rows=-1), dict(k=0), dict(n=0),
                                 dict(adapters=0), dict(rank=0), dict(xs=63), dict(xs=66), dict(ys=39), dict(os=39),
                                 dict(os=48), dict(x=P + 8), dict(a=P + 2), dict(b=P + 8)])
def test_lora_refuses(bad):
    assert lora(**bad) == -2


def test_lora_covers_ranks_of_eights_to_128_and_columns_of_32():
    assert lora(rank=12) == -4 and lora(rank=136) == -4 and lora(k=48, xs=48) == -4
    assert lora(rows=0, x=None) == 0


def logits(x=P, dtype=0, xs=64, out=P + 1024, os=64, rows=2, vocab=64, **rules):
    r = _lib.LogitsRules(**rules)
    return _lib.lib().zcu_process_logits(x, dtype, xs, out, os, rows, vocab, C.byref(r), None)


@pytest.mark.parametrize("bad", [dict(x=None), dict(out=None), dict(dtype=3), dict(dtype=-1), dict(rows=-1),
                                 dict(vocab=0), dict(xs=63), dict(os=63), dict(past=P, past_cap=4, past_count=2),
                                 dict(past=P, past_len=P, past_cap=-1, past_count=2),
                                 dict(past=P, past_len=P, past_cap=4, past_count=0),
                                 dict(bias_start=P, n_bias=3), dict(bias_start=P, n_bias=-1),
                                 dict(mask=P, masks=2, mask_stride=1), dict(mask=P, masks=0, mask_stride=2),
                                 dict(mask=P, masks=1, mask_stride=2), dict(out=P, dtype=1), dict(out=P, os=128)])
def test_logits_refuses(bad):
    assert logits(**bad) == -2


def test_logits_refuses_a_vocabulary_that_no_cluster_holds():
    assert logits(vocab=409601, xs=409632, os=409632) == -6
    assert logits(rows=0) == 0
    assert _lib.lib().zcu_process_logits(P, 0, 64, P, 64, 1, 64, None, None) == -2


@pytest.mark.parametrize("call,good", [
    (reserve, dict(max_rows=4, max_pages=8, num_pages=16, page=16, batch=2, tokens=8)),
    (trim, dict(max_rows=4, max_pages=8, num_pages=16, page=16, batch=2)),
    (append, dict(in_dtype=0, tokens=2, kv_dtype=1, hkv=2, hd=128, page=16, pages=4)),
    (sparse, dict(kv_dtype=1, table_rows=2, batch=2, hq=8, hkv=2, hd=128, page=16, max_pages=64, pages=128, max_ctx=1024,
                  budget=8, sink=1, recent=1)),
    (lora, dict(w=1, rows=2, k=64, n=40, adapters=3, rank=8)), (logits, dict(dtype=0, rows=2, vocab=64))])
def test_numbers_beyond_32_bits_are_refused_not_cut(call, good):
    """ctypes keeps the low 32 bits of a larger number; 2^32 + 16 must not pass for a page size of 16."""
    for name, v in good.items():
        for off in (1 << 32, -(1 << 32), 1 << 63):
            with pytest.raises(C.ArgumentError, match="32 bits"):
                call(**{name: v + off})


def test_dispatch_takes_cuda_tensors_only():
    """The binding module is built and loaded with the library; whatever it is given here it declines (host tensors, other
    objects, wrong counts), and the Python checks behind it name the fault."""
    import torch

    from zeroplatform_b200 import ops
    from zeroplatform_b200._lib import ZcError
    _lib.lib()
    d = _lib.dispatch
    assert d is not None
    t, n = torch.zeros(2, 3), None
    for f, count in ((d.reserve_pages, 13), (d.trim_pages, 7), (d.append_kv, 7), (d.sparse_paged_attention, 15),
                     (d.lora_add, 8), (d.process_logits, 14)):
        for args in ([t] * count, [n] * count, [3] * count, ["x"] * count, [np.zeros(3)] * count, [t] * (count - 1), []):
            assert f(*args) is False
    for call in (lambda: ops.process_logits(t), lambda: ops.lora_add(t, t, t, t, t), lambda: ops.append_kv(t, t, t, t, t),
                 lambda: ops.trim_pages(t, t, t, t, t, 16), lambda: ops.process_logits(np.zeros((2, 3))),
                 lambda: ops.sparse_paged_attention(t, t, t, t, t, t, t, 4)):
        with pytest.raises(ZcError):
            call()
