"""CPU: what the step tables, the rotation with several axes and cross attention refuse, before any launch."""
import ctypes as C

import pytest
import torch

bf = torch.bfloat16


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_rope_axes_refusals():
    from kessie_amd import ops
    q, k, pos, inv = torch.zeros(5, 4, 64, dtype=bf), torch.zeros(5, 2, 64, dtype=bf), i32(3, 5), torch.ones(32)
    s = (12, 10, 10)
    for err, args in [
        (ValueError, (q[0], k, pos, inv, s)), (ValueError, (q, k[:4], pos, inv, s)), (TypeError, (q, k.float(), pos, inv, s)),
        (ValueError, (q, k, pos[:2], inv, s)), (TypeError, (q, k, pos.float(), inv, s)), (ValueError, (q, k, pos[:, :4], inv, s)),
        (ValueError, (q, k, pos, torch.ones(33), s)), (ValueError, (q, k, pos, inv.double(), s)),
        (ValueError, (q, k, pos, torch.ones(64)[::2], s)), (ValueError, (q.transpose(1, 2).contiguous().transpose(1, 2), k, pos, inv, s)),
        (ValueError, (q, k, i32(6, 5)[:5], inv, (8, 8, 8, 4, 4))), (ValueError, (q, k, pos, inv, ())),
        (ValueError, (q, k, pos, inv, s)),  # not on the GPU
    ]:
        with pytest.raises(err):
            ops.rope_axes(*args)
    with pytest.raises(ValueError):
        ops.rope_axes(q, None, pos, inv, s, k_out=k)
    pool, slots = torch.zeros(3, 16, 2, 2, 64, dtype=bf), torch.zeros(5, dtype=torch.int64)
    for err, args in [
        (ValueError, (q, q, q, pos, pool, slots, inv, s)), (TypeError, (q, k.half(), k.half(), pos, pool, slots, inv, s)),
        (ValueError, (q, k, k[:4], pos, pool, slots, inv, s)), (ValueError, (q, k, k, pos, pool, slots[:4], inv, s)),
        (ValueError, (q, k, k, pos, pool, slots.int(), inv, s)), (ValueError, (q, k, k, pos, pool, slots, inv, s)),
    ]:
        with pytest.raises(err):
            ops.rope_axes_cache_write(*args)
    with pytest.raises(ValueError):
        ops.rope_remap_axes(pool, pos, pos, inv, s, page_list=i32(0))
    with pytest.raises(TypeError):
        ops.rope_remap_axes(pool, pos, pos.long(), inv, s, page_list=i32(1))
    with pytest.raises(ValueError):
        ops.rope_remap_axes(torch.zeros(4, 2, 64, dtype=bf), pos, pos, inv, s)


def _rope_status(sections, interleaved=0, d=64, r=64, t=0, dtype=1):
    from kessie_amd import _lib
    lib = _lib.load()
    sec = (C.c_int32 * max(1, len(sections)))(*sections)
    st = lib.kessie_rope_axes(None, 0, 0, None, 0, 0, 4, None, 0, 0, None, 0, 0, 0, None, 0, 0, None, sec, len(sections), interleaved, 0, 0,
                              t, d, r, dtype, None)
    return st, _lib.last_error()[1]


def test_rope_axes_refusals_at_the_c_entry():
    from kessie_amd import _lib
    assert _rope_status((12, 10, 10))[0] == _lib.OK
    assert _rope_status((0, 0, 32, 0))[0] == _lib.OK
    for sections, kw in [((12, 10, 11), {}), ((33, -1), {}), ((8, 8, 8, 4, 4), {}), ((), {}), ((16, 16), dict(r=63)), ((64,), dict(r=128)),
                         ((32,), dict(t=-1)), ((12, 10, 10), dict(d=0))]:
        assert _rope_status(sections, **kw)[0] == _lib.ERR_INVALID, (sections, kw)
    assert _rope_status((256,), d=512, r=512)[0] == _lib.ERR_UNSUPPORTED
    # Dealt out in turn, an axis other than the first cannot get more than its share.
    st, msg = _rope_status((2, 20, 10), interleaved=1)
    assert st == _lib.ERR_INVALID and "interleaved" in msg
    assert _rope_status((12, 10, 10), interleaved=1)[0] == _lib.OK


def test_cross_attention_refusals():
    from kessie_amd import _lib, ops
    q, k = torch.zeros(6, 4, 64, dtype=bf), torch.zeros(9, 2, 64, dtype=bf)
    qs, ks, kl = i32(3), i32(2), i32(2)
    ok = dict(q=q, k=k, v=k, query_start_loc=qs, max_query_len=3, kv_start=ks, kv_lens=kl, max_kv_len=9)
    for err, change in [
        (ValueError, dict(q=q[0])), (ValueError, dict(k=k[:, :, :32], v=k[:, :, :32])), (TypeError, dict(k=k.half())),
        (ValueError, dict(v=k[:8])), (TypeError, dict(v=k.float())), (ValueError, dict(q=torch.zeros(6, 3, 64, dtype=bf))),
        (TypeError, dict(query_start_loc=qs.long())), (TypeError, dict(kv_lens=kl.long())), (ValueError, dict(query_start_loc=qs[:2])),
        (ValueError, dict(kv_start=i32(1))), (ValueError, dict(max_query_len=-1)), (ValueError, dict(max_kv_len=-1)),
        (TypeError, dict(key_mask=torch.zeros(9))), (ValueError, dict(key_mask=torch.zeros(8, dtype=torch.bool))),
        (ValueError, dict(key_mask=torch.zeros(18, dtype=torch.bool)[::2])), (ValueError, dict(out=q[:5])), (TypeError, dict(out=q.float())),
        (ValueError, {}),  # not on the GPU
    ]:
        with pytest.raises(err):
            ops.cross_attention(**{**ok, **change})
    lib = _lib.load()

    def status(b=1, mq=1, mk=1, tq=1, tkv=1, hq=4, hkv=2, d=64, dtype=1, ptr=None):
        return lib.kessie_cross_attention(ptr, 0, 0, ptr, 0, 0, ptr, 0, 0, ptr, ptr, ptr, None, ptr, 0, 0, b, mq, mk, tq, tkv, hq, hkv, d, 0.1,
                                          dtype, None, 0, None)
    assert status() == _lib.ERR_INVALID  # null pointers
    assert status(b=0) == status(mq=0) == status(tq=0) == _lib.OK
    for kw in (dict(b=-1), dict(mq=-1), dict(mk=-1), dict(tq=-1), dict(tkv=-1), dict(hq=3), dict(hkv=0), dict(d=0)):
        assert status(**kw) == _lib.ERR_INVALID, kw
    for kw in (dict(d=257), dict(dtype=7), dict(hq=65536, hkv=1)):
        assert status(**kw) == _lib.ERR_UNSUPPORTED, kw


def test_step_tables_refusals():
    from kessie_amd import _lib, ops
    from kessie_amd.kessie_attention import KeSSieAttentionMetadata as Meta
    ok = dict(block_table=i32(2, 8), computed_lens=i32(2), new_lens=i32(2), page_size=16, num_token_rows=4, free_pages=i32(5),
              free_count=i32(1))
    for err, change in [
        (TypeError, dict(block_table=i32(2, 8).long())), (ValueError, dict(block_table=i32(1, 8))), (ValueError, dict(block_table=i32(8, 2).t())),
        (ValueError, dict(new_lens=i32(3))), (ValueError, dict(page_size=0)), (ValueError, dict(num_token_rows=-1)),
        (ValueError, dict(free_count=None)), (TypeError, dict(free_count=i32(1).long())), (TypeError, dict(free_pages=i32(5).long())),
        (ValueError, dict(position_delta=i32(3))), (TypeError, dict(page_valid=i32(9))), (TypeError, dict(page_positions=i32(9).long())),
        (ValueError, dict(page_valid=torch.zeros(8, dtype=torch.int8), page_positions=i32(9))),
        (ValueError, dict(out=(i32(3), i32(2), i32(4).long(), i32(4), i32(2)))), (ValueError, dict(computed_lens=i32(4)[::2])),
        (ValueError, {}),  # not on the GPU
    ]:
        with pytest.raises(err):
            ops.step_tables(**{**ok, **change})
    lib = _lib.load()

    def status(stride=8, width=8, max_free=0, b=2, p=16, rows=4, pages=0):
        return lib.kessie_step_tables(None, stride, width, None, None, None, None, None, max_free, b, p, rows, None, None, None, None, None,
                                      None, None, pages, None)
    for kw in ({}, dict(p=0), dict(b=-1), dict(rows=-1), dict(max_free=-1), dict(pages=-1), dict(width=-1)):
        assert status(**kw) == _lib.ERR_INVALID, kw
    for bad in (dict(new_lens=[1]), dict(new_lens=[1, -1]), dict(computed_lens=[-1, 0]), dict(new_lens=[17, 17], num_free=1),
                dict(computed_lens=[120, 0], new_lens=[9, 0]), dict(num_token_rows=1), dict(page_size=0), dict(position_delta=[1])):
        with pytest.raises(ValueError):
            Meta.build(**{**dict(block_table=i32(2, 8), computed_lens=[0, 0], new_lens=[1, 1], page_size=16, free_pages=i32(5)), **bad})


def test_rows_of_an_output_that_overlap_are_refused():
    """At the C entries, before any launch (the addresses are the host's)."""
    from kessie_amd import _lib
    lib = _lib.load()
    buf = torch.zeros(64, dtype=torch.int64)
    p, sec = buf.data_ptr(), (C.c_int32 * 1)(32)

    def rope(ts, hs, t=5, hq=4):
        return lib.kessie_rope_axes(p, 0, 0, p, ts, hs, hq, None, 0, 0, None, 0, 0, 0, None, 0, 0, None, sec, 1, 0, 0, 0, t, 64, 64, 1, None)

    def remap(ts, hs, pages=None):
        return lib.kessie_rope_remap_axes(p, 1 << 20, ts, hs, pages, 1, p, 0, None, 0, 0, None, sec, 1, 0, 0, 5, 4, 64, 64, 16, 1, None)

    def cross(ts, hs):
        return lib.kessie_cross_attention(p, 0, 0, p, 0, 0, p, 0, 0, p, p, p, None, p, ts, hs, 1, 5, 1, 5, 1, 4, 2, 64, 0.1, 1, None, 0, None)
    for call in (rope, remap, lambda ts, hs: remap(ts, hs, p), cross):
        for ts, hs in ((0, 64), (64, 0), (64, 64), (255, 64), (256, 63), (63, 64 * 5)):
            assert call(ts, hs) != _lib.OK
            assert "overlap" in _lib.last_error()[1], (ts, hs)
        for ts, hs in ((256, 64), (64, 64 * 16), (1000, 65)) if call is not cross else ():  # (a null pointer ends those)
            assert call(ts, hs) != _lib.OK and "overlap" not in _lib.last_error()[1], (ts, hs)
    assert rope(0, 64, t=1) != _lib.OK and "overlap" not in _lib.last_error()[1]
    assert rope(64, 0, hq=1) != _lib.OK and "overlap" not in _lib.last_error()[1]


@pytest.mark.parametrize("scale", [float("inf"), float("nan"), -3e38])
def test_scales_past_fp32(scale):
    from kessie_amd import _lib
    st = _lib.load().kessie_cross_attention(None, 0, 0, None, 0, 0, None, 0, 0, None, None, None, None, None, 0, 0, 1, 1, 1, 1, 1, 4, 2, 64,
                                            scale, 1, None, 0, None)
    assert st == _lib.ERR_INVALID and "sm_scale" in _lib.last_error()[1]


def test_workspace_of_an_unknown_type():
    from kessie_amd import _lib
    assert _lib.load().kessie_cross_attention_workspace_bytes(1, 1, 1, 60000, 8, 1, 64, 60000, 7) == 0


def test_step_tables_that_lie_over_each_other_are_refused():
    """In place (last step's seq_lens as computed_lens and out at once), and outputs that share memory: before any launch."""
    from kessie_amd import _lib
    lib = _lib.load()
    names = ["table", "computed", "new", "delta", "free", "count", "starts", "lens", "slots", "pos", "taken", "valid", "where"]
    own = {n: torch.zeros(64, dtype=torch.int64) for n in names}

    def status(**share):
        a = {n: own[share.get(n, n)].data_ptr() for n in names}
        st = lib.kessie_step_tables(a["table"], 8, 8, a["computed"], a["new"], a["delta"], a["free"], a["count"], 5, 2, 16, 4, a["starts"],
                                    a["lens"], a["slots"], a["pos"], a["taken"], a["valid"], a["where"], 5, None)
        return st, _lib.last_error()[1]
    for out in ("table", "starts", "lens", "slots", "pos", "taken", "valid", "where"):
        for other in names:
            if other != out:
                st, msg = status(**{out: other})
                assert st == _lib.ERR_INVALID and "over" in msg, (out, other)
