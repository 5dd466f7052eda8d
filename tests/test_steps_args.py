"""Arguments that the calls around a step refuse before anything is launched:
pkv_plan_*, pkv_rope_*, pkv_attn_packed, and their Python forms. CPU only."""
import pytest
import torch

import pkv

L = pkv._lib
A = 1 << 12  # an aligned address that is never read


def packed(**kw):
    a = dict(q=A, q_row=512, q_head=64, k=A, k_row=128, k_head=64, v=A, v_row=128, v_head=64, gate=None, g_row=0, g_head=0,
             out=A, o_row=512, o_head=64, cu=A, seqs=2, T=10, Hq=8, Hkv=2, D=64, dtype=0, scale=0.125, stream=None)
    a.update(kw)
    return L.pkv_attn_packed(*a.values())


@pytest.mark.parametrize("kw", [
    dict(T=-1), dict(seqs=-1), dict(Hq=0), dict(Hkv=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(cu=None), dict(cu=A + 2),
    dict(q=A + 8), dict(v=A + 2), dict(gate=A + 4), dict(q_row=-512), dict(k_row=100), dict(v_head=4), dict(o_row=32),
    dict(o_head=32), dict(o_row=64, o_head=64), dict(o_row=128, o_head=256), dict(k_row=(1 << 24) + 8), dict(gate=A, g_row=3)])
def test_packed_refuses(kw):
    assert packed(**kw) == pkv.ERR_INVALID


@pytest.mark.parametrize("kw", [dict(D=96), dict(D=0), dict(dtype=2), dict(Hq=7), dict(T=1 << 30, Hq=16, Hkv=2, o_row=1024)])
def test_packed_does_not_serve(kw):
    assert packed(**kw) == pkv.ERR_UNSUPPORTED


def test_nothing_to_do():
    assert packed(T=0, q=None, cu=None) == pkv.OK and packed(seqs=0) == pkv.OK
    assert L.pkv_rope_spans(None, None, 0, 0, None, None) == pkv.OK
    assert L.pkv_rope_positions(None, None, 0, None, None, None, 0, 0, None, 0, None) == pkv.OK
    assert rope(T=0, q=None) == pkv.OK and rope(Hq=0, Hkv=0) == pkv.OK
    assert L.pkv_plan_truncate(None, None, None, 0, None, 4, 16, 8, None, None, None) == pkv.OK


def plan(**kw):
    a = dict(len=A, held=A, ntok=A, nrows=3, table=A, max_blocks=4, bs=16, pool=8, fl=A, fc=A, T=5, pos=A, slot=A, seq=A,
             cu=A, limits=A, len_out=A, held_out=A, fo=A, status=A, stream=None)
    a.update(kw)
    return L.pkv_plan_step(*a.values())


@pytest.mark.parametrize("kw", [
    dict(nrows=-1), dict(T=-1), dict(max_blocks=0), dict(bs=0), dict(pool=0), dict(len=None), dict(held=None),
    dict(ntok=None), dict(table=None), dict(pos=None), dict(slot=None), dict(seq=None), dict(cu=None), dict(limits=None),
    dict(len_out=None), dict(held_out=None), dict(status=None), dict(fl=None), dict(fc=None), dict(fl=None, fc=None),
    dict(len=A + 1), dict(fo=A + 2), dict(nrows=0, cu=None)])
def test_plan_refuses(kw):
    assert plan(**kw) == pkv.ERR_INVALID


@pytest.mark.parametrize("kw", [dict(T=1 << 29), dict(pool=1 << 28, bs=16), dict(max_blocks=1 << 28),
                                dict(pool=1 << 29, bs=1)])
def test_plan_does_not_serve(kw):
    assert plan(**kw) == pkv.ERR_UNSUPPORTED


def test_truncate_refuses():
    a = [A, A, A, 3, A, 4, 16, 8, A, A, None]
    for i in (0, 1, 2, 4, 8, 9):
        assert L.pkv_plan_truncate(*(a[:i] + [None] + a[i + 1:])) == pkv.ERR_INVALID
    assert L.pkv_plan_truncate(*(a[:3] + [-1] + a[4:])) == pkv.ERR_INVALID
    assert L.pkv_plan_truncate(*(a[:7] + [1 << 30] + a[8:])) == pkv.ERR_UNSUPPORTED


def rope(**kw):
    a = dict(q=A, q_row=512, q_head=64, k=A, k_row=128, k_head=64, qo=A, qo_row=512, qo_head=64, ko=A, ko_row=128,
             ko_head=64, Hq=8, Hkv=2, D=64, dtype=0, qn=None, kn=None, eps=1e-6, rope=A, stride=10, axes=A, inv=A, rot=64,
             adj=0, T=10, stream=None)
    a.update(kw)
    return L.pkv_rope_rows(*a.values())


@pytest.mark.parametrize("kw", [
    dict(T=-1), dict(Hq=-1), dict(Hkv=-1), dict(rot=-16), dict(stride=9), dict(q=None), dict(k=None), dict(qo=None),
    dict(ko=None), dict(rope=None), dict(axes=None), dict(inv=None), dict(q=A + 2), dict(ko=A + 8), dict(q_row=4),
    dict(ko_head=-8), dict(qo_row=32), dict(ko_head=56), dict(qn=A + 2),
    dict(qo_row=448), dict(ko_row=64)])
def test_rope_rows_refuses(kw):
    assert rope(**kw) == pkv.ERR_INVALID


@pytest.mark.parametrize("kw", [dict(D=80), dict(dtype=5), dict(rot=72), dict(rot=128), dict(rot=8)])
def test_rope_rows_does_not_serve(kw):
    assert rope(**kw) == pkv.ERR_UNSUPPORTED


def test_positions_refuse():
    P, S = L.pkv_rope_positions, L.pkv_rope_spans
    assert S(A, A, -1, 3, A, None) == S(A, A, 2, -1, A, None) == S(None, A, 2, 3, A, None) == pkv.ERR_INVALID
    assert S(A, None, 2, 3, A, None) == S(A, A, 2, 3, None, None) == S(A, A + 1, 2, 3, A, None) == pkv.ERR_INVALID
    ok = [A, A, 4, A, A, A, 2, 3, A, 4, None]
    for i in (0, 1, 3, 4, 5, 8):
        assert P(*(ok[:i] + [None] + ok[i + 1:])) == pkv.ERR_INVALID
    assert P(*(ok[:9] + [3, None])) == pkv.ERR_INVALID


def raises(status, f, *a, **k):
    with pytest.raises(pkv.PkvError) as e:
        f(*a, **k)
    assert e.value.status == status, e.value
    return str(e.value)


def test_python_forms_check_their_tensors():
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    I, U = pkv.ERR_INVALID, pkv.ERR_UNSUPPORTED
    q, k, cu = bf(6, 4, 64), bf(6, 2, 64), i32(3)
    f = pkv.attn_packed
    assert "not on a GPU" in raises(I, f, q, k, k, cu, q, 0.1)
    raises(U, f, q.float(), k.float(), k.float(), cu, q.float(), 0.1)
    raises(I, f, q, k.half(), k, cu, q, 0.1)
    raises(I, f, q, k, k[:5], cu, q, 0.1)
    raises(I, f, q, k, bf(6, 2, 128), cu, q, 0.1)
    raises(I, f, q, k, k, cu.long(), q, 0.1)
    raises(I, f, q, k, k, i32(0), q, 0.1)
    raises(I, f, q, k, k, cu, bf(6, 3, 64), 0.1)
    raises(I, f, q, k, k, cu, bf(6, 64, 4).transpose(1, 2), 0.1)
    raises(I, f, q, k, k, cu, q, 0.1, gate=bf(6, 2, 64))
    raises(I, f, q[0], k, k, cu, q, 0.1)
    rope, axes, inv = i32(3, 6), i32(16), torch.zeros(16)
    f = pkv.rope_rows
    assert "not on a GPU" in raises(I, f, q, k, rope, axes, inv, q, k)
    raises(I, f, q, k, i32(3, 5), axes, inv, q, k)
    raises(I, f, q, k, i32(2, 6), axes, inv, q, k)
    raises(I, f, q, k, rope, axes, inv[:8], q, k)
    raises(I, f, q, k, rope, axes, inv.double(), q, k)
    raises(I, f, q, k, rope, axes, inv, q, k, q_norm=torch.zeros(32))
    raises(I, f, q, k, rope, axes, inv, q[:5], k)
    spans, scu, base = i32(4, 5), i32(3), i32(4)
    assert "not on a GPU" in raises(I, pkv.rope_spans, scu, spans, base)
    raises(I, pkv.rope_spans, scu, i32(4, 4), base)
    raises(I, pkv.rope_spans, i32(0), spans, base)
    raises(I, pkv.rope_spans, scu, spans, i32(3))
    pos = i32(6)
    assert "not on a GPU" in raises(I, pkv.rope_positions, pos, pos, scu, spans, base, rope)
    raises(I, pkv.rope_positions, pos, i32(5), scu, spans, base, rope)
    raises(I, pkv.rope_positions, pos, pos, scu, spans, base, i32(3, 5))
    raises(I, pkv.rope_positions, pos, pos, scu, spans, i32(2), rope)
    r3, table, t = i32(3), i32(3, 4), i32(9)
    step = lambda **kw: pkv.plan_step(**{**dict(len=r3, held=r3, ntok=r3, block_table=table, block_size=16, num_blocks=8,
                                                pos=t, slot_map=t, tok_seq=t, cu=i32(4), limits=r3, len_out=r3, held_out=r3,
                                                status=r3, free_list=i32(8), free_count=i32(1)), **kw})
    assert "not on a GPU" in raises(I, step)
    for kw in (dict(len=i32(2)), dict(cu=r3), dict(block_table=i32(12)), dict(slot_map=i32(8)), dict(free_list=i32(7)),
               dict(free_count=i32(2)), dict(status=r3.long()), dict(block_table=i32(4, 3).t())):
        raises(I, lambda: step(**kw))
    cut = lambda **kw: pkv.plan_truncate(**{**dict(new_len=r3, len=r3, held=r3, block_table=table, block_size=16,
                                                   num_blocks=8, free_list=i32(8), free_count=i32(1)), **kw})
    assert "not on a GPU" in raises(I, cut)
    for kw in (dict(new_len=i32(2)), dict(free_list=i32(7)), dict(free_count=r3), dict(block_table=i32(12))):
        raises(I, lambda: cut(**kw))
