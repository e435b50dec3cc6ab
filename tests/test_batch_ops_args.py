"""Arguments that the batched-decoding operators refuse, checked on the host before anything is launched (these run
without a GPU), and the rotation plans' limits."""
import ctypes as C
import math

import numpy as np
import pytest

import quillm_b200 as qb

EINVAL = -1
BUF = np.zeros(1 << 16, np.uint8)
A = (BUF.ctypes.data + 255) // 256 * 256  # an aligned address that is never read


def refused(rc, word=""):
    assert rc == EINVAL, rc
    assert word in qb.last_error(), qb.last_error()


def cache(**k):
    d = dict(k=A, v=A, dtype=qb.QMC_F16, n_layers=2, n_pages=8, page_size=4, n_kv_heads=2, head_dim=64)
    d.update(k)
    return qb.QmcPagedCache(*(d[f[0]] for f in qb.QmcPagedCache._fields_))


@pytest.mark.parametrize("bad", [
    dict(head_dim=127), dict(head_dim=0), dict(head_dim=258), dict(rot_dim=130), dict(rot_dim=3), dict(rot_dim=0),
    dict(layout=2), dict(layout=-1), dict(scaling=4), dict(scaling=-1), dict(theta=0.0), dict(theta=math.nan),
    dict(theta=math.inf), dict(scaling=1, factor=0.0), dict(scaling=1, factor=math.nan),
    dict(scaling=2, low=4.0, high=4.0), dict(scaling=2, low=0.0), dict(scaling=2, orig_ctx=0),
    dict(scaling=3, low=0.0), dict(scaling=3, low=5.0, high=4.0), dict(scaling=3, theta=1.0), dict(scaling=3, orig_ctx=-1)])
def test_rope_plan_refusals(bad):
    d = dict(head_dim=128, rot_dim=128, layout=0, scaling=0, theta=1e4, factor=2.0, low=1.0, high=4.0, orig_ctx=4096)
    d.update(bad)
    cfg = qb.QmcRopeConfig(*(d[f[0]] for f in qb.QmcRopeConfig._fields_))
    h = C.c_void_p(1)
    refused(qb.cuda().qmc_rope_plan_create(C.byref(cfg), C.byref(h)), "rope_plan_create")
    assert not h.value
    refused(qb.cuda().qmc_rope_plan_create(None, C.byref(h)))
    assert qb.cuda().qmc_rope_plan_free(None) == 0


def qk(plan, **k):
    d = dict(dtype=0, q=A, ldq=256, qo=A, ldqo=256, heads=2, k=A, ldk=128, ko=A, ldko=128, kv=1, qw=None, kw=None, eps=1e-5,
             pos=A, rows=3)
    d.update(k)
    return qb.cuda().qmc_qk_norm_rope(plan, d["dtype"], d["q"], d["ldq"], d["qo"], d["ldqo"], d["heads"], d["k"], d["ldk"],
                                      d["ko"], d["ldko"], d["kv"], d["qw"], d["kw"], d["eps"], d["pos"], d["rows"], None)


@pytest.mark.parametrize("bad", [
    dict(dtype=2), dict(dtype=5), dict(q=None), dict(qo=None), dict(k=None), dict(ko=None), dict(ldq=255), dict(ldqo=0),
    dict(ldk=127), dict(ldko=-128), dict(heads=-1), dict(kv=-1), dict(rows=-1), dict(rows=1 << 31), dict(eps=-1.0),
    dict(eps=math.nan), dict(pos=None), dict(q=A + 2), dict(dtype=1, k=A + 1)])
def test_qk_norm_rope_refusals(bad):
    p = qb.RopePlan(128)
    refused(qk(p.h, **bad), "qk_norm_rope")
    refused(qk(None), "plan")
    assert qk(p.h, rows=0) == 0 and qk(p.h, heads=0, kv=0, q=None, k=None) == 0  # nothing to do


def append(plan, c, **k):
    d = dict(layer=1, dtype=1, q=A, ldq=256, qo=A, ldqo=256, heads=4, k=A, ldk=128, v=A, ldv=128, qw=None, kw=None, eps=1e-5,
             seq=A, pos=A, table=A, n_seq=3, ld=4, rows=3)
    d.update(k)
    return qb.cuda().qmc_kv_append_paged(plan, C.addressof(c) if c else None, d["layer"], d["dtype"], d["q"], d["ldq"],
                                         d["qo"], d["ldqo"], d["heads"], d["k"], d["ldk"], d["v"], d["ldv"], d["qw"], d["kw"],
                                         d["eps"], d["seq"], d["pos"], d["table"], d["n_seq"], d["ld"], d["rows"], None)


BAD_CACHE = [dict(k=None), dict(v=None), dict(dtype=2), dict(dtype=9), dict(n_layers=0), dict(n_pages=0), dict(page_size=0),
             dict(n_kv_heads=0), dict(head_dim=0), dict(k=A + 1), dict(n_layers=1 << 30, n_pages=1 << 30, page_size=1 << 20)]


@pytest.mark.parametrize("bad", BAD_CACHE + [dict(head_dim=63), dict(head_dim=258)])
def test_append_refuses_caches(bad):
    refused(append(None, cache(**bad)), "kv_append_paged")
    refused(append(None, None), "null cache")


@pytest.mark.parametrize("bad", [
    dict(layer=2), dict(layer=-1), dict(dtype=3), dict(q=None), dict(heads=0), dict(heads=-1), dict(k=None), dict(v=None),
    dict(ldq=255), dict(ldk=127), dict(ldv=127), dict(rows=-1), dict(rows=1 << 31), dict(ld=0), dict(n_seq=-1),
    dict(pos=None), dict(table=None), dict(seq=None, rows=4), dict(eps=-1e-5)])
def test_append_refusals(bad):
    refused(append(None, cache(), **bad), "kv_append_paged")
    p = qb.RopePlan(128)
    refused(append(p.h, cache()), "plan")  # a plan of another head size
    assert append(None, cache(), rows=0) == 0


def attn(c, **k):
    d = dict(layer=0, dtype=1, q=A, ldq=256, out=A, ldo=256, heads=4, n_seq=3, scale=0.125, pages=A, prefix=9, table=A, ld=4,
             lens=A, ws=A, bytes=1 << 40)
    d.update(k)
    return qb.cuda().qmc_attn_prefix(C.addressof(c) if c else None, d["layer"], d["dtype"], d["q"], d["ldq"], d["out"],
                                     d["ldo"], d["heads"], d["n_seq"], d["scale"], d["pages"], d["prefix"], d["table"],
                                     d["ld"], d["lens"], d["ws"], d["bytes"], None)


@pytest.mark.parametrize("bad", BAD_CACHE + [dict(head_dim=257), dict(dtype=qb.QMC_F32), dict(dtype=qb.QMC_BF16)])
def test_attn_refuses_caches(bad):
    c, n = cache(**bad), C.c_size_t(7)
    refused(attn(c), "attn_prefix")
    refused(qb.cuda().qmc_attn_prefix_workspace(1, C.addressof(c), 3, 4, 9, 4, C.byref(n)), "attn_prefix_workspace")
    assert n.value == 0


@pytest.mark.parametrize("bad", [
    dict(layer=2), dict(layer=-1), dict(dtype=2), dict(dtype=4), dict(q=None), dict(out=None), dict(ldq=255), dict(ldo=255),
    dict(heads=3), dict(heads=0), dict(n_seq=-1), dict(scale=math.nan), dict(scale=math.inf), dict(scale=-0.5), dict(pages=None),
    dict(prefix=-1), dict(prefix=17), dict(table=None), dict(ld=0), dict(ld=1 << 30), dict(lens=None), dict(ws=None), dict(q=A + 1)])
def test_attn_refusals(bad):
    refused(attn(cache(), **bad), "attn_prefix")
    assert attn(cache(), n_seq=0) == 0
    c = cache()
    refused(qb.cuda().qmc_attn_prefix_workspace(1, C.addressof(c), 3, 4, 9, 4, None))


def test_attn_refuses_positions_near_the_end_of_int():
    c, n = cache(page_size=1, n_pages=1 << 20), C.c_size_t(0)
    refused(qb.cuda().qmc_attn_prefix_workspace(1, C.addressof(c), 1, 4, 0, (1 << 31) - 1, C.byref(n)), "positions")
    assert n.value == 0


def select(**k):
    d = dict(dtype=0, logits=A, ld=100, prompts=2, beams=3, vocab=100, scores=A, finished=A, eos=2, n_out=6, parents=A, tokens=A,
             out=A, ws=A, bytes=1 << 30)
    d.update(k)
    return qb.cuda().qmc_beam_select(d["dtype"], d["logits"], d["ld"], d["prompts"], d["beams"], d["vocab"], d["scores"],
                                     d["finished"], d["eos"], d["n_out"], d["parents"], d["tokens"], d["out"], d["ws"],
                                     d["bytes"], None)


@pytest.mark.parametrize("bad", [
    dict(dtype=2), dict(ld=99), dict(prompts=-1), dict(beams=0), dict(beams=65), dict(vocab=0), dict(n_out=0), dict(n_out=65),
    dict(vocab=1, beams=3, n_out=4, eos=0), dict(eos=-1), dict(eos=100), dict(logits=None), dict(scores=None),
    dict(parents=None), dict(tokens=None), dict(out=None), dict(ws=None), dict(bytes=100), dict(logits=A + 2),
    dict(prompts=30000), dict(beams=64, vocab=1 << 20, ld=1 << 20)])
def test_beam_select_refusals(bad):
    refused(select(**bad), "beam_select")
    assert select(prompts=0) == 0
    n = C.c_size_t(0)
    refused(qb.cuda().qmc_beam_workspace(2, 3, 100, 6, None))
    refused(qb.cuda().qmc_beam_workspace(2, 65, 100, 6, C.byref(n)))
    assert qb.beam_workspace(2, 3, 100, 6) > 0


def reorder(c, **k):
    d = dict(prompts=2, beams=3, parents=A, ldp=3, lens=A, table=A, out=A + 64, ld=4)
    d.update(k)
    return qb.cuda().qmc_beam_reorder(C.addressof(c) if c else None, d["prompts"], d["beams"], d["parents"], d["ldp"],
                                      d["lens"], d["table"], d["out"], d["ld"], None)


@pytest.mark.parametrize("bad", [
    dict(prompts=-1), dict(beams=0), dict(beams=65, ldp=65), dict(ldp=2), dict(ld=0), dict(parents=None), dict(lens=None),
    dict(table=None), dict(out=None), dict(out=A)])
def test_beam_reorder_refusals(bad):
    refused(reorder(cache(), **bad), "beam_reorder")
    assert reorder(cache(), prompts=0) == 0
    for c in BAD_CACHE:
        refused(reorder(cache(**c)), "beam_reorder")


def test_sizes_counted_in_32_bits_are_bounded():
    many = (1 << 20) + 1
    c = cache(n_layers=1, n_pages=1, page_size=1, n_kv_heads=1 << 24, head_dim=32)
    refused(reorder(c), "too large")
    refused(attn(c), "too large")
    p = qb.RopePlan(2)
    refused(qb.cuda().qmc_qk_norm_rope(p.h, 0, A, 1 << 30, A, 1 << 30, many, None, 0, None, 0, 0, None, None, 0.0, A, 1, None), "too many")
    refused(qb.cuda().qmc_qk_norm_rope(p.h, 0, None, 0, None, 0, 0, A, 1 << 30, A, 1 << 30, 2**31 - 1, None, None, 0.0, A, 1, None))


def test_beam_reorder_refuses_pages_of_too_many_pieces():
    c = cache(n_layers=1 << 20, n_pages=1, page_size=1 << 20, n_kv_heads=1, head_dim=256)
    refused(reorder(c, beams=64, ldp=64), "too many")


def test_attn_workspace_of_no_sequences():
    c, n = cache(), C.c_size_t(7)
    for prefix in (0, 9, 16):
        assert qb.cuda().qmc_attn_prefix_workspace(1, C.addressof(c), 0, 4, prefix, 4, C.byref(n)) == 0
        assert n.value == 0


@pytest.mark.parametrize("bad", [dict(theta=5e-324), dict(scaling=1, factor=1e-320), dict(scaling=2, factor=1e-320), dict(scaling=3, factor=1e-320)])
def test_rope_plan_refuses_frequencies_past_the_largest_number(bad):
    d = dict(head_dim=128, rot_dim=128, layout=0, scaling=0, theta=1e4, factor=2.0, low=1.0, high=4.0, orig_ctx=4096)
    d.update(bad)
    cfg = qb.QmcRopeConfig(*(d[f[0]] for f in qb.QmcRopeConfig._fields_))
    h = C.c_void_p(1)
    refused(qb.cuda().qmc_rope_plan_create(C.byref(cfg), C.byref(h)), "frequency")
    assert not h.value


@pytest.mark.parametrize("name", ["pos", "qw", "kw"])
def test_qk_norm_rope_refuses_misaligned(name):
    p = qb.RopePlan(128)
    refused(qk(p.h, **{name: A + 2}), "misaligned")


@pytest.mark.parametrize("name", ["pos", "seq", "table", "qw", "kw"])
def test_append_refuses_misaligned(name):
    refused(append(None, cache(), **{name: A + 2}), "misaligned")


@pytest.mark.parametrize("name", ["pages", "table", "lens"])
def test_attn_refuses_misaligned(name):
    refused(attn(cache(), **{name: A + 1}), "misaligned")


@pytest.mark.parametrize("name", ["scores", "parents", "tokens", "out"])
def test_beam_select_refuses_misaligned(name):
    refused(select(**{name: A + 2}), "misaligned")


@pytest.mark.parametrize("name", ["parents", "lens", "table", "out"])
def test_beam_reorder_refuses_misaligned(name):
    refused(reorder(cache(), **{name: A + 65}), "misaligned")


def test_attn_refuses_a_scale_past_the_largest_exponent():
    refused(attn(cache(), scale=3e38), "scale")  # as an exponent of two, times log2(e), it is infinite
