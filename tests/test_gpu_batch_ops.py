"""The batched-decoding operators against plain implementations in 64 bits: key / query norms with the rotation, the
append to a paged cache, attention over a shared prefix, beam selection and the reordering of states, and a
beam search that uses them together.

Tolerances, with u = 2^-24 and e the output type's half step (2^-24, 2^-11, 2^-8):
  rotation: cos and sin are off by the float angle (pi u), sincospi (2 steps, 4 u) and their rounding (u), 9 u in all; two
    products and a sum add 3 u of |a| + |b|, a norm 16 u (the sum of squares by lane and tree: 14 roundings, halved
    by the root, the root, the quotient and two products).  Together under 2^-19 m (|a| + |b|), plus e |out|.
  attention: a score is off by d_s <= (hd + 8) u scale sum_d |q k| (2^-21 more where a float query is split in
    two halves); a weight by 2 d_s + 2^-20 and, where weights are rounded to 16 bits for the product, e_P of that type;
    the sum of weights likewise (where a third of the exponentials come from a polynomial, 2^-13.7 for bf16 and 2^-18.5 for fp16
    join them, far below e_P, which the sum does not have).  o is off by at most 2 (2 d_s + 2^-20 + e_P) sum_p w_p |v_p|, plus e |o|.
  beam scores: exp is off by 2 u (1 + |x - m|) <= 2^-19 for the terms that count, the chunk's float sum by 21 u: 2^-18 in
    the log-sum-exp, plus u |score|."""
import math

import numpy as np
import pytest
import torch

import quillm_b200 as qb

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": qb.QMC_F32, "f16": qb.QMC_F16, "bf16": qb.QMC_BF16}
E = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}
TINY = {"f32": 2.0**-149, "f16": 2.0**-25, "bf16": 2.0**-133}
U = 2.0**-24


def lib():
    return qb.cuda()


def f64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def rand(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(DT[dtype])


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def clean():
    torch.cuda.synchronize()
    rc = lib().qmc_check_device_error()
    assert rc == 0, qb.last_error()


def flagged():
    """the device error word was set, and is clear now"""
    torch.cuda.synchronize()
    assert lib().qmc_check_device_error() == -1 and "out of range" in qb.last_error()
    assert lib().qmc_check_device_error() == 0


def strided(g, rows, n, dtype, pad, shift):
    """rows of n elements n + pad apart, the first `shift` elements into an allocation filled with 77"""
    base = torch.full((rows * (n + pad) + shift + 8,), 77.0, dtype=DT[dtype], device="cuda")
    view = base[shift:shift + rows * (n + pad)].view(rows, n + pad)[:, :n]
    view.copy_(rand(g, (rows, n), dtype))
    return base, view


# ------------------------------------------------------------------ rotation, 64 bits
def frequencies(rot, scaling, theta, factor, low, high, orig):
    f, m = [], 1.0
    if scaling == qb.QMC_ROPE_YARN:
        d = lambda t: rot * math.log(orig / (t * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        lo, hi = min(max(math.floor(d(high)), 0), rot - 1), min(max(math.ceil(d(low)), 0), rot - 1)
        m = 0.1 * math.log(factor) + 1
    for i in range(rot // 2):
        v = theta ** (-2.0 * i / rot)
        if scaling == qb.QMC_ROPE_LINEAR:
            v /= factor
        elif scaling == qb.QMC_ROPE_BANDS:
            t = orig * v / (2 * math.pi)
            s = min(max((t - low) / (high - low), 0.0), 1.0)
            v = v * s + v / factor * (1 - s)
        elif scaling == qb.QMC_ROPE_YARN:
            r = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            v = v / factor * r + v * (1 - r)
        f.append(v)
    return np.array(f), m


SCALED = {0: dict(), 1: dict(factor=4.0), 2: dict(factor=8.0, low=1.0, high=4.0, orig_ctx=4096),
          3: dict(factor=16.0, low=1.0, high=32.0, orig_ctx=4096)}


def ref_heads(x, pos, w, eps, rot, layout, scaling, theta=10000.0):
    """x [rows, heads, hd] in 64 bits -> (y, |a| + |b| of each element's pair)"""
    k = dict(factor=1.0, low=0.0, high=0.0, orig_ctx=0)
    k.update(SCALED[scaling])
    f, m = frequencies(rot, scaling, theta, k["factor"], k["low"], k["high"], k["orig_ctx"]) if rot else (np.zeros(0), 1.0)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    y, mag = x.copy(), np.abs(x)
    ang = pos.astype(np.float64)[:, None, None] * f
    c, s = m * np.cos(ang), m * np.sin(ang)
    ia = np.arange(rot // 2) * (2 if layout == 0 else 1)
    ib = ia + (1 if layout == 0 else rot // 2)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    mag[..., ia] = mag[..., ib] = m * (np.abs(a) + np.abs(b))
    return y, mag


def close(got, want, tol):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5].tolist(), got[bad][:5], want[bad][:5], np.broadcast_to(tol, got.shape)[bad][:5])


def check_heads(got, x, pos, w, eps, rot, layout, scaling, dtype):
    want, mag = ref_heads(x, pos, w, eps, rot, layout, scaling)
    close(got, want, 2.0**-19 * mag + E[dtype] * np.abs(want) + TINY[dtype])


def plan(hd, rot, layout, scaling):
    return qb.RopePlan(hd, rot, layout, 10000.0, scaling, **SCALED[scaling])


ROPE = [  # rows, heads, kv, hd, rot, pad, shift
    (1, 32, 32, 128, 128, 0, 0), (5, 64, 8, 128, 128, 0, 0), (333, 6, 6, 48, 20, 0, 0), (9, 7, 7, 80, 40, 8, 8),
    (17, 3, 1, 36, 12, 1, 3), (4, 12, 4, 256, 256, 0, 0), (3, 5, 2, 256, 130, 1, 1), (2, 2, 1, 2, 2, 0, 0), (40, 16, 1, 64, 32, 2, 2),
    (2, 300, 1, 6, 4, 0, 0), (1000, 8, 2, 96, 96, 16, 0)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", range(len(ROPE)))
def test_qk_norm_rope(cuda_dev, case, dtype):
    rows, heads, kv, hd, rot, pad, shift = ROPE[case]
    g = gen(case)
    pos = torch.randint(0, 100000, (rows,), generator=g, device="cuda", dtype=torch.int32)
    pos[0] = [0, 2**31 - 1, -(2**31), 1, -7][case % 5]
    qw, kw = (1 + 0.2 * torch.randn(hd, generator=g, device="cuda") for _ in range(2))
    for i, (layout, scaling, norm) in enumerate([(0, 0, False), (1, 2, True), (0, 3, True), (1, 1, False)]):
        _, q = strided(g, rows, heads * hd, dtype, pad, shift)
        _, k = strided(g, rows, kv * hd, dtype, pad, shift)
        qbase, qo = strided(g, rows, heads * hd, dtype, pad, shift)
        ko = torch.zeros(rows, kv * hd, dtype=DT[dtype], device="cuda")
        before = qbase.clone()
        p = plan(hd, rot, layout, scaling)
        qb.check(lib().qmc_qk_norm_rope(p.h, CODE[dtype], q.data_ptr(), heads * hd + pad, qo.data_ptr(), heads * hd + pad, heads,
                                        k.data_ptr(), kv * hd + pad, ko.data_ptr(), kv * hd, kv,
                                        qw.data_ptr() if norm else None, kw.data_ptr() if norm else None, 1e-5,
                                        pos.data_ptr(), rows, qb.torch_stream()))
        clean()
        pn = pos.cpu().numpy()
        check_heads(f64(qo).reshape(rows, heads, hd), f64(q).reshape(rows, heads, hd), pn, f64(qw) if norm else None, 1e-5, rot,
                    layout, scaling, dtype)
        check_heads(f64(ko).reshape(rows, kv, hd), f64(k).reshape(rows, kv, hd), pn, f64(kw) if norm else None, 1e-5, rot, layout,
                    scaling, dtype)
        qo.zero_()  # what lies between and around the rows is untouched
        keep = before.clone()
        keep[shift:shift + rows * (heads * hd + pad)].view(rows, heads * hd + pad)[:, :heads * hd].zero_()
        assert torch.equal(keep, qbase)


def test_rope_in_place_one_sided_and_like_qmc_rope(cuda_dev):
    g = gen(3)
    p = plan(128, 128, 0, 0)
    x = rand(g, (1, 32 * 128), "f32")
    a, b = x.clone(), x.clone()
    pos = torch.tensor([731], dtype=torch.int32, device="cuda")
    st = qb.torch_stream()
    # in place, queries only, keys only
    qb.check(lib().qmc_qk_norm_rope(p.h, 0, a.data_ptr(), 4096, a.data_ptr(), 4096, 32, None, 0, None, 0, 0, None, None, 0.0,
                                    pos.data_ptr(), 1, st))
    qb.check(lib().qmc_qk_norm_rope(p.h, 0, None, 0, None, 0, 0, b.data_ptr(), 4096, b.data_ptr(), 4096, 32, None, None, 0.0,
                                    pos.data_ptr(), 1, st))
    c = x.clone()
    qb.check(lib().qmc_rope(c.data_ptr(), 32, 128, 731, 10000.0, st))
    clean()
    assert torch.equal(a, b)
    mag = ref_heads(f64(x).reshape(1, 32, 128), np.array([731]), None, 0.0, 128, 0, 0)[1].reshape(1, -1)
    close(f64(a), f64(c), 2.0**-19 * mag)


# ------------------------------------------------------------------ append
def pools(g, layers, pages, page, kv, hd, dtype, fill=None):
    shape = (layers, pages, page, kv, hd)
    k, v = ((rand(g, shape, dtype) if fill is None else torch.full(shape, fill, dtype=DT[dtype], device="cuda")) for _ in range(2))
    return k, v, qb.PagedCache(k, v, CODE[dtype], *shape)


def do_append(p, c, layer, dtype, q, qo, heads, k, v, qw, kw, seq, pos, table, rows):
    dp = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    ld = lambda t: 0 if t is None else t.stride(0)  # noqa: E731
    qb.check(lib().qmc_kv_append_paged(p.h if p else None, c.ref, layer, CODE[dtype], dp(q), ld(q), dp(qo), ld(qo), heads, dp(k),
                                       ld(k), dp(v), ld(v), dp(qw), dp(kw), 1e-5, dp(seq), dp(pos), dp(table),
                                       table.shape[0], table.shape[1], rows, qb.torch_stream()))


APPEND = [  # seqs, each, heads, kv, hd, rot, page, pad, shift
    (8, 1, 32, 32, 128, 128, 16, 0, 0), (3, 50, 64, 8, 128, 64, 16, 0, 0), (7, 61, 6, 6, 48, 48, 12, 0, 0), (4, 9, 4, 2, 36, 20, 1, 1, 1),
    (2, 33, 3, 3, 256, 256, 7, 3, 5), (5, 5, 2, 1, 10, 2, 64, 2, 2)]


@pytest.mark.parametrize("dtype,cdt", [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("f16", "f32"),
                                       ("bf16", "bf16"), ("bf16", "f16")])
@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append(cuda_dev, case, dtype, cdt):
    seqs, each, heads, kv, hd, rot, page, pad, shift = APPEND[case]
    g, layout, norm = gen(100 + case), case % 2, case % 3 > 0
    width = -(-(each + 2 * seqs + 3) // page)
    n_pages = seqs * width + 3
    table = torch.randperm(n_pages, generator=g, device="cuda")[:seqs * width].to(torch.int32).view(seqs, width)
    n = (heads + 2 * kv) * hd
    _, x = strided(g, seqs * each + 2, n, dtype, pad, shift)
    q, k, v = x[:, :heads * hd], x[:, heads * hd:(heads + kv) * hd], x[:, (heads + kv) * hd:]
    seq = torch.arange(seqs, dtype=torch.int32, device="cuda").repeat_interleave(each)
    pos = (2 * torch.arange(seqs, device="cuda")[:, None] + 3 + torch.arange(each, device="cuda")).reshape(-1).to(torch.int32)
    # two rows of padding: a negative sequence, a negative position
    seq = torch.cat([seq, torch.tensor([-1, 0], dtype=torch.int32, device="cuda")])
    pos = torch.cat([pos, torch.tensor([0, -1], dtype=torch.int32, device="cuda")])
    order = torch.randperm(seqs * each + 2, generator=g, device="cuda")
    seq, pos = seq[order].contiguous(), pos[order].contiguous()
    qw, kw = (1 + 0.2 * torch.randn(hd, generator=g, device="cuda") for _ in range(2)) if norm else (None, None)
    kp, vp, c = pools(g, 2, n_pages, page, kv, hd, cdt, fill=55.0)
    qo = torch.full((x.shape[0], heads * hd), 33.0, dtype=DT[dtype], device="cuda")
    do_append(plan(hd, rot, layout, 2), c, 1, dtype, q, qo, heads, k, v, qw, kw, seq, pos, table, x.shape[0])
    clean()
    sn, pn = seq.cpu().numpy(), pos.cpu().numpy()
    ok = (sn >= 0) & (pn >= 0)
    assert (f64(qo)[~ok] == 33.0).all()
    w = lambda t: None if t is None else f64(t)  # noqa: E731
    check_heads(f64(qo)[ok].reshape(-1, heads, hd), f64(q)[ok].reshape(-1, heads, hd), pn[ok], w(qw), 1e-5, rot, layout, 2, dtype)
    slot = table.cpu().numpy()[sn[ok], pn[ok] // page].astype(np.int64) * page + pn[ok] % page
    gk, gv = (f64(t)[1].reshape(-1, kv, hd) for t in (kp, vp))
    check_heads(gk[slot], f64(k)[ok].reshape(-1, kv, hd), pn[ok], w(kw), 1e-5, rot, layout, 2, cdt)
    want = v.to(torch.float32).to(DT[cdt])  # values: one rounding to the cache's type
    assert np.array_equal(gv[slot], f64(want)[ok].reshape(-1, kv, hd))
    rest = np.setdiff1d(np.arange(n_pages * page), slot)
    assert (gk[rest] == 55.0).all() and (gv[rest] == 55.0).all() and (kp[0] == 55.0).all() and (vp[0] == 55.0).all()


def test_append_without_plan_or_queries_and_bad_slots(cuda_dev):
    g = gen(9)
    kp, vp, c = pools(g, 1, 6, 4, 2, 64, "f16", fill=55.0)
    k, v = (rand(g, (4, 128), "f16") for _ in range(2))
    table = torch.tensor([[0, 1], [2, 3], [4, 6], [-1, 5]], dtype=torch.int32, device="cuda")
    pos = torch.tensor([3, 4, 1, 5], dtype=torch.int32, device="cuda")
    do_append(None, c, 0, "f16", None, None, 0, k, v, None, None, None, pos, table, 4)  # sequence r is row r
    clean()
    for r, slot in enumerate([3, 3 * 4, 4 * 4 + 1, 5 * 4 + 1]):
        assert torch.equal(kp.view(-1, 128)[slot], k[r]) and torch.equal(vp.view(-1, 128)[slot], v[r])
    assert (kp == 55.0).sum() == 6 * 4 * 128 - 4 * 128
    # a page outside the pool on either side, a position past the table, a sequence past it: nothing is written
    before = kp.clone()
    seq = torch.tensor([2, 3, 0, 4], dtype=torch.int32, device="cuda")
    pos = torch.tensor([4, 0, 8, 0], dtype=torch.int32, device="cuda")
    do_append(None, c, 0, "f16", None, None, 0, k, v, None, None, seq, pos, table, 4)
    flagged()
    assert torch.equal(before, kp)


# ------------------------------------------------------------------ attention
def ref_attn(q, kp, vp, lens, prefix, prefix_pages, table, page, kv, hd, scale):
    """(o, sum of w |v|, largest scale sum |q k|) in 64 bits"""
    n_seq, heads = q.shape[0], q.shape[1] // hd
    group = heads // kv
    out, mag, big = (np.zeros((n_seq, heads, hd)) for _ in range(3))
    for b in range(n_seq):
        n = int(lens[b])
        if not n:
            continue
        p = np.arange(n)
        pages = np.where(p < prefix, prefix_pages[np.minimum(p // page, max(len(prefix_pages) - 1, 0))] if prefix else 0,
                         table[b][p // page])
        slot = pages.astype(np.int64) * page + p % page
        for h in range(heads):
            k, v = kp[slot, h // group], vp[slot, h // group]
            qh = q[b, h * hd:(h + 1) * hd]
            s = scale * (k @ qh)
            w = np.exp(s - s.max())
            w /= w.sum()
            out[b, h], mag[b, h] = w @ v, w @ np.abs(v)
            big[b, h] = (abs(scale) * (np.abs(k) @ np.abs(qh))).max()
    return out.reshape(n_seq, -1), mag.reshape(n_seq, -1), big.reshape(n_seq, -1)


def attn_setup(g, n_seq, heads, kv, hd, prefix, own, page, dtype, cdt, layers=1, stale=math.nan):
    """own: the sequences' own lengths, -1 for an empty row; slots that nobody may read hold `stale`"""
    width = max(1, -(-(prefix + max(max(own), 0) + 1) // page))
    shared, first = -(-prefix // page), prefix // page
    need = shared + n_seq * (width - first)
    n_pages = need + 2
    pages = torch.randperm(n_pages, generator=g, device="cuda")[:need].to(torch.int32)
    table = torch.full((n_seq, width), -9, dtype=torch.int32, device="cuda")
    table[:, first:] = pages[shared:].view(n_seq, -1)
    pp = pages[:shared].clone()
    kp, vp, c = pools(g, layers, n_pages, page, kv, hd, cdt, fill=stale)
    lens = torch.tensor([0 if o < 0 else prefix + o for o in own], dtype=torch.int32, device="cuda")
    tn, pn = table.cpu().numpy(), pp.cpu().numpy()
    for b in range(-1, n_seq):
        lo, hi = (0, prefix) if b < 0 else (prefix, int(lens[b]))
        p = np.arange(lo, max(lo, hi))
        slot = torch.from_numpy((pn if b < 0 else tn[b])[p // page].astype(np.int64) * page + p % page).cuda()
        for t in (kp, vp):
            t[layers - 1].view(-1, kv, hd)[slot] = rand(g, (len(p), kv, hd), cdt)
    return kp, vp, c, pp, table, lens


def do_attn(c, layer, dtype, q, out, heads, scale, pp, prefix, table, lens, ws=None, stream=None):
    n_seq = table.shape[0]
    if ws is None:
        ws = torch.full((qb.attn_prefix_workspace(CODE[dtype], c, n_seq, heads, prefix, table.shape[1]),), 255, dtype=torch.uint8,
                        device="cuda")
    qb.check(lib().qmc_attn_prefix(c.ref, layer, CODE[dtype], q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), heads, n_seq,
                                   scale, pp.data_ptr() if pp.numel() else None, prefix, table.data_ptr(), table.shape[1],
                                   lens.data_ptr(), ws.data_ptr(), ws.numel(), stream or qb.torch_stream()))
    return ws


def check_attn(got, q, kp, vp, lens, prefix, pp, table, page, kv, hd, scale, dtype, cdt):
    want, mag, big = ref_attn(f64(q), f64(kp).reshape(-1, kv, hd), f64(vp).reshape(-1, kv, hd), lens.cpu().numpy(), prefix,
                              pp.cpu().numpy(), table.cpu().numpy(), page, kv, hd, scale)
    ds = (hd + 8) * U * big + (2.0**-21 * big if dtype != cdt else 0)
    ep = E[cdt] if dtype == cdt and dtype != "f32" else 2.0**-20
    close(f64(got), want, 2 * (2 * ds + 2.0**-20 + ep) * mag + E[dtype] * np.abs(want) + TINY[dtype])


TYPES = [("f32", "f32"), ("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")]
ATTN = [  # seqs, heads, kv, hd, prefix, own lengths, page
    (4, 32, 32, 128, 128, [32, 1, 7, 20], 16), (1, 8, 8, 64, 1, [0], 16), (3, 6, 6, 48, 0, [5, 1, 300], 12),
    (5, 6, 6, 48, 205, [77, 0, -1, 1, 33], 12), (2, 64, 8, 128, 1000, [600, 12], 16), (7, 16, 1, 64, 333, [3, 0, 0, 9, -1, 64, 65], 32),
    (2, 40, 8, 80, 257, [128, 129], 1), (3, 5, 1, 20, 77, [4, 2, 1], 5), (2, 4, 2, 256, 200, [31, 100], 64), (2, 3, 3, 7, 40, [9, 20], 3),
    (33, 20, 1, 32, 129, list(range(33)), 50), (2, 2, 2, 250, 70, [1, 2], 8), (40, 32, 2, 128, 700, [i % 5 for i in range(40)], 16),
    (3, 8, 2, 96, 64, [-1, -1, -1], 16), (17, 32, 2, 64, 513, [2] * 17, 64), (20, 24, 1, 112, 300, [i * 3 for i in range(20)], 20)]


@pytest.mark.parametrize("dtype,cdt", TYPES)
@pytest.mark.parametrize("case", range(len(ATTN)))
def test_attn_prefix(cuda_dev, case, dtype, cdt):
    n_seq, heads, kv, hd, prefix, own, page = ATTN[case]
    g = gen(200 + case)
    layers = 1 + case % 2
    kp, vp, c, pp, table, lens = attn_setup(g, n_seq, heads, kv, hd, prefix, own, page, dtype, cdt, layers)
    pad, shift = [(0, 0), (8, 8), (3, 1)][case % 3]
    _, q = strided(g, n_seq, heads * hd, dtype, pad, shift)
    obase, out = strided(g, n_seq + 1, heads * hd, dtype, pad, shift)  # one row behind the last sequence
    before = obase.clone()
    scale = 1.0 / math.sqrt(hd)
    do_attn(c, layers - 1, dtype, q, out, heads, scale, pp, prefix, table, lens)
    clean()
    check_attn(out[:n_seq], q, kp[layers - 1], vp[layers - 1], lens, prefix, pp, table, page, kv, hd, scale, dtype, cdt)
    for b, o in enumerate(own):
        if o < 0:
            assert (out[b] == 0).all()
    again = out.clone()
    do_attn(c, layers - 1, dtype, q, out, heads, scale, pp, prefix, table, lens)  # the same bits every time
    clean()
    assert torch.equal(again, out)
    keep = before.clone()
    for t in (keep, obase):
        t[shift:shift + (n_seq + 1) * (heads * hd + pad)].view(n_seq + 1, -1)[:n_seq, :heads * hd].zero_()
    assert torch.equal(keep, obase)


@pytest.mark.parametrize("dtype,cdt", TYPES)
def test_attn_large_scores(cuda_dev, dtype, cdt):
    """scores in the hundreds, one position far above the others, late and early, so that maxima move by much"""
    n_seq, heads, kv, hd, prefix, page = 20, 16, 2, 128, 900, 16
    g = gen(77)
    kp, vp, c, pp, table, lens = attn_setup(g, n_seq, heads, kv, hd, prefix, [40] * n_seq, page, dtype, cdt)
    q = rand(g, (n_seq, heads * hd), dtype, 4.0)
    flat = kp.view(-1, kv, hd)
    for p in (3, 500, 899):
        flat[int(pp[p // page]) * page + p % page] = (q[1].view(kv, -1, hd)[:, p % 8] * (1 + p / 900)).to(DT[cdt])
    out = torch.zeros_like(q)
    do_attn(c, 0, dtype, q, out, heads, 0.1, pp, prefix, table, lens)
    clean()
    check_attn(out, q, kp, vp, lens, prefix, pp, table, page, kv, hd, 0.1, dtype, cdt)


def test_attn_bad_pages_and_lengths(cuda_dev):
    g = gen(5)
    for dtype, cdt, heads in [("f32", "f32", 4), ("f16", "f16", 4), ("bf16", "bf16", 128)]:
        kp, vp, c, pp, table, lens = attn_setup(g, 3, heads, 2, 64, 40, [9, 9, 9], 8, dtype, cdt, stale=0.0)
        q = rand(g, (3, heads * 64), dtype)
        out = torch.zeros_like(q)
        args = (heads, 0.125, pp, 40, table, lens)
        do_attn(c, 0, dtype, q, out, *args)
        clean()
        good = out.clone()
        for t, at, bad in ((table, (1, 5), 1 << 30), (table, (1, 6), -1), (pp, (2,), kp.shape[1]), (lens, (1,), 39),
                           (lens, (1,), 1 << 30), (lens, (1,), -5)):
            old = t[at].clone()
            t[at] = bad
            do_attn(c, 0, dtype, q, out, *args)
            flagged()
            t[at] = old
            if t is not pp:  # the other sequences have their results
                assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])
        do_attn(c, 0, dtype, q, out, *args)
        clean()
        assert torch.equal(out, good)


@pytest.mark.parametrize("dtype,cdt", TYPES)
def test_attn_captured_and_on_streams(cuda_dev, dtype, cdt):
    """a captured call replayed with other lengths and queries; two calls at once on streams of their own"""
    n_seq, heads, kv, hd, prefix, page = 6, 64, 2, 64, 300, 16
    g = gen(8)
    kp, vp, c, pp, table, lens = attn_setup(g, n_seq, heads, kv, hd, prefix, [50, 40, 30, 20, 10, 60], page, dtype, cdt)
    q = rand(g, (n_seq, heads * hd), dtype)
    outs = [torch.zeros_like(q) for _ in range(2)]
    wss = [do_attn(c, 0, dtype, q, o, heads, 0.125, pp, prefix, table, lens).clone() for o in outs]
    clean()
    graphs = []
    for o, ws in zip(outs, wss):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            do_attn(c, 0, dtype, q, o, heads, 0.125, pp, prefix, table, lens, ws)
        graphs.append(gr)
    for n in (301, 310):
        lens.copy_(torch.tensor([n, 0, 300, 317, 305, 302], dtype=torch.int32))
        q.copy_(rand(g, (n_seq, heads * hd), dtype))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        for s, gr in zip(streams, graphs):
            with torch.cuda.stream(s):
                for _ in range(5):
                    gr.replay()
        clean()
        assert torch.equal(outs[0], outs[1])
        check_attn(outs[0], q, kp, vp, lens, prefix, pp, table, page, kv, hd, 0.125, dtype, cdt)


def test_offsets_past_32_bits(cuda_dev):
    """a pool of more than 2^32 bytes and 2^31 elements: the last pages are appended to and read"""
    page, kv, hd, n_pages = 32, 8, 128, 68000
    kp, vp = (torch.empty((1, n_pages, page, kv, hd), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    assert kp.numel() > 1 << 31
    c = qb.PagedCache(kp, vp, qb.QMC_BF16, 1, n_pages, page, kv, hd)
    g = gen(6)
    last = n_pages - 1 - torch.arange(6, dtype=torch.int32, device="cuda")
    kp[0, n_pages - 8:] = 0
    vp[0, n_pages - 8:] = 0
    pp, table = last[:2].clone(), torch.stack([last[[0, 1, 2]], last[[0, 1, 3]]])
    heads, prefix = 64, 50
    n = 10
    pos = torch.cat([torch.arange(prefix), prefix + torch.arange(n), prefix + torch.arange(n)]).to(torch.int32).cuda()
    seq = torch.cat([torch.zeros(prefix + n), torch.ones(n)]).to(torch.int32).cuda()
    table[1, 1] = last[4]  # the prefix ends inside a page: positions 50 .. of sequence 1 lie in a page of its own
    x = rand(g, (prefix + 2 * n, 2 * kv * hd), "bf16")
    do_append(plan(hd, hd, 1, 0), c, 0, "bf16", None, None, 0, x[:, :kv * hd], x[:, kv * hd:], None, None, seq, pos, table,
              prefix + 2 * n)
    q = rand(g, (2, heads * hd), "bf16")
    out, lens = torch.zeros_like(q), torch.full((2,), prefix + n, dtype=torch.int32, device="cuda")
    do_attn(c, 0, "bf16", q, out, heads, 0.09, pp, prefix, table, lens)
    clean()
    lo = n_pages - 8
    check_attn(out, q, kp[0, lo:], vp[0, lo:], lens, prefix, pp - lo, table - lo, page, kv, hd, 0.09, "bf16", "bf16")
    pn = pos.cpu().numpy()
    sl = (table.cpu().numpy()[seq.cpu().numpy(), pn // page].astype(np.int64) - lo) * page + pn % page
    check_heads(f64(kp[0, lo:]).reshape(-1, kv, hd)[sl], f64(x[:, :kv * hd]).reshape(-1, kv, hd), pn, None, 0, hd, 1, 0, "bf16")


# ------------------------------------------------------------------ beams
def do_select(dtype, logits, vocab, prompts, beams, scores, finished, eos, n_out, ws=None):
    par, tok = (torch.full((prompts, n_out), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    out = torch.zeros(prompts, n_out, device="cuda")
    if ws is None:
        ws = torch.full((qb.beam_workspace(prompts, beams, vocab, n_out),), 255, dtype=torch.uint8, device="cuda")
    qb.check(lib().qmc_beam_select(CODE[dtype], logits.data_ptr(), logits.stride(0), prompts, beams, vocab, scores.data_ptr(),
                                   None if finished is None else finished.data_ptr(), eos, n_out, par.data_ptr(), tok.data_ptr(),
                                   out.data_ptr(), ws.data_ptr(), ws.numel(), qb.torch_stream()))
    return par, tok, out


def ref_select(x, scores, finished, eos, n_out, prompts, beams):
    """x [rows, vocab] in 64 bits"""
    vocab = x.shape[1]
    x = np.where(np.isnan(x), -np.inf, x)
    sc = np.full(x.shape, -np.inf)
    for r in range(x.shape[0]):
        cum = scores[r]
        if not cum > -np.inf:
            continue
        if finished is not None and finished[r]:
            sc[r, eos] = cum
            continue
        m = x[r].max()
        if m == np.inf:
            sc[r] = np.where(x[r] == np.inf, cum - np.log((x[r] == np.inf).sum()), -np.inf)
        elif m > -np.inf:
            sc[r] = cum + (x[r] - (m + np.log(np.exp(x[r] - m).sum())))
    flat = sc.reshape(prompts, beams * vocab)
    at = np.argsort(-flat, axis=1, kind="stable")[:, :n_out]
    return at // vocab, at % vocab, np.take_along_axis(flat, at, 1)


def check_select(got, want):
    (par, tok, sc), (wp, wt, ws) = got, want
    sc = f64(sc)
    fin = np.isfinite(ws)
    assert np.array_equal(sc[~fin], ws[~fin])
    close(sc[fin], ws[fin], 2.0**-18 + U * np.abs(ws[fin]))
    assert np.array_equal(par.cpu().numpy(), wp) and np.array_equal(tok.cpu().numpy(), wt)


BEAM = [(1, 4, 32000, 4), (3, 1, 300, 1), (2, 5, 4096, 10), (2, 3, 4097, 6), (4, 2, 17, 4), (1, 16, 1, 16), (1, 64, 5000, 64), (2, 8, 128000, 16),
        (1, 2, 3, 6), (5, 7, 999, 14), (1, 1, 100, 64), (2, 4, 63, 64), (300, 2, 50, 4)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", range(len(BEAM)))
def test_beam_select(cuda_dev, case, dtype):
    prompts, beams, vocab, n_out = BEAM[case]
    g, rows = gen(300 + case), prompts * beams
    _, x = strided(g, rows, vocab, dtype, [0, 3, 16][case % 3], [0, 1, 0][case % 3])
    x.mul_(3)
    scores = -torch.rand(rows, generator=g, device="cuda") * 5
    fin = (torch.rand(rows, generator=g, device="cuda") < 0.3).to(torch.uint8)
    eos = min(2, vocab - 1)
    for finished in (None, fin):
        got = do_select(dtype, x, vocab, prompts, beams, scores, finished, eos, n_out)
        clean()
        check_select(got, ref_select(f64(x), f64(scores), None if finished is None else fin.cpu().numpy(), eos, n_out, prompts, beams))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_beam_select_masks_and_ties(cuda_dev, dtype):
    g = gen(1)
    prompts, beams, vocab = 6, 4, 9000
    low = torch.finfo(DT[dtype]).min
    x = rand(g, (prompts * beams, vocab), dtype, 3.0)
    scores = -torch.rand(prompts * beams, generator=g, device="cuda") * 5
    x[0:4] = 1.5                    # all equal: the lowest tokens of the best beam
    x[4] = -math.inf                # a mask that leaves nothing
    x[5, 1:] = -math.inf            # or one token
    x[6, 7000:] = low               # or holds the type's lowest value
    x[7] = low
    x[8:12, ::2] = math.nan         # NaN never wins
    x[9] = math.nan
    x[10, 5] = math.inf
    x[11, 5] = x[11, 8000] = math.inf
    scores[12:16] = -math.inf       # no beam lives
    scores[17:20] = -math.inf       # the first step: one does
    scores[18] = math.nan
    x[20:24] = x[20]                # equal rows, equal scores: the lower beam
    scores[20:24] = -1.0
    x[20:24, 11] = 0.0
    x[22, 11] = -0.0
    for n_out in (1, 4, 8, 64):
        got = do_select(dtype, x, vocab, prompts, beams, scores, None, 0, n_out)
        clean()
        want = ref_select(f64(x), f64(scores), None, 0, n_out, prompts, beams)
        check_select([t[[0, 1, 3, 4, 5]] for t in got], [t[[0, 1, 3, 4, 5]] for t in want])
        # rows with infinities: the finite scores as the definition has them
        fin = np.isfinite(want[2][2])
        check_select([t[2:3][:, torch.from_numpy(fin).cuda()] for t in got], [t[2:3][:, fin] for t in want])


def test_beam_select_few_tokens_live(cuda_dev):
    """fewer finite continuations than asked for: the lowest others follow at -inf"""
    x = torch.full((2, 10000), -math.inf, device="cuda")
    x[0, 9000], x[1, 5] = 1.0, 2.0
    scores = torch.tensor([-1.0, -2.0], device="cuda")
    got = do_select("f32", x, 10000, 1, 2, scores, None, 0, 6)
    clean()
    check_select(got, ref_select(f64(x), f64(scores), None, 0, 6, 1, 2))


def ref_reorder(par, n, page, table, kp, vp):
    """plain loops over numpy arrays; par [prompts, beams]"""
    prompts, beams = par.shape
    out = table.copy()
    t, filled = n // page, n % page
    for p in range(prompts):
        seen, free = set(), [b for b in range(beams) if b not in set(par[p])]
        for j in range(beams):
            row, src = p * beams + j, p * beams + par[p, j]
            out[row, :t] = table[src, :t]
            if t >= table.shape[1]:
                continue
            if par[p, j] not in seen:
                seen.add(par[p, j])
                out[row, t] = table[src, t]
            else:
                give = table[p * beams + free.pop(0), t]
                out[row, t] = give
                for x in (kp, vp):
                    x[:, give, :filled] = x[:, table[src, t], :filled]
    return out


@pytest.mark.parametrize("case", range(8))
def test_beam_reorder(cuda_dev, case):
    prompts, beams, n, page, kv, hd, cdt, layers = [(1, 4, 150, 16, 32, 128, "f16", 3), (3, 8, 64, 16, 2, 64, "bf16", 2),
                                                    (2, 5, 7, 12, 1, 7, "f16", 2), (4, 1, 9, 4, 2, 8, "f32", 1),
                                                    (2, 64, 31, 32, 1, 16, "f32", 1), (2, 3, 0, 4, 1, 8, "f16", 1),
                                                    (2, 6, 16, 4, 1, 8, "f16", 2), (2, 16, 5, 1, 3, 5, "bf16", 2)][case]
    g = gen(400 + case)
    rows, width = prompts * beams, n // page + (0 if case == 6 else 3)
    n_pages = rows * max(width, 1) + 1
    table = torch.randperm(n_pages, generator=g, device="cuda")[:rows * width].to(torch.int32).view(rows, width)
    kp, vp, c = pools(g, layers, n_pages, page, kv, hd, cdt)
    par = torch.randint(0, beams, (prompts, beams + 2), generator=g, device="cuda", dtype=torch.int32)
    if case == 0:
        par[0, :4] = torch.tensor([1, 0, 0, 1], dtype=torch.int32)  # beams 0 and 1 swap, 2 and 3 end
    if case == 4:
        par[0, :beams] = 63
    lens = torch.full((rows,), -5, dtype=torch.int32, device="cuda")
    lens[::beams] = n  # the first beam's length is the prompt's
    out = torch.full_like(table, -3)
    wk, wv = f64(kp), f64(vp)
    want = ref_reorder(par[:, :beams].cpu().numpy(), n, page, table.cpu().numpy(), wk, wv)
    for _ in range(2):  # pages that are copied from are never copied to: once more changes nothing
        qb.check(lib().qmc_beam_reorder(c.ref, prompts, beams, par.data_ptr(), beams + 2, lens.data_ptr(), table.data_ptr(),
                                        out.data_ptr(), width, qb.torch_stream()))
        clean()
        assert np.array_equal(out.cpu().numpy(), want)
        assert np.array_equal(f64(kp), wk) and np.array_equal(f64(vp), wv)


def test_beam_reorder_bad_indices(cuda_dev):
    g = gen(2)
    kp, vp, c = pools(g, 1, 4, 4, 1, 8, "f16")
    before = kp.clone()
    out = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    for par, table, n in (([0, 2], [[0, 1], [2, 3]], 6), ([0, -1], [[0, 1], [2, 3]], 6), ([1, 1], [[0, 1], [2, 4]], 6),
                          ([1, 1], [[0, -1], [2, 3]], 6), ([0, 0], [[0, 1], [2, 3]], 9), ([0, 1], [[0, 1], [2, 3]], -1)):
        p, t = torch.tensor([par], dtype=torch.int32, device="cuda"), torch.tensor(table, dtype=torch.int32, device="cuda")
        lens = torch.tensor([n, n], dtype=torch.int32, device="cuda")
        qb.check(lib().qmc_beam_reorder(c.ref, 1, 2, p.data_ptr(), 2, lens.data_ptr(), t.data_ptr(), out.data_ptr(), 2,
                                        qb.torch_stream()))
        flagged()
        assert torch.equal(before, kp)


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("dtype,cdt", TYPES)
def test_beam_search_over_pages(cuda_dev, dtype, cdt):
    """a beam search with one attention layer and random projections: rotate, append, attend, select, reorder, against one in 64
    bits that keeps every beam's whole history.  The plain search follows the device's choices, and each
    choice must be within the scores' error of the best that it sees."""
    g = gen(11)
    beams, heads, kv, hd, page, vocab, prompt, steps = 4, 4, 2, 64, 8, 500, 21, 30
    dim = heads * hd
    emb = torch.randn(vocab, dim, generator=g, device="cuda")
    wqkv = torch.randn(dim, (heads + 2 * kv) * hd, generator=g, device="cuda") / math.sqrt(dim)
    wout = torch.randn(dim, vocab, generator=g, device="cuda") * 4 / math.sqrt(dim)
    qw, kw = (1 + 0.1 * torch.randn(hd, generator=g, device="cuda") for _ in range(2))
    first = prompt // page  # the prompt's last page is not full: each beam continues it in a page of its own
    width = -(-(prompt + steps) // page)
    shared = -(-prompt // page)
    table = torch.zeros(beams, width, dtype=torch.int32, device="cuda")
    pp = torch.arange(shared, dtype=torch.int32, device="cuda")
    table[:, first:] = shared + torch.arange(beams * (width - first), device="cuda").view(beams, -1)
    kp, vp, c = pools(g, 1, shared + beams * (width - first), page, kv, hd, cdt, fill=math.nan)
    p = plan(hd, hd, 1, 2)
    scale = 1 / math.sqrt(hd)

    def project(tokens):
        return (emb[tokens] @ wqkv).to(DT[dtype])

    x = project(torch.randint(0, vocab, (prompt,), generator=g, device="cuda"))
    zero, at = torch.zeros(prompt, dtype=torch.int32, device="cuda"), torch.arange(prompt, dtype=torch.int32, device="cuda")
    table0 = torch.zeros(1, width, dtype=torch.int32, device="cuda")
    table0[0, :shared] = pp
    nk = heads * hd
    do_append(p, c, 0, dtype, None, None, 0, x[:, nk:nk + kv * hd], x[:, nk + kv * hd:], qw, kw, zero, at, table0, prompt)

    def ref_kv(x, pos):
        x = f64(x).reshape(len(pos), heads + 2 * kv, hd)
        q = ref_heads(x[:, :heads], pos, f64(qw), 1e-5, hd, 1, 2)[0]
        k = ref_heads(x[:, heads:heads + kv], pos, f64(kw), 1e-5, hd, 1, 2)[0]
        return q, k, x[:, heads + kv:]

    _, k0, v0 = ref_kv(x, np.arange(prompt))
    hist = [(k0, v0)] * beams
    scores = torch.tensor([0.0] + [-math.inf] * (beams - 1), device="cuda")
    ref_scores = f64(scores)
    tokens = torch.full((beams,), 3, dtype=torch.int64, device="cuda")
    drift = 0.0
    for step in range(steps):
        n = prompt + step
        x = project(tokens)
        q = torch.zeros(beams, heads * hd, dtype=DT[dtype], device="cuda")
        pos = torch.full((beams,), n, dtype=torch.int32, device="cuda")
        do_append(p, c, 0, dtype, x[:, :nk], q, heads, x[:, nk:nk + kv * hd], x[:, nk + kv * hd:], qw, kw, None, pos, table, beams)
        lens, o = pos + 1, torch.zeros_like(q)
        do_attn(c, 0, dtype, q, o, heads, scale, pp, prompt, table, lens)
        logits = o.float() @ wout
        par, tok, sc = do_select("f32", logits, vocab, 1, beams, scores, None, 0, beams)
        out = torch.zeros_like(table)
        qb.check(lib().qmc_beam_reorder(c.ref, 1, beams, par.data_ptr(), beams, lens.data_ptr(), table.data_ptr(), out.data_ptr(),
                                        width, qb.torch_stream()))
        clean()
        # the same step in 64 bits on whole histories
        rq, rk, rv = ref_kv(x, np.full(beams, n))
        hist = [(np.concatenate([h[0], rk[b:b + 1]]), np.concatenate([h[1], rv[b:b + 1]])) for b, h in enumerate(hist)]
        ro, err = np.zeros((beams, heads, hd)), np.zeros((beams, heads, hd))
        for b in range(beams):
            for h in range(heads):
                k, v = hist[b][0][:, h // 2], hist[b][1][:, h // 2]
                s = scale * (k @ rq[b, h])
                w = np.exp(s - s.max())
                w /= w.sum()
                ro[b, h] = w @ v
                # the bound of the attention, with the roundings of q, k and v, which the plain search does without
                ds = (E[dtype] + E[cdt] + 2.0**-17) * scale * (np.abs(k) @ np.abs(rq[b, h])).max()
                ep = E[cdt] if dtype == cdt and dtype != "f32" else 2.0**-20
                err[b, h] = (2 * (2 * ds + 2.0**-20 + ep) + E[cdt]) * (w @ np.abs(v)) + E[dtype] * np.abs(ro[b, h])
        # a logit is off by the sum over the dimensions (and its own float sum), a score by twice the largest, and the scores add up
        drift += 2 * ((err.reshape(beams, -1) + 512 * U * np.abs(ro.reshape(beams, -1))) @ np.abs(f64(wout))).max() + 2.0**-18
        rl = ro.reshape(beams, -1) @ f64(wout)
        logp = rl - rl.max(1, keepdims=True)
        logp -= np.log(np.exp(logp).sum(1, keepdims=True))
        total = ref_scores[:, None] + logp
        pn, tn = par[0].cpu().numpy(), tok[0].cpu().numpy()
        chosen = total[pn, tn]
        best = np.sort(total.reshape(-1))[::-1][:beams]
        assert len(set(zip(pn.tolist(), tn.tolist()))) == beams
        assert np.abs(np.sort(chosen)[::-1] - best).max() <= 2 * drift, (step, chosen, best)
        close(f64(sc)[0], chosen, drift)
        hist = [hist[j] for j in pn]
        ref_scores, scores, tokens, table = chosen, sc[0].contiguous(), tok[0].long(), out


# ------------------------------------------------------------------ captured, at once, at the ends of the ranges
TC = [  # seqs, heads, kv, hd, prefix, own lengths, page: many rows, every padded head width, pages from one copy to many
    (20, 2, 2, 8, 1000, [3] * 20, 8), (5, 16, 2, 24, 2049, [0, 1, 7, 8, 9], 24), (40, 8, 1, 40, 129, [i for i in range(40)], 40),
    (9, 16, 1, 56, 128, [1] * 9, 128), (17, 8, 8, 72, 127, [2] * 17, 256), (130, 2, 1, 88, 777, [i % 3 for i in range(130)], 16),
    (12, 16, 1, 104, 3001, [5] * 12, 512), (33, 8, 1, 120, 640, [1] * 33, 64), (257, 1, 1, 128, 500, [0] * 257, 32),
    (18, 1, 1, 64, 5, [1] * 18, 8)]


@pytest.mark.parametrize("dtype,cdt", [("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("case", range(len(TC)))
def test_attn_many_rows(cuda_dev, case, dtype, cdt):
    n_seq, heads, kv, hd, prefix, own, page = TC[case]
    g = gen(500 + case)
    kp, vp, c, pp, table, lens = attn_setup(g, n_seq, heads, kv, hd, prefix, own, page, dtype, cdt)
    _, q = strided(g, n_seq, heads * hd, dtype, [0, 5][case % 2], [0, 3][case % 2])
    out = torch.zeros(n_seq, heads * hd, dtype=DT[dtype], device="cuda")
    scale = 1.0 / math.sqrt(hd)
    do_attn(c, 0, dtype, q, out, heads, scale, pp, prefix, table, lens)
    clean()
    check_attn(out, q, kp, vp, lens, prefix, pp, table, page, kv, hd, scale, dtype, cdt)


@pytest.mark.parametrize("dtype,cdt", TYPES)
def test_attn_pages_listed_more_than_once(cuda_dev, dtype, cdt):
    """two sequences with the same pages of their own, a prefix that repeats a page; on the library's own stream"""
    n_seq, heads, kv, hd, prefix, page = 3, 24, 1, 64, 96, 16
    g = gen(19)
    kp, vp, c, pp, table, lens = attn_setup(g, n_seq, heads, kv, hd, prefix, [30, 30, 17], page, dtype, cdt, stale=0.0)
    table[1] = table[0]
    pp[3:] = pp[0]
    q = rand(g, (n_seq, heads * hd), dtype)
    q[1] = q[0]
    out = torch.zeros_like(q)
    ws = torch.empty(qb.attn_prefix_workspace(CODE[dtype], c, n_seq, heads, prefix, table.shape[1]), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    qb.check(lib().qmc_attn_prefix(c.ref, 0, CODE[dtype], q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), heads, n_seq, 0.125,
                                   pp.data_ptr(), prefix, table.data_ptr(), table.shape[1], lens.data_ptr(), ws.data_ptr(), ws.numel(),
                                   None))
    qb.check(lib().qmc_sync())
    assert torch.equal(out[0], out[1])
    check_attn(out, q, kp, vp, lens, prefix, pp, table, page, kv, hd, 0.125, dtype, cdt)


def test_decoding_step_captured(cuda_dev):
    """append, attention, selection and reordering in one graph, replayed on another stream with other inputs, against the same
    calls one by one: the same bits"""
    prompts, beams, heads, kv, hd, page, width, prefix, vocab = 2, 3, 8, 2, 64, 8, 6, 13, 9001
    rows, g = prompts * beams, gen(23)
    n_pages = rows * width + 2
    p = plan(hd, hd, 1, 0)
    perm = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    pp, own = perm[:2].clone(), perm[2:2 + rows * (width - 1)].view(rows, width - 1)
    state = []
    for _ in range(2):  # [0] replayed, [1] one by one
        kp, vp, c = pools(gen(24), 2, n_pages, page, kv, hd, "f16")
        table = torch.cat([pp[:1].expand(rows, 1), own], 1).contiguous()
        state.append(dict(kp=kp, vp=vp, c=c, table=table, out=torch.zeros_like(table), lens=torch.full((rows,), 30, dtype=torch.int32, device="cuda"),
                          pos=torch.full((rows,), 29, dtype=torch.int32, device="cuda"), x=torch.zeros(rows, (heads + 2 * kv) * hd, device="cuda").half(),
                          y=torch.zeros(rows, heads * hd, device="cuda").half(), logits=torch.zeros(rows, vocab, device="cuda"),
                          scores=torch.zeros(rows, device="cuda"), par=torch.zeros(prompts, 5, dtype=torch.int32, device="cuda"),
                          tok=torch.zeros(prompts, 5, dtype=torch.int32, device="cuda"), best=torch.zeros(prompts, 5, device="cuda"),
                          w1=torch.full((qb.attn_prefix_workspace(qb.QMC_F16, c, rows, heads, prefix, width),), 255, dtype=torch.uint8, device="cuda"),
                          w2=torch.full((qb.beam_workspace(prompts, beams, vocab, 5),), 255, dtype=torch.uint8, device="cuda")))

    def step(s):
        k, v = s["x"][:, heads * hd:(heads + kv) * hd], s["x"][:, (heads + kv) * hd:]
        do_append(p, s["c"], 1, "f16", s["x"][:, :heads * hd], s["x"][:, :heads * hd], heads, k, v, None, None, None, s["pos"], s["table"], rows)
        do_attn(s["c"], 1, "f16", s["x"][:, :heads * hd], s["y"], heads, 0.125, pp, prefix, s["table"], s["lens"], s["w1"])
        qb.check(lib().qmc_beam_select(qb.QMC_F32, s["logits"].data_ptr(), vocab, prompts, beams, vocab, s["scores"].data_ptr(), None, 0, 5,
                                       s["par"].data_ptr(), s["tok"].data_ptr(), s["best"].data_ptr(), s["w2"].data_ptr(), s["w2"].numel(),
                                       qb.torch_stream()))
        qb.check(lib().qmc_beam_reorder(s["c"].ref, prompts, beams, s["par"].data_ptr(), 5, s["lens"].data_ptr(), s["table"].data_ptr(),
                                        s["out"].data_ptr(), width, qb.torch_stream()))

    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step(state[0])
    for n in (30, 33, 40):
        x, z = rand(g, (rows, (heads + 2 * kv) * hd), "f16"), rand(g, (rows, vocab), "f32", 3.0)
        for s in state:
            s["x"].copy_(x), s["logits"].copy_(z), s["lens"].fill_(n), s["pos"].fill_(n - 1)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        step(state[1])
        clean()
        for name in ("kp", "vp", "x", "y", "par", "tok", "best", "out"):
            a, b = (s[name].view(torch.int16) if s[name].dtype == torch.float16 else s[name] for s in state)
            assert torch.equal(a, b), name
        for s in state:
            s["table"].copy_(s["out"])
            s["scores"].copy_(s["best"][:, :beams].reshape(-1))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_beam_select_at_once(cuda_dev, dtype):
    """two selections at once, on streams and workspaces of their own"""
    g = gen(31)
    jobs = []
    for prompts, beams, vocab, n_out in ((3, 8, 40000, 16), (2, 5, 70001, 10)):
        x = rand(g, (prompts * beams, vocab), dtype, 3.0)
        jobs.append((x, vocab, prompts, beams, -torch.rand(prompts * beams, generator=g, device="cuda"), None, 0, n_out))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in jobs], [[] for _ in jobs]
    for _ in range(5):
        for i, (s, j) in enumerate(zip(streams, jobs)):
            with torch.cuda.stream(s):
                got[i].append(do_select(dtype, *j))
    clean()
    for all_of, (x, vocab, prompts, beams, scores, _, eos, n_out) in zip(got, jobs):
        want = ref_select(f64(x), f64(scores), None, eos, n_out, prompts, beams)
        for one in all_of:
            check_select(one, want)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_beam_select_largest(cuda_dev, dtype):
    """as many beams and logits as a call takes: 64 rows of 2^19, and all of one chunk's logits equal"""
    g = gen(37)
    x = rand(g, (64, 1 << 19), dtype, 2.0)
    x[5, :20000] = 9.0
    scores = -torch.rand(64, generator=g, device="cuda")
    scores[5] += 3.0
    got = do_select(dtype, x, 1 << 19, 1, 64, scores, None, 0, 64)
    clean()
    check_select(got, ref_select(f64(x), f64(scores), None, 0, 64, 1, 64))
