"""The batched-decoding operators where values are extreme and blocks have many tiles, against plain forms in 64 bits:
scores that rise far above a row's first tile, softmax weights far below the largest, infinities beside dimensions that
stay, rows of logits with infinities.

Tolerances as in test_gpu_batch_ops.py (u = 2^-24, e and e_P half steps of the output's and the weights' type); what a test
adds to them stands beside it."""
import math

import numpy as np
import pytest
import torch

import quillm_b200 as qb
from test_gpu_batch_ops import (CODE, DT, E, TINY, U, check_select, clean, do_append, do_attn, do_select, f64, gen, lib, plan, pools,
                                rand, ref_select)

pytestmark = pytest.mark.gpu
LOG2E = 1.4426950408889634


def shared(g, kv, hd, prefix, page, cdt, std=1.0):
    """a cache that holds one prefix of whole pages, the prefix's pages, and its keys and values as views by position"""
    n = prefix // page
    assert n * page == prefix
    kp, vp, c = pools(g, 1, n, page, kv, hd, cdt)
    kp.mul_(std)
    pp = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
    slot = (pp.long()[:, None] * page + torch.arange(page, device="cuda")).view(-1)
    return kp.view(-1, kv, hd), vp.view(-1, kv, hd), c, pp, slot


def ranges(c, dtype, n_seq, heads, hd, prefix, page):
    """position ranges that the prefix is split into: without own positions the workspace is [ranges][rows] (m, l) and o, and 256
    bytes over"""
    n = qb.attn_prefix_workspace(CODE[dtype], c, n_seq, heads, prefix, prefix // page)
    return (n - 256) // (n_seq * heads * (8 + 4 * hd))


def over_prefix(c, dtype, q, heads, hd, scale, pp, prefix, page):
    """the attention of rows that have the prefix alone, twice: the same bits"""
    n_seq, width = q.shape[0], prefix // page
    table = torch.full((n_seq, width), -9, dtype=torch.int32, device="cuda")
    lens = torch.full((n_seq,), prefix, dtype=torch.int32, device="cuda")
    outs = []
    for _ in range(2):
        outs.append(torch.full((n_seq, heads * hd), 77.0, dtype=DT[dtype], device="cuda"))
        do_attn(c, 0, dtype, q, outs[-1], heads, scale, pp, prefix, table, lens)
    clean()
    bits = [o.view(torch.int32 if dtype == "f32" else torch.int16) for o in outs]
    assert torch.equal(*bits)
    return outs[0]


def check_prefix(got, q, keys, values, slot, kv, hd, scale, dtype, cdt, floor=0.0):
    """floor: added, of the largest value, for weights far below the largest of their tile"""
    n_seq = q.shape[0]
    x = q.double().view(n_seq, kv, -1, hd).transpose(0, 1).flatten(1, 2)  # [kv, rows, hd]
    y = got.double().view(n_seq, kv, -1, hd).transpose(0, 1).flatten(1, 2)
    for h in range(kv):
        k, v = keys[slot, h].double(), values[slot, h].double()
        w = torch.softmax(scale * (x[h] @ k.T), 1)
        want, mag = w @ v, w @ v.abs()
        big = scale * (x[h].abs() @ k.abs().T).amax(1, keepdim=True)
        ds = (hd + 8) * U * big + (2.0**-21 * big if dtype != cdt else 0)
        ep = E[cdt] if dtype == cdt and dtype != "f32" else 2.0**-20
        tol = 2 * (2 * ds + 2.0**-20 + ep) * mag + E[dtype] * want.abs() + TINY[dtype] + floor * v.abs().max()
        bad = ~((y[h] - want).abs() <= tol)
        assert not bad.any(), (h, bad.nonzero()[:4].tolist(), y[h][bad][:4].tolist(), want[bad][:4].tolist(), tol[bad][:4].tolist())


# kernels of the prefix: type of rows and cache, sequences, query heads of a KV head, head_dim, page, positions of a tile; 148 KV heads fill
# the SMs, so that a block has several tiles
MANY = {"tc": ("f16", "f16", 20, 1, 64, 16, 128), "tc bf16": ("bf16", "bf16", 20, 1, 64, 16, 128),
        "tc pair": ("f16", "f16", 17, 8, 64, 32, 128), "tc pair bf16": ("bf16", "bf16", 17, 8, 64, 32, 128),
        "tc wide": ("f16", "f16", 5, 8, 128, 64, 128), "tc wide bf16": ("bf16", "bf16", 33, 4, 120, 8, 128),
        "warp": ("f16", "f16", 3, 4, 64, 16, 64), "warp bf16": ("bf16", "bf16", 2, 8, 128, 16, 64), "warp f32": ("f32", "f16", 4, 2, 128, 16, 64),
        "mma 32": ("f16", "f16", 20, 1, 64, 4, 64), "mma 64": ("bf16", "bf16", 20, 2, 128, 4, 64), "mma f32": ("f32", "f16", 20, 1, 64, 16, 64),
        "mma 256": ("f16", "f16", 3, 2, 256, 16, 64), "mma 256 f32": ("f32", "f16", 9, 4, 200, 16, 64),
        "vec": ("f32", "f32", 3, 2, 64, 16, 32), "rows": ("f16", "f16", 3, 2, 36, 16, 32)}


def many(name, prefix=1536, std=0.05):
    dtype, cdt, n_seq, group, hd, page, tile = MANY[name]
    kv, g = 148, gen(len(name) + 1000 * n_seq)
    keys, values, c, pp, slot = shared(g, kv, hd, prefix, page, cdt, std)
    q = rand(g, (n_seq, kv * group * hd), dtype)
    n = ranges(c, dtype, n_seq, kv * group, hd, prefix, page)
    assert -(-prefix // tile) // n >= 4, n  # a block has four tiles and more
    return dtype, cdt, n_seq, kv, group, hd, page, keys, values, c, pp, slot, q


@pytest.mark.parametrize("name", list(MANY))
def test_attn_scores_far_above_the_first_tile(cuda_dev, name):
    """for one row of a KV head a key scores 9 to 300 powers of two above what came before it, in every later tile of a block
    and at every offset modulo 16; the other rows, whose scores stay, do not move the reference for it"""
    prefix = 1536
    dtype, cdt, n_seq, kv, group, hd, page, keys, values, c, pp, slot, q = many(name, prefix)
    scale = 1.0 / math.sqrt(hd)
    x = q.view(n_seq, kv, group, hd)
    x[..., 0] = 0
    for h in range(kv):
        p = 128 * (1 + h % 11) + 16 * (h // 16 % 8) + h % 16
        up = [9, 60, 130, 200, 300][h % 5]
        x[h % n_seq, h, h % group, 0] = 8
        keys[slot[p], h] = 0
        keys[slot[p], h, 0] = up / LOG2E / (8 * scale)
    out = over_prefix(c, dtype, q, kv * group, hd, scale, pp, prefix, page)
    check_prefix(out, q, keys, values, slot, kv, hd, scale, dtype, cdt)


GAPS = [8, 11, 14, 16, 18, 20]  # natural exponents of a sink above the rest


def sinks(g, q, keys, values, slot, where, kv, hd, scale):
    """a KV head's key at position where(head), of value zero, scores GAPS[head % 6] above all others, which are nearly level and have
    values that do not cancel: what is left of the output is the others' share, e^-gap of a value each"""
    keys[..., 0] = 0
    values.copy_(64 + 16 * torch.randn(values.shape, generator=g, device="cuda"))
    q.view(q.shape[0], kv, -1, hd)[..., 0] = 8
    for h in range(kv):
        keys[slot[where(h)], h] = 0
        keys[slot[where(h)], h, 0] = GAPS[h % 6] / (8 * scale)
        values[slot[where(h)], h] = 0


# added, of the largest value: a weight is off by 2^-25 where that is more than half its own step, a row's largest of a tile stands at 2^10
# or above when the sink is in it, and up to 128 positions share the sink's tile: 2^7 2^-25 2^-10
SINK_FLOOR = 2.0**-28


@pytest.mark.parametrize("name", [n for n, case in MANY.items() if case[1] == "f16"])
def test_attn_small_weights_beside_a_sink(cuda_dev, name):
    prefix = 1536
    dtype, cdt, n_seq, kv, group, hd, page, keys, values, c, pp, slot, q = many(name, prefix)
    scale = 1.0 / math.sqrt(hd)
    sinks(gen(5), q, keys, values, slot, lambda h: [0, 700, 1535, 130][h // 6 % 4], kv, hd, scale)
    out = over_prefix(c, dtype, q, kv * group, hd, scale, pp, prefix, page)
    check_prefix(out, q, keys, values, slot, kv, hd, scale, dtype, cdt, SINK_FLOOR)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attn_small_weights_beside_a_sink_of_its_own(cuda_dev, hd, dtype):
    """the same in a sequence's own positions"""
    kv, group, page, own, n_seq = 60, 4, 16, 2048, 5
    g, scale, heads = gen(hd), 1.0 / math.sqrt(hd), 240
    keys, values, c, pages, slot = shared(g, kv, hd, n_seq * own, page, "f16", 0.05)
    q = rand(g, (n_seq, heads * hd), dtype)
    for b in range(n_seq):
        at = slot[b * own:(b + 1) * own]
        k, v = keys[at], values[at]
        sinks(g, q[b:b + 1], k, v, torch.arange(own), lambda h: [0, 900, 2000][h // 6 % 3], kv, hd, scale)
        keys[at], values[at] = k, v
    table = pages.view(n_seq, own // page).contiguous()
    lens = torch.tensor([own, own - 40, own, own - 47, own], dtype=torch.int32, device="cuda")
    out = torch.zeros_like(q)
    do_attn(c, 0, dtype, q, out, heads, scale, torch.empty(0), 0, table, lens)
    clean()
    for b, n in enumerate(lens.tolist()):
        check_prefix(out[b:b + 1], q[b:b + 1], keys, values, slot[b * own:b * own + n], kv, hd, scale, dtype, "f16", SINK_FLOOR)


# ------------------------------------------------------------------ rotation
def same(got, want):
    """equal values, infinities and NaN in the same places"""
    assert torch.equal(got.float().nan_to_num(1e30, 2e30, -2e30), want.float().nan_to_num(1e30, 2e30, -2e30))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [3, 1000])
@pytest.mark.parametrize("hd,rot,layout", [(128, 64, 1), (128, 64, 0), (64, 20, 0), (48, 20, 1), (36, 12, 1), (256, 2, 1), (10, 6, 0)])
def test_infinities_beside_dimensions_that_stay(cuda_dev, hd, rot, layout, rows, dtype):
    """dimensions past the rotated ones, and all of them without a plan, come through as they are, whatever stands beside them"""
    heads, kv, page, g = 16, 8, 16, gen(hd + rot)
    x = rand(g, (rows, (heads + 2 * kv) * hd), dtype)
    v3 = x.view(rows, heads + 2 * kv, hd)
    stay = torch.arange(rot, hd, device="cuda")
    for i, value in enumerate((math.inf, -math.inf, math.nan)):
        at = stay[torch.randint(0, hd - rot, (rows, heads + 2 * kv), generator=g, device="cuda")]
        pick = torch.randint(0, 3, (rows, heads + 2 * kv), generator=g, device="cuda") == i
        v3.scatter_(2, at[..., None], torch.where(pick[..., None], torch.tensor(value, device="cuda"), v3.gather(2, at[..., None]).float()).to(DT[dtype]))
    q, k, v = x[:, :heads * hd], x[:, heads * hd:(heads + kv) * hd], x[:, (heads + kv) * hd:]
    pos = torch.randint(0, 5000, (rows,), generator=g, device="cuda", dtype=torch.int32)
    qo, ko = torch.zeros(rows, heads * hd, dtype=DT[dtype], device="cuda"), torch.zeros(rows, kv * hd, dtype=DT[dtype], device="cuda")
    p = plan(hd, rot, layout, 0)
    qb.check(lib().qmc_qk_norm_rope(p.h, CODE[dtype], q.data_ptr(), x.stride(0), qo.data_ptr(), heads * hd, heads, k.data_ptr(), x.stride(0),
                                    ko.data_ptr(), kv * hd, kv, None, None, 0.0, pos.data_ptr(), rows, qb.torch_stream()))
    clean()
    same(qo.view(rows, heads, hd)[..., rot:], q.reshape(rows, heads, hd)[..., rot:])
    same(ko.view(rows, kv, hd)[..., rot:], k.reshape(rows, kv, hd)[..., rot:])
    assert torch.isfinite(qo.view(rows, heads, hd)[..., :rot]).all() and torch.isfinite(ko.view(rows, kv, hd)[..., :rot]).all()
    n_pages = -(-rows // page)
    kp, vp, c = pools(g, 1, n_pages, page, kv, hd, dtype, fill=55.0)
    at = torch.arange(rows, dtype=torch.int32, device="cuda")
    table = torch.arange(n_pages, dtype=torch.int32, device="cuda").view(1, -1)
    do_append(None, c, 0, dtype, q, qo, heads, k, v, None, None, torch.zeros_like(at), at, table, rows)
    clean()
    same(qo, q)
    same(kp.view(-1, kv * hd)[:rows], k)
    same(vp.view(-1, kv * hd)[:rows], v)


@pytest.mark.parametrize("factor", [1e-6, 0.5, 1.0, 1.5, 40.0])
def test_yarn_scales_only_longer_contexts(cuda_dev, factor):
    """the factor on cos and sin is 1 for factors up to 1: a turn then keeps the length of every pair"""
    rows, heads, hd, g = 50, 4, 64, gen(2)
    q = rand(g, (rows, heads * hd), "f32")
    out, pos = torch.zeros_like(q), torch.arange(rows, dtype=torch.int32, device="cuda") * 97
    p = qb.RopePlan(hd, hd, qb.QMC_ROPE_HALF, 10000.0, qb.QMC_ROPE_YARN, factor, 1.0, 32.0, 4096)
    qb.check(lib().qmc_qk_norm_rope(p.h, 0, q.data_ptr(), heads * hd, out.data_ptr(), heads * hd, heads, None, 0, None, 0, 0, None, None, 0.0,
                                    pos.data_ptr(), rows, qb.torch_stream()))
    clean()
    by = 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
    a, b = (t.view(rows, heads, 2, hd // 2).double().square().sum(2).sqrt() for t in (q, out))
    assert ((b - by * a).abs() <= 2.0**-18 * by * a).all()  # two elements, each off by 2^-19 m (|a| + |b|), up to sqrt(2) of the length


# ------------------------------------------------------------------ beams
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [5, 100, 4097, 30000])
def test_beam_select_fills_up_behind_infinities(cuda_dev, vocab, dtype):
    """in a row that holds +inf every other token scores -inf: where too few are left, the lowest of them follow"""
    prompts, beams, g = 7, 3, gen(vocab)
    x = rand(g, (prompts * beams, vocab), dtype, 3.0)
    scores = -torch.rand(prompts * beams, generator=g, device="cuda")
    last = vocab - 1
    x[0:3, min(50, last)] = math.inf                       # one in each beam
    x[3, 0] = x[3, 1] = x[3, last] = math.inf              # the lowest are infinite themselves
    x[4], x[5] = -math.inf, math.nan
    x[6, :] = math.inf                                     # as many as there are tokens
    x[7:9] = -math.inf
    x[9, ::2] = math.inf
    x[10, 1::3], x[10, 2::3] = math.nan, -math.inf
    x[10, last] = math.inf
    x[11] = x[10]
    scores[12] = -math.inf                                 # a dead beam below one that holds infinities
    x[13, 3] = x[14, 2] = math.inf
    finished = torch.zeros(prompts * beams, dtype=torch.uint8, device="cuda")
    finished[15] = 1                                       # and a finished one
    x[16, 1] = math.inf
    scores[17] = math.nan
    x[18, last] = math.inf                                 # beside rows of finite logits there are enough
    for n_out in (1, 3, 6, 15, 64):
        if n_out > beams * vocab:
            continue
        got = do_select(dtype, x, vocab, prompts, beams, scores, finished, 2, n_out)
        clean()
        check_select(got, ref_select(f64(x), f64(scores), finished.cpu().numpy(), 2, n_out, prompts, beams))


# ------------------------------------------------------------------ many tiles a block
@pytest.mark.parametrize("name", list(MANY))
def test_attn_many_tiles_a_block(cuda_dev, name):
    """rings of tiles used again and again, both streams of a block, maxima that creep up and fall, a last tile that is cut"""
    dtype, cdt, n_seq, group, hd, page, tile = MANY[name]
    for std, prefix in ((1.0, 1536), (3.0, 1536), (1.0, 1984 + page)):
        kv, g = 148, gen(int(10 * std) + prefix)
        prefix = prefix // page * page
        keys, values, c, pp, slot = shared(g, kv, hd, prefix, page, cdt, std)
        # scores that rise, fall and rise again along the prefix
        keys[slot] *= (1.0 + 0.8 * torch.sin(torch.arange(prefix, device="cuda") / 200)).to(DT[cdt])[:, None, None]
        q = rand(g, (n_seq, kv * group * hd), dtype)
        assert -(-prefix // tile) // ranges(c, dtype, n_seq, kv * group, hd, prefix, page) >= 4
        scale = 1.0 / math.sqrt(hd)
        out = over_prefix(c, dtype, q, kv * group, hd, scale, pp, prefix, page)
        check_prefix(out, q, keys, values, slot, kv, hd, scale, dtype, cdt, SINK_FLOOR if cdt == "f16" else 0.0)


@pytest.mark.parametrize("dtype,cdt", [("f16", "f16"), ("bf16", "bf16")])
def test_attn_repeats_its_bits(cuda_dev, dtype, cdt):
    """prefix and own positions beside each other, in several tiles each: the same bits from call to call"""
    n_seq, heads, kv, hd, page, prefix, own = 16, 64, 8, 128, 16, 8192, 512
    g = gen(3)
    width = (prefix + own) // page
    n_pages = prefix // page + n_seq * (own // page)
    kp, vp, c = pools(g, 1, n_pages, page, kv, hd, cdt)
    pages = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    pp = pages[:prefix // page].clone()
    table = torch.cat([pp.expand(n_seq, -1), pages[prefix // page:].view(n_seq, -1)], 1).contiguous()
    lens = (prefix + torch.randint(1, own + 1, (n_seq,), generator=g, device="cuda")).to(torch.int32)
    q = rand(g, (n_seq, heads * hd), dtype)
    outs = [torch.zeros_like(q) for _ in range(20)]
    for o in outs:
        do_attn(c, 0, dtype, q, o, heads, 0.09, pp, prefix, table, lens)
    clean()
    assert all(torch.equal(o.view(torch.int16), outs[0].view(torch.int16)) for o in outs)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_beam_select_ties_of_shifted_rows(cuda_dev, dtype):
    """rows of logits that differ by a constant have the same scores: the lower beam's come first"""
    prompts, beams, vocab, n_out = 40, 6, 9, 20
    g = gen(41)
    x = torch.randint(-4, 5, (prompts, 1, vocab), generator=g, device="cuda") + torch.randint(-30, 30, (prompts, beams, 1), generator=g, device="cuda")
    x = x.to(DT[dtype]).view(prompts * beams, vocab).contiguous()
    scores = torch.randint(-9, 0, (prompts, 1), generator=g, device="cuda").float().expand(-1, beams).reshape(-1).contiguous()
    par, tok, sc = do_select(dtype, x, vocab, prompts, beams, scores, None, 0, n_out)
    clean()
    # ordered by the logit above that of the row's first token, then by beam, then by token
    rel = (x.view(prompts, beams, vocab) - x.view(prompts, beams, vocab)[:, :, :1]).float().cpu().numpy().reshape(prompts, -1)
    at = np.argsort(-rel, axis=1, kind="stable")[:, :n_out]
    assert np.array_equal(par.cpu().numpy(), at // vocab) and np.array_equal(tok.cpu().numpy(), at % vocab)
    check_select((par, tok, sc), (at // vocab, at % vocab, ref_select(f64(x), f64(scores), None, 0, n_out, prompts, beams)[2]))


def best(x, scores, n_out, prompts, beams):
    """parents, tokens and scores in 64 bits, from the distances to a row's largest logit; x [rows, vocab], no NaN"""
    sc = np.full(x.shape, -np.inf)
    for r in range(x.shape[0]):
        m = x[r].max()
        if scores[r] > -np.inf and np.isfinite(m):
            sc[r] = scores[r] + ((x[r] - m) - np.log(np.exp(x[r] - m).sum()))
        elif scores[r] > -np.inf and m > 0:
            sc[r] = np.where(x[r] == np.inf, scores[r] - np.log((x[r] == np.inf).sum()), -np.inf)
    flat = sc.reshape(prompts, -1)
    at = np.argsort(-flat, axis=1, kind="stable")[:, :n_out]
    return at // x.shape[1], at % x.shape[1], np.take_along_axis(flat, at, 1)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_beam_select_rows_of_the_lowest_value(cuda_dev, dtype):
    """a mask of the type's lowest value over a whole row leaves every token the same share, 1 / vocab, not all of it"""
    prompts, beams, vocab, n_out, g = 2, 2, 9000, 8, gen(43)
    x = rand(g, (prompts * beams, vocab), dtype, 3.0)
    x[1] = x[2] = x[3] = torch.finfo(DT[dtype]).min
    scores = -torch.rand(prompts * beams, generator=g, device="cuda")
    got = do_select(dtype, x, vocab, prompts, beams, scores, None, 0, n_out)
    clean()
    check_select(got, best(f64(x), f64(scores), n_out, prompts, beams))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_beam_select_masked_rows_together(cuda_dev, dtype):
    """equal rows, masks of -inf and of the lowest value, NaN, infinities, dead beams and the first step in one call"""
    prompts, beams, vocab, g = 6, 4, 9000, gen(47)
    low = torch.finfo(DT[dtype]).min
    x = rand(g, (prompts * beams, vocab), dtype, 3.0)
    scores = -torch.rand(prompts * beams, generator=g, device="cuda") * 5
    x[0:4] = 1.5
    x[4] = -math.inf
    x[5, 1:] = -math.inf
    x[6, 7000:] = low
    x[7] = low
    x[8:12, ::2] = math.nan
    x[9] = math.nan
    x[10, 5] = math.inf
    x[11, 5] = x[11, 8000] = math.inf
    scores[12:16] = -math.inf
    scores[17:20] = -math.inf
    scores[18] = math.nan
    x[20:24] = x[20].clone()
    scores[20:24] = -1.0
    x[20:24, 11] = 0.0
    x[22, 11] = -0.0
    for n_out in (1, 4, 8, 64):
        got = do_select(dtype, x, vocab, prompts, beams, scores, None, 0, n_out)
        clean()
        check_select(got, best(np.nan_to_num(f64(x), nan=-np.inf, posinf=np.inf, neginf=-np.inf), f64(scores), n_out, prompts, beams))
