"""Measured cases of the batched-decoding operators: query / key norms with the rotation, the append to a
paged cache, attention of a batch over a shared prefix, and beam selection with the reordering of states.

`run` computes an operator in elementary torch operations, or, with `own` set, through libquillm_cuda."""
import math

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
CODE = {"f32": 0, "f16": 1, "bf16": 4}
LAYOUT = {"interleaved": 0, "half": 1}
SCALING = {"plain": 0, "linear": 1, "bands": 2, "yarn": 3}
EPS = 1e-5
# scaled contexts: an original length of 4096, low / high factors of the wavelength bands and of the ramp
ORIG = 4096
BANDS = (1.0, 4.0)
RAMP = (1.0, 32.0)


def listed():
    return [
        # one decoded token of the 7B shapes: launch latency
        rope_case(name="rope-1-token", rows=1, heads=32, kv=32, hd=128, rot=128, dtype="f32", layout="interleaved",
                  norm=False, scaling="plain", factor=1.0, far=700),
        # a batch's token of small heads, part of the head rotated, sizes no vector width divides
        rope_case(name="rope-odd", rows=333, heads=6, kv=6, hd=48, rot=20, dtype="f16", layout="half", norm=True,
                  scaling="linear", factor=4.0, far=20000),
        # a long prompt of the 70B shapes with key and query norms and a scaled rotation
        rope_case(name="rope-prompt", rows=8192, heads=64, kv=8, hd=128, rot=128, dtype="bf16", layout="half", norm=True,
                  scaling="bands", factor=8.0, far=100000),
        # the token of eight sequences of the 7B shapes, float rows into the fp16 cache
        append_case(name="append-8-tokens", seqs=8, each=1, start=700, heads=32, kv=32, hd=128, rot=128, page=16, layers=2,
                    dtype="f32", cache="f16", layout="interleaved", norm=False, scaling="plain", factor=1.0),
        # ragged pieces of prompts, small heads, a page size that is no power of two
        append_case(name="append-odd", seqs=7, each=61, start=9, heads=6, kv=6, hd=48, rot=48, page=12, layers=2,
                    dtype="f32", cache="f32", layout="interleaved", norm=True, scaling="yarn", factor=4.0),
        # prompts of the 70B shapes
        append_case(name="append-prompt", seqs=4, each=2048, start=0, heads=64, kv=8, hd=128, rot=128, page=32, layers=1,
                    dtype="bf16", cache="bf16", layout="half", norm=True, scaling="bands", factor=8.0),
        # four beams over a prompt of 128 tokens, the 7B shapes with the model's own types
        attn_case(name="attn-beams", seqs=4, heads=32, kv=32, hd=128, prefix=128, own_max=32, page=16, layers=2,
                  dtype="f32", cache="f16", empty=0),
        # small heads in full precision, a prefix that ends inside a page, one sequence that is done
        attn_case(name="attn-odd", seqs=5, heads=6, kv=6, hd=48, prefix=205, own_max=77, page=12, layers=2, dtype="f32",
                  cache="f32", empty=1),
        # sixteen samples of the 70B shapes over a document
        attn_case(name="attn-document", seqs=16, heads=64, kv=8, hd=128, prefix=8192, own_max=512, page=16, layers=1,
                  dtype="bf16", cache="bf16", empty=0),
        # a large batch behind one long context
        attn_case(name="attn-long", seqs=64, heads=64, kv=8, hd=128, prefix=32768, own_max=256, page=32, layers=1,
                  dtype="f16", cache="f16", empty=0),
        # four beams of one prompt, the vocabulary and layers of the 7B model
        beam_case(name="beam-4", prompts=1, beams=4, vocab=32000, n_out=4, dtype="f32", ended=0, first=False, length=150,
                  page=16, layers=32, kv=32, hd=128, cache="f16"),
        # many prompts, wide beams, a large vocabulary
        beam_case(name="beam-batch", prompts=24, beams=8, vocab=128000, n_out=16, dtype="bf16", ended=2, first=False,
                  length=1000, page=32, layers=16, kv=8, hd=128, cache="bf16"),
    ]


def rope_case(**k):
    return dict(kind="rope", **k)


def append_case(**k):
    return dict(kind="append", **k)


def attn_case(**k):
    return dict(kind="attn", **k)


def beam_case(**k):
    return dict(kind="beam", **k)


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(32, 32), (64, 8), (6, 6), (8, 8), (12, 4), (16, 1), (40, 8), (7, 7)]


def draw(rng):
    kind = rng.choice(["rope", "append", "attn", "attn", "beam"])
    heads, kv = rng.choice(HEADS)
    hd = rng.choice([32, 48, 64, 80, 96, 128, 128, 256])
    rotation = dict(rot=rng.choice([hd, hd, hd // 2, 2 * rng.randint(1, hd // 2)]), layout=rng.choice(list(LAYOUT)),
                    norm=rng.random() < 0.5, scaling=rng.choice(list(SCALING)), factor=rng.choice([2.0, 4.0, 8.0, 32.0]))
    page = rng.choice([8, 16, 16, 32, 64, rng.randint(1, 50)])
    if kind == "rope":
        dtype = rng.choice(list(DT))
        most = 8192 * 72 * 128 * 2 // ((heads + kv) * hd * SIZE[dtype])
        return rope_case(rows=_log(rng, 1, min(most, 16384)), heads=heads, kv=kv, hd=hd, dtype=dtype,
                         far=rng.choice([0, 5000, 100000, 1000000]), **rotation)
    if kind == "append":
        seqs, dtype, cache = _log(rng, 1, 64), rng.choice(list(DT)), rng.choice(list(DT))
        most = 8192 * 80 * 128 * 2 // ((heads + 2 * kv) * hd * seqs * max(SIZE[dtype], SIZE[cache]))
        return append_case(seqs=seqs, each=1 if rng.random() < 0.4 else _log(rng, 1, max(1, min(most, 2048))),
                           start=rng.randint(0, 3000), heads=heads, kv=kv, hd=hd, page=page, layers=rng.randint(1, 3),
                           dtype=dtype, cache=cache, **rotation)
    if kind == "attn":
        dtype, cache = rng.choice([("f32", "f32"), ("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "bf16")])
        seqs = _log(rng, 1, 64)
        prefix = rng.choice([0, _log(rng, 1, 32768), _log(rng, 1, 32768), _log(rng, 1, 32768)])
        own_max = _log(rng, 1, 1024)
        work = 64 * 64 * 128 * 32768 if cache != "f32" and dtype != "f32" else 64 * 64 * 128 * 4096
        prefix = min(prefix, work // (seqs * heads * hd), 32768 * 8 * 128 * 2 // (kv * hd * SIZE[cache]))
        own_max = min(own_max, max(1, 64 * 8 * 128 * 512 // (seqs * kv * hd * SIZE[cache])))
        return attn_case(seqs=seqs, heads=heads, kv=kv, hd=hd, prefix=prefix, own_max=own_max, page=page,
                         layers=rng.randint(1, 3), dtype=dtype, cache=cache,
                         empty=rng.choice([0, 0, 1]) if seqs > 1 else 0)
    beams, vocab, dtype = rng.choice([1, 2, 3, 4, 5, 8, 16]), _log(rng, 300, 128000), rng.choice(list(DT))
    most = 24 * 8 * 128000 // (beams * vocab * SIZE[dtype])
    return beam_case(prompts=_log(rng, 1, max(1, min(most, 24))), beams=beams, vocab=vocab,
                     n_out=beams if rng.random() < 0.5 else 2 * beams, dtype=dtype,
                     ended=rng.randint(0, beams - 1), first=rng.random() < 0.3, length=rng.randint(1, 1500), page=page,
                     layers=rng.randint(1, 16), kv=rng.choice([1, 2, 8]), hd=rng.choice([48, 64, 128]),
                     cache=rng.choice(list(DT)))


# ------------------------------------------------------------------------------------------------ inputs
def _random(g, shape, dtype, std=1.0):
    """normal values of a type, in pieces so that the float form of a large cache never exists whole"""
    t = torch.empty(shape, dtype=dtype, device="cuda")
    flat = t.view(-1)
    for i in range(0, flat.numel(), 1 << 27):
        n = min(1 << 27, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, generator=g, device="cuda") * std
    return t


def _ints(g, lo, hi, shape):
    return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int32)


def _pages(g, n):
    return torch.randperm(n, generator=g, device="cuda").to(torch.int32)


def _cdiv(a, b):
    return -(-a // b)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {"rope": _prepare_rope, "append": _prepare_append, "attn": _prepare_attn, "beam": _prepare_beam}[case["kind"]](case, g)


def _rows(case, g, rows):
    """packed [q | k | v] rows as a projection leaves them, norm weights near one"""
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    s = {"case": case, "qkv": _random(g, (rows, (heads + 2 * kv) * hd), DT[case["dtype"]]),
         "q_out": torch.zeros(rows, heads * hd, dtype=DT[case["dtype"]], device="cuda"), "qw": None, "kw": None}
    if case["norm"]:
        s["qw"] = 1 + 0.1 * torch.randn(hd, generator=g, device="cuda")
        s["kw"] = 1 + 0.1 * torch.randn(hd, generator=g, device="cuda")
    if own:
        import quillm_b200 as qb

        low, high = BANDS if case["scaling"] == "bands" else RAMP
        s["plan"] = qb.RopePlan(hd, case["rot"], LAYOUT[case["layout"]], 10000.0, SCALING[case["scaling"]], case["factor"],
                                low, high, ORIG)
    return s


def _prepare_rope(case, g):
    rows = case["rows"]
    s = _rows(case, g, rows)
    s["k_out"] = torch.zeros(rows, case["kv"] * case["hd"], dtype=DT[case["dtype"]], device="cuda")
    s["pos"] = torch.arange(rows, dtype=torch.int32, device="cuda") + case["far"]
    return s


def _cache(case, g, n_pages, std=1.0, zero=False):
    shape = (case["layers"], n_pages, case["page"], case["kv"], case["hd"])
    if zero:
        kv = [torch.zeros(shape, dtype=DT[case["cache"]], device="cuda") for _ in range(2)]
    else:
        kv = [_random(g, shape, DT[case["cache"]], std) for _ in range(2)]
    s = {"k": kv[0], "v": kv[1]}
    if own:
        import quillm_b200 as qb

        s["cache"] = qb.PagedCache(kv[0], kv[1], CODE[case["cache"]], *shape)
    return s


def _prepare_append(case, g):
    seqs, each, page = case["seqs"], case["each"], case["page"]
    # sequence i holds `start` + i tokens and gets `each` more
    width = _cdiv(case["start"] + seqs + each, page)
    s = _rows(case, g, seqs * each)
    s.update(_cache(case, g, seqs * width, zero=True))
    s["table"] = _pages(g, seqs * width).view(seqs, width)
    seq = torch.arange(seqs, dtype=torch.int32, device="cuda")
    s["seq"] = seq.repeat_interleave(each)
    s["pos"] = (case["start"] + seq[:, None] + torch.arange(each, dtype=torch.int32, device="cuda")[None]).reshape(-1)
    return s


def _prepare_attn(case, g):
    seqs, page, prefix = case["seqs"], case["page"], case["prefix"]
    shared, width = _cdiv(prefix, page), _cdiv(prefix + case["own_max"], page)
    first = prefix // page  # the first table entry that own positions reach
    pages = _pages(g, shared + seqs * (width - first))
    s = {"case": case, "q": _random(g, (seqs, case["heads"] * case["hd"]), DT[case["dtype"]])}
    s.update(_cache(case, g, pages.numel()))
    s["prefix_pages"] = pages[:shared].clone()
    s["table"] = torch.zeros(seqs, width, dtype=torch.int32, device="cuda")
    s["table"][:, :shared] = s["prefix_pages"]
    s["table"][:, first:] = pages[shared:].view(seqs, -1)
    lens = prefix + _ints(g, 1, case["own_max"] + 1, (seqs,))
    lens[0] = prefix + case["own_max"]
    if case["empty"]:
        lens[seqs - case["empty"]:] = 0
    s["lens"], s["out"] = lens, torch.zeros_like(s["q"])
    if own:
        import quillm_b200 as qb

        n = qb.attn_prefix_workspace(CODE[case["dtype"]], s["cache"], seqs, case["heads"], prefix, width)
        s["workspace"] = torch.empty(n, dtype=torch.uint8, device="cuda")
    return s


def _prepare_beam(case, g):
    prompts, beams, vocab, page = case["prompts"], case["beams"], case["vocab"], case["page"]
    rows, tail = prompts * beams, case["length"] // page
    s = {"case": case, "logits": _random(g, (rows, vocab), DT[case["dtype"]], 3.0)}
    s["scores"] = -torch.rand(rows, generator=g, device="cuda") * 4 - 5
    if case["first"]:  # the first step: one live beam a prompt
        s["scores"] = torch.where(torch.arange(rows, device="cuda") % beams == 0, 0.0, -math.inf).float()
    s["finished"] = (torch.arange(rows, device="cuda") % beams < case["ended"]).to(torch.uint8)
    if case["first"]:
        s["finished"].zero_()
    s.update(_cache(case, g, prompts * (tail + 2 * beams)))
    pages = _pages(g, prompts * (tail + 2 * beams)).view(prompts, -1)
    # full pages: shared within the prompt; the page being filled: each beam's own
    full = torch.randint(0, tail + beams, (prompts, beams, tail), generator=g, device="cuda")
    s["table"] = torch.cat([pages[:, None, :].expand(-1, beams, -1).gather(2, full), pages[:, tail + beams:, None]], 2)
    s["table"] = s["table"].reshape(rows, tail + 1).contiguous()
    s["lens"] = torch.full((rows,), case["length"], dtype=torch.int32, device="cuda")
    s["parents"] = torch.zeros(prompts, case["n_out"], dtype=torch.int32, device="cuda")
    s["tokens"] = torch.zeros_like(s["parents"])
    s["out_scores"] = torch.zeros(prompts, case["n_out"], device="cuda")
    s["table_out"] = torch.zeros_like(s["table"])
    if own:
        import quillm_b200 as qb

        n = qb.beam_workspace(prompts, beams, vocab, case["n_out"])
        s["workspace"] = torch.empty(n, dtype=torch.uint8, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"rope": _own_rope, "append": _own_append, "attn": _own_attn, "beam": _own_beam}[kind](s)
    return {"rope": _plain_rope, "append": _plain_append, "attn": _plain_attn, "beam": _plain_beam}[kind](s)


def _own_rope(s):
    import quillm_b200 as qb

    c, x = s["case"], s["qkv"]
    heads, kv, hd, e = c["heads"], c["kv"], c["hd"], SIZE[c["dtype"]]
    ld, p = (heads + 2 * kv) * hd, x.data_ptr()
    qb.check(qb.cuda().qmc_qk_norm_rope(
        s["plan"].h, CODE[c["dtype"]], p, ld, s["q_out"].data_ptr(), heads * hd, heads, p + heads * hd * e, ld,
        s["k_out"].data_ptr(), kv * hd, kv, None if s["qw"] is None else s["qw"].data_ptr(),
        None if s["kw"] is None else s["kw"].data_ptr(), EPS, s["pos"].data_ptr(), c["rows"], qb.torch_stream()))
    return {"q": s["q_out"], "k": s["k_out"]}


def _own_append(s):
    import quillm_b200 as qb

    c, x = s["case"], s["qkv"]
    heads, kv, hd, e = c["heads"], c["kv"], c["hd"], SIZE[c["dtype"]]
    ld, p = (heads + 2 * kv) * hd, x.data_ptr()
    qb.check(qb.cuda().qmc_kv_append_paged(
        s["plan"].h, s["cache"].ref, c["layers"] - 1, CODE[c["dtype"]], p, ld, s["q_out"].data_ptr(), heads * hd, heads,
        p + heads * hd * e, ld, p + (heads + kv) * hd * e, ld, None if s["qw"] is None else s["qw"].data_ptr(),
        None if s["kw"] is None else s["kw"].data_ptr(), EPS, s["seq"].data_ptr(), s["pos"].data_ptr(),
        s["table"].data_ptr(), s["table"].shape[0], s["table"].shape[1], x.shape[0], qb.torch_stream()))
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _own_attn(s):
    import quillm_b200 as qb

    c, w = s["case"], s["workspace"]
    n = c["heads"] * c["hd"]
    qb.check(qb.cuda().qmc_attn_prefix(
        s["cache"].ref, c["layers"] - 1, CODE[c["dtype"]], s["q"].data_ptr(), n, s["out"].data_ptr(), n, c["heads"],
        c["seqs"], 1.0 / math.sqrt(c["hd"]), s["prefix_pages"].data_ptr(), c["prefix"], s["table"].data_ptr(),
        s["table"].shape[1], s["lens"].data_ptr(), w.data_ptr(), w.numel(), qb.torch_stream()))
    return {"out": s["out"]}


def _own_beam(s):
    import quillm_b200 as qb

    c, w, lib, stream = s["case"], s["workspace"], qb.cuda(), qb.torch_stream()
    qb.check(lib.qmc_beam_select(
        CODE[c["dtype"]], s["logits"].data_ptr(), c["vocab"], c["prompts"], c["beams"], c["vocab"], s["scores"].data_ptr(),
        s["finished"].data_ptr(), 2, c["n_out"], s["parents"].data_ptr(), s["tokens"].data_ptr(),
        s["out_scores"].data_ptr(), w.data_ptr(), w.numel(), stream))
    qb.check(lib.qmc_beam_reorder(
        s["cache"].ref, c["prompts"], c["beams"], s["parents"].data_ptr(), c["n_out"], s["lens"].data_ptr(),
        s["table"].data_ptr(), s["table_out"].data_ptr(), s["table"].shape[1], stream))
    return {"parents": s["parents"], "tokens": s["tokens"], "scores": s["out_scores"], "table": s["table_out"],
            "k": s["k"], "v": s["v"]}


def _frequencies(c):
    """radians per position of each pair, in 64 bits, and the factor on cos and sin"""
    rot, factor = c["rot"], c["factor"]
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    f = 10000.0 ** (-2.0 * i / rot)
    if c["scaling"] == "linear":
        return f / factor, 1.0
    if c["scaling"] == "bands":
        low, high = BANDS
        smooth = ((ORIG * f / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        return f * smooth + f / factor * (1 - smooth), 1.0
    if c["scaling"] == "yarn":
        slow, fast = RAMP
        at = [rot * math.log(ORIG / (b * 2 * math.pi)) / (2 * math.log(10000.0)) for b in (fast, slow)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _norm_rotate(c, x, w, cos, sin):
    """x [rows, heads, hd] in 32 bits; cos, sin [rows, 1, rot / 2]"""
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    rot = c["rot"]
    y = x.clone()
    if c["layout"] == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, a * sin + b * cos
    return y


def _plain_qk(s):
    c = s["case"]
    heads, kv, hd = c["heads"], c["kv"], c["hd"]
    f, m = _frequencies(c)
    angle = s["pos"].double()[:, None] * f
    cos, sin = ((m * t).float()[:, None, :] for t in (torch.cos(angle), torch.sin(angle)))
    x = s["qkv"].float().view(-1, heads + 2 * kv, hd)
    q = _norm_rotate(c, x[:, :heads], s["qw"], cos, sin)
    k = _norm_rotate(c, x[:, heads:heads + kv], s["kw"], cos, sin)
    return q, k, x[:, heads + kv:]


def _plain_rope(s):
    q, k, _ = _plain_qk(s)
    t = s["qkv"].dtype
    return {"q": q.flatten(1).to(t), "k": k.flatten(1).to(t)}


def _plain_append(s):
    c = s["case"]
    q, k, v = _plain_qk(s)
    pos = s["pos"].long()
    pages = s["table"][s["seq"].long(), pos // c["page"]].long()
    for pool, x in ((s["k"], k), (s["v"], v)):
        pool[c["layers"] - 1][pages, pos % c["page"]] = x.to(pool.dtype)
    return {"q": q.flatten(1).to(s["qkv"].dtype), "k": s["k"], "v": s["v"]}


def _plain_attn(s):
    c = s["case"]
    seqs, heads, kv, hd, page, prefix = c["seqs"], c["heads"], c["kv"], c["hd"], c["page"], c["prefix"]
    group, layer = heads // kv, c["layers"] - 1
    q = s["q"].float().view(seqs, kv, group, hd) / math.sqrt(hd)
    # the prefix: one product of all queries with its keys
    kp, vp = (s[n][layer][s["prefix_pages"].long()].flatten(0, 1)[:prefix].float().transpose(0, 1) for n in ("k", "v"))
    sp = (q.transpose(0, 1).flatten(1, 2) @ kp.transpose(1, 2)).view(kv, seqs, group, prefix).transpose(0, 1)
    # own positions, padded to the longest
    pos = prefix + torch.arange(c["own_max"], device="cuda")
    seen = pos < s["lens"][:, None]  # [seqs, own_max]
    slot = s["table"][:, pos // page].long() * page + pos % page
    ko, vo = (s[n][layer].flatten(0, 1)[slot].float().permute(0, 2, 1, 3) for n in ("k", "v"))
    so = torch.where(seen[:, None, None, :], q @ ko.transpose(2, 3), -math.inf)
    m = so.amax(-1, keepdim=True)
    if prefix:
        m = torch.maximum(m, sp.amax(-1, keepdim=True))
    m = torch.where(m == -math.inf, 0.0, m)
    ep, eo = torch.exp(sp - m), torch.exp(so - m)
    total = ep.sum(-1, keepdim=True) + eo.sum(-1, keepdim=True)
    o = (ep.transpose(0, 1).flatten(1, 2) @ vp).view(kv, seqs, group, hd).transpose(0, 1) + eo @ vo
    o = torch.where((s["lens"] > 0)[:, None, None, None], o / total, 0.0)
    return {"out": o.reshape(seqs, heads * hd).to(s["q"].dtype)}


def _plain_beam(s):
    c = s["case"]
    prompts, beams, vocab, page = c["prompts"], c["beams"], c["vocab"], c["page"]
    x = s["logits"].double()
    m = x.amax(1, keepdim=True)
    logp = x - (m + torch.log(torch.exp(x - m).sum(1, keepdim=True)))
    cum = s["scores"].double()[:, None]
    token = torch.arange(vocab, device="cuda")
    ended = torch.where(token == 2, cum, -math.inf)  # a finished beam goes on as it is
    score = torch.where(s["finished"].bool()[:, None], ended, cum + logp).view(prompts, beams * vocab)
    score, at = torch.sort(score, dim=1, descending=True, stable=True)
    score, at = score[:, :c["n_out"]].float(), at[:, :c["n_out"]]
    parents = at // vocab
    # states: rows of the table by parent; the first child keeps the page being filled, the others copy it
    # into the pages of beams without a child
    par, tail, filled = parents[:, :beams], c["length"] // page, c["length"] % page
    same = par[:, :, None] == par[:, None, :]
    first = ~torch.tril(same, -1).any(2)
    childless = ~(par[:, :, None] == torch.arange(beams, device="cuda")).any(1)
    free = torch.argsort((~childless).int(), dim=1, stable=True)
    owner = torch.where(first, par, free.gather(1, ((~first).int().cumsum(1) - 1).clamp(min=0)))
    table = s["table"].view(prompts, beams, -1).gather(1, par[:, :, None].expand(-1, -1, tail + 1))
    last = s["table"].view(prompts, beams, -1)[:, :, tail]
    source, target = last.gather(1, par), last.gather(1, owner)
    table[:, :, tail] = target
    if filled:
        for pool in (s["k"], s["v"]):
            pool[:, target.flatten().long(), :filled] = pool[:, source.flatten().long(), :filled]
    return {"parents": parents.int(), "tokens": (at % vocab).int(), "scores": score, "table": table.reshape(prompts * beams, -1),
            "k": s["k"], "v": s["v"]}


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    c = case
    if c["kind"] in ("rope", "append"):
        e, hd = SIZE[c["dtype"]], c["hd"]
        rows = c["rows"] if c["kind"] == "rope" else c["seqs"] * c["each"]
        each = (c["heads"] + c["kv"]) * hd
        total = rows * (2 * each * e + 4)
        if c["kind"] == "append":
            kvd = c["kv"] * hd
            total = rows * (2 * c["heads"] * hd * e + 2 * kvd * (e + SIZE[c["cache"]]) + 12)
        return {"bytes": total, "flops": rows * each * (3 + (4 if c["norm"] else 0))}
    if c["kind"] == "attn":
        live = c["seqs"] - c["empty"]
        tokens = live * (c["own_max"] + 1) / 2  # own lengths are spread evenly
        kvd = c["kv"] * c["hd"]
        return {"bytes": 2 * (c["prefix"] + tokens) * kvd * SIZE[c["cache"]] + 2 * c["seqs"] * c["heads"] * c["hd"] * SIZE[c["dtype"]],
                "flops": 4 * c["heads"] * c["hd"] * (live * c["prefix"] + tokens)}
    live = c["prompts"] * (1 if c["first"] else c["beams"] - c["ended"])
    rows = c["prompts"] * c["beams"]
    # about a third of the beams copy the filled part of a page
    copied = rows / 3 * c["layers"] * 2 * (c["length"] % c["page"]) * c["kv"] * c["hd"] * SIZE[c["cache"]]
    return {"bytes": live * c["vocab"] * SIZE[c["dtype"]] + 2 * copied + 8 * rows * (c["length"] // c["page"] + 1),
            "flops": 4 * live * c["vocab"]}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "append": _exact_append, "attn": _exact_attn, "beam": _exact_beam}[case["kind"]](case, s)


def _exact_heads(c, x, w, turn):
    """x [rows, heads, hd] doubles; turn [rows, rot / 2] complex"""
    if w is not None:
        x = x / (x.square().sum(2, keepdim=True) / c["hd"] + EPS).sqrt() * w.double()
    half, rot = c["rot"] // 2, c["rot"]
    pairs = x[..., :rot].unflatten(2, (2, half)).transpose(2, 3) if c["layout"] == "half" else x[..., :rot].unflatten(2, (half, 2))
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn[:, None, :])
    z = z.transpose(2, 3) if c["layout"] == "half" else z
    return torch.cat([z.flatten(2), x[..., rot:]], 2)


def _exact_turn(c, pos):
    rot, out, m = c["rot"], [], 1.0
    if c["scaling"] == "yarn":
        m = 1.0 + math.log(c["factor"]) / 10.0
        edge = lambda turns: rot / 2 * math.log(ORIG / (2 * math.pi * turns), 10000.0)  # noqa: E731
        lo, hi = max(0, math.floor(edge(RAMP[1]))), min(rot - 1, math.ceil(edge(RAMP[0])))
    for i in range(rot // 2):
        f = math.exp(-math.log(10000.0) * 2 * i / rot)
        if c["scaling"] == "linear":
            f /= c["factor"]
        elif c["scaling"] == "bands":
            turns = ORIG / (2 * math.pi / f)
            part = min(1.0, max(0.0, (turns - BANDS[0]) / (BANDS[1] - BANDS[0])))
            f = part * f + (1 - part) * f / c["factor"]
        elif c["scaling"] == "yarn":
            part = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            f = part * f / c["factor"] + (1 - part) * f
        out.append(f)
    angle = pos.double()[:, None] * torch.tensor(out, dtype=torch.float64, device=pos.device)
    return torch.polar(torch.full_like(angle, m), angle)


def _exact_qk(c, s):
    heads, kv, hd = c["heads"], c["kv"], c["hd"]
    x, turn = s["qkv"].double().unflatten(1, (heads + 2 * kv, hd)), _exact_turn(c, s["pos"])
    return _exact_heads(c, x[:, :heads], s["qw"], turn), _exact_heads(c, x[:, heads:heads + kv], s["kw"], turn), x[:, heads + kv:]


def _exact_rope(c, s):
    q, k, _ = _exact_qk(c, s)
    return {"q": q.flatten(1), "k": k.flatten(1)}


def _exact_append(c, s):
    q, k, v = _exact_qk(c, s)
    pools = []
    for pool, x in ((s["k"].double(), k), (s["v"].double(), v)):
        flat = pool[c["layers"] - 1].flatten(0, 1)
        for i in range(c["seqs"]):  # sequence i's tokens follow one another
            at = torch.arange(c["each"], device="cuda") + c["start"] + i
            flat[s["table"][i][at // c["page"]].long() * c["page"] + at % c["page"]] = x[i * c["each"]:(i + 1) * c["each"]]
        pools.append(pool)
    return {"q": q.flatten(1), "k": pools[0], "v": pools[1]}


def _exact_attn(c, s):
    heads, kv, hd, prefix, page = c["heads"], c["kv"], c["hd"], c["prefix"], c["page"]
    out = torch.zeros(c["seqs"], heads, hd, dtype=torch.float64, device="cuda")
    keys, values = (s[n][c["layers"] - 1].flatten(0, 1) for n in ("k", "v"))
    for b, n in enumerate(s["lens"].tolist()):
        if not n:
            continue
        at = torch.arange(n, device="cuda")
        pages = s["table"][b].clone()
        pages[:prefix // page] = s["prefix_pages"][:prefix // page]
        slot = pages[at // page].long() * page + at % page
        if prefix % page:  # the prefix's last page is its own, the sequence goes on in another
            shared = (at >= prefix // page * page) & (at < prefix)
            slot = torch.where(shared, s["prefix_pages"][-1].long() * page + at % page, slot)
        for h in range(kv):
            q = s["q"][b].double().view(kv, -1, hd)[h]
            p = torch.softmax(q @ keys[slot, h].double().T / math.sqrt(hd), 1)
            out[b].view(kv, -1, hd)[h] = p @ values[slot, h].double()
    return {"out": out.flatten(1)}


def _exact_beam(c, s):
    scores, parents, tokens = [], [], []
    for p in range(c["prompts"]):
        rows = []
        for b in range(p * c["beams"], (p + 1) * c["beams"]):
            row = torch.log_softmax(s["logits"][b].double(), 0) + s["scores"][b].double()
            if s["finished"][b]:
                row = torch.full_like(row, -math.inf)
                row[2] = s["scores"][b].double()
            rows.append(row)
        flat = torch.cat(rows)
        at = torch.argsort(flat, descending=True, stable=True)[:c["n_out"]]
        scores.append(flat[at])
        parents.append((at // c["vocab"]).int())
        tokens.append((at % c["vocab"]).int())
    return {"parents": torch.stack(parents), "tokens": torch.stack(tokens), "scores": torch.stack(scores), "table": None,
            "k": None, "v": None}
