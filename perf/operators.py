"""Measured cases of the paged 8-bit key/value cache and of draft verification.

Operators:
  attend   attention of query rows over the 8-bit cache (one scale for each
           block of 16 tokens and KV head)
  append   float key/value rows quantised into the cache, and read back as the
           values the cache now stands for
  pages    fork / resize, compact and copy: bookkeeping of the cache's pages
  verify   drafted tokens checked against the target's probabilities

`own` false: elementary torch operations; true: the framework's calls.
"""
import importlib
import math
import random

import numpy as np
import torch

own = False

BLOCK = 16
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_context = []


def _hale():
    return importlib.import_module("hale-token_b200")


def _ctx():
    if not _context:
        _context.append(_hale().Context(torch.cuda.current_device()))
    return _context[0]


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _attend(name, seqs, run, lo, hi, nh, nkv, hd, page, dtype, window=0):
    c = dict(op="attend", seqs=seqs, run=run, lo=lo, hi=hi, nh=nh, nkv=nkv, hd=hd, page=page, dtype=dtype, window=window)
    return dict(c, name=name) if name else c


def _append(name, seqs, run, lo, hi, nkv, hd, page, dtype):
    c = dict(op="append", seqs=seqs, run=run, lo=lo, hi=hi, nkv=nkv, hd=hd, page=page, dtype=dtype)
    return dict(c, name=name) if name else c


def _pages(name, kind, seqs, lo, hi, nkv, hd, page, layers, width=2):
    c = dict(op="pages", kind=kind, seqs=seqs, lo=lo, hi=hi, nkv=nkv, hd=hd, page=page, layers=layers, width=width)
    return dict(c, name=name) if name else c


def _verify(name, seqs, drafts, vocab, dtype, probs, temperature):
    c = dict(op="verify", seqs=seqs, drafts=drafts, vocab=vocab, dtype=dtype, probs=probs, temperature=temperature)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user's chat: the latency of a single token's attention (Qwen3-30B-A3B heads)
        _attend("attend one chat", 1, 1, 517, 517, 32, 4, 128, 64, "f32"),
        # a server's decode step over requests of every age (Mixtral heads)
        _attend("attend batch decode", 64, 1, 1, 8191, 32, 8, 128, 64, "bf16"),
        # few requests with very long documents
        _attend("attend long documents", 3, 1, 90001, 131071, 32, 4, 128, 128, "f32"),
        # the rows of drafted tokens checked in one step, sliding window
        _attend("attend drafted rows", 16, 5, 700, 6001, 32, 4, 128, 16, "f16", 4000),
        # a prompt's chunk behind a long history
        _attend("attend prompt chunk", 2, 2048, 5000, 8192, 32, 4, 128, 64, "bf16"),
        # one decode step's new rows, most of them inside a block that is there already
        _append("append decode step", 64, 1, 1, 4000, 8, 128, 64, "bf16"),
        # whole prompts of different lengths
        _append("append prompts", 9, 1500, 0, 40, 4, 128, 64, "f32"),
        # parallel samples of running requests: fork, one step each, dropped again
        _pages("pages fork and step", "fork", 32, 100, 3000, 4, 128, 64, 8, 4),
        # half the requests ended: the rest moves together, new requests come in
        _pages("pages compact", "compact", 48, 500, 4000, 4, 128, 64, 16),
        # pages duplicated for another owner
        _pages("pages copy", "copy", 6, 65, 400, 8, 128, 32, 4),
        # one user's speculative step, draft without probabilities (a lookup draft)
        _verify("verify one lookup", 1, 4, 32000, "f32", False, 0.7),
        # a server's speculative step with a draft model (Qwen3-30B-A3B vocabulary)
        _verify("verify batch", 48, 5, 151936, "bf16", True, 1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "pages", "verify"])
    nkv, hd = rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 96, 128, 128, 192, 256])
    page, dtype = rng.choice([16, 32, 64, 128]), rng.choice(["f32", "f16", "bf16"])
    if op == "attend":
        group, run = rng.choice([1, 2, 3, 4, 7, 8, 16]), rng.choice([1, 1, 2, 5, 9, _log(rng, 16, 1500)])
        hi = _log(rng, run, 60000)
        # the largest listed case has about 2e10 bytes x queries of work: stay well below
        most = max(1, int(3e8 / (hi * nkv * hd * (1 + run * group / 512))))
        seqs = _log(rng, 1, min(128, most))
        return _attend(None, seqs, run, rng.randint(run, hi), hi, nkv * group, nkv, hd, page, dtype,
                       rng.choice([0, 0, 0, rng.randint(1, hi)]))
    if op == "append":
        run = rng.choice([1, 1, 3, _log(rng, 4, 3000)])
        seqs = _log(rng, 1, max(1, min(200, int(1.4e7 / (run * nkv * hd)))))
        lo = rng.randint(0, 300)
        return _append(None, seqs, run, lo, lo + rng.randint(0, 700), nkv, hd, page, dtype)
    if op == "pages":
        kind, lo = rng.choice(["fork", "compact", "copy"]), rng.randint(1, 600)
        hi = lo + _log(rng, 1, 2000)
        layers = rng.choice([1, 2, 4])
        seqs = _log(rng, 2, max(2, min(64, int(3e8 / (hi * nkv * hd * layers)))))
        return _pages(None, kind, seqs, lo, hi, nkv, hd, page, layers, rng.choice([1, 2, 3]))
    vocab = _log(rng, 1000, 152000)
    seqs = _log(rng, 1, max(1, min(100, int(4e7 / vocab / 4))))
    return _verify(None, seqs, rng.randint(1, 8), vocab, dtype, rng.random() < 0.6, round(rng.uniform(0.5, 1.3), 2))


def _lengths(case):
    """A length for each sequence in lo..hi, from the case alone."""
    r = random.Random(case["seqs"] * 1000003 + case["lo"] * 1009 + case["hi"])
    return [case["hi"]] + [r.randint(case["lo"], case["hi"]) for _ in range(case["seqs"] - 1)]


def _runs(case):
    """New rows for each sequence: `run` for the first, run/2..run for the others."""
    r = random.Random(case["seqs"] * 7919 + case["run"])
    return [case["run"]] + [r.randint((case["run"] + 1) // 2, case["run"]) for _ in range(case["seqs"] - 1)]


def _pages_of(n, page):
    return (n + page - 1) // page


def work(case):
    el = 4 if case.get("dtype") == "f32" else 2
    if case["op"] == "attend":
        held, pairs, rows = 0, 0, 0
        for n, run in zip(_lengths(case), _runs(case)):
            run = min(run, n)
            w = case["window"] or n
            first = max(0, n - run - w + 1)
            held += n - first
            pairs += sum(min(w, n - i) for i in range(run))
            rows += run
        token = case["nkv"] * (case["hd"] + 4.0 / BLOCK)
        return {"bytes": 2 * held * token + 2 * rows * case["nh"] * case["hd"] * el + 4 * rows * case["nh"],
                "flops": 4.0 * pairs * case["nh"] * case["hd"]}
    if case["op"] == "append":
        rows = sum(_runs(case))
        values = 2 * rows * case["nkv"] * case["hd"]
        # float rows in, codes out; codes in, f32 values out
        return {"bytes": values * (el + 1 + 1 + 4), "flops": 3.0 * values}
    if case["op"] == "pages":
        lens, page = _lengths(case), case["page"]
        each = 2 * case["layers"] * case["nkv"] * page * (case["hd"] + 4.0 / BLOCK)
        if case["kind"] == "fork":  # every sharer of a partly filled last page but one gets its own
            moved = sum(case["width"] for n in lens if n % page)
        elif case["kind"] == "compact":
            half = [_pages_of(n, page) for n in lens]
            moved = min(sum(half[0::2]), sum(half[1::2]))
        else:
            moved = sum(_pages_of(n, page) for n in lens)
        ints = sum(_pages_of(n, page) for n in lens)
        return {"bytes": 2 * moved * each + 8 * ints, "flops": float(ints)}
    rows = case["seqs"] * (case["drafts"] + 1)
    # every target row, and the draft's row at the one refused place
    return {"bytes": rows * case["vocab"] * el + (case["seqs"] * case["vocab"] * 4 if case["probs"] else 0),
            "flops": 3.0 * rows * case["vocab"]}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _quantise(x):
    """Codes and scales of [..., tokens, hd] floats, 16 tokens to a scale."""
    b = x.unflatten(-2, (x.shape[-2] // BLOCK, BLOCK))
    scale = (b.abs().amax((-1, -2)).double() / 127).float()
    codes = torch.round(b / scale[..., None, None]).clamp_(-127, 127)
    return codes.flatten(-3, -2).to(torch.int8), scale


def _cache(case, g, lens, extra, layers=1, n_seqs=None):
    """A filled cache: sequence b's pages scattered over the pool, `extra` pages free."""
    nkv, hd, page = case["nkv"], case["hd"], case["page"]
    need = [_pages_of(n, page) for n in lens]
    n_seqs = n_seqs or len(lens)
    n_pages, max_pages = sum(need) + extra, max(need) + 4
    k = torch.empty((layers, n_pages, nkv, page, hd), dtype=torch.int8, device="cuda")
    v = torch.empty_like(k)
    ks = torch.empty((layers, n_pages, nkv, page // BLOCK), dtype=torch.float32, device="cuda")
    vs = torch.empty_like(ks)
    # keys have a few channels that are much larger than the others, values less so
    channel = torch.exp(0.6 * torch.randn((nkv, 1, hd), device="cuda", generator=g))
    step = max(1, (1 << 26) // (nkv * page * hd))
    for l in range(layers):
        for p in range(0, n_pages, step):
            shape = (min(step, n_pages - p), nkv, page, hd)
            k[l, p:p + step], ks[l, p:p + step] = _quantise(torch.randn(shape, device="cuda", generator=g) * channel)
            token = torch.exp(0.5 * torch.randn(shape[:3] + (1,), device="cuda", generator=g))
            v[l, p:p + step], vs[l, p:p + step] = _quantise(torch.randn(shape, device="cuda", generator=g) * token)
    order = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((n_seqs, max_pages), -1, dtype=torch.int32, device="cuda")
    count = torch.zeros(n_seqs, dtype=torch.int64)
    count[:len(need)] = torch.tensor(need)
    held = torch.arange(max_pages)[None, :] < count[:, None]
    table[held.cuda()] = order[:sum(need)]
    refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    refs[order[:sum(need)].long()] = 1
    length = torch.zeros(n_seqs, dtype=torch.int32, device="cuda")
    length[:len(lens)] = torch.tensor(lens, dtype=torch.int32)
    return {"k": k, "v": v, "k_scale": ks, "v_scale": vs, "table": table, "lens": length, "refs": refs}


def _rows(lens, runs):
    """(sequence, position) of every new row, the last `run` positions of each sequence."""
    seqs = [b for b, r in enumerate(runs) for _ in range(r)]
    pos = [n - r + i for n, r in zip(lens, runs) for i in range(r)]
    place = [i for r in runs for i in range(r)]
    return [torch.tensor(t, dtype=torch.int32, device="cuda") for t in (seqs, pos, place)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    st = {"case": case}

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    if case["op"] == "attend":
        lens = _lengths(case)
        runs = [min(r, n) for r, n in zip(_runs(case), lens)]
        st["cache"] = _cache(case, g, lens, 3)
        st["seqs"], st["pos"], st["place"] = _rows(lens, runs)
        n = len(st["seqs"])
        st["q"] = (2.0 * randn(n, case["nh"], case["hd"])).to(TYPES[case["dtype"]])
        st["out"] = torch.empty_like(st["q"])
        st["lse"] = torch.empty((n, case["nh"]), device="cuda")
        st["scale"] = case["hd"] ** -0.5
    elif case["op"] == "append":
        lens, runs = _lengths(case), _runs(case)
        full = [n + r for n, r in zip(lens, runs)]
        st["cache"] = _cache(case, g, full, 3)
        st["seqs"], st["pos"], st["place"] = _rows(full, runs)
        n = len(st["seqs"])
        channel = torch.exp(0.6 * randn(case["nkv"], case["hd"]))
        st["new_k"] = (1.2 * randn(n, case["nkv"], case["hd"]) * channel).to(TYPES[case["dtype"]])
        st["new_v"] = (1.2 * randn(n, case["nkv"], case["hd"])).to(TYPES[case["dtype"]])
        st["k_out"] = torch.empty((n, case["nkv"], case["hd"]), device="cuda")
        st["v_out"] = torch.empty_like(st["k_out"])
    elif case["op"] == "pages":
        lens, page, B, w = _lengths(case), case["page"], case["seqs"], case["width"]
        total = sum(_pages_of(n, page) for n in lens)
        st["cache"] = _cache(case, g, lens, {"fork": 2 * B * (w + 1) + 2, "compact": 5, "copy": total + 1}[case["kind"]],
                             case["layers"], B * (w + 1))

        def ints(t):
            return torch.tensor(t, dtype=torch.int32, device="cuda")

        if case["kind"] == "fork":
            parents, children = list(range(B)), list(range(B, B * (w + 1)))
            st["parents"], st["children"] = ints(parents * w), ints(children)
            st["all"], st["grown"] = ints(parents + children), ints([lens[s % B] + 1 for s in parents + children])
            st["back"] = ints(lens + [0] * len(children))
        elif case["kind"] == "compact":
            st["sets"] = [(ints(range(h, B, 2)), ints(lens[h::2])) for h in (0, 1)]
            st["turn"] = 0
            st["zero"] = ints([0] * B)
            st["remap"] = torch.empty((2, len(st["cache"]["refs"])), dtype=torch.int32, device="cuda")
            st["live"] = torch.empty(1, dtype=torch.int32, device="cuda")
        else:
            st["src"] = torch.nonzero(st["cache"]["refs"] == 1)[:, 0].to(torch.int32)
            st["dst"] = torch.nonzero(st["cache"]["refs"] == 0)[:total, 0].to(torch.int32)
    else:
        B, K, V, dt = case["seqs"], case["drafts"], case["vocab"], TYPES[case["dtype"]]
        base = 2.2 * randn(B, K + 1, V)
        st["logits"] = base.to(dt)
        st["probs"] = None
        if case["probs"]:
            st["probs"] = torch.softmax((base[:, :K] + 0.6 * randn(B, K, V)) / case["temperature"], -1)
            st["draft"] = torch.multinomial(st["probs"].view(B * K, V), 1, generator=g).view(B, K).to(torch.int32)
        else:
            p = torch.softmax(base[:, :K] / (0.35 * case["temperature"]), -1)
            st["draft"] = torch.multinomial(p.view(B * K, V), 1, generator=g).view(B, K).to(torch.int32)
        st["n_draft"] = torch.randint((K + 1) // 2, K + 1, (B,), device="cuda", generator=g).to(torch.int32)
        st["u"] = torch.rand((B, K + 1), device="cuda", generator=g)
        st["tokens"] = torch.empty((B, K + 1), dtype=torch.int32, device="cuda")
        st["count"] = torch.empty(B, dtype=torch.int32, device="cuda")
        st["logp"] = torch.empty((B, K + 1), device="cuda")
    if own and "cache" in st:
        st["kv"] = _hale().Kv8(_ctx(), **st["cache"])
    elif own:
        _ctx()
    return st


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _flat(c, name, seqs):
    """[len(seqs), nkv, max_pages * page, hd] f32 values of the sequences' pages (missing pages: page 0)."""
    ids = c["table"][seqs].long().clamp(min=0)
    codes, scale = c[name][0][ids], c[name + "_scale"][0][ids]
    x = codes.float().unflatten(3, (scale.shape[-1], BLOCK)) * scale[..., None, None]
    return x.flatten(3, 4).transpose(1, 2).flatten(2, 3)


def _plain_attend(st):
    case, c = st["case"], st["cache"]
    B, run, nh, nkv, hd = case["seqs"], case["run"], case["nh"], case["nkv"], case["hd"]
    seqs, place = st["seqs"].long(), st["place"].long()
    q = torch.zeros((B, run, nh, hd), device="cuda")
    q[seqs, place] = st["q"].float()
    pos = torch.full((B, run), -1, dtype=torch.int64, device="cuda")
    pos[seqs, place] = st["pos"].long()
    every = torch.arange(B, device="cuda")
    k, v = _flat(c, "k", every), _flat(c, "v", every)
    t = torch.arange(k.shape[2], device="cuda")
    seen = t <= pos[..., None]
    if case["window"]:
        seen &= t > pos[..., None] - case["window"]
    q = q.view(B, run, nkv, nh // nkv, hd).permute(0, 2, 3, 1, 4).reshape(B, nkv, nh // nkv * run, hd)
    s = (q @ k.transpose(-1, -2)).view(B, nkv, nh // nkv, run, -1).mul_(st["scale"])
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    e = s.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    o = (e.flatten(2, 3) @ v).view(B, nkv, nh // nkv, run, hd) / total.clamp(min=1e-37)
    lse = (top + total.log())[..., 0]
    o = o.permute(0, 3, 1, 2, 4).reshape(B, run, nh, hd)[seqs, place]
    lse = lse.permute(0, 3, 1, 2).reshape(B, run, nh)[seqs, place]
    return o.to(st["q"].dtype), lse


def _plain_append(st):
    c, seqs, pos = st["cache"], st["seqs"].long(), st["pos"].long()
    page = st["case"]["page"]
    ids = c["table"][seqs, pos // page].long()
    slot, block = pos % page, (pos % page) // BLOCK
    # the blocks that are written, and each row's place among them
    blocks, which = torch.unique(ids * (page // BLOCK) + block, return_inverse=True)
    bp, bb = blocks // (page // BLOCK), blocks % (page // BLOCK)
    outs = []
    for name, x in (("k", st["new_k"].float()), ("v", st["new_v"].float())):
        codes, scale = c[name][0], c[name + "_scale"][0]
        n, nkv, hd = x.shape
        amax = torch.zeros((len(blocks), nkv), device="cuda")
        amax.index_reduce_(0, which, x.abs().amax(-1), "amax")
        fresh = torch.zeros(len(blocks), dtype=torch.bool, device="cuda")
        fresh[which[pos % BLOCK == 0]] = True
        old = torch.where(fresh[:, None], 0.0, scale[bp, :, bb])
        want = (amax.double() / 127).float()
        want = torch.where(amax > 0, want.clamp(min=2.0 ** -100), 0.0)
        new = torch.maximum(old, want)
        rows = (bb * BLOCK)[:, None] + torch.arange(BLOCK, device="cuda")
        held = codes[bp[:, None], :, rows]
        grown = new > old
        ratio = held.double() * (old.double())[:, None, :, None] / torch.where(grown, new, 1.0).double()[:, None, :, None]
        codes[bp[:, None], :, rows] = torch.where(grown[:, None, :, None], torch.round(ratio), held.double()).to(torch.int8)
        scale[bp, :, bb] = new
        s = new[which]
        value = torch.round(x.double() / torch.where(s > 0, s, 1.0).double()[..., None]).clamp(-127, 127)
        codes[ids, :, slot] = value.to(torch.int8)
        outs.append(codes[ids, :, slot].float() * scale[ids, :, block][..., None])
    return tuple(outs)


def _copy(c, src, dst):
    for name in ("k", "v", "k_scale", "v_scale"):
        c[name][:, dst] = c[name][:, src]


def _plain_resize(c, seqs, new):
    page = c["k"].shape[3]
    seqs, new = seqs.long(), new.long()
    old = c["lens"][seqs].long()
    po, pn = (old + page - 1) // page, (new + page - 1) // page
    rows, refs = c["table"][seqs].long(), c["refs"]
    j = torch.arange(rows.shape[1], device="cuda")[None, :]
    drop = (j >= pn[:, None]) & (j < po[:, None])
    gone = rows[drop]
    refs.index_add_(0, gone, torch.full_like(gone, -1, dtype=torch.int32))
    rows[drop] = -1
    grow = new > old
    partial = grow & (old % page != 0)
    last = rows.gather(1, (po - 1).clamp(min=0)[:, None])[:, 0]
    place = torch.arange(len(seqs), device="cuda")
    before = ((last[:, None] == last[None, :]) & partial[None, :] & (place[None, :] < place[:, None])).sum(1)
    own_page = partial & (refs[last.clamp(min=0)].long() - before > 1)
    left = last[own_page]
    refs.index_add_(0, left, torch.full_like(left, -1, dtype=torch.int32))
    demand = own_page.long() + torch.where(grow, pn - po, 0)
    at = demand.cumsum(0) - demand
    free = torch.nonzero(refs == 0)[:, 0]
    fresh = free[at[own_page]]
    _copy(c, left, fresh)
    rows[own_page, (po - 1)[own_page]] = fresh
    refs[fresh] = 1
    add = (j >= po[:, None]) & (j < pn[:, None]) & grow[:, None]
    more = free[(at + own_page.long())[:, None].add(j - po[:, None])[add]]
    rows[add] = more
    refs[more] = 1
    c["table"][seqs] = rows.to(torch.int32)
    c["lens"][seqs] = new.to(torch.int32)


def _plain_fork(c, parents, children):
    parents, children, refs = parents.long(), children.long(), c["refs"]
    gone = c["table"][children]
    gone = gone[gone >= 0].long()
    refs.index_add_(0, gone, torch.full_like(gone, -1, dtype=torch.int32))
    rows = c["table"][parents]
    held = rows[rows >= 0].long()
    refs.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    c["table"][children] = rows
    c["lens"][children] = c["lens"][parents]


def _plain_compact(c, remap, live):
    refs = c["refs"]
    used = refs > 0
    n = int(used.sum())
    at = torch.arange(len(refs), device="cuda")
    holes, movers = at[:n][~used[:n]], at[n:][used[n:]]
    remap[0] = torch.where(used, at, -1).to(torch.int32)
    remap[0, movers] = holes.to(torch.int32)
    remap[1] = torch.where(at < n, at, -1).to(torch.int32)
    remap[1, holes] = movers.to(torch.int32)
    _copy(c, movers, holes)
    refs[holes] = refs[movers]
    refs[movers] = 0
    t = c["table"]
    c["table"].copy_(torch.where(t >= 0, remap[0][t.long().clamp(min=0)], t))
    live.fill_(n)


def _plain_verify(st):
    case, T = st["case"], st["case"]["temperature"]
    B, K, V = case["seqs"], case["drafts"], case["vocab"]
    x = st["logits"].double() / T
    x = x - x.amax(-1, keepdim=True)
    e = x.exp()
    total = e.sum(-1, keepdim=True)
    draft, n, u = st["draft"].long(), st["n_draft"].long(), st["u"].double()
    rank = torch.arange(K + 1, device="cuda")[None, :]
    p_x = (e[:, :K].gather(-1, draft[..., None]) / total[:, :K])[..., 0]
    q_x = st["probs"].gather(-1, draft[..., None])[..., 0].double() if case["probs"] else torch.ones_like(p_x)
    took = (u[:, :K] * q_x < p_x) & (rank[:, :K] < n[:, None])
    count = took.long().cumprod(1).sum(1)
    every = torch.arange(B, device="cuda")
    mass = e[every, count] / total[every, count]
    refused = count < n
    at = count.clamp(max=K - 1)
    if case["probs"]:
        q = st["probs"][every, at].double()
    else:
        q = torch.zeros_like(mass).scatter_(1, draft[every, at][:, None], 1.0)
    rest = (mass - q).clamp(min=0)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, mass)
    mass = torch.where(refused[:, None], rest, mass)
    cum = mass.cumsum(1)
    # the lowest index whose cumulated mass is above the number drawn
    last = (cum > (u[:, K] * cum[:, -1])[:, None]).to(torch.int8).argmax(1)
    tokens = torch.where(rank < count[:, None], torch.nn.functional.pad(draft, (0, 1)), -1)
    tokens[every, count] = last
    logp = (x - total.log()).gather(-1, tokens.clamp(min=0)[..., None])[..., 0]
    logp = torch.where(tokens >= 0, logp, 0.0)
    return tokens.to(torch.int32), (count + 1).to(torch.int32), logp.float()


def _held(c):
    """The cache's whole state; codes as the words they are stored in."""
    return {"table": c["table"], "lens": c["lens"], "refs": c["refs"], "k": c["k"].view(torch.int64),
            "v": c["v"].view(torch.int64), "k_scale": c["k_scale"], "v_scale": c["v_scale"]}


def run(st):
    case = st["case"]
    if case["op"] == "attend":
        if not own:
            return _plain_attend(st)
        st["kv"].attention(0, st["q"], st["out"], st["pos"], st["seqs"], scale=st["scale"], window=case["window"],
                           run=case["run"], lse=st["lse"])
        return st["out"], st["lse"]
    if case["op"] == "append":
        if not own:
            return _plain_append(st)
        st["kv"].append(0, st["new_k"], st["new_v"], st["pos"], st["seqs"])
        st["kv"].read(0, st["k_out"], st["v_out"], st["pos"], st["seqs"])
        return st["k_out"], st["v_out"]
    if case["op"] == "verify":
        if not own:
            return _plain_verify(st)
        _hale().verify_drafts(_ctx(), st["logits"], st["draft"], st["u"], st["tokens"], st["count"],
                              draft_probs=st["probs"], n_draft=st["n_draft"], temperature=case["temperature"],
                              out_logp=st["logp"])
        return st["tokens"], st["count"], st["logp"]
    c, kv = st["cache"], st.get("kv")
    if case["kind"] == "fork":
        if not own:
            _plain_fork(c, st["parents"], st["children"])
            _plain_resize(c, st["all"], st["grown"])
            _plain_resize(c, st["all"], st["back"])
        else:
            kv.fork(st["parents"], st["children"])
            kv.resize(st["grown"], st["all"])
            kv.resize(st["back"], st["all"])
        return _held(c)
    if case["kind"] == "copy":
        if not own:
            _copy(c, st["src"].long(), st["dst"].long())
        else:
            kv.copy_pages(st["src"], st["dst"])
        return _held(c)
    ended, lens = st["sets"][st["turn"]]
    st["turn"] ^= 1
    if not own:
        _plain_resize(c, ended, st["zero"][:len(ended)])
        _plain_compact(c, st["remap"], st["live"])
        _plain_resize(c, ended, lens)
    else:
        kv.resize(st["zero"][:len(ended)], ended)
        kv.compact(st["remap"], st["live"])
        kv.resize(lens, ended)
    return dict(_held(c), remap=st["remap"], live=st["live"])


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_attend(st):
    case, c = st["case"], st["cache"]
    nh, nkv, page = case["nh"], case["nkv"], case["page"]
    group = nh // nkv
    seqs, pos, table = st["seqs"].cpu().numpy(), st["pos"].cpu().numpy(), c["table"].cpu().numpy()
    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(st["lse"].shape, dtype=torch.float64, device="cuda")
    for b in range(case["seqs"]):
        rows = np.flatnonzero(seqs == b)
        n = int(pos[rows].max()) + 1
        ids = torch.tensor(table[b, :_pages_of(n, page)], dtype=torch.int64, device="cuda")
        p = torch.tensor(pos[rows], dtype=torch.int64, device="cuda")
        t = torch.arange(n, device="cuda")
        hidden = t[None, :] > p[:, None]
        if case["window"]:
            hidden |= t[None, :] <= p[:, None] - case["window"]
        r = torch.tensor(rows, device="cuda")
        for h in range(nkv):
            kv = []
            for name in ("k", "v"):
                f = c[name + "_scale"][0][ids, h].double().repeat_interleave(BLOCK, 1)
                kv.append((c[name][0][ids, h].double() * f[..., None]).reshape(-1, case["hd"])[:n])
            for i in range(0, len(rows), 512):
                part = r[i:i + 512]
                q = st["q"][part, h * group:(h + 1) * group].double()
                s = torch.einsum("rgd,td->rgt", q, kv[0]) * st["scale"]
                s = s.masked_fill(hidden[i:i + 512, None], -math.inf)
                z = torch.logsumexp(s, -1)
                out[part, h * group:(h + 1) * group] = torch.einsum("rgt,td->rgd", torch.exp(s - z[..., None]), kv[1])
                lse[part, h * group:(h + 1) * group] = z
    return out, lse


def _exact_append(st):
    case, c = st["case"], st["cache"]
    page, nkv, hd = case["page"], case["nkv"], case["hd"]
    seqs, pos, table = st["seqs"].cpu().numpy(), st["pos"].cpu().numpy(), c["table"].cpu().numpy()
    ids = table[seqs, pos // page]
    outs = []
    for name in ("k", "v"):
        x = st["new_" + name].double().cpu().numpy()
        was = c[name + "_scale"][0].cpu().numpy()
        out = np.empty((len(seqs), nkv, hd))
        # rows are in order: a block's rows stand together
        start = np.flatnonzero(np.r_[True, (np.diff(seqs) != 0) | (np.diff(pos // BLOCK) != 0)])
        for a, z in zip(start, np.r_[start[1:], len(seqs)]):
            part = x[a:z]
            scale = (np.abs(part).max((0, 2)) / 127).astype(np.float32)
            if pos[a] % BLOCK:
                scale = np.maximum(scale, was[ids[a], :, pos[a] % page // BLOCK])
            f = scale.astype(np.float64)[None, :, None]
            out[a:z] = np.rint(part / f) * f
        outs.append(torch.from_numpy(out))
    return tuple(outs)


def _exact_verify(st):
    case = st["case"]
    B, K, T = case["seqs"], case["drafts"], case["temperature"]
    draft, n, u = st["draft"].cpu().numpy(), st["n_draft"].cpu().numpy(), st["u"].cpu().numpy().astype(np.float64)
    tokens, count, logp = np.full((B, K + 1), -1, np.int32), np.empty(B, np.int32), np.zeros((B, K + 1))
    for b in range(B):
        lp = torch.log_softmax(st["logits"][b].double() / T, -1).cpu().numpy()
        i = 0
        while i < n[b]:
            x = draft[b, i]
            q = float(st["probs"][b, i, x]) if case["probs"] else 1.0
            if not u[b, i] * q < math.exp(lp[i, x]):
                break
            tokens[b, i] = x
            i += 1
        mass = np.exp(lp[i])
        if i < n[b]:
            rest = mass.copy()
            if case["probs"]:
                rest = np.maximum(mass - st["probs"][b, i].double().cpu().numpy(), 0)
            else:
                rest[draft[b, i]] = 0
            mass = rest if rest.sum() > 0 else mass
        cum = np.cumsum(mass)
        tokens[b, i] = np.searchsorted(cum, u[b, K] * cum[-1], side="right")
        count[b] = i + 1
        for j in range(i + 1):
            logp[b, j] = lp[j, tokens[b, j]]
    return torch.from_numpy(tokens), torch.from_numpy(count), torch.from_numpy(logp)


def exact(case, seed):
    if case["op"] == "pages":
        return None  # whole numbers and moved bytes: nothing is computed
    global own
    kept, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = kept
    return {"attend": _exact_attend, "append": _exact_append, "verify": _exact_verify}[case["op"]](st)
