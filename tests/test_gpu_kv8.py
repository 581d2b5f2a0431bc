"""The paged 8-bit key/value cache on the GPU against plain 64-bit
computations: rows quantised in and read back, attention over the cache,
pages resized, forked, compacted and copied, and refusals."""
import importlib
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

hale = importlib.import_module("hale-token_b200")

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    c = hale.Context(0)
    yield c
    c.check()
    c.close()


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def filled(ctx, rng, lens, nkv, hd, page, layers=1, spare=3, max_pages=None, garbage=False):
    """A cache of random codes and scales; sequence s holds lens[s] tokens in
    shuffled pages. garbage: scales of blocks behind a sequence's end are NaN."""
    need = [-(-n // page) for n in lens]
    n_pages = sum(need) + spare
    max_pages = max_pages or max(need + [1]) + 1
    kv = hale.Kv8.empty(ctx, layers, n_pages, nkv, hd, page, len(lens), max_pages)
    g = np.random.default_rng(rng)
    order = g.permutation(n_pages)
    table = np.full((len(lens), max_pages), -1, np.int32)
    refs = np.zeros(n_pages, np.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        refs[order[at:at + n]] = 1
        at += n
    shape = tuple(kv.k.shape)
    for t in (kv.k, kv.v):
        t.copy_(torch.from_numpy(g.integers(-127, 128, shape, dtype=np.int8)))
    for t in (kv.k_scale, kv.v_scale):
        sc = np.exp(g.normal(-4.0, 0.7, tuple(t.shape))).astype(np.float32)
        if garbage:
            sc[:, refs == 0] = np.nan
            for s, n in enumerate(lens):
                if n % page:
                    sc[:, table[s, n // page], :, -(-(n % page) // 16):] = np.nan
        t.copy_(torch.from_numpy(sc))
    kv.table.copy_(torch.from_numpy(table))
    kv.refs.copy_(torch.from_numpy(refs))
    kv.lens.copy_(ints(lens))
    return kv


def values(kv, layer, seq, n):
    """k, v [n, nkv, hd] in f64 of a sequence's first n tokens."""
    page = kv.page_tokens
    ids = kv.table[seq, :-(-n // page)].long().cpu().numpy()
    out = []
    for codes, scale in ((kv.k, kv.k_scale), (kv.v, kv.v_scale)):
        c = codes[layer].cpu().numpy()[ids].astype(np.float64)
        s = np.repeat(scale[layer].cpu().numpy()[ids].astype(np.float64), 16, axis=2)
        with np.errstate(invalid="ignore"):
            x = (c * s[..., None]).transpose(0, 2, 1, 3).reshape(-1, kv.n_kv_heads, kv.head_dim)
        out.append(x[:n])
    return out


def attention64(kv, layer, q, seqs, pos, scale, window):
    """out, lse in f64, and per element a bound on a correct kernel's error."""
    n, nh, hd = q.shape
    group = nh // kv.n_kv_heads
    out, lse = np.zeros((n, nh, hd)), np.full((n, nh), -np.inf)
    worst, top = np.zeros((n, nh)), np.zeros((n, nh))
    for s in sorted(set(seqs)):
        rows = [r for r in range(n) if seqs[r] == s and pos[r] >= 0]
        if s < 0 or not rows:
            continue
        k, v = values(kv, layer, s, max(pos[r] for r in rows) + 1)
        for r in rows:
            lo = max(0, pos[r] - window + 1) if window else 0
            for h in range(nh):
                kk, vv = k[lo:pos[r] + 1, h // group], v[lo:pos[r] + 1, h // group]
                sc = scale * (kk @ q[r, h])
                m = sc.max()
                e = np.exp(sc - m)
                out[r, h] = (e / e.sum()) @ vv
                lse[r, h] = m + math.log(e.sum())
                worst[r, h] = abs(scale) * (np.abs(kk) @ np.abs(q[r, h])).max()
                top[r, h] = np.abs(vv).max()
    return out, lse, worst, top


def check_attention(out, lse, want, dtype):
    """A score is a sum of up to 256 products, formed in 32 bits in at most 32
    truncating steps of 2^-23 of sum |q k| each, q itself held to 2^-22: off by
    2^-18 of it. exp and the sums (under 2^7 adds a lane, 2^-24 each) add
    2^-16. A weighted mean of values up to `top` is off by twice that times
    top. With 16-bit q the weights may be rounded to 11 bits (2^-12 each, 2^-11
    with the sum's), and the result is rounded once to its type."""
    o, z, worst, top = want
    tol = top * (2 * worst * 2.0 ** -18 + 2.0 ** -15)
    if dtype != "f32":
        tol = tol + top * 2.0 ** -11
    tol = tol[..., None] + np.abs(o) * torch.finfo(DT[dtype]).eps / 2
    got = out.double().cpu().numpy()
    assert np.isfinite(got).all()
    assert (np.abs(got - o) <= tol).all(), float((np.abs(got - o) - tol).max())
    if lse is not None:
        g = lse.double().cpu().numpy()
        empty = np.isneginf(z)
        assert np.array_equal(np.isneginf(g), empty)
        g, z, worst = g[~empty], z[~empty], worst[~empty]
        assert (np.abs(g - z) <= worst * 2.0 ** -18 + 2.0 ** -15 + np.abs(z) * 2.0 ** -23).all()


def run_attention(ctx, kv, rng, dtype, nh, seqs, pos, window=0, run=1, layer=0, seed=3):
    g = np.random.default_rng(seed)
    n = len(seqs)
    q = torch.from_numpy(g.normal(0, 1.5, (n, nh, kv.head_dim)).astype(np.float32)).cuda().to(DT[dtype])
    out, lse = torch.full_like(q, 7.0), torch.full((n, nh), 7.0, device="cuda")
    kv.attention(layer, q, out, ints(pos), ints(seqs), window=window, run=run, lse=lse)
    ctx.check()
    scale = np.float64(np.float32(kv.head_dim ** -0.5))
    return out, lse, attention64(kv, layer, q.double().cpu().numpy(), seqs, pos, scale, window)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("nh,nkv,hd,page,lens", [
    (8, 2, 128, 64, [1, 2, 15, 16, 17, 63, 64, 65, 300, 1000]),
    (3, 3, 16, 16, [33, 1, 129]),
    (7, 1, 80, 32, [257, 40]),
    (16, 1, 64, 128, [700, 5]),
    (20, 2, 192, 256, [511, 100]),
    (12, 3, 256, 16, [90, 333]),
    (40, 2, 96, 64, [190]),
])
def test_single_rows(ctx, dtype, nh, nkv, hd, page, lens):
    kv = filled(ctx, 1, lens, nkv, hd, page, garbage=True)
    out, lse, want = run_attention(ctx, kv, 1, dtype, nh, list(range(len(lens))), [n - 1 for n in lens])
    check_attention(out, lse, want, dtype)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("nh,nkv,hd,page,runs,hist,window", [
    (4, 1, 128, 64, [5, 1, 3], [40, 0, 77], 0),
    (8, 2, 128, 16, [17, 40, 33], [0, 100, 31], 0),
    (8, 8, 64, 32, [130, 7], [3, 60], 50),
    (6, 2, 80, 64, [70], [200], 1),
    (16, 2, 256, 128, [33, 20], [0, 300], 90),
    (14, 2, 192, 16, [9, 64], [513, 0], 0),
])
def test_runs_of_rows(ctx, dtype, nh, nkv, hd, page, runs, hist, window):
    """Several rows of a sequence, each seeing up to itself; runs of other
    lengths than announced give the same."""
    lens = [h + r for h, r in zip(hist, runs)]
    kv = filled(ctx, 2, lens, nkv, hd, page, garbage=True)
    seqs = [s for s, r in enumerate(runs) for _ in range(r)]
    pos = [h + i for h, r in zip(hist, runs) for i in range(r)]
    for run in (max(runs), 1, 4096):
        out, lse, want = run_attention(ctx, kv, 2, dtype, nh, seqs, pos, window, run)
        check_attention(out, lse, want, dtype)


@pytest.mark.parametrize("run", [1, 8, 500])
@pytest.mark.parametrize("dtype", list(DT))
def test_rows_in_any_order_empty_rows_and_rows_left_out(ctx, dtype, run):
    kv = filled(ctx, 4, [200, 90, 31], 2, 64, 32, garbage=True)
    seqs = [2, 0, 0, 1, -1, 0, 1, 1, 0, 2, -1, 0]
    pos = [30, 199, 0, 17, 5, -1, 89, 3, 64, -7, -1, 120]
    out, lse, want = run_attention(ctx, kv, 4, dtype, 4, seqs, pos, run=run)
    left = [r for r, s in enumerate(seqs) if s < 0]
    keep = [r for r in range(len(seqs)) if r not in left]
    assert (out[left] == 7).all() and (lse[left] == 7).all()
    check_attention(out[keep], lse[keep], [w[keep] for w in want], dtype)
    assert (out[[5, 9]] == 0).all() and torch.isneginf(lse[[5, 9]]).all()


@pytest.mark.parametrize("dtype", list(DT))
def test_long_sequences_split_over_the_gpu(ctx, dtype):
    lens = [20011, 1, 4097]
    kv = filled(ctx, 5, lens, 2, 128, 64)
    for seqs, pos in (([0, 1, 2], [20010, 0, 4096]), ([0], [20010])):
        out, lse, want = run_attention(ctx, kv, 5, dtype, 8, seqs, pos)
        check_attention(out, lse, want, dtype)
    pos = list(range(20011 - 6, 20011))
    for run in (1, 6):
        out, lse, want = run_attention(ctx, kv, 5, dtype, 8, [0] * 6, pos, run=run)
        check_attention(out, lse, want, dtype)


@pytest.mark.parametrize("run", [1, 64])
@pytest.mark.parametrize("dtype", list(DT))
def test_scales_far_apart_and_zero(ctx, dtype, run):
    """Blocks whose scales differ by 10^6, blocks of zeros, queries of zeros
    and of very large and small size."""
    kv = filled(ctx, 6, [150], 1, 64, 16)
    kv.v_scale.mul_(torch.tensor([1e-3, 1.0, 0.0, 1e3] * 4, device="cuda")[:kv.n_pages].view(1, -1, 1, 1))
    kv.k_scale[:, int(kv.table[0, 1])] = 0.0
    g = np.random.default_rng(8)
    q = g.normal(0, 1, (6, 2, 64)).astype(np.float32)
    q[1] = 0
    q[2] *= 1e-6
    q[3] *= 12
    q[4, :, 5:] *= 1e-5
    qt = torch.from_numpy(q).cuda().to(DT[dtype])
    out, lse = torch.empty_like(qt), torch.empty((6, 2), device="cuda")
    pos = [149, 149, 149, 149, 100, 15]
    kv.attention(0, qt, out, ints(pos), ints([0] * 6), scale=0.25, run=run, lse=lse)
    ctx.check()
    check_attention(out, lse, attention64(kv, 0, qt.double().cpu().numpy(), [0] * 6, pos, 0.25, 0), dtype)


@pytest.mark.parametrize("run", [1, 16])
@pytest.mark.parametrize("dtype", list(DT))
def test_a_query_that_is_no_number_spoils_its_own_head_alone(ctx, dtype, run):
    kv = filled(ctx, 9, [300], 2, 64, 32)
    g = np.random.default_rng(4)
    q = torch.from_numpy(g.normal(0, 1, (3, 4, 64)).astype(np.float32)).cuda().to(DT[dtype])
    q[1, 2, 7] = float("nan")
    q[2, 0, 5] = float("inf")
    out, lse = torch.zeros_like(q), torch.zeros((3, 4), device="cuda")
    kv.attention(0, q, out, ints([299, 120, 7]), ints([0, 0, 0]), run=run, lse=lse)
    ctx.check()
    bad = torch.zeros((3, 4), dtype=torch.bool)
    bad[1, 2] = bad[2, 0] = True
    assert torch.equal(out.float().isnan().all(-1).cpu(), bad) and torch.equal(out.float().isnan().any(-1).cpu(), bad)
    assert torch.equal(lse.isnan().cpu(), bad)
    clean = torch.where(bad[..., None].cuda(), torch.zeros_like(q), q)
    want = attention64(kv, 0, clean.double().cpu().numpy(), [0] * 3, [299, 120, 7], np.float64(np.float32(64 ** -0.5)), 0)
    keep = (~bad).numpy()
    o, z, worst, top = want
    check_attention(out.cpu()[torch.from_numpy(keep)], lse.cpu()[torch.from_numpy(keep)], (o[keep], z[keep], worst[keep], top[keep]), dtype)


def test_rows_apart_other_layers_and_other_streams(ctx):
    """q and out as slices of wider rows, a middle layer, a side stream, and
    the same call twice: the same bits."""
    kv = filled(ctx, 7, [300, 80], 2, 32, 32, layers=3)
    g = np.random.default_rng(9)
    wide = torch.from_numpy(g.normal(0, 1, (7, 4 + 2 * 2, 32)).astype(np.float32)).cuda()
    q, big = wide[:, :4], torch.full((7, 9, 32), 5.0, device="cuda")
    out = big[:, 3:7]
    seqs, pos = [0, 0, 0, 1, 1, 0, 1], [299, 298, 5, 79, 0, 150, 33]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        kv.attention(1, q, out, ints(pos), ints(seqs), run=2)
    st.synchronize()
    first = big.clone()
    kv.attention(1, q, out, ints(pos), ints(seqs), run=2)
    ctx.check()
    assert torch.equal(first, big)
    assert (big[:, :3] == 5).all() and (big[:, 7:] == 5).all()
    want = attention64(kv, 1, q.double().cpu().numpy(), seqs, pos, np.float64(np.float32(32 ** -0.5)), 0)
    check_attention(out, None, want, "f32")


def test_bad_pages_are_reported_and_left_out(ctx):
    """A missing page, a page number out of range, a sequence and a position
    out of range: reported, and the other rows are right."""
    kv = filled(ctx, 8, [200, 100, 50], 2, 64, 32)
    kv.table[1, 1] = -1
    kv.table[2, 1] = kv.n_pages
    g = np.random.default_rng(3)
    q = torch.from_numpy(g.normal(0, 1, (5, 4, 64)).astype(np.float32)).cuda()
    for run in (1, 16):
        for seqs, pos in (([0, 1, 0, 0, 0], [199, 99, 10, 0, 3]), ([0, 0, 2, 0, 0], [5, 199, 49, 1, 3]),
                          ([0, 0, 0, 3, 0], [5, 199, 49, 1, 3]), ([0, 0, 0, 0, 0], [5, 199, 49, 1, 10 ** 9])):
            out = torch.zeros_like(q)
            kv.attention(0, q, out, ints(pos), ints(seqs), run=run)
            with pytest.raises(hale.HaleError) as e:
                ctx.check()
            assert e.value.status == hale.E_DEVICE_CHECK
            ok = [r for r in range(5) if seqs[r] == 0 and pos[r] < 200]
            want = attention64(kv, 0, q.double().cpu().numpy()[ok], [0] * len(ok), [pos[r] for r in ok],
                               np.float64(np.float32(64 ** -0.5)), 0)
            check_attention(out[ok], None, want, "f32")


# ---------------------------------------------------------------------------
# append and read
# ---------------------------------------------------------------------------
class Model:
    """The cache's codes and scales in plain Python: {(seq, block, head, which): (scale, codes[16, hd])}."""

    def __init__(self, nkv, hd):
        self.nkv, self.hd, self.d = nkv, hd, {}

    def append(self, k, v, seqs, pos):
        rows = {}
        for r, (s, p) in enumerate(zip(seqs, pos)):
            if s >= 0 and p >= 0:
                rows.setdefault((s, p // 16), {})[p % 16] = r
        for (s, b), members in rows.items():
            for which, x in (("k", k), ("v", v)):
                for h in range(self.nkv):
                    old, codes = self.d.get((s, b, h, which), (np.float32(0), np.zeros((16, self.hd))))
                    part = {t: x[r, h].astype(np.float64) for t, r in members.items()}
                    finite = [np.abs(p[np.isfinite(p)]).max(initial=0) for p in part.values()]
                    a = np.float32(max(finite))
                    want = np.float32(0) if a == 0 else max(np.float32(np.float64(a) / 127), np.float32(2.0 ** -100))
                    if 0 in part:
                        old = np.float32(0)
                    new = max(old, want)
                    if old > 0 and new > old:
                        codes = np.rint(codes * np.float64(old) / np.float64(new))
                    codes = codes.copy()
                    for t, p in part.items():
                        with np.errstate(invalid="ignore", divide="ignore"):
                            c = np.rint(p / np.float64(new)) if new > 0 else np.where(np.isinf(p), np.inf * np.sign(p), 0 * p)
                        codes[t] = np.clip(np.nan_to_num(c, nan=0.0, posinf=127, neginf=-127), -127, 127)
                    self.d[s, b, h, which] = (new, codes)

    def check(self, kv, layer, tokens):
        k, v = kv.k[layer].cpu().numpy(), kv.v[layer].cpu().numpy()
        ks, vs = kv.k_scale[layer].cpu().numpy(), kv.v_scale[layer].cpu().numpy()
        table = kv.table.cpu().numpy()
        for s, p in tokens:
            page, slot = table[s, p // kv.page_tokens], p % kv.page_tokens
            for which, c, sc in (("k", k, ks), ("v", v, vs)):
                for h in range(self.nkv):
                    scale, codes = self.d[s, p // 16, h, which]
                    assert sc[page, h, slot // 16] == scale, (s, p, h, which)
                    assert np.array_equal(c[page, h, slot], codes[p % 16]), (s, p, h, which)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("nkv,hd,page", [(2, 128, 64), (1, 16, 16), (3, 80, 32), (2, 256, 128), (1, 192, 16)])
def test_append_codes_and_scales(ctx, dtype, nkv, hd, page):
    """Prompts, then single tokens whose size grows and shrinks, rows in any
    order, a row twice, rows left out: codes and scales to the bit."""
    lens = [70, 33, 16]
    kv = filled(ctx, 11, lens, nkv, hd, page, layers=2)
    was = [t[0].clone() for t in (kv.k, kv.v, kv.k_scale, kv.v_scale)]
    m = Model(nkv, hd)
    g = np.random.default_rng(12)
    todo = [([0] * 37 + [1] * 20 + [2] * 1, list(range(37)) + list(range(20)) + [0])]
    for i in range(5):
        todo.append(([2, 0, -1, 1], [1 + i, 37 + i, 0, 20 + i]))
    todo.append(([0, 0, 1, 0, 0, 1, 2, 0], [47, 42, 25, 45, 43, -3, 6, 47]))
    todo.append(([0] * 4, [48, 51, 49, 50]))
    done = set()
    for i, (seqs, pos) in enumerate(todo):
        x = [torch.from_numpy((g.normal(0, 1, (len(seqs), nkv, hd)) * 2.0 ** g.integers(-3, 3)).astype(np.float32)).cuda().to(DT[dtype])
             for _ in range(2)]
        kv.append(1, x[0], x[1], ints(pos), ints(seqs))
        ctx.check()
        m.append(x[0].double().cpu().numpy(), x[1].double().cpu().numpy(), seqs, pos)
        done |= {(s, p) for s, p in zip(seqs, pos) if s >= 0 and p >= 0}
    m.check(kv, 1, sorted(done))
    for a, t in zip(was, (kv.k, kv.v, kv.k_scale, kv.v_scale)):
        assert torch.equal(a, t[0])  # the other layer is as it was
    tokens = sorted(done)
    seqs, pos = [s for s, _ in tokens] + [-1, 0], [p for _, p in tokens] + [0, -1]
    for name, odt in DT.items():
        ko, vo = (torch.full((len(seqs), nkv, hd), 9.0, device="cuda", dtype=odt) for _ in range(2))
        kv.read(1, ko, vo, ints(pos), ints(seqs))
        ctx.check()
        for which, got in (("k", ko), ("v", vo)):
            want = np.stack([[np.float32(m.d[s, p // 16, h, which][0]) * m.d[s, p // 16, h, which][1][p % 16].astype(np.float32)
                              for h in range(nkv)] for s, p in tokens])
            assert torch.equal(got[:-2].cpu(), torch.from_numpy(want).to(odt))
            assert (got[-2:] == 9).all()


def test_append_ties_tiny_and_non_finite_values(ctx):
    kv = filled(ctx, 13, [64], 1, 16, 16)
    m = Model(1, 16)
    k, v = torch.zeros((5, 1, 16), device="cuda"), torch.zeros((5, 1, 16), device="cuda")
    k[0, 0, :6] = torch.tensor([127.0, 2.5, -3.5, 0.5, 1.5, 126.5])      # scale 1: halves go to even
    k[1, 0, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), 1e30])
    k[2, 0, :3] = torch.tensor([1e-44, -3e-44, 0.0])                      # far below the smallest scale
    k[3, 0, :3] = torch.tensor([float("inf"), float("nan"), 0.0])         # no finite size at all
    k[4, 0, :3] = torch.tensor([3.4e38, -3.4028235e38, 1e37])
    v[0, 0, :3] = torch.tensor([6.35, 0.025, 0.075])
    seqs, pos = [0] * 5, [0, 16, 32, 48, 35]
    kv.append(0, k, v, ints(pos), ints(seqs))
    ctx.check()
    m.append(k.double().cpu().numpy(), v.double().cpu().numpy(), seqs, pos)
    m.check(kv, 0, list(zip(seqs, pos)))


def test_append_long_lists_and_rows_apart(ctx):
    """Over 1024 rows (several rows a CTA), k and v slices of one wide row."""
    lens = [900, 700]
    kv = filled(ctx, 14, lens, 2, 32, 64)
    m = Model(2, 32)
    g = np.random.default_rng(15)
    seqs, pos = [0] * 900 + [1] * 700, list(range(900)) + list(range(700))
    order = g.permutation(1600)
    for seqs, pos in ((seqs, pos), ([seqs[i] for i in order], [pos[i] for i in order])):
        wide = torch.from_numpy(g.normal(0, 1, (1600, 8, 32)).astype(np.float32)).cuda()
        kv.append(0, wide[:, 4:6], wide[:, 6:8], ints(pos), ints(seqs))
        ctx.check()
        m.append(wide[:, 4:6].cpu().numpy(), wide[:, 6:8].cpu().numpy(), seqs, pos)
        m.check(kv, 0, list(zip(seqs, pos)))


def test_append_reports_missing_pages(ctx):
    kv = filled(ctx, 16, [20, 40], 1, 16, 16)
    k = torch.ones((2, 1, 16), device="cuda")
    for seqs, pos in (([0, 1], [33, 0]), ([2, 1], [0, 1]), ([0, 1], [10 ** 8, 2])):
        kv.append(0, k, k, ints(pos), ints(seqs))
        with pytest.raises(hale.HaleError) as e:
            ctx.check()
        assert e.value.status == hale.E_DEVICE_CHECK


# ---------------------------------------------------------------------------
# pages
# ---------------------------------------------------------------------------
class Pages:
    """resize, fork and compact restated on Python lists; data[page] names what a page holds."""

    def __init__(self, kv):
        self.pt, self.cap = kv.page_tokens, kv.max_pages
        self.lens = kv.lens.cpu().tolist()
        self.rows = [[p for p in r if p >= 0] for r in kv.table.cpu().tolist()]
        self.refs = kv.refs.cpu().tolist()

    def resize(self, seqs, new):
        rows, refs = [list(r) for r in self.rows], list(self.refs)
        copies = []
        for s, n in zip(seqs, new):
            keep = -(-n // self.pt)
            if n < self.lens[s]:
                for p in rows[s][keep:]:
                    refs[p] -= 1
                rows[s] = rows[s][:keep]
        want = []
        for s, n in zip(seqs, new):
            if n > self.lens[s]:
                if self.lens[s] % self.pt and refs[rows[s][-1]] > 1:
                    refs[rows[s][-1]] -= 1
                    want.append((s, True))
                want += [(s, False)] * (-(-n // self.pt) - len(rows[s]))
        free = [p for p, c in enumerate(refs) if c == 0]
        if len(free) < len(want):
            return None
        for (s, own), p in zip(want, free):
            if own:
                copies.append((rows[s][-1], p))
                rows[s][-1] = p
            else:
                rows[s].append(p)
            refs[p] = 1
        self.rows, self.refs = rows, refs
        for s, n in zip(seqs, new):
            self.lens[s] = n
        return copies

    def fork(self, parents, children):
        for c in children:
            for p in self.rows[c]:
                self.refs[p] -= 1
        for a, c in zip(parents, children):
            self.rows[c], self.lens[c] = list(self.rows[a]), self.lens[a]
            for p in self.rows[a]:
                self.refs[p] += 1

    def compact(self):
        used = [p for p, c in enumerate(self.refs) if c > 0]
        n = len(used)
        pairs = list(zip([p for p in used if p >= n], [p for p in range(n) if self.refs[p] == 0]))
        to = dict(pairs)
        for s, d in pairs:
            self.refs[d], self.refs[s] = self.refs[s], 0
        self.rows = [[to.get(p, p) for p in r] for r in self.rows]
        return pairs, n

    def check(self, kv):
        assert kv.lens.cpu().tolist() == self.lens
        assert kv.refs.cpu().tolist() == self.refs
        assert kv.table.cpu().tolist() == [r + [-1] * (self.cap - len(r)) for r in self.rows]


def snapshot(kv):
    return [t.clone() for t in (kv.k, kv.v, kv.k_scale, kv.v_scale)]


def after(snap, pairs):
    out = [t.clone() for t in snap]
    for s, d in pairs:
        for t, o in zip(snap, out):
            o[:, d] = t[:, s]
    return out


def same(kv, want):
    for t, w in zip((kv.k, kv.v, kv.k_scale, kv.v_scale), want):
        assert torch.equal(t, w)


@pytest.mark.parametrize("page,nkv,hd,layers", [(16, 1, 16, 1), (64, 2, 128, 3), (32, 3, 80, 2), (256, 1, 256, 1)])
def test_random_page_work(ctx, page, nkv, hd, layers):
    lens = [3 * page + 5, page, 2 * page - 1, 0, 0, 0, 7, 0]
    kv = filled(ctx, 21, lens, nkv, hd, page, layers, spare=14, max_pages=9)
    m = Pages(kv)
    g = np.random.default_rng(22)
    remap, live = torch.zeros((2, kv.n_pages), dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    for step in range(60):
        snap, what = snapshot(kv), g.integers(0, 4)
        if what <= 1:
            seqs = g.permutation(8)[:g.integers(1, 9)].tolist()
            new = [int(np.clip(m.lens[s] + g.integers(-2 * page, 2 * page + 1) * g.integers(0, 2) + g.integers(-2, 3), 0, 9 * page)) for s in seqs]
            pairs = m.resize(seqs, new)
            kv.resize(ints(new), ints(seqs))
            if pairs is None:
                with pytest.raises(hale.HaleError) as e:
                    ctx.check()
                assert e.value.status == hale.E_DEVICE_CHECK
                pairs = []
        elif what == 2:
            p = g.permutation(8)
            n = int(g.integers(1, 5))
            children, parents = p[:n].tolist(), [int(x) for x in g.choice(p[n:], n)]
            m.fork(parents, children)
            kv.fork(ints(parents), ints(children))
            pairs = []
        else:
            old_refs = list(m.refs)
            pairs, n = m.compact()
            kv.compact(remap, live)
            to = [p if c > 0 else -1 for p, c in enumerate(old_refs)]
            for s, d in pairs:
                to[s] = d
            back = [-1] * kv.n_pages
            for p, d in enumerate(to):
                if d >= 0:
                    back[d] = p
            assert live.item() == n and remap.cpu().tolist() == [to, back]
        ctx.check()
        m.check(kv)
        same(kv, after(snap, pairs))


def test_many_sharers_grow_in_one_call(ctx):
    """300 forks of two parents, all lengthened at once with their parents."""
    kv = filled(ctx, 23, [37, 50] + [0] * 300, 1, 16, 16, spare=700, max_pages=5)
    m = Pages(kv)
    children = list(range(2, 302))
    parents = [c % 2 for c in children]
    m.fork(parents, children)
    kv.fork(ints(parents), ints(children))
    order = np.random.default_rng(5).permutation(302).tolist()
    new = [m.lens[s] + 1 + s % 20 for s in order]
    snap = snapshot(kv)
    pairs = m.resize(order, new)
    kv.resize(ints(new), ints(order))
    ctx.check()
    assert len(pairs) == 300
    m.check(kv)
    same(kv, after(snap, pairs))


def test_copy_pages(ctx):
    kv = filled(ctx, 24, [64, 64], 2, 48, 16, layers=2)
    snap = snapshot(kv)
    src, dst = [0, 3, 5, 3, 7], [1, 2, 5, 4, 6]
    kv.copy_pages(ints(src), ints(dst))
    ctx.check()
    same(kv, after(snap, list(zip(src, dst))))


def test_page_refusals_change_nothing(ctx):
    kv = filled(ctx, 25, [40, 30, 20], 1, 32, 16, max_pages=4)
    m, snap = Pages(kv), snapshot(kv)
    bad = [lambda: kv.resize(ints([50, 20]), ints([1, 1])), lambda: kv.resize(ints([65]), ints([0])),
           lambda: kv.resize(ints([-1]), ints([0])), lambda: kv.resize(ints([5]), ints([3])),
           lambda: kv.resize(ints([5, 1]), ints([0, -1])), lambda: kv.resize(ints([64, 64, 64])),
           lambda: kv.fork(ints([0, 1]), ints([2, 2])), lambda: kv.fork(ints([0, 1]), ints([1, 2])),
           lambda: kv.fork(ints([3]), ints([1])), lambda: kv.fork(ints([0]), ints([-1])), lambda: kv.fork(ints([0]), ints([0])),
           lambda: kv.copy_pages(ints([0, 1]), ints([2, 2])), lambda: kv.copy_pages(ints([0, 1]), ints([1, 2])),
           lambda: kv.copy_pages(ints([0]), ints([kv.n_pages])), lambda: kv.copy_pages(ints([-1]), ints([0]))]
    for call in bad:
        call()
        with pytest.raises(hale.HaleError) as e:
            ctx.check()
        assert e.value.status == hale.E_DEVICE_CHECK
        m.check(kv)
        same(kv, snap)


def test_argument_refusals(ctx):
    kv = filled(ctx, 26, [40], 2, 32, 16)
    q, out, one = torch.zeros((1, 4, 32), device="cuda"), torch.zeros((1, 4, 32), device="cuda"), ints([0])
    k = torch.zeros((1, 2, 32), device="cuda")
    bad = [lambda: kv.attention(1, q, out, one), lambda: kv.attention(0, q[:, :3], out[:, :3], one),
           lambda: kv.attention(0, q, out, one, run=0), lambda: kv.attention(0, q, out, one, scale=float("nan")),
           lambda: kv.append(2, k, k, one), lambda: kv.resize(ints([1, 1])), lambda: kv.fork(ints([0]), ints([0]))]
    for call in bad:
        with pytest.raises(hale.HaleError) as e:
            call()
        assert e.value.status == hale.E_INVALID_ARGUMENT
    odd = torch.zeros(1 + 4 * 32, device="cuda")[1:].view(1, 4, 32)
    with pytest.raises(hale.HaleError, match="16-byte"):
        kv.attention(0, odd, out, one)
    for call in (lambda: kv.attention(0, q.double(), out.double(), one), lambda: kv.attention(0, q, out, one.long()),
                 lambda: kv.attention(0, q.cpu(), out, one), lambda: kv.append(0, k, k.half(), one),
                 lambda: kv.attention(0, q, out, ints([0, 1])), lambda: kv.read(0, k.double(), None, one)):
        with pytest.raises(ValueError):
            call()
    for change in (dict(head_dim=24), dict(head_dim=272), dict(page_tokens=48), dict(page_tokens=8), dict(n_pages=0),
                   dict(n_seqs=0), dict(max_pages=1 << 28), dict(n_kv_heads=0), dict(k=None), dict(refs=None),
                   dict(n_pages=(1 << 20) + 1)):
        c = hale.Kv8Struct.from_buffer_copy(kv.c)
        for name, v in change.items():
            setattr(c, name, v)
        st = hale.lib().hale_kv8_resize(ctx.h, hale.C.byref(c), None, hale.ptr(one), 1, None)
        assert st == hale.E_INVALID_ARGUMENT, change
    ctx.check()
    empty = torch.zeros((0, 4, 32), device="cuda")
    kv.attention(0, empty, empty, ints([]))
    kv.append(0, empty[:, :2], empty[:, :2], ints([]))
    ctx.check()
