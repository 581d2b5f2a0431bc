"""Draft verification on the GPU against its definition in 64 bits."""
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


def verify64(logits, draft, u, probs, n_draft, T):
    """tokens, counts, log p by the definition."""
    B, R, V = logits.shape
    tokens, count, logp = np.full((B, R), -1), np.zeros(B, int), np.zeros((B, R))
    x = np.where(np.isnan(logits), -np.inf, logits).astype(np.float64)
    for b in range(B):
        def dist(i):
            top = x[b, i].max()
            if np.isneginf(top):
                return None, None
            d = np.where(x[b, i] == top, 0.0, (x[b, i] - (0.0 if np.isinf(top) else top)) / (T if T > 0 else 1.0))
            if np.isinf(top):
                d = np.where(x[b, i] == top, 0.0, -np.inf)
            e = np.exp(d)
            return e / e.sum(), d - math.log(e.sum())
        i = 0
        while True:
            p, lp = dist(i)
            if p is None:
                break
            if i < n_draft[b]:
                t = draft[b, i]
                if T > 0:
                    q = probs[b, i, t].astype(np.float64) if probs is not None else 1.0
                    kept = 0 <= t < V and float(u[b, i]) * q < p[t]
                else:
                    kept = t == int(np.argmax(x[b, i]))
                if kept:
                    tokens[b, i], logp[b, i] = t, lp[t]
                    i += 1
                    continue
            if T > 0:
                mass = p.copy()
                if i < n_draft[b]:
                    if probs is not None:
                        mass = np.maximum(p - probs[b, i].astype(np.float64), 0)
                    else:
                        mass[draft[b, i]] = 0
                    if mass.sum() == 0:
                        mass = p
                cum = np.cumsum(mass)
                t = int(np.argmax(cum > float(u[b, -1]) * cum[-1]))
            else:
                t = int(np.argmax(x[b, i]))
            tokens[b, i], logp[b, i] = t, lp[t]
            i += 1
            break
        count[b] = i
    return tokens, count, logp


def run(ctx, logits, draft, u, probs=None, n_draft=None, T=1.0, stride=None):
    B, R, V = logits.shape
    tokens = torch.full((B, R), 99, dtype=torch.int32, device="cuda")
    count, logp = torch.full((B,), 99, dtype=torch.int32, device="cuda"), torch.full((B, R), 99.0, device="cuda")
    i32 = lambda a: None if a is None else torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")  # noqa: E731
    f32 = lambda a: None if a is None else torch.tensor(np.asarray(a), dtype=torch.float32, device="cuda")  # noqa: E731
    hale.verify_drafts(ctx, logits, i32(draft), f32(u), tokens, count, draft_probs=f32(probs), n_draft=i32(n_draft),
                       temperature=T, out_logp=logp)
    return tokens, count, logp


def check(got, want):
    """Whole numbers are equal; log p is formed in 64 bits from exact logits and
    the row's sum, and rounded once (2^-24 of it). The sum's terms are 32-bit
    exponentials: 2^-22 from the function, and from its argument, x log2 e / T
    rounded once at up to 2^5 where a term still counts, 2^5 2^-24 ln 2; terms
    below 2^-32 of the largest change the sum of 10^5 of them by less than
    2^-15 of their own error. Adding 32 of them rounds 5 times 2^-24 in a tree
    or 31 times in a row: together under 2^-18 of the sum, so of log p in absolute terms."""
    tokens, count, logp = (t.cpu().numpy() for t in got)
    assert np.array_equal(tokens, want[0]), (tokens, want[0])
    assert np.array_equal(count, want[1])
    assert (np.abs(logp - want[2]) <= 2.0 ** -24 * np.abs(want[2]) + 2.0 ** -18).all()


def inputs(seed, B, K, V, dtype, with_probs, sharp=2.5, T=1.0):
    g = np.random.default_rng(seed)
    base = g.normal(0, sharp, (B, K + 1, V)).astype(np.float32)
    logits = torch.from_numpy(base).cuda().to(DT[dtype])
    noisy = base[:, :K].astype(np.float64) / T + g.normal(0, 0.7, (B, K, V))
    p = np.exp(noisy - noisy.max(-1, keepdims=True)) if K else noisy
    p = (p / p.sum(-1, keepdims=True)).astype(np.float32) if K else p.astype(np.float32)
    draft = np.array([[g.choice(V, p=p[b, i].astype(np.float64) / p[b, i].astype(np.float64).sum()) for i in range(K)]
                      for b in range(B)], dtype=np.int64).reshape(B, K)
    u = g.random((B, K + 1)).astype(np.float32)
    return logits, draft, u, p if with_probs else None, g.integers(0, K + 1, B)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("B,K,V,with_probs,T", [(1, 4, 1000, True, 1.0), (5, 3, 257, False, 0.7), (3, 8, 8193, True, 1.3),
                                                (2, 1, 50257, True, 0.6), (7, 0, 999, False, 1.0), (4, 64, 33, True, 1.0),
                                                (40, 2, 1, False, 1.0), (1, 2, 151936, True, 1.0)])
def test_against_the_definition(ctx, dtype, B, K, V, with_probs, T):
    logits, draft, u, probs, n = inputs(V + B, B, K, V, dtype, with_probs, T=T)
    for n_draft in (None, n):
        got = run(ctx, logits, draft, u, probs, n_draft, T)
        ctx.check()
        check(got, verify64(logits.float().cpu().numpy(), draft, u, probs, [K] * B if n_draft is None else n, T))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("V", [5, 8192, 20001])
def test_greedy(ctx, dtype, V):
    """The largest logit, the lowest of equals; a draft that follows it is kept."""
    g = np.random.default_rng(V)
    x = np.round(g.normal(0, 2, (4, 4, V))).astype(np.float32)
    draft = x[:, :3].argmax(-1)
    draft[1, 2] = (draft[1, 2] + 1) % V
    draft[2, 0] = V - 1 - draft[2, 0]
    logits = torch.from_numpy(x).cuda().to(DT[dtype])
    for T in (0.0, -1.0):
        got = run(ctx, logits, draft, None, T=T)
        ctx.check()
        check(got, verify64(x, draft, np.zeros((4, 4)), None, [3] * 4, T))


def test_masked_infinite_and_empty_rows(ctx):
    inf, V = math.inf, 3000
    g = np.random.default_rng(1)
    x = g.normal(0, 1, (6, 3, V)).astype(np.float32)
    x[0, :, 7:] = -inf                       # a cut made by the caller
    x[1, 0] = -inf                           # nothing at all
    x[2, 1] = math.nan
    x[3, 0, [5, 2000]] = inf                 # two certain tokens
    x[4, :, :2990] = math.nan
    x[5, 0, 1:] = -inf
    draft = np.array([[3, 9], [1, 1], [int(np.argmax(x[2, 0])), 4], [2000, 1], [2995, 2996], [0, 0]])
    u = np.array([[0.001, 0.0, 0.999], [0, 0, 0.5], [0, 0, 0.5], [0.3, 0.9, 0.2], [0.01, 0.2, 0.7], [0.9999, 0.99, 0.0]], np.float32)
    for T in (1.0, 0.0):
        got = run(ctx, torch.from_numpy(x).cuda(), draft, u, T=T)
        ctx.check()
        check(got, verify64(x, draft, u, None, [2] * 6, T))


def test_the_ends_of_the_unit_interval(ctx):
    """u = 0 takes the lowest token with any mass, u just under 1 the highest;
    a draft equal to the target is always kept, and one refused by rounding
    alone is drawn from the target."""
    V = 700
    x = np.full((3, 2, V), -math.inf, np.float32)
    x[:, :, 100:600] = np.random.default_rng(2).normal(0, 1, 500).astype(np.float32)
    p = np.exp(x[:, :1].astype(np.float64) - x[:, :1].max())
    p = (p / p.sum(-1, keepdims=True)).astype(np.float32)
    u = np.array([[1.0 - 2.0 ** -24, 0.0], [0.5, 1.0 - 2.0 ** -24], [0.0, 0.5]], np.float32)
    draft = np.array([[150], [150], [150]])
    got = run(ctx, torch.from_numpy(x).cuda(), draft, u, p)
    ctx.check()
    tokens = got[0].cpu().numpy()
    assert tokens[0].tolist() == [150, 100] and tokens[1].tolist() == [150, 599] and tokens[2, 0] == 150
    big = np.ones_like(p)                      # q >= p everywhere: nothing is left of p - q
    got = run(ctx, torch.from_numpy(x).cuda(), draft, np.full((3, 2), 0.99, np.float32), big)
    ctx.check()
    check(got, verify64(x, draft, np.full((3, 2), 0.99, np.float32), big, [1] * 3, 1.0))


def test_rows_apart_and_the_same_bits_twice(ctx):
    logits, draft, u, probs, n = inputs(4, 6, 3, 5001, "f16", True)
    wide = torch.full((6, 4, 5123), 77.0, device="cuda", dtype=torch.float16)
    wide[:, :, 3:5004] = logits
    pw = torch.full((6, 3, 5200), 5.0, device="cuda")
    pw[:, :, 1:5002] = torch.from_numpy(probs)
    want = verify64(logits.float().cpu().numpy(), draft, u, probs, n, 1.0)
    outs = []
    for _ in range(2):
        tokens, count = torch.empty((6, 4), dtype=torch.int32, device="cuda"), torch.empty(6, dtype=torch.int32, device="cuda")
        logp = torch.empty((6, 4), device="cuda")
        hale.verify_drafts(ctx, wide[:, :, 3:5004], torch.tensor(draft, dtype=torch.int32, device="cuda"),
                           torch.from_numpy(u).cuda(), tokens, count, draft_probs=pw[:, :, 1:5002],
                           n_draft=torch.tensor(n, dtype=torch.int32, device="cuda"), out_logp=logp)
        outs.append((tokens, count, logp))
    ctx.check()
    check(outs[0], want)
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_drafts_and_counts_out_of_range_are_reported(ctx):
    logits, draft, u, probs, n = inputs(9, 3, 2, 300, "f32", False)
    draft[0, 0], draft[1, 1] = 300, -5
    got = run(ctx, logits, draft, u)
    with pytest.raises(hale.HaleError) as e:
        ctx.check()
    assert e.value.status == hale.E_DEVICE_CHECK
    assert got[1][0].item() == 1 and got[1][1].item() <= 2
    logits, draft, u, probs, n = inputs(9, 3, 2, 300, "f32", False)
    for count in ([3, 0, 1], [0, -1, 1]):
        got = run(ctx, logits, draft, u, n_draft=count)
        with pytest.raises(hale.HaleError):
            ctx.check()
        check(got, verify64(logits.cpu().numpy(), draft, u, None, np.clip(count, 0, 2), 1.0))


def test_argument_refusals(ctx):
    logits, draft, u, _, _ = inputs(3, 2, 2, 50, "f32", False)
    for change in (dict(T=math.nan), dict(T=math.inf), dict(u=None)):
        with pytest.raises(hale.HaleError) as e:
            run(ctx, logits, draft, change.get("u", u), T=change.get("T", 1.0))
        assert e.value.status == hale.E_INVALID_ARGUMENT
    with pytest.raises(hale.HaleError):
        run(ctx, torch.zeros((1, 66, 4), device="cuda"), np.zeros((1, 65)), np.zeros((1, 66)))
    with pytest.raises(ValueError):
        run(ctx, logits.double(), draft, u)
    with pytest.raises(ValueError):
        run(ctx, logits[:, :2], draft, u)
    ctx.check()
