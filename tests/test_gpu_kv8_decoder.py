"""A decoder over the paged 8-bit cache, and the cache, its pages and draft
verification used together, as a server would."""
import importlib
import json
import os

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

hale = importlib.import_module("hale-token_b200")
fmt = importlib.import_module("hale-token_b200.formats")
loader = importlib.import_module("hale-token_b200.loader")
GOLDEN = os.path.join(os.path.dirname(__file__), "golden")


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


class Toy:
    """A dense model (no experts) with random f32 weights, on the GPU and in 64 bits."""

    def __init__(self, seed, hidden, nh, nkv, hd, layers, vocab, inter, norms):
        g = np.random.default_rng(seed)
        self.nh, self.nkv, self.hd, self.theta, self.eps = nh, nkv, hd, 10000.0, 1e-5

        def mat(r, c):
            return (g.standard_normal((r, c)) / np.sqrt(c)).astype(np.float32)

        def vec(n):
            return (1 + 0.1 * g.standard_normal(n)).astype(np.float32)
        self.layers = []
        for _ in range(layers):
            L = dict(input_norm=vec(hidden), post_norm=vec(hidden), q=mat(nh * hd, hidden), k=mat(nkv * hd, hidden),
                     v=mat(nkv * hd, hidden), o=mat(hidden, nh * hd), dense_gate=mat(inter, hidden), dense_up=mat(inter, hidden),
                     dense_down=mat(hidden, inter))
            if norms:
                L.update(q_norm=vec(hd), k_norm=vec(hd))
            self.layers.append(L)
        self.embed, self.head, self.final = mat(vocab, hidden), mat(vocab, hidden), vec(hidden)
        self.dims = dict(hidden=hidden, n_layers=layers, n_heads=nh, n_kv_heads=nkv, head_dim=hd, vocab=vocab,
                         eps=self.eps, rope_theta=self.theta)

    def decoder(self, ctx, kv, max_len, max_batch):
        def enc(m):
            return (fmt.F32, m.shape[0], m.shape[1], m.view(np.uint8).reshape(m.shape[0], -1))
        layers = [{k: (enc(v) if v.ndim == 2 else v) for k, v in L.items()} for L in self.layers]
        return hale.Decoder(ctx, self.dims, layers, enc(self.embed), enc(self.head), self.final, None, max_len,
                            max_batch=max_batch, kv8=kv)

    def norm(self, x, w):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.eps) * w

    def rope(self, x, pos):
        h = self.hd // 2
        ang = pos * self.theta ** (-2.0 * np.arange(h) / self.hd)
        a, b, c, s = x[..., :h], x[..., h:], np.cos(ang), np.sin(ang)
        return np.concatenate([a * c - b * s, b * c + a * s], -1)

    def row(self, token, pos, cached):
        """Logits of one token, attending over the values cached(layer) = (k, v)
        [pos + 1, nkv, hd] gives; and its own k, v of each layer."""
        x = self.embed[token].astype(np.float64)
        made = []
        for i, L in enumerate(self.layers):
            W = {k: v.astype(np.float64) for k, v in L.items()}
            n = self.norm(x, W["input_norm"])
            q = (W["q"] @ n).reshape(self.nh, self.hd)
            k, v = ((W[m] @ n).reshape(self.nkv, self.hd) for m in "kv")
            if "q_norm" in W:
                q, k = self.norm(q, W["q_norm"]), self.norm(k, W["k_norm"])
            q, k = self.rope(q, pos), self.rope(k, pos)
            made.append((k, v))
            kc, vc = cached(i)
            out = []
            for h in range(self.nh):
                s = kc[:, h // (self.nh // self.nkv)] @ q[h] * self.hd ** -0.5
                e = np.exp(s - s.max())
                out.append((e / e.sum()) @ vc[:, h // (self.nh // self.nkv)])
            x = x + W["o"] @ np.concatenate(out)
            n = self.norm(x, W["post_norm"])
            gate = W["dense_gate"] @ n
            x = x + W["dense_down"] @ (gate / (1 + np.exp(-gate)) * (W["dense_up"] @ n))
        return self.head.astype(np.float64) @ self.norm(x, self.final), made


def cached_rows(ctx, kv, seq, n):
    """The values the cache stands for, by layer: (k, v) [n, nkv, hd]."""
    out = []
    for layer in range(kv.n_layers):
        k, v = (torch.zeros((n, kv.n_kv_heads, kv.head_dim), device="cuda") for _ in range(2))
        kv.read(layer, k, v, ints(range(n)), ints([seq] * n))
        out.append((k.double().cpu().numpy(), v.double().cpu().numpy()))
    ctx.check()
    return out


# Each step rounds in 32 bits: products of up to 192 terms (2^-24 each, about
# 2^-20 of sum |a b| in the worst order), norms, exponentials. Two layers of
# some ten such steps, the values of order 1: 1e-4 is 2^-20 a hundred times over.
NEAR = 1e-4


@pytest.mark.parametrize("nh,nkv,hd,page,norms", [(4, 2, 16, 16, False), (8, 1, 64, 32, True), (6, 2, 48, 64, False)])
def test_decoder_over_the_paged_cache(ctx, nh, nkv, hd, page, norms):
    """Prompts in chunks of several sequences, then single rows one step at a
    time: every row's logits against 64 bits over the cached values, and the
    cached values within half a code of the keys and values themselves."""
    toy = Toy(nh, 64, nh, nkv, hd, 2, 50, 96, norms)
    kv = hale.Kv8.empty(ctx, 2, 24, nkv, hd, page, 3, 6)
    dec = toy.decoder(ctx, kv, 90, 16)
    g = np.random.default_rng(hd)
    text = {s: g.integers(0, 50, 40).tolist() for s in range(3)}
    done = {0: 0, 1: 0, 2: 0}
    last = {}
    steps = [{0: 10, 2: 5}, {0: 3, 1: 12}, {0: 1, 1: 1, 2: 1}, {1: 1}, {2: 14}, {0: 1, 2: 1}]
    for step in steps:
        rows = [(s, done[s] + i) for s, n in step.items() for i in range(n)]
        kv.resize(ints([done[s] + n for s, n in step.items()]), ints(list(step)))
        logits = torch.zeros((len(rows), 50), device="cuda")
        dec.step([text[s][p] for s, p in rows], [p for _, p in rows], [s for s, _ in rows], logits)
        ctx.check()
        for s, n in step.items():
            done[s] += n
        cache = {s: cached_rows(ctx, kv, s, done[s]) for s in step}
        for r, (s, p) in enumerate(rows):
            want, made = toy.row(text[s][p], p, lambda layer: tuple(x[:p + 1] for x in cache[s][layer]))
            assert np.abs(logits[r].cpu().numpy() - want).max() < NEAR, (step, s, p)
            last[s] = want
            for layer, (k, v) in enumerate(made):
                for got, x, scale in ((cache[s][layer][0][p], k, kv.k_scale), (cache[s][layer][1][p], v, kv.v_scale)):
                    sc = scale[layer, int(kv.table[s, p // page]), :, p % page // 16].double().cpu().numpy()
                    # half a code, and the 32-bit error of the value
                    assert (np.abs(got - x) <= 0.5 * sc[:, None] + NEAR).all()
    # sequence 0 alone through the one-row path, eager and replayed
    one = torch.zeros(50, device="cuda")
    for i in range(3):
        p = done[0]
        kv.resize(ints([p + 1]), ints([0]))
        dec.forward(text[0][p], p, one)
        ctx.check()
        done[0] += 1
        cache = cached_rows(ctx, kv, 0, p + 1)
        want, _ = toy.row(text[0][p], p, lambda layer: cache[layer])
        assert np.abs(one.cpu().numpy() - want).max() < NEAR
    dec.close()


def test_decoder_refusals(ctx):
    toy = Toy(1, 64, 4, 2, 16, 2, 50, 96, False)
    for kv in (hale.Kv8.empty(ctx, 1, 4, 2, 16, 16, 1, 4), hale.Kv8.empty(ctx, 2, 4, 1, 16, 16, 1, 4),
               hale.Kv8.empty(ctx, 2, 4, 2, 32, 16, 1, 4), hale.Kv8.empty(ctx, 2, 4, 2, 16, 16, 1, 3)):
        with pytest.raises(hale.HaleError) as e:
            toy.decoder(ctx, kv, 64, 4)
        assert e.value.status == hale.E_INVALID_ARGUMENT
    kv = hale.Kv8.empty(ctx, 2, 4, 2, 16, 16, 1, 4)
    dec = toy.decoder(ctx, kv, 64, 4)
    dec.step([1, 2], [0, 1])  # no pages yet
    with pytest.raises(hale.HaleError) as e:
        ctx.check()
    assert e.value.status == hale.E_DEVICE_CHECK
    dec.close()


@pytest.mark.parametrize("name", ["tiny-qwen3-moe", "tiny-mixtral"])
def test_generation_of_the_fixture_models_runs(ctx, name):
    """The fixtures through the loader and generate()."""
    d = os.path.join(GOLDEN, name)
    with open(os.path.join(d, "expected.json")) as f:
        prompt = json.load(f)["prompt"]
    plain, pool, _ = loader.load_decoder(ctx, d, max_len=len(prompt) + 8, max_batch=4)
    hd = plain.dims["head_dim"]
    kv = hale.Kv8.empty(ctx, plain.dims["n_layers"], 8, plain.dims["n_kv_heads"], hd, 16, 1, 8)
    dec, pool2, _ = loader.load_decoder(ctx, d, max_len=len(prompt) + 8, max_batch=4, kv8=kv)
    kv.resize(ints([len(prompt) + 6]))
    greedy = hale.SamplingParams(0.0, 1.0, 0, 1.0)
    got, _, _ = dec.generate(prompt, greedy, 1, 6)
    ctx.check()
    assert len(got) == 6 and all(0 <= t < dec.dims["vocab"] for t in got)
    plain.close()
    dec.close()


def test_speculative_serving(ctx):
    """Two prompts; forks of one; drafted tokens of every sequence in one step,
    verified, the refused ones taken back; a compaction in between. The tokens
    are those of the target's distribution by definition, and the cache stays
    what a plain bookkeeping says."""
    from test_gpu_kv8 import Pages
    from test_gpu_verify import verify64
    toy = Toy(5, 64, 8, 2, 32, 2, 40, 64, True)
    kv = hale.Kv8.empty(ctx, 2, 40, 2, 32, 16, 5, 8)
    pages = Pages(kv)
    dec = toy.decoder(ctx, kv, 128, 32)
    g = np.random.default_rng(6)
    text = {0: g.integers(0, 40, 13).tolist(), 1: g.integers(0, 40, 16).tolist()}

    def resize(lens):
        assert pages.resize(list(lens), list(lens.values())) is not None
        kv.resize(ints(list(lens.values())), ints(list(lens)))
    resize({s: len(t) for s, t in text.items()})
    rows = [(s, p) for s, t in text.items() for p in range(len(t))]
    dec.step([text[s][p] for s, p in rows], [p for _, p in rows], [s for s, _ in rows])
    pages.fork([0, 0, 1], [2, 3, 4])
    kv.fork(ints([0, 0, 1]), ints([2, 3, 4]))
    for child, parent in ((2, 0), (3, 0), (4, 1)):
        text[child] = list(text[parent])
    K, B = 3, 5
    for turn in range(8):
        # the last token of each sequence, not yet in the cache, and K drafted ones
        start = {s: len(text[s]) for s in range(B)}
        first = g.integers(0, 40, B)
        draft = g.integers(0, 40, (B, K))
        resize({s: start[s] + K + 1 for s in range(B)})
        rows = [(s, start[s] + i) for s in range(B) for i in range(K + 1)]
        toks = [int(first[s]) if p == start[s] else int(draft[s, p - start[s] - 1]) for s, p in rows]
        logits = torch.zeros((B * (K + 1), 40), device="cuda")
        dec.step(toks, [p for _, p in rows], [s for s, _ in rows], logits)
        q = g.dirichlet(np.ones(40), (B, K)).astype(np.float32)
        u = g.random((B, K + 1)).astype(np.float32)
        out, count = torch.zeros((B, K + 1), dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
        T = (1.0, 0.0)[turn % 2]
        hale.verify_drafts(ctx, logits.view(B, K + 1, 40), ints(draft), torch.from_numpy(u).cuda(), out, count,
                           draft_probs=torch.from_numpy(q).cuda(), temperature=T)
        ctx.check()
        want = verify64(logits.view(B, K + 1, 40).cpu().numpy(), draft, u, q, [K] * B, T)
        assert np.array_equal(out.cpu().numpy(), want[0]) and np.array_equal(count.cpu().numpy(), want[1])
        kept = count.cpu().numpy() - 1
        resize({s: start[s] + 1 + int(kept[s]) for s in range(B)})
        for s in range(B):
            text[s] += [int(first[s])] + draft[s, :kept[s]].tolist()
            assert len(text[s]) == pages.lens[s]
        if turn == 3:
            remap, live = torch.zeros((2, 40), dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
            pages.compact()
            kv.compact(remap, live)
        if turn == 5:  # sequence 3 ends, 4 becomes a copy of 2
            resize({3: 0})
            text[3] = []
            pages.fork([2], [4])
            kv.fork(ints([2]), ints([4]))
            text[4] = list(text[2])
        ctx.check()
        pages.check(kv)
    for s in range(B):  # a last row of each sequence over what its cache now holds
        p = len(text[s])
        resize({s: p + 1})
        logits = torch.zeros((1, 40), device="cuda")
        dec.step([7], [p], [s], logits)
        cache = cached_rows(ctx, kv, s, p + 1)
        want, _ = toy.row(7, p, lambda layer: cache[layer])
        assert np.abs(logits[0].cpu().numpy() - want).max() < NEAR
    dec.close()


def test_captured_steps_replay_with_the_days_lengths(ctx):
    """append, attention, verify and resize in one graph, replayed with other
    positions, equal the same calls made one by one; two graphs in turn."""
    g = np.random.default_rng(8)
    caches = [hale.Kv8.empty(ctx, 1, 64, 2, 64, 16, 4, 16) for _ in range(2)]
    q, k, v = (torch.from_numpy(g.normal(0, 1, (4, n, 64)).astype(np.float32)).cuda() for n in (8, 2, 2))
    logits = torch.from_numpy(g.normal(0, 2, (4, 3, 100)).astype(np.float32)).cuda()
    draft, u = ints(g.integers(0, 100, (4, 2))), torch.rand((4, 3), device="cuda")
    pos, lens = ints([0] * 4), ints([1] * 4)

    def bufs():
        return dict(out=torch.zeros_like(q), lse=torch.zeros((4, 8), device="cuda"),
                    tokens=torch.zeros((4, 3), dtype=torch.int32, device="cuda"), count=ints([0] * 4))

    def work(kv, b):
        kv.resize(lens)
        kv.append(0, k, v, pos, ints_seqs)
        kv.attention(0, q, b["out"], pos, ints_seqs, lse=b["lse"])
        hale.verify_drafts(ctx, logits, draft, u, b["tokens"], b["count"])
    ints_seqs = ints(range(4))
    eager, replayed = bufs(), bufs()
    work(caches[0], eager)  # the context's workspace
    caches[0].resize(ints([0] * 4))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            work(caches[1], replayed)
        graphs.append(graph)
    for step in range(70):
        pos.fill_(step)
        lens.fill_(step + 1)
        k.mul_(1.02)
        work(caches[0], eager)
        graphs[step % 2].replay()
        ctx.check()
        for name in eager:
            assert torch.equal(eager[name], replayed[name]), (step, name)
    for a, b in zip(caches[0].__dict__.values(), caches[1].__dict__.values()):
        if isinstance(a, torch.Tensor):
            assert torch.equal(a, b)
