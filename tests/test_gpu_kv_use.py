"""The head norms, cache appends and paged attention as a serving loop uses them
together: prompts in chunks and then tokens, a captured decode step replayed with other
inputs, calls on streams of their own, caches past 32-bit offsets.  Attention is checked
against 64 bits over what the cache holds (test_gpu_kv_attention.py has the tolerance)."""
import numpy as np
import pytest

import kv_inputs as K
import mxfp4_inputs as X

pytestmark = pytest.mark.gpu
H, G, D, PAGE = 8, 2, 128, 16


@pytest.fixture(scope="module")
def M():
    import minirun_hip as M

    M.load()
    return M


class Layer:
    """What lies between a layer's projections, for the sequences of one cache."""

    def __init__(self, M, seed, mxfp4, pages=64, positions=512, d=D):
        import torch

        rng = np.random.default_rng(seed)
        self.M, self.rng, self.d = M, rng, d
        self.cache = M.KVCache.zeros(pages, G, PAGE, d, mxfp4=mxfp4)
        freqs = np.array(M.rope_frequencies(d))
        angle = np.arange(positions)[:, None] * freqs
        self.cos, self.sin = X.dev(np.cos(angle).astype(np.float32)), X.dev(np.sin(angle).astype(np.float32))
        self.wq, self.wk = (X.dev(1 + 0.1 * rng.standard_normal(d).astype(np.float32)) for _ in range(2))

    def rows(self, tokens):
        """Queries, keys and values of a projection, next to each other."""
        x, _ = K.values_of(self.rng, (tokens, (H + 2 * G) * self.d), False)
        d = self.d
        return (x[:, :H * d].view(tokens, H, d), x[:, H * d:(H + G) * d].view(tokens, G, d),
                x[:, (H + G) * d:].view(tokens, G, d))

    def step(self, q, k, v, positions, slots, table, lens, offsets=None, **kw):
        M = self.M
        how = dict(cos_t=self.cos, sin_t=self.sin, positions=positions, halves=True)
        q = M.head_norm_rope(q, q_weight=self.wq, **how)
        M.kv_append(self.cache, k, v, slots, normalize=True, norm_weight=self.wk, **how)
        return q, M.kv_attention(q, self.cache, table, lens, scale=self.d ** -0.5, q_offsets=offsets, **kw)

    def check(self, q, out, table, lens, offsets=None):
        k, v = (X.host(t) for t in self.cache.values())
        want, _, weight, terms = K.attention(X.host(q), k, v, table, lens, offsets, self.d ** -0.5)
        tol = weight * (X.BF16_ROUND + 2 * (self.d + 2) * K.MFMA * terms[..., None] + (max(lens) + 8) * K.MFMA)
        assert (np.abs(X.host(out) - want) <= tol + X.BF16_ROUND * np.abs(want)).all()


def i32(a):
    return X.dev(np.asarray(a, np.int32))


@pytest.mark.parametrize("mxfp4", [False, True])
def test_prompts_in_chunks_and_then_tokens(M, mxfp4):
    layer = Layer(M, 1, mxfp4)
    table = layer.rng.permutation(64)[:40].reshape(2, 20).astype(np.int32)
    lens = np.zeros(2, np.int64)
    # tokens of the two sequences in each call: chunks of prompts, drafts, single tokens
    for counts in ([100, 30], [40, 3], [1, 5], [1, 1], [0, 1], [1, 0], [60, 70], [1, 1]):
        offsets = np.cumsum([0] + counts)
        positions = np.concatenate([lens[b] + np.arange(c) for b, c in enumerate(counts)]).astype(np.int64)
        owner = np.repeat([0, 1], counts)
        slots = table[owner, positions // PAGE] * PAGE + positions % PAGE
        lens += counts
        single = counts == [1, 1]
        q, out = layer.step(*layer.rows(int(offsets[-1])), i32(positions), i32(slots), i32(table), i32(lens),
                            None if single else i32(offsets))
        layer.check(q, out, table, lens, None if single else offsets)


def test_a_prompt_is_its_tokens_one_by_one(M):
    """The same rows in one call and token by token: the caches hold the same bits."""
    import torch

    caches = []
    for chunk in (37, 1):
        layer = Layer(M, 2, True)
        q, k, v = layer.rows(37)
        table = i32([[5, 1, 3]])
        for t in range(0, 37, chunk):
            at = np.arange(t, t + chunk)
            slots = np.array([5, 1, 3])[at // PAGE] * PAGE + at % PAGE
            layer.step(q[t:t + chunk], k[t:t + chunk], v[t:t + chunk], i32(at), i32(slots), table, i32([t + chunk]),
                       i32([0, chunk]))
        caches.append(layer.cache)
    for a, b in zip(*([c.k, c.v, c.k_scales, c.v_scales] for c in caches)):
        assert torch.equal(a, b)


def capture(fn):
    import torch

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        fn()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = fn()
    torch.cuda.synchronize()
    return g, out


@pytest.mark.parametrize("hint", [40, 300000])
def test_captured_steps_replay_with_other_inputs(M, hint):
    """Two captured decode steps (of one layer each, their workspaces their own), replayed in
    turn while sequences grow, against the same step called eagerly."""
    import torch

    layers = [Layer(M, 3 + i, True, pages=4096) for i in range(2)]
    table = (np.arange(3)[:, None] * 20 + np.arange(20)).astype(np.int32)
    wide = np.full((3, 20000), -1, np.int32)
    wide[:, :20] = table
    state = []
    for layer in layers:
        q, k, v = (t.clone() for t in layer.rows(3))
        pos, slots, lens = i32([0, 0, 0]), i32([0, 0, 0]), i32([1, 1, 1])
        state.append([layer, q, k, v, pos, slots, lens, i32(wide)])
    graphs = [capture(lambda s=s: s[0].step(*s[1:6], s[7], s[6], max_kv_len=hint)) for s in state]
    at = np.array([0, 15, 200])
    for turn in range(4):
        for (g, (gq, gout)), s in zip(graphs, state):
            layer = s[0]
            for dst, src in zip(s[1:4], layer.rows(3)):
                dst.copy_(src)
            s[4].copy_(i32(at))
            s[5].copy_(i32(table[np.arange(3), at // PAGE] * PAGE + at % PAGE))
            s[6].copy_(i32(at + 1))
            gout.fill_(float("nan"))
            g.replay()
            torch.cuda.synchronize()
            kept = [gout.clone()] + [t.clone() for t in (layer.cache.k, layer.cache.v, layer.cache.k_scales, layer.cache.v_scales)]
            _, eager = layer.step(s[1], s[2], s[3], s[4], s[5], s[7], s[6], max_kv_len=hint)  # writes the same rows again
            torch.cuda.synchronize()
            for a, b in zip(kept, (eager, layer.cache.k, layer.cache.v, layer.cache.k_scales, layer.cache.v_scales)):
                assert torch.equal(a, b), turn
        at += 1


@pytest.mark.parametrize("hint", [0, 100])  # the keys in parts, joined, and whole
def test_captured_prompts_replay_with_other_lengths(M, hint):
    """A captured step of 300 tokens, replayed while they belong to other sequences of other lengths."""
    import torch

    layer = Layer(M, 12, True, pages=200, positions=1200)
    table = np.stack([np.arange(70) + 70 * b for b in range(2)]).astype(np.int32)
    q, k, v = (t.clone() for t in layer.rows(300))
    pos, slots, lens, offsets = i32(np.zeros(300)), i32(np.full(300, -1)), i32([0, 0]), i32([0, 0, 0])
    step = lambda: layer.step(q, k, v, pos, slots, i32_table, lens, offsets, max_kv_len=hint)
    i32_table = i32(table)
    g, (_, gout) = capture(step)
    have = np.zeros(2, np.int64)
    for counts in ([200, 100], [299, 0], [1, 250], [150, 150]):
        at = np.concatenate([have[b] + np.arange(c) for b, c in enumerate(counts)])
        owner = np.repeat([0, 1], counts)
        pad = 300 - len(at)
        have += counts
        for dst, src in zip((q, k, v), layer.rows(300)):
            dst.copy_(src)
        pos.copy_(i32(np.append(at, np.zeros(pad))))
        slots.copy_(i32(np.append(table[owner, at // PAGE] * PAGE + at % PAGE, np.full(pad, -1))))
        lens.copy_(i32(have))
        offsets.copy_(i32(np.cumsum([0] + counts)))
        gout.fill_(7)
        g.replay()
        torch.cuda.synchronize()
        got = gout.clone()
        _, eager = step()
        torch.cuda.synchronize()
        assert torch.equal(got[:len(at)], eager[:len(at)]) and (got[len(at):] == 7).all()


def test_captured_backward_replays(M):
    import torch

    T = 300
    rng = np.random.default_rng(8)
    q, k, dq, dk = (K.values_of(rng, (T, h, 64), False)[0] for h in (6, 2, 6, 2))
    w = X.dev(np.ones(64, np.float32))
    fn = lambda: M.head_norm_rope_backward(dq, q, dk, k, q_weight=w, k_weight=w)
    g, outs = capture(fn)
    for turn in range(4):
        dq.mul_(-1.5)
        for o in outs:
            o.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, fn())), turn
        torch.cuda.synchronize()


def test_calls_on_streams_of_their_own(M):
    """Two attentions at once, and a third thread's, give what they give alone."""
    import threading

    import torch

    layer = Layer(M, 4, True, pages=512)
    table = i32(np.arange(500).reshape(2, 250))
    layer.cache.k.random_()
    layer.cache.v.random_()
    layer.cache.k_scales.fill_(126)
    layer.cache.v_scales.fill_(126)
    lens = i32([4000, 3111])
    q = [layer.rows(2)[0].contiguous() for _ in range(3)]
    call = lambda i: M.kv_attention(q[i], layer.cache, table, lens, scale=0.1)
    want = [call(i) for i in range(3)]
    torch.cuda.synchronize()
    for _ in range(3):
        got, streams = [None] * 3, [torch.cuda.Stream() for _ in range(3)]

        def go(i):
            with torch.cuda.stream(streams[i]):
                for _ in range(20):
                    got[i] = call(i)

        threads = [threading.Thread(target=go, args=(i,)) for i in range(3)]
        [t.start() for t in threads]
        [t.join() for t in threads]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("mxfp4", [False, True])
def test_offsets_past_32_bits(M, mxfp4):
    """Pages that begin past 4 GiB of keys."""
    import torch

    page, dim = 64, 256
    pages = 2 ** 33 // (page * G * dim * (1 if mxfp4 else 4)) + 40
    cache = M.KVCache.zeros(pages, G, page, dim, mxfp4=mxfp4)
    rng = np.random.default_rng(6)
    T = 90
    k, k64 = K.values_of(rng, (T, G, dim), False)
    v, v64 = K.values_of(rng, (T, G, dim), False)
    table = np.array([[pages - 1, pages - 7]], np.int32)
    at = np.arange(T)
    M.kv_append(cache, k, v, i32(table[0, at // page].astype(np.int64) * page + at % page))
    few = M.KVCache(*(None if t is None else t[-7:].contiguous() for t in (cache.k, cache.v, cache.k_scales, cache.v_scales)))
    q, q64 = K.values_of(rng, (1, H, dim), False)
    a = M.kv_attention(q, cache, i32(table), i32([T]), scale=0.06)
    b = M.kv_attention(q, few, i32([[6, 0]]), i32([T]), scale=0.06)
    assert torch.equal(a, b) and torch.isfinite(a).all() and (a != 0).all()
    many, _ = K.values_of(rng, (T, H, dim), False)
    a = M.kv_attention(many, cache, i32(table), i32([T]), scale=0.06, q_offsets=i32([0, T]))
    b = M.kv_attention(many, few, i32([[6, 0]]), i32([T]), scale=0.06, q_offsets=i32([0, T]))
    assert torch.equal(a, b) and torch.isfinite(a).all()
    kk, vv = few.values()
    where = lambda x: np.concatenate([x[6], x[0]], 1)[:, :T]
    stored = where(X.host(kk)), where(X.host(vv))
    for got, x in zip(stored, (k64, v64)):
        x = np.moveaxis(x, 1, 0)
        if mxfp4:
            words, scales = K.quantize64(x.reshape(-1, dim))
            x = X.values(words, scales).reshape(x.shape)
        assert np.array_equal(got, x)


def test_norms_past_32_bits(M):
    """Rows that begin past 2^31 elements of the queries."""
    import torch

    T, D_ = 2 ** 16 + 3, 512  # 2^31 elements and some
    x = torch.randn(T, 64, D_, device="cuda", dtype=torch.bfloat16)
    y = M.head_norm_rope(x)
    for rows in (slice(0, 5), slice(T - 5, T)):
        assert torch.equal(y[rows], M.head_norm_rope(x[rows]))
