"""Heads whose product leaves the rows' statistics and no logits: sizes taken from the choice itself. Rows and weights are
small whole numbers, so that the logits are exact in fp32 and held to the tolerances of given logits."""
import ctypes

import pytest
import torch

from aegist_mixer import _lib, ops

INF = float("inf")
# vocabularies that end 1 column into a tile's first or second half, in the middle of one, and at one's end
SIZES = [(200, 32769, 64), (400, 32897, 128), (1000, 9001, 192), (2000, 4225, 64), (769, 10007, 192), (515, 16385, 128),
         (1300, 8193, 320), (257, 50257, 64), (1000, 32768, 2048), (1025, 8193, 128)]


def _by_statistics(T, V, K, ldx=0):
    fn = _lib.lib()._ZN6aegist17proj_is_gemm_bf16EPKvixS1_iPKtiii
    fn.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p] + [ctypes.c_int] * 3
    fn.restype = ctypes.c_bool
    return V >= 256 and fn(256, _lib.BF16, ldx or K, 256, _lib.BF16, None, T, V, K)


def test_sizes_reach_the_statistics():
    for T, V, K in SIZES:
        assert _by_statistics(T, V, K) and _by_statistics(T, V, K, K + 64)
        # whole numbers up to 4 against up to 3: partial sums below 2^24
        assert K * 12 < 2 ** 24


def _whole(shape, most, seed, dev):
    g = torch.Generator(dev).manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g, device=dev).bfloat16()


def _check(x, w, tok, top, r, rows=slice(None), scale=1.0):
    """Of given logits: logprob and alternative within 2^-16 + (|logprob| + 1) 2^-22, the entropy within 30 2^-16 (sums of V
    terms and their exponentials), ids equal, the lower token of equal logits."""
    logits = x[rows].double() @ w.double().t()
    V = w.shape[0]
    lse = torch.logsumexp(logits, 1)
    t = tok[rows].long()
    inside = (t >= 0) & (t < V)
    lp = logits.gather(1, t.clamp(0, V - 1).unsqueeze(1))[:, 0] - lse
    got = r.logprob[rows].double()
    assert (got[t < 0] == 0).all() and torch.isnan(got[t >= V]).all()
    out = inside & torch.isinf(lp)
    assert torch.equal(got[out], lp[out])
    ok = inside & ~out
    assert ((got - lp).abs() <= 2.0 ** -16 + (lp.abs() + 1) * 2.0 ** -22)[ok].all()
    p = torch.exp(logits - lse.unsqueeze(1))
    ent = -(p * (logits - lse.unsqueeze(1))).nan_to_num(nan=0.0).sum(1)
    assert ((r.entropy[rows].double() - ent).abs() <= 30 * 2.0 ** -16).all()
    if top:
        m = logits.amax(1)
        first = torch.where(logits == m.unsqueeze(1), torch.arange(V, device=x.device), V).amin(1)
        assert torch.equal(r.top_ids[rows][:, 0].long(), first)
        best = m - lse
        assert ((r.top_logprobs[rows][:, 0].double() - best).abs() <= 2.0 ** -16 + (best.abs() + 1) * 2.0 ** -22).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,K", SIZES)
@pytest.mark.parametrize("top", [0, 1])
def test_statistics(dev, T, V, K, top):
    """Against 64 bits: tokens of every column of the last tiles and outside the vocabulary, the largest logit in the last
    column and twice (once on either side of a tile's edge), rows of zeros, and rows with a NaN or an infinity."""
    x, w = _whole((T, K), 4, T, dev), _whole((V, K), 3, V, dev)
    w[V - 1] = 3 * torch.sign(x[9] + 0.5)
    edge = (V - 1) // 256 * 256
    w[edge - 1] = w[edge - 200] = w[3] = 3 * torch.sign(x[10] + 0.5)
    x[0] = x[T - 1] = 0
    tok = torch.randint(0, V, (T,), device=dev, dtype=torch.int32)
    n = min(130, T // 2)
    tok[20:20 + n] = V - 1 - torch.arange(n, device=dev, dtype=torch.int32)
    for i, t in enumerate((-1, -2 ** 31, V, 2 ** 31 - 1, V - 1, 0, V - 1, 3)):
        tok[4 + i] = t
    r = ops.head_logprobs(x, w, tok, top)
    _check(x, w, tok, top, r)
    if top:
        assert r.top_ids[9, 0] == V - 1 and r.top_ids[10, 0] == 3 and r.top_ids[0, 0] == 0 and r.top_ids[T - 1, 0] == 0
    xb = x.clone()
    bad = (1, 2, T - 2)
    xb[1, 3], xb[2, K - 1], xb[T - 2, 0] = float("nan"), INF, -INF
    b = ops.head_logprobs(xb, w, tok, top)
    keep = torch.ones(T, dtype=torch.bool, device=dev)
    keep[list(bad)] = False
    for p, q in zip(b, r):
        if p is not None:
            assert torch.equal(p[keep].nan_to_num(nan=7.0), q[keep].nan_to_num(nan=7.0))
    for t in bad:
        assert torch.isnan(b.logprob[t]) and torch.isnan(b.entropy[t])
        if top:
            assert torch.isnan(b.top_logprobs[t]).all()
    if top:
        assert b.top_ids[1, 0] == 0  # every logit is NaN


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,K", [(200, 32769, 64), (400, 32897, 128), (1000, 9001, 192)])
def test_infinite_logits_beside_the_end(dev, T, V, K):
    """Logits of -inf, of NaN and of +inf in the last tiles, whose columns past the vocabulary are masked."""
    x, w = _whole((T, K), 4, T, dev).abs() + 1, _whole((V, K), 3, V, dev)
    tok = torch.randint(0, V, (T,), device=dev, dtype=torch.int32)
    tok[:4] = torch.tensor([V - 1, V - 2, 0, V - 130], dtype=torch.int32)
    wm = w.clone()
    wm[[V - 1, V - 130, 0]] = -3e38  # (a product of it and 2 or more is -inf)
    x[:, 0] = 4
    r = ops.head_logprobs(x, wm, tok, 1)
    assert (r.logprob[[0, 2, 3]] == -INF).all() and torch.isfinite(r.entropy).all()
    masked = wm.clone()
    masked[[V - 1, V - 130, 0]] = 0
    logits = x.double() @ masked.double().t()
    logits[:, [V - 1, V - 130, 0]] = -INF
    lse = torch.logsumexp(logits, 1)
    lp = logits.gather(1, tok.long().unsqueeze(1))[:, 0] - lse
    fin = torch.isfinite(lp)
    assert torch.equal(torch.isfinite(r.logprob), fin) and ((r.logprob.double() - lp).abs() <= 2.0 ** -16 + (lp.abs() + 1) * 2.0 ** -22)[fin].all()
    assert torch.equal(logits.gather(1, r.top_ids.long())[:, 0], logits.amax(1))
    for value, name in ((float("nan"), "nan"), (3e38, "inf")):
        for at in (V - 1, V - 130, 0):
            wb = w.clone()
            wb[at] = value
            r = ops.head_logprobs(x, wb, tok, 1)
            assert (r.top_ids[:, 0] == at).all(), (name, at)
            assert all(torch.isnan(v).all() for v in (r.logprob, r.entropy, r.top_logprobs))


@pytest.mark.gpu
@pytest.mark.parametrize("top", [0, 1])
def test_statistics_of_strided_rows_in_graphs_and_on_two_streams(dev, top):
    """Rows of a wider matrix, captured and replayed between eager calls of another size, and two streams at once."""
    T, V, K = 400, 32897, 128
    w = _whole((V, K), 3, 1, dev)
    wides = [_whole((T, K + 64), 4, i, dev) for i in range(2)]
    xs = [wide[:, 64:] for wide in wides]
    tok = torch.randint(0, V, (T,), device=dev, dtype=torch.int32)
    same = lambda a, b: all(p is None or torch.equal(p, q) for p, q in zip(a, b))  # noqa: E731
    want = [ops.head_logprobs(x.contiguous(), w, tok, top) for x in xs]
    _check(xs[0], w, tok, top, want[0])
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.head_logprobs(xs[i], w, tok, top))
    torch.cuda.synchronize()
    assert all(same(g, want[i]) for i in range(2) for g in got[i])
    graphs, outs = [], []
    for x in xs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.head_logprobs(x, w, tok, top))
        graphs.append(gr)
    for i in range(3):
        for wide, x, gr, o in zip(wides, xs, graphs, outs):
            wide.copy_(_whole((T, K + 64), 4, 10 + i, dev))
            gr.replay()
            ops.head_logprobs(_whole((T + 300, K), 4, 5, dev), w, torch.zeros(T + 300, device=dev, dtype=torch.int32), top)
            torch.cuda.synchronize()
            assert same(o, ops.head_logprobs(x.contiguous(), w, tok, top))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [2049, 2500])
def test_statistics_in_blocks(dev, T):
    """More rows than 256 MiB of logits have: a block by its statistics, then one of one row or of many."""
    V, K = 32771, 64
    block = 2 ** 28 // (4 * V)
    assert _by_statistics(block, V, K) and T > block
    x, w = _whole((T, K), 4, 3, dev), _whole((V, K), 3, 4, dev)
    tok = torch.randint(0, V, (T,), device=dev, dtype=torch.int32)
    r = ops.head_logprobs(x, w, tok, 1)
    for t in (slice(0, 300), slice(block - 100, min(T, block + 100)), slice(T - 100, T)):
        _check(x, w, tok, 1, r, t)
