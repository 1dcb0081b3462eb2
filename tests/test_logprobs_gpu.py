"""Log probabilities of given tokens, entropy and alternatives: against log-softmax in 64 bits."""
import math

import pytest
import torch

from aegist_mixer import ops
from oracle import mixer_ref as R

pytestmark = pytest.mark.gpu
INF = float("inf")


def _ref(x, tokens, top):
    """fp64 on the CPU; rows that nothing is left of by their rule."""
    x = x.double().cpu()
    m = x.amax(1, keepdim=True)
    d = x - torch.where(torch.isinf(m), 0.0, m)  # (a sum of 3e38 and ln V is 3e38 in doubles too)
    lse = torch.logsumexp(d, 1, keepdim=True)
    lp = torch.where(torch.isinf(lse), -INF, d - lse)
    ent = -(lp.exp() * lp).nan_to_num(nan=0.0).sum(1)
    ent = torch.where(torch.isinf(lse[:, 0]), 0.0, ent)
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    return lp.gather(1, tokens.long().cpu().unsqueeze(1))[:, 0], ent, ids, lp.gather(1, ids), x


def _check(x, tokens, top, got):
    """Tolerances: x - m is exact to 2^-24 |x - m|, e^(x - m) is within |x - m| 2^-24 and 2 units of itself, where terms
    with |x - m| > 30 count for nothing; the sum of V terms in chains of at most 2^12 and a tree, each rounding
    2^-24 of the sum: at worst (30 + 2 + 2^12) 2^-24, at random far less: 2^-16 stands for both. The
    entropy's terms carry up to |x - m| <= 30 more."""
    lp, ent, ids, lps, xd = _ref(x, tokens, top)
    span = torch.where(torch.isfinite(lp), lp.abs(), 0.0) + 1
    fin = torch.isfinite(lp)
    a = got.logprob.cpu().double()
    assert torch.equal(torch.isfinite(a), fin) and torch.equal(a[~fin], lp[~fin])
    assert ((a - lp).abs()[fin] <= (2.0 ** -16 + span * 2.0 ** -22)[fin]).all()
    assert ((got.entropy.cpu().double() - ent).abs() <= 30 * 2.0 ** -16).all()
    if not top:
        assert got.top_ids is None and got.top_logprobs is None
        return
    assert torch.equal(got.top_ids.cpu().long(), ids)
    b = got.top_logprobs.cpu().double()
    fin = torch.isfinite(lps)
    assert torch.equal(b[~fin], lps[~fin])
    assert ((b - lps).abs()[fin] <= (2.0 ** -16 + (lps.abs() + 1) * 2.0 ** -22)[fin]).all()


def _case(T, V, dtype, seed=0, std=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, V, generator=g) * std).to(dtype), torch.randint(0, V, (T,), generator=g, dtype=torch.int32)


@pytest.mark.parametrize("T", [1, 2, 3, 61, 300])
@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 1000, 4099, 20000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_logprobs(dev, T, V, dtype):
    x, tok = _case(T, V, dtype, T + V)
    for top in sorted({0, 1, min(5, V), min(64, V)}):
        _check(x, tok, top, ops.token_logprobs(x.to(dev), tok.to(dev), top))


@pytest.mark.parametrize("T,V,top", [(1, 131072, 20), (1, 262147, 64), (7, 100003, 5), (130, 100003, 3), (1, 1_000_003, 10)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_logprobs_large(dev, T, V, top, dtype):
    x, tok = _case(T, V, dtype, T + V)
    _check(x, tok, top, ops.token_logprobs(x.to(dev), tok.to(dev), top))


@pytest.mark.parametrize("V", [5, 300, 9000, 70001])
@pytest.mark.parametrize("T", [1, 9, 300])
def test_ties_order_and_extremes(dev, T, V):
    """Rows that selection finds hard: all alike, ascending, descending, few distinct values, one peak, -0 beside +0."""
    g = torch.Generator().manual_seed(1)
    top = min(V, 64)
    rows = [torch.zeros(V), torch.arange(V) * 1e-3, -torch.arange(V) * 1e-3, torch.randint(0, 3, (V,), generator=g).float(),
            torch.where(torch.arange(V) == V - 1, 50.0, 0.0), torch.where(torch.arange(V) % 2 == 0, -0.0, 0.0),
            (torch.arange(V) % 256) * 0.01, (torch.arange(V) // 64) * -0.01, torch.full((V,), -3e38)]
    x = torch.stack([rows[t % len(rows)] for t in range(T)]) if T > 1 else rows[3].unsqueeze(0)
    tok = torch.randint(0, V, (T,), generator=g, dtype=torch.int32)
    _check(x, tok, top, ops.token_logprobs(x.to(dev), tok.to(dev), top))
    xb = x.bfloat16()
    _check(xb, tok, top, ops.token_logprobs(xb.to(dev), tok.to(dev), top))


@pytest.mark.parametrize("T,V", [(127, 16385), (128, 30001), (383, 32769), (384, 33001), (3, 8192), (3, 8193), (5, 16384)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_where_the_cutting_changes(dev, T, V, dtype):
    x, tok = _case(T, V, dtype, V)
    for top in (0, 6):
        _check(x, tok, top, ops.token_logprobs(x.to(dev), tok.to(dev), top))


@pytest.mark.parametrize("V", [4096, 16384, 65536])
@pytest.mark.parametrize("T", [2, 400])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_alternatives_side_by_side(dev, V, T, dtype):
    """The alternatives lie close together: in fours 1024 apart (one lane's logits), in one run of 64, all at the end."""
    x, tok = _case(T, V, dtype, V)
    at = torch.arange(V)
    x[0][(at % 1024 // 4 == 37)] += 40
    x[1, V // 2 - 9:V // 2 + 55] += 40
    x[T - 1, V - 64:] += 40
    _check(x, tok, 64, ops.token_logprobs(x.to(dev), tok.to(dev), 64))


@pytest.mark.parametrize("V", [7, 500, 40000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_rows(dev, V, dtype):
    """-inf in most places, in all but one, in all; the token itself ruled out; masks of the type's lowest value."""
    T, top = 12, min(V, 20)
    x, tok = _case(T, V, dtype, V)
    g = torch.Generator().manual_seed(2)
    x[:6].masked_fill_(torch.rand(6, V, generator=g) < 0.95, -INF)
    x[6], x[7] = -INF, -INF
    x[7, V - 1] = 1.0
    x[8, int(tok[8])] = -INF
    x[9, : V - 2] = torch.finfo(dtype).min
    x[10] = torch.finfo(dtype).min
    x[11] = torch.finfo(dtype).max
    _check(x, tok, top, ops.token_logprobs(x.to(dev), tok.to(dev), top))
    r = ops.token_logprobs(x.to(dev), tok.to(dev), top)
    assert r.logprob[6] == -INF and r.entropy[6] == 0 and r.top_ids[6].tolist() == list(range(top))
    assert r.entropy[7] == 0 and r.top_logprobs[7, 0] == 0


@pytest.mark.parametrize("V", [70, 30000])
@pytest.mark.parametrize("T", [5, 400])
def test_nan_infinity_and_other_tokens(dev, T, V):
    x, tok = _case(T, V, torch.float32, 3)
    x[0, 3], x[1, V - 1], x[2, 0] = float("nan"), INF, float("nan")
    x[2, 1:] = -INF
    tok[3], tok[4] = -1, V
    r = ops.token_logprobs(x.to(dev), tok.to(dev), 4)
    for t in range(3):
        assert all(torch.isnan(v[t]).all() for v in (r.logprob, r.entropy, r.top_logprobs))
    assert r.top_ids[0, 0] == 3 and r.top_ids[1, 0] == V - 1 and r.top_ids[2].tolist() == [0, 1, 2, 3]
    assert r.logprob[3] == 0 and torch.isnan(r.logprob[4])
    assert torch.isfinite(r.entropy[3:]).all() and torch.isfinite(r.top_logprobs[3:]).all()
    keep = tok.clone()
    keep[3:5] = 0
    _check(x[3:], keep[3:], 4, ops.token_logprobs(x[3:].to(dev), keep[3:].to(dev), 4))


@pytest.mark.parametrize("dtype,bits", [(torch.float32, 0x7f800001), (torch.float32, -0x400001), (torch.bfloat16, 0x7f81), (torch.bfloat16, -0x7f)])
@pytest.mark.parametrize("V", [300, 9001, 70001])
@pytest.mark.parametrize("top", [0, 1, 7])
def test_nan_of_either_kind(dev, dtype, bits, V, top):
    """Signaling NaNs of either sign, which maxima treat as they do not treat quiet ones."""
    x, tok = _case(6, V, dtype, 9)
    raw = x.view(torch.int32 if dtype == torch.float32 else torch.int16)
    raw[1, V // 3] = raw[4, V - 1] = bits
    assert torch.isnan(x[1, V // 3])
    r = ops.token_logprobs(x.to(dev), tok.to(dev), top)
    for t, at in ((1, V // 3), (4, V - 1)):
        assert torch.isnan(r.logprob[t]) and torch.isnan(r.entropy[t])
        if top:
            assert r.top_ids[t, 0] == at and torch.isnan(r.top_logprobs[t]).all()
    keep = torch.tensor([0, 2, 3, 5])
    _check(x[keep], tok[keep], top, type(r)(*(f if f is None else f[keep.to(dev)] for f in r)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [4, 300])
def test_strides_and_odd_places(dev, T, dtype):
    """Rows of a wider matrix, starting at any element."""
    wide, tok = _case(T, 5000, dtype, 4)
    for a, b in ((0, 4999), (1, 4500), (3, 1030), (7, 4097)):
        x = wide.to(dev)[:, a:b]
        t = (tok % (b - a)).to(dev)
        _check(wide[:, a:b], t.cpu(), 6, ops.token_logprobs(x, t, 6))
    lead = ops.token_logprobs(wide.to(dev).view(2, T // 2, 5000), tok.to(dev).view(2, T // 2), 3)
    flat = ops.token_logprobs(wide.to(dev), tok.to(dev), 3)
    assert lead.top_ids.shape == (2, T // 2, 3) and all(torch.equal(a.flatten(), b.flatten()) for a, b in zip(lead, flat))


def test_no_rows(dev):
    r = ops.token_logprobs(torch.empty(0, 9, device=dev), torch.empty(0, dtype=torch.int32, device=dev), 3)
    assert r.logprob.shape == (0,) and r.top_ids.shape == (0, 3)


def _head(kind, V, K, seed, dev):
    """(weight argument, scale argument, fp64 matrix)"""
    g = torch.Generator().manual_seed(seed)
    if kind == "q4":
        codes = torch.randint(0, 256, (V, K // 2), generator=g, dtype=torch.uint8)
        sc = (0.007 * (0.5 + torch.rand(V, K // 64, generator=g))).half()
        mn = (-7.5 * sc.float()).half()
        return ops.q4_pack(codes.to(dev), sc.to(dev), mn.to(dev)), None, R.q4_dequantize(codes, sc, mn, 64)
    w = torch.randn(V, K, generator=g) * 0.03
    if kind == "int8":
        q, s = R.qlinear_quantize(w)
        return q.to(dev), s.to(dev), q.double() * s.double().unsqueeze(1)
    return w.bfloat16().to(dev), None, w.bfloat16().double()


@pytest.mark.parametrize("kind", ["q4", "bf16", "int8"])
@pytest.mark.parametrize("T,V,K,top", [(1, 1000, 64, 5), (3, 5003, 128, 3), (17, 32768, 256, 1), (90, 4100, 192, 2), (700, 9001, 128, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_head_logprobs(dev, kind, T, V, K, top, dtype):
    """Against fp64 logits. A logit is off by at most (2^-16 (fp32 rows of int8 and bf16 weights count with 16 bits) +
    K 2^-24) sum |x w|; ids are compared where the logits of the list stand further apart than that."""
    w, s, wd = _head(kind, V, K, V + K, dev)
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, K, generator=g).to(dtype)
    tok = torch.randint(0, V, (T,), generator=g, dtype=torch.int32)
    r = ops.head_logprobs(x.to(dev), w, tok.to(dev), top, scale=s)
    logits = x.double() @ wd.t()
    # (q4: the minimum's and the codes' terms are summed apart, 16 scales at most where the weight is under 8.5)
    off = ((2.0 ** -16 + K * 2.0 ** -24) * 2 * (x.double().abs() @ wd.abs().t())).amax(1)
    lp, ent, ids, lps, _ = _ref(logits, tok, min(top + 1, V))
    assert ((r.logprob.cpu().double() - lp).abs() <= 2 * off + 2.0 ** -15).all()
    assert ((r.entropy.cpu().double() - ent).abs() <= 40 * off + 30 * 2.0 ** -16).all()
    gap = (lps[:, :-1] - lps[:, 1:]) > 2 * off.unsqueeze(1)
    sure = gap & torch.cat([torch.ones(T, 1, dtype=torch.bool), gap[:, :-1]], 1)
    assert sure.float().mean() > 0.5
    assert (r.top_ids.cpu().long() == ids[:, :top])[sure].all()
    assert ((r.top_logprobs.cpu().double() - lps[:, :top]).abs() <= 2 * off.unsqueeze(1) + 2.0 ** -15).all()


@pytest.mark.parametrize("V,T", [(65537, 1024), (131073, 513), (131073, 1535)])
@pytest.mark.parametrize("top", [0, 3])
def test_head_logprobs_in_blocks(dev, V, T, top):
    """More rows than 256 MiB of logits have: the last block, of one row, two or three, is cut into other splits than the
    blocks before it. Against the logits of bf16 products, exact in fp32 but for the order of 64 sums (the bounds
    of the test above, rows of bf16 values)."""
    K = 64
    w, _, wd = _head("bf16", V, K, 1, dev)
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, K, generator=g).bfloat16()
    tok = torch.randint(0, V, (T,), generator=g, dtype=torch.int32)
    r = ops.head_logprobs(x.to(dev), w, tok.to(dev), top)
    for t in (slice(0, 3), slice(T // 2, T // 2 + 2), slice(T - 4, T)):  # (rows of every block)
        xs = x[t].double()
        off = (K * 2.0 ** -23 * (xs.abs() @ wd.abs().t())).amax(1)
        lp, ent, _, lps, _ = _ref(xs @ wd.t(), tok[t], top)
        assert ((r.logprob[t].cpu().double() - lp).abs() <= 2 * off + 2.0 ** -15).all()
        assert ((r.entropy[t].cpu().double() - ent).abs() <= 40 * off + 30 * 2.0 ** -16).all()
        if top:
            assert ((r.top_logprobs[t].cpu().double() - lps).abs() <= 2 * off.unsqueeze(1) + 2.0 ** -15).all()
    one = ops.head_logprobs(x[T // 3:T // 3 + 1].to(dev), w, tok[T // 3:T // 3 + 1].to(dev), top)
    assert (one.logprob - r.logprob[T // 3:T // 3 + 1]).abs().max() < 1e-3


@pytest.mark.parametrize("T", [1, 20, 300])
def test_quantize_project_score_together(dev, T):
    """A head quantised, multiplied and scored: the head's answers are those of the logits that linear_q4 makes of
    the same rows, whichever way the vocabulary is cut."""
    V, K = 20011, 256
    w4 = ops.q4_quantize(0.05 * torch.randn(V, K, device=dev), 32)
    x = torch.randn(T, K, device=dev)
    tok = torch.randint(0, V, (T,), device=dev, dtype=torch.int32)
    a = ops.head_logprobs(x, w4, tok, 8)
    logits = ops.linear_q4(x, w4)
    b = ops.token_logprobs(logits, tok, 8)
    # the product may be cut into other tiles: the bound of two ways of adding K products in fp32
    off = 2 * (K * 2.0 ** -24) * (x.abs().double() @ (ops.q4_dequantize(w4).abs().double().t() + 0.3)).amax()
    assert (a.logprob - b.logprob).abs().max() <= 2 * off and (a.top_logprobs - b.top_logprobs).abs().max() <= 2 * off
    ref = torch.log_softmax(x.double() @ ops.q4_dequantize(w4).double().t(), 1)
    assert (a.logprob.double() - ref.gather(1, tok.long().unsqueeze(1))[:, 0]).abs().max() <= 2 * off + 2.0 ** -15


@pytest.mark.parametrize("T", [1, 70, 600])
def test_same_bits_again_and_in_graphs(dev, T):
    V, K, top = 30011, 128, 7
    w4 = ops.q4_quantize(0.05 * torch.randn(V, K, device=dev))
    x = torch.randn(T, K, device=dev)
    tok = torch.randint(0, V, (T,), device=dev, dtype=torch.int32)
    xs, graphs, outs = [x.clone(), x.clone()], [], []
    first = ops.head_logprobs(x, w4, tok, top)
    assert all(torch.equal(a, b) for a, b in zip(first, ops.head_logprobs(x, w4, tok, top)))
    for xi in xs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append((ops.head_logprobs(xi, w4, tok, top), ops.token_logprobs(xi, tok % K, top)))
        graphs.append(gr)
    for _ in range(3):
        for xi, gr, o in zip(xs, graphs, outs):
            xi.copy_(torch.randn(T, K, device=dev))
            gr.replay()
            ops.head_logprobs(torch.randn(T + 5, K, device=dev), w4, torch.zeros(T + 5, device=dev, dtype=torch.int32), top)
            torch.cuda.synchronize()
            for a, b in zip(o[0] + o[1], ops.head_logprobs(xi, w4, tok, top) + ops.token_logprobs(xi, tok % K, top)):
                assert torch.equal(a, b)


def test_more_rows_than_a_grid(dev):
    """2^20 rows and some, and tokens at the ends of their type."""
    T, V = 2 ** 20 + 7, 5
    x = torch.randn(T, V, device=dev)
    tok = torch.randint(0, V, (T,), device=dev, dtype=torch.int32)
    tok[::1000] = -2 ** 31
    tok[1::1000] = 2 ** 31 - 1
    r = ops.token_logprobs(x, tok, 2)
    assert (r.logprob[::1000] == 0).all() and torch.isnan(r.logprob[1::1000]).all()
    for t in (slice(2, 900), slice(T - 20, T)):
        ok = (tok[t] >= 0) & (tok[t] < V)
        keep = torch.where(ok, tok[t], 0)
        _check(x[t].cpu()[ok.cpu()], keep.cpu()[ok.cpu()], 2, type(r)(*(f[t][ok] for f in r)))


@pytest.mark.parametrize("top", [0, 5])
def test_logits_past_32_bits(dev, top):
    """More than 2^31 logits: the rows on both sides of the offsets 2^31 and 2^32 bytes, and the last."""
    V, T = 131072 + 3, 16500
    x = torch.empty(T, V, device=dev, dtype=torch.bfloat16)
    x[:64].normal_()
    for t in range(64, T, 64):
        x[t:t + 64] = x[:min(64, T - t)]
    tok = torch.randint(0, V, (T,), device=dev, dtype=torch.int32)
    r = ops.token_logprobs(x, tok, top)
    for t in (0, 2 ** 30 // V, 2 ** 31 // V, T - 2):
        t = slice(t, t + 2)
        _check(x[t].cpu(), tok[t].cpu(), top, type(r)(*(f if f is None else f[t] for f in r)))


@pytest.mark.parametrize("T", [1, 40])
def test_two_calls_at_once(dev, T):
    """Calls on two streams, each with a workspace of its own, do not disturb each other."""
    V, K, top = 60001, 256, 9
    w4 = ops.q4_quantize(0.05 * torch.randn(V, K, device=dev))
    xs = [torch.randn(T, K, device=dev) for _ in range(2)]
    tok = torch.randint(0, V, (T,), device=dev, dtype=torch.int32)
    want = [ops.head_logprobs(x, w4, tok, top) + (ops.linear_q4(x, w4),) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.head_logprobs(xs[i], w4, tok, top) + (ops.linear_q4(xs[i], w4),))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i]))


@pytest.mark.parametrize("kind", ["q4", "bf16", "int8"])
def test_head_takes_strides_and_leading_dimensions(dev, kind):
    """Rows of a wider matrix, a batch of sequences padded with -1, and the same answers as packed rows."""
    V, K, top = 3001, 128, 4
    w, s, _ = _head(kind, V, K, 3, dev)
    wide = torch.randn(2, 9, K + 64, device=dev).bfloat16()
    x = wide[..., 64:]
    tok = torch.randint(0, V, (2, 9), device=dev, dtype=torch.int32)
    tok[0, 5:] = -1
    r = ops.head_logprobs(x, w, tok, top, scale=s)
    flat = ops.head_logprobs(x.reshape(18, K).contiguous(), w, tok.flatten(), top, scale=s)
    assert r.logprob.shape == (2, 9) and r.top_ids.shape == (2, 9, top)
    assert all(torch.equal(a.flatten(), b.flatten()) for a, b in zip(r, flat))
    assert (r.logprob[0, 5:] == 0).all() and (r.logprob[0, :5] < 0).all() and torch.isfinite(r.entropy).all()


def test_head_scales_bf16_rows(dev):
    """A bf16 head with a scale per row, as the projections take it."""
    V, K, T = 2003, 64, 5
    w, _, wd = _head("bf16", V, K, 4, dev)
    sc = (0.5 + torch.rand(V, generator=torch.Generator().manual_seed(1))).bfloat16()
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(2))
    tok = torch.arange(T, dtype=torch.int32) * 400
    r = ops.head_logprobs(x.to(dev), w, tok.to(dev), scale=sc.to(dev))
    wd = wd * sc.double().unsqueeze(1)
    off = ((2.0 ** -16 + K * 2.0 ** -24) * 2 * (x.abs().double() @ wd.abs().t())).amax(1)
    lp, ent, _, _, _ = _ref(x.double() @ wd.t(), tok, 0)
    assert ((r.logprob.cpu().double() - lp).abs() <= 2 * off + 2.0 ** -15).all()
    assert ((r.entropy.cpu().double() - ent).abs() <= 40 * off + 30 * 2.0 ** -16).all()


@pytest.mark.parametrize("T,V,K", [(70, 20000, 64), (300, 2053, 128), (257, 9001, 192), (1000, 32768, 64), (515, 4225, 2048)])
@pytest.mark.parametrize("top", [0, 1])
def test_head_of_many_rows_without_logits(dev, T, V, K, top):
    """Rows whose statistics the product itself leaves: the answers of the logits that linear makes of the same rows (the
    same sums in the same order, so the same ids), also where a row is NaN, infinite or all alike."""
    g = torch.Generator().manual_seed(V)
    w = (torch.randn(V, K, generator=g) * 0.05).bfloat16().to(dev)
    x = torch.randn(T, K, generator=g).bfloat16()
    x[1], x[2, 3], x[3, K - 1], x[T - 1] = 0, float("nan"), INF, 0
    w[V - 1], w[V // 2] = w[5], w[5]  # equal logits: the lowest token
    tok = torch.randint(0, V, (T,), generator=g, dtype=torch.int32)
    tok[4], tok[5], tok[6], tok[7] = -1, V, V - 1, 0
    x, tok = x.to(dev), tok.to(dev)
    a, b = ops.head_logprobs(x, w, tok, top), ops.token_logprobs(ops.linear(x, w), tok, top)
    # both are within the bounds of _check of the same logits
    for p, q, off in zip(a, b, (2.0 ** -15, 60 * 2.0 ** -16, 0, 2.0 ** -15)):
        if p is None:
            assert q is None
        elif p.dtype == torch.int32:
            assert torch.equal(p, q)
        else:
            assert torch.equal(torch.isnan(p), torch.isnan(q)) and torch.isnan(p[2]).all() and torch.isnan(p[3]).all()
            ok = ~torch.isnan(p)
            assert ((p - q).abs()[ok] <= off + q.abs()[ok] * 2.0 ** -21).all()
    assert abs(float(a.logprob[1]) + math.log(V)) < 1e-4 and abs(float(a.entropy[T - 1]) - math.log(V)) < 1e-3
    assert a.logprob[4] == 0 and torch.isnan(a.logprob[5])
    if top:
        assert a.top_ids[1, 0] == 0 and a.top_ids[2, 0] == 0 and (a.top_ids[8:] != V - 1).all()
    again = ops.head_logprobs(x, w, tok, top)
    assert all(p is None or torch.equal(p.nan_to_num(nan=7.0), q.nan_to_num(nan=7.0)) for p, q in zip(a, again))


def test_many_rows_of_a_wider_matrix_in_a_graph(dev):
    """Rows with a stride, and the statistics of the product captured and replayed between eager calls."""
    T, V, K = 300, 9001, 128
    w = (torch.randn(V, K, device=dev) * 0.05).bfloat16()
    wide = torch.randn(T, K + 64, device=dev).bfloat16()
    x = wide[:, 64:]
    tok = torch.randint(0, V, (T,), device=dev, dtype=torch.int32)
    ops.head_logprobs(x, w, tok, 1)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = ops.head_logprobs(x, w, tok, 1)
    for _ in range(3):
        wide.copy_(torch.randn(T, K + 64, device=dev))
        gr.replay()
        ops.head_logprobs(torch.randn(T + 70, K, device=dev).bfloat16(), w, torch.zeros(T + 70, device=dev, dtype=torch.int32), 1)
        torch.cuda.synchronize()
        for a, b in zip(out, ops.head_logprobs(x.contiguous(), w, tok, 1)):
            assert torch.equal(a, b)


def test_one_row_without_leading_dimensions(dev):
    x, tok = _case(1, 700, torch.float32, 5)
    a, b = ops.token_logprobs(x[0].to(dev), tok[0].to(dev), 3), ops.token_logprobs(x.to(dev), tok.to(dev), 3)
    assert a.logprob.shape == () and a.top_ids.shape == (3,)
    assert all(torch.equal(p, q[0]) for p, q in zip(a, b))


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("T", [1, 2, 3, 16, 70, 300, 1000])
@pytest.mark.parametrize("V", [1003, 9001])
def test_head_counts_fp32_rows_with_all_their_bits(dev, kind, T, V):
    """Values 1 + i 2^-7 + 2^-8 + 2^-17 against weights of 0 and 1: every partial sum is a multiple of 2^-17 below 2^7, so
    the logits are exact in fp32 in any order, and held to the tolerances of given logits. The first 16 bits of a value
    alone are 2^-17 off, up to 64 2^-17 in the difference of two logits: 16 of those tolerances. Beside them rows at the
    ends of fp32's range, of zeros and with a NaN or an infinity."""
    K, top = 64, 5
    g = torch.Generator().manual_seed(T + V)
    x = 1 + torch.randint(0, 64, (T, K), generator=g) * 2.0 ** -7 + 2.0 ** -8 + 2.0 ** -17
    x *= torch.where(torch.arange(T) % 3 == 2, -1.0, 1.0).unsqueeze(1)
    w = (torch.arange(K) < torch.randint(0, K + 1, (V, 1), generator=g)).float()
    tok = torch.randint(0, V, (T,), generator=g, dtype=torch.int32)
    if T > 10:
        x[3], x[4], x[5] = 0, 0, 1e-38
        x[4, 20] = 3.3e38
    args = (w.to(dev).to(torch.bfloat16), None) if kind == "bf16" else (w.to(dev).to(torch.int8), torch.ones(V, device=dev).bfloat16())
    r = ops.head_logprobs(x.to(dev), args[0], tok.to(dev), top, scale=args[1])
    keep = torch.arange(T) != 5  # (logits next to 0: ties by the order of their sums)
    _check((x.double() @ w.double().t())[keep], tok[keep], top, type(r)(*(f[keep.to(dev)] for f in r)))
    if T > 10:
        assert abs(float(r.logprob[5]) + math.log(V)) < 1e-4
        xb = x.clone()
        xb[0, 3], xb[T - 1, K - 1] = float("nan"), INF
        b = ops.head_logprobs(xb.to(dev), args[0], tok.to(dev), top, scale=args[1])
        for p, q in zip(b, r):
            assert torch.equal(p[1:T - 1], q[1:T - 1])
        assert all(torch.isnan(p[t]).all() for p in (b.logprob, b.entropy, b.top_logprobs) for t in (0, T - 1))


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_head_of_fp32_rows_takes_strides_and_graphs(dev, kind):
    """Rows of a wider matrix, replayed between eager calls, and a last block that is smaller than the ones before it."""
    T, V, K, top = 40, 5003, 128, 3
    w, s, _ = _head(kind, V, K, 3, dev)
    wide = torch.randn(T, K + 64, device=dev)
    x = wide[:, 64:]
    tok = torch.randint(0, V, (T,), device=dev, dtype=torch.int32)
    ops.head_logprobs(x, w, tok, top, scale=s)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = ops.head_logprobs(x, w, tok, top, scale=s)
    for _ in range(3):
        wide.copy_(torch.randn(T, K + 64, device=dev))
        gr.replay()
        ops.head_logprobs(torch.randn(3 * T, K, device=dev), w, torch.zeros(3 * T, device=dev, dtype=torch.int32), top, scale=s)
        torch.cuda.synchronize()
        for a, b in zip(out, ops.head_logprobs(x.contiguous(), w, tok, top, scale=s)):
            assert torch.equal(a, b)
    V = 2 ** 22 + 5  # 15 rows to a block of 256 MiB: 2 blocks and one row
    w = (torch.randn(V, 16, device=dev) * 0.05).bfloat16()
    x, tok = torch.randn(31, 16, device=dev), torch.randint(0, V, (31,), device=dev, dtype=torch.int32)
    a, b = ops.head_logprobs(x, w, tok, top), ops.head_logprobs(x[28:].contiguous(), w, tok[28:], top)
    # 16 products in another order
    off = 2 * 16 * 2.0 ** -24 * 2 * float((x.abs() @ w.float().abs().t()).amax()) + 2.0 ** -15
    assert (a.logprob[28:] - b.logprob).abs().max() <= off and (a.top_logprobs[28:] - b.top_logprobs).abs().max() <= off


def test_head_refuses_rows_that_are_not_aligned(dev):
    V, K = 100, 64
    w, tok = torch.zeros(V, K, device=dev).bfloat16(), torch.zeros(4, device=dev, dtype=torch.int32)
    wide = torch.zeros(4, K + 6, device=dev)
    for x in (wide[:, :K], torch.zeros(4, K + 4, device=dev)[:, 1:1 + K]):
        with pytest.raises(ops.AegistError, match="aligned"):
            ops.head_logprobs(x, w, tok)
    with pytest.raises(ops.AegistError, match="multiple of 16"):
        ops.head_logprobs(torch.zeros(4, 24, device=dev), torch.zeros(V, 24, device=dev).bfloat16(), tok)


@pytest.mark.parametrize("V", [100, 3000, 9001, 40000, 70001])
@pytest.mark.parametrize("T", [10, 400])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_logits_alike(dev, V, T, dtype):
    """Most of a row equal, at the type's lowest value or in the middle, with few or many above it and others below it
    among the first tokens, in the middle or nowhere."""
    g = torch.Generator().manual_seed(V)
    low, at = torch.finfo(dtype).min, torch.arange(V)
    live = torch.randperm(V, generator=g)[:16]
    rows = [torch.full((V,), low) for _ in range(4)] + [torch.zeros(V) for _ in range(5)]
    for r in rows[:2]:
        r[live[:3]] = torch.tensor([1.0, 2.0, 2.0])
    rows[1][:min(200, V // 2)] = -INF                       # none of the first tokens is at the mask
    rows[2][at % 2 == 0] = -INF
    rows[3][V - min(1000, V // 2):] = torch.randn(min(1000, V // 2), generator=g)
    rows[4][live] = torch.arange(16) * 0.25 + 0.25          # above the others, fewer than asked for
    rows[5][torch.randperm(V, generator=g)[:min(300, V // 2)]] = 3.0   # two values alike, one more often than asked for
    rows[6][:min(150, V // 2)] = -1.0                       # the lowest tokens are below
    rows[7][at % 2 == 0] = -0.0
    rows[7][live[:5]] = 1e-3
    rows[8][live] = -1.0
    rows.append(torch.full((V,), torch.finfo(dtype).max))
    x = torch.stack([rows[t % 10] for t in range(T)]).to(dtype)
    tok = torch.where(torch.arange(T) % 2 == 0, live[torch.arange(T) % 16], torch.randint(0, V, (T,), generator=g)).int()
    for top in (1, 3, 20, 64):
        _check(x, tok, top, ops.token_logprobs(x.to(dev), tok.to(dev), top))


def test_masks_of_the_lowest_value_cost_about_what_minus_infinity_costs(dev):
    """(By maxima one after the other 20 alternatives took 18 times as long, 64 of them 50 times.)"""
    T, V, top = 1000, 32768, 20
    x = torch.randn(T, V, device=dev)
    keep = torch.rand(T, V, device=dev) < 16 / V
    tok = torch.zeros(T, dtype=torch.int32, device=dev)
    def us(mask):
        y, best = torch.where(keep, x, mask), INF
        for _ in range(8):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(8):
                ops.token_logprobs(y, tok, top)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best
    assert us(torch.finfo(torch.float32).min) < 6 * us(-INF)


def test_head_of_fp32_rows_in_blocks_of_what_they_are_split_into(dev):
    """A short vocabulary and long rows: blocks of 682 rows by the split rows. Logits exact in fp32, as above."""
    T, V, K = 700, 100, 65536
    g = torch.Generator().manual_seed(1)
    x, w = torch.zeros(T, K), (torch.rand(V, K, generator=g) < 0.5).float()
    x[:, 5::1024] = 1 + torch.randint(0, 64, (T, 64), generator=g) * 2.0 ** -7 + 2.0 ** -8 + 2.0 ** -17
    tok = torch.randint(0, V, (T,), generator=g, dtype=torch.int32)
    r = ops.head_logprobs(x.to(dev), w.to(dev).bfloat16(), tok.to(dev), 4)
    _check(x[:, 5::1024].double() @ w[:, 5::1024].double().t(), tok, 4, r)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("T,V", [(64, 3001), (65, 3001), (129, 1001), (127 + 30, 2 ** 19 + 3), (2 * 127 + 65, 2 ** 19 + 3)])
def test_head_where_the_split_rows_stop_being_stacked(dev, kind, T, V):
    """64 rows and more, and last blocks of 30 and 65 rows behind ones of 127. Logits exact in fp32, as above."""
    K, top = 64, 3
    g = torch.Generator().manual_seed(T)
    x = 1 + torch.randint(0, 64, (T, K), generator=g) * 2.0 ** -7 + 2.0 ** -8 + 2.0 ** -17
    w = (torch.arange(K) < torch.randint(0, K + 1, (V, 1), generator=g)).to(dev)
    tok = torch.randint(0, V, (T,), generator=g, dtype=torch.int32)
    args = (w.bfloat16(), None) if kind == "bf16" else (w.to(torch.int8), torch.ones(V, device=dev).bfloat16())
    r = ops.head_logprobs(x.to(dev), args[0], tok.to(dev), top, scale=args[1])
    rows = torch.tensor([0, 1, 63, T - 31, T - 30, T - 29, T - 1])
    _check(x[rows].double() @ w.cpu().double().t(), tok[rows], top, type(r)(*(f[rows.to(dev)] for f in r)))
