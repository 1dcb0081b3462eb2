"""4-bit weights: quantising, packing, reading back and the product, against the definitions in 64 bits."""
import numpy as np
import pytest
import torch

from aegist_mixer import _lib, ops
from oracle import mixer_ref as R

pytestmark = pytest.mark.gpu


def _weight(N, K, G, seed, mins=True):
    """Random codes, scales and minima on the CPU, and the fp64 matrix they stand for."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    scale = (0.007 * (0.5 + torch.rand(N, K // G, generator=g))).half()
    mn = (-(7 + torch.rand(N, K // G, generator=g)) * scale.float()).half()
    w = R.q4_dequantize(codes, scale, mn if mins else -8 * scale.double(), G)
    return codes, scale, mn if mins else None, w


def _pack(codes, scale, mn, dev):
    return ops.q4_pack(codes.to(dev), scale.to(dev), None if mn is None else mn.to(dev))


def _bound(x, codes, scale, mn, G):
    """What rounding can put an output off by: an activation counts with 22 bits below itself (and 34 below the
    largest of its row); the products and the sums of a group's x are exact or rounded to 24 bits, added in
    chains of at most 128 and then K / G; the scale and the minimum are applied with a rounding each."""
    N, K = codes.shape[0], 2 * codes.shape[1]
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(1).double()
    s = scale.double().abs().repeat_interleave(G, 1)
    m = (mn.double().abs() if mn is not None else 8 * scale.double()).repeat_interleave(G, 1)
    xa = x.double().abs()
    wa = (c * s + m).t()
    return (2.0 ** -22 + (128 + K // G + 8) * 2.0 ** -24) * (xa @ wa) + 2.0 ** -34 * xa.amax(1, keepdim=True) * wa.sum(0)


def _check(x, w4, wt, dev, **kw):
    codes, scale, mn, w = wt
    y = ops.linear_q4(x.to(dev) if not x.is_cuda else x, w4, **kw)
    ref = x.cpu().double() @ w.t()
    off = (y.cpu().double() - ref).abs()
    assert (off <= _bound(x.cpu(), codes, scale, mn, w4.group)).all(), (off / _bound(x.cpu(), codes, scale, mn, w4.group)).max()
    return y


@pytest.mark.parametrize("N,K,G", [(1, 32, 32), (16, 64, 64), (17, 96, 32), (33, 128, 128), (100, 320, 64), (7, 1152, 128),
                                   (256, 2048, 64)])
@pytest.mark.parametrize("mins", [True, False])
def test_pack_and_dequantize(dev, N, K, G, mins):
    codes, scale, mn, w = _weight(N, K, G, N + K, mins)
    back = ops.q4_dequantize(_pack(codes, scale, mn, dev))
    # one product and one sum in fp32, rounded once or twice: of c s and m, each at most 16 |s| here
    assert ((back.cpu().double() - w).abs() <= 2 * 2.0 ** -24 * 16 * scale.double().repeat_interleave(G, 1)).all()


@pytest.mark.parametrize("M", [1, 2, 3, 5, 8, 9, 16, 17, 31, 33, 64, 65, 130, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,K,G", [(1, 32, 32), (17, 96, 32), (33, 128, 128), (100, 320, 64), (530, 640, 128), (48, 2048, 64)])
def test_linear_q4(dev, M, dtype, N, K, G):
    wt = _weight(N, K, G, 3 * N + K, mins=M % 2 == 1)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(dtype)
    _check(x, _pack(*wt[:3], dev), wt, dev)


@pytest.mark.parametrize("M,N,K,G", [(1, 8192, 2048, 64), (5, 4096, 2048, 32), (16, 2048, 4096, 64), (61, 8192, 2048, 32),
                                     (300, 1024, 2048, 128), (1030, 2064, 512, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_q4_model_sizes(dev, M, N, K, G, dtype):
    wt = _weight(N, K, G, M, mins=True)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(1)).to(dtype)
    _check(x, _pack(*wt[:3], dev), wt, dev)


@pytest.mark.parametrize("M", [1, 3, 16, 40, 200])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_q4_accumulates_and_takes_strides(dev, M, dtype):
    N, K, G = 70, 256, 64
    wt = _weight(N, K, G, 5)
    w4 = _pack(*wt[:3], dev)
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(M, K + 64, generator=g).to(dtype).to(dev)
    x = wide[:, 32:32 + K]  # rows of another matrix
    y = _check(x, w4, wt, dev)
    res = torch.randn(M, N, generator=g).to(dev)
    both = ops.linear_q4(x, w4, out=res.clone(), accumulate=True)
    assert torch.equal(both, res + y)  # the product is rounded to fp32 before it is added
    lead = ops.linear_q4(x.reshape(1, M, K), w4)
    assert lead.shape == (1, M, N) and torch.equal(lead[0], y)


@pytest.mark.parametrize("M", [1, 4, 20, 150])
def test_linear_q4_rows_of_any_size(dev, M):
    """Rows from the smallest to the largest activations; rows of zeros; values far below their row's largest."""
    N, K, G = 40, 256, 64
    wt = _weight(N, K, G, 6)
    w4 = _pack(*wt[:3], dev)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(3))
    x[0] = 0
    _check(x, w4, wt, dev)
    assert (ops.linear_q4(x.to(dev), w4)[0] == 0).all()
    for e in (-120, -60, 60, 110):
        _check(x * 2.0 ** e, w4, wt, dev)
    x[:, ::7] *= 2.0 ** -30
    x[:, 5] = 1000.0
    _check(x, w4, wt, dev)
    _check(x.bfloat16(), w4, wt, dev)


@pytest.mark.parametrize("M", [1, 2, 7, 40, 700])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("G", [32, 64, 128])
def test_linear_q4_sums_of_large_rows(dev, M, dtype, G):
    """Rows whose groups sum to more than fp32 holds, although every output is far inside it."""
    N, K = 40, 256
    codes, scale, mn, _ = _weight(N, K, G, 16)
    scale, mn = (scale.float() / 64).half(), (mn.float() / 64).half()
    wt = (codes, scale, mn, R.q4_dequantize(codes, scale, mn, G))
    x = 1e38 * (1 + torch.rand(M, K, generator=torch.Generator().manual_seed(5))).to(dtype)
    assert torch.isinf(x.float()[:, :G].sum(1)).all() and (x.double() @ wt[3].t()).abs().max() < 1e38
    _check(x.to(dtype), _pack(*wt[:3], dev), wt, dev)


@pytest.mark.parametrize("M", [2, 9, 33, 140])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_q4_keeps_bad_rows_apart(dev, M, dtype):
    """A NaN or infinity stays in its row of x, and a NaN minimum or infinite scale in its row of the weight."""
    N, K, G = 50, 192, 64
    codes, scale, mn, w = _weight(N, K, G, 7)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(4)).to(dtype)
    good = ops.linear_q4(x.to(dev), _pack(codes, scale, mn, dev))
    for bad in (float("nan"), float("inf"), float("-inf")):
        xb = x.clone()
        xb[M // 2, 70] = bad
        y = ops.linear_q4(xb.to(dev), _pack(codes, scale, mn, dev))
        keep = torch.arange(M) != M // 2
        assert not torch.isfinite(y[M // 2]).any() and torch.equal(y[keep], good[keep])
    mb, sb = mn.clone(), scale.clone()
    mb[3, 1], sb[31, 2] = float("nan"), float("inf")
    y = ops.linear_q4(x.to(dev), _pack(codes, sb, mb, dev))
    keep = (torch.arange(N) != 3) & (torch.arange(N) != 31)
    assert not torch.isfinite(y[:, ~keep]).any() and torch.equal(y[:, keep], good[:, keep])


def test_linear_q4_of_more_rows_than_a_launch(dev):
    """2^19 rows and some: blocks of rows, accumulating into the output's strides; offsets of X past 2^32 bytes."""
    M, N, K, G = 2 ** 19 + 21, 24, 4608, 128
    wt = _weight(N, K, G, 10)
    w4 = _pack(*wt[:3], dev)
    x = torch.randn(2 ** 16, K, device=dev).bfloat16().repeat(9, 1)[:M]
    out = torch.full((M, N + 8), 2.0, device=dev)
    need = _lib.lib().aegist_linear_q4_workspace_bytes(_lib.BF16, M, N, K, G)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    # (the library's own call: columns 3 to 3 + N of a wider output)
    _lib.call("aegist_linear_q4", x.data_ptr(), _lib.BF16, K, w4.data.data_ptr(), out.data_ptr() + 12, N + 8, M, N, K, G, 1,
              ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert (out[:, :3] == 2).all() and (out[:, 3 + N:] == 2).all()
    for t in (0, 2 ** 18 - 5, 2 ** 19 - 8, 2 ** 19, M - 16):
        xs = x[t:t + 16].cpu()
        off = (out[t:t + 16, 3:3 + N].cpu().double() - 2 - xs.double() @ wt[3].t()).abs()
        # (the sum with 2 rounds once more)
        assert (off <= _bound(xs, wt[0], wt[1], wt[2], G) + 2.0 ** -24 * (off + 2 + (xs.double() @ wt[3].t()).abs())).all()


@pytest.mark.parametrize("M", [1, 3, 40, 140])
def test_linear_q4_of_a_weight_past_32_bits(dev, M):
    """Codes of more than 4 GiB, scales and minima behind them: the first and the last rows' outputs."""
    N, K, G = 2 ** 20 + 40, 8448, 64
    g = torch.Generator(dev).manual_seed(11)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8, device=dev)
    scale = (0.007 * (0.5 + torch.rand(N, K // G, generator=g, device=dev))).half()
    mn = (-7.5 * scale.float()).half()
    w4 = ops.q4_pack(codes, scale, mn)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(1)).bfloat16()
    y = ops.linear_q4(x.to(dev), w4)
    for n in (0, N // 2, N - 24):
        c, s, m = (t[n:n + 24].cpu() for t in (codes, scale, mn))
        ref = x.double() @ R.q4_dequantize(c, s, m, G).t()
        assert ((y[:, n:n + 24].cpu().double() - ref).abs() <= _bound(x, c, s, m, G)).all()


@pytest.mark.parametrize("M", [2, 5, 17, 150])
@pytest.mark.parametrize("K", [4224, 8192 + 64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_q4_long_rows(dev, M, K, dtype):
    """K past what a workgroup's waves hold at a time, where later parts add to the earlier ones' output."""
    N, G = 150, 32
    wt = _weight(N, K, G, K)
    w4 = _pack(*wt[:3], dev)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(dtype)
    y = _check(x, w4, wt, dev)
    res = torch.randn(M, N, generator=torch.Generator().manual_seed(2))
    both = ops.linear_q4(x.to(dev), w4, out=res.to(dev), accumulate=True)
    # a rounding of the sum per part of K (at most 5 of them), of what is there then
    size = res.abs().double() + x.abs().double() @ wt[3].abs().t()
    assert ((both - y).cpu().double() - res.double()).abs().le(6 * 2.0 ** -24 * 2 * size).all()


def test_linear_q4_empty(dev):
    wt = _weight(20, 64, 64, 8)
    assert ops.linear_q4(torch.empty(0, 64, device=dev), _pack(*wt[:3], dev)).shape == (0, 20)
    none = ops.q4_quantize(torch.empty(0, 64, device=dev))
    assert ops.linear_q4(torch.ones(3, 64, device=dev), none).shape == (3, 0)
    assert ops.q4_dequantize(none).shape == (0, 64)


@pytest.mark.parametrize("M", [1, 16, 70, 600])
def test_linear_q4_same_bits_again_and_in_graphs(dev, M):
    """Bit-identical from call to call, on a side stream, and in two captured graphs replayed between eager work."""
    N, K, G = 1000, 512, 64
    wt = _weight(N, K, G, 9)
    w4 = _pack(*wt[:3], dev)
    x = torch.randn(M, K, device=dev)
    y = ops.linear_q4(x, w4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(ops.linear_q4(x, w4), y)
    torch.cuda.current_stream().wait_stream(side)
    graphs, xs, outs = [], [x.clone(), x.clone()], []
    for xi in xs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.linear_q4(xi, w4))
        graphs.append(gr)
    for i in range(3):
        for xi, gr, o in zip(xs, graphs, outs):
            xi.copy_(torch.randn(M, K, device=dev))
            gr.replay()
            other = ops.linear_q4(torch.randn(3 * M, K, device=dev), w4)  # eager work between the replays
            torch.cuda.synchronize()
            assert torch.equal(o, ops.linear_q4(xi, w4)), i
            del other


def _quantize_ref(w, G):
    """The definition, in numpy doubles with one rounding to fp16."""
    w = w.double().numpy().reshape(w.shape[0], -1, G)
    mn = w.min(-1).astype(np.float16)
    sc = np.maximum((w.max(-1) - mn.astype(np.float64)) / 15, 0).astype(np.float16)
    m, s = mn.astype(np.float64)[..., None], sc.astype(np.float64)[..., None]
    code = np.where(s > 0, np.clip(np.rint((w - m) / np.where(s > 0, s, 1)), 0, 15), 0)
    return code.reshape(w.shape[0], -1).astype(np.uint8), sc, mn


@pytest.mark.parametrize("N,K,G", [(1, 32, 32), (16, 64, 64), (17, 96, 32), (33, 128, 128), (100, 320, 64), (70, 2048, 128),
                                   (512, 4096, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_is_exact(dev, N, K, G, dtype):
    """The packed block is, byte for byte, that of the codes, scales and minima of the definition."""
    g = torch.Generator().manual_seed(N + K)
    w = (0.02 * torch.randn(N, K, generator=g) * torch.exp(torch.randn(N, 1, generator=g))).to(dtype)
    w[0, :G] = 0.25                                   # a group of one value
    w[N // 2, K - G:] *= 2.0 ** -20                   # one whose scale is an fp16 subnormal
    if N > 2:
        w[2, :G] = (torch.arange(G) % 31).to(dtype) / 2   # halves of a step: ties
        w[1, :G] += 30000.0
    q4 = ops.q4_quantize(w.to(dev), G)
    code, sc, mn = _quantize_ref(w, G)
    want = ops.q4_pack(R.pack_codes(torch.from_numpy(code)).to(dev), torch.from_numpy(sc).to(dev), torch.from_numpy(mn).to(dev))
    assert torch.equal(q4.data, want.data)
    assert q4.shape == (N, K) and q4.group == G


def test_quantize_takes_strides_and_shows_bad_groups(dev):
    w = torch.randn(20, 300, device=dev)
    part = w[:, 4:260]
    assert torch.equal(ops.q4_quantize(part, 32).data, ops.q4_quantize(part.contiguous(), 32).data)
    w = torch.randn(20, 256, device=dev)
    good = ops.q4_dequantize(ops.q4_quantize(w))
    for bad in (float("nan"), float("inf"), -float("inf"), 7e4):
        wb = w.clone()
        wb[5, 70] = bad
        back = ops.q4_dequantize(ops.q4_quantize(wb))
        assert torch.isnan(back[5, 64:128]).all()
        back[5, 64:128] = good[5, 64:128]
        assert torch.equal(back, good)


def test_quantize_error_is_half_a_step(dev):
    """|w - w4| is at most half the group's scale and what the fp16 minimum and the scale's rounding leave at the ends."""
    w = torch.randn(64, 512, device=dev)
    back = ops.q4_dequantize(ops.q4_quantize(w, 64)).view(64, 8, 64)
    wg = w.view(64, 8, 64)
    step = (wg.amax(-1) - wg.amin(-1)) / 15
    # fp16 roundings: the minimum by 2^-11 of itself (half a unit), the 15 steps by 2^-11 of the range
    slack = 2.0 ** -11 * (wg.abs().amax(-1) + 15 * step) + 2.0 ** -11 * step
    assert ((back - wg).abs() <= (step / 2 + slack).unsqueeze(-1)).all()
