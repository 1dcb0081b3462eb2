"""The 4-bit product on each of its tiles: sizes taken from the choice itself, so that every tile height, type and group
runs. (A weight narrow enough for a quick test mostly goes to the kernel that streams it.)"""
import ctypes

import pytest
import torch

from aegist_mixer import _lib, ops
from oracle import mixer_ref as R

DT = {_lib.F32: torch.float32, _lib.BF16: torch.bfloat16}
# (type of X, 16-row tiles of a workgroup, group): (M, N, K) of few rows, of more than 8 tiles of rows, of more than 32 groups.
# No M, N or K fills the tiles (but for K in groups of 128)
CASES = {
    (_lib.F32, 2, 32): [(83, 16001, 544), (515, 2053, 544), (1031, 1000, 1184)],
    (_lib.F32, 2, 64): [(17, 60001, 576), (515, 1999, 576), (263, 4100, 2240)],
    (_lib.F32, 2, 128): [(83, 16001, 640), (263, 2053, 1152), (300, 4100, 4352)],
    (_lib.F32, 4, 32): [(61, 60001, 96), (1500, 1999, 96), (1031, 1999, 1184)],
    (_lib.F32, 4, 64): [(150, 32771, 64), (700, 4100, 64), (1000, 2053, 2240)],
    (_lib.F32, 4, 128): [(61, 60001, 128), (1500, 2053, 128), (263, 8201, 4352)],
    (_lib.F32, 8, 32): [(107, 60001, 1184), (1500, 4100, 1184), (390, 16001, 1184)],
    (_lib.F32, 8, 64): [(125, 60001, 832), (4001, 1999, 832), (390, 16001, 2240)],
    (_lib.F32, 8, 128): [(107, 60001, 896), (1500, 4100, 1152), (390, 16001, 4352)],
    (_lib.BF16, 2, 32): [(83, 32771, 96), (1500, 1999, 96), (515, 2053, 1184)],
    (_lib.BF16, 2, 64): [(17, 131075, 64), (390, 8201, 64), (263, 2053, 2240)],
    (_lib.BF16, 2, 128): [(17, 60001, 384), (1500, 2053, 128), (300, 4100, 4352)],
    (_lib.BF16, 4, 32): [(45, 60001, 544), (1031, 2053, 544), (1031, 1999, 1184)],
    (_lib.BF16, 4, 64): [(150, 16001, 832), (515, 4100, 576), (1000, 2053, 2240)],
    (_lib.BF16, 4, 128): [(61, 60001, 640), (1000, 2053, 640), (515, 4100, 4352)],
    (_lib.BF16, 8, 32): [(125, 60001, 160), (4001, 1999, 224), (390, 16001, 1184)],
    (_lib.BF16, 8, 64): [(107, 60001, 320), (1500, 4100, 320), (390, 16001, 2240)],
    (_lib.BF16, 8, 128): [(125, 60001, 384), (4001, 1999, 640), (1500, 4100, 4352)],
}
ALL = [(xd, tile, G, *size) for (xd, tile, G), sizes in CASES.items() for size in sizes]
FIRST = [(xd, tile, G, *sizes[0]) for (xd, tile, G), sizes in CASES.items()]


def _form(xd, M, N, K, G):
    fn = _lib.lib()._ZN6aegist14linear_q4_formEiiiii
    fn.argtypes = [ctypes.c_int] * 5
    return fn(xd, M, N, K, G)


def test_sizes_reach_the_tiles():
    assert len({k for k in CASES}) == 18
    for xd, tile, G, M, N, K in ALL:
        assert _form(xd, M, N, K, G) == tile, (xd, tile, G, M, N, K)
        assert M % (16 * tile) and N % 256 and K % G == 0
        assert _lib.lib().aegist_linear_q4_workspace_bytes(xd, M, N, K, G) > 0


def _weight(N, K, G, seed, dev):
    """Codes, scales, minima and their fp64 matrix on the device."""
    g = torch.Generator(dev).manual_seed(seed)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8, device=dev)
    scale = (0.007 * (0.5 + torch.rand(N, K // G, generator=g, device=dev))).half()
    mn = (-(7 + torch.rand(N, K // G, generator=g, device=dev)) * scale.float()).half()
    return codes, scale, mn, R.q4_dequantize(codes, scale, mn, G).double()


def _bound(x, codes, scale, mn, G):
    """An activation counts with 22 bits, half a step off at most, and down to 2^-34 of the largest of its row; products and
    sums of a group's x are exact or rounded to 24 bits, added in chains of at most 128 (twice, for its two parts, of
    which the second is 2^-11 of the first) and then K / G; scale and minimum are applied with a rounding each."""
    K = 2 * codes.shape[1]
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(1).double()
    wa = (c * scale.double().abs().repeat_interleave(G, 1) + mn.double().abs().repeat_interleave(G, 1)).t()
    xa = x.double().abs()
    return (2.0 ** -22 + (128 + K // G + 8) * 2.0 ** -24) * (xa @ wa) + 2.0 ** -34 * xa.amax(1, keepdim=True) * wa.sum(0)


def _close(y, x, wt, G):
    off = (y.double() - x.double() @ wt[3].t()).abs()
    return bool((off <= _bound(x, *wt[:3], G)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("xd,tile,G,M,N,K", ALL)
def test_tiles(dev, xd, tile, G, M, N, K):
    """Rows of a wider matrix against 64 bits; the same product added into columns of a wider output; the same bits again."""
    wt = _weight(N, K, G, M + N, dev)
    w4 = ops.q4_pack(*wt[:3])
    g = torch.Generator(dev).manual_seed(K)
    x = torch.randn(M, K + 64, generator=g, device=dev).to(DT[xd])[:, 32:32 + K]
    assert _form(xd, M, N, K, G) == tile
    y = ops.linear_q4(x, w4)
    assert _close(y, x, wt, G)
    assert torch.equal(ops.linear_q4(x.contiguous(), w4), y)
    out = torch.randn(M + 1, N + 9, generator=g, device=dev)
    want = out.clone()
    want[:M, 4:4 + N] += y  # the product is rounded to fp32 before it is added
    need = _lib.lib().aegist_linear_q4_workspace_bytes(xd, M, N, K, G)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _lib.call("aegist_linear_q4", x.data_ptr(), xd, K + 64, w4.data.data_ptr(), out.data_ptr() + 16, N + 9, M, N, K, G, 1,
              ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("xd,tile,G,M,N,K", FIRST)
def test_tiles_keep_bad_rows_apart(dev, xd, tile, G, M, N, K):
    """A NaN or infinity stays in its row of x, a NaN minimum or infinite scale in its row of the weight; rows of zeros."""
    codes, scale, mn, w = _weight(N, K, G, 7, dev)
    w4 = ops.q4_pack(codes, scale, mn)
    x = torch.randn(M, K, generator=torch.Generator(dev).manual_seed(4), device=dev).to(DT[xd])
    x[0] = 0
    good = ops.linear_q4(x, w4)
    assert (good[0] == 0).all()
    rows = (M // 2, M - 1)
    keep = torch.ones(M, dtype=torch.bool, device=dev)
    keep[list(rows)] = False
    for bad in (float("nan"), float("inf"), float("-inf")):
        xb = x.clone()
        xb[rows[0], K - 1], xb[rows[1], 0] = bad, bad
        y = ops.linear_q4(xb, w4)
        assert not torch.isfinite(y[~keep]).any() and torch.equal(y[keep], good[keep])
    mb, sb = mn.clone(), scale.clone()
    mb[3, 0], mb[N - 1, K // G - 1], sb[31, K // G - 1] = float("nan"), float("nan"), float("inf")
    keep = torch.ones(N, dtype=torch.bool, device=dev)
    keep[[3, 31, N - 1]] = False
    y = ops.linear_q4(x, ops.q4_pack(codes, sb, mb))
    assert not torch.isfinite(y[1:, ~keep]).any() and torch.equal(y[:, keep], good[:, keep])


@pytest.mark.gpu
@pytest.mark.parametrize("xd,tile,G,M,N,K", FIRST)
def test_tiles_take_rows_of_any_size(dev, xd, tile, G, M, N, K):
    """Rows near the ends of fp32's range give the same bits, shifted; values far below their row's largest; groups that sum
    to more than fp32 holds."""
    wt = _weight(N, K, G, 6, dev)
    w4 = ops.q4_pack(*wt[:3])
    x = torch.randn(M, K, generator=torch.Generator(dev).manual_seed(3), device=dev).to(DT[xd])
    y = ops.linear_q4(x, w4)
    for e in (100, -100):  # (powers of two: x 2^e is exact, and the result is rounded where it was)
        assert torch.equal(ops.linear_q4(x * 2.0 ** e, w4), y * 2.0 ** e)
    x[:, ::7] *= 2.0 ** -30
    x[:, 5] = 1000.0
    assert _close(ops.linear_q4(x, w4), x, wt, G)
    codes, scale, mn = wt[0], (wt[1].float() / 256).half(), (wt[2].float() / 256).half()
    wt = (codes, scale, mn, R.q4_dequantize(codes, scale, mn, G).double())
    x = (1e38 * (1 + torch.rand(M, K, generator=torch.Generator(dev).manual_seed(5), device=dev))).to(DT[xd])
    assert torch.isinf(x[:, :G].sum(1, dtype=torch.float32)).all() and (x.double() @ wt[3].t()).abs().max() < 1e38
    assert _close(ops.linear_q4(x, ops.q4_pack(codes, scale, mn)), x, wt, G)


@pytest.mark.gpu
@pytest.mark.parametrize("xd,tile,G,M,N,K", FIRST[::2])
def test_tiles_in_graphs_and_on_two_streams(dev, xd, tile, G, M, N, K):
    """Two captured graphs replayed between eager work, and two streams at once, each with a workspace of its own."""
    wt = _weight(N, K, G, 9, dev)
    w4 = ops.q4_pack(*wt[:3])
    xs = [torch.randn(M, K, device=dev).to(DT[xd]) for _ in range(2)]
    want = [ops.linear_q4(x, w4) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.linear_q4(xs[i], w4))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])
    graphs, outs = [], []
    for x in xs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.linear_q4(x, w4))
        graphs.append(gr)
    for _ in range(3):
        for x, gr, o in zip(xs, graphs, outs):
            x.copy_(torch.randn(M, K, device=dev))
            gr.replay()
            ops.linear_q4(torch.randn(M + 40, K, device=dev).to(DT[xd]), w4)
            torch.cuda.synchronize()
            assert torch.equal(o, ops.linear_q4(x, w4))


@pytest.mark.gpu
@pytest.mark.parametrize("xd,M,N,K,G,tiles", [(_lib.BF16, 2 ** 19 + 3001, 1000, 128, 64, (2, 2)), (_lib.F32, 2 ** 19 + 3001, 1000, 128, 64, (4, 4)),
                                              (_lib.BF16, 2 ** 19 + 21, 200, 4608, 128, (8, 0))])
def test_tiles_of_more_rows_than_a_launch(dev, xd, M, N, K, G, tiles):
    """2^19 rows and some in one workspace, block after block; the last case's operands pass 2^32 bytes."""
    assert (_form(xd, M, N, K, G), _form(xd, M - 2 ** 19, N, K, G)) == tiles
    wt = _weight(N, K, G, 10, dev)
    w4 = ops.q4_pack(*wt[:3])
    P = 2 ** 16 + 8
    x = torch.randn(P, K, device=dev).to(DT[xd]).repeat(9, 1)[:M]
    y = ops.linear_q4(x, w4)
    # a row's result does not depend on its place in the tiles
    for t in range(P, 2 ** 19, P):
        n = min(P, 2 ** 19 - t)
        assert torch.equal(y[t:t + n], y[:n])
    for t in (0, 2 ** 18 - 50, 2 ** 19 - 60, M - 100):
        assert _close(y[t:t + 100], x[t:t + 100], wt, G)
