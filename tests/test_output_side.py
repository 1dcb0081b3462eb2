"""CPU checks of the 4-bit projections and the log probabilities: what is refused before any launch, the sizes of
packed weights, and the device and stream that a call is made on. No kernel is launched here."""
import pytest
import torch

from aegist_mixer import _lib, ops


class _OnGpu(torch.Tensor):
    is_cuda = property(lambda self: True)


def _t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_OnGpu)


@pytest.fixture
def launches(monkeypatch):
    seen = []
    monkeypatch.setattr(ops, "call", lambda name, *args: seen.append((name, args)))
    monkeypatch.setattr(ops, "_stream", lambda device=None: 0)
    return seen


def _w4(N=16, K=64, group=64):
    return ops.Q4Weight(_t(max(1, _lib.lib().aegist_q4_bytes(N, K, group)), dtype=torch.uint8), (N, K), group)


def test_packed_bytes():
    L = _lib.lib()
    # codes in tiles of 16 x 128, scale and minimum in blocks of 16 rows x 8 groups of 2 bytes
    assert L.aegist_q4_bytes(8192, 2048, 64) == 8192 * 2048 // 2 + 2 * 8192 * 32 * 2
    assert L.aegist_q4_bytes(1, 32, 32) == 1024 + 2 * 256
    assert L.aegist_q4_bytes(17, 1152, 128) == 2 * (9 * 1024 + 2 * 2 * 256)
    assert L.aegist_q4_bytes(2 ** 20, 2 ** 14, 128) == 2 ** 33 + 2 * 2 ** 20 * 2 ** 8
    for N, K, G in ((-1, 64, 64), (8, 0, 64), (8, 96, 64), (8, 64, 16), (8, 64, 0), (8, -64, 64)):
        assert L.aegist_q4_bytes(N, K, G) == 0


def test_q4_entry_points_refuse():
    L = _lib.lib()
    assert L.aegist_q4_quantize(None, 0, 64, None, 8, 64, 48, None) == -1 and "32, 64 or 128" in _lib.last_error()
    assert L.aegist_q4_quantize(None, 2, 64, None, 8, 64, 64, None) == -3
    assert L.aegist_q4_quantize(None, 0, 64, None, 8, 64, 64, None) == -1
    assert L.aegist_q4_quantize(64, 0, 63, 64, 8, 64, 64, None) == -1   # rows overlap
    assert L.aegist_q4_quantize(64, 0, 66, 64, 8, 64, 64, None) == -1   # rows not 16-byte aligned
    assert L.aegist_q4_quantize(64, 0, 64, 72, 8, 64, 64, None) == -1   # block not aligned
    assert L.aegist_q4_pack(64, None, None, 64, 8, 64, 64, None) == -1
    assert L.aegist_q4_pack(66, 64, None, 64, 8, 64, 64, None) == -1
    assert L.aegist_q4_dequantize(64, 72, 8, 64, 64, None) == -1
    assert L.aegist_linear_q4(64, 0, 64, 64, 64, 8, 2, 8, 96, 64, 0, None, 0, None) == -1
    assert L.aegist_linear_q4(64, 3, 64, 64, 64, 8, 2, 8, 64, 64, 0, None, 0, None) == -3
    assert L.aegist_linear_q4(64, 0, 60, 64, 64, 8, 2, 8, 64, 64, 0, None, 0, None) == -1   # ldx < K
    assert L.aegist_linear_q4(64, 0, 66, 64, 64, 8, 2, 8, 64, 64, 0, None, 0, None) == -1   # rows not aligned
    assert L.aegist_linear_q4(64, 0, 64, 64, 64, 7, 2, 8, 64, 64, 0, None, 0, None) == -1   # ldy < N
    assert L.aegist_linear_q4(None, 0, 64, 64, 64, 8, 2, 8, 64, 64, 0, None, 0, None) == -1
    assert L.aegist_linear_q4(64, 0, 64, 64, 64, 8, -1, 8, 64, 64, 0, None, 0, None) == -1
    for N, M in ((0, 3), (8, 0)):
        assert L.aegist_linear_q4(None, 0, 64, None, None, 8, M, N, 64, 64, 0, None, 0, None) == 0
    assert L.aegist_q4_quantize(None, 0, 64, None, 0, 64, 64, None) == 0


def test_logprob_entry_points_refuse():
    L = _lib.lib()
    def lp(dtype=0, ld=100, out=64, ids=64, T=4, V=100, top=3, tokens=64, logits=64):
        return L.aegist_token_logprobs(logits, dtype, ld, tokens, out, out, ids, ids, T, V, top, None, 0, None)
    assert lp(dtype=2) == -3
    assert lp(top=65) == -1 and lp(top=-1) == -1 and lp(V=2, ld=2) == -1   # more alternatives than tokens
    assert lp(ld=99) == -1 and lp(V=0) == -1 and lp(T=-1) == -1
    assert lp(out=None) == -1 and lp(ids=None) == -1 and lp(tokens=None) == -1 and lp(logits=None) == -1
    assert lp(T=0, logits=None, out=None) == 0

    def head(xd=0, wd=1, K=64, group=0, W=64, ws=None, n=0, T=4, V=100, top=3):
        return L.aegist_head_logprobs(64, xd, K, W, wd, None, 64, 64, 64, 64, 64, T, V, K, group, top, ws, n, None)
    assert head(xd=2) == -3 and head(wd=0) == -3 and head(wd=4) == -3
    assert head(wd=3, group=48) == -1 and head(W=None) == -1 and head(top=65) == -1
    assert head() == -2 and "workspace" in _lib.last_error()
    need = L.aegist_head_logprobs_workspace_bytes(0, 1, 4, 100, 64, 0, 3)
    assert need > 0 and head(ws=256, n=need - 1) == -2 and head(ws=264, n=need) == -2
    assert head(T=0) == 0


def test_workspace_never_falls_short_of_a_smaller_call():
    """A workspace sized for the largest call serves the smaller ones."""
    L = _lib.lib()
    for xd in (0, 1):
        for N, K, G in ((8192, 2048, 64), (100, 96, 32)):
            sizes = [L.aegist_linear_q4_workspace_bytes(xd, M, N, K, G) for M in list(range(1, 70)) + [100, 500, 4000, 9000]]
            assert sizes == sorted(sizes)
    for V in (1000, 131072):
        for top in (0, 20):
            sizes = [L.aegist_token_logprobs_workspace_bytes(T, V, top) for T in (1, 2, 8, 30, 64, 200, 256, 1000, 4000)]
            assert max(sizes) < 1 << 28
            assert L.aegist_head_logprobs_workspace_bytes(1, 1, 4000, V, 2048, 0, top) < 1 << 30


@pytest.mark.parametrize("host", [None, "x", "weight", "out"])
def test_linear_q4_refuses_host_operands(launches, host):
    def on(what, t):
        return t.as_subclass(torch.Tensor) if what == host else t
    w = _w4()
    w.data = on("weight", w.data)
    x, o = on("x", _t(2, 64)), on("out", _t(2, 16))
    if host is None:
        ops.linear_q4(x, w, out=o)
        assert [n for n, _ in launches] == ["aegist_linear_q4"]
        return
    with pytest.raises(ops.AegistError, match="not on a GPU"):
        ops.linear_q4(x, w, out=o)
    assert not launches


def test_linear_q4_refuses_what_does_not_fit(launches):
    for x, kw in ((_t(2, 96), {}), (_t(2, 64), dict(out=_t(2, 8))), (_t(2, 64), dict(accumulate=True)),
                  (_t(2, 64), dict(out=_t(2, 16, dtype=torch.bfloat16))), (_t(64, 2).t(), {}),
                  (_t(2, 64), dict(out=_t(16, 2).t())), (_t(2, 64, dtype=torch.float16), {})):
        with pytest.raises(ops.AegistError):
            ops.linear_q4(x, _w4(), **kw)
    assert not launches


def test_q4_makers_refuse_what_does_not_fit(launches):
    u8, f16 = torch.uint8, torch.float16
    for codes, scale, mins in ((_t(4, 32, dtype=u8), _t(4, 1), None), (_t(4, 32, dtype=u8), _t(3, 1, dtype=f16), None),
                               (_t(4, 32, dtype=u8), _t(4, 1, dtype=f16), _t(4, 2, dtype=f16)),
                               (_t(4, 32), _t(4, 1, dtype=f16), None), (_t(4, 32, dtype=u8), _t(4, 3, dtype=f16), None),
                               (_t(4, 32, dtype=u8), _t(4, 4, dtype=f16), None), (_t(4, 32, dtype=u8), _t(4, 0, dtype=f16), None),
                               (_t(32, 4, dtype=u8).t(), _t(4, 1, dtype=f16), None),
                               (torch.zeros(4, 32, dtype=u8), _t(4, 1, dtype=f16), None)):
        with pytest.raises(ops.AegistError):
            ops.q4_pack(codes, scale, mins)
    for w, group in ((_t(4, 64), 48), (_t(4, 96), 64), (_t(64, 4).t(), 64), (_t(4, 64, dtype=torch.float16), 64), (_t(64), 64),
                     (torch.zeros(4, 64), 64), (_t(4, 0), 64)):
        with pytest.raises(ops.AegistError):
            ops.q4_quantize(w, group)
    assert not launches


def test_logprobs_refuse_what_does_not_fit(launches):
    i32 = torch.int32
    for x, t in ((_t(3, 10), _t(3, dtype=torch.int64)), (_t(3, 10), _t(4, dtype=i32)), (_t(10, 3).t(), _t(3, dtype=i32)),
                 (_t(3, 10, dtype=torch.float16), _t(3, dtype=i32)), (_t(3, 0), _t(3, dtype=i32)),
                 (torch.zeros(3, 10), _t(3, dtype=i32)), (_t(3, 10), torch.zeros(3, dtype=i32)),
                 (_t(3, 10), _t(6, dtype=i32)[::2])):
        with pytest.raises(ops.AegistError):
            ops.token_logprobs(x, t)
    bf = torch.bfloat16
    for x, w, t, s in ((_t(3, 64), _t(9, 32, dtype=bf), _t(3, dtype=i32), None), (_t(3, 64), _t(9, 64), _t(3, dtype=i32), None),
                       (_t(3, 64), _t(9, 64, dtype=torch.int8), _t(3, dtype=i32), _t(8, dtype=bf)),
                       (_t(3, 64), _w4(), _t(3, dtype=i32), _t(16, dtype=bf)), (_t(3, 64), _w4(), _t(2, dtype=i32), None),
                       (_t(3, 64), torch.zeros(9, 64, dtype=bf), _t(3, dtype=i32), None)):
        with pytest.raises(ops.AegistError):
            ops.head_logprobs(x, w, t, scale=s)
    assert not launches


def test_a_row_stride_below_the_row_reaches_the_library(monkeypatch):
    """Broadcast rows (stride 0) are not taken for packed ones: the library refuses them."""
    monkeypatch.setattr(ops, "_stream", lambda device=None: 0)
    x = _t(1, 64).expand(3, 64)
    with pytest.raises(ops.AegistError, match="ldx >= K"):
        ops.linear_q4(x, _w4(), out=_t(3, 16))
    with pytest.raises(ops.AegistError, match="ld < V"):
        ops.token_logprobs(_t(1, 10).expand(3, 10), _t(3, dtype=torch.int32))


def test_call_is_made_on_the_tensors_device(monkeypatch, launches):
    entered = []

    class On:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            entered.append(self.dev.index)

        def __exit__(self, *a):
            pass
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(ops, "_stream", lambda device=None: 100 + device.index)
    ops._call_on(torch.device("cuda", 0), "f", 1)
    ops._call_on(torch.device("cuda", 1), "f", 2)
    assert entered == [1] and launches == [("f", (1, 100)), ("f", (2, 101))]


def test_tensors_of_two_devices_are_refused():
    with pytest.raises(ops.AegistError, match="one device"):
        ops._one_device(torch.empty(1), None, torch.empty(1, device="meta"))


@pytest.mark.parametrize("V", [1, 1000, 4097, 50257, 131072, 2 ** 20 + 1, 2 ** 27, 2 ** 30])
def test_logprob_workspace_serves_every_smaller_batch(V):
    """Few rows are cut into more splits than many, which need no workspace at all: what is asked for T rows covers
    every smaller batch, so also the last block of a head's rows."""
    L = _lib.lib()
    for top in (0, 1, min(V, 64)):
        sizes = [L.aegist_token_logprobs_workspace_bytes(T, V, top) for T in list(range(1, 800, 7)) + [1536, 1537, 2 ** 20]]
        assert sizes == sorted(sizes)
        if V >= 50257:
            assert sizes[0] > 0
        # the logits of a block of 256 MiB (at least one row) and behind them what any number of its rows needs
        rows = max(1, 2 ** 28 // (4 * V))
        logits = -(-rows * V * 4 // 256) * 256
        blocks = L.aegist_head_logprobs_workspace_bytes(1, 1, 3 * rows + 1, V, 64, 0, top) - logits
        assert blocks >= max(L.aegist_token_logprobs_workspace_bytes(m, V, top) for m in (1, (rows + 1) // 2, rows))


def test_logprobs_refuse_a_vocabulary_past_the_index(launches):
    L = _lib.lib()
    V = 2 ** 30 + 1
    assert L.aegist_token_logprobs(64, 0, V, 64, 64, 64, 64, 64, 1, V, 1, None, 0, None) == -1 and "2^30" in _lib.last_error()
    assert L.aegist_head_logprobs(64, 0, 64, 64, 1, None, 64, 64, 64, 64, 64, 1, V, 64, 0, 1, None, 0, None) == -1
    assert L.aegist_token_logprobs_workspace_bytes(1, V, 1) == 0


def test_q4_sizes_past_the_index_are_refused():
    L = _lib.lib()
    for N, K in ((2 ** 28 + 1, 64), (8, 2 ** 28 + 64), (2 ** 31 - 1, 2 ** 31 - 64)):
        assert L.aegist_q4_bytes(N, K, 64) == 0 and "2^28" in _lib.last_error()
        assert L.aegist_linear_q4_workspace_bytes(1, 8, N, K, 64) == 0
        assert L.aegist_linear_q4(64, 0, K, 64, 64, N, 1, N, K, 64, 0, None, 0, None) == -1
    # rows go in blocks: the workspace of a projection is no larger for 2^31 of them than for 2^19
    assert L.aegist_linear_q4_workspace_bytes(1, 2 ** 31 - 1, 64, 64, 64) == L.aegist_linear_q4_workspace_bytes(1, 2 ** 19, 64, 64, 64)


def test_linear_q4_refuses_an_output_that_overlaps():
    L = _lib.lib()
    def call(x, w, y, M=2, N=64, K=64):
        return L.aegist_linear_q4(x, 0, K, w, y, N, M, N, K, 64, 0, None, 0, None)
    base, w = 1 << 20, L.aegist_q4_bytes(64, 64, 64)
    for x, q, y in ((base, base << 1, base), (base, base << 1, base + 256 + 252), (base + 252 + 4, base << 1, base),
                    (base, base << 1, (base << 1) + w - 4), (base, base << 1, (base << 1) - 508)):
        assert call(x, q, y) == -1 and "overlaps" in _lib.last_error()


def test_head_refuses_a_workspace_without_the_operands_of_a_4_bit_product():
    L = _lib.lib()
    T, V, K = 4000, 8192, 2048  # (tiles, with rows as operands in the workspace)
    need = L.aegist_head_logprobs_workspace_bytes(1, 3, T, V, K, 64, 0)
    assert need > L.aegist_head_logprobs_workspace_bytes(1, 1, T, V, K, 64, 0)   # (bf16: logits alone)
    def call(n):
        return L.aegist_head_logprobs(1 << 40, 1, K, 1 << 41, 3, None, 64, 64, 64, None, None, T, V, K, 64, 0, 1 << 42, n, None)
    assert call(need - 1) == -2 and "linear_q4" in _lib.last_error()
    assert call(100) == -2 and "head_logprobs" in _lib.last_error()


def test_sizes_past_32_bits_are_refused(launches):
    """ctypes would pass them on modulo 2^32: a vocabulary of 2^32 + 5 as one of 5."""
    def m(*shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device="meta").as_subclass(_OnGpu)
    big, u8, i32, f16, bf = 2 ** 32, torch.uint8, torch.int32, torch.float16, torch.bfloat16
    w4 = ops.Q4Weight(m(2048, dtype=u8), (16, 64), 64)
    for call in (lambda: ops.q4_pack(m(big + 16, 32, dtype=u8), m(big + 16, 1, dtype=f16)),
                 lambda: ops.q4_quantize(m(big + 16, 64)), lambda: ops.q4_quantize(m(16, big + 64)),
                 lambda: ops.q4_quantize(m(16, 64), big + 64), lambda: ops.Q4Weight(m(2048, dtype=u8), (big + 16, 64), 64), lambda: ops.linear_q4(m(big + 2, 64), w4),
                 lambda: ops.linear_q4(m(2, big // 4, 1, 64), w4),
                 lambda: ops.token_logprobs(m(1, big + 5), m(1, dtype=i32)),
                 lambda: ops.token_logprobs(m(big + 3, 5), m(big + 3, dtype=i32)),
                 lambda: ops.token_logprobs(m(3, 5), m(3, dtype=i32), big + 2), lambda: ops.token_logprobs(m(3, 5), m(3, dtype=i32), -1),
                 lambda: ops.head_logprobs(m(3, 64), m(big + 7, 64, dtype=bf), m(3, dtype=i32)),
                 lambda: ops.head_logprobs(m(big + 3, 64), w4, m(big + 3, dtype=i32))):
        with pytest.raises(ops.AegistError):
            call()
    assert not launches


def test_head_workspace_of_fp32_rows():
    """fp32 rows are split beside the logits, in blocks of 256 MiB however short the vocabulary is."""
    L = _lib.lib()
    def need(xd, wd, T, V=1000, K=8192, group=0):
        return L.aegist_head_logprobs_workspace_bytes(xd, wd, T, V, K, group, 1)
    for wd in (1, 2):
        assert need(0, wd, 10 ** 6) < 1 << 30 and need(0, wd, 10 ** 6, V=5) < 1 << 30
        assert need(0, wd, 100) >= need(1, wd, 100) + 6 * 100 * 8192
        assert need(0, wd, 1) == need(1, wd, 1)
        assert need(0, wd, 7, V=2 ** 27, K=2 ** 28) < 1 << 30   # a row at a time
    assert need(0, 1, 2) == need(1, 1, 2) and need(0, 2, 2) > need(1, 2, 2)
    sizes = [need(0, 1, T) for T in (1, 2, 3, 50, 1000, 5461, 5462, 20000, 10 ** 6)]
    assert sizes == sorted(sizes)
    def call(n, T=100):
        return L.aegist_head_logprobs(256, 0, 8192, 256, 1, None, 64, 64, 64, 64, 64, T, 1000, 8192, 0, 1, 1 << 40, n, None)
    assert call(need(0, 1, 100) - 1) == -2 and "head_logprobs" in _lib.last_error()


def test_packed_weight_of_other_bytes_is_refused():
    """A block that is shorter than its shape's would be read past its end."""
    u8, need = torch.uint8, _lib.lib().aegist_q4_bytes(40, 192, 32)
    w = ops.Q4Weight(_t(need, dtype=u8), [40, 192], 32)
    assert w.shape == (40, 192) and w.group == 32
    for data, shape, group in ((_t(need - 1, dtype=u8), (40, 192), 32), (_t(need, dtype=u8), (49, 192), 32), (_t(need, dtype=u8), (40, 320), 32),
                               (_t(need), (40, 192), 32), (_t(2 * need, dtype=u8)[::2], (40, 192), 32), (_t(need, dtype=u8), (40, 192), 128),
                               (_t(need, dtype=u8), (40, 192), 48), (_t(need, dtype=u8), (-40, 192), 32)):
        with pytest.raises(ops.AegistError):
            ops.Q4Weight(data, shape, group)
