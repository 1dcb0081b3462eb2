"""The output side of a served model, as measurable cases: projections and the output head with 4-bit
weights, and the log probabilities that a model answers with.

Four kinds: a weight matrix quantised to 4 bits and read back (a converter that checks what it wrote), the
projection with 4-bit weights, the log probabilities of given tokens with entropy and top alternatives from
logits, and the same straight from the hidden rows, where the logits are never whole. Sizes are those of the
hybrid that this repository is configured for (d_model 2048, DeltaNet qkv 8192, out projections 2048 x 4096,
a generic head of 32768 tokens), with tokens from one to a few thousand, odd row counts and vocabularies.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DM = 2048
VOCAB = 32768  # a generic output head
_DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _ops():
    for p in (str(Path.cwd()), str(Path.cwd() / "aegist-optimized-ai-library-_amd")):
        if p not in sys.path:
            sys.path.insert(0, p)
    from aegist_mixer import ops
    return ops


def listed():
    return [
        # An out projection quantised on load: the checkpoint's bf16 to 4 bits, and back to see what was lost.
        dict(name="quantize_out", kind="quantize", N=2048, K=4096, G=64, w="bf16"),
        # The output head, from fp32 masters, in long groups and with a vocabulary that fills no tile.
        dict(name="quantize_head", kind="quantize", N=32771, K=2048, G=128, w="f32"),
        # The engine's single-token projection: the smallest product, where latency counts.
        dict(name="linear_m1", kind="linear", M=1, N=8192, K=2048, G=64, x="f32", mins=True),
        # Three users' tokens through the output head, symmetric weights: the weight stream alone.
        dict(name="linear_head_m3", kind="linear", M=3, N=131072, K=2048, G=128, x="bf16", mins=False),
        # The out projection of a batch-16 decode step.
        dict(name="linear_m16", kind="linear", M=16, N=2048, K=4096, G=64, x="bf16", mins=True),
        # A mid-size batch of an odd count of rows, fp32 activations, short groups.
        dict(name="linear_m61", kind="linear", M=61, N=8192, K=2048, G=32, x="f32", mins=True),
        # A prefill projection of a ragged batch of prompt tokens.
        dict(name="linear_m4000", kind="linear", M=4000, N=8192, K=2048, G=64, x="bf16", mins=True),
        # One sampled token with its 20 best alternatives, as a serving interface returns them.
        dict(name="logprobs_t1", kind="logprobs", T=1, V=131072, top=20, dtype="f32", masked=0.0),
        # A decode batch under a grammar that rules most of an odd vocabulary out (and, in one row, all of it).
        dict(name="logprobs_t61_masked", kind="logprobs", T=61, V=100003, top=5, dtype="bf16", masked=0.9),
        # The logits of a long prompt scored token by token.
        dict(name="logprobs_t2000", kind="logprobs", T=2000, V=131072, top=8, dtype="f32", masked=0.0),
        # A batch-16 decode step's answer: 4-bit head, log probability and 5 alternatives.
        dict(name="head_t16", kind="head", T=16, V=131072, K=2048, G=64, x="bf16", w="q4", top=5),
        # A 1000-token prompt scored against a bf16 head, with the token that greedy decoding would take.
        dict(name="head_t1000", kind="head", T=1000, V=VOCAB, K=2048, G=0, x="bf16", w="bf16", top=1),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "linear", "logprobs", "logprobs", "head"])
    G = rng.choice([32, 64, 128])
    if kind == "quantize":
        return dict(kind=kind, N=_log_int(rng, 16, 32768), K=128 * rng.randint(1, 16), G=G, w=rng.choice(["bf16", "f32"]))
    if kind == "linear":
        if rng.random() < 0.6:
            N, K = rng.choice([(8192, 2048), (4096, 2048), (1024, 2048), (512, 2048), (2048, 4096), (2048, 512), (VOCAB, 2048)])
        else:
            N, K = _log_int(rng, 1, 16384), G * rng.randint(1, 4096 // G)
        M = _log_int(rng, 1, max(1, min(4000, (4000 * 8192 * 1024) // (N * K))))
        return dict(kind=kind, M=M, N=N, K=K, G=G, x=rng.choice(["f32", "bf16"]), mins=rng.choice([True, True, False]))
    if kind == "logprobs":
        V = _log_int(rng, 100, 200000)
        return dict(kind=kind, T=_log_int(rng, 1, max(1, min(4000, 200_000_000 // V))), V=V, top=min(V, rng.choice([0, 0, 1, 5, 20, rng.randint(1, 64)])),
                    dtype=rng.choice(["f32", "bf16"]), masked=rng.choice([0.0, 0.0, 0.5, 0.99]))
    # the ids come from computed logits: short lists, so that no two of them stand closer than fp32 sums do
    w, T = rng.choice(["q4", "bf16"]), _log_int(rng, 1, 1000)
    V = _log_int(rng, 1000, 131072 if T <= 64 else VOCAB)
    return dict(kind=kind, T=T, V=V, K=DM, G=G if w == "q4" else 0, x="bf16" if w == "bf16" else rng.choice(["bf16", "f32"]), w=w,
                top=rng.choice([0, 1, 5]) if T <= 16 else rng.choice([0, 1]))


# --- inputs -----------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed & 0x7fffffff)


def _codes(g, N, K, G, mins):
    """A 4-bit weight in the engine's layout: two codes to a byte, the even element low; fp16 scale and minimum
    of G values. Weights of std 0.02, so 15 steps span about 0.1; None for the minima: (code - 8) * scale."""
    codes = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    scale = (0.1 / 15 * (0.5 + torch.rand(N, K // G, generator=g, device="cuda"))).half()
    mn = (-(7 + torch.rand(N, K // G, generator=g, device="cuda")) * scale.float()).half() if mins else None
    return codes, scale, mn


def _tokens(g, T, V):
    return torch.randint(0, V, (T,), generator=g, device="cuda", dtype=torch.int32)


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    rn = lambda *s, std=1.0: torch.randn(*s, generator=g, device="cuda").mul_(std)  # noqa: E731
    s = dict(case=case)
    if kind == "quantize":
        # rows of different size, as trained weights have
        s["w"] = (rn(case["N"], case["K"], std=0.02) * torch.exp(rn(case["N"], 1, std=0.5))).to(_DT[case["w"]])
    elif kind == "linear":
        s["x"] = rn(case["M"], case["K"]).to(_DT[case["x"]])
        s["w"] = _codes(g, case["N"], case["K"], case["G"], case["mins"])
        if own:
            s["w4"] = _ops().q4_pack(*s["w"])  # weights are laid out once, on load
    elif kind == "logprobs":
        T, V = case["T"], case["V"]
        x = rn(T, V, std=2.5)
        s["tokens"] = _tokens(g, T, V)
        if case["masked"]:
            keep = torch.rand(T, V, generator=g, device="cuda") >= case["masked"]
            keep[torch.arange(T, device="cuda"), s["tokens"].long()] = True
            if T > 2:
                keep[T // 2] = False
            x.masked_fill_(~keep, -math.inf)
        s["logits"] = x.to(_DT[case["dtype"]])
    else:
        T, V, K = case["T"], case["V"], case["K"]
        s["x"] = rn(T, K).to(_DT[case["x"]])
        s["tokens"] = _tokens(g, T, V)
        if case["w"] == "q4":
            s["w"] = _codes(g, V, K, case["G"], True)
            if own:
                s["w4"] = _ops().q4_pack(*s["w"])
        else:
            s["w"] = rn(V, K, std=0.03).to(torch.bfloat16)
    return s


# --- the plain forms --------------------------------------------------------------------------------

def _to_half(x):
    """Doubles rounded once to fp16: to fp32 by rounding to odd, whose last bit then holds what was cut off."""
    f = x.float()
    bits = f.view(torch.int32)
    bits = torch.where(f.double().abs() > x.abs(), bits - 1, bits)
    cut = bits.view(torch.float32)
    return torch.where(cut.double() != x, bits | 1, bits).view(torch.float32).half()


def _quantize(w, G):
    w = w.double().view(w.shape[0], -1, G)
    lo, hi = w.amin(-1), w.amax(-1)
    mn = _to_half(lo)
    scale = _to_half(((hi - mn.double()) / 15).clamp(min=0))
    d = torch.where(scale > 0, scale.double(), math.inf).unsqueeze(-1)
    return torch.round((w - mn.double().unsqueeze(-1)) / d).clamp(0, 15), scale, mn


def _dequantize(codes, scale, mn):
    """fp32 weights from packed codes."""
    c = torch.stack([codes & 15, codes >> 4], -1).view(codes.shape[0], scale.shape[1], -1).float()
    s = scale.float().unsqueeze(-1)
    return (c * s + (mn.float().unsqueeze(-1) if mn is not None else -8 * s)).flatten(1)


def _logprobs(x, tokens, top):
    x = x.float()
    V = x.shape[1]
    m = x.amax(1, keepdim=True)
    d = x - torch.where(torch.isinf(m), 0.0, m)
    e = torch.exp(d)
    z = e.sum(1)
    lz = torch.log(z)
    lp = d.gather(1, tokens.long().unsqueeze(1)).squeeze(1) - lz
    ent = lz - torch.where(e > 0, e * d, 0.0).sum(1) / z
    empty = z == 0  # nothing left: no token has a probability
    lp, ent = torch.where(empty, -math.inf, lp), torch.where(empty, 0.0, ent)
    if not top:
        return lp, ent
    # one order for all: the value first, then the lower token
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7fffffff), bits) * 2 ** 32 + (V - 1 - torch.arange(V, device=x.device))
    ids = V - 1 - (torch.topk(key, top, dim=1).values & 0xffffffff)
    return lp, ent, ids.int(), torch.where(empty.unsqueeze(1), -math.inf, d.gather(1, ids) - lz.unsqueeze(1))


def run(state):
    c = state["case"]
    kind = c["kind"]
    if own:
        ops = _ops()
        if kind == "quantize":
            return ops.q4_dequantize(ops.q4_quantize(state["w"], c["G"]))
        if kind == "linear":
            return ops.linear_q4(state["x"], state["w4"])
        if kind == "logprobs":
            return _some(ops.token_logprobs(state["logits"], state["tokens"], c["top"]))
        return _some(ops.head_logprobs(state["x"], state["w4"] if c["w"] == "q4" else state["w"], state["tokens"], c["top"]))
    if kind == "quantize":
        code, scale, mn = _quantize(state["w"], c["G"])
        return (code.float() * scale.float().unsqueeze(-1) + mn.float().unsqueeze(-1)).flatten(1)
    if kind == "linear":
        return state["x"].float() @ _dequantize(*state["w"]).t()
    if kind == "logprobs":
        return _logprobs(state["logits"], state["tokens"], c["top"])
    w = _dequantize(*state["w"]) if c["w"] == "q4" else state["w"].float()
    return _logprobs(state["x"].float() @ w.t(), state["tokens"], c["top"])


def _some(out):
    """Without the alternatives where none were asked for."""
    return tuple(out) if out[2] is not None else tuple(out)[:2]


# --- the definitions in 64 bits ---------------------------------------------------------------------

def _exact_weight(codes, scale, mn):
    N, half = codes.shape
    w = torch.empty(N, 2 * half, dtype=torch.float64, device=codes.device)
    w[:, 0::2] = codes % 16
    w[:, 1::2] = torch.div(codes, 16, rounding_mode="floor")
    G = 2 * half // scale.shape[1]
    s = scale.double().repeat_interleave(G, 1)
    return w.mul_(s).add_(mn.double().repeat_interleave(G, 1)) if mn is not None else w.sub_(8).mul_(s)


def _exact_logprobs(x, tokens, top):
    lse = torch.logsumexp(x, 1)
    lp = x[torch.arange(x.shape[0], device=x.device), tokens.long()] - lse
    p = torch.exp(x - lse.unsqueeze(1))
    lp = torch.where(torch.isinf(lse), -math.inf, lp)
    # the terms of tokens that are ruled out are zero (0 times minus infinity)
    ent = torch.where(torch.isinf(lse), 0.0, -(p * (x - lse.unsqueeze(1))).nan_to_num(nan=0.0).sum(1))
    if not top:
        return lp, ent
    v = torch.topk(x, top, dim=1).values
    return lp, ent, None, torch.where(torch.isinf(lse).unsqueeze(1), -math.inf, v - lse.unsqueeze(1))


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    kind = case["kind"]
    if kind == "quantize":
        import numpy as np
        w = s["w"].double().cpu().numpy().reshape(case["N"], -1, case["G"])
        mn = w.min(-1).astype(np.float16)
        scale = np.maximum((w.max(-1) - mn.astype(np.float64)) / 15, 0).astype(np.float16)
        m64, s64 = mn.astype(np.float64)[..., None], scale.astype(np.float64)[..., None]
        with np.errstate(divide="ignore", invalid="ignore"):
            code = np.where(s64 > 0, np.clip(np.rint((w - m64) / s64), 0, 15), 0)
        return (code * s64 + m64).reshape(case["N"], case["K"])
    if kind == "linear":
        return s["x"].double() @ _exact_weight(*s["w"]).t()
    if kind == "logprobs":
        parts = [_exact_logprobs(x.double(), t, case["top"]) for x, t in zip(s["logits"].split(256), s["tokens"].split(256))]
        return tuple(None if p[0] is None else torch.cat(p) for p in zip(*parts))
    w = _exact_weight(*s["w"]) if case["w"] == "q4" else s["w"].double()
    return _exact_logprobs(s["x"].double() @ w.t(), s["tokens"], case["top"])


def work(case):
    kind = case["kind"]
    q4 = lambda N, K, G: N * K // 2 + 4 * N * (K // G)  # noqa: E731  codes, fp16 scale and minimum of each group
    size = {"f32": 4, "bf16": 2}
    if kind == "quantize":
        N, K = case["N"], case["K"]
        return dict(bytes=N * K * (size[case["w"]] + 4), flops=6 * N * K)
    if kind == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        w = q4(N, K, case["G"]) - (0 if case["mins"] else 2 * N * (K // case["G"]))
        return dict(bytes=w + M * K * size[case["x"]] + 4 * M * N, flops=2 * M * N * K)
    out = case["T"] * (12 + 8 * case["top"])  # the token, its log probability, the entropy, the alternatives
    if kind == "logprobs":
        return dict(bytes=case["T"] * case["V"] * size[case["dtype"]] + out, flops=4 * case["T"] * case["V"])
    T, V, K = case["T"], case["V"], case["K"]
    w = q4(V, K, case["G"]) if case["w"] == "q4" else 2 * V * K
    return dict(bytes=w + T * K * size[case["x"]] + out, flops=2 * T * V * K)
