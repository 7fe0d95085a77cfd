"""The fp8 operators' cases: what is measured and their plain forms.

rms_norm_fp8 / quantize_fp8  residual add + RMSNorm + e4m3 codes with a scale per 128 features
Fp8Linear                    product of e4m3 matrices, scales per 1x128 (rows) and 128x128 (weight)
Fp8MoELayer                  router + top-k + e4m3 experts + weighted sum for a few tokens

The shapes are the two model geometries of this repository (Qwen3: d 2048, d_ff 768, 128 experts,
top 8; gpt-oss: d 2880, d_ff 2880, 128 experts, top 4) and their attention projections.
"""
import math

import torch

own = False

BLOCK = 128
TINY = 2.0 ** -100
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one decode token between two sub-layers: the smallest call, all latency
        dict(name="norm_token", op="norm", T=1, d=2048, dtype="bf16", residual=True),
        # a speculative batch of odd length; 2880 = 22 groups and a half one
        dict(name="norm_odd", op="norm", T=37, d=2880, dtype="fp16", residual=True),
        # a prefill of 16384 tokens, the largest batch this repository measures
        dict(name="norm_prefill", op="norm", T=16384, d=2880, dtype="bf16", residual=True),
        # the attention output (64 heads of 64) before its projection: codes only, no norm
        dict(name="quant_rows", op="quant", T=4099, d=4096, dtype="bf16"),
        # one decode token through the qkv projection of 32 + 2*4 heads of 128
        dict(name="linear_token", op="linear", M=1, N=5120, K=2048, out="bf16", bias=False),
        # sixteen sequences through an output projection with a bias
        dict(name="linear_batch", op="linear", M=16, N=2880, K=4096, out="bf16", bias=True),
        # a ragged chunk through a qkv projection (64 + 2*8 heads of 64), K = 22.5 blocks
        dict(name="linear_chunk", op="linear", M=333, N=5120, K=2880, out="fp32", bias=True),
        # the whole prefill batch through the same projection: the largest product
        dict(name="linear_prefill", op="linear", M=16384, N=5120, K=2880, out="bf16", bias=True),
        # one decode token through a whole Qwen3 layer
        dict(name="moe_token", op="moe", model="qwen3", T=1, d=2048, f=768, E=128, k=8, residual=True),
        # five tokens of a multi-token verify through a gpt-oss layer (half blocks, biases)
        dict(name="moe_verify", op="moe", model="gptoss", T=5, d=2880, f=2880, E=128, k=4, residual=False),
        # sixteen sequences decoding together
        dict(name="moe_batch", op="moe", model="qwen3", T=16, d=2048, f=768, E=128, k=8, residual=True),
        # the largest few-token batch, an odd one: every expert is read
        dict(name="moe_many", op="moe", model="qwen3", T=61, d=2048, f=768, E=128, k=8, residual=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "quant", "linear", "linear", "moe", "moe"])
    if op in ("norm", "quant"):
        T, d = _log(rng, 1, 16384), _log(rng, 64, 8192)
        if rng.random() < 0.7:
            d = (d + 15) // 16 * 16
        T = max(1, min(T, 16384 * 2880 // d))
        c = dict(op=op, T=T, d=d, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
        if c["dtype"] == "fp32":
            c["T"] = max(1, T // 2)
        if op == "norm":
            c["residual"] = rng.random() < 0.7
        return c
    if op == "linear":
        M, N, K = _log(rng, 1, 16384), _log(rng, 64, 8192), _log(rng, 64, 8192)
        if rng.random() < 0.7:
            N, K = (N + 63) // 64 * 64, (K + 63) // 64 * 64
        M = max(1, min(M, 16384 * 5120 * 2880 // (N * K)))
        return dict(op=op, M=M, N=N, K=K, out=rng.choice(["bf16", "bf16", "fp16", "fp32"]), bias=rng.random() < 0.5)
    model = rng.choice(["qwen3", "gptoss"])
    E = rng.choice([8, 16, 32, 60, 64, 128])
    d, f = 16 * _log(rng, 8, 180), 16 * _log(rng, 8, 180)
    while E * d * f > 128 * 2048 * 768:
        d, f = max(128, d // 32 * 16), max(128, f // 32 * 16)
    return dict(op=op, model=model, T=_log(rng, 1, 64), d=d, f=f, E=E, k=rng.randint(1, 8), residual=rng.random() < 0.5)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _code_rows(v, scale):
    """e4m3 codes of v / scale in rows whose stride is a multiple of 16 bytes."""
    q = torch.zeros(*v.shape[:-1], (v.shape[-1] + 15) // 16 * 16, dtype=torch.uint8, device="cuda")
    q[..., : v.shape[-1]] = (v / scale).to(torch.float8_e4m3fn).view(torch.uint8)
    return q.view(torch.float8_e4m3fn)[..., : v.shape[-1]]


def _over(s, n, dim):
    """Block scales s spread over n elements of dimension dim."""
    return s.repeat_interleave(BLOCK, dim=dim).narrow(dim, 0, n)


def _weight(g, *shape):
    """A weight N(0, 0.02) as e4m3 codes with a scale per 128x128 block."""
    w = _randn(g, *shape) * 0.02
    n, k = shape[-2], shape[-1]
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    p = torch.nn.functional.pad(w, (0, kb * BLOCK - k, 0, nb * BLOCK - n))
    s = p.reshape(*shape[:-2], nb, BLOCK, kb, BLOCK).abs().amax(dim=(-3, -1)).clamp_min(1e-12) / 448.0
    return _code_rows(w, _over(_over(s, n, -2), k, -1)), s.contiguous()


def _experts(g, E, n, k):
    q = torch.empty(E, n, k, dtype=torch.float8_e4m3fn, device="cuda")
    s = torch.empty(E, -(-n // BLOCK), -(-k // BLOCK), device="cuda")
    step = max(1, (1 << 27) // (n * k))
    for e in range(0, E, step):
        m = min(step, E - e)
        q[e:e + m], s[e:e + m] = _weight(g, m, n, k)
    return q, s


def _stream_values(g, T, d):
    """Hidden states as they come: N(0, 1) with a few features many times larger."""
    return _randn(g, T, d) * (1.0 + 15.0 * (torch.rand(d, generator=g, device="cuda") < 0.01))


def prepare(case, seed):
    g = _gen(seed)
    c = dict(case)
    if c["op"] in ("norm", "quant"):
        dt = DTYPES[c["dtype"]]
        c["x"] = _stream_values(g, c["T"], c["d"]).to(dt)
        if c["op"] == "norm":
            c["w"] = (1.0 + 0.2 * _randn(g, c["d"])).to(dt)
            c["r"] = _stream_values(g, c["T"], c["d"]).to(dt) if c["residual"] else None
        if own:
            from moe_stream_b200 import fp8
            c["call"] = fp8
    elif c["op"] == "linear":
        M, N, K = c["M"], c["N"], c["K"]
        x = _stream_values(g, M, K)
        kb = -(-K // BLOCK)
        s = torch.nn.functional.pad(x, (0, kb * BLOCK - K)).reshape(M, kb, BLOCK).abs().amax(-1) / 448.0
        c["xq"], c["xs"] = _code_rows(x, _over(s, K, -1)), s.contiguous()
        c["wq"], c["ws"] = _weight(g, N, K)
        c["b"] = (0.5 * _randn(g, N)).to(torch.bfloat16) if c["bias"] else None
        if own:
            from moe_stream_b200 import fp8
            c["call"] = fp8.Fp8Linear(c["wq"], c["ws"], bias=c["b"])
    else:
        T, d, f, E = c["T"], c["d"], c["f"], c["E"]
        x = _randn(g, T, d)
        c["x"] = (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)).to(torch.bfloat16)
        c["r"] = _randn(g, T, d).to(torch.bfloat16) if c["residual"] else None
        c["router"] = (_randn(g, E, d) * 0.02).to(torch.bfloat16)
        c["gate"], c["up"], c["down"] = _experts(g, E, f, d), _experts(g, E, f, d), _experts(g, E, d, f)
        oss = c["model"] == "gptoss"
        c["router_bias"] = (0.1 * _randn(g, E)).to(torch.bfloat16) if oss else None
        c["biases"] = [(0.02 * _randn(g, E, n)).to(torch.bfloat16) if oss else None for n in (f, f, d)]
        if own:
            from moe_stream_b200 import fp8
            gb, ub, db = c["biases"]
            c["call"] = fp8.Fp8MoELayer(
                c["model"], c["router"], gate=(*c["gate"], gb), up=(*c["up"], ub), down=(*c["down"], db),
                top_k=c["k"], router_bias=c["router_bias"], norm_topk_prob=True)
    return c


# ------------------------------------------------------------- plain forms
def _groups(v):
    n = -(-v.shape[-1] // BLOCK)
    v = torch.nn.functional.pad(v, (0, n * BLOCK - v.shape[-1]))
    return v.reshape(*v.shape[:-1], n, BLOCK)


def _quantize(v):
    """(e4m3 codes, scales) of float32 v: per 128 features the scale is the smallest power of two s with
    max|v| <= 448 s (max|v| taken as 2^-100 at least), the code e4m3(v / s); NaN where max|v| is not finite."""
    g = _groups(v)
    a = g.abs().amax(dim=-1, keepdim=True).clamp_min(TINY)
    bits = a.view(torch.int32)        # a = 1.m * 2^(e - 127), 448 = 1.75 * 2^8
    e = (bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()
    s = torch.where(torch.isfinite(a), (e << 23).view(torch.float32), math.nan)
    q = (g / s).to(torch.float8_e4m3fn)
    return q.reshape(*v.shape[:-1], -1)[..., : v.shape[-1]], s.squeeze(-1)


def _dequantize(q, s):
    return q.float() * _over(s, q.shape[-1], -1)


def _dequantize_weight(q, s):
    return q.float() * _over(_over(s, q.shape[-2], -2), q.shape[-1], -1)


def _plain_norm(c):
    h = c["x"] if c["r"] is None else (c["x"].float() + c["r"].float()).to(c["x"].dtype)
    v = h.float()
    # 64 bits: a value next to a border between two codes or scales must not cross it
    rms = (1.0 / torch.sqrt(v.double().square().mean(-1, keepdim=True) + 1e-6)).float()
    y = v * rms * c["w"].float()
    q, s = _quantize(y)
    return dict(q=q, s=s, h=h)


def _plain_linear(c):
    y = _dequantize(c["xq"], c["xs"]) @ _dequantize_weight(c["wq"], c["ws"]).T
    if c["b"] is not None:
        y = y + c["b"].float()
    return y.to(DTYPES[c["out"]])


def _pick(q, at):
    return q.view(torch.uint8)[at].view(torch.float8_e4m3fn)


def _plain_moe(c):
    oss, T, k, E = c["model"] == "gptoss", c["T"], c["k"], c["E"]
    # 64 bits: a logit next to another must not change places
    logits = c["x"].double() @ c["router"].double().T
    if oss:
        logits = logits + c["router_bias"].double()
    logits = logits.float()
    top, at = torch.sort(logits, dim=-1, descending=True, stable=True)
    top, at = top[:, :k], at[:, :k]
    p = torch.softmax(top, dim=-1)   # also softmax over all E, top k, renormalised
    xv = _dequantize(*_quantize(c["x"].float()))
    bg, bu, bd = c["biases"]

    def act(g, u):
        if not oss:
            return g * torch.sigmoid(g) * u
        g, u = g.clamp(max=7.0), u.clamp(-7.0, 7.0)
        return g * torch.sigmoid(1.702 * g) * (u + 1.0)

    if T * k < E:                     # the pairs' experts, one by one
        at = at.reshape(-1)
        xv = xv.repeat_interleave(k, dim=0).unsqueeze(-1)
        pick = lambda m: _dequantize_weight(_pick(m[0], at), m[1][at])  # noqa: E731
        add = lambda b: b.float()[at] if oss else 0.0                    # noqa: E731
        h = act((pick(c["gate"]) @ xv).squeeze(-1) + add(bg), (pick(c["up"]) @ xv).squeeze(-1) + add(bu))
        h = _dequantize(*_quantize(h)).unsqueeze(-1)
        y = (pick(c["down"]) @ h).squeeze(-1) + add(bd)
        y = (p.unsqueeze(-1) * y.reshape(T, k, -1)).sum(1)
    else:                             # every expert is asked for: all of them at once
        full = torch.zeros(T, E, device=p.device).scatter_(1, at, p)
        add = lambda b: b.float().unsqueeze(1) if oss else 0.0           # noqa: E731
        h = act(xv @ _dequantize_weight(*c["gate"]).mT + add(bg), xv @ _dequantize_weight(*c["up"]).mT + add(bu))
        h = _dequantize(*_quantize(h))
        y = h @ _dequantize_weight(*c["down"]).mT + add(bd)
        y = (full.T.unsqueeze(-1) * y).sum(0)
    if c["r"] is not None:
        y = y + c["r"].float()
    return y.to(torch.bfloat16)


def run(state):
    c = state
    if c["op"] == "norm":
        if own:
            q, s, h = c["call"].rms_norm_fp8(c["x"], c["w"], eps=1e-6, residual=c["r"])
            return dict(q=q, s=s, h=h)
        return _plain_norm(c)
    if c["op"] == "quant":
        q, s = c["call"].quantize_fp8(c["x"]) if own else _quantize(c["x"].float())
        return dict(q=q, s=s)
    if c["op"] == "linear":
        return c["call"](c["xq"], c["xs"], out_dtype=DTYPES[c["out"]]) if own else _plain_linear(c)
    return c["call"](c["x"], residual=c["r"]) if own else _plain_moe(c)


def work(case):
    c = case
    if c["op"] in ("norm", "quant"):
        b = BYTES[c["dtype"]]
        n = c["T"] * c["d"]
        per = b + 1 + (2 * b if c.get("residual") else 0)
        norm = c["op"] == "norm"
        return {"bytes": n * per + 4 * c["T"] * -(-c["d"] // BLOCK) + (b * c["d"] if norm else 0),
                "flops": n * (6 if norm else 2)}
    if c["op"] == "linear":
        M, N, K = c["M"], c["N"], c["K"]
        kb = -(-K // BLOCK)
        return {"bytes": M * K + N * K + 4 * kb * (M + -(-N // BLOCK)) + M * N * BYTES[c["out"]] + 2 * N * c["bias"],
                "flops": 2 * M * N * K}
    T, d, f, E, k = c["T"], c["d"], c["f"], c["E"], c["k"]
    # distinct experts that T tokens of k each ask for when every expert is as likely as any other
    distinct = E * (1.0 - (1.0 - k / E) ** T)
    return {"bytes": distinct * 3 * d * f + 2 * E * d + 2 * T * d * (3 if c["residual"] else 2),
            "flops": 2 * T * k * 3 * d * f + 2 * T * E * d}


# ---------------------------------------------------------- in 64 bits
def _e4m3(v):
    """v (64 bits, |v| <= 464) to the nearest e4m3 value, ties to even."""
    e = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6)))
    step = torch.exp2(e - 3.0)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def _quantize64(v):
    cut = list(range(0, v.shape[-1], BLOCK))
    a = torch.stack([v[..., i:i + BLOCK].abs().amax(-1) for i in cut], -1).clamp_min(TINY)
    m, e = torch.frexp(a / 448.0)
    s = torch.ldexp(torch.ones_like(a), e - (m == 0.5).int())   # 2^ceil(log2(a / 448))
    q = torch.cat([_e4m3(v[..., i:i + BLOCK] / s[..., j:j + 1]) for j, i in enumerate(cut)], -1)
    return q, s


def _value64(q, s):
    """Codes times their block scales: s has one row per code row, or one per 128 of them."""
    rows = torch.arange(q.shape[0], device=q.device)
    if s.shape[0] != q.shape[0]:
        rows = rows // BLOCK
    return q.double() * s.double()[rows][:, torch.arange(q.shape[1], device=q.device) // BLOCK]


def exact(case, seed):
    c = prepare(case, seed)
    if c["op"] in ("norm", "quant"):
        v = c["x"].double()
        out = {}
        if c["op"] == "norm":
            if c["r"] is not None:
                v = (v + c["r"].double()).to(c["x"].dtype).double()
            out["h"] = v
            v = v / torch.sqrt((v * v).sum(-1, keepdim=True) / c["d"] + 1e-6) * c["w"].double()
        q, s = _quantize64(v)
        return dict(out, q=q, s=s)
    if c["op"] == "linear":
        y = torch.matmul(_value64(c["xq"], c["xs"]), _value64(c["wq"], c["ws"]).t())
        return y if c["b"] is None else y + c["b"].double()
    oss = c["model"] == "gptoss"
    x = c["x"].double()
    l = torch.matmul(x, c["router"].double().t())
    if oss:
        l = l + c["router_bias"].double()
    best = l.topk(c["k"], dim=-1)
    p = torch.exp(best.values - best.values.max(-1, keepdim=True).values)
    p = p / p.sum(-1, keepdim=True)
    xq, xs = _quantize64(x)
    xv = _value64(xq, xs)
    y = torch.zeros_like(x)
    for e in best.indices.unique().tolist():
        t, j = (best.indices == e).nonzero(as_tuple=True)
        g = xv[t] @ _value64(c["gate"][0][e], c["gate"][1][e]).t()
        u = xv[t] @ _value64(c["up"][0][e], c["up"][1][e]).t()
        if oss:
            g, u = g + c["biases"][0][e].double(), u + c["biases"][1][e].double()
            g, u = torch.minimum(g, torch.full_like(g, 7.0)), torch.minimum(torch.maximum(u, torch.full_like(u, -7.0)), torch.full_like(u, 7.0))
            h = g / (1.0 + torch.exp(-1.702 * g)) * (u + 1.0)
        else:
            h = g / (1.0 + torch.exp(-g)) * u
        hq, hs = _quantize64(h)
        o = _value64(hq, hs) @ _value64(c["down"][0][e], c["down"][1][e]).t()
        if oss:
            o = o + c["biases"][2][e].double()
        y.index_add_(0, t, o * p[t, j].unsqueeze(-1))
    return y if c["r"] is None else y + c["r"].double()
