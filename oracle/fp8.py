"""The block-scaled fp8 operators in 64 bits (test infrastructure only).

No reference counterpart: the reference's experts are 4-bit affine. Written
from the definitions in include/moestream.h, in torch float64 on the inputs'
device, with the error bounds of a 32-bit implementation beside the values.
"""
import torch

BLOCK = 128
TINY = 2.0 ** -100
U32 = 2.0 ** -24          # half a step of a 32-bit float


def blocks(n):
    return -(-n // BLOCK)


def spread(s, n, dim=-1):
    """Block scales spread over n elements."""
    return s.repeat_interleave(BLOCK, dim).narrow(dim, 0, n)


def group_max(v):
    """max |v| per 128 features, NaN where one is."""
    pad = torch.nn.functional.pad(v, (0, blocks(v.shape[-1]) * BLOCK - v.shape[-1]))
    return pad.reshape(*v.shape[:-1], -1, BLOCK).abs().amax(-1)


def scale_of(a):
    """The smallest power of two s with max(a, 2^-100) <= 448 s; NaN where a
    is not finite."""
    a = a.double().clamp_min(TINY)
    m, e = torch.frexp(a / 448.0)                # m in [0.5, 1)
    s = torch.ldexp(torch.ones_like(a), torch.where(m == 0.5, e - 1, e))
    return torch.where(torch.isfinite(a), s, torch.full_like(s, float("nan")))


def e4m3_step(v):
    """Distance of neighbouring e4m3 values around |v|."""
    return torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3.0)


def e4m3(v):
    """v to the nearest e4m3 value (ties to even), as float64; NaN stays."""
    step = e4m3_step(v)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def quantize(v):
    """(codes as float64 values, scales) of v [..., d]."""
    v = v.double()
    s = scale_of(group_max(v))
    return e4m3(v / spread(s, v.shape[-1])), s


def rms_norm(x, weight, eps, residual=None):
    """(h in x's type, y float64)."""
    h = x if residual is None else (x.double() + residual.double()).float().to(x.dtype)
    v = h.double()
    return h, v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps) * weight.double()


def rows_value(q, s):
    return q.double() * spread(s.double(), q.shape[-1])


def weight_value(q, s):
    n, k = q.shape[-2:]
    return q.double() * spread(spread(s.double(), n, -2), k, -1)


def product(x, w, kb):
    """(x w^T, error bound of 32-bit sums): products of e4m3 codes are exact
    in 32 bits; a block adds at most 128 of them and the result sums kb blocks
    after two scale products each, every step off by at most a whole step of a
    32-bit float (2^-23: an adder that truncates) of the magnitudes' sum."""
    y = x @ w.mT
    return y, (BLOCK + kb + 4) * 2 * U32 * (x.abs() @ w.abs().mT)


def product_likely(x, w, kb):
    """(x w^T, error that a 32-bit computation stays within in all likelihood):
    the roundings of one sum are independent, so they add up as the root of
    their number. A block takes at most 128 of them at random signs, or 16 of
    an adder of 32 products that truncates; kb blocks and four scale products
    follow. Each is at most 2^-23 of a partial sum, which is about the root of
    the products' squares; eight times that."""
    y = x @ w.mT
    return y, 8.0 * 2 * U32 * (16 + kb ** 0.5 + 4) * torch.sqrt(x.square() @ w.square().mT)


def quantize_bound(v, e):
    """(value of the quantised v, how far the quantised value of anything
    within e of v may be from it)."""
    d = v.shape[-1]
    q, s = quantize(v)
    s0 = scale_of(group_max((v.abs() - e).clamp_min(0.0)))
    s1 = scale_of(group_max(v.abs() + e))
    sv = spread(s, d)
    moves = e4m3((v - e) / sv) != e4m3((v + e) / sv)
    off = torch.where(moves, e4m3_step((v.abs() + e) / sv) * sv, torch.zeros_like(v))
    # another scale changes what is below the normal range of the larger one
    big = spread(s1, d)
    other = spread((s0 != s1).double(), d) > 0
    off = torch.where(other, off + e4m3_step((v.abs() + e) / big) * big, off)
    return q * sv, off


def route(x, router, bias, k, model, norm):
    """(indices [T, k], probabilities, their relative error bound [T, 1], per
    token whether the choice is beyond the logits' error bound). The bound: a warp's 32 lanes sum d / 32 products each (exact in 32
    bits: bf16 times bf16) and join them in five steps, then the bias; up to
    three more joins where the sum is split over warps."""
    x, router = x.double(), router.double()
    logits = x @ router.T
    mag = x.abs() @ router.abs().T
    if bias is not None:
        logits = logits + bias.double()
        mag = mag + bias.double().abs()
    err = ((x.shape[-1] / 32 + 9) * U32 * mag).amax(-1)
    order = torch.sort(logits, dim=-1, descending=True, stable=True)
    top, at = order.values[:, :k], order.indices[:, :k]
    sure = top[:, -1] - order.values[:, k] > 2 * err if k < logits.shape[-1] else err >= 0
    if model == "gptoss" or norm:
        p = torch.softmax(top, -1)
    else:
        p = torch.softmax(logits, -1).gather(1, at)
    return at, p, (4 * err + 600 * U32).unsqueeze(-1), sure


def moe_layer(x, router, router_bias, gate, up, down, k, model, norm=True, residual=None):
    """(y float64, bound of |bf16 result - y|, per token whether its experts
    are beyond doubt). gate, up, down: (codes, scales, bias or None)."""
    T, d = x.shape
    f = gate[0].shape[1]
    at, p, p_err, sure = route(x, router, router_bias, k, model, norm)
    q, s = quantize(x)
    xv = rows_value(q, s)
    y = torch.zeros(T, d, dtype=torch.float64, device=x.device)
    tol, mag = torch.zeros_like(y), torch.zeros_like(y)
    for e in at.unique().tolist():
        t, j = (at == e).nonzero(as_tuple=True)
        g, ge = product_likely(xv[t], weight_value(gate[0][e], gate[1][e]), blocks(d))
        u, ue = product_likely(xv[t], weight_value(up[0][e], up[1][e]), blocks(d))
        if gate[2] is not None:
            g, ge = g + gate[2][e].double(), ge + U32 * (g.abs() + gate[2][e].double().abs())
        if up[2] is not None:
            u, ue = u + up[2][e].double(), ue + U32 * (u.abs() + up[2][e].double().abs())
        a = 1.0
        if model == "gptoss":             # beyond a clamp no error passes
            ge = torch.where(g - ge > 7.0, torch.zeros_like(ge), ge)
            ue = torch.where(u.abs() - ue > 7.0, torch.zeros_like(ue), ue)
            g, u, a = g.clamp(max=7.0), u.clamp(-7.0, 7.0), 1.702
        sig = 1.0 / (1.0 + torch.exp(-a * g))
        sg, v = g * sig, u + 1.0 if model == "gptoss" else u
        h = sg * v
        # slope of g sigmoid(a g), whose own slope is at most a / 2; a dozen
        # roundings and exp's own error on the way
        slope = (sig + a * g * sig * (1.0 - sig)).abs() + ge
        he = slope * v.abs() * ge + (sg.abs() + slope * ge) * ue + 32 * U32 * (h.abs() + sg.abs())
        hv, off = quantize_bound(h, he)
        w = weight_value(down[0][e], down[1][e])
        o, oe = product_likely(hv, w, blocks(f))
        # codes that may have moved do so by themselves: their sum is within
        # six times the root of their squares' sum
        oe = oe + 6.0 * torch.sqrt(off.square() @ w.square().mT)
        if down[2] is not None:
            o, oe = o + down[2][e].double(), oe + U32 * (o.abs() + down[2][e].double().abs())
        pe = p[t, j].unsqueeze(-1)
        y.index_add_(0, t, pe * o)
        tol.index_add_(0, t, pe * (oe + p_err[t] * (o.abs() + oe)))
        mag.index_add_(0, t, (pe * o).abs())
    if residual is not None:
        y, mag = y + residual.double(), mag + residual.double().abs()
    tol = tol + (k + 2) * U32 * mag
    # one rounding to bf16: 2^-8 of the value that is rounded
    return y, tol + 2.0 ** -8 * (y.abs() + tol), sure
