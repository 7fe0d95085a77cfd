"""Block-scaled fp8: the norm, the dense products and the MoE layer of models
whose weights are e4m3 codes with a scale per 128 x 128 block.

The pool's experts are 4-bit affine blobs streamed into slots (``MoEBlock``);
these operators are for checkpoints in the other common serving format, held
in HBM whole. They chain as a decoder layer does:

    q, s, h = rms_norm_fp8(x, norm_weight, residual=h)   # add, norm, codes
    qkv     = Fp8Linear(w, w_scales)(q, s)               # projection
    q, s    = quantize_fp8(attention_output)
    q, s, h, y = rms_norm_fp8(Fp8Linear(...)(q, s), norm2, residual=h, with_norm=True)
    h       = Fp8MoELayer(...)(y, residual=h)            # whole MoE layer

A matrix is (codes, scales): codes float8_e4m3fn, scales float32, one per row
and 128 features of activations, one per 128 x 128 block of weights (e4m3
code times scale is the value). The quantiser's scales are powers of two; the
products take any scales whose products, a row's with a weight block's, stay in
the normal range of 32 bits.

Everything is asynchronous on the current stream of the inputs' device (or on
``stream=``, which the caller has made to wait for the inputs), allocates only through torch, keeps no state between calls and
can be captured into a CUDA graph. As in the rest of the package there is no
CPU implementation and no backward pass.
"""
import ctypes
import struct

import torch

from . import _lib

BLOCK = 128
MAX_TOKENS = 64           # MS_FP8_MAX_TOKENS
MAX_FEATURES = 16384      # MS_FP8_MAX_FEATURES
MAX_ROWS = 2 ** 31 - 2 ** 16   # MS_FP8_MAX_ROWS
_DT = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_E4M3 = torch.float8_e4m3fn

# ms_fp8_norm, ms_fp8_linear, ms_fp8_moe as the header declares them
_NORM = struct.Struct("@7P5qd4i")
_LINEAR = struct.Struct("@6P4q6i")
_MOE = struct.Struct("@3P3P3P3P3PQ8i")


def _blocks(n):
    return -(-n // BLOCK)


def _stream(device, stream=None):
    """Raw handle of `stream`, or of the current stream of device `device`."""
    return torch._C._cuda_getCurrentRawStream(device) if stream is None else stream.cuda_stream


def _on_stream(call, stream, device, *args, keep=(), captured=None):
    """call(*args) with `stream` current, behind the event `captured`: the
    tensors it makes belong to the stream that writes them. The tensors it
    reads (args, and `keep`) may be dropped once it returns: their memory is
    not used again before `stream` has come past the call."""
    if stream.device.index != device:
        raise ValueError(f"stream is on {stream.device}, the inputs on cuda:{device}")
    with torch.cuda.stream(stream):
        if captured is not None and torch.cuda.is_current_stream_capturing():
            stream.wait_event(captured)
        out = call(*args)
    for t in (*args, *keep):
        if isinstance(t, torch.Tensor):
            t.record_stream(stream)
    return out


def _rows(name, t, d=None, dtype=None):
    """t as [rows, features] with contiguous rows (a view where it is one)."""
    if not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if dtype is not None and t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    rank = t.dim()
    if rank == 0:
        raise ValueError(f"{name} must have a feature dimension")
    n = t.shape[-1]
    if d is not None and n != d:
        raise ValueError(f"{name} has {n} features, expected {d}")
    if rank != 2:
        t = t.reshape(-1, n) if t.numel() else t.reshape(0, n)
    if n > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t


def _row_stride(t):
    """Elements between the rows of a [rows, n] tensor (of one row: any)."""
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], t.stride(0))


def _out(name, t, shape, dtype, device):
    if t.dtype is not dtype or t.device.index != device or not t.is_cuda:
        raise TypeError(f"{name} must be a {dtype} tensor on cuda:{device}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def _codes_like(lead, d, device):
    """Uninitialised codes [..., d] whose rows start on 16-byte boundaries, as
    the products read them."""
    pad = (d + 15) // 16 * 16
    q = torch.empty((*lead, pad), dtype=_E4M3, device=device)
    return q if pad == d else q[..., :d]


def _like(name, t, x, dev):
    """t, a tensor that goes with x row by row, as contiguous rows."""
    if t.get_device() != dev:
        raise TypeError(f"{name} must be on x's device")
    if t.dtype is not x.dtype:
        raise TypeError(f"{name} must be {x.dtype}, got {t.dtype}")
    if t.shape != x.shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, x {tuple(x.shape)}")
    return t if t.is_contiguous() else _rows(name, t)


def _norm_call(x, weight, eps, residual, h_out, with_norm):
    # A call of a few rows takes less time on the GPU than here: contiguous
    # inputs, the ordinary case, go through with no views made of them.
    dt = _DT.get(x.dtype)
    if dt is None:
        raise TypeError(f"x must be bfloat16, float16 or float32, got {x.dtype}")
    if x.is_contiguous() and x.is_cuda and x.dim():
        x2, shape = x, x.shape
        d = xs = shape[-1]
    else:
        x2 = _rows("x", x)
        shape, d, xs = x.shape, x2.shape[1], _row_stride(x2)
    if not 1 <= d <= MAX_FEATURES:
        raise ValueError(f"x has {d} features, supported are 1 to {MAX_FEATURES}")
    T = x.numel() // d
    if T > MAX_ROWS:
        raise ValueError(f"x has {T} rows, at most {MAX_ROWS} per call")
    dev = x.get_device()
    wp = rp = hp = yp = rs = 0
    h = y = None
    if weight is not None:
        if weight.dtype is not x.dtype or weight.get_device() != dev:
            raise TypeError("weight must have x's dtype and device")
        if weight.shape != (d,):
            raise ValueError(f"weight has shape {tuple(weight.shape)}, expected ({d},)")
        if not eps >= 0.0:
            raise ValueError(f"eps must not be negative, got {eps}")
        if not weight.is_contiguous():
            weight = weight.contiguous()
        wp = weight.data_ptr()
    if residual is not None:
        res = _like("residual", residual, x, dev)
        rp, rs = res.data_ptr(), d if res.is_contiguous() else _row_stride(res)
        if h_out is None:
            h = torch.empty_like(x, memory_format=torch.contiguous_format)
        else:
            h = _out("h_out", h_out, shape, x.dtype, dev)
        hp = h.data_ptr()
    elif h_out is not None:
        raise ValueError("h_out needs a residual")
    if d % 16:
        q = _codes_like(shape[:-1], d, x.device)
    else:
        q = torch.empty_like(x, dtype=_E4M3, memory_format=torch.contiguous_format)
    s = x.new_empty((*shape[:-1], (d + 127) // 128), dtype=torch.float32)
    if with_norm:
        y = torch.empty_like(x, memory_format=torch.contiguous_format)
        yp = y.data_ptr()
    if T:
        args = _NORM.pack(x2.data_ptr(), rp, wp, hp, yp, q.data_ptr(), s.data_ptr(),
                          xs, rs, d, d, (d + 15) // 16 * 16, eps, T, d, dt, dev)
        rc = _lib.load().ms_rms_norm_fp8(args, _stream(dev))
        if rc:
            _lib.check(rc)
    return q, s, (x if h is None else h), y


def rms_norm_fp8(x, weight, eps=1e-6, residual=None, h_out=None, with_norm=False, stream=None):
    """Residual add, RMSNorm and quantisation in one pass: returns (q, scales,
    h[, y]) for x [..., d] in bf16, fp16 or fp32 (weight and residual alike).

    h = round(x + residual) (x itself without a residual),
    y = h / sqrt(mean(h^2) + eps) * weight (returned, rounded to x's type, if
    with_norm), q the e4m3 codes and scales [..., ceil(d/128)] of the
    unrounded y: per 128 features the smallest power of two with
    max|y| <= 448 * scale. A group with a NaN or an infinity is NaN whole.
    h_out may be x or residual (in place)."""
    if weight is None:
        raise TypeError("weight must be a tensor (quantize_fp8 quantises without a norm)")
    args = (x, weight, eps, residual, h_out, with_norm)
    q, s, h, y = _norm_call(*args) if stream is None else _on_stream(_norm_call, stream, x.device.index, *args)
    return (q, s, h, y) if with_norm else (q, s, h)


def quantize_fp8(x, stream=None):
    """(codes, scales) of x [..., d] as rms_norm_fp8 quantises."""
    args = (x, None, 0.0, None, None, False)
    q, s, _, _ = _norm_call(*args) if stream is None else _on_stream(_norm_call, stream, x.device.index, *args)
    return q, s


def status(device=None, stream=None):
    """Raise if a bounded wait inside an fp8 kernel on `device` ran out since
    the last call (its output is not valid). Waits for the stream."""
    dev = None if device is None else torch.device(device).index
    if dev is None:
        dev = torch.cuda.current_device()
    st = ctypes.c_int()
    _lib.check(_lib.load().ms_fp8_status(dev, ctypes.byref(st), ctypes.c_void_p(_stream(dev, stream))))


def quantize_weight_fp8(w):
    """(codes, scales) of a weight [..., n, k], one scale max|block| / 448 per
    128 x 128 block, as checkpoints hold them. Runs in torch, on w's device."""
    n, k = w.shape[-2:]
    nb, kb = _blocks(n), _blocks(k)
    w = w.float()
    p = torch.nn.functional.pad(w, (0, kb * BLOCK - k, 0, nb * BLOCK - n))
    s = p.reshape(*w.shape[:-2], nb, BLOCK, kb, BLOCK).abs().amax(dim=(-3, -1)).clamp_min(2.0 ** -100) / 448.0
    return (w / spread_scales(s, n, k)).clamp(-448.0, 448.0).to(_E4M3), s


def spread_scales(s, n, k):
    """Block scales [..., ceil(n/128), ceil(k/128)] spread over [..., n, k]."""
    return s.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]


def _bias(b, shape, device):
    if b is None:
        return None
    if tuple(b.shape) != tuple(shape):
        raise ValueError(f"bias has shape {tuple(b.shape)}, expected {tuple(shape)}")
    return b.detach().to(device=device, dtype=torch.float32).contiguous()


def _weight(name, codes, scales, rank, device=None):
    """Checked (codes, scales) with contiguous scales and 16-byte rows."""
    if codes.dtype is not _E4M3 or not codes.is_cuda or codes.dim() != rank:
        raise TypeError(f"{name} must be a {rank}-dimensional float8_e4m3fn CUDA tensor")
    if scales.dtype is not torch.float32:
        raise TypeError(f"{name}'s scales must be float32")
    if scales.device != codes.device or (device is not None and codes.device != device):
        raise TypeError(f"{name} and its scales must be on one device")
    want = (*codes.shape[:-2], _blocks(codes.shape[-2]), _blocks(codes.shape[-1]))
    if tuple(scales.shape) != want:
        raise ValueError(f"{name}'s scales have shape {tuple(scales.shape)}, expected {want}")
    return codes, scales.contiguous()


def _wait_for_copies(device, given, used):
    """Calls may come on any stream, so the copies that a constructor has
    queued are waited for. Inside a capture they are part of the graph, and so
    are the calls that may read them: the event behind them is returned."""
    if any(u is not None and u.data_ptr() != g.data_ptr() for g, u in zip(given, used)):
        with torch.cuda.device(device):
            if torch.cuda.is_current_stream_capturing():
                return torch.cuda.current_stream().record_event()
            torch.cuda.current_stream().synchronize()
    return None


class Fp8Linear:
    """y = x w^T (+ bias) for a weight w [N, K] in codes and block scales.

    A weight whose rows are contiguous and start on 16-byte boundaries is used
    where it is; another is copied once, here, as are scales that are not
    contiguous and a bias that is not float32. The copies are waited for, so
    the layer may be called on any stream; a layer that copies inside a capture
    belongs to that graph."""

    def __init__(self, weight, scales, bias=None):
        w, self.scales = _weight("weight", weight, scales, 2)
        self.out_features, self.in_features = N, K = w.shape
        if N < 1 or K < 1:
            raise ValueError("weight must not be empty")
        if max(N, K) > MAX_ROWS:
            raise ValueError(f"weight has {N} rows of {K}, supported are {MAX_ROWS} of either")
        if (K > 1 and w.stride(1) != 1) or w.data_ptr() % 16 or _row_stride(w) % 16 or _row_stride(w) < K:
            p = _codes_like((N,), K, w.device)
            p.copy_(w)
            w = p
        self.weight = w
        self.bias = _bias(bias, (N,), w.device)
        self.device = w.device
        self._captured = _wait_for_copies(w.device, (weight, scales, bias), (w, self.scales, self.bias))
        self._w = (w.data_ptr(), self.scales.data_ptr(), 0 if self.bias is None else self.bias.data_ptr())
        self._ld = _row_stride(w)
        self._dims = (K, N, _blocks(K), w.get_device())
        self._call = _lib.load().ms_linear_fp8

    def __call__(self, q, scales, out_dtype=torch.bfloat16, out=None, stream=None):
        """[..., N] of codes q [..., K] and scales [..., ceil(K/128)], in
        bf16, fp16 or fp32."""
        if stream is not None:
            return _on_stream(self._forward, stream, self.device.index, q, scales, out_dtype, out,
                              keep=(self.weight, self.scales, self.bias), captured=self._captured)
        return self._forward(q, scales, out_dtype, out)

    def _forward(self, q, scales, out_dtype, out):
        K, N, KB, dev = self._dims
        if q.get_device() != dev or scales.get_device() != dev:
            raise TypeError(f"codes and scales must be on the weight's device, {self.device}")
        dt = _DT.get(out_dtype)
        if dt is None:
            raise TypeError(f"out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
        lead = q.shape[:-1]
        if scales.shape[:-1] != lead:
            raise ValueError(f"scales have shape {tuple(scales.shape)} for codes {tuple(q.shape)}")
        x = _rows("codes", q, K, _E4M3)
        s = _rows("scales", scales, KB, torch.float32)
        M, ld, ls = x.shape[0], (K + 15) // 16 * 16, KB
        if M > MAX_ROWS:
            raise ValueError(f"codes have {M} rows, at most {MAX_ROWS} per call")
        if M > 1:
            ld, ls = x.stride(0), s.stride(0)
            if ls < KB:
                s, ls = s.contiguous(), KB
        if x.data_ptr() % 16 or ld % 16 or ld < K:
            p = _codes_like((M,), K, x.device)
            p.copy_(x)
            x, ld = p, (K + 15) // 16 * 16
        if out is None:
            out = s.new_empty((*lead, N), dtype=out_dtype)
        else:
            _out("out", out, (*lead, N), out_dtype, dev)
        if M:
            w, ws, b = self._w
            args = _LINEAR.pack(x.data_ptr(), s.data_ptr(), w, ws, b, out.data_ptr(),
                                ld, ls, self._ld, N, M, N, K, dt, dev, 0)
            rc = self._call(args, _stream(dev))
            if rc:
                _lib.check(rc)
        return out


class Fp8MoELayer:
    """A whole mixture-of-experts layer for up to 64 tokens over experts that
    are resident as e4m3 codes: router, top-k, the three products of every
    routed expert, the weighted sum and the residual.

    model: "qwen3" (softmax over all experts, top-k, renormalised if
    norm_topk_prob; silu(g) * u) or "gptoss" (top-k, softmax of those; clamped
    SwiGLU). router: bf16 [E, d] (and router_bias [E]); gate, up: (codes
    [E, f, d], scales[, bias [E, f]]); down: (codes [E, d, f], scales[, bias
    [E, d]]). d and f are multiples of 16. The logits are kept in 32 bits
    (MoEBlock rounds them to bf16 as the reference does). Weights that are
    contiguous and 16-byte aligned are used where they are; copies are made and
    waited for as Fp8Linear's."""

    def __init__(self, model, router, gate, up, down, top_k, router_bias=None, norm_topk_prob=True):
        if model not in ("qwen3", "gptoss"):
            raise ValueError(f"unknown model {model!r}")
        if router.dtype is not torch.bfloat16 or not router.is_cuda or router.dim() != 2:
            raise TypeError("router must be a two-dimensional bf16 CUDA tensor")
        self.model, self.top_k, self.norm_topk_prob = model, int(top_k), bool(norm_topk_prob)
        self.device = router.device
        E, d = router.shape
        f = gate[0].shape[-2] if gate[0].dim() == 3 else 0
        self.n_experts, self.d_model, self.d_ff = E, d, f
        if not 1 <= E <= 256:
            raise ValueError(f"{E} experts, supported are 1 to 256")
        if not 1 <= self.top_k <= min(32, E):
            raise ValueError(f"top_k must be in [1, {min(32, E)}], got {top_k}")
        for name, n in (("d_model", d), ("d_ff", f)):
            if n % 16 or not 16 <= n <= MAX_FEATURES:
                raise ValueError(f"{name} must be a multiple of 16 in [16, {MAX_FEATURES}], got {n}")
        self.router = self._aligned(router)
        self.router_bias = _bias(router_bias, (E,), self.device)
        parts = []
        for name, m, n, k in (("gate", gate, f, d), ("up", up, f, d), ("down", down, d, f)):
            codes, scales = _weight(name, m[0], m[1], 3, self.device)
            if tuple(codes.shape) != (E, n, k):
                raise ValueError(f"{name} has shape {tuple(codes.shape)}, expected {(E, n, k)}")
            parts.append((self._aligned(codes), scales, _bias(m[2] if len(m) > 2 else None, (E, n), self.device)))
        self.gate, self.up, self.down = parts
        given = [t for m in (gate, up, down) for t in (*m[:2], m[2] if len(m) > 2 else None)]
        self._captured = _wait_for_copies(self.device, (router, router_bias, *given),
                                          (self.router, self.router_bias, *(t for p in parts for t in p)))
        ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
        self._ptrs = (*(ptr(p[0]) for p in parts), *(ptr(p[1]) for p in parts), *(ptr(p[2]) for p in parts))
        self._router = (ptr(self.router), ptr(self.router_bias))
        self._model = _lib.MODEL_GPTOSS if model == "gptoss" else _lib.MODEL_QWEN3
        lib = _lib.load()
        self._call = lib.ms_moe_fp8_layer
        self._dev = self.router.get_device()
        self._tail = (self.d_model, self.d_ff, self.n_experts, self.top_k, self.norm_topk_prob, self._dev)
        self._ws = [0] * (MAX_TOKENS + 1)
        n = ctypes.c_size_t()
        for T in range(1, MAX_TOKENS + 1):
            _lib.check(lib.ms_moe_fp8_workspace(self._pack(0, 0, 0, 0, 0, T), ctypes.byref(n)))
            self._ws[T] = n.value

    @staticmethod
    def _aligned(t):
        if not t.is_contiguous():
            t = t.contiguous()
        return t.clone() if t.data_ptr() % 16 else t

    def _pack(self, x, residual, y, ws, ws_bytes, T):
        return _MOE.pack(x, *self._router, *self._ptrs, residual, y, ws, ws_bytes, self._model, T, *self._tail)

    def __call__(self, x, residual=None, out=None, stream=None):
        """x [..., d] bf16 -> y [..., d] bf16, residual (like x) added. out
        may be x or residual."""
        if stream is not None:
            return _on_stream(self._forward, stream, self.device.index, x, residual, out,
                              keep=(self.router, self.router_bias, *self.gate, *self.up, *self.down),
                              captured=self._captured)
        return self._forward(x, residual, out)

    def _forward(self, x, residual, out):
        d, dev = self.d_model, self._dev
        if x.get_device() != dev:
            raise TypeError(f"x must be on the layer's device, {self.device}")
        x2 = _rows("x", x, d, torch.bfloat16)
        if not x2.is_contiguous() or x2.data_ptr() % 16:
            x2 = self._aligned(x2)
        T = x2.shape[0]
        if T > MAX_TOKENS:
            raise ValueError(f"{T} tokens, at most {MAX_TOKENS} per call")
        rp = 0
        if residual is not None:
            r2 = self._aligned(_like("residual", residual, x, dev))
            rp = r2.data_ptr()
        if out is None:
            out = torch.empty_like(x, memory_format=torch.contiguous_format)
        else:
            _out("out", out, x.shape, torch.bfloat16, dev)
            if out.data_ptr() % 16:
                raise ValueError("out must start on a 16-byte boundary")
        if T:
            nb = self._ws[T]
            ws = x.new_empty(nb, dtype=torch.uint8)
            rc = self._call(self._pack(x2.data_ptr(), rp, out.data_ptr(), ws.data_ptr(), nb, T), _stream(dev))
            if rc:
                _lib.check(rc)
        return out
