"""Layer operators of a text tower on torch device tensors, over the C ABI (include/shodh_hip.h, "layer operators"): RMS norm with residual and 8-bit
output, dense layers on 4-bit weights, attention with a sliding window and always-visible first tokens. They run on the tensors' device, on its
current stream unless `stream` names another (a raw hipStream_t, made the current one for the call: new tensors are that stream's), and can be captured
into a graph. They are for inference: results carry no gradients, and inputs that require one are refused while torch records (torch.no_grad() takes them).
Nothing here computes on the host."""
import collections
import ctypes as C
import functools

import torch

from . import _lib as L

_DTYPES = {torch.float32: L.DTYPE_FP32, torch.bfloat16: L.DTYPE_BF16, torch.float16: L.DTYPE_FP16}
_QUANT = {"int8": (L.DTYPE_INT8, torch.int8), "e4m3": (L.DTYPE_E4M3, torch.float8_e4m3fn)}

RmsNorm = collections.namedtuple("RmsNorm", "y q scale sum")


def _refuse(msg, code=L.ERR_INVALID):
    raise L.ShodhError(code, msg)


def _u32(code=L.ERR_UNSUPPORTED, **sizes):
    """sizes that the C boundary takes in 32 bits (ctypes would cut them off without a word)"""
    for name, n in sizes.items():
        if not 0 <= n < 2 ** 32:
            _refuse("%s %d is no 32-bit number" % (name, n), code)


def _gradient():
    if torch.is_grad_enabled():
        _refuse("an input requires a gradient, which a layer operator does not give: call it under torch.no_grad()", L.ERR_UNSUPPORTED)


def _dtype(t, name):
    d = _DTYPES.get(t.dtype)
    if d is None:
        _refuse("%s is %s: fp32, bf16 or fp16 is taken" % (name, t.dtype))
    return d


def _on(t, device, name):
    if t.device != device:
        _refuse("%s is on %s, not on %s" % (name, t.device, device))


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)         # (0.1 us; the Stream object of the line below takes 2 us to make)


def _stream(device):
    return _raw_stream(device.index) if _raw_stream is not None else torch.cuda.current_stream(device).cuda_stream


def _current(stream, device):
    """`stream` as the current one for a call"""
    if device.type != "cuda":
        _refuse("a stream for tensors on %s" % device)
    return torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device))


def _like(t, dtype=None):
    """a contiguous tensor of t's shape (empty_like takes 1.2 us, new_empty 1.8)"""
    return torch.empty_like(t, dtype=dtype) if t.is_contiguous() else t.new_empty(t.shape, dtype=dtype)


def _new(rows, cols, dtype, device):
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)


def _matrix(t, name):
    """(rows, columns, row stride) of [..., columns] with neighbouring elements next to each other: a view of rows at one distance."""
    if t.dim() == 2:
        rows, cols = t.shape
        step, one = t.stride()
        if cols > 1 and one != 1:
            _refuse("%s: the last dimension has to be contiguous" % name)
        if rows > 1:
            if step == 0:
                _refuse("%s: rows at distance 0 (an expanded tensor)" % name)
            return rows, cols, step
        return rows, cols, cols
    if t.dim() == 0:
        _refuse("%s has no dimension" % name)
    cols = t.shape[-1]
    rows = t.numel() // cols if cols else 0
    if not t.is_contiguous():
        _refuse("%s: more than two dimensions have to be contiguous" % name)
    return rows, cols, cols


def rms_norm(x, weight, eps=1e-6, residual=None, want_y=True, quant=None, group=0, sum_out=None, stream=None):
    """h = x + residual; y = h / sqrt(mean(h^2) + eps) * weight over the last dimension (shodh_rms_norm_device).
    quant "int8" / "e4m3": the row in 8 bits, with a scale per `group` values (0: per row; 32, 64, 128, 256): y ~ q * scale.
    -> RmsNorm(y, q, scale, sum): what was not asked for is None; sum (with a residual) = h in x's type, written to `sum_out` (it may be
    `residual` itself: in place) or a new tensor; scale f32 [rows, groups]."""
    device = x.device
    if stream is not None:
        with _current(stream, device):
            return rms_norm(x, weight, eps, residual, want_y, quant, group, sum_out)
    if device.type != "cuda":
        _refuse("x is on %s: there is no CPU fallback" % device, L.ERR_DEVICE)
    if x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad) or (sum_out is not None and sum_out.requires_grad):
        _gradient()
    dt = _dtype(x, "x")
    rows, dim, xs = _matrix(x, "x")
    if dim >= 2 ** 32 or not 0 <= group < 2 ** 32:
        _u32(dim=dim, group=group)
    if weight.dim() != 1 or weight.shape[0] != dim or (dim > 1 and weight.stride(0) != 1):
        _refuse("weight has to be contiguous [%d]" % dim, L.ERR_DIM)
    _on(weight, device, "weight")
    wd = _dtype(weight, "weight")
    rs = ss = 0
    total = None
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            _refuse("residual has to be of x's shape and type", L.ERR_DIM)
        _on(residual, device, "residual")
        rs = _matrix(residual, "residual")[2]
        if sum_out is None:
            total = _like(x)
        else:
            total = sum_out
            if total.shape != x.shape or total.dtype != x.dtype:
                _refuse("sum_out has to be of x's shape and type", L.ERR_DIM)
            _on(total, device, "sum_out")
            ss = _matrix(total, "sum_out")[2]
    elif sum_out is not None:
        _refuse("sum_out without a residual")
    y = _like(x) if want_y else None
    q = scale = None
    qd = L.DTYPE_INT8
    if quant is not None:
        if quant not in _QUANT:
            _refuse("quant %r is neither 'int8' nor 'e4m3'" % (quant,))
        qd, qt = _QUANT[quant]
        q = _like(x, qt)
        scale = _new(rows, -(-dim // group) if group else 1, torch.float32, device)
    if rows == 0:
        return RmsNorm(y, q, scale, total)
    cfg = L.RmsNormCfg(rows, xs, rs, ss, 0, 0, dim, dt, wd, qd, group, eps)
    L.check(L.lib().shodh_rms_norm_device(device.index, C.byref(cfg), x.data_ptr(), residual.data_ptr() if residual is not None else None, weight.data_ptr(),
                                          total.data_ptr() if total is not None else None, y.data_ptr() if want_y else None,
                                          q.data_ptr() if q is not None else None, scale.data_ptr() if q is not None else None, _stream(device)))
    return RmsNorm(y, q, scale, total)


class W4Weight:
    """A dense layer's weights in 4 bits with group scales, laid out on the device once (shodh_w4_weight). The handle is read-only: any number of
    threads and streams may use it. It has to outlive the captured graphs that do. Made from device tensors it cannot be while their stream is captured."""

    def __init__(self, handle, device):
        self._h, self.device = handle, device
        n, k, g, b = C.c_uint32(), C.c_uint32(), C.c_uint32(), C.c_uint64()
        L.check(L.lib().shodh_w4_weight_shape(handle, C.byref(n), C.byref(k), C.byref(g), C.byref(b)))
        self.n, self.k, self.group, self.nbytes = n.value, k.value, g.value, b.value

    @staticmethod
    def _scale_dtype(scale_dtype):
        d = {torch.float16: L.DTYPE_FP16, torch.bfloat16: L.DTYPE_BF16}.get(scale_dtype)
        if d is None:
            _refuse("scales are kept in fp16 or bf16")
        return d

    @classmethod
    def quantize(cls, w, group=128, zeros=False, scale_dtype=torch.float16, device=0):
        """f32 weights [N, K] (host) rounded to 4 bits by the library."""
        w = torch.as_tensor(w, dtype=torch.float32, device="cpu").contiguous()
        if w.dim() != 2:
            _refuse("the weight has to be [N, K]", L.ERR_DIM)
        _u32(outputs=w.shape[0], inputs=w.shape[1], group=group)
        h = C.c_void_p()
        L.check(L.lib().shodh_w4_weight_quantize(int(device), w.data_ptr(), w.shape[0], w.shape[1], group, int(bool(zeros)), cls._scale_dtype(scale_dtype), C.byref(h)))
        return cls(h, torch.device("cuda", int(device)))

    @classmethod
    def from_quantized(cls, q, scale, zeros=None, k=None, group=128, scale_dtype=None, device=0):
        """q uint8 [N, ceil(K / 2)] (two inputs a byte, the even one in the low bits), scale [N, ceil(K / group)], zeros uint8 of scale's shape or None (8):
        device tensors (their device is used) or host tensors / arrays (`device`). Scales are kept as they are in fp16 and bf16, others in fp16 unless
        scale_dtype says otherwise; those that the type cannot hold to half a step are refused."""
        q, scale = torch.as_tensor(q), torch.as_tensor(scale)
        zeros = None if zeros is None else torch.as_tensor(zeros)
        if q.dim() != 2 or q.dtype != torch.uint8:
            _refuse("q has to be uint8 [N, ceil(K / 2)]")
        n = q.shape[0]
        k = 2 * q.shape[1] if k is None else int(k)
        if q.shape[1] != (k + 1) // 2:
            _refuse("q has %d bytes a row, %d inputs need %d" % (q.shape[1], k, (k + 1) // 2), L.ERR_DIM)
        if group not in (32, 64, 128):
            _refuse("group %r is none of 32, 64, 128" % (group,), L.ERR_UNSUPPORTED)
        _u32(outputs=n, inputs=k)
        shape = (n, -(-k // group))
        if tuple(scale.shape) != shape or (zeros is not None and (tuple(zeros.shape) != shape or zeros.dtype != torch.uint8)):
            _refuse("scale (and uint8 zeros) have to be %s" % (shape,), L.ERR_DIM)
        sd = cls._scale_dtype(scale_dtype or (torch.bfloat16 if scale.dtype == torch.bfloat16 else torch.float16))
        for t, name in ((scale, "scale"), (zeros, "zeros")):
            if t is not None:
                _on(t, q.device, name)
        q, scale = q.contiguous(), scale.float().contiguous()
        zeros = None if zeros is None else zeros.contiguous()
        h, zp = C.c_void_p(), zeros.data_ptr() if zeros is not None else None
        if q.device.type == "cuda":
            L.check(L.lib().shodh_w4_weight_create_device(q.device.index, q.data_ptr(), scale.data_ptr(), zp, n, k, group, sd, _stream(q.device), C.byref(h)))
            return cls(h, q.device)
        L.check(L.lib().shodh_w4_weight_create(int(device), q.data_ptr(), scale.data_ptr(), zp, n, k, group, sd, C.byref(h)))
        return cls(h, torch.device("cuda", int(device)))

    def dequantize(self):
        """the weights as the products see them: f32 [N, K] (host)"""
        out = torch.empty((self.n, self.k), dtype=torch.float32)
        L.check(L.lib().shodh_w4_weight_dequantize(self._h, out.data_ptr()))
        return out

    def dense(self, x, x_scale=None, bias=None, out_dtype=None, out=None, stream=None):
        """x [..., K] -> [..., N]: x @ W^T (* x_scale per row) + bias. x fp32, bf16, fp16, or int8 with x_scale f32 [rows] (or [rows, 1]);
        the result is of x's type (bf16 for int8 rows) unless out_dtype or `out` says otherwise. A row that holds a NaN or an infinity gives NaN in all its
        outputs (16-bit rows with an f32 result: what the formula gives)."""
        if self._h is None:
            _refuse("the weight is closed", L.ERR_STATE)
        if stream is not None:
            with _current(stream, self.device):
                return self.dense(x, x_scale, bias, out_dtype, out)
        if x.requires_grad or (bias is not None and bias.requires_grad) or (x_scale is not None and x_scale.requires_grad) or (out is not None and out.requires_grad):
            _gradient()
        rows, k, xs = _matrix(x, "x")
        if k != self.k:
            _refuse("x has %d columns, the weight %d inputs" % (k, self.k), L.ERR_DIM)
        if rows >= 2 ** 32:
            _u32(rows=rows)
        _on(x, self.device, "x")
        sp = bp = None
        if x.dtype == torch.int8:
            xd = L.DTYPE_INT8
            if x_scale is None or x_scale.dtype != torch.float32 or x_scale.numel() != rows or not x_scale.is_contiguous():
                _refuse("int8 rows come with x_scale, contiguous f32 [%d]" % rows)
            _on(x_scale, self.device, "x_scale")
            sp = x_scale.data_ptr()
        else:
            xd = _dtype(x, "x")
            if x_scale is not None:
                _refuse("x_scale belongs to int8 rows")
        if bias is not None:
            if bias.dtype != torch.float32 or bias.shape != (self.n,) or not bias.is_contiguous():
                _refuse("bias has to be contiguous f32 [%d]" % self.n, L.ERR_DIM)
            _on(bias, self.device, "bias")
            bp = bias.data_ptr()
        if out is None:
            dtype = out_dtype or (torch.bfloat16 if xd == L.DTYPE_INT8 else x.dtype)
            out = _new(rows, self.n, dtype, self.device) if x.dim() == 2 else x.new_empty(x.shape[:-1] + (self.n,), dtype=dtype)
            os_ = self.n
        else:
            shape = x.shape[:-1] + (self.n,)
            if out.shape != shape or (out_dtype is not None and out.dtype != out_dtype):
                _refuse("out has to be %s" % (tuple(shape),), L.ERR_DIM)
            _on(out, self.device, "out")
            os_ = _matrix(out, "out")[2]
        if rows == 0:
            return out
        L.check(L.lib().shodh_w4_dense_device(self._h, x.data_ptr(), xd, xs, sp, rows, bp, out.data_ptr(), _dtype(out, "out"), os_,
                                              _stream(self.device)))
        return out

    def close(self):
        """Frees the device copy (the runtime waits for what was started on it). Captured graphs that hold a product of this weight may not run afterwards."""
        if self._h is not None:
            h, self._h = self._h, None
            L.lib().shodh_w4_weight_destroy(h)

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _heads(t, name, device, dtype):
    """(token stride, head stride) of [tokens, heads, head_dim] with neighbouring features next to each other"""
    if t.dim() != 3 or t.dtype != dtype or t.device != device:
        _refuse("%s has to be [tokens, heads, head_dim], %s, on %s (got %s, %s, %s)" % (name, dtype, device, tuple(t.shape), t.dtype, t.device))
    n, h, d = t.shape
    s, hs, one = t.stride()
    if (d > 1 and one != 1) or (n > 1 and s == 0) or (h > 1 and hs == 0):
        _refuse("%s: the last dimension has to be contiguous, no dimension expanded" % name)
    return s if n > 1 else max(s, h * d), hs if h > 1 else d


def _descriptor(t, name, device, dtype, n):
    if t.dtype != dtype or t.device != device or t.shape != (n,) or not t.is_contiguous():
        _refuse("%s has to be contiguous %s [%d] on %s" % (name, dtype, n, device))
    return t.data_ptr()


@functools.lru_cache(maxsize=1024)
def _attention_workspace(device, n, kn, dt, heads, kv_heads, dim, seqs, sinks, left, right):
    """shodh_window_attention_workspace: a function of sizes alone"""
    cfg = L.AttentionCfg(n, kn, 0, 0, 0, 0, 0, 0, 0, 0, dt, heads, kv_heads, dim, seqs, sinks, left, right, 0.0, 0)
    need = C.c_uint64()
    L.check(L.lib().shodh_window_attention_workspace(device, C.byref(cfg), C.byref(need)))
    return need.value


def window_attention(q, k, v, cu, left=-1, right=-1, sinks=0, kv_start=None, kv_len=None, scale=None, return_lse=False, out=None, stream=None):
    """Attention over a sliding window plus the first `sinks` tokens of each sequence (shodh_window_attention_device).
    q [tokens, heads, head_dim] of all sequences one after another, sequence b = cu[b] .. cu[b + 1] (int32, device). k, v [kv_tokens, kv_heads, head_dim]:
    the same tokens, or with kv_start (int64) and kv_len (int32) a cache in which sequence b has the keys kv_start[b] .. + kv_len[b], its queries
    being the last ones. Query i of Lq stands at p = i + Lk - Lq and sees key j iff j <= p + right and (j >= p - left or j < sinks); a negative
    bound is none; causal: right=0. bf16 or fp16, head_dim a multiple of 8 up to 128, any strides of tokens and heads.
    -> out like q (and with return_lse the log of the sum of exponentials, f32 [tokens, heads]); tokens behind cu[-1] are left as they were."""
    device = q.device
    if stream is not None:
        with _current(stream, device):
            return window_attention(q, k, v, cu, left, right, sinks, kv_start, kv_len, scale, return_lse, out)
    if device.type != "cuda":
        _refuse("q is on %s: there is no CPU fallback" % device, L.ERR_DEVICE)
    if q.requires_grad or k.requires_grad or v.requires_grad or (out is not None and out.requires_grad):
        _gradient()
    dt = _dtype(q, "q")
    qs, qh = _heads(q, "q", device, q.dtype)
    ks, kh = _heads(k, "k", device, q.dtype)
    vs, vh = _heads(v, "v", device, q.dtype)
    n, heads, dim = q.shape
    kn, kv_heads, kd = k.shape
    if v.shape != k.shape or kd != dim:
        _refuse("k %s and v %s have to be [kv_tokens, kv_heads, %d] alike" % (tuple(k.shape), tuple(v.shape), dim), L.ERR_DIM)
    if cu.dim() != 1 or cu.shape[0] < 1:
        _refuse("cu has to be int32 [sequences + 1]")
    seqs = cu.shape[0] - 1
    cup = _descriptor(cu, "cu", device, torch.int32, seqs + 1)
    if (kv_start is None) != (kv_len is None):
        _refuse("kv_start and kv_len come together")
    sp = lp = None
    if kv_start is not None:
        sp, lp = _descriptor(kv_start, "kv_start", device, torch.int64, seqs), _descriptor(kv_len, "kv_len", device, torch.int32, seqs)
    if out is None:
        out = _like(q)
        os_, oh = heads * dim, dim
    else:
        if out.shape != q.shape:
            _refuse("out has to be of q's shape", L.ERR_DIM)
        os_, oh = _heads(out, "out", device, q.dtype)
    if not 0 <= sinks < 2 ** 31 or not -2 ** 31 <= left < 2 ** 31 or not -2 ** 31 <= right < 2 ** 31:
        _refuse("left, right and sinks are 32-bit numbers, sinks 0 or more")
    if heads >= 2 ** 32 or kv_heads >= 2 ** 32 or dim >= 2 ** 32 or seqs >= 2 ** 32:
        _u32(heads=heads, kv_heads=kv_heads, head_dim=dim, sequences=seqs)
    if scale is not None and not C.c_float(scale).value != 0:
        _refuse("scale 0 in f32 (or no number)")
    lse = _new(n, heads, torch.float32, device) if return_lse else None
    if n and seqs:
        cfg = L.AttentionCfg(n, kn, qs, qh, ks, kh, vs, vh, os_, oh, dt, heads, kv_heads, dim, seqs, sinks, left, right, scale or 0.0, 0)
        need = _attention_workspace(device.index, n, kn, dt, heads, kv_heads, dim, seqs, sinks, left, right)
        work = q.new_empty(need, dtype=torch.uint8) if need else None
        L.check(L.lib().shodh_window_attention_device(device.index, C.byref(cfg), q.data_ptr(), k.data_ptr(), v.data_ptr(), cup, sp, lp, out.data_ptr(),
                                                      lse.data_ptr() if return_lse else None, work.data_ptr() if work is not None else None, need,
                                                      _stream(device)))
    return (out, lse) if return_lse else out
