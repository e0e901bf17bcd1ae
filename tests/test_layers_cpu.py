"""The layer operators' checks of their arguments, through the C ABI and the Python functions, without a device: a call that cannot be right is an error
before anything is launched. (The pointers are never followed.)"""
import ctypes as C

import pytest
import torch

P = 4096          # some address, a multiple of every element size


@pytest.fixture(scope="module")
def L():
    from shodh_memory_amd import _lib
    return _lib


def rms(L, x=P, residual=None, weight=P, total=None, y=P, q=None, scale=None, **kw):
    cfg = L.RmsNormCfg()
    L.lib().shodh_rms_norm_cfg_default(C.byref(cfg))
    cfg.rows, cfg.dim = 4, 64
    for k, v in kw.items():
        setattr(cfg, k, v)
    return L.lib().shodh_rms_norm_device(0, C.byref(cfg), x, residual, weight, total, y, q, scale, None)


def test_rms_norm_defaults(L):
    cfg = L.RmsNormCfg()
    L.lib().shodh_rms_norm_cfg_default(C.byref(cfg))
    assert (cfg.dtype, cfg.weight_dtype, cfg.q_dtype, cfg.q_group, cfg.rows, cfg.dim) == (L.DTYPE_BF16, L.DTYPE_BF16, L.DTYPE_INT8, 0, 0, 0)
    assert abs(cfg.eps - 1e-6) < 1e-12 and C.sizeof(cfg) == 72


@pytest.mark.parametrize("kw,code", [
    (dict(dim=0), -1), (dict(dim=32769), -8), (dict(dtype=2), -1), (dict(dtype=4), -1), (dict(dtype=9), -1), (dict(weight_dtype=3), -1), (dict(eps=0.0), -1), (dict(eps=-1.0), -1),
    (dict(eps=float("nan")), -1), (dict(eps=float("inf")), -1), (dict(q=P), -1), (dict(scale=P), -1), (dict(y=None), -1), (dict(total=P), -1), (dict(weight=None), -1), (dict(x=None), -1),
    (dict(q=P, scale=P, q_dtype=0), -1), (dict(q=P, scale=P, q_dtype=1), -1), (dict(q=P, scale=P, q_group=16), -8), (dict(q=P, scale=P, q_group=96), -8), (dict(y_stride=63), -1),
    (dict(q=P, scale=P, q_stride=10), -1), (dict(residual=P, total=P, sum_stride=63), -1), (dict(x=P + 1), -1), (dict(y=P + 1), -1), (dict(q=P, scale=P + 2), -1),
    (dict(weight=P + 2, weight_dtype=0), -1)])
def test_rms_norm_refuses(L, kw, code):
    assert rms(L, **kw) == code and L.last_error()


def test_rms_norm_of_no_rows_needs_no_device(L):
    assert rms(L, rows=0, x=None, y=None) == 0


def w4_create(L, q=P, scale=P, n=16, k=64, group=32, dt=3, out=True):
    h = C.c_void_p(1234)
    rc = L.lib().shodh_w4_weight_create(0, q, scale, None, n, k, group, dt, C.byref(h) if out else None)
    return rc, h.value


@pytest.mark.parametrize("kw,code", [(dict(q=None), -1), (dict(scale=None), -1), (dict(n=0), -1), (dict(k=0), -1), (dict(group=16), -8), (dict(group=0), -8), (dict(group=256), -8), (dict(dt=0), -1),
                                     (dict(dt=2), -1), (dict(n=(1 << 20)), -1), (dict(k=(1 << 24) + 1), -1)])
def test_w4_weight_refuses(L, kw, code):
    rc, h = w4_create(L, **kw)
    assert rc == code and h is None and L.last_error()


def test_w4_null_handles(L):
    assert w4_create(L, out=False)[0] == -1
    assert L.lib().shodh_w4_dense_device(None, P, 1, 0, None, 1, None, P, 1, 0, None) == -1
    assert L.lib().shodh_w4_weight_dequantize(None, P) == -1
    assert L.lib().shodh_w4_weight_shape(None, None, None, None, None) == -1
    assert L.lib().shodh_w4_weight_quantize(0, None, 16, 64, 32, 0, 3, C.byref(C.c_void_p())) == -1
    L.lib().shodh_w4_weight_destroy(None)


def test_python_functions_take_device_tensors_only(L):
    from shodh_memory_amd import ShodhError, layers
    x, w = torch.randn(2, 64), torch.ones(64)
    with pytest.raises(ShodhError):
        layers.rms_norm(x, w)
    with pytest.raises(ShodhError):
        layers.W4Weight.from_quantized(torch.zeros(4, 16, dtype=torch.int8), torch.ones(4, 1))
    with pytest.raises(ShodhError):
        layers.W4Weight.from_quantized(torch.zeros(4, 16, dtype=torch.uint8), torch.ones(4, 2), group=32)
    if not torch.cuda.is_available():
        with pytest.raises(ShodhError) as e:
            layers.W4Weight.from_quantized(torch.zeros(4, 16, dtype=torch.uint8), torch.ones(4, 1), group=32)
        assert e.value.code == L.ERR_DEVICE and "no CPU fallback" in str(e.value)


def attn(L, q=P, k=P, v=P, cu=P, start=None, length=None, out=P, lse=None, work=None, nwork=0, **kw):
    cfg = L.AttentionCfg()
    L.lib().shodh_attention_cfg_default(C.byref(cfg))
    cfg.q_tokens = cfg.kv_tokens = 8
    cfg.heads, cfg.kv_heads, cfg.head_dim, cfg.seqs = 4, 2, 64, 1
    for name, value in kw.items():
        setattr(cfg, name, value)
    return L.lib().shodh_window_attention_device(0, C.byref(cfg), q, k, v, cu, start, length, out, lse, work, nwork, None)


def test_attention_defaults(L):
    cfg = L.AttentionCfg()
    L.lib().shodh_attention_cfg_default(C.byref(cfg))
    assert (cfg.dtype, cfg.left, cfg.right, cfg.sinks, cfg.scale, cfg.heads) == (L.DTYPE_BF16, -1, -1, 0, 0.0, 0) and C.sizeof(cfg) == 120


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=0), -8), (dict(dtype=2), -8), (dict(heads=0), -1), (dict(kv_heads=0), -1), (dict(heads=5), -1), (dict(head_dim=0), -8), (dict(head_dim=60), -8), (dict(head_dim=136), -8),
    (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(q_tokens=1 << 31), -8), (dict(kv_tokens=(1 << 40) + 1), -8), (dict(sinks=1 << 31), -8), (dict(seqs=1 << 30), -8),
    (dict(heads=65536), -8), (dict(q=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(cu=None), -1), (dict(out=None), -1), (dict(start=P), -1), (dict(length=P), -1),
    (dict(kv_tokens=9), -2), (dict(out_stride=63), -2), (dict(out_head_stride=8), -2), (dict(out_stride=64), -2), (dict(q=P + 1), -1), (dict(out=P + 1), -1), (dict(cu=P + 2), -1),
    (dict(lse=P + 2), -1), (dict(work=P + 8), -1), (dict(start=P + 4, length=P), -1)])
def test_attention_refuses(L, kw, code):
    assert attn(L, **kw) == code and L.last_error()


@pytest.mark.parametrize("kw", [dict(scale=2.5e38), dict(scale=-2.5e38), dict(q_tokens=(1 << 31) - 100, heads=1, kv_heads=1)])
def test_attention_refuses_what_f32_and_places_cannot_hold(L, kw):
    assert attn(L, **kw) in (-1, -8) and L.last_error()


def test_attention_of_nothing_needs_no_device(L):
    assert attn(L, seqs=0, cu=None) == 0 and attn(L, q_tokens=0, kv_tokens=0, q=None, k=None, v=None, out=None) == 0
    n = C.c_uint64(7)
    assert L.lib().shodh_window_attention_workspace(0, None, C.byref(n)) == -1 and n.value == 0
    assert L.lib().shodh_window_attention_workspace(0, C.byref(L.AttentionCfg()), None) == -1
