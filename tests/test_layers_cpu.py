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


def workspace(L, **kw):
    cfg = L.AttentionCfg()
    L.lib().shodh_attention_cfg_default(C.byref(cfg))
    for name, value in kw.items():
        setattr(cfg, name, value)
    n = C.c_uint64()
    return L.lib().shodh_window_attention_workspace(0, C.byref(cfg), C.byref(n)), n.value


@pytest.mark.parametrize("texts,tokens,heads,kv_heads,dim,left,right", [
    (1024, 20, 32, 32, 128, -1, -1), (10000, 30, 12, 12, 32, -1, -1), (10000, 30, 32, 32, 128, -1, -1), (10000, 30, 32, 32, 128, 4095, 0), (4096, 8, 32, 8, 128, -1, 0),
    (100000, 12, 32, 8, 128, -1, -1), (20000, 31, 12, 12, 64, -1, -1)])
def test_attention_workspace_of_many_short_texts(L, texts, tokens, heads, kv_heads, dim, left, right):
    """parts for what fills the card (8 rounds of at most 4 workgroups a CU, 32 rows each), not for what the longest sequence could be in all rows"""
    n = texts * tokens
    rc, need = workspace(L, q_tokens=n, kv_tokens=n, seqs=texts, heads=heads, kv_heads=kv_heads, head_dim=dim, left=left, right=right)
    resident = 256 * (2 if dim == 128 else 4)
    assert rc == 0 and need <= 16 + (8 * resident * 32 + 2 * kv_heads) * ((dim + 2) * 4 + 8)


@pytest.mark.parametrize("tokens,keys,heads,kv_heads,seqs", [(900, 32768, 32, 8, 1), (4000, 4000, 8, 1, 1), (256, 256 * 32768, 32, 8, 256), (5, 1 << 20, 64, 8, 1)])
def test_attention_workspace_of_prompts_and_caches(L, tokens, keys, heads, kv_heads, seqs):
    rc, need = workspace(L, q_tokens=tokens, kv_tokens=keys, seqs=seqs, heads=heads, kv_heads=kv_heads, head_dim=128, right=0)
    assert rc == 0 and need <= 16 + (8 * 512 * 32 + 2 * kv_heads) * (130 * 4 + 8)
    if tokens < 100:          # (few rows: no more than every row's parts take)
        assert need <= 16 + tokens * heads * 64 * (130 * 4 + 8)


@pytest.mark.parametrize("kw", [dict(q_tokens=1 << 21, kv_tokens=1 << 21, seqs=1 << 18, heads=32, kv_heads=8, head_dim=64), dict(q_tokens=(1 << 26), kv_tokens=(1 << 26), seqs=1, heads=8, kv_heads=8, head_dim=8),
                                dict(q_tokens=1 << 25, kv_tokens=1 << 25, seqs=1 << 20, heads=64, kv_heads=64, head_dim=128)])
def test_attention_workspace_is_given_for_calls_that_are_taken(L, kw):
    """the question and the call have the same limits (no device here: a call that is taken ends at that)"""
    if torch.cuda.is_available():
        pytest.skip("pointers of no memory")
    rc, need = workspace(L, **kw)
    got = attn(L, work=1 << 48 if need else None, nwork=need, k=1 << 45, v=1 << 46, out=1 << 47, **kw)
    assert (rc, got) in ((0, L.ERR_DEVICE), (-8, -8))


X = 1 << 30          # (64 values of 2 bytes x 4 rows are 512 bytes)


@pytest.mark.parametrize("taken,kw", [
    (False, dict(y=X + 2)), (False, dict(y=X - 2)), (False, dict(y=X + 510)), (True, dict(y=X + 512)), (True, dict(y=X - 512)), (True, dict(y=X)), (False, dict(y=X, y_stride=65)), (False, dict(y=X, x_stride=70)),
    (True, dict(y=X, x_stride=70, y_stride=70)), (True, dict(y=X + 128, x_stride=128, y_stride=128)), (False, dict(y=X + 126, x_stride=128, y_stride=128)), (False, dict(y=X + 130, x_stride=128, y_stride=128)),
    (True, dict(y=X - 128, x_stride=128, y_stride=128)), (False, dict(y=X - 130, x_stride=128, y_stride=128)), (False, dict(y=X + 128, x_stride=128, y_stride=127)),
    (True, dict(residual=2 * X, total=2 * X)), (True, dict(residual=2 * X, total=X)), (False, dict(residual=2 * X, total=2 * X + 2)), (False, dict(residual=2 * X, total=2 * X + 128)),
    (True, dict(residual=2 * X, total=2 * X, y=X)), (True, dict(residual=2 * X, total=X, y=2 * X)), (False, dict(residual=2 * X, total=X, y=X)), (False, dict(residual=2 * X, total=4 * X, y=4 * X + 256)),
    (False, dict(y=None, q=X, scale=4 * X)), (False, dict(y=None, q=X + 511, scale=4 * X)), (True, dict(y=None, q=X + 512, scale=4 * X)), (False, dict(y=None, q=4 * X, scale=4 * X + 252)), (False, dict(y=None, q=4 * X, scale=X + 4)),
    (False, dict(y=None, q=4 * X, scale=8 * X, weight=8 * X + 8)), (True, dict(y=None, q=4 * X, scale=4 * X + 256, q_group=32)), (False, dict(y=3 * X + 64, weight=3 * X)), (False, dict(rows=1, y=X + 2)), (True, dict(rows=1, y=X + 128))])
def test_rms_norm_outputs_that_overlap(L, taken, kw):
    if torch.cuda.is_available():
        pytest.skip("pointers of no memory")
    kw = dict(dict(x=X, weight=3 * X, y=5 * X), **kw)
    assert rms(L, **kw) == (L.ERR_DEVICE if taken else -1) and ("overlap" in L.last_error()) == (not taken)


# q|k|v of 8 tokens side by side: 4 + 2 + 2 heads of 64 values, 1024 bytes a token
QKV = dict(q=X, k=X + 512, v=X + 768, q_stride=512, k_stride=512, v_stride=512)


@pytest.mark.parametrize("taken,kw", [
    (True, dict(out=2 * X)), (True, dict(QKV, out=X, out_stride=512)), (False, dict(QKV, out=X)), (False, dict(QKV, out=X + 512, out_stride=512)), (False, dict(QKV, out=X + 256, out_stride=512)), (False, dict(QKV, out=X + 2, out_stride=512)),
    (True, dict(q=X, k=X + 512, v=X + 768, q_stride=1024, k_stride=1024, v_stride=1024, out=X + 1024, out_stride=1024)), (False, dict(q=X, k=X + 512, v=X + 768, q_stride=1024, k_stride=1024, v_stride=1024, out=X + 1022, out_stride=1024)),
    (True, dict(q=X, k=X + 4096, v=X + 6144, out=X)), (False, dict(q=X, k=X + 4096, v=X + 6144, out=X + 128)), (False, dict(out=2 * X, lse=2 * X + 4092)), (True, dict(out=2 * X, lse=2 * X + 4096)), (False, dict(out=2 * X, lse=X)),
    (False, dict(out=2 * X, lse=3 * X, cu=3 * X + 4)), (False, dict(out=2 * X, cu=2 * X + 4)), (False, dict(out=2 * X, start=2 * X + 8, length=P)),
    # head by head: q, k, v and out of a head one after another, and each other head's place in between
    (True, dict(kv_heads=4, q=X, k=X + 1024, v=X + 2048, out=X + 2048 + 1024, q_stride=64, k_stride=64, v_stride=64, out_stride=64, q_head_stride=2048, k_head_stride=2048, v_head_stride=2048, out_head_stride=2048)),
    (False, dict(kv_heads=4, q=X, k=X + 1024, v=X + 2048, out=X + 2048 + 1022, q_stride=64, k_stride=64, v_stride=64, out_stride=64, q_head_stride=2048, k_head_stride=2048, v_head_stride=2048, out_head_stride=2048))])
def test_attention_outputs_that_overlap(L, taken, kw):
    if torch.cuda.is_available():
        pytest.skip("pointers of no memory")
    kw = dict(dict(q=X, k=X + 8192, v=X + 16384, cu=7 * X), **kw)
    assert attn(L, **kw) == (L.ERR_DEVICE if taken else -1) and ("overlap" in L.last_error()) == (not taken)
