"""RMS norm with residual and 8-bit output against its definition in 64 bits (GPU).

Tolerances. Inside, everything is f32: with u = 2^-24, the sum of squares is a tree of at most 64 roundings per value, the mean, the square root, the
quotient and two products add six: y is off by at most 70 u |y| before its one rounding to its type, eps(type) / 2. (The square root halves the
sum's share: the bound is safe.) A scale is off by as much. q: a value v = y / scale is off by (70 + 3) u |v| before it is rounded by at most half a
step: 1/2 for int8; 2^-4 |v| or half the smallest step, 2^-10, for e4m3."""
import numpy as np
import pytest
import torch

from .conftest import needs_capture

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def layers():
    from shodh_memory_amd import layers
    return layers


def half_step(t):
    return torch.finfo(t).eps / 2


def defined(x, weight, residual, eps):
    h = x.double() + (residual.double() if residual is not None else 0)
    return h, weight.double() * h / torch.sqrt(h.pow(2).mean(-1, keepdim=True) + eps)


def check_rounded(got, want, t, relative):
    """every value within its rounding and `relative` f32 noise; values below the type's normal range within its smallest step"""
    tol = want.abs() * (half_step(t) * (1 + 2 * relative) + relative) + (2.0 ** -25 if t == torch.float16 else 2.0 ** -133)
    assert ((got.double() - want).abs() <= tol).all()


def check_q(r, y, group, kind):
    dim = y.shape[-1]
    g = group or dim
    y = y.reshape(-1, dim)
    amax = torch.stack([p.abs().amax(1) for p in y.split(g, 1)], 1)
    want = amax / (127 if kind == "int8" else 448)
    assert r.scale.shape == want.shape
    assert ((r.scale.double() - want).abs() <= 73 * U * want).all()
    each = r.scale.double().repeat_interleave(g, 1)[:, :dim]
    v = torch.where(each > 0, y / each.clamp(min=1e-300), 0.0)
    q = r.q.reshape(-1, dim).to(torch.float64) if kind == "int8" else r.q.reshape(-1, dim).float().double()
    noise = 150 * U * v.abs()          # v's own error here holds the scale's as well
    tol = 0.5 + noise if kind == "int8" else torch.maximum(v.abs() * 2.0 ** -4, torch.full_like(v, 2.0 ** -10)) + noise
    assert ((q - v).abs() <= tol).all()
    assert q.abs().max() <= (127 if kind == "int8" else 448)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 7), (5, 64), (1, 384), (33, 511), (2, 512), (7, 771), (4, 1024), (300, 1025), (2, 2048), (5, 2049), (3, 4096),
                                      (2, 4099), (1, 8192), (2, 8200), (2, 16384), (1, 16391), (1, 32768)])
def test_against_the_definition(layers, rows, dim, dtype):
    t = TYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(rows * 100003 + dim)
    x = torch.randn(rows, dim, generator=g, device="cuda").to(t)
    res = (3 * torch.randn(rows, dim, generator=g, device="cuda")).to(t)
    w = (1 + 0.3 * torch.randn(dim, generator=g, device="cuda")).to(t)
    for residual, quant, group, weight in [(None, None, 0, w), (res, "int8", 0, w), (res, "e4m3", 128, w.float()), (None, "int8", 32, w), (res, "e4m3", 0, w),
                                           (None, "e4m3", 256, w.float()), (res, "int8", 64, w)]:
        r = layers.rms_norm(x, weight, eps=1e-5, residual=residual, quant=quant, group=group)
        h, y = defined(x, weight, residual, 1e-5)
        check_rounded(r.y, y, t, 70 * U)
        if residual is not None:
            check_rounded(r.sum, h, t, U)
        else:
            assert r.sum is None
        if quant:
            check_q(r, y, group, quant)
        else:
            assert r.q is None and r.scale is None


def test_in_place_and_views(layers):
    """sum over the residual, x as columns of a wider tensor at an odd place, y not asked for: the same numbers, nothing else touched"""
    g = torch.Generator(device="cuda").manual_seed(5)
    wide = torch.randn(9, 1500, generator=g, device="cuda").bfloat16()
    before = wide.clone()
    x = wide[:, 3:3 + 777]
    w = torch.ones(777, device="cuda")
    res = torch.randn(9, 777, generator=g, device="cuda").bfloat16()
    a = layers.rms_norm(x.contiguous(), w, residual=res.clone(), quant="int8")
    mine = res.clone()
    b = layers.rms_norm(x, w, residual=mine, sum_out=mine, want_y=False, quant="int8")
    assert b.sum is mine and b.y is None
    assert torch.equal(a.sum, mine) and torch.equal(a.q, b.q) and torch.equal(a.scale, b.scale)
    out = torch.full((9, 1500), 7.0, device="cuda").bfloat16()
    layers.rms_norm(x, w, residual=res, sum_out=out[:, 5:5 + 777])
    assert torch.equal(out[:, 5:5 + 777], a.sum) and (out[:, :5] == 7).all() and (out[:, 782:] == 7).all()
    assert torch.equal(wide, before)


def test_three_dimensions_and_no_rows(layers):
    x = torch.randn(2, 3, 64, device="cuda")
    w = torch.rand(64, device="cuda")
    r = layers.rms_norm(x, w, quant="e4m3", group=32)
    s = layers.rms_norm(x.view(6, 64), w, quant="e4m3", group=32)
    assert r.y.shape == x.shape and r.q.shape == x.shape and r.scale.shape == (6, 2)
    assert torch.equal(r.y.view(6, 64), s.y) and torch.equal(r.scale, s.scale) and torch.equal(r.q.view(torch.uint8).view(6, 64), s.q.view(torch.uint8))
    e = layers.rms_norm(x[:0], w, quant="int8")
    assert e.y.shape == (0, 3, 64) and e.q.numel() == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_values_whose_squares_pass_f32(layers, dtype):
    t = TYPES[dtype]
    x = torch.randn(4, 1000, device="cuda").to(t)
    x[0] *= 1e25
    x[1, 17] = 3e38
    x[2] = 0
    w = torch.ones(1000, device="cuda")
    r = layers.rms_norm(x, w, quant="int8", group=64)
    _, y = defined(x, w, None, 1e-6)
    check_rounded(r.y, y, t, 70 * U)
    assert (r.y[2] == 0).all() and (r.scale[2] == 0).all() and (r.q[2] == 0).all()
    assert float(r.y[1, 17]) == pytest.approx(1000 ** 0.5, rel=0.01)


def test_nan_and_infinity_stay_in_their_group_and_row(layers):
    x = torch.randn(3, 256, device="cuda")
    x[0, 70] = float("nan")
    x[1, 200] = float("inf")
    w = torch.ones(256, device="cuda")
    r = layers.rms_norm(x, w, quant="e4m3", group=64)
    assert torch.isnan(r.y[0]).all() and torch.isnan(r.scale[0]).all()              # the mean of a row with a NaN is one
    assert torch.isnan(r.y[1, 200]) and (r.y[1, :200] == 0).all()                    # inf / inf, and x / inf
    assert torch.isnan(r.scale[1, 3]) and (r.scale[1, :3] == 0).all()
    assert (r.q[:2].float() == 0).all()
    _, y = defined(x[2:], w, None, 1e-6)
    check_rounded(r.y[2:], y, torch.float32, 70 * U)


def test_many_rows_each_its_own(layers):
    """more rows than workgroups: every row is what it is alone"""
    x = torch.randn(70001, 40, device="cuda").half()
    w = torch.rand(40, device="cuda").half()
    r = layers.rms_norm(x, w, quant="int8")
    at = torch.tensor([0, 1, 2047, 32768, 65535, 65536, 70000], device="cuda")
    s = layers.rms_norm(x[at].contiguous(), w, quant="int8")
    assert torch.equal(r.y[at], s.y) and torch.equal(r.q[at], s.q) and torch.equal(r.scale[at], s.scale)
    _, y = defined(x, w, None, 1e-6)
    check_rounded(r.y, y, torch.float16, 70 * U)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_more_data_than_the_caches_hold(layers, dtype):
    """the form that goes past the caches: rows are what they are alone"""
    x = torch.randn(66000, 1024, device="cuda").to(TYPES[dtype])
    res, w = x.flip(0).contiguous(), torch.rand(1024, device="cuda").to(TYPES[dtype])
    r = layers.rms_norm(x, w, residual=res, quant="e4m3", group=128)
    at = torch.tensor([0, 1, 33000, 65999], device="cuda")
    s = layers.rms_norm(x[at].contiguous(), w, residual=res[at].contiguous(), quant="e4m3", group=128)
    assert torch.equal(r.y[at], s.y) and torch.equal(r.sum[at], s.sum) and torch.equal(r.scale[at], s.scale)
    assert torch.equal(r.q.view(torch.uint8)[at], s.q.view(torch.uint8))
    h, y = defined(x, w, res, 1e-6)
    check_rounded(r.y, y, TYPES[dtype], 70 * U)


def test_more_rows_than_a_launch_has_workgroups(layers):
    """70 million rows of one value: y = x / sqrt(x^2 + eps) w, the tolerance of any y"""
    x = torch.randn(70_000_001, 1, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").bfloat16()
    w = torch.full((1,), 1.5, device="cuda")
    y = layers.rms_norm(x, w, eps=1e-3).y
    for part in (slice(0, 1000), slice(33_554_000, 33_555_000), slice(67_108_000, 67_110_000), slice(69_999_000, None)):
        check_rounded(y[part], defined(x[part], w, None, 1e-3)[1], torch.bfloat16, 70 * U)


@needs_capture
def test_streams_and_graph(layers):
    x, w = torch.randn(50, 1024, device="cuda").bfloat16(), torch.rand(1024, device="cuda").bfloat16()
    res = torch.randn(50, 1024, device="cuda").bfloat16()
    want = layers.rms_norm(x, w, residual=res, quant="int8")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layers.rms_norm(x, w, residual=res, quant="int8")
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = layers.rms_norm(x, w, residual=res, quant="int8")
    for k in range(3):
        x.copy_(torch.randn(50, 1024, device="cuda"))
        want = layers.rms_norm(x, w, residual=res, quant="int8")
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held)), k


def test_refusals(layers):
    from shodh_memory_amd import ShodhError
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    for call in [lambda: layers.rms_norm(x, w[:32]), lambda: layers.rms_norm(x.double(), w), lambda: layers.rms_norm(x, w.half()), lambda: layers.rms_norm(x, w, eps=0.0),
                 lambda: layers.rms_norm(x, w, eps=float("nan")), lambda: layers.rms_norm(x, w, quant="int4"), lambda: layers.rms_norm(x, w, quant="int8", group=48),
                 lambda: layers.rms_norm(x, w, residual=x[:2]), lambda: layers.rms_norm(x, w, residual=x.half()), lambda: layers.rms_norm(x.t(), torch.ones(4, device="cuda")),
                 lambda: layers.rms_norm(x, w, want_y=False), lambda: layers.rms_norm(x, w, sum_out=x), lambda: layers.rms_norm(x[:1].expand(4, 64), w),
                 lambda: layers.rms_norm(x, w.cpu()), lambda: layers.rms_norm(torch.randn(1, 32769, device="cuda"), torch.ones(32769, device="cuda")),
                 lambda: layers.rms_norm(x, w, residual=x, sum_out=torch.empty(1, 64, device="cuda").expand(4, 64))]:
        with pytest.raises(ShodhError):
            call()
    torch.cuda.synchronize()


def test_sizes_that_32_bits_cannot_hold(layers):
    """(a group of 2^32 + 32 would be taken as 32, and scales written for it where one a row has room)"""
    from shodh_memory_amd import ShodhError
    x, w = torch.randn(4, 256, device="cuda"), torch.ones(256, device="cuda")
    for group in (2 ** 32, 2 ** 32 + 32, -32, -2 ** 32 + 64):
        with pytest.raises(ShodhError):
            layers.rms_norm(x, w, quant="int8", group=group)
    wide = torch.empty(2 ** 32 + 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ShodhError):
        layers.rms_norm(wide[None], wide)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,dim", [(300, 64), (5, 1000), (40, 4096), (3, 20000)])
def test_in_place_through_the_c_boundary(layers, dtype, rows, dim):
    """sum and y over x or the residual themselves, element for element; any other overlap is refused and leaves what was there"""
    import ctypes as C

    from shodh_memory_amd import _lib as L
    t = TYPES[dtype]
    x0, r0 = (torch.randn(rows, dim, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda").to(t) for i in (1, 2))
    w = torch.rand(dim, device="cuda").to(t)
    want = layers.rms_norm(x0, w, residual=r0)
    kind = {"f32": L.DTYPE_FP32, "bf16": L.DTYPE_BF16}[dtype]
    cfg = L.RmsNormCfg(rows, 0, 0, 0, 0, 0, dim, kind, kind, L.DTYPE_INT8, 0, 1e-6)

    def call(x, r, total, y):
        return L.lib().shodh_rms_norm_device(0, C.byref(cfg), x.data_ptr(), r.data_ptr(), w.data_ptr(), total, y, None, None, torch.cuda.current_stream().cuda_stream)
    for total_at, y_at in (("r", "x"), ("x", "r"), ("r", None), (None, "x"), (None, "r"), ("x", "new")):
        x, r, new = x0.clone(), r0.clone(), torch.empty_like(x0)
        at = {"x": x, "r": r, "new": new}
        assert call(x, r, at[total_at].data_ptr() if total_at else None, at[y_at].data_ptr() if y_at else None) == 0
        if total_at:
            assert torch.equal(at[total_at], want.sum)
        if y_at:
            assert torch.equal(at[y_at], want.y)
    x, r = x0.clone(), r0.clone()
    one = x.element_size()
    assert call(x, r, x.data_ptr(), x.data_ptr()) == L.ERR_INVALID and call(x, r, r.data_ptr() + one, None) == L.ERR_INVALID and call(x, r, None, x.data_ptr() + dim * one) == L.ERR_INVALID
    torch.cuda.synchronize()
    assert torch.equal(x, x0) and torch.equal(r, r0)
