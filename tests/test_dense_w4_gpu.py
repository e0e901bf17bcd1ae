"""Dense layers on 4-bit weights against their definition in 64 bits (GPU).

Tolerance. A group's sum is formed as sum x (16 + q) - (16 + z) sum x. With u = 2^-23 (one unit in the last place per addition: the matrix unit's own order and
rounding of its sums is not specified), a sum of G products of bf16 / fp16 / split f32 numbers is off by at most G u sum |x| (16 + q), sum |x|
likewise, and the steps behind it (the difference, the scale, the sum over K / G groups, at most 8 waves, bias) by one u each of what has been added up:
    |y - exact| <= (G + K / G + 16) u T + eps(type) / 2 |exact|,   T = sum_k |x| (32 + q + z) s  (+ |bias|)
f32 rows: three parts of x, three sums each: 3 G. int8 rows: the groups' sums are exact, T = sum |x| |q - z| s and no G."""
import numpy as np
import pytest
import torch

from .conftest import needs_capture

pytestmark = pytest.mark.gpu
U = 2.0 ** -23
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def layers():
    from shodh_memory_amd import layers
    return layers


def make(n, k, group, zeros, seed, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    ng = -(-k // group)
    scale = (0.01 + 0.02 * torch.rand(n, ng, generator=g)).half().float()
    z = torch.randint(0, 16, (n, ng), generator=g, dtype=torch.uint8) if zeros else None
    p = torch.nn.functional.pad(q, (0, k % 2))
    return q, (p[:, 0::2] | (p[:, 1::2] << 4)).contiguous().to(device), scale.to(device), z.to(device) if zeros else None


def exact(x, xs, q, scale, z, bias, group):
    """(values, T) in 64 bits on the host"""
    k = q.shape[1]
    at = torch.arange(k) // group
    s = scale.cpu().double()[:, at]
    zz = z.cpu().double()[:, at] if z is not None else torch.full_like(s, 8.0)
    x = x.cpu().double()
    y = x @ ((q.double() - zz) * s).t()
    t = x.abs() @ (((q.double() - zz).abs() if xs is not None else 32 + q.double() + zz) * s).t()
    if xs is not None:
        y, t = y * xs.cpu().double()[:, None], t * xs.cpu().double()[:, None]
    if bias is not None:
        y, t = y + bias.cpu().double(), t + bias.cpu().double().abs()
    return y, t


def check(got, y, t, x_dtype, k, group):
    adds = {torch.int8: 0, torch.float32: 3 * group}.get(x_dtype, group) + -(-k // group) + 16
    tol = adds * U * t + torch.finfo(got.dtype).eps / 2 * y.abs() * (1 + 1e-6) + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    off = (got.cpu().double() - y).abs()
    assert (off <= tol).all(), float((off / tol).max())


def rows_of(kind, m, k, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(m, k, generator=g, device="cuda")
    if kind == "int8":
        xs = x.abs().amax(1).clamp(min=1e-6) / 127
        return torch.round(x / xs[:, None]).to(torch.int8), xs
    return x.to(TYPES[kind]), None


SHAPES = [(1, 1, 1), (1, 16, 32), (1, 384, 384), (1, 17, 129), (2, 33, 31), (3, 100, 255), (5, 1001, 1234), (16, 64, 256), (17, 48, 1000), (31, 130, 513), (32, 31, 128), (33, 20, 2048),
          (64, 96, 640), (65, 40, 300), (130, 35, 1025)]


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32", "int8"])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_against_the_definition(layers, kind, group):
    for i, (m, n, k) in enumerate(SHAPES):
        for zeros in (False, True):
            q, packed, scale, z = make(n, k, group, zeros, 7 * i + group)
            w = layers.W4Weight.from_quantized(packed, scale, z, k=k, group=group)
            x, xs = rows_of(kind, m, k, i)
            bias = torch.randn(n, device="cuda") if i % 2 else None
            out = w.dense(x, x_scale=xs, bias=bias)
            assert out.dtype == (torch.bfloat16 if kind == "int8" else x.dtype) and out.shape == (m, n)
            y, t = exact(x, xs, q, scale, z, bias, group)
            check(out, y, t, x.dtype, k, group)
            check(w.dense(x, x_scale=xs, bias=bias, out_dtype=torch.float32), y, t, x.dtype, k, group)
            w.close()


# many outputs and rows: the kernels that share a block of rows among 2 or 4 waves (by rows, outputs and type), with whole blocks of 128 inputs in odd and even
# numbers, a part of a block behind them, and nothing but a part
MANY = [(20, 10000, 384), (20, 17000, 257), (32, 30000, 129), (33, 5000, 1408), (64, 9000, 700), (49, 17000, 513), (64, 30001, 100), (130, 5003, 300), (257, 2050, 1157)]


@pytest.mark.parametrize("kind", ["bf16", "f16", "int8"])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_many_rows_and_outputs(layers, kind, group):
    for i, (m, n, k) in enumerate(MANY):
        zeros = bool((i + group // 32) % 2)
        q, packed, scale, z = make(n, k, group, zeros, 11 * i + group)
        w = layers.W4Weight.from_quantized(packed, scale, z, k=k, group=group, scale_dtype=torch.float16)
        x, xs = rows_of(kind, m, k + 3, i)
        x = x[:, 3:]                               # a stride of its own, no alignment
        bias = torch.randn(n, device="cuda") if i % 2 else None
        out = torch.full((m + 1, n + 5), 7.0, device="cuda")
        w.dense(x, x_scale=xs, bias=bias, out=out[:m, :n])
        assert (out[m] == 7).all() and (out[:, n:] == 7).all()
        y, t = exact(x, xs, q, scale, z, bias, group)
        check(out[:m, :n], y, t, x.dtype, k, group)
        if kind != "int8":
            x = x.clone()
            clean = w.dense(x)
            x[m // 2, k - 1] = float("nan")
            got = w.dense(x)
            assert torch.isnan(got[m // 2]).all()
            keep = torch.arange(m, device="cuda") != m // 2
            assert torch.equal(got[keep], clean[keep])
        w.close()


def test_host_data_and_dequantize(layers):
    q, packed, scale, z = make(37, 200, 64, True, 3, device="cpu")
    want = (q.double() - z.double()[:, torch.arange(200) // 64]) * scale.double()[:, torch.arange(200) // 64]
    for zeros in (z, None):
        host = layers.W4Weight.from_quantized(packed, scale, zeros, k=200, group=64)
        dev = layers.W4Weight.from_quantized(packed.cuda(), scale.cuda(), zeros.cuda() if zeros is not None else None, k=200, group=64)
        ref = want if zeros is not None else (q.double() - 8) * scale.double()[:, torch.arange(200) // 64]
        assert torch.equal(host.dequantize(), ref.float()) and torch.equal(dev.dequantize(), ref.float())
        x = torch.randn(4, 200, device="cuda").half()
        assert torch.equal(host.dense(x), dev.dense(x))
    assert (host.n, host.k, host.group) == (37, 200, 64)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("scale_dtype", [torch.float16, torch.bfloat16])
def test_quantize(layers, zeros, scale_dtype):
    """half a step of the group's scale (its rounding to 16 bits moves the largest values by a little more), zeros stay zeros"""
    g = torch.Generator().manual_seed(1)
    w = 0.02 * torch.randn(50, 333, generator=g)
    w[7, 32:64] = 0
    h = layers.W4Weight.quantize(w, group=32, zeros=zeros, scale_dtype=scale_dtype)
    p = torch.nn.functional.pad(w, (0, 352 - 333)).view(50, 11, 32)
    step = ((p.amax(2).clamp(min=0) - p.amin(2).clamp(max=0)) / 15 if zeros else p.abs().amax(2) / 7).repeat_interleave(32, 1)[:, :333]
    rounding = torch.finfo(scale_dtype).eps / 2
    # rounded to half a step, and the scale's own rounding times the number in front of it; with zero points the two ends can lie half a step outside
    tol = step * (1 + rounding) * (0.5 + (0.5 if zeros else 0)) + 15 * rounding * step + 1e-6
    assert ((h.dequantize() - w).abs() <= tol).all()
    assert (h.dequantize()[7, 32:64] == 0).all()


def test_views_columns_and_out(layers):
    q, packed, scale, z = make(70, 391, 128, True, 9)
    w = layers.W4Weight.from_quantized(packed, scale, z, k=391, group=128)
    wide = torch.randn(6, 1000, device="cuda").bfloat16()
    x = wide[:, 5:396]
    want = w.dense(x.contiguous())
    assert torch.equal(w.dense(x), want)
    out = torch.full((6, 200), 3.0, device="cuda").bfloat16()
    w.dense(x, out=out[:, 11:81])
    assert torch.equal(out[:, 11:81], want) and (out[:, :11] == 3).all() and (out[:, 81:] == 3).all()
    assert torch.equal(w.dense(x.contiguous().view(2, 3, 391)).view(6, 70), want)
    for m in range(6):          # a row does not depend on its neighbours
        assert torch.equal(w.dense(x[m:m + 1]), want[m:m + 1])
    assert w.dense(x[:0]).shape == (0, 70)


def test_nan_and_infinity_stay_in_their_row(layers):
    q, packed, scale, z = make(40, 256, 64, False, 2)
    w = layers.W4Weight.from_quantized(packed, scale, z, group=64)
    for t in (torch.float32, torch.bfloat16, torch.float16):
        x = torch.randn(5, 256, device="cuda").to(t)
        clean = w.dense(x)
        x[1, 100], x[3, 0] = float("nan"), float("inf")
        out = w.dense(x)
        assert torch.isnan(out[1]).all() and torch.isnan(out[3]).all()
        assert torch.equal(out[[0, 2, 4]], clean[[0, 2, 4]])


def test_f32_rows_keep_their_24_bits(layers):
    """weights of one (q - z = 1, scale 1) at single places: the products are x itself, bit for bit"""
    n = k = 64
    q = torch.full((n, k), 8, dtype=torch.uint8)
    q[torch.arange(n), torch.arange(n)] = 9
    w = layers.W4Weight.from_quantized((q[:, 0::2] | (q[:, 1::2] << 4)).cuda(), torch.ones(n, 2, device="cuda"), group=32)
    x = torch.zeros(64, k, device="cuda")
    v = torch.randn(64, device="cuda")
    x[torch.arange(64), torch.arange(64)] = v
    got = w.dense(x)
    # one value a row: 17 x - 16 ... : sums of 25 x's parts in f32, off by at most the 25 |x| u of the two sums
    assert ((got.diagonal().double() - v.double()).abs() <= 50 * U * v.double().abs()).all()
    assert (got - torch.diag(got.diagonal())).abs().max() <= 48 * U * v.abs().max()


@needs_capture
def test_streams_threads_and_graph(layers):
    import threading
    q, packed, scale, z = make(300, 1024, 128, True, 4)
    w = layers.W4Weight.from_quantized(packed, scale, z, group=128)
    xs = [torch.randn(3, 1024, device="cuda").half() for _ in range(4)]
    want = [w.dense(x) for x in xs]
    torch.cuda.synchronize()
    wrong = []

    def caller(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(20):
                if not torch.equal(w.dense(xs[i]), want[i]):
                    wrong.append(i)
        st.synchronize()
    th = [threading.Thread(target=caller, args=(i,)) for i in range(4)]
    [t.start() for t in th]
    [t.join() for t in th]
    assert not wrong
    x = xs[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = w.dense(x)
    for k in range(4):
        x.copy_(xs[k])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want[k]), k


@needs_capture
def test_a_captured_stream_lays_out_no_weights(layers):
    from shodh_memory_amd import ShodhError
    q, packed, scale, z = make(64, 128, 64, True, 6)
    w = layers.W4Weight.from_quantized(packed, scale, z, group=64)
    x = torch.randn(2, 128, device="cuda").half()
    want = w.dense(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = w.dense(x)
        with pytest.raises(ShodhError):
            layers.W4Weight.from_quantized(packed, scale, z, group=64)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, want)


def test_refusals(layers):
    from shodh_memory_amd import ShodhError
    q, packed, scale, z = make(32, 128, 64, True, 1)
    W = layers.W4Weight
    w = W.from_quantized(packed, scale, z, group=64)
    x = torch.randn(2, 128, device="cuda")
    bad_scale = scale.clone()
    bad_scale[3, 1] = float("inf")
    big = scale.clone()
    big[0, 0] = 1e6                                # no number of fp16
    for call in [lambda: W.from_quantized(packed, scale, z, group=48), lambda: W.from_quantized(packed, scale[:, :1], z, group=64), lambda: W.from_quantized(packed, scale, z, k=200, group=64),
                 lambda: W.from_quantized(packed, scale, z + 16, group=64), lambda: W.from_quantized(packed, bad_scale, z, group=64), lambda: W.from_quantized(packed, big, z, group=64),
                 lambda: W.from_quantized(packed, scale, z.cpu(), group=64), lambda: W.from_quantized(packed, scale, z, group=64, scale_dtype=torch.float32),
                 lambda: W.quantize(torch.full((4, 32), float("nan")), group=32), lambda: w.dense(x[:, :100]), lambda: w.dense(x.cpu()), lambda: w.dense(x.double()),
                 lambda: w.dense(x, x_scale=torch.ones(2, device="cuda")), lambda: w.dense(x.to(torch.int8)), lambda: w.dense(x.to(torch.int8), x_scale=torch.ones(3, device="cuda")),
                 lambda: w.dense(x, bias=torch.zeros(31, device="cuda")), lambda: w.dense(x, out=torch.empty(2, 31, device="cuda")), lambda: w.dense(x.t()),
                 lambda: w.dense(x, out_dtype=torch.float64), lambda: w.dense(x[:1].expand(2, 128))]:
        with pytest.raises(ShodhError):
            call()
    W.from_quantized(packed, big, z, group=64, scale_dtype=torch.bfloat16).close()
    w.close()
    with pytest.raises(ShodhError):
        w.dense(x)
    torch.cuda.synchronize()


def test_out_that_overlaps_is_refused(layers):
    """the result over its own inputs would be read by other workgroups; beside them in one buffer it is as good as anywhere"""
    from shodh_memory_amd import ShodhError
    q, packed, scale, z = make(128, 128, 64, True, 12)
    w = layers.W4Weight.from_quantized(packed, scale, z, group=64)
    wide = torch.randn(9, 300, device="cuda").half()
    x, want = wide[:, :128], w.dense(wide[:, :128].contiguous())
    bias, x8 = torch.zeros(9 * 128, device="cuda"), torch.ones(9, 128, dtype=torch.int8, device="cuda")
    for call in [lambda: w.dense(x, out=x), lambda: w.dense(x, out=wide[:, 100:228]), lambda: w.dense(x[1:], out=wide[:-1, :128]), lambda: w.dense(x, bias=bias[:128], out=bias.view(9, 128)),
                 lambda: w.dense(x8, x_scale=bias[:9], out=bias.view(9, 128))]:
        with pytest.raises(ShodhError):
            call()
    assert w.dense(x, out=wide[:, 128:256]).shape == (9, 128) and torch.equal(wide[:, 128:256], want)
    square = torch.randn(5, 128, device="cuda").half()
    assert torch.equal(w.dense(square, out=torch.empty_like(square)), w.dense(square))
    torch.cuda.synchronize()


@pytest.mark.parametrize("n,rows", [(16, 32 * 65535 + 50), (1048560, 2100)])
def test_more_rows_than_a_launch_takes(layers, n, rows):
    """in turns: every row is what it is in a call of its own"""
    g = torch.Generator(device="cuda").manual_seed(1)
    packed = torch.randint(0, 256, (n, 16), generator=g, dtype=torch.uint8, device="cuda")
    w = layers.W4Weight.from_quantized(packed, torch.full((n, 1), 0.03, device="cuda"), group=32)
    x = torch.randn(rows, 32, generator=g, device="cuda").bfloat16()
    out = w.dense(x)
    for r in (0, 2047, 2048, 2099, rows - 50, rows - 1):
        assert torch.equal(out[r:r + 1], w.dense(x[r:r + 1])), r
    x8, xs = torch.randint(-127, 128, (rows, 32), generator=g, device="cuda").to(torch.int8), torch.rand(rows, generator=g, device="cuda")
    w.dense(x8, x_scale=xs, out=out)
    for r in (0, 2048, rows - 1):
        assert torch.equal(out[r:r + 1], w.dense(x8[r:r + 1], x_scale=xs[r:r + 1])), r


def test_sizes_that_32_bits_cannot_hold(layers):
    from shodh_memory_amd import ShodhError
    q, packed, scale, z = make(16, 32, 32, False, 1)
    w = layers.W4Weight.from_quantized(packed, scale, group=32)
    held = torch.zeros(2 ** 32 + 64, dtype=torch.bfloat16, device="cuda")
    for call in [lambda: w.dense(held.as_strided((2 ** 32 + 1, 32), (1, 1))), lambda: w.dense(held.as_strided((2 ** 32, 32), (1, 1))), lambda: layers.W4Weight.quantize(torch.zeros(16, 32), group=2 ** 32 + 32),
                 lambda: layers.W4Weight.quantize(torch.zeros(16, 32), group=-32)]:
        with pytest.raises(ShodhError):
            call()


def test_scales_keep_their_type(layers):
    """bf16 scales are kept as they are, however small; scales that a type cannot hold to half its step are refused in it"""
    from shodh_memory_amd import ShodhError
    W = layers.W4Weight
    q, packed, _, z = make(16, 96, 32, True, 5)
    each = (q.double() - z.cpu().double()[:, torch.arange(96) // 32])
    for value in (1.0, 1e-6, 1e-7, 2e-8, 1e-20, 3e38, 0.0):
        for scale in (torch.full((16, 3), value, device="cuda").bfloat16(), torch.full((16, 3), value).bfloat16()):
            zz, pp = (z, packed) if scale.is_cuda else (z.cpu(), packed.cpu())
            w = W.from_quantized(pp, scale, zz, group=32) if value < 1e38 else None
            if w is not None:
                assert torch.equal(w.dequantize(), (each * scale.cpu().double()[:, torch.arange(96) // 32]).float())
        half = torch.full((16, 3), value, device="cuda").half()
        if torch.isfinite(half).all():           # what is a number of fp16 already stays what it is, the smallest ones too
            w = W.from_quantized(packed, half, z, group=32)
            assert torch.equal(w.dequantize(), (each * half.cpu().double()[:, torch.arange(96) // 32]).float())
        for dtype, least in ((None, 2.0 ** -14), (torch.float16, 2.0 ** -14), (torch.bfloat16, 2.0 ** -126)):
            f = torch.full((16, 3), 0.05, device="cuda")
            f[7, 2] = value
            largest = 65504 if dtype is not torch.bfloat16 else 3.38e38
            if value and not least <= value <= largest:
                with pytest.raises(ShodhError):
                    W.from_quantized(packed, f, z, group=32, scale_dtype=dtype)
            else:
                d = W.from_quantized(packed, f, z, group=32, scale_dtype=dtype).dequantize().double()
                want = each * f.cpu().double()[:, torch.arange(96) // 32]
                over = want.abs() > 3.5e38           # 2 x 3e38 and more: no numbers of dequantize's f32 (its largest is 3.403e38), but infinities of their sign
                assert torch.equal(d[over], torch.sign(want[over]) * float("inf"))
                assert ((d - want).abs() <= torch.finfo(dtype or torch.float16).eps / 2 * want.abs() * (1 + 1e-6))[~over].all()
    w = 1e-9 * torch.randn(8, 64)
    assert ((W.quantize(w, group=32, scale_dtype=torch.bfloat16).dequantize() - w).abs().max() <= 1e-9 * 0.4)
    torch.cuda.synchronize()


@needs_capture
@pytest.mark.parametrize("elsewhere", [True, False])
def test_weights_come_and_go_beside_a_capture(layers, elsewhere):
    """made from host data, read back and freed while a graph is captured, by another thread or the same one: the capture is what it would be without"""
    import threading
    q, packed, scale, z = make(64, 128, 64, True, 6, device="cpu")
    w = layers.W4Weight.from_quantized(packed, scale, z, group=64)
    f, held_weights = torch.randn(40, 96, generator=torch.Generator().manual_seed(3)), [layers.W4Weight.from_quantized(packed, scale, z, group=64) for _ in range(2)]
    x = torch.randn(2, 128, device="cuda").half()
    want, made, wrong = w.dense(x), [], []

    def work():
        try:
            made.append(layers.W4Weight.from_quantized(packed, scale, z, group=64))
            made.append(layers.W4Weight.quantize(f, group=32))
            made.append(made[0].dequantize())
            held_weights.pop()                       # (collected)
            held_weights.pop().close()
        except Exception as e:
            wrong.append(e)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = w.dense(x)
        if elsewhere:
            th = threading.Thread(target=work)
            th.start()
            th.join()
        else:
            work()
        second = w.dense(x)
    assert not wrong and not held_weights
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, want) and torch.equal(second, want)
        assert torch.equal(made[0].dense(x), want) and torch.equal(made[2], w.dequantize())
        x.mul_(0.5)
        want = w.dense(x)
    assert torch.equal(made[1].dequantize(), layers.W4Weight.quantize(f, group=32).dequantize())


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 2, 3, 5, 16, 17, 64, 100])
def test_f32_rows_come_through_bit_for_bit(layers, group, rows):
    """one weight of 1 for each output, all others 0: a row's three parts times 1 add up to the value itself without a rounding, the rest to 0"""
    for k, n in ((31, 20), (128, 100), (300, 333), (1161, 50)):
        g = torch.Generator().manual_seed(k + rows)
        place = torch.randint(0, k, (n,), generator=g)
        place[0], place[-1] = 0, k - 1
        z = torch.randint(0, 15, (n, -(-k // group)), generator=g, dtype=torch.uint8)
        q = z.repeat_interleave(group, 1)[:, :k].contiguous()
        q[torch.arange(n), place] += 1
        p = torch.nn.functional.pad(q, (0, k % 2))
        w = layers.W4Weight.from_quantized(p[:, 0::2] | (p[:, 1::2] << 4), torch.ones(n, z.shape[1]), z, k=k, group=group)
        x = (torch.randn(rows, k, generator=g) * torch.exp(4 * torch.randn(rows, k, generator=g))).cuda()
        assert torch.equal(w.dense(x), x[:, place.cuda()])


@pytest.mark.parametrize("group", [32, 64, 128])
def test_f32_rows_against_the_definition_without_the_16s(layers, group):
    """f32 rows multiply q - z itself. A product of a part of x (8 bits) with q - z (5 bits) is exact; a group's three sums of G of them, the scale, the sum over
    groups, the waves and the bias are one u = 2^-23 of what has been added up each: |y - exact| <= (3 G + K / G + 16) u sum |x| |q - z| s (+ |bias|) + u / 2 |exact|.
    That is a tenth and less of what the form 16 + q would need; rows of one sign and weights whose sum is near 0 would show it."""
    for i, (m, n, k) in enumerate(SHAPES):
        for zeros in (False, True):
            q, packed, scale, z = make(n, k, group, zeros, 13 * i + group)
            w = layers.W4Weight.from_quantized(packed, scale, z, k=k, group=group)
            x = rows_of("f32", m, k, i)[0]
            if i % 2:
                x = x.abs() + 1
            y, _ = exact(x, None, q, scale, z, None, group)
            _, t = exact(x, torch.ones(m), q, scale, z, None, group)
            off = (w.dense(x).cpu().double() - y).abs()
            tol = (3 * group + -(-k // group) + 16) * U * t + U / 2 * y.abs()
            assert (off <= tol).all(), float((off / tol).max())


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32", "int8"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(1, 50, 1000), (4, 33, 384), (16, 100, 700), (33, 40, 513), (64, 9000, 384), (20, 17000, 257), (49, 30000, 300)])
def test_large_values_that_meet_no_weight(layers, kind, group, m, n, k):
    """every other input is huge, its weights are 0 (q = z); the others are whole numbers that f32 adds up exactly: an f32 result is that sum, without a trace of
    the rounding of the large ones. (|sum| <= 1000 / 2 x 120 x 15 < 2^24, scale 1)"""
    g = torch.Generator().manual_seed(m + group)
    z = torch.randint(0, 16, (n, -(-k // group)), generator=g, dtype=torch.uint8)
    q = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    q[:, ::2] = z.repeat_interleave(group, 1)[:, :k:2]
    p = torch.nn.functional.pad(q, (0, k % 2))
    w = layers.W4Weight.from_quantized((p[:, 0::2] | (p[:, 1::2] << 4)).cuda(), torch.ones(n, z.shape[1], device="cuda"), z.cuda(), k=k, group=group)
    x = torch.randint(-120, 121, (m, k), generator=g).float()
    want = x[:, 1::2].double() @ (q.double() - z.repeat_interleave(group, 1)[:, :k].double())[:, 1::2].t()
    x[:, ::2] = {"bf16": 2.0 ** 40, "f16": 2.0 ** 15, "f32": 2.0 ** 40, "int8": 127}[kind]
    if kind == "int8":
        got = w.dense(x.to(torch.int8).cuda(), x_scale=torch.ones(m, device="cuda"), out_dtype=torch.float32)
    else:
        got = w.dense(x.to(TYPES[kind]).cuda(), out_dtype=torch.float32)
    assert torch.equal(got.cpu().double(), want)
