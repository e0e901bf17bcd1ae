"""Attention with a sliding window and always-visible first tokens against its definition in 64 bits (GPU).

Tolerance. Inputs are numbers of a 16-bit type, so scores are exact products summed in f32: with u = 2^-23 a score s is off by at most
(D + 2) u scale sum |q k|, call it e; a probability by the factor exp(+- 2 e) (its own score and the sum's) and a few u of exp2 and the sums (at most
(64 + 16) u: tiles, halves, waves and parts are added one after another). For the product with V a probability is rounded to the 16-bit type, by half a
step h = eps(type) / 2 relative (fp16: or 2^-25, half its smallest step, of the largest; keys in number n), and the result once more:
    |out - exact| <= (h + 2 e + 80 u (1 + n / 4096)) sum p |v| + [fp16] n 2^-25 max |v| + h |exact|
lse is off by at most e + 80 u + u |lse|."""
import math
import os

import pytest
import torch

from .conftest import needs_capture

pytestmark = pytest.mark.gpu
U = 2.0 ** -23
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def layers():
    from shodh_memory_amd import layers
    return layers


def exact(q, k, v, nq, nk, left, right, sinks, starts=None, scale=None):
    """(out, lse, tolerance of out, tolerance of lse) in 64 bits on the host"""
    t = q.dtype
    q, k, v = q.cpu().double(), k.cpu().double(), v.cpu().double()
    heads, kv, d = q.shape[1], k.shape[1], q.shape[2]
    scale = d ** -0.5 if scale is None else scale
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    lse, ltol = torch.full(q.shape[:2], -math.inf, dtype=torch.float64), torch.zeros(q.shape[:2], dtype=torch.float64)
    h2 = torch.finfo(t).eps / 2
    at = 0
    for b, (a, n) in enumerate(zip(nq, nk)):
        f = at if starts is None else starts[b]
        p, j = torch.arange(a)[:, None] + n - a, torch.arange(n)[None]
        seen = torch.ones(a, n, dtype=torch.bool)
        if right >= 0:
            seen &= j <= p + right
        if left >= 0:
            seen &= (j >= p - left) | (j < sinks)
        for h in range(heads):
            hk = h * kv // heads
            kk, vv = k[f:f + n, hk], v[f:f + n, hk]
            s = (scale * (q[at:at + a, h] @ kk.t())).masked_fill(~seen, -math.inf)
            size = (abs(scale) * (q[at:at + a, h].abs() @ kk.abs().t())).masked_fill(~seen, 0)
            e = (d + 2) * U * (size.amax(1) if n else torch.zeros(a, dtype=torch.float64))
            if n:
                l = torch.logsumexp(s, 1)
                w = torch.exp(s - torch.where(torch.isinf(l), 0.0, l)[:, None])
                w = torch.where(seen, w, 0.0)
                vz = vv.masked_fill(~seen.any(0)[:, None], 0) if a else vv
                o = w @ vz
                lse[at:at + a, h], out[at:at + a, h] = l, o
                ltol[at:at + a, h] = e + 80 * U + U * torch.where(torch.isinf(l), 0.0, l).abs()
                cnt = seen.sum(1).double()[:, None]
                top = (seen.double()[:, :, None] * vz.abs()[None]).amax(1) if a * n * d < 3e7 else vz.abs().amax()
                tol[at:at + a, h] = (h2 + 2 * e[:, None] + 80 * U * (1 + cnt / 4096)) * (w @ vz.abs()) + (cnt * 2.0 ** -25 * top if t == torch.float16 else 0) + h2 * o.abs() + 1e-30
        at += a
    return out, lse, tol, ltol


def check(got, lse, ref):
    o, l, tol, ltol = ref
    got, lse = got.cpu().double(), lse.cpu().double()
    off = (got - o).abs()
    assert (off <= tol * (1 + 1e-6) + (2.0 ** -25 if got.dtype == torch.float16 else 0)).all(), float((off / tol.clamp(min=1e-30)).max())
    none = torch.isinf(l)
    assert torch.equal(torch.isinf(lse), none) and (lse[none] < 0).all() and (got[none] == 0).all()
    assert ((lse - l).abs()[~none] <= ltol[~none]).all()


def cu_of(nq):
    return torch.tensor([sum(nq[:i]) for i in range(len(nq) + 1)], dtype=torch.int32, device="cuda")


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv,dim", [(2, 2, 32), (4, 1, 64), (3, 3, 128), (6, 2, 40), (5, 1, 8), (8, 2, 96)])
@pytest.mark.parametrize("left,right,sinks", [(-1, -1, 0), (-1, 0, 0), (31, 0, 4), (0, 0, 0), (10, 7, 1), (64, 64, 3), (100, -1, 70), (5, 0, 300)])
def test_texts(layers, dtype, heads, kv, dim, left, right, sinks):
    """ragged self-attention, q|k|v as parts of one tensor"""
    nq = [1, 0, 33, 200, 2, 129, 64, 31, 1, 300]
    qkv = normal(1, sum(nq), heads + 2 * kv, dim).to(TYPES[dtype])
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    out, lse = layers.window_attention(q, k, v, cu_of(nq), left=left, right=right, sinks=sinks, return_lse=True)
    assert out.shape == q.shape and out.is_contiguous()
    check(out, lse, exact(q, k, v, nq, nq, left, right, sinks))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv,dim", [(2, 2, 32), (16, 4, 64), (8, 1, 128), (12, 12, 64), (40, 1, 72)])
@pytest.mark.parametrize("left,right,sinks", [(-1, 0, 0), (63, 0, 4), (1000, 0, 1), (0, 0, 2), (700, 0, 900)])
def test_single_tokens_over_a_cache(layers, dtype, heads, kv, dim, left, right, sinks):
    nk = [1, 0, 1500, 64, 65, 31, 700, 33, 4000, 5]
    nq = [1, 1, 1, 1, 1, 2, 5, 1, 1, 0]
    starts = [sum(nk[:i]) + 3 * i for i in range(len(nk))]
    total = starts[-1] + nk[-1] + 2
    q, k, v = normal(2, sum(nq), heads, dim).to(TYPES[dtype]), normal(3, total, kv, dim).to(TYPES[dtype]), normal(4, total, kv, dim).to(TYPES[dtype])
    out, lse = layers.window_attention(q, k, v, cu_of(nq), left=left, right=right, sinks=sinks, kv_start=torch.tensor(starts, device="cuda"),
                                       kv_len=torch.tensor(nk, dtype=torch.int32, device="cuda"), return_lse=True)
    check(out, lse, exact(q, k, v, nq, nk, left, right, sinks, starts))


@pytest.mark.parametrize("nq,nk", [([40], [10]), ([300, 1], [100, 0]), ([3], [2]), ([700], [1300])])
def test_more_queries_than_keys_and_parts(layers, nq, nk):
    """queries ahead of the first key see nothing: zeros and -inf"""
    starts = [sum(nk[:i]) for i in range(len(nk))]
    q, k, v = normal(5, sum(nq), 4, 64).bfloat16(), normal(6, sum(nk) + 1, 2, 64).bfloat16(), normal(7, sum(nk) + 1, 2, 64).bfloat16()
    for left, right, sinks in [(-1, 0, 0), (20, 0, 2), (-1, -1, 0), (4, 3, 0)]:
        out, lse = layers.window_attention(q, k, v, cu_of(nq), left=left, right=right, sinks=sinks, kv_start=torch.tensor(starts, device="cuda"),
                                           kv_len=torch.tensor(nk, dtype=torch.int32, device="cuda"), return_lse=True)
        check(out, lse, exact(q, k, v, nq, nk, left, right, sinks, starts))


def test_long_document(layers):
    q, k, v = normal(8, 3001, 16, 128).bfloat16(), normal(9, 3001, 8, 128).bfloat16(), normal(10, 3001, 8, 128).bfloat16()
    cu = cu_of([3001])
    for left, sinks in [(511, 4), (-1, 0)]:
        out, lse = layers.window_attention(q, k, v, cu, left=left, right=0, sinks=sinks, return_lse=True)
        check(out, lse, exact(q, k, v, [3001], [3001], left, 0, sinks))


@pytest.mark.parametrize("lq", [1, 900])
def test_growing_scores_and_scale(layers, lq):
    """scores that rise along the keys by far more than 8 powers of two move the reference maximum tile after tile; a scale of one's own"""
    n = 2000
    q = torch.ones(lq, 2, 64, device="cuda").half()
    k = (torch.linspace(-4, 4, n, device="cuda")[:, None, None] * torch.ones(n, 2, 64, device="cuda")).half()
    v = normal(11, n, 2, 64).half()
    for kk in (k, k.flip(0).contiguous()):
        for scale in (0.3, -0.05):
            out, lse = layers.window_attention(q, kk, v, cu_of([lq]), scale=scale, kv_start=torch.zeros(1, dtype=torch.int64, device="cuda"),
                                               kv_len=torch.tensor([n], dtype=torch.int32, device="cuda"), return_lse=True)
            check(out, lse, exact(q, kk, v, [lq], [n], -1, -1, 0, [0], scale))


@pytest.mark.parametrize("nq,nk", [([400, 37], [400, 37]), ([1, 2], [900, 77])])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_what_masked_keys_hold_does_not_matter(layers, nq, nk, bad, dim):
    """rows that do not see the spoiled keys are, bit for bit, what they are without them; those that see them are spoiled"""
    starts = [sum(nk[:i]) + 7 * i for i in range(len(nk))]
    total = starts[-1] + nk[-1] + 7
    q, k, v = normal(12, sum(nq), 4, dim).bfloat16(), normal(13, total, 2, dim).bfloat16(), normal(14, total, 2, dim).bfloat16()
    args = dict(left=50, right=0, sinks=2, kv_start=torch.tensor(starts, device="cuda"), kv_len=torch.tensor(nk, dtype=torch.int32, device="cuda"), return_lse=True)
    clean, clse = layers.window_attention(q, k, v, cu_of(nq), **args)
    spoiled = [j for j in (2, 20, 21, 199, 300, 845, 846, 860) if j < nk[0]]
    k2, v2 = k.clone(), v.clone()
    for j in spoiled:
        v2[j] = bad
        if j != 300:
            k2[j] = float("nan")
    gap = starts[1] - 7
    k2[gap:gap + 7] = float("nan")
    v2[gap:gap + 7] = bad                 # between the sequences
    out, lse = layers.window_attention(q, k2, v2, cu_of(nq), **args)
    at = 0
    for b, (a, n) in enumerate(zip(nq, nk)):
        for i in range(a):
            p = i + n - a
            hit = b == 0 and any(j <= p and (j >= p - 50 or j < 2) for j in spoiled)
            if hit:
                assert not torch.isfinite(out[at + i]).any()
            else:
                assert torch.equal(out[at + i], clean[at + i]) and torch.equal(lse[at + i], clse[at + i]), (b, i)
        at += a


def test_one_row_is_what_it_is_in_any_batch(layers):
    """a sequence's values do not depend on its neighbours in the batch where the form is the same"""
    nq = [70, 130, 256, 1, 90] * 30
    q, k, v = normal(15, sum(nq), 4, 64).bfloat16(), normal(16, sum(nq), 4, 64).bfloat16(), normal(17, sum(nq), 4, 64).bfloat16()
    a = layers.window_attention(q, k, v, cu_of(nq), left=40, right=40)
    n = sum(nq) // 2
    b = layers.window_attention(q[:n].contiguous(), k[:n].contiguous(), v[:n].contiguous(), cu_of(nq[:75]), left=40, right=40)
    assert torch.equal(a[:n], b)


def test_strides_out_and_rows_behind_the_last(layers):
    nq = [50, 3]
    base_q, base_kv = normal(18, 4, 60, 72).half(), normal(19, 60, 2, 150).half()
    q = base_q.transpose(0, 1)[:, :, 1:65]                              # head-major, odd start
    k, v = base_kv[:, :, 3:67], base_kv[:, :, 81:145]
    want, wl = layers.window_attention(q.contiguous(), k.contiguous(), v.contiguous(), cu_of(nq), left=9, right=2, sinks=1, return_lse=True)
    out = torch.full((60, 4, 70), 9.0, device="cuda").half()
    got, gl = layers.window_attention(q, k, v, cu_of(nq), left=9, right=2, sinks=1, return_lse=True, out=out[:, :, 2:66])
    assert torch.equal(out[:53, :, 2:66], want[:53]) and (out[53:] == 9).all() and (out[:, :, :2] == 9).all() and (out[:, :, 66:] == 9).all()
    assert torch.equal(gl[:53], wl[:53])
    # head-major output, and the split form's rows behind the last sequence
    hm = torch.full((4, 60, 64), 9.0, device="cuda").half()
    layers.window_attention(q, k, v, cu_of(nq), left=9, right=2, sinks=1, out=hm.transpose(0, 1))
    assert torch.equal(hm.transpose(0, 1)[:53], want[:53]) and (hm[:, 53:] == 9).all()
    one = torch.full((3, 4, 64), 9.0, device="cuda").half()
    layers.window_attention(q[:3], base_kv[:, :, 3:67], base_kv[:, :, 81:145], torch.tensor([0, 1], dtype=torch.int32, device="cuda"), out=one,
                            kv_start=torch.zeros(1, dtype=torch.int64, device="cuda"), kv_len=torch.tensor([60], dtype=torch.int32, device="cuda"))
    assert (one[1:] == 9).all() and (one[0] != 9).all()


def test_offsets_past_32_bits(layers):
    """a cache of more than 2^32 elements, one sequence at its end"""
    total, kv, d = (1 << 32) // 128 + 4096, 1, 128
    k = torch.zeros(total, kv, d, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(total, kv, d, dtype=torch.bfloat16, device="cuda")
    n = 300
    k[-n:], v[-n:] = normal(20, n, kv, d).bfloat16(), normal(21, n, kv, d).bfloat16()
    q = normal(22, 1, 4, d).bfloat16()
    out, lse = layers.window_attention(q, k, v, cu_of([1]), left=100, right=0, sinks=3, kv_start=torch.tensor([total - n], device="cuda"),
                                       kv_len=torch.tensor([n], dtype=torch.int32, device="cuda"), return_lse=True)
    check(out, lse, exact(q, k[-n:], v[-n:], [1], [n], 100, 0, 3, [0]))


def test_bad_descriptors_stay_in_bounds(layers):
    """ranges outside the cache have no keys; a bad cu leaves its neighbours right"""
    q, k, v = normal(23, 4, 2, 64).bfloat16(), normal(24, 100, 2, 64).bfloat16(), normal(25, 100, 2, 64).bfloat16()
    start = torch.tensor([0, 90, -5, 10], device="cuda")
    length = torch.tensor([40, 11, 10, -1], dtype=torch.int32, device="cuda")
    out, lse = layers.window_attention(q, k, v, cu_of([1, 1, 1, 1]), kv_start=start, kv_len=length, return_lse=True)
    ref = exact(q[:1], k, v, [1], [40], -1, -1, 0, [0])
    check(out[:1], lse[:1], ref)
    assert (out[1:] == 0).all() and torch.isinf(lse[1:]).all()
    cu = torch.tensor([0, 2, 4, 9], dtype=torch.int32, device="cuda")
    out = layers.window_attention(q, k[:4].contiguous(), v[:4].contiguous(), cu)
    good = layers.window_attention(q, k[:4].contiguous(), v[:4].contiguous(), cu[:3].contiguous())
    assert torch.equal(out, good)
    torch.cuda.synchronize()


@pytest.mark.parametrize("seqs", [65, 256, 300, 4200])
def test_many_sequences(layers, seqs):
    """ragged texts, and single tokens over caches: more sequences than one load of cu, than one round of its search, than one table of parts"""
    g = torch.Generator().manual_seed(seqs)
    most = 6 if seqs > 1000 else 80
    nq = [int(n) for n in torch.randint(0, most, (seqs,), generator=g)]
    nq[seqs // 2], nq[-1] = 140, 0
    q, k, v = normal(30, sum(nq), 2, 32).bfloat16(), normal(31, sum(nq), 1, 32).bfloat16(), normal(32, sum(nq), 1, 32).bfloat16()
    out, lse = layers.window_attention(q, k, v, cu_of(nq), left=20, right=3, sinks=2, return_lse=True)
    check(out, lse, exact(q, k, v, nq, nq, 20, 3, 2))
    nk = [int(n) for n in torch.randint(0, most, (seqs,), generator=g)]
    nk[1], nk[seqs // 3], nk[-2] = 2500, 0, 900
    nq = [int(n) for n in torch.randint(0, 3, (seqs,), generator=g)]
    starts = [sum(nk[:i]) for i in range(seqs)]
    q, k, v = normal(33, sum(nq), 2, 32).half(), normal(34, sum(nk), 1, 32).half(), normal(35, sum(nk), 1, 32).half()
    for left in (-1, 700):
        out, lse = layers.window_attention(q, k, v, cu_of(nq), left=left, right=0, sinks=3, kv_start=torch.tensor(starts, device="cuda"),
                                           kv_len=torch.tensor(nk, dtype=torch.int32, device="cuda"), return_lse=True)
        check(out, lse, exact(q, k, v, nq, nk, left, 0, 3, starts))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [32, 56, 64, 128])
@pytest.mark.parametrize("nq,nk", [([150, 1, 40], [150, 1, 40]), ([1, 3], [700, 260])])
def test_odd_places(layers, dtype, dim, nq, nk):
    """q, k and v at places and distances that are no multiples of 16 bytes, in both forms"""
    starts = [sum(nk[:i]) + i for i in range(len(nk))]
    t = TYPES[dtype]
    q = normal(36, sum(nq), 4, dim + 3).to(t)[:, :, 1:1 + dim]
    k, v = normal(37, sum(nk) + 3, 2, dim + 5).to(t)[:, :, 3:3 + dim], normal(38, sum(nk) + 3, 2, 2 * dim + 1).to(t)[:, :, dim:2 * dim]
    for left, right, sinks in [(-1, 0, 0), (60, 0, 3), (33, 10, 0)]:
        out, lse = layers.window_attention(q, k, v, cu_of(nq), left=left, right=right, sinks=sinks, kv_start=torch.tensor(starts, device="cuda"),
                                           kv_len=torch.tensor(nk, dtype=torch.int32, device="cuda"), return_lse=True)
        check(out, lse, exact(q, k, v, nq, nk, left, right, sinks, starts))


@pytest.mark.parametrize("nq,nk", [([300, 5], [300, 5]), ([1, 1], [3000, 12])])
def test_over_the_queries(layers, nq, nk):
    """out = q itself: each row of q is read by those that write its output alone, before they write"""
    q = normal(42, sum(nq), 4, 64).bfloat16()
    k, v = normal(43, sum(nk), 2, 64).bfloat16(), normal(44, sum(nk), 2, 64).bfloat16()
    args = dict(left=900, right=0, kv_start=torch.tensor([0, nk[0]], device="cuda"), kv_len=torch.tensor(nk, dtype=torch.int32, device="cuda"))
    want = layers.window_attention(q, k, v, cu_of(nq), **args)
    got = q.clone()
    assert layers.window_attention(got, k, v, cu_of(nq), out=got, **args) is got
    assert torch.equal(got, want)


def test_no_keys_at_all_and_the_largest_bounds(layers):
    none = torch.empty(0, 2, 64, device="cuda", dtype=torch.bfloat16)
    start, length = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    for n in (1, 500):
        out, lse = layers.window_attention(normal(45, n, 4, 64).bfloat16(), none, none, cu_of([n]), kv_start=start, kv_len=length, return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all()
    big = 2 ** 31 - 1
    q, k, v = normal(46, 200, 4, 64).bfloat16(), normal(47, 200, 2, 64).bfloat16(), normal(48, 200, 2, 64).bfloat16()
    for left, right, sinks in [(big, big, 0), (big, 0, big), (0, big, big), (-2 ** 31, -2 ** 31, 0)]:
        for a, b in ((200, 200), (3, 200)):
            out, lse = layers.window_attention(q[:a], k, v, cu_of([a]), left=left, right=right, sinks=sinks, kv_start=start, kv_len=length + b, return_lse=True)
            check(out, lse, exact(q[:a], k, v, [a], [b], left, right, sinks, [0]))


def test_a_cache_in_many_parts(layers):
    nk = [60000, 1, 33333]
    starts = [0, 60000, 60001]
    q, k, v = normal(39, 4, 8, 64).bfloat16(), normal(40, sum(nk), 1, 64).bfloat16(), normal(41, sum(nk), 1, 64).bfloat16()
    for left in (-1, 50000):
        out, lse = layers.window_attention(q, k, v, cu_of([1, 1, 2]), left=left, right=0, sinks=5, kv_start=torch.tensor(starts, device="cuda"),
                                           kv_len=torch.tensor(nk, dtype=torch.int32, device="cuda"), return_lse=True)
        check(out, lse, exact(q, k, v, [1, 1, 2], nk, left, 0, 5, starts))


@needs_capture
def test_streams_and_two_graphs(layers):
    """two captured graphs and eager calls in between, with lengths that change from replay to replay"""
    q = normal(26, 2, 8, 64).bfloat16()
    k, v = normal(27, 9000, 2, 64).bfloat16(), normal(28, 9000, 2, 64).bfloat16()
    start, cu = torch.tensor([0, 4500], device="cuda"), cu_of([1, 1])
    length = torch.tensor([3000, 4000], dtype=torch.int32, device="cuda")

    def call():
        return layers.window_attention(q, k, v, cu, left=2500, right=0, sinks=4, kv_start=start, kv_len=length, return_lse=True)
    call()
    torch.cuda.synchronize()
    graphs, held = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(call())
        graphs.append(g)
    for n in (1, 2999, 4500, 64):
        length.copy_(torch.tensor([n, 4500 - n // 2], dtype=torch.int32))
        want = call()
        for g in graphs:
            g.replay()
        want2 = call()
        torch.cuda.synchronize()
        for h in held:
            assert torch.equal(h[0], want[0]) and torch.equal(h[1], want[1]) and torch.equal(want2[0], want[0]), n
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    raw = layers.window_attention(q, k, v, cu, left=2500, right=0, sinks=4, kv_start=start, kv_len=length, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(raw, want[0])


def test_refusals(layers):
    from shodh_memory_amd import ShodhError
    q, k, v, cu = normal(1, 6, 4, 64).bfloat16(), normal(2, 6, 2, 64).bfloat16(), normal(3, 6, 2, 64).bfloat16(), cu_of([6])
    A = layers.window_attention
    st, ln = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    wide = torch.randn(6, 4, 136, device="cuda").bfloat16()
    for call in [lambda: A(q.float(), k.float(), v.float(), cu), lambda: A(q, k.half(), v, cu), lambda: A(q, k, v[:, :1], cu), lambda: A(q, k[:, :, :32], v[:, :, :32], cu),
                 lambda: A(q[:, :3], k, v, cu), lambda: A(wide, wide[:, :2], wide[:, :2], cu), lambda: A(q[:, :, :60], k[:, :, :60], v[:, :, :60], cu), lambda: A(q, k, v, cu.long()),
                 lambda: A(q, k, v, cu.cpu()), lambda: A(q, k[:5], v[:5], cu), lambda: A(q, k, v, cu, kv_start=st), lambda: A(q, k, v, cu, kv_start=st, kv_len=ln.long()),
                 lambda: A(q, k, v, cu, kv_start=st.int(), kv_len=ln), lambda: A(q, k, v, cu, sinks=-1), lambda: A(q, k, v, cu, scale=0.0), lambda: A(q, k, v, cu, scale=float("nan")),
                 lambda: A(q, k, v, cu, scale=float("inf")), lambda: A(q, k, v, cu, out=q[:5]), lambda: A(q, k, v, cu, out=q[:1].expand(6, 4, 64)), lambda: A(q.transpose(1, 2), k, v, cu),
                 lambda: A(q[:, :1].expand(6, 4, 64), k, v, cu), lambda: A(q.cpu(), k, v, cu), lambda: A(q, k.cpu(), v, cu), lambda: A(q[0], k, v, cu)]:
        with pytest.raises(ShodhError):
            call()
    assert A(q[:0], k[:0], v[:0], cu_of([0])).shape == (0, 4, 64)
    torch.cuda.synchronize()


@pytest.mark.parametrize("lq,heads", [(1, 2), (3, 2), (700, 2), (1024, 32)])
@pytest.mark.parametrize("above", [10.0, 14.0, 16.0, 17.5, 20.0])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_what_a_dominant_sink_leaves_over(layers, dtype, above, lq, heads):
    """a first key with nearly all the weight and a value of zero: the output is what the many others make of the small rest. A probability in fp16 is
    off by half its type's step relative, or by half of the smallest step: 2^-25 of 2^7 at least, the place of the largest (bf16 has that range):
        |out - exact| <= (h + 2 e + 160 u) sum p |v| + h |exact| + [fp16] 2^-32 sum |v| + 2^-25
    with scores of one exact product each: e = 66 u |s|, |s| <= above."""
    t, n, d = TYPES[dtype], 4096, 64
    q = torch.zeros(lq, heads, d, device="cuda", dtype=t)
    q[:, :, 0] = 1
    k = torch.zeros(n, heads, d, device="cuda", dtype=t)
    k[1:, :, 0] = (0.02 * normal(60, n - 1, 1)).to(t)
    k[0, :, 0] = above
    v = normal(61, n, 1, d).to(t).expand(n, heads, d).contiguous()
    v[:, :, :8] = 1                                            # rest after rest on the same side: nothing averages out
    v[0] = 0
    out = layers.window_attention(q, k, v, cu_of([lq]), left=n, right=n, sinks=1, scale=1.0, kv_start=torch.zeros(1, dtype=torch.int64, device="cuda"),
                                  kv_len=torch.tensor([n], dtype=torch.int32, device="cuda"))
    p, v0 = torch.softmax(k[:, 0, 0].double(), 0), v[:, 0].double()
    want, size = p @ v0, p @ v0.abs()
    h = torch.finfo(t).eps / 2
    tol = (h + 2 * 66 * U * above + 160 * U) * size + h * want.abs() + ((2.0 ** -32 * v0.abs().sum(0) + 2.0 ** -25) if t == torch.float16 else 0)
    assert ((out.double() - want).abs() <= tol * (1 + 1e-6)).all(), float(((out.double() - want).abs() / tol).max())


def used_by(call):
    """(result, most bytes of device memory taken meanwhile; 0 under the guard's allocator, which does not count them)"""
    if os.environ.get("SHODH_GUARD", "0") not in ("", "0"):
        return call(), 0
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = call()
    torch.cuda.synchronize()
    return out, torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("dtype,heads,kv,dim,lq,nk,left", [("bf16", 8, 1, 128, 1500, 9000, -1), ("f16", 8, 1, 128, 1500, 9000, 6000), ("bf16", 24, 1, 64, 611, 30011, -1), ("bf16", 32, 8, 32, 300, 33000, -1)])
def test_a_prompt_over_a_long_cache(layers, dtype, heads, kv, dim, lq, nk, left):
    """hundreds of new tokens behind tens of thousands: more parts are wanted than there are places for"""
    t = TYPES[dtype]
    q, k, v = normal(70, lq, heads, dim).to(t), normal(71, nk + 5, kv, dim).to(t), normal(72, nk + 5, kv, dim).to(t)
    start, length = torch.tensor([5], device="cuda"), torch.tensor([nk], dtype=torch.int32, device="cuda")
    (out, lse), most = used_by(lambda: layers.window_attention(q, k, v, cu_of([lq]), left=left, right=0, sinks=3, kv_start=start, kv_len=length, return_lse=True))
    assert most <= 160 << 20
    some = slice(lq - 40, lq)            # (the last queries, as a shorter prompt over the same keys, and the first ones)
    ref = exact(q[some], k[5:], v[5:], [40], [nk], left, 0, 3, [0])
    check(out[some], lse[some], ref)
    ref = exact(q[:40], k[5:], v[5:], [40], [nk - lq + 40], left, 0, 3, [0])
    check(out[:40], lse[:40], ref)


@pytest.mark.parametrize("heads,kv,dim,seqs,lq,nk", [(16, 2, 128, 70, 2, 20000), (32, 4, 128, 300, 4, 2100), (8, 8, 32, 1500, 1, 5000)])
def test_sequences_that_share_their_keys(layers, heads, kv, dim, seqs, lq, nk):
    """every sequence over the same cache: the keys are read far more often than there are of them"""
    q, k, v = normal(73, seqs * lq, heads, dim).bfloat16(), normal(74, nk, kv, dim).bfloat16(), normal(75, nk, kv, dim).bfloat16()
    start = torch.zeros(seqs, dtype=torch.int64, device="cuda")
    length = torch.full((seqs,), nk, dtype=torch.int32, device="cuda")
    for cut in (0, 2):                   # all alike; or of every length, some of them of none
        if cut:
            length[::3], length[1::7] = nk // 2, 0
        (out, lse), most = used_by(lambda: layers.window_attention(q, k, v, cu_of([lq] * seqs), kv_start=start, kv_len=length, return_lse=True))
        assert most <= 160 << 20
        for n in (nk, nk // 2, 0):
            at = (length == n).repeat_interleave(lq)
            if at.any():
                rows = int(at.sum())
                check(out[at][:200], lse[at][:200], exact(q[at][:200], k, v, [min(rows, 200)], [n], -1, -1, 0, [0]))
                check(out[at][-50:], lse[at][-50:], exact(q[at][-50:], k, v, [min(rows, 50)], [n], -1, -1, 0, [0]))


@pytest.mark.parametrize("heads,kv,dim", [(12, 12, 32), (4, 1, 128)])
def test_thousands_of_short_texts_without_a_window(layers, heads, kv, dim):
    """and one long text among them"""
    g = torch.Generator().manual_seed(9)
    nq = [int(n) for n in torch.randint(0, 51, (10000,), generator=g)]
    for long in (None, 7001):
        if long:
            nq[long] = 3000
        n = sum(nq)
        q, k, v = normal(76, n, heads, dim).bfloat16(), normal(77, n, kv, dim).bfloat16(), normal(78, n, kv, dim).bfloat16()
        (out, lse), most = used_by(lambda: layers.window_attention(q, k, v, cu_of(nq), return_lse=True))
        assert most <= (160 << 20) + 2 * out.numel() * 2
        for b in (0, 1, 63, 64, 65, 4999, 7000, 7001, 7002, 9998, 9999):
            f, c = sum(nq[:b]), nq[b]
            few = min(c, 60)
            check(out[f:f + few], lse[f:f + few], exact(q[f:f + few], k[f:f + c], v[f:f + c], [few], [c], -1, -1, 0, [0]))


def test_numbers_that_32_bits_cannot_hold(layers):
    from shodh_memory_amd import ShodhError
    q, k, v, cu = normal(1, 6, 4, 64).bfloat16(), normal(2, 6, 2, 64).bfloat16(), normal(3, 6, 2, 64).bfloat16(), cu_of([6])
    for kw in [dict(sinks=2 ** 32 + 4), dict(sinks=2 ** 32), dict(sinks=2 ** 31), dict(left=2 ** 31), dict(left=-2 ** 31 - 1), dict(right=2 ** 32), dict(scale=1e-46), dict(scale=-1e-60), dict(scale=1e39)]:
        with pytest.raises(ShodhError):
            layers.window_attention(q, k, v, cu, **kw)
    torch.cuda.synchronize()


def test_sequences_out_of_order_and_their_parts(layers):
    """a cu that is not rising: rows that one sequence alone claims are right, nothing outside them is touched"""
    q, k, v = normal(80, 6, 8, 128).bfloat16(), normal(81, 9000, 1, 128).bfloat16(), normal(82, 9000, 1, 128).bfloat16()
    start = torch.zeros(4, dtype=torch.int64, device="cuda")
    length = torch.full((4,), 9000, dtype=torch.int32, device="cuda")
    good = layers.window_attention(q, k, v, cu_of([4, 0, 0, 0]), kv_start=start, kv_len=length)
    for order in ([0, 4, 1, 2, 2], [0, 4, 0, -3, 9], [0, 4, 2, 3, 1]):
        out = torch.full_like(q, 5.0)
        layers.window_attention(q, k, v, torch.tensor(order, dtype=torch.int32, device="cuda"), kv_start=start, kv_len=length, out=out)
        assert torch.equal(out[0], good[0]) and torch.equal(out[3], good[3]) and (out[4:] == 5).all(), order
    torch.cuda.synchronize()


@needs_capture
def test_a_graph_whose_lengths_need_larger_parts(layers):
    """how many parts there are is found anew in every run: lengths that grow and shrink between replays, of a capture made at any of them"""
    seqs, heads, kv, dim, nk = 400, 32, 4, 128, 2500
    q, k, v = normal(83, seqs, heads, dim).bfloat16(), normal(84, nk, kv, dim).bfloat16(), normal(85, nk, kv, dim).bfloat16()
    start, cu = torch.zeros(seqs, dtype=torch.int64, device="cuda"), cu_of([1] * seqs)
    length = torch.full((seqs,), 40, dtype=torch.int32, device="cuda")

    def call():
        return layers.window_attention(q, k, v, cu, kv_start=start, kv_len=length, return_lse=True)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for i, n in enumerate((2500, 40, 1300, 0, 2500)):
        length.fill_(n)
        length[i::7] = 2500 - n
        want = call()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1]), n
        at = length == n
        check(want[0][at][:64], want[1][at][:64], exact(q[at][:64], k, v, [64], [n], -1, -1, 0, [0]))
