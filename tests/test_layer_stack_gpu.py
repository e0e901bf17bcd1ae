"""The layer operators one after another, as a text tower would run them (GPU): norm with 8-bit rows -> q|k|v on 4-bit weights -> attention -> output product ->
norm with the residual and 8-bit rows -> up and down on 4-bit weights -> norm; then the same for single tokens over a cache that the first run filled. Each operator's
result is compared with its definition in 64 bits on what it was given, within the tolerance of its own tests: so no error of one hides in the next one's."""
import pytest
import torch

from . import test_dense_w4_gpu as W4
from . import test_rms_norm_gpu as NORM
from . import test_window_attention_gpu as ATTN
from .conftest import needs_capture

pytestmark = pytest.mark.gpu
HEADS, KV, DIM, HIDDEN, UP = 6, 2, 64, 392, 1000


@pytest.fixture(scope="module")
def layers():
    from shodh_memory_amd import layers
    return layers


class Dense:
    def __init__(self, layers, n, k, group, zeros, seed):
        self.group, self.bias = group, 0.1 * ATTN.normal(seed, n)
        self.q, packed, self.scale, self.z = W4.make(n, k, group, zeros, seed)
        self.w = layers.W4Weight.from_quantized(packed, self.scale, self.z, k=k, group=group)

    def __call__(self, x, xs=None, dtype=None):
        return self.w.dense(x, x_scale=xs, bias=self.bias, out_dtype=dtype)

    def check(self, got, x, xs=None):
        y, t = W4.exact(x, xs, self.q, self.scale, self.z, self.bias, self.group)
        W4.check(got, y, t, x.dtype, self.q.shape[1], self.group)


class Block:
    def __init__(self, layers, dtype):
        self.layers, self.dtype = layers, dtype
        self.norms = [(1 + 0.2 * ATTN.normal(50 + i, HIDDEN)).to(dtype) for i in range(3)]
        self.qkv = Dense(layers, (HEADS + 2 * KV) * DIM, HIDDEN, 128, True, 60)
        self.out = Dense(layers, HIDDEN, HEADS * DIM, 64, False, 61)
        self.up = Dense(layers, UP, HIDDEN, 32, True, 62)
        self.down = Dense(layers, HIDDEN, UP, 128, False, 63)

    def __call__(self, x, attend):
        L, s = self.layers, {"x": x}
        s["n1"] = L.rms_norm(x, self.norms[0], want_y=False, quant="int8")
        s["qkv"] = self.qkv(s["n1"].q, s["n1"].scale, self.dtype)
        s["attn"], s["lse"] = attend(s["qkv"].view(-1, HEADS + 2 * KV, DIM))
        s["out"] = self.out(s["attn"].view(-1, HEADS * DIM))
        s["n2"] = L.rms_norm(s["out"], self.norms[1], residual=x, quant="int8")
        s["up"] = self.up(s["n2"].q, s["n2"].scale, self.dtype)
        s["down"] = self.down(s["up"])
        s["n3"] = L.rms_norm(s["down"], self.norms[2], residual=s["n2"].sum)
        return s

    def check(self, s, attention):
        def normed(r, x, w, residual=None, quant=False):
            h, y = NORM.defined(x, w, residual, 1e-6)
            if r.y is not None:
                NORM.check_rounded(r.y, y, self.dtype, 70 * NORM.U)
            if residual is not None:
                NORM.check_rounded(r.sum, h, self.dtype, NORM.U)
            if quant:
                NORM.check_q(r, y, 0, "int8")
        normed(s["n1"], s["x"], self.norms[0], quant=True)
        self.qkv.check(s["qkv"], s["n1"].q, s["n1"].scale.view(-1))
        ATTN.check(s["attn"], s["lse"], attention(s["qkv"].view(-1, HEADS + 2 * KV, DIM)))
        self.out.check(s["out"], s["attn"].view(-1, HEADS * DIM))
        normed(s["n2"], s["out"], self.norms[1], residual=s["x"], quant=True)
        self.up.check(s["up"], s["n2"].q, s["n2"].scale.view(-1))
        self.down.check(s["down"], s["up"])
        normed(s["n3"], s["down"], self.norms[2], residual=s["n2"].sum)


def parts(qkv):
    return qkv[:, :HEADS], qkv[:, HEADS:HEADS + KV], qkv[:, HEADS + KV:]


@pytest.mark.parametrize("captured", [False, pytest.param(True, marks=needs_capture)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_block_on_texts_then_on_single_tokens(layers, dtype, captured):
    block = Block(layers, dtype)
    nq, left, sinks = [70, 1, 150, 0, 33], 40, 3
    tokens, room = sum(nq), 8
    x = ATTN.normal(70, tokens, HIDDEN).to(dtype)
    cu = ATTN.cu_of(nq)
    s = block(x, lambda qkv: layers.window_attention(*parts(qkv), cu, left=left, right=0, sinks=sinks, return_lse=True))
    block.check(s, lambda qkv: ATTN.exact(*parts(qkv), nq, nq, left, 0, sinks))

    # the texts' keys and values become a cache with room behind each; every sequence goes on by one token a step (the step captured once, or not)
    starts = [sum(nq[:i]) + room * i for i in range(len(nq))]
    total = tokens + room * len(nq)
    ck, cv = (torch.full((total, KV, DIM), float("nan"), device="cuda", dtype=dtype) for _ in range(2))
    at = 0
    for f, n in zip(starts, nq):
        ck[f:f + n], cv[f:f + n] = parts(s["qkv"].view(-1, HEADS + 2 * KV, DIM)[at:at + n])[1:]
        at += n
    start = torch.tensor(starts, device="cuda")
    length = torch.tensor(nq, dtype=torch.int32, device="cuda")
    one = ATTN.cu_of([1] * len(nq))
    xt = torch.zeros(len(nq), HIDDEN, device="cuda", dtype=dtype)

    def attend(qkv):
        q, k, v = parts(qkv)
        place = start + length
        ck.index_copy_(0, place, k)
        cv.index_copy_(0, place, v)
        return layers.window_attention(q, ck, cv, one, left=left, right=0, sinks=sinks, kv_start=start, kv_len=length + 1, return_lse=True)
    if captured:
        block(xt, attend)                     # (written over by the first step)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = block(xt, attend)
    lens = list(nq)
    for step in range(4):
        xt.copy_(ATTN.normal(80 + step, len(nq), HIDDEN).to(dtype))
        if captured:
            graph.replay()
        else:
            held = block(xt, attend)
        torch.cuda.synchronize()
        lens = [n + 1 for n in lens]
        block.check(held, lambda qkv: ATTN.exact(parts(qkv)[0], ck, cv, [1] * len(nq), lens, left, 0, sinks, starts))
        eager = block(xt, attend)
        for name in ("qkv", "attn", "lse", "out", "up", "down"):
            assert torch.equal(eager[name], held[name]), name
        assert torch.equal(eager["n3"].y, held["n3"].y) and torch.equal(eager["n3"].sum, held["n3"].sum)
        length += 1
        torch.cuda.synchronize()


def test_inputs_that_require_a_gradient(layers):
    """no gradient is lost without a word: such inputs are refused while torch records, and taken where it does not"""
    from shodh_memory_amd import ShodhError
    w4 = layers.W4Weight.quantize(torch.randn(32, 64), group=32)
    x, g, bias = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda"), torch.zeros(32, device="cuda")
    q, k, v, cu = ATTN.normal(1, 4, 2, 32).half(), ATTN.normal(2, 4, 1, 32).half(), ATTN.normal(3, 4, 1, 32).half(), ATTN.cu_of([4])

    def leaf(t):
        return t.clone().requires_grad_()
    calls = [lambda: layers.rms_norm(leaf(x), g).y, lambda: layers.rms_norm(x, torch.nn.Parameter(g)).y, lambda: layers.rms_norm(x, g, residual=leaf(x)).y, lambda: w4.dense(leaf(x)), lambda: w4.dense(x, bias=leaf(bias)),
             lambda: w4.dense((2 * leaf(x)).half()), lambda: layers.window_attention(leaf(q), k, v, cu), lambda: layers.window_attention(q, leaf(k), v, cu), lambda: layers.window_attention(q, k, leaf(v), cu)]
    plain = [layers.rms_norm(x, g).y, layers.rms_norm(x, g).y, layers.rms_norm(x, g, residual=x).y, w4.dense(x), w4.dense(x, bias=bias), w4.dense((2 * x).half())] + [layers.window_attention(q, k, v, cu)] * 3
    for call, want in zip(calls, plain):
        with pytest.raises(ShodhError):
            call()
        with torch.no_grad():
            assert torch.equal(call(), want)
        with torch.inference_mode():
            assert torch.equal(call(), want)
    for call in [lambda: layers.rms_norm(x, g, residual=x, sum_out=leaf(x)), lambda: w4.dense(x, out=leaf(x[:, :32])), lambda: layers.window_attention(q, k, v, cu, out=leaf(q))]:
        with pytest.raises(ShodhError):
            call()
