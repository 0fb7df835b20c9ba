"""The decoder-layer operators as a program runs them, one after the other.

Norm, query/key/value projection with adapters, head norms with rotation in
place on the projection's output, attention (plain torch, outside this
library), output projection with adapters, norm, router product, expert layer:
eagerly, and captured in one CUDA graph whose inputs change between replays.
Every stage is checked against its fp64 form on the inputs that it was given,
with the per-operator bounds of the operators' own tests.
"""

import numpy as np
import pytest
import torch

from flashattentionanycard_b200 import _native
from flashattentionanycard_b200.kernels import gemm, lora_gemm, moe_decode, qk_norm_rope, rmsnorm
from oracle import decoder
from tests.test_gpu_lora_gemm import Case
from tests.test_gpu_moe_decode import bound as moe_bound
from tests.test_gpu_qk_norm_rope import check_forward

pytestmark = pytest.mark.gpu

EPS = 1e-6
BF = torch.bfloat16


@pytest.fixture(autouse=True)
def clean_status(cuda_device):
    _native.device_status(reset=True)
    yield
    assert _native.device_status(reset=True)[0] == 0


def f64(t):
    return t.detach().cpu().double().numpy()


class Layer:
    def __init__(self, t, hidden=256, heads=4, kv_heads=2, d=64, experts=8, inner=136, topk=2):
        g = torch.Generator().manual_seed(t)
        self.t, self.heads, self.kv, self.d, self.topk = t, heads, kv_heads, d, topk
        self.qkv = Case(t, hidden, (heads + 2 * kv_heads) * d, 6, 16, seed=1)
        self.proj = Case(t, heads * d, hidden, 6, 8, seed=2)

        def randn(*shape, scale=1.0):
            return (torch.randn(*shape, generator=g) * scale).to(BF).cuda()

        self.norms = [1 + randn(hidden, scale=0.1) for _ in range(2)]
        self.q_weight, self.k_weight = 1 + randn(d, scale=0.1), 1 + randn(d, scale=0.1)
        self.router = randn(hidden, experts, scale=hidden**-0.5)
        self.w_gate_up = randn(experts, hidden, 2 * inner, scale=hidden**-0.5)
        self.w_down = randn(experts, inner, hidden, scale=inner**-0.5)
        self.table = qk_norm_rope.rope_table(512, d, device="cuda")
        self.positions = torch.randint(512, (t,), generator=g).to(torch.int32).cuda()
        self.x = randn(t, hidden)
        new = lambda *s: torch.empty(*s, dtype=BF, device="cuda")  # noqa: E731
        self.xn, self.xm, self.attn = new(t, hidden), new(t, hidden), new(t, heads * d)
        self.qkv_out, self.raw = new(t, (heads + 2 * kv_heads) * d), new(t, (heads + 2 * kv_heads) * d)
        self.o, self.logits, self.out = new(t, hidden), new(t, experts), new(t, hidden)

    def views(self):
        v = self.qkv_out.view(self.t, self.heads + 2 * self.kv, self.d)
        return v[:, :self.heads], v[:, self.heads:self.heads + self.kv], v[:, self.heads + self.kv:]

    def step(self):
        norm = {"ROWS_PER_CTA": 1, "num_warps": 4}
        rmsnorm.launch(self.x, self.norms[0], self.xn, norm, EPS)
        lora_gemm.launch(self.xn, self.qkv.w, self.qkv.bank, self.qkv.ids, self.qkv_out)
        self.raw.copy_(self.qkv_out)
        q, k, v = self.views()
        qk_norm_rope.launch(q, k, self.q_weight, self.k_weight, self.positions, self.table, q, k, EPS)
        # Every token attends to all (the mask is not this test's matter).
        rep = self.heads // self.kv
        kk, vv = k.float().repeat_interleave(rep, 1), v.float().repeat_interleave(rep, 1)
        p = torch.softmax(torch.einsum("thd,shd->hts", q.float(), kk) * self.d**-0.5, -1)
        self.attn.copy_(torch.einsum("hts,shd->thd", p, vv).reshape(self.t, -1))
        lora_gemm.launch(self.attn, self.proj.w, self.proj.bank, self.proj.ids, self.o)
        rmsnorm.launch(self.o, self.norms[1], self.xm, norm, EPS)
        gemm.launch(self.xm, self.router, self.logits, {})
        moe_decode.launch(self.xm, self.logits, self.w_gate_up, self.w_down, self.out, self.topk)

    def check(self):
        self.qkv.x, self.proj.x = self.xn, self.attn
        self.qkv.check(self.raw)
        raw = self.raw.view(self.t, -1, self.d)
        q, k, v = self.views()
        a = {"q": raw[:, :self.heads], "k": raw[:, self.heads:self.heads + self.kv], "q_weight": self.q_weight,
             "k_weight": self.k_weight, "positions": self.positions, "cos_sin": self.table}
        check_forward(a, q, k, "bf16")
        assert torch.equal(v, raw[:, self.heads + self.kv:])
        self.proj.check(self.o)
        ref, tol = moe_bound({"x": self.xm, "logits": self.logits, "w_gate_up": self.w_gate_up,
                              "w_down": self.w_down}, self.topk, True, "bf16")
        assert np.all(np.abs(f64(self.out) - ref) <= tol)


@pytest.mark.parametrize("t", [1, 7, 40, 128])
def test_eager(t, cuda_device):
    layer = Layer(t)
    layer.step()
    layer.check()


@pytest.mark.parametrize("t", [1, 40])
def test_captured_with_changing_inputs(t, cuda_device):
    layer = Layer(t)
    layer.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.step()
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        layer.x.copy_(torch.randn(layer.x.shape, generator=g).to(BF))
        layer.positions.copy_(torch.randint(512, (t,), generator=g).to(torch.int32))
        ids = torch.randint(-1, 6, (t,), generator=g).to(torch.int32)
        layer.qkv.ids.copy_(ids)
        layer.proj.ids.copy_(ids)
        graph.replay()
        torch.cuda.synchronize()
        layer.check()


def test_training_pair_of_norm_and_rotation(cuda_device):
    """Forward, then the gradients of a squared loss from its own output: the
    loss's change along a random direction of q, from differences of the fp64
    forward form, equals the gradient's product with it.

    The gradient is rounded to bf16 (2^-8 of each term) and its g = q_out is the
    rounded output (2^-8 more): 2^-7 of the sum of the terms' absolute values."""
    t, h, d = 20, 3, 64
    g = torch.Generator().manual_seed(0)
    q = torch.randn(t, h, d, generator=g).to(BF).cuda()
    k = q[:, :1].contiguous()
    w = torch.ones(d, dtype=BF, device="cuda")
    table = qk_norm_rope.rope_table(64, d, device="cuda")
    pos = torch.arange(t, dtype=torch.int32, device="cuda")
    target = torch.randn(t, h, d, generator=g).to(BF).cuda()
    q_out, k_out, dq, dk = (torch.empty_like(x) for x in (q, k, q, k))
    dw = [torch.empty(d, device="cuda") for _ in range(2)]
    qk_norm_rope.launch(q, k, w, w, pos, table, q_out, k_out, 1e-3)
    dout = (q_out.float() - target.float()).to(BF)
    qk_norm_rope.launch_backward(dout, torch.zeros_like(k), q, k, w, w, pos, table, dq, dk, dw[0], dw[1], 1e-3)

    def loss(x):
        y = decoder.qk_norm_rope(x, f64(w), np.arange(t), f64(table), 1e-3)
        return 0.5 * ((y - f64(target)) ** 2).sum()

    x, step = f64(q), 1e-6
    way = np.random.default_rng(0).normal(size=x.shape)
    slope = (loss(x + step * way) - loss(x - step * way)) / (2 * step)
    terms = f64(dq) * way
    size = (np.abs(f64(dout)) + np.abs(f64(q_out)) * 2.0**-8).max() * np.abs(way).sum()
    assert abs(terms.sum() - slope) <= 2.0**-7 * size
    assert not dk.any() and not dw[1].any()


def test_operators_of_several_streams_at_once(cuda_device):
    """Persistent, clustered and small kernels of five streams share the SMs;
    every result keeps its bits."""
    from tests import test_gpu_moe_decode as moe

    cases = []
    for t, e, k, inner, topk in ((1, 8, 512, 1024, 2), (12, 16, 264, 520, 3), (90, 30, 256, 768, 5), (128, 64, 512, 256, 8)):
        a = moe.make(t, e, k, inner, seed=t)
        cases.append(lambda a=a, topk=topk: moe.run(a, topk))
    for t in (5, 200, 900):
        c = Case(t, 512, 1032, 9, 24, seed=t)
        cases.append(c.run)
    layer = Layer(60)
    a, b = torch.randn(300, 512, device="cuda").to(BF), torch.randn(512, 264, device="cuda").to(BF)
    odd = torch.randn(37, 77, device="cuda").to(BF), torch.randn(77, 93, device="cuda").to(BF)

    def product(x, w):
        out = torch.empty(x.shape[0], w.shape[1], dtype=BF, device="cuda")
        gemm.launch(x, w, out, {})
        return out

    cases += [lambda: product(a, b), lambda: product(*odd)]
    layer.step()
    want = [c() for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(5)]
    got = []
    for turn in range(6):
        for i, c in enumerate(cases):
            s = streams[(i + turn) % len(streams)]
            with torch.cuda.stream(s):
                got.append((i, c()))
    torch.cuda.synchronize()
    for i, out in got:
        assert torch.equal(out, want[i]), i


def test_training_pair_along_its_own_gradient(cuda_device):
    """As above, along the fp64 gradient with noise, where a gradient of zero or
    of the wrong sign is far off.

    dq is rounded (2^-8 of every term).  Its g is rounded twice, as q_out and as
    the difference: 2^-8 (|q_out| + |g|) of every element, which moves the slope
    by its product with the forward form's change along the direction."""
    t, h, d = 20, 3, 64
    g = torch.Generator().manual_seed(0)
    q = torch.randn(t, h, d, generator=g).to(BF).cuda()
    k = q[:, :1].contiguous()
    w = (1 + 0.2 * torch.randn(d, generator=g)).to(BF).cuda()
    table = qk_norm_rope.rope_table(64, d, device="cuda")
    pos = torch.arange(t, dtype=torch.int32, device="cuda")
    target = torch.randn(t, h, d, generator=g).to(BF).cuda()
    q_out, k_out, dq, dk = (torch.empty_like(x) for x in (q, k, q, k))
    dw = [torch.empty(d, device="cuda") for _ in range(2)]
    qk_norm_rope.launch(q, k, w, w, pos, table, q_out, k_out, 1e-3)
    dout = (q_out.float() - target.float()).to(BF)
    qk_norm_rope.launch_backward(dout, torch.zeros_like(k), q, k, w, w, pos, table, dq, dk, dw[0], dw[1], 1e-3)

    def form(x, weight):
        return decoder.qk_norm_rope(x, weight, np.arange(t), f64(table), 1e-3)

    x, weight, goal, step = f64(q), f64(w), f64(target), 1e-6
    rng = np.random.default_rng(0)
    full = decoder.qk_norm_rope_backward(form(x, weight) - goal, x, weight, np.arange(t), f64(table), 1e-3)
    round_g = 2.0**-8 * (np.abs(f64(q_out)) + np.abs(f64(dout)))
    for mine, grad, move, rounding in ((f64(dq), full[0], lambda s, way: form(x + s * way, weight), 2.0**-8),
                                       (f64(dw[0]), full[1], lambda s, way: form(x, weight + s * way), 1e-5)):
        way = grad + 0.3 * np.sqrt((grad * grad).mean()) * rng.normal(size=grad.shape)
        up, down = move(step, way), move(-step, way)
        slope = 0.5 * (((up - goal) ** 2).sum() - ((down - goal) ** 2).sum()) / (2 * step)
        tol = rounding * np.abs(mine * way).sum() + (round_g * np.abs(up - down)).sum() / (2 * step) + 1e-4
        assert abs((mine * way).sum() - slope) <= tol
        assert abs(slope) > 4 * tol  # zero, or the other sign, would not pass
