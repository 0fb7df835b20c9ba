"""Query/key norm + rotation, forward and backward, against the fp64 form.

Tolerances.  The forward result is rounded once (half a step, eps / 2 of the
value; fp16 below its normal range half a subnormal step, 2^-25).  Before that,
in fp32 (u = 2^-24): the mean of D squares is a sum of positive terms, at most
D / 8 + 13 roundings deep on any path (8 per lane, then shuffles; 32 per lane
in the strided kernel), so relative error (D / 8 + 13) u / 2 after the root;
rsqrt 2 ulp; two products; the rotation two more on each of its two terms.
That is under (D / 16 + 20) u of |y_a| + |y_b|.  Backward: the same per factor
and a mean of D products (D / 8 + 13 deep, of their absolute values); under
(D / 4 + 64) u of r (|g w| + |n| mean |g w n|).  A weight gradient adds at most
rows + 64 terms in sequence: (rows + 64 + D / 16 + 20) u of the sum of |g n|.
"""

import numpy as np
import pytest
import torch

from flashattentionanycard_b200 import _native
from flashattentionanycard_b200.kernels import qk_norm_rope
from oracle import decoder

pytestmark = pytest.mark.gpu

U = 2.0**-24
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
SUB = {"bf16": 2.0**-134, "fp16": 2.0**-25}


@pytest.fixture(autouse=True)
def clean_status(cuda_device):
    _native.device_status(reset=True)
    yield
    assert _native.device_status(reset=True)[0] == 0


def f64(t):
    return t.detach().cpu().double().numpy()


def make(t, h, hk, d, rot, dtype, seed=0, table=64, packed=True, pad=0, i64=False, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    dt = DTYPES[dtype]
    qkv = torch.randn(t, h + 2 * hk, d + pad, generator=g).to(dt).to(device)
    q, k = qkv[:, :h, :d], qkv[:, h:h + hk, :d]
    if not packed:
        q, k = q.contiguous(), k.contiguous()
    pos = torch.randint(table, (t,), generator=g)
    return {"q": q, "k": k, "q_weight": (1 + 0.2 * torch.randn(d, generator=g)).to(dt).to(device),
            "k_weight": (1 + 0.2 * torch.randn(d, generator=g)).to(dt).to(device),
            "positions": pos.to(torch.int64 if i64 else torch.int32).to(device),
            "cos_sin": torch.from_numpy(decoder.rope_table(table, rot)).float().to(device)}, g


def check_forward(a, q_out, k_out, dtype, eps=1e-6, interleaved=False, rows=slice(None)):
    d = a["q"].shape[2]
    half = torch.finfo(DTYPES[dtype]).eps / 2
    for x, w, out in ((a["q"], a["q_weight"], q_out), (a["k"], a["k_weight"], k_out)):
        pos, cs = f64(a["positions"]).astype(int)[rows], f64(a["cos_sin"])
        x, w = f64(x)[rows], f64(w)
        ref = decoder.qk_norm_rope(x, w, pos, cs, eps, interleaved)
        y = np.abs(x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w)
        near = y + y[..., partner(d, cs.shape[1], interleaved)]
        err = np.abs(f64(out)[rows] - ref)
        assert np.all(err <= half * np.abs(ref) * (1 + 1e-3) + SUB[dtype] + (d / 16 + 20) * U * near)


def partner(d, rot, interleaved):
    p = np.arange(d)
    a, b = decoder._pairs(rot, interleaved)
    p[a], p[b] = b, a
    return p


def forward(a, interleaved=False, eps=1e-6):
    q_out = torch.full_like(a["q"].contiguous(), float("nan"))
    k_out = torch.full_like(a["k"].contiguous(), float("nan"))
    qk_norm_rope.launch(**a, q_out=q_out, k_out=k_out, epsilon=eps, interleaved=interleaved)
    return q_out, k_out


SHAPES = [
    # t, h, hk, d, rot
    (1, 32, 8, 128, 128), (1, 1, 1, 8, 2), (7, 3, 1, 64, 64), (130, 5, 2, 80, 32), (33, 6, 3, 256, 64),
    (19, 4, 4, 200, 200), (600, 33, 9, 128, 96), (5, 2, 1, 2, 2), (9, 3, 2, 37, 36), (11, 2, 1, 300, 130),
    (3, 2, 2, 1024, 512), (64, 17, 1, 24, 16), (2500, 8, 2, 96, 48),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(shape, dtype, interleaved, cuda_device):
    a, _ = make(*shape, dtype, seed=sum(shape), i64=shape[0] % 2 == 0)
    q_out, k_out = forward(a, interleaved)
    check_forward(a, q_out, k_out, dtype, interleaved=interleaved)


def backward(a, dq_out, dk_out, interleaved=False, eps=1e-6, dq=None, dk=None):
    d = a["q"].shape[2]
    dq = torch.full_like(dq_out, float("nan")) if dq is None else dq
    dk = torch.full_like(dk_out, float("nan")) if dk is None else dk
    dw = [torch.full((d,), float("nan"), device=dq.device) for _ in range(2)]
    qk_norm_rope.launch_backward(dq_out, dk_out, **a, dq=dq, dk=dk, dq_weight=dw[0], dk_weight=dw[1],
                                 epsilon=eps, interleaved=interleaved)
    return dq, dk, dw[0], dw[1]


def check_backward(a, grads, got, dtype, eps=1e-6, interleaved=False):
    d = a["q"].shape[2]
    half = torch.finfo(DTYPES[dtype]).eps / 2
    pos, cs = f64(a["positions"]).astype(int), f64(a["cos_sin"])
    for x, w, g, dx, dw in ((a["q"], a["q_weight"], grads[0], got[0], got[2]),
                            (a["k"], a["k_weight"], grads[1], got[1], got[3])):
        x, w, g = f64(x), f64(w), f64(g)
        ref, dref = decoder.qk_norm_rope_backward(g, x, w, pos, cs, eps, interleaved)
        r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        n = np.abs(x * r)
        ga = np.abs(g) + np.abs(g)[..., partner(d, cs.shape[1], interleaved)]
        gw = ga * np.abs(w)
        scale = r * (gw + n * (gw * n).mean(-1, keepdims=True))
        assert np.all(np.abs(f64(dx) - ref) <= half * np.abs(ref) * (1 + 1e-3) + SUB[dtype]
                      + (d / 4 + 64) * U * scale)
        depth = x.shape[0] * x.shape[1] + 84 + d / 16
        assert np.all(np.abs(f64(dw) - dref) <= depth * U * (ga * n).sum((0, 1)))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(shape, dtype, interleaved, cuda_device):
    a, g = make(*shape, dtype, seed=sum(shape))
    grads = [torch.randn(*a[n].shape, generator=g).to(DTYPES[dtype]).to(cuda_device) for n in ("q", "k")]
    got = backward(a, *grads, interleaved)
    check_backward(a, grads, got, dtype, interleaved=interleaved)
    again = backward(a, *grads, interleaved)
    assert all(torch.equal(x, y) for x, y in zip(got, again))  # fixed order of sums


def test_backward_against_differences(cuda_device):
    """d loss / d x[i] from the forward form's differences; bf16 rounding of dx
    (2^-8) and the differences' own error (1e-6) bound the distance."""
    a, g = make(2, 2, 1, 16, 16, "bf16", seed=5)
    grads = [torch.randn(*a[n].shape, generator=g).bfloat16().to(cuda_device) for n in ("q", "k")]
    dq = f64(backward(a, *grads)[0])
    pos, cs, w, x = f64(a["positions"]).astype(int), f64(a["cos_sin"]), f64(a["q_weight"]), f64(a["q"])
    step = 1e-5
    for i in np.ndindex(x.shape):
        e = np.zeros_like(x)
        e[i] = step
        up, down = (decoder.qk_norm_rope(x + s * e, w, pos, cs, 1e-6) for s in (1, -1))
        want = ((up - down) * f64(grads[0])).sum() / (2 * step)
        assert abs(dq[i] - want) <= 2.0**-8 * abs(want) + 1e-5


@pytest.mark.parametrize("pad", [0, 8, 3])
def test_strided_in_place_and_neighbours_untouched(pad, cuda_device):
    t, h, hk, d, rot = 21, 4, 2, 64, 32
    a, _ = make(t, h, hk, d, rot, "bf16", seed=pad, pad=pad)
    want = forward(a)
    base = a["q"]._base.clone()
    qkv = base.clone()
    q, k = qkv[:, :h, :d], qkv[:, h:h + hk, :d]
    qk_norm_rope.launch(q, k, a["q_weight"], a["k_weight"], a["positions"], a["cos_sin"], q, k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(qkv[:, h + hk:], base[:, h + hk:]) and torch.equal(qkv[..., d:], base[..., d:])


def test_backward_in_place_gradient(cuda_device):
    a, g = make(50, 6, 2, 128, 128, "bf16")
    grads = [torch.randn(*a[n].shape, generator=g).bfloat16().to(cuda_device) for n in ("q", "k")]
    want = backward(a, *grads)
    got = backward(a, *grads, dq=grads[0], dk=grads[1])
    assert all(torch.equal(x, y) for x, y in zip(want, got))


def test_broadcast_input_and_head_major_layout(cuda_device):
    """An input may repeat memory (expanded) and lie head-major; the output too."""
    a, g = make(40, 4, 4, 64, 64, "bf16", packed=False)
    one = a["q"][:, :1]
    a["q"] = one.expand(-1, 4, -1)
    a["k"] = a["k"].transpose(0, 1).contiguous().transpose(0, 1)
    q_out = torch.empty(4, 40, 64, dtype=torch.bfloat16, device=cuda_device).transpose(0, 1)
    k_out = torch.empty_like(a["k"])
    qk_norm_rope.launch(**a, q_out=q_out, k_out=k_out)
    check_forward(a, q_out, k_out, "bf16")


@pytest.mark.parametrize("t, h, hk", [(0, 4, 2), (5, 0, 2), (5, 3, 0)])
def test_empty(t, h, hk, cuda_device):
    d = 32
    a, g = make(t, h, hk, d, d, "bf16")
    q_out, k_out = forward(a)
    check_forward(a, q_out, k_out, "bf16")
    grads = [torch.randn(*a[n].shape, generator=g).bfloat16().to(cuda_device) for n in ("q", "k")]
    got = backward(a, *grads)
    if t * h == 0:
        assert torch.equal(got[2], torch.zeros_like(got[2]))
    if t * hk == 0:
        assert torch.equal(got[3], torch.zeros_like(got[3]))


def test_positions_outside_the_table_are_reported_and_skipped(cuda_device):
    for d in (64, 37):
        a, g = make(9, 3, 2, d, 16, "bf16", table=20)
        a["positions"][2], a["positions"][6] = -1, 20
        q_out, k_out = forward(a)
        torch.cuda.synchronize()
        assert _native.device_status(reset=True) in ((5, 2), (5, 6))
        bad = [2, 6]
        good = [i for i in range(9) if i not in bad]
        assert torch.isnan(q_out[bad]).all() and torch.isnan(k_out[bad]).all()
        check_forward(a, q_out, k_out, "bf16", rows=good)
        grads = [torch.randn(*a[n].shape, generator=g).bfloat16().to(cuda_device) for n in ("q", "k")]
        got = backward(a, *grads)
        assert _native.device_status(reset=True)[0] == 5
        assert torch.isnan(got[0][bad]).all() and torch.isfinite(got[2]).all()
        sub = {k: (v[good] if v.shape[0] == 9 and k in ("q", "k", "positions") else v) for k, v in a.items()}
        check_backward(sub, [x[good] for x in grads], (got[0][good], got[1][good], got[2], got[3]), "bf16")


def test_values_that_are_not_finite_stay_in_their_row(cuda_device):
    a, _ = make(6, 3, 1, 64, 32, "bf16")
    clean = forward(a)
    a["q"][2, 1, 5] = float("inf")
    a["q"][3, 0, 0] = float("nan")
    a["q"][4, 2] = 0
    got = forward(a)
    keep = torch.ones(6, 3, dtype=torch.bool)
    keep[2, 1] = keep[3, 0] = keep[4, 2] = False
    assert torch.equal(got[0][keep], clean[0][keep]) and torch.equal(got[1], clean[1])
    # x / inf is 0, inf / inf is NaN; past rot nothing mixes.
    assert torch.isnan(got[0][3, 0]).all() and torch.isnan(got[0][2, 1, 5])
    assert torch.equal(got[0][2, 1, 32:], torch.zeros_like(got[0][2, 1, 32:]))
    assert torch.equal(got[0][4, 2], torch.zeros_like(got[0][4, 2]))


def test_other_stream_graph_and_two_graphs(cuda_device):
    a, g = make(300, 8, 2, 128, 128, "bf16")
    grads = [torch.randn(*a[n].shape, generator=g).bfloat16().to(cuda_device) for n in ("q", "k")]
    want, wantg = forward(a), backward(a, *grads)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = forward(a)
    side.synchronize()
    assert torch.equal(got[0], want[0])
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append((forward(a), backward(a, *grads)))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for f, b in outs:
        assert torch.equal(f[0], want[0]) and torch.equal(f[1], want[1])
        assert all(torch.equal(x, y) for x, y in zip(b, wantg))


def test_rope_table(cuda_device):
    """fp64 angles: one fp32 rounding (2^-24 of at most 1) plus fp64 dust, at
    positions whose fp32 angle would be off by whole turns' fractions too."""
    rows, rot = 200_000, 64
    got = qk_norm_rope.rope_table(rows, rot, 500000.0, cuda_device)
    assert np.abs(f64(got) - decoder.rope_table(rows, rot, 500000.0)).max() <= U + 1e-9
    assert qk_norm_rope.rope_table(0, 8, device=cuda_device).shape == (0, 8)


def test_offsets_past_32_bits(cuda_device):
    """Token rows 2^31 elements apart and more."""
    t, h, d = 3, 2, 64
    far = (1 << 30) + 64
    base = torch.empty(far * 2 + 4096, dtype=torch.bfloat16, device=cuda_device)
    q = base.as_strided((t, h, d), (far, d, 1))
    k = base.as_strided((t, 1, d), (far, d, 1), 2 * d + 1024)
    a, _ = make(t, h, 1, d, d, "bf16")
    want = forward(a)
    q.copy_(a["q"])
    k.copy_(a["k"])
    qk_norm_rope.launch(q, k, a["q_weight"], a["k_weight"], a["positions"], a["cos_sin"], q, k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


@pytest.mark.parametrize("shape", [(7, 3, 1, 64, 64), (130, 5, 2, 80, 32), (2500, 7, 3, 96, 48), (9, 3, 2, 37, 36)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_no_epsilon(shape, interleaved, cuda_device):
    """Heads that do not fill a unit: its idle rows must add nothing where
    rsqrt(0 + epsilon) is infinite."""
    a, g = make(*shape, "bf16", seed=3)
    q_out, k_out = forward(a, interleaved, eps=0.0)
    check_forward(a, q_out, k_out, "bf16", eps=0.0, interleaved=interleaved)
    grads = [torch.randn(a[n].shape, generator=g).bfloat16().cuda() for n in ("q", "k")]
    got = backward(a, *grads, interleaved=interleaved, eps=0.0)
    check_backward(a, grads, got, "bf16", eps=0.0, interleaved=interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("t, d, rot", [(6, 64, 32), (6, 80, 16), (700, 256, 64), (5, 37, 12)])
def test_infinities_past_the_rotation_stay_in_their_column(t, d, rot, interleaved, cuda_device):
    """Past rot nothing mixes: an infinity there reaches no other column, in
    either form of the pairs, from the values, the weights or the gradient."""
    h, col = 20 if t > 100 else 3, rot + 3
    a, g = make(t, h, 1, d, rot, "bf16")
    a["q"], a["k"] = a["q"].contiguous(), a["k"].contiguous()
    grads = [torch.randn(*a[n].shape, generator=g).bfloat16().to(cuda_device) for n in ("q", "k")]
    others = [c for c in range(d) if c != col]
    clean, clean_grad = forward(a, interleaved), backward(a, *grads, interleaved)

    bad = {**a, "q": a["q"].clone()}
    bad["q"][2, 1, col] = float("inf")  # x / inf is 0, inf / inf is NaN
    out = forward(bad, interleaved)[0]
    assert torch.equal(out[2, 1, others], torch.zeros_like(out[2, 1, others])) and torch.isnan(out[2, 1, col])
    # Backward the row's statistics are gone; it adds to no other column of the weights' gradient.
    silent = [grads[0].clone(), grads[1]]
    silent[0][2, 1] = 0
    without, got = backward(a, *silent, interleaved)[2], backward(bad, *grads, interleaved)
    assert torch.equal(got[2][others], without[others]) and torch.isnan(got[2][col])

    bad = {**a, "q_weight": a["q_weight"].clone()}
    bad["q_weight"][col] = float("inf")
    out = forward(bad, interleaved)[0]
    assert torch.equal(out[..., others], clean[0][..., others]) and torch.isinf(out[..., col]).all()

    grads[0][2, 1, col] = float("inf")
    got = backward(a, *grads, interleaved)
    assert torch.equal(got[2][others], clean_grad[2][others]) and torch.isinf(got[2][col])
    assert torch.equal(got[1], clean_grad[1]) and torch.equal(got[3], clean_grad[3])
    rows = torch.ones(t, h, dtype=torch.bool)
    rows[2, 1] = False
    assert torch.equal(got[0][rows], clean_grad[0][rows])


def test_outputs_over_other_operands_are_refused(cuda_device):
    """Any memory in common but a side's own view, whole, is an error, and nothing runs."""
    t, h, hk, d = 30, 4, 2, 64
    a, g = make(t, h, hk, d, d, "bf16")
    want = forward(a)
    buf = torch.zeros(4 * t, h + hk, d, dtype=torch.bfloat16, device=cuda_device)
    q_out, k_out = buf[:t, :h], buf[:t, h:]
    shifted = a["q"]._base[1:, :h], a["q"]._base[1:, h:h + hk]
    for over in (dict(k_out=buf[:t, 1:1 + hk]), dict(k_out=buf[1:1 + t, :hk]), dict(q_out=a["q"]._base[:, hk:h + hk]),
                 dict(k_out=a["q"][:, :hk]), dict(q_out=a["q"]._base[:, 1:1 + h]), dict(k_out=q_out[:, 2:])):
        before = a["q"]._base.clone(), buf.clone()
        with pytest.raises(ValueError, match="must not overlap"):
            qk_norm_rope.launch(**{**a, "q_out": q_out, "k_out": k_out, **over})
        assert torch.equal(a["q"]._base, before[0]) and torch.equal(buf, before[1])
    short = {**a, "q": a["q"][:-1], "k": a["k"][:-1], "positions": a["positions"][:-1]}
    for over in (dict(q_out=shifted[0]), dict(k_out=shifted[1])):
        with pytest.raises(ValueError, match="must not overlap"):
            qk_norm_rope.launch(**{**short, "q_out": q_out[:-1], "k_out": k_out[:-1], **over})
    grads = [torch.randn(*a[n].shape, generator=g).bfloat16().to(cuda_device) for n in ("q", "k")]
    dw = [torch.empty(d, device=cuda_device) for _ in range(2)]
    into = dict(dq_out=grads[0], dk_out=grads[1], dq=q_out, dk=k_out, dq_weight=dw[0], dk_weight=dw[1])
    for over in (dict(dk=grads[0][:, :hk]), dict(dq=a["q"]._base[:, hk:h + hk]), dict(dk=q_out[:, 1:1 + hk]),
                 dict(dq_weight=buf.flatten()[2 * d:4 * d].view(torch.float32)),
                 dict(dk_weight=buf.flatten()[h * d:(h + 2) * d].view(torch.float32))):
        with pytest.raises(ValueError, match="must not overlap"):
            qk_norm_rope.launch_backward(**{**a, **into, **over})
    # Beside each other in one buffer they are taken.
    qk_norm_rope.launch(**a, q_out=q_out, k_out=k_out)
    assert torch.equal(q_out, want[0]) and torch.equal(k_out, want[1]) and not buf[t:].any()


@pytest.mark.parametrize("d", [128, 37])
def test_gradient_over_the_values(d, cuda_device):
    a, g = make(300, 6, 2, d, 16, "bf16")
    grads = [torch.randn(*a[n].shape, generator=g).bfloat16().to(cuda_device) for n in ("q", "k")]
    want = backward(a, *grads)
    got = backward(a, *grads, dq=a["q"], dk=a["k"])
    assert all(torch.equal(x, y) for x, y in zip(want, got))


def test_two_heads_per_side_in_every_layout(cuda_device):
    """q, k and v beside each other in every head, in place; heads in front of tokens."""
    t, h, d = 50, 4, 64
    a, _ = make(t, h, h, d, 32, "bf16", packed=False)
    want = forward(a)
    for shape, order in (((t, h, 3, d), (2, 0, 1, 3)), ((h, t, 3, d), (2, 1, 0, 3)), ((3, h, t, d), (0, 2, 1, 3))):
        buf = torch.zeros(shape, dtype=torch.bfloat16, device=cuda_device)
        q, k, v = buf.permute(order)
        q.copy_(a["q"])
        k.copy_(a["k"])
        qk_norm_rope.launch(q, k, a["q_weight"], a["k_weight"], a["positions"], a["cos_sin"], q, k)
        assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and not v.any()


def torch_forms(a, side, g, interleaved, eps=1e-6):
    """fp64 on the GPU, apart from the kernels and from the oracle's indexing:
    (forward, gradient of x, gradient of w, and the sums of absolute values that
    the bounds are taken from), heads of one side."""
    x, w, g = a[side].double(), a[side + "_weight"].double(), g.double()
    d, rot = x.shape[2], a["cos_sin"].shape[1]
    cs = a["cos_sin"].double()[a["positions"].long()][:, None]
    turn = torch.complex(cs[..., : rot // 2], cs[..., rot // 2:])

    def rotate(v, by, size=False):
        z = v[..., :rot]
        lo, hi = (z[..., 0::2], z[..., 1::2]) if interleaved else z.split(rot // 2, -1)
        if size:
            lo = hi = lo.abs() + hi.abs()
        else:
            z = torch.complex(lo, hi) * by
            lo, hi = z.real, z.imag
        z = torch.stack([lo, hi], -1).flatten(-2) if interleaved else torch.cat([lo, hi], -1)
        rest = v[..., rot:]
        return torch.cat([z, 2 * rest.abs() if size else rest], -1)

    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = x * r
    back = rotate(g, turn.conj())
    gw, ga = back * w, rotate(g, None, size=True)
    dx = r * (gw - n * (gw * n).mean(-1, keepdim=True))
    gaw = ga * w.abs()
    size = r * (gaw + n.abs() * (gaw * n.abs()).mean(-1, keepdim=True))
    return rotate(n * w, turn), rotate(n * w, None, size=True), dx, size, (back * n).sum((0, 1)), (ga * n.abs()).sum((0, 1))


def close(got, ref, tol):
    assert got.shape == ref.shape and bool(((got.double() - ref).abs() <= tol).all())


# Enough head rows that a warp takes two or four batches of a token's heads
# behind one load of the angles, on 8, 16 and 32 lanes a row; heads that do not
# fill the batches.
MANY = [(16500, 9, 3, 128, 96), (30100, 17, 3, 64, 32), (22000, 5, 2, 256, 64), (21900, 14, 2, 80, 80),
        (61000, 9, 2, 48, 16)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", MANY)
def test_many_head_rows(shape, interleaved, cuda_device):
    """Both directions over several batches a unit.

    The weights' gradient: a lane adds its four rows of a batch and then the
    batches of its units (two a unit; 296 blocks of 8 warps share the units); a
    block adds the rows of at most 32 lane groups, and the last kernel at most
    296 / 32 + 1 blocks and then 32 sums: depth 4 + batches + 32 + 10 + 32."""
    t, h, hk, d, rot = shape
    a, g = make(t, h, hk, d, rot, "bf16", seed=t)
    grads = [torch.randn(*a[n].shape, generator=g).bfloat16().to(cuda_device) for n in ("q", "k")]
    outs, got = forward(a, interleaved), backward(a, *grads, interleaved)
    half = torch.finfo(torch.bfloat16).eps / 2 * (1 + 1e-3)
    heads = 2 * 4 * 32 // (8 if d <= 64 else 16 if d <= 128 else 32)  # of a unit
    depth = 78 + 2 * -(-t * (-(-h // heads) - (-hk // heads)) // (296 * 8))
    for i, side in enumerate(("q", "k")):
        y, near, dx, size, dw, dw_size = torch_forms(a, side, grads[i], interleaved)
        close(outs[i], y, half * y.abs() + (d / 16 + 20) * U * near)
        close(got[i], dx, half * dx.abs() + (d / 4 + 64) * U * size)
        close(got[2 + i], dw, (depth + d / 16 + 20) * U * dw_size)
        # A bound that a missing batch would not pass: one row's share of the sum.
        assert float(((depth + d / 16 + 20) * U * dw_size).max()) < 0.05 * float(dw.abs().mean())
    again = backward(a, *grads, interleaved)
    assert all(torch.equal(x, y) for x, y in zip(got, again))


@pytest.mark.parametrize("d", [64, 37])
def test_every_position_is_outside_an_empty_table(d, cuda_device):
    a, g = make(5, 3, 2, d, 16, "bf16")
    a["cos_sin"] = qk_norm_rope.rope_table(0, 16, device=cuda_device)
    q_out, k_out = forward(a)
    assert _native.device_status(reset=True)[0] == 5
    assert torch.isnan(q_out).all() and torch.isnan(k_out).all()
    grads = [torch.randn(*a[n].shape, generator=g).bfloat16().to(cuda_device) for n in ("q", "k")]
    dq, dk, *dw = backward(a, *grads)
    assert _native.device_status(reset=True)[0] == 5
    assert torch.isnan(dq).all() and torch.isnan(dk).all() and not dw[0].any() and not dw[1].any()
