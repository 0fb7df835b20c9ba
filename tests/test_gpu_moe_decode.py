"""The few-token MoE layer against its fp64 form.

Tolerance, element by element (``bound``).  A tensor-core sum of n exact
products in fp32 is off by at most n v S with v = 2^-23 (each addition cut or
rounded to 24 bits) and S the sum of the products' absolute values.  With dg, du
that bound for the gate and up columns: h = silu(g) u is off by
1.1 |u| dg + |silu(g)| du (|silu'| <= 1.1) plus 8 v |h| of arithmetic, and is
rounded to the element type: half a step of |h|, or half a subnormal step.  The
down product adds I v S again; the gates (softmax over E logits, all terms
positive) are off by (E + 16) v relative; the gate-weighted sum of k terms by
k v; the result is rounded once.
"""

import numpy as np
import pytest
import torch

from flashattentionanycard_b200 import _native
from flashattentionanycard_b200.kernels import moe_decode
from oracle import decoder

pytestmark = pytest.mark.gpu

V = 2.0**-23
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
SUB = {"bf16": 2.0**-134, "fp16": 2.0**-25}


@pytest.fixture(autouse=True)
def clean_status(cuda_device):
    _native.device_status(reset=True)
    yield
    assert _native.device_status(reset=True)[0] == 0


def f64(t):
    return t.detach().cpu().double().numpy()


def make(t, e, k, inner, dtype="bf16", logits=torch.float32, seed=0, skew=0.0):
    g = torch.Generator().manual_seed(seed + t + e)
    dt = DTYPES[dtype]
    z = 2 * torch.randn(t, e, generator=g)
    z[:, 0] += skew
    return {"x": torch.randn(t, k, generator=g).to(dt).cuda(), "logits": z.to(logits).cuda(),
            "w_gate_up": (torch.randn(e, k, 2 * inner, generator=g) * k**-0.5).to(dt).cuda(),
            "w_down": (torch.randn(e, inner, k, generator=g) * inner**-0.5).to(dt).cuda()}


def run(a, topk, renormalize=True, **kw):
    out = torch.full_like(a["x"], float("nan"))
    moe_decode.launch(**a, out=out, topk=topk, renormalize=renormalize, **kw)
    return out


def bound(a, topk, renormalize, dtype):
    """(fp64 result, allowed distance)."""
    x, z, gu, dn = (f64(a[n]) for n in ("x", "logits", "w_gate_up", "w_down"))
    half = torch.finfo(DTYPES[dtype]).eps / 2
    t, k = x.shape
    e, inner = dn.shape[:2]
    ids, gates = decoder.moe_gate(z, topk, renormalize)
    ref, tol = np.zeros((t, k)), np.zeros((t, k))
    for ex in np.unique(ids):
        rows, slot = np.nonzero(ids == ex)
        w = gates[rows, slot][:, None]
        s = x[rows] @ gu[ex]
        ds = k * V * (np.abs(x[rows]) @ np.abs(gu[ex]))
        g, u = s[:, :inner], s[:, inner:]
        silu = g / (1 + np.exp(-g))
        h = silu * u
        dh = 1.1 * np.abs(u) * ds[:, :inner] + np.abs(silu) * ds[:, inner:] + 8 * V * np.abs(h)
        dh = dh + half * (np.abs(h) + dh) + SUB[dtype]
        y = h @ dn[ex]
        hy = np.abs(h) @ np.abs(dn[ex])
        dy = dh @ np.abs(dn[ex]) + inner * V * hy
        np.add.at(ref, rows, w * y)
        np.add.at(tol, rows, w * (dy + (e + 16 + topk) * V * np.abs(y)))
    return ref, tol + half * (np.abs(ref) + tol) + SUB[dtype]


def check(a, topk, out, dtype, renormalize=True, rows=slice(None)):
    ref, tol = bound(a, topk, renormalize, dtype)
    assert np.all(np.abs(f64(out) - ref)[rows] <= tol[rows])


SHAPES = [
    # t, e, k, inner, topk
    (1, 1, 8, 8, 1), (1, 8, 64, 64, 2), (2, 3, 72, 40, 3), (16, 16, 256, 128, 4), (17, 5, 264, 136, 3),
    (31, 33, 520, 264, 5), (33, 12, 1032, 1000, 3), (48, 40, 136, 328, 6), (64, 130, 256, 96, 8),
    (100, 2, 128, 520, 2), (128, 8, 512, 256, 2), (128, 300, 64, 24, 8), (65, 1024, 72, 16, 7),
    (1, 16, 2048, 4096, 8), (5, 4, 4096, 8, 1), (5, 4, 8, 4096, 2),
    # sixteen tokens and fewer on either kernel: more assignments, long runs, wide outputs
    (9, 64, 128, 72, 8), (16, 64, 256, 1024, 4), (16, 3, 2056, 136, 2), (8, 40, 4104, 24, 8),
    (13, 600, 264, 40, 4), (2, 2, 20000, 16, 2),
    # the largest lists
    (128, 1024, 8, 8, 8), (128, 1024, 72, 136, 8), (128, 8, 264, 72, 8), (16, 4, 264, 2056, 4),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_layer(shape, dtype, cuda_device):
    t, e, k, inner, topk = shape
    a = make(t, e, k, inner, dtype)
    out = run(a, topk)
    check(a, topk, out, dtype)
    assert torch.equal(out, run(a, topk))


@pytest.mark.parametrize("logits", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("renormalize", [False, True])
def test_gate_types_ties_and_renormalisation(logits, renormalize, cuda_device):
    a = make(40, 24, 64, 48, logits=logits)
    a["logits"][3] = a["logits"][3, 0]  # all equal: the lowest indices
    a["logits"][4, ::2] = 0.0
    a["logits"][4, 1::2] = -0.0  # equal to it
    a["logits"][5, 7:] = float("-inf")
    a["logits"][6] = torch.finfo(logits).min
    a["logits"][6, 11] = 0
    out = run(a, 4, renormalize)
    check(a, 4, out, "bf16", renormalize)


@pytest.mark.parametrize("t, skew", [(128, 100.0), (37, 3.0), (16, 100.0), (5, 3.0)])
def test_one_hot_expert(t, skew, cuda_device):
    a = make(t, 9, 200, 72, skew=skew)
    check(a, 3, run(a, 3), "bf16")


def test_fewer_finite_logits_than_picks(cuda_device):
    """Picks of probability zero add nothing."""
    a = make(4, 6, 64, 32)
    a["logits"][:, 1:] = float("-inf")
    check(a, 3, run(a, 3), "bf16")


@pytest.mark.parametrize("t", [20, 14])
def test_rows_without_a_distribution_are_nan_and_alone(t, cuda_device):
    a = make(t, 6, 64, 32)
    clean = run(a, 2)
    a["logits"][3] = float("-inf")
    a["logits"][7, 2] = float("nan")
    a["logits"][9, 2] = float("inf")
    a["x"][11, 5] = float("nan")
    a["x"][12, 5] = float("inf")
    out = run(a, 2)
    bad = [3, 7, 9, 11]
    good = [i for i in range(t) if i not in bad + [12]]
    assert torch.isnan(out[bad]).all()
    assert not torch.isfinite(out[12]).any()
    assert torch.equal(out[good], clean[good])


def test_experts_nobody_picked_are_not_touched(cuda_device):
    a = make(10, 8, 64, 40)
    a["logits"][:, 3] = -100.0
    a["logits"][:, 7] = -100.0
    clean = run(a, 2)
    for e in (3, 7):
        a["w_gate_up"][e] = float("nan")
        a["w_down"][e] = float("inf")
    assert torch.equal(run(a, 2), clean)


@pytest.mark.parametrize("t", [30, 15])
def test_weights_that_are_not_finite_reach_their_tokens_only(t, cuda_device):
    a = make(t, 4, 64, 136)
    clean = run(a, 1)
    a["w_gate_up"][2] = float("nan")
    out = run(a, 1)
    hit = (a["logits"].argmax(1) == 2)
    assert hit.any() and torch.isnan(out[hit]).all() and torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("t", [3, 50])
def test_output_over_the_input(t, cuda_device):
    a = make(t, 8, 264, 136)
    want = run(a, 2)
    moe_decode.launch(**a, out=a["x"], topk=2)
    assert torch.equal(a["x"], want)


def test_no_tokens(cuda_device):
    a = make(0, 4, 64, 32)
    assert run(a, 2).shape == (0, 64)


@pytest.mark.parametrize("t", [23, 11])
def test_dirty_workspace_and_guard_bytes(t, cuda_device):
    a = make(t, 10, 264, 136)
    want = run(a, 3)
    need = moe_decode.workspace_bytes(t, 10, 264, 136, 3)
    for fill in (0, 255, 127):
        ws = torch.full((need + 4096,), fill, dtype=torch.uint8, device=cuda_device)
        out = torch.zeros(40, 264, dtype=torch.bfloat16, device=cuda_device)
        moe_decode.launch(**a, out=out[8:8 + t], topk=3, workspace=ws[:need])
        assert torch.equal(out[8:8 + t], want)
        assert not out[:8].any() and not out[8 + t:].any() and (ws[need:] == fill).all()
    with pytest.raises(ValueError, match="workspace"):
        run(a, 3, workspace=ws[:need - 1])
    with pytest.raises(RuntimeError, match="aligned"):
        run(a, 3, workspace=ws[16:16 + need])


def test_unaligned_tensors_are_refused(cuda_device):
    a = make(4, 4, 64, 32)
    flat = torch.zeros(4 * 64 + 1, dtype=torch.bfloat16, device=cuda_device)
    with pytest.raises(RuntimeError, match="aligned"):
        moe_decode.launch(**a, out=flat[1:].view(4, 64), topk=2)


def test_streams_graphs_and_two_calls_at_once(cuda_device):
    a, b = make(16, 16, 512, 512), make(90, 30, 256, 768, seed=3)
    want = run(a, 2), run(b, 5)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, data, k, o in zip(streams, (a, b), (2, 5), outs):
            with torch.cuda.stream(s):
                o.append(run(data, k))
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(x, w) for x in o)
    graphs = []
    for data, k in ((a, 2), (b, 5)):
        out = torch.full_like(data["x"], float("nan"))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            moe_decode.launch(**data, out=out, topk=k)
            moe_decode.launch(**data, out=out, topk=k)
        graphs.append((g, out))
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for (_, o), w in zip(graphs, want))


def test_matches_the_routed_chain(cuda_device):
    """The same layer through the framework's routed operators (their outputs
    are rounded between the steps: y to bf16, half a step of each term more)."""
    from flashattentionanycard_b200.kernels import moe_grouped_gemm
    from flashattentionanycard_b200.kernels.moe_routing import MoeRouter, combine, gather_rows, topk_gate

    t, e, k, inner, topk = 96, 8, 256, 384, 2
    a = make(t, e, k, inner)
    ids = torch.empty(t, topk, dtype=torch.int32, device=cuda_device)
    gates = torch.empty(t, topk, device=cuda_device)
    topk_gate(a["logits"], topk, ids, gates)
    router = MoeRouter(t * topk, e, cuda_device)(ids.reshape(-1))
    bf = dict(dtype=torch.bfloat16, device=cuda_device)
    xp, gu = torch.empty(t * topk, k, **bf), torch.empty(t * topk, 2 * inner, **bf)
    y, out = torch.empty(t * topk, k, **bf), torch.empty(t, k, **bf)
    gather_rows(a["x"], router.perm, xp, topk)
    sms = torch.cuda.get_device_properties(cuda_device).multi_processor_count
    moe_grouped_gemm.launch(xp, a["w_gate_up"], router.offsets, gu, {"CTA_MULTIPLIER": 1}, sms)
    h = (torch.nn.functional.silu(gu[:, :inner].float()) * gu[:, inner:].float()).bfloat16()
    moe_grouped_gemm.launch(h, a["w_down"], router.offsets, y, {"CTA_MULTIPLIER": 1}, sms)
    combine(y, gates, out, router.inv_perm)
    mine = f64(run(a, topk))
    assert np.linalg.norm(f64(out) - mine) <= 2.0**-7 * np.linalg.norm(mine)


def picked(a, topk):
    """Experts of every token, fp64 order."""
    return decoder.moe_gate(f64(a["logits"]), topk)[0]


def cuts_tiles(t, k, inner, active):
    """Whether the persistent kernel's first phase cuts its tiles: its rule on the device's SMs."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    tiles, steps = active * -(-inner // 128), -(-k // 64)
    return t > 16 and -(-tiles // sms) * steps > tiles * steps // sms + 12


# Few wide tiles, each shared by 16 and by 32 runs of k-steps (more than one
# round of the partial sums' loads), and runs that end one tile and begin the
# next; an expert of one or two rows beside ones of many.
CUT = [(20, 4, 4096, 136, 2, 0.0), (17, 2, 8192, 72, 1, 3.0), (128, 160, 1032, 120, 8, 0.0), (33, 9, 2056, 264, 2, 4.0)]


def make_cut(t, e, k, inner, topk, skew, dtype="bf16"):
    a = make(t, e, k, inner, dtype, skew=skew)
    ids = picked(a, topk)
    assert cuts_tiles(t, k, inner, len(np.unique(ids)))
    return a, np.bincount(ids.ravel(), minlength=e)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", CUT)
def test_layer_of_cut_tiles(shape, dtype, cuda_device):
    t, e, k, inner, topk, skew = shape
    a, rows = make_cut(*shape, dtype)
    if skew:
        assert rows.max() > 2 and ((rows > 0) & (rows <= 2)).any()
    out = run(a, topk)
    check(a, topk, out, dtype)
    for _ in range(10):
        assert torch.equal(out, run(a, topk))


@pytest.mark.parametrize("shape", CUT)
def test_cut_tiles_dirty_workspace_and_rows_that_are_not_finite(shape, cuda_device):
    t, e, k, inner, topk, skew = shape
    a, _ = make_cut(*shape)
    want = run(a, topk)
    need = moe_decode.workspace_bytes(t, e, k, inner, topk)
    ids = picked(a, topk)
    bad = {**a, "x": a["x"].clone()}
    bad["x"][5, 3] = float("nan")
    bad["x"][11, k - 1] = float("inf")
    good = [i for i in range(t) if i not in (5, 11)]
    for fill in (0, 255, 127):
        ws = torch.full((need + 4096,), fill, dtype=torch.uint8, device=cuda_device)
        out = torch.zeros(t + 16, k, dtype=torch.bfloat16, device=cuda_device)
        moe_decode.launch(**a, out=out[8:8 + t], topk=topk, workspace=ws[:need])
        assert torch.equal(out[8:8 + t], want)
        assert not out[:8].any() and not out[8 + t:].any() and (ws[need:] == fill).all()
        ws[:need] = fill
        got = run(bad, topk, workspace=ws[:need])
        assert torch.equal(got[good], want[good])
        assert torch.isnan(got[5]).all() and not torch.isfinite(got[11]).any()
    spoiled = int(ids[0, 0])
    hit = torch.from_numpy((ids == spoiled).any(1))
    a["w_gate_up"][spoiled, k - 1] = float("nan")
    got = run(a, topk)
    assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], want[~hit])


def test_cut_tiles_on_streams_and_in_graphs(cuda_device):
    cases = [(make_cut(*s)[0], s[4]) for s in CUT]
    want = [run(a, k) for a, k in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = []
    for turn in range(8):
        for i, (a, k) in enumerate(cases):
            with torch.cuda.stream(streams[(i + turn) % len(streams)]):
                outs.append((i, run(a, k)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i, o in outs)
    graphs = []
    for a, k in cases:
        out = torch.full_like(a["x"], float("nan"))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            moe_decode.launch(**a, out=out, topk=k)
            moe_decode.launch(**a, out=out, topk=k)
        graphs.append((graph, out))
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for (_, o), w in zip(graphs, want))
