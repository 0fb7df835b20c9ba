"""The projection with adapters against its fp64 form.

Tolerance, element by element: a tensor-core sum of n exact products in fp32 is
off by at most n v S, v = 2^-23, S the sum of the products' absolute values.
H = s (x A^T) is off by K v of its S and 4 v of arithmetic and is rounded to the
element type (half a step of |H|, or half a subnormal step); it meets |B|. The
accumulator adds K + rank + 8 terms' v (the cluster's partial sums included) of
the whole S, and the result is rounded once.
"""

import numpy as np
import pytest
import torch

from flashattentionanycard_b200 import _native
from flashattentionanycard_b200.kernels import lora_gemm
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


class Case:
    def __init__(self, t, k, n, slots, rank, dtype="bf16", seed=0, runs=None, bare=0.2):
        g = torch.Generator().manual_seed(seed + t + n)
        dt = DTYPES[dtype]
        self.dtype, self.slots = dtype, slots
        self.x = torch.randn(t, k, generator=g).to(dt).cuda()
        self.w = (torch.randn(k, n, generator=g) * k**-0.5).to(dt).cuda()
        self.a, self.b, self.scales = [], [], []
        self.bank = lora_gemm.AdapterBank(slots, k, n, rank, dt, "cuda")
        for s in range(slots):
            r = max(1, rank - 3 * (s % 4)) if s % 5 else rank
            self.a.append((torch.randn(r, k, generator=g) * k**-0.5).to(dt))
            self.b.append((0.3 * torch.randn(r, n, generator=g)).to(dt))
            self.scales.append(float(torch.rand((), generator=g)) + 0.5)
            self.bank.load(s, self.a[s].cuda(), self.b[s].cuda(), self.scales[s])
        pick = torch.randint(slots, (t,), generator=g)
        if runs:  # neighbouring rows share an adapter
            pick = pick[:runs].repeat_interleave(-(-t // runs))[:t]
        pick[torch.rand(t, generator=g) < bare] = -1
        self.ids = pick.to(torch.int32).cuda()

    def run(self, **kw):
        out = torch.full((self.x.shape[0], self.w.shape[1]), float("nan"), dtype=self.x.dtype, device="cuda")
        return lora_gemm.launch(self.x, self.w, self.bank, self.ids, out, **kw)

    def bound(self, ids=None):
        x, w = f64(self.x), f64(self.w)
        ids = self.ids.cpu().numpy() if ids is None else ids
        half = torch.finfo(DTYPES[self.dtype]).eps / 2
        ref = decoder.lora_gemm(x, w, [f64(a) for a in self.a], [f64(b) for b in self.b],
                                np.float32(self.scales).astype(np.float64), ids)
        size, tol = np.abs(x) @ np.abs(w), np.zeros_like(ref)
        for s in np.unique(ids[ids >= 0]):
            rows, a, b = ids == s, f64(self.a[s]), np.abs(f64(self.b[s]))
            h = np.abs(self.scales[s] * x[rows] @ a.T)
            dh = (x.shape[1] + 4) * V * self.scales[s] * np.abs(x[rows]) @ np.abs(a).T
            dh = dh + half * (h + dh) + SUB[self.dtype]
            size[rows] += (h + dh) @ b
            tol[rows] += dh @ b
        tol += (x.shape[1] + 128 + 8) * V * size
        return ref, tol + half * (np.abs(ref) + tol) + SUB[self.dtype]

    def check(self, out, rows=slice(None), ids=None):
        ref, tol = self.bound(ids)
        assert np.all(np.abs(f64(out) - ref)[rows] <= tol[rows])


SHAPES = [
    # t, k, n, slots, rank, runs
    (1, 8, 8, 1, 1, None), (1, 4096, 512, 8, 16, None), (2, 72, 136, 3, 4, None),
    (16, 64, 128, 4, 16, None), (17, 1000, 264, 40, 24, None), (64, 512, 1032, 64, 16, None),
    (100, 264, 2056, 12, 64, 7), (128, 136, 256, 200, 8, None), (129, 520, 128, 5, 100, None),
    (200, 128, 4096, 33, 32, 20), (256, 328, 200, 1000, 16, None), (257, 64, 64, 2, 16, None),
    (300, 1000, 520, 300, 16, None), (1000, 256, 1000, 9, 128, 11), (2100, 200, 776, 30, 33, 40),
    (5000, 72, 256, 4, 64, 3), (63, 2048, 20000, 6, 16, None), (1500, 8, 8, 3, 8, 2),
    # the longest lists: every row of a tile its own adapter
    (256, 72, 264, 1024, 128, None), (520, 136, 72, 1024, 128, None), (700, 64, 520, 700, 64, None),
    (128, 256, 20000, 500, 32, None),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_projection(shape, dtype, cuda_device):
    t, k, n, slots, rank, runs = shape
    c = Case(t, k, n, slots, rank, dtype, runs=runs)
    out = c.run()
    c.check(out)
    assert torch.equal(out, c.run())


@pytest.mark.parametrize("t", [40, 600])
def test_no_adapter_and_one_adapter(t, cuda_device):
    c = Case(t, 256, 384, 4, 16, bare=0.0)
    c.ids.fill_(-1)
    c.check(c.run())
    c.ids.fill_(3)
    c.check(c.run())


@pytest.mark.parametrize("t", [40, 600])
def test_bad_ids_and_empty_slots_are_reported(t, cuda_device):
    c = Case(t, 128, 256, 6, 16, bare=0.0)
    ids = c.ids.cpu().numpy().copy()
    c.bank.unload(2)
    c.ids[3], c.ids[17], c.ids[t - 1] = 6, -2, 2
    ids = c.ids.cpu().numpy().copy()
    ids[(ids == 2) | (ids == 6) | (ids == -2)] = -1
    out = c.run()
    torch.cuda.synchronize()
    code, detail = _native.device_status(reset=True)
    assert code == 6 and ids[detail] == -1
    c.check(out, ids=ids)


@pytest.mark.parametrize("t", [50, 500])
def test_rows_that_are_not_finite_stay_alone(t, cuda_device):
    c = Case(t, 136, 264, 7, 16)
    c.ids[30] = 1
    clean = c.run()
    c.x[5, 3] = float("nan")
    c.x[30, 9] = float("inf")
    out = c.run()
    keep = torch.ones(t, dtype=torch.bool)
    keep[5] = keep[30] = False
    assert torch.equal(out[keep], clean[keep])
    assert torch.isnan(out[5]).all() and not torch.isfinite(out[30]).any()


def test_row_past_the_adapters_rank_stays_zero(cuda_device):
    """An infinite x against the bank's zero padding is no NaN: the row is
    infinite where the projection and its own adapter agree in sign."""
    c = Case(20, 64, 128, 3, 64, bare=0.0)
    c.ids.fill_(0)
    c.bank.load(0, torch.ones(1, 64, dtype=torch.bfloat16).cuda(), torch.ones(1, 128, dtype=torch.bfloat16).cuda())
    c.w.fill_(1)
    c.x[4, 7] = float("inf")
    out = c.run()
    assert torch.isinf(out[4]).all() and torch.isfinite(out[:4]).all()


def test_no_rows(cuda_device):
    c = Case(1, 64, 128, 3, 16)
    out = torch.empty(0, 128, dtype=torch.bfloat16, device=cuda_device)
    lora_gemm.launch(c.x[:0], c.w, c.bank, c.ids[:0], out)


@pytest.mark.parametrize("t", [90, 700])
def test_dirty_workspace_and_guard_rows(t, cuda_device):
    c = Case(t, 264, 520, 20, 24)
    want = c.run()
    need = lora_gemm.workspace_bytes(t, c.bank)
    for fill in (0, 255, 127):
        ws = torch.full((need + 4096,), fill, dtype=torch.uint8, device=cuda_device)
        out = torch.zeros(t + 32, 520, dtype=torch.bfloat16, device=cuda_device)
        lora_gemm.launch(c.x, c.w, c.bank, c.ids, out[16:16 + t], workspace=ws[:need])
        assert torch.equal(out[16:16 + t], want)
        assert not out[:16].any() and not out[16 + t:].any() and (ws[need:] == fill).all()
    with pytest.raises(ValueError, match="workspace"):
        c.run(workspace=ws[:need - 1])
    with pytest.raises(RuntimeError, match="aligned"):
        c.run(workspace=ws[16:16 + need])


def test_unaligned_tensors_are_refused(cuda_device):
    c = Case(4, 64, 128, 3, 16)
    flat = torch.zeros(4 * 128 + 1, dtype=torch.bfloat16, device=cuda_device)
    with pytest.raises(RuntimeError, match="aligned"):
        lora_gemm.launch(c.x, c.w, c.bank, c.ids, flat[1:].view(4, 128))


def test_output_over_the_input_is_refused(cuda_device):
    c = Case(4, 64, 64, 3, 16)
    with pytest.raises(ValueError, match="overlap"):
        lora_gemm.launch(c.x, c.w, c.bank, c.ids, c.x)


def test_adapter_changed_between_calls(cuda_device):
    c = Case(30, 64, 128, 4, 16)
    c.run()
    g = torch.Generator().manual_seed(9)
    c.a[1], c.b[1] = torch.randn(5, 64, generator=g).bfloat16(), torch.randn(5, 128, generator=g).bfloat16()
    c.scales[1] = 0.25
    c.bank.load(1, c.a[1].cuda(), c.b[1].cuda(), 0.25)
    c.check(c.run())


def test_back_to_back_calls_chain_on_one_stream(cuda_device):
    """The product starts on x before its own shrink kernel is done: x written
    by the call just before must be seen whole."""
    g = torch.Generator().manual_seed(1)
    for t in (24, 512):
        c = Case(t, 512, 512, 5, 16)
        d = Case(t, 512, 512, 5, 16, seed=7)
        mid, out = torch.empty_like(c.x), torch.empty_like(c.x)
        lora_gemm.launch(c.x, c.w, c.bank, c.ids, mid)
        torch.cuda.synchronize()
        lora_gemm.launch(mid, d.w, d.bank, d.ids, out)
        torch.cuda.synchronize()
        want = out.clone()
        for _ in range(20):
            mid.copy_(torch.randn(mid.shape, generator=g))
            torch.cuda.synchronize()
            lora_gemm.launch(c.x, c.w, c.bank, c.ids, mid)
            lora_gemm.launch(mid, d.w, d.bank, d.ids, out)
            assert torch.equal(out, want)


def test_streams_graphs_and_two_calls_at_once(cuda_device):
    cases = [Case(33, 512, 1024, 9, 16), Case(700, 256, 512, 9, 32, runs=6)]
    want = [c.run() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [[], []]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, c, o in zip(streams, cases, outs):
            with torch.cuda.stream(s):
                o.append(c.run())
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(x, w) for x in o)
    graphs = []
    for c in cases:
        out = torch.full_like(want[len(graphs)], float("nan"))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(2):
                lora_gemm.launch(c.x, c.w, c.bank, c.ids, out)
        graphs.append((g, out))
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for (_, o), w in zip(graphs, want))


# Either side of the choices of the product (streamed W or pair tiles) and of the shrink.
EDGES = [
    (257, 136, 4608, 40, 16, 9), (384, 264, 6400, 12, 32, 7), (1024, 520, 2304, 9, 16, 30),
    (1024, 136, 2440, 300, 64, None), (1025, 264, 128, 17, 24, None), (1152, 64, 8, 1024, 128, None),
    (9345, 72, 8, 3, 16, 5),
]


@pytest.mark.parametrize("shape", EDGES)
def test_projection_at_the_edges_of_its_variants(shape, cuda_device):
    t, k, n, slots, rank, runs = shape
    c = Case(t, k, n, slots, rank, runs=runs)
    out = c.run()
    c.check(out)
    assert torch.equal(out, c.run())


def test_pair_tiles_report_bad_ids_and_keep_other_rows(cuda_device):
    c = Case(1300, 136, 520, 20, 24)
    need = lora_gemm.workspace_bytes(1300, c.bank)
    c.bank.unload(2)
    c.ids[3], c.ids[300], c.ids[1299] = 20, -2, 2
    ids = c.ids.cpu().numpy().copy()
    ids[(ids == 2) | (ids == 20) | (ids == -2)] = -1
    clean = c.run()
    torch.cuda.synchronize()
    code, detail = _native.device_status(reset=True)
    assert code == 6 and ids[detail] == -1
    c.check(clean, ids=ids)
    c.ids[30] = 1
    clean = c.run()
    c.x[5, 3] = float("nan")
    c.x[30, 9] = float("inf")
    keep = torch.ones(1300, dtype=torch.bool)
    keep[5] = keep[30] = False
    for fill in (0, 255, 127):
        ws = torch.full((need + 4096,), fill, dtype=torch.uint8, device=cuda_device)
        out = torch.zeros(1332, 520, dtype=torch.bfloat16, device=cuda_device)
        lora_gemm.launch(c.x, c.w, c.bank, c.ids, out[16:1316], workspace=ws[:need])
        assert torch.equal(out[16:1316][keep], clean[keep])
        assert torch.isnan(out[21]).all() and not torch.isfinite(out[46]).any()
        assert not out[:16].any() and not out[1316:].any() and (ws[need:] == fill).all()
    torch.cuda.synchronize()
    assert _native.device_status(reset=True)[0] == 6


def test_pair_tiles_on_streams_and_in_graphs(cuda_device):
    g = torch.Generator().manual_seed(1)
    c, d = Case(1100, 512, 512, 5, 16), Case(1100, 512, 512, 5, 16, seed=7)
    mid, out = torch.empty_like(c.x), torch.empty_like(c.x)
    c.run(), d.run()
    lora_gemm.launch(c.x, c.w, c.bank, c.ids, mid)
    torch.cuda.synchronize()
    lora_gemm.launch(mid, d.w, d.bank, d.ids, out)
    want = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lora_gemm.launch(c.x, c.w, c.bank, c.ids, mid)
        lora_gemm.launch(mid, d.w, d.bank, d.ids, out)
    other = torch.cuda.Stream()
    alone = d.run()
    for _ in range(10):
        mid.copy_(torch.randn(mid.shape, generator=g))
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            beside = d.run()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(beside, alone)


def test_offsets_past_32_bits(cuda_device):
    """x and out of more than 2^31 elements: 1000 rows over and over.  Odd waves
    of pair tiles walk K downwards, so a row's sum may be taken in either order:
    every repeat is held to the bound, which covers any order."""
    c = Case(1000, 8192, 8192, 12, 16)
    t = 263_000
    x, ids = c.x.repeat(t // 1000, 1), c.ids.repeat(t // 1000)
    assert x.numel() > 2**31
    out = torch.full_like(x, float("nan"))
    lora_gemm.launch(x, c.w, c.bank, ids, out)
    del x
    some = torch.arange(0, 1000, 37)
    c.x, c.ids = c.x[some], c.ids[some]
    ref, tol = (torch.from_numpy(v).cuda() for v in c.bound())
    for block in out.view(t // 1000, 1000, -1):
        assert ((block[some].double() - ref).abs() <= tol).all()
    assert torch.isfinite(out[:1000]).all() and torch.isfinite(out[-1000:]).all()


def parts(scale, b_size, x_size=1.0, t=40, k=264, n=136, rank=16, seed=3):
    """One fp16 adapter on every row of a zero projection, so that the result is the adapter's alone."""
    g = torch.Generator().manual_seed(seed)
    x = (x_size * torch.randn(t, k, generator=g)).half().cuda()
    a = (torch.randn(rank, k, generator=g) * k**-0.5 * x_size**0.5).half().cuda()
    b = (b_size * torch.randn(rank, n, generator=g)).half().cuda()
    bank = lora_gemm.AdapterBank(3, k, n, rank, torch.float16, "cuda")
    bank.load(1, a, b, scale)
    out = torch.full((t, n), float("nan"), dtype=torch.float16, device="cuda")
    w, ids = torch.zeros(k, n, dtype=torch.float16, device="cuda"), torch.ones(t, dtype=torch.int32, device="cuda")
    lora_gemm.launch(x, w, bank, ids, out)
    return f64(x), f64(a), f64(b), f64(out), k


@pytest.mark.parametrize("t", [40, 700])
@pytest.mark.parametrize("scale, b_size, x_size", [
    (1e6, 2e-6, 1.0), (-3e5, 1e-4, 1.0), (1.5, 1e-3, 3e3), (1.0, 6e-8, 3e3),  # x A^T, or its scaled form, past 65504
    (2e-7, 3e3, 1.0), (1e-9, 6e4 / 6, 30.0), (3e-3, 200.0, 1e-3),              # below the smallest normal number
    (1.0, 0.3, 1.0), (0.7, 1e3, 1e-2),
])
def test_fp16_scales_and_adapters_of_any_size(scale, b_size, x_size, t, cuda_device):
    """What the scale and the second factor multiply to is in range, so the
    result is, whatever each of them is.

    With 2^e the power of two between the factors, h = scale 2^-e (x A^T) is off
    by (K + 4) v of its absolute sum, half a step of |h| and half a subnormal
    step, 2^-25; b = B 2^e by 2^-25 where e < 0 made it subnormal; the sum adds
    (rank + 136) v of its size; the result is rounded once.  Whichever e is
    taken, one that serves leaves |b| at most 2 where |scale| > 1, and |h| no
    larger than x A^T where B is moved down."""
    x, a, b, out, k = parts(scale, b_size, x_size, t)
    sc = float(np.float32(scale))
    up = max(0, -int(np.floor(np.log2(np.abs(b).max()))))
    down = max(0, min(int(np.floor(np.log2(np.abs(b).max()))), -int(np.floor(np.log2(abs(sc))))))
    e = up - down
    h, bb = sc * 2.0**-e * (x @ a.T), np.abs(b) * 2.0**e
    dh = (k + 4) * V * abs(sc) * 2.0**-e * (np.abs(x) @ np.abs(a).T)
    dh = dh + 2.0**-11 * (np.abs(h) + dh) + 2.0**-25
    db = 2.0**-25 if e < 0 else 0.0
    size = (np.abs(h) + dh) @ (bb + db)
    tol = dh @ (bb + db) + np.abs(h).sum(1, keepdims=True) * db + 152 * V * size
    ref = sc * (x @ a.T) @ b
    assert np.abs(ref).max() < 60000
    assert np.all(np.abs(out - ref) <= tol + 2.0**-11 * (np.abs(ref) + tol) + 2.0**-25)
    # The bound says something: it is a small part of the result's size.
    assert np.median(tol) < 0.02 * np.sqrt((ref * ref).mean()) + 2.0**-25 * 16
