"""A shared projection with the low-rank adapters of many requests at once (sm_100a).

The dense GEMM of the reference's ``bo_kernel_tuner/kernels/gemm.py:7-40`` with
one adapter per row beside it (the reference has none):

    out[t] = x[t] @ w + scale_a * (x[t] @ A_a.T) @ B_a     a = ids[t], -1: none

An ``AdapterBank`` keeps the adapters of a projection in slots on the device, as
a serving program loads them; ``launch`` runs a batch in which every row names
its slot, in two kernels: the rows' low-rank vectors, then the projection, whose
K loop goes on over the adapters that the row tile uses.  With few rows (or few
tiles) the second kernel streams ``w`` against the tokens (decode); else it is
the CTA-pair GEMM (prefill).
"""

import math

from flashattentionanycard_b200 import _native

MAX_SLOTS, MAX_SIZE, RANKS = 1024, 1 << 30, (16, 32, 64, 128)


def _moved_exponent(largest, scale):
    """e of the power of two that an fp16 adapter's slot takes from its scale into b.

    The kernels round scale (x @ A.T) to fp16, which holds 2^-24 to 65504.  With
    the largest value of b 2^e in [1, 2), and its rows of like size, that product
    is past 65504 only where the adapter's result is too, and what it loses below
    the smallest normal number is a step of 2^-25 of the result.  Up, b 2^e is
    exact.  Down it may lose bits of its smallest values, so b goes down only to
    bring a scale below one up to it."""
    if not largest or not scale:
        return 0
    up = 1 - math.frexp(largest)[1]
    return max(up, min(0, math.frexp(scale)[1] - 1))


class AdapterBank:
    """Adapters of one [K, N] projection in ``slots`` device slots, ranks up to ``max_rank``.

    ``load`` copies an adapter in (on the current stream) and refuses values
    that are not finite: rows of other adapters meet them as zero factors.  In
    fp16 the slot's b and scale may differ from the loaded ones by a power of
    two that their product does not see."""

    def __init__(self, slots, k, n, max_rank, dtype, device):
        import torch

        self.slots, self.k, self.n = int(slots), int(k), int(n)
        if not 1 <= self.slots <= MAX_SLOTS:
            raise ValueError(f"slots must be in [1, {MAX_SLOTS}], got {slots}")
        if self.k < 8 or self.n < 8 or self.k % 8 or self.n % 8:
            raise ValueError(f"K and N must be positive multiples of 8 (got {k} and {n})")
        if self.k > MAX_SIZE or self.n > MAX_SIZE:
            raise ValueError(f"K and N must be at most {MAX_SIZE} (got {k} and {n})")
        if not 1 <= int(max_rank) <= RANKS[-1]:
            raise ValueError(f"max_rank must be in [1, {RANKS[-1]}], got {max_rank}")
        _native.dtype_code(dtype)
        self.rank = next(r for r in RANKS if r >= int(max_rank))
        self.max_rank = int(max_rank)
        self.a = torch.zeros(self.slots, self.rank, self.k, dtype=dtype, device=device)
        self.b = torch.zeros(self.slots, self.rank, self.n, dtype=dtype, device=device)
        self.scales = torch.zeros(self.slots, dtype=torch.float32, device=device)
        self.ranks = torch.zeros(self.slots, dtype=torch.int32, device=device)
        self.dtype, self.device = dtype, self.a.device

    def _slot(self, slot):
        if not 0 <= int(slot) < self.slots:
            raise ValueError(f"slot must be in [0, {self.slots}), got {slot}")
        return int(slot)

    def load(self, slot, a, b, scale=1.0):
        """Put the adapter a [r, K], b [r, N] with its scale into ``slot``."""
        import torch

        slot = self._slot(slot)
        r = a.shape[0] if a.dim() else 0
        if a.dim() != 2 or b.dim() != 2 or not 1 <= r <= self.max_rank \
                or a.shape != (r, self.k) or b.shape != (r, self.n):
            raise ValueError(f"shape mismatch: a {tuple(a.shape)}, b {tuple(b.shape)}; expected [r, {self.k}] "
                             f"and [r, {self.n}] with r in [1, {self.max_rank}]")
        a, b = a.detach(), b.detach()  # trained parameters leave no graph on the bank
        if a.dtype != self.dtype or b.dtype != self.dtype:
            raise ValueError(f"the adapter must have the bank's dtype {self.dtype}")
        scale = float(scale)
        if not abs(scale) <= 3.4028234663852886e38:
            raise ValueError("scale must be a finite fp32 value")
        # The largest magnitudes: NaN and infinity stay what they are in a maximum.
        largest = torch.linalg.vector_norm(a, float("inf")) + torch.linalg.vector_norm(b, float("inf")) * 0
        if not math.isfinite(largest.item()):
            raise ValueError("the adapter holds values that are not finite")
        if self.dtype == torch.float16:
            e = _moved_exponent(torch.linalg.vector_norm(b, float("inf")).item(), scale)
            if e:
                b, scale = b * 2.0**e, scale * 2.0**-e
        into_a, into_b = self.a[slot], self.b[slot]
        into_a[:r].copy_(a)
        into_b[:r].copy_(b)
        if r < self.rank:
            into_a[r:].zero_()
            into_b[r:].zero_()
        self.scales[slot].fill_(scale)
        self.ranks[slot].fill_(r)

    def unload(self, slot):
        slot = self._slot(slot)
        self.ranks[slot] = 0
        self.scales[slot] = 0
        self.a[slot].zero_()
        self.b[slot].zero_()


def workspace_bytes(m, bank):
    """Device scratch of one call with m rows on the current device: sized for a
    batch that uses as many of the bank's slots as it can, about
    2 m rank min(slots, 256) bytes for many rows (8192 rows and 256 slots of rank
    128: 0.5 GB)."""
    lib = _native.load()
    n = int(lib.bokt_lora_gemm_workspace_bytes(int(m), bank.n, bank.k, bank.slots, bank.rank))
    if n < 0:
        raise RuntimeError(f"bokt_lora_gemm_workspace_bytes: {lib.bokt_last_error().decode()}")
    return n


def launch(x, w, bank, ids, out, workspace=None):
    """out[T, N] = x[T, K] @ w[K, N] plus every row's adapter; ids int32 [T], -1 for none.

    An id outside [-1, slots) or of an empty slot sets the device status word
    (``_native.device_status``), and its row gets the projection alone.
    ``workspace``: a uint8 tensor of ``workspace_bytes`` (calls that may overlap
    on the GPU need one each); by default the call takes a fresh one from
    torch's allocator."""
    import torch

    if x.dim() != 2 or w.dim() != 2:
        raise ValueError(f"x and w must have two dimensions, got {tuple(x.shape)} and {tuple(w.shape)}")
    m, k = x.shape
    n = w.shape[1]
    if w.shape[0] != k or out.shape != (m, n):
        raise ValueError(f"shape mismatch: x {tuple(x.shape)}, w {tuple(w.shape)}, out {tuple(out.shape)}")
    if m > MAX_SIZE:
        raise ValueError(f"at most {MAX_SIZE} rows (got {m})")
    if k != bank.k or n != bank.n:
        raise ValueError(f"the bank's adapters are for a [{bank.k}, {bank.n}] projection, not [{k}, {n}]")
    if ids.dtype != torch.int32 or ids.shape != (m,) or not ids.is_contiguous():
        raise ValueError(f"ids must be a contiguous int32 tensor of {m} elements")
    dtype = x.dtype
    if not (dtype == w.dtype == out.dtype == bank.dtype):
        raise ValueError("x, w, out and the bank must share one dtype")
    if not (x.is_contiguous() and w.is_contiguous() and out.is_contiguous()):
        raise ValueError("x, w and out must be contiguous row-major tensors")
    index = x.get_device()
    if index < 0 or not (w.get_device() == out.get_device() == ids.get_device() == bank.a.get_device() == index):
        raise ValueError("all tensors and the bank must be on one CUDA device")
    xp, outp = x.data_ptr(), out.data_ptr()
    if xp < outp + 2 * m * n and outp < xp + 2 * m * k:
        raise ValueError("out must not overlap x: finished columns are written while others still read x")
    if torch._C._cuda_getDevice() != index:  # the library launches on the current device
        with torch.cuda.device(index):
            return launch(x, w, bank, ids, out, workspace)
    scratch, nbytes = _native.workspace("bokt_lora_gemm_workspace_bytes", (m, n, k, bank.slots, bank.rank),
                                        index, workspace)
    rc = _native.load().bokt_lora_gemm(
        xp, w.data_ptr(), bank.a.data_ptr(), bank.b.data_ptr(), bank.scales.data_ptr(),
        bank.ranks.data_ptr(), ids.data_ptr(), outp, m, n, k, bank.slots, bank.rank,
        _native.dtype_code(dtype), scratch.data_ptr(), nbytes, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _native.check(rc, "bokt_lora_gemm")
    return out
