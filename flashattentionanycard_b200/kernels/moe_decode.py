"""A whole mixture-of-experts layer for a few tokens, in two kernels (sm_100a).

For the decode batches of a served model: where the routed chain
(``moe_routing.topk_gate``, ``MoeRouter``, ``gather_rows``,
``moe_grouped_gemm.launch`` twice, the activation, ``combine``) is bound by its
launches, ``launch`` runs the layer from router logits to combined output at
the rate at which the weights of the experts in use arrive from HBM:

    p = softmax(logits[t]);  e_1..e_k the k largest (ties to the lower index)
    out[t] = sum_j g_j (silu(x[t] @ Wg[e_j]) * (x[t] @ Wu[e_j])) @ Wd[e_j]

with ``w_gate_up`` [E, K, 2 I] holding the gate columns and then the up columns
of every expert, ``w_down`` [E, I, K], and g_j = p[e_j], divided by their sum
with ``renormalize``.  silu(..) * (..) is rounded to the element type between the
products (in fp16 within 65,504), the result once more.  The reference has the
grouped product alone (``bo_kernel_tuner/kernels/moe_grouped_gemm.py:61-65``)
and leaves the rest of the layer outside.
"""

from flashattentionanycard_b200 import _native

MAX_TOKENS, MAX_TOPK, MAX_EXPERTS = 128, 8, 1024


def workspace_bytes(tokens, experts, k, inner, topk):
    """Device scratch of one call on the current device (contents free before and after)."""
    lib = _native.load()
    n = int(lib.bokt_moe_decode_workspace_bytes(int(tokens), int(experts), int(k), int(inner), int(topk)))
    if n < 0:
        raise RuntimeError(f"bokt_moe_decode_workspace_bytes: {lib.bokt_last_error().decode()}")
    return n


def launch(x, logits, w_gate_up, w_down, out, topk, renormalize=True, workspace=None):
    """out[T, K] = the layer's output for x [T, K] and logits [T, E] (T <= 128);
    out may be x itself.

    ``workspace``: a uint8 tensor of ``workspace_bytes`` (calls that may overlap
    on the GPU need one each); by default the call takes a fresh one from
    torch's allocator."""
    import torch

    xs, gs, ds, ls = x.shape, w_gate_up.shape, w_down.shape, logits.shape
    if len(xs) != 2 or len(gs) != 3 or len(ds) != 3 or len(ls) != 2:
        raise ValueError("x and logits must have two dimensions, the weights three")
    t, k = xs
    e, inner, _ = ds
    topk = int(topk)
    if gs != (e, k, 2 * inner) or ds != (e, inner, k):
        raise ValueError(f"shape mismatch: x {tuple(xs)}, w_gate_up {tuple(gs)} "
                         f"(expected [E, K, 2 I]), w_down {tuple(ds)} (expected [E, I, K])")
    if ls != (t, e) or out.shape != xs:
        raise ValueError(f"shape mismatch: logits {tuple(ls)}, out {tuple(out.shape)}")
    if not 1 <= topk <= min(e, MAX_TOPK):
        raise ValueError(f"topk must be in [1, {min(e, MAX_TOPK)}], got {topk}")
    if t > MAX_TOKENS or e > MAX_EXPERTS:
        raise ValueError(f"at most {MAX_TOKENS} tokens and {MAX_EXPERTS} experts (got {t} and {e}): "
                         "larger batches go through moe_routing and moe_grouped_gemm")
    if k % 8 or inner % 8:
        raise ValueError(f"K and I must be multiples of 8 (got {k} and {inner})")
    if not (x.dtype == w_gate_up.dtype == w_down.dtype == out.dtype):
        raise ValueError("x, the weights and out must share one dtype")
    logits_dtype = 2 if logits.dtype == torch.float32 else _native.dtype_code(logits.dtype)
    dtype = _native.dtype_code(x.dtype)
    if not (x.is_contiguous() and logits.is_contiguous() and w_gate_up.is_contiguous()
            and w_down.is_contiguous() and out.is_contiguous()):
        raise ValueError("x, logits, the weights and out must be contiguous")
    index = x.get_device()
    if index < 0 or not (logits.get_device() == w_gate_up.get_device() == w_down.get_device()
                         == out.get_device() == index):
        raise ValueError("all tensors must be on one CUDA device")
    if torch._C._cuda_getDevice() != index:  # the library launches on the current device
        with torch.cuda.device(index):
            return launch(x, logits, w_gate_up, w_down, out, topk, renormalize, workspace)
    scratch, nbytes = _native.workspace("bokt_moe_decode_workspace_bytes", (t, e, k, inner, topk), index,
                                        workspace)
    rc = _native.load().bokt_moe_decode(
        x.data_ptr(), logits.data_ptr(), logits_dtype, w_gate_up.data_ptr(), w_down.data_ptr(),
        out.data_ptr(), t, e, k, inner, topk, 1 if renormalize else 0, dtype, scratch.data_ptr(), nbytes,
        torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _native.check(rc, "bokt_moe_decode")
    return out
