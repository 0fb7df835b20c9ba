"""Operators of a decoder layer around its attention, and the cases they are measured on.

Three operators, in the order in which a serving or training step meets them:

``lora``  the shared projection of a batch of requests, each with a low-rank
          adapter of its own (or none): out = x @ w + scale_a * (x @ A_a) @ B_a
``qk``    RMSNorm of every query and key head followed by the rotary position
          rotation, forward and backward
``moe``   a whole mixture-of-experts layer for a few tokens: top-k softmax gate,
          gated-SiLU experts and the gate-weighted sum

``run`` computes them in elementary fp32 torch operations, or with this
repository's kernels where ``own`` is set.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One sequence decoding through a small expert layer: all latency.
        {"name": "moe_one_token", "op": "moe", "t": 1, "e": 8, "k": 1024, "i": 2048, "top": 2, "dtype": "bf16"},
        # A decode batch over the widest experts: every expert's weights are read once.
        {"name": "moe_wide_32", "op": "moe", "t": 32, "e": 16, "k": 4096, "i": 14336, "top": 2, "dtype": "bf16"},
        # Many small experts, eight per token.
        {"name": "moe_fine_64", "op": "moe", "t": 64, "e": 128, "k": 2048, "i": 768, "top": 8, "dtype": "fp16"},
        # Odd batch and sizes that end inside every tile.
        {"name": "moe_odd_37", "op": "moe", "t": 37, "e": 12, "k": 1032, "i": 1000, "top": 3, "dtype": "bf16"},
        # One request with its adapter: latency.
        {"name": "lora_one_token", "op": "lora", "t": 1, "k": 4096, "n": 4096, "slots": 8, "rank": 16, "requests": 1,
         "dtype": "bf16"},
        # A decode batch: one token per request, adapters spread over the bank.
        {"name": "lora_decode_64", "op": "lora", "t": 64, "k": 4096, "n": 14336, "slots": 32, "rank": 16, "requests": 64,
         "dtype": "bf16"},
        # Short prefills and decodes together, sizes that end inside every tile.
        {"name": "lora_odd_203", "op": "lora", "t": 203, "k": 1000, "n": 2056, "slots": 12, "rank": 24, "requests": 37,
         "dtype": "fp16"},
        # Prefill: nine prompts of uneven lengths.
        {"name": "lora_prefill_4096", "op": "lora", "t": 4096, "k": 4096, "n": 4096, "slots": 16, "rank": 32, "requests": 9,
         "dtype": "bf16"},
        # A decode batch far into long sequences.
        {"name": "qk_decode_64", "op": "qk", "t": 64, "heads": 32, "kv_heads": 8, "d": 128, "rot": 128, "table": 131072,
         "pairs": False, "grad": False, "dtype": "bf16"},
        # Prefill.
        {"name": "qk_prefill_16384", "op": "qk", "t": 16384, "heads": 32, "kv_heads": 8, "d": 128, "rot": 128, "table": 16384,
         "pairs": False, "grad": False, "dtype": "bf16"},
        # A training step's backward pass.
        {"name": "qk_grad_8192", "op": "qk", "t": 8192, "heads": 32, "kv_heads": 8, "d": 128, "rot": 128, "table": 8192,
         "pairs": False, "grad": True, "dtype": "bf16"},
        # Backward with an odd length, one shared key head and a partial rotation of neighbouring pairs.
        {"name": "qk_grad_odd_1111", "op": "qk", "t": 1111, "heads": 5, "kv_heads": 1, "d": 80, "rot": 32, "table": 4096,
         "pairs": True, "grad": True, "dtype": "fp16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["moe", "lora", "qk"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "moe":
        k, i = 8 * _log(rng, 32, 512), 8 * _log(rng, 32, 512)
        e = min(_log(rng, 2, 128), max(2, int(4e9 / (6 * k * i))))
        return {"op": op, "t": _log(rng, 1, 128), "e": e, "k": k, "i": i, "top": rng.randint(1, min(e, 8)), "dtype": dtype}
    if op == "lora":
        t = _log(rng, 1, 4096)
        return {"op": op, "t": t, "k": 8 * _log(rng, 32, 512), "n": 8 * _log(rng, 32, 512), "slots": _log(rng, 1, 32),
                "rank": _log(rng, 4, 64), "requests": t if t <= 64 and rng.random() < 0.5 else _log(rng, 1, min(t, 64)),
                "dtype": dtype}
    d = 16 * rng.randint(2, 16)
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 3, 4, 5])
    t = min(_log(rng, 1, 16384), max(1, 60_000_000 // (d * (heads + kv))))
    return {"op": op, "t": t, "heads": heads, "kv_heads": kv, "d": d, "rot": d if rng.random() < 0.5 else 16 * rng.randint(1, d // 16),
            "table": 16384, "pairs": rng.random() < 0.3, "grad": rng.random() < 0.5, "dtype": dtype}


def _expected_experts(case):
    return case["e"] * (1 - (1 - case["top"] / case["e"]) ** case["t"])


def work(case):
    t = case["t"]
    if case["op"] == "moe":
        k, i, top = case["k"], case["i"], case["top"]
        weights = _expected_experts(case) * 3 * k * i * 2
        return {"bytes": int(weights + 2 * t * k * 2 + t * case["e"] * 4), "flops": 2 * 3 * k * i * t * top}
    if case["op"] == "lora":
        k, n, s = case["k"], case["n"], case["slots"]
        rank = sum(_rank(case, j) for j in range(s)) / s
        used = s * (1 - (1 - 1 / s) ** (case["requests"] * 7 / 8))
        return {"bytes": int(2 * (t * k + k * n + t * n + used * rank * (k + n))), "flops": int(2 * t * (k * n + 7 / 8 * rank * (k + n)))}
    rows, d = t * (case["heads"] + case["kv_heads"]), case["d"]
    angles = min(t, case["table"]) * case["rot"] * 4
    # forward: values in and out; backward: values and gradients in, gradients out.
    return {"bytes": (3 if case["grad"] else 2) * rows * d * 2 + angles, "flops": rows * d * (20 if case["grad"] else 9)}


# ------------------------------------------------------------------ inputs
def _rank(case, slot):
    """Adapters of one bank differ in rank: the full one, a half and a quarter in turn."""
    return max(1, case["rank"] >> (slot % 3))


def prepare(case, seed):
    dtype = DTYPES[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, scale=1.0, dtype=dtype):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype).mul_(scale)

    t = case["t"]
    if case["op"] == "moe":
        e, k, i = case["e"], case["k"], case["i"]
        state = {"case": case, "x": randn(t, k), "logits": randn(t, e, scale=2.0, dtype=torch.float32),
                 "w_gate_up": randn(e, k, 2 * i, scale=k**-0.5), "w_down": randn(e, i, k, scale=i**-0.5),
                 "out": torch.empty(t, k, device="cuda", dtype=dtype)}
        return state
    if case["op"] == "lora":
        k, n, s, r = case["k"], case["n"], case["slots"], case["rank"]
        ranks = torch.tensor([_rank(case, j) for j in range(s)], device="cuda")
        held = (torch.arange(r, device="cuda")[None, :] < ranks[:, None])[:, :, None]
        # Requests are runs of neighbouring tokens; one in eight has no adapter.
        cuts = torch.randperm(max(t - 1, 1), generator=g, device="cuda")[: case["requests"] - 1] + 1
        request = torch.zeros(t, dtype=torch.int64, device="cuda").index_fill_(0, cuts, 1).cumsum(0) if case["requests"] > 1 \
            else torch.zeros(t, dtype=torch.int64, device="cuda")
        adapter = torch.randint(s, (case["requests"],), generator=g, device="cuda")
        bare = torch.rand(case["requests"], generator=g, device="cuda") < 0.125
        bare[0] = False
        state = {"case": case, "x": randn(t, k), "w": randn(k, n, scale=k**-0.5), "a": randn(s, r, k, scale=k**-0.5) * held,
                 "b": randn(s, r, n, scale=0.1) * held, "ids": torch.where(bare, -1, adapter)[request].to(torch.int32),
                 "scales": 0.5 + torch.rand(s, generator=g, device="cuda"), "out": torch.empty(t, n, device="cuda", dtype=dtype)}
        if own:
            # The bank a serving program keeps: adapters are loaded when a request first brings them.
            from flashattentionanycard_b200.kernels import lora_gemm

            bank = lora_gemm.AdapterBank(s, k, n, r, dtype, state["x"].device)
            for j in range(s):
                rank = _rank(case, j)
                bank.load(j, state["a"][j, :rank], state["b"][j, :rank], float(state["scales"][j]))
            state["bank"] = bank
        return state
    h, hk, d, rot, p = case["heads"], case["kv_heads"], case["d"], case["rot"], case["table"]
    # Queries, keys and values of a token lie side by side, as the projection leaves them.
    qkv = randn(t, h + 2 * hk, d)
    # A decode batch has every token somewhere in a sequence of its own; a longer one is a prompt.
    positions = torch.randint(p, (t,), generator=g, device="cuda") if t <= 64 else torch.arange(t, device="cuda") % p
    power = torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot
    angle = torch.arange(p, device="cuda", dtype=torch.float64)[:, None] * 10000.0**-power
    state = {"case": case, "q": qkv[:, :h], "k": qkv[:, h:h + hk], "positions": positions.to(torch.int32),
             "q_weight": 1 + randn(d, scale=0.1), "k_weight": 1 + randn(d, scale=0.1),
             "cos_sin": torch.cat([angle.cos(), angle.sin()], 1).float()}
    if case["grad"]:
        state |= {"dq_out": randn(t, h, d), "dk_out": randn(t, hk, d), "dq": torch.empty(t, h, d, device="cuda", dtype=dtype),
                  "dk": torch.empty(t, hk, d, device="cuda", dtype=dtype), "dqw": torch.empty(d, device="cuda", dtype=torch.float32),
                  "dkw": torch.empty(d, device="cuda", dtype=torch.float32)}
    else:
        state |= {"q_out": torch.empty(t, h, d, device="cuda", dtype=dtype), "k_out": torch.empty(t, hk, d, device="cuda", dtype=dtype)}
    return state


EPS = 1e-6


# ------------------------------------------------------------------ plain forms
def _moe(s):
    case, x = s["case"], s["x"].float()
    t, top, i = case["t"], case["top"], case["i"]
    p = torch.softmax(s["logits"], dim=1)
    gates, ids = torch.sort(p, dim=1, descending=True, stable=True)
    gates, ids = gates[:, :top], ids[:, :top]
    gates = gates / gates.sum(1, keepdim=True)
    if t * top <= case["e"]:
        # Few assignments: each meets its own expert's weights.
        flat = ids.reshape(-1)
        gu = torch.bmm(x.repeat_interleave(top, 0)[:, None, :], s["w_gate_up"][flat].float())
        h = gu[..., :i] * torch.sigmoid(gu[..., :i]) * gu[..., i:]
        y = torch.bmm(h, s["w_down"][flat].float()).view(t, top, -1)
        return (gates[:, :, None] * y).sum(1).to(s["x"].dtype)
    # Many: every expert sees every token, and the gate keeps what was routed.
    weight = torch.zeros(t, case["e"], device=x.device).scatter_(1, ids, gates)
    gu = torch.matmul(x, s["w_gate_up"].float())
    h = gu[..., :i] * torch.sigmoid(gu[..., :i]) * gu[..., i:]
    y = torch.bmm(h, s["w_down"].float())
    return (weight.t()[:, :, None] * y).sum(0).to(s["x"].dtype)


def _lora(s):
    x, ids = s["x"].float(), s["ids"].long()
    slots, r = s["a"].shape[:2]
    mine = (ids[:, None] == torch.arange(slots, device=x.device)) * s["scales"]
    h = (x @ s["a"].float().flatten(0, 1).t()).view(-1, slots, r) * mine[:, :, None]
    return (x @ s["w"].float() + h.flatten(1) @ s["b"].float().flatten(0, 1)).to(s["x"].dtype)


def _halves(v, rot, pairs):
    return (v[..., 0:rot:2], v[..., 1:rot:2]) if pairs else (v[..., : rot // 2], v[..., rot // 2:rot])


def _join(a, b, rest, pairs):
    turned = torch.stack([a, b], -1).flatten(-2) if pairs else torch.cat([a, b], -1)
    return torch.cat([turned, rest], -1)


def _angles(s):
    cs = s["cos_sin"][s["positions"].long()][:, None, :]
    return cs.chunk(2, -1)


def _qk_one(x, w, c, sn, rot, pairs):
    v = x.float()
    y = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * w.float()
    a, b = _halves(y, rot, pairs)
    return _join(a * c - b * sn, b * c + a * sn, y[..., rot:], pairs).to(x.dtype)


def _qk_one_grad(do, x, w, c, sn, rot, pairs):
    v, g = x.float(), do.float()
    a, b = _halves(g, rot, pairs)
    g = _join(a * c + b * sn, b * c - a * sn, g[..., rot:], pairs)
    r = torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    n, gw = v * r, g * w.float()
    dx = r * (gw - n * (gw * n).mean(-1, keepdim=True))
    return dx.to(x.dtype), (g * n).sum((0, 1), dtype=torch.float64).float()


def run(state):
    case = state["case"]
    if case["op"] == "moe":
        if own:
            from flashattentionanycard_b200.kernels import moe_decode

            moe_decode.launch(state["x"], state["logits"], state["w_gate_up"], state["w_down"], state["out"], case["top"])
            return state["out"]
        return _moe(state)
    if case["op"] == "lora":
        if own:
            from flashattentionanycard_b200.kernels import lora_gemm

            lora_gemm.launch(state["x"], state["w"], state["bank"], state["ids"], state["out"])
            return state["out"]
        return _lora(state)
    rot, pairs = case["rot"], case["pairs"]
    q, k, qw, kw = state["q"], state["k"], state["q_weight"], state["k_weight"]
    if own:
        from flashattentionanycard_b200.kernels import qk_norm_rope

        if case["grad"]:
            qk_norm_rope.launch_backward(state["dq_out"], state["dk_out"], q, k, qw, kw, state["positions"], state["cos_sin"],
                                         state["dq"], state["dk"], state["dqw"], state["dkw"], epsilon=EPS, interleaved=pairs)
            return state["dq"], state["dk"], state["dqw"], state["dkw"]
        qk_norm_rope.launch(q, k, qw, kw, state["positions"], state["cos_sin"], state["q_out"], state["k_out"], epsilon=EPS,
                            interleaved=pairs)
        return state["q_out"], state["k_out"]
    c, sn = _angles(state)
    if case["grad"]:
        dq, dqw = _qk_one_grad(state["dq_out"], q, qw, c, sn, rot, pairs)
        dk, dkw = _qk_one_grad(state["dk_out"], k, kw, c, sn, rot, pairs)
        return dq, dk, dqw, dkw
    return _qk_one(q, qw, c, sn, rot, pairs), _qk_one(k, kw, c, sn, rot, pairs)


# ------------------------------------------------------------------ 64-bit results
def _exact_moe(s):
    case = s["case"]
    t, top, i = case["t"], case["top"], case["i"]
    logits = s["logits"].double()
    out = torch.zeros(t, case["k"], dtype=torch.float64, device="cuda")
    order = torch.argsort(-logits, dim=1, stable=True)[:, :top]
    picked = torch.gather(logits, 1, order)
    share = torch.exp(picked - picked[:, :1])
    share = share / share.sum(1, keepdim=True)
    for e in torch.unique(order).tolist():
        rows, slot = torch.nonzero(order == e, as_tuple=True)
        up = s["x"][rows].double() @ s["w_gate_up"][e].double()
        act = up[:, :i] / (1 + torch.exp(-up[:, :i])) * up[:, i:]
        out.index_add_(0, rows, share[rows, slot][:, None] * (act @ s["w_down"][e].double()))
    return out


def _exact_lora(s):
    x = s["x"].double()
    out = x @ s["w"].double()
    for j in torch.unique(s["ids"]).tolist():
        if j >= 0:
            rows = torch.nonzero(s["ids"] == j)[:, 0]
            out[rows] += float(s["scales"][j]) * ((x[rows] @ s["a"][j].double().t()) @ s["b"][j].double())
    return out


def _exact_qk(s):
    case = s["case"]
    rot, d, pairs = case["rot"], case["d"], case["pairs"]
    low = torch.arange(0, rot, 2) if pairs else torch.arange(rot // 2)
    high = low + 1 if pairs else low + rot // 2
    cs = s["cos_sin"][s["positions"].long()].double()
    turn = torch.complex(cs[:, : rot // 2], cs[:, rot // 2:])[:, None, :]
    outs, sums = [], []
    for name in ("q", "k"):
        x, w = s[name].double(), s[name + "_weight"].double()
        size = torch.sqrt((x * x).sum(-1, keepdim=True) / d + EPS)
        if not case["grad"]:
            y = x / size * w
            z = torch.complex(y[..., low], y[..., high]) * turn
            y[..., low], y[..., high] = z.real, z.imag
            outs.append(y)
            continue
        g = s["d" + name + "_out"].double()
        z = torch.complex(g[..., low], g[..., high]) * turn.conj()
        g[..., low], g[..., high] = z.real, z.imag
        sums.append((g * x / size).sum((0, 1)))
        outs.append(g * w / size - x * (g * w * x).sum(-1, keepdim=True) / (d * size**3))
    return tuple(outs + sums)


def exact(case, seed):
    state = prepare(case, seed)
    return {"moe": _exact_moe, "lora": _exact_lora, "qk": _exact_qk}[case["op"]](state)
