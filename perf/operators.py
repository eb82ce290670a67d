"""The operators that a rank of an expert-parallel model runs around the MoE exchange, with inputs
to measure them on and their plain forms.

* `ffn`    the experts' gated feed-forward block on the rows that the dispatch left grouped by
           expert (serving): y = (act(x Wg^T) * (x Wu^T)) Wo^T, each row with its expert's weights.
* `train`  the same block's training step: y, and from dy the gradients dx, dw_in and dw_out.
* `clip`   the global 2-norm over many gradient tensors, and the gradients scaled to a limit.

With `own` false, `run` computes them with elementary torch operations in 32 bits; with `own`
true it calls `ugdr_b200.ops`.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    def block(op, name, experts, rows, hidden, inner, dtype="bf16", act="silu", skew=0.0, slack=0):
        return {"name": name, "op": op, "experts": experts, "rows": rows, "hidden": hidden, "inner": inner,
                "dtype": dtype, "act": act, "skew": skew, "slack": slack}

    def clip(name, tensors, total, dtype, out, under, packed):
        return {"name": name, "op": "clip", "tensors": tensors, "total": total, "dtype": dtype, "out": out,
                "under": under, "packed": packed}

    return [
        # One token through one dense block: the latency of single-token serving.
        block("ffn", "ffn one token dense", 1, 1, 2048, 5632),
        # A decode step of a rank that owns 32 of 256 experts of the 7168-wide MoE workload.
        block("ffn", "ffn decode 32 experts", 32, 48, 7168, 2048),
        # A prefill chunk on the same rank: about 256 rows per expert.
        block("ffn", "ffn prefill 32 experts", 32, 8192, 7168, 2048),
        # Odd sizes, the other type and activation, skewed routing, a receive area larger than used.
        block("ffn", "ffn odd fp16 gelu", 6, 777, 1000, 1416, "fp16", "gelu", 1.0, 100),
        # A small model's block: launches and short loops count.
        block("train", "train small", 4, 96, 512, 1024),
        # Odd sizes with an expert or two that nearly nobody chose.
        block("train", "train odd fp16 gelu", 9, 1531, 1032, 712, "fp16", "gelu", 1.5, 77),
        # A fine-grained MoE layer of a mid-sized model.
        block("train", "train mid 16 experts", 16, 16384, 2048, 1408),
        # The 7168-wide MoE workload: half of a rank's rows when 8 ranks send 16,384 tokens, top-8.
        block("train", "train large 32 experts", 32, 65536, 7168, 2048),
        # Norm weights and biases: the smallest call.
        clip("clip small", 24, 40_000, "bf16", "fp32", False, False),
        # Hundreds of tensors of mixed types, packed back to back, under the limit, in place.
        clip("clip odd mixed in place", 400, 30_000_001, "mixed", "same", True, True),
        # One layer's gradients in 32 bits, scaled into another buffer.
        clip("clip layer fp32", 40, 180_000_000, "fp32", "same", False, False),
        # A rank's whole gradient in bf16, scaled into the optimizer's 32-bit buffers.
        clip("clip large bf16 to fp32", 300, 1_400_000_000, "bf16", "fp32", False, False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["ffn", "train", "clip"])
    if op == "clip":
        tensors = _log(rng, 1, 500)
        return {"op": op, "tensors": tensors, "total": max(tensors, _log(rng, 2_000, 600_000_000)),
                "dtype": rng.choice(["bf16", "fp16", "fp32", "mixed"]), "out": rng.choice(["same", "fp32"]),
                "under": rng.random() < 0.3, "packed": rng.random() < 0.5}
    while True:
        experts, rows = _log(rng, 1, 64), _log(rng, 1, 40_000)
        hidden, inner = 8 * _log(rng, 8, 896), 8 * _log(rng, 8, 704)
        if 18 * rows * hidden * inner <= 8e12 and 3 * experts * hidden * inner <= 1.2e9:
            break
    return {"op": op, "experts": experts, "rows": rows, "hidden": hidden, "inner": inner,
            "dtype": rng.choice(["bf16", "fp16"]), "act": rng.choice(["silu", "gelu"]),
            "skew": rng.choice([0.0, 0.5, 1.5]), "slack": rng.choice([0, 0, 64, 201])}


# ---- inputs --------------------------------------------------------------------------------------


def _sizes(case):
    """Sizes of a model's gradient tensors, the same for every seed: log-normal, at least one
    element each, `total` in all."""
    n, total = case["tensors"], case["total"]
    rng = np.random.default_rng(n + total)
    share = np.exp(1.5 * rng.standard_normal(n))
    sizes = 1 + np.floor(share / share.sum() * (total - n)).astype(np.int64)
    sizes[int(rng.integers(n))] += total - int(sizes.sum())
    return [int(v) for v in sizes]


def _flat_views(sizes, dtype, packed):
    """One flat buffer and the tensors in it: back to back, or each at a multiple of 128 elements."""
    step = 1 if packed else 128
    at, starts = 0, []
    for n in sizes:
        starts.append(at)
        at += -(-n // step) * step
    flat = torch.zeros(at, dtype=dtype, device="cuda")
    return flat, [flat[a:a + n] for a, n in zip(starts, sizes)]


def _prepare_clip(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    sizes = _sizes(case)
    if case["dtype"] == "mixed":
        parts = [(torch.bfloat16, sizes[0::2]), (torch.float32, sizes[1::2])]
    else:
        parts = [(_TYPES[case["dtype"]], sizes)]
    flats, outs, grads, into = [], [], [], []
    scale = np.exp(np.random.default_rng(seed + 1).standard_normal(len(sizes))) * 1e-2
    for dtype, part in parts:
        flat, views = _flat_views(part, dtype, case["packed"])
        for v, k in zip(views, scale):
            v.normal_(0.0, float(k), generator=gen)
        flats.append(flat)
        grads += views
        if not case["under"]:  # scaled into a buffer of its own, so that a pass can be repeated
            out, views = _flat_views(part, torch.float32 if case["out"] == "fp32" else dtype, case["packed"])
            outs.append(out)
            into += views
    state = {"op": "clip", "grads": grads, "into": into or None, "result": outs or flats,
             # A limit far above any norm, or one that the norm is some ten times over.
             "max_norm": 1e30 if case["under"] else 3e-3 * math.sqrt(case["total"])}
    if own:
        from ugdr_b200.ops import GradClip

        state["plan"] = GradClip(grads, out=into or None)
    return state


def _counts(case, seed):
    """Rows of each expert: rows thrown by a router whose preferences are as uneven as `skew`."""
    rng = np.random.default_rng(seed)
    pull = np.exp(case["skew"] * rng.standard_normal(case["experts"]))
    return rng.multinomial(case["rows"], pull / pull.sum())


def prepare(case, seed):
    if case["op"] == "clip":
        return _prepare_clip(case, seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, experts, hidden, inner = _TYPES[case["dtype"]], case["experts"], case["hidden"], case["inner"]
    counts = _counts(case, seed)
    rows = case["rows"] + case["slack"]

    def normal(scale, *shape):
        return torch.empty(*shape, dtype=dtype, device="cuda").normal_(0.0, scale, generator=gen)

    state = {"op": case["op"], "act": case["act"], "most": int(counts.max()),
             "counts": torch.from_numpy(counts.astype(np.int32)).cuda(),
             "x": normal(1.0, rows, hidden),
             "w_in": normal(hidden ** -0.5, experts, 2, inner, hidden),
             "w_out": normal(inner ** -0.5, experts, hidden, inner),
             # Rows behind the last group stay as they were: the outputs go into buffers of zeros.
             "y": torch.zeros(rows, hidden, dtype=dtype, device="cuda")}
    if case["op"] == "train":
        state["dy"] = normal(0.1, rows, hidden)
        state["dx"] = torch.zeros(rows, hidden, dtype=dtype, device="cuda")
    return state


# ---- one pass ------------------------------------------------------------------------------------


def run(state):
    if state["op"] == "clip":
        return _run_clip(state)
    if not own:
        return _plain_block(state)
    from ugdr_b200 import ops

    x, counts, w_in, w_out, act = (state[k] for k in ("x", "counts", "w_in", "w_out", "act"))
    if state["op"] == "ffn":
        return ops.expert_ffn(x, counts, w_in, w_out, act=act, out=state["y"])
    y, saved = ops.expert_ffn_train(x, counts, w_in, w_out, act=act, out=state["y"])
    dx, dw_in, dw_out = ops.expert_ffn_backward(state["dy"], x, counts, w_in, w_out, saved, act=act, dx=state["dx"])
    return {"y": y, "dx": dx, "dw_in": dw_in, "dw_out": dw_out}


def _run_clip(state):
    if own:
        norm = state["plan"].clip(state["max_norm"])
    else:
        grads, into = state["grads"], state["into"] or state["grads"]
        squares = torch.stack([g.float().square().sum(dtype=torch.float64) for g in grads])
        norm = squares.sum().sqrt().float()
        coef = torch.clamp(state["max_norm"] / (norm + 1e-6), max=1.0)
        [o.copy_(g.float() * coef) for g, o in zip(grads, into)]
    return {"norm": norm, "grads": state["result"]}


def _act(g, act):
    """The activation and its derivative."""
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    p = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return g * p, p + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_block(s):
    """Every expert's rows side by side in a padded batch, one batched product per projection."""
    x, counts, dtype = s["x"], s["counts"].long(), s["x"].dtype
    ends = counts.cumsum(0)
    starts = ends - counts
    place = torch.arange(s["most"], device=x.device)
    live = place < counts[:, None]  # [experts, most]
    slot = torch.where(live, starts[:, None] + place, 0)
    row = torch.arange(x.shape[0], device=x.device)
    expert = torch.searchsorted(ends, row, right=True).clamp(max=counts.numel() - 1)
    back = (row - starts[expert]).clamp(max=s["most"] - 1)
    used = (row < ends[-1])[:, None]

    def padded(t):
        return torch.where(live[..., None], t[slot].float(), 0.0)

    def rows_of(t, into):
        return into.copy_(torch.where(used, t[expert, back].to(dtype), into))

    xp = padded(x)
    wg, wu, wo = s["w_in"][:, 0].float(), s["w_in"][:, 1].float(), s["w_out"].float()
    g, u = torch.bmm(xp, wg.transpose(1, 2)), torch.bmm(xp, wu.transpose(1, 2))
    a, da = _act(g, s["act"])
    h = a * u
    y = rows_of(torch.bmm(h, wo.transpose(1, 2)), s["y"])
    if s["op"] == "ffn":
        return y
    dyp = padded(s["dy"])
    dh = torch.bmm(dyp, wo)
    dw_out = torch.bmm(dyp.transpose(1, 2), h).to(dtype)
    dg, du = dh * u * da, dh * a
    dw_in = torch.stack([torch.bmm(dg.transpose(1, 2), xp), torch.bmm(du.transpose(1, 2), xp)], 1).to(dtype)
    dx = rows_of(torch.bmm(dg, wg) + torch.bmm(du, wu), s["dx"])
    return {"y": y, "dx": dx, "dw_in": dw_in, "dw_out": dw_out}


# ---- what a pass cannot do without, and what it gives in 64 bits ---------------------------------


def work(case):
    if case["op"] == "clip":
        parts = {"mixed": 3.0, "bf16": 2.0, "fp16": 2.0, "fp32": 4.0}[case["dtype"]]
        written = 0.0 if case["under"] else 4.0 if case["out"] == "fp32" else parts
        return {"bytes": case["total"] * (parts + written), "flops": 3.0 * case["total"]}
    experts, rows, block = case["experts"], case["rows"], case["hidden"] * case["inner"]
    chosen = experts * (1.0 - (1.0 - 1.0 / experts) ** rows)  # experts that have a row, on average
    weights, acts = 2.0 * 3 * chosen * block, 2.0 * rows * case["hidden"]
    if case["op"] == "ffn":
        return {"bytes": weights + 2 * acts, "flops": 6.0 * rows * block}
    return {"bytes": weights + 2.0 * 3 * experts * block + 4 * acts, "flops": 18.0 * rows * block}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        total = torch.zeros((), dtype=torch.float64, device="cuda")
        for g in s["grads"]:
            total += torch.dot(g.double(), g.double())
        norm = total.sqrt()
        coef = min(1.0, s["max_norm"] / (float(norm) + 1e-6))
        return {"norm": norm, "grads": [f.double() * coef for f in _sources(s)]}
    y = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
    dx = torch.zeros_like(y)
    dws = [[], []]
    at = 0
    for e, n in enumerate(s["counts"].tolist()):
        x = s["x"][at:at + n].double().requires_grad_()
        w_in, w_out = s["w_in"][e].double().requires_grad_(), s["w_out"][e].double().requires_grad_()
        gate, up = x @ w_in[0].T, x @ w_in[1].T
        gate = torch.nn.functional.silu(gate) if case["act"] == "silu" else torch.nn.functional.gelu(gate)
        out = (gate * up) @ w_out.T
        y[at:at + n] = out.detach()
        if case["op"] == "train":
            grads = torch.autograd.grad(out, (x, w_in, w_out), s["dy"][at:at + n].double())
            dx[at:at + n] = grads[0]
            dws[0].append(grads[1].float())
            dws[1].append(grads[2].float())
        at += n
    if case["op"] == "ffn":
        return y
    return {"y": y, "dx": dx, "dw_in": torch.stack(dws[0]), "dw_out": torch.stack(dws[1])}


def _sources(s):
    """The flat buffers that the gradients lie in, laid out as the results are."""
    return [g._base for g in {g._base.data_ptr(): g for g in s["grads"]}.values()]
