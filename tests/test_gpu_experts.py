"""The experts' gated feed-forward block, forward and backward, against its formulas in fp64.

Tolerances are bounds, element by element, derived from what the operator rounds: h, dg and du
once to the type (half a step: eps / 2 of the value, or half the smallest subnormal), the output
once, and fp32 sums of n products, off by at most n * 2^-23 of the sum of the products' sizes
(either way of rounding an addition)."""
from __future__ import annotations

import math

import pytest

from conftest import gpu_count

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def one_gpu():
    if gpu_count() < 1:
        pytest.skip("no GPU")
    torch.cuda.set_device(0)


def act64(g, act):
    """a(g), a'(g)."""
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    p = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
    return g * p, p + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def rounding(t, dtype):
    """How far a value as large as |t| is off after one rounding to dtype."""
    f = torch.finfo(dtype)
    return t.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2


def oracle(x, w_in, w_out, act, dy=None):
    """One expert: {name: (value, bound of the error)} in fp64."""
    dtype = x.dtype
    x, w_in, w_out = x.double(), w_in.double(), w_out.double()
    wg, wu = w_in[0], w_in[1]
    (F, H), n, step = wg.shape, x.shape[0], 2.0 ** -23
    g, u = x @ wg.T, x @ wu.T
    eg, eu = H * step * (x.abs() @ wg.abs().T), H * step * (x.abs() @ wu.abs().T)
    a, da = act64(g, act)
    h = a * u
    # |a'| <= 1.13 and |a''| <= 0.8 for both activations; evaluating them costs a few fp32 steps.
    eh = 1.13 * eg * (u.abs() + eu) + a.abs() * eu + 16 * step * h.abs()
    eh = eh + rounding(h.abs() + eh, dtype)
    y = h @ w_out.T
    ey = eh @ w_out.abs().T + F * step * ((h.abs() + eh) @ w_out.abs().T)
    out = {"y": (y, ey + rounding(y.abs() + ey, dtype))}
    if dy is None:
        return out
    dy = dy.double()
    dh = dy @ w_out
    edh = H * step * (dy.abs() @ w_out.abs())
    dg, du = dh * u * da, dh * a
    edg = edh * (u.abs() + eu) * 1.13 + dh.abs() * (eu * (da.abs() + 0.8 * eg) + u.abs() * 0.8 * eg)
    edu = edh * (a.abs() + 1.13 * eg) + dh.abs() * 1.13 * eg
    # The derivatives are sums of terms up to |a'| + |g|: a few fp32 steps of those.
    edg = edg + 16 * step * (dh * u).abs() * (1 + g.abs())
    edu = edu + 16 * step * du.abs()
    edg, edu = edg + rounding(dg.abs() + edg, dtype), edu + rounding(du.abs() + edu, dtype)
    dx = dg @ wg + du @ wu
    edx = edg @ wg.abs() + edu @ wu.abs()
    edx = edx + 2 * F * step * ((dg.abs() + edg) @ wg.abs() + (du.abs() + edu) @ wu.abs())
    xa = x.abs()
    dw_in = torch.stack([dg.T @ x, du.T @ x])
    edw = torch.stack([edg.T @ xa, edu.T @ xa])
    edw = edw + n * step * torch.stack([(dg.abs() + edg).T @ xa, (du.abs() + edu).T @ xa])
    dw_out = dy.T @ h
    edo = dy.abs().T @ eh + n * step * (dy.abs().T @ (h.abs() + eh))
    for name, v, e in (("dx", dx, edx), ("dw_in", dw_in, edw), ("dw_out", dw_out, edo)):
        out[name] = (v, e + rounding(v.abs() + e, dtype))
    return out


def inputs(counts, hidden, inner, dtype, slack=0, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed + sum(counts) + hidden)
    rows, nexp = sum(counts) + slack, len(counts)

    def normal(scale, *shape):
        return torch.empty(*shape, dtype=dtype, device="cuda").normal_(0, scale, generator=gen)

    return (normal(1, rows, hidden), torch.tensor(counts, dtype=torch.int32, device="cuda"),
            normal(hidden ** -0.5, nexp, 2, inner, hidden), normal(inner ** -0.5, nexp, hidden, inner),
            normal(0.1, rows, hidden))


def near(got, want, bound, what):
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound, first at "
                                 f"{bad.nonzero()[0].tolist()}, worst {float((off / bound).nan_to_num(1e9).max()):.3g} of it")


def compare(x, counts, w_in, w_out, act, dy, got):
    """Every expert's part of got (a dict of y, dx, dw_in, dw_out) against the oracle's."""
    at = 0
    for e, n in enumerate(counts.tolist()):
        rows = slice(at, at + n)
        for name, (v, b) in oracle(x[rows], w_in[e], w_out[e], act, dy[rows]).items():
            if name in got:
                near(got[name][e] if name.startswith("dw") else got[name][rows], v, b, f"expert {e}: {name}")
        at += n


def step(x, counts, w_in, w_out, act, dy, **kw):
    from ugdr_b200 import ops

    y, saved = ops.expert_ffn_train(x, counts, w_in, w_out, act=act, **kw)
    dx, dw_in, dw_out = ops.expert_ffn_backward(dy, x, counts, w_in, w_out, saved, act=act, **kw)
    return {"y": y, "dx": dx, "dw_in": dw_in, "dw_out": dw_out}


CASES = [
    # counts, hidden, inner: one row and one column group; tiles' edges; experts nobody chose
    ([1], 8, 8), ([1], 64, 128), ([3], 264, 72), ([0, 5, 0, 1, 0], 128, 64), ([0, 0], 64, 64),
    ([15, 16, 17, 31, 32, 33], 136, 200), ([63, 64, 65, 127, 128, 129], 256, 128),
    ([255, 256, 257], 128, 264), ([511, 1, 513], 520, 136), ([700], 1000, 712),
    # few tiles and long sums, which pairs of CTAs share
    ([2500], 144, 264), ([5, 40, 0, 300], 1800, 520), ([1900], 1032, 1032), ([1100, 0, 31], 200, 72), ([33], 1160, 136), ([2], 72, 2056), ([700, 900], 72, 136),
    ([1] * 40, 72, 520), ([2, 0, 300, 7, 0, 0, 90], 1032, 1416), ([130], 2048, 24), ([40, 9], 24, 2056),
]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("counts,hidden,inner", CASES)
def test_block_matches_the_formulas(counts, hidden, inner, dtype, act):
    from ugdr_b200 import ops

    x, c, w_in, w_out, dy = inputs(counts, hidden, inner, getattr(torch, dtype))
    got = step(x, c, w_in, w_out, act, dy)
    compare(x, c, w_in, w_out, act, dy, got)
    assert torch.equal(ops.expert_ffn(x, c, w_in, w_out, act=act), got["y"])
    ops.check_status()


def test_many_experts_with_few_rows():
    counts = [(7 * e) % 4 for e in range(1000)]
    x, c, w_in, w_out, dy = inputs(counts, 64, 40, torch.bfloat16)
    compare(x, c, w_in, w_out, "silu", dy, step(x, c, w_in, w_out, "silu", dy))


def test_rows_behind_the_last_group_stay():
    from ugdr_b200 import ops

    counts = [5, 0, 70, 12]
    x, c, w_in, w_out, dy = inputs(counts, 136, 264, torch.bfloat16, slack=150)
    used = sum(counts)
    for t in (x, dy):  # whatever lies there reaches no result
        t[used:used + 50] = float("nan")
        t[used + 50:] = float("inf")
    y, dx = torch.full_like(x, 7.0), torch.full_like(x, -3.0)
    _, saved = ops.expert_ffn_train(x, c, w_in, w_out, out=y)
    _, dw_in, dw_out = ops.expert_ffn_backward(dy, x, c, w_in, w_out, saved, dx=dx)
    compare(x, c, w_in, w_out, "silu", dy, {"y": y, "dx": dx, "dw_in": dw_in, "dw_out": dw_out})
    assert bool((y[used:] == 7.0).all()) and bool((dx[used:] == -3.0).all())


def test_a_group_of_nans_reaches_no_other_expert():
    counts = [33, 20, 75]
    x, c, w_in, w_out, dy = inputs(counts, 72, 136, torch.float16)
    x[33:53], dy[33:53] = float("nan"), float("inf")
    got = step(x, c, w_in, w_out, "silu", dy)
    for e, rows in ((0, slice(0, 33)), (2, slice(53, 128))):
        for name, (v, b) in oracle(x[rows], w_in[e], w_out[e], "silu", dy[rows]).items():
            near(got[name][e] if name.startswith("dw") else got[name][rows], v, b, f"expert {e}: {name}")
    assert bool(got["y"][33:53].isnan().all()) and bool(got["dw_in"][1].isnan().any())


def test_large_gates_saturate():
    """Gates far out on both sides: a(g) -> g and -> 0 with no NaN from the exponential."""
    x, c, w_in, w_out, dy = inputs([40], 64, 64, torch.bfloat16)
    for act in ("silu", "gelu"):
        got = step(x * 200, c, w_in, w_out, act, dy)
        compare(x * 200, c, w_in, w_out, act, dy, got)


def test_in_place_in_the_receive_area():
    """y over x when serving; dx over dy or x when training: the same bits as apart."""
    from ugdr_b200 import ops

    x, c, w_in, w_out, dy = inputs([9, 300, 41], 264, 200, torch.bfloat16)
    want = step(x, c, w_in, w_out, "silu", dy)
    over = x.clone()
    assert ops.expert_ffn(over, c, w_in, w_out, out=over) is over
    assert torch.equal(over, want["y"])
    for which in ("dy", "x"):
        x2, dy2 = x.clone(), dy.clone()
        _, saved = ops.expert_ffn_train(x2, c, w_in, w_out)
        dx, dw_in, dw_out = ops.expert_ffn_backward(dy2, x2, c, w_in, w_out, saved, dx=dy2 if which == "dy" else x2)
        assert torch.equal(dx, want["dx"]) and torch.equal(dw_in, want["dw_in"]) and torch.equal(dw_out, want["dw_out"])


def test_runs_repeat_bit_for_bit_and_outputs_go_where_asked():
    from ugdr_b200 import ops

    x, c, w_in, w_out, dy = inputs([3, 290, 17], 520, 328, torch.bfloat16)
    a, b = step(x, c, w_in, w_out, "gelu", dy), step(x, c, w_in, w_out, "gelu", dy)
    assert all(torch.equal(a[k], b[k]) for k in a)
    given = [torch.empty_like(t) for t in (x, w_in, w_out)]
    _, saved = ops.expert_ffn_train(x, c, w_in, w_out, act="gelu")
    got = ops.expert_ffn_backward(dy, x, c, w_in, w_out, saved, "gelu", *given)
    for g, t, name in zip(got, given, ("dx", "dw_in", "dw_out")):
        assert g is t and torch.equal(g, a[name])


def test_two_streams_at_once():
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    sets = [inputs([200, 0, 57], 264, 264, torch.bfloat16, seed=k) for k in (1, 2)]
    want = [step(*t[:4], "silu", t[4]) for t in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        got.append([step(*t[:4], "silu", t[4], stream=s) for t, s in zip(sets, (s1, s2))])
    torch.cuda.synchronize()
    for pair in got:
        for w, g in zip(want, pair):
            assert all(torch.equal(w[k], g[k]) for k in w)


def test_inputs_on_a_chosen_stream_are_kept_until_it_is_through():
    """Inputs dropped right after the call: their memory is not given out while a busy stream has
    yet to read them."""
    from ugdr_b200 import ops

    x, c, w_in, w_out, _ = inputs([64, 64], 256, 256, torch.bfloat16)
    want = ops.expert_ffn(x, c, w_in, w_out)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        again = x.clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)  # some 10 ms
        got = ops.expert_ffn(again, c, w_in, w_out, stream=side)
        del again
        others = [torch.full_like(x, float("nan")) for _ in range(4)]
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        del others


def test_another_device_than_the_current_one():
    if gpu_count() < 2:
        pytest.skip("needs 2 GPUs")
    x, c, w_in, w_out, dy = (t.to("cuda:1") for t in inputs([20, 45], 72, 136, torch.bfloat16))
    got = step(x, c, w_in, w_out, "silu", dy)
    assert torch.cuda.current_device() == 0 and all(t.device.index == 1 for t in got.values())
    compare(x, c, w_in, w_out, "silu", dy, got)


def test_offsets_past_32_bits():
    """More than 2^32 elements kept for the backward pass: the first and the last rows are right, and
    the weights' gradients when only the last rows have one."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of free GPU memory")
    rows, hidden, inner = 70_001, 64, 32_768
    x, c, w_in, w_out, dy = inputs([rows - 3, 3], hidden, inner, torch.bfloat16)
    dy[:rows - 7] = 0
    got = step(x, c, w_in, w_out, "silu", dy)
    assert 2 * rows * inner > 1 << 32
    for e, r in ((0, slice(0, 5)), (0, slice(rows - 7, rows - 3)), (1, slice(rows - 3, rows))):
        o = oracle(x[r], w_in[e], w_out[e], "silu", dy[r])
        near(got["y"][r], *o["y"], "y")
        near(got["dx"][r], *o["dx"], "dx")
        if r.start > 5:
            near(got["dw_in"][e], *o["dw_in"], "dw_in")
            near(got["dw_out"][e], *o["dw_out"], "dw_out")


def test_captured_steps_follow_their_inputs():
    """Two graphs of a training step, replayed in turn with new rows and new counts."""
    sets = [inputs([20, 100], 136, 136, torch.bfloat16, seed=k) for k in (1, 2)]
    for t in sets:
        step(*t[:4], "silu", t[4])
    torch.cuda.synchronize()
    graphs = []
    for t in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*t[:4], "silu", t[4])
        graphs.append((g, out))
    for counts in ([20, 100], [0, 120], [77, 3]):
        for (g, out), t in zip(graphs, sets):
            t[1].copy_(torch.tensor(counts, dtype=torch.int32))
            t[0].copy_(t[0].roll(1, 0))
            g.replay()
        torch.cuda.synchronize()
        for (_, out), t in zip(graphs, sets):
            used = sum(counts)
            want = step(*t[:4], "silu", t[4])
            for k in want:
                a, b = (want[k], out[k]) if k.startswith("dw") else (want[k][:used], out[k][:used])
                assert torch.equal(a, b), k


def test_bad_counts_are_recorded_and_stay_in_bounds():
    from ugdr_b200 import ops

    x, c, w_in, w_out, dy = inputs([10, 10], 64, 64, torch.bfloat16)
    want = ops.expert_ffn(x, c, w_in, w_out)
    for counts in ([10, 1000], [10, 2 ** 31 - 1]):  # rows past the end are dropped
        got = ops.expert_ffn(x, torch.tensor(counts, dtype=torch.int32, device="cuda"), w_in, w_out)
        assert torch.equal(got, want)
        with pytest.raises(RuntimeError, match="counts"):
            ops.check_status()
    got = step(x, torch.tensor([-5, 20], dtype=torch.int32, device="cuda"), w_in, w_out, "silu", dy)
    with pytest.raises(RuntimeError, match="counts"):
        ops.check_status(0)
    assert bool((got["dw_in"][0] == 0).all())
    compare(x, torch.tensor([0, 20]), w_in, w_out, "silu", dy, got)
    ops.check_status()


def test_no_rows():
    from ugdr_b200 import ops

    _, _, w_in, w_out, _ = inputs([1, 1], 64, 40, torch.bfloat16)
    x, c = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    got = step(x, c, w_in, w_out, "silu", x)
    assert got["y"].shape == (0, 64) and got["dx"].shape == (0, 64)
    assert bool((got["dw_in"] == 0).all()) and bool((got["dw_out"] == 0).all())
    assert ops.expert_ffn(x, c, w_in, w_out).shape == (0, 64)


def test_gradients_against_differences():
    """Directional derivatives: <kernel's gradient, v> against central differences of the fp64
    forward, off by the gradient's own bound summed over v (and the differences' h^2 term)."""
    x, c, w_in, w_out, dy = inputs([6, 11], 40, 56, torch.float16)
    got = step(x, c, w_in, w_out, "gelu", dy)
    gen = torch.Generator(device="cuda").manual_seed(5)

    def loss(x_, wi, wo):
        total, at = 0.0, 0
        for e, n in enumerate(c.tolist()):
            r = slice(at, at + n)
            a, _ = act64(x_[r] @ wi[e, 0].T, "gelu")
            total = total + ((a * (x_[r] @ wi[e, 1].T)) @ wo[e].T * dy[r].double()).sum()
            at += n
        return total

    bounds = {k: [] for k in ("dx", "dw_in", "dw_out")}
    at = 0
    for e, n in enumerate(c.tolist()):
        r = slice(at, at + n)
        o = oracle(x[r], w_in[e], w_out[e], "gelu", dy[r])
        for k in bounds:
            bounds[k].append(o[k][1])
        at += n
    base = [t.double() for t in (x, w_in, w_out)]
    for i, k in enumerate(("dx", "dw_in", "dw_out")):
        bound = torch.cat(bounds[k]) if k == "dx" else torch.stack(bounds[k])
        v = torch.randn(base[i].shape, dtype=torch.float64, device="cuda", generator=gen)
        eps = 1e-5
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + eps * v, base[i] - eps * v
        numeric = float((loss(*up) - loss(*down)) / (2 * eps))
        mine = float((got[k].double() * v).sum())
        assert abs(mine - numeric) <= float((bound * v.abs()).sum()) + 1e-6 * (1 + abs(numeric)), k


def test_refusals():
    from ugdr_b200 import ops

    x, c, w_in, w_out, dy = inputs([4, 4], 64, 64, torch.bfloat16)
    y, saved = ops.expert_ffn_train(x, c, w_in, w_out)
    bad = [
        dict(x=x.float()), dict(x=x[:, :60]), dict(x=x.t()), dict(x=x.cpu()), dict(x=x.half()),
        dict(counts=c.long()), dict(counts=c.cpu()), dict(counts=c[:1]), dict(counts=c[:0]),
        dict(w_in=w_in[:, :1]), dict(w_in=w_in.transpose(2, 3)), dict(w_out=w_out[:1]), dict(w_out=w_out.half()),
        dict(act="relu"), dict(out=y[:3]), dict(out=y.half()), dict(out=w_out.view(-1, 64)[:8]),
    ]
    for change in bad:
        args = dict(x=x, counts=c, w_in=w_in, w_out=w_out) | change
        with pytest.raises(ValueError):
            ops.expert_ffn(**args)
    shifted = torch.empty(8 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(8, 64)
    with pytest.raises(ValueError, match="aligned"):
        ops.expert_ffn(shifted, c, w_in, w_out)
    buf = torch.empty(9, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        ops.expert_ffn(buf[:8], c, w_in, w_out, out=buf[1:])
    with pytest.raises(ValueError, match="overlap"):
        ops.expert_ffn_train(x, c, w_in, w_out, out=x)
    for kw in (dict(dx=saved.h[:, :64]), dict(dw_in=w_in), dict(dw_out=w_out), dict(dx=x[:4])):
        with pytest.raises(ValueError):
            ops.expert_ffn_backward(dy, x, c, w_in, w_out, saved, **kw)
    with pytest.raises(ValueError):
        ops.expert_ffn_backward(dy, x, c, w_in, w_out, ops.ExpertFFNSaved(saved.h[:4], saved.gu))
    with pytest.raises(ValueError):
        ops.expert_ffn_backward(dy[:4], x, c, w_in, w_out, saved)


def test_kernel_reports_name_the_operators():
    from ugdr_b200 import ops

    names = [a["name"] for a in ops.kernel_attributes()]
    for want in ("expert_kernel<bf16, up>", "expert_kernel<fp16, grad in>", "expert_split_kernel<bf16, down>",
                 "grad_norm_kernel", "grad_scale_kernel"):
        assert want in names, names
    assert all(a["local_bytes_per_thread"] == 0 and a["blocks_per_sm"] == 1 for a in ops.kernel_attributes()
               if a["name"].startswith("expert"))


def test_moe_layer_trains_through_the_exchange():
    """A rank's MoE layer with real experts, as a training step runs it: dispatch, experts, combine,
    the gradients back the same way, the weights' gradients clipped; against fp64.  One expert per
    (token, k) row; the tolerance adds the roundings of the combine and of dy * w to the experts'."""
    from ugdr_b200 import ops
    from ugdr_b200.models.moe import route
    from ugdr_b200.parallel.collectives import MoEAllToAll
    from ugdr_b200.parallel.peers import PeerGroup

    tokens, hidden, inner, experts = 300, 128, 192, 8
    recv = tokens + 100
    g = PeerGroup(MoEAllToAll.required_bytes(1, experts, hidden, recv), 0, 1, lambda v: [v])
    moe = MoEAllToAll(g, tokens, hidden, 1, experts, recv)
    x, _, w_in, w_out, dout = inputs([tokens] + [0] * (experts - 1), hidden, inner, torch.bfloat16)
    ids, _ = route(tokens, experts, 1, seed=3)
    w = torch.rand(tokens, 1, device="cuda") + 0.5

    moe.dispatch(x, ids)
    counts = moe.expert_rows()
    rows = moe.recv_view().clone()
    _, saved = ops.expert_ffn_train(rows, counts, w_in, w_out, out=moe.recv_view())
    moe.ready()
    out = moe.combine(w)
    dyt = (dout.float() * w).to(torch.bfloat16)
    moe.dispatch(dyt, ids)
    dx, dw_in, dw_out = ops.expert_ffn_backward(moe.recv_view(), rows, counts, w_in, w_out, saved,
                                                dx=moe.recv_view())
    moe.ready()
    dxt = moe.combine(torch.ones_like(w))
    torch.cuda.synchronize()
    g.check_status()
    ops.check_status()
    assert counts.tolist() == torch.bincount(ids.reshape(-1).long(), minlength=experts).tolist()
    half = torch.finfo(torch.bfloat16).eps / 2
    grads = []
    for e in range(experts):
        mine = (ids.reshape(-1) == e).nonzero().reshape(-1)
        o = oracle(x[mine], w_in[e], w_out[e], "silu", dyt[mine])
        y, b = o["y"]
        we = w[mine].double()
        near(out[mine], y * we, (b * we + (y.abs() + b) * we * half) * 1.001, f"out of expert {e}")
        v, b = o["dx"]
        near(dxt[mine], v, b + (v.abs() + b) * half, f"dx of expert {e}")
        for name, t in (("dw_in", dw_in), ("dw_out", dw_out)):
            near(t[e], *o[name], f"{name} of expert {e}")
            grads.append(o[name][0])
    before = [t.clone() for t in (dw_in, dw_out)]
    total = math.sqrt(sum(float((t.double() ** 2).sum()) for t in before))
    norm = ops.GradClip([dw_in, dw_out]).clip(0.5 * total)
    assert abs(float(norm) - total) <= 1e-6 * total
    for t, b in zip((dw_in, dw_out), before):
        near(t, b.double() * 0.5, b.double().abs() * 0.5 * (half + 1e-6) + 1e-38, "clipped")

    # Serving: the experts in place in the receive area.
    moe.dispatch(x, ids)
    ops.expert_ffn(moe.recv_view(), moe.expert_rows(), w_in, w_out, out=moe.recv_view())
    moe.ready()
    assert torch.equal(moe.combine(w), out)
