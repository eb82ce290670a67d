"""The global gradient norm and clipping against fp64.

Tolerances: the sum of squares is built from fp32 sums of 8 squares (8 roundings of 2^-24) added in
fp64, so the norm is within 4 * 2^-24 plus its own rounding of 2^-24; the factor is rounded to
fp32, the product to fp32 and the output to its type (eps / 2, or half the smallest subnormal)."""
from __future__ import annotations

import math

import pytest

from conftest import gpu_count

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

NORM_REL = 6 * 2.0 ** -24
SCALE_REL = 9 * 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def one_gpu():
    if gpu_count() < 1:
        pytest.skip("no GPU")
    torch.cuda.set_device(0)


def tensors(sizes, dtypes, scale=1.0, offset=0, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        dtype = getattr(torch, dtypes[i % len(dtypes)])
        t = torch.empty(n + offset, dtype=dtype, device="cuda")[offset:]
        out.append(t.normal_(0, scale, generator=gen))
    return out


def norm64(grads):
    return math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))


def check_scaled(out, before, coef):
    for o, b in zip(out, before):
        f = torch.finfo(o.dtype)
        want = b.double() * coef
        tol = want.abs() * (f.eps / 2 + SCALE_REL) + f.smallest_normal * f.eps / 2
        assert bool(((o.double() - want).abs() <= tol).all()), (o.shape, o.dtype)


SIZES = [[1], [7], [8], [4095, 4096, 4097], [1, 2, 3, 0, 5, 8191], [0], [0, 0, 9, 0], [1_000_003],
         [3] * 700, [100_000, 1, 65536, 12_345, 0, 777]]


@pytest.mark.parametrize("dtypes", [["bfloat16"], ["float16"], ["float32"], ["bfloat16", "float32", "float16"]])
@pytest.mark.parametrize("sizes", SIZES)
def test_norm_and_scaling(sizes, dtypes):
    from ugdr_b200.ops import GradClip

    for offset in (0, 1, 3):
        grads = tensors(sizes, dtypes, 0.3, offset)
        before = [g.clone() for g in grads]
        want = norm64(before)
        into = [torch.empty(g.numel() + offset, device="cuda")[offset:] for g in grads]
        limit = 0.25 * want
        coef = min(1.0, limit / (want + 1e-6))
        for out in (None, into, [torch.empty_like(g) for g in grads]):
            plan = GradClip(grads, out)
            assert abs(float(plan.sum_squares()) - want ** 2) <= 2 * NORM_REL * want ** 2
            # Within the limit: in place nothing changes, elsewhere they are copied.
            assert abs(float(plan.clip(2 * want + 1)) - want) <= NORM_REL * want
            assert all(torch.equal(o, b.to(o.dtype)) for o, b in zip(plan.out, before))
            assert abs(float(plan.clip(limit)) - want) <= NORM_REL * want
            check_scaled(plan.out, before, coef)
            for g, b in zip(grads, before):
                g.copy_(b)


def test_memory_around_the_tensors_stays():
    from ugdr_b200.ops import GradClip

    for dtype in (torch.bfloat16, torch.float32):
        for lead, n, tail in ((1, 4099, 5), (7, 13, 1), (3, 1, 3), (8, 8192, 8)):
            flat = torch.full((lead + n + tail,), 9.0, dtype=dtype, device="cuda")
            flat[lead:lead + n] = 1.0
            GradClip([flat[lead:lead + n]]).clip(0.0)
            assert bool((flat[lead:lead + n] == 0).all())
            assert bool((flat[:lead] == 9).all()) and bool((flat[lead + n:] == 9).all())


def test_out_of_another_alignment():
    from ugdr_b200.ops import GradClip

    g = tensors([10_001], ["bfloat16"], 1.0, 3)[0]
    for lead in range(8):
        out = torch.zeros(10_020, dtype=torch.float32, device="cuda")
        GradClip([g], [out[lead:lead + 10_001]]).clip(1e9)
        assert torch.equal(out[lead:lead + 10_001], g.float())
        assert not bool(out[:lead].any()) and not bool(out[lead + 10_001:].any())


@pytest.mark.parametrize("scale", [1e-30, 1e-22, 1e-15, 1e15, 3e18, 1e25, 1e30])
def test_ranges_where_fp32_squares_leave_their_type(scale):
    from ugdr_b200.ops import GradClip

    for dtype in ("float32", "bfloat16"):
        grads = tensors([5000, 33], [dtype], scale)
        grads[1].zero_()
        grads[1][3] = scale
        want = norm64(grads)
        assert abs(float(GradClip(grads).clip(float("inf"))) - want) <= NORM_REL * want


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("scale", [1e-30, 1.0])
def test_groups_of_zeros_between_others(dtype, scale):
    """Groups of zeros of either sign between numbers whose squares fp32 holds, or does not."""
    from ugdr_b200.ops import GradClip

    dtype = getattr(torch, dtype)
    if dtype == torch.float16 and scale < 1:
        scale = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # its smallest number
    for n in (40, 8 * 4096 + 5, 3_000_007):
        g = torch.zeros(n, dtype=dtype, device="cuda")
        g[torch.arange(n, device="cuda") % 48 < 16] = -0.0
        g[::40] = scale
        g[n // 2:n // 2 + 3] = 2 * scale
        want = norm64([g])
        assert want > 0 and abs(float(GradClip([g]).clip(float("inf"))) - want) <= NORM_REL * want


def test_zeros_infinities_and_nans():
    from ugdr_b200.ops import GradClip

    z = torch.zeros(1000, device="cuda")
    assert float(GradClip([z]).clip(1.0)) == 0.0
    g = torch.ones(1000, device="cuda")
    g[10] = float("inf")
    assert float(GradClip([g]).clip(1.0)) == float("inf")  # scaled by 0: inf * 0 is a NaN
    assert bool(g[10].isnan()) and bool((g[:10] == 0).all()) and bool((g[11:] == 0).all())
    g = torch.ones(1000, dtype=torch.bfloat16, device="cuda")
    g[999] = float("nan")
    assert math.isnan(float(GradClip([g]).clip(1.0))) and bool(g.isnan().all())


def test_total_of_other_ranks():
    """The norm over this rank's and others' gradients: the sums of squares added, then clipped."""
    from ugdr_b200.ops import GradClip

    mine, theirs = tensors([5000, 77], ["bfloat16"], 0.1, seed=1), tensors([9000], ["float32"], 0.2, seed=2)
    before, want = [g.clone() for g in mine], norm64(mine + theirs)
    a, b = GradClip(mine), GradClip(theirs)
    total = a.sum_squares() + b.sum_squares()
    assert abs(float(a.clip(1.0, sum_squares=total)) - want) <= NORM_REL * want
    check_scaled(mine, before, 1.0 / (want + 1e-6))


def test_repeats_streams_and_graphs():
    from ugdr_b200.ops import GradClip

    grads = tensors([300_000, 17, 4096 * 50 + 1], ["bfloat16", "float32"], 0.5)
    out = [torch.empty(g.numel(), device="cuda") for g in grads]
    out2 = [torch.empty(g.numel(), device="cuda") for g in grads]
    plan, plan2 = GradClip(grads, out), GradClip(grads, out2)
    first = plan.clip(1.0)
    want = [o.clone() for o in out]
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    norms = []
    for _ in range(20):
        norms += [plan.clip(1.0, stream=s1), plan2.clip(1.0, stream=s2)]
    torch.cuda.synchronize()
    assert all(torch.equal(n, first) for n in norms)
    assert all(torch.equal(a, w) and torch.equal(b, w) for a, b, w in zip(out, out2, want))
    graphs = []
    for p in (plan, plan2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            n = p.clip(1.0)
        graphs.append((g, n))
    for g in grads:
        g.mul_(3.0)
    now = norm64(grads)
    torch.cuda.synchronize()
    for (g, _), s in zip(graphs, (s1, s2)):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    for _, n in graphs:
        assert abs(float(n) - now) <= NORM_REL * now
    check_scaled(out, grads, 1.0 / (now + 1e-6))
    assert all(torch.equal(a, b) for a, b in zip(out, out2))


def test_after_an_allreduce_in_the_symmetric_buffer():
    """Gradients summed in the peer group's buffer, clipped there through views of it."""
    from ugdr_b200.ops import GradClip
    from ugdr_b200.parallel.collectives import allreduce_bf16
    from ugdr_b200.parallel.peers import PeerGroup

    sizes = [4096, 1000, 24]
    group = PeerGroup(2 * sum(sizes), 0, 1, lambda v: [v])
    flat = group.view(torch.bfloat16, sum(sizes))
    flat.normal_(0, 1)
    before = flat.clone()
    plan = GradClip(list(flat.split(sizes)))
    allreduce_bf16(group, flat.numel())
    norm = plan.clip(2.0)
    torch.cuda.synchronize()
    group.check_status()
    want = norm64([before])
    assert abs(float(norm) - want) <= NORM_REL * want
    check_scaled([flat], [before], 2.0 / (want + 1e-6))


def test_more_than_2_to_the_32_elements():
    from ugdr_b200.ops import GradClip

    n = (1 << 32) + 4101
    if torch.cuda.mem_get_info()[0] < 3 * n:
        pytest.skip("needs 13 GB of free GPU memory")
    g = torch.full((n,), 2.0 ** -8, dtype=torch.bfloat16, device="cuda")
    want = math.sqrt(n) * 2.0 ** -8
    assert abs(float(GradClip([g]).clip(want / 4)) - want) <= NORM_REL * want
    for part in (g[:5000], g[1 << 31:(1 << 31) + 5000], g[-5000:]):
        assert bool((part == 2.0 ** -10).all())


def test_refusals():
    from ugdr_b200.ops import GradClip

    g = torch.ones(64, device="cuda")
    for grads, out in (([], None), ([g.double()], None), ([g.cpu()], None), ([g[::2]], None), ([None], None),
                       ([g], []), ([g], [g[:32]]), ([g], [g.half()]), ([g.half()], [g.bfloat16()]),
                       ([g[:32]], [g[16:48]]), ([g, g], None), ([g[:32], g[16:48]], None),
                       ([g[:32], g[32:]], [torch.empty_like(g[:32]), g[:32]]), ([g[:16], g[16:32]], [g[32:48], g[40:56]])):
        with pytest.raises(ValueError):
            GradClip(grads, out)
    plan = GradClip([g])
    for limit in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            plan.clip(limit)
    for total in (torch.zeros((), device="cuda"), torch.zeros((), dtype=torch.float64), 1.0,
                  torch.zeros(2, dtype=torch.float64, device="cuda")):
        with pytest.raises(ValueError):
            plan.clip(1.0, sum_squares=total)
    other = [torch.empty_like(g), torch.empty_like(g)]
    GradClip([g, g], other).clip(1.0)  # read twice, written apart
    assert torch.equal(other[0], other[1])
