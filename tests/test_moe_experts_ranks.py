"""Experts between the exchange's dispatch and combine with more than one rank: the counts that a rank takes
from the table (on the host), and whole steps with uneven routing in which one rank's experts are late
(one process per GPU; the same steps on one rank as well)."""
from __future__ import annotations

import datetime
import json
import os
import subprocess
import sys
import threading
import types

import pytest

from conftest import REPO, gpu_count

torch = pytest.importorskip("torch")

TOKENS, HIDDEN, INNER, EXPERTS, TOPK, STEPS = 200, 128, 192, 8, 3, 4


@pytest.mark.parametrize("world,rank", [(1, 0), (2, 0), (2, 1), (4, 2)])
def test_expert_rows_are_the_sums_over_all_sources_of_this_ranks_experts(world, rank):
    from ugdr_b200.parallel.collectives import MoEAllToAll

    table = torch.arange(world * EXPERTS, dtype=torch.int32).view(world, EXPERTS) ** 2
    a2a = MoEAllToAll.__new__(MoEAllToAll)
    a2a.g = types.SimpleNamespace(world=world, rank=rank, view=lambda dtype, n, offset: table.reshape(-1).view(dtype)[
        offset // 4:offset // 4 + n])
    a2a.nexp, a2a.exp_per_rank, a2a.table_off = EXPERTS, EXPERTS // world, 0
    want = [sum(int(table[s, e]) for s in range(world)) for e in range(rank * EXPERTS // world, (rank + 1) * EXPERTS // world)]
    got = a2a.expert_rows()
    assert got.dtype == torch.int32 and got.tolist() == want


def test_the_benchmarks_check_sees_a_wrong_row_on_any_rank():
    """Two ranks as threads: right outputs pass on both, and a row whose last expert was missed, or that has
    another's result, fails on the rank that has it."""
    from ugdr_b200.parallel.bench import _experts_right

    world, tokens, hidden, inner, experts, topk = 2, 5, 64, 48, 6, 3
    gen = torch.Generator().manual_seed(3)
    w_in, w_out = (torch.randn(*s, generator=gen) * s[-1] ** -0.5 for s in ((experts, 2, inner, hidden), (experts, hidden, inner)))
    xs = [torch.randn(tokens, hidden, generator=gen).to(torch.bfloat16) for _ in range(world)]
    ids = [torch.stack([torch.randperm(experts, generator=gen)[:topk] for _ in range(tokens)]).to(torch.int32) for _ in range(world)]
    ws = [torch.rand(tokens, topk, generator=gen) + 0.5 for _ in range(world)]

    def layer(r, k_used=topk):
        out = torch.zeros(tokens, hidden)
        for t in range(tokens):
            for k in range(k_used):
                gate, up = w_in[ids[r][t, k]] @ xs[r][t].float()
                out[t] += ws[r][t, k] * (w_out[ids[r][t, k]] @ (torch.nn.functional.silu(gate) * up))
        return out.to(torch.bfloat16)

    barrier, box = threading.Barrier(world, timeout=60), [None] * world

    def verdicts(outs):
        got = [None] * world

        def rank(r):
            def exchange(obj):
                box[r] = obj
                barrier.wait()
                everyone = list(box)
                barrier.wait()
                return everyone

            own = slice(r * experts // world, (r + 1) * experts // world)
            got[r] = _experts_right(r, exchange, xs[r], ids[r], ws[r], w_in[own], w_out[own], outs[r])

        threads = [threading.Thread(target=rank, args=(r,)) for r in range(world)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        return got

    right = [layer(r) for r in range(world)]
    assert verdicts(right) == [True, True]
    missed = right[1].clone()
    missed[2] = layer(1, topk - 1)[2]
    assert verdicts([right[0], missed]) == [True, False]
    swapped = right[0].clone()
    swapped[[0, 1]] = swapped[[1, 0]]
    assert verdicts([swapped, right[1]]) == [False, True]


def routes(rank, step):
    """Uneven routing, another in every step: low experts are liked best, and some have no rows at all."""
    gen = torch.Generator().manual_seed(1000 * step + rank)
    logits = torch.rand(TOKENS, EXPERTS, generator=gen) - 0.15 * torch.arange(EXPERTS)
    logits[:, (step + 5) % EXPERTS] = -9.0
    return torch.topk(logits, TOPK, dim=-1).indices.to(torch.int32), torch.rand(TOKENS, TOPK, generator=gen) + 0.25


def steps_are_right(rank, world, exchange):
    """Steps of dispatch, experts in place, ready, combine, all of them before the first check, so that every
    rank takes every step; each against fp64.  The tolerance adds to an expert's the roundings of the
    weighted sum: TOPK products and sums in fp32, and one to bf16."""
    from test_gpu_experts import inputs, near, oracle
    from ugdr_b200 import ops
    from ugdr_b200.parallel.collectives import MoEAllToAll
    from ugdr_b200.parallel.peers import PeerGroup

    recv = TOKENS * TOPK * world + 64
    g = PeerGroup(MoEAllToAll.required_bytes(world, EXPERTS, HIDDEN, recv), rank, world, exchange)
    a2a = MoEAllToAll(g, TOKENS, HIDDEN, TOPK, EXPERTS, recv)
    _, _, w_in, w_out, _ = inputs([1] * EXPERTS, HIDDEN, INNER, torch.bfloat16)  # all ranks': the same everywhere
    own = slice(rank * EXPERTS // world, (rank + 1) * EXPERTS // world)
    mine = w_in[own].contiguous(), w_out[own].contiguous()
    taken = []
    for step in range(STEPS):
        gen = torch.Generator().manual_seed(77 + 1000 * step + rank)
        x = torch.randn(TOKENS, HIDDEN, generator=gen).to(torch.bfloat16).cuda()
        ids, w = (t.cuda() for t in routes(rank, step))
        a2a.dispatch(x, ids)
        counts, rows = a2a.expert_rows(), a2a.recv_view()
        if step % world == rank:
            torch.cuda._sleep(40_000_000)  # some 20 ms late with its experts
        ops.expert_ffn(rows, counts, *mine, out=rows)
        a2a.ready()
        taken.append((x, ids, w, counts, a2a.combine(w)))
    torch.cuda.synchronize()
    g.check_status()
    ops.check_status()
    half = torch.finfo(torch.bfloat16).eps / 2
    for step, (x, ids, w, counts, out) in enumerate(taken):
        everyone = torch.stack([routes(r, step)[0].reshape(-1) for r in range(world)]).reshape(-1).long()
        assert counts.tolist() == torch.bincount(everyone, minlength=EXPERTS)[own].tolist()
        want, bound, size = (torch.zeros(TOKENS, HIDDEN, dtype=torch.float64, device="cuda") for _ in range(3))
        for k in range(TOPK):
            for e in range(EXPERTS):
                t = (ids[:, k] == e).nonzero().reshape(-1)
                if t.numel():
                    y, b = oracle(x[t], w_in[e], w_out[e], "silu")["y"]
                    we = w[t, k:k + 1].double()
                    want[t] += y * we
                    bound[t] += b * we
                    size[t] += (y.abs() + b) * we
        bound += size * (TOPK + 1) * 2.0 ** -23
        near(out, want, bound + (want.abs() + bound) * half, f"step {step} on rank {rank}")
    g.close()


def _worker(rank, world, port, q):
    try:
        import torch.distributed as dist

        os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
        torch.cuda.set_device(rank)
        dist.init_process_group("gloo", rank=rank, world_size=world, timeout=datetime.timedelta(seconds=60))

        def exchange(obj):
            out = [None] * world
            dist.all_gather_object(out, obj)
            return out

        steps_are_right(rank, world, exchange)
        dist.barrier()
        q.put((rank, "ok"))
    except BaseException as e:  # report to the parent
        q.put((rank, repr(e)))


@pytest.mark.gpu
def test_steps_on_one_rank():
    if gpu_count() < 1:
        pytest.skip("no GPU")
    torch.cuda.set_device(0)
    steps_are_right(0, 1, lambda v: [v])


@pytest.mark.gpu
@pytest.mark.parametrize("world", [2, 4, 8])
def test_steps_on_several_ranks(world):
    if gpu_count() < world:
        pytest.skip(f"needs {world} GPUs")
    import torch.multiprocessing as mp

    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = 29850 + world + os.getpid() % 200
    ps = [ctx.Process(target=_worker, args=(r, world, port, q)) for r in range(world)]
    for p in ps:
        p.start()
    results = {}
    try:
        for _ in ps:
            r, msg = q.get(timeout=300)
            results[r] = msg
    finally:
        for p in ps:
            p.join(60)
            if p.is_alive():
                p.kill()
    assert results == {r: "ok" for r in range(world)}, results


@pytest.mark.gpu
def test_the_benchmark_checks_the_experts_results():
    if gpu_count() < 1:
        pytest.skip("no GPU")
    run = subprocess.run([sys.executable, "-m", "torch.distributed.run", "--nproc-per-node", "1", "--master-addr", "127.0.0.1",
                          "--master-port", str(30100 + os.getpid() % 200), "-m", "ugdr_b200.parallel.bench", "--op", "moe",
                          "--tokens", "256", "--inner", "64", "--iters", "1", "--warmup", "1"], cwd=REPO, timeout=240,
                         capture_output=True, text=True)
    assert run.returncode == 0, run.stderr[-2000:]
    line = json.loads(run.stdout.strip().splitlines()[-1])
    assert line["correct"] is True and line["experts_correct"] is True, line
