"""Log probabilities of a vocabulary that is split over ranks: the host's part on two gloo ranks, the kernels replaced by
plain 64-bit stand-ins that keep the records' meaning (maximum, sums, the given token's logit, the largest keys)."""
import os
import subprocess
import sys
import textwrap

from conftest import ROOT

WORKER = textwrap.dedent("""
    import os, sys, types
    import torch, torch.distributed as dist
    sys.path.insert(0, {root!r})
    from dynaflow_b200 import ops
    from dynaflow_b200.decoder import TensorParallelDecoder

    rank, world = int(os.environ["RANK"]), int(os.environ["WORLD_SIZE"])
    dist.init_process_group("gloo")
    rows, vocab, top = 5, 40, 3
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(rows, vocab, generator=g, dtype=torch.float64)
    ids = torch.tensor([0, 19, 20, 39, 7])
    per = vocab // world

    def shard(lg, chosen, start, k, record, workspace):
        assert start == rank * per and lg.shape[1] == per
        here = (chosen >= start) & (chosen < start + per)
        x = torch.where(here, lg.gather(1, (chosen - start).clamp(0, per - 1)[:, None])[:, 0], -torch.inf)
        value, at = lg.sort(1, descending=True)
        record.copy_(torch.cat([lg.exp().sum(1), x, value[:, :k].flatten(), (at[:, :k] + start).double().flatten()]).view(torch.uint8))
        return record

    def join(records, parts, n, k):
        assert parts == world
        r = records.view(torch.float64).view(parts, -1)
        s, x = r[:, :n].sum(0), r[:, n:2 * n].amax(0)
        value = r[:, 2 * n:(2 + k) * n].view(parts, n, k).transpose(0, 1).reshape(n, -1)
        at = r[:, (2 + k) * n:].view(parts, n, k).transpose(0, 1).reshape(n, -1)
        best, i = value.sort(1, descending=True)
        return x - s.log(), s, at.gather(1, i)[:, :k].int(), best[:, :k] - s.log()[:, None]

    ops.token_logprobs_shard, ops.token_logprobs_join = shard, join
    ops.token_logprobs_record = lambda n, k, device: torch.empty(8 * n * (2 + 2 * k), dtype=torch.uint8)
    ops.token_logprobs_workspace = lambda *a: None
    dec = types.SimpleNamespace(world=world, rank=rank, d_cuts=[0, 2, rows])
    mine = logits[:, rank * per:(rank + 1) * per]
    lp, _, top_ids, top_lp = TensorParallelDecoder.token_logprobs(dec, [mine[:2], mine[2:]], ids, top)
    want = torch.log_softmax(logits, -1)
    assert torch.allclose(lp, want.gather(1, ids[:, None])[:, 0])
    assert torch.equal(top_ids.long(), want.sort(1, descending=True).indices[:, :top])
    assert torch.allclose(top_lp, want.sort(1, descending=True).values[:, :top])
    dist.barrier()
    dist.destroy_process_group()
    if rank == 0:
        print("SPLIT_VOCABULARY_OK")
""")


def test_records_of_two_ranks_are_gathered_in_rank_order(tmp_path):
    script = tmp_path / "worker.py"
    script.write_text(WORKER.format(root=ROOT))
    env = dict(os.environ, OMP_NUM_THREADS="1")
    port = 29500 + os.getpid() % 400
    r = subprocess.run([sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node", "2", "--master-addr", "127.0.0.1",
                        "--master-port", str(port), str(script)], capture_output=True, text=True, timeout=240, env=env)
    assert r.returncode == 0 and "SPLIT_VOCABULARY_OK" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]
