"""The paged operators with thousands of requests."""
import os
import random
import subprocess
import sys
import textwrap

import pytest
import test_gpu_paged_attention as attention
import torch

from conftest import ROOT
from dynaflow_b200 import ops

pytestmark = pytest.mark.gpu

PLAN_WORKER = textwrap.dedent("""
    import random, sys
    import torch
    sys.path.insert(0, {root!r})
    from dynaflow_b200 import ops
    from oracle import paged_oracle as oracle

    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    for requests in {sizes}:
        rng = random.Random(requests)
        page, max_pages = 16, 3
        lens, fresh = [], []
        for _ in range(requests):
            lens.append(rng.randint(0, 40))
            fresh.append(rng.randint(0, min(lens[-1], 3)))
        order = list(range(requests * max_pages))
        rng.shuffle(order)
        state = [[-1] * max_pages for _ in range(requests)], [0] * requests, order, len(order)
        table, held, free, count = map(i32, (state[0], state[1], order, [len(order)]))
        for step in range(2):
            rows = sum(fresh) + 5
            starts, slots, positions = (torch.full((n,), -7, dtype=torch.int32, device="cuda") for n in (requests + 1, rows, rows))
            ops.page_plan(i32(lens), i32(fresh), table, held, free, count, starts, slots, positions, page_size=page)
            torch.cuda.synchronize()
            want = oracle.page_plan(lens, fresh, *state, page, rows)
            got = (table.tolist(), held.tolist(), free.tolist(), count.item(), starts.tolist(), slots.tolist(), positions.tolist())
            assert all(g == w for g, w in zip(got, want)), (requests, step)
            state = want[:4]
            lens = [n + 1 if rng.random() < 0.7 else n // 2 for n in lens]
            fresh = [min(1, n) for n in lens]
        ops.check_status()
    print("PLANS_OK")
""")


@pytest.mark.parametrize("sizes", [(4064, 2, 8192), (4095, 4063), (4096, 4064)])
def test_plan_of_thousands_of_requests_first_in_its_process(native_lib, tmp_path, sizes):
    """From 4064 requests on the prefix sums and the kernel's own shared memory pass what a launch has without asking; an
    earlier larger call in the process would have asked already."""
    script = tmp_path / "worker.py"
    script.write_text(PLAN_WORKER.format(root=ROOT, sizes=sizes))
    r = subprocess.run([sys.executable, str(script)], capture_output=True, text=True, timeout=240, cwd=ROOT, env=dict(os.environ))
    assert r.returncode == 0 and "PLANS_OK" in r.stdout, r.stdout[-1000:] + r.stderr[-2000:]


# more requests than have their lengths and prefix sums in shared memory (1024), around that number and odd
@pytest.mark.parametrize("requests,max_ctas", [(1024, 0), (1025, 0), (1025, 3), (3001, 0), (3001, 1)])
@pytest.mark.parametrize("several", [False, True])
def test_attention_of_thousands_of_requests(native_lib, requests, max_ctas, several):
    """Empty requests, one token, several pages; one long one, which is cut; with several new tokens some without any."""
    rng = random.Random(requests + max_ctas)
    lens = [rng.choice([0, 1, 15, 16, 17, 40]) for _ in range(requests)]
    lens[requests // 3] = 1500
    case = attention.Case(lens, 1, 16, requests)
    fresh = [min(n, rng.choice([0, 1, 1, 2, 3])) for n in lens] if several else [1] * requests
    starts = [sum(fresh[:b]) for b in range(requests + 1)] if several else list(range(requests + 1))
    rows = starts[-1] + (3 if several else 0)
    q = torch.randn(rows, 4 * 128, generator=torch.Generator().manual_seed(requests)).bfloat16()
    more = dict(fresh=fresh, starts=starts, max_new=3) if several else {}
    got = attention._run(ops, case, q, 4, max_ctas=max_ctas, **more)
    want, tol = attention._want(case, q, starts, fresh, 4, 128 ** -0.5)
    served = torch.zeros(rows, dtype=torch.bool)
    served[:starts[-1]] = True
    attention._check(got, want, tol, served)
