"""The paged operators with thousands of requests."""
import os
import subprocess
import sys
import textwrap

import pytest

from conftest import ROOT

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
