"""The paged 4-bit key/value cache on the GPU: page plan and rotary + quantising append against plain
restatements (``oracle/paged_oracle.py``), 64 bits, one element at a time."""
import random

import pytest
import torch

from oracle import paged_oracle as oracle

pytestmark = pytest.mark.gpu

HD = 128


@pytest.fixture(scope="module")
def ops(native_lib):
    from dynaflow_b200 import ops as _ops

    return _ops


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Plan:
    """Device state of a page pool next to the oracle's lists."""

    def __init__(self, ops, requests, max_pages, num_pages, page, seed):
        self.ops, self.page, self.rng = ops, page, random.Random(seed)
        order = list(range(num_pages))
        self.rng.shuffle(order)
        self.lists = [[[-1] * max_pages for _ in range(requests)], [0] * requests, order, num_pages]
        self.table, self.held, self.free, self.count = _i32(self.lists[0]), _i32(self.lists[1]), _i32(order), _i32([num_pages])

    def step(self, lens, fresh, rows, per_request=0):
        starts = torch.full((len(lens) + 1,), -7, dtype=torch.int32, device="cuda")
        slots, positions = torch.full((rows,), -7, dtype=torch.int32, device="cuda"), torch.full((rows,), -7, dtype=torch.int32, device="cuda")
        self.ops.page_plan(_i32(lens), _i32(fresh), self.table, self.held, self.free, self.count, starts, slots, positions,
                           page_size=self.page, rows_per_request=per_request)
        torch.cuda.synchronize()
        want = oracle.page_plan(lens, fresh, *self.lists, self.page, rows, per_request)
        got = (self.table.tolist(), self.held.tolist(), self.free.tolist(), self.count.item(), starts.tolist(), slots.tolist(), positions.tolist())
        for name, g, w in zip(("table", "held", "free", "count", "starts", "slots", "positions"), got, want):
            assert g == w, name
        self.lists = list(want[:4])
        return slots, positions, starts


# requests: one, odd, more than one block of the prefix sum, many; rows that make the plan one CTA or a cluster
@pytest.mark.parametrize("requests,page,longest", [(1, 16, 1), (3, 64, 200), (33, 48, 700), (1025, 16, 40), (2500, 16, 20)])
def test_plan_follows_requests_through_their_lives(ops, requests, page, longest):
    """Prompts, single tokens, several tokens at once, finished requests and rejected tokens, step by step."""
    max_pages = -(-longest // page) + 4
    plan = Plan(ops, requests, max_pages, requests * max_pages, page, requests)
    rng = plan.rng
    lens = [0] * requests
    for step in range(6):
        fresh = []
        for b in range(requests):
            kind = rng.random()
            if lens[b] == 0:
                new = rng.randint(1, longest) if kind < 0.7 else 0
            elif kind < 0.15:
                lens[b], new = 0, 0                                     # finished
            elif kind < 0.3:
                lens[b], new = rng.randint(1, lens[b]), 0               # drafted tokens taken back
            else:
                new = rng.choice([0, 1, 1, 4])
            lens[b] += new
            fresh.append(new)
        most = max(fresh)
        if step % 2:
            plan.step(lens, fresh, requests * max(most, 1) + rng.choice([0, 5]), max(most, 1))
        else:
            plan.step(lens, fresh, sum(fresh) + rng.choice([0, 3]))
    ops.check_status()


def test_plan_taken_back_restores_the_free_list(ops):
    plan = Plan(ops, 5, 8, 30, 16, 1)
    plan.step([20, 0, 33, 1, 64], [20, 0, 33, 1, 64], 118)
    before = (plan.table.clone(), plan.held.clone(), plan.free.clone(), plan.count.clone())
    plan.step([60, 40, 34, 17, 80], [40, 40, 1, 16, 16], 113)
    plan.step([20, 0, 33, 1, 64], [0] * 5, 0)
    for a, b in zip((plan.table, plan.held, plan.count), (before[0], before[1], before[3])):
        assert torch.equal(a, b)
    n = int(before[3])
    assert torch.equal(plan.free[:n], before[2][:n])
    ops.check_status()


def test_plan_reports_too_few_pages_and_gives_none(ops):
    plan = Plan(ops, 3, 8, 6, 16, 2)
    plan.step([32, 16, 0], [32, 16, 0], 48)
    ops.check_status()
    # 2 + 1 held, 3 free: request 0 wants 2 more and request 2 wants 2; request 1 is over and gives one back: 4 for 4
    plan.step([64, 0, 32], [32, 0, 32], 64)
    ops.check_status()
    plan.step([65, 0, 32], [1, 0, 0], 1)                 # nothing is left
    with pytest.raises(ops.DeviceStatusError, match="pages missing"):
        ops.check_status()
    ops.check_status()                                   # cleared


def test_plan_reports_a_full_table_row(ops):
    plan = Plan(ops, 2, 2, 8, 16, 3)
    plan.step([33, 5], [33, 5], 38)
    with pytest.raises(ops.DeviceStatusError, match="table row full"):
        ops.check_status()


def test_plan_reports_missing_rows(ops):
    plan = Plan(ops, 2, 4, 8, 16, 4)
    plan.step([20, 5], [20, 5], 22)
    with pytest.raises(ops.DeviceStatusError, match="rows missing"):
        ops.check_status()
    plan.step([22, 5], [2, 0], 2, 1)                     # two new tokens, one row a request
    with pytest.raises(ops.DeviceStatusError, match="rows missing"):
        ops.check_status()


@pytest.mark.parametrize("lens,fresh", [([-5, 2 ** 31 - 1], [3, 2 ** 31 - 1]), ([2 ** 31 - 1] * 2, [2 ** 31 - 1] * 2), ([5, 7], [-1, 9])])
def test_plan_with_senseless_lengths_stays_in_its_buffers(ops, lens, fresh):
    guard = torch.full((64,), 77, dtype=torch.int32, device="cuda")
    table, held, free = guard[8:16].view(2, 4), guard[16:18], guard[24:32]
    table.fill_(-1), held.fill_(0), free.copy_(torch.arange(8))
    count, starts, slots, positions = guard[33:34].fill_(8), guard[36:39], guard[44:48], guard[52:56]
    ops.page_plan(_i32(lens), _i32(fresh), table, held, free, count, starts, slots, positions, page_size=16)
    torch.cuda.synchronize()
    for a, b in ((0, 8), (18, 24), (32, 33), (34, 36), (39, 44), (48, 52), (56, 64)):
        assert (guard[a:b] == 77).all()
    assert ((table >= -1) & (table < 8)).all() and ((slots >= -1) & (slots < 128)).all() and 0 <= count.item() <= 8
    ops.read_status()
    ops._native.load().df_status_clear(ops.status_block().data_ptr(), None)
    torch.cuda.synchronize()


def test_plan_in_a_graph(ops):
    plan = Plan(ops, 4, 8, 32, 16, 5)
    lens, fresh = _i32([0] * 4), _i32([1] * 4)
    starts, slots, positions = _i32([0] * 5), _i32([0] * 4), _i32([0] * 4)

    def step():
        lens.add_(1)
        ops.page_plan(lens, fresh, plan.table, plan.held, plan.free, plan.count, starts, slots, positions, page_size=16, rows_per_request=1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        ops.status_block()
        with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
            step()
    torch.cuda.current_stream().wait_stream(side)
    for n in range(1, 40):
        graph.replay()
        torch.cuda.synchronize()
        want = oracle.page_plan([n] * 4, [1] * 4, *plan.lists, 16, 4, 1)
        assert slots.tolist() == want[5] and positions.tolist() == want[6] and plan.table.tolist() == want[0]
        plan.lists = list(want[:4])
    ops.check_status()


# ------------------------------------------------------------------ append
def _append(ops, rows, hq, hkv, page, seed, *, scale=1.0, pad=(), in_place=False, wide=0, theta=10000.0, longest=5000):
    g = torch.Generator().manual_seed(seed)
    cols = (hq + 2 * hkv) * HD
    qkv = (torch.randn(rows, cols, generator=g) * scale).bfloat16()
    pages = -(-rows // page) + 2
    slots = torch.randperm(pages * page, generator=g)[:rows].to(torch.int32)
    positions = torch.randint(0, longest, (rows,), generator=g, dtype=torch.int32)
    positions[-1] = longest - 1
    for r in pad:
        slots[r] = -1
    room = torch.full((rows, cols + wide), 3.0, dtype=torch.bfloat16, device="cuda")
    room[:, :cols] = qkv.cuda()
    src = room[:, :cols]
    cache = torch.full((pages, hkv, page * 136), 0xAB, dtype=torch.uint8, device="cuda")
    out = src if in_place else torch.full((rows, cols), 5.0, dtype=torch.bfloat16, device="cuda")
    ops.rope_append_paged4(src, positions.cuda(), slots.cuda(), ops.rope_angles(longest, theta), hq, hkv, cache, page_size=page, out=out)
    torch.cuda.synchronize()
    if not in_place:
        assert torch.equal(src.cpu(), qkv)
    if wide:
        assert (room[:, cols:] == 3.0).all()
    return qkv, positions, slots, cache.cpu(), out.cpu()


def _check_append(qkv, positions, slots, cache, out, hq, hkv, page, theta=10000.0, untouched=5.0):
    """The rotated rows are within one rounding (bf16: half a step, 2^-8 of the value) and 3 fp32 operations of the 64-bit
    ones; the cache holds the quantisation of exactly the bf16 keys and values, and ``out`` what the cache stands for."""
    rows = qkv.shape[0]
    x = qkv.view(rows, hq + 2 * hkv, HD)
    want = oracle.rotate(x[:, :hq + hkv], positions, theta)
    got = out.view(rows, hq + 2 * hkv, HD)
    real = slots >= 0
    assert (got[~real] == (x[~real] if untouched is None else untouched)).all()
    # |error| <= 2^-8 |value| + 2^-21 (|u| + |v|): angles and products in fp32 (half a step 2^-24 each, four of them)
    room = x[:, :hq + hkv].double().abs()
    room = (room[..., :64] + room[..., 64:]).repeat(1, 1, 2)
    err = (got[:, :hq].double() - want[:, :hq]).abs()[real]
    assert (err <= want[:, :hq].abs()[real] * 2 ** -8 + room[:, :hq][real] * 2 ** -21).all()
    key_rows = want[:, hq:].bfloat16()
    free = torch.ones(cache.shape[0] * page, dtype=torch.bool)
    free[slots[real].long()] = False
    for r in [i for i in range(rows) if real[i]][:: max(1, rows // 40)]:
        for h in range(hkv):
            k, v = oracle.read_token(cache, int(slots[r]), h, page)
            assert torch.equal(got[r, hq + h].double(), k.bfloat16().double()) and torch.equal(got[r, hq + hkv + h].double(), v.bfloat16().double())
            codes, step, low = oracle.quantise(x[r, hq + hkv + h])
            assert torch.equal(v, step * codes + low)
            # both are within half a step of their key (and 15 steps' rounding of the scale, 15 * 2^-9 of a step, at the ends);
            # the two keys are at most one bf16 step (2^-7) apart, the two scales at most that
            codes, step, low = oracle.quantise(key_rows[r, h])
            assert ((k - (step * codes + low)).abs() <= step * (1 + 2 ** -7) * (1 + 15 * 2 ** -8) + key_rows[r, h].double().abs() * 2 ** -7).all()
    # slots that no row has keep their bytes
    for s in free.nonzero()[:, 0].tolist()[:30]:
        page_id, at = divmod(s, page)
        granule, r = divmod(at, 16)
        for base in (0, 1088):
            o = granule * 2176 + base
            assert (cache[page_id, :, o + r * 64:o + r * 64 + 64] == 0xAB).all() and (cache[page_id, :, o + 1024 + r * 4:o + 1028 + r * 4] == 0xAB).all()


@pytest.mark.parametrize("rows,hq,hkv,page", [(1, 1, 1, 16), (2, 4, 1, 64), (37, 6, 2, 48), (130, 32, 8, 32), (700, 3, 3, 128), (5, 0, 2, 16)])
def test_append_quantises_into_the_slots(ops, rows, hq, hkv, page):
    case = _append(ops, rows, hq, hkv, page, rows)
    _check_append(*case, hq, hkv, page)


def test_append_in_place_with_padding_rows_and_a_wider_buffer(ops):
    case = _append(ops, 50, 8, 2, 32, 3, pad=(0, 17, 49), in_place=True, wide=72)
    _check_append(*case, 8, 2, 32, untouched=None)


def test_append_keeps_padding_rows_of_the_output(ops):
    case = _append(ops, 9, 4, 1, 16, 4, pad=(3, 8))
    _check_append(*case, 4, 1, 16)


def test_append_at_far_positions(ops):
    case = _append(ops, 20, 4, 2, 16, 5, longest=1 << 20, theta=500000.0)
    _check_append(*case, 4, 2, 16, theta=500000.0)


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 1e30])
def test_append_of_tiny_and_huge_values(ops, scale):
    case = _append(ops, 20, 4, 2, 16, 6, scale=scale)
    _check_append(*case, 4, 2, 16)


def test_append_of_constant_and_nan_rows(ops):
    hq, hkv, page = 1, 1, 16
    qkv = torch.zeros(3, 3 * HD, dtype=torch.bfloat16, device="cuda")
    qkv[0, 2 * HD:] = 2.5                                 # a constant value: scale 0
    qkv[1, 2 * HD + 7] = float("nan")
    qkv[2, HD:] = torch.randn(2 * HD)
    cache = ops.paged4_cache(1, hkv, page).zero_()
    ops.rope_append_paged4(qkv, _i32([0, 0, 0]), _i32([3, 4, 5]), ops.rope_angles(4, 10000.0), hq, hkv, cache, page_size=page)
    torch.cuda.synchronize()
    assert (qkv[0, 2 * HD:] == 2.5).all()
    assert torch.isnan(qkv[1, 2 * HD:]).all()             # a NaN in a value is not lost
    assert torch.isfinite(qkv[2].float()).all()
    k, v = oracle.read_token(cache.cpu(), 3, 0, page)
    assert (v == 2.5).all() and (k == 0).all()


def test_append_with_slots_and_positions_out_of_range_is_padding(ops):
    qkv = torch.randn(4, 3 * HD).bfloat16().cuda()
    before = qkv.clone()
    cache = ops.paged4_cache(2, 1, 16).fill_(0xAB)
    ops.rope_append_paged4(qkv, _i32([0, -1, 8, 1]), _i32([32, 1, 2, 2 ** 31 - 1]), ops.rope_angles(8, 10000.0), 1, 1, cache, page_size=16)
    torch.cuda.synchronize()
    assert torch.equal(qkv, before) and (cache == 0xAB).all()
