"""Token log probabilities against 64-bit log-softmax, entropies and sorted logits."""
import math
import random

import pytest
import torch

from oracle import paged_oracle as oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(native_lib):
    from dynaflow_b200 import ops as _ops

    return _ops


def _check(got, logits, ids, top):
    """Ids are equal. A log probability is (x - m) - log S in fp32: exp of a difference d is within 2^-22 + 2^-23 |d| log2(e)
    of its value, of the terms that count |d| <= 24 (those below e^-24 of the largest sum to less than 2^-17 of 2^18 of them,
    and are as exact as that again): S is within 2^-18, and each fp32 step adds 2^-24 of the numbers it handles."""
    lp, ent, tid, tlp = [t.cpu() for t in got]
    rows = list(range(logits.shape[0]))
    wlp, went, wtid, wtlp = oracle.token_logprobs(logits, ids, top)
    for name, g, w in (("logprob", lp, wlp), ("entropy", ent, went), ("top_logprobs", tlp, wtlp)):
        same = (g.double() == w) | (torch.isnan(g) & torch.isnan(w))
        room = 2.0 ** -18 + 2.0 ** -22 * w.abs()
        bad = ~(same | ((g.double() - w).abs() <= room))
        assert not bad.any(), (name, rows, g[bad][:4], w[bad][:4])
    assert torch.equal(tid, wtid)


def _run(ops, logits, ids, top, id_dtype=torch.int64):
    got = ops.token_logprobs(logits, torch.tensor(ids, dtype=id_dtype, device="cuda"), top)
    torch.cuda.synchronize()
    return got


@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 5, 5), (3, 100, 0), (2, 8191, 7), (1, 8193, 32), (2, 20000, 20), (700, 40, 3), (3, 65537, 5)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_against_64_bits(ops, rows, vocab, top, dtype):
    g = torch.Generator().manual_seed(rows + vocab)
    logits = (torch.randn(rows, vocab, generator=g) * 3).to(dtype)
    ids = torch.randint(0, vocab, (rows,), generator=g).tolist()
    _check(_run(ops, logits.cuda(), ids, top), logits, ids, top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab,ld,shift", [(100, 103, 1), (8200, 8207, 3), (33000, 33001, 5), (50, 64, 0)])
def test_rows_at_any_address(ops, vocab, ld, shift, dtype):
    """Row strides and a first element that no vector load fits."""
    rows = 5
    g = torch.Generator().manual_seed(ld)
    room = torch.full((rows * ld + shift,), 1e4, dtype=dtype, device="cuda")       # what lies around the rows is large
    logits = torch.randn(rows, vocab, generator=g).to(dtype)
    view = room[shift:].view(rows, ld)[:, :vocab]
    view.copy_(logits)
    ids = [0, vocab - 1, 3, 4, 5]
    _check(_run(ops, view, ids, 10, torch.int32), logits, ids, 10)


@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "two values", "rising fp32 ties"])
@pytest.mark.parametrize("top", [1, 20, 32])
def test_orders_that_defeat_a_threshold(ops, kind, top):
    """All logits equal, growing along the row (every chunk brings a new top), runs of ties: the lower index first."""
    vocab = 30000
    i = torch.arange(vocab)
    row = {"equal": torch.full((vocab,), 1.5), "rising": i / 1000, "falling": -i / 1000, "two values": (i % 7 == 3).float(),
           "rising fp32 ties": (i // 100) / 100}[kind].float()
    logits = torch.stack([row, row.flip(0)])
    for dtype in (torch.float32, torch.bfloat16):
        x = logits.to(dtype)
        _check(_run(ops, x.cuda(), [7, 29999], top), x, [7, 29999], top)


def test_zero_and_minus_zero_are_equal(ops):
    x = torch.full((1, 50), -5.0)
    x[0, 10], x[0, 20], x[0, 30] = -0.0, 0.0, -0.0
    _check(_run(ops, x.cuda(), [20], 5), x, [20], 5)


@pytest.mark.parametrize("allowed", [0, 1, 3, 40])
def test_forbidden_tokens(ops, allowed):
    """-inf logits take no part; fewer allowed tokens than asked for, and none at all."""
    vocab, top = 17000, 8
    g = torch.Generator().manual_seed(allowed)
    x = torch.full((2, vocab), -math.inf)
    for r in range(2):
        at = torch.randperm(vocab, generator=g)[:allowed]
        x[r, at] = torch.randn(allowed, generator=g)
    ids = [int(x[r].argmax()) for r in range(2)]
    ids[1] = 5 if allowed < 40 else ids[1]
    for dtype in (torch.float32, torch.bfloat16):
        y = x.to(dtype)
        _check(_run(ops, y.cuda(), ids, top), y, ids, top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masks_of_the_lowest_value(ops, dtype):
    """Forbidden by the type's lowest value instead of -inf; both kinds; a row of nothing but lowest values is uniform."""
    vocab, top = 20000, 12
    low = torch.finfo(dtype).min
    x = torch.full((4, vocab), low, dtype=torch.float64)
    x[0, [5, 19000, 700]] = torch.tensor([1.0, 2.0, 0.5], dtype=torch.float64)
    x[1, 3:] = -math.inf
    x[1, [100, 9000]] = torch.tensor([-3.0, 4.0], dtype=torch.float64)
    x[3, ::2] = -math.inf
    x = x.to(dtype)
    ids = [700, 9000, 123, 1]
    _check(_run(ops, x.cuda(), ids, top), x, ids, top)


def test_a_very_long_row(ops):
    """So long that a row is cut into more slices than a cluster has; the slices' records go through the workspace."""
    vocab = 1_300_000
    x = (torch.randn(1, vocab, generator=torch.Generator().manual_seed(12)) * 3).bfloat16()
    assert ops.token_logprobs_workspace(1, vocab, 20).numel() > 1000
    _check(_run(ops, x.cuda(), [vocab - 1], 20), x, [vocab - 1], 20)


def test_nan_and_infinity_are_not_lost(ops):
    x = torch.randn(4, 9000)
    x[0, 4000] = float("nan")
    x[1, 8999] = math.inf
    x[3] = -math.inf
    x[3, 17] = float("nan")
    for dtype in (torch.float32, torch.bfloat16):
        got = _run(ops, x.to(dtype).cuda(), [1, 2, 3, 4], 2)
        for t in (got[0], got[1]):
            assert torch.isnan(t[[0, 1, 3]]).all() and torch.isfinite(t[2]).all()


@pytest.mark.parametrize("scale", [1e-30, 50.0, 1e30])
def test_flat_and_sharp_rows(ops, scale):
    g = torch.Generator().manual_seed(4)
    x = (torch.randn(2, 12000, generator=g).double() * scale).float()
    ids = [int(x[0].argmax()), 77]
    _check(_run(ops, x.cuda(), ids, 4), x, ids, 4)


def test_ids_outside_the_vocabulary(ops):
    x = torch.randn(4, 60)
    got = _run(ops, x.cuda(), [-1, 60, 2 ** 40, 59], 0)
    assert (got[0][:3] == -math.inf).all() and torch.isfinite(got[0][3])
    assert got[2].shape == (4, 0)


@pytest.mark.parametrize("parts", [1, 2, 5])
def test_shards_give_what_the_whole_row_gives(ops, parts):
    """The vocabulary cut into shards (one launch each, their records joined): same ids, same numbers within the bound."""
    vocab, rows, top = 25000, 3, 20
    g = torch.Generator().manual_seed(parts)
    x = (torch.randn(rows, vocab, generator=g) * 3).bfloat16()
    ids = [0, 12345, vocab - 1]
    d, dids = x.cuda(), torch.tensor(ids, device="cuda")
    cuts = [vocab * i // parts for i in range(parts + 1)]
    records = []
    for a, b in zip(cuts, cuts[1:]):
        ws = ops.token_logprobs_workspace(rows, b - a, top)
        records.append(ops.token_logprobs_shard(d[:, a:b], dids, a, top, ops.token_logprobs_record(rows, top), ws))
    got = ops.token_logprobs_join(torch.cat(records), parts, rows, top)
    torch.cuda.synchronize()
    _check(got, x, ids, top)


def test_same_bits_every_time_and_in_a_graph(ops):
    x = torch.randn(5, 40000, generator=torch.Generator().manual_seed(9)).bfloat16().cuda()
    ids = torch.arange(5, device="cuda")
    want = [t.clone() for t in ops.token_logprobs(x, ids, 20)]
    for _ in range(5):
        for a, b in zip(ops.token_logprobs(x, ids, 20), want):
            assert torch.equal(a, b)
    out, ws = ops.token_logprobs_out(5, 20), ops.token_logprobs_workspace(5, 40000, 20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
            ops.token_logprobs(x, ids, 20, out=out, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    for t in out:
        t.fill_(0)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, want):
        assert torch.equal(a, b)


def test_random_shapes(ops):
    rng = random.Random(11)
    for case in range(12):
        rows, vocab = rng.randint(1, 30), int(math.exp(rng.uniform(0, math.log(30000))))
        top, dtype = rng.randint(0, min(32, vocab)), rng.choice([torch.bfloat16, torch.float32])
        g = torch.Generator().manual_seed(case)
        x = (torch.randn(rows, vocab, generator=g) * rng.choice([0.1, 2.0, 10.0])).to(dtype)
        ids = torch.randint(0, vocab, (rows,), generator=g).tolist()
        _check(_run(ops, x.cuda(), ids, top), x, ids, top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [31, 33, 255, 257, 534, 745, 1024, 1361, 1637, 2047, 2049, 8193, 8200, 17000])
@pytest.mark.parametrize("top", [1, 7, 32])
def test_rows_that_leave_warps_without_logits(ops, vocab, top, dtype):
    # fewer vectors than threads, in the row or in its last slice: the threshold comes from the warps that have logits
    top = min(top, vocab)
    for rows in (3, 300):
        g = torch.Generator().manual_seed(3 * vocab + rows)
        logits = torch.randn(rows, vocab, generator=g).to(dtype)
        logits[:, ::5] = -math.inf
        ids = torch.randint(0, vocab, (rows,), generator=g).tolist()
        got = _run(ops, logits.cuda(), ids, top)
        some = slice(None, None, max(rows // 5, 1))
        _check([t[some] for t in got], logits[some], ids[some], top)
