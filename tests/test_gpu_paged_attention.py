"""Attention over the paged 4-bit cache against 64-bit attention over the numbers the cache stands for."""
import math
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


class Case:
    """A cache whose requests' pages are scattered, bytes of all ones (NaN parameters) wherever no token was written."""

    def __init__(self, lens, hkv, page, seed, *, spare=1, key_scale=1.0, value_scale=1.0, value_shift=0.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.hkv, self.page = lens, hkv, page
        held = [-(-n // page) for n in lens]
        pages = sum(held) + spare
        order = torch.randperm(pages, generator=g).tolist()
        self.width = max(held + [1])
        self.table = [[-1] * self.width for _ in lens]
        cache = torch.full((pages, hkv, page // 16, 2176), 0xFF, dtype=torch.uint8)
        self.keys, self.values = [], []
        for b, n in enumerate(lens):
            room = -(-n // 16) * 16
            ks, vs = torch.zeros(hkv, n, HD, dtype=torch.float64), torch.zeros(hkv, n, HD, dtype=torch.float64)
            for j in range(held[b]):
                self.table[b][j] = order.pop()
            for h in range(hkv):
                if n == 0:
                    continue
                k = (torch.randn(room, HD, generator=g) * key_scale).bfloat16()
                v = (torch.randn(room, HD, generator=g) * value_scale + value_shift).bfloat16()
                data, kd, vd = oracle.pack_granules(k, v)
                for i in range(room // 16):
                    at = i * 16
                    dst = cache[self.table[b][at // page], h, (at % page) // 16]
                    dst.copy_(data[i])
                    for r in range(max(0, n - at), 16):              # tokens past the end: all ones
                        for base in (0, 1088):
                            dst[base + r * 64:base + r * 64 + 64] = 0xFF
                            dst[base + 1024 + 4 * r:base + 1028 + 4 * r] = 0xFF
                ks[h], vs[h] = kd[:n], vd[:n]
            self.keys.append(ks)
            self.values.append(vs)
        self.cache = cache.view(pages, hkv, page * 136)


def _want(case, q, starts, fresh, group, scale, missing=()):
    """64-bit result of every row, and how far fp32 sums and the two fp16 roundings may take the kernel from it:
    * the result is rounded to bf16: half a step, 2^-8 |o|;
    * a score is a sum of 128 products and 2 terms in fp32, whose terms sum to at most A in magnitude: 2^-23 * 24 * A
      (8 matrix steps of 16, each sum off by at most two truncations), hence every weight by that factor, numerator and denominator;
    * p s_v is rounded to fp16 (2^-11), values reach R = 15 s + |m| in magnitude;
    * n keys are summed 16 at a time: 2^-23 (n / 16 + 40) R; exp2 is within 2^-21."""
    out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b, n in enumerate(case.lens):
        for j in range(fresh[b]):
            row, last = starts[b] + j, n - fresh[b] + j + 1
            for h in range(q.shape[1] // HD):
                kvh = h // group
                cols = slice(h * HD, (h + 1) * HD)
                k, v = case.keys[b][kvh][:max(last, 0)], case.values[b][kvh][:max(last, 0)]
                if missing:
                    keep = torch.tensor([i // case.page not in missing for i in range(k.shape[0])], dtype=torch.bool)
                    k, v = k[keep], v[keep]
                x = q[row, cols].double()
                o = oracle.attend(x[None], k, v, scale)[0]
                out[row, cols] = o
                if k.shape[0]:
                    size = x.abs().sum() * 2 * k.abs().max() * scale + (x.abs() @ k.abs().T).max() * scale     # |s n| <= |k| + |m|
                    reach = 2 * v.abs().max()
                    off = 2 * (2.0 ** -23 * 24 * size + 2.0 ** -21) + 2.0 ** -11 + 2.0 ** -23 * (k.shape[0] / 16 + 40)
                    tol[row, cols] = 2.0 ** -8 * o.abs() + off * reach
    return out, tol


def _run(ops, case, q, group, *, fresh=None, starts=None, max_new=1, scale=None, max_ctas=0, wide=0, page_table=None):
    rows, cols = q.shape
    hq = cols // HD
    room = torch.full((rows, cols + wide), 9.0, dtype=torch.bfloat16, device="cuda")
    room[:, :cols] = q.cuda()
    out_room = torch.full((rows, cols + wide), 7.0, dtype=torch.bfloat16, device="cuda")
    out = out_room[:, :cols]
    ws = ops.attention_paged4_workspace(len(case.lens), hq, case.hkv, max_new)
    ws[640:].fill_(0xFF)                 # all but the counters
    more = dict(row_starts=_i32(starts), new_lens=_i32(fresh), max_new=max_new) if fresh is not None else {}
    args = (room[:, :cols], case.cache.cuda(), _i32(page_table or case.table), _i32(case.lens), out, ws)
    ops.attention_paged4(*args, page_size=case.page, scale=scale, max_ctas=max_ctas, **more)
    first = out.clone()
    out_room.fill_(7.0)
    ops.attention_paged4(*args, page_size=case.page, scale=scale, max_ctas=max_ctas, **more)      # the same bits again
    torch.cuda.synchronize()
    ops.check_status()
    assert torch.equal(out, first)
    assert (out_room[:, cols:] == 7.0).all()
    return out.cpu()


def _check(got, want, tol, served):
    assert torch.isfinite(got[served].float()).all()
    err = (got.double() - want).abs()
    worst = (err[served] / tol[served].clamp(min=1e-300)).max().item() if served.any() else 0.0
    assert (err[served] <= tol[served]).all(), worst
    assert (got[~served] == 7.0).all()


def _decode(ops, lens, hkv, group, page, seed, **kw):
    run = {k: kw.pop(k) for k in ("max_ctas", "wide", "scale") if k in kw}
    case = Case(lens, hkv, page, seed, **kw)
    q = torch.randn(len(lens), hkv * group * HD, generator=torch.Generator().manual_seed(seed + 1)).bfloat16()
    got = _run(ops, case, q, group, **run)
    want, tol = _want(case, q, list(range(len(lens))), [1] * len(lens), group, run.get("scale") or HD ** -0.5)
    _check(got, want, tol, torch.ones(len(lens), dtype=torch.bool))
    return got


@pytest.mark.parametrize("lens,hkv,group,page", [
    ([1], 1, 1, 16), ([16], 1, 4, 16), ([17], 1, 4, 16), ([333], 1, 4, 16), ([5, 64, 65, 1000], 2, 4, 64), ([300, 77], 1, 3, 48),
    ([129, 1, 512, 31], 2, 8, 32), ([200, 333], 2, 12, 128), ([640, 15], 1, 16, 16), ([40, 700], 1, 20, 64), ([2100], 2, 5, 256)])
def test_one_new_token_a_request(ops, lens, hkv, group, page):
    _decode(ops, lens, hkv, group, page, len(lens) + group)


def test_many_short_requests(ops):
    """More requests than warps walk in one go, most of them inside one warp's part."""
    rng = random.Random(5)
    _decode(ops, [rng.randint(1, 40) for _ in range(700)], 2, 4, 16, 51)


def test_requests_without_keys_get_zeros(ops):
    got = _decode(ops, [0, 50, 0, 0, 17, 0], 2, 4, 32, 52)
    assert (got[0] == 0).all() and (got[5] == 0).all()
    assert (_decode(ops, [0], 1, 4, 16, 53) == 0).all()


@pytest.mark.parametrize("max_ctas", [1, 3, 40])
def test_on_few_sms(ops, max_ctas):
    _decode(ops, [900, 1024, 333, 64, 1, 512], 2, 4, 64, 54, max_ctas=max_ctas)


def test_strided_rows_and_another_scale(ops):
    _decode(ops, [90, 411], 2, 4, 32, 55, wide=264, scale=0.25)


@pytest.mark.parametrize("value_scale,value_shift", [(1e-9, 0.0), (1e9, 0.0), (1.0, 100.0)])
def test_size_of_the_values_does_not_matter(ops, value_scale, value_shift):
    _decode(ops, [500, 33], 1, 4, 32, 56, value_scale=value_scale, value_shift=value_shift)


def test_large_scores_move_the_reference(ops):
    """Scores up to a few hundred: the running maximum moves many times, in every order."""
    _decode(ops, [1500, 40], 1, 4, 16, 57, key_scale=20.0)


def test_growing_scores_and_scales(ops):
    """Keys aligned with the query and growing along the cache; values whose scale grows too."""
    n, page = 600, 32
    case = Case([n], 1, page, 58)
    q = torch.randn(1, 4 * HD, generator=torch.Generator().manual_seed(59)).bfloat16()
    ramp = torch.linspace(0.1, 4.0, 608).view(-1, 1)
    g = torch.Generator().manual_seed(60)
    k = (q[0, :HD].float() * ramp).bfloat16()
    v = (torch.randn(608, HD, generator=g) * torch.logspace(-6, 6, 608).view(-1, 1)).bfloat16()
    data, kd, vd = oracle.pack_granules(k, v)
    view = case.cache.view(-1, 1, page // 16, 2176)
    for i in range(38):
        view[case.table[0][i * 16 // page], 0, (i * 16 % page) // 16] = data[i]
    case.keys, case.values = [kd[None, :n]], [vd[None, :n]]
    got = _run(ops, case, q, 4, max_ctas=1)
    want, tol = _want(case, q, [0], [1], 4, HD ** -0.5)
    _check(got, want, tol, torch.ones(1, dtype=torch.bool))


@pytest.mark.parametrize("lens,fresh,hkv,group,page,max_new", [
    ([100], [4], 1, 4, 16, 4), ([100, 3, 65], [2, 3, 1], 2, 4, 32, 4), ([50, 40, 0, 17], [0, 7, 0, 17], 2, 1, 16, 17),
    ([300, 20], [5, 20], 1, 8, 64, 20), ([1, 2, 33], [1, 2, 3], 1, 16, 48, 3)])
@pytest.mark.parametrize("gap", [0, 2])
def test_several_new_tokens_are_causal_among_themselves(ops, lens, fresh, hkv, group, page, max_new, gap):
    case = Case(lens, hkv, page, 61)
    if gap:
        starts = [b * (max_new + gap) for b in range(len(lens) + 1)]       # fixed rows a request, some without a token
    else:
        starts = [sum(fresh[:b]) for b in range(len(lens) + 1)]
    rows = starts[-1] + 2
    q = torch.randn(rows, hkv * group * HD, generator=torch.Generator().manual_seed(62)).bfloat16()
    got = _run(ops, case, q, group, fresh=fresh, starts=starts, max_new=max_new)
    want, tol = _want(case, q, starts, fresh, group, HD ** -0.5)
    served = torch.zeros(rows, dtype=torch.bool)
    for b, n in enumerate(fresh):
        served[starts[b]:starts[b] + n] = True
    _check(got, want, tol, served)


def test_more_new_tokens_than_served(ops):
    """Rows past max_new are left; those served see the keys they would see with all of them there."""
    case = Case([40, 30], 1, 16, 63)
    fresh, starts = [6, 2], [0, 6, 8]
    q = torch.randn(8, 4 * HD, generator=torch.Generator().manual_seed(64)).bfloat16()
    got = _run(ops, case, q, 4, fresh=fresh, starts=starts, max_new=3)
    want, tol = _want(case, q, starts, fresh, 4, HD ** -0.5)
    served = torch.tensor([True] * 3 + [False] * 3 + [True] * 2)
    _check(got, want, tol, served)


def test_a_later_token_with_nan_does_not_reach_an_earlier_row(ops):
    case = Case([20], 1, 16, 65)
    page = case.cache.view(-1, 1, 1, 2176)[case.table[0][1], 0, 0]
    for base in (1024, 1088 + 1024):                                       # token 19: NaN scale and minimum, key and value
        page[base + 3 * 4:base + 4 * 4] = 0xFF
    q = torch.randn(2, 4 * HD, generator=torch.Generator().manual_seed(66)).bfloat16()
    got = _run_nan(ops, case, q)
    want, tol = _want(case, q, [0], [2], 4, HD ** -0.5)
    assert ((got[0].double() - want[0]).abs() <= tol[0]).all()
    assert torch.isnan(got[1].float()).all()                               # the row that sees it has it


def _run_nan(ops, case, q):
    out = torch.zeros(q.shape, dtype=torch.bfloat16, device="cuda")
    ws = ops.attention_paged4_workspace(1, 4, 1, 2)
    ops.attention_paged4(q.cuda(), case.cache.cuda(), _i32(case.table), _i32(case.lens), out, ws, page_size=case.page,
                         row_starts=_i32([0, 2]), new_lens=_i32([2]), max_new=2)
    torch.cuda.synchronize()
    ops.check_status()
    return out.cpu()


@pytest.mark.parametrize("bad", [-1, 10 ** 9, -2 ** 31])
def test_missing_pages_do_not_count(ops, bad):
    case = Case([100, 50], 2, 16, 67)
    table = [list(r) for r in case.table]
    table[0][2] = table[1][2] = bad
    q = torch.randn(2, 8 * HD, generator=torch.Generator().manual_seed(68)).bfloat16()
    got = _run(ops, case, q, 4, page_table=table)
    want, tol = _want(case, q, [0, 1], [1, 1], 4, HD ** -0.5, missing=(2,))
    _check(got, want, tol, torch.ones(2, dtype=torch.bool))


def test_senseless_lengths_and_rows_stay_in_their_buffers(ops):
    """Lengths past the table, negative ones, rows outside q: the table's end limits the first, the rest has no rows."""
    case = Case([64, 64, 64], 1, 16, 69)
    q = torch.randn(3, 4 * HD, generator=torch.Generator().manual_seed(70)).bfloat16().cuda()
    out = torch.full((3, 4 * HD), 7.0, dtype=torch.bfloat16, device="cuda")
    ws = ops.attention_paged4_workspace(3, 4, 1, 2)
    ops.attention_paged4(q, case.cache.cuda(), _i32(case.table), _i32([2 ** 31 - 1, -5, 64]), out, ws, page_size=16,
                         row_starts=_i32([0, 1, 2 ** 31 - 1, 0]), new_lens=_i32([1, 1, -3]), max_new=2)
    torch.cuda.synchronize()
    ops.check_status()
    assert (out[1] == 0).all() and (out[2] == 7.0).all()


def test_long_cache_past_32_bit_offsets(ops):
    """A pool of 4.6 GB whose last pages hold the request, 40000 tokens long."""
    page, hkv, n = 256, 2, 40000
    small = Case([n], hkv, page, 71, spare=0)
    held = len(small.table[0])
    pages = 4600 * 1000 * 1000 // (hkv * page * 136)
    cache = torch.empty(pages, hkv, page * 136, dtype=torch.uint8, device="cuda")
    cache[pages - held:] = small.cache.cuda()
    table = _i32([[p + pages - held for p in small.table[0]]])
    q = torch.randn(1, 8 * HD, generator=torch.Generator().manual_seed(72)).bfloat16()
    out = torch.empty(1, 8 * HD, dtype=torch.bfloat16, device="cuda")
    ops.attention_paged4(q.cuda(), cache, table, _i32([n]), out, ops.attention_paged4_workspace(1, 8, hkv), page_size=page)
    torch.cuda.synchronize()
    ops.check_status()
    want, tol = _want(small, q, [0], [1], 4, HD ** -0.5)
    _check(out.cpu(), want, tol, torch.ones(1, dtype=torch.bool))


def test_random_shapes(ops):
    rng = random.Random(73)
    for case in range(10):
        hkv, group, page = rng.choice([1, 2, 3]), rng.choice([1, 2, 3, 4, 5, 7, 8, 9, 16]), rng.choice([16, 32, 48, 64, 128])
        longest = int(math.exp(rng.uniform(0, math.log(1500))))
        lens = [rng.randint(0, longest) for _ in range(rng.randint(1, 9))]
        _decode(ops, lens, hkv, group, page, 100 + case, max_ctas=rng.choice([0, 0, 7]))


def test_in_a_graph_with_growing_lengths(ops):
    case = Case([90, 31], 1, 16, 74)
    q = torch.randn(2, 4 * HD, generator=torch.Generator().manual_seed(75)).bfloat16()
    dq, cache, table, lens = q.cuda(), case.cache.cuda(), _i32(case.table), _i32([1, 1])
    out = torch.zeros(2, 4 * HD, dtype=torch.bfloat16, device="cuda")
    ws = ops.attention_paged4_workspace(2, 4, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        ops.status_block()
        with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
            ops.attention_paged4(dq, cache, table, lens, out, ws, page_size=16)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in ((1, 1), (16, 17), (90, 31), (7, 0)):
        lens.copy_(_i32([a, b]))
        graph.replay()
        torch.cuda.synchronize()
        ops.check_status()
        part = Case.__new__(Case)
        part.lens, part.page, part.hkv = [a, b], 16, 1
        part.keys, part.values = [k[:, :n] for k, n in zip(case.keys, (a, b))], [v[:, :n] for v, n in zip(case.values, (a, b))]
        want, tol = _want(part, q, [0, 1], [1, 1], 4, HD ** -0.5)
        _check(out.cpu(), want, tol, torch.ones(2, dtype=torch.bool))


def test_two_streams_with_a_workspace_each(ops):
    case = Case([800, 300], 2, 64, 76)
    q = torch.randn(2, 8 * HD, generator=torch.Generator().manual_seed(77)).bfloat16()
    want = _run(ops, case, q, 4)
    dq, cache, table, lens = q.cuda(), case.cache.cuda(), _i32(case.table), _i32(case.lens)
    outs = [torch.zeros(2, 8 * HD, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    wss = [ops.attention_paged4_workspace(2, 8, 2) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, o, w in zip(streams, outs, wss):
            with torch.cuda.stream(s):
                ops.attention_paged4(dq, cache, table, lens, o, w, page_size=64)
    torch.cuda.synchronize()
    ops.check_status()
    assert torch.equal(outs[0].cpu(), want) and torch.equal(outs[1].cpu(), want)
