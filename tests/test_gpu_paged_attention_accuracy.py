"""How near the attention over the paged 4-bit cache comes to the 64-bit result, relative to the result's own size, where
one warp walks a whole row of keys."""
import pytest
import torch

from oracle import paged_oracle as oracle

pytestmark = pytest.mark.gpu

HD, HEADS, PAGE = 128, 16, 64          # sixteen heads on one SM: one for each of its warps


@pytest.fixture(scope="module")
def ops(native_lib):
    from dynaflow_b200 import ops as _ops

    return _ops


def _errors(ops, q, keys, values, group=1):
    """``q [16, 128]`` (a key/value head each; with ``group`` 16 all of one head, in eight heads alike) against the same ``keys,
    values [n, 128]``: for every query the distance to the 64-bit result and its bound, both relative to the result's norm. The
    bound is the sum of
    * the result's rounding to bf16, 2^-8;
    * what the keys' weights are off by: the rounding of p s to fp16 (2^-11), and as derived for every row elsewhere, the score's
      fp32 sum and exp2, 2 (2^-23 24 A + 2^-21), A the sum of the score's terms in magnitude. These errors are independent from
      key to key, at most d each, so that their sum over the keys has a standard deviation of at most d sqrt(sum |p v|^2),
      with the two parts of v, s (n - 7.5) and the middle m + 7.5 s, each on its own; four of them are allowed;
    * where p s is far below the largest one it is no normal fp16 number: 2^-25 of what stands for 2^10 at least, on codes of at
      most 7.5, again independent: four standard deviations of n keys;
    * the matrix unit's fp32 sums: at most two steps of 2^-23 of the largest partial sum for each 16 keys; in a sum there are also
      the codes' means, 7.5, of what the halves of at most 512 keys' granules differ in weight;
    * the fp32 sums of p and of p (m + 7.5 s): a lane adds n / 8 terms, half a step (2^-24) of the largest partial sum each,
      independent: sqrt(n / 8) of them, four standard deviations."""
    n = keys.shape[0]
    data, kd, vd = oracle.pack_granules(keys, values)
    codes, step, low = oracle.quantise(values)
    pages = n // PAGE
    kv = HEADS if group == 1 else 8
    cache = data.view(pages, 1, PAGE // 16, 2176).expand(pages, kv, PAGE // 16, 2176).contiguous().view(pages, kv, PAGE * 136).cuda()
    table = torch.arange(pages, dtype=torch.int32, device="cuda").view(1, pages)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    rows = q.view(1, -1).repeat(1, kv * group // HEADS).cuda()
    out = torch.zeros_like(rows)
    ops.attention_paged4(rows, cache, table, lens, out, ops.attention_paged4_workspace(1, kv * group, kv), page_size=PAGE, max_ctas=1)
    torch.cuda.synchronize()
    ops.check_status()
    got = out.cpu().double().view(-1, HEADS, HD)
    got = got[-1] if group > 1 else got[0]
    scale = HD ** -0.5
    wave, middle = step * (codes - 7.5), low + 7.5 * step
    found = []
    for h in range(HEADS):
        x = q[h].double()
        p = torch.softmax(kd @ x * scale, 0)[:, None]
        o = (p * vd).sum(0)
        size = (x.abs().sum() * 2 * kd.abs().max() + (kd.abs() @ x.abs()).max()) * scale
        each = 2.0 ** -11 + 2 * (2.0 ** -23 * 24 * size + 2.0 ** -21)
        spread = ((p * wave).norm() ** 2 + HD * (p * middle).norm() ** 2).sqrt()
        tilt = (p * step).view(-1, 2, 8).sum(2).diff(dim=1).view(-1, 32).cumsum(1).abs().max() * 2 * 7.5 * HD ** 0.5
        cut = n / 16 * 2.0 ** -22 * ((p * wave).cumsum(0).abs().amax(0).norm() + tilt)
        lane = 4 * (n / 8) ** 0.5 * 2.0 ** -24 * (HD ** 0.5 * (p * middle).cumsum(0).abs().max() + o.norm())
        floor = 4 * n ** 0.5 * 2.0 ** -35 * (p * step).max() * 7.5 * HD ** 0.5
        found.append(((got[h] - o).norm() / o.norm(), 2.0 ** -8 + (4 * each * spread + floor + cut + lane) / o.norm()))
    return torch.tensor(found, dtype=torch.float64)


def _check(found):
    assert torch.isfinite(found).all()
    assert (found[:, 0] <= found[:, 1]).all(), found


def _inputs(n, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(HEADS, HD, generator=g).bfloat16(), torch.randn(n, HD, generator=g), torch.randn(n, HD, generator=g))


@pytest.mark.parametrize("n,shift", [(4096, 0.0), (16384, 0.0), (65536, 0.0), (65536, 3.0)])
def test_long_rows_of_equal_keys(ops, n, shift):
    """Results that shrink with the number of keys: nothing that grows with it may be left over."""
    q, k, v = _inputs(n, n + int(shift))
    _check(_errors(ops, q, k.bfloat16(), (v + shift).bfloat16()))


def test_keys_that_count_in_one_half_of_every_sixteen(ops):
    """The keys in places 8 to 15 of each granule have no weight."""
    n = 65536
    q, k, v = _inputs(n, 7)
    base = torch.randn(HD, generator=torch.Generator().manual_seed(9))
    q = (0.8 * base + 0.6 * q.float()).bfloat16()
    k.view(-1, 16, HD)[:, 8:] -= 4 * base
    _check(_errors(ops, q, k.bfloat16(), v.bfloat16()))


def _towards(q, n, weight):
    """Queries with a direction in common, and the key along it that gets ``weight`` times the weight of ``n`` others of N(0, 1)."""
    base = torch.randn(HD, generator=torch.Generator().manual_seed(9))
    q = (0.8 * base + 0.6 * q.float()).bfloat16()
    score = torch.log(torch.tensor(weight * n * 1.65))             # of N(0, 1) scores the mean weight is e^(1/2)
    return q, base * (score / ((q.float() @ base).mean() * HD ** -0.5))


@pytest.mark.parametrize("group", [1, 16])
@pytest.mark.parametrize("n,weight,size,at", [(16384, 999.0, 0.02, 0.0), (65536, 999.0, 0.02, 0.0), (65536, 99.0, 0.02, 0.4), (16384, 999.0, 0.0, 0.0),
                                              (16384, 999.0, 0.0, 1.0), (16384, 1e9, 0.0, 0.7)])
def test_one_key_with_nearly_all_of_the_weight_and_a_small_value(ops, n, weight, size, at, group):
    """The other keys' weights are small, but what they add up to is much of the result, or all of it."""
    q, k, v = _inputs(n, n + 1)
    i = int(at * (n - 1))
    q, k[i] = _towards(q, n, weight)
    v[i] *= size
    _check(_errors(ops, q, k.bfloat16(), v.bfloat16(), group))


@pytest.mark.parametrize("group", [1, 16])
@pytest.mark.parametrize("size,weight", [(1e5, 1e-11), (1e6, 1e-13), (1e-6, 10.0), (1e20, 1e-30)])
@pytest.mark.parametrize("at", [0.0, 0.6])
def test_one_value_of_another_size_with_another_weight(ops, size, weight, at, group):
    n = 16384
    q, k, v = _inputs(n, 5)
    i = int(at * (n - 1))
    q, k[i] = _towards(q, n, weight / n)
    v[i] *= size
    _check(_errors(ops, q, k.bfloat16(), v.bfloat16(), group))


def test_values_near_the_end_of_the_range(ops):
    q, k, v = _inputs(4096, 6)
    _check(_errors(ops, q, k.bfloat16(), (v * 2.0 ** 120).bfloat16()))
    _check(_errors(ops, q, k.bfloat16(), (v * 2.0 ** -100).bfloat16()))


@pytest.mark.parametrize("n", [1, 40])
def test_one_key_with_all_of_the_weight_gives_its_value(ops, n):
    """The largest weight is 1 and is not rounded: the result is the value's numbers, s n + m, rounded once. (They and the middle
    m + 7.5 s fit into fp32: 8 bits each, 15 / 2 times at most, and the exponents are close.)"""
    q, k, v = _inputs(48, 11)
    k[n - 1] = 40 * q[0].float()
    k, v = k.bfloat16(), v.bfloat16()
    data, _, vd = oracle.pack_granules(k, v)
    out = torch.zeros(1, 4 * HD, dtype=torch.bfloat16, device="cuda")
    ops.attention_paged4(q[:1].repeat(1, 4).cuda(), data.view(1, 1, 48 * 136).cuda(), torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                         torch.tensor([n], dtype=torch.int32, device="cuda"), out, ops.attention_paged4_workspace(1, 4, 1), page_size=48)
    torch.cuda.synchronize()
    ops.check_status()
    assert torch.equal(out.cpu().view(4, HD), vd[n - 1].bfloat16().expand(4, HD))
