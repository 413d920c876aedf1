"""The paged cache's own calls, one after the other, with places of the batch that are free."""
import pytest
import torch

from oracle import paged_oracle as oracle

pytestmark = pytest.mark.gpu

HD = 128


@pytest.mark.parametrize("per,several", [(0, False), (1, False), (3, False), (0, True), (3, True)])
def test_plan_append_attend_with_free_places(native_lib, per, several):
    """Whatever layout the plan gives the rows, every new token's row is its own request's attention."""
    from dynaflow_b200 import ops
    from dynaflow_b200.paged import PagedKVCache4

    hq, hkv, page = 4, 2, 16
    lens = [[20, 0, 33, 5], [22, 0, 34, 8] if several else [21, 0, 34, 6]]
    fresh = [[20, 0, 33, 5], [2, 0, 1, 3] if several else [1, 0, 1, 1]]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    cache = PagedKVCache4(1, hkv, num_pages=12, page_size=page, max_requests=4, max_len=64, max_rows=64, device="cuda")
    g = torch.Generator().manual_seed(per + 10 * several)
    prompt = torch.randn(sum(fresh[0]), (hq + 2 * hkv) * HD, generator=g).bfloat16().cuda()
    cache.plan(i32(lens[0]), i32(fresh[0]))
    cache.append(0, prompt, hq)
    cache.plan(i32(lens[1]), i32(fresh[1]), rows_per_request=per)
    rows = 4 * per if per else sum(fresh[1]) + 2
    step = torch.randn(rows, (hq + 2 * hkv) * HD, generator=g).bfloat16().cuda()
    cache.append(0, step, hq)
    out = torch.full((rows, hq * HD), 7.0, dtype=torch.bfloat16, device="cuda")
    max_new = 3 if several else 1
    ws = ops.attention_paged4_workspace(4, hq, hkv, max_new)
    cache.attend(0, step[:, :hq * HD], out, ws, i32(lens[1]), **({} if per == 1 else dict(new_lens=i32(fresh[1]), max_new=max_new)))
    torch.cuda.synchronize()
    ops.check_status()
    raw, table, q, got = cache.layers[0].cpu(), cache.page_table.tolist(), step.cpu().double(), out.cpu().double()
    left = set(range(rows))
    at = 0
    for b in range(4):
        for j in range(fresh[1][b]):
            row = b * per + j if per else at + j
            left.discard(row)
            for h in range(hq):
                seen = [oracle.read_token(raw, table[b][i // page] * page + i % page, h // 2, page) for i in range(lens[1][b] - fresh[1][b] + j + 1)]
                want = oracle.attend(q[row, h * HD:(h + 1) * HD][None], torch.stack([k for k, _ in seen]), torch.stack([v for _, v in seen]), HD ** -0.5)[0]
                # half a step of the bf16 result, and the rounding of the weights to fp16 (2^-11) on values below 5
                assert ((got[row, h * HD:(h + 1) * HD] - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -11 * 5).all(), (b, j, h)
        at += fresh[1][b]
    for row in left:             # no token: left as it was, or zeros where every request has a row
        assert (got[row] == (0.0 if per == 1 else 7.0)).all()
