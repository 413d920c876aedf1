"""The buffers of the paged 4-bit cache, on the host."""
import os

import pytest
import torch

from conftest import ROOT
from dynaflow_b200 import ops
from dynaflow_b200.paged import PagedKVCache4


@pytest.mark.parametrize("max_len,page", [(100, 64), (128, 64), (1, 16), (17, 16), (300, 48)])
def test_every_position_that_can_have_a_slot_has_its_angles(max_len, page):
    """A request may grow to the end of its last page."""
    cache = PagedKVCache4(1, 1, num_pages=8, page_size=page, max_requests=1, max_len=max_len, max_rows=4, rope_theta=500.0, device="cpu")
    room = cache.page_table.shape[1] * page
    assert room >= max_len and cache.angles.shape == (room, 128)
    assert (cache.angles == ops.rope_angles(room, 500.0, "cpu")).all()


@pytest.mark.parametrize("several", [False, True])
def test_attend_finds_the_rows_where_the_plan_put_them(monkeypatch, several):
    """One row a request, or the plan's row starts of these requests with their token counts."""
    calls = []
    monkeypatch.setattr(ops, "attention_paged4", lambda *a, **kw: calls.append((a, kw)))
    cache = PagedKVCache4(2, 1, num_pages=8, page_size=16, max_requests=4, max_len=32, max_rows=16, device="cpu")
    cache.row_starts.copy_(torch.tensor([0, 3, 3, 4, 9]))
    lens, fresh = (torch.tensor(x, dtype=torch.int32) for x in ([5, 0, 7, 9], [3, 0, 1, 5]))
    q = torch.zeros(16, 128)
    for first, n in ((0, 4), (2, 2), (1, 1)):
        more = dict(new_lens=fresh[first:first + n], max_new=5) if several else {}
        cache.attend(1, q, q, None, lens[first:first + n], first, **more)
        (got_q, layer, table, got_lens, *_), kw = calls.pop()
        assert got_q is q and layer is cache.layers[1] and torch.equal(table, cache.page_table[first:first + n]) and len(got_lens) == n
        if several:
            assert torch.equal(kw["row_starts"], cache.row_starts[first:first + n + 1]) and kw["new_lens"] is more["new_lens"] and kw["max_new"] == 5
        else:
            assert kw["row_starts"] is None and kw["new_lens"] is None and kw["max_new"] == 1


def _documented_calls():
    """The lines of the example of the paged cache, up to the log probabilities."""
    text = open(os.path.join(ROOT, "INTEGRATION.md")).read()
    lines = text[text.index("cache = PagedKVCache4("):].split("```")[0].splitlines()
    return [line.split("#")[0].strip() for line in lines[1:] if line.startswith(("cache.", "ws"))]


def test_the_documented_sequence_pairs_every_row_with_its_request(monkeypatch):
    """The calls of the example, run with places of the batch that are free: an attention that is not told where a request's
    rows are comes after a plan that gives every request one."""
    layout = {}

    def plan(*args, rows_per_request=0, **kw):
        layout["per"] = rows_per_request

    def attention(q, *args, row_starts=None, new_lens=None, **kw):
        assert new_lens is not None and row_starts is not None or layout["per"] == 1
        layout["attentions"] = layout.get("attentions", 0) + 1

    monkeypatch.setattr(ops, "page_plan", plan)
    monkeypatch.setattr(ops, "rope_append_paged4", lambda *a, **kw: None)
    monkeypatch.setattr(ops, "attention_paged4", attention)
    monkeypatch.setattr(ops, "attention_paged4_workspace", lambda *a, **kw: None)
    cache = PagedKVCache4(1, 1, num_pages=8, page_size=64, max_requests=4, max_len=64, max_rows=16, device="cpu")
    names = dict(cache=cache, ops=ops, layer=0, q_heads=4, kv_heads=1, q_cols=512, qkv=torch.zeros(4, 768), q=torch.zeros(4, 512), out=None,
                 seq_lens=torch.zeros(4, dtype=torch.int32), new_lens=torch.zeros(4, dtype=torch.int32))
    for line in _documented_calls():
        exec(line, names)
    assert layout["attentions"] >= 2
