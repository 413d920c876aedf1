"""Plain restatements, in 64 bits and one element or request at a time, of the operators of a decode step over a
paged 4-bit key/value cache: page plan, rotary + quantise, attention, token log probabilities."""
from __future__ import annotations

import math

import torch

GRANULE, GRANULE_BYTES, HALF = 16, 2176, 1088


def page_plan(lens, fresh, table, held, free, count, page_size, rows, rows_per_request=0):
    """Lists in, lists out: ``(table, held, free, count, row_starts, slots, positions)``. ``free`` is the whole list,
    ``count`` how many of its first entries are free pages."""
    table, held, free = [list(r) for r in table], list(held), list(free)
    B = len(lens)
    need = [-(-n // page_size) for n in lens]
    need = [h if n > len(table[0]) else n for n, h in zip(need, held)]
    leaving = [(b, j) for b in range(B) for j in range(need[b], held[b])]
    for k, (b, j) in enumerate(reversed(leaving)):
        free[count + k] = table[b][j]
        table[b][j] = -1
    count += len(leaving)
    missing = [(b, j) for b in range(B) for j in range(held[b], need[b])]
    enough = len(missing) <= count
    if enough:
        for b, j in missing:
            count -= 1
            table[b][j] = free[count]
    held = [need[b] if need[b] <= held[b] or enough else held[b] for b in range(B)]
    starts, slots, positions = [0], [-1] * rows, [0] * rows
    for b in range(B):
        starts.append(starts[-1] + (rows_per_request or fresh[b]))
        for i in range(min(fresh[b], rows_per_request) if rows_per_request else fresh[b]):
            row, pos = starts[b] + i, lens[b] - fresh[b] + i
            if row >= rows:
                break
            positions[row] = pos
            if pos // page_size < held[b]:
                slots[row] = table[b][pos // page_size] * page_size + pos % page_size
    return table, held, free, count, starts, slots, positions


def rotate(x: torch.Tensor, positions: torch.Tensor, theta: float) -> torch.Tensor:
    """``x [rows, heads, 128]`` (any dtype) -> rotated, 64 bits, not rounded."""
    freq = theta ** (-torch.arange(64, dtype=torch.float64) / 64)
    a = positions.double().view(-1, 1, 1) * freq
    u, v = x.double()[..., :64], x.double()[..., 64:]
    return torch.cat([u * a.cos() - v * a.sin(), v * a.cos() + u * a.sin()], -1)


def quantise(x: torch.Tensor):
    """Rows ``[..., 128]`` of bf16 values -> codes (int64), scale and minimum (64 bits; both bf16 values)."""
    x = x.double()
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((high - low) / 15).bfloat16().double()
    codes = torch.where(scale > 0, ((x - low) / scale.clamp(min=1e-300)).round().clamp(0, 15), torch.zeros_like(x))
    return codes.long(), scale, low


def read_token(cache: torch.Tensor, slot: int, head: int, page_size: int):
    """Key and value (64 bits) that the bytes of one token of a cache ``[pages, kv_heads, page_size * 136]`` stand for."""
    page, at = divmod(slot, page_size)
    granule, r = divmod(at, GRANULE)
    raw = cache[page, head, granule * GRANULE_BYTES:(granule + 1) * GRANULE_BYTES]
    out = []
    for base in (0, HALF):
        value = torch.empty(128, dtype=torch.float64)
        scale, low = raw[base + 1024 + r * 4:base + 1024 + r * 4 + 4].clone().view(torch.bfloat16).double().tolist()
        for d in range(128):
            byte = d // 2
            place = (byte // 16) ^ ((r >> 1) & 3)
            b = int(raw[base + r * 64 + place * 16 + byte % 16])
            value[d] = scale * (b & 15 if d % 2 == 0 else b >> 4) + low
        out.append(value)
    return out


def write_tokens(cache: torch.Tensor, slots, head: int, page_size: int, keys: torch.Tensor, values: torch.Tensor) -> None:
    """Quantises ``keys, values [n, 128]`` (bf16 values) into the slots of one head."""
    for base, x in ((0, keys), (HALF, values)):
        codes, scale, low = quantise(x)
        packed = (codes[:, 0::2] | (codes[:, 1::2] << 4)).to(torch.uint8)
        params = torch.cat([scale, low], 1).bfloat16().view(torch.uint8)
        for i, slot in enumerate(slots):
            page, at = divmod(int(slot), page_size)
            granule, r = divmod(at, GRANULE)
            raw = cache[page, head]
            o = granule * GRANULE_BYTES + base
            for c in range(4):
                place = c ^ ((r >> 1) & 3)
                raw[o + r * 64 + place * 16:o + r * 64 + place * 16 + 16] = packed[i, c * 16:c * 16 + 16]
            raw[o + 1024 + r * 4:o + 1024 + r * 4 + 4] = params[i]


def attend(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, scale: float) -> torch.Tensor:
    """``q [heads, 128]`` against ``keys, values [n, 128]``, 64 bits; no keys: zeros."""
    if keys.shape[0] == 0:
        return torch.zeros(q.shape, dtype=torch.float64)
    return torch.softmax(q.double() @ keys.double().T * scale, -1) @ values.double()


def token_logprobs(logits: torch.Tensor, ids, top_k: int):
    """``(logprob, entropy, top_ids, top_logprobs)`` of rows of logits, 64 bits; of equal logits the lower index first. A row
    without a finite logit has no distribution: log probabilities -inf, entropy 0."""
    lp, ent, tid, tlp = [], [], [], []
    for row, i in zip(logits.double().cpu(), ids):
        order = sorted(range(row.numel()), key=lambda j: (-row[j].item(), j))[:top_k] if top_k else []
        if (row == -math.inf).all():
            logp, h = torch.full_like(row, -math.inf), torch.tensor(0.0, dtype=torch.float64)
        else:
            logp = torch.log_softmax(row, -1)
            p = logp.exp()
            h = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum()
        lp.append(logp[i] if 0 <= i < row.numel() else torch.tensor(-math.inf, dtype=torch.float64))
        ent.append(h)
        tid.append(torch.tensor(order, dtype=torch.int32))
        tlp.append(logp[torch.tensor(order, dtype=torch.long)] if order else torch.zeros(0, dtype=torch.float64))
    return torch.stack(lp), torch.stack(ent), torch.stack(tid), torch.stack(tlp)


def pack_granules(keys: torch.Tensor, values: torch.Tensor):
    """``keys, values [16 n, 128]`` (bf16 values) -> the bytes ``uint8 [n, 2176]`` and the numbers (64 bits) they stand for."""
    halves, stands = [], []
    for x in (keys, values):
        codes, scale, low = quantise(x)
        b = (codes[:, 0::2] | (codes[:, 1::2] << 4)).to(torch.uint8).view(-1, GRANULE, 4, 16)
        placed = torch.empty_like(b)
        for r in range(GRANULE):
            for c in range(4):
                placed[:, r, c ^ ((r >> 1) & 3)] = b[:, r, c]
        params = torch.cat([scale, low], 1).bfloat16().view(torch.uint8).view(-1, GRANULE * 4)
        halves.append(torch.cat([placed.flatten(1), params], 1))
        stands.append(scale * codes + low)
    return torch.cat(halves, 1), stands[0], stands[1]
