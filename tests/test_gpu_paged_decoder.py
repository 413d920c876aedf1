"""The paged 4-bit cache under the decoder: prompts, decode steps, log probabilities and pages that come and go, together."""
import pytest
import torch

from oracle import paged_oracle as oracle

pytestmark = pytest.mark.gpu

TOL = 2e-2
HD = 128


def _decoder(batch, seq, micro_batches=2, seed=21):
    from dynaflow_b200.decoder import DecoderShape, TensorParallelDecoder, reference_weights

    shape = DecoderShape(hidden=256, intermediate=512, heads=4, kv_heads=2, head_dim=128, layers=2, vocab=512)
    weights = reference_weights(shape, seed=seed)
    return shape, weights, TensorParallelDecoder(shape, max_rows=batch * seq, micro_batches=micro_batches, weights=weights)


def _held(paged, layer, request, length):
    """What the cache holds of a request's first ``length`` tokens: keys and values ``[kv heads, length, 128]``, 64 bits."""
    ps = paged.page_size
    cache, table = paged.layers[layer].cpu(), paged.page_table[request].tolist()
    pages = cache[torch.tensor(table[:-(-length // ps)])]                                # [pages, kv heads, bytes]
    raw = pages.view(len(pages), paged.kv_heads, ps // 16, 2176).transpose(0, 1).reshape(paged.kv_heads, -1, 2176)
    r, c = torch.arange(16).view(16, 1), torch.arange(4).view(1, 4)
    out = []
    for base in (0, 1088):
        b = raw[..., base:base + 1024].unflatten(-1, (16, 4, 16))[:, :, r.expand(16, 4), c ^ ((r >> 1) & 3)].flatten(-2)
        codes = torch.stack([b & 15, b >> 4], -1).flatten(-2).double()
        params = raw[..., base + 1024:base + 1088].contiguous().view(torch.bfloat16).unflatten(-1, (16, 2)).double()
        out.append((params[..., :1] * codes + params[..., 1:]).flatten(1, 2)[:, :length])
    return out


def _rel(got, want):
    return ((got.float() - want.float()).abs().max() / want.float().abs().max()).item()


def test_prompts_then_steps_match_a_contiguous_cache_of_the_same_numbers(native_lib):
    """Prefill into pages, then a decode step: the same step on a contiguous bf16 cache that holds the numbers the pages stand
    for. They differ by the bf16 rounding of those numbers (2^-8) and by the new token's key and value, which the pages hold in
    4 bits: one of L = 101 keys, off by 1/30 of its range, 1e-3 of the result."""
    from dynaflow_b200 import ops
    from dynaflow_b200.decoder import TensorParallelDecoder

    B, S, max_len = 5, 100, 160
    shape, weights, dec = _decoder(B, S)
    ids = torch.randint(0, shape.vocab, (B, S), generator=torch.Generator().manual_seed(3)).cuda()
    dec.init_decode_paged(B, max_len, page_size=32)
    hidden = dec.prefill_paged(ids)
    torch.cuda.synchronize()
    ops.check_status()
    assert torch.isfinite(hidden.float()).all() and dec.paged.page_counts.tolist() == [4] * B
    assert dec.paged.free_count.item() == B * 5 - B * 4
    twin = TensorParallelDecoder(shape, max_rows=B * S, micro_batches=2, weights=weights)
    twin.init_decode(B, max_len, context_len=S + 1, fill_seed=None)
    for layer in range(shape.layers):
        for b in range(B):
            k, v = _held(dec.paged, layer, b, S)
            twin.k_cache[layer, b, :S] = k.transpose(0, 1).reshape(S, -1).bfloat16().cuda()
            twin.v_cache[layer, b, :S] = v.transpose(0, 1).reshape(S, -1).bfloat16().cuda()
    # layer 0's keys are the quantised rotated projections of the normalised embeddings
    x = weights["embed"][ids.cpu()].float()
    x = (x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + shape.eps)).bfloat16().float() * weights["l0.norm1"].float()
    key = (x.bfloat16().double() @ weights["l0.k"].double().T).view(B, S, 2, HD)
    want = torch.stack([oracle.rotate(key[b], torch.arange(S), shape.rope_theta) for b in range(B)])
    k0 = torch.stack([_held(dec.paged, 0, b, S)[0].transpose(0, 1) for b in range(B)])
    step = (want.amax(-1, keepdim=True) - want.amin(-1, keepdim=True)) / 15
    # half a step of the code, and the bf16 roundings of the projection's input, its result and the rotation
    assert ((k0 - want).abs() <= 0.6 * step + want.abs() * 2 ** -6 + want.abs().amax(-1, keepdim=True) * 2 ** -7).all()
    last = torch.randint(0, shape.vocab, (B,), generator=torch.Generator().manual_seed(4)).cuda()
    dec.seq_lens.add_(1)
    got = torch.cat(dec.decode_step(last)).clone()
    want = torch.cat(twin.decode_step(last))
    torch.cuda.synchronize()
    ops.check_status()
    assert _rel(got, want) <= TOL
    # log probabilities of the step's own logits
    top = 4
    lp, entropy, top_ids, top_lp = dec.token_logprobs([got[dec.d_cuts[i]:dec.d_cuts[i + 1]] for i in range(2)], last, top)
    wlp, went, wid, wtlp = oracle.token_logprobs(got, last.tolist(), top)
    assert torch.equal(top_ids.cpu(), wid)
    for g, w in ((lp, wlp), (entropy, went), (top_lp, wtlp)):
        assert ((g.cpu().double() - w).abs() <= 2.0 ** -18 + 2.0 ** -22 * w.abs()).all()


def test_generation_eagerly_and_from_one_graph(native_lib):
    """Greedy generation across page borders, the step captured once and replayed: the same tokens and the same bits as eager
    steps; then one sequence ends, its pages go back, another takes them."""
    from dynaflow_b200 import ops

    B, S, max_len, steps = 4, 30, 64, 17
    shape, _, dec = _decoder(B, S, seed=22)
    ids = torch.randint(0, shape.vocab, (B, S), generator=torch.Generator().manual_seed(5)).cuda()

    def start():
        dec.init_decode_paged(B, max_len, page_size=16, num_pages=14)
        hidden = dec.prefill_paged(ids)
        return ops.gemm_bf16(hidden.view(B, S, -1)[:, -1].contiguous(), dec.lm_head).float().argmax(-1)

    def run(step, token):
        tokens, logits = [token.clone()], []
        for _ in range(steps):
            dec.seq_lens.add_(1)
            lg = step(token)
            token.copy_(dec.token_logprobs(lg, token.clone(), 1)[2][:, 0])
            tokens.append(token.clone())
            logits.append(torch.cat(lg).clone())
        torch.cuda.synchronize()
        ops.check_status()
        return torch.stack(tokens), torch.stack(logits)

    eager_tokens, eager_logits = run(dec.decode_step, start())
    assert dec.paged.page_counts.tolist() == [3] * B           # 47 tokens each, from two pages
    token = start()
    dec.seq_lens.add_(1)                         # (the capture's own eager step needs a row for the new token)
    replay, out = dec.capture_decode(token)
    dec.seq_lens.sub_(1)

    def replayed(_):
        replay()
        return out

    graph_tokens, graph_logits = run(replayed, token)
    assert torch.equal(graph_tokens, eager_tokens) and torch.equal(graph_logits, eager_logits)
    # sequence 0 ends: its pages go back
    free = dec.paged.free_count.item()
    dec.seq_lens[0] = 0
    replay()
    torch.cuda.synchronize()
    ops.check_status()
    assert dec.paged.page_counts[0].item() == 0 and dec.paged.free_count.item() > free
    assert (dec.attn_out[0][0] == 0).all()       # no keys: zeros, and nothing of the ended sequence is written


def test_a_pool_that_is_too_small_is_reported(native_lib):
    from dynaflow_b200 import ops

    B, S = 3, 20
    shape, _, dec = _decoder(B, S, micro_batches=1, seed=23)
    dec.init_decode_paged(B, 64, page_size=16, num_pages=5)      # two pages each would be six
    dec.prefill_paged(torch.zeros(B, S, dtype=torch.int64, device="cuda"))
    with pytest.raises(ops.DeviceStatusError, match="pages missing"):
        ops.check_status()
    with pytest.raises(ValueError, match="prefill_paged"):
        dec.prefill_paged(torch.zeros(B, 65, dtype=torch.int64, device="cuda"))
