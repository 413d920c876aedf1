"""The decoder over the paged cache: sequences that grow past the length it was made for, and a forward pass during a prefill."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _decoder(batch, seq):
    from dynaflow_b200.decoder import DecoderShape, TensorParallelDecoder, reference_weights

    shape = DecoderShape(hidden=256, intermediate=512, heads=4, kv_heads=2, head_dim=128, layers=2, vocab=512)
    return shape, TensorParallelDecoder(shape, max_rows=batch * seq, micro_batches=2, weights=reference_weights(shape, seed=31))


def test_steps_past_max_len_inside_the_last_page(native_lib):
    """28 is no multiple of the page: up to 32 tokens every step is the one that a cache made for 32 takes, bit for bit; the
    33rd token has no page, and that is reported."""
    from dynaflow_b200 import ops

    B, S, page = 2, 27, 16
    runs = []
    for max_len in (28, 32):
        shape, dec = _decoder(B, S)
        ids = torch.randint(0, shape.vocab, (B, S), generator=torch.Generator().manual_seed(6)).cuda()
        dec.init_decode_paged(B, max_len, page_size=page)
        for cache in dec.paged.layers:
            cache.fill_(0xFF)                       # NaN parameters wherever nothing is written
        dec.prefill_paged(ids)
        logits = []
        for step in range(5):
            dec.seq_lens.add_(1)
            logits.append(torch.cat(dec.decode_step(ids[:, step].contiguous())).clone())
        torch.cuda.synchronize()
        ops.check_status()
        runs.append(torch.stack(logits))
        dec.seq_lens.add_(1)
        dec.decode_step(ids[:, 0].contiguous())
        with pytest.raises(ops.DeviceStatusError, match="table row full"):
            ops.check_status()
    assert torch.isfinite(runs[0].float()).all() and torch.equal(runs[0], runs[1])


def test_a_forward_pass_during_a_prefill_leaves_the_pages_alone(native_lib):
    """Whether keys and values go into the pages is the call's, not the object's: a forward pass that another thread starts
    while prompts are brought in does not append."""
    import threading

    from dynaflow_b200 import ops

    B, S = 2, 20
    shape, dec = _decoder(B, S)
    ids = torch.randint(0, shape.vocab, (B, S), generator=torch.Generator().manual_seed(8)).cuda()
    dec.init_decode_paged(B, 32, page_size=16)
    append, calls = dec.paged.append, []

    def counted(*args):
        calls.append(threading.current_thread())
        if len(calls) == 1:
            other = threading.Thread(target=dec.forward, args=(ids,))
            other.start()
            other.join()
        append(*args)

    dec.paged.append = counted
    dec.prefill_paged(ids)
    torch.cuda.synchronize()
    ops.check_status()
    assert len(calls) == shape.layers * 2 and set(calls) == {threading.current_thread()}
