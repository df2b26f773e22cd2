"""Which parts of a page decoder's prefill DECODER_INT8_ACTIVATIONS moves to
int8 activations, by rows: the projections always, the MoE blocks above 16.

With an output projection of zeros the attention adds exactly nothing to the
residual, so that what is left of a layer is its MoE block: the logits are then
the same bits with and without the flag where that block is weight-only."""
import numpy as np
import pytest

import decoder_oracle as D
import uocr_moe as M
from test_decoder_gpu import _device_layer, _run

pytestmark = pytest.mark.gpu

DIMS = D.DecoderDims(512, 1, 4, 2, 128, 512, 8, 2, 128, 256)


def prefill_logits(torch, cuda, rows, flags, zero_output):
    d = DIMS
    w = D.synth_weights(d, 5, int8=False, norm_sigma=0.1)
    dec = M.Decoder(d.hidden, d.layers, d.heads, d.kv_heads, d.vocab, max_positions=rows + 2, max_prefill=rows,
                    experts=d.experts, top_k=d.top_k, ffn=d.ffn, shared_ffn=d.shared_ffn,
                    weight_format=M.WEIGHT_INT8, flags=flags)
    layer = _device_layer(torch, cuda, w.layers[0])
    if zero_output:
        layer["wo"].zero_()
    f = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(cuda)  # noqa: E731
    head = (f(w.embed), f(w.final_norm), f(w.lm_head))
    dec.set_layer(0, layer, dtype=M.DTYPE_F32)
    dec.set_head(*head, dtype=M.DTYPE_F32)
    torch.cuda.synchronize()
    logits, _, _, _ = _run(torch, cuda, dec, D.synth_prompt(d, 5, rows), d.vocab, 1, torch.cuda.Stream())
    dec.close()
    return logits


@pytest.mark.parametrize("rows", [1, 9, 16, 17, 40])
def test_moe_block_is_int8_above_16_rows(cuda, rows):
    import torch
    plain, flagged = (prefill_logits(torch, cuda, rows, flags, True) for flags in (0, M.DECODER_INT8_ACTIVATIONS))
    assert np.array_equal(plain, flagged) == (rows <= 16)


@pytest.mark.parametrize("rows", [9, 40])
def test_projections_are_int8_at_any_rows(cuda, rows):
    import torch
    plain, flagged = (prefill_logits(torch, cuda, rows, flags, False) for flags in (0, M.DECODER_INT8_ACTIVATIONS))
    assert not np.array_equal(plain, flagged)
