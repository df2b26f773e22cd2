"""Beam search on the page decoder (uocr_decoder_beam_search): the operators for
sequences that share a page, run together.

The device's hypotheses are scored anew by the CPU restatement of the decoder
(oracle/decoder_oracle.py), token after token. Its logits agree with the device's
within max_rel <= 2e-2 (bf16) and 5e-2 (int8) of the largest logit, the decoder's
own bars; a log-probability moves by at most twice a logit's change, so a score
of n tokens by 2 n tol max|logit|."""
import copy

import numpy as np
import pytest

import decoder_oracle as D
import uocr_moe as M
from test_decoder_gpu import TOL, _build

pytestmark = pytest.mark.gpu

# (hidden, layers, heads, kv_heads, vocab, experts, top_k, ffn, shared, prefill rows, decode steps)
SHAPES = [(512, 2, 4, 1, 1024, 8, 2, 128, 256, 20, 9), (1024, 2, 8, 4, 777, 16, 4, 128, 128, 17, 6)]


def _search(torch, dec, beams, steps, eos=-1, stream=None):
    tokens = torch.full((beams, steps), -7, dtype=torch.int32, device="cuda")
    lengths = torch.full((beams,), -7, dtype=torch.int32, device="cuda")
    scores = torch.full((beams,), 9.0, device="cuda")
    torch.cuda.synchronize()
    dec.beam_search(beams, steps, tokens, scores, lengths, eos=eos, stream=stream)
    dec.check(stream=stream)
    torch.cuda.synchronize()
    return tokens.cpu().numpy(), scores.cpu().numpy(), lengths.cpu().numpy()


def _log_softmax(z):
    z = z.astype(np.float64)
    return z - z.max() - np.log(np.exp(z - z.max()).sum())


class _Scored:
    """Log-probabilities of token sequences behind a prompt, by the oracle; remembers what it has computed."""

    def __init__(self, dims, weights, prompt):
        first = D.DecoderOracle(dims, weights)
        self.seen = {(): (first, first.prefill(prompt))}
        self.largest = 0.0

    def logits(self, prefix):
        if prefix not in self.seen:
            ora = copy.copy(self.state(prefix[:-1]))
            ora.k_cache, ora.v_cache = list(ora.k_cache), list(ora.v_cache)  # a step makes new arrays
            self.seen[prefix] = (ora, ora.step(prefix[-1]))
        self.largest = max(self.largest, float(np.abs(self.seen[prefix][1]).max()))
        return self.seen[prefix][1]

    def state(self, prefix):
        self.logits(prefix)
        return self.seen[prefix][0]

    def score(self, tokens):
        return sum(_log_softmax(self.logits(tuple(tokens[:i])))[t] for i, t in enumerate(tokens))

    def search(self, beams, steps):
        """Beam search on the oracle's logits: [(score, tokens)], best first."""
        alive = [(0.0, ())]
        for _ in range(steps):
            cand = []
            for score, tokens in alive:
                lp = score + _log_softmax(self.logits(tokens))
                cand += [(lp[t], tokens + (int(t),)) for t in np.argsort(-lp)[:beams]]
            alive = sorted(cand, key=lambda c: -c[0])[:beams]
        return alive


@pytest.mark.parametrize("fmt,flags", [(M.WEIGHT_BF16, 0), (M.WEIGHT_INT8, 0),
                                       (M.WEIGHT_INT8, M.DECODER_INT8_ACTIVATIONS)])
@pytest.mark.parametrize("rows", [2, 17])
@pytest.mark.parametrize("shape", SHAPES)
def test_beam_search_against_the_oracle(cuda, shape, rows, fmt, flags):
    import torch
    dims, dec, weights = _build(torch, cuda, shape, fmt, flags=flags)
    steps, beams = shape[-1], 5
    prompt = D.synth_prompt(dims, 5, rows)
    dec.prefill(torch.from_numpy(prompt).to(cuda))
    tokens, scores, lengths = _search(torch, dec, beams, steps)
    ora = _Scored(dims, weights, prompt)
    want = [ora.score(t) for t in tokens.tolist()]
    tol = 2 * steps * TOL[fmt] * ora.largest
    print(f"beam search {shape} fmt {fmt}: scores {scores} against {np.array(want)}, tolerance {tol:.3f}")
    assert np.abs(scores - want).max() <= tol
    assert (np.diff(scores) <= 0).all() and (lengths == steps).all()
    assert len({tuple(t) for t in tokens.tolist()}) == beams
    # No search on logits this close finds less than the oracle's by more than the two errors.
    best = ora.search(beams, steps)
    assert scores[0] >= best[0][0] - 2 * tol
    dec.close()


def test_beam_search_keeps_the_sequence_and_repeats_itself(cuda):
    import torch
    shape = SHAPES[0]
    dims, dec, _ = _build(torch, cuda, shape, M.WEIGHT_BF16)
    x = torch.from_numpy(D.synth_prompt(dims, 5, 12)).to(cuda)
    toks = [torch.empty(6, dtype=torch.int32, device=cuda) for _ in range(2)]
    side = torch.cuda.Stream()
    dec.prefill(x)
    dec.decode(6, toks[0])
    dec.prefill(x)
    torch.cuda.synchronize()
    first = _search(torch, dec, 4, 7)
    again = _search(torch, dec, 4, 7, stream=side)
    assert all(np.array_equal(a, b) for a, b in zip(first, again))
    dec.decode(3, toks[1])
    after = _search(torch, dec, 3, 4)  # behind decoded tokens
    dec.decode(3, toks[1][3:])
    assert torch.equal(toks[0], toks[1])
    # One beam is the greedy sequence; the tokens of the search behind three decoded ones begin where they ended.
    greedy, score, _ = _search(torch, dec, 1, 1)
    dec.prefill(x)
    one, _, _ = _search(torch, dec, 1, 7)
    token = torch.empty(1, dtype=torch.int32, device=cuda)
    dec.prefill(x, token=token)
    assert one[0, 0] == token.item() and score[0] <= 0 and after[0].shape == (3, 4) and greedy.shape == (1, 1)
    dec.close()


def test_beam_search_ends_beams(cuda):
    import torch
    shape = SHAPES[0]
    dims, dec, weights = _build(torch, cuda, shape, M.WEIGHT_BF16)
    prompt = D.synth_prompt(dims, 5, 6)
    dec.prefill(torch.from_numpy(prompt).to(cuda))
    free, _, _ = _search(torch, dec, 6, 8)
    eos = int(free[0, 2])
    tokens, scores, lengths = _search(torch, dec, 6, 8, eos=eos)
    ora = _Scored(dims, weights, prompt)
    ended = 0
    for t, s, n in zip(tokens.tolist(), scores, lengths):
        ended += n < 8
        assert (n == 8 or t[n - 1] == eos) and eos not in t[:n - 1] and all(v == eos for v in t[n:])
        assert abs(ora.score(t[:n]) - s) <= 2 * 8 * TOL[M.WEIGHT_BF16] * ora.largest
    assert ended > 0 and (np.diff(scores) <= 0).all()
    dec.close()


def test_beam_search_refusals(cuda):
    import torch
    shape = (512, 1, 4, 1, 256, 8, 2, 128, 256, 20, 2)
    dims, dec, _ = _build(torch, cuda, shape, M.WEIGHT_BF16)  # 25 positions

    def refused(beams, steps, **kw):
        with pytest.raises(M.UocrError) as e:
            _search(torch, dec, beams, steps, **kw)
        assert e.value.code == 1
        return str(e.value)
    assert "prefill" in refused(2, 2)
    dec.prefill(torch.from_numpy(D.synth_prompt(dims, 5, 20)).to(cuda))
    assert "beams" in refused(17, 2) and "max_positions" in refused(2, 6) and "eos" in refused(2, 2, eos=256)
    assert "beams" in refused(0, 2) and "steps" in refused(2, 26)
    assert "eos" in refused(2, 2, eos=-2)
    need = torch.empty(1 << 20, dtype=torch.uint8, device=cuda)
    out = torch.empty(8, dtype=torch.int32, device=cuda)
    import ctypes
    base = (need.data_ptr() + 255) // 256 * 256
    for workspace, size in ((None, 1 << 19), (base, 100), (base + 16, 1 << 19)):
        args = M.BeamSearchArgs(2, 2, -1, 0, out.data_ptr(), out.data_ptr(), None, workspace, size)
        assert M.lib().uocr_decoder_beam_search(dec.h, ctypes.byref(args), None) == 1
    _search(torch, dec, 16, 5)
    with pytest.raises(ValueError):
        dec.beam_search(2, 2, torch.empty(2, 2, dtype=torch.int64, device=cuda), torch.empty(2, device=cuda))
    dec.close()


@pytest.mark.parametrize("beams", [3, 8])
def test_a_captured_search_repeats_itself(cuda, beams):
    """Its replays continue the sequence that it was captured with, whatever else was searched between them."""
    import torch
    dims, dec, _ = _build(torch, cuda, SHAPES[0], M.WEIGHT_BF16)
    dec.prefill(torch.from_numpy(D.synth_prompt(dims, 5, 12)).to(cuda))
    want = _search(torch, dec, beams, 5)
    tokens = torch.zeros(beams, 5, dtype=torch.int32, device="cuda")
    scores = torch.zeros(beams, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dec.beam_search(beams, 5, tokens, scores)
    for _ in range(2):
        tokens.zero_()
        graph.replay()
        dec.check()
        assert np.array_equal(tokens.cpu().numpy(), want[0]) and np.array_equal(scores.cpu().numpy(), want[1])
        _search(torch, dec, 2, 3)
    del graph
    dec.close()


@pytest.mark.parametrize("fmt", [M.WEIGHT_BF16, M.WEIGHT_INT8])
def test_a_search_behind_decoded_tokens_continues_them(cuda, fmt):
    """Its scores are those of its tokens behind the prompt and the decoded tokens, and no worse than the oracle's best."""
    import torch
    shape = SHAPES[0]
    dims, dec, weights = _build(torch, cuda, shape, fmt)
    prompt = D.synth_prompt(dims, 5, 12)
    first, toks = (torch.empty(n, dtype=torch.int32, device=cuda) for n in (1, 3))
    dec.prefill(torch.from_numpy(prompt).to(cuda), token=first)
    dec.decode(3, toks)
    torch.cuda.synchronize()
    consumed = (first.item(), *toks[:2].tolist())  # the third is chosen, not yet part of the sequence
    tokens, scores, _ = _search(torch, dec, 4, 5)
    ora = _Scored(dims, weights, prompt)

    def score(t):
        return sum(_log_softmax(ora.logits(consumed + tuple(t[:i])))[v] for i, v in enumerate(t))
    want = [score(t) for t in tokens.tolist()]
    tol = 2 * 5 * TOL[fmt] * ora.largest
    # A search elsewhere (one decoded token less, or none) would have other scores: the test can tell.
    elsewhere = [abs(sum(_log_softmax(ora.logits(consumed[:n] + tuple(t[:i])))[v] for i, v in enumerate(t)) - w)
                 for t, w in zip(tokens.tolist(), want) for n in (0, 2)]
    print(f"search behind decoded tokens, fmt {fmt}: {np.abs(scores - want).max():.4f} off, tolerance {tol:.3f}, "
          f"elsewhere {min(elsewhere):.3f} to {max(elsewhere):.3f} off")
    assert np.abs(scores - want).max() <= tol and max(elsewhere) > 2 * tol
    alive = [(0.0, ())]
    for _ in range(5):
        cand = [(s + lp[t], h + (int(t),)) for s, h in alive
                for lp in [_log_softmax(ora.logits(consumed + h))] for t in np.argsort(-lp)[:4]]
        alive = sorted(cand, key=lambda c: -c[0])[:4]
    assert scores[0] >= alive[0][0] - 2 * tol
    dec.close()


@pytest.mark.parametrize("decoded", [0, 3])
def test_one_beam_is_the_greedy_sequence(cuda, decoded):
    """Token by token, up to one that the oracle's logits cannot tell from the other's within both errors."""
    import torch
    shape = SHAPES[0]
    dims, dec, weights = _build(torch, cuda, shape, M.WEIGHT_BF16)
    prompt = D.synth_prompt(dims, 5, 12)
    x = torch.from_numpy(prompt).to(cuda)
    first, before, greedy = (torch.empty(n, dtype=torch.int32, device=cuda) for n in (1, 3, 8))
    dec.prefill(x, token=first)
    if decoded:
        dec.decode(decoded, before)
    one, _, _ = _search(torch, dec, 1, 7)
    dec.decode(7, greedy)
    torch.cuda.synchronize()
    start = (first.item(), *before.tolist())[:decoded]
    # The greedy sequence's next token is the one chosen last; decode() says those after it.
    chosen = before[-1].item() if decoded else first.item()
    sequence = [chosen, *greedy.tolist()]
    ora = _Scored(dims, weights, prompt)
    for i, (a, b) in enumerate(zip(one[0].tolist(), sequence)):
        if a != b:
            z = ora.logits(start + tuple(sequence[:i]))
            assert abs(z[a] - z[b]) <= 2 * TOL[M.WEIGHT_BF16] * np.abs(z).max(), (i, a, b)
            break
    assert one[0, 0] == chosen
    dec.close()


@pytest.mark.parametrize("beams", [3, 8])
@pytest.mark.parametrize("rows", [1100, 2500])
def test_a_search_behind_a_long_page(cuda, rows, beams):
    """A prefix that many blocks share, by the attention kernels for few and for many rows."""
    import torch
    shape = (512, 2, 4, 1, 1024, 8, 2, 128, 256, rows, 5)
    dims, dec, weights = _build(torch, cuda, shape, M.WEIGHT_BF16)
    prompt = D.synth_prompt(dims, 5, rows)
    dec.prefill(torch.from_numpy(prompt).to(cuda))
    tokens, scores, lengths = _search(torch, dec, beams, 5)
    ora = _Scored(dims, weights, prompt)
    want = [ora.score(t) for t in tokens.tolist()]
    tol = 2 * 5 * TOL[M.WEIGHT_BF16] * ora.largest
    print(f"search behind {rows} rows, {beams} beams: {np.abs(scores - want).max():.4f} off, tolerance {tol:.3f}")
    assert np.abs(scores - want).max() <= tol and (lengths == 5).all() and (np.diff(scores) <= 0).all()
    assert scores[0] >= ora.search(beams, 5)[0][0] - 2 * tol
    dec.close()
