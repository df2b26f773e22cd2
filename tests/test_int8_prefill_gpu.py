"""int8 activations on the prefill path: the MoE plan
(PLAN_INT8_ACTIVATIONS) and the page decoder (DECODER_INT8_ACTIVATIONS).

Two bars for a layer. Against the oracle on the dequantised weights, the int8
bar of 5e-2 (max_rel): a row's int8 step is 1/127 of its largest value, about
4 / 127 of its rms, so each of the two quantisations adds 4 / (127 sqrt(12)) =
0.9 % of noise to a product. Against a 64-bit restatement with the same
roundings, 1e-2: what differs is an activation whose bf16 or int8 rounding goes
the other way because of an ulp in front of it, some 1e-4 of them; one step of
one of F activations moves an output by at most 3 * 4 / 127 / sqrt(F) of its rms
(a weight of 3 sigma), 0.8 % at F = 128, and the largest output is over 2 rms."""
import numpy as np
import pytest

import decoder_oracle as D
import oracle as O
import uocr_moe as M
from conftest import max_rel
from test_decode_gpu import INT8_TOL, _tiny_layer, _upload, check_ids, run_plan, to_np
from test_decoder_gpu import _device_layer, _run

pytestmark = pytest.mark.gpu


def quantized(x):
    """Rows in int8 values with uocr_quantize_tokens' scales, as float64 (q * s)."""
    x = np.asarray(x, np.float32)
    peak = np.abs(x).max(axis=1, keepdims=True)
    s = np.where(peak > 0, peak * (np.float32(1) / np.float32(127)), np.float32(1)).astype(np.float32)
    return np.rint(x / s).astype(np.float64) * s


def dequantized(w):
    q, s = O.quantize_q8(w)
    return O.dequantize_q8(q, s).astype(np.float64)


def swiglu(g, u):
    return O.round_bf16((g / (1.0 + np.exp(-g)) * u).astype(np.float32)).reshape(g.shape)


def restated(w, x, want: O.MoeResult):
    """The layer with int8 weights and activations in 64 bits, given the routing."""
    E, F, H = w.router.shape[0], w.gate.shape[0] // w.router.shape[0], x.shape[1]
    gate, up, down = (dequantized(m) for m in (w.gate, w.up, w.down))
    xq = quantized(x)
    y = np.zeros(x.shape)
    for e in range(E):
        t, j = np.nonzero(want.ids == e)
        if t.size == 0:
            continue
        f = slice(e * F, (e + 1) * F)
        a = quantized(swiglu(xq[t] @ gate[f].T, xq[t] @ up[f].T))
        y[t] += want.weights[t, j][:, None] * (a @ down[e * H:(e + 1) * H].T)
    if w.shared_gate.size:
        a = quantized(swiglu(xq @ dequantized(w.shared_gate).T, xq @ dequantized(w.shared_up).T))
        y += a @ dequantized(w.shared_down).T
    return y


@pytest.mark.parametrize("T,H,E,K,F,S", [(40, 256, 16, 4, 128, 128), (300, 512, 64, 6, 256, 256),
                                         (129, 256, 8, 2, 128, 0), (17, 256, 128, 8, 128, 128),
                                         (700, 512, 4, 1, 384, 128)])
def test_plan_prefill(cuda, T, H, E, K, F, S):
    import torch
    rng = np.random.default_rng(T * 3 + E)
    w = _tiny_layer(rng, H, E, F, S)
    x = rng.standard_normal((T, H)).astype(np.float32)
    plan = M.Plan(M.Dims(H, E, K, F, S), max_rows=max(T, 32), weight_format=M.WEIGHT_INT8,
                  flags=M.PLAN_INT8_ACTIVATIONS)
    plain = M.Plan(M.Dims(H, E, K, F, S), max_rows=max(T, 32), weight_format=M.WEIGHT_INT8)
    assert plan.bytes()[1] < plain.bytes()[1]  # no expanded weights
    _upload(plan, w, torch, cuda)
    xd = torch.from_numpy(x).to(cuda)
    y, ids, wts = run_plan(plan, 0, xd, K, torch)
    deq = {n: (dequantized(getattr(w, n)).astype(np.float32) if getattr(w, n).size else getattr(w, n))
           for n in ("gate", "up", "down", "shared_gate", "shared_up", "shared_down")}
    want = O.moe_forward(O.MoeWeights(w.router, *deq.values()), x, K, renormalize=True)
    check_ids(ids, want)
    assert max_rel(y, want.y) <= INT8_TOL
    got = O.MoeResult(**{**want.__dict__, "ids": ids, "weights": wts})
    assert max_rel(y, restated(w, x, got)) <= 1e-2
    again, _, _ = run_plan(plan, 0, xd, K, torch)
    assert np.array_equal(y, again)
    # up to 16 rows are weight-only, with and without the flag
    _upload(plain, w, torch, cuda)
    a, _, _ = run_plan(plan, 0, xd[:16].contiguous(), K, torch)
    b, _, _ = run_plan(plain, 0, xd[:16].contiguous(), K, torch)
    assert np.array_equal(a, b)


def test_plan_stack_replays_as_a_graph(cuda):
    import torch
    rng = np.random.default_rng(3)
    H, E, K, F, S, T, L = 256, 16, 4, 128, 128, 90, 3
    plan = M.Plan(M.Dims(H, E, K, F, S, L), max_rows=T, weight_format=M.WEIGHT_INT8,
                  flags=M.PLAN_INT8_ACTIVATIONS | M.PLAN_PRE_NORM)
    for i in range(L):
        _upload(plan, _tiny_layer(rng, H, E, F, S), torch, cuda, layer=i)
    x = torch.from_numpy(rng.standard_normal((T, H)).astype(np.float32)).to(cuda)
    plain = x.clone()
    for i in range(L):  # layer by layer, h <- h + MoE(RMSNorm(h))
        y = torch.empty_like(plain)
        plan.forward(i, plain, y)
        plain = plain + y
    side = torch.cuda.Stream()
    h = torch.empty_like(x)
    for _ in range(3):  # captured, then replayed
        h.copy_(x)
        side.wait_stream(torch.cuda.current_stream())
        plan.forward_stack(h, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        plan.check(stream=side)
        # the stack adds its residual in the combine, one fp32 rounding earlier
        assert max_rel(to_np(h), to_np(plain)) <= 1e-2


def test_plan_prefill_of_few_rows_and_many_experts(cuda):
    """Rows between the decode limit and a tile: every expert has a row or none."""
    import torch
    rng = np.random.default_rng(8)
    H, E, K, F, S, T = 256, 128, 2, 128, 128, 18
    w = _tiny_layer(rng, H, E, F, S)
    x = rng.standard_normal((T, H)).astype(np.float32)
    plan = M.Plan(M.Dims(H, E, K, F, S), max_rows=64, weight_format=M.WEIGHT_INT8, flags=M.PLAN_INT8_ACTIVATIONS)
    _upload(plan, w, torch, cuda)
    y, ids, wts = run_plan(plan, 0, torch.from_numpy(x).to(cuda), K, torch)
    want = O.moe_forward(w, x, K, renormalize=True)
    check_ids(ids, want)
    assert max_rel(y, restated(w, x, O.MoeResult(**{**want.__dict__, "ids": ids, "weights": wts}))) <= 1e-2


@pytest.mark.parametrize("shape", [(512, 2, 4, 1, 1024, 8, 2, 128, 256, 70, 6), (1024, 2, 8, 4, 768, 16, 4, 128, 128, 17, 5),
                                   (512, 1, 4, 2, 512, 8, 2, 128, 256, 9, 4)])
def test_decoder_prefill(cuda, shape):
    """The page decoder with int8 activations against the oracle on the dequantised weights, at the int8 bar."""
    import torch
    H, layers, heads, kv, vocab, E, K, F, S, n, steps = shape
    dims = D.DecoderDims(H, layers, heads, kv, 128, vocab, E, K, F, S)
    w_dev = D.synth_weights(dims, 5, int8=False, norm_sigma=0.1)
    dec = M.Decoder(H, layers, heads, kv, vocab, max_positions=n + steps + 3, max_prefill=n, experts=E, top_k=K, ffn=F,
                    shared_ffn=S, weight_format=M.WEIGHT_INT8, flags=M.DECODER_INT8_ACTIVATIONS)
    keep = [_device_layer(torch, cuda, L) for L in w_dev.layers]
    for i, t in enumerate(keep):
        dec.set_layer(i, t, dtype=M.DTYPE_F32)
    f = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(cuda)  # noqa: E731
    head = (f(w_dev.embed), f(w_dev.final_norm), f(w_dev.lm_head))
    dec.set_head(*head, dtype=M.DTYPE_F32)
    torch.cuda.synchronize()
    prompt = D.synth_prompt(dims, 5, n)
    side = torch.cuda.Stream()
    l0, t0, toks, lg = _run(torch, cuda, dec, prompt, vocab, steps, side)
    ora = D.DecoderOracle(dims, D.synth_weights(dims, 5, int8=True, norm_sigma=0.1))
    errs = [max_rel(l0, ora.prefill(prompt))]
    for s, token in enumerate([t0] + toks.tolist()[:-1]):
        errs.append(max_rel(lg[s], ora.step(token)))
    print(f"decoder {shape} int8 activations: max_rel {[f'{e:.1e}' for e in errs]}")
    assert max(errs) <= INT8_TOL, errs
    again = _run(torch, cuda, dec, prompt, vocab, steps, side)
    assert np.array_equal(l0, again[0]) and np.array_equal(lg, again[3])
    dec.close()
