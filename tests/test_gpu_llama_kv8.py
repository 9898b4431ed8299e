"""The decoder over an 8-bit cache: its two ways through a prompt, its pages, and how far it is from the fp16 cache."""
import numpy as np
import pytest
import torch

from antares_b200 import ops
from antares_b200.llama import LlamaConfig, LlamaInt4Decoder, SynthWeights, synth_prompt

pytestmark = pytest.mark.gpu


def _decoder(cuda, cfg, **kw):
    return LlamaInt4Decoder(cfg, cuda, weights=SynthWeights(cfg, centered=True, scale_mul=0.25), **kw)


def _feed(dec, toks, upto):
    """Token by token through the public call; the logits after each."""
    dec.reset(torch.from_numpy(toks[:1]).to(dec.dev))
    out = []
    for t in toks[:upto]:
        dec.step(int(t))
        out.append(dec.logits.clone())
    return torch.stack(out)


def _rel(a, b):
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize("n", [5, 70, 130])
def test_prompt_in_one_pass_and_token_by_token(cuda, n):
    cfg = LlamaConfig(n_layers=2, max_seq=256)
    toks = synth_prompt(cfg, n, 3)
    dec = _decoder(cuda, cfg, kv_bits=8)
    dec.capture(1)
    one = _feed(dec, toks, n)[-1]
    k_one, s_one = dec.k_cache.clone(), dec.k_scale.clone()
    dec.prefill(toks)
    k_all, s_all = dec.k_cache, dec.k_scale
    used = -(-n // 16)
    # the same scales but for the projections' own difference (another kernel: fp16 rounding of every value, 2^-10 of it)
    a, b = (s.permute(0, 1, 3, 2).reshape(2, -1, cfg.n_heads)[:, :used] for s in (s_one, s_all))
    assert _rel(a, b) <= 5e-3
    # a block's rows were rounded again whenever its scale grew, at most half a step a time: codes lie close together
    rows = [k.permute(0, 1, 3, 2, 4).reshape(2, -1, cfg.n_heads, 128)[:, :n].float() for k in (k_one, k_all)]
    assert (rows[0] - rows[1]).abs().mean() <= 1.5
    # both are this model at 8-bit precision: each is as far from the other as from the fp16 cache, see below
    assert _rel(one, dec.logits) <= 0.03
    # replayed, the recorded pass gives the same bits
    first = dec.logits.clone()
    dec.prefill(toks)
    assert torch.equal(first, dec.logits)
    assert ops.kernel_status() == 0


def test_close_to_the_fp16_cache(cuda):
    """A code is off by at most 1/254 of its block's largest value, about 1/85 of the spread of normal values at 3 sigma: each
    key and value 0.7 % in the mean, averaged over the keys that a row attends to; 3 % of the logits leaves room for two layers."""
    cfg = LlamaConfig(n_layers=2, max_seq=128)
    toks = synth_prompt(cfg, 90, 5)
    dec8, dec16 = _decoder(cuda, cfg, kv_bits=8), _decoder(cuda, cfg)
    dec8.capture(1)
    dec16.capture(1)
    a, b = _feed(dec8, toks, 90), _feed(dec16, toks, 90)
    assert _rel(a[0], b[0]) <= 0.03 and _rel(a, b) <= 0.03
    assert not torch.equal(a, b)


def test_pages_in_any_order_change_nothing(cuda):
    cfg = LlamaConfig(n_layers=2, max_seq=200)
    toks = synth_prompt(cfg, 100, 7)
    table = np.random.default_rng(0).permutation(7).astype(np.int32)
    outs = []
    for kw in (dict(kv_page_rows=32), dict(kv_page_rows=32, kv_page_table=table), dict(kv_page_rows=128)):
        dec = _decoder(cuda, cfg, kv_bits=8, **kw)
        dec.capture(1)
        dec.prefill(toks)
        for t in (11, 12, 13):
            dec.step(t)
        outs.append(dec.logits.clone())
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_generate_and_the_end_of_the_cache(cuda):
    cfg = LlamaConfig(n_layers=2, max_seq=40)
    dec = _decoder(cuda, cfg, kv_bits=8)
    prompt = synth_prompt(cfg, 6, 1)
    toks = dec.generate(prompt, 20)
    assert len(toks) == 26 and list(toks) == list(dec.generate(prompt, 20))
    assert len(dec.generate(prompt, 20, batched_prefill=True)) == 26
    dec.reset(torch.from_numpy(prompt).to(cuda))
    for _ in range(40):
        dec.step(5)
    with pytest.raises(IndexError):
        dec.step(5)
    assert dec.step_bytes(39) < LlamaInt4Decoder.step_bytes(_decoder(cuda, cfg), 39)
    assert ops.kernel_status() == 0


def test_refusals(cuda):
    cfg = LlamaConfig(n_layers=1, max_seq=64)
    for kw in (dict(kv_bits=4), dict(kv_bits=8, kv_page_rows=24), dict(kv_bits=8, kv_page_rows=8)):
        with pytest.raises(ValueError):
            _decoder(cuda, cfg, **kw)
