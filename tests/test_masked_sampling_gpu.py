"""The samplers on rows with masked (-inf) logits, as grammar masks leave them."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _sample(logits, temps, filtered, top_k=-1, top_p=1.0):
    from libra_b200 import ops

    B = logits.shape[0]
    dev = logits.device
    t = torch.tensor(temps, device=dev)
    seeds = torch.arange(B, device=dev) + 11
    pos = torch.arange(B, device=dev)
    tok = torch.full((B,), -1, dtype=torch.long, device=dev)
    lp = torch.full((B,), math.nan, device=dev)
    x = logits.clone()  # (the fp32 sampler clears its input)
    if filtered:
        ops.sample_tokens_filtered(x, t, torch.full((B,), top_p, device=dev),
                                   torch.full((B,), top_k, dtype=torch.long, device=dev), seeds, pos, tok, lp)
    else:
        ops.sample_tokens(x, t, seeds, pos, tok, lp)
    return tok.cpu(), lp.double().cpu()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("filtered", [False, True])
def test_masked_rows_sample_an_allowed_token_with_its_logprob(dtype, filtered):
    g = torch.Generator().manual_seed(3)
    V, temps = 9000, [1.0, 0.7, 0.0, 1.3]
    z = torch.randn(4, V, generator=g)
    keep = torch.rand(4, V, generator=g) < 0.01
    keep[1] = False
    keep[1, V - 1] = True  # one token left, behind every thread's first elements
    keep[3, :V // 2] = False
    z = torch.where(keep, z, -math.inf).to(dtype).cuda()
    tok, lp = _sample(z, temps, filtered, top_k=50 if filtered else -1, top_p=0.99 if filtered else 1.0)
    for b in range(4):
        assert bool(keep[b, tok[b]]), "a masked token was drawn"
        x = z[b].double().cpu() / (temps[b] or 1.0)
        want = float(torch.log_softmax(x, 0)[tok[b]])
        # fp32 sums of at most 100 terms and logarithms of values below 16: 2^-24 of a few hundred
        assert abs(float(lp[b]) - want) < 500 * 2.0 ** -24, (b, float(lp[b]), want)
    assert int(tok[1]) == V - 1 and float(lp[1]) == 0.0


@pytest.mark.parametrize("filtered", [False, True])
def test_row_of_nothing_but_masked_logits(filtered):
    z = torch.full((2, 500), -math.inf, device="cuda")
    z[1, 7] = 1.0
    tok, lp = _sample(z, [1.0, 1.0], filtered, top_k=5 if filtered else -1)
    assert float(lp[0]) == -math.inf and int(tok[1]) == 7 and float(lp[1]) == 0.0
