"""Vocabulary scans over logits whose rows, vectors or first entries hold nothing finite: tokens masked out with -inf, rows masked
out as a whole, NaN.  Softmax of such a row is what torch.softmax gives (NaN as soon as the row holds a NaN or nothing but
-inf); its token is an index of the vocabulary all the same.

Tolerance: a sum of exponentials below 1, each off by a step of the exponential and by the rounding of its argument (2^-22 of 1 in
all), added in chains of V / 256 and at most 64 + 12 joins, 2^-24 each; the logarithm another 2^-22 of the result."""
import pytest
import torch

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def make(dev, v):
    gen = torch.Generator().manual_seed(v)
    z = (3 * torch.randn((12, v), generator=gen)).to(torch.bfloat16)
    z[1] = NAN
    z[2] = -INF
    z[3, : max(1, v // 2)] = -INF                       # the first half masked out
    z[4] = -INF
    z[4, v - 1] = 1.0                                   # one token left
    z[5, :8] = NAN                                      # the first vector, the rest as it is
    z[6, : v - 1] = -INF
    z[6, v - 1] = NAN
    z[7, ::3] = -INF
    z[8] = 0                                            # all tie
    z[9] = torch.finfo(torch.bfloat16).min              # the type's lowest value everywhere
    z[10, v // 2] = NAN
    return z.to(dev)


def clear_of_nan(z):
    return ~torch.isnan(torch.softmax(z.double(), 1)).any(1)


def check_conf(conf, tok, z):
    v = z.shape[1]
    err = (v / 256 + 76) * 2.0 ** -24 + 2.0 ** -22
    ok = clear_of_nan(z)
    assert torch.equal(torch.isnan(conf), ~ok)
    want = torch.softmax(z[ok].double(), 1).amax(1)
    assert bool(((conf[ok].double() / want - 1).abs() <= err).all())
    assert torch.equal(tok[ok].cpu(), z[ok].float().cpu().argmax(1))
    assert bool((tok >= 0).all()) and bool((tok < v).all()) and int(tok[1]) == 0 and int(tok[2]) == 0


@pytest.mark.parametrize("shifted", [0, 1])
@pytest.mark.parametrize("v", [1, 7, 8, 300, 5001, 20000])
def test_scans_without_a_finite_maximum(dev, v, shifted):
    from prefilling_dllm_amd import ops
    z = make(dev, v)
    if shifted:                                         # rows that begin at an odd element
        wide = torch.zeros((z.shape[0], v + 1), dtype=torch.bfloat16, device=dev)
        wide[:, 1:] = z
        z = wide[:, 1:]
    conf, tok = ops.conf_argmax(z, 1)
    check_conf(conf, tok, z)
    ids = torch.full((z.shape[0], 1), -5, dtype=torch.int64, device=dev)
    conf2, tok2, tr, left = ops.denoise_unmask(z, ids, -5, 0.9)
    assert torch.equal(tok, tok2) and torch.equal(conf[clear_of_nan(z)], conf2[clear_of_nan(z)])
    assert bool(tr.all()) and torch.equal(ids.flatten(), tok) and int(left.sum()) == 0
    labels = torch.full((z.shape[0],), v - 1, dtype=torch.int64, device=dev)
    logp = ops.selfinfo_logprob(z, labels)
    want = torch.log_softmax(z.double(), 1)[:, v - 1]
    assert torch.equal(torch.isnan(logp), torch.isnan(want))
    ok = ~torch.isnan(want)
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(logp), inf)
    ok &= ~inf
    err = (v / 256 + 76) * 2.0 ** -24 + 2.0 ** -22
    assert bool(((logp[ok].double() - want[ok]).abs() <= err + want[ok].abs() * 2.0 ** -22).all())


def test_confidence_of_a_row_without_logits_reaches_no_threshold(dev):
    """A block with one row of NaN and one of -inf: both confidences are NaN, so neither is transferred for its size."""
    from prefilling_dllm_amd import ops
    z = torch.randn((3 * 16, 1000), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    z[20], z[25] = NAN, -INF
    conf, tok = ops.conf_argmax(z, 16)
    assert bool(torch.isnan(conf[20])) and bool(torch.isnan(conf[25])) and not bool(torch.isinf(conf).any())
