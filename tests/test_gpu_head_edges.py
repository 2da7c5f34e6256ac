"""The vocabulary head's rows whose logits leave fp32: a label of -inf, every entry -inf.  (A logit overflows where the product of
two bf16 numbers does: 2^100 * -2^100.)"""
import pytest
import torch

pytestmark = pytest.mark.gpu

BIG = 2.0 ** 100
HALF_BF16 = 2.0 ** -8   # half a step of bf16 relative to the value


@pytest.mark.parametrize("n,v", [(20, 700), (100, 9000), (300, 20000)])
def test_label_of_minus_infinity(dev, n, v):
    """logp is -inf, lse that of the other entries, and the row's gradient g ([v = label] - p) finite."""
    from prefilling_dllm_amd import ops
    d = 72
    gen = torch.Generator(device=dev).manual_seed(n)
    h = torch.randn((n, d), generator=gen, device=dev).to(torch.bfloat16)
    w = (torch.randn((v, d), generator=gen, device=dev) * 0.3).to(torch.bfloat16)
    h[:, 0], w[:, 0] = 0, 0
    labels = torch.randint(0, v - 1, (n,), generator=gen, device=dev)
    rows = torch.tensor([3, n - 1], device=dev)
    h[rows, 0], w[v - 1, 0], labels[rows] = BIG, -BIG, v - 1
    g = torch.randn(n, generator=gen, device=dev)
    z = h.double() @ w.double().t()
    logp, lse = ops.head_selfinfo_logprob(h, w, labels, return_lse=True)
    assert bool((logp[rows] == float("-inf")).all())
    # sums of 72 products below 8 and of v exponentials: far below 1e-4
    assert bool(((lse.double() - torch.logsumexp(z, 1)).abs() < 1e-4).all())
    gh, gw = ops.head_selfinfo_grad(h, w, labels, logp, lse, g)
    p = torch.softmax(z, 1)
    p[torch.arange(n, device=dev), labels] -= 1
    p *= -g.double().unsqueeze(1)
    # d rounded to bf16 (up to 64 rows with its remainder) and off by the error of lse, the result rounded to bf16
    rel = HALF_BF16 + 2e-4
    for got, want, size in ((gh, p @ w.double(), p.abs() @ w.double().abs()), (gw, p.t() @ h.double(), p.abs().t() @ h.double().abs())):
        assert bool(torch.isfinite(got).all())
        assert bool(((got.double() - want).abs() <= want.abs() * HALF_BF16 + size * rel * (1 + HALF_BF16) + 2.0 ** -30).all())


@pytest.mark.parametrize("n,v", [(20, 300), (100, 40000), (300, 20000)])
def test_every_entry_minus_infinity(dev, n, v):
    """Softmax of such a row is NaN, so its confidence reaches no threshold; its token is 0."""
    from prefilling_dllm_amd import ops
    d = 72
    gen = torch.Generator(device=dev).manual_seed(n)
    h = torch.randn((n, d), generator=gen, device=dev).to(torch.bfloat16)
    w = (torch.randn((v, d), generator=gen, device=dev) * 0.3).to(torch.bfloat16)
    h[:, 0], w[:, 0] = 0, BIG
    h[[2, n - 1], 0] = -BIG
    conf, tok = ops.head_conf_argmax(h, w, n)
    nan = torch.zeros(n, dtype=torch.bool, device=dev)
    nan[[2, n - 1]] = True
    assert torch.equal(torch.isnan(conf), nan) and bool((tok[nan] == 0).all()) and bool((conf[~nan] <= 1).all())
    ids = torch.full((1, n), -1, dtype=torch.int64, device=dev)
    _, _, tr, left = ops.head_denoise_unmask(h, w, ids, -1, 2.0)
    assert tr[0].nonzero().flatten().tolist() == [2] and int(left) == n - 1
    labels = torch.zeros(n, dtype=torch.int64, device=dev)
    logp, lse = ops.head_selfinfo_logprob(h, w, labels, return_lse=True)
    assert torch.equal(torch.isnan(logp), nan) and bool((lse[nan] == float("-inf")).all()) and bool(torch.isfinite(lse[~nan]).all())
