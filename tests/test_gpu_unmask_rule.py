"""The transfer rule of a denoise step where confidences are NaN: the order is the reference's torch.topk (NaN above every number),
ties to the lowest index, so a block forces exactly one position however its NaN lie."""
import pytest
import torch

pytestmark = pytest.mark.gpu

MASK = 7
NAN = float("nan")
LEAST = 0.875   # exact in fp32


def plain(conf, ids, threshold):
    """transfer [n, block] by the definition, one block after the other on the CPU."""
    out = torch.zeros(ids.shape, dtype=torch.bool)
    for b in range(ids.shape[0]):
        masked = [i for i in range(ids.shape[1]) if int(ids[b, i]) == MASK]
        if not masked:
            continue
        c = [float(conf[b, i]) for i in masked]
        nans = [i for i, v in zip(masked, c) if v != v]
        out[b, nans[0] if nans else masked[c.index(max(c))]] = True
        for i, v in zip(masked, c):
            if v >= threshold:
                out[b, i] = True
    return out


def check(ids, conf, tok, tr, left, after, threshold):
    ids, conf, tok, tr, left, after = (t.cpu() for t in (ids, conf, tok, tr, left, after))
    conf, tok = conf.view(ids.shape), tok.view(ids.shape)
    want = plain(conf, ids, threshold)
    assert torch.equal(tr.bool(), want)
    assert torch.equal(after, torch.where(want, tok, ids))
    assert torch.equal(left.long(), (ids == MASK).sum(1) - want.sum(1))


def test_one_nan_forces_one_position(dev):
    """NaN at 0, the largest confidence at 16, the next one at 8, all below the threshold."""
    from prefilling_dllm_amd import ops
    conf = torch.full((32,), 0.1, device=dev)
    conf[0], conf[16], conf[8] = NAN, 0.5, 0.4
    tok = torch.arange(100, 132, device=dev)
    ids = torch.full((1, 32), MASK, dtype=torch.int64, device=dev)
    tr, left = ops.threshold_unmask(conf, tok, ids, MASK, LEAST)
    assert tr[0].nonzero().flatten().tolist() == [0] and int(left) == 31 and int(ids[0, 0]) == 100


@pytest.mark.parametrize("block", [1, 2, 5, 32, 33, 64, 65, 130])
@pytest.mark.parametrize("share", [0.0, 0.1, 0.6, 1.0])
def test_threshold_unmask_with_nan(dev, block, share):
    from prefilling_dllm_amd import ops
    n = 40
    gen = torch.Generator().manual_seed(block * 10 + int(10 * share))
    conf = (torch.randint(-3, 12, (n, block), generator=gen).float() / 10)     # many ties, some negative, some above the threshold
    conf[torch.rand((n, block), generator=gen) < 0.05] = float("-inf")
    conf[torch.rand((n, block), generator=gen) < 0.05] = -0.0
    conf[torch.rand((n, block), generator=gen) < share] = NAN
    sign = torch.rand((n, block), generator=gen) < 0.5
    conf = torch.where(torch.isnan(conf) & sign, -conf, conf)                  # NaN of either sign
    ids = torch.randint(100, 200, (n, block), generator=gen)
    ids[torch.rand((n, block), generator=gen) < 0.7] = MASK
    ids[0] = 100                                                               # a block without a masked position
    tok = torch.randint(200, 300, (n * block,), generator=gen)
    after = ids.to(dev)
    tr, left = ops.threshold_unmask(conf.view(-1).to(dev), tok.to(dev), after, MASK, LEAST)
    check(ids, conf, tok, tr, left, after, LEAST)


@pytest.mark.parametrize("n,block", [(3, 32), (40, 33)])
def test_denoise_steps_with_nan_states(dev, n, block):
    """A NaN in some states, through the steps from logits and from states, with the transfers in the joining launch (up to 32
    blocks) and in one of their own."""
    from prefilling_dllm_amd import ops
    v, d = 900, 64
    gen = torch.Generator(device=dev).manual_seed(n)
    w = (torch.randn((v, d), generator=gen, device=dev) * 0.3).to(torch.bfloat16)
    h = torch.randn((n * block, d), generator=gen, device=dev).to(torch.bfloat16)
    h[torch.rand(n * block, generator=gen, device=dev) < 0.1, 3] = NAN
    ids = torch.randint(100, 200, (n, block), generator=gen, device=dev)
    ids[torch.rand((n, block), generator=gen, device=dev) < 0.7] = MASK
    logits = (h.float() @ w.float().t()).to(torch.bfloat16)
    for call in (lambda t: ops.head_denoise_unmask(h, w, t, MASK, LEAST), lambda t: ops.denoise_unmask(logits, t, MASK, LEAST)):
        after = ids.clone()
        conf, tok, tr, left = call(after)
        assert bool(torch.isnan(conf).any())
        check(ids, conf, tok, tr, left, after, LEAST)
