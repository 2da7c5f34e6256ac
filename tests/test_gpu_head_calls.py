"""Calls of the vocabulary head's functions as the engine's own steps make them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(dev, n, v, d, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    h = torch.randn((n, d), generator=gen, device=dev).to(torch.bfloat16)
    w = (torch.randn((v, d), generator=gen, device=dev) * (2.5 / d ** 0.5)).to(torch.bfloat16)
    return h, w, torch.randint(0, v, (n,), generator=gen, device=dev)


@pytest.mark.parametrize("topk", [None, 0, -1, 1, 6, 7, 100])
def test_chunk_selection_takes_what_the_selection_from_logits_takes(dev, topk):
    """None and numbers that are not positive select every chunk, in both forms."""
    from prefilling_dllm_amd import engine_ops
    c, j, v, d = 7, 3, 900, 64
    h, w, labels = make(dev, c * j, v, d)
    scores, idx = engine_ops.select_chunks_from_hidden(h.view(c, j, d), w, labels.view(c, j), topk)
    want = scores.cpu().argsort(descending=True, stable=True)[: topk if topk and topk > 0 else c].sort().values
    assert torch.equal(idx.cpu(), want)
    logits = (h.float() @ w.float().t()).to(torch.bfloat16).view(c, j, v)
    assert engine_ops.select_chunks_from_logits(logits, labels.view(c, j), topk)[1].shape == idx.shape
