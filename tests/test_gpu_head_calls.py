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


@pytest.mark.parametrize("n,v,d", [(1, 300, 64), (40, 900, 72), (130, 3000, 264)])
def test_logprob_carries_its_gradient(dev, n, v, d):
    """A loss on the log-probabilities, with terms beside it, gives the states and the weight the gradient of head_selfinfo_grad."""
    from prefilling_dllm_amd import ops
    h, w, labels = make(dev, n, v, d, seed=n)
    if n > 4:
        labels[2] = -100
    rows = labels >= 0
    g = torch.randn(n, generator=torch.Generator().manual_seed(n)).to(dev)
    logp, lse = ops.head_selfinfo_logprob(h, w, labels, return_lse=True)
    assert not logp.requires_grad
    want = ops.head_selfinfo_grad(h, w, labels, logp, lse, g)
    x, head = h.clone().requires_grad_(), torch.nn.Parameter(w.clone())
    # (a row without a label is -inf: left out of the sum, its gradient is 0)
    for with_lse in (False, True):
        got = ops.head_selfinfo_logprob(x, head, labels, return_lse=with_lse)
        got = got[0] if with_lse else got
        assert torch.equal(got.detach(), logp)
        a, b = torch.autograd.grad((got[rows] * g[rows]).sum() + 0 * x.float().sum(), (x, head))
        g0 = torch.where(rows, g, torch.zeros_like(g))
        ref = ops.head_selfinfo_grad(h, w, labels, logp, lse, g0)
        assert torch.equal(a, ref[0]) and torch.equal(b, ref[1]) and torch.equal(a, want[0])
    # one of the two alone, a mean, gradients that add up over two backward passes
    ops.head_selfinfo_logprob(h, head, labels)[rows].mean().backward()
    once = head.grad.clone()
    ops.head_selfinfo_logprob(h, head, labels)[rows].mean().backward()
    assert torch.equal(head.grad, once + once) and bool((once != 0).any())
    with torch.no_grad():
        assert not ops.head_selfinfo_logprob(x, head, labels).requires_grad
    # states from a layer in front
    proj = torch.eye(d, dtype=torch.bfloat16, device=dev).requires_grad_()
    ops.head_selfinfo_logprob(h @ proj, w, labels)[rows].sum().backward()
    assert proj.grad.shape == (d, d) and bool(torch.isfinite(proj.grad).all()) and bool((proj.grad != 0).any())


def test_what_the_gradient_does_not_cover_raises(dev):
    from prefilling_dllm_amd import ops
    h, w, labels = make(dev, 12, 300, 64)
    h.requires_grad_()
    logp, lse = ops.head_selfinfo_logprob(h, w, labels, return_lse=True)
    with pytest.raises(NotImplementedError, match="log sum exp"):
        (logp.sum() + lse.square().sum()).backward()
    logp = ops.head_selfinfo_logprob(h, w, labels)
    (g,) = torch.autograd.grad(logp.sum(), h, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    logp = ops.head_selfinfo_logprob(h, w, labels)
    with torch.no_grad():
        h.mul_(2)
    with pytest.raises(RuntimeError, match="modified"):
        logp.sum().backward()


def test_every_launch_is_made_on_the_device_of_its_tensors(dev, monkeypatch):
    """The device of the tensors is current around every launch of these functions (here told by the guard that makes it so)."""
    import contextlib

    from prefilling_dllm_amd import engine_ops, ops
    inside, launches = [0], []

    @contextlib.contextmanager
    def guard(device):
        assert device == dev
        inside[0] += 1
        yield
        inside[0] -= 1

    class Library:
        def __getattr__(self, name):
            f = getattr(real, name)
            if name.endswith("_bytes"):
                return f

            def call(*a):
                launches.append((name, inside[0] > 0))
                return f(*a)
            return call

    real = ops.lib
    monkeypatch.setattr(ops, "lib", Library())
    monkeypatch.setattr(ops, "_on", guard)
    h, w, labels = make(dev, 12, 300, 64)
    ids = torch.full((3, 4), 7, dtype=torch.int64, device=dev)
    engine_ops.select_chunks_from_hidden(h.view(3, 4, 64), w, labels.view(3, 4), 2)
    engine_ops.denoise_unmask_step_from_hidden(h, w, ids, mask_token_id=7, threshold=0.9)
    logp, lse = ops.head_selfinfo_logprob(h, w, labels, return_lse=True)
    ops.head_selfinfo_grad(h, w, labels, logp, lse, logp)
    ops.head_conf_argmax(h, w, 4)
    ops.chunk_score_reduce(logp, 3)
    wq, ws = ops.quantize_fp8_blocks(w)
    xq, xs = ops.quantize_fp8_rows(h)
    ops.fp8_block_linear(h, wq, ws)
    ops.fp8_block_linear(xq, wq, ws, x_scale=xs)
    assert len(launches) == 12 and [name for name, on in launches if not on] == []


def test_a_head_without_entries_is_refused(dev):
    """By every call with the library's own error, and block_ids stay as they were."""
    from prefilling_dllm_amd import ops
    h, w, labels = make(dev, 8, 300, 64)
    none = w[:0]
    ids = torch.full((2, 4), 7, dtype=torch.int64, device=dev)
    for call in (lambda: ops.head_selfinfo_logprob(h, none, labels), lambda: ops.head_conf_argmax(h, none, 4),
                 lambda: ops.head_denoise_unmask(h, none, ids, 7, 0.9),
                 lambda: ops.head_selfinfo_grad(h, none, labels, *(labels.float() for _ in range(3)))):
        with pytest.raises(ValueError, match="SHAPE"):
            call()
    assert bool((ids == 7).all())


def test_a_backward_pass_under_capture_is_refused(dev, monkeypatch):
    """(told by the question that the backward pass asks, not by a capture)"""
    from prefilling_dllm_amd import ops
    h, w, labels = make(dev, 12, 300, 64)
    h.requires_grad_()
    logp = ops.head_selfinfo_logprob(h, w, labels)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="call head_selfinfo_grad"):
        logp.sum().backward()
    assert h.grad is None


def test_scores_of_a_parameter_replay_from_a_graph(dev):
    """A weight that requires a gradient, scored under capture: the values of the eager call at every replay."""
    from prefilling_dllm_amd import ops
    h, w, labels = make(dev, 40, 900, 72)
    head = torch.nn.Parameter(w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.head_selfinfo_logprob(h, head, labels)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = ops.head_selfinfo_logprob(h, head, labels, return_lse=True)
    for seed in (1, 2, 3):
        h.copy_(make(dev, 40, 900, 72, seed=seed)[0])
        want = ops.head_selfinfo_logprob(h, w, labels, return_lse=True)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.detach(), want[0]) and torch.equal(lse.detach(), want[1])
        torch.randn(1 << 20, device=dev).sum().item()
