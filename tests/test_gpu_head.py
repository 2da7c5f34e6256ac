"""The vocabulary head from hidden states (log-probability of labels, its gradient, confidence / token, denoise step)
against the definitions in 64 bits.

Tolerances.  A logit is a sum of D products of bf16 numbers, exact in fp32, added in fp32: its error is below
D * 2^-24 * sum |h w| (every partial sum off by half a step).  logp, lse and log(conf) move by at most twice the largest
error of a row's logits, plus the error of exponential, sum over V terms in chains of at most 128 and about 64 joins, and
logarithm: 256 * 2^-24 + 2^-20.  A gradient is a sum whose terms are rounded to bf16 once, then rounded to bf16 itself.  bf16
keeps 8 significant bits: numbers in [1, 2) are 2^-7 apart, so a rounding is off by at most half of that, 2^-8 relative.
Up to 64 rows a second plane carries the remainder of the terms' rounding, itself rounded to bf16: 2^-8 * 2^-8 = 2^-16."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_BF16 = 2.0 ** -8   # half a step of bf16 relative to the value


def make(dev, n, v, d, seed=0, scale=2.5):
    gen = torch.Generator(device=dev).manual_seed(seed)
    h = torch.randn((n, d), generator=gen, device=dev).to(torch.bfloat16)
    w = (torch.randn((v, d), generator=gen, device=dev) * (scale / d ** 0.5)).to(torch.bfloat16)
    labels = torch.randint(0, v, (n,), generator=gen, device=dev)
    g = torch.randn(n, generator=gen, device=dev)
    return h, w, labels, g


def logit_error(h, w):
    """Per row: the bound on the error of its logits."""
    a = h.double().abs() @ w.double().abs().t()
    return a.amax(1) * h.shape[1] * 2.0 ** -24


def stat_error(h, w):
    return 2 * logit_error(h, w) + 256 * 2.0 ** -24 + 2.0 ** -20


def exact(h, w, labels, g):
    v = w.shape[0]
    z = h.double() @ w.double().t()
    inside = (labels >= 0) & (labels < v)
    at = labels.clamp(0, v - 1).unsqueeze(1)
    lp = torch.log_softmax(z, 1)
    picked = lp.gather(1, at).squeeze(1)
    d = -lp.exp()
    d.scatter_(1, at, -torch.expm1(picked).unsqueeze(1))
    d *= g.double().unsqueeze(1)
    d[~inside] = 0
    logp = torch.where(inside, picked, torch.full_like(picked, float("-inf")))
    return z, logp, torch.logsumexp(z, 1), d


def check_logp(logp, lse, h, w, want_logp, want_lse):
    err = stat_error(h, w)
    inf = torch.isinf(want_logp)
    assert torch.equal(torch.isinf(logp), inf) and bool((logp[inf] < 0).all())
    assert bool(((logp.double() - want_logp).abs()[~inf] <= err[~inf] + want_logp.abs()[~inf] * 2.0 ** -22).all())
    assert bool(((lse.double() - want_lse).abs() <= err + want_lse.abs() * 2.0 ** -22).all())


def check_grad(gh, gw, h, w, d):
    """The result is off by its own rounding and by what the rounding of d and the errors of z carry into the sum."""
    n = h.shape[0]
    rel = 2.0 ** -16 if n <= 64 else HALF_BF16
    dz = stat_error(h, w).unsqueeze(1)                      # relative error of exp(z - lse)
    carried = d.abs() * (rel + dz) + 2.0 ** -40
    for got, want, slack in ((gh, d @ w.double(), carried @ w.double().abs()),
                             (gw, d.t() @ h.double(), carried.t() @ h.double().abs())):
        assert got.dtype == torch.bfloat16
        tol = want.abs() * HALF_BF16 + slack * (1 + HALF_BF16) + 2.0 ** -30
        assert bool(((got.double() - want).abs() <= tol).all())


# every tile of the kernels (32, 64, 128, 256 rows), one row to several tiles, ragged in every direction, one entry
SHAPES = [(1, 1, 8), (1, 300, 64), (5, 1000, 520), (31, 127, 72), (32, 129, 64), (33, 2570, 136), (64, 3000, 256),
          (65, 257, 8), (128, 1025, 1032), (129, 3001, 512), (300, 2571, 136), (1030, 700, 200), (2, 40000, 64),
          # one piece of few entries (no sum of partial results), just more than that, the last row of the small tiles
          (20, 1024, 520), (20, 1030, 520), (256, 2000, 264), (257, 2001, 264), (200, 20000, 72),
          # just more than 32 tiles of 256 x 256; the large tiles of the gradient, ragged in every direction
          (1025, 1700, 72), (300, 25001, 264), (257, 50100, 72), (300, 25001, 384),
          (300, 25001, 392),
          # rows behind the last whole column: in pieces or as a column of their own
          (384, 17000, 64), (600, 17000, 64), (700, 9000, 72)]


@pytest.mark.parametrize("n,v,d", SHAPES)
def test_logprob_and_gradient(dev, n, v, d):
    from prefilling_dllm_amd import ops
    h, w, labels, g = make(dev, n, v, d, seed=n + v)
    if n > 4:
        labels[0], labels[n - 1], labels[2] = v, -1, -100
        labels[3] = labels[1]                               # the same entry twice
    z, want, want_lse, dz = exact(h, w, labels, g)
    logp, lse = ops.head_selfinfo_logprob(h, w, labels, return_lse=True)
    check_logp(logp, lse, h, w, want, want_lse)
    assert torch.equal(ops.head_selfinfo_logprob(h, w, labels), logp)
    gh, gw = ops.head_selfinfo_grad(h, w, labels, logp, lse, g)
    check_grad(gh, gw, h, w, dz)


def test_gradient_in_pieces(dev):
    """A workspace that holds a few hundred entries at a time gives the result of the whole vocabulary at once."""
    from prefilling_dllm_amd import _lib, ops
    for n in (40, 200):
        h, w, labels, g = make(dev, n, 5000, 264, seed=n)
        labels[5] = -1
        _, _, _, d = exact(h, w, labels, g)
        logp, lse = ops.head_selfinfo_logprob(h, w, labels, return_lse=True)
        full = ops.head_selfinfo_grad(h, w, labels, logp, lse, g)
        need = int(_lib.lib.pdllm_head_selfinfo_grad_workspace_bytes(n, 5000, 264))
        # a copy of the states, a piece of 256 entries, fp32 sums; up to 64 rows: rounded up to 32 or 64, twice, and the piece twice
        rows, copies = (128, 2) if n <= 64 else (n, 1)
        least = 2 * rows * 264 + 2 * rows * 256 * copies + 4 * n * 264 + 3 * 256
        for have in (need // 2, least + 2 * rows * 256 * copies, least):
            got = ops.head_selfinfo_grad(h, w, labels, logp, lse, g, max_workspace_bytes=have)
            check_grad(*got, h, w, d)
            assert torch.equal(got[1], full[1])             # grad_w does not depend on the pieces
        with pytest.raises(RuntimeError, match="WORKSPACE"):
            ops.head_selfinfo_grad(h, w, labels, logp, lse, g, max_workspace_bytes=2 * n * 264)


def test_gradient_against_differences(dev):
    """(f(x + e) - f(x - e)) / 2e of f = sum g logp in 64 bits, along a direction in each argument."""
    from prefilling_dllm_amd import ops
    h, w, labels, g = make(dev, 70, 500, 64, seed=3)
    logp, lse = ops.head_selfinfo_logprob(h, w, labels, return_lse=True)
    gh, gw = ops.head_selfinfo_grad(h, w, labels, logp, lse, g)

    def f(hh, ww):
        z = torch.log_softmax(hh @ ww.t(), 1)
        return float((g.double() * z.gather(1, labels.unsqueeze(1)).squeeze(1)).sum())

    gen = torch.Generator(device=dev).manual_seed(9)
    for x, grad, call in ((h, gh, lambda u: f(u, w.double())), (w, gw, lambda u: f(h.double(), u))):
        u = torch.randn(x.shape, generator=gen, device=dev, dtype=torch.float64)
        e = 1e-5
        num = (call(x.double() + e * u) - call(x.double() - e * u)) / (2 * e)
        ana = float((grad.double() * u).sum())
        # each element off by its own rounding and by that of its terms, 2^-8 each; along a random direction: their root sum of squares, 6 sigma
        tol = 6 * float(((grad.double() * u) ** 2).sum() ** 0.5) * 2.0 ** -7 + 1e-6
        assert abs(num - ana) <= tol


def test_nearly_certain_labels_keep_their_digits(dev):
    """logp of -1e-6 .. -1e-1 is right to a few parts in 10^5 of itself (log_softmax in fp32 loses the digits of the small ones),
    and so is 1 - p."""
    from prefilling_dllm_amd import ops
    n, v, d = 24, 400, 64
    h, w, labels, g = make(dev, n, v, d, seed=5, scale=1.0)
    boost = torch.linspace(10, 25, n, device=dev)
    wl = w[labels].float()
    h = (h.float() + boost.unsqueeze(1) * wl / (wl * wl).sum(1, keepdim=True)).to(torch.bfloat16)
    _, want, _, dz = exact(h, w, labels, g)
    logp, lse = ops.head_selfinfo_logprob(h, w, labels, return_lse=True)
    assert float(want.max()) > -1e-5 and float(want.min()) < -1e-2      # the inputs cover the range
    assert bool(((logp.double() - want).abs() <= want.abs() * stat_error(h, w)).all())
    gh, gw = ops.head_selfinfo_grad(h, w, labels, logp, lse, g)
    rel = lambda a, b: float((a.double() - b).abs().max() / b.abs().max())
    assert rel(gh, dz @ w.double()) <= 2 * HALF_BF16 and rel(gw, dz.t() @ h.double()) <= 2 * HALF_BF16


def test_rows_without_a_label_do_not_reach_the_gradient(dev):
    """States of NaN and infinity in rows whose label lies outside the vocabulary (a padded batch)."""
    from prefilling_dllm_amd import ops
    for n in (10, 150):
        h, w, labels, g = make(dev, n, 700, 72, seed=n)
        bad = torch.zeros(n, dtype=torch.bool, device=dev)
        bad[1::3] = True
        labels[bad] = -100
        h[bad] = float("nan")
        h[1] = float("inf")
        g[bad] = float("nan")
        logp, lse = ops.head_selfinfo_logprob(h, w, labels, return_lse=True)
        assert bool((logp[bad] == float("-inf")).all()) and bool(torch.isfinite(logp[~bad]).all())
        gh, gw = ops.head_selfinfo_grad(h, w, labels, logp, lse, g)
        assert bool((gh[bad] == 0).all())
        hk, lk, gk = h[~bad], labels[~bad], g[~bad]
        _, _, _, d = exact(hk, w, lk, gk)
        slack = (d.abs() * (HALF_BF16 + stat_error(hk, w).unsqueeze(1))).t() @ hk.double().abs()
        want = d.t() @ hk.double()
        assert bool(((gw.double() - want).abs() <= want.abs() * HALF_BF16 + 1.01 * slack + 1e-9).all())
        # every label outside: no gradient at all
        none = torch.full_like(labels, -1)
        gh, gw = ops.head_selfinfo_grad(h, w, none, logp, lse, g)
        assert int(torch.count_nonzero(gh)) == 0 and int(torch.count_nonzero(gw)) == 0


def test_extreme_logits(dev):
    """Rows of zeros (all entries tie), logits of +-1e4, and NaN in one row only."""
    from prefilling_dllm_amd import ops
    h, w, labels, g = make(dev, 40, 300, 64, seed=8)
    h[0] = 0
    h[1] = h[1] * 4096
    h[2, 5] = float("nan")
    logp, lse = ops.head_selfinfo_logprob(h, w, labels, return_lse=True)
    assert bool(torch.isnan(logp[2])) and bool(torch.isnan(lse[2]))
    keep = torch.arange(40, device=dev) != 2
    _, want, want_lse, _ = exact(h[keep], w, labels[keep], g[keep])
    check_logp(logp[keep], lse[keep], h[keep], w, want, want_lse)
    conf, tok = ops.head_conf_argmax(h, w, 1)
    assert int(tok[0]) == 0 and abs(float(conf[0]) - 1 / 300) < 1e-8      # ties go to the lowest index
    assert bool(torch.isnan(conf[2])) and 0 <= int(tok[2]) < 300


@pytest.mark.parametrize("n,v", [(1030, 17200), (130, 3000), (384, 17000), (60, 700)])
def test_equal_rows_have_equal_results(dev, n, v):
    """The same states in whole tiles, in pieces of them and behind them: the same bits, so that of two equally confident positions
    a block transfers the first."""
    from prefilling_dllm_amd import ops
    h, w, labels, _ = make(dev, n, v, 72, seed=n)
    again = torch.arange(n, device=dev) % 37
    h, labels = (h * torch.rand((n, 1), device=dev)).to(torch.bfloat16)[again], labels[again]
    logp, lse = ops.head_selfinfo_logprob(h, w, labels, return_lse=True)
    assert torch.equal(logp, logp[again]) and torch.equal(lse, lse[again])
    conf, tok = ops.head_conf_argmax(h, w, 1)
    assert torch.equal(conf, conf[again]) and torch.equal(tok, tok[again])
    # one state everywhere: the first position of each block
    ids = torch.full((2, n // 2), v - 1, dtype=torch.int64, device=dev)
    _, _, tr, _ = ops.head_denoise_unmask(h[:1].expand(n, 72).contiguous(), w, ids, v - 1, 2.0, shift=True)
    assert bool(tr[:, 0].all()) and int(tr.sum()) == 2


def test_views_and_strides(dev):
    """States that are columns of a wider tensor, a weight that is a slice of rows, int32 labels, a single row of any stride."""
    from prefilling_dllm_amd import ops
    h, w, labels, g = make(dev, 50, 600, 128, seed=2)
    hv = torch.full((50, 200), float("nan"), dtype=torch.bfloat16, device=dev)
    hv[:, 8:136] = h
    wv = torch.full((700, 136), float("nan"), dtype=torch.bfloat16, device=dev)
    wv[100:, :128] = w
    a = ops.head_selfinfo_logprob(h, w, labels, return_lse=True)
    b = ops.head_selfinfo_logprob(hv[:, 8:136], wv[100:, :128], labels.to(torch.int32), return_lse=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for x, y in zip(ops.head_selfinfo_grad(h, w, labels, *a, g),
                    ops.head_selfinfo_grad(hv[:, 8:136], wv[100:, :128], labels, *a, g)):
        assert torch.equal(x, y)
    one = ops.head_selfinfo_logprob(hv[7:8, 8:136], w, labels[7:8])
    assert torch.equal(one, ops.head_selfinfo_logprob(h[7:8], w, labels[7:8]))


def plain_shift(h, block, last):
    hb = h.view(-1, block, h.shape[1])
    first = hb[:, :1] if last is None else last.unsqueeze(1)
    return torch.cat((first, hb[:, :-1]), 1).reshape(h.shape)


@pytest.mark.parametrize("n_seqs,block,v,d,shift,with_last",
                         [(1, 1, 50, 8, True, True), (1, 32, 5000, 512, True, True), (3, 33, 4001, 264, True, False),
                          (2, 32, 1000, 64, False, False), (5, 64, 2000, 136, True, True), (1, 7, 1, 64, True, True),
                          (1, 3, 40000, 64, True, True), (32, 5, 300, 64, True, False), (40, 33, 1500, 64, True, True),
                          (33, 1, 40001, 72, False, False)])
def test_denoise_step(dev, n_seqs, block, v, d, shift, with_last):
    from prefilling_dllm_amd import ops
    n = n_seqs * block
    gen = torch.Generator(device=dev).manual_seed(n + v)
    _, w, token, _ = make(dev, n, v, d, seed=n * 3 + v)
    boost = 10 + 20 * torch.rand(n, generator=gen, device=dev)
    wt = w[token].float()
    h = (torch.randn((n, d), generator=gen, device=dev) + boost.unsqueeze(1) * wt / (wt * wt).sum(1, keepdim=True)).to(torch.bfloat16)
    last = torch.randn((n_seqs, d), generator=gen, device=dev).to(torch.bfloat16) if with_last else None
    hs = plain_shift(h, block, last) if shift else h
    z = hs.double() @ w.double().t()
    want_conf = torch.exp(z.amax(1) - torch.logsumexp(z, 1))
    conf, tok = ops.head_conf_argmax(h, w, block, shift=shift, last_hidden=last)
    assert bool(((conf.double() / want_conf - 1).abs() <= stat_error(hs, w) * 1.01).all())
    # the token is right wherever the two largest logits are further apart than their errors
    top = z.topk(min(2, v), 1)
    clear = torch.ones(n, dtype=torch.bool, device=dev) if v == 1 else \
        (top.values[:, 0] - top.values[:, 1]) > 2 * logit_error(hs, w)
    assert bool(clear.float().mean() > 0.9)
    assert torch.equal(tok[clear], z.argmax(1)[clear])
    mask_id = v - 1
    ids = torch.randint(0, v, (n_seqs, block), generator=gen, device=dev)
    ids[:, ::2] = mask_id
    want_ids = ids.clone()
    want_tr, want_left = ops.threshold_unmask(conf, tok, want_ids, mask_id, 0.9)
    got_ids = ids.clone()
    c2, t2, tr, left = ops.head_denoise_unmask(h, w, got_ids, mask_id, 0.9, shift=shift, last_hidden=last)
    for a, b in ((conf, c2), (tok, t2), (want_tr, tr), (want_left, left), (want_ids, got_ids)):
        assert torch.equal(a, b)


def test_empty_calls(dev):
    from prefilling_dllm_amd import ops
    h, w, labels, g = make(dev, 4, 300, 64)
    logp, lse = ops.head_selfinfo_logprob(h[:0], w, labels[:0], return_lse=True)
    assert logp.shape == (0,) and lse.shape == (0,)
    gh, gw = ops.head_selfinfo_grad(h[:0], w, labels[:0], logp, lse, g[:0])
    assert gh.shape == (0, 64) and gw.shape == (300, 64) and int(torch.count_nonzero(gw)) == 0
    conf, tok = ops.head_conf_argmax(h[:0], w, 8)
    assert conf.numel() == 0 and tok.numel() == 0
    conf, tok, tr, left = ops.head_denoise_unmask(h[:0], w, torch.empty((0, 8), dtype=torch.int64, device=dev), 1, 0.9)
    assert tr.shape == (0, 8) and left.shape == (0,)


@pytest.mark.parametrize("n,v,d", [(96, 3000, 256), (32, 3000, 72), (320, 25000, 264)])
def test_graph_replays_against_new_states(dev, n, v, d):
    """Logp, gradient and denoise step of one capture, replayed with new states and eager work in between."""
    from prefilling_dllm_amd import ops
    h, w, labels, g = make(dev, n, v, d, seed=1)
    ids0 = torch.full((n // 32, 32), 7, dtype=torch.int64, device=dev)

    def step(ids):
        logp, lse = ops.head_selfinfo_logprob(h, w, labels, return_lse=True)
        gh, gw = ops.head_selfinfo_grad(h, w, labels, logp, lse, g)
        return (logp, lse, gh, gw, ids) + ops.head_denoise_unmask(h, w, ids, 7, 0.5, shift=True)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(ids0.clone())
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    ids = ids0.clone()
    with torch.cuda.graph(graph):
        out = step(ids)
    for seed in (11, 12, 13):
        h.copy_(make(dev, n, v, d, seed=seed)[0])
        want = step(ids0.clone())
        ids.copy_(ids0)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
        (torch.randn(1 << 20, device=dev) * 2).sum().item()


def test_another_stream_gives_the_same(dev):
    from prefilling_dllm_amd import ops
    h, w, labels, g = make(dev, 200, 3000, 512, seed=4)
    a = ops.head_selfinfo_logprob(h, w, labels, return_lse=True)
    ga = ops.head_selfinfo_grad(h, w, labels, *a, g)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for s in (s1, s2):                                       # two calls at once, each with its own scratch
        with torch.cuda.stream(s):
            b = ops.head_selfinfo_logprob(h, w, labels, return_lse=True)
            outs.append(b + ops.head_selfinfo_grad(h, w, labels, *b, g))
    torch.cuda.synchronize()
    for o in outs:
        for x, y in zip(a + ga, o):
            assert torch.equal(x, y)


@pytest.mark.parametrize("n,v,d", [(20, 1100, 264), (100, 1100, 264), (300, 25000, 264), (20, 300, 72)])
def test_gradients_with_strides_of_their_own(dev, n, v, d):
    """The C entry with gradients whose rows begin at multiples of 8 bytes only: the same values, nothing written beside them."""
    from prefilling_dllm_amd import _lib, ops
    h, w, labels, g = make(dev, n, v, d, seed=n)
    logp, lse = ops.head_selfinfo_logprob(h, w, labels, return_lse=True)
    want = ops.head_selfinfo_grad(h, w, labels, logp, lse, g)
    gh = torch.full((n + 2, d + 4), 7.0, dtype=torch.bfloat16, device=dev)
    gw = torch.full((v + 2, d + 12), 7.0, dtype=torch.bfloat16, device=dev)
    need = int(_lib.lib.pdllm_head_selfinfo_grad_workspace_bytes(n, v, d))
    ws = torch.full((need + 256,), 255, dtype=torch.uint8, device=dev)     # (what it held before, NaN here, does not matter)
    st = _lib.lib.pdllm_head_selfinfo_grad(
        h.data_ptr(), d, w.data_ptr(), d, labels.data_ptr(), logp.data_ptr(), lse.data_ptr(), g.data_ptr(), n, v, d,
        ws.data_ptr(), need, gh[1:, 4:].data_ptr(), d + 4, gw[1:, 4:].data_ptr(), d + 12, torch.cuda.current_stream().cuda_stream)
    assert st == 0
    assert torch.equal(gh[1:n + 1, 4:4 + d], want[0]) and torch.equal(gw[1:v + 1, 4:4 + d], want[1])
    gh[1:n + 1, 4:4 + d] = 7
    gw[1:v + 1, 4:4 + d] = 7
    assert bool((gh == 7).all()) and bool((gw == 7).all()) and bool((ws[need:] == 255).all())


def test_head_scores_rank_chunks_like_the_logits(dev):
    """The chunk scoring of the engine from states: head_selfinfo_logprob -> mean per chunk -> top-k, next to the logits path."""
    from prefilling_dllm_amd import engine_ops, ops
    n_chunks, n_labels, v, d = 12, 4, 5000, 256
    h, w, labels, _ = make(dev, n_chunks * n_labels, v, d, seed=6)
    scores, idx = engine_ops.select_chunks_from_hidden(h.view(n_chunks, n_labels, d), w, labels.view(n_chunks, n_labels), 5)
    z = h.double() @ w.double().t()
    want = torch.log_softmax(z, 1).gather(1, labels.unsqueeze(1)).view(n_chunks, n_labels).mean(1)
    assert bool(((scores.double() - want).abs() <= stat_error(h, w).max() + want.abs() * 2.0 ** -21).all())
    assert sorted(want.topk(5).indices.tolist()) == idx.tolist()
    logits = (h @ w.t()).view(n_chunks, n_labels, v)
    ref_scores, _ = ops.chunk_select_from_logits(logits, labels.view(n_chunks, n_labels), 5)
    # the logits path rounds every logit to bf16: half a step of the largest, twice
    assert bool(((scores - ref_scores).abs() <= 2 * float(z.abs().max()) * HALF_BF16).all())


def test_denoise_loop_from_states(dev):
    """A block denoised to its end, step by step: the step from states and the step from fp32-exact logits take the same path."""
    from prefilling_dllm_amd import engine_ops, ops
    v, d, block, mask_id = 2000, 128, 16, 1999
    gen = torch.Generator(device=dev).manual_seed(21)
    w = (torch.randn((v, d), generator=gen, device=dev) * (2.5 / d ** 0.5)).to(torch.bfloat16)
    w[mask_id] = 0
    emb = torch.randn((v, d), generator=gen, device=dev)
    ids = torch.full((1, block), mask_id, dtype=torch.int64, device=dev)
    ids2 = ids.clone()
    last = torch.randn((1, d), generator=gen, device=dev).to(torch.bfloat16)
    for step in range(block):
        mix = torch.randn((block, block), generator=gen, device=dev)
        h = (3 * (mix @ emb[ids.view(-1)]) / block ** 0.5).to(torch.bfloat16)
        transfer, left = engine_ops.denoise_unmask_step_from_hidden(h, w, ids, mask_token_id=mask_id, threshold=0.9,
                                                                    last_context_hidden=last)
        conf, tok = ops.head_conf_argmax(h, w, block, shift=True, last_hidden=last)
        t2, l2 = ops.threshold_unmask(conf, tok, ids2, mask_id, 0.9)
        assert torch.equal(transfer, t2) and torch.equal(left, l2) and torch.equal(ids, ids2)
        if int(left) == 0:
            break
    assert int(left) == 0 and not bool((ids == mask_id).any())
