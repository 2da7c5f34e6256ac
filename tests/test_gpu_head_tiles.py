"""The vocabulary head in the tiles that only large vocabularies and many rows take, against the definitions in 64 bits
(tolerances as in test_gpu_head).

Which tile a call takes: 128 entries high up to 64 rows or up to 512 tiles of 128 x 64, else 256 high: 128 rows wide up to 128
rows, 256 wide above.  A last round of the 256 compute units that pieces of 64 rows would fill at most once is cut into them, and so are
up to 128 rows behind the last whole column (beside a single column up to 64, while the weight has at most 256 MB)."""
import pytest
import test_gpu_head as head
import torch

pytestmark = pytest.mark.gpu


def up(a, b):
    return -(-a // b)


def plan(n, v, d):
    """(width of the tiles, whole tiles, tiles cut into pieces, columns of pieces behind the whole columns)."""
    assert n > 64 and up(v, 128) * up(n, 64) > 512
    tn = 128 if n <= 128 else 256
    rest = n % tn
    again = n >= 2 * tn or up(v, 256) * 512 * d <= 256 << 20
    cols = up(rest, 64) if 0 < rest <= (tn // 2 if n >= 2 * tn else tn // 4) and again else 0
    whole = up(v, 256) * (n // tn + (rest > 0 and cols == 0))
    cut = whole % 256 if tn // 64 * (whole % 256) <= 256 else 0
    return tn, whole - cut, cut, cols


@pytest.mark.parametrize("n,v,d,want", [
    (97, 33001, 72, (128, 129, 0, 0)), (128, 33025, 264, (128, 130, 0, 0)),     # 128 wide, one round
    (100, 70001, 72, (128, 256, 18, 0)), (65, 65700, 8, (128, 256, 1, 0)),      # and a round of pieces: 64 rows and 36, 64 and 1
    (128, 90000, 136, (128, 256, 96, 0)),
    (1320, 9001, 72, (256, 180, 0, 1)),                                         # 256 wide: rows behind the last whole column
    (1320, 13500, 72, (256, 256, 9, 1)),                                        # beside a round of pieces
    (300, 70001, 72, (256, 256, 18, 1)), (257, 33000, 136, (256, 129, 0, 1)),   # behind a single column
    (290, 140000, 1032, (256, 1094, 0, 0)),                                    # no: the weight has more than 256 MB
    (200, 70001, 520, (256, 256, 18, 0)),
])
def test_large_tiles(dev, n, v, d, want):
    assert plan(n, v, d) == want
    head.test_logprob_and_gradient(dev, n, v, d)


@pytest.mark.parametrize("n_seqs,block,v,d,want", [(3, 33, 33001, 72, (128, 129, 0, 0)), (4, 25, 70001, 72, (128, 256, 18, 0)),
                                                   (40, 33, 9001, 72, (256, 180, 0, 1)), (40, 33, 13500, 136, (256, 256, 9, 1)),
                                                   (9, 32, 70001, 72, (256, 256, 18, 1))])
@pytest.mark.parametrize("shift,with_last", [(False, False), (True, False), (True, True)])
def test_denoise_in_large_tiles(dev, n_seqs, block, v, d, want, shift, with_last):
    assert plan(n_seqs * block, v, d) == want
    head.test_denoise_step(dev, n_seqs, block, v, d, shift, with_last)


@pytest.mark.parametrize("pieces", [3, 5])
def test_large_gradient_tiles_in_pieces(dev, pieces):
    """Pieces of 24576 or 12288 entries in tiles of 256 x 256 and a last one of 400 in tiles of 128 x 64, in a workspace that held
    NaN: grad_w as from one piece, grad_h within the bounds, nothing behind the workspace."""
    from prefilling_dllm_amd import _lib, ops
    n, v, d = 330, 49552, 264
    piece = (v - 400) // (pieces - 1)
    assert v == (pieces - 1) * piece + 400 and up(piece, 128) * up(n, 64) > 512 >= up(400, 128) * up(n, 64)
    assert n > 256 and up(d, 256) * up(v, 256) >= 192                        # (not the small tiles of the products)
    h, w, labels, g = head.make(dev, n, v, d, seed=pieces)
    labels[5] = -1
    labels[6], labels[7] = v - 1, piece                                      # in the last piece, the first entry of the second
    _, _, _, want = head.exact(h, w, labels, g)
    logp, lse = ops.head_selfinfo_logprob(h, w, labels, return_lse=True)
    full = ops.head_selfinfo_grad(h, w, labels, logp, lse, g)
    head.check_grad(*full, h, w, want)
    # the states' copy, a piece of d, the accumulators of its splits (at least 256 entries each, 256 workgroups in all)
    splits = min(piece // 256, 256 // (up(d, 256) * up(n, 256)))
    a256 = lambda x: up(x, 256) * 256
    have = a256(2 * n * d) + a256(2 * n * piece) + a256(4 * splits * n * d)
    ws = torch.full((have + 512,), 255, dtype=torch.uint8, device=dev)
    gh = torch.full((n, d), float("nan"), dtype=torch.bfloat16, device=dev)
    gw = torch.full((v, d), float("nan"), dtype=torch.bfloat16, device=dev)
    st = _lib.lib.pdllm_head_selfinfo_grad(
        h.data_ptr(), d, w.data_ptr(), d, labels.data_ptr(), logp.data_ptr(), lse.data_ptr(), g.data_ptr(), n, v, d,
        ws.data_ptr(), have, gh.data_ptr(), d, gw.data_ptr(), d, torch.cuda.current_stream().cuda_stream)
    assert st == 0
    assert torch.equal(gw, full[1]) and bool((ws[have:] == 255).all())
    head.check_grad(gh, gw, h, w, want)
    ws.fill_(255)                                                            # once more: the same bits
    gh2, gw2 = ops.head_selfinfo_grad(h, w, labels, logp, lse, g, max_workspace_bytes=have)
    assert torch.equal(gh2, gh) and torch.equal(gw2, gw)


def chunked(h, w, labels, g):
    """The definitions in 64 bits, the vocabulary 16384 entries at a time: logp, lse, the bound of their errors (a row each) and
    the gradient of the logits."""
    step = 16384
    hd = h.double()
    z = torch.cat([hd @ w[a:a + step].double().t() for a in range(0, w.shape[0], step)], 1)
    lse = torch.logsumexp(z, 1)
    logp = z.gather(1, labels.unsqueeze(1)).squeeze(1) - lse
    err = torch.zeros(h.shape[0], dtype=torch.float64, device=h.device)
    for a in range(0, w.shape[0], step):
        err = torch.maximum(err, (hd.abs() @ w[a:a + step].double().abs().t()).amax(1))
    err = 2 * err * h.shape[1] * 2.0 ** -24 + 256 * 2.0 ** -24 + 2.0 ** -20
    d = z.sub_(lse.unsqueeze(1)).exp_().neg_()
    d[torch.arange(h.shape[0], device=h.device), labels] = -torch.expm1(logp)
    return logp, lse, err, d.mul_(g.double().unsqueeze(1))


@pytest.mark.parametrize("n", [128, 1100])
def test_full_vocabulary_and_width(dev, n):
    """152064 entries of 3584 columns: the whole weight at 16 bits, at 1100 rows the gradient in two pieces of the workspace that
    the library asks for."""
    from prefilling_dllm_amd import _lib, ops
    v, d, step = 152064, 3584, 16384
    if n > 1000:
        assert 2 * n * v > 256 << 20
    h, w, labels, g = head.make(dev, n, v, d, seed=n)
    labels[0], labels[1] = 0, v - 1
    logp, lse = ops.head_selfinfo_logprob(h, w, labels, return_lse=True)
    gh, gw = ops.head_selfinfo_grad(h, w, labels, logp, lse, g)
    want_logp, want_lse, err, dz = chunked(h, w, labels, g)
    assert bool(((logp.double() - want_logp).abs() <= err + want_logp.abs() * 2.0 ** -22).all())
    assert bool(((lse.double() - want_lse).abs() <= err + want_lse.abs() * 2.0 ** -22).all())
    half = head.HALF_BF16
    carried_h = torch.zeros(h.shape, dtype=torch.float64, device=dev)
    want_h = torch.zeros_like(carried_h)
    for a in range(0, v, step):
        dc, wc = dz[:, a:a + step], w[a:a + step].double()
        carried = dc.abs() * (half + err.unsqueeze(1)) + 2.0 ** -40
        want_h += dc @ wc
        carried_h += carried @ wc.abs()
        want_w, slack = dc.t() @ h.double(), carried.t() @ h.double().abs()
        assert bool(((gw[a:a + step].double() - want_w).abs() <= want_w.abs() * half + slack * (1 + half) + 2.0 ** -30).all()), a
    assert bool(((gh.double() - want_h).abs() <= want_h.abs() * half + carried_h * (1 + half) + 2.0 ** -30).all())


def test_weight_beyond_two_gigabytes(dev):
    """152064 entries of 8192 columns, 2.3 GiB: scores of labels at the end of the weight, tokens wherever they lie."""
    from prefilling_dllm_amd import ops
    v, d, n, step = 152064, 8192, 40, 16384
    gen = torch.Generator(device=dev).manual_seed(7)
    w = torch.empty((v, d), dtype=torch.bfloat16, device=dev)
    for a in range(0, v, step):
        w[a:a + step] = torch.randn((min(step, v - a), d), generator=gen, device=dev) * (2.5 / d ** 0.5)
    token = torch.randint(0, v, (n,), generator=gen, device=dev)
    token[:4] = torch.tensor([v - 1, v - 2, 0, v - 130], device=dev)
    wt = w[token].float()
    h = (torch.randn((n, d), generator=gen, device=dev) + 40 * wt / (wt * wt).sum(1, keepdim=True)).to(torch.bfloat16)
    one = torch.ones(n, device=dev)
    want_logp, want_lse, err, _ = chunked(h, w, token, one)
    for rows in (slice(0, n), slice(0, 1)):
        logp, lse = ops.head_selfinfo_logprob(h[rows], w, token[rows], return_lse=True)
        assert bool(((logp.double() - want_logp[rows]).abs() <= err[rows] + want_logp[rows].abs() * 2.0 ** -22).all())
        assert bool(((lse.double() - want_lse[rows]).abs() <= err[rows] + want_lse[rows].abs() * 2.0 ** -22).all())
        conf, tok = ops.head_conf_argmax(h[rows], w, 1)
        assert torch.equal(tok, token[rows])          # a lead of 40 is far beyond the largest of the others, 2.5 * 4.5
    big = h.repeat(4, 1)                               # 160 rows: the tiles of 256
    logp4 = ops.head_selfinfo_logprob(big, w, token.repeat(4))
    assert bool(((logp4.double() - want_logp.repeat(4)).abs() <= err.repeat(4) + want_logp.repeat(4).abs() * 2.0 ** -22).all())
    assert torch.equal(ops.head_conf_argmax(big, w, 1)[1], token.repeat(4))
