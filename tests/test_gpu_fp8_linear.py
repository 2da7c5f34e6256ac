"""Products of e4m3 operands with a scale for each block of 128 against the definition in 64 bits, and the quantisers bit by
bit.

Tolerances.  The matrix instruction adds eight neighbouring products exactly but for what lies below 2^-13 of the largest
of them (at most 7 products are cut, each by less than that), and the groups in fp32.  With T = sum over groups of the largest
|sx sw xq wq| and S = the sum over all: error below 7 * 2^-13 T + (16 + 3 + 2 ceil(K / 128)) * 2^-24 S, then half a step of bf16,
2^-8 of the value.  That is the worst case; in the root mean square the cuts are far apart in sign and the result is as near
as its bf16 rounding, at most 2^-8 / sqrt(3) of the values: half as much again is allowed."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def quantize_ref(x, rows, cols=128):
    """The quantiser's definition on the CPU: blocks of rows x 128, smallest power of two s with amax / s <= 448."""
    n, k = x.shape
    nb, kb = -(-n // rows), -(-k // cols)
    xp = torch.zeros((nb * rows, kb * cols), dtype=torch.float64)
    xp[:n, :k] = x.double()
    b = xp.view(nb, rows, kb, cols).permute(0, 2, 1, 3).reshape(nb, kb, -1)
    amax = b.abs().amax(2)
    frac, e = torch.frexp(amax / 448.0)
    s = torch.where(amax > 0, torch.exp2((e - (frac == 0.5).int()).double()).clamp(min=2.0 ** -126), torch.ones_like(amax))
    q = (xp / s.repeat_interleave(rows, 0).repeat_interleave(cols, 1))[:n, :k].float().to(torch.float8_e4m3fn)
    return q, s.float()


def check_linear(out, xq, xs, wq, ws):
    n, k = wq.shape
    a = xq.double() * xs.double().repeat_interleave(128, 1)[:, :k]
    b = wq.double() * ws.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    want = a @ b.t()
    top = lambda x: x.abs().view(x.shape[0], k // 8, 8).amax(2)
    tol = 7 * 2.0 ** -13 * (top(a) @ top(b).t()) + (19 + 2 * -(-k // 128)) * 2.0 ** -24 * (a.abs() @ b.abs().t())
    assert out.shape == want.shape and out.dtype == torch.bfloat16
    err = out.double() - want
    assert bool((err.abs() <= (want.abs() + tol) * 2.0 ** -8 + tol + 2.0 ** -130).all())
    if out.numel() > 1000:
        assert float(err.norm()) <= 1.5 * 2.0 ** -8 / 3 ** 0.5 * float(want.norm())


def operands(dev, m, n, k, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn((m, k), generator=gen, device=dev) * torch.exp2(torch.randint(-6, 7, (m, 1), generator=gen, device=dev).float())
    wq = (torch.randn((n, k), generator=gen, device=dev) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    ws = (0.3 + torch.rand((-(-n // 128), -(-k // 128)), generator=gen, device=dev)) * 0.01
    return x.to(torch.bfloat16), wq, ws


# every tile (32, 64, 128, 256 rows), one row to several tiles, blocks and vectors that end early, one feature
@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 4096, 4096), (3, 127, 128), (32, 129, 272), (33, 300, 144), (64, 1000, 1168),
                                   (65, 2201, 400), (128, 256, 2048), (129, 513, 1024), (333, 2201, 1168), (600, 130, 5120),
                                   (17, 40, 18944), (2, 20001, 64),
                                   # up to 32 rows: kept in shared memory beside many features, or streamed with them
                                   (5, 16400, 1040), (17, 20001, 1168), (32, 16385, 2064), (4, 16384, 1024), (9, 16384, 896), (1, 16390, 1040), (18, 12300, 1040), (16, 4100, 2064), (17, 4100, 2064),
                                   (20, 8200, 272),
                                   # few tiles of a long k, streamed 32 rows at a time: ragged rows and features, either width
                                   (59, 280, 8304), (97, 1003, 2048), (65, 8400, 144), (130, 17, 4112)])
def test_linear(dev, m, n, k):
    from prefilling_dllm_amd import ops
    x, wq, ws = operands(dev, m, n, k, seed=m + n + k)
    xq, xs = ops.quantize_fp8_rows(x)
    rq, rs = quantize_ref(x.cpu(), 1)
    assert torch.equal(xq.cpu().view(torch.uint8), rq.view(torch.uint8)) and torch.equal(xs.cpu(), rs)
    out = ops.fp8_block_linear(xq, wq, ws, x_scale=xs)
    check_linear(out, xq, xs, wq, ws)
    assert torch.equal(out, ops.fp8_block_linear(x, wq, ws))


@pytest.mark.parametrize("n,k", [(1, 16), (128, 128), (300, 400), (1000, 1168)])
def test_quantize_blocks(dev, n, k):
    from prefilling_dllm_amd import ops
    gen = torch.Generator().manual_seed(n)
    w = (torch.randn((n, k), generator=gen) * torch.exp2(torch.randint(-20, 20, (n, k), generator=gen).float())).to(torch.bfloat16)
    w[:, : k // 2] = torch.where(torch.rand((n, k // 2), generator=gen) < 0.5, 0.0, w[:, : k // 2].float()).to(torch.bfloat16)
    q, s = ops.quantize_fp8_blocks(w.to(dev))
    rq, rs = quantize_ref(w, 128)
    assert torch.equal(s.cpu(), rs)
    assert torch.equal(q.cpu().view(torch.uint8), rq.view(torch.uint8))


def test_quantize_edges(dev):
    """Zeros, values at the border of a power of two (448 and the number above it), the smallest and largest numbers, halves
    between two e4m3 values (to the even one), infinities and NaN."""
    from prefilling_dllm_amd import ops
    x = torch.zeros((9, 256))
    x[1, 0], x[2, 0], x[3, 0] = 448.0, 450.0, -896.0
    x[4] = 1e-39
    x[5, :128] = 3e38
    x[6, 0] = 256.0
    x[6, 1:9] = torch.tensor([17.0, 19.0, 21.0, 1.0625, 2.0 ** -10, 3 * 2.0 ** -10, -17.0, 2.0 ** -9])
    x[7, 3] = float("inf")
    x[8, 200] = float("nan")
    x = x.to(torch.bfloat16)
    q, s = ops.quantize_fp8_rows(x.to(dev))
    rq, rs = quantize_ref(x[:7], 1)
    assert torch.equal(s[:7].cpu(), rs)
    assert torch.equal(q[:7].cpu().float(), rq.float())
    assert bool(torch.isnan(s[7, 0])) and float(s[7, 1]) == 1.0 and bool(torch.isnan(s[8, 1])) and float(s[8, 0]) == 1.0
    # a row that holds one comes out NaN, the others do not see it
    _, wq, ws = operands(dev, 1, 40, 256)
    out = ops.fp8_block_linear(x.to(dev), wq, ws)
    assert bool(torch.isnan(out[7:]).all()) and bool(torch.isfinite(out[:5]).all()) and int(torch.count_nonzero(out[0])) == 0


def test_strides_and_out(dev):
    """Operands and output that are columns of wider tensors, an odd row stride of the output, scales of any stride."""
    from prefilling_dllm_amd import ops
    m, n, k = 70, 200, 400
    x, wq, ws = operands(dev, m, n, k, seed=5)
    xq, xs = ops.quantize_fp8_rows(x)
    want = ops.fp8_block_linear(x, wq, ws)
    xw = torch.full((m, 512), float("nan"), dtype=torch.bfloat16, device=dev)
    xw[:, 16:16 + k] = x
    wide = torch.zeros((n + 5, 432), dtype=torch.uint8, device=dev)
    wide[5:, :k] = wq.view(torch.uint8)
    wv = wide.view(torch.float8_e4m3fn)[5:, :k]
    wst = ws.t().contiguous().t()
    for pad in (0, 3, 8):
        buf = torch.full((m, n + pad + 8), 7.0, dtype=torch.bfloat16, device=dev)
        out = ops.fp8_block_linear(xw[:, 16:16 + k], wv, wst, out=buf[:, pad:pad + n])
        assert torch.equal(out, want)
        assert bool((buf[:, :pad] == 7).all()) and bool((buf[:, pad + n:] == 7).all())      # nothing beside it
    assert torch.equal(ops.fp8_block_linear(xq, wq, ws, x_scale=xs.contiguous()), want)
    rows = torch.full((m + 10, n), 7.0, dtype=torch.bfloat16, device=dev)
    ops.fp8_block_linear(x, wq, ws, out=rows[:m])
    assert bool((rows[m:] == 7).all())
    # a single row of a tensor whose rows begin anywhere
    odd = torch.zeros(2 * 403, dtype=torch.bfloat16, device=dev)[:403 * 2].view(2, 403)[:1, :400]
    odd.copy_(x[:1])
    assert torch.equal(ops.fp8_block_linear(odd, wq, ws, out=buf[:1, 3:3 + n]), ops.fp8_block_linear(x[:1], wq, ws))


@pytest.mark.parametrize("m,n,k", [(40, 300, 256), (9, 17000, 1040), (300, 5000, 400)])
def test_empty_rows_and_graph(dev, m, n, k):
    from prefilling_dllm_amd import ops
    x, wq, ws = operands(dev, m, n, k, seed=1)
    assert ops.fp8_block_linear(x[:0], wq, ws).shape == (0, n)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.fp8_block_linear(x, wq, ws)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.fp8_block_linear(x, wq, ws)
    for seed in (2, 3, 4):
        x.copy_(operands(dev, m, n, k, seed=seed)[0])
        want = ops.fp8_block_linear(x, wq, ws)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        torch.randn(1 << 20, device=dev).sum().item()


def test_eight_bit_head_feeds_the_denoise_step(dev):
    """A head in 8 bits: quantised weight -> logits in bf16 -> denoise_unmask and chunk scores, next to the 16-bit head read
    from the states.  An e4m3 rounding is off by at most 2^-4 of the value (or of the smallest normal number, 2^-6, times
    the scale), so a logit moves by less than the sum of 2 * 2^-4 + 2^-8 of its terms, and by a bf16 rounding."""
    from prefilling_dllm_amd import ops
    v, d, n_seqs, block = 3000, 512, 4, 32
    gen = torch.Generator(device=dev).manual_seed(3)
    w = (torch.randn((v, d), generator=gen, device=dev) * (2.5 / d ** 0.5)).to(torch.bfloat16)
    token = torch.randint(0, v - 1, (n_seqs * block,), generator=gen, device=dev)
    wt = w[token].float()
    h = (torch.randn((n_seqs * block, d), generator=gen, device=dev) + 60 * wt / (wt * wt).sum(1, keepdim=True)).to(torch.bfloat16)
    wq, ws = ops.quantize_fp8_blocks(w)
    logits = ops.fp8_block_linear(h, wq, ws)
    z = h.double() @ w.double().t()
    slack = (2 * 2.0 ** -4 + 2.0 ** -8) * (h.double().abs() @ w.double().abs().t()) + z.abs() * 2.0 ** -8
    assert bool(((logits.double() - z).abs() <= slack).all())
    ids = torch.full((n_seqs, block), v - 1, dtype=torch.int64, device=dev)
    ids8 = ids.clone()
    _, tok8, tr8, left8 = ops.denoise_unmask(logits, ids8, v - 1, 0.9)
    _, tok, tr, left = ops.head_denoise_unmask(h, w, ids, v - 1, 0.9)
    assert torch.equal(tok8, token) and torch.equal(tok, token)      # a lead of 60 is far beyond the noise of 8 bits
    assert torch.equal(ids8, ids) and torch.equal(tr8, tr) and torch.equal(left8, left)
    scores = ops.chunk_scores_from_logits(logits.view(n_seqs, block, v), token.view(n_seqs, block))
    want = ops.chunk_score_reduce(ops.head_selfinfo_logprob(h, w, token), n_seqs)
    assert bool(((scores - want).abs() <= 1e-4).all())
