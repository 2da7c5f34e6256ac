"""The e4m3 product in its large tiles, against the definition in 64 bits (tolerances as in test_gpu_fp8_linear).

Above 32 rows the tile is the one of the fewest weighted rounds of the compute units: 20 for a round of 256 tiles of 256 x 256, 13
for one of 256 x 128, 10 for 512 of 128 x 64."""
import pytest
import test_gpu_fp8_linear as fp8
import torch

pytestmark = pytest.mark.gpu


def up(a, b):
    return -(-a // b)


def tile(m, n):
    tiles = lambda tm, tn: up(n, tm) * up(m, tn)
    l, mid, s = 20 * up(tiles(256, 256), 256), 13 * up(tiles(256, 128), 256), 10 * up(tiles(128, 64), 512)
    return "256x256" if l <= mid and l <= s else "256x128" if mid <= s else "128x64"


# rows and features that end inside a tile, an odd number of features, one to many stages of 128 columns, the last one short
CASES = [("256x128", 300, 14001, k) for k in (16, 80, 128, 144, 400, 1040)] + \
        [("256x256", 600, 18945, k) for k in (16, 80, 128, 144, 272, 1040)] + \
        [("256x128", 385, 14100, 256), ("256x256", 513, 20000, 384), ("256x128", 4100, 4097, 400), ("256x256", 8200, 4000, 272),
         ("256x128", 1030, 18944, 3584), ("256x256", 2050, 18000, 1024)]


@pytest.mark.parametrize("want,m,n,k", CASES)
def test_large_tiles(dev, want, m, n, k):
    from prefilling_dllm_amd import ops
    assert tile(m, n) == want
    x, wq, ws = fp8.operands(dev, m, n, k, seed=m + n + k)
    xq, xs = ops.quantize_fp8_rows(x)
    out = ops.fp8_block_linear(xq, wq, ws, x_scale=xs)
    fp8.check_linear(out, xq, xs, wq, ws)
    assert torch.equal(out, ops.fp8_block_linear(x, wq, ws))


@pytest.mark.parametrize("want,m,n,k", [("256x128", 300, 14001, 400), ("256x256", 600, 18945, 272)])
def test_large_tiles_in_wider_tensors(dev, want, m, n, k):
    """Operands that are columns of wider tensors, outputs whose rows begin at any element, scales by rows and by blocks."""
    from prefilling_dllm_amd import ops
    assert tile(m, n) == want
    x, wq, ws = fp8.operands(dev, m, n, k, seed=5)
    xq, xs = ops.quantize_fp8_rows(x)
    plain = ops.fp8_block_linear(xq, wq, ws, x_scale=xs)
    fp8.check_linear(plain, xq, xs, wq, ws)
    xw = torch.full((m, k + 48), 0x7f, dtype=torch.uint8, device=dev)         # NaN beside the operands
    xw[:, 16:16 + k] = xq.view(torch.uint8)
    ww = torch.full((n + 3, k + 32), 0x7f, dtype=torch.uint8, device=dev)
    ww[3:, 16:16 + k] = wq.view(torch.uint8)
    xv, wv = xw.view(torch.float8_e4m3fn)[:, 16:16 + k], ww.view(torch.float8_e4m3fn)[3:, 16:16 + k]
    for pad in (0, 1, 4, 8):
        buf = torch.full((m + 2, n + pad + 7), 7.0, dtype=torch.bfloat16, device=dev)
        ops.fp8_block_linear(xv, wv, ws.t().contiguous().t(), x_scale=xs.contiguous(), out=buf[1:m + 1, pad:pad + n])
        assert torch.equal(buf[1:m + 1, pad:pad + n], plain)
        buf[1:m + 1, pad:pad + n] = 7
        assert bool((buf == 7).all())


@pytest.mark.parametrize("want,m,n,k", [("256x128", 300, 14001, 400), ("256x256", 600, 18945, 272)])
def test_large_tiles_in_a_graph(dev, want, m, n, k):
    from prefilling_dllm_amd import ops
    assert tile(m, n) == want
    x, wq, ws = fp8.operands(dev, m, n, k, seed=1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.fp8_block_linear(x, wq, ws)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.fp8_block_linear(x, wq, ws)
    for seed in (2, 3, 4):
        x.copy_(fp8.operands(dev, m, n, k, seed=seed)[0])
        want_out = ops.fp8_block_linear(x, wq, ws)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want_out)
        torch.randn(1 << 20, device=dev).sum().item()


def test_rows_of_nan_and_zero_in_large_tiles(dev):
    """A row that holds an infinity or a NaN comes out NaN, one of zeros zero, and the others do not see them."""
    from prefilling_dllm_amd import ops
    for m, n, k in ((300, 14001, 400), (600, 18945, 272)):
        x, wq, ws = fp8.operands(dev, m, n, k, seed=9)
        want = ops.fp8_block_linear(x, wq, ws)
        bad = x.clone()
        bad[[1, m - 1]] = float("nan")
        bad[128, 5] = float("inf")
        bad[[2, 255]] = 0
        out = ops.fp8_block_linear(bad, wq, ws)
        keep = torch.ones(m, dtype=torch.bool, device=dev)
        keep[[1, 2, 128, 255, m - 1]] = False
        assert torch.equal(out[keep], want[keep]) and bool(torch.isnan(out[[1, 128, m - 1]]).all())
        assert int(torch.count_nonzero(out[[2, 255]])) == 0
