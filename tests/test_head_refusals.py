"""Calls of the head and fp8 operators that are refused, on the host, before any launch: no GPU is needed."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from prefilling_dllm_amd import _lib
    return _lib.lib


@pytest.fixture(scope="module")
def p():
    buf = (ctypes.c_char * 8192)()
    p.keep = buf
    return (ctypes.addressof(buf) + 255) & ~255


def test_head_sizes_and_pointers(lib, p):
    f = lib.pdllm_head_selfinfo_logprob
    ok = dict(h=p, hs=64, w=p, ws=64, lab=p, n=4, v=100, d=64, ws_p=p, ws_n=1 << 20, out=p)

    def call(**kw):
        a = {**ok, **kw}
        return f(a["h"], a["hs"], a["w"], a["ws"], a["lab"], a["n"], a["v"], a["d"], a["ws_p"], a["ws_n"], a["out"], None, None)

    assert call(n=0) == 0                                            # nothing to do
    for kw, st in ((dict(h=None), -1), (dict(w=None), -1), (dict(lab=None), -1), (dict(out=None), -1),
                   (dict(n=-1), -2), (dict(v=0), -2), (dict(d=0), -2), (dict(d=60), -2), (dict(n=(1 << 24) + 1), -2),
                   (dict(v=(1 << 30) + 1), -2), (dict(d=(1 << 20) + 8, hs=1 << 21, ws=1 << 21), -2),
                   (dict(hs=56), -3), (dict(ws=56), -3), (dict(hs=68), -3), (dict(ws=68), -3), (dict(h=p + 8), -3),
                   (dict(w=p + 8), -3), (dict(ws=1 << 22), -3),
                   (dict(ws_p=None), -5), (dict(ws_n=8), -5), (dict(ws_p=p + 4), -5)):
        assert call(**kw) == st, kw
    assert lib.pdllm_head_workspace_bytes(-1, 10) == -2 and lib.pdllm_head_workspace_bytes(1, 0) == -2
    assert lib.pdllm_head_workspace_bytes(0, 10) == 0
    # a row's parts: 8 bytes and a position each, of 128 entries up to 64 rows and of 256 above
    for n in (1, 32, 33, 64, 65, 128, 129, 5000):
        assert lib.pdllm_head_workspace_bytes(n, 152064) >= n * (152064 // (128 if n <= 64 else 256)) * 12


def test_gradient_sizes_and_pointers(lib, p):
    f = lib.pdllm_head_selfinfo_grad
    need = lib.pdllm_head_selfinfo_grad_workspace_bytes(4, 100, 64)
    assert need > 0 and lib.pdllm_head_selfinfo_grad_workspace_bytes(0, 100, 64) == 0
    ok = dict(h=p, hs=64, w=p, ws=64, lab=p, lp=p, lse=p, g=p, n=4, v=100, d=64, ws_p=p, ws_n=need, gh=p, ghs=64, gw=p, gws=64)

    def call(**kw):
        a = {**ok, **kw}
        return f(a["h"], a["hs"], a["w"], a["ws"], a["lab"], a["lp"], a["lse"], a["g"], a["n"], a["v"], a["d"], a["ws_p"],
                 a["ws_n"], a["gh"], a["ghs"], a["gw"], a["gws"], None)

    for kw, st in ((dict(lp=None), -1), (dict(lse=None), -1), (dict(g=None), -1), (dict(gh=None), -1), (dict(gw=None), -1),
                   (dict(ghs=60), -3), (dict(gws=66), -3), (dict(gh=p + 4), -3), (dict(gw=p + 4), -3), (dict(d=20), -2),
                   (dict(ws_p=None), -5), (dict(ws_p=p + 16), -5), (dict(ws_n=1024), -5)):
        assert call(**kw) == st, kw
    for bad in ((-1, 10, 8), (1, 0, 8), (1, 10, 12), (1, 10, 0)):
        assert lib.pdllm_head_selfinfo_grad_workspace_bytes(*bad) == -2
    # 4096 rows against the full head: the pieces keep the scratch far below the 1.2 GB that the whole gradient of the logits takes
    assert lib.pdllm_head_selfinfo_grad_workspace_bytes(4096, 152064, 3584) < 450 << 20


def test_denoise_sizes_and_pointers(lib, p):
    f = lib.pdllm_head_denoise_unmask
    ok = dict(h=p, hs=64, last=None, ls=64, w=p, ws=64, ns=2, bl=4, v=100, d=64, ids=p, ws_p=p, ws_n=1 << 20, conf=p, tok=p, tr=p)

    def call(**kw):
        a = {**ok, **kw}
        return f(a["h"], a["hs"], a["last"], a["ls"], a["w"], a["ws"], a["ns"], a["bl"], a["v"], a["d"], 1, a["ids"], 5, 0.9,
                 a["ws_p"], a["ws_n"], a["conf"], a["tok"], a["tr"], None, None)

    assert call(ns=0) == 0
    for kw, st in ((dict(ids=None), -1), (dict(tr=None), -1), (dict(conf=None), -1), (dict(tok=None), -1), (dict(ns=-1), -2),
                   (dict(bl=0), -2), (dict(ns=1 << 20, bl=1 << 20), -2), (dict(last=p, ls=32), -3), (dict(last=p + 2), -3),
                   (dict(ws_n=16), -5)):
        assert call(**kw) == st, kw


def test_fp8_sizes_and_pointers(lib, p):
    f = lib.pdllm_fp8_linear
    ok = dict(x=p, xs=64, sx=p, sxr=1, sxb=4, w=p, ws=64, sw=p, swr=1, swb=1, m=4, n=8, k=64, out=p, os=8)

    def call(**kw):
        a = {**ok, **kw}
        return f(a["x"], a["xs"], a["sx"], a["sxr"], a["sxb"], a["w"], a["ws"], a["sw"], a["swr"], a["swb"], a["m"], a["n"],
                 a["k"], a["out"], a["os"], None)

    assert call(m=0) == 0
    for kw, st in ((dict(x=None), -1), (dict(sx=None), -1), (dict(w=None), -1), (dict(sw=None), -1), (dict(out=None), -1),
                   (dict(m=-1), -2), (dict(n=0), -2), (dict(k=0), -2), (dict(k=40), -2), (dict(k=(1 << 20) + 16), -2),
                   (dict(xs=48), -3), (dict(ws=72), -3), (dict(x=p + 8), -3), (dict(w=p + 4), -3), (dict(os=7), -3),
                   (dict(out=p + 1), -3), (dict(sxr=-1), -3), (dict(swb=-1), -3), (dict(ws=1 << 23), -3)):
        assert call(**kw) == st, kw
    g = lib.pdllm_fp8_linear_bf16
    need = lib.pdllm_fp8_linear_bf16_workspace_bytes(40, 64)
    assert need == 40 * 64 + 4 * 40 and lib.pdllm_fp8_linear_bf16_workspace_bytes(16, 64) == 0
    for bad in ((-1, 64), (4, 0), (4, 40), (4, (1 << 20) + 16), ((1 << 24) + 1, 64)):
        assert lib.pdllm_fp8_linear_bf16_workspace_bytes(*bad) == -2
    ok.update(m=40, ws_p=p, ws_n=need)

    def call16(**kw):
        a = {**ok, **kw}
        return g(a["x"], a["xs"], a["w"], a["ws"], a["sw"], a["swr"], a["swb"], a["m"], a["n"], a["k"], a["ws_p"], a["ws_n"],
                 a["out"], a["os"], None)

    assert call16(m=0) == 0
    for kw, st in ((dict(x=None), -1), (dict(w=None), -1), (dict(sw=None), -1), (dict(out=None), -1), (dict(m=-1), -2),
                   (dict(n=0), -2), (dict(k=40), -2), (dict(xs=48), -3), (dict(xs=68), -3), (dict(x=p + 8), -3), (dict(ws=72), -3),
                   (dict(os=7), -3), (dict(swr=-1), -3), (dict(xs=1 << 22), -3), (dict(ws_p=None), -5), (dict(ws_p=p + 4), -5),
                   (dict(ws_n=need - 1), -5)):
        assert call16(**kw) == st, kw
    for q in (lib.pdllm_fp8_quantize_rows, lib.pdllm_fp8_quantize_blocks):
        assert q(p, 64, 0, 64, p, 64, p, 1, 1, None) == 0
        assert q(None, 64, 2, 64, p, 64, p, 1, 1, None) == -1 and q(p, 64, 2, 64, None, 64, p, 1, 1, None) == -1
        assert q(p, 64, 2, 64, p, 64, None, 1, 1, None) == -1
        assert q(p, 64, -1, 64, p, 64, p, 1, 1, None) == -2 and q(p, 64, 2, 24, p, 64, p, 1, 1, None) == -2
        assert q(p, 60, 2, 64, p, 64, p, 1, 1, None) == -3 and q(p, 64, 2, 64, p, 72, p, 1, 1, None) == -3
        assert q(p + 2, 64, 2, 64, p, 64, p, 1, 1, None) == -3 and q(p, 64, 2, 64, p, 64, p, -1, 1, None) == -3


def test_python_layer_needs_device_tensors():
    from prefilling_dllm_amd import engine_ops, ops
    h, w = torch.zeros((4, 64), dtype=torch.bfloat16), torch.zeros((10, 64), dtype=torch.bfloat16)
    lab = torch.zeros(4, dtype=torch.int64)
    f = torch.zeros(4)
    for call in (lambda: ops.head_selfinfo_logprob(h, w, lab), lambda: ops.head_selfinfo_grad(h, w, lab, f, f, f),
                 lambda: ops.head_conf_argmax(h, w, 4), lambda: ops.head_denoise_unmask(h, w, lab.view(1, 4), 1, 0.9),
                 lambda: ops.quantize_fp8_rows(h), lambda: ops.quantize_fp8_blocks(w),
                 lambda: ops.fp8_block_linear(h, w, f), lambda: ops.chunk_score_reduce(f, 2),
                 lambda: engine_ops.denoise_unmask_step_from_hidden(h, w, lab.view(1, 4), mask_token_id=1, threshold=0.9)):
        with pytest.raises(ValueError, match="device tensors"):
            call()
    with pytest.raises(ValueError, match="n_chunks"):
        engine_ops.select_chunks_from_hidden(h, w, lab, 2)
