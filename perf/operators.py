"""The operators of the vocabulary head: their plain forms, the calls of the library and the cases they are timed on.

  selfinfo   log-probability of a label per row, from hidden states and the head's weight (no logits in memory)
  grad       the same with the gradients of the hidden states and of the weight
  denoise    one denoise step (confidence, token, transfer) from hidden states and the head's weight
  fp8        matrix product of bf16 rows with an e4m3 weight that has one scale for each block of 128 x 128

`own` selects the library's calls (True) or elementary torch operations in 32 bits (False).
"""
import math

import torch

own = False

MASK_ID = 5          # the mask token of the denoise cases
THRESHOLD = 0.9      # the engine's confidence threshold


# ------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------

def listed():
    return [
        # a handful of labels over the toy vocabulary of the tests: the latency of the call
        {"name": "selfinfo_tiny", "op": "selfinfo", "rows": 12, "vocab": 9000, "dim": 512},
        # chunk scoring of a long prompt: 32 chunks x 4 label tokens, the 28-head model's width and vocabulary
        {"name": "selfinfo_32_chunks", "op": "selfinfo", "rows": 128, "vocab": 152064, "dim": 3584},
        # perplexity of two chunks of 1025 tokens and one more, the 32-head model's width and vocabulary
        {"name": "selfinfo_long", "op": "selfinfo", "rows": 2051, "vocab": 126464, "dim": 4096},
        # a training step of a toy model, odd everywhere
        {"name": "grad_tiny", "op": "grad", "rows": 97, "vocab": 9001, "dim": 520},
        # a sequence of a small model, every second token masked out of the loss
        {"name": "grad_1000", "op": "grad", "rows": 1000, "vocab": 50021, "dim": 1032},
        # a batch of 4096 tokens against the full head: the largest training step
        {"name": "grad_4096", "op": "grad", "rows": 4096, "vocab": 152064, "dim": 3584},
        # one block of 32 masked tokens behind a cached prompt: every denoise step of one request
        {"name": "denoise_block", "op": "denoise", "seqs": 1, "block": 32, "vocab": 152064, "dim": 3584,
         "shift": True, "last": True},
        # 61 requests of an odd block length, without a state in front of the block
        {"name": "denoise_61x33", "op": "denoise", "seqs": 61, "block": 33, "vocab": 50021, "dim": 3584,
         "shift": True, "last": False},
        # one token through a square projection: the smallest call of a decode step
        {"name": "fp8_one_row", "op": "fp8", "rows": 1, "k": 4096, "n": 4096},
        # sizes that end inside a tile, a block of scales and a vector
        {"name": "fp8_odd", "op": "fp8", "rows": 333, "k": 1168, "n": 2201},
        # one block of 32 rows against the full head in 8 bits (the weight is all the traffic)
        {"name": "fp8_block_head", "op": "fp8", "rows": 32, "k": 3584, "n": 152064},
        # eight chunks of 1025 tokens through the widest projection of the 28-head model: prefill
        {"name": "fp8_prefill", "op": "fp8", "rows": 8200, "k": 3584, "n": 18944},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["selfinfo", "grad", "denoise", "fp8"])
    while True:
        if op == "fp8":
            case = {"op": op, "rows": _log(rng, 1, 8200), "k": 16 * _log(rng, 4, 1184), "n": _log(rng, 64, 152064)}
            if case["rows"] * case["k"] * case["n"] <= 8200 * 3584 * 18944:
                return case
            continue
        vocab, dim = _log(rng, 257, 152064), 8 * _log(rng, 8, 512)
        if op == "denoise":
            case = {"op": op, "seqs": _log(rng, 1, 64), "block": _log(rng, 1, 64), "vocab": vocab, "dim": dim,
                    "shift": rng.random() < 0.6, "last": rng.random() < 0.5}
            rows = case["seqs"] * case["block"]
        else:
            rows = _log(rng, 1, 4096)
            case = {"op": op, "rows": rows, "vocab": vocab, "dim": dim}
        if rows * vocab * dim <= 4096 * 152064 * 3584:
            return case


def work(case):
    if case["op"] == "fp8":
        m, k, n = case["rows"], case["k"], case["n"]
        kb, nb = -(-k // 128), -(-n // 128)
        return {"bytes": 2 * m * k + n * k + 4 * nb * kb + 2 * m * n, "flops": 2 * m * k * n}
    v, d = case["vocab"], case["dim"]
    if case["op"] == "denoise":
        rows = case["seqs"] * case["block"]
        last = case["seqs"] * d * 2 if case["shift"] and case["last"] else 0
        return {"bytes": 2 * rows * d + last + 2 * v * d + rows * (4 + 8 + 1 + 16) + 4 * case["seqs"], "flops": 2 * rows * v * d}
    rows = case["rows"]
    if case["op"] == "selfinfo":
        return {"bytes": 2 * rows * d + 2 * v * d + rows * (8 + 4), "flops": 2 * rows * v * d}
    return {"bytes": 4 * rows * d + 4 * v * d + rows * (8 + 4 + 4), "flops": 6 * rows * v * d}


# ------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------

def _head(gen, vocab, dim, dev):
    """A head whose logits against states of unit variance have a deviation of 2.5 (a piece at a time: the fp32 draw is
    twice the size of the weight)."""
    w = torch.empty((vocab, dim), dtype=torch.bfloat16, device=dev)
    for a in range(0, vocab, 16384):
        b = min(vocab, a + 16384)
        w[a:b] = torch.randn((b - a, dim), generator=gen, device=dev) * (2.5 / math.sqrt(dim))
    return w


def _states(gen, rows, w, token, boost, dev):
    """States of unit variance that lean towards the output vector of one token: its logit is `boost` higher."""
    h = torch.randn((rows, w.shape[1]), generator=gen, device=dev)
    wt = w[token].float()
    return (h + boost.unsqueeze(1) * wt / (wt * wt).sum(1, keepdim=True)).to(torch.bfloat16)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    if case["op"] == "fp8":
        m, k, n = case["rows"], case["k"], case["n"]
        kb, nb = -(-k // 128), -(-n // 128)
        # activations with a few channels ten times as large as the others; the weight as the program keeps it
        x = torch.randn((m, k), generator=gen, device=dev)
        x *= torch.where(torch.rand(k, generator=gen, device=dev) < 0.02, 10.0, 1.0)
        wq = torch.empty((n, k), dtype=torch.float8_e4m3fn, device=dev)
        for a in range(0, n, 16384):
            b = min(n, a + 16384)
            wq[a:b] = (torch.randn((b - a, k), generator=gen, device=dev) * 100.0).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
        ws = (0.5 + torch.rand((nb, kb), generator=gen, device=dev)) * (0.01 / math.sqrt(k))
        return {"op": "fp8", "x": x.to(torch.bfloat16), "wq": wq, "ws": ws}
    vocab = case["vocab"]
    w = _head(gen, vocab, case["dim"], dev)
    rows = case["seqs"] * case["block"] if case["op"] == "denoise" else case["rows"]
    token = torch.randint(0, vocab, (rows,), generator=gen, device=dev)
    if case["op"] == "denoise":
        # from unsure positions (confidence around a third) to certain ones; three quarters still masked
        boost = 13.0 + 17.0 * torch.rand(rows, generator=gen, device=dev)
        h = _states(gen, rows, w, token, boost, dev)
        last = None
        if case["shift"] and case["last"]:
            t0 = torch.randint(0, vocab, (case["seqs"],), generator=gen, device=dev)
            last = _states(gen, case["seqs"], w, t0, 13.0 + 17.0 * torch.rand(case["seqs"], generator=gen, device=dev), dev)
        ids = torch.randint(0, vocab, (case["seqs"], case["block"]), generator=gen, device=dev)
        ids[torch.rand(ids.shape, generator=gen, device=dev) < 0.75] = MASK_ID
        return {"op": "denoise", "h": h, "w": w, "ids": ids, "shift": case["shift"], "last": last}
    boost = 24.0 * torch.rand(rows, generator=gen, device=dev)
    h = _states(gen, rows, w, token, boost, dev)
    other = torch.randint(0, vocab, (rows,), generator=gen, device=dev)
    labels = torch.where(torch.rand(rows, generator=gen, device=dev) < 0.7, token, other)
    state = {"op": case["op"], "h": h, "w": w, "labels": labels}
    if case["op"] == "grad":
        # gradient of a mean over the masked positions weighted by 1 / masking rate; the other half has weight 0
        g = (torch.rand(rows, generator=gen, device=dev) < 0.5).float() * (-2.0 / rows)
        g[0] = -2.0 / rows
        state["g"] = g * (0.5 + torch.rand(rows, generator=gen, device=dev))
    return state


# ------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------

def _plain_quantize(x):
    """One scale for each row and 128 columns, the smallest power of two with amax / scale <= 448 (so that the division
    is exact); values rounded to e4m3."""
    m, k = x.shape
    kb = -(-k // 128)
    xb = torch.nn.functional.pad(x.float(), (0, kb * 128 - k)).view(m, kb, 128)
    frac, e = torch.frexp(xb.abs().amax(2))
    scale = torch.where(frac > 0, torch.exp2((e - torch.where(frac > 0.875, 8, 9)).float()), 1.0)
    q = (xb / scale.unsqueeze(2)).to(torch.float8_e4m3fn).float()
    return (q * scale.unsqueeze(2)).view(m, kb * 128)[:, :k]


def _plain_fp8(s):
    n, k = s["wq"].shape
    w = s["wq"].float()
    w *= s["ws"].repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return (_plain_quantize(s["x"]) @ w.t()).to(torch.bfloat16)


def _log1pexp(x):
    return x.clamp(min=0.0) + torch.log1p(torch.exp(-x.abs()))


def _plain_selfinfo(s):
    """logp = -log(1 + exp(lse of the other tokens - logit of the label)): exact also where the label is all but certain
    and 1 - p is far below the spacing of the numbers next to 1."""
    logits = s["h"].float() @ s["w"].float().t()
    labels = s["labels"].unsqueeze(1)
    x = logits.gather(1, labels).squeeze(1)
    rest = logits.scatter(1, labels, float("-inf"))
    m = rest.amax(1)
    rest = m + torch.log(rest.sub_(m.unsqueeze(1)).exp_().sum(1))
    logp = -_log1pexp(rest - x)
    return logp, x - logp, logits


def _plain_grad(s):
    logp, lse, d = _plain_selfinfo(s)
    g = s["g"].unsqueeze(1)
    d.sub_(lse.unsqueeze(1)).exp_().mul_(-g)
    d.scatter_(1, s["labels"].unsqueeze(1), -g * torch.expm1(logp).unsqueeze(1))
    return logp, (d @ s["w"].float()).to(torch.bfloat16), (d.t() @ s["h"].float()).to(torch.bfloat16)


def _plain_denoise(s):
    ids = s["ids"].clone()
    n, block = ids.shape
    h = s["h"]
    if s["shift"]:
        hb = h.view(n, block, -1)
        first = hb[:, :1] if s["last"] is None else s["last"].unsqueeze(1)
        h = torch.cat((first, hb[:, :-1]), 1).reshape(n * block, -1)
    logits = h.float() @ s["w"].float().t()
    top, token = logits.max(1)
    conf = 1.0 / torch.exp(logits - top.unsqueeze(1)).sum(1)
    masked = ids == MASK_ID
    c = torch.where(masked, conf.view(n, block), -1.0)
    best = torch.zeros_like(masked).scatter_(1, c.argmax(1, keepdim=True), True)
    transfer = masked & (best | (conf.view(n, block) >= THRESHOLD))
    ids = torch.where(transfer, token.view(n, block), ids)
    left = (masked.sum(1) - transfer.sum(1)).to(torch.int32)
    return conf, token, transfer, left, ids


def run(state):
    op = state["op"]
    if own:
        from prefilling_dllm_amd import ops
        if op == "selfinfo":
            return ops.head_selfinfo_logprob(state["h"], state["w"], state["labels"])
        if op == "grad":
            logp, lse = ops.head_selfinfo_logprob(state["h"], state["w"], state["labels"], return_lse=True)
            gh, gw = ops.head_selfinfo_grad(state["h"], state["w"], state["labels"], logp, lse, state["g"])
            return logp, gh, gw
        if op == "denoise":
            ids = state["ids"].clone()
            conf, token, transfer, left = ops.head_denoise_unmask(state["h"], state["w"], ids, MASK_ID, THRESHOLD,
                                                                  shift=state["shift"], last_hidden=state["last"])
            return conf, token, transfer, left, ids
        return ops.fp8_block_linear(state["x"], state["wq"], state["ws"])
    if op == "selfinfo":
        return _plain_selfinfo(state)[0]
    if op == "grad":
        return _plain_grad(state)
    if op == "denoise":
        return _plain_denoise(state)
    return _plain_fp8(state)


# ------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------

def _e4m3_64(v):
    """v (fp64, |v| <= 448 up to rounding) rounded to the nearest e4m3 value, ties to the even one."""
    _, e = torch.frexp(v)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3.0)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "fp8":
        x, wq, ws = s["x"].double(), s["wq"], s["ws"].double()
        (m, k), n = x.shape, wq.shape[0]
        out = torch.zeros((m, n), dtype=torch.float64, device=x.device)
        for b, a in enumerate(range(0, k, 128)):
            xb = x[:, a:a + 128]
            amax = xb.abs().amax(1, keepdim=True)
            scale = torch.where(amax > 0, torch.exp2(torch.ceil(torch.log2(amax / 448.0) - 1e-9)), 1.0)
            xb = _e4m3_64(xb / scale) * scale
            for c in range(0, n, 16384):
                rows = torch.arange(c, min(n, c + 16384), device=x.device)
                out[:, c:c + 16384] += xb @ (wq[rows, a:a + 128].double() * ws[rows // 128, b].unsqueeze(1)).t()
        return out
    h, w = s["h"].double(), s["w"]
    if case["op"] == "denoise":
        if s["shift"]:
            rows = torch.arange(h.shape[0], device=h.device)
            head = rows % case["block"] == 0
            src = torch.where(head, rows, rows - 1)
            hs = h[src]
            if s["last"] is not None:
                hs[head] = s["last"].double()
            h = hs
        z = torch.cat([h @ w[a:a + 16384].double().t() for a in range(0, w.shape[0], 16384)], 1)
        conf = torch.exp(z.amax(1) - torch.logsumexp(z, 1))
        return conf, None, None, None, None
    z = torch.cat([h @ w[a:a + 16384].double().t() for a in range(0, w.shape[0], 16384)], 1)
    logp = torch.log_softmax(z, 1)
    picked = logp[torch.arange(h.shape[0], device=h.device), s["labels"]]
    if case["op"] == "selfinfo":
        return picked
    del z
    d = logp.exp_().neg_()
    d[torch.arange(h.shape[0], device=h.device), s["labels"]] = -torch.expm1(picked)
    d *= s["g"].double().unsqueeze(1)
    gh = torch.zeros_like(h)
    gw = torch.empty(w.shape, dtype=torch.float64, device=w.device)
    for a in range(0, w.shape[0], 16384):
        gh += d[:, a:a + 16384] @ w[a:a + 16384].double()
        gw[a:a + 16384] = d[:, a:a + 16384].t() @ h
    return picked, gh, gw
