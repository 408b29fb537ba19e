"""What is measured of the token table and the 8-bit floating point products: cases, inputs, plain forms, exact values.

Four operators of a model whose vocabulary table is looked up on the way in and whose linear layers run in 8-bit
floating point with one fp32 scale for each block of 128:

  embedding        out[t] = scale * table[ids[t]]
  embedding_grad   grad_table[v] = scale * sum of grad_out[t] over the tokens t with ids[t] == v, 0 where there is none
  quantize         a group G of x (1 x 128 or 128 x 128 values): s = 2^e with the smallest e such that max|G| <= top * 2^e
                   (top = 448 for e4m3, 57344 for e5m2), q = x / s rounded to nearest even
  gemm             C = act(sum over blocks b of 128 of K: sa[., b] * sb[b, .] * (A[:, b] @ B[b, :]) + bias)

`own` = False runs them as elementary torch operations in 32 bits, `own` = True as calls of accera_b200.runtime.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
TOP = {"e4m3": 448.0, "e5m2": 57344.0}


def listed():
    return [
        # the token step of a small serving batch: eight rows of a 32000-word table, latency alone
        {"name": "embedding_step", "op": "embedding", "tokens": 8, "vocab": 32000, "dim": 4096, "type": "bf16", "scale": 64.0},
        # a prompt batch through the same table
        {"name": "embedding_prompt", "op": "embedding", "tokens": 16384, "vocab": 32000, "dim": 4096, "type": "bf16", "scale": 64.0},
        # gradient of a short fine-tuning sequence, odd token count, a row length that is no multiple of a vector
        {"name": "embedding_grad_short", "op": "embedding_grad", "tokens": 509, "vocab": 4099, "dim": 1001, "grad": "f16", "type": "f32", "scale": 1.0},
        # a training batch of 4 x 4096 tokens, frequent words as in text, bf16 gradients into an fp32 master gradient
        {"name": "embedding_grad_batch", "op": "embedding_grad", "tokens": 16384, "vocab": 32000, "dim": 4096, "grad": "bf16", "type": "f32", "scale": 64.0},
        # a large training batch over a 128000-word vocabulary
        {"name": "embedding_grad_large", "op": "embedding_grad", "tokens": 65536, "vocab": 128000, "dim": 4096, "grad": "bf16", "type": "bf16", "scale": 1.0},
        # activations on their way into a product: one scale per row and 128 columns, ragged in both directions
        {"name": "quantize_rows", "op": "quantize", "rows": 1000, "cols": 5000, "block": 1, "across": False, "from": "bf16", "to": "e4m3"},
        # gradients for the weight-gradient product: groups run down the columns, result stored transposed
        {"name": "quantize_across", "op": "quantize", "rows": 16384, "cols": 8192, "block": 1, "across": True, "from": "bf16", "to": "e5m2"},
        # the logits of one token: every byte of a 32000 x 4096 head is read once
        {"name": "gemm_token", "op": "gemm", "form": "forward", "m": 1, "n": 32000, "k": 4096, "a": "e4m3", "b": "e4m3", "c": "f32", "act": False},
        # a serving batch of 48 sequences through one linear layer with bias and ReLU
        {"name": "gemm_step", "op": "gemm", "form": "forward", "m": 48, "n": 4096, "k": 4096, "a": "e4m3", "b": "e4m3", "c": "bf16", "act": True},
        # gradient of a layer's input, ragged: the weights are read along their other direction, no transposed copy
        {"name": "gemm_input_grad", "op": "gemm", "form": "input_grad", "m": 1000, "n": 4112, "k": 5000, "a": "e5m2", "b": "e4m3", "c": "bf16", "act": False},
        # forward product of a training batch
        {"name": "gemm_forward", "op": "gemm", "form": "forward", "m": 8192, "n": 8192, "k": 8192, "a": "e4m3", "b": "e4m3", "c": "bf16", "act": False},
        # weight gradient over 16384 tokens: both sides scaled along the tokens, fp32 result
        {"name": "gemm_weight_grad", "op": "gemm", "form": "weight_grad", "m": 4096, "n": 8192, "k": 16384, "a": "e5m2", "b": "e4m3", "c": "f32", "act": False},
    ]


def draw(rng):
    def size(lo, hi):
        v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return max(lo, min(hi, v if rng.random() < 0.5 or v < 64 else (v + 8) // 16 * 16))

    op = rng.choice(["embedding", "embedding_grad", "quantize", "gemm"])
    if op == "embedding":
        return {"op": op, "tokens": size(1, 32768), "vocab": size(1000, 128000), "dim": size(64, 4096),
                "type": rng.choice(["f32", "f16", "bf16"]), "scale": rng.choice([1.0, 0.125, 64.0])}
    if op == "embedding_grad":
        return {"op": op, "tokens": size(1, 65536), "vocab": size(1000, 128000), "dim": size(64, 4096), "grad": rng.choice(["f32", "bf16", "f16"]),
                "type": rng.choice(["f32", "bf16"]), "scale": rng.choice([1.0, 0.125, 64.0])}
    if op == "quantize":
        return {"op": op, "rows": size(1, 16384), "cols": size(64, 8192), "block": rng.choice([1, 1, 128]), "across": rng.random() < 0.5,
                "from": rng.choice(["f32", "bf16", "f16"]), "to": rng.choice(["e4m3", "e5m2"])}
    form = rng.choice(["forward", "forward", "input_grad", "weight_grad"])
    m = size(1, 8192) if form == "forward" else size(128, 8192)
    return {"op": op, "form": form, "m": m, "n": size(256, 8192), "k": size(256, 8192), "a": "e4m3" if form == "forward" else "e5m2", "b": "e4m3",
            "c": "f32" if form == "weight_grad" else rng.choice(["bf16", "f16", "f32"]), "act": form == "forward" and rng.random() < 0.5}


def _up(a, b):
    return -(-a // b)


def _quantised(x, kind, rows):
    """8-bit values and fp32 scales max / top of the groups of `rows` x 128 values of x: a checkpoint's or another kernel's output."""
    m, k = x.shape
    kb, mb = _up(k, 128), _up(m, rows)
    padded = torch.nn.functional.pad(x, (0, kb * 128 - k, 0, mb * rows - m)).view(mb, rows, kb, 128)
    s = padded.abs().amax(dim=(1, 3)).clamp_min(1e-30) / TOP[kind]
    q = (padded / s[:, None, :, None]).view(mb * rows, kb * 128)[:m, :k].contiguous().to(TYPES[kind])
    return q, s.contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 17)
    c = dict(case)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if c["op"] in ("embedding", "embedding_grad"):
        # word frequencies fall like one over the rank, as in text: the most frequent word is several percent of all tokens
        u = torch.rand(c["tokens"], device="cuda", generator=g, dtype=torch.float64)
        c["ids"] = (float(c["vocab"]) ** u - 1.0).long().clamp_(0, c["vocab"] - 1)
        t = TYPES[c["type"]]
        if c["op"] == "embedding":
            c["table"] = (randn(c["vocab"], c["dim"]) * 0.02).to(t)
            c["out"] = torch.empty(c["tokens"], c["dim"], device="cuda", dtype=t)
        else:
            c["grad_out"] = (randn(c["tokens"], c["dim"]) * 0.05).to(TYPES[c["grad"]])
            c["out"] = torch.empty(c["vocab"], c["dim"], device="cuda", dtype=t)
    elif c["op"] == "quantize":
        # activations and gradients: a common size for each row and column, a few columns far above the rest
        x = randn(c["rows"], c["cols"]) * torch.exp(randn(c["rows"], 1)) * torch.exp(2.0 * randn(1, c["cols"]).clamp_(-2.0, 2.0))
        c["x"] = (x * 0.05).to(TYPES[c["from"]])
        m, k = (c["cols"], c["rows"]) if c["across"] else (c["rows"], c["cols"])
        c["q"] = torch.empty(m, k, device="cuda", dtype=TYPES[c["to"]])
        c["s"] = torch.empty(_up(m, c["block"]), _up(k, 128), device="cuda")
    else:
        m, n, k = c["m"], c["n"], c["k"]
        c["A"], c["sa"] = _quantised(randn(m, k) * torch.exp(randn(m, 1)), c["a"], 1)
        if c["form"] == "input_grad":      # weights as they are stored, [contraction, n]: n contiguous
            c["B"], s = _quantised(torch.nn.functional.pad(randn(k, n) / k ** 0.5, (0, _up(n, 128) * 128 - n)), c["b"], 128)
            c["B"], c["sb"] = c["B"][:, :n].contiguous(), s
        else:                              # [n, contraction], handed over as its transposed view
            q, s = _quantised(randn(n, k) / k ** 0.5, c["b"], 128 if c["form"] == "forward" else 1)
            c["B"], c["sb"] = q.t(), s.t()
        c["bias"] = randn(n) if c["act"] else None
        c["C"] = torch.empty(m, n, device="cuda", dtype=TYPES[c["c"]])
    return c


def _spread(s, dim, count, block):
    """The scale of each row or column from the scales of the blocks of `block` of them."""
    return s if s.shape[dim] == count else s.repeat_interleave(block, dim=dim).narrow(dim, 0, count)


def _groups(x, block):
    m, k = x.shape
    mb, kb = _up(m, block), _up(k, 128)
    return torch.nn.functional.pad(x, (0, kb * 128 - k, 0, mb * block - m)).view(mb, block, kb, 128)


def _plain_quantize(s):
    x = s["x"].t() if s["across"] else s["x"]
    m, k = x.shape
    g = _groups(x.float(), s["block"])
    top = g.abs().amax(dim=(1, 3))
    # a logarithm next to a whole number may be off by its last bit, so the exponent is settled by comparing, in 64 bits
    e = torch.floor(torch.log2(top.double() / TOP[s["to"]]) + 0.5)
    e = e - 1 + (top > TOP[s["to"]] * torch.exp2(e - 1)).double() + (top > TOP[s["to"]] * torch.exp2(e)).double()
    scale = torch.exp2(torch.where(top > 0, e.clamp(-126, 127), torch.zeros_like(e)))
    q = (g.double() / scale[:, None, :, None]).float().reshape(g.shape[0] * g.shape[1], -1)[:m, :k]
    return q.to(TYPES[s["to"]]), scale.float()


def _plain_gemm(s):
    m, n, k = s["m"], s["n"], s["k"]
    a = s["A"].float() * _spread(_spread(s["sa"], 1, k, 128), 0, m, 128)
    b = s["B"].float() * _spread(_spread(s["sb"], 0, k, 128), 1, n, 128)
    c = a @ b
    if s["act"]:
        c = torch.clamp_min(c + s["bias"], 0.0)
    return c.to(TYPES[s["c"]])


def run(state):
    s = state
    if own:
        from accera_b200 import runtime as rt
        if s["op"] == "embedding":
            rt.embedding(s["table"], s["ids"], s["out"], scale=s["scale"])
            return s["out"]
        if s["op"] == "embedding_grad":
            rt.embedding_grad(s["grad_out"], s["ids"], s["out"], scale=s["scale"])
            return s["out"]
        if s["op"] == "quantize":
            rt.quantize_fp8(s["x"].t() if s["across"] else s["x"], s["q"], s["s"])
            return {"q": s["q"], "s": s["s"]}
        rt.gemm_fp8(s["A"], s["B"], s["C"], s["sa"], s["sb"], bias=s["bias"], beta=0.0, relu=s["act"])
        return s["C"]
    if s["op"] == "embedding":
        return (s["table"][s["ids"]].float() * s["scale"]).to(s["table"].dtype)
    if s["op"] == "embedding_grad":
        total = torch.zeros(s["vocab"], s["dim"], device="cuda").index_add_(0, s["ids"], s["grad_out"].float())
        return (total * s["scale"]).to(s["out"].dtype)
    if s["op"] == "quantize":
        q, scale = _plain_quantize(s)
        return {"q": q, "s": scale}
    return _plain_gemm(s)


def exact(case, seed):
    """What run() returns, from the definitions in 64 bits."""
    s = prepare(case, seed)
    if s["op"] == "embedding":
        return torch.index_select(s["table"].double(), 0, s["ids"]) * s["scale"]
    if s["op"] == "embedding_grad":
        # tokens ordered by word; a word's sum is a difference of two running sums, a few columns at a time
        order = torch.argsort(s["ids"], stable=True)
        words, counts = torch.unique_consecutive(s["ids"][order], return_counts=True)
        last = torch.cumsum(counts, 0) - 1
        out = torch.zeros(s["vocab"], s["dim"], device="cuda", dtype=torch.float64)
        for c0 in range(0, s["dim"], 512):
            sums = torch.cumsum(s["grad_out"][order, c0:c0 + 512].double(), 0)[last]
            out[words, c0:c0 + 512] = torch.diff(sums, dim=0, prepend=torch.zeros_like(sums[:1])) * s["scale"]
        return out
    if s["op"] == "quantize":
        x = (s["x"].t() if s["across"] else s["x"]).double()
        m, k = x.shape
        bits, low, top = (3, -6, 448.0) if s["to"] == "e4m3" else (2, -14, 57344.0)
        q = torch.empty_like(x)
        scales = torch.empty_like(s["s"], dtype=torch.float64)
        for b in range(_up(k, 128)):
            part = x[:, b * 128:(b + 1) * 128]
            amax = part.abs().amax(dim=1)
            if s["block"] != 1:
                amax = torch.stack([v.amax() for v in amax.split(s["block"])])
            mant, e = torch.frexp(amax)                                   # amax = mant * 2^e, mant in [0.5, 1)
            lead, top_e = math.frexp(top)
            e = torch.where(mant <= lead, e - top_e, e - top_e + 1)
            e = torch.where(amax > 0, e.clamp(-126, 127), torch.zeros_like(e))
            scales[:, b] = torch.ldexp(torch.ones_like(amax), e)
            y = part / (scales[:, b].repeat_interleave(s["block"])[:m, None])
            _, ey = torch.frexp(y)
            step = torch.ldexp(torch.ones_like(y), (ey - 1).clamp_min(low) - bits)
            q[:, b * 128:(b + 1) * 128] = torch.round(y / step) * step    # round() goes to even
        return {"q": q, "s": scales}
    m, n, k = s["m"], s["n"], s["k"]
    c = torch.zeros(m, n, device="cuda", dtype=torch.float64)
    for b in range(_up(k, 128)):
        part = s["A"][:, b * 128:(b + 1) * 128].double() @ s["B"][b * 128:(b + 1) * 128].double()
        sb = s["sb"][b].double()
        sb = sb if sb.numel() == n else sb.repeat_interleave(128)[:n]
        c += part * s["sa"][:, b, None].double() * sb
    if s["act"]:
        c = torch.relu(c + s["bias"].double())
    return c


def work(case):
    c = case
    size = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1, "e5m2": 1}
    if c["op"] == "embedding":
        n, d, e = c["tokens"], c["dim"], size[c["type"]]
        return {"bytes": n * 8 + min(n, c["vocab"]) * d * e + n * d * e, "flops": n * d}
    if c["op"] == "embedding_grad":
        n, d = c["tokens"], c["dim"]
        return {"bytes": n * 8 + n * d * size[c["grad"]] + c["vocab"] * d * size[c["type"]], "flops": n * d}
    if c["op"] == "quantize":
        m, k = (c["cols"], c["rows"]) if c["across"] else (c["rows"], c["cols"])
        return {"bytes": m * k * (size[c["from"]] + 1) + _up(m, c["block"]) * _up(k, 128) * 4, "flops": 3 * m * k}
    m, n, k = c["m"], c["n"], c["k"]
    nb = n if c["form"] == "weight_grad" else _up(n, 128)
    return {"bytes": m * k + n * k + 4 * _up(k, 128) * (m + nb) + m * n * size[c["c"]] + (4 * n if c["act"] else 0), "flops": 2 * m * n * k}
