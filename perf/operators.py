"""Cases that measure the 8-bit layer operators and the windowed attention.

The operators: rms_norm (root-mean-square norm with the residual's addition, its
output in the input's type or in e4m3 with a scale for each 128 columns),
quantize_e4m3 (rows in groups of 128 columns, or weights in 128 x 128 blocks),
linear_e4m3 (the product of what the two produce) and attention_window (sliding
window, first tokens that stay visible, grouped heads, a cache that is longer
than the queries).  `run` computes their plain forms, or calls the library's
kernels where `own` is set; `exact` gives the same results from the definitions
in 64 bits.
"""

import importlib.util
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

GROUP = 128
E4M3_MAX = 448.0
TINY = 2.0 ** -126  # smallest scale: a group of zeros is divided by it
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _package():
    """The package directory's name is no identifier: import it by its path."""
    name = "omni_tokenizer_b200"
    if name not in sys.modules:
        at = Path(__file__).resolve().parents[1] / "omni-tokenizer_b200"
        spec = importlib.util.spec_from_file_location(name, at / "__init__.py", submodule_search_locations=[str(at)])
        module = importlib.util.module_from_spec(spec)
        sys.modules[name] = module
        spec.loader.exec_module(module)
    return sys.modules[name]


# ------------------------------------------------------------------- cases
def listed():
    return [
        # One token's activations on the way to the next layer's product: latency.
        dict(name="norm_token", op="norm", rows=1, cols=4096, dtype="bf16", residual=True, quantize=True),
        # A long prompt's activations, a layer's norm in bandwidth.
        dict(name="norm_prompt", op="norm", rows=16384, cols=8192, dtype="bf16", residual=True, quantize=True),
        # What enters an audio encoder's second product: 16 segments of 1500 rows.
        dict(name="quant_audio", op="quant", rows=24000, cols=4096, dtype="bf16", block_rows=1),
        # A weight of the image encoder, laid out when it is loaded (4304 is no multiple of 128).
        dict(name="quant_weight", op="quant", rows=4304, cols=1152, dtype="f32", block_rows=128),
        # One token through one projection: the weight's bytes.
        dict(name="linear_token", op="linear", m=1, n=4096, k=4096, out="bf16", bias=False),
        # A small batch of tokens, odd sizes, the image encoder's feed-forward shape.
        dict(name="linear_batch", op="linear", m=61, n=4304, k=1152, out="f16", bias=True),
        # The audio encoder's first feed-forward product over 16 segments.
        dict(name="linear_audio", op="linear", m=24000, n=4096, k=1024, out="bf16", bias=True),
        # A long prompt through a wide projection: matrix throughput.
        dict(name="linear_prompt", op="linear", m=8192, n=8192, k=4096, out="bf16", bias=False),
        # One token of one sequence against its cache: latency.
        dict(name="attn_token", op="attn", batch=1, heads=16, kv_heads=2, q_len=1, kv_len=2048, dim=64, window=512,
             right=0, sinks=4, ragged=False, layout="tokens", dtype="bf16"),
        # A serving batch's next tokens against long caches of several lengths.
        dict(name="attn_tokens", op="attn", batch=64, heads=32, kv_heads=8, q_len=1, kv_len=16384, dim=128,
             window=4096, right=0, sinks=4, ragged=True, layout="heads", dtype="bf16"),
        # An audio batch of several lengths, local attention to both sides.
        dict(name="attn_audio", op="attn", batch=16, heads=16, kv_heads=16, q_len=1500, kv_len=1500, dim=64,
             window=257, right=256, sinks=1, ragged=True, layout="tokens", dtype="f16"),
        # A long prompt, causal.
        dict(name="attn_prompt", op="attn", batch=1, heads=32, kv_heads=8, q_len=8192, kv_len=8192, dim=128,
             window=1024, right=0, sinks=4, ragged=False, layout="heads", dtype="bf16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "quant", "linear", "attn"])
    if op == "norm":
        cols = _log_int(rng, 64, 8192)
        rows = _log_int(rng, 1, min(65536, 16384 * 8192 // cols))
        quantize = rng.random() < 0.6
        return dict(op=op, rows=rows, cols=cols, dtype=rng.choice(["bf16", "f16", "f32"]) if cols * rows < 2**25
                    else rng.choice(["bf16", "f16"]), residual=rng.random() < 0.7, quantize=quantize)
    if op == "quant":
        cols = _log_int(rng, 64, 8192)
        rows = _log_int(rng, 1, min(65536, 24000 * 4096 // cols))
        return dict(op=op, rows=rows, cols=cols, dtype=rng.choice(["bf16", "f16", "f32"]),
                    block_rows=rng.choice([1, 128]))
    if op == "linear":
        n, k = _log_int(rng, 64, 8192), _log_int(rng, 64, 8192)
        m = _log_int(rng, 1, min(32768, 8192 * 8192 * 4096 // (n * k)))
        return dict(op=op, m=m, n=n, k=k, out=rng.choice(["bf16", "f16"]), bias=rng.random() < 0.5)
    kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([32, 64, 72, 80, 96, 128])
    dtype, layout = rng.choice(["bf16", "f16"]), rng.choice(["heads", "tokens"])
    sinks = rng.choice([0, 1, 4, 5, 64, 130])
    window = rng.choice([0, 1]) * _log_int(rng, 1, 4096)
    if rng.random() < 0.5:  # next tokens against a cache
        q_len = rng.choice([1, 1, 1, 2, 4, 7])
        kv_len = _log_int(rng, 8, 16384)
        batch = _log_int(rng, 1, max(1, min(64, 64 * 8 * 4096 // (kv_heads * kv_len))))
        right = 0
    else:  # prompts and encoders
        kv_len = _log_int(rng, 9, 4096)
        q_len = kv_len if rng.random() < 0.6 else rng.randint(1, kv_len)
        batch = _log_int(rng, 1, max(1, min(32, 2**29 // (heads * q_len * kv_len))))
        right = rng.choice([0, 0, 1]) * rng.randint(1, kv_len)
    return dict(op="attn", batch=batch, heads=heads, kv_heads=kv_heads, q_len=q_len, kv_len=kv_len, dim=dim,
                window=window, right=right, sinks=sinks, ragged=rng.random() < 0.6, layout=layout, dtype=dtype)


# ------------------------------------------------------------------ inputs
def _groups(cols):
    return (cols + GROUP - 1) // GROUP


def _activations(rows, cols, dtype, gen, dev):
    """Activations with a few wide channels, as residual streams have them."""
    wide = torch.exp(1.2 * torch.randn(cols, generator=gen, device=dev))
    return (torch.randn(rows, cols, generator=gen, device=dev) * wide).to(dtype)


def _padded(q):
    """Rows of e4m3 whose pitch is a multiple of 16 bytes."""
    rows, cols = q.shape
    if cols % 16 == 0:
        return q
    wide = torch.zeros(rows, (cols + 15) // 16 * 16, dtype=torch.uint8, device=q.device).view(torch.float8_e4m3fn)
    wide[:, :cols].copy_(q)
    return wide[:, :cols]


def _lengths(case):
    """(keys held, queries) of each sequence, before the seed orders them."""
    b, kv, q = case["batch"], case["kv_len"], case["q_len"]
    if not case["ragged"]:
        return np.full(b, kv), np.full(b, q)
    held = np.linspace(kv, max(1, kv // 8), b).round().astype(np.int64)
    if q < kv and q <= 8:  # next tokens: as many for each sequence
        return np.maximum(held, min(q, kv)), np.full(b, q)
    return held, np.minimum(np.maximum(1, (held * q) // kv), held)


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    op = case["op"]
    if op == "norm":
        dt = DTYPES[case["dtype"]]
        x = _activations(case["rows"], case["cols"], dt, gen, dev)
        res = _activations(case["rows"], case["cols"], dt, gen, dev) if case["residual"] else None
        w = (1 + 0.1 * torch.randn(case["cols"], generator=gen, device=dev)).to(dt)
        return dict(case=case, x=x, residual=res, weight=w)
    if op == "quant":
        return dict(case=case, x=_activations(case["rows"], case["cols"], DTYPES[case["dtype"]], gen, dev))
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        a, a_scales = _plain_quantize(_activations(m, k, torch.float32, gen, dev), 1)
        w, w_scales = _plain_quantize(torch.randn(n, k, generator=gen, device=dev) / math.sqrt(k), 128)
        bias = torch.randn(n, generator=gen, device=dev).to(DTYPES[case["out"]]) if case["bias"] else None
        return dict(case=case, a=_padded(a), a_scales=a_scales, w=_padded(w), w_scales=w_scales, bias=bias)
    dt, b, d = DTYPES[case["dtype"]], case["batch"], case["dim"]

    def tensor(heads, tokens):
        if case["layout"] == "tokens":
            return torch.randn(b, tokens, heads, d, generator=gen, device=dev).to(dt).transpose(1, 2)
        return torch.randn(b, heads, tokens, d, generator=gen, device=dev).to(dt)

    q = tensor(case["heads"], case["q_len"])
    k, v = (tensor(case["kv_heads"], case["kv_len"]) for _ in range(2))
    out = tensor(case["heads"], case["q_len"])  # rows past a sequence's queries keep this
    order = np.random.RandomState(seed % (1 << 31)).permutation(b)
    held, queries = (torch.from_numpy(n[order].astype(np.int32)).to(dev) for n in _lengths(case))
    return dict(case=case, q=q, k=k, v=v, out=out, lengths=held, q_lengths=queries)


# ------------------------------------------------------------- plain forms
def _plain_quantize(x, block_rows):
    """e4m3 values and scales = max |x| / 448 of each group (block_rows x 128)."""
    rows, cols = x.shape
    padded = torch.zeros(-(-rows // block_rows) * block_rows, _groups(cols) * GROUP, device=x.device)
    padded[:rows, :cols] = x
    grouped = padded.view(-1, block_rows, _groups(cols), GROUP)
    scales = (grouped.abs().amax(dim=(1, 3)) / E4M3_MAX).clamp_min(TINY)
    q = (grouped / scales[:, None, :, None]).view(padded.shape)[:rows, :cols]
    return q.to(torch.float8_e4m3fn), scales


def _plain_norm(s):
    case, x = s["case"], s["x"]
    h = x.float()
    if case["residual"]:
        h = h + s["residual"].float()
    y = h * torch.rsqrt(h.square().mean(dim=1, keepdim=True) + 1e-6) * s["weight"].float()
    out = dict(zip(("q", "scales"), _plain_quantize(y, 1))) if case["quantize"] else {"y": y.to(x.dtype)}
    if case["residual"]:
        out["residual"] = h.to(x.dtype)
    return out


def _dequantized(q, scales, block_rows, dtype):
    rows, cols = q.shape
    wide = scales.to(dtype).repeat_interleave(block_rows, 0)[:rows].repeat_interleave(GROUP, 1)[:, :cols]
    return q.to(dtype) * wide


def _plain_linear(s):
    y = _dequantized(s["a"], s["a_scales"], 1, torch.float32) @ _dequantized(s["w"], s["w_scales"], 128, torch.float32).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(DTYPES[s["case"]["out"]])


def _visible(case, held, queries, device):
    """[batch, q_len, kv_len]: which keys a query sees.  Query i of a sequence of n
    keys and m queries stands at position p = n - m + i."""
    i = torch.arange(case["q_len"], device=device).view(1, -1, 1)
    key = torch.arange(case["kv_len"], device=device).view(1, 1, -1)
    held, queries = held.view(-1, 1, 1).long(), queries.view(-1, 1, 1).long()
    p = held - queries + i
    seen = (key < held) & (key <= p + case["right"])
    if case["window"] > 0:
        seen &= (key > p - case["window"]) | (key < case["sinks"])
    return seen


def _plain_attention(s):
    case, q, k, v = s["case"], s["q"], s["k"], s["v"]
    b, h, lq, d = q.shape
    kvh, lk = k.shape[1:3]
    scores = (q.float().reshape(b, kvh, (h // kvh) * lq, d) * d**-0.5) @ k.float().transpose(2, 3)
    scores = scores.view(b, h, lq, lk)
    seen = _visible(case, s["lengths"], s["q_lengths"], q.device)[:, None]
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(dim=3, keepdim=True).clamp_min(-3e38)
    weights = scores.sub_(top).exp_()
    total = weights.sum(dim=3, keepdim=True)
    y = (weights.view(b, kvh, (h // kvh) * lq, lk) @ v.float()).view(b, h, lq, d) / total.clamp_min(TINY)
    mine = (torch.arange(lq, device=q.device)[None] < s["q_lengths"][:, None])[:, None, :, None]
    return torch.where(mine, y.to(q.dtype), s["out"])


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        if op == "norm":
            return _plain_norm(state)
        if op == "quant":
            return dict(zip(("q", "scales"), _plain_quantize(state["x"].float(), case["block_rows"])))
        return _plain_linear(state) if op == "linear" else _plain_attention(state)
    ob = _package()
    if op == "norm":
        if case["quantize"]:
            q, scales, residual = ob.rms_norm_e4m3(state["x"], state["weight"], residual=state["residual"], eps=1e-6)
            out = {"q": q, "scales": scales}
        else:
            y, residual = ob.rms_norm(state["x"], state["weight"], residual=state["residual"], eps=1e-6)
            out = {"y": y}
        if case["residual"]:
            out["residual"] = residual
        return out
    if op == "quant":
        return dict(zip(("q", "scales"), ob.quantize_e4m3(state["x"], block_rows=case["block_rows"])))
    if op == "linear":
        return ob.linear_e4m3(state["a"], state["a_scales"], state["w"], state["w_scales"], bias=state["bias"],
                              out_dtype=DTYPES[case["out"]])
    return ob.attention_window(state["q"], state["k"], state["v"], window=case["window"], sinks=case["sinks"],
                               right=case["right"], lengths=state["lengths"], q_lengths=state["q_lengths"],
                               out=state["out"])


# --------------------------------------------------------------- the floor
def work(case):
    op = case["op"]
    size = {"bf16": 2, "f16": 2, "f32": 4}
    if op == "norm":
        n, e = case["rows"] * case["cols"], size[case["dtype"]]
        out = n + 4 * case["rows"] * _groups(case["cols"]) if case["quantize"] else n * e
        return {"bytes": n * e * (3 if case["residual"] else 1) + out + case["cols"] * e, "flops": 5 * n}
    if op == "quant":
        n = case["rows"] * case["cols"]
        scales = -(-case["rows"] // case["block_rows"]) * _groups(case["cols"])
        return {"bytes": n * size[case["dtype"]] + n + 4 * scales, "flops": 3 * n}
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        scales = (m + -(-n // 128)) * _groups(k)
        return {"bytes": m * k + n * k + 4 * scales + 2 * m * n + 2 * n * case["bias"], "flops": 2 * m * n * k}
    pairs = keys = rows = 0
    for n, m in zip(*_lengths(case)):
        p = np.arange(n - m, n)
        high = np.clip(p + case["right"] + 1, 0, n)
        low = np.clip(p - case["window"] + 1, 0, high) if case["window"] > 0 else np.zeros_like(high)
        pairs += int((high - low + np.minimum(case["sinks"], low)).sum())
        keys += int(high[-1] - low[0] + min(case["sinks"], low[0]))
        rows += int(m)
    d = case["dim"]
    return {"bytes": 2 * d * (2 * rows * case["heads"] + 2 * keys * case["kv_heads"]), "flops": 4 * d * pairs * case["heads"]}


# ------------------------------------------------------------- 64-bit forms
def _exact_quantize(y, block_rows):
    """Scale of each group and the e4m3 value nearest to y / scale, group after group of columns."""
    rows, cols = y.shape
    scales = torch.empty(-(-rows // block_rows), _groups(cols), dtype=torch.float64, device=y.device)
    q = torch.empty_like(y)
    whole = rows // block_rows * block_rows
    for g in range(_groups(cols)):
        part = y[:, g * GROUP:(g + 1) * GROUP]
        top = part.abs().amax(dim=1)
        tops = top[:whole].view(-1, block_rows).amax(dim=1)
        if whole < rows:
            tops = torch.cat([tops, top[whole:].amax().view(1)])
        scales[:, g] = torch.clamp(tops / E4M3_MAX, min=TINY)
        q[:, g * GROUP:(g + 1) * GROUP] = part / scales[:, g].repeat_interleave(block_rows)[:rows, None]
    # Nearest e4m3 (ties to even): 3 mantissa bits above 2^-6, steps of 2^-9 below.
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0**-6))) - 3)
    return torch.round(q / step) * step, scales


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        h = s["x"].double()
        if case["residual"]:
            h = h + s["residual"].double()
        y = h / torch.sqrt((h * h).sum(dim=1, keepdim=True) / case["cols"] + 1e-6)
        y = y * s["weight"].double()
        out = dict(zip(("q", "scales"), _exact_quantize(y, 1))) if case["quantize"] else {"y": y}
        if case["residual"]:
            out["residual"] = h
        return out
    if op == "quant":
        return dict(zip(("q", "scales"), _exact_quantize(s["x"].double(), case["block_rows"])))
    if op == "linear":
        m, n = case["m"], case["n"]
        y = torch.zeros(m, n, dtype=torch.float64, device="cuda")
        rows = torch.arange(n, device="cuda") // 128
        for g in range(_groups(case["k"])):
            cut = slice(g * GROUP, (g + 1) * GROUP)
            part = s["a"][:, cut].double() @ s["w"][:, cut].double().t()
            y += part * s["a_scales"][:, g, None].double() * s["w_scales"][rows, g].double()
        return y if s["bias"] is None else y + s["bias"].double()
    y = s["out"].double()
    group = case["heads"] // case["kv_heads"]
    held, queries = s["lengths"].tolist(), s["q_lengths"].tolist()
    for b in range(case["batch"]):
        n, m = held[b], queries[b]
        p = torch.arange(n - m, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")[None]
        hidden = key > p + case["right"]
        if case["window"] > 0:
            hidden |= (key <= p - case["window"]) & (key >= case["sinks"])
        for h in range(case["kv_heads"]):
            k, v = s["k"][b, h, :n].double(), s["v"][b, h, :n].double()
            for j in range(h * group, (h + 1) * group):
                e = torch.einsum("id,jd->ij", s["q"][b, j, :m].double(), k) / math.sqrt(case["dim"])
                e = torch.softmax(e.masked_fill(hidden, -math.inf), dim=1)
                y[b, j, :m] = torch.nan_to_num(e) @ v
    return y
