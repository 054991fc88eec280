"""Cases that measure rotary positions and the 4-bit key/value cache.

The operators: rotary (positions of one or more axes turned into q and k, or out of
their gradients), cache_write_e2m1 and cache_read_e2m1 (a cache of e2m1 values with a
scale for each 32 columns, in pages or in one piece) and attention_window_e2m1
(attention of a sequence's last queries over such a cache).  `run` computes their plain
forms, or calls the library's kernels where `own` is set; `exact` gives the same results
from the definitions in 64 bits.

A cache is bytes [pages, kv_heads, page].  A page holds blocks of 16 tokens, one after the
other; a block, with D the head dimension rounded up to a multiple of 32 and G = D / 32:
  keys    8 D bytes: a token's D values in their order, two in a byte, the first one low;
  values  8 D bytes: of each 16 columns and lane (g, c) of a warp one word, its bytes
          columns g and g + 8 of tokens (2c, 2c + 1), then of tokens (2c + 8, 2c + 9), the
          even token low; a lane's words lie 4 together (2 where D is no multiple of 64);
  scales  of the keys 32 G bytes, f16 [token % 8, group, token / 8];
  scales  of the values 32 G bytes, f16 [group, (token % 8) / 2, token / 8, token % 2].
"""

import importlib.util
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

GROUP, BLOCK = 32, 16
SMALLEST, LARGEST = 2.0**-14, 10752.0  # of a scale
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
POSITIONS = {"i32": torch.int32, "i64": torch.int64, "f32": torch.float32}


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
        # One new token far into a sequence: latency.
        dict(name="rotary_token", op="rotary", batch=1, heads=32, kv_heads=8, tokens=1, dim=128, pairs=64, axes=1,
             layout="tokens", adjacent=False, inverse=False, positions="i32", dtype="bf16"),
        # A long prompt of images and text, time, height and width.
        dict(name="rotary_prompt", op="rotary", batch=1, heads=32, kv_heads=8, tokens=8192, dim=128, pairs=64, axes=3,
             layout="tokens", adjacent=False, inverse=False, positions="i64", dtype="bf16"),
        # An image encoder's gradients of q and k on their way back, height and width.
        dict(name="rotary_images", op="rotary", batch=32, heads=16, kv_heads=16, tokens=729, dim=72, pairs=36, axes=2,
             layout="heads", adjacent=True, inverse=True, positions="f32", dtype="f16"),
        # A serving batch's new keys and values on their way into the pages.
        dict(name="write_tokens", op="write", batch=64, kv_heads=8, q_len=1, kv_len=4096, dim=128, page=64,
             ragged=True, layout="tokens", dtype="bf16"),
        # A long prompt's keys and values, one piece of memory for the sequence.
        dict(name="write_prompt", op="write", batch=1, kv_heads=8, q_len=8191, kv_len=8192, dim=128, page=0,
             ragged=False, layout="tokens", dtype="bf16"),
        # A cached prefix on its way into another use.
        dict(name="read_prefix", op="read", batch=1, kv_heads=8, q_len=16384, kv_len=16384, dim=128, page=256,
             ragged=False, layout="heads", dtype="bf16"),
        # The last tokens of several sequences, an odd head dimension.
        dict(name="read_batch", op="read", batch=9, kv_heads=4, q_len=157, kv_len=2000, dim=80, page=16,
             ragged=True, layout="tokens", dtype="f16"),
        # One token of one sequence against its cache: latency.
        dict(name="attn_token", op="attn", batch=1, heads=16, kv_heads=2, q_len=1, kv_len=2048, dim=64, page=0,
             window=0, right=0, sinks=0, ragged=False, layout="tokens", dtype="bf16"),
        # A serving batch's next tokens against long caches of several lengths.
        dict(name="attn_tokens", op="attn", batch=64, heads=32, kv_heads=8, q_len=1, kv_len=16384, dim=128, page=64,
             window=0, right=0, sinks=0, ragged=True, layout="tokens", dtype="bf16"),
        # One sequence with a very long cache: work split over its length.
        dict(name="attn_long", op="attn", batch=1, heads=32, kv_heads=8, q_len=1, kv_len=131072, dim=128, page=128,
             window=0, right=0, sinks=0, ragged=False, layout="heads", dtype="f16"),
        # Several drafted tokens a sequence, a window and first tokens that stay visible.
        dict(name="attn_draft", op="attn", batch=16, heads=32, kv_heads=8, q_len=5, kv_len=8192, dim=128, page=32,
             window=4096, right=0, sinks=4, ragged=True, layout="tokens", dtype="bf16"),
        # The second half of a long prompt, over the first half's cache and its own.
        dict(name="attn_prompt", op="attn", batch=1, heads=32, kv_heads=8, q_len=4096, kv_len=8192, dim=128, page=64,
             window=0, right=0, sinks=0, ragged=False, layout="tokens", dtype="bf16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    op = rng.choice(["rotary", "write", "read", "attn", "attn"])
    layout, dtype = rng.choice(["tokens", "heads"]), rng.choice(["bf16", "f16"])
    dim = rng.choice([32, 64, 72, 80, 96, 128])
    if op == "rotary":
        heads = rng.choice([1, 4, 16, 32, 40])
        kv_heads = rng.choice([0, 1, heads])
        pairs = rng.choice([dim // 2, dim // 2, dim // 4, rng.randint(1, dim // 2)])
        batch = rng.choice([1, 1, 2, 7, 32])
        tokens = _log_int(rng, 1, 2**23 // (batch * (heads + kv_heads) * 32))
        return dict(op=op, batch=batch, heads=heads, kv_heads=kv_heads, tokens=tokens, dim=dim, pairs=pairs,
                    axes=rng.choice([1, 2, 3, 4]), layout=layout, adjacent=rng.random() < 0.5,
                    inverse=rng.random() < 0.5, positions=rng.choice(["i32", "i64", "f32"]),
                    dtype=rng.choice(["bf16", "f16", "f32"]) if tokens < 2000 else dtype)
    kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
    page = rng.choice([0, 16, 32, 48, 64, 128, 256])
    if op in ("write", "read"):
        kv_len = _log_int(rng, 16, 16384)
        batch = _log_int(rng, 1, max(1, min(64, 8 * 16384 // (kv_heads * kv_len))))
        q_len = rng.choice([1, rng.randint(1, kv_len), _log_int(rng, 1, kv_len), kv_len])
        return dict(op=op, batch=batch, kv_heads=kv_heads, q_len=q_len, kv_len=kv_len, dim=dim, page=page,
                    ragged=rng.random() < 0.6, layout=layout, dtype=dtype)
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    sinks = rng.choice([0, 0, 1, 4, 5, 64, 130])
    window = rng.choice([0, 1]) * _log_int(rng, 1, 4096)
    right = 0
    if rng.random() < 0.65:  # next tokens against a cache
        q_len = rng.choice([1, 1, 1, 2, 4, 7])
        kv_len = _log_int(rng, 16, 65536)
        batch = _log_int(rng, 1, max(1, min(64, 64 * 8 * 8192 // (kv_heads * kv_len))))
    else:  # prompts
        kv_len = _log_int(rng, 24, 8192)
        q_len = kv_len if rng.random() < 0.4 else rng.randint(1, kv_len)
        batch = _log_int(rng, 1, max(1, min(32, 2**29 // (heads * q_len * kv_len))))
        right = rng.choice([0, 0, 1]) * rng.randint(1, kv_len)
    return dict(op="attn", batch=batch, heads=heads, kv_heads=kv_heads, q_len=q_len, kv_len=kv_len, dim=dim, page=page,
                window=window, right=right, sinks=sinks, ragged=rng.random() < 0.6, layout=layout, dtype=dtype)


# ------------------------------------------------------------------ inputs
def _axes(case):
    """Axis of each pair: one run of pairs for each axis, as even as they go."""
    return [i * case["axes"] // case["pairs"] for i in range(case["pairs"])]


def _lengths(case):
    """(tokens held, last ones of them that a call is about) of each sequence, before the seed orders them."""
    b, kv, q = case["batch"], case["kv_len"], case["q_len"]
    if not case["ragged"]:
        return np.full(b, kv), np.full(b, q)
    held = np.linspace(kv, max(1, kv // 8), b).round().astype(np.int64)
    if q < kv and q <= 8:  # next tokens: as many for each sequence
        return np.maximum(held, min(q, kv)), np.full(b, q)
    return held, np.minimum(np.maximum(1, (held * q) // kv), held)


def _pages(case):
    """(tokens of a page, pages of a sequence, pages of the cache)."""
    page = case["page"] or -(-case["kv_len"] // BLOCK) * BLOCK
    each = -(-case["kv_len"] // page)
    return page, each, each * case["batch"]


def _sizes(case):
    wide = -(-case["dim"] // GROUP) * GROUP
    return wide, wide // GROUP, 4 if wide % 64 == 0 else 2


def _quantized(x):
    """Codes of 0 to 7, signs and scales [..., groups] of the columns of x, a multiple of 32."""
    parts = x.float().unflatten(-1, (-1, GROUP))
    top = parts.abs().amax(dim=-1)
    ratio = top / torch.full_like(top, 6.0)  # a division: a product with 1/6 misses the middle of two scales
    unit = torch.exp2(torch.frexp(ratio)[1].float() - 6)  # six significant bits
    scales = (torch.round(ratio / unit) * unit).clamp(SMALLEST, LARGEST)
    q = (parts.abs() / scales[..., None]).clamp_max(6.0)
    step = torch.where(q < 2, 0.5, torch.where(q < 4, 1.0, 2.0))
    q = (torch.round(q / step) * step).clamp_max(6.0)
    codes = torch.where(q < 2, q * 2, torch.where(q < 4, q + 2, q / 2 + 4))
    return codes.to(torch.uint8), parts < 0, scales


def _packed(k, v):
    """Blocks [..., bytes] of keys and values [..., 16, D], D a multiple of 32."""
    wide = k.shape[-1]
    words = 4 if wide % 64 == 0 else 2
    lead = k.shape[:-2]
    codes, signs, k_scales = _quantized(k)
    nibbles = (codes + 8 * signs.to(torch.uint8)).flatten(-2).unflatten(-1, (-1, 2))
    k_bytes = (nibbles[..., 0] + 16 * nibbles[..., 1]).flatten(-2)
    codes, signs, v_scales = _quantized(v)
    n = len(lead)
    # tokens (half, c, parity) x columns (vector, word, upper, g) -> [vector, g, c, word, half, upper, parity]
    nibbles = (codes + 8 * signs.to(torch.uint8)).flatten(-2).reshape(*lead, 2, 4, 2, wide // 16 // words, words, 2, 8)
    nibbles = nibbles.permute(*range(n), n + 3, n + 6, n + 1, n + 4, n, n + 5, n + 2)
    v_bytes = (nibbles[..., 0] + 16 * nibbles[..., 1]).flatten(n)
    k_scales = k_scales.half().unflatten(-2, (2, 8)).permute(*range(n), n + 1, n + 2, n).flatten(n)
    v_scales = v_scales.half().unflatten(-2, (2, 4, 2)).permute(*range(n), n + 3, n + 1, n, n + 2).flatten(n)
    return torch.cat([k_bytes, v_bytes, k_scales.view(torch.uint8), v_scales.view(torch.uint8)], dim=-1)


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    op, dt, b, d = case["op"], DTYPES[case["dtype"]], case["batch"], case["dim"]

    def tensor(heads, tokens, spread=False):
        x = torch.randn(b, tokens, heads, d, generator=gen, device=dev)
        if spread:  # some channels of a head are wider than others
            x = x * torch.exp(0.8 * torch.randn(1, 1, heads, d, generator=gen, device=dev))
        x = x.to(dt)
        return x.transpose(1, 2) if case["layout"] == "tokens" else x.transpose(1, 2).contiguous()

    if op == "rotary":
        t, a = case["tokens"], case["axes"]
        rows = torch.arange(t, device=dev)
        start = torch.randint(0, 100000, (1, b, 1), generator=gen, device=dev)
        if a == 1:
            positions = start + rows.view(1, 1, t)
        else:  # time stands still within an image, height and width run over it
            side = max(1, math.isqrt(t))
            grid = torch.stack([rows // (side * side), rows // side % side, rows % side, rows][-a if a < 4 else 0:])
            positions = start + grid[:a].view(a, 1, t)
        run = torch.arange(case["pairs"], device=dev, dtype=torch.float64)
        return dict(case=case, q=tensor(case["heads"], t), k=tensor(case["kv_heads"], t) if case["kv_heads"] else None,
                    positions=positions.to(POSITIONS[case["positions"]]).contiguous(), axes=bytes(_axes(case)),
                    frequencies=(10000.0 ** (-run / case["pairs"])).float())

    page, each, pages = _pages(case)
    wide, groups, _ = _sizes(case)
    order = np.random.RandomState(seed % (1 << 31)).permutation(b)
    held, count = (torch.from_numpy(n[order].astype(np.int32)).to(dev) for n in _lengths(case))
    table = None
    if case["page"]:
        table = torch.randperm(pages, generator=gen, device=dev).to(torch.int32).view(b, each)
    cache = torch.empty(pages, case["kv_heads"], page // BLOCK, 16 * wide + 64 * groups, dtype=torch.uint8, device=dev)
    per = max(1, 2**26 // cache[0].numel())
    for at in range(0, pages, per):  # what stands in it: keys and values of the head dimension, zeros behind
        shape = (*cache[at:at + per].shape[:3], BLOCK, wide)
        k, v = (torch.randn(shape, generator=gen, device=dev, dtype=torch.bfloat16) for _ in range(2))
        k[..., d:], v[..., d:] = 0, 0
        cache[at:at + per] = _packed(k, v)
    state = dict(case=case, cache=cache.flatten(2), table=table, lengths=held, counts=count)
    if op == "attn":
        state.update(q=tensor(case["heads"], case["q_len"]), out=tensor(case["heads"], case["q_len"]))
    else:  # rows past a sequence's last ones keep what out holds
        state.update(out=(tensor(case["kv_heads"], case["q_len"]), tensor(case["kv_heads"], case["q_len"])))
    if op == "write":
        state.update(k=tensor(case["kv_heads"], case["q_len"], True), v=tensor(case["kv_heads"], case["q_len"], True))
    return state


# ------------------------------------------------------------- plain forms
def _turned(x, cos, sin, case):
    """x [batch, heads, tokens, D] with its pairs turned by angles [batch, tokens, pairs]."""
    x, n = x.float(), case["pairs"]
    head, tail = x[..., :2 * n], x[..., 2 * n:]
    x0, x1 = (head[..., ::2], head[..., 1::2]) if case["adjacent"] else (head[..., :n], head[..., n:])
    cos, sin = cos[:, None], sin[:, None]
    y0, y1 = x0 * cos - x1 * sin, x1 * cos + x0 * sin
    head = torch.stack([y0, y1], dim=-1).flatten(-2) if case["adjacent"] else torch.cat([y0, y1], dim=-1)
    return torch.cat([head, tail], dim=-1).to(DTYPES[case["dtype"]])


def _plain_rotary(s):
    case = s["case"]
    of_pair = s["positions"].double()[torch.tensor(list(s["axes"]), device="cuda")]  # [pairs, batch, tokens]
    angle = of_pair.permute(1, 2, 0) * s["frequencies"].double()  # 32 bits lose the angles of far positions
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    sin = -sin if case["inverse"] else sin
    return [_turned(x, cos, sin, case) for x in (s["q"], s["k"]) if x is not None]


def _values(scales, codes, signs):
    table = torch.tensor(E2M1, device="cuda")
    return ((table[codes.int()] * (1 - 2 * signs.float())) * scales[..., None]).flatten(-2)


def _plain_stored(x, dim):
    """What the cache stands for once x is in it."""
    codes, signs, scales = _quantized(torch.nn.functional.pad(x, (0, -dim % GROUP)))
    return _values(scales, codes, signs)[..., :dim]


def _unpacked(s):
    """Keys and values [batch, kv_heads, capacity, D] that the cache holds, in 32 bits."""
    case, cache = s["case"], s["cache"]
    wide, groups, words = _sizes(case)
    blocks = cache.unflatten(2, (-1, 16 * wide + 64 * groups))  # [pages, kv_heads, blocks, bytes]
    two = torch.tensor([[x, y] for y in E2M1 + [-e for e in E2M1] for x in E2M1 + [-e for e in E2M1]], device="cuda")
    if s["table"] is None:
        blocks = blocks[:case["batch"], None]
    else:
        blocks = blocks[s["table"].long()]  # [batch, pages of a sequence, kv_heads, blocks, bytes]
    blocks = blocks.transpose(1, 2).flatten(2, 3)
    at = np.cumsum([0, 8 * wide, 8 * wide, 32 * groups, 32 * groups])
    k, v, k_scales, v_scales = (blocks[..., i:j] for i, j in zip(at[:-1], at[1:]))
    k_scales = k_scales.contiguous().view(torch.float16).float().unflatten(-1, (8, groups, 2)).permute(0, 1, 2, 5, 3, 4)
    v_scales = v_scales.contiguous().view(torch.float16).float().unflatten(-1, (groups, 4, 2, 2))
    v_scales = v_scales.permute(0, 1, 2, 5, 4, 6, 3)  # [.., half, c, parity, group]
    k = two[k.int()].flatten(-2).unflatten(-1, (BLOCK, groups, GROUP))
    k = (k * k_scales.flatten(3, 4)[..., None]).flatten(2, 3).flatten(-2)
    v = two[v.int()].unflatten(-2, (-1, 8, 4, words, 2, 2))  # [.., vector, g, c, word, half, upper, parity]
    v = v.permute(0, 1, 2, 7, 5, 9, 3, 6, 8, 4)  # [.., half, c, parity, vector, word, upper, g]
    v = v.flatten(6).flatten(3, 5).unflatten(-1, (groups, GROUP))
    v = (v * v_scales.flatten(3, 5)[..., None]).flatten(2, 3).flatten(-2)
    return k[..., :case["dim"]], v[..., :case["dim"]]


def _last(x, s):
    """The last counts[b] of the lengths[b] tokens of x [batch, kv_heads, capacity, D], from row 0 on."""
    first = (s["lengths"] - s["counts"]).long()[:, None, None, None]
    row = torch.arange(s["case"]["q_len"], device="cuda")[None, None, :, None]
    return torch.gather(x, 2, (first + row).clamp_max(x.shape[2] - 1).expand(-1, x.shape[1], -1, x.shape[3]))


def _mine(s):
    return (torch.arange(s["case"]["q_len"], device="cuda")[None] < s["counts"][:, None])[:, None, :, None]


def _visible(case, held, queries, keys):
    """[batch, q_len, keys]: which keys a query sees.  Query i of a sequence of n
    keys and m queries stands at position p = n - m + i."""
    i = torch.arange(case["q_len"], device="cuda").view(1, -1, 1)
    key = torch.arange(keys, device="cuda").view(1, 1, -1)
    held, queries = held.view(-1, 1, 1).long(), queries.view(-1, 1, 1).long()
    p = held - queries + i
    seen = (key < held) & (key <= p + case["right"])
    if case["window"] > 0:
        seen &= (key > p - case["window"]) | (key < case["sinks"])
    return seen


def _plain_attention(s):
    case, q = s["case"], s["q"]
    k, v = _unpacked(s)
    b, h, lq, d = q.shape
    kvh, lk = k.shape[1:3]
    scores = (q.float().reshape(b, kvh, (h // kvh) * lq, d) * d**-0.5) @ k.transpose(2, 3)
    scores = scores.view(b, h, lq, lk)
    seen = _visible(case, s["lengths"], s["counts"], lk)[:, None]
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(dim=3, keepdim=True).clamp_min(-3e38)
    weights = scores.sub_(top).exp_()
    total = weights.sum(dim=3, keepdim=True)
    y = (weights.view(b, kvh, (h // kvh) * lq, lk) @ v).view(b, h, lq, d) / total.clamp_min(2.0**-126)
    return torch.where(_mine(s), y.to(q.dtype), s["out"])


def run(state):
    case, s = state["case"], state
    op = case["op"]
    if not own:
        if op == "rotary":
            return _plain_rotary(s)
        if op == "attn":
            return _plain_attention(s)
        rows = [_plain_stored(x, case["dim"]) for x in (s["k"], s["v"])] if op == "write" else [
            _last(x, s) for x in _unpacked(s)]
        return [torch.where(_mine(s), x.to(o.dtype), o) for x, o in zip(rows, s["out"])]
    ob = _package()
    if op == "rotary":
        return [x for x in ob.rotary(s["q"], s["k"], s["positions"], s["frequencies"], axes=s["axes"],
                                     adjacent=case["adjacent"], inverse=case["inverse"]) if x is not None]
    if op == "attn":
        return ob.attention_window_e2m1(s["q"], s["cache"], s["lengths"], q_lengths=s["counts"], table=s["table"],
                                        window=case["window"], sinks=case["sinks"], right=case["right"], out=s["out"])
    if op == "write":
        ob.cache_write_e2m1(s["k"], s["v"], s["cache"], s["lengths"], q_lengths=s["counts"], table=s["table"])
    return list(ob.cache_read_e2m1(s["cache"], case["dim"], s["lengths"], q_lengths=s["counts"], table=s["table"],
                                   out=s["out"]))


# --------------------------------------------------------------- the floor
def work(case):
    op, e, d = case["op"], {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]], case["dim"]
    if op == "rotary":
        n = case["batch"] * (case["heads"] + case["kv_heads"]) * case["tokens"]
        ids = case["axes"] * case["batch"] * case["tokens"] * (8 if case["positions"] == "i64" else 4)
        return {"bytes": 2 * e * n * d + ids + 4 * case["pairs"], "flops": 6 * n * case["pairs"]}
    row = d / 2 + 2 * -(-d // GROUP)  # bytes of a token's keys, or values, in the cache
    held, count = _lengths(case)
    if op in ("read", "write"):
        rows = int(count.sum()) * case["kv_heads"] * 2
        moved = {"read": row + e * d, "write": e * d + row + e * d}[op]
        return {"bytes": rows * moved, "flops": rows * d * (1 if op == "read" else 4)}
    pairs = keys = rows = 0
    for n, m in zip(held, count):
        p = np.arange(n - m, n)
        high = np.clip(p + case["right"] + 1, 0, n)
        low = np.clip(p - case["window"] + 1, 0, high) if case["window"] > 0 else np.zeros_like(high)
        pairs += int((high - low + np.minimum(case["sinks"], low)).sum())
        keys += int(high[-1] - low[0] + min(case["sinks"], low[0]))
        rows += int(m)
    return {"bytes": 2 * row * keys * case["kv_heads"] + 2 * e * d * rows * case["heads"],
            "flops": 4 * d * pairs * case["heads"]}


# ------------------------------------------------------------- 64-bit forms
def _exact_value(x):
    """The nearest value of a group's e2m1 multiples (to the even code in the middle), x [rows, D]."""
    out = torch.empty_like(x)
    values = torch.tensor(E2M1, dtype=torch.float64, device="cuda")
    for at in range(0, x.shape[1], GROUP):
        part = x[:, at:at + GROUP]
        top = part.abs().amax(dim=1)
        # Twice the scale's last place is a power of two: compare 6 * (s + half a step) with top, which is exact.
        size = torch.exp2(torch.floor(torch.log2((top / 6).clamp_min(1e-30))) - 5)
        low = torch.floor(top / 6 / size)
        low = torch.where(6 * (low + 1) * size <= top, low + 1, torch.where(6 * low * size > top, low - 1, low))
        rest = top - 6 * low * size  # of a step of 6 * size
        up = (rest > 3 * size) | ((rest == 3 * size) & (low % 2 == 1))
        scale = ((low + up) * size).clamp(SMALLEST, LARGEST)[:, None]
        got = torch.zeros_like(part)
        for code in range(1, 8):  # past the middle between two values, or on it where the upper code is even
            middle = (values[code - 1] + values[code]) / 2 * scale
            past = (part.abs() >= middle) if code % 2 == 0 else (part.abs() > middle)
            got = torch.where(past, values[code] * scale, got)
        out[:, at:at + GROUP] = torch.sign(part) * got
    return out


def _exact_cached(s, b, h, tokens):
    """Keys and values [tokens, D] of a sequence's head, token after token as the layout says."""
    case = s["case"]
    wide, groups, words = _sizes(case)
    page = _pages(case)[0]
    at = torch.arange(tokens, device="cuda")
    which = torch.full_like(at, b) if s["table"] is None else s["table"][b].long()[at // page]
    size = 16 * wide + 64 * groups
    flat, base = s["cache"].reshape(-1), (which * case["kv_heads"] + h) * (page // BLOCK * size)
    base = (base + at % page // BLOCK * size)[:, None]
    t, col = (at % BLOCK)[:, None], torch.arange(case["dim"], device="cuda")[None]
    values = torch.tensor(E2M1 + [-x for x in E2M1], dtype=torch.float64, device="cuda")

    def half(offset):
        return (flat[offset].int() + 256 * flat[offset + 1].int()).to(torch.int16).view(torch.float16).double()

    key = (flat[base + t * (wide // 2) + col // 2].int() >> (col % 2 * 4)) & 15
    keys = values[key] * half(base + 16 * wide + 2 * ((t % 8 * groups + col // GROUP) * 2 + t // 8))
    tile, g, c = col // 16, col % 8, t % 8 // 2
    place = tile // words * 128 * words + (4 * g + c) * 4 * words + tile % words * 4 + t // 8 * 2 + col % 16 // 8
    value = (flat[base + 8 * wide + place].int() >> (t % 2 * 4)) & 15
    scale = col // GROUP * 16 + c * 4 + t // 8 * 2 + t % 2
    return keys, values[value] * half(base + 16 * wide + 32 * groups + 2 * scale)


def exact(case, seed):
    s = prepare(case, seed)
    op, d = case["op"], case["dim"]
    if op == "rotary":
        got = []
        position = s["positions"].double()
        for x in (s["q"], s["k"]):
            if x is None:
                continue
            y = x.double()
            for i, axis in enumerate(_axes(case)):
                turn = torch.polar(torch.ones_like(position[axis]), position[axis] * s["frequencies"][i].double())[:, None]
                turn = turn.conj() if case["inverse"] else turn
                i0, i1 = (2 * i, 2 * i + 1) if case["adjacent"] else (i, i + case["pairs"])
                z = torch.complex(x[..., i0].double(), x[..., i1].double()) * turn
                y[..., i0], y[..., i1] = z.real, z.imag
            got.append(y)
        return got
    held, count = s["lengths"].tolist(), s["counts"].tolist()
    if op != "attn":
        got = [x.double() for x in s["out"]]
        for b in range(case["batch"]):
            n, m = held[b], count[b]
            for h in range(case["kv_heads"]):
                if op == "write":
                    rows = [_exact_value(x[b, h, :m].double()) for x in (s["k"], s["v"])]
                else:
                    rows = [x[n - m:] for x in _exact_cached(s, b, h, n)]
                got[0][b, h, :m], got[1][b, h, :m] = rows
        return got
    y = s["out"].double()
    group = case["heads"] // case["kv_heads"]
    for b in range(case["batch"]):
        n, m = held[b], count[b]
        p = torch.arange(n - m, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")[None]
        hidden = key > p + case["right"]
        if case["window"] > 0:
            hidden |= (key <= p - case["window"]) & (key >= case["sinks"])
        for h in range(case["kv_heads"]):
            k, v = _exact_cached(s, b, h, n)
            for j in range(h * group, (h + 1) * group):
                e = torch.einsum("id,jd->ij", s["q"][b, j, :m].double(), k) / math.sqrt(d)
                e = torch.softmax(e.masked_fill(hidden, -math.inf), dim=1)
                y[b, j, :m] = torch.nan_to_num(e) @ v
    return y
