"""The operators of a decoder layer held in 8 and 4 bits, as cases that can be timed.

Weights and activations of the linear layers are 8-bit floating point (e4m3) with
one f32 scale for each block of 128; keys and values lie in a cache of 4-bit codes
with an f16 scale and lowest value for each group of 32.  A decoder layer quantizes
its activations, multiplies them by its weights, rotates queries and keys, appends
keys and values to the cache and attends over it.

Kinds of cases and the ranges they stand for
  quantize   f32, f16 or bf16 to e4m3 with a scale for every 1 x 128 block
             (activations: 1 .. 8192 rows) or every 128 x 128 block (weights);
             rows of 128 .. 11008 elements
  product    a [M, K] times b [N, K] transposed, both e4m3 with their scales:
             1 .. 4096 rows, K and N from 256 to 11008, with and without bias
  rotary     rotary positions on queries or keys: both layouts of pairs, all of a
             head or a part of it, tables for long contexts, near and far positions
  append     1 .. 2048 new tokens of 1 .. 64 sequences into their pages
  attention  queries of 1 .. 2048 new tokens against caches of 1 .. 131072
             tokens: many query heads for one of keys, pages in any order, causal
             or not, windows, sequences padded on the left
"""
import math
import os
import sys

import torch

own = False

BLOCK, GROUP = 128, 32
F16_MAX, F8_MAX, TINY = 65504.0, 448.0, 2.0 ** -126
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}

# What a drawn case may cost at most: the largest listed ones.
MAX_ELEMENTS = 4096 * 11008
MAX_MACS = 2048 * 4096 * 11008
MAX_ROTARY = 4096 * 32 * 128
MAX_APPEND = 2048 * 8 * 128
MAX_CACHE = 131072 * 8 * 128
MAX_SCORES = 2048 * 4096 * 32 * 128


def listed():
    return [
        # One token's activations on their way into a layer: a launch.
        {"name": "quantize_token", "kind": "quantize", "M": 1, "K": 4096, "rows": 1, "dtype": "bf16"},
        # The activations of a prompt of 4096 tokens between the feed-forward layers.
        {"name": "quantize_prompt", "kind": "quantize", "M": 4096, "K": 11008, "rows": 1, "dtype": "f32"},
        # A 7B-sized model generating one token: a feed-forward layer, bound by its weights.
        {"name": "product_decode", "kind": "product", "M": 1, "K": 4096, "N": 11008, "dtype": "bf16", "bias": False, "act": 0},
        # The same model reading a prompt of 2048 tokens.
        {"name": "product_prefill", "kind": "product", "M": 2048, "K": 4096, "N": 11008, "dtype": "bf16", "bias": False, "act": 0},
        # Sizes that are multiples of nothing: the last block of 128 holds 9.
        {"name": "product_ragged", "kind": "product", "M": 4099, "K": 777, "N": 1001, "dtype": "f32", "bias": True, "act": 2},
        # Queries of sixteen sequences that generate a token each.
        {"name": "rotary_decode", "kind": "rotary", "batch": 16, "seq": 1, "heads": 32, "dim": 128, "rot": 128, "pairs": "half",
         "layout": "bshd", "far": 30000, "dtype": "bf16"},
        # Queries of a prompt, neighbouring pairs, half of the head rotated.
        {"name": "rotary_prompt", "kind": "rotary", "batch": 2, "seq": 2048, "heads": 32, "dim": 128, "rot": 64, "pairs": "interleaved",
         "layout": "bhsd", "far": 2048, "dtype": "f32"},
        # Keys and values of sixteen sequences that generate, in pages of 16 tokens.
        {"name": "append_decode", "kind": "append", "batch": 16, "seq": 1, "heads": 8, "dim": 128, "past": 4000, "page": 16,
         "layout": "bshd", "ragged": False, "dtype": "bf16"},
        # Prompts of up to 512 tokens, each of its own length.
        {"name": "append_prompts", "kind": "append", "batch": 4, "seq": 512, "heads": 8, "dim": 128, "past": 100, "page": 64,
         "layout": "bshd", "ragged": True, "dtype": "f16"},
        # One sequence far into a long context: work that has to be split over its keys.
        {"name": "attend_long", "kind": "attention", "batch": 1, "seq": 1, "heads": 32, "kv": 8, "dim": 128, "past": 131071, "page": 0,
         "layout": "bshd", "causal": True, "window": 0, "padded": False, "dtype": "bf16"},
        # Thirty-two sequences of different lengths, in pages.
        {"name": "attend_batch", "kind": "attention", "batch": 32, "seq": 1, "heads": 32, "kv": 8, "dim": 128, "past": 4000, "page": 16,
         "layout": "bshd", "causal": True, "window": 0, "padded": False, "dtype": "f16"},
        # The second half of a prompt of 4096 tokens, the first half in the cache already.
        {"name": "attend_prompt", "kind": "attention", "batch": 1, "seq": 2048, "heads": 32, "kv": 8, "dim": 128, "past": 2048, "page": 64,
         "layout": "bshd", "causal": True, "window": 0, "padded": False, "dtype": "bf16"},
    ]


# ---------------------------------------------------------------------------
# drawn cases
# ---------------------------------------------------------------------------
def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A layer's width: mostly a multiple of 64 as models have them, sometimes of
    16, sometimes any number."""
    n, r = _log(rng, lo, hi), rng.random()
    step = 64 if r < 0.5 else 16 if r < 0.7 else 1
    return max(lo, n // step * step)


def draw(rng):
    kind = rng.choice(["quantize", "product", "product", "product", "rotary", "append", "attention", "attention", "attention"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    while True:
        if kind == "quantize":
            c = {"kind": kind, "M": _log(rng, 1, 8192), "K": _width(rng, 128, 11008), "rows": rng.choice([1, 1, 128]), "dtype": dtype}
            if c["M"] * c["K"] <= MAX_ELEMENTS:
                return c
        elif kind == "product":
            c = {"kind": kind, "M": _log(rng, 1, 4096), "K": _width(rng, 256, 11008), "N": _width(rng, 256, 11008), "dtype": dtype,
                 "bias": rng.random() < 0.5, "act": rng.choice([0, 0, 1, 2])}
            if c["M"] * c["K"] * c["N"] <= MAX_MACS:
                return c
        elif kind == "rotary":
            dim = rng.choice([64, 80, 96, 128, 192, 256])
            c = {"kind": kind, "batch": _log(rng, 1, 64), "seq": _log(rng, 1, 4096), "heads": _log(rng, 1, 64), "dim": dim,
                 "rot": rng.choice([dim, dim, dim // 2]), "pairs": rng.choice(["half", "interleaved"]),
                 "layout": rng.choice(["bshd", "bhsd"]), "far": _log(rng, 1, 120000), "dtype": dtype}
            if c["batch"] * c["seq"] * c["heads"] * dim <= MAX_ROTARY:
                return c
        elif kind == "append":
            c = {"kind": kind, "batch": _log(rng, 1, 64), "seq": _log(rng, 1, 2048), "heads": _log(rng, 1, 16),
                 "dim": rng.choice([64, 64, 96, 128, 128, 256]), "past": _log(rng, 1, 8192), "page": rng.choice([0, 16, 16, 64, 48]),
                 "layout": rng.choice(["bshd", "bhsd"]), "ragged": rng.random() < 0.5, "dtype": dtype}
            if c["batch"] * c["seq"] * c["heads"] * c["dim"] <= MAX_APPEND and c["batch"] * c["past"] * c["heads"] * c["dim"] <= MAX_CACHE:
                return c
        else:
            kv = _log(rng, 1, 16)
            c = {"kind": kind, "batch": _log(rng, 1, 64), "seq": 1 if rng.random() < 0.6 else _log(rng, 1, 2048),
                 "heads": kv * rng.choice([1, 2, 4, 4, 7, 8]), "kv": kv, "dim": rng.choice([64, 64, 96, 128, 128, 128, 256]),
                 "past": _log(rng, 1, 131071), "page": rng.choice([0, 16, 16, 64, 48]), "layout": rng.choice(["bshd", "bhsd"]),
                 "causal": rng.random() < 0.8, "window": rng.choice([0, 0, 0, 500]), "padded": rng.random() < 0.25, "dtype": dtype}
            length = c["past"] + c["seq"]
            if (c["batch"] * length * kv * c["dim"] <= MAX_CACHE and c["batch"] * c["seq"] * length * c["heads"] * c["dim"] <= MAX_SCORES
                    and c["batch"] * c["seq"] * length * c["heads"] <= MAX_SCORES // 128):
                return c


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _pad(x, dim, step):
    """x with zeros behind it in `dim`, to a multiple of `step`."""
    n = -x.shape[dim] % step
    shape = list(x.shape)
    shape[dim] = n
    return torch.cat([x, x.new_zeros(shape)], dim) if n else x


def _quantize8(x, rows):
    """e4m3 values and f32 scales of x [M, K] in blocks of rows x 128."""
    M, K = x.shape
    x = x.float()
    blocks = _pad(_pad(x, 0, rows), 1, BLOCK).unflatten(1, (-1, BLOCK)).unflatten(0, (-1, rows))
    scale = (blocks.abs().amax((1, 3)) / F8_MAX).clamp_min(TINY)
    y = (blocks / scale[:, None, :, None]).clamp(-F8_MAX, F8_MAX)
    return y.flatten(0, 1).flatten(1, 2)[:M, :K].to(torch.float8_e4m3fn), scale


def _spread(values, scale, rows):
    """f32 values of e4m3 ones [M, K] with a scale for each block of rows x 128."""
    M, K = values.shape
    s = scale.repeat_interleave(rows, 0)[:M] if rows > 1 else scale
    return values.float() * s.repeat_interleave(BLOCK, 1)[:, :K]


def _activate(y, act):
    return y.clamp_min(0) if act == 1 else 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5))) if act == 2 else y


def _rotate(x, cos, sin, rot, interleaved):
    """x [B, H, S, D]; cos, sin [B, S, rot / 2]."""
    cos, sin, t = cos[:, None], sin[:, None], x[..., :rot]
    a, b = (t[..., 0::2], t[..., 1::2]) if interleaved else (t[..., :rot // 2], t[..., rot // 2:])
    p, q = a * cos - b * sin, b * cos + a * sin
    t = torch.stack([p, q], -1).flatten(-2) if interleaved else torch.cat([p, q], -1)
    return torch.cat([t, x[..., rot:]], -1)


def _quantize4(x):
    """Codes [.., D / 2] and (scale, lowest) [.., D / 32, 2] of x [.., D] in f32.

    Byte n * G + g of a row holds elements 32 g + 2 n (low half) and 32 g + 2 n + 1."""
    g = x.clamp(-F16_MAX, F16_MAX).unflatten(-1, (-1, GROUP))
    low = g.amin(-1, keepdim=True).half()
    scale = ((g.amax(-1, keepdim=True) - low.float()) / 15).clamp_min(0).half()
    c = ((g - low.float()) / scale.float()).round().clamp(0, 15)
    c = torch.where(scale > 0, c, 0).to(torch.uint8).unflatten(-1, (GROUP // 2, 2))
    return (c[..., 0] | c[..., 1] << 4).transpose(-1, -2).flatten(-2), torch.cat([scale, low], -1)


def _spread4(codes, pairs):
    """f32 values [.., D] of codes and (scale, lowest)."""
    c = codes.unflatten(-1, (GROUP // 2, -1)).transpose(-1, -2)
    c = torch.stack([c & 15, c >> 4], -1).flatten(-2).float()
    return (c * pairs[..., :1].float() + pairs[..., 1:].float()).flatten(-2)


def _gather(pages, table):
    """[B, H, tokens, ..] of the pages [pages, H, size, ..] of each sequence."""
    return pages[table.long()].transpose(1, 2).flatten(2, 3)


def _attend(s, q, k, v):
    """q [B, H, S, D] against k, v [B, KV, L, D], all f32, under the masks of s."""
    (B, H, S, D), (KV, L) = q.shape, k.shape[1:3]
    keys = torch.arange(L, device=q.device)
    at = s.past[:, None].long() + torch.arange(S, device=q.device)
    last = at if s.case["causal"] else (s.past.long() + S - 1)[:, None].expand(B, S)
    seen = keys <= last[..., None]
    if s.case["window"]:
        seen = seen & (keys > at[..., None] - s.case["window"])
    if s.starts is not None:
        seen = seen & (keys >= s.starts[:, None, None])
    seen = seen[:, None, None]  # [B, 1, 1, S, L]
    q = q.view(B, KV, H // KV, S, D).flatten(2, 3)
    p = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(B, KV, H // KV, S, L) / math.sqrt(D)
    p = p.masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(torch.isinf(top), 0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v).view(B, KV, H // KV, S, D)
    return (o / torch.where(total > 0, total, 1)).flatten(1, 2)


# ---------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------
class State:
    """The tensors of a case; `call`: the framework's calls, bound to them once."""

    def __init__(self, case, seed):
        self.case, self.call = case, None
        self.rng = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, shape, sigma=1.0):
        return torch.randn(shape, device="cuda", generator=self.rng).mul_(sigma)

    def whole(self, lo, hi, shape):
        return torch.randint(lo, hi + 1, shape, device="cuda", generator=self.rng, dtype=torch.int32)

    def activations(self, shape):
        """Normal values, some channels (the last dimension's) much larger than the rest."""
        x = self.normal(shape)
        return x.mul_(1 + 15 * (torch.rand(shape[-1:], device="cuda", generator=self.rng) < 0.01))

    def heads(self, x):
        """x, laid out [B, H, S, D], in the case's layout and type."""
        x = x.to(TYPES[self.case["dtype"]])
        return x.transpose(1, 2).flatten(2).contiguous() if self.case["layout"] == "bshd" else x.contiguous()

    def pages(self, capacity):
        """The page table of caches that hold `capacity` tokens, and the pages' number and size."""
        B, size = self.case["batch"], self.case["page"]
        if not size:
            return None, B, capacity
        each = -(-capacity // size)
        order = torch.randperm(B * each, device="cuda", generator=self.rng)
        return order.view(B, each).to(torch.int32), B * each, size

    def cache(self, heads, capacity):
        """Codes and scales of keys and values, every place filled."""
        D = self.case["dim"]
        self.table, count, size = self.pages(capacity)
        self.k_codes, self.k_scales = _quantize4(self.activations((count, heads, size, D)))
        self.v_codes, self.v_scales = _quantize4(self.normal((count, heads, size, D)))

    def lengths(self):
        """Tokens that the cache of each sequence holds before the call."""
        B, past = self.case["batch"], self.case["past"]
        return self.whole(past // 2, past, (B,)) if B > 1 else torch.full((B,), past, dtype=torch.int32, device="cuda")

    def places(self):
        """The page table, also where each sequence has one page."""
        if self.table is not None:
            return self.table
        return torch.arange(self.case["batch"], device="cuda", dtype=torch.int32)[:, None]


def _tables(far, rot, base=10000.0, stretch=4.0):
    """cos and sin of positions 0 .. far, linearly scaled for a context `stretch` times as long."""
    rate = base ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot) / stretch
    angle = torch.arange(far + 1, device="cuda", dtype=torch.float64)[:, None] * rate
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    s, kind = State(case, seed), case["kind"]
    dtype = TYPES[case["dtype"]]
    if kind == "quantize":
        M, K, rows = case["M"], case["K"], case["rows"]
        s.x = s.activations((M, K)).to(dtype)
        s.y = torch.empty((M, K), dtype=torch.float8_e4m3fn, device="cuda")
        s.scale = torch.empty((-(-M // rows), -(-K // BLOCK)), device="cuda")
    elif kind == "product":
        M, K, N = case["M"], case["K"], case["N"]
        s.a, s.a_scale = _quantize8(s.activations((M, K)), 1)
        s.b, s.b_scale = _quantize8(s.normal((N, K), 0.02), BLOCK)
        s.a, s.b = s.a.contiguous(), s.b.contiguous()
        s.bias = s.normal((N,), 0.1) if case["bias"] else None
        s.y = torch.empty((M, N), dtype=dtype, device="cuda")
    elif kind == "rotary":
        B, S = case["batch"], case["seq"]
        s.x = s.heads(s.normal((B, case["heads"], S, case["dim"])))
        s.y = torch.empty_like(s.x)
        s.cos, s.sin = _tables(case["far"] + S, case["rot"])
        s.at = (s.whole(0, case["far"], (B, 1)) + torch.arange(S, device="cuda")).long()
    elif kind == "append":
        B, S, H, D = case["batch"], case["seq"], case["heads"], case["dim"]
        s.cache(H, case["past"] + S)
        s.k, s.v = (s.heads(s.activations((B, H, S, D))) for _ in range(2))
        s.past = s.lengths()
        s.counts = s.whole(0, S, (B,)) if case["ragged"] else None
    elif kind == "attention":
        B, S, D = case["batch"], case["seq"], case["dim"]
        s.cache(case["kv"], case["past"] + S)
        s.q = s.heads(s.normal((B, case["heads"], S, D)))
        s.y = torch.empty_like(s.q)
        s.past = s.lengths()
        # padding on the left; at times it is as long as the sequence, and rows see nothing
        s.starts = s.whole(0, max(1, case["past"] // 2 + S // 4), (B,)) if case["padded"] else None
    else:
        raise ValueError(kind)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _split(x, case):
    """[B, H, S, D] of a tensor in the case's layout."""
    return x.unflatten(2, (-1, case["dim"])).transpose(1, 2) if case["layout"] == "bshd" else x


def _plain(s):
    case, kind = s.case, s.case["kind"]
    if kind == "quantize":
        y, scale = _quantize8(s.x, case["rows"])
        return {"y": y, "scale": scale}
    if kind == "product":
        y = torch.matmul(_spread(s.a, s.a_scale, 1), _spread(s.b, s.b_scale, BLOCK).t())
        if s.bias is not None:
            y += s.bias
        return {"y": _activate(y, case["act"]).to(s.y.dtype)}
    if kind == "rotary":
        y = _rotate(_split(s.x, case).float(), s.cos[s.at], s.sin[s.at], case["rot"], case["pairs"] == "interleaved")
        return {"y": s.heads(y)}
    if kind == "append":
        B, S, size = case["batch"], case["seq"], s.k_codes.shape[2]
        i = torch.arange(S, device="cuda")
        at = s.past[:, None].long() + i
        page, slot = s.places().long().gather(1, at // size), at % size
        new = (i < s.counts[:, None] if s.counts is not None else torch.ones_like(at, dtype=torch.bool))[..., None, None]
        for x, codes, pairs in ((s.k, s.k_codes, s.k_scales), (s.v, s.v_codes, s.v_scales)):
            c, p = _quantize4(_split(x, case).transpose(1, 2).float())
            codes[page, :, slot] = torch.where(new, c, codes[page, :, slot])
            pairs[page, :, slot] = torch.where(new[..., None], p, pairs[page, :, slot])
        return {"k_codes": s.k_codes, "k_scales": s.k_scales, "v_codes": s.v_codes, "v_scales": s.v_scales}
    k = _spread4(_gather(s.k_codes, s.places()), _gather(s.k_scales, s.places()))
    v = _spread4(_gather(s.v_codes, s.places()), _gather(s.v_scales, s.places()))
    return {"y": s.heads(_attend(s, _split(s.q, case).float(), k, v))}


def _bind(s):
    """The framework's call of a case on the tensors of its state, and what it gives."""
    sys.path.insert(0, os.path.join(os.getcwd(), "onnx-mlir_amd"))
    import om_mi355x as om

    kinds = {torch.float32: "float32", torch.int32: "int32", torch.int64: "int64", torch.uint8: "uint8", torch.float16: "float16",
             torch.bfloat16: om.bfloat16, torch.float8_e4m3fn: om.float8_e4m3fn}

    def t(x):
        return None if x is None else om.DeviceArray.wrap(x.data_ptr(), tuple(x.shape), kinds[x.dtype], owner=x)

    case, kind = s.case, s.case["kind"]
    if kind == "quantize":
        call = om.PreparedCall("om_mi355x_DynamicQuantizeBlocks", t(s.y), t(s.scale), t(s.x), case["rows"])
        return call, {"y": s.y, "scale": s.scale}
    if kind == "product":
        call = om.PreparedCall("om_mi355x_MatMulBlocks", t(s.y), t(s.a), t(s.a_scale), t(s.b), t(s.b_scale), t(s.bias), case["act"])
        return call, {"y": s.y}
    if kind == "rotary":
        call = om.PreparedCall("om_mi355x_RotaryEmbedding", t(s.y), t(s.x), t(s.cos), t(s.sin), t(s.at),
                               int(case["pairs"] == "interleaved"), case["heads"], case["rot"])
        return call, {"y": s.y}
    caches = [t(s.k_codes), t(s.k_scales), t(s.v_codes), t(s.v_scales)]
    if kind == "append":
        call = om.PreparedCall("om_mi355x_CacheAppend4", *caches, t(s.k), t(s.v), t(s.table), t(s.past), t(s.counts))
        return call, {"k_codes": s.k_codes, "k_scales": s.k_scales, "v_codes": s.v_codes, "v_scales": s.v_scales}
    call = om.PreparedCall("om_mi355x_CacheAttention4", t(s.y), t(s.q), *caches, t(s.table), t(s.past), None, t(s.starts), None,
                           int(case["causal"]), case["window"])
    return call, {"y": s.y}


def run(state):
    if not own:
        return _plain(state)
    if state.call is None:
        state.call, state.out = _bind(state)
    state.call()
    return state.out


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind, size = case["kind"], {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
    if kind == "quantize":
        n = case["M"] * case["K"]
        return {"bytes": n * (size + 1) + 4 * -(-case["M"] // case["rows"]) * -(-case["K"] // BLOCK), "flops": 3.0 * n}
    if kind == "product":
        M, K, N = case["M"], case["K"], case["N"]
        blocks = -(-K // BLOCK)
        scales = 4 * blocks * (M + -(-N // BLOCK)) + (4 * N if case["bias"] else 0)
        return {"bytes": M * K + N * K + scales + size * M * N, "flops": 2.0 * M * N * K}
    if kind == "rotary":
        n = case["batch"] * case["seq"] * case["heads"]
        tables = case["batch"] * case["seq"] * (8 + 8 * (case["rot"] // 2))
        return {"bytes": 2 * n * case["dim"] * size + tables, "flops": 3.0 * n * case["rot"]}
    row = case["dim"] // 2 + case["dim"] // GROUP * 4  # a token's codes and scales in one head
    if kind == "append":
        n = case["batch"] * case["seq"] * case["heads"] * (0.5 if case["ragged"] else 1)
        return {"bytes": 2 * n * (case["dim"] * size + row), "flops": 8.0 * n * case["dim"]}
    B, S, past = case["batch"], case["seq"], case["past"] if case["batch"] == 1 else 0.75 * case["past"]
    reach = min(past + S, case["window"] + S) if case["window"] else past + S
    keys = past + S / 2 if case["causal"] else past + S
    keys = min(keys, case["window"]) if case["window"] else keys
    return {"bytes": 2 * B * case["heads"] * S * case["dim"] * size + 2 * B * reach * case["kv"] * row,
            "flops": 4.0 * B * S * keys * case["heads"] * case["dim"]}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_scales(scale, rows, M, K):
    i, j = torch.arange(M, device=scale.device) // rows, torch.arange(K, device=scale.device) // BLOCK
    return scale.double()[i[:, None], j[None]]


def _exact_cache(codes, pairs):
    """[.., D] in 64 bits: element d is the half d % 2 of byte (d % 32 // 2) G + d // 32."""
    G = pairs.shape[-2]
    d = torch.arange(G * GROUP, device=codes.device)
    byte = codes[..., d % GROUP // 2 * G + d // GROUP].to(torch.int64)
    return torch.where(d % 2 == 1, byte // 16, byte % 16).double() * pairs[..., d // GROUP, 0].double() + pairs[..., d // GROUP, 1].double()


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "quantize":
        M, K, rows = case["M"], case["K"], case["rows"]
        x = s.x.double()
        i, j = torch.arange(M, device=x.device) // rows, torch.arange(K, device=x.device) // BLOCK
        flat = (i[:, None] * s.scale.shape[1] + j).flatten()
        top = torch.zeros(s.scale.numel(), dtype=torch.float64, device=x.device).scatter_reduce_(0, flat, x.abs().flatten(), "amax")
        scale = (top / F8_MAX).clamp_min(TINY)
        v = x / scale[flat].view(M, K)
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
        return {"y": torch.clamp(torch.round(v / step) * step, -F8_MAX, F8_MAX), "scale": scale.view_as(s.scale)}
    if kind == "product":
        M, K, N = case["M"], case["K"], case["N"]
        a = s.a.double() * _exact_scales(s.a_scale, 1, M, K)
        y = a @ (s.b.double() * _exact_scales(s.b_scale, BLOCK, N, K)).T
        y = y + (s.bias.double() if s.bias is not None else 0)
        return {"y": torch.maximum(y, torch.zeros_like(y)) if case["act"] == 1 else y * torch.special.ndtr(y) if case["act"] == 2 else y}
    if kind == "rotary":
        x, rot = _split(s.x, case).double(), case["rot"]
        turn = torch.complex(s.cos.double(), s.sin.double())[s.at][:, None]
        half = torch.arange(rot // 2, device=x.device)
        first, second = (2 * half, 2 * half + 1) if case["pairs"] == "interleaved" else (half, half + rot // 2)
        z = torch.complex(x[..., first], x[..., second]) * turn
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return {"y": y.transpose(1, 2).flatten(2) if case["layout"] == "bshd" else y}
    if kind == "append":  # (the codes are whole numbers: they round what 32 bits give)
        out = {"k_codes": None, "v_codes": None}
        for name, x, pairs in (("k_scales", s.k, s.k_scales), ("v_scales", s.v, s.v_scales)):
            x, pairs = _split(x, case).double(), pairs.double()
            for b in range(case["batch"]):
                for i in range(case["seq"] if s.counts is None else int(s.counts[b])):
                    page, slot = divmod(int(s.past[b]) + i, pairs.shape[2])
                    rows = x[b, :, i].unflatten(-1, (-1, GROUP))
                    low = rows.min(-1).values.half().double()
                    pairs[s.places()[b, page], :, slot] = torch.stack([(rows.max(-1).values - low).clamp(min=0) / 15, low], -1)
            out[name] = pairs
        return out if case["batch"] * case["seq"] <= 4096 else None
    B, S, H, D = case["batch"], case["seq"], case["heads"], case["dim"]
    q, table = _split(s.q, case).double(), s.places().tolist()
    past = s.past.tolist()
    y = torch.zeros((B, H, S, D), dtype=torch.float64, device=q.device)
    for b in range(B):
        for h in range(H):
            rows = [_exact_cache(c[table[b], h * case["kv"] // H].flatten(0, 1), p[table[b], h * case["kv"] // H].flatten(0, 1))
                    for c, p in ((s.k_codes, s.k_scales), (s.v_codes, s.v_scales))]
            key, i = torch.arange(rows[0].shape[0], device=q.device)[None], torch.arange(S, device=q.device)[:, None]
            seen = key <= past[b] + (i if case["causal"] else S - 1)
            seen &= (key > past[b] + i - case["window"]) if case["window"] else True
            seen &= (key >= s.starts[b]) if s.starts is not None else True
            score = torch.where(seen, q[b, h] @ rows[0].T / math.sqrt(D), -math.inf)
            y[b, h] = torch.nan_to_num(torch.softmax(score, -1)) @ rows[1]
    return {"y": y.transpose(1, 2).flatten(2) if case["layout"] == "bshd" else y}
