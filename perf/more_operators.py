"""The key-value cache and the attention that reads it, as cases that can be timed: what a program that serves a model asks of this
library between a layer's fused Q/K/V projection and its output projection, and when it forks or compacts sequences.

The cache is one layer's: k and v [pages][kv_heads][page_tokens][head_dim] in f16 or in e4m3 (with a scale per head); a sequence's
tokens lie in the pages that its row of the table names.  A call's rows are the last tokens of their sequences, packed.

op          a pass is
append      fused rows [q | k | v] of new tokens: q and k rotated by their tokens' positions (a table of cosines and sines), q stored
            as f16 rows, k and v into their pages
decode      one new token a sequence: out = softmax(scale * q K^T) V over the whole sequence, or its last `window` tokens; query
            heads share key-value heads in groups
prompt      the same for several new tokens a sequence, each of which sees the tokens up to itself
copy        whole pages of every layer to other pages: what forking a sequence (its last page) and compacting a pool do
"""
import math

import torch

own = False

E4M3_MAX = 448.0


def listed():
    return [
        # one user's next token in a small model, f32 rows as the 4-bit projections give them: a launch and little else
        {"name": "append_1_14x64", "op": "append", "seqs": 1, "rows": 1, "longest": 777, "q_heads": 14, "kv_heads": 2, "dim": 64,
         "page": 16, "cache": "f16", "x": "f32", "rotary": 64, "interleaved": False},
        # a few prompts of a 7B model, packed, into an 8-bit cache
        {"name": "append_2048_28x128_e4m3", "op": "append", "seqs": 5, "rows": 2048, "longest": 1100, "q_heads": 28, "kv_heads": 4, "dim": 128,
         "page": 64, "cache": "e4m3", "x": "f16", "rotary": 128, "interleaved": False},
        # one user's next token in a small model, some hundred tokens into the conversation
        {"name": "decode_1_777_14x64", "op": "decode", "seqs": 1, "longest": 777, "q_heads": 14, "kv_heads": 2, "dim": 64, "page": 16,
         "cache": "f16", "window": 0},
        # and at the end of a long document in a 7B model: one row, and all of the card has to read
        {"name": "decode_1_32768_28x128", "op": "decode", "seqs": 1, "longest": 32768, "q_heads": 28, "kv_heads": 4, "dim": 128, "page": 16,
         "cache": "f16", "window": 0},
        # a batch of users in the midst of conversations of very different lengths
        {"name": "decode_32_8192_28x128", "op": "decode", "seqs": 32, "longest": 8192, "q_heads": 28, "kv_heads": 4, "dim": 128, "page": 16,
         "cache": "f16", "window": 0},
        # a larger one on a model whose heads share nothing, with an 8-bit cache
        {"name": "decode_48_4096_32x128_e4m3", "op": "decode", "seqs": 48, "longest": 4096, "q_heads": 32, "kv_heads": 32, "dim": 128, "page": 64,
         "cache": "e4m3", "window": 0},
        # a short question to a small model
        {"name": "prompt_37_14x64", "op": "prompt", "seqs": 1, "rows": 37, "longest": 37, "context": 0, "q_heads": 14, "kv_heads": 2, "dim": 64,
         "page": 16, "cache": "f16", "window": 0},
        # prompts of several users, packed
        {"name": "prompt_2048_in_7_28x128", "op": "prompt", "seqs": 7, "rows": 2048, "longest": 700, "context": 0, "q_heads": 28, "kv_heads": 4, "dim": 128,
         "page": 16, "cache": "f16", "window": 0},
        # a long document in one piece
        {"name": "prompt_8192_28x128", "op": "prompt", "seqs": 1, "rows": 8192, "longest": 8192, "context": 0, "q_heads": 28, "kv_heads": 4, "dim": 128,
         "page": 64, "cache": "f16", "window": 0},
        # the next piece of two long documents, of which an 8-bit cache holds the beginning; wide heads that look back a thousand tokens
        {"name": "prompt_1500_after_5000_16x256_e4m3", "op": "prompt", "seqs": 2, "rows": 1500, "longest": 800, "context": 5000, "q_heads": 16,
         "kv_heads": 8, "dim": 256, "page": 32, "cache": "e4m3", "window": 1024},
        # a sequence forked: its last page, in every layer
        {"name": "copy_1_of_28_layers", "op": "copy", "pairs": 1, "layers": 28, "kv_heads": 4, "dim": 128, "page": 16, "cache": "f16"},
        # a pool compacted
        {"name": "copy_500_of_28_layers", "op": "copy", "pairs": 500, "layers": 28, "kv_heads": 4, "dim": 128, "page": 16, "cache": "f16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prompt", "prompt", "copy"])
    dim = rng.choice([64, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 5, 8, 32])
    group = rng.choice([1, 2, 3, 4, 7, 8]) if kv < 32 else 1
    c = {"op": op, "page": rng.choice([16, 32, 64, 128]), "cache": rng.choice(["f16", "f16", "e4m3"]), "kv_heads": kv, "dim": dim}
    if op == "copy":
        c["layers"] = rng.choice([1, 24, 28, 32])
        page_bytes = c["page"] * kv * dim
        c["pairs"] = min(_log_int(rng, 1, 500), max(1, 28 * 500 * 16 * 4 * 128 // (c["layers"] * page_bytes)))
        return c
    c["q_heads"] = kv * group
    c["seqs"] = _log_int(rng, 1, 48)
    if op == "append":
        most = 2048 * 36 * 128 // ((c["q_heads"] + 2 * kv) * dim)
        c["rows"] = max(c["seqs"], min(_log_int(rng, 1, 2048), most))
        c["seqs"] = min(c["seqs"], c["rows"], most)
        c["rows"] = min(c["rows"], max(most, c["seqs"]))
        c["longest"] = min(8192, max(c["rows"], _log_int(rng, 1, 8192)))
        c["rotary"] = rng.choice([dim, dim, dim // 2])
        c["interleaved"] = rng.random() < 0.3
        c["x"] = rng.choice(["f32", "f16"])
        return c
    c["window"] = rng.choice([0, 0, 0, _log_int(rng, 1, 2048)])
    if op == "decode":
        # tokens x heads x bytes of the largest listed one
        most = 24 * 4096 * 32 * 128 // (kv * dim * (1 if c["cache"] == "e4m3" else 2))
        c["longest"] = _log_int(rng, 1, 32768)
        while sum(_lengths(c)[1]) > most or c["seqs"] * c["longest"] > 8 * most:
            c["longest"] = c["longest"] * 3 // 4
        return c
    # rows x keys x heads x values of the longest prompt
    c["rows"] = _log_int(rng, 1, 8192)
    c["seqs"] = min(c["seqs"], c["rows"], 16)
    c["context"] = rng.choice([0, 0, _log_int(rng, 1, 16384)]) // c["seqs"]
    while c["rows"] > 1 and c["rows"] * (c["rows"] / 2 + c["context"] * c["seqs"]) * c["q_heads"] * dim > 0.5 * 8192 * 8192 * 28 * 128:
        c["rows"] = max(1, c["rows"] * 3 // 4)
    c["seqs"] = min(c["seqs"], c["rows"])
    c["longest"] = min(c["rows"], max(-(-c["rows"] // c["seqs"]), int(1.7 * c["rows"] / c["seqs"])))
    return c


# ---- lengths, which the case alone decides --------------------------------------------------------------------------

def _spread_out(count, longest):
    """`count` lengths up to `longest`, spread evenly, the first one the longest."""
    return [max(1, int(longest * (1.0 - (i * 0.6180339887498949) % 1.0))) for i in range(count)]


def _lengths(c):
    """(new tokens, tokens in the cache with them) of each sequence."""
    n = c["seqs"]
    if c["op"] == "decode":
        return [1] * n, _spread_out(n, c["longest"])
    if c["op"] == "append":
        # as many new tokens each, the rest to the first; any of them may continue a longer sequence
        new = [c["rows"] // n] * n
        new[0] += c["rows"] - sum(new)
        return new, [max(a, b) for a, b in zip(new, _spread_out(n, c["longest"]))]
    share = _spread_out(n, c["longest"])
    new = [max(1, int(v * c["rows"] / sum(share))) for v in share]
    left = c["rows"] - sum(new)
    for i in range(n):   # what rounding left over, or took too much
        step = left if i == n - 1 else left // (n - i) if left >= 0 else -min(new[i] - 1, -left)
        step = max(step, 1 - new[i])
        new[i] += step
        left -= step
    return new, [v + c["context"] for v in new]


# ---- inputs ---------------------------------------------------------------------------------------------------------

_TYPES = {"f32": torch.float32, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}


def _cached(gen, c, shape, scales):
    """Keys or values as a cache holds them: order one, a few large channels."""
    x = torch.randn(shape, device="cuda", generator=gen)
    x[..., torch.randint(0, c["dim"], (max(1, c["dim"] // 64),), device="cuda", generator=gen)] *= 3.0
    if c["cache"] == "f16":
        return x.half()
    return (x / scales[:, None, None]).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    c, s = case, {"case": dict(case)}
    kv, dim, page = c["kv_heads"], c["dim"], c["page"]
    # an 8-bit cache's scales: calibrated, one for each head
    s["k_scales"], s["v_scales"] = ((0.02 + 0.02 * torch.rand(kv, device="cuda", generator=gen)) if c["cache"] == "e4m3" else None for _ in range(2))
    if c["op"] == "copy":
        pages = 2 * c["pairs"] + 3
        shape = (c["layers"], pages, kv, page, dim)
        s["k"], s["v"] = _cached(gen, c, shape, s["k_scales"]), _cached(gen, c, shape, s["v_scales"])
        order = torch.randperm(pages, device="cuda", generator=gen)[:2 * c["pairs"]]
        s["sources"], s["targets"] = order[:c["pairs"]].tolist(), order[c["pairs"]:].tolist()
        s["sources_dev"], s["targets_dev"] = order[:c["pairs"]].contiguous(), order[c["pairs"]:].contiguous()
        torch.cuda.synchronize()
        return s
    new, lengths = _lengths(c)
    used = [-(-v // page) for v in lengths]
    s["width"], pages = max(used), sum(used) + 2
    shape = (pages, kv, page, dim)
    s["k"], s["v"] = _cached(gen, c, shape, s["k_scales"]), _cached(gen, c, shape, s["v_scales"])
    order = torch.randperm(pages, device="cuda", generator=gen).tolist()
    tables, at = [], 0
    for n in used:
        tables.append(order[at:at + n] + [-1] * (s["width"] - n))
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s["tables"] = torch.tensor(tables, dtype=torch.int32, device="cuda")
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    rows, heads = starts[-1], c["q_heads"]
    s["rows"] = rows
    # what the host of such a program knows of the call: every row's sequence and position, every cached token's
    s["row_seq"] = torch.repeat_interleave(torch.arange(c["seqs"], device="cuda"), torch.tensor(new, device="cuda"))
    s["row_position"] = torch.arange(rows, device="cuda") - s["starts"].long()[s["row_seq"]] + (s["lengths"] - s["starts"].diff()).long()[s["row_seq"]]
    if c["op"] == "append":
        s["qkv"] = (1.5 * torch.randn(rows, (heads + 2 * kv) * dim, device="cuda", generator=gen)).to(_TYPES[c["x"]])
        half = c["rotary"] // 2
        angle = torch.arange(max(lengths), dtype=torch.float64, device="cuda")[:, None] * 1e6 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()
        s["q"] = torch.empty(rows, heads * dim, dtype=torch.float16, device="cuda")
    else:
        s["q"] = (1.5 * torch.randn(rows, heads * dim, device="cuda", generator=gen)).half()
        s["out"] = torch.empty(rows, heads * dim, dtype=torch.float16, device="cuda")
        s["scale"] = dim ** -0.5
    torch.cuda.synchronize()
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------------

def _rotated(x, cos, sin, interleaved):
    """x [rows, heads, dim] with its first 2 * half values turned by cos, sin [rows, half]."""
    half = cos.shape[1]
    cos, sin = cos[:, None], sin[:, None]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        both = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        both = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([both, rest], -1)


def _store(s, name, y, at_page, at_token):
    scales = s[name + "_scales"]
    if scales is None:
        s[name][at_page, :, at_token] = y.half()
    else:
        codes = (y / scales[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        s[name].view(torch.uint8)[at_page, :, at_token] = codes.view(torch.uint8)


def _plain_append(s):
    c, page = s["case"], s["case"]["page"]
    kv, heads, dim, half = c["kv_heads"], c["q_heads"], c["dim"], c["rotary"] // 2
    x = s["qkv"].float().view(s["rows"], heads + 2 * kv, dim)
    angle = s["cos_sin"][s["row_position"]]
    turned = _rotated(x[:, :heads + kv], angle[:, :half], angle[:, half:], c["interleaved"])
    at_page, at_token = s["tables"][s["row_seq"], s["row_position"] // page].long(), s["row_position"] % page
    _store(s, "k", turned[:, heads:], at_page, at_token)
    _store(s, "v", x[:, heads + kv:], at_page, at_token)
    return {"q": turned[:, :heads].reshape(s["rows"], heads * dim).half(), "k": s["k"], "v": s["v"]}


def _gathered(s, name, tokens_page, tokens_at):
    """A cache's tokens [..., kv_heads, dim] in f32."""
    x = s[name]
    scales = s[name + "_scales"]
    if scales is None:
        return x[tokens_page, :, tokens_at].float()
    return x.view(torch.uint8)[tokens_page, :, tokens_at].view(torch.float8_e4m3fn).float() * scales[:, None]


def _softmax_rows(scores, seen):
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top > -math.inf, top, 0.0))
    return p, p.sum(-1, keepdim=True)


def _plain_decode(s):
    c, page = s["case"], s["case"]["page"]
    kv, group, dim, n = c["kv_heads"], c["q_heads"] // c["kv_heads"], c["dim"], c["seqs"]
    at = torch.arange(s["width"] * page, device="cuda")
    pages = s["tables"].clamp_min(0).long()[:, at // page]
    k, v = (_gathered(s, name, pages, (at % page)[None].expand_as(pages)) for name in ("k", "v"))
    q = s["q"].float().view(n, kv, group, dim) * s["scale"]
    scores = q @ k.permute(0, 2, 3, 1)
    length = s["lengths"].long()[:, None]
    seen = at[None] < length
    if c["window"]:
        seen = seen & (at[None] >= length - c["window"])
    p, total = _softmax_rows(scores, seen[:, None, None])
    return ((p @ v.transpose(1, 2)) / total).reshape(n, -1).half()


def _plain_prompt(s):
    # every row against every cached token of the call, those of other sequences masked
    c, page = s["case"], s["case"]["page"]
    kv, group, dim, rows = c["kv_heads"], c["q_heads"] // c["kv_heads"], c["dim"], s["rows"]
    lengths = s["lengths"].long()
    seq = torch.repeat_interleave(torch.arange(c["seqs"], device="cuda"), lengths)
    at = torch.arange(seq.numel(), device="cuda") - (lengths.cumsum(0) - lengths)[seq]
    pages = s["tables"][seq, at // page].long()
    k, v = (_gathered(s, name, pages, at % page) for name in ("k", "v"))
    q = s["q"].float().view(rows, kv, group, dim).permute(1, 2, 0, 3) * s["scale"]
    scores = (q.reshape(kv, group * rows, dim) @ k.permute(1, 2, 0)).view(kv, group, rows, -1)
    position = s["row_position"][:, None]
    seen = (seq[None] == s["row_seq"][:, None]) & (at[None] <= position)
    if c["window"]:
        seen = seen & (at[None] > position - c["window"])
    p, total = _softmax_rows(scores, seen)
    o = (p.view(kv, group * rows, -1) @ v.transpose(0, 1)).view(kv, group, rows, dim) / total
    return o.permute(2, 0, 1, 3).reshape(rows, -1).half()


def _plain_copy(s):
    k, v = s["k"].view(torch.uint8), s["v"].view(torch.uint8)
    k[:, s["targets_dev"]] = k[:, s["sources_dev"]]
    v[:, s["targets_dev"]] = v[:, s["sources_dev"]]
    return {"k": s["k"], "v": s["v"]}


_PLAIN = {"append": _plain_append, "decode": _plain_decode, "prompt": _plain_prompt, "copy": _plain_copy}


# ---- the framework's operators ---------------------------------------------------------------------------------------

_NAMES = {torch.float32: "f32", torch.float16: "f16", torch.int32: "i32", torch.float8_e4m3fn: "u8"}
_LEGACY_STREAM = 1  # hipStreamLegacy: the null stream as a handle (a null pointer is the context's own stream)
_device = None


class _Rows:
    """A torch tensor as the library's functions take their arguments: a pointer and the name of the element type."""

    def __init__(self, t):
        self.tensor, self.ptr, self.dtype, self.numel = t, t.data_ptr(), _NAMES[t.dtype], t.numel()


def _dev():
    """The process's one context, its work in the order of torch's: on the stream that is torch's current one at the first call."""
    global _device
    if _device is None:
        import tensorwarp_amd as T
        _device = T.WarpDevice(0)
        _device.with_stream(torch.cuda.current_stream().cuda_stream or _LEGACY_STREAM)
    return _device


def _rows(t):
    return None if t is None else _Rows(t)


def _handles(s):
    """The cache's and the batch's descriptions, which a serving program makes once and keeps."""
    import tensorwarp_amd as T
    c, h = s["case"], {"T": T}

    def cache(k, v):
        return T.KvCache(_Rows(k), _Rows(v), c["page"], c["kv_heads"], c["dim"], k_scales=_rows(s["k_scales"]), v_scales=_rows(s["v_scales"]))

    if c["op"] == "copy":
        h["layers"] = T.kv_layers([cache(k, v) for k, v in zip(s["k"].unbind(0), s["v"].unbind(0))])
        return h
    h["cache"] = cache(s["k"], s["v"])
    h["seqs"] = T.KvSequences(_Rows(s["tables"]), _Rows(s["lengths"]), c["seqs"], s["width"], starts=None if c["op"] == "decode" else _Rows(s["starts"]))
    for name in ("qkv", "q", "cos_sin", "out"):
        if name in s:
            h[name] = _Rows(s[name])
    return h


def _own(s):
    c, dev = s["case"], _dev()
    h = s.get("handles")
    if h is None:
        h = s["handles"] = _handles(s)
    T = h["T"]
    if c["op"] == "append":
        T.kv_append(dev, h["cache"], h["seqs"], h["qkv"], s["rows"], c["q_heads"], h["q"], cos_sin=h["cos_sin"], positions=s["cos_sin"].shape[0],
                    rotary_dim=c["rotary"], interleaved=c["interleaved"])
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    if c["op"] == "copy":
        T.kv_copy_pages(dev, h["layers"], s["sources"], s["targets"])
        return {"k": s["k"], "v": s["v"]}
    if c["op"] == "decode":
        T.attention_decode(dev, h["cache"], h["seqs"], h["q"], c["q_heads"], h["out"], scale=s["scale"], window=c["window"])
    else:
        T.attention_prompt(dev, h["cache"], h["seqs"], h["q"], s["rows"], c["q_heads"], h["out"], scale=s["scale"], window=c["window"])
    return s["out"]


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    c = case
    kv, dim, es = c["kv_heads"], c["dim"], 1 if c["cache"] == "e4m3" else 2
    if c["op"] == "copy":
        return {"bytes": 2 * 2 * c["pairs"] * c["layers"] * kv * c["page"] * dim * es, "flops": 0}
    new, lengths = _lengths(c)
    heads, rows = c["q_heads"], sum(new)
    if c["op"] == "append":
        xs = 4 if c["x"] == "f32" else 2
        return {"bytes": rows * dim * ((heads + 2 * kv) * xs + heads * 2 + 2 * kv * es) + 4 * rows * c["rotary"],
                "flops": 3 * rows * (heads + kv) * c["rotary"]}
    w = c["window"] or 1 << 30
    tokens = sum(min(t, n + w - 1) for n, t in zip(new, lengths))   # tokens that some row sees
    # scores: row i of a sequence's new ones sees min(position + 1, window) tokens
    scores = sum(_seen(t, w) - _seen(t - n, w) for n, t in zip(new, lengths))
    return {"bytes": 2 * tokens * kv * dim * es + 4 * rows * heads * dim, "flops": 4 * heads * dim * scores}


def _seen(t, w):
    """Sum over the first t positions of the tokens that each sees."""
    return t * (t + 1) // 2 if t <= w else w * (w + 1) // 2 + (t - w) * w


# ---- from the definitions, in 64 bits --------------------------------------------------------------------------------

def exact(case, seed):
    s, c = prepare(case, seed), case
    kv, dim, page = c["kv_heads"], c["dim"], c["page"]
    if c["op"] == "copy":
        out = {}
        for name in ("k", "v"):
            whole = s[name].float().cpu()
            after = whole.clone()
            for a, b in zip(s["sources"], s["targets"]):
                after[:, b] = whole[:, a]
            out[name] = after.double()
        return out
    heads = c["q_heads"]
    group = heads // kv
    new, lengths = _lengths(c)
    tables = s["tables"].tolist()
    if c["op"] == "append":
        x = s["qkv"].double()
        half = c["rotary"] // 2
        out_q = x[:, :heads * dim].clone()
        out = {"q": out_q, "k": s["k"].float().double(), "v": s["v"].float().double()}
        row = 0
        for i in range(c["seqs"]):
            at = torch.arange(lengths[i] - new[i], lengths[i], device="cuda")
            rows = slice(row, row + new[i])
            row += new[i]
            turn = torch.complex(s["cos_sin"][at, :half].double(), s["cos_sin"][at, half:].double())
            pages = torch.tensor(tables[i], device="cuda")[at // page]
            for h in range(heads + 2 * kv):
                y = x[rows, h * dim:(h + 1) * dim].clone()
                if h < heads + kv:
                    first = slice(0, 2 * half, 2) if c["interleaved"] else slice(0, half)
                    second = slice(1, 2 * half, 2) if c["interleaved"] else slice(half, 2 * half)
                    z = torch.complex(y[:, first], y[:, second]) * turn
                    y[:, first], y[:, second] = z.real.clone(), z.imag.clone()
                if h < heads:
                    out_q[rows, h * dim:(h + 1) * dim] = y
                else:
                    name, g = ("k", h - heads) if h < heads + kv else ("v", h - heads - kv)
                    if s[name + "_scales"] is not None:
                        y = y / s[name + "_scales"][g].double()
                        y = torch.minimum(torch.maximum(y, torch.tensor(-E4M3_MAX, device="cuda")), torch.tensor(E4M3_MAX, device="cuda"))
                    out[name][pages, g, at % page] = y
        return out
    result = torch.zeros(s["rows"], heads, dim, dtype=torch.float64, device="cuda")
    row = 0
    for i in range(c["seqs"]):
        n, length = new[i], lengths[i]
        count = -(-length // page)
        pages = torch.tensor(tables[i][:count], device="cuda")
        first = max(0, length - n + 1 - c["window"]) if c["window"] else 0   # the first token that any row sees
        for g in range(kv):
            k, v = (s[name].view(torch.uint8)[pages, g].view(s[name].dtype).reshape(-1, dim)[first:length].float().double() for name in ("k", "v"))
            if s["k_scales"] is not None:
                k, v = k * s["k_scales"][g].double(), v * s["v_scales"][g].double()
            for part in range(0, n, 2048):
                m = min(2048, n - part)
                where = torch.arange(length - n + part, length - n + part + m, device="cuda")[:, None]
                token = torch.arange(first, length, device="cuda")[None]
                hidden = (token > where) | ((token <= where - c["window"]) if c["window"] else token < 0)
                q = s["q"][row + part:row + part + m].double().view(m, heads, dim)
                for h in range(g * group, (g + 1) * group):
                    a = torch.softmax((q[:, h] @ k.t()).mul_(s["scale"]).masked_fill_(hidden, -math.inf), 1)
                    result[row + part:row + part + m, h] = a @ v
        row += n
    return result.view(s["rows"], -1)
