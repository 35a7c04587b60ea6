"""The 8-bit activation path and the token sampler, as cases that can be timed: what a program that serves a model with
weights in 8-bit floating point (e4m3, one f32 scale per block of 128 x 128) asks of this library per layer and per token.

op          a pass is
gemm        C[m, n] = sum over blocks b of 128 features of a_scales[m, b] * w_scales[n // 128, b] * (A_b x W_b^T), A [m, k] and
            W [n, k] in e4m3 as the checkpoint holds them, sums in 32 bits, C in f32 or f16
norm        s = x + residual, y = s / sqrt(mean(s^2) + eps) * weight, and y as e4m3 rows with one f32 scale per row and 128
            columns: scale = max|y| / 448 over the block, q = e4m3(y / scale); s comes back in f32, y in f16 where asked for
gated       y = act(gate) * up of fused [gate | up] rows (or of rows in the paired order: 32 gate columns, their 32 up columns, and
            so on), as e4m3 rows with scales as above; act is silu or the tanh form of gelu
sample      one token per row of f32 logits from the row's own uniform number u: weights exp((x - max x) / temperature); of the
            tokens in descending order (equal ones by index) the first top_k, of these the shortest run that holds top_p of their
            sum, of these the ones of at least min_p times the largest; the token is the first, by index, at which the running sum
            of what is left exceeds u times the whole.  temperature 0 takes the largest logit
"""
import math

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0


def listed():
    return [
        # one token through the output projection of a small model: a launch and little else
        {"name": "gemm_896x896_m1", "op": "gemm", "m": 1, "n": 896, "k": 896, "out": "f32"},
        # one token through gate and up of a 7B model: the weights once through memory
        {"name": "gemm_3584x37888_m1", "op": "gemm", "m": 1, "n": 37888, "k": 3584, "out": "f32"},
        # a few users' tokens through a down projection
        {"name": "gemm_11008x4096_m13", "op": "gemm", "m": 13, "n": 4096, "k": 11008, "out": "f32"},
        # a prompt of odd length through a deep, narrow projection
        {"name": "gemm_18944x3584_m333", "op": "gemm", "m": 333, "n": 3584, "k": 18944, "out": "f16"},
        # a long prompt through gate and up: matrix instructions and nothing else
        {"name": "gemm_4096x22016_m2048", "op": "gemm", "m": 2048, "n": 22016, "k": 4096, "out": "f16"},
        # the norm ahead of one token's projections
        {"name": "norm_1x896", "op": "norm", "rows": 1, "cols": 896, "x": "f32", "residual": True, "normed": False},
        # ahead of a long prompt's, with the f16 rows that 4-bit projections of the same layer take
        {"name": "norm_2048x4096", "op": "norm", "rows": 2048, "cols": 4096, "x": "f16", "residual": True, "normed": True},
        # the gate of eight routed experts for one token
        {"name": "gated_8x704_gelu", "op": "gated", "rows": 8, "dim": 704, "x": "f32", "paired": True, "act": "gelu"},
        # and of a long prompt's feed-forward block
        {"name": "gated_2048x11008_silu", "op": "gated", "rows": 2048, "dim": 11008, "x": "f16", "paired": False, "act": "silu"},
        # the next token of one user
        {"name": "sample_1x152064", "op": "sample", "rows": 1, "cols": 152064, "mix": "plain"},
        # of a decode batch whose users asked for different things, some rows under a grammar's mask
        {"name": "sample_32x152064", "op": "sample", "rows": 32, "cols": 152064, "mix": "masked"},
        # of many short-vocabulary rows
        {"name": "sample_256x32000", "op": "sample", "rows": 256, "cols": 32000, "mix": "plain"},
    ]


def _log_int(rng, lo, hi, step=1):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def draw(rng):
    op = rng.choice(["gemm", "gemm", "gemm", "norm", "gated", "sample"])
    if op == "gemm":
        # k in whole 16-byte pieces (its last block often cut short), n of any size
        k, n = _log_int(rng, 256, 18944, 16), _log_int(rng, 256, 37888)
        n = min(n, 3584 * 37888 // k)
        m = min(_log_int(rng, 1, 2048), max(1, 2048 * 22016 * 4096 // (n * k)))
        return {"op": op, "m": m, "n": n, "k": k, "out": rng.choice(["f32", "f16"])}
    if op == "norm":
        cols = _log_int(rng, 256, 8192)
        return {"op": op, "rows": min(_log_int(rng, 1, 2048), 2048 * 4096 // cols), "cols": cols, "x": rng.choice(["f32", "f16"]),
                "residual": rng.random() < 0.75, "normed": rng.random() < 0.5}
    if op == "gated":
        paired = rng.random() < 0.5
        dim = _log_int(rng, 352, 18944, 32 if paired else 1)
        return {"op": op, "rows": min(_log_int(rng, 1, 2048), 2048 * 11008 // dim), "dim": dim, "x": rng.choice(["f32", "f16"]),
                "paired": paired, "act": rng.choice(["silu", "gelu"])}
    cols = _log_int(rng, 1000, 152064)
    return {"op": op, "rows": min(_log_int(rng, 1, 256), 256 * 32000 // cols), "cols": cols, "mix": rng.choice(["plain", "masked"])}


# ---- inputs -------------------------------------------------------------------------------------------------------

_TYPES = {"f32": torch.float32, "f16": torch.float16}


def _blocks(n):
    return -(-n // BLOCK)


def _activations(gen, rows, cols):
    """Normalized rows: order one, with the few large channels that trained models have."""
    a = torch.randn(rows, cols, device="cuda", generator=gen)
    a[:, torch.randint(0, cols, (max(1, cols // 256),), device="cuda", generator=gen)] *= 12.0
    return a


def _e4m3_rows(x):
    """f32 rows as e4m3 with a scale per row and 128 columns."""
    rows, cols = x.shape
    kb = _blocks(cols)
    y = torch.zeros(rows, kb * BLOCK, device=x.device)
    y[:, :cols] = x
    y = y.view(rows, kb, BLOCK)
    scales = y.abs().amax(2).clamp_min(1e-30) / E4M3_MAX
    q = (y / scales[:, :, None]).view(rows, kb * BLOCK)[:, :cols].to(torch.float8_e4m3fn).contiguous()
    return q, scales


def _e4m3_weight(gen, n, k):
    """Normally distributed weights as a checkpoint holds them: [n, k] in e4m3, f32 scales [ceil(n / 128), ceil(k / 128)]."""
    w = 0.02 * torch.randn(n, k, device="cuda", generator=gen)
    nb, kb = _blocks(n), _blocks(k)
    scales = torch.full((nb, kb), 0.02 * 4.5 / E4M3_MAX, device="cuda") * (0.75 + 0.5 * torch.rand(nb, kb, device="cuda", generator=gen))
    w.div_(scales.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]).clamp_(-E4M3_MAX, E4M3_MAX)
    return w.to(torch.float8_e4m3fn), scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    c, s = case, {"case": dict(case)}
    if c["op"] == "gemm":
        s["a"], s["a_scales"] = _e4m3_rows(_activations(gen, c["m"], c["k"]))
        s["w"], s["w_scales"] = _e4m3_weight(gen, c["n"], c["k"])
        s["c"] = torch.empty(c["m"], c["n"], dtype=_TYPES[c["out"]], device="cuda")
    elif c["op"] == "norm":
        rows, cols = c["rows"], c["cols"]
        s["x"] = _activations(gen, rows, cols).to(_TYPES[c["x"]])
        s["residual"] = 3.0 * _activations(gen, rows, cols) if c["residual"] else None
        s["weight"] = 1.0 + 0.2 * torch.randn(cols, device="cuda", generator=gen)
        s["eps"] = 1e-6
        s["sum"] = torch.empty(rows, cols, device="cuda") if c["residual"] else None
        s["normed"] = torch.empty(rows, cols, dtype=torch.float16, device="cuda") if c["normed"] else None
        s["q"] = torch.empty(rows, cols, dtype=torch.float8_e4m3fn, device="cuda")
        s["scales"] = torch.empty(rows, _blocks(cols), device="cuda")
    elif c["op"] == "gated":
        rows, dim = c["rows"], c["dim"]
        s["gate_up"] = (1.5 * torch.randn(rows, 2 * dim, device="cuda", generator=gen)).to(_TYPES[c["x"]])
        s["q"] = torch.empty(rows, dim, dtype=torch.float8_e4m3fn, device="cuda")
        s["scales"] = torch.empty(rows, _blocks(dim), device="cuda")
    else:
        rows, cols = c["rows"], c["cols"]
        # a language model's logits: a broad body and a few candidates that stand out
        x = 2.0 * torch.randn(rows, cols, device="cuda", generator=gen)
        at = torch.randint(0, cols, (rows, 24), device="cuda", generator=gen)
        x.scatter_(1, at, 6.0 + 4.0 * torch.rand(rows, 24, device="cuda", generator=gen))
        if c["mix"] == "masked":  # every second row allows one token in eight
            out = torch.rand(rows, cols, device="cuda", generator=gen) > 0.125
            out[1::2] = False
            out[:, 0] = False
            x.masked_fill_(out, -math.inf)
        pick = torch.rand(4, rows, device="cuda", generator=gen)
        s["logits"] = x
        s["uniform"] = torch.rand(rows, device="cuda", generator=gen)
        s["temperature"] = 0.5 + torch.rand(rows, device="cuda", generator=gen)
        s["top_p"] = torch.where(pick[1] < 0.7, 0.8 + 0.19 * torch.rand(rows, device="cuda", generator=gen), 1.0)
        s["top_k"] = torch.where(pick[2] < 0.5, torch.randint(1, 100, (rows,), device="cuda", generator=gen), 0).to(torch.int32)
        s["min_p"] = torch.where(pick[3] < 0.3, 0.1 * torch.rand(rows, device="cuda", generator=gen), 0.0)
        if rows > 1:  # in a batch some users decode greedily
            s["temperature"] = torch.where(pick[0] < 0.1, 0.0, s["temperature"])
        s["tokens"] = torch.empty(rows, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------

def _spread(scales, rows, cols):
    return scales.repeat_interleave(BLOCK, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]


def _plain_gemm(s):
    m, n, k = (s["case"][d] for d in ("m", "n", "k"))
    a = s["a"].float() * s["a_scales"].repeat_interleave(BLOCK, 1)[:, :k]
    w = s["w"].float() * _spread(s["w_scales"], n, k)
    return (a @ w.t()).to(s["c"].dtype)


def _quantize(y):
    rows, cols = y.shape
    kb = _blocks(cols)
    y = torch.nn.functional.pad(y, (0, kb * BLOCK - cols)).view(rows, kb, BLOCK)
    scales = y.abs().amax(2).clamp_min(1e-30) / E4M3_MAX
    return {"q": (y / scales[:, :, None]).view(rows, kb * BLOCK)[:, :cols].to(torch.float8_e4m3fn), "scales": scales}


def _plain_norm(s):
    t = s["x"].float()
    if s["residual"] is not None:
        t = t + s["residual"]
    y = t * torch.rsqrt((t * t).mean(1, keepdim=True) + s["eps"]) * s["weight"]
    out = _quantize(y)
    if s["residual"] is not None:
        out["sum"] = t
    if s["normed"] is not None:
        out["normed"] = y.to(torch.float16)
    return out


def _halves(gate_up, paired):
    rows, dim = gate_up.shape[0], gate_up.shape[1] // 2
    if paired:
        v = gate_up.view(rows, dim // 32, 2, 32)
        return v[:, :, 0].reshape(rows, dim), v[:, :, 1].reshape(rows, dim)
    return gate_up[:, :dim], gate_up[:, dim:]


def _plain_gated(s):
    g, u = _halves(s["gate_up"].float(), s["case"]["paired"])
    if s["case"]["act"] == "silu":
        y = g / (1.0 + torch.exp(-g)) * u
    else:
        y = 0.5 * g * (1.0 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g))) * u
    return _quantize(y)


def _plain_sample(s):
    # in 64 bits: a token is decided by where u falls among up to 10^5 borders
    x = s["logits"].double()
    rows, cols = x.shape
    order = torch.sort(x, dim=1, descending=True, stable=True)
    largest = order.values[:, :1]
    t = s["temperature"].double()[:, None]
    w = torch.exp((order.values - largest) / torch.where(t > 0, t, 1.0))
    place = torch.arange(cols, device=x.device)[None]
    k = s["top_k"][:, None]
    k = torch.where(k > 0, k, cols)
    k = torch.where(t > 0, k, 1)
    w = torch.where(place < k, w, 0.0)
    before = torch.cumsum(w, 1) - w
    mass = w.sum(1, keepdim=True)
    kept = (place < k) & (before < s["top_p"].double()[:, None] * mass) & (w >= s["min_p"].double()[:, None]) | (place == 0)
    by_index = torch.zeros_like(w).scatter_(1, order.indices, torch.where(kept, w, 0.0))
    run_sum = torch.cumsum(by_index, 1)
    past = run_sum > s["uniform"].double()[:, None] * run_sum[:, -1:]
    return torch.argmax(past.to(torch.int8), dim=1).to(torch.int32)


_PLAIN = {"gemm": _plain_gemm, "norm": _plain_norm, "gated": _plain_gated, "sample": _plain_sample}


# ---- the framework's operators -------------------------------------------------------------------------------------

_NAMES = {torch.float32: "f32", torch.float16: "f16", torch.int32: "i32", torch.float8_e4m3fn: "u8"}
_device = None


class _Rows:
    """A torch tensor as the library's functions take their arguments: a pointer and the name of the element type."""

    def __init__(self, t):
        self.tensor, self.ptr, self.dtype, self.numel = t, t.data_ptr(), _NAMES[t.dtype], t.numel()


_LEGACY_STREAM = 1  # hipStreamLegacy: the null stream as a handle (a null pointer is the context's own stream)


def _dev():
    """The process's one context, its work in the order of torch's: on the stream that is torch's current one at the first call."""
    global _device
    if _device is None:
        import tensorwarp_amd as T
        _device = T.WarpDevice(0)
        _device.with_stream(torch.cuda.current_stream().cuda_stream or _LEGACY_STREAM)
    return _device


def _row(s, name):
    t = s[name]
    return None if t is None else _Rows(t)


def _own(s):
    import tensorwarp_amd as T
    c, dev = s["case"], _dev()
    if c["op"] == "gemm":
        T.gemm_fp8(dev, _row(s, "a"), _row(s, "a_scales"), _row(s, "w"), _row(s, "w_scales"), c["m"], c["n"], c["k"], _row(s, "c"))
        return s["c"]
    if c["op"] == "norm":
        T.add_rms_norm_fp8(dev, _row(s, "x"), _row(s, "residual"), _row(s, "weight"), s["eps"], c["rows"], c["cols"],
                           _row(s, "q"), _row(s, "scales"), sum=_row(s, "sum"), normed=_row(s, "normed"))
        return {name: s[name] for name in ("q", "scales", "sum", "normed") if s[name] is not None}
    if c["op"] == "gated":
        gated = T.swiglu_rows_fp8 if c["act"] == "silu" else T.geglu_rows_fp8
        gated(dev, _row(s, "gate_up"), _row(s, "q"), _row(s, "scales"), c["dim"], c["rows"], paired=c["paired"])
        return {"q": s["q"], "scales": s["scales"]}
    T.sample(dev, _row(s, "logits"), _row(s, "uniform"), _row(s, "tokens"), c["rows"], c["cols"], temperature=_row(s, "temperature"),
             top_k=_row(s, "top_k"), top_p=_row(s, "top_p"), min_p=_row(s, "min_p"))
    return s["tokens"]


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "gemm":
        m, n, k = c["m"], c["n"], c["k"]
        scales = 4 * _blocks(k) * (m + _blocks(n))
        return {"bytes": m * k + n * k + scales + m * n * (4 if c["out"] == "f32" else 2), "flops": 2 * m * n * k}
    if c["op"] == "sample":
        return {"bytes": 4 * c["rows"] * c["cols"] + 24 * c["rows"], "flops": 2 * c["rows"] * c["cols"]}
    es = 4 if c["x"] == "f32" else 2
    if c["op"] == "norm":
        rows, cols = c["rows"], c["cols"]
        per = es + 1 + (8 if c["residual"] else 0) + (2 if c["normed"] else 0)
        return {"bytes": rows * cols * per + 4 * cols + 4 * rows * _blocks(cols), "flops": 6 * rows * cols}
    return {"bytes": c["rows"] * c["dim"] * (2 * es + 1) + 4 * c["rows"] * _blocks(c["dim"]), "flops": 10 * c["rows"] * c["dim"]}


# ---- from the definitions, in 64 bits ------------------------------------------------------------------------------

def _exact_rows(y):
    """Scales and the values that the 8-bit codes stand for in units of them, before their rounding."""
    rows, cols = y.shape
    scales = torch.stack([part.abs().max(dim=1).values / E4M3_MAX for part in torch.split(y, BLOCK, dim=1)], dim=1)
    column_block = torch.arange(cols, device=y.device).div(BLOCK, rounding_mode="floor")
    return {"q": y / scales.clamp_min(1e-300)[:, column_block], "scales": scales}


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "gemm":
        total = torch.zeros(c["m"], c["n"], dtype=torch.float64, device="cuda")
        row_block = torch.arange(c["n"], device="cuda").div(BLOCK, rounding_mode="floor")
        for b in range(_blocks(c["k"])):
            at = slice(b * BLOCK, min((b + 1) * BLOCK, c["k"]))
            part = s["a"][:, at].float().double() @ s["w"][:, at].float().double().t().contiguous()
            total += part * s["a_scales"][:, b].double()[:, None] * s["w_scales"][:, b].double()[row_block][None]
        return total
    if c["op"] == "norm":
        v = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
        y = v / torch.sqrt(torch.linalg.vector_norm(v, dim=1, keepdim=True) ** 2 / c["cols"] + s["eps"]) * s["weight"].double()
        out = _exact_rows(y)
        if s["residual"] is not None:
            out["sum"] = v
        if s["normed"] is not None:
            out["normed"] = y
        return out
    if c["op"] == "gated":
        v, dim = s["gate_up"].double(), c["dim"]
        j = torch.arange(dim, device="cuda")
        gate_at, up_at = ((j // 32) * 64 + j % 32, (j // 32) * 64 + j % 32 + 32) if c["paired"] else (j, j + dim)
        g, u = v[:, gate_at], v[:, up_at]
        act = g * torch.sigmoid(g) if c["act"] == "silu" else g * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3))
        return _exact_rows(act * u)
    import numpy as np
    x = s["logits"].double().cpu().numpy()
    par = {name: s[name].double().cpu().numpy() for name in ("uniform", "temperature", "top_p", "top_k", "min_p")}
    tokens = np.zeros(c["rows"], np.int32)
    for r in range(c["rows"]):
        if par["temperature"][r] <= 0:
            tokens[r] = np.argmax(x[r])
            continue
        order = np.lexsort((np.arange(c["cols"]), -x[r]))
        if par["top_k"][r] > 0:
            order = order[:int(par["top_k"][r])]
        w = np.exp((x[r][order] - x[r][order[0]]) / par["temperature"][r])
        sums = np.concatenate([[0.0], np.cumsum(w)])
        count = max(1, min(int(np.searchsorted(sums[:-1], par["top_p"][r] * sums[-1], side="left")), int((w >= par["min_p"][r]).sum())))
        by_index = np.argsort(order[:count])
        sums = np.cumsum(w[:count][by_index])
        at = int(np.searchsorted(sums, par["uniform"][r] * sums[-1], side="right"))
        tokens[r] = order[:count][by_index][min(at, count - 1)]
    return torch.from_numpy(tokens)
