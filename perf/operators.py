"""The token end of a training step as cases that can be timed and compared: embedding lookup with scaling and
dropout, its gradient by sorted tokens, and dropout from a counter-based generator.

Tables have the shapes of the configurations the package is benchmarked and tested on (GPT-2 small: 50257 x 768,
Llama-3-8B: 128256 x 4096, an odd 2999 x 1777 matrix) and relatives of them.  Token ids follow the frequencies of
text (1 / rank), with a share of places without a token (negative ids: padding) and, where a case says so, a
share of one id (an end-of-text token used as padding).
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
MAX_ELEMENTS = 134_217_728  # of a drawn case's activations: the largest listed one's
MAX_TABLE = 525_336_576  # of a drawn case's table
M32 = 0xFFFFFFFF


def _embed(tokens, rows, dim, **more):
    return {"what": "embed", "tokens": tokens, "rows": rows, "dim": dim, "dtype": "bf16", "ecc": 0, "scale": 1.0, "p": 0.0, "pad": 0.0,
            "hot": 0.0, "ids": 64, **more}


def _grad(tokens, rows, dim, **more):
    return {"what": "grad", "tokens": tokens, "rows": rows, "dim": dim, "dtype": "bf16", "scale": 1.0, "p": 0.0, "pad": 0.0, "hot": 0.0,
            "ids": 64, "tied": False, **more}


def _dropout(rows, dim, **more):
    return {"what": "dropout", "rows": rows, "dim": dim, "dtype": "bf16", "p": 0.1, "residual": False, **more}


def listed():
    return [
        # one token of a generation loop: latency of a call
        dict(_embed(1, 50257, 768), name="embed_one_token"),
        # GPT-2 small's micro-batch of 8 x 1024 tokens, embedding dropout included
        dict(_embed(8192, 50257, 768, p=0.1), name="embed_gpt2_dropout"),
        # two sequences of 8192 tokens of Llama-3-8B with the embeddings scaled by sqrt(dim)
        dict(_embed(16384, 128256, 4096, scale=64.0), name="embed_llama"),
        # evaluation on master weights: rows of an odd-width fp16 table with 16-bit error-correction codes, to fp32
        dict(_embed(5003, 2999, 1777, dtype="f16", ecc=16, ids=32), name="embed_master_odd"),
        # a handful of tokens into a small fp32 table (adapters, tests): latency of the gradient
        dict(_grad(33, 8192, 1024, dtype="f32"), name="grad_few_tokens"),
        # GPT-2 small's batch of 16 x 1024 tokens through embedding dropout
        dict(_grad(16384, 50257, 768, p=0.1), name="grad_gpt2_dropout"),
        # Llama-3-8B's table, four sequences of 8192 tokens (the largest)
        dict(_grad(32768, 128256, 4096), name="grad_llama"),
        # a padded batch whose padding is an ordinary id, odd everywhere, fp32
        dict(_grad(8191, 2999, 1777, dtype="f32", hot=0.4, pad=0.1, scale=0.5, ids=32), name="grad_padded_odd"),
        # tied embeddings: added to the gradient that the output head left in the same leaf
        dict(_grad(8192, 128256, 4096, tied=True), name="grad_tied"),
        # the attention output of one short sequence
        dict(_dropout(256, 768), name="dropout_small"),
        # the end of a block of a large model: dropout and the residual addition in one pass
        dict(_dropout(16384, 4096, residual=True), name="dropout_residual"),
        # fp32 activations of odd width, as many dropped as kept
        dict(_dropout(9001, 1777, dtype="f32", p=0.5), name="dropout_f32_odd"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    what = rng.choice(["embed", "embed", "grad", "grad", "grad", "dropout"])
    dim = rng.choice([8 * _log(rng, 8, 512), _log(rng, 65, 4095)])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    p = rng.choice([0.0, 0.1, rng.uniform(0.01, 0.9)])
    if what == "dropout":
        return _dropout(_log(rng, 1, min(32768, MAX_ELEMENTS // dim)), dim, dtype=dtype, p=p or 0.3, residual=rng.random() < 0.5)
    rows = _log(rng, 100, min(128256, MAX_TABLE // dim // (2 if dtype == "f32" else 1)))
    tokens = _log(rng, 1, min(65536, MAX_ELEMENTS // dim // (2 if dtype == "f32" else 1)))
    more = dict(dtype=dtype, p=p, scale=rng.choice([1.0, math.sqrt(dim)]), pad=rng.choice([0.0, 0.0, 0.2]),
                hot=rng.choice([0.0, 0.0, rng.uniform(0.0, 0.6)]), ids=rng.choice([32, 64]))
    if what == "embed":
        return _embed(tokens, rows, dim, ecc=0 if dtype == "f32" else rng.choice([0, 0, 8, 16]), **more)
    return _grad(tokens, rows, dim, tied=rng.random() < 0.3, **more)


def _shares(case, device):
    """How often each id comes, in 64 bits."""
    share = 1.0 / (torch.arange(case["rows"], dtype=torch.float64, device=device) + 2.7)
    share *= (1.0 - case["hot"]) / share.sum()
    share[0] += case["hot"]
    return share


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std, dt=dtype):
        return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dt)

    state = {**case, "seed": 0x9E3779B97F4A7C15 ^ seed, "offset": seed % 1000}
    if case["what"] == "dropout":
        state["x"] = normal(case["rows"], case["dim"], std=1.0)
        state["add"] = normal(case["rows"], case["dim"], std=2.0) if case["residual"] else None
        return state
    n = case["tokens"]
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    ids = torch.searchsorted(torch.cumsum(_shares(case, "cuda"), 0), u).clamp_(max=case["rows"] - 1)
    if case["pad"]:
        ids[torch.rand(n, generator=g, device="cuda") < case["pad"]] = -1
    state["tokens_"] = ids.to(torch.int32 if case["ids"] == 32 else torch.int64)
    if case["what"] == "embed":
        state["table"] = normal(case["rows"], case["dim"], std=0.02)
        if case["ecc"]:
            top = 127 if case["ecc"] == 8 else 32767
            code = torch.int8 if case["ecc"] == 8 else torch.int16
            state["codes"] = torch.randint(-top, top + 1, (case["rows"], case["dim"]), generator=g, device="cuda", dtype=torch.int32).to(code)
        else:
            state["codes"] = None
    else:
        state["dy"] = normal(n, case["dim"], std=1e-2)
        state["grad"] = normal(case["rows"], case["dim"], std=1e-3) if case["tied"] else None
    return state


def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    """The calls that a user makes."""
    import flashoptim_jax_b200 as fo

    if s["what"] == "dropout":
        return fo.dropout(s["x"], s["p"], s["seed"], s["offset"], residual=s["add"])
    if s["what"] == "embed":
        return fo.embed(s["table"], s["tokens_"], scale=s["scale"], ecc=s["codes"], p=s["p"], seed=s["seed"], offset=s["offset"])
    return fo.embed_grad(s["dy"], s["tokens_"], s["rows"], scale=s["scale"], p=s["p"], seed=s["seed"], offset=s["offset"],
                         out=s["grad"], accumulate=s["tied"])


def _times(a, b):
    """(high, low) 32 bits of the product of 32-bit whole numbers held in 64 bits; `b` is a Python number."""
    low = a * (b & 0xFFFF)  # below 2^48
    high = a * (b >> 16) + (low >> 16)  # below 2^49
    return high >> 16, ((high & 0xFFFF) << 16) | (low & 0xFFFF)


def _philox(n, seed, offset, second, device):
    """16 bits for each of n elements: Philox4x32-10 (Salmon et al., Parallel random numbers: as easy as 1, 2, 3, 2011) of
    the counter (element / 8, offset), eight elements to a block; `second` marks the stream that settles ties."""
    block = torch.arange((n + 7) // 8, dtype=torch.int64, device=device)
    c0, c1 = block & M32, (block >> 32) | (second << 31)
    c2, c3 = torch.full_like(block, offset & M32), torch.full_like(block, (offset >> 32) & M32)
    k0, k1 = seed & M32, (seed >> 32) & M32
    for _ in range(10):
        (h0, l0), (h1, l1) = _times(c0, 0xD2511F53), _times(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    words = torch.stack([c0, c1, c2, c3], 1)
    return torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:n]


def _kept(s, shape, device):
    """1 / (1 - p) where an element stays, 0 where it is dropped, in 32 bits."""
    n = math.prod(shape)
    bits = (_philox(n, s["seed"], s["offset"], 0, device) << 16) | _philox(n, s["seed"], s["offset"], 1, device)
    return ((bits >= round(s["p"] * 2**32)).float() * (1.0 / (1.0 - s["p"]))).reshape(shape)


def _plain(s):
    if s["what"] == "dropout":
        y = s["x"].float() * _kept(s, s["x"].shape, s["x"].device)
        return (y if s["add"] is None else y + s["add"].float()).to(s["x"].dtype)
    ids = s["tokens_"].long()
    some = ids >= 0
    if s["what"] == "embed":
        at = ids.clamp(min=0)
        y = s["table"][at]
        dtype = y.dtype
        if s["codes"] is None:
            y = y.float()
        else:  # the stored value and code / top of half its unit in the last place
            digits, least, top = 8 if dtype == torch.bfloat16 else 11, -126 if dtype == torch.bfloat16 else -14, 2 ** (s["ecc"] - 1) - 1
            y = y.float()
            exponent = torch.where(y == 0, float(least), torch.frexp(y)[1].float() - 1).clamp(min=least)
            y = y + (s["codes"][at].float() / top) * torch.exp2(exponent - digits)
            dtype = torch.float32
        y = y * (s["scale"] * some.float()[:, None])
        if s["p"]:
            y = y * _kept(s, y.shape, y.device)
        return y.to(dtype)
    dy = s["dy"].float() * s["scale"]
    if s["p"]:
        dy = dy * _kept(s, dy.shape, dy.device)
    if s["tied"]:
        total = s["grad"].float()
    else:
        total = torch.zeros((s["rows"], s["dim"]), dtype=torch.float32, device=dy.device)
    total.index_add_(0, ids.clamp(min=0), dy * some.float()[:, None])
    if s["tied"]:
        return s["grad"].copy_(total)
    return total.to(s["dy"].dtype)


def work(case):
    e = BYTES[case["dtype"]]
    if case["what"] == "dropout":
        n = case["rows"] * case["dim"]
        return {"bytes": (3 if case["residual"] else 2) * n * e, "flops": 2 * n}
    n, dim = case["tokens"], case["dim"]
    distinct = float((1.0 - (1.0 - (1.0 - case["pad"]) * _shares(case, "cpu")) ** n).sum())  # rows that some token names
    some = (1.0 - case["pad"]) * n
    if case["what"] == "embed":
        out = 4 if case["ecc"] else e
        return {"bytes": n * case["ids"] / 8 + distinct * dim * (e + case["ecc"] / 8) + n * dim * out, "flops": 2 * some * dim}
    table = 2 * distinct if case["tied"] else case["rows"]
    return {"bytes": n * case["ids"] / 8 + some * dim * e + table * dim * e, "flops": 2 * some * dim}


def _mask64(n, s):
    """Which elements stay, from the definition: the 32-bit uniform of an element, from products in 16-bit limbs."""
    def limbs(x, y):  # x tensor, y number, both below 2^32: the 64-bit product as its two halves
        x0, x1, y0, y1 = x & 0xFFFF, x >> 16, y & 0xFFFF, y >> 16
        cross = x1 * y0 + ((x0 * y0) >> 16)
        rest = x0 * y1 + (cross & 0xFFFF)
        return x1 * y1 + (cross >> 16) + (rest >> 16), (((rest & 0xFFFF) << 16) + ((x0 * y0) & 0xFFFF))

    keep = torch.empty(n, dtype=torch.bool, device="cuda")
    threshold, part = round(s["p"] * 2**32), 1 << 25
    for first in range(0, n, part):
        count = min(part, n - first)
        elements = torch.arange(first, first + count, device="cuda")
        blocks = torch.arange(first >> 3, ((first + count - 1) >> 3) + 1, device="cuda")
        halves = []
        for stream in (0, 1):
            x = [blocks % 2**32, blocks // 2**32 + stream * 2**31, torch.zeros_like(blocks) + s["offset"] % 2**32, torch.zeros_like(blocks) + s["offset"] // 2**32 % 2**32]
            for r in range(10):
                key0, key1 = (s["seed"] + r * 0x9E3779B9) % 2**32, (s["seed"] // 2**32 + r * 0xBB67AE85) % 2**32
                a, b = limbs(x[0], 0xD2511F53), limbs(x[2], 0xCD9E8D57)
                x = [b[0] ^ x[1] ^ key0, b[1], a[0] ^ x[3] ^ key1, a[1]]
            word = torch.stack(x)[(elements % 8) // 2, (elements >> 3) - (first >> 3)]
            halves.append((word >> (16 * (elements % 2))) % 65536)
        keep[first : first + count] = halves[0] * 65536 + halves[1] >= threshold
    return keep


def exact(case, seed):
    s = prepare(case, seed)
    if case["what"] == "dropout":
        x = s["x"].double()
        y = torch.where(_mask64(x.numel(), s).reshape(x.shape), x / (1.0 - s["p"]), 0.0)
        return y if s["add"] is None else y.add_(s["add"])
    ids = s["tokens_"]
    if case["what"] == "embed":
        y = torch.zeros((case["tokens"], case["dim"]), dtype=torch.float64, device="cuda")
        named = torch.nonzero(ids >= 0)[:, 0]
        rows = s["table"][ids[named].long()].double()
        if case["ecc"]:  # neighbours of a 16-bit float are whole steps of its bits apart
            digits, least = (7, 2.0**-126) if case["dtype"] == "bf16" else (10, 2.0**-14)
            step = torch.pow(2.0, torch.floor(torch.log2(rows.abs().clamp(min=least)))) * 2.0**-digits
            rows += s["codes"][ids[named].long()].double() * (step / 2) / (2 ** (case["ecc"] - 1) - 1)
        y[named] = rows * s["scale"]
        if s["p"]:
            y = torch.where(_mask64(y.numel(), s).reshape(y.shape), y / (1.0 - s["p"]), 0.0)
        return y
    total = s["grad"].double() if case["tied"] else torch.zeros((case["rows"], case["dim"]), dtype=torch.float64, device="cuda")
    dy = s["dy"].double() * s["scale"]
    if s["p"]:
        dy = torch.where(_mask64(dy.numel(), s).reshape(dy.shape), dy / (1.0 - s["p"]), 0.0)
    order = torch.argsort(ids, stable=True)
    order = order[ids[order] >= 0]
    return total.index_put_((ids[order].long(),), dy[order], accumulate=True)
