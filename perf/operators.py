"""The 8-bit serving operators: what they compute, and the cases they are measured on.

Four operators that follow one another in a layer that serves in 8 bits: the RMS norm that adds
the residual and leaves 8-bit codes with a scale for each token, the 8-bit integer product with
scales for each token and channel, the K/V cache that is quantised as it is written (a scale for
each block of tokens and head) and read back, and attention over that cache. `run` computes them
in plain torch operations, or through `kinomlx_b200.ops_q8` where `own` is true.

int8 codes come back as bf16 values of the codes (whole numbers up to 127 are exact there) beside
their scales; e4m3 codes as the float8 tensors they are.
"""

from __future__ import annotations

import math

import torch

own = False

BF16 = torch.bfloat16
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}
LEAST_SCALE = 2.0**-126  # below it a group counts as zero
EPS = 1e-6


# ---------------------------------------------------------------- cases
def listed() -> list[dict]:
    return [
        # a decode batch of 16 tokens at the video model's width: latency
        dict(name="norm_tokens16", op="norm", rows=16, dim=4096, dtype="e4m3", residual=True,
             weight=True),
        # every video token of one step
        dict(name="norm_video", op="norm", rows=9216, dim=4096, dtype="e4m3", residual=True,
             weight=True),
        # the fused q, k, v projection of four decoded tokens: streams the weight
        dict(name="product_tokens4", op="product", m=4, n=12288, k=4096, bias=False),
        # the audio stream's feed-forward: 126 tokens, ragged against every tile
        dict(name="product_audio", op="product", m=126, n=8192, k=2048, bias=True),
        # the video stream's feed-forward
        dict(name="product_video", op="product", m=9216, n=16384, k=4096, bias=True),
        # one new token for each of 64 sequences, blocks part full
        dict(name="cache_append", op="write", batch=64, new=1, ragged=False, cached=2048, heads=8,
             dim=128, block=64, dtype="e4m3"),
        # the keys and values of an image and its text, written at once
        dict(name="cache_fill", op="write", batch=2, new=4608, ragged=False, cached=0, heads=24,
             dim=128, block=64, dtype="e4m3"),
        # a cache taken back to bf16
        dict(name="cache_read", op="read", batch=4, cached=9216, heads=8, dim=128, block=32,
             dtype="int8"),
        # a small decode batch over short caches: latency
        dict(name="attend_tokens", op="attend", batch=8, new=1, ragged=False, cached=1000, heads=8,
             group=4, dim=128, block=64, dtype="int8", causal=True),
        # long caches, one token each: the cache's bytes
        dict(name="attend_long", op="attend", batch=16, new=1, ragged=False, cached=32768, heads=8,
             group=4, dim=128, block=64, dtype="int8", causal=True),
        # prompts of several lengths taken in by chunks
        dict(name="attend_chunk", op="attend", batch=4, new=1024, ragged=True, cached=8192, heads=8,
             group=4, dim=128, block=32, dtype="e4m3", causal=True),
        # image and text queries over their own and a reference image's keys
        dict(name="attend_image", op="attend", batch=1, new=4608, ragged=False, cached=9216,
             heads=24, group=1, dim=128, block=128, dtype="int8", causal=False),
    ]


def _log(rng, low: int, high: int) -> int:
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng) -> dict:
    op = rng.choice(["norm", "product", "write", "read", "attend"])
    dtype = rng.choice(["int8", "e4m3"])
    if op == "norm":
        dim = 8 * _log(rng, 8, 1024)
        return dict(op=op, rows=_log(rng, 1, min(32768, 9216 * 4096 // dim)), dim=dim, dtype=dtype,
                    residual=rng.random() < 0.6, weight=rng.random() < 0.7)
    if op == "product":
        n, k = 8 * _log(rng, 8, 2048), 16 * _log(rng, 4, 1024)
        return dict(op=op, m=_log(rng, 1, min(9216, 9216 * 16384 * 4096 // (n * k))), n=n, k=k,
                    bias=rng.random() < 0.5)
    shape = dict(dim=rng.choice([64, 128]), block=rng.choice([16, 32, 64, 128]), dtype=dtype)
    if op == "write":
        batch, heads = _log(rng, 1, 64), rng.randint(1, 24)
        new = _log(rng, 1, max(1, 9216 // batch))
        return dict(op=op, batch=batch, new=new, ragged=rng.random() < 0.5,
                    cached=_log(rng, 1, 2048) - 1, heads=heads, **shape)
    if op == "read":
        batch, heads = _log(rng, 1, 16), rng.randint(1, 16)
        return dict(op=op, batch=batch, cached=_log(rng, 1, 4 * 9216 * 8 // (batch * heads)),
                    heads=heads, **shape)
    group, heads = rng.choice([1, 1, 2, 3, 4, 5, 6, 7, 8]), rng.randint(1, 12)
    batch = _log(rng, 1, 32)
    new = 1 if rng.random() < 0.4 else _log(rng, 1, 2048)
    most = min(32768, 16 * 32768 * 8 // (2 * batch * heads),
               24 * 4608 * 9216 // (batch * heads * group * new))
    new = min(new, max(1, most))
    cached = max(new, _log(rng, 1, max(2, most)))
    return dict(op=op, batch=batch, new=new, ragged=rng.random() < 0.5, cached=cached, heads=heads,
                group=group, causal=rng.random() < 0.7, **shape)


# ---------------------------------------------------------------- lengths: a case's own, not the seed's
def _new_tokens(c: dict) -> list[int]:
    """New tokens of each sequence: `new`, or spread from 1 to `new`."""
    if not c["ragged"]:
        return [c["new"]] * c["batch"]
    return [max(1, c["new"] - (b * 37 + c["new"] // 3 * b) % c["new"]) for b in range(c["batch"])]


def _lengths(c: dict) -> list[int]:
    """Tokens that each sequence has in the cache (for `write`: before it), the first one `cached`."""
    spread = max(1, c["cached"] // 2)
    return [c["cached"] - (b * 97 + b * b * 13) % spread for b in range(c["batch"])]


def _tokens(c: dict) -> tuple[list[int], list[int]]:
    """New tokens, and the cache's lengths when the operator is done."""
    if c["op"] == "read":
        return [0] * c["batch"], _lengths(c)
    new = _new_tokens(c)
    if c["op"] == "write":
        return new, [n + length for n, length in zip(new, _lengths(c))]
    return new, [max(n, length) for n, length in zip(new, _lengths(c))]


def _pairs(c: dict) -> int:
    """Query-key pairs of one head that the mask leaves."""
    new, total = _tokens(c)
    if not c["causal"]:
        return sum(n * t for n, t in zip(new, total))
    return sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, total))


def work(case: dict) -> dict:
    c = case
    if c["op"] == "norm":
        e = c["rows"] * c["dim"]
        nbytes = e * (7 if c["residual"] else 3) + 4 * c["rows"] + 2 * c["dim"] * c["weight"]
        return {"bytes": nbytes, "flops": 6 * e}
    if c["op"] == "product":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": m * k + n * k + 2 * m * n + 4 * (m + n) + 2 * n * c["bias"],
                "flops": 2 * m * n * k}
    new, total = _tokens(c)
    width = c["heads"] * c["dim"]
    if c["op"] == "write":
        blocks = sum((t - 1) // c["block"] - (t - n) // c["block"] + 1 for n, t in zip(new, total))
        return {"bytes": 2 * 3 * sum(new) * width + 2 * 8 * blocks * c["heads"],
                "flops": 2 * 3 * sum(new) * width}
    blocks = sum(-(-t // c["block"]) for t in total)
    if c["op"] == "read":
        return {"bytes": 2 * sum(total) * width + 2 * 2 * c["batch"] * max(total) * width
                + 2 * 4 * blocks * c["heads"], "flops": 2 * sum(total) * width}
    q = sum(new) * width * c["group"]
    return {"bytes": 2 * sum(total) * width + 2 * 4 * blocks * c["heads"] + 4 * q,
            "flops": 4 * c["dim"] * c["heads"] * c["group"] * _pairs(c)}


# ---------------------------------------------------------------- inputs
def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, g, std=1.0, dtype=BF16) -> torch.Tensor:
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _random_codes(shape, dtype: str, g) -> torch.Tensor:
    """Codes of normal values whose largest of a few thousand takes the top code."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16)
    if dtype == "int8":
        return (x * 33).round().clamp(-127, 127).to(torch.int8)
    return (x * 118).clamp(-448, 448).to(torch.float8_e4m3fn)


def _random_scales(shape, dtype: str, g) -> torch.Tensor:
    spread = torch.rand(shape, generator=g, device="cuda") + 0.5
    return spread * (4.0 / TOP[dtype])


def _int32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case: dict, seed: int) -> dict:
    c, g = case, _generator(seed)
    if c["op"] == "norm":
        s = {"x": _normal((c["rows"], c["dim"]), g), "residual": None, "weight": None}
        if c["residual"]:
            s["residual"] = _normal((c["rows"], c["dim"]), g, 3.0)
        if c["weight"]:
            s["weight"] = 1 + _normal((c["dim"],), g, 0.2)
        return {"case": c, **s}
    if c["op"] == "product":
        return {
            "case": c,
            "codes": _random_codes((c["m"], c["k"]), "int8", g),
            "scales": _random_scales((c["m"],), "int8", g),
            "w_codes": _random_codes((c["n"], c["k"]), "int8", g),
            "w_scales": _random_scales((c["n"],), "int8", g) * c["k"] ** -0.5,
            "bias": _normal((c["n"],), g, 0.1) if c["bias"] else None,
        }
    new, total = _tokens(c)
    per = [max(1, -(-t // c["block"])) for t in total]
    pages = torch.randperm(sum(per), generator=g, device="cuda").to(torch.int32)
    # the blocks of every sequence in any order, and one block more that no sequence has
    table = torch.full((c["batch"], max(per)), sum(per), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = pages[at:at + n]
        at += n
    shape = (sum(per) + 1, c["heads"], c["block"], c["dim"])
    s = {"case": c, "table": table, "most_new": max(new), "most": max(total)}
    for name in ("k", "v"):
        s[name + "_codes"] = _random_codes(shape, c["dtype"], g)
        s[name + "_scales"] = _random_scales(shape[:2], c["dtype"], g)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s["starts"] = _int32(starts) if c.get("ragged") else None
    s["lengths"] = _int32([t - n for n, t in zip(new, total)] if c["op"] == "write" else total)
    if c["op"] == "write":
        s["k"] = _normal((sum(new), c["heads"], c["dim"]), g)
        s["v"] = _normal((sum(new), c["heads"], c["dim"]), g, 0.7)
    if c["op"] == "attend":
        s["q"] = _normal((sum(new), c["heads"] * c["group"], c["dim"]), g)
    return s


# ---------------------------------------------------------------- plain forms
def _values(codes: torch.Tensor) -> torch.Tensor:
    """What run() returns for codes: int8 as bf16 values, e4m3 as they are."""
    return codes.to(BF16) if codes.dtype == torch.int8 else codes


def _encode(y: torch.Tensor, dtype: str) -> torch.Tensor:
    if dtype == "int8":
        return y.round().clamp(-127, 127).to(torch.int8)
    return y.clamp(-448, 448).to(torch.float8_e4m3fn)


def _scale_of(amax: torch.Tensor, dtype: str) -> torch.Tensor:
    scale = amax / TOP[dtype]
    scale = torch.where(scale < LEAST_SCALE, 0.0, scale)
    return torch.where(amax.isfinite(), scale, math.nan)


def _inverse(scale: torch.Tensor) -> torch.Tensor:
    return torch.where(scale > 0, 1.0 / scale, 0.0)


def _norm(s: dict):
    c, x = s["case"], s["x"]
    hidden = x if s["residual"] is None else (x.float() + s["residual"].float()).to(BF16)
    y = hidden.double()  # values next to a border of the codes
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)
    if s["weight"] is not None:
        y = y * s["weight"].double()
    scale = _scale_of(y.abs().amax(-1), c["dtype"])
    codes = _encode((y * _inverse(scale)[:, None]).float(), c["dtype"])
    return {"codes": _values(codes), "scales": scale.float(), "hidden": hidden}


def _product(s: dict):
    acc = s["codes"].float() @ s["w_codes"].float().T
    out = acc * s["scales"][:, None] * s["w_scales"][None, :]
    if s["bias"] is not None:
        out = out + s["bias"].float()
    return out.to(BF16)


def _row_of(s: dict, rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(first row, rows) of each sequence."""
    if s["starts"] is None:
        each = rows // s["case"]["batch"]
        first = torch.arange(s["case"]["batch"], device="cuda") * each
        return first, torch.full_like(first, each)
    return s["starts"][:-1].long(), (s["starts"][1:] - s["starts"][:-1]).long()


def _write_one(s: dict, name: str) -> None:
    c, x = s["case"], s[name]
    codes, scales, block = s[name + "_codes"], s[name + "_scales"], c["block"]
    first, new = _row_of(s, x.shape[0])
    length = s["lengths"].long()
    touched = (s["most_new"] + block - 2) // block + 1  # blocks that a sequence's tokens may fall into
    index = length[:, None] // block + torch.arange(touched, device="cuda")
    at = index[..., None] * block + torch.arange(block, device="cuda")  # positions (batch, blocks, slots)
    fresh = (at >= length[:, None, None]) & (at < (length + new)[:, None, None])
    earlier = at < length[:, None, None]
    some = fresh.any(-1)
    page = s["table"].long().gather(1, index.clamp(max=s["table"].shape[1] - 1))
    page = torch.where(some, page, codes.shape[0] - 1)
    row = (first[:, None, None] + at - length[:, None, None]).clamp(0, x.shape[0] - 1)
    values = torch.where(fresh[..., None, None], x[row].float(), 0.0)  # (batch, blocks, slots, heads, dim)
    before = torch.where(earlier.any(-1)[..., None], scales[page], 0.0)
    scale = torch.maximum(_scale_of(values.abs().amax((2, 4)), c["dtype"]), before)
    grown = torch.where(scale > before, before * _inverse(scale), 1.0)  # of the earlier codes
    old = codes[page].transpose(2, 3).float()
    mixed = torch.where(fresh[..., None, None], values * _inverse(scale)[:, :, None, :, None],
                        old * grown[:, :, None, :, None])
    kept = codes.view(torch.uint8)[page].transpose(2, 3)
    fill = torch.where((fresh | earlier)[..., None, None],
                       _encode(mixed, c["dtype"]).view(torch.uint8), kept)
    codes.view(torch.uint8)[page] = fill.transpose(2, 3).contiguous()
    scales[page] = scale


def _cache_out(s: dict) -> dict:
    out = {}
    for name in ("k", "v"):  # without the block that no sequence has
        out[name + "_codes"] = _values(s[name + "_codes"][:-1])
        out[name + "_scales"] = s[name + "_scales"][:-1]
    return out


def _write(s: dict):
    _write_one(s, "k")
    _write_one(s, "v")
    return _cache_out(s)


def _dense(s: dict, name: str) -> torch.Tensor:
    """(batch, heads, tokens, dim) fp32 values of the cache, zeros past the lengths."""
    page, most = s["table"].long(), s["most"]
    x = s[name + "_codes"][page].float() * s[name + "_scales"][page][..., None, None]
    x = x.transpose(1, 2).flatten(2, 3)[:, :, :most]
    inside = torch.arange(most, device="cuda") < s["lengths"][:, None]
    return torch.where(inside[:, None, :, None], x, 0.0)


def _read(s: dict):
    return tuple(_dense(s, name).transpose(1, 2).to(BF16).contiguous() for name in ("k", "v"))


def _attend(s: dict):
    c, q, most = s["case"], s["q"], s["most"]
    first, new = _row_of(s, q.shape[0])
    token = torch.arange(s["most_new"], device="cuda")
    row = (first[:, None] + token).clamp(max=q.shape[0] - 1)
    x = q[row].float().unflatten(2, (c["heads"], c["group"]))  # (batch, tokens, heads, group, dim)
    x = x.permute(0, 2, 3, 1, 4).flatten(2, 3) * c["dim"] ** -0.5
    scores = x @ _dense(s, "k").transpose(2, 3)  # (batch, heads, group * tokens, keys)
    seen = torch.arange(most, device="cuda") < s["lengths"][:, None, None]
    if c["causal"]:
        position = s["lengths"][:, None].long() - new[:, None] + token
        seen = seen & (torch.arange(most, device="cuda") <= position[..., None])
    scores = scores.unflatten(2, (c["group"], s["most_new"]))
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top.isfinite(), top, 0.0)).exp_()
    total = scores.sum(-1, keepdim=True)
    y = scores.flatten(2, 3) @ _dense(s, "v")
    y = y.unflatten(2, (c["group"], s["most_new"])) / torch.where(total > 0, total, 1.0)
    y = y.permute(0, 3, 1, 2, 4).flatten(2, 3).to(BF16)  # (batch, tokens, query heads, dim)
    at = torch.arange(q.shape[0], device="cuda")
    batch = torch.searchsorted(first + new, at, right=True)
    return y[batch, at - first[batch]]


PLAIN = {"norm": _norm, "product": _product, "write": _write, "read": _read, "attend": _attend}


# ---------------------------------------------------------------- the framework's calls
def _run_own(s: dict):
    from kinomlx_b200 import ops_q8

    c = s["case"]
    if c["op"] == "norm":
        codes, scales, hidden = ops_q8.rms_norm_quantize(
            s["x"], s["weight"], EPS, residual=s["residual"], dtype=CODES[c["dtype"]])
        return {"codes": _values(codes), "scales": scales, "hidden": hidden}
    if c["op"] == "product":
        return ops_q8.linear_int8(s["codes"], s["scales"], s["w_codes"], s["w_scales"], s["bias"])
    cache = ops_q8.KVCache(s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"])
    if c["op"] == "write":
        ops_q8.kv_cache_write(cache, s["k"], s["v"], s["table"], s["lengths"], s["starts"])
        return _cache_out(s)
    if c["op"] == "read":
        return ops_q8.kv_cache_read(cache, s["table"], s["lengths"], s["most"])
    return ops_q8.kv_cache_attention(s["q"], cache, s["table"], s["lengths"], s["starts"],
                                     causal=c["causal"])


def run(state: dict):
    if own:
        return _run_own(state)
    return PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------- the definition in 64 bits
def _exact_code(y: torch.Tensor, dtype: str) -> torch.Tensor:
    """The code's value nearest to y, ties to even."""
    if dtype == "int8":
        return y.round().clamp(-127, 127)
    _, exponent = torch.frexp(y.abs().clamp(max=448.0, min=2.0**-6))
    step = torch.ldexp(torch.ones_like(y), exponent - 4)  # four significant bits, least 2^-9
    return ((y / step).round() * step).clamp(-448, 448)


def _exact_block(old: torch.Tensor, before: torch.Tensor, x: torch.Tensor, dtype: str):
    """Codes of one block (heads, slots, dim) after tokens x (heads, tokens, dim) follow the old
    ones (heads, slots, dim), with its scale for each head."""
    scale = x.abs().amax((1, 2)) / TOP[dtype]
    scale = torch.maximum(scale, before)
    ratio = (before / scale)[:, None, None]
    old = torch.where(ratio < 1, _exact_code(old * ratio, dtype), old)
    return torch.cat([old, _exact_code(x / scale[:, None, None], dtype)], 1), scale


def exact(case: dict, seed: int):
    c, s = case, prepare(case, seed)
    if c["op"] == "norm":
        full = s["x"].double() + (s["residual"].double() if c["residual"] else 0)
        h = full.to(BF16).double()  # what the norm takes is what the next layer reads
        y = h / torch.sqrt(h.pow(2).mean(-1, keepdim=True) + EPS)
        if c["weight"]:
            y = y * s["weight"].double()
        scale = y.abs().max(-1).values / TOP[c["dtype"]]
        return {"codes": _exact_code(y / scale[:, None], c["dtype"]), "scales": scale,
                "hidden": full}
    if c["op"] == "product":
        w = s["w_codes"].double() * s["w_scales"].double()[:, None]
        out = torch.mm(s["codes"].double() * s["scales"].double()[:, None], w.t())
        return out + s["bias"].double() if c["bias"] else out
    new, total = _tokens(c)
    table, block = s["table"].tolist(), c["block"]
    if c["op"] == "write":
        if sum((t - 1) // block - (t - n) // block + 1 for n, t in zip(new, total)) > 2000:
            return None
        out = {}
        for name in ("k", "v"):
            codes = s[name + "_codes"][:-1].double()
            scales = s[name + "_scales"][:-1].double()
            at = 0
            for b, (n, t) in enumerate(zip(new, total)):
                x = s[name][at:at + n].double().transpose(0, 1)
                at += n
                for j in range((t - n) // block, (t - 1) // block + 1):
                    begin, end = max(t - n, j * block), min(t, (j + 1) * block)
                    held, page = begin - j * block, table[b][j]
                    piece, scale = _exact_block(
                        codes[page, :, :held], scales[page] if held else 0 * scales[page],
                        x[:, begin - (t - n):end - (t - n)], c["dtype"])
                    codes[page, :, :end - j * block] = piece
                    scales[page] = scale
            out |= {name + "_codes": codes, name + "_scales": scales}
        return out

    def cached(name: str, b: int) -> torch.Tensor:  # (heads, tokens, dim)
        blocks = [s[name + "_codes"][p].double() * s[name + "_scales"][p].double()[:, None, None]
                  for p in table[b][:-(-total[b] // block)]]
        if not blocks:
            return torch.zeros((c["heads"], 0, c["dim"]), dtype=torch.float64, device="cuda")
        return torch.cat(blocks, 1)[:, :total[b]]

    if c["op"] == "read":
        out = []
        for name in ("k", "v"):
            y = torch.zeros((c["batch"], max(total), c["heads"], c["dim"]), dtype=torch.float64,
                            device="cuda")
            for b in range(c["batch"]):
                y[b, :total[b]] = cached(name, b).transpose(0, 1)
            out.append(y)
        return tuple(out)
    out, at = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for b, (n, t) in enumerate(zip(new, total)):
        k, v = cached("k", b), cached("v", b)
        mask = torch.zeros((n, t), dtype=torch.float64, device="cuda")
        if c["causal"]:
            mask += torch.full((n, t), -math.inf, dtype=torch.float64,
                               device="cuda").triu(t - n + 1)
        for h in range(c["heads"] * c["group"]):
            kv = h // c["group"]
            score = s["q"][at:at + n, h].double() @ k[kv].T / math.sqrt(c["dim"]) + mask
            out[at:at + n, h] = torch.softmax(score, -1) @ v[kv]
        at += n
    return out
