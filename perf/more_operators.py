"""Operators that models as they are published need of this path, as measurable cases: rotary
positions in either pair layout, over a part of the head and with frequencies scaled for long
contexts (new tokens, tokens appended to a paged cache, donor K/V scattered into one, K shifted in
place), and products with 4-bit weights that have a scale and a zero point per group.

With ``own`` false, ``run`` computes them from elementary torch operations in 32 bits (angles in
64); with ``own`` true it calls ``semblend_amd.rotary``, ``semblend_amd.quantized`` and the entry
points that take a rotary embedding.

Definitions. f_i are the model's fp32 frequencies, n of them: they turn the first 2n elements of a
head and leave the others as they are.
  * pairs: interleaved (2i, 2i + 1) or half (i, i + n); the angle is p * f_i, unrounded, and cosine
    and sine are multiplied by the embedding's factor (1 where a cached K is shifted, which holds it
    already).
  * scaled frequencies: with w_i = 2 pi / f_i the wavelength and L the trained length, f_i / s where
    w_i > L / lo, f_i where w_i < L / hi, and between them (1 - t) f_i / s + t f_i with
    t = (L / w_i - lo) / (hi - lo).
  * append: a token at position p goes to page ``table[p // bs]``, slot ``p % bs``, K (and Q) turned
    by p. Scatter: donor row d to position t, K turned by t - d. Shift: K at position p turned by
    its delta.
  * 4-bit weights: w[n, k] = (code[n, k] - zero[n, k // g]) * scale[n, k // g], codes and zeros whole
    numbers of 0 to 15 (8 where there are no zeros), scales in 16 bits; y = x w^T + bias.

Shapes: Qwen2.5-7B (28 query / 4 KV heads x 128, hidden 3584, 28 layers), Qwen2.5-0.5B (14 / 2 x
64) and Llama-3-8B (32 / 8 x 128, hidden 4096, 32 layers), as in the tests and the benchmark; the
other widths of weights are generic.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
QWEN7B = {"hq": 28, "hkv": 4, "d": 128, "base": 1e6}
QWEN05B = {"hq": 14, "hkv": 2, "d": 64, "base": 1e6}
LLAMA8B = {"hq": 32, "hkv": 8, "d": 128, "base": 5e5}
SHAPES = (QWEN7B, QWEN05B, LLAMA8B)


def listed() -> list[dict]:
    return [
        # One decode step's Q and K of a serving batch, turned before they are cached (latency).
        {"name": "rotate_decode_32", "kind": "rotate", "dtype": "bf16", "rows": 32, "ctx": 4000,
         "pairs": "half", "turned": 128, "scaled": False, "factor": 1.0, **QWEN7B},
        # Q and K of a long prompt, frequencies scaled for it.
        {"name": "rotate_prefill_8k", "kind": "rotate", "dtype": "bf16", "rows": 8192,
         "ctx": 131072, "pairs": "half", "turned": 128, "scaled": True, "factor": 1.0, **LLAMA8B},
        # A head of which the first half is turned, in fp32.
        {"name": "rotate_part_fp32", "kind": "rotate", "dtype": "fp32", "rows": 1501, "ctx": 4096,
         "pairs": "interleaved", "turned": 32, "scaled": False, "factor": 1.0, **QWEN05B},
        # One layer's K/V and Q of a batch of prompts, with a factor on cosine and sine.
        {"name": "append_half_4k", "kind": "append", "dtype": "bf16", "bs": 16, "requests": 4,
         "rows": 4602, "ctx": 9000, "pairs": "half", "turned": 128, "scaled": True, "factor": 1.21,
         **LLAMA8B},
        # A donor request's K/V of every layer into the new request's pages.
        {"name": "scatter_half_28_layers", "kind": "scatter", "dtype": "bf16", "bs": 16,
         "layers": 28, "rows": 6963, "ctx": 8192, "pairs": "half", "turned": 128, "scaled": False,
         "factor": 1.0, **QWEN7B},
        # K of loaded pages shifted in place, token by token.
        {"name": "shift_half_32_layers", "kind": "shift", "dtype": "fp16", "bs": 16, "layers": 32,
         "rows": 3001, "ctx": 4096, "pairs": "half", "turned": 128, "scaled": False, "factor": 1.0,
         **LLAMA8B},
        # The QKV projection of one chat's token (latency).
        {"name": "w4_qkv_1", "kind": "w4", "dtype": "bf16", "rows": 1, "inputs": 3584,
         "features": 4608, "group": 128, "zeros": True, "bias": True},
        # A wide layer of a small batch's decode step.
        {"name": "w4_wide_8", "kind": "w4", "dtype": "bf16", "rows": 8, "inputs": 3584,
         "features": 37888, "group": 128, "zeros": True, "bias": False},
        # A deep layer of a decode step, groups of 64.
        {"name": "w4_deep_16", "kind": "w4", "dtype": "bf16", "rows": 16, "inputs": 18944,
         "features": 3584, "group": 64, "zeros": True, "bias": False},
        # One token's logits over a large vocabulary, symmetric weights.
        {"name": "w4_head_1", "kind": "w4", "dtype": "fp16", "rows": 1, "inputs": 4096,
         "features": 131072, "group": 128, "zeros": False, "bias": False},
        # The QKV projection of a large batch's decode step, groups of 32.
        {"name": "w4_qkv_64", "kind": "w4", "dtype": "fp16", "rows": 64, "inputs": 4096,
         "features": 6144, "group": 32, "zeros": True, "bias": False},
        # The QKV projection of the rows that a 16K prompt does not reuse.
        {"name": "w4_prefill_2458", "kind": "w4", "dtype": "bf16", "rows": 2458, "inputs": 3584,
         "features": 4608, "group": 128, "zeros": True, "bias": True},
    ]


def _log(rng, lo: int, hi: int) -> int:
    """An integer spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    if rng.random() < 0.5:
        rows = rng.choice((rng.randint(1, 16), _log(rng, 1, 64), _log(rng, 65, 2400)))
        inputs = 32 * _log(rng, 8, 300 if rows > 64 else 600)
        features = _log(rng, 64, 8000 if rows > 64 else 40000)
        group = rng.choice([g for g in (32, 64, 128, 128) if inputs % g == 0])
        return {"kind": "w4", "dtype": rng.choice(("bf16", "bf16", "fp16")), "rows": rows,
                "inputs": inputs, "features": features, "group": group,
                "zeros": rng.random() < 0.7, "bias": rng.random() < 0.5}
    shape = dict(rng.choice(SHAPES))
    c = {"kind": rng.choice(("rotate", "rotate", "append", "scatter", "shift")),
         "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")), "bs": rng.choice((16, 16, 32)),
         "pairs": rng.choice(("half", "half", "interleaved")),
         "turned": shape["d"] // rng.choice((1, 1, 2)), "scaled": rng.random() < 0.5,
         "factor": 1.0, **shape}
    if c["kind"] == "rotate":
        c.update(rows=_log(rng, 1, 6000), ctx=_log(rng, 6000, 131072),
                 factor=rng.choice((1.0, 1.0, 1.21)))
    elif c["kind"] == "append":
        n = rng.choice((1, 1, 5, 33))
        c.update(requests=n, rows=rng.choice((n, _log(rng, n, 6000))), ctx=_log(rng, 300, 12000),
                 factor=rng.choice((1.0, 1.21)))
    else:
        rows = _log(rng, 1, 5000)
        c.update(rows=rows, ctx=rows + _log(rng, 1, 4000),
                 layers=rng.randint(1, max(1, min(32, 60000 // rows // (2 if c["dtype"] == "fp32"
                                                                        else 1)))))
    return c


# ---- inputs --------------------------------------------------------------------------------

def _frequencies(c) -> torch.Tensor:
    """The fp32 frequencies as a model keeps them."""
    n = c["turned"]
    f = 1.0 / (c["base"] ** (torch.arange(0, n, 2, dtype=torch.float32) / n))
    if not c["scaled"]:
        return f
    factor, lo, hi, length = 8.0, 1.0, 4.0, 8192.0
    wave = 2 * math.pi / f
    t = (length / wave - lo) / (hi - lo)
    between = (1 - t) * f / factor + t * f
    return torch.where(wave > length / lo, f / factor,
                       torch.where(wave < length / hi, f, between))


def _lengths(c) -> tuple[list[int], list[int]]:
    """(context length, new rows) of each request: contexts fall to a few per cent of the longest,
    every request has a row, and the rows left over go to every second request."""
    n, ctx = c["requests"], c["ctx"]
    lens = [max(1, int(ctx * (1.0 - 0.97 * i / max(1, n - 1)))) for i in range(n)]
    rows, left = [1] * n, c["rows"] - n
    for i in range(0, n, 2):
        take = min(left if i + 2 >= n else left // 2, lens[i] - 1)
        rows[i] += take
        left -= take
    return lens, rows


def _inputs(case, seed: int) -> dict:
    c = case
    host = torch.Generator("cpu").manual_seed(seed)
    gpu = torch.Generator("cuda").manual_seed(seed)
    dt = DTYPES[c["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=gpu, device="cuda", dtype=dt)

    s = {"case": dict(c)}
    if c["kind"] == "w4":
        n, k, g = c["features"], c["inputs"], c["group"]
        s["x"] = randn(c["rows"], k)
        # codes as a rounded normal weight leaves them: the middle ones more often than the ends
        codes = torch.empty((n, k), dtype=torch.uint8, device="cuda")
        for part in codes.view(-1).split(1 << 26):
            w = torch.randn(part.shape, generator=gpu, device="cuda", dtype=torch.float16)
            part.copy_(w.mul_(2.8).add_(8.0).round_().clamp_(0, 15))
        s["codes"] = codes
        u = torch.rand((n, k // g), generator=gpu, device="cuda")
        s["scales"] = ((0.5 + u) * (0.36 / math.sqrt(k))).to(dt)
        s["zeros"] = torch.randint(5, 11, (n, k // g), generator=gpu, device="cuda",
                                   dtype=torch.int32).to(torch.uint8) if c["zeros"] else None
        s["bias"] = randn(n) if c["bias"] else None
        return s
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    s["freq"] = _frequencies(c)
    if c["kind"] == "rotate":
        pos = torch.randint(0, c["ctx"], (1,), generator=host)
        pos = torch.randint(0, c["ctx"], (c["rows"],), generator=host) if c["rows"] <= 64 else \
            (pos + torch.arange(c["rows"])) % c["ctx"]
        s["pos"] = pos.to(torch.int32).cuda()
        s["q"], s["k"] = randn(c["rows"], hq, d), randn(c["rows"], hkv, d)
        return s
    bs = c["bs"]
    lens, rows = _lengths(c) if c["kind"] == "append" else ([c["ctx"]], [c["rows"]])
    need = [-(-n // bs) for n in lens]
    pool = sum(need) + sum(need) // 16 + 3
    perm = torch.randperm(pool, generator=host).to(torch.int32)
    tables = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for i, b in enumerate(need):
        tables[i, :b] = perm[at:at + b]
        at += b
    s["tables"] = tables.cuda()
    if c["kind"] == "append":
        s["single"] = max(rows) == 1
        s["starts"] = torch.tensor([0] + rows).cumsum(0).to(torch.int32).cuda()
        s["pos"] = torch.cat([torch.arange(n - r, n) for n, r in zip(lens, rows)]
                             ).to(torch.int32).cuda()
        total = sum(rows)
        s["cache"] = randn(pool, 2, hkv, bs, d)
        s["q"], s["k"], s["v"] = randn(total, hq, d), randn(total, hkv, d), randn(total, hkv, d)
        return s
    # one tensor holds every layer's cache; a layer's pages lie as an engine keeps them
    s["caches"] = torch.cat([randn(1, 2, pool, bs, hkv, d) for _ in range(c["layers"])])
    chosen = torch.randperm(c["ctx"], generator=host)[:c["rows"]].sort().values
    delta = torch.randint(-2048, 2049, (c["ctx"] // 256 + 1,), generator=host)[chosen // 256]
    if c["kind"] == "shift":
        s["pos"], s["delta"] = chosen.to(torch.int32), delta.to(torch.int32)   # the host's lists
    else:
        s["to"] = chosen.to(torch.int32).cuda()
        s["from"] = torch.remainder(chosen - delta, c["ctx"]).to(torch.int32).cuda()
        s["donors"] = torch.cat([randn(1, 2, hkv, c["ctx"], d) for _ in range(c["layers"])])
    return s


def prepare(case, seed: int) -> dict:
    s = _inputs(case, seed)
    if own and case["kind"] == "w4":
        from semblend_amd import quantized

        s["api"] = quantized
        s["handle"] = quantized.QuantizedLinear(s["codes"], s["scales"], s["zeros"])
    elif own:
        from semblend_amd import paged_cache, rope_correction, rotary

        s["api"] = {"rotate": rotary, "append": paged_cache}.get(case["kind"], rope_correction)
        s["rotary"] = rotary.RotaryEmbedding(s["freq"], case["d"], layout=case["pairs"],
                                             factor=case["factor"])
        if "caches" in s:
            s["layers"] = [x.permute(1, 0, 3, 2, 4) for x in s["caches"].unbind(0)]
        if "donors" in s:
            s["donor_layers"] = list(s["donors"].unbind(0))
    return s


# ---- one pass ------------------------------------------------------------------------------

def _run_own(s):
    api, kind = s["api"], s["case"]["kind"]
    if kind == "w4":
        return api.quantized_linear(s["x"], s["handle"], bias=s["bias"])
    if kind == "rotate":
        return api.apply_rotary(s["q"], s["pos"], s["rotary"], key=s["k"])
    if kind == "append":
        q = api.append_kv_paged(s["cache"], s["k"], s["v"], s["tables"], s["pos"],
                                row_starts=None if s["single"] else s["starts"],
                                rotary=s["rotary"], query=s["q"])
        return q, s["cache"]
    if kind == "scatter":
        api.rope_correct_scatter_paged_layers(s["layers"], s["donor_layers"], s["tables"][0],
                                              s["from"], s["to"], rotary=s["rotary"])
    else:
        api.apply_rope_deltas_inplace_layers(s["layers"], s["tables"][0], s["pos"], s["delta"],
                                             layout="standard", rotary=s["rotary"])
    return s["caches"]


def _turn(s, x: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
    """x [..., T, H, D] turned by pos [T], in 32 bits; angles, cosine and sine in 64."""
    c = s["case"]
    n = c["turned"]
    angle = pos.double()[:, None] * s["freq"].cuda().double()
    cos = (angle.cos() * c["factor"]).float()[:, None]
    sin = (angle.sin() * c["factor"]).float()[:, None]
    x = x.float()
    if c["pairs"] == "half":
        a, b = x[..., :n // 2], x[..., n // 2:n]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    else:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    return torch.cat([turned, x[..., n:]], dim=-1)


def _run_plain(s):
    c = s["case"]
    kind = c["kind"]
    dt = DTYPES[c["dtype"]]
    if kind == "w4":
        zero = s["zeros"].float() if c["zeros"] else torch.full_like(s["scales"], 8.0).float()
        w = s["codes"].float().unflatten(1, (-1, c["group"]))
        w = ((w - zero[..., None]) * s["scales"].float()[..., None]).flatten(1)
        y = s["x"].float() @ w.t()
        return (y + s["bias"].float() if c["bias"] else y).to(dt)
    if kind == "rotate":
        return _turn(s, s["q"], s["pos"]).to(dt), _turn(s, s["k"], s["pos"]).to(dt)
    bs = c["bs"]
    if kind == "append":
        p = s["pos"].long()
        req = torch.repeat_interleave(torch.arange(s["tables"].shape[0], device="cuda"),
                                      s["starts"].diff().long(), output_size=p.shape[0])
        page, slot = s["tables"].long()[req, p // bs], p % bs
        s["cache"][page, 0, :, slot] = _turn(s, s["k"], p).to(dt)
        s["cache"][page, 1, :, slot] = s["v"]
        return _turn(s, s["q"], p).to(dt), s["cache"]
    if kind == "scatter":
        t, d = s["to"].long(), s["from"].long()
        page, slot = s["tables"][0].long()[t // bs], t % bs
        rows = s["donors"][:, :, :, d].transpose(2, 3)                  # [L, 2, T, H, D]
        s["caches"][:, 0, page, slot] = _turn(s, rows[:, 0], t - d).to(dt)
        s["caches"][:, 1, page, slot] = rows[:, 1]
        return s["caches"]
    p, delta = s["pos"].cuda().long(), s["delta"].cuda()
    page, slot = s["tables"][0].long()[p // bs], p % bs
    s["caches"][:, 0, page, slot] = _turn(s, s["caches"][:, 0, page, slot], delta).to(dt)
    return s["caches"]


def run(s):
    return _run_own(s) if own else _run_plain(s)


# ---- work ----------------------------------------------------------------------------------

def work(case) -> dict:
    c = case
    es = 4 if c["dtype"] == "fp32" else 2
    if c["kind"] == "w4":
        m, n, k = c["rows"], c["features"], c["inputs"]
        groups = n * (k // c["group"])
        weights = n * k / 2 + groups * (2 + (0.5 if c["zeros"] else 0))
        return {"bytes": int(weights) + (m * k + m * n + (n if c["bias"] else 0)) * es,
                "flops": 2 * m * n * k}
    hq, hkv, d, n = c["hq"], c["hkv"], c["d"], c["turned"]
    if c["kind"] == "rotate":
        rows = c["rows"] * (hq + hkv)
        return {"bytes": 2 * rows * d * es, "flops": 3 * rows * n}
    if c["kind"] == "append":
        total = sum(_lengths(c)[1])
        return {"bytes": 2 * total * (hq + 2 * hkv) * d * es, "flops": 3 * total * (hq + hkv) * n}
    rows = c["rows"] * c["layers"] * hkv
    if c["kind"] == "scatter":
        return {"bytes": 4 * rows * d * es, "flops": 3 * rows * n}
    return {"bytes": 2 * rows * n * es, "flops": 3 * rows * n}


# ---- the same in 64 bits -------------------------------------------------------------------

def _exact_turn(c, freq: torch.Tensor, x: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
    """x [T, H, D]: each pair a complex number, times factor * exp(i angle), in 64 bits."""
    n = c["turned"]
    z = x.double()
    first = torch.arange(0, n, 2) if c["pairs"] == "interleaved" else torch.arange(n // 2)
    second = first + (1 if c["pairs"] == "interleaved" else n // 2)
    w = torch.polar(torch.full((), c["factor"], dtype=torch.float64, device=x.device),
                    torch.outer(pos.double(), freq.double().to(x.device)))
    pair = torch.complex(z[..., first], z[..., second]) * w[:, None, :]
    z[..., first], z[..., second] = pair.real, pair.imag
    return z


def exact(case, seed: int):
    s = _inputs(case, seed)
    c = case
    if c["kind"] == "w4":
        n, k, g = c["features"], c["inputs"], c["group"]
        x = s["x"].double()
        parts = []
        for a in range(0, n, 16384):
            rows = slice(a, min(n, a + 16384))
            scale = s["scales"][rows].double().repeat_interleave(g, dim=1)
            if c["zeros"]:
                off = s["zeros"][rows].double().repeat_interleave(g, dim=1) * scale
            else:
                off = 8 * scale
            parts.append(torch.addmm(torch.zeros((), dtype=torch.float64, device="cuda"), x,
                                     (s["codes"][rows].double() * scale - off).t().contiguous()))
        y = torch.cat(parts, dim=1)
        return y if s["bias"] is None else y + s["bias"].double()
    freq = s["freq"]
    if c["kind"] == "rotate":
        return _exact_turn(c, freq, s["q"], s["pos"]), _exact_turn(c, freq, s["k"], s["pos"])
    bs = c["bs"]
    if c["kind"] == "append":
        cache = s["cache"].double()
        k, at = _exact_turn(c, freq, s["k"], s["pos"]), 0
        for i, r in enumerate(_lengths(c)[1]):
            p = s["pos"][at:at + r].long()
            page = s["tables"][i].long().index_select(0, torch.div(p, bs, rounding_mode="floor"))
            cache[page, 0, :, p % bs] = k[at:at + r]
            cache[page, 1, :, p % bs] = s["v"][at:at + r].double()
            at += r
        return _exact_turn(c, freq, s["q"], s["pos"]), cache
    caches = s["caches"].double()
    p = (s["to"] if c["kind"] == "scatter" else s["pos"].cuda()).long()
    page = s["tables"][0].long().index_select(0, torch.div(p, bs, rounding_mode="floor"))
    for layer in range(c["layers"]):
        if c["kind"] == "scatter":
            d = s["from"].long()
            k = s["donors"][layer, 0].index_select(1, d).transpose(0, 1)
            caches[layer, 0, page, p % bs] = _exact_turn(c, freq, k, p - d)
            caches[layer, 1, page, p % bs] = \
                s["donors"][layer, 1].index_select(1, d).transpose(0, 1).double()
        else:
            k = caches[layer, 0, page, p % bs]
            caches[layer, 0, page, p % bs] = _exact_turn(c, freq, k, s["delta"].cuda())
    return caches
