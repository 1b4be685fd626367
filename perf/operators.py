"""Rotary positions, the paged 4-bit cache and the attention that reads it, as measurable cases.

Three operators, each through the public entry points where ``own`` is set
and in elementary torch operations where it is not:

  rotary  ``apply_rotary_positions``: rotation of q and k by their positions,
          half or interleaved pairs, the whole head or its first columns,
          frequencies scaled for long contexts; forward, or forward and
          backward of a training step.
  append  ``append_paged``: the keys and values of new tokens, the keys
          rotated on the way, into a paged cache held in 4 bits (and the new
          queries rotated beside them), then ``read_paged`` of the stored
          rows: the values that the 4 bits stand for.
  attend  ``attend_paged``: attention of the newest queries over that cache.

The cache: page ids come from a table (B, pages a sequence) of int32; a page
holds P tokens of every key/value head as e2m1 values (1 sign, 2 exponent, 1
mantissa bit) in blocks of 32 along D that share a power of two:

  k_codes  (N, Hk, P, D / 2)            token t, byte d / 2, low half: even d
  k_scales (N, Hk, P, D / 32)           exponent + 127
  v_codes  (N, Hk, P / 4, 16, 4, D/32)  token 4a + r, d = (D / 16) m + j at
                                        [a, m, r, j / 2], low half: even j
  v_scales (N, Hk, P / 4, D / 32, 4)    token 4a + r at [a, block, r]

A block's exponent is floor(log2 max|x|) - 2, its values x / 2^exponent
rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code,
6 above).
"""
from __future__ import annotations

import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "flash-attn-volta_amd"))

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
FACTOR, ORIGINAL = 8.0, 8192        # context scaling: 8 times the 8192 positions trained on
BASE = 500000.0


def _rotary(B, S, H, Hk, D, R, pairs, scaling, first, train, dtype, layout="bshd"):
    return {"op": "rotary", "B": B, "S": S, "H": H, "Hk": Hk, "D": D, "R": R, "pairs": pairs,
            "scaling": scaling, "first": first, "train": train, "dtype": dtype, "layout": layout}


def _append(B, S, held, H, Hk, D, R, P, ragged, dtype, pairs="half"):
    return {"op": "append", "B": B, "S": S, "held": held, "H": H, "Hk": Hk, "D": D, "R": R, "P": P,
            "ragged": ragged, "pairs": pairs, "scaling": "wavelength", "dtype": dtype}


def _attend(B, Sq, L, H, Hk, D, P, ragged, dtype):
    return {"op": "attend", "B": B, "Sq": Sq, "L": L, "H": H, "Hk": Hk, "D": D, "P": P,
            "ragged": ragged, "dtype": dtype}


def listed():
    cases = {
        # the new tokens of 32 users at far positions of a context-scaled
        # model: the smallest rotation, launches and latency are the time
        "rotary_step": _rotary(32, 1, 32, 8, 128, 128, "half", "wavelength", 60000, False, "bf16"),
        # the training step of a 4k grouped-query layer
        "rotary_train": _rotary(1, 4096, 32, 8, 128, 128, "half", "yarn", 0, True, "bf16"),
        # interleaved pairs on a quarter of the head, odd length, tensors as
        # transposed (B, heads, S, D) views
        "rotary_part": _rotary(8, 1001, 12, 12, 64, 16, "interleaved", "none", 0, True, "fp16",
                               "bhsd"),
        # one user's next token into the cache: the smallest call
        "append_one": _append(1, 1, 4096, 32, 8, 128, 128, 64, False, "bf16"),
        # the next tokens of prompts of several lengths, 28 query heads on 4
        "append_ragged": _append(12, 250, 700, 28, 4, 128, 128, 16, True, "bf16"),
        # a whole prompt of odd length into an empty cache
        "append_prompt": _append(1, 6001, 0, 32, 8, 128, 64, 64, False, "fp16"),
        # one user's next token against 4k cached: latency
        "attend_one": _attend(1, 1, 4096, 32, 8, 128, 64, False, "bf16"),
        # 32 users' next tokens, caches of up to 3001: reading the cache
        "attend_batch": _attend(32, 1, 3001, 32, 8, 128, 64, True, "bf16"),
        # four speculated tokens a user, 14 query heads on 2 of 64 columns
        "attend_draft": _attend(16, 4, 5000, 14, 2, 64, 16, True, "fp16"),
        # two users' next tokens against the longest contexts
        "attend_long": _attend(2, 1, 131072, 32, 8, 128, 128, False, "fp16"),
        # the next 256 tokens of a long prompt
        "attend_chunk": _attend(1, 256, 8448, 32, 8, 128, 64, False, "bf16"),
        # a long prompt's last 2048 tokens: the largest amount of arithmetic
        "attend_prompt": _attend(1, 2048, 8192, 32, 8, 128, 64, False, "bf16"),
    }
    return [dict(c, name=n) for n, c in cases.items()]


# Head counts (query, key/value) and columns that models use.
HEADS = ((32, 8, 128), (28, 4, 128), (16, 8, 128), (14, 2, 64), (64, 8, 128), (32, 4, 128),
         (12, 12, 64), (4, 4, 32), (8, 8, 32), (32, 32, 128))


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """One more case of an operator of listed(), its sizes anew."""
    op = rng.choice(("rotary", "append", "attend", "attend"))
    most = [max(work(c)[k] for c in listed() if c["op"] == op) for k in ("bytes", "flops")]
    while True:
        c = _draw(rng, op)
        w = work(c)
        if w["bytes"] <= most[0] and w["flops"] <= most[1]:
            return c


def _draw(rng, op):
    H, Hk, D = rng.choice(HEADS)
    dtype = rng.choice(("fp16", "bf16"))
    R = rng.choice((D, D, D // 2, D // 4, 3 * D // 4))
    P = rng.choice((16, 32, 64, 128))
    pairs = rng.choice(("half", "half", "interleaved"))
    if op == "rotary":
        return _rotary(_log_int(rng, 1, 64), _log_int(rng, 1, 8192), H, Hk, D, R, pairs,
                       rng.choice(("none", "linear", "ntk", "yarn", "wavelength")),
                       rng.choice((0, 1000, 100003, 1000003)), rng.random() < 0.5, dtype,
                       rng.choice(("bshd", "bhsd")))
    if op == "append":
        return _append(_log_int(rng, 1, 64), _log_int(rng, 1, 8192), rng.choice((0, 3, 77, 1030)),
                       H, Hk, D, R, P, rng.random() < 0.5, dtype, pairs)
    Sq = rng.choice((1, 1, 1, 2, 5, _log_int(rng, 8, 2048)))
    return _attend(_log_int(rng, 1, 64), Sq, Sq + _log_int(rng, 1, 131072) - 1, H, Hk, D, P,
                   rng.random() < 0.5, dtype)


# -- inputs ------------------------------------------------------------------------

def _lengths(c, most, least):
    """B lengths: all `most`, or spread evenly from `least` to `most`."""
    if not c["ragged"] or c["B"] == 1:
        return [most] * c["B"]
    return [least + (most - least) * b // (c["B"] - 1) for b in range(c["B"])]


def _frequencies(c):
    """(radians a position of each pair, the factor on cos and sin)."""
    R = c["R"]
    base = BASE
    if c["scaling"] == "ntk":
        base *= FACTOR ** (R / max(R - 2, 1))
    f = [base ** (-2.0 * j / R) for j in range(R // 2)]
    if c["scaling"] == "linear":
        return [x / FACTOR for x in f], 1.0
    if c["scaling"] == "yarn":
        # pairs that turn over 32 times in the original context keep their
        # frequency, those that turn less than once get it divided
        lo, hi = (R * math.log(ORIGINAL / (2 * math.pi * turns)) / (2 * math.log(BASE))
                  for turns in (32.0, 1.0))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), R - 1)
        ramp = [min(max((j - lo) / max(hi - lo, 1e-3), 0.0), 1.0) for j in range(R // 2)]
        return [x / FACTOR * r + x * (1 - r) for x, r in zip(f, ramp)], 0.1 * math.log(FACTOR) + 1
    if c["scaling"] == "wavelength":
        # wavelengths under a quarter of the original context stay, those
        # over it are divided, between them the two are mixed
        out = []
        for x in f:
            s = min(max((ORIGINAL * x / (2 * math.pi) - 1.0) / (4.0 - 1.0), 0.0), 1.0)
            out.append((1 - s) * x / FACTOR + s * x)
        return out, 1.0
    return f, 1.0


def _randn(shape, dtype, gen):
    return torch.randn(shape, dtype=torch.float32, device="cuda", generator=gen).to(dtype)


def _tensor(c, S, heads, gen):
    """(B, S, heads, D) of the case's dtype and layout."""
    if c.get("layout") == "bhsd":
        return _randn((c["B"], heads, S, c["D"]), DTYPES[c["dtype"]], gen).transpose(1, 2)
    return _randn((c["B"], S, heads, c["D"]), DTYPES[c["dtype"]], gen)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pages(c, tokens, gen):
    """A page table for `tokens` tokens of each sequence, its pages scattered
    over a pool, and the pool full of earlier, finished sequences' values."""
    B, P, Hk, D = c["B"], c["P"], c["Hk"], c["D"]
    width = -(-tokens // P)
    n = B * width + 3
    table = torch.randperm(n, device="cuda", generator=gen)[:B * width].to(torch.int32)
    k, ks = _quantise(_randn((n, Hk, P, D), torch.float32, gen))
    v, vs = _quantise(_randn((n, Hk, P, D), torch.float32, gen))
    v = v.view(n, Hk, P // 4, 4, 16, D // 32).transpose(3, 4).contiguous()
    vs = vs.view(n, Hk, P // 4, 4, D // 32).transpose(3, 4).contiguous()
    return {"table": table.view(B, width), "k_codes": k, "k_scales": ks, "v_codes": v,
            "v_scales": vs}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    c = case
    s = dict(c)
    if c["op"] != "attend":
        freq, factor = _frequencies(c)
        s["freq"] = torch.tensor(freq, dtype=torch.float64, device="cuda")
        s["factor"] = factor
    if c["op"] == "rotary":
        s["q"], s["k"] = _tensor(c, c["S"], c["H"], gen), _tensor(c, c["S"], c["Hk"], gen)
        if c["train"]:
            s["gq"], s["gk"] = _tensor(c, c["S"], c["H"], gen), _tensor(c, c["S"], c["Hk"], gen)
        # each sequence continues at a position of its own
        at = torch.randint(0, 1000, (c["B"], 1), device="cuda", generator=gen) + c["first"]
        s["positions"] = (at + torch.arange(c["S"], device="cuda")).to(torch.int32)
    elif c["op"] == "append":
        s["q"], s["k"], s["v"] = (_tensor(c, c["S"], h, gen) for h in (c["H"], c["Hk"], c["Hk"]))
        s["start"] = _ints(_lengths(c, c["held"], 0))
        s["counts"] = _ints(_lengths(c, c["S"], 1)) if c["ragged"] else None
        s.update(_pages(c, c["held"] + c["S"], gen))
    else:
        s["q"] = _tensor(c, c["Sq"], c["H"], gen)
        s["lengths"] = _ints(_lengths(c, c["L"], max(c["L"] // 4, 1)))
        s.update(_pages(c, c["L"], gen))
    if own:
        from flash_attn_volta import PagedKVCache, RotaryPositions
        if c["op"] != "attend":
            scaling = {"linear": {"type": "linear", "factor": FACTOR},
                       "ntk": {"type": "ntk", "factor": FACTOR},
                       "yarn": {"type": "yarn", "factor": FACTOR, "original_length": ORIGINAL},
                       "wavelength": {"type": "wavelength", "factor": FACTOR, "low": 1.0,
                                      "high": 4.0, "original_length": ORIGINAL}}
            s["rotary"] = RotaryPositions(c["R"], base=BASE, scaling=scaling.get(c["scaling"]),
                                          interleaved=c["pairs"] == "interleaved", device="cuda")
        if c["op"] != "rotary":
            s["cache"] = PagedKVCache.from_tensors(s["k_codes"], s["k_scales"], s["v_codes"],
                                                   s["v_scales"], DTYPES[c["dtype"]])
        if c["op"] == "rotary" and c["train"]:
            s["q"].requires_grad_()
            s["k"].requires_grad_()
    return s


# -- the pass ----------------------------------------------------------------------

def run(state):
    s = state
    if own:
        return _run_own(s)
    if s["op"] == "rotary":
        cos, sin = _angles(s, s["positions"], torch.float32)
        dt = s["q"].dtype
        out = {n: _rotate(s, s[n].float(), cos, sin).to(dt) for n in ("q", "k")}
        if s["train"]:
            out |= {"d" + n: _rotate(s, s["g" + n].float(), cos, -sin).to(dt) for n in ("q", "k")}
        return out
    return _append_plain(s) if s["op"] == "append" else _attend_plain(s)


def _run_own(s):
    from flash_attn_volta import append_paged, apply_rotary_positions, attend_paged, read_paged
    if s["op"] == "rotary":
        q, k = apply_rotary_positions(s["q"], s["k"], s["positions"], s["rotary"])
        if not s["train"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["gq"], s["gk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    if s["op"] == "append":
        q = append_paged(s["cache"], s["k"], s["v"], s["table"], s["start"], s["counts"],
                         q=s["q"], rotary=s["rotary"])
        k, v = read_paged(s["cache"], s["table"], s["start"], s["S"], s["counts"])
        return {"q": q, "k": k, "v": v}
    return attend_paged(s["q"], s["cache"], s["table"], s["lengths"])


def _angles(s, positions, dtype):
    """cos and sin (B, S, 1, R / 2), the angles in 64 bits."""
    a = positions.double()[..., None, None] * s["freq"]
    return (a.cos() * s["factor"]).to(dtype), (a.sin() * s["factor"]).to(dtype)


def _rotate(s, x, cos, sin):
    R = s["R"]
    if s["pairs"] == "half":
        a, b = x[..., :R // 2], x[..., R // 2:R]
        parts = (a * cos - b * sin, b * cos + a * sin)
    else:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        parts = (torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2),)
    return torch.cat((*parts, x[..., R:]), dim=-1)


def _quantise(x):
    """(codes (.., D / 2), scales (.., D / 32)) of x (.., D)."""
    x = x.unflatten(-1, (-1, 32))
    e = torch.frexp(x.abs().amax(-1, keepdim=True))[1].clamp(-123, 128) - 3
    a = torch.ldexp(x.abs(), -e)
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5)
            + (a >= 3.5) + (a > 5.0) + 8 * (x < 0)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8).squeeze(-1)


def _values(codes, scales):
    """float32 (.., D) of codes (.., D / 2) and scales (.., D / 32)."""
    lut = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float32, device=codes.device)
    v = lut[torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).int()]
    return (v.unflatten(-1, (-1, 32)) * torch.exp2(scales.float() - 127)[..., None]).flatten(-2)


def _slots(s, positions):
    """(page, slot in the page) of positions (B, n)."""
    page = torch.gather(s["table"].long(), 1, positions // s["P"])
    return page, positions % s["P"]


def _held(s, positions):
    """k, v (B, n, Hk, D) in float32 of the cached tokens at positions (B, n)."""
    page, t = _slots(s, positions)
    k = _values(s["k_codes"][page, :, t], s["k_scales"][page, :, t])
    v = s["v_codes"][page, :, t // 4, :, t % 4].flatten(-2)
    return k, _values(v, s["v_scales"][page, :, t // 4, :, t % 4])


def _append_plain(s):
    dt = s["q"].dtype
    new = torch.arange(s["S"], device="cuda")[None]
    positions = s["start"].long()[:, None] + new
    cos, sin = _angles(s, positions, torch.float64)
    q = _rotate(s, s["q"].float(), cos.float(), sin.float()).to(dt)
    k, ks = _quantise(_rotate(s, s["k"].double(), cos, sin))      # codes next to a border
    v, vs = _quantise(s["v"].float())
    v = v.unflatten(-1, (16, -1))
    page, t = _slots(s, positions)
    at_k, at_v = (page, slice(None), t), (page, slice(None), t // 4, slice(None), t % 4)
    stored = (("k_codes", at_k, k), ("k_scales", at_k, ks), ("v_codes", at_v, v),
              ("v_scales", at_v, vs))
    real = None if s["counts"] is None else new < s["counts"][:, None]
    for name, at, x in stored:
        if real is not None:
            x = torch.where(real.view(real.shape + (1,) * (x.dim() - 2)), x, s[name][at])
        s[name][at] = x
    k, v = _held(s, positions)
    if real is not None:
        k, v = k * real[..., None, None], v * real[..., None, None]
    return {"q": q, "k": k.to(dt), "v": v.to(dt)}


def _attend_plain(s):
    B, Sq, H, Hk, D, L = (s[n] for n in ("B", "Sq", "H", "Hk", "D", "L"))
    positions = torch.arange(L, device="cuda")
    k, v = _held(s, positions.expand(B, L))
    q = s["q"].float().unflatten(2, (Hk, H // Hk)).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)
    scores = q @ k.permute(0, 2, 3, 1) * D ** -0.5                   # (B, Hk, G * Sq, L)
    last = s["lengths"].long()[:, None] - Sq + torch.arange(Sq, device="cuda")     # (B, Sq)
    seen = (positions <= last[..., None]).repeat(1, H // Hk, 1)[:, None]
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = p @ v.transpose(1, 2) / torch.where(total == 0, 1.0, total)
    out = out.view(B, Hk, H // Hk, Sq, D).permute(0, 3, 1, 2, 4).reshape(B, Sq, H, D)
    return out.to(s["q"].dtype)


# -- what a pass cannot do without ---------------------------------------------------

def work(case):
    c = case
    D, Hk = c["D"], c["Hk"]
    token = Hk * (D + D // 16)          # bytes of a token's keys and values in the cache
    if c["op"] == "rotary":
        n = c["B"] * c["S"]
        passes = 2 if c["train"] else 1
        return {"bytes": passes * (2 * n * (c["H"] + Hk) * D * 2 + 4 * n),
                "flops": passes * n * (c["H"] + Hk) * c["R"] * 3}
    if c["op"] == "append":
        n = sum(_lengths(c, c["S"], 1)) if c["ragged"] else c["B"] * c["S"]
        # new q, k, v in; q, the cache's rows and, read back, their values out
        return {"bytes": n * (2 * c["H"] * D * 2 + 4 * Hk * D * 2 + 2 * token),
                "flops": n * ((c["H"] + Hk) * c["R"] * 3 + 6 * Hk * D)}
    pairs = held = 0
    for n in _lengths(c, c["L"], max(c["L"] // 4, 1)):
        first = max(0, c["Sq"] - n)     # queries before it see no key
        k = c["Sq"] - first
        pairs += k * (n - c["Sq"] + first + 1) + k * (k - 1) // 2
        held += n
    return {"bytes": held * token + 2 * c["B"] * c["Sq"] * c["H"] * D * 2,
            "flops": 4 * D * c["H"] * pairs}


# -- the definition in 64 bits -------------------------------------------------------

def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "attend":
        return _exact_attend(c, s)
    if c["op"] == "rotary":
        turn = _turns(c, s["positions"])
        out = {n: _exact_rotate(c, s[n].detach().double(), turn) for n in ("q", "k")}
        if c["train"]:
            out |= {"d" + n: _exact_rotate(c, s["g" + n].double(), turn.conj())
                    for n in ("q", "k")}
        return out
    at = s["start"].long()[:, None] + torch.arange(c["S"], device="cuda")
    turn = _turns(c, at)
    k, v = _exact_stored(_exact_rotate(c, s["k"].double(), turn)), _exact_stored(s["v"].double())
    if s["counts"] is not None:
        for b, n in enumerate(s["counts"].tolist()):
            k[b, n:] = 0
            v[b, n:] = 0
    return {"q": _exact_rotate(c, s["q"].double(), turn), "k": k, "v": v}


def _turns(c, positions):
    """factor * exp(i position frequency), (B, S, 1, R / 2)."""
    freq, factor = _frequencies(c)
    freq = torch.tensor(freq, dtype=torch.float64, device=positions.device)
    angle = torch.outer(positions.double().flatten(), freq).view(*positions.shape, 1, -1)
    return torch.polar(torch.full_like(angle, factor), angle)


def _exact_rotate(c, x, turn):
    y = x.clone()
    R = c["R"]
    re, im = ((slice(0, R // 2), slice(R // 2, R)) if c["pairs"] == "half"
              else (slice(0, R, 2), slice(1, R, 2)))
    z = torch.complex(x[..., re].contiguous(), x[..., im].contiguous()) * turn
    y[..., re], y[..., im] = z.real, z.imag
    return y


def _exact_stored(x):
    """x as the cache's 4 bits hold it: steps of half the value's power of
    two, at least 0.5, in units of the block's."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    top = b.abs().max(dim=-1, keepdim=True).values
    unit = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -124))) - 2)
    y = b / unit
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=1.0))) - 1)
    return (torch.round(y / step) * step).clamp(-6, 6).mul(unit).reshape(x.shape)


def _exact_attend(c, s):
    B, Sq, H, Hk, D, P = (c[n] for n in ("B", "Sq", "H", "Hk", "D", "P"))
    G = H // Hk
    grid = torch.tensor(E2M1 + E2M1, dtype=torch.float64, device="cuda")
    grid[8:] *= -1

    def decode(codes, scales):
        x = torch.empty(codes.shape[0], D, dtype=torch.float64, device="cuda")
        x[:, 0::2], x[:, 1::2] = grid[(codes % 16).long()], grid[(codes // 16).long()]
        return x * torch.exp2(scales.double() - 127).repeat_interleave(32, dim=1)

    out = torch.zeros(B, Sq, H, D, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lengths"].tolist()):
        if n == 0:
            continue
        pages = s["table"][b, :-(-n // P)].long()
        i = torch.arange(max(0, Sq - n), Sq, device="cuda")
        hidden = torch.arange(n, device="cuda")[None] > (i + n - Sq)[:, None]
        for h in range(Hk):
            k = decode(s["k_codes"][pages, h].reshape(-1, D // 2),
                       s["k_scales"][pages, h].reshape(-1, D // 32))[:n]
            v = decode(s["v_codes"][pages, h].transpose(2, 3).reshape(-1, D // 2),
                       s["v_scales"][pages, h].transpose(2, 3).reshape(-1, D // 32))[:n]
            for g in range(h * G, (h + 1) * G):
                w = (s["q"][b, i, g].double() @ k.T) / math.sqrt(D)
                out[b, i, g] = torch.softmax(w.masked_fill(hidden, -math.inf), dim=-1) @ v
    return out
