"""Timed cases of the serving-side operators around the paged attention: rotary
tables and rotations, the paged key-value cache (written quantised, read back)
and the decode that reads it in 8 bits.

``own = False`` runs each operator in elementary torch operations in fp32 (fp64
for angles); ``own = True`` runs the library's calls on the same inputs.

The 8-bit cache: a row (one token, one KV head, K or V) x[0..D) is stored as
e4m3 codes c = e4m3(x / 2^e) and one byte e + 127, e the smallest integer with
max|x| <= 448 * 2^e (clamped to [-100, 120]; 0 for a row of zeros).  Scale bytes
are [pages, Hkv, 2, page_size] (0: K, 1: V).
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
F8 = torch.float8_e4m3fn


def _bw():
    import blackwell_b200 as bw

    return bw


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # A table for a 4096-token window, rotary over a whole head of 64: made once at start-up.
        {"name": "table 4k", "op": "table", "length": 4096, "R": 64, "base": 10000.0, "scaling": "none", "factor": 1.0,
         "orig": 0, "first": 0},
        # A table for the 131072-token context, YaRN-scaled from 8192: angles of far positions.
        {"name": "table 128k yarn", "op": "table", "length": 131072, "R": 128, "base": 500000.0, "scaling": "yarn",
         "factor": 16.0, "orig": 8192, "first": 0},
        # One decode step of 8 sequences at unrelated positions: latency.
        {"name": "rope decode 8", "op": "rope", "B": 1, "S": 8, "Hq": 32, "Hkv": 8, "D": 128, "R": 128, "dtype": "bf16",
         "layout": "thd", "interleaved": False, "inverse": False, "length": 8192, "base": 500000.0},
        # Prefill of 4 x 4096 tokens, heads of 128, BSHD as a projection leaves it.
        {"name": "rope prefill 4x4096", "op": "rope", "B": 4, "S": 4096, "Hq": 32, "Hkv": 8, "D": 128, "R": 128,
         "dtype": "bf16", "layout": "bshd", "interleaved": False, "inverse": False, "length": 8192, "base": 500000.0},
        # Gradient of an interleaved rotation of half of a 64-wide head, fp32, odd length, BHSD.
        {"name": "rope grad f32 partial", "op": "rope", "B": 3, "S": 1777, "Hq": 12, "Hkv": 4, "D": 64, "R": 32,
         "dtype": "f32", "layout": "bhsd", "interleaved": True, "inverse": True, "length": 2048, "base": 10000.0},
        # One decode step of 64 sequences: K rotated, K and V quantised into their pages.
        {"name": "append 64", "op": "append", "B": 64, "lo": 100, "hi": 1000, "Hkv": 8, "D": 128, "R": 128, "page": 16,
         "fp8": True, "interleaved": False},
        # A 2048-token chunk written at the end of a 32768-token sequence, all of it read back for the chunk's attention.
        {"name": "chunk 2k at 30k", "op": "chunk", "B": 1, "n": 2048, "lo": 32768, "hi": 32768, "Hkv": 8, "D": 128,
         "R": 128, "page": 64, "fp8": True, "interleaved": False},
        # Ragged chunks of 5 sequences in 8-token pages, heads of 64, half of the head rotated; the bf16 cache.
        {"name": "chunk ragged bf16", "op": "chunk", "B": 5, "n": 129, "lo": 130, "hi": 1501, "Hkv": 4, "D": 64, "R": 32,
         "page": 8, "fp8": False, "interleaved": True},
        # One short sequence: the latency of a decode step.
        {"name": "decode 1x517", "op": "decode", "B": 1, "lo": 517, "hi": 517, "Hkv": 8, "G": 4, "D": 128, "page": 16},
        # A batch of ragged sequences, heads of 64, groups of 3.
        {"name": "decode 16 ragged D64", "op": "decode", "B": 16, "lo": 1, "hi": 4099, "Hkv": 4, "G": 3, "D": 64,
         "page": 64},
        # One 131072-token context: the split over the cache's length.
        {"name": "decode 1x128k", "op": "decode", "B": 1, "lo": 131072, "hi": 131072, "Hkv": 8, "G": 8, "D": 128,
         "page": 32},
        # The framework's decode workload: 64 sequences of 1024 to 32768 tokens.
        {"name": "decode 64x(1k..32k)", "op": "decode", "B": 64, "lo": 1024, "hi": 32768, "Hkv": 8, "G": 8, "D": 128,
         "page": 64},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["table", "rope", "rope", "append", "chunk", "decode", "decode", "decode"])
    D = rng.choice([64, 128])
    R = 16 * rng.randint(1, D // 16)
    if op == "table":
        scaling = rng.choice(["none", "linear", "ntk", "yarn", "bands"])
        return {"op": op, "length": _log_int(rng, 1, 131072), "R": 2 * rng.randint(2, 64),
                "base": rng.choice([10000.0, 500000.0, 1000000.0]), "scaling": scaling,
                "factor": 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0, 40.0]),
                "orig": 0 if scaling == "none" else rng.choice([2048, 4096, 8192]), "first": rng.choice([0, rng.randint(1, 1 << 20)])}
    if op == "rope":
        Hkv = rng.randint(1, 16)
        Hq = Hkv * rng.randint(1, 8)
        D = 8 * rng.randint(2, 32)
        R = 16 * rng.randint(1, D // 16)
        most = 4 * 4096 * 40 * 128 // ((Hq + Hkv) * D)
        tokens = _log_int(rng, 1, most // 2)
        B = rng.randint(1, min(5, tokens))
        layout = rng.choice(["thd", "bshd", "bhsd"])
        S = tokens // B
        return {"op": op, "B": 1 if layout == "thd" else B, "S": S, "Hq": Hq, "Hkv": Hkv, "D": D, "R": R,
                "dtype": rng.choice(["bf16", "bf16", "f32"]), "layout": layout, "interleaved": rng.random() < 0.5,
                "inverse": rng.random() < 0.5, "length": _log_int(rng, 256, 32768), "base": 10000.0}
    Hkv = rng.choice([1, 2, 3, 4, 5, 8, 16])
    page = rng.choice([8, 16, 32, 64, 128, 256])
    if op == "append":
        B = _log_int(rng, 1, 300)
        lo = rng.randint(1, 200)
        return {"op": op, "B": B, "lo": lo, "hi": lo + rng.randint(0, 400), "Hkv": Hkv, "D": D, "R": R, "page": page,
                "fp8": rng.random() < 0.7, "interleaved": rng.random() < 0.5}
    if op == "chunk":
        B = rng.randint(1, 6)
        hi = _log_int(rng, 20, 32768 // B)
        lo = rng.randint(1, hi)
        return {"op": op, "B": B, "n": rng.randint(1, lo), "lo": lo, "hi": hi, "Hkv": Hkv, "D": D, "R": R, "page": page,
                "fp8": rng.random() < 0.7, "interleaved": rng.random() < 0.5}
    B = _log_int(rng, 1, 128)
    G = rng.randint(1, 16)
    hi = _log_int(rng, 2, min(131072, 64 * 16384 * 8 // (B * Hkv * max(1, G // 8))))
    return {"op": op, "B": B, "lo": rng.randint(0, hi), "hi": hi, "Hkv": Hkv, "G": G, "D": D, "page": page}


# ------------------------------------------------------------------ inputs

def _lens(c, g):
    """B lengths evenly from lo to hi (so that every seed has the same work), in the seed's order."""
    B = c["B"]
    t = torch.linspace(c["lo"], c["hi"], B, dtype=torch.float64).round().long() if B > 1 else torch.tensor([c["hi"]])
    return t[torch.randperm(B, generator=g)]


def _paged(c, g, gd):
    """Lengths, a block table whose pages lie in random order (-1 where a sequence has no page), and the cache's pages."""
    lens = _lens(c, g)
    page = c["page"]
    need = (lens + page - 1) // page
    num = int(need.sum()) + 3
    width = max(1, int(need.max()))
    first = torch.cumsum(need, 0) - need
    col = torch.arange(width)
    perm = torch.randperm(num, generator=gd, device=DEV).int()
    at = (first[:, None] + col[None]).clamp(max=num - 1).to(DEV)
    table = torch.where((col[None] < need[:, None]).to(DEV), perm[at], torch.full((), -1, dtype=torch.int32, device=DEV))
    return lens, table.contiguous(), num


def _codes(shape, gd):
    """Codes as a quantised cache holds them: the row's largest between 224 and 448 or a little less."""
    out = torch.empty(shape, dtype=F8, device=DEV)
    flat = out.view(-1)
    step = 1 << 28
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        flat[i:i + n] = (torch.randn(n, generator=gd, device=DEV) * 100.0).clamp_(-448.0, 448.0).to(F8)
    return out


def prepare(case, seed):
    c = case
    g = torch.Generator().manual_seed(int(seed))
    gd = torch.Generator(device=DEV).manual_seed(int(seed))
    s = {"case": c}
    if c["op"] == "table":
        # another seed is another stretch of positions
        s["first"] = c["first"] + int(torch.randint(0, 1000, (1,), generator=g))
        s["out"] = torch.empty(c["length"], c["R"], dtype=torch.float32, device=DEV)
        return s
    if c["op"] == "rope":
        dt = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32
        B, S, D = c["B"], c["S"], c["D"]

        def make(H):
            x = torch.randn(B, S, H, D, generator=gd, device=DEV).to(dt)
            if c["layout"] == "thd":
                return x.view(S, H, D)
            return x.transpose(1, 2) if c["layout"] == "bshd" else x.transpose(1, 2).contiguous()

        s["q"], s["k"] = make(c["Hq"]), make(c["Hkv"])
        s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        s["table"] = _angles_table(c["length"], c["R"], c["base"])
        if c["layout"] == "thd":  # a token of each of S sequences
            s["pos"] = torch.randint(0, c["length"], (S,), generator=g).int().to(DEV)
        else:  # B prompts, each behind a prefix of its own
            room = max(1, c["length"] - S)
            s["pos"] = (torch.randint(0, room, (B, 1), generator=g) + torch.arange(S)[None]).int().to(DEV)
        return s
    Hkv, D, page = c["Hkv"], c["D"], c["page"]
    lens, s["block_table"], num = _paged(c, g, gd)
    s["lens"] = lens.int().to(DEV)
    shape = (num, page, Hkv, D)
    if c["op"] == "decode" or c["fp8"]:
        s["k_cache"], s["v_cache"] = _codes(shape, gd), _codes(shape, gd)
        s["scales"] = torch.randint(118, 123, (num, Hkv, 2, page), generator=gd, device=DEV).to(torch.uint8)
    else:
        s["k_cache"] = torch.randn(shape, generator=gd, device=DEV).bfloat16()
        s["v_cache"] = torch.randn(shape, generator=gd, device=DEV).bfloat16()
        s["scales"] = None
    if c["op"] == "decode":
        Hq = Hkv * c["G"]
        s["q"] = torch.randn(c["B"], Hq, D, generator=gd, device=DEV).bfloat16()
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(c["B"], Hq, dtype=torch.float32, device=DEV)
        # room for the partial results of a split cache, kept from call to call as a server keeps it
        room = (2048 + c["B"] * Hkv) * c["G"] * (D + 2) * 4 + 8 * (c["B"] + 1) + 4096
        s["workspace"] = torch.empty(room, dtype=torch.uint8, device=DEV)
        return s
    # the new tokens: the last n of each sequence (1 of each in a decode step), K and V out of one projection
    n = c.get("n", 1)
    seq = torch.arange(c["B"]).repeat_interleave(n)
    pos = (lens - n)[:, None] + torch.arange(n)[None]
    pos = pos.reshape(-1)
    T = pos.numel()
    kv = torch.randn(T, 2 * Hkv * D, generator=gd, device=DEV)
    kv = kv * torch.exp(0.5 * torch.randn(2 * Hkv * D, generator=gd, device=DEV))  # channels of unlike size
    kv = kv.bfloat16()
    s["k"], s["v"] = kv[:, :Hkv * D].view(T, Hkv, D), kv[:, Hkv * D:].view(T, Hkv, D)
    s["pos"] = pos.int().to(DEV)
    seq, pos = seq.to(DEV), pos.to(DEV)
    s["slots"] = s["block_table"][seq, pos // page].long() * page + pos % page
    s["table"] = _angles_table(int(lens.max()) + 1, c["R"], 10000.0)
    if c["op"] == "chunk":
        total = int(lens.sum())
        s["offsets"] = (torch.cumsum(lens, 0) - lens).to(DEV)
        s["k_out"] = torch.empty(total, Hkv, D, dtype=torch.bfloat16, device=DEV)
        s["v_out"] = torch.empty(total, Hkv, D, dtype=torch.bfloat16, device=DEV)
    return s


# ------------------------------------------------------------------ the plain forms

def _frequencies(R, base, scaling, factor, orig):
    """Angles per position of the R / 2 pairs, fp64, and the factor on cos and sin."""
    i = torch.arange(0, R, 2, dtype=torch.float64, device=DEV)
    if scaling == "ntk":
        base = base * factor ** (R / (R - 2))
    f = base ** (-i / R)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "yarn":
        def dim(turns):
            return R * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(base))

        low, high = max(math.floor(dim(32.0)), 0), min(math.ceil(dim(1.0)), R - 1)
        ramp = ((i / 2 - low) / (high - low if high != low else 0.001)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    if scaling == "bands":
        turns = orig * f / (2 * math.pi)
        mix = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f / factor * (1 - mix) + f * mix, 1.0
    return f, 1.0


def _table64(first, length, R, base, scaling="none", factor=1.0, orig=0):
    f, m = _frequencies(R, base, scaling, factor, orig)
    a = torch.arange(first, first + length, dtype=torch.float64, device=DEV)[:, None] * f[None]
    return torch.cat([torch.cos(a) * m, torch.sin(a) * m], 1)


def _angles_table(length, R, base):
    return _table64(0, length, R, base).float()


def _rotate(x, pos, table, interleaved, inverse):
    """fp32 rotation of the last axis; pos has x's leading axes but the heads', which are at axis -2 here."""
    R = table.shape[1]
    inside = ((pos >= 0) & (pos < table.shape[0]))[..., None, None]
    cs = table[pos.clamp(0, table.shape[0] - 1).long()][..., None, :]
    c, sn = cs[..., :R // 2], cs[..., R // 2:]
    if inverse:
        sn = -sn
    x = x.float()
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    u, w = a * c - b * sn, a * sn + b * c
    turned = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    return torch.where(inside, torch.cat([turned, x[..., R:]], -1), x)


def _power(e):
    return ((e + 127) << 23).view(torch.float32)


def _quantise(x):
    """fp32 rows -> (e4m3 codes, scale bytes)."""
    finite = torch.isfinite(x)
    top = torch.where(finite, x.abs(), torch.zeros_like(x)).amax(-1)
    m, e = torch.frexp(top)
    e = torch.where(top > 0, (e - 9 + (m > 0.875).int()).clamp(-100, 120), torch.zeros_like(e)).int()
    code = torch.where(finite, x * _power(-e)[..., None], torch.full_like(x, float("nan"))).to(F8)
    return code, (e + 127).to(torch.uint8)


def _write_plain(s):
    c = s["case"]
    page, Hkv, D = c["page"], c["Hkv"], c["D"]
    k = _rotate(s["k"], s["pos"], s["table"], c["interleaved"], False)
    v = s["v"].float()
    rows = lambda t: t.view(torch.uint8 if c["fp8"] else t.dtype).view(-1, Hkv, D)  # noqa: E731
    if c["fp8"]:
        (kc, ke), (vc, ve) = _quantise(k), _quantise(v)
        rows(s["k_cache"])[s["slots"]] = kc.view(torch.uint8)
        rows(s["v_cache"])[s["slots"]] = vc.view(torch.uint8)
        s["scales"][s["slots"] // page, :, :, s["slots"] % page] = torch.stack([ke, ve], -1)
    else:
        rows(s["k_cache"])[s["slots"]] = k.bfloat16()
        rows(s["v_cache"])[s["slots"]] = v.bfloat16()


def _values(s, which, page, slot):
    """fp32 values of the cache rows (page, slot) of K (0) or V (1)."""
    cache = s["v_cache"] if which else s["k_cache"]
    if s["scales"] is None:
        return cache[page, slot].float()
    scale = _power(s["scales"][page, :, which, slot].int() - 127)
    return cache.view(torch.uint8)[page, slot].view(F8).float() * scale[..., None]


def _read_plain(s):
    lens, page = s["lens"].long(), s["case"]["page"]
    total = s["k_out"].shape[0]
    row = torch.arange(total, device=DEV)
    seq = torch.searchsorted(s["offsets"] + lens, row, right=True)
    tok = row - s["offsets"][seq]
    pg = s["block_table"][seq, tok // page].long()
    s["k_out"].copy_(_values(s, 0, pg, tok % page))
    s["v_out"].copy_(_values(s, 1, pg, tok % page))


def _decode_plain(s):
    c = s["case"]
    B, Hkv, G, D, page = c["B"], c["Hkv"], c["G"], c["D"], c["page"]
    tok = torch.arange(max(1, c["hi"]), device=DEV)
    pg = s["block_table"][:, tok // page].long().clamp(min=0)
    slot = (tok % page)[None].expand_as(pg)
    seen = (tok[None] < s["lens"][:, None])[:, None, None]
    q = s["q"].float().view(B, Hkv, G, D)
    x = torch.matmul(q, _values(s, 0, pg, slot).permute(0, 2, 3, 1)) * (1.0 / math.sqrt(D))
    x = torch.where(seen, x, torch.full((), -math.inf, device=DEV))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, _values(s, 1, pg, slot).permute(0, 2, 1, 3))
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.view(B, Hkv * G, D).bfloat16(), (top + torch.log(total)).view(B, Hkv * G)


# ------------------------------------------------------------------ one pass

def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if op == "table":
        if own:
            return _bw().rope_table(c["length"], c["R"], base=c["base"], scaling=c["scaling"], factor=c["factor"],
                                    original_length=c["orig"], first=s["first"], out=s["out"])
        return _table64(s["first"], c["length"], c["R"], c["base"], c["scaling"], c["factor"], c["orig"]).float()
    if op == "rope":
        if own:
            return _bw().rope(s["q"], s["k"], s["table"], positions=s["pos"], interleaved=c["interleaved"],
                              inverse=c["inverse"], q_out=s["q_out"], k_out=s["k_out"])
        if c["layout"] == "thd":
            return tuple(_rotate(x, s["pos"], s["table"], c["interleaved"], c["inverse"]).to(x.dtype)
                         for x in (s["q"], s["k"]))
        return tuple(_rotate(x.transpose(1, 2), s["pos"], s["table"], c["interleaved"], c["inverse"]).to(x.dtype)
                     .transpose(1, 2) for x in (s["q"], s["k"]))
    if op == "decode":
        if own:
            return _bw().gqa_decode_paged_fp8(s["q"], s["k_cache"], s["v_cache"], s["scales"], s["block_table"],
                                              s["lens"], workspace=s["workspace"], out=s["out"], lse=s["lse"])
        return _decode_plain(s)
    if own:
        _bw().kv_cache_write(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], scales=s["scales"],
                             cos_sin_cache=s["table"], positions=s["pos"], interleaved=c["interleaved"])
    else:
        _write_plain(s)
    if op == "append":  # the updated cache
        return [s["k_cache"], s["v_cache"]] + ([s["scales"]] if c["fp8"] else [])
    if own:
        return _bw().kv_cache_read(s["k_cache"], s["v_cache"], s["block_table"], s["lens"], s["offsets"],
                                   scales=s["scales"], k_out=s["k_out"], v_out=s["v_out"])
    _read_plain(s)
    return s["k_out"], s["v_out"]


def work(case):
    c = case
    if c["op"] == "table":
        n = c["length"] * c["R"]
        return {"bytes": 4 * n, "flops": 20 * n}
    if c["op"] == "rope":
        n = c["B"] * c["S"] * (c["Hq"] + c["Hkv"]) * c["D"]
        touched = min(c["length"], c["B"] * c["S"])
        return {"bytes": 2 * n * (2 if c["dtype"] == "bf16" else 4) + 4 * touched * c["R"] + 4 * c["B"] * c["S"],
                "flops": 3 * n * c["R"] // c["D"]}
    lens = np.round(np.linspace(c["lo"], c["hi"], c["B"])) if c["B"] > 1 else np.array([c["hi"]])
    tokens, row = float(lens.sum()), c["Hkv"] * c["D"]
    if c["op"] == "decode":
        q = c["B"] * c["Hkv"] * c["G"]
        return {"bytes": tokens * 2 * (row + c["Hkv"]) + q * (4 * c["D"] + 4),
                "flops": 4 * tokens * c["G"] * row}
    held = 2 * row + 2 * c["Hkv"] if c["fp8"] else 4 * row
    new = c["B"] * c.get("n", 1)
    b = new * (4 * row + held + 4 * c["R"])
    if c["op"] == "chunk":
        b += tokens * (held + 4 * row)
    return {"bytes": b, "flops": 6 * new * row}


# ------------------------------------------------------------------ in 64 bits

def _two_to(e):
    """fp64 2^e for whole e (pow may be a last bit off)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _round_e4m3(y):
    """fp64 -> the nearest e4m3 value, ties to even (|y| <= 448)."""
    _, e = torch.frexp(y)
    q = _two_to((e - 1).clamp(min=-6) - 3)
    return torch.round(y / q) * q


def _exact_rows(x):
    """fp64 rows -> (code values, scales), both fp64."""
    top = x.abs().amax(-1)
    e = torch.ceil(torch.log2(top / 448.0)).clamp(-1000, 1000)
    e = torch.where(448.0 * _two_to(e - 1) >= top, e - 1, e)
    e = torch.where(448.0 * _two_to(e) < top, e + 1, e)
    sc = torch.where(top > 0, _two_to(e.clamp(-100, 120)), torch.ones_like(top))
    return _round_e4m3(x / sc[..., None]), sc


def _exact_turn(x, pos, table, interleaved, inverse):
    """Rotation as a complex product, pair by pair, in fp64; x [tokens, heads, D]."""
    R = table.shape[1]
    x = x.double()
    t = table.double()
    ok = (pos >= 0) & (pos < t.shape[0])
    row = t[torch.where(ok, pos, torch.zeros_like(pos)).long()]
    z = torch.complex(row[:, :R // 2], row[:, R // 2:])
    z = torch.where(ok[:, None], z, torch.ones_like(z))
    z = (z.conj() if inverse else z)[:, None]
    out = x.clone()
    if interleaved:
        out[..., :R] = torch.view_as_real(torch.view_as_complex(x[..., :R].reshape(*x.shape[:2], R // 2, 2).contiguous()) * z).flatten(-2)
    else:
        w = torch.complex(x[..., :R // 2].contiguous(), x[..., R // 2:R].contiguous()) * z
        out[..., :R // 2], out[..., R // 2:R] = w.real, w.imag
    return out


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    op = c["op"]
    if op == "table":
        R, L, F, N = c["R"], c["length"], c["factor"], c["orig"]
        base = c["base"] * (F ** (R / (R - 2)) if c["scaling"] == "ntk" else 1.0)
        freq, m = [], 1.0
        for i in range(R // 2):
            f = math.exp(-2.0 * i / R * math.log(base))
            if c["scaling"] == "linear":
                f /= F
            elif c["scaling"] == "yarn":
                m = 1.0 + 0.1 * math.log(F)
                edge = [R / 2 * math.log(N / (2 * math.pi * t)) / math.log(base) for t in (32.0, 1.0)]
                low, high = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), R - 1)
                r = min(1.0, max(0.0, (i - low) / ((high - low) or 0.001)))
                f = f * (r / F + 1.0 - r)
            elif c["scaling"] == "bands":
                wave = 2 * math.pi / f
                if wave > N:
                    f /= F
                elif wave >= N / 4.0:
                    r = (N / wave - 1.0) / 3.0
                    f = f * (r + (1 - r) / F)
            freq.append(f)
        p = np.arange(s["first"], s["first"] + L, dtype=np.float64)[:, None] * np.array(freq)[None]
        return torch.from_numpy(np.concatenate([m * np.cos(p), m * np.sin(p)], 1))
    if op == "rope":
        outs = []
        for x in (s["q"], s["k"]):
            if c["layout"] == "thd":
                outs.append(_exact_turn(x, s["pos"], s["table"], c["interleaved"], c["inverse"]))
                continue
            B, H, S, D = x.shape
            y = torch.empty(B, H, S, D, dtype=torch.float64, device=DEV)
            for b in range(B):
                y[b] = _exact_turn(x[b].transpose(0, 1), s["pos"][b], s["table"], c["interleaved"], c["inverse"]).transpose(0, 1)
            outs.append(y)
        return tuple(outs)
    if op == "decode":
        B, Hkv, G, D, page = c["B"], c["Hkv"], c["G"], c["D"], c["page"]
        o = torch.zeros(B, Hkv * G, D, dtype=torch.float64, device=DEV)
        lse = torch.full((B, Hkv * G), -math.inf, dtype=torch.float64, device=DEV)
        for b in range(B):
            L = int(s["lens"][b])
            if L == 0:
                continue
            t = torch.arange(L, device=DEV)
            pg, sl = s["block_table"][b, t // page].long(), t % page
            kv = []
            for w, cache in enumerate((s["k_cache"], s["v_cache"])):
                sc = _two_to(s["scales"][pg, :, w, sl].long() - 127)
                kv.append((cache.view(torch.uint8)[pg, sl].view(F8).double() * sc[..., None]).transpose(0, 1))
            x = s["q"][b].double().view(Hkv, G, D) @ kv[0].transpose(1, 2) / math.sqrt(D)
            lse[b] = torch.logsumexp(x, -1).view(-1)
            o[b] = (torch.softmax(x, -1) @ kv[1]).view(Hkv * G, D)
        return o, lse
    # the cache after the write, as fp64 code values and scales
    page, Hkv, D = c["page"], c["Hkv"], c["D"]
    pg, sl = s["slots"] // page, s["slots"] % page
    new = [_exact_turn(s["k"], s["pos"], s["table"], c["interleaved"], False), s["v"].double()]
    held, sc = [], None
    if c["fp8"]:
        sc = _two_to(s["scales"].long() - 127)
    for w, cache in enumerate((s["k_cache"], s["v_cache"])):
        t = cache.to(torch.float32).double()
        if c["fp8"]:
            t[pg, sl], sc[pg, :, w, sl] = _exact_rows(new[w])
        else:
            t[pg, sl] = new[w]
        held.append(t)
    if op == "append":
        return held + ([None] if c["fp8"] else [])
    out = []
    for w in range(2):
        parts = []
        for b in range(c["B"]):
            t = torch.arange(int(s["lens"][b]), device=DEV)
            p_, s_ = s["block_table"][b, t // page].long(), t % page
            parts.append(held[w][p_, s_] * (sc[p_, :, w, s_][..., None] if c["fp8"] else 1.0))
        out.append(torch.cat(parts))
    return tuple(out)
