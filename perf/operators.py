"""Cases of the paged key/value cache: writing it (plain append, and the fused norm / rotation prologue), reading rows
back, and attention of a few new tokens over it, each in a plain form (elementary torch operations in 32 bits) and as
the framework's calls.

Layouts: cache pages [pages, kv heads, page_size, D], bf16 or e4m3 with one power-of-two scale per row (its biased
exponent in ``scales`` [pages, kv heads, page_size, 2], K's and V's); page tables int32 [B, pages per sequence]; lengths
and start positions int32 [B] on the device.
"""
import math

import torch

own = False

PAD = -1  # table entry of a page that a sequence does not own


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def _attn(name, B, T, Hq, Hkv, D, length, ragged, bits, page, causal, stats=False):
    return {"name": name, "kind": "attn", "B": B, "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "length": length, "ragged": ragged,
            "bits": bits, "page": page, "causal": causal, "stats": stats}


def _write(name, kind, B, L, Hq, Hkv, D, history, ragged, bits, page, norm="none", halves=False):
    return {"name": name, "kind": kind, "B": B, "L": L, "Hq": Hq, "Hkv": Hkv, "D": D, "history": history,
            "ragged": ragged, "bits": bits, "page": page, "norm": norm, "halves": halves}


def listed():
    return [
        # the first token of two prompts (with and without the condition): nothing but latency
        _attn("attn first scale", 2, 1, 16, 16, 128, 1, False, 16, 64, False),
        # the 8 x 8 token scale of eight guided prompts, every token sees all 121 cached ones
        _attn("attn scale 8x8", 16, 64, 16, 16, 128, 121, False, 8, 64, False),
        # one token for each of 32 sequences of any length up to a whole image, grouped heads, 8-bit cache
        _attn("attn decode ragged", 32, 1, 32, 8, 128, 10521, True, 8, 64, True),
        # few sequences with a very long cache: the split over the cache's length carries it
        _attn("attn long", 3, 1, 16, 2, 128, 131071, False, 16, 64, True, True),
        # five tokens at once with a causal order, seven query heads to a key head, small pages
        _attn("attn draft tokens", 16, 5, 28, 4, 128, 4121, True, 16, 16, True),
        # the small head dimension, as many key heads as query heads, many sequences
        _attn("attn d64", 64, 1, 16, 16, 64, 2521, True, 8, 32, False),
        # the largest: whole images for 24 sequences at full heads in bf16
        _attn("attn largest", 24, 1, 16, 16, 128, 10521, False, 16, 128, False),
        # a decoding step's norms, rotation and cache rows for 64 sequences at different positions
        _write("prologue decode", "prologue", 64, 1, 32, 8, 128, 1000, True, 16, 64, "rms", True),
        # the 64 x 64 token scale of a guided prompt
        _write("prologue scale 64x64", "prologue", 2, 4096, 16, 16, 128, 6425, False, 16, 64, "l2", False),
        # the 32 x 32 token scale into an 8-bit cache, and the whole cache back for the many-token attention kernels
        _write("prologue and read 8 bit", "prologue_read", 8, 1024, 16, 16, 128, 1497, False, 8, 64, "l2", False),
        # projected text keys of ragged length into an 8-bit cache and back
        _write("append text and read", "append_read", 16, 64, 20, 20, 64, 0, True, 8, 16),
        # a finished prefix moves from contiguous buffers into pages
        _write("append prefix", "append", 4, 6425, 16, 16, 128, 0, False, 16, 64),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "prologue", "prologue_read", "append_read", "append"])
    D, bits, page = rng.choice([64, 128]), rng.choice([8, 16]), rng.choice([16, 32, 48, 64, 128])
    B, ragged = _log(rng, 1, 64), rng.random() < 0.5
    Hkv = rng.choice([1, 2, 3, 4, 5, 8, 16])
    G = rng.choice([1, 1, 2, 4, 7, 8])
    if kind == "attn":
        T = _log(rng, 1, 64)
        length = _log(rng, 1, 131072)
        while B * Hkv * length * D * bits > 1.0e9 * 8:
            B, length = max(1, B // 2), max(1, length * 3 // 4)
        while B * Hkv * G * T * length > 1.0e8:  # scores of the plain form
            T, length = max(1, T // 2), max(1, length * 3 // 4)
        return {k: v for k, v in _attn("", B, T, Hkv * G, Hkv, D, length, ragged, bits, page, rng.random() < 0.5,
                                       rng.random() < 0.3).items() if k != "name"}
    L, history = _log(rng, 1, 4096), rng.choice([0, _log(rng, 1, 6425)])
    while B * (L + history) * (G + 2) * Hkv * D > 1.0e8:
        B, L, history = max(1, B // 2), max(1, L * 3 // 4), history * 3 // 4
    if kind in ("append", "prologue"):
        bits = 16
    norm = rng.choice(["l2", "rms", "none"]) if kind.startswith("prologue") else "none"
    return {k: v for k, v in _write("", kind, B, L, Hkv * G, Hkv, D, history, ragged, bits, page, norm,
                                    rng.random() < 0.5).items() if k != "name"}


def _spread(n, most, ragged):
    """n lengths up to `most`: all alike, or spread over 0 .. most, the longest and (of eight or more) an empty one among
    them."""
    if not ragged:
        return [most] * n
    spread = [int((most + 1) * ((i * 0.6180339887) % 1.0)) for i in range(n)]
    spread[0] = most
    return spread if n < 8 else spread[:-1] + [0]


def _pages_per_sequence(case):
    most = case["length"] if case["kind"] == "attn" else case["history"] + case["L"]
    return -(-most // case["page"])


def work(case):
    B, Hq, Hkv, D, bits = case["B"], case["Hq"], case["Hkv"], case["D"], case["bits"]
    row = 2 * (D * bits // 8 + (1 if bits == 8 else 0))  # K and V of one token and head in the cache
    if case["kind"] == "attn":
        T, lens = case["T"], _spread(B, case["length"], case["ragged"])
        seen = sum(sum(max(0, n - T + t + 1) for t in range(T)) if case["causal"] else T * n for n in lens)
        out = 2 * B * Hq * T * D * 2 + (8 * B * Hq * T if case["stats"] else 0)
        return {"bytes": sum(lens) * Hkv * row + out, "flops": 4.0 * D * Hq * seen}
    new = sum(_spread(B, case["L"], case["ragged"])) if case["kind"].startswith("append") else B * case["L"]
    old = sum(_spread(B, case["history"], case["ragged"]))
    plain = 2 * 2 * D * Hkv  # K and V of one token in bf16
    if case["kind"] == "append":
        return {"bytes": new * (plain + row * Hkv), "flops": 0.0}
    if case["kind"] == "append_read":
        return {"bytes": new * (plain + 2 * row * Hkv) + B * case["L"] * plain + old * (plain + row * Hkv), "flops": 0.0}
    moved = new * (2 * 2 * D * Hq + plain + row * Hkv)
    flops = 8.0 * new * (Hq + Hkv) * D
    if case["kind"] == "prologue":
        return {"bytes": moved, "flops": flops}
    return {"bytes": moved + (old + new) * row * Hkv + B * (case["history"] + case["L"]) * plain, "flops": flops}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _quantised(x):
    """Rows of x (fp32) as e4m3 with a power-of-two scale: (e4m3 values, biased exponents uint8 [..., 1])."""
    fine = torch.isfinite(x)
    most = torch.where(fine, x.abs(), torch.zeros_like(x)).amax(-1, keepdim=True)
    m, e = torch.frexp(most)
    e = torch.where(m > 0.875, e - 8, e - 9)  # 448 = 0.875 * 2^9: the least e with most * 2^-e <= 448
    e = torch.where(most > 0, e, torch.full_like(e, -100)).clamp(-100, 120).to(torch.int32)
    scaled = torch.where(fine, x, torch.full_like(x, math.nan)) * ((127 - e) << 23).view(torch.float32)
    return scaled.to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _exponents(b):
    """2^(b - 127) in fp32 for biased exponents of normal numbers."""
    return (b.to(torch.int32) << 23).view(torch.float32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, Hq, Hkv, D, page, bits = case["B"], case["Hq"], case["Hkv"], case["D"], case["page"], case["bits"]
    per = _pages_per_sequence(case)
    pages = B * per + 3
    attn = case["kind"] == "attn"
    loud = torch.exp(0.6 * torch.randn(Hkv, 1, D, generator=g, device="cuda"))  # some channels of K are louder than others

    def values(channel):
        x = torch.randn(pages, Hkv, page, D, generator=g, device="cuda")
        if channel:
            x = x * loud
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True))
        return x

    s = {"case": dict(case)}
    shuffled = torch.randperm(pages, generator=g, device="cuda")
    order, free = shuffled[: B * per].view(B, per).to(torch.int32), shuffled[B * per:]
    if attn:
        lens = _spread(B, case["length"], case["ragged"])
    else:
        lens = _spread(B, case["history"], case["ragged"])
    lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    turn = torch.randperm(B, generator=g, device="cuda")
    lens = lens[turn]
    if attn:  # pages that no token uses are not owned
        order = torch.where(torch.arange(per, device="cuda")[None] * page < lens[:, None], order, torch.full_like(order, PAD))
    s["table"], s["lens"] = order.contiguous(), lens
    if bits == 8:
        k8, ke = _quantised(values(True))
        v8, ve = _quantised(values(False))
        s["k"], s["v"], s["scales"] = k8, v8, torch.cat([ke, ve], -1).contiguous()
    else:
        s["k"], s["v"], s["scales"] = values(True).bfloat16(), values(False).bfloat16(), None
        if attn:  # nobody's pages hold anything
            s["k"][free], s["v"][free] = math.nan, math.nan
    if attn:
        s["q"] = (1.5 * torch.randn(B, Hq, case["T"], D, generator=g, device="cuda")).bfloat16()
        s["scale"] = D ** -0.5
    else:
        L = case["L"]
        x = torch.randn(B, L, Hq + 2 * Hkv, D, generator=g, device="cuda").bfloat16()  # one projection's output
        s["xq"], s["xk"], s["xv"] = x[:, :, :Hq], x[:, :, Hq:Hq + Hkv], x[:, :, Hq + Hkv:]
        counts = _spread(B, L, case["ragged"]) if case["kind"].startswith("append") else [L] * B
        s["count"] = torch.tensor(counts, dtype=torch.int32, device="cuda")[turn]
        s["scale_mul"] = torch.rand(Hq, generator=g, device="cuda") * 3.0 + 1.0
        s["wq"] = 1.0 + 0.2 * torch.randn(D, generator=g, device="cuda")
        s["wk"] = 1.0 + 0.2 * torch.randn(D, generator=g, device="cuda")
        most = case["history"] + L
        freq = 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64, device="cuda") * 2.0 / D)
        angle = torch.arange(most, dtype=torch.float64, device="cuda")[:, None] * freq[None]
        s["cos"], s["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
        s["most"] = most
        s["after"] = lens + s["count"]
    return s


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------
def _rows_plain(s, which, n):
    """Rows 0 .. n-1 of every sequence of the cache in fp32, [B, Hkv, n, D]; zeros where a sequence has no page."""
    data, table = s[which], s["table"].long()
    B, per = table.shape
    page, D = data.shape[2], data.shape[3]
    at = table.clamp(min=0)
    if s["scales"] is None:
        x = data[at].float()
    else:
        x = data.view(torch.uint8)[at].view(torch.float8_e4m3fn).float()
        x = x * _exponents(s["scales"][..., 0 if which == "k" else 1][at]).unsqueeze(-1)
    x = x.permute(0, 2, 1, 3, 4).reshape(B, data.shape[1], per * page, D)[:, :, :n]
    return x


def _attn_plain(s):
    c, q, lens = s["case"], s["q"], s["lens"]
    B, Hq, T, D = q.shape
    Hkv, n = c["Hkv"], c["length"]
    G = Hq // Hkv
    j = torch.arange(n, device=q.device)
    there = (j[None] < lens[:, None])[:, None, :, None]
    k = torch.where(there, _rows_plain(s, "k", n), 0.0)
    v = torch.where(there, _rows_plain(s, "v", n), 0.0)
    x = torch.matmul(q.float().view(B, Hkv, G * T, D), k.transpose(2, 3)) * s["scale"]
    x = x.view(B, Hkv, G, T, n)
    limit = lens[:, None].expand(B, T)
    if c["causal"]:
        limit = lens[:, None] - T + 1 + torch.arange(T, device=q.device)[None]
    x = torch.where(j < limit[:, None, None, :, None], x, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Hkv, G * T, n), v).view(B, Hkv, G, T, D) / torch.where(total > 0, total, 1.0)
    o = o.reshape(B, Hq, T, D).bfloat16()
    if not c["stats"]:
        return o
    return o, (m * math.log2(math.e)).reshape(B, Hq, T), total.reshape(B, Hq, T)


def _rotated(x, cos, sin, halves):
    D = x.shape[-1]
    if halves:
        a, b = x[..., : D // 2], x[..., D // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)


def _put_plain(s, k, v):
    """Writes rows (fp32 [B, L, Hkv, D]) at positions lens + l of every sequence where l < count."""
    B, L, Hkv, D = k.shape
    page = s["k"].shape[2]
    l = torch.arange(L, device=k.device)
    pos = s["lens"][:, None].long() + l[None]
    b, l = torch.nonzero(l[None] < s["count"][:, None], as_tuple=True)
    pos = pos[b, l]
    at, row = s["table"].long()[b, pos // page], pos % page
    for i, (which, x) in enumerate((("k", k), ("v", v))):
        x = x[b, l]
        if s["scales"] is None:
            s[which][at, :, row] = x.bfloat16()
        else:
            x8, e = _quantised(x)
            s[which].view(torch.uint8)[at, :, row] = x8.view(torch.uint8)
            s["scales"][at, :, row, i] = e[..., 0]


def _read_plain(s):
    j = torch.arange(s["most"], device=s["lens"].device)
    there = (j[None] < s["after"][:, None])[:, None, :, None]
    return [torch.where(there, _rows_plain(s, w, s["most"]), 0.0).bfloat16() for w in ("k", "v")]


def _prologue_plain(s):
    c = s["case"]
    q, k, v = s["xq"].float(), s["xk"].float(), s["xv"].float()
    if c["norm"] == "l2":
        q = q / torch.sqrt(q.square().sum(-1, keepdim=True)).clamp(min=1e-12) * s["scale_mul"][:, None]
        k = k / torch.sqrt(k.square().sum(-1, keepdim=True)).clamp(min=1e-12)
    elif c["norm"] == "rms":
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * s["wq"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + 1e-6) * s["wk"]
    pos = s["lens"][:, None].long() + torch.arange(c["L"], device=q.device)[None]
    cos, sin = s["cos"][pos].unsqueeze(2), s["sin"][pos].unsqueeze(2)
    q, k = _rotated(q, cos, sin, c["halves"]), _rotated(k, cos, sin, c["halves"])
    _put_plain(s, k, v)
    return q.transpose(1, 2).contiguous().bfloat16()


def _run_plain(s):
    kind = s["case"]["kind"]
    if kind == "attn":
        return _attn_plain(s)
    if kind.startswith("prologue"):
        q = _prologue_plain(s)
        return [q, s["k"], s["v"]] if kind == "prologue" else [q] + _read_plain(s)
    _put_plain(s, s["xk"].float(), s["xv"].float())
    return [s["k"], s["v"]] if kind == "append" else _read_plain(s)


# ------------------------------------------------------------------------------------------------
# the framework's calls
# ------------------------------------------------------------------------------------------------
def _run_own(s):
    from lvar_b200 import kernels as K
    c, k, v, table, scales = s["case"], s["k"], s["v"], s["table"], s["scales"]
    kind = c["kind"]
    if kind == "attn":
        return K.paged_attn_fwd(s["q"], k, v, table, s["lens"], s["scale"], scales=scales, causal=c["causal"],
                                max_len=c["length"], return_stats=c["stats"])
    if kind.startswith("prologue"):
        norm = {"l2": {"scale_mul": s["scale_mul"]}, "rms": {"q_weight": s["wq"], "k_weight": s["wk"], "eps": 1e-6},
                "none": {}}[c["norm"]]
        q = K.paged_qkv_prologue(s["xq"], s["xk"], s["xv"], k, v, table, s["lens"], scales=scales, rope_cos=s["cos"],
                                 rope_sin=s["sin"], rope_halves=c["halves"], **norm)
        return [q, k, v] if kind == "prologue" else [q, *K.paged_kv_read(k, v, table, s["after"], s["most"], scales=scales)]
    K.paged_kv_append(s["xk"].transpose(1, 2), s["xv"].transpose(1, 2), k, v, table, s["lens"], scales=scales, count=s["count"])
    return [k, v] if kind == "append" else list(K.paged_kv_read(k, v, table, s["after"], s["most"], scales=scales))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------
# 64-bit values from the definitions
# ------------------------------------------------------------------------------------------------
def _sequence64(s, which, b, n):
    """The first n rows of sequence b, fp64 [Hkv, n, D]."""
    page = s["k"].shape[2]
    ids = s["table"][b, : -(-n // page)].long()
    raw = s[which].view(torch.uint8)[ids] if s["scales"] is not None else s[which][ids]
    x = (raw.view(torch.float8_e4m3fn) if s["scales"] is not None else raw).double()
    if s["scales"] is not None:
        x = x * torch.exp2(s["scales"][ids][..., 0 if which == "k" else 1].double() - 127.0)[..., None]
    return x.transpose(0, 1).flatten(1, 2)[:, :n]


def _exact_attn(s):
    c, q = s["case"], s["q"].double()
    B, Hq, T, D = q.shape
    G = Hq // c["Hkv"]
    o = torch.zeros(B, Hq, T, D, dtype=torch.float64, device="cuda")
    M = torch.full((B, Hq, T), -math.inf, dtype=torch.float64, device="cuda")
    total = torch.zeros(B, Hq, T, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        k, v = _sequence64(s, "k", b, n), _sequence64(s, "v", b, n)
        for t in range(T):
            see = max(0, n - (T - 1 - t)) if c["causal"] else n
            if see == 0:
                continue
            x = torch.einsum("hgd,hnd->hgn", q[b, :, t].view(-1, G, D), k[:, :see]) * (s["scale"] * math.log2(math.e))
            top = x.max(-1, keepdim=True).values
            w = torch.exp2(x - top)
            total[b, :, t], M[b, :, t] = w.sum(-1).flatten(), top.flatten()
            o[b, :, t] = (torch.einsum("hgn,hnd->hgd", w, v[:, :see]) / w.sum(-1, keepdim=True)).flatten(0, 1)
    return (o, M, total) if c["stats"] else o


def _stored64(x):
    """What an 8-bit row keeps of x (fp64): the nearest e4m3 multiple of the row's power of two, ties to even."""
    most = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(most.clamp(min=1e-300) / 448.0))
    e = torch.where(most * torch.exp2(-e) > 448.0, e + 1, torch.where(most * torch.exp2(1 - e) <= 448.0, e - 1, e)).clamp(-100, 120)
    y = x * torch.exp2(-e)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * torch.exp2(e)


def _exact_write(s):
    c = s["case"]
    q, k, v = s["xq"].double(), s["xk"].double(), s["xv"].double()
    D = c["D"]
    if c["norm"] == "l2":
        q = q / q.norm(dim=-1, keepdim=True).clamp(min=1e-12) * s["scale_mul"].double()[:, None]
        k = k / k.norm(dim=-1, keepdim=True).clamp(min=1e-12)
    elif c["norm"] == "rms":
        q = q / (q.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * s["wq"].double()
        k = k / (k.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * s["wk"].double()
    if c["kind"].startswith("prologue"):
        i = torch.arange(D // 2, device="cuda")
        first, second = (i, i + D // 2) if c["halves"] else (2 * i, 2 * i + 1)
        for b, n in enumerate(s["lens"].tolist()):
            turn = torch.complex(s["cos"][n:n + c["L"]].double(), s["sin"][n:n + c["L"]].double())[:, None]
            for x in (q, k):
                z = torch.complex(x[b][..., first], x[b][..., second]) * turn
                x[b, ..., first], x[b, ..., second] = z.real, z.imag
    if c["bits"] == 8:
        k, v = _stored64(k), _stored64(v)
    page, lens, count, after = c["page"], s["lens"].tolist(), s["count"].tolist(), s["after"].tolist()
    out = [q.transpose(1, 2)] if c["kind"].startswith("prologue") else []
    for which, x in (("k", k), ("v", v)):
        if c["kind"] in ("prologue", "append"):
            pool = s[which].double()
            for b in range(c["B"]):
                for p in range(lens[b] // page, -(-after[b] // page)):
                    lo, hi = max(lens[b], p * page), min(after[b], (p + 1) * page)
                    pool[s["table"][b, p].long(), :, lo - p * page:hi - p * page] = x[b, lo - lens[b]:hi - lens[b]].transpose(0, 1)
            out.append(pool)
        else:
            rows = torch.zeros(c["B"], c["Hkv"], s["most"], D, dtype=torch.float64, device="cuda")
            for b in range(c["B"]):
                if lens[b]:
                    rows[b, :, :lens[b]] = _sequence64(s, which, b, lens[b])
                rows[b, :, lens[b]:after[b]] = x[b, :count[b]].transpose(0, 1)
            out.append(rows)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_attn(s) if case["kind"] == "attn" else _exact_write(s)
