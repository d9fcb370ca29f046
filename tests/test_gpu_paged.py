"""The paged cache on the GPU against the 64-bit oracle.

Bounds (u = half a step of a rounding, relative): bf16 2^-8, fp16 2^-11, fp32 2^-24.
"""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import paged as op  # noqa: E402

U16, UH, U32 = 2.0 ** -8, 2.0 ** -11, 2.0 ** -24


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from lvar_b200 import kernels
    return kernels


def make_cache(B, H, D, page, most, bits, seed, heads_last=False):
    """Random pages, a shuffled table that covers `most` rows per sequence, and NaN in the pages nobody owns."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    per = max(1, -(-most // page))
    n = B * per + 2

    def pool(loud):
        shape = (n, page, H, D) if heads_last else (n, H, page, D)
        x = torch.randn(shape, generator=g, device="cuda")
        if loud:
            x = x * torch.exp(0.5 * torch.randn(D, generator=g, device="cuda"))
        return x.transpose(1, 2) if heads_last else x

    k, v, scales = pool(True), pool(False), None
    order = torch.randperm(n, generator=g, device="cuda")
    table = order[:B * per].view(B, per).to(torch.int32).contiguous()
    if bits == 8:
        # every row with a scale of its own, over several octaves
        k, v = (x * torch.exp2(torch.randint(-3, 4, (*x.shape[:3], 1), generator=g, device="cuda").float()) for x in (k, v))
        packed, ex = [], []
        for x in (k, v):
            y, e = op.quantise(x)
            packed.append(y.float().to(torch.float8_e4m3fn))
            ex.append(e + 127)
        if heads_last:
            packed = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in packed]
        k, v = packed
        scales = torch.cat(ex, -1).to(torch.uint8).contiguous()
    else:
        k, v = k.bfloat16(), v.bfloat16()
        k[order[B * per:]] = math.nan
        v[order[B * per:]] = math.nan
    return k, v, scales, table


def bound(o, A, S, n, D, bits):
    """|error| of an output element: the last rounding, the weights' rounding (fp16 weights also lose up to 2^-25 of the
    largest, scaled by 2^15, a key: n 2^-39), and fp32: a score is off by at most (D + 8) u S (products are exact, D sums,
    four factors), which a weight and the sum of weights both take over, and exp2 by 2^-22; n sums."""
    w = (U16 if bits == 16 else UH + n * 2.0 ** -39) + 2 * (2 * (D + 8) * U32 * S + 2.0 ** -21) + n * U32
    return U16 * o.abs() + w.unsqueeze(-1) * A * (1 + U16) + 1e-30


def check_attn(K, q, k, v, table, lens, scale, scales=None, causal=False, **kw):
    bits = 8 if scales is not None else 16
    st = K.new_status("cuda")
    got, M, L = K.paged_attn_fwd(q, k, v, table, lens, scale, scales=scales, causal=causal, return_stats=True, status=st, **kw)
    o, Mr, Lr, A, S = op.attention(q, k, v, table, lens.tolist(), scale, scales, causal)
    assert K.read_status(st)[0] == 0
    D, n = q.shape[-1], max(1, int(lens.max()))
    assert torch.isfinite(got).all()
    err, tol = (got.double() - o).abs(), bound(o, A, S, n, D, bits)
    assert (err <= tol).all(), f"off by up to {(err / tol).max().item():.2f} bounds"
    empty = Mr == -math.inf
    assert torch.equal(M == -math.inf, empty) and (L[empty] == 0).all() and (got[empty] == 0).all()
    full = ~empty
    dm = ((D + 8) * U32 * S * math.log2(math.e) + 2 * U32 * Mr.abs())[full]
    assert ((M.double() - Mr).abs()[full] <= dm + 1e-30).all()
    # L is relative to the kernel's own M
    want = (Lr * torch.exp2(torch.where(empty, 0.0, Mr - M.double())))[full]
    assert ((L.double()[full] - want).abs() <= (2 * (D + 8) * U32 * S[full] + 2.0 ** -21 + n * U32) * want).all()
    return got


LENGTHS = [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257, 1000]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("Hq,H,T,page,causal", [(4, 4, 1, 64, False), (4, 1, 1, 16, True), (6, 2, 5, 48, True),
                                                (8, 1, 4, 32, True), (3, 3, 17, 128, False), (14, 2, 9, 64, True),
                                                (2, 1, 40, 512, True)])
def test_attention_over_many_lengths(K, bits, D, Hq, H, T, page, causal):
    """Rows per key head: 1, 4, 15, 32, 17, 63 and 80 (one, two or four warps of rows, one or two row tiles); lengths that
    end anywhere in tiles and pages, an empty sequence, and with `causal` tokens that see nothing."""
    B = len(LENGTHS)
    k, v, scales, table = make_cache(B, H, D, page, 1000, bits, 100 * T + D + bits)
    q = torch.randn(B, Hq, T, D, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").bfloat16()
    lens = torch.tensor(LENGTHS, dtype=torch.int32, device="cuda")
    a = check_attn(K, q, k, v, table, lens, D ** -0.5, scales, causal)
    # a cap on the lengths that shapes the launch differently changes roundings only; the same call repeats its bits
    assert torch.equal(a, K.paged_attn_fwd(q, k, v, table, lens, D ** -0.5, scales=scales, causal=causal))


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("max_len", [0, 1, 64, 128, 129, 256, 257])
def test_attention_short_bounds(K, bits, max_len):
    """Launches without a split (few tiles) and with one."""
    lens = torch.tensor([max_len, 0, (max_len + 1) // 2], dtype=torch.int32, device="cuda")
    k, v, scales, table = make_cache(3, 4, 128, 16, max_len, bits, max_len)
    q = torch.randn(3, 8, 2, 128, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").bfloat16()
    check_attn(K, q, k, v, table, lens, 0.3, scales, True, max_len=max_len)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("B,H,G,T,most", [(1, 1, 1, 1, 20011), (1, 1, 8, 1, 20011), (2, 3, 1, 20, 9000), (5, 2, 4, 2, 6000),
                                          (40, 2, 1, 1, 700), (150, 1, 2, 1, 300)])
def test_attention_split_over_the_length(K, bits, B, H, G, T, most):
    """One item over all CTAs, several items per CTA, more sequences than threads in a scan step."""
    r = random.Random(B * most)
    lens = torch.tensor([most] + [r.choice([0, 1, r.randint(1, most)]) for _ in range(B - 1)], dtype=torch.int32, device="cuda")
    k, v, scales, table = make_cache(B, H, 128, 64, most, bits, most + B)
    q = 2 * torch.randn(B, H * G, T, 128, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    check_attn(K, q.bfloat16(), k, v, table, lens, 128 ** -0.5, scales, True)


@pytest.mark.parametrize("bits", [16, 8])
def test_attention_strides(K, bits):
    """Pages with the heads inside the rows, a table with spare columns, q and out as views, a wide value range."""
    B, H, T, D, page, n = 3, 2, 3, 64, 32, 333
    k, v, scales, table = make_cache(B, H, D, page, n, bits, 8, heads_last=True)
    assert not k.is_contiguous()
    wide = torch.full((B, table.shape[1] + 5), 10 ** 9, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + table.shape[1]] = table
    table = wide[:, 2:]
    q = torch.randn(B, T, 2 * H, D + 8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6)).bfloat16()
    q = q[..., :D].transpose(1, 2)
    lens = torch.tensor([n, 65, 1], dtype=torch.int32, device="cuda")
    out = torch.full((B, T, 2 * H, 2 * D), 7.0, dtype=torch.bfloat16, device="cuda")
    view = out[..., D:].transpose(1, 2)
    got = check_attn(K, q, k, v, table, lens, D ** -0.5, scales, True, out=view)
    assert got.data_ptr() == view.data_ptr() and (out[..., :D] == 7).all()


@pytest.mark.parametrize("bits", [16, 8])
def test_attention_extreme_scores(K, bits):
    """Scores of several hundred (one key carries a row) and V rows 2^60 apart."""
    B, H, D, n = 2, 2, 128, 500
    k, v, scales, table = make_cache(B, H, D, 64, n, bits, 9)
    q = 30 * torch.randn(B, H, 2, D, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda").bfloat16()
    lens = torch.tensor([n, 77], dtype=torch.int32, device="cuda")
    check_attn(K, q, k, v, table, lens, 1.0, scales)
    if bits == 8:
        up = torch.randint(-30, 31, scales.shape[:3], generator=torch.Generator(device="cuda").manual_seed(8), device="cuda")
        scales[..., 1] = (scales[..., 1].int() + up).to(torch.uint8)
    else:
        v.mul_(torch.exp2(torch.randint(-30, 31, (*v.shape[:3], 1), generator=torch.Generator(device="cuda").manual_seed(8),
                                        device="cuda").float()).bfloat16())
    check_attn(K, q, k, v, table, lens, 1.0, scales)
    check_attn(K, q * 0, k, v, table, lens, 1.0, scales)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("G,T", [(1, 3), (8, 4), (4, 16)])
def test_values_that_a_row_does_not_see_stay_out(K, bits, G, T):
    """NaN and infinities behind the end of a sequence and in keys that only later tokens see do not reach a row; where a
    row sees one, it does."""
    B, H, D, page, n = 2, 2, 128, 32, 150
    k, v, scales, table = make_cache(B, H, D, page, n, bits, 11)
    q = torch.randn(B, H * G, T, D, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda").bfloat16()
    lens = torch.tensor([n - 30, n - 60], dtype=torch.int32, device="cuda")
    clean = K.paged_attn_fwd(q, k, v, table, lens, 0.1, scales=scales, causal=True)

    def poison(x, pos, value, where=slice(None)):
        for b in range(B):
            p = int(lens[b]) + pos
            x[int(table[b, p // page]), :, p % page, where] = value
    bad = math.nan if bits == 8 else math.inf
    for pos in range(0, 30):
        poison(k, pos, bad)
        poison(v, pos, bad)
    assert torch.equal(clean, K.paged_attn_fwd(q, k, v, table, lens, 0.1, scales=scales, causal=True))
    poison(k, -1, math.nan)
    poison(v, -1, bad, slice(40, 60))
    got = K.paged_attn_fwd(q, k, v, table, lens, 0.1, scales=scales, causal=True)
    assert torch.equal(clean[:, :, :T - 1], got[:, :, :T - 1]) and torch.isnan(got[:, :, T - 1]).all()
    # a row that sees an infinite V with weight > 0 takes it, in its columns only
    k, v, scales, table = make_cache(B, H, D, page, n, bits, 11)
    poison(v, -1, bad, slice(40, 60))
    got = K.paged_attn_fwd(q, k, v, table, lens, 0.1, scales=scales, causal=True)
    assert torch.equal(clean[:, :, :T - 1], got[:, :, :T - 1])
    last = got[:, :, T - 1]
    assert (torch.isnan(last) if bits == 8 else last == math.inf)[..., 40:60].all()
    assert torch.equal(last[..., :40], clean[:, :, T - 1, :40]) and torch.equal(last[..., 60:], clean[:, :, T - 1, 60:])


def test_bad_pages_and_lengths_set_the_status(K):
    k, v, _, table = make_cache(2, 2, 64, 16, 100, 16, 12)
    k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    q = torch.randn(2, 2, 1, 64, device="cuda").bfloat16()
    lens = torch.tensor([100, 50], dtype=torch.int32, device="cuda")
    st = K.new_status("cuda")
    got = K.paged_attn_fwd(q, k, v, table, lens, max_len=60, status=st)
    assert K.read_status(st)[0] == 5  # the first sequence is cut at 60 keys
    cut = torch.tensor([60, 50], dtype=torch.int32, device="cuda")
    assert torch.equal(got, K.paged_attn_fwd(q, k, v, table, cut, max_len=60))
    for page in (-1, k.shape[0], 2 ** 31 - 1):
        t = table.clone()
        t[0, 1] = page
        for call in (lambda s: K.paged_attn_fwd(q, k, v, t, lens, status=s),
                     lambda s: K.paged_kv_read(k, v, t, lens, 100, status=s)):
            st = K.new_status("cuda")
            call(st)
            assert K.read_status(st)[0] == 5
    t = table.clone()
    t[0, 1] = -1
    rk, rv = K.paged_kv_read(k, v, t, lens, 100)
    assert (rk[0, :, 16:32] == 0).all() and (rv[0, :, 16:32] == 0).all() and (rk[0, :, 32:] != 0).any()
    # entries behind a sequence's end are not looked at
    t = table.clone()
    t[1, 4:] = 2 ** 31 - 1
    st = K.new_status("cuda")
    assert torch.equal(K.paged_attn_fwd(q, k, v, t, lens, status=st), K.paged_attn_fwd(q, k, v, table, lens))
    K.paged_kv_read(k, v, t, lens, 100, status=st)
    assert K.read_status(st)[0] == 0


# -- writing and reading -----------------------------------------------------------------------------
def empty_cache(n, H, page, D, bits):
    if bits == 8:
        k = torch.full((n, H, page, D), 0x31, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        return k, k.clone(), torch.full((n, H, page, 2), 99, dtype=torch.uint8, device="cuda")
    k = torch.full((n, H, page, D), 7.0, dtype=torch.bfloat16, device="cuda")
    return k, k.clone(), None


def place(table, page, start, b, l):
    p = int(start[b]) + l
    return int(table[b, p // page]), p % page


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("B,H,L,D,page", [(1, 1, 1, 128, 16), (3, 5, 37, 64, 16), (2, 3, 70, 128, 48), (4, 2, 300, 64, 64), (3, 1, 51, 64, 16), (2, 1, 33, 128, 32)])
def test_append_and_read(K, bits, B, H, L, D, page):
    """Exact: rows, their scales, everything around them, and the way back."""
    g = torch.Generator(device="cuda").manual_seed(L + D)
    x = torch.randn(B, L, 2, H, D, generator=g, device="cuda") * torch.exp2(
        torch.randint(-40, 41, (B, L, 2, H, 1), generator=g, device="cuda").float())
    x[0, 0, 0, 0] = 0.0
    if L > 30:
        x[0, 3, 0, 0, 5], x[0, 4, 1, 0, 6], x[0, 5, 0, 0] = math.nan, math.inf, -math.inf
        x[0, 6, 0, 0], x[0, 7, 0, 0] = 1e-35, 3e38
        x[0, 8, 0, 0], x[0, 9, 0, 0, :2] = 448.0, torch.tensor([450.0, -2.0])
    x = x.bfloat16()
    k, v = x[:, :, 0].transpose(1, 2), x[:, :, 1].transpose(1, 2)
    start = torch.tensor([(11 * b + 5) % 40 for b in range(B)], dtype=torch.int32, device="cuda")
    count = torch.tensor([L if b == 0 else (L * b) // B for b in range(B)], dtype=torch.int32, device="cuda")
    per = -(-(40 + L) // page)
    kp, vp, sc = empty_cache(B * per + 1, H, page, D, bits)
    table = torch.randperm(B * per + 1, generator=g, device="cuda")[:B * per].view(B, per).to(torch.int32)
    st = K.new_status("cuda")
    K.paged_kv_append(k, v, kp, vp, table, start, scales=sc, count=count, status=st)
    assert K.read_status(st)[0] == 0
    wk, wv, ws = empty_cache(B * per + 1, H, page, D, bits)
    n = int((start + count).max()) + 3
    back = torch.zeros(2, B, H, n, D, dtype=torch.float64, device="cuda")
    for i, (src, pool) in enumerate(((k, wk), (v, wv))):
        if bits == 8:
            y, e = op.quantise(src)
        for b in range(B):
            for l in range(int(count[b])):
                pg, row = place(table, page, start, b, l)
                if bits == 8:
                    pool[pg, :, row] = y[b, :, l].float().to(torch.float8_e4m3fn)
                    ws[pg, :, row, i] = (e[b, :, l, 0] + 127).to(torch.uint8)
                    back[i, b, :, int(start[b]) + l] = y[b, :, l] * torch.exp2(e[b, :, l].double())
                else:
                    pool[pg, :, row] = src[b, :, l]
                    back[i, b, :, int(start[b]) + l] = src[b, :, l].double()
    if bits == 8:
        nan = [(a.view(torch.uint8) & 0x7F) == 0x7F for a in (kp, vp, wk, wv)]
        assert torch.equal(nan[0], nan[2]) and torch.equal(nan[1], nan[3])
        assert torch.equal(kp.view(torch.uint8)[~nan[0]], wk.view(torch.uint8)[~nan[0]])
        assert torch.equal(vp.view(torch.uint8)[~nan[1]], wv.view(torch.uint8)[~nan[1]])
        assert torch.equal(sc, ws)
    else:
        assert torch.equal(kp.view(torch.int16), wk.view(torch.int16)) and torch.equal(vp.view(torch.int16), wv.view(torch.int16))
    # back: from the first written row on (what lies before is another owner's), zeros behind the end
    end = start + count
    for first in (0, 17):
        rk, rv = K.paged_kv_read(kp, vp, table, end, n, scales=sc, start=first, status=st)
        assert K.read_status(st)[0] == 0
        for i, r in enumerate((rk, rv)):
            for b in range(B):
                lo, hi = max(first, int(start[b])), min(int(end[b]), n)
                want = back[i, b, :, lo:hi].bfloat16()
                got = r[b, :, lo - first:max(lo, hi) - first]
                assert torch.equal(got.nan_to_num(9e9, 8e9, -8e9), want.nan_to_num(9e9, 8e9, -8e9))
                assert (r[b, :, max(0, int(end[b]) - first):] == 0).all()


@pytest.mark.parametrize("bits", [16, 8])
def test_read_into_views(K, bits):
    B, H, D, n = 2, 3, 128, 130
    k, v, sc, table = make_cache(B, H, D, 32, n, bits, 21, heads_last=True)
    lens = torch.tensor([n, 77], dtype=torch.int32, device="cuda")
    buf = torch.full((2, B, n + 4, H, D), 7.0, dtype=torch.bfloat16, device="cuda")
    out = (buf[0, :, 2:2 + n].transpose(1, 2), buf[1, :, 2:2 + n].transpose(1, 2))
    got = K.paged_kv_read(k, v, table, lens, n, scales=sc, out=out)
    assert got[0].data_ptr() == out[0].data_ptr()
    for b in range(B):
        for i, pool in enumerate((k, v)):
            assert torch.equal(out[i][b, :, :int(lens[b])].double(), op.rows(pool, sc, i, table, b, int(lens[b])))
            assert (out[i][b, :, int(lens[b]):] == 0).all()
    assert (buf[:, :, :2] == 7).all() and (buf[:, :, 2 + n:] == 7).all()


NORMS = ["none", "l2", "rms", "rms plain"]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("norm", NORMS)
@pytest.mark.parametrize("B,L,Hq,H,D", [(3, 1, 8, 2, 128), (2, 19, 5, 5, 64), (2, 9, 3, 1, 128), (1, 700, 16, 16, 128)])
def test_prologue(K, bits, halves, norm, B, L, Hq, H, D):
    """fp32 arithmetic on the widened inputs, rounded once: an element is off by its last rounding and by 32 u of the
    magnitudes that its rotation adds (at most 12 sums and a root in the norm, three factors, the rotation's two products)."""
    page = 16
    g = torch.Generator(device="cuda").manual_seed(31 + L)
    x = torch.randn(B, L, Hq + 2 * H, D, generator=g, device="cuda").bfloat16()
    if L > 1:
        x[0, 1, :, :] = 0.0
    q, k, v = x[:, :, :Hq], x[:, :, Hq:Hq + H], x[:, :, Hq + H:]
    start = torch.tensor([3 + 13 * b for b in range(B)], dtype=torch.int32, device="cuda")
    per = -(-(3 + 13 * B + L) // page)
    kp, vp, sc = empty_cache(B * per, H, page, D, bits)
    table = torch.randperm(B * per, generator=g, device="cuda").view(B, per).to(torch.int32)
    angle = torch.arange(per * page, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (
        -torch.arange(D // 2, dtype=torch.float64, device="cuda") * 2 / D)
    kw = {"rope_cos": angle.cos().float(), "rope_sin": angle.sin().float(), "rope_halves": halves}
    ref = {"cos": kw["rope_cos"], "sin": kw["rope_sin"], "halves": halves}
    if norm == "none":
        kw, ref = ({}, {}) if halves else (kw, ref)
    elif norm == "l2":
        kw["scale_mul"] = ref["scale_mul"] = torch.rand(Hq, generator=g, device="cuda") + 0.5
    else:
        kw["eps"] = ref["eps"] = 1e-6
        if norm == "rms":
            for n in ("q_weight", "k_weight"):
                kw[n] = ref[n] = torch.randn(D, generator=g, device="cuda")
    st = K.new_status("cuda")
    got = K.paged_qkv_prologue(q, k, v, kp, vp, table, start, scales=sc, status=st, **kw)
    assert K.read_status(st)[0] == 0
    wq, wk, sq, sk = op.prologue(q, k, start=start.tolist(), **ref)
    assert ((got.transpose(1, 2).double() - wq).abs() <= U16 * wq.abs() + 33 * U32 * sq + 1e-38).all()
    if norm == "none" and halves:
        assert torch.equal(got, q.transpose(1, 2))
    for b in range(B):
        for l in range(0, L, 1 if L < 50 else 97):
            pg, row = place(table, page, start, b, l)
            if bits == 16:
                assert torch.equal(vp[pg, :, row], v[b, l])
                assert ((kp[pg, :, row].double() - wk[b, l]).abs() <= U16 * wk[b, l].abs() + 33 * U32 * sk[b, l] + 1e-38).all()
            else:
                y, e = op.quantise(v[b, l])
                assert torch.equal(vp[pg, :, row].double(), y) and torch.equal(sc[pg, :, row, 1].int() - 127, e[:, 0].int())
                e = sc[pg, :, row, 0].double() - 127
                most = wk[b, l].abs().amax(-1)
                slack = 33 * U32 * sk[b, l].amax(-1)
                assert ((most - slack) * torch.exp2(-e) <= 448).all()
                assert (((most + slack) * torch.exp2(1 - e) > 448) | (e == op.E_MIN)).all()
                up = torch.exp2(e)[:, None]
                tol = torch.maximum(2.0 ** -4 * wk[b, l].abs(), 2.0 ** -10 * up) + 40 * U32 * sk[b, l]
                assert ((kp[pg, :, row].double() * up - wk[b, l]).abs() <= tol).all()


def test_prologue_is_the_contiguous_one_with_pages(K):
    """The same arguments through the contiguous prologue: equal but for rare flips of the last bf16 bit (the contiguous
    form divides by the norm and rounds the rotation's products one by one)."""
    B, L, H, D = 2, 64, 4, 128
    g = torch.Generator(device="cuda").manual_seed(41)
    qkv = torch.randn(B, L, 3, H, D, generator=g, device="cuda").bfloat16()
    mul = torch.rand(H, generator=g, device="cuda") + 1
    ang = torch.rand(100, D // 2, generator=g, device="cuda") * 6
    cos, sin = ang.cos(), ang.sin()
    kc, vc = (torch.zeros(B, H, 100, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q0 = K.qkv_prologue(qkv, mul, cos, sin, 10, kc, vc, 10)
    kp, vp, _ = empty_cache(2 * 7, H, 16, D, 16)
    table = torch.randperm(14, generator=g, device="cuda").view(2, 7).to(torch.int32)
    start = torch.full((B,), 10, dtype=torch.int32, device="cuda")
    q1 = K.paged_qkv_prologue(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], kp, vp, table, start, scale_mul=mul, rope_cos=cos, rope_sin=sin)
    k1, v1 = K.paged_kv_read(kp, vp, table, start + L, L, start=10)
    for a, b in ((q0, q1), (kc[:, :, 10:10 + L], k1)):
        a, b = a.double(), b.double()
        # two roundings of values at most 70 u32 of the rotated magnitudes apart
        assert ((a - b).abs() <= 2 * U16 * a.abs() + 70 * U32 * 4).all() and (a == b).double().mean() > 0.99
    assert torch.equal(vc[:, :, 10:10 + L], v1)


def test_padding_and_places_without_a_page(K):
    """Rows behind `count` are not written and give q = 0; positions without a page or a table row set the status."""
    B, L, H, D, page = 3, 4, 2, 64, 16
    x = torch.randn(B, L, 3 * H, D, device="cuda").bfloat16()
    q, k, v = x[:, :, :H], x[:, :, H:2 * H], x[:, :, 2 * H:]
    table = torch.tensor([[0, 1], [2, -1], [3, 7]], dtype=torch.int32, device="cuda")
    count = torch.tensor([2, 0, 4], dtype=torch.int32, device="cuda")
    start = torch.tensor([14, 30, 0], dtype=torch.int32, device="cuda")
    cos = torch.ones(18, D // 2, device="cuda")
    for bits in (16, 8):
        kp, vp, sc = empty_cache(4, H, page, D, bits)
        st = K.new_status("cuda")
        o = K.paged_qkv_prologue(q, k, v, kp, vp, table, start, scales=sc, count=count, rope_cos=cos, rope_sin=0 * cos, status=st)
        assert K.read_status(st)[0] == 0
        assert (o[0, :, 2:] == 0).all() and (o[1] == 0).all() and torch.equal(o[2], q[2].transpose(0, 1))
        before = [t.clone() for t in (kp, vp)]
        for s in ([32, 0, 0], [-1, 0, 0], [2 ** 31 - 1, 0, 0]):  # behind the table, negative, past every bound
            st = K.new_status("cuda")
            K.paged_kv_append(k.transpose(1, 2)[:1], v.transpose(1, 2)[:1], kp, vp, table[:1],
                              torch.tensor(s[:1], dtype=torch.int32, device="cuda"), scales=sc, status=st)
            assert K.read_status(st)[0] == 5
        st = K.new_status("cuda")
        K.paged_kv_append(k.transpose(1, 2)[1:], v.transpose(1, 2)[1:], kp, vp, table[1:],
                          torch.tensor([16, 16], dtype=torch.int32, device="cuda"), scales=sc, status=st)
        assert K.read_status(st)[0] == 5  # pages -1 and 7 of 4
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, (kp, vp)))


# -- a run of them together --------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [16, 8])
def test_generation_steps_in_a_graph(K, bits):
    """Ragged sequences, a prompt through the prologue, then steps of one token: prologue, attention and the lengths' update
    captured once and replayed; every step against the oracle on the cache read back.  Two graphs of the same stream replay
    at the same time on two streams."""
    B, Hq, H, D, page, most = 5, 8, 2, 128, 16, 400
    g = torch.Generator(device="cuda").manual_seed(51)
    per = -(-most // page)
    ang = torch.arange(most, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (
        -torch.arange(D // 2, dtype=torch.float64, device="cuda") * 2 / D)
    cos, sin = ang.cos().float(), ang.sin().float()
    wq, wk = (1 + 0.1 * torch.randn(D, generator=g, device="cuda") for _ in range(2))

    def world(seed):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        kp, vp, sc = empty_cache(B * per, H, page, D, bits)
        table = torch.randperm(B * per, generator=gen, device="cuda").view(B, per).to(torch.int32)
        w = {"kp": kp, "vp": vp, "sc": sc, "table": table, "lens": torch.zeros(B, dtype=torch.int32, device="cuda"),
             "x": torch.zeros(B, 1, Hq + 2 * H, D, dtype=torch.bfloat16, device="cuda"), "gen": gen}
        prompt = torch.randn(B, 300, Hq + 2 * H, D, generator=gen, device="cuda").bfloat16()
        count = torch.tensor([300, 1, 0, 299, 64], dtype=torch.int32, device="cuda")
        step(w, prompt, count)
        w["lens"] += count
        return w

    def step(w, x, count=None):
        q = K.paged_qkv_prologue(x[:, :, :Hq], x[:, :, Hq:Hq + H], x[:, :, Hq + H:], w["kp"], w["vp"], w["table"], w["lens"],
                                 scales=w["sc"], eps=1e-5, q_weight=wq, k_weight=wk, rope_cos=cos, rope_sin=sin, rope_halves=True,
                                 count=count)
        return q

    def decode(w):
        q = step(w, w["x"])
        w["lens"] += 1
        return q, K.paged_attn_fwd(q, w["kp"], w["vp"], w["table"], w["lens"], scales=w["sc"], causal=True)

    def capture(w):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            w["q"], w["o"] = decode(w)
        return graph

    worlds = [world(1), world(2)]
    graphs = [capture(w) for w in worlds]
    streams = [torch.cuda.Stream() for _ in worlds]
    for _ in range(4):
        for w in worlds:
            w["x"].copy_(torch.randn(w["x"].shape, generator=w["gen"], device="cuda"))
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for w in worlds:
            lens = w["lens"].tolist()
            o, _, _, A, S = op.attention(w["q"], w["kp"], w["vp"], w["table"], lens, D ** -0.5, w["sc"])
            assert ((w["o"].double() - o).abs() <= bound(o, A, S, max(lens), D, bits)).all()
            # the newest row is in the cache
            k, v = K.paged_kv_read(w["kp"], w["vp"], w["table"], w["lens"], max(lens), scales=w["sc"])
            for b, n in enumerate(lens):
                want, _ = op.quantise(w["x"][b, 0, Hq + H:]) if bits == 8 else (w["x"][b, 0, Hq + H:], None)
                if bits == 8:
                    want = want * torch.exp2(_.double())
                assert torch.equal(v[b, :, n - 1].double(), want.double())


def test_calls_on_two_streams_at_once(K):
    """Eager calls of one shape on two streams share nothing."""
    k, v, _, table = make_cache(4, 2, 128, 64, 5000, 16, 61)
    q = torch.randn(4, 8, 1, 128, device="cuda").bfloat16()
    lens = torch.tensor([5000, 4000, 17, 1200], dtype=torch.int32, device="cuda")
    want = [K.paged_attn_fwd(x, k, v, table, lens) for x in (q, -q)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(K.paged_attn_fwd(q if i == 0 else -q, k, v, table, lens))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_offsets_beyond_32_bits(K):
    """A page whose byte offset passes 2^32 and, with heads apart, 2^31 elements."""
    page, H, D = 512, 8, 128
    n = 2 ** 32 // (H * page * D * 2) + 40
    k = torch.empty(n, H, page, D, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    g = torch.Generator(device="cuda").manual_seed(71)
    table = torch.tensor([[n - 1, 1, n - 3]], dtype=torch.int32, device="cuda")
    x = torch.randn(1, H, 1100, D, generator=g, device="cuda").bfloat16()
    K.paged_kv_append(x, -x, k, v, table, torch.zeros(1, dtype=torch.int32, device="cuda"))
    lens = torch.tensor([1100], dtype=torch.int32, device="cuda")
    rk, rv = K.paged_kv_read(k, v, table, lens, 1100)
    assert torch.equal(rk, x) and torch.equal(rv, -x)
    q = torch.randn(1, H, 1, D, generator=g, device="cuda").bfloat16()
    check_attn(K, q, k, v, table, lens, D ** -0.5)


def test_refusals(K):
    k, v, sc, table = make_cache(2, 2, 64, 16, 64, 8, 81)
    kb, vb, _, _ = make_cache(2, 2, 64, 16, 64, 16, 81)
    n = torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    q = torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16, device="cuda")
    x = torch.zeros(2, 2, 1, 64, dtype=torch.bfloat16, device="cuda")
    t = torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16, device="cuda")
    cos = torch.zeros(70, 32, device="cuda")
    one = torch.ones(2, device="cuda")
    w = torch.ones(64, device="cuda")
    bad = [
        lambda: K.paged_attn_fwd(q, k, v, table, n), lambda: K.paged_attn_fwd(q, kb, vb, table, n, scales=sc),
        lambda: K.paged_attn_fwd(q.half(), kb, vb, table, n), lambda: K.paged_attn_fwd(q[:, :3], kb, vb, table, n),
        lambda: K.paged_attn_fwd(q, kb, vb, table.long(), n), lambda: K.paged_attn_fwd(q, kb, vb, table, n.long()),
        lambda: K.paged_attn_fwd(q, kb, vb, table, n[:1]), lambda: K.paged_attn_fwd(q, kb, vb, table[:1], n),
        lambda: K.paged_attn_fwd(q, kb, vb, table, n.cpu()), lambda: K.paged_attn_fwd(q, kb, vb[:3], table, n),
        lambda: K.paged_attn_fwd(q, k, v, table, n, scales=sc[:3]), lambda: K.paged_attn_fwd(q, kb, vb, table, n, 0.0),
        lambda: K.paged_attn_fwd(q, kb, vb, table, n, max_len=-1), lambda: K.paged_attn_fwd(q, kb, vb, table, n, out=q[:1]),
        lambda: K.paged_attn_fwd(torch.zeros(2, 4, 1, 32, dtype=torch.bfloat16, device="cuda"), kb, vb, table, n),
        lambda: K.paged_attn_fwd(q, kb, vb, table, n, status=torch.zeros(1, device="cuda")),
        lambda: K.paged_kv_append(x, x[:1], kb, vb, table, n), lambda: K.paged_kv_append(q, q, kb, vb, table, n),
        lambda: K.paged_kv_append(x, x, kb, vb, table, n, count=n.float()),
        lambda: K.paged_attn_fwd(q, kb, vb, table, n, max_len=1 << 40), lambda: K.paged_kv_read(kb, vb, table, n, 1 << 40),
        lambda: K.paged_kv_read(kb, vb, table, n, 5, start=-1), lambda: K.paged_kv_read(kb, vb, table, n, -1),
        lambda: K.paged_kv_read(kb, vb, table, n, 5, out=(x, x)),
        lambda: K.paged_qkv_prologue(t, t, t, kb, vb, table, n, scale_mul=one, eps=1e-6),
        lambda: K.paged_qkv_prologue(t, t, t, kb, vb, table, n, q_weight=w),
        lambda: K.paged_qkv_prologue(t, t, t, kb, vb, table, n, rope_cos=cos),
        lambda: K.paged_qkv_prologue(t, t, t, kb, vb, table, n, rope_cos=cos[:, :16], rope_sin=cos[:, :16]),
        lambda: K.paged_qkv_prologue(t, t, t, kb, vb, table, n, scale_mul=one.double()),
        lambda: K.paged_qkv_prologue(t, t, t, kb, vb, table, n, eps=1e-6, k_weight=w[:32]),
        lambda: K.paged_qkv_prologue(t[:, :, :1], t, t, kb, vb, table, n),
        lambda: K.paged_qkv_prologue(t[..., ::2], t, t, kb, vb, table, n),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was not refused")
    # nothing to do is no error
    assert K.paged_attn_fwd(q[:, :, :0], kb, vb, table, n).shape == (2, 4, 0, 64)
    assert K.paged_kv_read(kb, vb, table, n, 0)[0].shape == (2, 2, 0, 64)
    K.paged_kv_append(x[:, :, :0], x[:, :, :0], kb, vb, table, n)


def test_padding_stays_zero_without_eps(K):
    """A root-mean-square norm without eps is 0 / 0 for a row of zeros, but a row of padding is 0."""
    x = torch.zeros(2, 3, 6, 64, dtype=torch.bfloat16, device="cuda")
    kp, vp, _ = empty_cache(2, 2, 16, 64, 16)
    table = torch.tensor([[0], [1]], dtype=torch.int32, device="cuda")
    zero, count = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    o = K.paged_qkv_prologue(x[:, :, :2], x[:, :, 2:4], x[:, :, 4:], kp, vp, table, zero, eps=0.0, count=count)
    assert torch.isnan(o[0, :, 0]).all() and (o[0, :, 1:] == 0).all() and (o[1] == 0).all()
    assert torch.isnan(kp[0, :, 0]).all() and (kp[0, :, 1:] == 7).all() and (kp[1] == 7).all()


@pytest.mark.parametrize("bits", [16, 8])
def test_many_sequences(K, bits):
    """Thousands of sequences, most of them empty or of a few keys."""
    r = random.Random(5)
    B = 3001
    n = [r.choice([0, 0, 1, r.randint(1, 30), 300]) for _ in range(B)]
    k, v, scales, _ = make_cache(40, 1, 64, 16, 300, bits, 101)
    if bits == 16:
        k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    table = torch.randint(0, k.shape[0], (B, 19), generator=torch.Generator(device="cuda").manual_seed(6), device="cuda").to(torch.int32)
    q = torch.randn(B, 2, 1, 64, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda").bfloat16()
    check_attn(K, q, k, v, table, torch.tensor(n, dtype=torch.int32, device="cuda"), 0.125, scales)


@pytest.mark.parametrize("bits", [16, 8])
def test_a_million_keys(K, bits):
    """One sequence whose table names the same few pages over and over."""
    n = 1200003
    k, v, scales, _ = make_cache(30, 1, 64, 512, 512, bits, 103)
    if bits == 16:
        k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    table = (torch.arange(-(-n // 512), device="cuda") * 7 % k.shape[0]).to(torch.int32)[None]
    q = 2 * torch.randn(1, 4, 2, 64, generator=torch.Generator(device="cuda").manual_seed(8), device="cuda")
    check_attn(K, q.bfloat16(), k, v, table, torch.tensor([n], dtype=torch.int32, device="cuda"), 0.125, scales, True)


def test_cache_object_and_table(K):
    """Sequences that come, grow and go over fewer pages than all of them at full length would take."""
    from lvar_b200.paged import PagedKVCache, PageTable
    table = PageTable(3, 200, page_size=16, num_pages=20)
    for dtype in (torch.bfloat16, torch.float8_e4m3fn):
        cache = PagedKVCache(20, 2, 64, 16, dtype)
        g = torch.Generator(device="cuda").manual_seed(91)
        held = [torch.zeros(2, 0, 64, device="cuda") for _ in range(3)]
        for grow in ([30, 100, 0], [40, 0, 90], [0, -1, 0], [33, 60, 17]):
            for s, n in enumerate(grow):
                if n < 0:
                    table.release(s)
                    held[s] = held[s][:, :0]
            start = torch.tensor([h.shape[1] for h in held], dtype=torch.int32, device="cuda")
            count = torch.tensor([max(n, 0) for n in grow], dtype=torch.int32, device="cuda")
            table.reserve_all({s: held[s].shape[1] + max(n, 0) for s, n in enumerate(grow)})
            if max(grow) > 0:
                x = torch.randn(3, 2, max(grow), 64, generator=g, device="cuda").bfloat16()
                st = K.new_status("cuda")
                cache.append(x, x, table.table, start, count=count, status=st)
                assert K.read_status(st)[0] == 0
                for s, n in enumerate(grow):
                    held[s] = torch.cat([held[s], x[s, :, :max(n, 0)].float()], 1)
        lens = torch.tensor([h.shape[1] for h in held], dtype=torch.int32, device="cuda")
        k, v = cache.read(table.table, lens, int(lens.max()))
        for s in range(3):
            want = held[s].double()
            if dtype != torch.bfloat16:
                y, e = op.quantise(want)
                want = y * torch.exp2(e.double())
            assert torch.equal(k[s, :, :int(lens[s])].double(), want) and torch.equal(k[s], v[s])
        q = torch.randn(3, 4, 1, 64, generator=g, device="cuda").bfloat16()
        assert torch.equal(cache.attend(q, table.table, lens, 0.2), K.paged_attn_fwd(q, cache.k, cache.v, table.table, lens, 0.2,
                                                                                    scales=cache.scales))
        for s in range(3):
            table.release(s)


def test_a_wait_that_runs_out_ends_in_a_status(K):
    """A wait limit of zero: the call gives up at its first unfinished wait and returns, and the next one is whole."""
    for bits in (16, 8):
        for T, G in ((1, 1), (5, 7)):
            for n in (100, 9000):
                k, v, sc, table = make_cache(2, 2, 128, 64, n, bits, 95)
                q = torch.randn(2, 2 * G, T, 128, device="cuda").bfloat16()
                lens = torch.tensor([n, n // 3], dtype=torch.int32, device="cuda")
                st = K.new_status("cuda")
                K.paged_attn_fwd(q, k, v, table, lens, scales=sc, status=st, wait_limit_ns=0)
                assert K.read_status(st)[0] in (0, 6)  # 0: nothing had to wait
                check_attn(K, q, k, v, table, lens, 128 ** -0.5, sc)


def loop_of(cache, mode, seed=1):
    from lvar_b200 import infinity_loop as IL
    lc = IL.LoopConfig(depth=4, width=256, heads=2, ffn=512, text_dim=64, text_len=8, code_dim=8, scales=(1, 2, 4, 8, 16, 24),
                       attn_mode=mode, cache=cache)
    return IL.InfinityLoop(lc, batch=2, seed=seed)


@pytest.mark.parametrize("mode", ["sparse", "dense"])
def test_generation_loop_over_pages(K, mode):
    """The generation loop with its cache in pages: the routes are the contiguous one's, a captured graph replays the eager
    result bit for bit, and after the same layer inputs a layer's cache is the contiguous one's up to roundings (with e4m3
    pages: up to those of the rows)."""
    from lvar_b200 import sparse_attn_config as cfg
    saved = dict(cfg.GLOBAL_CONFIG["attn"])
    try:
        cfg.GLOBAL_CONFIG["attn"].update(decision_scale=3, bound_layer=1, top_keys=0.3, cs4a_ws=[1, 1, 1, 1, 3, 5],
                                         attn_sink=2, win_size=[-1, -1, 1, 1, 3, 5])
        text = torch.randn(2, 8, 64, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
        base = loop_of("contiguous", mode)
        base.generate(text, seed=4)
        routes = dict(base.routes)
        for cache in ("paged", "paged_e4m3"):
            loop = loop_of(cache, mode)
            out = loop.generate(text, seed=4).clone()
            assert loop.routes == routes and torch.isfinite(out).all()
            assert torch.equal(loop.generate(text, seed=4), out)
            loop.capture(text, seed=4)
            assert torch.equal(loop.replay(), out)
            # one layer's step on the same projection: contiguous and paged caches with the same history
            for si in range(len(base.cum) - 1):
                gen = torch.Generator(device="cuda").manual_seed(si)
                xn = torch.randn(4, base.cum[si + 1] - base.cum[si], 256, generator=gen, device="cuda").bfloat16()
                for x in (base, loop):
                    assert torch.isfinite(x._self_attention(x.blocks[3], 3, xn, si)).all()
                k, v = loop.paged[3].read(loop.pages.table, loop.lens[si + 1], base.cum[si + 1])
                kc, vc = base.k_cache[3][:, :, :base.cum[si + 1]], base.v_cache[3][:, :, :base.cum[si + 1]]
                assert torch.equal(loop.lens[si], torch.full_like(loop.lens[si], base.cum[si]))
                if cache == "paged":
                    assert torch.equal(v, vc)
                    # two roundings of values at most 70 u32 of the rotated magnitudes (below 1) apart
                    assert ((k.double() - kc.double()).abs() <= 2 * U16 * kc.double().abs() + 140 * U32).all()
                else:
                    for x, y in ((k, kc), (v, vc)):
                        # e4m3 rounds by 2^-4 of an element or half the row's smallest step, 2^-10 * 2^e with
                        # 2^e <= max / 224; the bf16 rounding of the other side comes on top
                        most = y.double().abs().amax(-1, keepdim=True)
                        assert ((x.double() - y.double()).abs() <= (2.0 ** -4 + 2 * U16) * y.double().abs() + most / 224 * 2.0 ** -9 + 140 * U32).all()
    finally:
        cfg.GLOBAL_CONFIG["attn"].clear()
        cfg.GLOBAL_CONFIG["attn"].update(saved)


class _TakesNothing:
    """The compiled entry as it answers calls that it leaves to the checks in Python."""

    @staticmethod
    def _none(*_):
        return None
    attn = append = prologue = read = _none


@pytest.mark.parametrize("bits", [16, 8])
def test_both_entries_make_the_same_call(K, bits, monkeypatch):
    """The compiled entry and the Python one: the same launches from the same arguments, bit for bit."""
    B, L, Hq, H, D, page = 3, 5, 6, 2, 64, 32
    g = torch.Generator(device="cuda").manual_seed(111)
    x = torch.randn(B, L, Hq + 2 * H, D, generator=g, device="cuda").bfloat16()
    q, k, v = x[:, :, :Hq], x[:, :, Hq:Hq + H], x[:, :, Hq + H:]
    start = torch.tensor([0, 40, 17], dtype=torch.int32, device="cuda")
    count = torch.tensor([5, 2, 0], dtype=torch.int32, device="cuda")
    table = torch.arange(6, device="cuda").view(3, 2).to(torch.int32)
    ang = torch.rand(64, D // 2, generator=g, device="cuda")
    kinds = [{}, {"scale_mul": torch.rand(Hq, generator=g, device="cuda")}, {"eps": 1e-5},
             {"eps": 1e-5, "q_weight": torch.rand(D, generator=g, device="cuda"), "k_weight": torch.rand(D, generator=g, device="cuda")}]

    def all_of_them():
        out = []
        for kw in kinds:
            for rope in ({}, {"rope_cos": ang, "rope_sin": ang, "rope_halves": True}):
                kp, vp, sc = empty_cache(6, H, page, D, bits)
                st = K.new_status("cuda")
                out.append(K.paged_qkv_prologue(q, k, v, kp, vp, table, start, scales=sc, count=count, status=st, **kw, **rope))
                K.paged_kv_append(k.transpose(1, 2), v.transpose(1, 2), kp, vp, table, start + 6, scales=sc, status=st)
                out += [kp, vp, st] + ([] if sc is None else [sc])
                out += K.paged_kv_read(kp, vp, table, start + 11, 60, scales=sc, start=1, status=st)
                qh = q.transpose(1, 2)
                out.append(K.paged_attn_fwd(qh, kp, vp, table, start + 11, scales=sc, status=st))
                out += K.paged_attn_fwd(qh, kp, vp, table, start + 11, 0.3, scales=sc, causal=True, max_len=60, return_stats=True,
                                        status=st, wait_limit_ns=10 ** 9)
                out += K.paged_attn_fwd(qh, kp, vp, table.repeat(1, 20), start + 11, scales=sc, return_stats=True)
                assert K.read_status(st)[0] == 0
        return [t.clone().view(torch.uint8) for t in out]
    a = all_of_them()
    monkeypatch.setattr(K, "_paged_host", _TakesNothing)
    b = all_of_them()
    assert len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_the_compiled_entry_leaves_wrong_calls_alone(K):
    """It answers None, raises only where a number is none, and keeps no reference that it should not."""
    import sys
    from lvar_b200 import _paged_host as host
    k, v, sc, table = make_cache(2, 2, 64, 16, 64, 16, 81)
    n = torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    q = torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16, device="cuda")
    good = [q, k, v, table, n, 0.1, None, False, None, False, None, None]
    for i, wrong in ((0, q.cpu()), (0, q.half()), (0, None), (0, q[:, :3]), (1, k[:, :, :, ::2]), (3, table.long()), (4, n.long()),
                     (4, None), (6, torch.zeros(1)), (8, -1), (8, 1 << 40), (8, "x"), (10, q), (11, -1)):
        args = list(good)
        args[i] = wrong
        assert host.attn(*args) is None, i
    with pytest.raises(TypeError):
        host.attn(*good[:-1])
    with pytest.raises(TypeError):
        host.attn(*good[:5], "scale", *good[6:])
    before = [sys.getrefcount(x) for x in (q, k, v, table, n)]
    for _ in range(50):
        host.attn(*good)
    assert before == [sys.getrefcount(x) for x in (q, k, v, table, n)]
    assert sys.getrefcount(host.attn(*good)) <= 2


@pytest.mark.parametrize("bits,D", [(16, 128), (8, 128), (16, 64), (8, 64)])
@pytest.mark.parametrize("G,T", [(1, 1), (2, 5), (4, 8), (7, 5)])
def test_a_wait_that_runs_out_many_tiles_into_a_ring(K, bits, D, G, T):
    """Every CTA has more tiles than its ring has stages: a call whose waits run out ends with a status (always, where the
    limit is zero; one that ends without a status is whole), and the next call has the bits it had before."""
    B, H, n = 2, 4, 80000
    k, v, sc, table = make_cache(B, H, D, 64, n, bits, 191)
    q = torch.randn(B, H * G, T, D, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda").bfloat16()
    lens = torch.tensor([n, n - 777], dtype=torch.int32, device="cuda")
    good = K.new_status("cuda")
    want = K.paged_attn_fwd(q, k, v, table, lens, scales=sc, causal=True, status=good)
    for limit in (0, 0, 0, 1000, 5000, 20000, 0):
        st = K.new_status("cuda")
        got = K.paged_attn_fwd(q, k, v, table, lens, scales=sc, causal=True, status=st, wait_limit_ns=limit)
        code = K.read_status(st)[0]
        if limit == 0:
            assert code == 6
        else:
            assert code in (0, 1, 3)
            assert code != 0 or torch.equal(got, want)
        assert torch.equal(K.paged_attn_fwd(q, k, v, table, lens, scales=sc, causal=True, status=good), want)
    assert K.read_status(good)[0] == 0


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D,G,T", [(128, 1, 1), (64, 8, 1), (128, 4, 4), (64, 3, 3), (128, 5, 7), (64, 8, 8)])
def test_infinite_values_wherever_they_lie(K, D, G, T, causal):
    """An element of V that is +inf or -inf makes the output's element the same infinity (its weight is positive), and two
    of opposite signs make NaN, whatever the key's place in a tile, whatever the weights' last bits and however many rows
    share the key; the other columns keep their bits.  Rows of 1, 8, 16, 9, 35 and 64; every place of two tiles and some
    behind them."""
    H, page, n = 2, 32, 400
    at = list(range(0, 150)) + list(range(150, n - T, 23)) + [n - T]
    B = len(at)
    k, v, _, _ = make_cache(B, H, D, page, n, 16, 11)
    per = -(-n // page)
    table = torch.arange(B * per, device="cuda").view(B, per).to(torch.int32)
    k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    q = torch.randn(B, H * G, T, D, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda").bfloat16()
    lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
    clean = K.paged_attn_fwd(q, k, v, table, lens, 0.1, causal=causal)
    for b, p in enumerate(at):
        row = v[int(table[b, p // page]), :, p % page]
        row[:, 20:30], row[:, 30:40], row[:, 40:41] = math.inf, -math.inf, math.inf
        p2 = (p + 37) % (n - T)  # another key that every token sees
        if p2 != p:
            v[int(table[b, p2 // page]), :, p2 % page, 40] = -math.inf
    got = K.paged_attn_fwd(q, k, v, table, lens, 0.1, causal=causal)
    assert (got[..., 20:30] == math.inf).all() and (got[..., 30:40] == -math.inf).all() and torch.isnan(got[..., 40]).all()
    assert torch.equal(got[..., :20], clean[..., :20]) and torch.equal(got[..., 41:], clean[..., 41:])


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("B,L,Hq,H,D", [(1, 2, 3, 1, 128), (2, 5, 4, 4, 64), (1, 900, 16, 16, 128), (1, 1100, 16, 16, 64)])
def test_norms_of_rows_that_are_not_finite(K, bits, B, L, Hq, H, D):
    """A NaN makes its row's norm NaN and with it the whole row; an infinity makes its own element NaN and the others 0, with
    either norm.  Few and many rows per lane."""
    g = torch.Generator(device="cuda").manual_seed(131 + L)
    clean = torch.randn(B, L, Hq + 2 * H, D, generator=g, device="cuda").bfloat16()
    x = clean.clone()
    x[0, 0, 0, 3] = math.nan                 # a query row
    x[0, L - 1, Hq, D - 1] = math.nan        # a key row
    x[B - 1, 1, Hq - 1, 7] = -math.inf
    x[B - 1, 0, Hq + H - 1, 0] = math.inf
    x[0, L // 2, Hq + H, 1] = math.nan       # a value row
    page = 16
    per = -(-L // page)
    table = torch.arange(B * per, device="cuda").view(B, per).to(torch.int32)
    start, lens = (torch.full((B,), n, dtype=torch.int32, device="cuda") for n in (0, L))
    for kw in ({"scale_mul": torch.rand(Hq, generator=g, device="cuda") + 0.5}, {"eps": 1e-6}):
        out = []
        for y in (clean, x):
            kp, vp, sc = empty_cache(B * per, H, page, D, bits)
            q = K.paged_qkv_prologue(y[:, :, :Hq], y[:, :, Hq:Hq + H], y[:, :, Hq + H:], kp, vp, table, start, scales=sc, **kw)
            out.append((q, *K.paged_kv_read(kp, vp, table, lens, L, scales=sc)))
        wq, wk, _, _ = op.prologue(x[:, :, :Hq], x[:, :, Hq:Hq + H], start=[0] * B, **kw)
        wv = x[:, :, Hq + H:].double()
        for i, want in enumerate((wq, wk, wv)):
            want = want.transpose(1, 2)
            bad = ~torch.isfinite(x[:, :, (0, Hq, Hq + H)[i]:(Hq, Hq + H, Hq + 2 * H)[i]]).all(-1).transpose(1, 2)
            a, b = out[0][i], out[1][i]
            assert bad.any() and torch.equal(a[~bad], b[~bad])
            assert torch.equal(torch.isnan(b[bad]), torch.isnan(want[bad])), i
            if i < 2:
                assert (b[bad].nan_to_num(0.0) == 0).all()


@pytest.mark.parametrize("B,H,L,D", [(1, 1, 3, 128), (1, 3, 5, 64), (1, 16, 1600, 128), (1, 16, 1600, 64), (1, 8, 3000, 64)])
def test_scale_of_rows_without_a_finite_element(K, B, H, L, D):
    """Elements that are not finite take no part in a row's maximum: a row of nothing else has the least exponent, whatever
    the rows beside it hold."""
    g = torch.Generator(device="cuda").manual_seed(141)
    per = -(-L // 16)
    table = torch.arange(per, device="cuda").view(1, per).to(torch.int32)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    for rows in ([math.nan], [math.nan, math.inf], [-math.inf]):
        x = torch.randn(B, H, L, D, generator=g, device="cuda").bfloat16()
        for i, value in enumerate(rows):
            x[0, (H - 1) * (1 - i), i::3] = value
        kp, vp, sc = empty_cache(per, H, 16, D, 8)
        K.paged_kv_append(x, x.flip(1), kp, vp, table, zero, scales=sc)
        for i, y in enumerate((x, x.flip(1))):
            _, e = op.quantise(y)
            got = sc[..., i].transpose(0, 1).reshape(H, -1)[:, :L]
            assert torch.equal(got.int() - 127, e[0, :, :, 0].int())
        qkv = x.transpose(1, 2)
        K.paged_qkv_prologue(qkv, qkv, qkv, kp, vp, table, zero, scales=sc, scale_mul=torch.ones(H, device="cuda"))
        bad = ~torch.isfinite(x[0]).any(-1)
        got = sc.transpose(0, 1).reshape(H, -1, 2)[:, :L]
        assert bad.any() and (got[bad] == 27).all() and (got[~bad] > 100).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,H,T,n", [(2, 2, 1, 2), (8, 1, 1, 64), (16, 2, 2, 130), (3, 3, 5, 1000), (4, 1, 4, 20000)])
def test_weights_of_few_rows_are_not_rounded_once(K, D, Hq, H, T, n):
    """Up to 16 rows per key head over a bf16 cache: a weight is the sum of two bf16 numbers.  The first leaves at most 2^-8
    of it (half a step), the second rounds that by 2^-9 of its own value (it lies below the half step of 1, or is exact), so
    2^-17 of the weight is lost in place of 2^-8.  V rows come in pairs x, -x and scores are small, so that what an output
    element has is the difference of nearly equal weights and its own rounding hides nothing."""
    k, v, _, table = make_cache(2, H, D, 64, n, 16, 161)
    k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    v[:, :, 1::2] = -v[:, :, 0::2]
    q = torch.randn(2, Hq, T, D, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda").bfloat16()
    lens = torch.tensor([n, (n + 1) // 2], dtype=torch.int32, device="cuda")
    scale = 0.1 / D
    got = K.paged_attn_fwd(q, k, v, table, lens, scale)
    o, _, _, A, S = op.attention(q, k, v, table, lens.tolist(), scale)
    fp32 = 2 * (2 * (D + 8) * U32 * S + 2.0 ** -21) + n * U32
    tol = U16 * o.abs() + (2.0 ** -17 + fp32).unsqueeze(-1) * A * (1 + U16) + 1e-30
    err = (got.double() - o).abs()
    assert (err <= tol).all(), f"off by up to {(err / tol).max().item():.2f} bounds"


def scatter(pool, table, page, start, count, rows):
    """Puts rows [B, L, H, ...] (l < count[b]) at positions start[b] + l of a pool [pages, H, page, ...]."""
    b, l = torch.nonzero(torch.arange(rows.shape[1], device="cuda")[None] < count[:, None], as_tuple=True)
    pos = start.long()[b] + l
    rows = rows.to(pool.dtype)
    if pool.dtype == torch.float8_e4m3fn:
        pool, rows = pool.view(torch.uint8), rows.view(torch.uint8)
    pool[table.long()[b, pos // page], :, pos % page] = rows[b, l]


def same(a, b):
    """Equal bytes, but for which NaN stands where both have one."""
    if a.dtype == torch.float8_e4m3fn:
        a, b = a.view(torch.uint8), b.view(torch.uint8)
        return bool(((a == b) | (((a & 0x7F) == 0x7F) & ((b & 0x7F) == 0x7F))).all())
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def with_odd_rows(x, g):
    """x [B, L, H, D] in which every eleventh row or so is zero, tiny, huge, or has NaN and infinities in it."""
    kind = torch.randint(0, 77, (*x.shape[:-1], 1), generator=g, device="cuda")
    col = torch.arange(x.shape[-1], device="cuda")
    for i, value in enumerate((0.0, 1e-35, 3e38, math.nan, math.inf, -math.inf)):
        x = torch.where((kind == i) if i < 3 else (kind == i) & (col % 9 == i), torch.full_like(x, value), x)
    return x.bfloat16()


# The heads that make a lane take four or two rows (whole and partial last groups), and calls just large enough for that.
MANY = [(64, 16, 1500), (64, 13, 1900), (64, 8, 3000), (64, 7, 3400), (128, 8, 1500), (128, 7, 1800), (128, 4, 3000), (128, 3, 4000)]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("D,H,L", MANY)
def test_append_with_several_rows_per_lane(K, bits, D, H, L):
    """Exact, everything around the rows included; NaN and infinities among the rows of a warp."""
    g = torch.Generator(device="cuda").manual_seed(171 + H)
    B, page = 2, 48
    x = torch.randn(B, L, 2 * H, D, generator=g, device="cuda") * torch.exp2(
        torch.randint(-40, 41, (B, L, 2 * H, 1), generator=g, device="cuda").float())
    x = with_odd_rows(x, g)
    k, v = x[:, :, :H], x[:, :, H:]
    start = torch.tensor([5, 50], dtype=torch.int32, device="cuda")
    count = torch.tensor([L, L - 77], dtype=torch.int32, device="cuda")
    per = -(-(50 + L) // page)
    table = torch.randperm(B * per + 1, generator=g, device="cuda")[:B * per].view(B, per).to(torch.int32)
    kp, vp, sc = empty_cache(B * per + 1, H, page, D, bits)
    wk, wv, ws = empty_cache(B * per + 1, H, page, D, bits)
    st = K.new_status("cuda")
    K.paged_kv_append(k.transpose(1, 2), v.transpose(1, 2), kp, vp, table, start, scales=sc, count=count, status=st)
    assert K.read_status(st)[0] == 0
    for i, (src, pool) in enumerate(((k, wk), (v, wv))):
        if bits == 8:
            y, e = op.quantise(src)
            scatter(pool, table, page, start, count, y.float().to(torch.float8_e4m3fn))
            scatter(ws[..., i], table, page, start, count, (e + 127)[..., 0])
        else:
            scatter(pool, table, page, start, count, src)
    assert same(kp, wk) and same(vp, wv) and (bits == 16 or same(sc, ws))


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("norm", ["l2", "rms", "none"])
@pytest.mark.parametrize("D,Hq,H,L", [(64, 16, 16, 600), (64, 20, 5, 900), (64, 8, 8, 1100), (128, 8, 8, 600), (128, 10, 5, 700),
                                      (128, 4, 4, 1100)])
def test_prologue_with_several_rows_per_lane(K, bits, halves, norm, D, Hq, H, L):
    """The bounds of test_prologue, for every row."""
    g = torch.Generator(device="cuda").manual_seed(181 + Hq)
    B, page = 2, 48
    x = torch.randn(B, L, Hq + 2 * H, D, generator=g, device="cuda").bfloat16()
    odd = with_odd_rows(x[:, :, Hq + H:].float(), g)
    q, k, v = x[:, :, :Hq], x[:, :, Hq:Hq + H], odd
    start = torch.tensor([3, 16], dtype=torch.int32, device="cuda")
    per = -(-(16 + L) // page)
    table = torch.randperm(B * per, generator=g, device="cuda").view(B, per).to(torch.int32)
    angle = torch.arange(per * page, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (
        -torch.arange(D // 2, dtype=torch.float64, device="cuda") * 2 / D)
    kw = {"rope_cos": angle.cos().float(), "rope_sin": angle.sin().float(), "rope_halves": halves}
    ref = {"cos": kw["rope_cos"], "sin": kw["rope_sin"], "halves": halves}
    if norm == "l2":
        kw["scale_mul"] = ref["scale_mul"] = torch.rand(Hq, generator=g, device="cuda") + 0.5
    elif norm == "rms":
        kw["eps"] = ref["eps"] = 1e-6
        for n in ("q_weight", "k_weight"):
            kw[n] = ref[n] = torch.randn(D, generator=g, device="cuda")
    kp, vp, sc = empty_cache(B * per, H, page, D, bits)
    st = K.new_status("cuda")
    got = K.paged_qkv_prologue(q, k, v, kp, vp, table, start, scales=sc, status=st, **kw)
    assert K.read_status(st)[0] == 0
    wq, wk, sq, sk = op.prologue(q, k, start=start.tolist(), **ref)
    assert ((got.transpose(1, 2).double() - wq).abs() <= U16 * wq.abs() + 33 * U32 * sq + 1e-38).all()
    pos = start.long()[:, None] + torch.arange(L, device="cuda")
    at = table.long().gather(1, pos // page)
    rows = [t.view(torch.uint8)[at, :, pos % page].view(t.dtype) if bits == 8 else t[at, :, pos % page] for t in (kp, vp)]
    if bits == 16:
        assert ((rows[0].double() - wk).abs() <= U16 * wk.abs() + 33 * U32 * sk + 1e-38).all()
        assert same(rows[1], v)
    else:
        e = sc[at, :, pos % page].double() - 127
        y, ev = op.quantise(v)
        assert torch.equal(e[..., 1], ev[..., 0].double()) and same(rows[1], y.float().to(torch.float8_e4m3fn))
        most, slack, up = wk.abs().amax(-1), 33 * U32 * sk.amax(-1), torch.exp2(e[..., :1])
        assert ((most - slack) * torch.exp2(-e[..., 0]) <= 448).all()
        assert ((most + slack) * torch.exp2(1 - e[..., 0]) > 448).all()
        tol = torch.maximum(2.0 ** -4 * wk.abs(), 2.0 ** -10 * up) + 40 * U32 * sk
        assert ((rows[0].double() * up - wk).abs() <= tol).all()
