"""The paged cache without a GPU: the 64-bit oracle, the C structs' mirrors, the exact page division, and what the library
refuses before it touches a device."""
import ctypes as C
import math
import re
from pathlib import Path

import pytest
import torch

from oracle import paged as op

ROOT = Path(__file__).resolve().parent.parent


def test_nearest_e4m3_is_torchs_conversion():
    y = torch.cat([torch.linspace(-448, 448, 20001), torch.linspace(-2.0 ** -5, 2.0 ** -5, 20001)]).float()
    assert torch.equal(op.nearest_e4m3(y.double()), y.to(torch.float8_e4m3fn).double())


def test_exponent_is_the_least_that_fits():
    most = torch.tensor([448.0, 448.5, 447.9, 1.0, 2.0 ** -20, 3.0e38, 1e-40, 0.0, 224.0, 225.0], dtype=torch.float64)
    e = op.exponent(most)
    for m, x in zip(most.tolist(), e.tolist()):
        if m and op.E_MIN < x:
            assert m * 2.0 ** -x <= 448.0 < m * 2.0 ** (1 - x)
    assert e.tolist()[:2] == [0, 1] and e[7] == op.E_MIN and e[6] == op.E_MIN


def test_quantised_rows_are_bf16_numbers():
    x = torch.randn(64, 128, generator=torch.Generator().manual_seed(0)) * torch.logspace(-6, 6, 64)[:, None]
    y, e = op.quantise(x)
    value = y * torch.exp2(e.double())
    assert torch.equal(value.bfloat16().double(), value)
    assert ((value - x.double()).abs() <= torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * torch.exp2(e.double()))).all()


def test_attention_oracle_is_softmax():
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(3, 2, 16, 64, generator=g).bfloat16() for _ in range(2))
    q = torch.randn(1, 4, 3, 64, generator=g).bfloat16()
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32)
    n = 37
    kk, vv = (torch.cat([x[2], x[0], x[1]], 1)[:, :n].double().repeat_interleave(2, 0) for x in (k, v))
    for causal in (False, True):
        o, M, L, _, _ = op.attention(q, k, v, table, [n], 0.2, causal=causal)
        x = torch.einsum("htd,hnd->htn", q[0].double(), kk) * 0.2
        if causal:
            x = x.masked_fill(torch.arange(n)[None, None] > n - 3 + torch.arange(3)[None, :, None], -math.inf)
        assert torch.allclose(o[0], torch.softmax(x, -1) @ vv, atol=1e-12)
        assert torch.allclose(M[0] + L[0].log2(), torch.logsumexp(x, -1) * math.log2(math.e), atol=1e-12)


@pytest.mark.parametrize("name,mirror", [("lvar_paged_cache", "PagedCache"), ("lvar_paged_write_args", "PagedWriteArgs"),
                                         ("lvar_paged_read_args", "PagedReadArgs"), ("lvar_paged_attn_args", "PagedAttnArgs")])
def test_struct_mirrors_follow_the_header(name, mirror):
    from lvar_b200 import _lib
    text = (ROOT / "include" / "lvar_b200.h").read_text()
    start = text.index(f"typedef struct {name} {{") + len(f"typedef struct {name} {{")
    body = re.sub(r"/\*.*?\*/", "", text[start:text.index(f"}} {name};")], flags=re.S)
    kinds = {"uint64_t": C.c_uint64, "int64_t": C.c_int64, "int32_t": C.c_int32, "float": C.c_float, "lvar_paged_cache": _lib.PagedCache}
    want = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        first, *rest = decl.split(",")
        kind = C.c_void_p if "*" in first else kinds[first.split()[0]]
        want += [(x.split()[-1].lstrip("*"), kind) for x in [first, *rest]]
    assert want == [tuple(f) for f in getattr(_lib, mirror)._fields_]


@pytest.mark.parametrize("mirror", ["PagedWriteArgs", "PagedReadArgs", "PagedAttnArgs"])
def test_packed_bytes_are_the_struct(mirror):
    from lvar_b200 import _lib
    kind = getattr(_lib, mirror)

    def leaves(s):
        for name, k in s._fields_:
            yield from leaves(k) if issubclass(k, C.Structure) else [k]
    kinds = list(leaves(kind))
    values = [0.5 * i if k is C.c_float else i + 1 for i, k in enumerate(kinds)]
    data = _lib.packer(kind)(*values)
    back = kind.from_buffer_copy(data)

    def read(s):
        for name, k in s._fields_:
            x = getattr(s, name)
            yield from read(x) if isinstance(x, C.Structure) else [x]
    assert list(read(back)) == values


def test_page_division_is_exact():
    """The kernels divide a group of 16 rows by the groups per page with one multiplication."""
    g = torch.Generator().manual_seed(2)
    for groups in range(2, 33):
        magic = ((1 << 32) + groups - 1) // groups
        at = torch.randint(0, 1 << 27, (4000,), generator=g).tolist() + [0, groups - 1, groups, (1 << 27) - 1]
        at += [x // groups * groups + d for x in at for d in (-1, 0) if x >= groups]
        assert all((n * magic) >> 32 == n // groups for n in at)


def _cache(**kw):
    """A description that passes every check; the pointers are never followed."""
    from lvar_b200 import _lib
    f = dict(k=1 << 20, k_sp=8 * 64 * 128, k_sh=64 * 128, k_sl=128, v=1 << 21, v_sp=8 * 64 * 128, v_sh=64 * 128, v_sl=128,
             table=1 << 22, t_sb=4, num_pages=16, page_size=64, Hkv=8, D=128, B=2, max_pages=4)
    f.update(kw)
    return _lib.PagedCache(**f)


BAD_CACHES = [("non-null", dict(k=None)), ("non-null", dict(table=None)), ("Head dimension", dict(D=96)),
              ("page_size", dict(page_size=24)), ("page_size", dict(page_size=8)), ("page_size", dict(page_size=1024)),
              ("strides", dict(k_sl=132)), ("strides", dict(v_sp=-64)), ("aligned", dict(v=(1 << 21) + 8)),
              ("sizes", dict(num_pages=0)), ("sizes", dict(max_pages=0)),
              ("strides", dict(scales=1 << 23, k_sl=136)),  # 8-bit rows: multiples of 16
              ("scales", dict(scales=(1 << 23) + 2)), ("scales", dict(scales=1 << 23, s_sh=130))]


def _calls(cache):
    """The three entry points with otherwise good arguments."""
    from lvar_b200 import _lib
    lib = _lib.lib
    p = 1 << 24
    w = _lib.PagedWriteArgs(cache=cache, k=p, k_sb=1024, k_sl=128, k_sh=128, v=p, v_sb=1024, v_sl=128, v_sh=128, start=p, L=1)
    r = _lib.PagedReadArgs(cache=cache, k=p, k_sb=1024, k_sh=128, k_sl=128, v=p, v_sb=1024, v_sh=128, v_sl=128, lens=p, n=1)
    a = _lib.PagedAttnArgs(cache=cache, q=p, q_sb=1024, q_sh=128, q_sl=128, o=p, o_sb=1024, o_sh=128, o_sl=128, lens=p,
                           scale=0.1, Hq=8, T=1, max_len=64)
    return [(lib.lvar_paged_write, w), (lib.lvar_paged_read, r), (lib.lvar_paged_attn, a)]


@pytest.mark.parametrize("word,bad", BAD_CACHES)
def test_bad_caches_are_refused(word, bad):
    from lvar_b200 import _lib
    for fn, args in _calls(_cache(**bad)):
        rc = fn(C.byref(args), None)
        assert rc in (-1, -2), rc
        assert word in _lib.lib.lvar_last_error().decode()


@pytest.mark.parametrize("i,word,bad", [
    (0, "non-null", dict(k=None)), (0, "non-null", dict(start=None)), (0, "go together", dict(q=1 << 24)),
    (0, "number of tokens", dict(L=0)), (0, "norm", dict(norm=3)), (0, "eps", dict(norm=2, eps=-1.0)),
    (0, "go together", dict(rope_cos=1 << 24)), (0, "no rows", dict(rope_cos=1 << 24, rope_sin=1 << 24, rope_rows=0)),
    (0, "strides", dict(k_sl=132)), (0, "aligned", dict(v=(1 << 24) + 4)), (0, "too many", dict(L=1 << 30)),
    (0, "scale_mul", dict(q=1 << 24, q_out=1 << 24, Hq=8, norm=1)),
    (1, "non-null", dict(lens=None)), (1, "row range", dict(n=0)), (1, "row range", dict(start=-1)),
    (1, "row range", dict(start=1 << 30)), (1, "strides", dict(k_sl=132)), (1, "aligned", dict(k=(1 << 24) + 8)),
    (2, "non-null", dict(lens=None)), (2, "go together", dict(M=1 << 24)), (2, "multiple", dict(Hq=12)), (2, "multiple", dict(T=0)),
    (2, "scale", dict(scale=0.0)), (2, "scale", dict(scale=math.nan)), (2, "scale", dict(scale=math.inf)),
    (2, "max_len", dict(max_len=-1)), (2, "max_len", dict(max_len=(1 << 30) + 1)), (2, "strides", dict(o_sl=4)),
    (2, "aligned", dict(q=(1 << 24) + 8)), (2, "too many", dict(Hq=8, T=1 << 28))])
def test_bad_arguments_are_refused(i, word, bad):
    from lvar_b200 import _lib
    fn, args = _calls(_cache())[i]
    for k, v in bad.items():
        setattr(args, k, v)
    rc = fn(C.byref(args), None)
    assert rc in (-1, -2, -4), rc
    assert word in _lib.lib.lvar_last_error().decode()


def test_null_arguments_are_refused():
    from lvar_b200 import _lib
    for fn, _ in _calls(_cache()):
        assert fn(None, None) == -1
    assert _lib.lib.lvar_paged_attn_workspace(0, 8, 8, 1, 128, 0, 64) == -1
    assert _lib.lib.lvar_paged_attn_workspace(1, 9, 8, 1, 128, 0, 64) == -1


def test_cpu_tensors_are_refused():
    from lvar_b200 import kernels as K
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    table, n = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16)
    for call in (lambda: K.paged_kv_append(x, x, k, k, table, n), lambda: K.paged_qkv_prologue(x, x, x, k, k, table, n),
                 lambda: K.paged_kv_read(k, k, table, n, 1), lambda: K.paged_attn_fwd(x, k, k, table, n)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
