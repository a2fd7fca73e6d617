"""The paged-cache operators' refusals on the CPU: the C ABI with addresses that
are never dereferenced, and the Python surface. Nothing here launches a kernel."""
import copy
import ctypes

import pytest
import torch

from headshot_amd import _lib, context
from headshot_amd.paged import PagedKV

L = _lib.load()
F16, F32 = _lib.HS_F16, _lib.HS_F32
OK, EINVAL, EUNSUPPORTED = _lib.HS_OK, _lib.HS_EINVAL, _lib.HS_EUNSUPPORTED


def at(i):
    """The i-th of some buffers 256 MiB apart."""
    return ctypes.c_void_p(0x10000000 * (i + 1))


def refused(status, code, needle):
    assert status == code, _lib.status_name(status)
    assert needle in L.hs_last_error().decode(), L.hs_last_error().decode()


def append(dt=F16, q=at(0), qs=256, k=at(1), ks=128, v=at(2), vs=128, qw=None, qb=None, kw=None, kb=None,
           sn=None, cs=None, rows=0, pos=None, off=at(3), table=at(4), lens=at(5), qo=at(6), ko=at(7),
           kc=at(8), vc=at(9), n=10, b=2, h=4, h_kv=2, d=64, page=16, n_pages=8, max_pages=4, eps=1e-5):
    return L.hs_kv_append(None, dt, q, qs, k, ks, v, vs, qw, qb, kw, kb, sn, cs, rows, pos, off, table, lens,
                          qo, ko, kc, vc, n, b, h, h_kv, d, page, n_pages, max_pages, eps)


def test_append_refusals():
    refused(append(dt=7), EINVAL, "dtype")
    refused(append(h=3), EINVAL, "heads")
    refused(append(h_kv=0), EINVAL, "heads")
    refused(append(d=32), EUNSUPPORTED, "head_dim")
    refused(append(page=24), EUNSUPPORTED, "power of two")
    refused(append(page=0), EINVAL, "page")
    refused(append(n=-1), EINVAL, "negative")
    refused(append(off=None), EINVAL, "one token per sequence")
    refused(append(qw=at(10)), EINVAL, "weight and bias")
    refused(append(kb=at(10)), EINVAL, "weight and bias")
    refused(append(sn=at(10)), EINVAL, "sin and cos")
    refused(append(pos=at(10)), EINVAL, "positions")
    refused(append(kw=at(10), kb=at(11), eps=0.0), EINVAL, "eps")
    refused(append(k=None), EINVAL, "null k")
    refused(append(v=None), EINVAL, "null v")
    refused(append(qo=None), EINVAL, "null q_out")
    refused(append(kc=None), EINVAL, "null cache")
    refused(append(lens=None), EINVAL, "null cache")
    refused(append(ks=120), EINVAL, "overlap")
    refused(append(ks=132), EUNSUPPORTED, "16-byte")
    refused(append(k=ctypes.c_void_p(0x20000008)), EUNSUPPORTED, "16-byte")
    refused(append(kc=ctypes.c_void_p(0x90000008)), EUNSUPPORTED, "16-byte")
    refused(append(ko=at(1)), EINVAL, "overlaps an input")
    refused(append(kc=at(2)), EINVAL, "overlaps an input")
    refused(append(vc=at(8)), EINVAL, "outputs overlap")
    refused(append(qo=at(9)), EINVAL, "outputs overlap")
    refused(append(n=1 << 29), EINVAL, "2^30")
    refused(append(page=1 << 20, max_pages=1 << 10), EINVAL, "2^30")
    refused(append(n_pages=1 << 30), EINVAL, "too large")
    assert append(n=0, q=None, k=None, v=None, qo=None, ko=None, kc=None, vc=None, lens=None) == OK
    assert append(n=0, b=0, off=None) == OK


def packed(dt=F16, q=at(0), qs=256, k=at(1), ks=128, v=at(2), vs=128, off=at(3), koff=at(4), out=at(5), ws=at(6),
           nbytes=1 << 27, n=10, m=12, b=2, h=4, h_kv=2, d=64, causal=1, scale=0.125):
    return L.hs_attention_packed(None, dt, q, qs, k, ks, v, vs, off, koff, out, ws, nbytes, n, m, b, h, h_kv, d,
                                 causal, scale)


def test_packed_refusals():
    refused(packed(dt=2), EINVAL, "dtype")
    refused(packed(h=5), EINVAL, "heads")
    refused(packed(d=96), EUNSUPPORTED, "head_dim")
    refused(packed(causal=-1), EINVAL, "causal")
    refused(packed(m=-1), EINVAL, "negative")
    refused(packed(koff=None), EINVAL, "k_offsets")
    refused(packed(off=None), EINVAL, "null")
    refused(packed(out=None), EINVAL, "null")
    refused(packed(q=None), EINVAL, "null q")
    refused(packed(qs=248), EINVAL, "overlap")
    refused(packed(ks=1 << 22), EINVAL, "2^22")
    refused(packed(scale=float("inf")), EINVAL, "finite")
    refused(packed(scale=float("nan")), EINVAL, "finite")
    refused(packed(qs=260), EUNSUPPORTED, "16-byte")
    refused(packed(v=ctypes.c_void_p(0x30000004)), EUNSUPPORTED, "16-byte")
    refused(packed(out=ctypes.c_void_p(0x60000008)), EUNSUPPORTED, "16-byte")
    refused(packed(out=at(2)), EINVAL, "overlaps")
    refused(packed(n=1 << 29), EINVAL, "2^30")
    refused(packed(ws=ctypes.c_void_p(0x70000008)), EUNSUPPORTED, "16-byte")
    if L.hs_attention_packed_workspace(F16, 10, 5000, 2, 4, 2, 64, 1) > 0:
        refused(packed(m=5000, nbytes=0), EINVAL, "workspace")
        refused(packed(m=5000, ws=None), EINVAL, "workspace")
        refused(packed(m=5000, ws=at(1)), EINVAL, "workspace overlaps")
        refused(packed(m=5000, ws=at(5)), EINVAL, "workspace overlaps")
    assert packed(n=0, koff=at(4)) == OK
    assert packed(b=0) == OK


def paged(dt=F16, q=at(0), qs=256, kc=at(1), vc=at(2), table=at(3), lens=at(4), out=at(5), ws=at(6),
          nbytes=1 << 27, b=2, h=4, h_kv=2, d=64, page=16, n_pages=8, max_pages=4, scale=0.125):
    return L.hs_attention_paged(None, dt, q, qs, kc, vc, table, lens, out, ws, nbytes, b, h, h_kv, d, page,
                                n_pages, max_pages, scale)


def test_paged_refusals():
    refused(paged(dt=2), EINVAL, "dtype")
    refused(paged(h=5), EINVAL, "heads")
    refused(paged(d=256), EUNSUPPORTED, "head_dim")
    refused(paged(b=-1), EINVAL, "negative")
    refused(paged(page=48), EUNSUPPORTED, "power of two")
    refused(paged(q=None), EINVAL, "null q")
    refused(paged(out=None), EINVAL, "null")
    refused(paged(lens=None), EINVAL, "null")
    refused(paged(table=None), EINVAL, "null")
    refused(paged(qs=200), EINVAL, "overlap")
    refused(paged(scale=float("nan")), EINVAL, "finite")
    refused(paged(qs=260), EUNSUPPORTED, "16-byte")
    refused(paged(out=at(0)), EINVAL, "overlaps")
    refused(paged(b=1 << 21, qs=256), EINVAL, "2^23")
    if L.hs_attention_paged_workspace(2, 4, 2, 64) > 0:
        refused(paged(nbytes=0), EINVAL, "workspace")
        refused(paged(ws=None), EINVAL, "workspace")
        refused(paged(ws=at(1)), EINVAL, "overlaps")
        refused(paged(ws=ctypes.c_void_p(0x70000008)), EUNSUPPORTED, "16-byte")
    assert paged(b=0) == OK


def test_workspace_of_refused_shapes():
    f = L.hs_attention_paged_workspace
    assert f(0, 4, 2, 64) == 0 and f(2, 5, 2, 64) == 0 and f(2, 4, 0, 64) == 0 and f(2, 4, 2, 80) == 0
    assert f(2, 8192, 2, 64) == 0
    g = L.hs_attention_packed_workspace
    assert g(F16, 0, 5000, 2, 4, 2, 64, 1) == 0 and g(F16, 10, -1, 2, 4, 2, 64, 1) == 0
    assert g(F16, 10, 5000, 0, 4, 2, 64, 1) == 0 and g(F16, 10, 5000, 2, 5, 2, 64, 1) == 0
    assert g(F16, 10, 5000, 2, 4, 2, 80, 1) == 0 and g(7, 10, 5000, 2, 4, 2, 64, 1) == 0
    assert g(F32, 10, 5000, 2, 4, 2, 64, -1) == 0 and g(F32, 1 << 29, 5000, 2, 4, 2, 64, 1) == 0
    refused(paged(h=8192, qs=8192 * 64), EINVAL, "4096")


# ------------------------------------------------------------ the Python surface


@pytest.fixture
def surface(monkeypatch):
    """A HipContext whose launches are recorded: CPU tensors stand in."""
    calls = []
    monkeypatch.setattr(context, "_device", lambda: -1)  # what get_device() says of a CPU tensor
    ctx = context.HipContext.__new__(context.HipContext)
    ctx.lib, ctx.device, ctx.last_launch = L, torch.device("cpu"), None
    ctx._launch_held = lambda name, fn, held, *args: calls.append((name, args))
    return ctx, calls


def cache(pages=4, h=2, page=16, d=64, dtype=torch.float16, b=2, max_pages=3):
    return PagedKV.empty(pages, h, page, d, dtype, torch.zeros((b, max_pages), dtype=torch.int32),
                         torch.zeros(b, dtype=torch.int32))


def test_python_append(surface):
    ctx, calls = surface
    f16 = torch.float16
    wide = torch.zeros((5, (4 + 2 + 2) * 64), dtype=f16)
    q, k, v = wide.split([256, 128, 128], 1)
    off = torch.tensor([0, 3, 5], dtype=torch.int32)
    qo, ko = ctx.kv_append(cache(), k, v, off, q=q, k_rows=True)
    assert qo.shape == (5, 256) and ko.shape == (5, 128) and calls[-1][0] == "kv_append"
    assert calls[-1][1][2] == 512 and calls[-1][1][4] == 512  # rows of the wide product
    assert ctx.kv_append(cache(), k, v, off) == (None, None)
    # head-major columns of one token
    ctx.kv_append(cache(), k[:2].unflatten(1, (2, 64)), v[:2].unflatten(1, (2, 64)))
    bad = [
        lambda: ctx.kv_append(cache(), k.float(), v.float(), off),
        lambda: ctx.kv_append(cache(), k, v[:4], off),
        lambda: ctx.kv_append(cache(), k, v, off.long()),
        lambda: ctx.kv_append(cache(), k, v, off[:2]),
        lambda: ctx.kv_append(cache(), k, v),                          # 5 tokens, 2 sequences
        lambda: ctx.kv_append(cache(), k[:, :64], v, off),
        lambda: ctx.kv_append(cache(), k[:, ::2], v, off),
        lambda: ctx.kv_append(cache(), k[:1].expand(5, 128), v, off),  # rows on each other
        lambda: ctx.kv_append(cache(), k, v, off, q=q[:4]),
        lambda: ctx.kv_append(cache(), k, v, off, qn=(torch.ones(64), torch.ones(64))),
        lambda: ctx.kv_append(cache(), k, v, off, kn=(torch.ones(32), torch.ones(32))),
        lambda: ctx.kv_append(cache(), k, v, off, rope=(torch.ones(9, 64), torch.ones(8, 64))),
        lambda: ctx.kv_append(cache(), k, v, off, positions=torch.zeros(5, dtype=torch.int32)),
        lambda: ctx.kv_append(cache(), k, v, off, q=q, out_q=torch.zeros(5, 255, dtype=f16)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(AssertionError):
            f()
            pytest.fail(f"call {i} was taken")


def test_python_attention(surface):
    ctx, calls = surface
    f16 = torch.float16
    off = torch.tensor([0, 3, 5], dtype=torch.int32)
    q, k = torch.zeros((5, 4, 64), dtype=f16), torch.zeros((5, 2, 64), dtype=f16)
    assert ctx.attention_packed(q, k, k, off).shape == (5, 256)
    assert ctx.attention_paged(q[:2], cache()).shape == (2, 256)
    assert ctx.attention_paged(q[:2].flatten(1), cache()).shape == (2, 256)
    for i, f in enumerate([
        lambda: ctx.attention_packed(q.flatten(1), k, k, off),
        lambda: ctx.attention_packed(q, k.float(), k, off),
        lambda: ctx.attention_packed(q, k[:4], k[:4], off),
        lambda: ctx.attention_packed(q, k, k[:4], off, off),
        lambda: ctx.attention_packed(q.transpose(1, 2).contiguous().transpose(1, 2), k, k, off),
        lambda: ctx.attention_packed(q, k, k, off.long()),
        lambda: ctx.attention_packed(q, k, k, off, off[:2]),
        lambda: ctx.attention_packed(q, k, k, off, out=torch.zeros(5, 256)),
        lambda: ctx.attention_packed(q, k, k, off, workspace=torch.zeros(64)),
        lambda: ctx.attention_packed(q, k, k, off, causal=-1),
        lambda: ctx.attention_packed(q, k, k, off, causal=2 ** 32 + 1),  # 1 in 32 bits
        lambda: ctx.attention_paged(q, cache()),
        lambda: ctx.attention_paged(q[:2].float(), cache()),
        lambda: ctx.attention_paged(q[:2], cache(), workspace=torch.zeros(4)),
        lambda: ctx.attention_paged(q[:2], cache(), out=torch.zeros(2, 128, dtype=f16)),
    ]):
        with pytest.raises(AssertionError):
            f()
            pytest.fail(f"call {i} was taken")


def test_python_cache():
    """A cache is checked when it is made and when a tensor of it is replaced."""
    c = cache()
    assert (c.heads, c.page, c.head_dim) == (2, 16, 64) and c.shape == (4, 2, 16, 64, 2, 3)
    c.lens += 1  # in place
    assert c.lens.tolist() == [1, 1]
    c.lens = torch.tensor([5, 6], dtype=torch.int32)
    c.page_table = torch.zeros((2, 9), dtype=torch.int32)
    assert c.shape[5] == 9
    kept = c.lens
    for name, t in [("lens", torch.zeros(3, dtype=torch.int32)), ("lens", torch.zeros(2, dtype=torch.int64)),
                    ("page_table", torch.zeros(6, dtype=torch.int32)), ("k", c.k[:3]), ("v", c.v.float()),
                    ("k", c.k.transpose(1, 2).contiguous().transpose(1, 2)), ("v", c.v[0])]:
        with pytest.raises(AssertionError):
            setattr(c, name, t)
    assert c.lens is kept and c.k.shape == c.v.shape
    with pytest.raises(AssertionError):
        PagedKV(c.k.double(), c.v.double(), c.page_table, c.lens)


def test_python_cache_copies():
    """A shallow copy shares the pages, a deep one has its own."""
    c = cache()
    near, far = copy.copy(c), copy.deepcopy(c)
    assert near.shape == far.shape == c.shape and near.k is c.k and near.lens is c.lens
    far.lens += 1
    assert far.k is not c.k and c.lens.tolist() == [0, 0]


def test_tensors_of_another_device():
    """The launch goes to the current device's stream: a tensor elsewhere is
    refused before it."""
    with pytest.raises(AssertionError, match="current device"):
        context._here(torch.zeros(3), 0, "k")

    class Elsewhere:
        def get_device(self):
            return 1

        def data_ptr(self):
            return 16

    assert context._here(Elsewhere(), 1, "k") == 16
    with pytest.raises(AssertionError, match="current device"):
        context._here(Elsewhere(), 0, "k")


def test_cache_of_another_device(surface, monkeypatch):
    ctx, _ = surface
    c, rows = cache(), torch.zeros((2, 128), dtype=torch.float16)
    monkeypatch.setattr(context, "_device", lambda: 1)
    for f in (lambda: ctx.kv_append(c, rows, rows), lambda: ctx.attention_paged(rows, c)):
        with pytest.raises(AssertionError, match="current device"):
            f()
