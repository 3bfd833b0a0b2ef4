"""What the calls for chunks of new tokens refuse, and with which words; no GPU is asked (the checks come before any launch)."""
import pytest
import torch

from omchat_b200 import lib

P = 1 << 20   # an aligned address that nobody follows


@pytest.fixture(scope="module")
def L():
    from omchat_b200 import build
    build.build()
    return lib.load()


def _said(L):
    return L.omc_last_error().decode()


def _rotary(L, **kw):
    a = dict(x=P, fp32=0, ldx=256, pos=P, T=4, heads=2, head=128, turns=P, rot=128, y=P, ldy=256)
    a.update(kw)
    return L.omc_rotary_rows(a["x"], a["fp32"], a["ldx"], a["pos"], a["T"], a["heads"], a["head"], a["turns"], a["rot"], 1, 0, 1.0, a["y"], a["ldy"], None)


@pytest.mark.parametrize("kw,rc,word", [(dict(rot=3), -2, "even"), (dict(rot=130), -2, "even"), (dict(rot=-2), -2, "even"), (dict(head=0), -2, "heads"), (dict(head=258), -2, "heads"),
                                        (dict(heads=0), -2, "no heads"), (dict(T=-1), -2, "negative"), (dict(turns=None), -1, "frequencies"), (dict(x=None), -1, "null"),
                                        (dict(pos=None), -1, "null"), (dict(ldx=255), -2, "overlap"), (dict(ldy=128), -2, "overlap")])
def test_rotary(L, kw, rc, word):
    assert _rotary(L, **kw) == rc and word in _said(L)
    assert _rotary(L, T=0) == 0


def _append(L, **kw):
    a = dict(qkv=P, ld=8 * 128, pos=P, T=4, hq=4, hkv=2, head=128, turns=P, rot=128, q=P, ldq=512, pool=P, pages=9, table=P, seqs=1, max_pages=3, page=64)
    a.update(kw)
    return L.omc_rotary_kv_append(a["qkv"], a["ld"], a["pos"], None, a["T"], a["hq"], a["hkv"], a["head"], a["turns"], a["rot"], 1, 1.0, a["q"], a["ldq"], a["pool"], a["pages"],
                                  a["table"], a["seqs"], a["max_pages"], a["page"], None)


@pytest.mark.parametrize("kw,rc,word", [(dict(hq=0), -2, "no heads"), (dict(hkv=0), -2, "no heads"), (dict(page=0), -1, "paging"), (dict(pages=0), -1, "paging"),
                                        (dict(max_pages=0), -1, "paging"), (dict(seqs=0), -1, "paging"), (dict(pool=None), -1, "null"), (dict(table=None), -1, "null"),
                                        (dict(ld=1000), -2, "overlap"), (dict(ldq=511), -2, "overlap"), (dict(rot=129), -2, "even")])
def test_append(L, kw, rc, word):
    assert _append(L, **kw) == rc and word in _said(L)
    assert _append(L, T=0) == 0


def _attend(L, **kw):
    a = dict(q=P, ldq=512, pool=P, pages=9, table=P, max_pages=3, page=64, cu=P, ctx=P, n_seq=2, T=4, max_new=3, max_ctx=100, hq=4, hkv=2, head=128, scale=0.1, out=P, ldo=512, ws=None, wsb=0)
    a.update(kw)
    return L.omc_paged_chunk_attn(a["q"], a["ldq"], a["pool"], a["pages"], a["table"], a["max_pages"], a["page"], a["cu"], a["ctx"], a["n_seq"], a["T"], a["max_new"], a["max_ctx"],
                                  a["hq"], a["hkv"], a["head"], a["scale"], a["out"], a["ldo"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("kw,rc,word", [(dict(head=96), -2, "64 or 128"), (dict(hq=3), -2, "multiple"), (dict(hkv=0), -2, "multiple"), (dict(page=0), -1, "paging"),
                                        (dict(pages=1 << 24), -2, "2^31"), (dict(n_seq=-1), -2, "negative"), (dict(max_new=-1), -2, "negative"), (dict(scale=0.0), -1, "scale"),
                                        (dict(scale=-0.1), -1, "scale"), (dict(scale=float("nan")), -1, "scale"), (dict(scale=float("inf")), -1, "scale"), (dict(q=P + 2), -3, "16-byte"),
                                        (dict(out=P + 8), -3, "16-byte"), (dict(ldq=516), -3, "multiples of 8"), (dict(ldq=504), -2, "overlap"), (dict(cu=None), -1, "null"),
                                        (dict(table=None), -1, "null"), (dict(T=1 << 20, max_new=1 << 20, max_ctx=1 << 30), -2, "2^31 products"),
                                        (dict(T=1 << 20, max_new=1 << 30), -2, "2^31 rows"), (dict(max_ctx=(1 << 30) + 1), -2, "2^30"),
                                        (dict(max_ctx=100000), -1, "workspace"), (dict(max_ctx=100000, ws=P, wsb=1000), -1, "workspace"),
                                        (dict(max_ctx=100000, ws=P + 8, wsb=1 << 40), -1, "workspace")])
def test_attention(L, kw, rc, word):
    assert _attend(L, **kw) == rc and word in _said(L)
    assert _attend(L, T=0) == 0 and _attend(L, n_seq=0) == 0 and _attend(L, max_new=0) == 0


def test_workspace_bytes(L):
    size = lambda *a: L.omc_paged_chunk_attn_workspace_bytes(*a)  # noqa: E731
    assert size(1, 1, 300, 28, 4, 128) == 0 < size(1, 1, 40960, 28, 4, 128)   # nothing is cut: nothing is joined
    assert size(1, 1, 40960, 28, 4, 128) < 1 << 24 and size(1, 1, 4096, 28, 4, 96) < 0 and "64 or 128" in _said(L)
    assert L.omc_wait_failed() == 0
    lib.check_waits()


def test_host_tensors_are_refused():
    x, i, d = torch.zeros(2, 256, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32), torch.zeros(64, dtype=torch.float64)
    pool, table = torch.zeros(3, 2, 1, 16, 128, dtype=torch.bfloat16), torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(lib.OmcError):
        lib.rotary(x, i, d, 2, 128)
    with pytest.raises(lib.OmcError):
        lib.rotary_kv_append(torch.zeros(2, 512, dtype=torch.bfloat16), i, None, d, 2, pool, table)
    with pytest.raises(lib.OmcError):
        lib.paged_attention(x, pool, table, i, i[:1], 1, 1, 2, 0.1)
