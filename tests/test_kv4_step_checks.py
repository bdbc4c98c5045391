"""What the operators around a step of the 4-bit cache refuse.  The host's checks
come before any launch, so tensors on the CPU and addresses that hold nothing
show them."""

import pytest
import torch

from tests.test_kv4_checks import BASE, cache_args, kv4, lib_cache  # noqa: F401
from tests.test_kv4_checks import lib_query
from tests.test_kv4_host import Codes, library  # noqa: F401
from tests.test_rotary_checks import host  # noqa: F401


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def reserve_args():
    return dict(grow=i32(3), lengths=i32(3), table=i32(3, 4), free=i32(9), count=i32(1), page_size=16, n=5)


@pytest.mark.parametrize("how,message", [
    (dict(grow=i32(2)), "grow must be"), (dict(grow=torch.zeros(3)), "grow must be"), (dict(lengths=i32(3, 1)), "lengths must be"),
    (dict(lengths=torch.zeros(3)), "lengths must be"), (dict(table=i32(2, 4)), "table must be"), (dict(table=i32(3)), "table must be"),
    (dict(table=i32(4, 3).t()), "table must be"), (dict(table=i32(3, 4).long()), "table must be"),
    (dict(table=i32(3, 4).to("meta")), "table is on"), (dict(free=i32(9, 1)), "free must be"),
    (dict(free=torch.zeros(9)), "free must be"), (dict(free=i32(18)[::2]), "free must be"), (dict(count=i32(2)), "count must be"),
    (dict(count=i32(1).to("meta")), "count is on"), (dict(n=-1), "-1 new tokens")])
def test_reserve_refusals(kv4, host, how, message):  # noqa: F811
    kv4.kv4_reserve(**reserve_args())
    with pytest.raises(ValueError, match=message):
        kv4.kv4_reserve(**dict(reserve_args(), **how))
    assert host == ["vqx_kv4_reserve"]


def accept_args():
    codes, scales, lengths, table = cache_args()
    i64 = torch.zeros(6, dtype=torch.int64)
    return dict(tree=i64, drafts=i64, sampled=i64, codes=codes, scales=scales, lengths=lengths, table=table)


@pytest.mark.parametrize("how,message", [
    (dict(tree=i32(6)), "tree must be"), (dict(tree=torch.zeros(2, 3).long()), "tree must be"), (dict(drafts=i32(6)), "drafts must be"),
    (dict(drafts=torch.zeros(5).long()), "drafts must be"), (dict(sampled=torch.zeros(12).long()[::2]), "sampled must be"),
    (dict(sampled=torch.zeros(6, device="meta").long()), "sampled is on"), (dict(cu=i32(2)), "cu must be"),
    (dict(tree=torch.zeros(5).long()), "need cu")])
def test_accept_refusals(kv4, host, how, message):  # noqa: F811
    kv4.kv4_accept(**accept_args())
    with pytest.raises(ValueError, match=message):
        kv4.kv4_accept(**dict(accept_args(), **how))
    assert host == ["vqx_kv4_accept"]


@pytest.mark.parametrize("n,how,message", [
    (6, dict(tree=i32(6)), "tree must be"), (6, dict(tree=torch.zeros(5).long()), "tree must be"),
    (6, dict(tree=torch.zeros(12).long()[::2]), "tree must be"), (6, dict(tree=torch.zeros(6, device="meta").long()), "tree is on"),
    (130, {}, "up to 65"), (65, dict(cu=i32(3)), "up to 65"), (70, dict(cu=i32(3), most=66), "up to 66"), (6, dict(window=-1), "window")])
def test_tree_refusals(kv4, host, monkeypatch, n, how, message):  # noqa: F811
    monkeypatch.setattr(kv4, "_workspace_bytes", lambda *a: 0)
    codes, scales, lengths, table = cache_args()

    def call(n, **how):
        return kv4.kv4_tree_attention(torch.zeros(n, 4, 128), codes, scales, lengths, table=table,
                                      **dict(dict(tree=torch.zeros(n, dtype=torch.int64)), **how))

    call(128), call(70, cu=i32(3), most=64), call(0, cu=i32(3)), call(64, cu=i32(3))
    assert host == ["vqx_kv4_tree_attention"] * 4
    with pytest.raises(ValueError, match=message):
        call(n, **how)
    assert len(host) == 4


def test_tree_holds_its_workspace(kv4, library):  # noqa: F811
    codes, scales, lengths, table = cache_args()
    kv4.kv4_tree_attention(torch.zeros(2, 4, 128), codes.as_subclass(Codes), scales, lengths, torch.zeros(2).long(),
                           table=table)
    assert library == [("vqx_kv4_tree_attention", 4096, True)]


def test_fake_shapes(vqx):
    o = torch.ops.quantized_ops
    cu, positions, slots = o.kv4_reserve(*(t.to("meta") for t in list(reserve_args().values())[:5]), 16, 5)
    assert cu.shape == (4,) and positions.shape == slots.shape == (5,) and cu.dtype == positions.dtype == torch.int32
    assert slots.dtype == torch.int64
    a = {k: t.to("meta") for k, t in accept_args().items()}
    q = torch.zeros(6, 4, 128, dtype=torch.float16, device="meta")
    out, lse = o.kv4_tree_attention(q, a["codes"], a["scales"], a["lengths"], a["tree"], None, None, a["table"])
    assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (6, 4) and lse.dtype == torch.float32
    path, count, follows = o.kv4_accept(**a)
    assert path.shape == (6,) and path.dtype == count.dtype == torch.int32 and count.shape == follows.shape == (2,)
    assert follows.dtype == torch.int64


# the library's own checks -------------------------------------------------------
@pytest.mark.parametrize("how,error,message", [
    (dict(seqs=-1), ValueError, "sequences"), (dict(seqs=1 << 24), ValueError, "sequences"), (dict(per=0), ValueError, "pages of"),
    (dict(size=0), ValueError, "0 tokens"), (dict(pages=1 << 31), ValueError, "pages in all"),
    (dict(per=1 << 20, size=1 << 10), RuntimeError, "2\\^30 tokens"), (dict(n=-1), ValueError, "new tokens"),
    (dict(n=1 << 30), ValueError, "new tokens"), (dict(count=None), ValueError, "null"), (dict(free=None), ValueError, "null"),
    (dict(grow=None), ValueError, "null"), (dict(slots=None), ValueError, "null"), (dict(grow=BASE + 4096), ValueError, "one tensor")])
def test_library_reserve_refusals(vqx, how, error, message):
    a = dict(grow=BASE, lengths=BASE + 4096, table=BASE, free=BASE, count=BASE, seqs=2, per=3, pages=9, size=16, n=4, cu=BASE,
             positions=BASE, slots=BASE)
    a.update(how)
    with pytest.raises(error, match=message):
        vqx._lib.call("vqx_kv4_reserve", *a.values(), 0)


@pytest.mark.parametrize("how,message", [
    (dict(tree=None), "null"), (dict(drafts=None), "null"), (dict(sampled=None), "null"), (dict(path=None), "null"),
    (dict(accepted=None), "null"), (dict(next=None), "null"), (dict(n=3), "without offsets"), (dict(n=-2), "new tokens")])
def test_library_accept_refusals(vqx, how, message):
    a = dict(tree=BASE, drafts=BASE, sampled=BASE, n=4, cu=None, path=BASE, accepted=BASE, next=BASE)
    a.update(how)
    with pytest.raises(ValueError, match=message):
        vqx._lib.call("vqx_kv4_accept", lib_cache(vqx._lib), *a.values(), 0)


@pytest.mark.parametrize("q,how,message", [
    (dict(n=130), {}, "65 new tokens"), (dict(n=70, cu=BASE), {}, "70 new tokens"), (dict(n=70, cu=BASE, most=65), {}, "65 new tokens"),
    ({}, dict(tree=None), "null"), ({}, dict(out=None), "null"), ({}, dict(lse=None), "null"), ({}, dict(out=BASE + 8), "aligned"),
    (dict(heads=3), {}, "3 query heads")])
def test_library_tree_refusals(vqx, q, how, message):
    L = vqx._lib
    a = dict(tree=BASE, out=BASE, lse=BASE, workspace=None, bytes=0)
    a.update(how)
    with pytest.raises(ValueError, match=message):
        L.call("vqx_kv4_tree_attention", lib_cache(L), lib_query(L, **q), *a.values(), 0)


def test_library_tree_workspace(vqx):
    """A long room needs one, and a call without it is refused."""
    L = vqx._lib
    cache, query, n = lib_cache(L, pages=4096, pages_per_seq=2048), lib_query(L, n=16), L.ctypes.c_int64(-1)
    L.call("vqx_kv4_tree_attention_workspace_size", cache, query, n)
    assert n.value > 0
    with pytest.raises(ValueError, match="workspace"):
        L.call("vqx_kv4_tree_attention", cache, query, BASE, BASE, BASE, BASE, n.value - 1, 0)
