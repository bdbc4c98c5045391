"""What the host side of the 4-bit cache's operators hands to the library, with
the library replaced by a stand-in: no GPU needed."""

import weakref

import pytest
import torch

from tests.test_kv4_checks import cache_args, kv4  # noqa: F401


class Codes(torch.Tensor):
    """Notes the memory that is allocated like it."""
    made = []

    def new_empty(self, *args, **kwargs):
        t = torch.empty(*args, dtype=torch.uint8)
        Codes.made.append((t.data_ptr(), weakref.ref(t)))
        return t


@pytest.fixture
def library(kv4, monkeypatch):  # noqa: F811
    """Records of (entry point, whether its workspace is still held)."""
    calls = []
    Codes.made.clear()

    def call(name, *args):
        if name.endswith("workspace_size"):
            args[-1].value = 4096
        else:
            held = {at: ref() is not None for at, ref in Codes.made}
            calls.append((name, args[-2], held.get(args[-3])))

    monkeypatch.setattr(kv4._lib, "call", call)
    monkeypatch.setattr(kv4._lib, "require_device", lambda *a: None)
    monkeypatch.setattr(kv4._lib, "stream_of", lambda t: 0)
    monkeypatch.setattr(kv4, "_workspace_bytes", lambda *a: 4096)
    return calls


def test_attention_holds_its_workspace(kv4, library):  # noqa: F811
    codes, scales, lengths, table = cache_args()
    kv4.kv4_attention(torch.zeros(2, 4, 128), codes.as_subclass(Codes), scales, lengths, table=table)
    assert library == [("vqx_kv4_attention", 4096, True)]


def test_evict_holds_its_workspace(kv4, library):  # noqa: F811
    codes, scales, lengths, table = cache_args()
    out = cache_args()
    kv4.kv4_evict(codes.as_subclass(Codes), scales, torch.zeros(2, 2, 32), lengths, 8, 2, out[0], out[1],
                  torch.zeros(2, 2, 8), table, out[3])
    assert library == [("vqx_kv4_evict", 4096, True)]


def test_library_evict_refuses_lengths_over_its_input(vqx):
    """The first head of a sequence writes its new length, the others read the
    old one: the same place for both would give each head another selection."""
    L = vqx._lib
    base, seqs = 1 << 20, 2

    def cache(at, lengths):
        return L.VqxKv4Cache(codes=at, scales=at, table=base, lengths=lengths, pages=4, pages_per_seq=2, kv_heads=2,
                             page_size=16, dim=128, seqs=seqs)

    for new in (base, base + 4 * seqs - 4, base - 4 * seqs + 4):
        with pytest.raises(ValueError, match="new lengths go to another tensor"):
            L.call("vqx_kv4_evict", cache(base, base), base, 32, 8, 2, cache(base << 20, new), base, base << 21, None, 0, None)


INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("how,message", [
    (dict(scale=NAN), "scale is finite"), (dict(scale=INF), "scale is finite"), (dict(scale=-INF), "scale is finite"),
    (dict(scale=1e39), "scale is finite"), (dict(softcap=1e-46), "too small"), (dict(softcap=1e-39), "too small"),
    (dict(scale=1e8, softcap=1e-35), "too small"), (dict(scale=-1e8, softcap=1e-35), "too small")])
def test_scale_refusals(kv4, how, message):  # noqa: F811
    args = cache_args()
    d = dict(scale=None, softcap=0.0)
    d.update(how)
    with pytest.raises(ValueError, match=message):
        kv4._query(torch.zeros(6, 4, 128), kv4._cache(*args, "x"), args[0].device, None, None, d["scale"], d["softcap"],
                   0, None, "x")


@pytest.mark.parametrize("scale,softcap,message", [
    (NAN, 0.0, "not finite"), (INF, 0.0, "not finite"), (-INF, 30.0, "not finite"), (1.0, 1e-39, "too small"),
    (-1e8, 1e-35, "too small")])
def test_library_scale_refusals(vqx, scale, softcap, message):
    L = vqx._lib
    base, n = 1 << 20, L.ctypes.c_int64(-1)
    cache = L.VqxKv4Cache(codes=base, scales=base, table=base, lengths=base, pages=4, pages_per_seq=2, kv_heads=2,
                          page_size=16, dim=128, seqs=2)
    q = L.VqxKv4Query(q=base, cu=None, slopes=None, n=2, stride_n=512, stride_h=128, dtype=1, heads=4, most=0, window=0,
                      scale=scale, softcap=softcap)
    with pytest.raises(ValueError, match=message):
        L.call("vqx_kv4_attention_workspace_size", cache, q, n)
    for scale, softcap in ((0.0, 30.0), (-3e38, 0.0), (-3e38, 3e38), (1e-30, 1e-37)):
        q.scale, q.softcap = scale, softcap
        L.call("vqx_kv4_attention_workspace_size", cache, q, n)
