"""What the 4-bit cache's operators refuse.  The host's checks come before any
launch, so tensors on the CPU and addresses that hold nothing show them."""

import pytest
import torch

BASE = 1 << 20


def cache_args(seqs=2, kv=2, dim=128, size=16, pages=5, per=2):
    return [torch.zeros(2, pages, kv, size, dim // 2, dtype=torch.uint8),
            torch.zeros(2, pages, kv, size, dim // 32, dtype=torch.uint8),
            torch.zeros(seqs, dtype=torch.int32), torch.zeros(seqs, per, dtype=torch.int32)]


@pytest.fixture
def kv4(vqx):
    from voyager_compiler_amd.ops import kv4 as module
    return module


def test_a_sound_cache(kv4):
    args = cache_args()
    c = kv4._cache(*args, "x")
    assert (c.pages, c.pages_per_seq, c.kv_heads, c.page_size, c.dim, c.seqs) == (5, 2, 2, 16, 128, 2)
    assert c.codes == args[0].data_ptr() and c.table == args[3].data_ptr()
    assert kv4._cache(*args[:3], None, "x").table is None


@pytest.mark.parametrize("i,change,message", [
    (0, lambda t: t.to(torch.int8), "uint8"), (1, lambda t: t.float(), "uint8"),
    (0, lambda t: t[0], "codes must be"), (0, lambda t: t[:1], "codes must be"),
    (0, lambda t: t[..., :48].contiguous(), "codes must be"), (0, lambda t: t[:, :4].contiguous(), "scales must be"),
    (1, lambda t: t[..., :2].contiguous(), "scales must be"), (1, lambda t: t[..., 0], "scales must be"),
    (0, lambda t: t.transpose(1, 2).contiguous().transpose(1, 2), "contiguous"),
    (1, lambda t: t.transpose(2, 3).contiguous().transpose(2, 3), "contiguous"),
    (1, lambda t: t.to("meta"), "scales are on"),
    (2, lambda t: t.long(), "lengths must be"), (2, lambda t: t[:, None], "lengths must be"),
    (2, lambda t: torch.zeros(4, dtype=torch.int32)[::2], "lengths must be"),
    (2, lambda t: t.to("meta"), "lengths is on"),
    (3, lambda t: t.long(), "table must be"), (3, lambda t: t[:1], "table must be"), (3, lambda t: t[0], "table must be"),
    (3, lambda t: t.t(), "table must be"), (3, lambda t: t[:, :0].contiguous(), "no pages")])
def test_cache_refusals(kv4, i, change, message):
    args = cache_args()
    args[i] = change(args[i])
    with pytest.raises(ValueError, match=message):
        kv4._cache(*args, "x")


def query(kv4, q, cu=None, most=None, scale=None, softcap=0.0, window=0, slopes=None):
    args = cache_args()
    return kv4._query(q, kv4._cache(*args, "x"), args[0].device, cu, most, scale, softcap, window, slopes, "x")[:2]


def test_a_sound_query(kv4):
    q = torch.zeros(6, 9, 128, dtype=torch.bfloat16)[:, 1:5]
    s, held = query(kv4, q)
    assert held is q and (s.n, s.heads, s.stride_n, s.stride_h, s.most) == (6, 4, 9 * 128, 128, 0)
    s, held = query(kv4, torch.zeros(6, 4, 130)[..., 1:129])
    assert held.is_contiguous() and s.q == held.data_ptr()


@pytest.mark.parametrize("q,how,message", [
    (torch.zeros(6, 128), {}, "query must be"), (torch.zeros(6, 4, 64), {}, "query must be"),
    (torch.zeros(6, 4, 128, dtype=torch.float64), {}, "float32, bfloat16 or float16"),
    (torch.zeros(6, 4, 128, device="meta"), {}, "query is on"),
    (torch.zeros(6, 3, 128), {}, "3 query heads"), (torch.zeros(6, 0, 128), {}, "0 query heads"),
    (torch.zeros(5, 4, 128), {}, "need cu"), (torch.zeros(6, 4, 128), dict(cu=torch.zeros(2, dtype=torch.int32)), "cu must be"),
    (torch.zeros(6, 4, 128), dict(cu=torch.zeros(3)), "cu must be"), (torch.zeros(6, 4, 128), dict(most=0), "most is 0"),
    (torch.zeros(6, 4, 128), dict(window=-1), "window"), (torch.zeros(6, 4, 128), dict(softcap=-1.0), "softcap"),
    (torch.zeros(6, 4, 128), dict(softcap=float("inf")), "softcap"), (torch.zeros(6, 4, 128), dict(softcap=float("nan")), "softcap"),
    (torch.zeros(6, 4, 128), dict(slopes=torch.zeros(2)), "slopes must be"),
    (torch.zeros(6, 4, 128), dict(slopes=torch.zeros(4, dtype=torch.float64)), "slopes must be"),
    (torch.zeros(6, 4, 128), dict(slopes=torch.zeros(4, device="meta")), "slopes are on")])
def test_query_refusals(kv4, q, how, message):
    with pytest.raises(ValueError, match=message):
        query(kv4, q, **how)


def test_weights_refusals(kv4):
    for w in (torch.zeros(2, 2, 9).double(), torch.zeros(2, 3, 9), torch.zeros(2, 2), torch.zeros(2, 9, 2).mT):
        with pytest.raises(ValueError, match="weights must be"):
            kv4._weights(w, 2, 2, "weights", "x", w.device)


def test_cpu_tensors_are_refused(kv4):
    args = cache_args()
    with pytest.raises(NotImplementedError):
        torch.ops.quantized_ops.kv4_attention(torch.zeros(2, 4, 128), *args[:3])


def test_fake_shapes(kv4):
    o = torch.ops.quantized_ops
    codes, scales, lengths, table = (t.to("meta") for t in cache_args())
    q = torch.zeros(6, 4, 128, dtype=torch.float16, device="meta")
    out, lse = o.kv4_attention(q, codes, scales, lengths, None, None, table)
    assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (6, 4) and lse.dtype == torch.float32
    k, v = o.kv4_read(codes, scales, lengths, 6, None, table, torch.float32)
    assert k.shape == v.shape == (6, 2, 128) and k.dtype == torch.float32
    w = torch.zeros(2, 2, 32, device="meta")
    index, kept = o.kv4_evict(codes, scales, w, lengths, 8, 2, codes, scales, w[..., :8], table, table)
    assert index.shape == (2, 2, 8) and index.dtype == kept.dtype == torch.int32 and kept.shape == (2,)
    assert o.kv4_append(k, v, codes, scales, lengths, None, table) is None


# the library's own checks -------------------------------------------------------
def lib_cache(L, **how):
    d = dict(codes=BASE, scales=BASE, table=BASE, lengths=BASE, pages=4, pages_per_seq=2, kv_heads=2, page_size=16,
             dim=128, seqs=2)
    d.update(how)
    return L.VqxKv4Cache(**d)


def lib_query(L, **how):
    d = dict(q=BASE, cu=None, slopes=None, n=2, stride_n=512, stride_h=128, dtype=1, heads=4, most=0, window=0,
             scale=1.0, softcap=0.0)
    d.update(how)
    return L.VqxKv4Query(**d)


def workspace(L, cache, q):
    n = L.ctypes.c_int64(-1)
    L.call("vqx_kv4_attention_workspace_size", cache, q, n)
    return n.value


@pytest.mark.parametrize("how,error,message", [
    (dict(codes=None), ValueError, "null"), (dict(scales=None), ValueError, "null"),
    (dict(lengths=None), ValueError, "null"), (dict(pages=0), ValueError, "no pages"), (dict(dim=96), ValueError, "64, 128 or 256"),
    (dict(codes=BASE + 8), ValueError, "aligned"), (dict(scales=BASE + 2), ValueError, "aligned"),
    (dict(kv_heads=0), ValueError, "sizes"), (dict(page_size=0), ValueError, "sizes"), (dict(seqs=-1), ValueError, "sizes"),
    (dict(table=None, pages=1), ValueError, "without a table"),
    (dict(pages=1 << 31), RuntimeError, "2\\^32 rows"), (dict(pages=1 << 30, page_size=32), RuntimeError, "2\\^32 rows"),
    (dict(pages_per_seq=1 << 26), RuntimeError, "2\\^30 tokens"), (dict(seqs=1 << 24), RuntimeError, "2\\^24 heads"),
    (dict(kv_heads=1 << 17), RuntimeError, "131072 kv heads")])
def test_library_cache_refusals(vqx, how, error, message):
    L = vqx._lib
    with pytest.raises(error, match=message):
        workspace(L, lib_cache(L, **how), lib_query(L, n=how.get("seqs", 2)))


@pytest.mark.parametrize("how,message", [
    (dict(dtype=3), "dtype 3"), (dict(n=3), "without offsets"), (dict(n=-2), "new tokens"), (dict(heads=3), "3 query heads"),
    (dict(heads=0), "0 query heads"), (dict(q=None), "null"), (dict(q=BASE + 4), "16 bytes"), (dict(stride_n=516), "16 bytes"),
    (dict(stride_h=4), "16 bytes"), (dict(softcap=-1.0), "softcap"), (dict(softcap=float("nan")), "softcap"),
    (dict(window=-1), "window"), (dict(window=1 << 30), "window"), (dict(n=1 << 30), "new tokens"), (dict(most=-1), "most")])
def test_library_query_refusals(vqx, how, message):
    L = vqx._lib
    with pytest.raises(ValueError, match=message):
        workspace(L, lib_cache(L), lib_query(L, **how))


def test_library_refuses_a_small_workspace(vqx):
    L = vqx._lib
    cache, q = lib_cache(L, pages=4096, pages_per_seq=2048), lib_query(L)
    need = workspace(L, cache, q)
    assert need > 0
    for ws, size in ((None, 0), (BASE, need - 1), (BASE + 4, need)):
        with pytest.raises(ValueError, match="workspace"):
            L.call("vqx_kv4_attention", cache, q, BASE, BASE, ws, size, None)
    for out, lse in ((None, BASE), (BASE, None)):
        with pytest.raises(ValueError, match="null"):
            L.call("vqx_kv4_attention", cache, q, out, lse, BASE, need, None)


def test_library_append_and_read_refusals(vqx):
    L = vqx._lib
    c = lib_cache(L)
    append = lambda key=BASE, value=BASE, dtype=1, n=2, sn=256, sh=128: L.call(  # noqa: E731
        "vqx_kv4_append", c, key, value, dtype, n, sn, sh, 256, 128, None, None)
    for how, message in ((dict(key=None), "null"), (dict(value=None), "null"), (dict(dtype=4), "dtype 4"),
                         (dict(n=3), "without offsets"), (dict(key=BASE + 2), "16 bytes"), (dict(sn=129), "16 bytes"),
                         (dict(sh=1), "16 bytes")):
        with pytest.raises(ValueError, match=message):
            append(**how)
    for args, message in (((None, BASE, 1, 2), "null"), ((BASE, BASE + 2, 1, 2), "aligned"), ((BASE, BASE, 3, 2), "dtype 3"),
                          ((BASE, BASE, 1, 1), "without offsets")):
        with pytest.raises(ValueError, match=message):
            L.call("vqx_kv4_read", c, *args, None, None)


def test_library_evict_refusals(vqx):
    L = vqx._lib
    far = BASE << 20

    def evict(budget=8, recent=2, weights=BASE, length=32, index=BASE, ow=far, codes=far, scales=far, **out):
        L.call("vqx_kv4_evict", lib_cache(L), weights, length, budget, recent,
               lib_cache(L, codes=codes, scales=scales, **out), index, ow, None, 0, None)

    for how, message in ((dict(budget=0), "budget of 0"), (dict(budget=33), "room for 32"), (dict(recent=-1), "-1 latest"),
                         (dict(recent=9), "9 latest"), (dict(weights=None), "null"), (dict(index=None), "null"),
                         (dict(ow=None), "null"), (dict(length=-1), "weights of -1"), (dict(kv_heads=4), "differ"),
                         (dict(dim=64), "differ"), (dict(seqs=1), "differ"), (dict(codes=BASE), "another cache"),
                         (dict(codes=BASE + 4096), "another cache"), (dict(scales=BASE + 64), "another cache"),
                         (dict(ow=BASE), "another tensor"), (dict(ow=BASE + 4 * 32 * 4 - 4), "another tensor")):
        with pytest.raises(ValueError, match=message):
            evict(**how)
    big, n = lib_cache(L, pages=1 << 20, pages_per_seq=1 << 16), L.ctypes.c_int64(-1)
    L.call("vqx_kv4_evict_workspace_size", big, 1 << 16, n)
    assert n.value > 0
    for ws, size in ((None, 0), (BASE, n.value - 1), (BASE + 4, n.value)):
        with pytest.raises(ValueError, match="workspace"):
            L.call("vqx_kv4_evict", big, BASE, 1 << 16, 8, 2, lib_cache(L, codes=1 << 40, scales=1 << 41), BASE, 1 << 42,
                   ws, size, None)
    L.call("vqx_kv4_evict_workspace_size", big, 8192, n)
    assert n.value == 0
    with pytest.raises(ValueError, match="weights of -1"):
        L.call("vqx_kv4_evict_workspace_size", big, -1, n)
