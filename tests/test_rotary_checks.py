"""What the rotary operators refuse, and the frequencies they are given.  The
host's checks come before any launch, so tensors on the CPU show them."""

import math

import pytest
import torch

from tests.test_kv4_checks import BASE, cache_args, kv4, lib_cache  # noqa: F401


@pytest.mark.parametrize("freqs,pos,factor,message", [
    (torch.zeros(4, dtype=torch.float64), None, 1.0, "freqs must be"), (torch.zeros(2, 2), None, 1.0, "freqs must be"),
    (torch.zeros(8)[::2], None, 1.0, "freqs must be"), (torch.zeros(0), None, 1.0, "0 frequencies"),
    (torch.zeros(33), None, 1.0, "33 frequencies"), (torch.zeros(4, device="meta"), None, 1.0, "freqs are on"),
    (torch.zeros(4), torch.zeros(5), 1.0, "positions must be"), (torch.zeros(4), torch.zeros(4).int(), 1.0, "positions must be"),
    (torch.zeros(4), torch.zeros(5, device="meta").int(), 1.0, "positions is on"),
    (torch.zeros(4), None, math.inf, "finite"), (torch.zeros(4), None, math.nan, "finite")])
def test_turn_refusals(kv4, freqs, pos, factor, message):  # noqa: F811
    with pytest.raises(ValueError, match=message):
        kv4._turn(freqs, pos, 5, 64, False, factor, False, "x", torch.device("cpu"))


def test_a_sound_turn(kv4):  # noqa: F811
    freqs, pos = torch.zeros(32), torch.zeros(5).int()
    t = kv4._turn(freqs, pos, 5, 64, True, 0.5, False, "x", torch.device("cpu"))
    assert (t.freqs, t.positions, t.pairs, t.interleaved, t.back, t.factor) == (
        freqs.data_ptr(), pos.data_ptr(), 32, 1, 0, 0.5)


@pytest.fixture
def host(kv4, monkeypatch):  # noqa: F811
    monkeypatch.setattr(kv4._lib, "require_device", lambda *a: None)
    calls = []
    monkeypatch.setattr(kv4, "_launch", lambda name, *a: calls.append(name))
    return calls


@pytest.mark.parametrize("shape", [(4, 64), (4, 2, 60), (4, 2, 1032), (4, 2, 0)])
def test_rotary_refuses_shapes(vqx, host, shape):
    with pytest.raises(ValueError, match="x must be"):
        vqx.ops.rotary(torch.zeros(shape), torch.zeros(4).int(), torch.zeros(2))
    assert not host


def test_append_rotary_refusals(kv4, host):  # noqa: F811
    codes, scales, lengths, table = cache_args()
    q, k, f = torch.zeros(2, 4, 128), torch.zeros(2, 2, 128), torch.zeros(64)

    def call(q=q, k=k, v=k, f=f, **how):
        return kv4.kv4_append_rotary(q, k, v, codes, scales, lengths, f, None, table, **how)

    call()
    assert host == ["vqx_kv4_append_rotary"]
    for how, message in [(dict(q=q[:1]), "differ"), (dict(q=q.half()), "differ"), (dict(v=k.half()), "differ"),
                         (dict(q=q[..., :64]), "query must be"), (dict(k=k[:, :1]), "key must be"),
                         (dict(q=q[:, :0]), "0 query heads"), (dict(f=torch.zeros(65)), "65 frequencies"),
                         (dict(positions=torch.zeros(3).int()), "positions must be")]:
        with pytest.raises(ValueError, match=message):
            call(**how)
    assert len(host) == 1


def test_cpu_tensors_are_refused(vqx):
    with pytest.raises(NotImplementedError):
        torch.ops.quantized_ops.rotary(torch.zeros(2, 4, 128), torch.zeros(2).int(), torch.zeros(2))


def test_frequencies_have_no_gradient(vqx):
    with pytest.raises(ValueError, match="no gradient"):
        torch.ops.quantized_ops.rotary(torch.zeros(2, 4, 8, device="meta"), torch.zeros(2, device="meta").int(),
                                       torch.zeros(2, device="meta", requires_grad=True))


def test_fake_shapes(vqx):
    codes, scales, lengths, table = (t.to("meta") for t in cache_args())
    q, k = torch.zeros(2, 4, 128, device="meta"), torch.zeros(2, 2, 128, device="meta")
    o = torch.ops.quantized_ops
    assert o.rotary(q.half(), lengths, torch.zeros(3, device="meta")).dtype == torch.float16
    assert o.kv4_append_rotary(q, k, k, codes, scales, lengths, torch.zeros(3, device="meta"), None, table).shape == q.shape


# the library's own checks ---------------------------------------------------
def turn(L, **how):
    d = dict(freqs=BASE, positions=BASE, pairs=4, interleaved=0, back=0, factor=1.0)
    d.update(how)
    return L.VqxTurn(**d)


@pytest.mark.parametrize("how,t,message", [
    (dict(dtype=3), {}, "float32, bfloat16"), (dict(dim=12), {}, "multiple of 8"), (dict(dim=2048), {}, "multiple of 8"),
    (dict(n=-1), {}, "tokens"), (dict(n=1 << 30), {}, "tokens"), (dict(heads=1 << 21), {}, "heads"),
    ({}, dict(freqs=None), "null"), ({}, dict(positions=None), "null"), ({}, dict(pairs=0), "0 pairs"),
    ({}, dict(pairs=5), "5 pairs"), ({}, dict(factor=math.inf), "finite"), (dict(x=None), {}, "null"),
    (dict(out=None), {}, "null"), (dict(out=BASE + 8), {}, "aligned"), (dict(out=BASE), {}, "not x"),
    (dict(x=BASE + 8), {}, "16 bytes"), (dict(sn=4), {}, "16 bytes")])
def test_library_rotary_refusals(vqx, how, t, message):
    L = vqx._lib
    a = dict(x=BASE, dtype=1, n=2, heads=2, dim=8, sn=16, sh=8, out=2 * BASE)
    a.update(how)
    with pytest.raises(ValueError, match=message):
        L.call("vqx_rotary", a["x"], a["dtype"], a["n"], a["heads"], a["dim"], a["sn"], a["sh"], turn(L, **t), a["out"], 0)


@pytest.mark.parametrize("how,message", [
    (dict(heads=0), "0 query heads"), (dict(n=3), "without offsets"), (dict(q=None), "null"), (dict(out=None), "null"),
    (dict(out=BASE), "not the query"), (dict(k=BASE + 4), "16 bytes"), (dict(v=BASE + 4), "16 bytes"),
    (dict(dtype=3), "float32, bfloat16"), (dict(turn=dict(pairs=65)), "65 pairs")])
def test_library_append_rotary_refusals(vqx, how, message):
    L = vqx._lib
    a = dict(q=BASE, k=BASE, v=BASE, heads=4, dtype=1, n=2, out=2 * BASE, turn={})
    a.update(how)
    with pytest.raises(ValueError, match=message):
        L.call("vqx_kv4_append_rotary", lib_cache(L), turn(L, **a["turn"]), a["q"], a["heads"], 512, 128, a["k"], 256, 128,
               a["v"], 256, 128, a["dtype"], a["n"], None, a["out"], 0)


# the frequencies --------------------------------------------------------------
def test_frequencies(vqx):
    f = vqx.ops.rotary_frequencies(8, 10000.0)
    assert f.dtype == torch.float32 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001]), rtol=2.0 ** -23)
    assert torch.equal(vqx.ops.rotary_frequencies(8, stretch=4.0), f / 4)
    g = vqx.ops.rotary_frequencies(8, stretch=8.0, trained=1000)  # 159, 15.9, 1.59 and 0.159 turns
    assert torch.equal(g[:2], f[:2]) and torch.equal(g[3], f[3] / 8) and f[2] / 8 < g[2] < f[2]


@pytest.mark.parametrize("args,how", [((3,), {}), ((0,), {}), ((8, 0.0), {}), ((8,), dict(stretch=0.0)),
                                      ((8,), dict(trained=-1)), ((8,), dict(slow=4.0))])
def test_frequency_refusals(vqx, args, how):
    with pytest.raises(ValueError, match="rotary_frequencies"):
        vqx.ops.rotary_frequencies(*args, **how)
