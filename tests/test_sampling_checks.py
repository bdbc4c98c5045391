"""What sample_tokens refuses."""

import pytest
import torch

from tests.test_kv4_checks import BASE, kv4  # noqa: F401
from tests.test_rotary_checks import host  # noqa: F401


@pytest.mark.parametrize("how,message", [
    (dict(logits=torch.zeros(4)), "logits must be"), (dict(logits=torch.zeros(4, 0)), "logits must be"),
    (dict(logits=torch.zeros(1, 2 ** 22 + 1, dtype=torch.float16)), "logits must be"),
    (dict(logits=torch.zeros(4, 9, dtype=torch.float64)), "float32, bfloat16"), (dict(random=None), "one number"),
    (dict(random=torch.zeros(3)), "random must be"), (dict(random=torch.zeros(4).double()), "random must be"),
    (dict(random=torch.zeros(4, device="meta")), "random is on"), (dict(temperature=torch.zeros(4, 1)), "temperature must be"),
    (dict(top_k=torch.zeros(4)), "top_k must be"), (dict(top_k=torch.zeros(4).long()), "top_k must be"),
    (dict(top_p=torch.zeros(8)[::2]), "top_p must be"), (dict(min_p=torch.zeros(4).half()), "min_p must be")])
def test_refusals(vqx, host, monkeypatch, how, message):  # noqa: F811
    from voyager_compiler_amd.ops import sampling

    monkeypatch.setattr(sampling, "_workspace_bytes", lambda *a: 0)
    args = dict(logits=torch.zeros(4, 9), random=torch.zeros(4))
    vqx.ops.sample_tokens(**args)
    with pytest.raises(ValueError, match=message):
        vqx.ops.sample_tokens(**dict(args, **how))
    assert host == ["vqx_sample_tokens"]


def test_cpu_tensors_are_refused(vqx):
    with pytest.raises(NotImplementedError):
        torch.ops.quantized_ops.sample_tokens(torch.zeros(4, 9), torch.zeros(4))


def test_fake_shapes(vqx):
    tokens, chances = torch.ops.quantized_ops.sample_tokens(torch.zeros(4, 9, device="meta").half(), torch.zeros(4, device="meta"))
    assert tokens.shape == chances.shape == (4,) and tokens.dtype == torch.int64 and chances.dtype == torch.float32


@pytest.mark.parametrize("how,message", [
    (dict(dtype=3), "float32, bfloat16"), (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(vocab=0), "2\\^22"),
    (dict(vocab=(1 << 22) + 1), "2\\^22"), (dict(logits=None), "null"), (dict(random=None), "null"), (dict(tokens=None), "null"),
    (dict(chances=None), "null"), (dict(logits=BASE + 1), "aligned"),
    (dict(vocab=100000, bytes=1 << 20), "workspace"), (dict(vocab=100000, workspace=BASE), "workspace"),
    (dict(vocab=100000, workspace=BASE + 8, bytes=1 << 20), "workspace")])
def test_library_refusals(vqx, how, message):
    a = dict(logits=BASE, dtype=1, rows=2, vocab=9, stride=9, random=BASE, temperature=None, top_k=None, top_p=None, min_p=None,
             tokens=BASE, chances=BASE, workspace=None, bytes=0)
    a.update(how)
    with pytest.raises(ValueError, match=message):
        vqx._lib.call("vqx_sample_tokens", *a.values(), 0)


def test_library_workspace(vqx):
    """Few long rows without top_k have launches of their own before."""
    L = vqx._lib

    def need(rows, vocab, by_count, dtype=1):
        n = L.ctypes.c_int64(-1)
        L.call("vqx_sample_tokens_workspace_size", dtype, rows, vocab, by_count, n)
        return n.value

    assert need(1, 100000, 0) > 0 and need(8, 100000, 0) == 8 * need(1, 100000, 0)
    assert need(1, 100000, 1) == need(1, 5000, 0) == need(1000, 100000, 0) == need(0, 100000, 0) == 0
    with pytest.raises(ValueError, match="2\\^22"):
        need(1, 0, 0)
