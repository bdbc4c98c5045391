"""How the 4-bit cache's attention cuts a call up: the plan that sizes the workspace
against the ranges that the kernels work out of lengths and offsets on the device,
both compiled for the host (no GPU needed)."""

import ctypes
import os
import random
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = ctypes.c_void_p


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    out = tmp_path_factory.mktemp("host") / "kv4_ranges_host.so"
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    subprocess.run([hipcc, "-x", "hip", "--offload-host-only", "-no-hip-rt", "-O1", "-std=c++17", "-fPIC", "-shared",
                    "-Wno-everything", "-I", os.path.join(ROOT, "voyager-compiler_amd", "csrc"),
                    os.path.join(ROOT, "tests", "native", "kv4_ranges_host.cpp"), "-o", str(out)], check=True)
    return ctypes.CDLL(str(out))


def ranges(lib, room, kv, dim, group, kind, news, most, window, tree, lengths):
    """(rows of a tile, tiles, tokens of a split, splits), [sequences, tiles, (lo,
    hi, splits joined)]."""
    cu = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    given = np.array(lengths, np.int32)
    n = int(cu[-1])
    most = min(most, n)
    plan, tiles = np.zeros(4, np.int32), most * group // 16 + 2
    out = np.zeros(len(news) * tiles * 3, np.int32)
    lib.vqx_host_kv4_ranges(ctypes.c_int64(room), len(news), kv, dim, group, kind, n, cu.ctypes.data_as(P), most, window,
                            int(tree), given.ctypes.data_as(P), plan.ctypes.data_as(P), out.ctypes.data_as(P))
    return plan, out[:len(news) * int(plan[1]) * 3].reshape(len(news), int(plan[1]), 3)


def check(lib, room, kv, dim, group, kind, news, most, window, tree, lengths):
    case = (room, kv, dim, group, kind, news, most, window, tree, lengths)
    (rows, tiles, chunk, splits), found = ranges(lib, *case)
    for b, (new, length) in enumerate(zip(news, lengths)):
        count, base = min(new, most), min(max(length, 0), 1 << 30) - new
        for t in range(tiles):
            lo, hi, joined = (int(x) for x in found[b, t])
            if t * rows >= count * group:
                assert joined == 0, case
                continue
            # no more than were planned, and those cover the range
            assert 1 <= joined <= splits and hi - lo <= splits * chunk, (case, b, t, joined, splits)
            assert 0 <= lo <= hi <= room, case
            # nothing that a row may see lies outside
            first, last = t * rows // group, (min((t + 1) * rows, count * group) - 1) // group
            if tree:
                first, last = -1, count - 1
            least = max(0, base + first - window + 1) if window else 0
            end = min(room, max(0, base + last + 1))
            assert end <= hi and (lo <= least or least >= end), (case, b, t, lo, hi, least, end)


# more new tokens than `most` says, a window, and several splits
@pytest.mark.parametrize("room,kv,news,most,window,length", [
    (65536, 1, [3000], 64, 1990, 5000), (65536, 2, [64, 64], 8, 1976, 10000), (65536, 2, [128, 128], 64, 1920, 10000),
    (65536, 2, [200, 200], 16, 4000, 10000), (131072, 1, [70, 1], 1, 100000, 131000)])
@pytest.mark.parametrize("tree", [True, False])
def test_more_new_tokens_than_most(host, room, kv, news, most, window, length, tree):
    check(host, room, kv, 64, 1, 1, news, most, window, tree, [length] * len(news))


@pytest.mark.parametrize("seed", range(300))
def test_drawn_calls(host, seed):
    r = random.Random(seed)
    seqs, room = r.choice([1, 1, 2, 5, 40]), r.choice([64, 1000, 5000, 40000, 1 << 17, 1 << 20])
    tree = r.random() < 0.6
    news = [r.choice([0, 1, r.randint(1, 64), r.randint(1, 64 if tree else 800), r.randint(65, 4000)]) for _ in range(seqs)]
    if not sum(news):
        news[0] = 1
    most = r.choice([1, 8, 63, 64]) if tree else r.choice([1, 16, 100, max(news)])
    window = r.choice([0, 0, 1, 31, 33, r.randint(64, 4200), r.randint(64, max(65, room))])
    lengths = [r.choice([0, -5, new, r.randint(0, room), r.randint(0, room), room, room + r.randint(0, 1000), 2 ** 31 - 1])
               for new in news]
    check(host, room, r.choice([1, 2, 8, 16]), r.choice([64, 128, 256]), r.choice([1, 2, 5, 8]), r.choice([0, 1, 2]), news, most,
          window, tree, lengths)


def test_windows_have_several_splits(host):
    """So that the GPU's tests of windows join some."""
    from tests.test_gpu_kv4_tree_windows import BEYOND, WINDOWS

    for kind, dim, kv, group, lengths, news, most, window, page, _ in WINDOWS + BEYOND:
        room = -(-max(lengths) // page) * page if page else max(lengths)
        case = (room, kv, dim, group, dict(f32=0, bf16=1, f16=2)[kind], news, most, window, True, lengths)
        check(host, *case)
        assert int(ranges(host, *case)[0][3]) > 1, case
