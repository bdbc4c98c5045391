"""Pages for new tokens and the acceptance of drafted ones, against loops over
Python lists.  All of it is whole numbers: everything has to be equal."""

import random

import pytest
import torch

from tests import kv4_reference as ref
from tests.test_gpu_kv4 import make_cache, on, same

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(scope="module")
def ops(vqx):
    return torch.ops.quantized_ops


# ---------------------------------------------------------------------------
# reserve
# ---------------------------------------------------------------------------
def reserved(grow, lengths, table, free, count, size, n):
    """What kv4_reserve leaves and returns, from lists."""
    pages, per = len(free), len(table[0]) if table else 0
    for b, g in enumerate(grow):
        if g < 0:
            for page in table[b]:
                if 0 <= page < pages and count < pages:
                    free[count] = page
                    count += 1
            table[b], lengths[b] = [-1] * per, 0
    stock, needed, tokens = count, 0, 0
    cu, positions, slots = [0], [], []
    for b, g in enumerate(grow):
        g = max(g, 0)
        if lengths[b] >= 0 and lengths[b] + g <= per * size:
            places = range(lengths[b], lengths[b] + g)
            lack = sorted({t // size for t in places if not 0 <= table[b][t // size] < pages})
            needed, tokens = needed + len(lack), tokens + g
            if (not lack or needed <= stock) and tokens <= n:
                for j in lack:
                    count -= 1
                    table[b][j] = free[count]
                positions += places
                slots += [table[b][t // size] * size + t % size for t in places]
                lengths[b] += g
        cu.append(len(positions))
    rest = [-1] * (n - len(positions))
    return cu, positions + rest, slots + rest, lengths, table, free, count


def check_reserve(ops, grow, lengths, table, free, count, size, n):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    state = [i32(lengths), i32(table).reshape(len(grow), len(table[0]) if table else 2), i32(free), i32([count])]
    made = ops.kv4_reserve(i32(grow), *state, size, n)
    torch.cuda.synchronize()
    want = reserved(list(grow), list(lengths), [list(r) for r in table], list(free), count, size, n)
    for name, got, w in zip(("cu", "positions", "slots", "lengths", "table", "free", "count"), (*made, *state), want):
        same(got, torch.tensor(w, dtype=got.dtype).reshape(got.shape), name)
    return made, state


def scene(seed, seqs, per, size, spare, ending=0.2, most=50):
    """A server's state: rows filled up to their lengths, the other pages free."""
    r = random.Random(seed)
    lengths = [r.randrange(per * size + 1) for _ in range(seqs)]
    used = sum(-(-x // size) for x in lengths)
    ids = list(range(used + spare))
    r.shuffle(ids)
    table, at = [], 0
    for x in lengths:
        k = -(-x // size)
        table.append(ids[at:at + k] + [-1] * (per - k))
        at += k
    free = ids[at:] + [7] * used
    grow = [-1 if r.random() < ending else r.choice([0, 1, 1, r.randrange(most)]) for _ in range(seqs)]
    return grow, lengths, table, free, spare, size


@pytest.mark.parametrize("seqs,per,size,spare", [
    (1, 1, 1, 1), (1, 5, 16, 3), (16, 64, 64, 40), (63, 3, 7, 20), (64, 70, 16, 200), (65, 130, 4, 10), (300, 9, 32, 100),
    (1024, 5, 16, 500), (1025, 5, 16, 2000), (2500, 3, 8, 900)])
@pytest.mark.parametrize("seed", [0, 1])
def test_reserve(ops, seqs, per, size, spare, seed):
    s = scene(seed, seqs, per, size, spare)
    check_reserve(ops, *s, sum(max(g, 0) for g in s[0]))


@pytest.mark.parametrize("n", [0, 1, 17, 4096, 4097, 60000])
def test_reserve_room_for_tokens(ops, n):
    """Less room than tokens: the first that does not fit ends it; more: -1."""
    check_reserve(ops, *scene(5, 200, 40, 16, 4000, most=300), n)


def test_reserve_pages_run_out(ops):
    """Nobody overtakes the first that lacks a page, but who needs none is served;
    one without the room in its row is passed over."""
    table = [[0, -1, -1], [1, -1, -1], [2, -1, -1], [3, -1, -1], [4, 5, 6]]
    (cu, *_), (lengths, _, _, count) = check_reserve(
        ops, [9, 40, 3, 1, 1], [16, 2, 2, 16, 48], table, list(range(7, 10)) + [0] * 7, 3, 16, 100)
    # the second, 42 tokens, takes the two pages that the first left; the third needs none, the
    # fourth finds none, and the last, 49 tokens, has not the room
    assert cu.tolist() == [0, 9, 49, 52, 52, 52] and count.item() == 0 and lengths.tolist() == [25, 42, 5, 16, 48]
    (cu, *_), (lengths, _, _, count) = check_reserve(
        ops, [9, 50, 3, 1, 1], [16, 2, 2, 16, 48], table, list(range(7, 10)) + [0] * 7, 3, 16, 100)
    # here the second has not the room, and the fourth is served
    assert cu.tolist() == [0, 9, 9, 12, 13, 13] and count.item() == 1 and lengths.tolist() == [25, 2, 5, 17, 48]
    (cu, *_), (_, _, _, count) = check_reserve(
        ops, [9, 30, 3, 1, 1], [16, 2, 2, 16, 47], table, [9] + [0] * 9, 1, 16, 100)
    assert cu.tolist() == [0, 9, 9, 12, 12, 13] and count.item() == 0


def test_reserve_pages_behind_the_length(ops):
    """Pages that a row still has are used before others are taken, holes filled."""
    table = [[3, 4, 5, -1], [6, -1, 7, 99]]
    check_reserve(ops, [40, 50], [10, 4], table, [8, 9, 0, 1, 2] + [0] * 5, 5, 16, 90)


def test_reserve_all_end(ops):
    grow, lengths, table, free, spare, size = scene(3, 130, 12, 8, 0)
    made, state = check_reserve(ops, [-1] * 130, lengths, table, free, 0, size, 5)
    assert state[3].item() == len(free) and sorted(state[2].tolist()) == list(range(len(free)))
    assert made[1].tolist() == [-1] * 5


def test_reserve_many_entries(ops):
    """More entries of rows than are looked at together, of rows that end and of
    rows that grow; holes in them."""
    grow, lengths, table, free, spare, size = scene(4, 1100, 45, 4, 12000, ending=0.0)
    r = random.Random(2)
    lengths = [min(n, 100) for n in lengths]
    for row in table[::7]:
        row[r.randrange(45)] = -1
    check_reserve(ops, [r.choice([-1, 70, 61, 0]) for _ in range(1100)], lengths, table, free, spare, size, 80000)
    check_reserve(ops, [r.choice([77, 3]) for _ in range(1100)], lengths, table, free, spare, size, 30000)


def test_reserve_long_rows(ops):
    check_reserve(ops, [9000, -1, 20000], [100, 9999, 0], [[*range(7)] + [-1] * 1400, [*range(7, 632)] + [-1] * 782,
                                                         [-1] * 1407], list(range(632, 3000)) + [0] * 632, 2368, 16, 30000)


def test_reserve_what_is_given_back_is_taken(ops):
    check_reserve(ops, [-3, 33], [32, 0], [[0, 1, -1], [-1, -1, -1]], [2, 5, 5], 1, 16, 40)


def test_reserve_counts_that_are_wrong(ops):
    """A count or length outside its range, and pages that come back twice, reach
    no memory that is not theirs."""
    check_reserve(ops, [1, 1], [-5, 3], [[-1], [0]], [1, 0], 0, 16, 9)
    free = torch.full((4,), 9, dtype=torch.int32, device=DEV)
    for count in (-7, 100):
        state = [torch.tensor([40, 16], device=DEV).int(), torch.tensor([[0, 1, 2], [0, 1, -1]], device=DEV).int(), free[:3],
                 torch.tensor([count], device=DEV).int()]
        ops.kv4_reserve(torch.tensor([-1, -1], device=DEV).int(), *state, 16, 0)
        assert state[0].tolist() == [0, 0] and state[3].item() == 3 and free[3].item() == 9


def test_reserve_no_sequences(ops):
    cu, positions, slots = check_reserve(ops, [], [], [], [1, 0], 2, 16, 3)[0]
    assert cu.tolist() == [0] and positions.tolist() == [-1] * 3


def test_reserve_graph(ops):
    """A captured step hands pages out as sequences grow."""
    grow, lengths, table, free, spare, size = scene(8, 40, 30, 8, 300, ending=0.1)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    state = [i32(lengths), i32(table), i32(free), i32([spare])]
    dev = i32(grow)
    first = [t.clone() for t in state]
    ops.kv4_reserve(dev, *state, size, 64)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = ops.kv4_reserve(dev, *state, size, 64)
    for t, f in zip(state, first):
        t.copy_(f)
    want = (lengths, table, free, spare)
    r = random.Random(1)
    for i in range(5):
        grow = [r.choice([-1, 0, 1, 1, 1, 5]) for _ in range(40)]
        dev.copy_(i32(grow))
        graph.replay()
        torch.cuda.synchronize()
        out = reserved(list(grow), *(list(map(list, x)) if x is want[1] else list(x) if isinstance(x, list) else x
                                     for x in want), size, 64)
        for name, got, w in zip(("cu", "positions", "slots", "lengths", "table", "free", "count"), (*made, *state), out):
            same(got, torch.tensor(w, dtype=got.dtype).reshape(got.shape), f"{name} of replay {i}")
        want = out[3:]


# ---------------------------------------------------------------------------
# accept
# ---------------------------------------------------------------------------
def forest(news, seed, likely=0.6):
    """(tree, drafts, sampled) of drafted tokens; most of what is sampled is a
    child's number, some children have the same number."""
    r = random.Random(seed)
    tree, drafts, sampled = [], [], []
    for c in news:
        masks = []
        for j in range(c):
            parent = j - 1 if r.random() < 0.6 else r.randrange(j) if j else 0
            masks.append((masks[parent] | 1 << j if j else 1) if j < 64 else 0)
        ids = [r.randrange(6) for _ in range(c)]
        say = [r.randrange(6) for _ in range(c)]
        for j in range(1, min(c, 64)):
            parent = (masks[j] ^ 1 << j).bit_length() - 1
            if r.random() < likely:
                say[parent] = ids[j]
        tree += masks
        drafts += ids
        sampled += say
    return tree, drafts, sampled


def signed(x):
    return x - (1 << 64) if x >> 63 else x


def accepted(tree, drafts, sampled, spans):
    path, counts, follows = [-1] * len(tree), [], []
    for first, end in spans:
        c, line = min(end - first, 64), []
        if c:
            line = [0]
            while True:
                at = line[-1]
                child = [j for j in range(at + 1, c) if tree[first + j] == tree[first + at] | 1 << j
                         and drafts[first + j] == sampled[first + at]]
                if not child:
                    break
                line.append(child[0])
        path[first:first + len(line)] = line
        counts.append(len(line))
        follows.append(sampled[first + line[-1]] if line else -1)
    return path, counts, follows


def check_accept(ops, news, lengths, kv, dim, page, seed=0, even=False, behind=0, spoil=None, made=None):
    seqs, n = len(news), sum(news) + behind
    codes, scales, table = make_cache(seqs, kv, dim, max(lengths), page, seed)
    if spoil:
        spoil(table)
    tree, drafts, sampled = made or forest(news, seed)
    more = [0] * behind
    cu = None if even else torch.tensor([0] + news).cumsum(0).int()
    lens = torch.tensor(lengths).int()
    want_codes, want_scales = codes.clone(), scales.clone()
    spans = ref.spans(sum(news), seqs, cu)
    path, counts, follows = accepted(tree, drafts, sampled, spans)
    pages, size = codes.shape[1], codes.shape[3]
    for b, (first, end) in enumerate(spans):
        base = lengths[b] - (end - first)
        for i in range(counts[b]):
            if path[first + i] == i:
                continue
            to = ref.places(table, size, pages, b, [base + i] if 0 <= base + i < ref.room(codes, table) else [])
            for _, p, s in to:
                t = base + path[first + i]
                source = ref.places(table, size, pages, b, [t] if t < ref.room(codes, table) else [])
                for made, was in ((want_codes, codes), (want_scales, scales)):
                    made[:, p, :, s] = was[:, source[0][1], :, source[0][2]] if source else 0
    dev = on(torch.tensor([signed(x) for x in tree] + more), torch.tensor(drafts + more), torch.tensor(sampled + more), codes,
             scales, lens, cu, table)
    got = ops.kv4_accept(*dev)
    torch.cuda.synchronize()
    same(got[0], torch.tensor(path + [-1] * behind).int(), "path")
    same(got[1], torch.tensor(counts).int(), "accepted")
    same(got[2], torch.tensor(follows), "next")
    same(dev[5], torch.tensor([x - c + k for x, c, k in zip(lengths, news, counts)]).int(), "lengths")
    same(dev[3], want_codes, "codes")
    same(dev[4], want_scales, "scales")
    return counts


ACCEPT = [
    # new tokens, lengths, kv heads, dim, page
    ([1], [1], 1, 64, 0), ([2, 7], [2, 40], 2, 128, 16), ([8, 0, 3, 5], [100, 9, 3, 5], 3, 64, 7),
    ([64, 63, 33], [64, 700, 90], 4, 128, 64), ([64], [1000], 2, 256, 100), ([20] * 9, [60] * 9, 1, 256, 0),
    ([30, 41], [31, 300], 5, 128, 32)]


@pytest.mark.parametrize("news,lengths,kv,dim,page", ACCEPT)
@pytest.mark.parametrize("seed", range(4))
def test_accept(ops, news, lengths, kv, dim, page, seed):
    check_accept(ops, news, lengths, kv, dim, page, seed)


def test_accept_long_lines(ops):
    """Every second token in a line to the last, and all of a chain."""
    apart = [sum(1 << i for i in range(j % 2, j + 1, 2)) | 1 for j in range(64)]
    say = [5 if j % 2 == 0 else 6 for j in range(64)]
    assert check_accept(ops, [64], [100], 2, 64, 16, made=(apart, say, say)) == [32]
    chain = [(2 << j) - 1 for j in range(64)]
    assert check_accept(ops, [64], [64], 2, 128, 16, made=(chain, list(range(64)), list(range(1, 65)))) == [64]


def test_accept_even_offsets(ops):
    check_accept(ops, [6, 6, 6], [6, 30, 17], 2, 64, 16, even=True)


def test_accept_tokens_of_no_sequence(ops):
    check_accept(ops, [6, 2], [6, 30], 2, 64, 16, behind=70)


def test_accept_more_than_64(ops):
    check_accept(ops, [90, 5], [200, 20], 2, 64, 16)


def test_accept_places_before_the_beginning(ops):
    """A length below the number of new tokens: those before place 0 are not there."""
    check_accept(ops, [20, 9], [11, 0], 2, 64, 16, seed=2)


def test_accept_missing_pages(ops):
    def spoil(table):
        table[0, 1], table[1, 0] = -1, 10 ** 6
    for seed in range(4):
        check_accept(ops, [20, 20], [40, 30], 2, 64, 8, seed, spoil=spoil)


def test_accept_no_tokens(ops):
    codes, scales, table = make_cache(2, 1, 64, 32, 16)
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    dev = on(codes, scales, torch.tensor([5, 0]).int(), None, table)
    path, counts, follows = ops.kv4_accept(none, none, none, *dev)
    assert path.shape == (0,) and counts.tolist() == [0, 0] and follows.tolist() == [-1, -1]
    assert dev[2].tolist() == [5, 0]


def test_accept_graph(ops):
    """A captured acceptance follows what was drafted and sampled."""
    news, lengths = [12, 30, 1], [50, 31, 7]
    cu = torch.tensor([0] + news).cumsum(0).int()
    codes, scales, table = make_cache(3, 2, 128, 64, 16)
    i64 = lambda x: torch.tensor([signed(v) for v in x], device=DEV)  # noqa: E731
    state = [i64(x) for x in forest(news, 0)]
    dcodes, dscales, dlens, dcu, dt = on(codes, scales, torch.tensor(lengths).int(), cu, table)
    ops.kv4_accept(*state, dcodes, dscales, dlens, dcu, dt)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.kv4_accept(*state, dcodes, dscales, dlens, dcu, dt)
    for seed in range(1, 5):
        for t, x in zip(state, forest(news, seed)):
            t.copy_(i64(x))
        dlens.copy_(torch.tensor(lengths))
        dcodes.copy_(codes), dscales.copy_(scales)
        graph.replay()
        torch.cuda.synchronize()
        again = on(codes, scales, torch.tensor(lengths).int())
        want = ops.kv4_accept(*state, *again, dcu, dt)
        for name, got, w in zip(("path", "accepted", "next", "codes", "scales", "lengths"), (*out, dcodes, dscales, dlens),
                                (*want, *again)):
            same(got, w.cpu(), f"{name} of seed {seed}")
