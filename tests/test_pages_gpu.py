"""Pages between sequences (csrc/pages.cu) against the rules carried out one row after the other."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
BS = 16


def pages_of(n, stride):
    return min((max(n, 0) + BS - 1) // BS, stride)


def fork_rules(table, lens, parents, refs, out):
    """the rules of b200q_pages_fork, row by row: (table, refs, slots, pairs, status)"""
    stride, refs0, refs, out = len(table[0]) if table else 0, list(refs), list(refs), [list(r) for r in out]
    slots, pairs, fresh, no_column, seen = [], [], [], 0, set()
    for i, p in enumerate(parents):
        slots.append(-1)
        pairs.append([-1, -1])
        if not 0 <= p < len(table):
            continue
        n = min(max(lens[p], 0), stride * BS)
        if n // BS >= stride:
            no_column += 1
        elif n % BS == 0 or p in seen or refs0[table[p][n // BS]] != 1:
            fresh.append(i)
        seen.add(p)
    free = [q for q, c in enumerate(refs0) if c == 0]
    if len(fresh) > len(free):
        return out, refs, [-1] * len(parents), [[-1, -1]] * len(parents), [len(fresh) - len(free), no_column]
    given = dict(zip(fresh, free))
    for i, p in enumerate(parents):
        if not 0 <= p < len(table):
            continue
        n = min(max(lens[p], 0), stride * BS)
        last = n // BS
        out[i][: pages_of(n, stride)] = table[p][: pages_of(n, stride)]
        if last < stride:
            if i in given:
                out[i][last] = given[i]
                if n % BS:
                    pairs[i] = [table[p][last], given[i]]
            slots[i] = out[i][last] * BS + n % BS
        for q in out[i][: max(pages_of(n, stride), min(last + 1, stride))]:
            refs[q] += 1
    for p, row in enumerate(table):
        for q in row[: pages_of(lens[p], stride)]:
            refs[q] -= 1
    return out, refs, slots, pairs, [0, no_column]


def make_state(rng, groups, beams, lens_of, spare, stride, others=0):
    """groups of rows that share their first pages, some pages held by rows outside (others)"""
    rows, lens, held = [], [], 0
    for g in range(groups):
        n = lens_of(g)
        pages = pages_of(n, stride)
        shared = rng.randint(0, pages)
        common = list(range(held, held + shared))
        held += shared
        for _ in range(beams):
            rows.append(common + list(range(held, held + pages - shared)))
            held += pages - shared
            lens.append(n)
    blocks = held + spare
    perm = list(range(blocks))
    rng.shuffle(perm)
    refs = [0] * blocks
    table = []
    for row in rows:
        row = [perm[q] for q in row]
        for q in row:
            refs[q] += 1
        table.append(row + [rng.randrange(blocks) for _ in range(stride - len(row))])
    for _ in range(others):
        q = rng.randrange(blocks)
        if refs[q]:
            refs[q] += 1
    return table, lens, refs


def ints(v, cuda):
    return torch.tensor(v, dtype=torch.int32, device=cuda)


def fork(lib, cuda, table, lens, parents, refs, stride, out=None):
    n = len(parents)
    t = {"table": ints(table, cuda).view(-1, stride), "lens": ints(lens, cuda), "refs": ints(refs, cuda), "out": ints(out, cuda).view(-1, stride),
         "slots": ints([7] * n, cuda), "pairs": torch.full((n, 2), 7, dtype=torch.int32, device=cuda), "status": ints([9, 9], cuda)}
    lib.pages_fork(t["table"], t["lens"], ints(parents, cuda), t["refs"], t["out"], t["slots"], t["pairs"], t["status"])
    return t


@pytest.mark.parametrize("groups,beams,stride,spare", [(1, 1, 1, 3), (1, 5, 6, 9), (3, 4, 9, 40), (40, 8, 5, 400), (300, 4, 30, 2000), (2, 3, 400, 20000), (4, 4, 7, 0),
                                                       (1500, 3, 4, 5000)])
@pytest.mark.parametrize("seed", [0, 1])
def test_fork(cuda, groups, beams, stride, spare, seed):
    from llmq_b200 import lib
    rng = random.Random(seed + groups)
    table, lens, refs = make_state(rng, groups, beams, lambda g: rng.choice((0, 1, 15, 16, 17, rng.randint(0, stride * BS), stride * BS, stride * BS - 1)), spare,
                                   stride, others=groups // 2)
    rows = len(table)
    parents = [b * beams + rng.randrange(beams) for b in range(groups) for _ in range(beams)]
    if seed:   # rows that end, and a parent that there is not
        parents = [rng.choice((-1, p, p, p)) for p in parents] + [rows, rows + 5]
    out = [[-3] * stride for _ in parents]
    want = fork_rules(table, lens, parents, refs, out)
    t = fork(lib, cuda, table, lens, parents, refs, stride, out)
    for name, w in zip(("out", "refs", "slots", "pairs", "status"), want):
        assert t[name].cpu().tolist() == w, name
    assert t["table"].cpu().tolist() == table


def test_first_step_and_end(cuda):
    """one row of a prompt becomes six beams, and the other way round; then everything is given back"""
    from llmq_b200 import lib
    for n in (32, 33):
        pages = pages_of(n, 4)
        table, refs = [[5, 3, 8][:pages] + [0] * (4 - pages)], [0] * 20
        for q in table[0][:pages]:
            refs[q] = 1
        want = fork_rules(table, [n], [0] * 6, refs, [[0] * 4 for _ in range(6)])
        t = fork(lib, cuda, table, [n], [0] * 6, refs, 4, [[0] * 4 for _ in range(6)])
        assert t["refs"].cpu().tolist() == want[1] and t["out"].cpu().tolist() == want[0] and t["pairs"].cpu().tolist() == want[3]
        back = fork(lib, cuda, want[0], [n + 1] * 6, [4], want[1], 4, [[0] * 4])
        want2 = fork_rules(want[0], [n + 1] * 6, [4], want[1], [[0] * 4])
        assert back["refs"].cpu().tolist() == want2[1] and back["out"].cpu().tolist() == want2[0]
        lib.pages_free(back["out"], ints([n + 2], cuda), back["refs"])
        assert back["refs"].cpu().tolist() == [0] * 20
        none = fork(lib, cuda, want[0], [n + 1] * 6, [], want[1], 4, [[0] * 4])   # no row goes on: all pages are given back
        assert none["refs"].cpu().tolist() == [0] * 20


def test_free(cuda):
    from llmq_b200 import lib
    rng = random.Random(3)
    table, lens, refs = make_state(rng, 30, 4, lambda g: rng.randint(0, 200), 11, 13)
    ends = [rng.randint(0, 1) for _ in table]
    want = list(refs)
    for row, n, e in zip(table, lens, ends):
        for q in row[: pages_of(n, 13)] if e else []:
            want[q] -= 1
    r = ints(refs, cuda)
    lib.pages_free(ints(table, cuda), ints(lens, cuda), r, ends=ints(ends, cuda))
    assert r.cpu().tolist() == want
    lib.pages_free(ints(table, cuda), ints(lens, cuda), r, ends=ints([1 - e for e in ends], cuda))
    assert r.cpu().tolist() == [0] * len(refs)


@pytest.mark.parametrize("dtype,width", [(torch.uint8, 16), (torch.uint8, 2304), (torch.bfloat16, 40000), (torch.float32, 4)])
@pytest.mark.parametrize("n", [1, 37])
def test_copy(cuda, dtype, width, n):
    from llmq_b200 import lib
    rng = random.Random(n)
    layers, blocks = 3, 100
    kv = torch.randint(0, 200, (layers, blocks, width), generator=torch.Generator().manual_seed(1)).to(dtype)
    ids = list(range(blocks))
    rng.shuffle(ids)
    pairs = [[ids[i % 10], ids[20 + i]] for i in range(n)]   # (a page may be copied to several places)
    pairs += [[-1, ids[90]], [ids[2], -1], [blocks, ids[91]], [ids[1], blocks]]
    want = kv.clone()
    for s, d in pairs[:n]:
        want[:, d] = kv[:, s]
    got = kv.to(cuda)
    lib.pages_copy(got, ints(pairs, cuda))
    assert torch.equal(got.cpu(), want)
    got = kv.to(cuda)
    for count in (0, -3, n // 2, 1000):
        lib.pages_copy(got, ints(pairs, cuda), ints([count], cuda))
        part = kv.clone()
        for s, d in pairs[: min(max(count, 0), n)]:
            part[:, d] = kv[:, s]
        assert torch.equal(got.cpu(), part)


def test_copy_of_far_pages(cuda):
    from llmq_b200 import lib
    kv = torch.zeros(2, 70000, 16 * 1024, dtype=torch.uint8, device=cuda)   # 2.3 GB
    kv[1, 3], kv[0, 3] = 5, 6
    lib.pages_copy(kv, ints([[3, 69999]], cuda))
    assert (kv[0, 69999] == 6).all() and (kv[1, 69999] == 5).all() and int(kv[:, 4:69999].max()) == 0


@pytest.mark.parametrize("blocks,live", [(1, 0.0), (1, 1.0), (5, 0.5), (4099, 0.3), (4100, 0.97), (50001, 0.1), (50001, 0.6), (50001, 0.0), (40000, 1.0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(cuda, blocks, live, in_place):
    from llmq_b200 import lib
    rng = random.Random(blocks)
    refs = [rng.randint(1, 9) if rng.random() < live else 0 for _ in range(blocks)]
    used = [q for q, c in enumerate(refs) if c]
    n = len(used)
    source, to = [q for q in used if q >= n], [q for q in range(n) if refs[q] == 0]
    where = [q if refs[q] and q < n else -1 for q in range(blocks)]
    for s, d in zip(source, to):
        where[s] = d
    counts = [0] * blocks
    for q in used:
        counts[where[q]] = refs[q]
    stride = 7
    lens = [rng.randint(0, 8 * BS) if used else 0 for _ in range(200)]
    table = [[rng.choice(used) if used and c < pages_of(n_, stride) else -5 for c in range(stride)] for n_ in lens]
    want = [[where[q] if c < pages_of(n_, stride) else -5 for c, q in enumerate(row)] for n_, row in zip(lens, table)]
    t, r = ints(table, cuda), ints(refs, cuda)
    t_out, r_out = (t, r) if in_place else (t.clone(), torch.full_like(r, 77))
    page_map, pairs, status = torch.full_like(r, 55), torch.full((blocks // 2 + 1, 2), -9, dtype=torch.int32, device=cuda), ints([4, 4], cuda)
    lib.pages_compact(t, ints(lens, cuda), r, t_out, r_out, page_map, pairs, status)
    assert status.cpu().tolist() == [n, len(to)]
    assert pairs.cpu().tolist() == [[s, d] for s, d in zip(source, to)] + [[-9, -9]] * (blocks // 2 + 1 - len(to))
    assert page_map.cpu().tolist() == where and r_out.cpu().tolist() == counts and t_out.cpu().tolist() == want


@pytest.mark.parametrize("n", [2 ** 31 - 1, 2 ** 31 - 15, 2 ** 31 - 16, 7 * BS + 1])
def test_lengths_beyond_the_table(cuda, n):
    """they count as the table's width, up to the largest there are"""
    from llmq_b200 import lib
    stride, rows, blocks = 7, 3, 60
    table = [[20 + 7 * r + c - r * (c == 0) for c in range(stride)] for r in range(rows)]   # (the rows' first pages: 20, 26, 32)
    refs = [0] * blocks
    for row in table:
        for q in row:
            refs[q] += 1
    used = [q for q in range(blocks) if refs[q]]
    where = {q: i for i, q in enumerate([q for q in used if q < len(used)])}
    free = [q for q in range(len(used)) if refs[q] == 0]
    where = {q: q for q in used if q < len(used)} | dict(zip([q for q in used if q >= len(used)], free))
    t, r, lens = ints(table, cuda), ints(refs, cuda), ints([n, 0, n], cuda)
    t_out, r_out, page_map = t.clone(), torch.zeros_like(r), torch.zeros_like(r)
    pairs, status = torch.zeros(blocks // 2 + 1, 2, dtype=torch.int32, device=cuda), ints([0, 0], cuda)
    lib.pages_compact(t, lens, r, t_out, r_out, page_map, pairs, status)
    assert t_out.cpu().tolist() == [[where[q] for q in table[0]], table[1], [where[q] for q in table[2]]]
    lib.pages_free(t, lens, r)
    want = list(refs)
    for q in table[0] + table[2]:
        want[q] -= 1
    assert r.cpu().tolist() == want
    out = [[-3] * stride for _ in range(rows)]
    f = fork(lib, cuda, table, [n, 5, n], [0, 2, 0], refs, stride, out)
    w = fork_rules(table, [n, 5, n], [0, 2, 0], refs, out)
    for name, x in zip(("out", "refs", "slots", "pairs", "status"), w):
        assert f[name].cpu().tolist() == x, name


def test_unaligned_counts(cuda):
    """counts that do not begin on a 16-byte boundary"""
    from llmq_b200 import lib
    rng = random.Random(8)
    table, lens, refs = make_state(rng, 5, 3, lambda g: rng.randint(0, 60), 33, 6)
    parents = [b * 3 + rng.randrange(3) for b in range(5) for _ in range(3)]
    out = [[-3] * 6 for _ in parents]
    want = fork_rules(table, lens, parents, refs, out)
    big = ints([4] + refs, cuda)
    r = big[1:]
    o, slots, pairs, status = ints(out, cuda), ints([0] * 15, cuda), torch.zeros(15, 2, dtype=torch.int32, device=cuda), ints([0, 0], cuda)
    lib.pages_fork(ints(table, cuda), ints(lens, cuda), ints(parents, cuda), r, o, slots, pairs, status)
    assert (o.cpu().tolist(), r.cpu().tolist(), slots.cpu().tolist(), pairs.cpu().tolist(), status.cpu().tolist()) == tuple(want) and int(big[0]) == 4
