"""GPU: the tables of an engine step (ops.step_tables) against a plain loop over the requests, exactly; and
KeSSieAttentionMetadata.build on top of it."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

FILL = -77


def plain(table, have, new, page, rows, free, delta):
    """table (list of lists, changed in place), start_loc, seq_lens, slots, positions, pages taken."""
    start, lens, slots, positions, used, upto = [0], [], [-1] * rows, [0] * rows, 0, 0
    for b, (c, n) in enumerate(zip(have, new)):
        c, n = max(c, 0), max(n, 0)
        first, held, total = start[-1], -(-c // page), -(-(c + n) // page)
        start.append(first + n)
        fits = total <= len(table[b]) and c + n < 1 << 31
        need = total - held if fits else 0
        upto += need
        ok = fits and first + n <= rows and (need == 0 or upto <= len(free))
        if ok:
            for i in range(need):
                table[b][held + i] = free[upto - need + i]
            used = upto if need else used
        lens.append(c + n if ok else c)
        for j in range(n):
            if first + j < rows:
                p = c + j
                positions[first + j] = min(p, (1 << 31) - 1) + delta[b]  # (positions saturate)
                pg = table[b][p // page] if ok else -1
                slots[first + j] = pg * page + p % page if pg >= 0 else -1
    return start, lens, slots, positions, used


def run(dev, have, new, page, width, rows, free, extra_free=0, delta=None, count=None, pages=None):
    from kessie_amd import ops

    b = len(have)
    i32 = dict(dtype=torch.int32, device=dev)
    table = [[1000 + 37 * r + i if i < -(-max(c, 0) // page) else FILL for i in range(width)] for r, c in enumerate(have)]
    got = torch.tensor(table, **i32).view(b, width)
    pages = 4096 if pages is None else pages
    valid, where = torch.zeros(pages, dtype=torch.int8, device=dev), torch.full((pages,), FILL, **i32)
    r = ops.step_tables(got, torch.tensor(have, **i32), torch.tensor(new, **i32), page, rows,
                        torch.tensor(list(free) + [5] * extra_free, **i32),
                        torch.tensor([len(free) if count is None else count], **i32),
                        position_delta=None if delta is None else torch.tensor(delta, **i32), page_valid=valid, page_positions=where)
    before = [list(x) for x in table]
    d = delta or [0] * b
    start, lens, slots, positions, used = plain(table, have, new, page, rows, list(free), d)
    assert r.query_start_loc.tolist() == start
    assert r.seq_lens.tolist() == lens
    assert r.slot_mapping.tolist() == slots
    assert r.positions.tolist() == positions
    assert r.taken.tolist() == [used]
    assert got.tolist() == table
    for b in range(len(have)):
        for i, (x, y) in enumerate(zip(before[b], table[b])):
            if x != y and 0 <= y < pages:  # a page taken
                assert valid[y] == 1 and where[y] == i * page + d[b]
    assert int(valid.sum()) == len({y for a, z in zip(before, table) for x, y in zip(a, z) if x != y and 0 <= y < pages})
    return r


@pytest.mark.parametrize("have,new,page,rows", [
    ([0], [1], 16, 1), ([15], [1], 16, 1), ([16], [1], 16, 4), ([0], [0], 16, 3), ([5, 0, 31, 32], [1, 40, 1, 1], 16, 43),
    ([0, 0, 0], [0, 17, 0], 16, 20), ([3, 3], [0, 0], 16, 0), ([-4, 7], [3, -2], 16, 8), ([100, 1], [1, 600], 1, 640),
    ([63, 64, 65, 127], [2, 63, 64, 1], 64, 300), ([10, 20], [7, 9], 48, 16),
])
def test_small_steps(dev, have, new, page, rows):
    run(dev, have, new, page, 700 // page + 2, rows, range(200, 200 + 700))


@pytest.mark.parametrize("count", [0, 1, 2, 3, 5, 6, 40, -3])
def test_a_free_list_that_does_not_suffice(dev, count):
    """Needs 1, 0, 2, 0, 3, 0: requests are granted in order while their running sum is within the list; those that
    need no page always are."""
    free = list(range(50, 56))[:max(0, min(count, 6))]
    run(dev, [16, 3, 0, 5, 0, 1], [1, 1, 20, 2, 48, 3], 16, 8, 75, free, extra_free=6 - len(free), count=count)


def test_rows_and_tables_that_do_not_suffice(dev):
    # The second request exceeds its table (8 pages) and takes nothing; the last one its token rows.
    run(dev, [0, 100, 0, 16], [20, 40, 17, 30], 16, 8, 100, range(9, 40))
    # A length that leaves 31 bits is refused like one that leaves the table.
    run(dev, [(1 << 31) - 2, 4], [5, 2], 1 << 20, 1 << 12, 9, range(9, 40))
    # Without a free list, requests go on within the pages they have.
    from kessie_amd import ops
    i32 = dict(dtype=torch.int32, device=dev)
    table = torch.tensor([[7, -1], [8, -1]], **i32)
    r = ops.step_tables(table, torch.tensor([3, 16], **i32), torch.tensor([2, 1], **i32), 16, 3)
    assert r.slot_mapping.tolist() == [7 * 16 + 3, 7 * 16 + 4, -1] and r.seq_lens.tolist() == [5, 16]
    assert r.taken.tolist() == [0] and table.tolist() == [[7, -1], [8, -1]]


def test_page_ids_outside_the_pool(dev):
    """A negative id gives its tokens no slot; ids outside page_valid are written to the table but set no flag."""
    run(dev, [0, 0], [16, 33], 16, 4, 60, [-5, 4090, 9000, 3], pages=4096)


def test_no_requests(dev):
    from kessie_amd import ops
    i32 = dict(dtype=torch.int32, device=dev)
    e = torch.empty(0, **i32)
    r = ops.step_tables(torch.empty(0, 4, **i32), e, e, 16, 5)
    assert r.query_start_loc.tolist() == [0] and r.slot_mapping.tolist() == [-1] * 5 and r.positions.tolist() == [0] * 5
    assert r.taken.tolist() == [0] and r.seq_lens.numel() == 0


@pytest.mark.parametrize("b,longest,page", [(1, 5000, 16), (255, 9, 16), (256, 40, 32), (1023, 3, 16), (1024, 30, 16), (1025, 12, 16),
                                            (2500, 1, 16), (5000, 7, 64)])
def test_many_requests(dev, b, longest, page):
    """The scan's edges (1,024 requests a pass), empty requests among them, padded rows, deltas."""
    rng = random.Random(b)
    have = [rng.choice([0, rng.randrange(0, 200)]) for _ in range(b)]
    new = [rng.choice([0, 1, 1, rng.randrange(0, longest + 1)]) for _ in range(b)]
    rows = sum(new) + rng.choice([0, 1, 300])
    need = sum(-(-(c + n) // page) - -(-c // page) for c, n in zip(have, new))
    width = -(-(200 + longest) // page)
    run(dev, have, new, page, width, rows, [rng.randrange(0, 1 << 20) for _ in range(need)], delta=[rng.randrange(-99, 99) for _ in have],
        pages=0)
    run(dev, have, new, page, width, max(0, rows // 2), [rng.randrange(0, 1 << 20) for _ in range(need // 3)], pages=0)


def test_strided_table_views_and_reused_outputs(dev):
    from kessie_amd import ops
    i32 = dict(dtype=torch.int32, device=dev)
    whole = torch.full((6, 12), FILL, **i32)
    table = whole[1:4, 2:7]
    out = (torch.empty(4, **i32), torch.empty(3, **i32), torch.empty(40, dtype=torch.int64, device=dev), torch.empty(40, **i32),
           torch.empty(1, **i32))
    args = (torch.tensor([0, 0, 0], **i32), torch.tensor([5, 17, 9], **i32), 16, 40, torch.arange(90, 99, **i32), torch.tensor([9], **i32))
    r = ops.step_tables(table, *args, out=out)
    assert r.slot_mapping.data_ptr() == out[2].data_ptr()
    want = torch.full((6, 12), FILL, dtype=torch.int32)
    want[1, 2], want[2, 2], want[2, 3], want[3, 2] = 90, 91, 92, 93
    assert torch.equal(whole.cpu(), want)
    assert r.slot_mapping.tolist() == [90 * 16 + i for i in range(5)] + [91 * 16 + i for i in range(16)] + [92 * 16] + \
        [93 * 16 + i for i in range(9)] + [-1] * 9
    with pytest.raises(ValueError, match="out must be"):
        ops.step_tables(table, *args, out=out[:3] + (out[3][:39], out[4]))


def test_captured_step_follows_its_inputs(dev):
    """A graph of the step, replayed with other lengths and another free list."""
    from kessie_amd import ops
    i32 = dict(dtype=torch.int32, device=dev)
    table, have, new = torch.full((3, 9), FILL, **i32), torch.zeros(3, **i32), torch.zeros(3, **i32)
    free, count = torch.arange(40, 60, **i32), torch.zeros(1, **i32)
    out = ops.step_tables(table, have, new, 16, 64, free, count)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.step_tables(table, have, new, 16, 64, free, count, out=out)
    for c, n, f in (([0, 0, 0], [20, 1, 3], 20), ([20, 1, 3], [1, 15, 14], 16), ([5, 5, 5], [30, 30, 1], 2)):
        table.fill_(FILL)
        for b, x in enumerate(c):
            table[b, :-(-x // 16)] = torch.arange(100 + 10 * b, 100 + 10 * b + -(-x // 16), **i32)
        plain_table = table.tolist()
        have.copy_(torch.tensor(c)), new.copy_(torch.tensor(n)), count.fill_(f)
        g.replay()
        start, lens, slots, positions, used = plain(plain_table, c, n, 16, 64, free.tolist()[:f], [0, 0, 0])
        assert out.query_start_loc.tolist() == start and out.seq_lens.tolist() == lens and out.slot_mapping.tolist() == slots
        assert out.positions.tolist() == positions and out.taken.tolist() == [used] and table.tolist() == plain_table


def test_metadata_build(dev):
    from kessie_amd.kessie_attention import KeSSieAttentionMetadata as Meta
    i32 = dict(dtype=torch.int32, device=dev)
    table = torch.full((4, 6), FILL, **i32)
    free = torch.arange(10, 30, **i32)
    m = Meta.build(table, [0, 0, 0], [18, 1, 40], 16, free, num_token_rows=64)
    assert (m.num_actual_tokens, m.max_query_len, m.max_seq_len, m.pages_taken) == (59, 40, 40, 6)
    assert m.query_start_loc.tolist() == m.query_start_loc_cpu.tolist() == [0, 18, 19, 59]
    assert m.seq_lens.tolist() == m.seq_lens_cpu.tolist() == [18, 1, 40]
    assert m.block_table.tolist() == [[10, 11] + [FILL] * 4, [12] + [FILL] * 5, [13, 14, 15] + [FILL] * 3]
    assert m.slot_mapping.tolist() == [160 + i for i in range(18)] + [12 * 16] + [13 * 16 + i for i in range(40)] + [-1] * 5
    m = Meta.build(table, [18, 1, 40], [1, 1, 1], 16, free[m.pages_taken:], position_delta=[0, 7, -2])
    assert m.positions.tolist() == [18, 8, 38] and m.pages_taken == 0 and m.slot_mapping.tolist() == [178, 193, 13 * 16 + 40]
    for bad in (dict(num_free=0), dict(num_token_rows=10)):
        with pytest.raises(ValueError):
            Meta.build(table, [32, 16, 40], [1, 1, 30], 16, free, **bad)
    with pytest.raises(ValueError, match="exceeds the block table"):
        Meta.build(table, [32, 16, 90], [1, 1, 30], 16, free)
