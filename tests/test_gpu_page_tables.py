"""GPU: page tables and slots of requests that grow, against a loop over requests and tokens."""
import pytest
import torch

from rwkv_cuda_amd import page_tables as PT
from _gpu_util import DEV
from _mixers_util import graph_of

pytestmark = pytest.mark.gpu


def definition(lens, more, table, pool, taken, page, n):
    """slots, starts, held, taken and the table, in whole numbers of any size."""
    table, slots, starts, held = [list(r) for r in table], [], [0], []
    for b, (a, m) in enumerate(zip(lens, more)):
        a = max(a, 0)
        m = max(0, min(max(m, 0), len(table[b]) * page - a))
        for c in range(-(-a // page), -(-(a + m) // page)):
            table[b][c] = pool[taken] if 0 <= taken < len(pool) else -1
            taken += 1
        for t in range(a, a + m):
            if len(slots) < n:
                slot = table[b][t // page] * page + t % page if table[b][t // page] >= 0 else -1
                slots.append(slot if slot < 2 ** 31 else -1)
        starts.append(starts[-1] + m)
        held.append(a + m)
    return slots + [-1] * (n - len(slots)), starts, held, [taken], table


def check(lens, more, table, pool, taken, page, n):
    want = definition(lens, more, table, pool, taken, page, n)
    dev = [torch.tensor(z, dtype=torch.int32, device=DEV) for z in (lens, more, table, pool, [taken])]
    version = dev[2]._version
    got = PT.EXTEND(*dev, page, n)
    torch.cuda.synchronize()
    for name, g, w in zip(("slots", "starts", "held", "taken", "table"), (*got, dev[2]), want):
        assert g.dtype == torch.int32 and g.tolist() == w, name
    assert dev[2]._version > version
    return got


def requests(B, longest, tokens, M, page, seed, spare=7):
    g = torch.Generator().manual_seed(seed)
    draw = lambda hi: torch.randint(0, hi + 1, (B,), generator=g).tolist()
    lens, more = draw(longest), draw(tokens)
    pages = [min(M, -(-a // page)) for a in lens]
    pool = torch.randperm(sum(pages) + sum(-(-m // page) + 1 for m in more) + spare, generator=g).tolist()
    table, at = [], 0
    for c in pages:
        table.append(pool[at:at + c] + [-9] * (M - c))
        at += c
    return lens, more, table, pool, at


@pytest.mark.parametrize("B,longest,tokens,M,page", [(1, 0, 1, 1, 1), (1, 100, 1, 8, 16), (3, 50, 40, 9, 16), (17, 5, 3, 4, 2), (256, 300, 1, 40, 16), (300, 20, 700, 90, 8), (1023, 64, 1, 70, 1),
                                                     (1024, 9, 9, 3, 8), (1025, 9, 9, 3, 8), (3000, 40, 11, 60, 1), (5, 3000, 9000, 200, 64)])
def test_against_a_loop(lib, B, longest, tokens, M, page):
    lens, more, table, pool, taken = requests(B, longest, tokens, M, page, seed=B)
    total = sum(max(0, min(m, M * page - a)) for a, m in zip(lens, more))
    for n in (total, total + 100, max(0, total - 1), total // 2):
        check(lens, more, table, pool, taken, page, n)


def test_what_is_not_there(lib):
    """Counts below 0, rows that are full, no tokens at all, pools that are too short or behind, pages that no table may name, and no slots."""
    lens, more, table, pool, taken = requests(9, 40, 60, 8, 16, seed=1)
    lens[0], lens[1], more[2], more[3], lens[4], more[4] = -5, 128, -3, 2 ** 31 - 1, 126, 100
    lens[5], more[5] = 4000, 10                                  # more than the table has pages for
    table[6][0] = -2 ** 31
    table[7][0] = 2 ** 31 - 1
    lens[6], lens[7], more[6], more[7] = 3, 3, 5, 5
    check(lens, more, table, pool, taken, 16, 400)
    check(lens, more, table, pool, len(pool) - 2, 16, 400)
    check(lens, more, table, pool, 2 ** 31 - 40, 16, 400)
    check(lens, more, table, pool, -3, 16, 400)
    check(lens, [0] * 9, table, pool, taken, 16, 5)
    check(lens, more, table, pool, taken, 16, 0)


def test_starts_stay_within_31_bits(lib):
    B, M, page = 5, 1 << 11, 1 << 19
    lens, more = [0] * B, [2 ** 30] * B
    table = torch.zeros(B, M, dtype=torch.int32, device=DEV)
    dev = [torch.tensor(z, dtype=torch.int32, device=DEV) for z in (lens, more)]
    pool, taken = torch.arange(B * M, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    slots, starts, held, out = PT.EXTEND(*dev, table, pool, taken, page, 1000)
    torch.cuda.synchronize()
    assert starts.tolist() == [0, 2 ** 30, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1] and held.tolist() == more and out.tolist() == [B * M]
    assert slots.tolist() == list(range(1000)) and torch.equal(table.flatten(), pool)


def test_captured_and_replayed(lib):
    """Steps of a token a row, captured; the results are put back where the next step reads them, as a serving loop does."""
    B, M, page, steps = 33, 6, 4, 18
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    more, taken = torch.ones_like(lens), torch.zeros(1, dtype=torch.int32, device=DEV)
    more[5] = 0
    table = torch.full((B, M), -1, dtype=torch.int32, device=DEV)
    pool = torch.randperm(B * M, generator=torch.Generator().manual_seed(2)).to(torch.int32).to(DEV)

    def step():
        slots, starts, held, out = PT.EXTEND(lens, more, table, pool, taken, page, B)
        lens.copy_(held), taken.copy_(out)
        return slots, starts
    graph, (slots, starts) = graph_of(step)
    torch.cuda.synchronize()
    lens.zero_(), taken.zero_(), table.fill_(-1)
    host = [[0] * B, [-1] * 0, [[-1] * M for _ in range(B)], 0]
    for i in range(steps):
        graph.replay()
        torch.cuda.synchronize()
        want = definition(host[0], more.tolist(), host[2], pool.tolist(), host[3], page, B)
        host[0], host[2], host[3] = want[2], want[4], want[3][0]
        assert slots.tolist() == want[0] and starts.tolist() == want[1] and table.tolist() == want[4] and taken.tolist() == want[3], i
