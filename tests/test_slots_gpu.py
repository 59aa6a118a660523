"""Pages and slot maps (mla_build_slots) against a request-by-request loop: whole
numbers, so everything has to be equal."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def plan_by_hand(lens, news, table, free, head, page, num_tokens):
    table, width = [list(r) for r in table], len(table[0]) if table else 0
    slots, positions, cu = [], [], [0]
    at = head
    for b, (n, m) in enumerate(zip(lens, news)):
        n, m = max(n, 0), max(m, 0)
        have, want = min(width, -(-n // page)), min(width, -(-(n + m) // page))
        for blk in range(have, want):
            table[b][blk] = free[at] if 0 <= at < len(free) else -1
            at += 1
        for p in range(n, n + m):
            pg = table[b][p // page] if p // page < width else -1
            slots.append(pg * page + p % page if pg >= 0 else -1)
            positions.append(p)
        cu.append(cu[-1] + m)
    pad = max(0, num_tokens - len(slots))
    return (slots[:num_tokens] + [-1] * pad, positions[:num_tokens] + [0] * pad, cu,
            [max(n, 0) + max(m, 0) for n, m in zip(lens, news)], at, table)


def check(lens, news, page, width, num_free, head=0, num_tokens=None, seed=0, stride=None):
    import ada_mla

    g = torch.Generator().manual_seed(seed)
    pages = torch.randperm(1 << 20, generator=g).to(torch.int32)
    free, pages = pages[:num_free], pages[num_free:].tolist()
    table = torch.full((len(lens), width), -7, dtype=torch.int32)
    for b, n in enumerate(lens):
        for blk in range(min(width, -(-max(n, 0) // page))):
            table[b, blk] = pages.pop()
    total = sum(max(m, 0) for m in news)
    num_tokens = total if num_tokens is None else num_tokens
    want = plan_by_hand(lens, news, table.tolist(), free.tolist(), head, page, num_tokens)
    wide = torch.full((len(lens), stride or width), -9, dtype=torch.int32, device="cuda")
    dev = wide[:, :width]
    dev.copy_(table)
    args = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lens, news)]
    for _ in range(2):  # planning a step again gives the same
        p = ada_mla.mla_build_slots(*args, dev, free.cuda(), page, num_tokens,
                                    free_head=torch.tensor([head], dtype=torch.int32, device="cuda") if head else None)
        got = (p.slots.tolist(), p.positions.tolist(), p.cu_new.tolist(), p.seq_lens.tolist(), int(p.free_head), dev.tolist())
        for name, a, b in zip(("slots", "positions", "cu_new", "seq_lens", "free_head", "table"), got, want):
            assert a == b, name
    assert p.slots.dtype == torch.int64
    if stride:
        assert bool((wide[:, width:] == -9).all())


@pytest.mark.parametrize("batch", [1, 2, 31, 256, 1023, 1025, 3000])
@pytest.mark.parametrize("page", [1, 32, 64])
def test_decode_step(batch, page):
    g = torch.Generator().manual_seed(batch + page)
    lens = torch.randint(0, 300, (batch,), generator=g).tolist()
    check(lens, [1] * batch, page, 320 // page + 1, batch + 3, head=2, seed=batch)


@pytest.mark.parametrize("seed", range(4))
def test_prompts_of_mixed_lengths(seed):
    g = torch.Generator().manual_seed(seed)
    news = torch.randint(0, 3000, (37,), generator=g).tolist()
    news[3] = news[4] = 0
    news[5] = 1
    lens = (torch.randint(0, 200, (37,), generator=g) * torch.randint(0, 2, (37,), generator=g)).tolist()
    check(lens, news, 48, 80, 37 * 80, head=5, seed=seed, stride=91)


def test_one_token_one_page_and_nothing():
    check([0], [1], 64, 1, 1)
    check([63], [1], 64, 2, 1)   # fills its page
    check([64], [1], 64, 2, 1)   # opens the next
    check([0, 0, 0], [0, 0, 0], 64, 2, 1)
    check([], [], 64, 4, 2)
    check([5], [0], 64, 1, 0, num_tokens=4)


def test_list_and_table_run_out():
    check([0, 10, 0], [100, 100, 100], 32, 4, 5)            # 4 + 3 + 4 pages asked for, 5 free
    check([0, 0], [500, 40], 32, 4, 20)                     # the table is 4 pages wide
    check([300], [10], 32, 4, 20)                           # longer than its table already
    check([1, 2], [40, 50], 32, 8, 20, num_tokens=1500)     # room for more tokens than come
    check([1, 2], [40, 50], 32, 8, 20, num_tokens=60)       # and for fewer
    check([-4, 6], [3, -2], 32, 8, 20)                      # counts below zero are zero


def test_refusals():
    import ada_mla

    i32 = dict(dtype=torch.int32, device="cuda")
    lens, table, free = torch.zeros(2, **i32), torch.zeros(2, 4, **i32), torch.zeros(3, **i32)
    ok = (lens, lens, table, free, 64, 0)
    ada_mla.mla_build_slots(*ok)
    for at, bad in [(0, lens.long()), (0, lens.cpu()), (1, torch.zeros(3, **i32)), (2, table.t().contiguous().t()), (2, table[:1]),
                    (2, table.float()), (3, free[None]), (3, free.cpu()), (4, 0), (5, -1), (5, 1 << 31)]:
        args = list(ok)
        args[at] = bad
        with pytest.raises((RuntimeError, TypeError)):
            ada_mla.mla_build_slots(*args)
    with pytest.raises(RuntimeError):
        ada_mla.mla_build_slots(*ok, free_head=torch.zeros(2, **i32))


def test_other_stream():
    import ada_mla

    s = torch.cuda.Stream()
    lens = torch.full((8,), 3, dtype=torch.int32, device="cuda")
    table, free = torch.zeros(8, 4, dtype=torch.int32, device="cuda"), torch.arange(64, dtype=torch.int32, device="cuda")
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        p = ada_mla.mla_build_slots(lens, torch.full_like(lens, 100), table, free, 64, 800)
    s.synchronize()
    assert p.cu_new.tolist() == list(range(0, 801, 100)) and int(p.free_head) == 8


@pytest.mark.parametrize("tokens", [1, 256, 4096, 4097, 100000])
def test_what_a_caller_keeps_is_small(tokens):
    """The lengths and the head go on to the next step: what they keep alive does not grow
    with the step's tokens."""
    import ada_mla

    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    table, free = torch.zeros(3, 2000, dtype=torch.int32, device="cuda"), torch.arange(2000, dtype=torch.int32, device="cuda")
    p = ada_mla.mla_build_slots(lens, torch.tensor([tokens, 0, 0], dtype=torch.int32, device="cuda"), table, free, 64, tokens)
    assert p.seq_lens.tolist() == [tokens, 0, 0] and int(p.free_head) == -(-tokens // 64)
    assert p.slots[-1].item() == tokens - 1 and p.positions[-1].item() == tokens - 1
    for kept in (p.seq_lens, p.free_head, p.cu_new):
        assert kept.untyped_storage().nbytes() <= 12 * 4096 + 256
