"""Draft-tree decode (mla_decode_tree) against the definition in 64 bits.

Bound of one output element, with u the unit roundoff of the inputs' type (2^-11 fp16,
2^-8 bf16), p the softmax row and A = sum_j p_j |c_j|: the weights go into the second
product rounded to that type (u A, and at most 2^-25 each for fp16 weights below its
normal numbers, relative to a largest weight of at least 1), the output is rounded once
(u |o|), and fp32 logits and sums (576 and N terms) stay below 2^-13 A for the sizes
here; fp32 output drops the output's rounding.  LSE: fp32 logits of size below 16,
accumulated over 576 terms: 2^-14."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SCALE = 192.0 ** -0.5
LSE_TOL = 2.0 ** -14


def problem(batch, k, heads, lens, page, dtype, seed, spare=2):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(batch, k, heads, 576, generator=g).to(dtype)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    pool = torch.randn(pages, page, 576, generator=g).to(dtype)
    perm = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((batch, max(max(need), 1) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return q, pool, table, torch.tensor(lens, dtype=torch.int32)


def rows_of(pool, table, b, n):
    page = pool.shape[1]
    t = torch.arange(n)
    return pool.view(-1, 576)[table[b].long()[t // page] * page + t % page]


def expect(q, pool, table, lens, mask, dtype, out_dtype=None):
    batch, k, heads, _ = q.shape
    out = torch.zeros(batch, k, heads, 512, dtype=torch.float64)
    lse = torch.full((batch, k, heads), float("-inf"), dtype=torch.float64)
    tol = torch.zeros_like(out)
    u = U[dtype]
    for b in range(batch):
        n = int(lens[b])
        c = rows_of(pool, table, b, n).double()
        for i in range(k):
            m = (2 << i) - 1 if mask is None else int(mask[b, i] if mask.dim() == 2 else mask[i]) & ((1 << 64) - 1)
            see = [t for t in range(n) if t < n - k or (m >> (t - (n - k))) & 1]
            if not see:
                continue
            cs = c[see]
            x = q[b, i].double() @ cs.t() * SCALE
            p = torch.softmax(x, 1)
            out[b, i] = p @ cs[:, :512]
            lse[b, i] = torch.logsumexp(x, 1)
            a = p @ cs[:, :512].abs()
            tol[b, i] = (u + 2.0 ** -13) * a + 2.0 ** -25 * cs[:, :512].abs().sum(0)
            if out_dtype != torch.float32:
                tol[b, i] += u * out[b, i].abs() + 2.0 ** -24
    return out, lse, tol


def check(q, pool, table, lens, mask=None, num_splits=-1, out_dtype=None, want=None):
    import ada_mla

    dev = [t.cuda() for t in (q, pool, table, lens)]
    got, lse = ada_mla.mla_decode_tree(*dev, None if mask is None else mask.cuda(), max_seq_len=int(lens.max()) if len(lens) else 0,
                                       softmax_scale=SCALE, num_splits=num_splits, return_lse=True, out_dtype=out_dtype)
    assert ada_mla.mla_get_device_error() == 0
    w, wl, tol = expect(q, pool, table, lens, mask, q.dtype, out_dtype) if want is None else want
    diff = (got.double().cpu() - w).abs()
    assert bool((diff <= tol).all()), float((diff / tol.clamp(min=1e-30)).max())
    none = torch.isinf(wl)
    assert bool((torch.isneginf(lse.cpu()) == none).all())
    assert bool(((lse.cpu().double() - wl)[~none].abs() <= LSE_TOL).all())
    return got, lse


def random_tree(batch, k, seed):
    import ada_mla

    g = torch.Generator().manual_seed(seed)
    parents = (torch.rand(batch, k, generator=g) * (torch.arange(k) + 1)).long() - 1
    return ada_mla.tree_mask(parents)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,k,heads,lens,page", [
    (1, 1, 1, [1], 32), (1, 1, 128, [500], 64), (1, 8, 16, [4096], 64), (3, 7, 16, [7, 96, 1000], 32), (2, 5, 32, [97, 640], 96),
    (2, 3, 128, [333, 65], 64), (1, 64, 2, [700], 64), (2, 64, 16, [64, 911], 128), (9, 2, 20, [2, 3, 31, 32, 33, 95, 96, 97, 191], 32),
    (4, 4, 96, [500, 4, 1000, 12], 64)])
def test_random_trees(dtype, batch, k, heads, lens, page):
    q, pool, table, n = problem(batch, k, heads, lens, page, dtype, seed=batch * 100 + k)
    check(q, pool, table, n, random_tree(batch, k, seed=k))


@pytest.mark.parametrize("num_splits", [1, 2, 5, 100])
def test_explicit_splits_and_fp32_output(num_splits):
    q, pool, table, n = problem(2, 6, 16, [900, 300], 64, torch.float16, seed=3)
    mask = random_tree(2, 6, seed=1)
    check(q, pool, table, n, mask, num_splits=num_splits, out_dtype=torch.float32)
    q, pool, table, n = problem(1, 6, 16, [900], 64, torch.bfloat16, seed=3)
    check(q, pool, table, n, mask[:1], num_splits=num_splits)


def test_chain_matches_multi_token_decode_and_shared_mask():
    import ada_mla

    q, pool, table, n = problem(2, 4, 16, [256, 256], 64, torch.float16, seed=5)
    a, la = check(q, pool, table, n, None)
    chain = torch.tensor([(2 << i) - 1 for i in range(4)])
    b, lb = check(q, pool, table, n, chain)
    assert torch.equal(a, b) and torch.equal(la, lb)
    dense = torch.stack([rows_of(pool, table, i, 256) for i in range(2)]).cuda()
    m, lm = ada_mla.mla_decode_mtp(q.cuda(), dense, softmax_scale=SCALE, return_lse=True)
    assert float((m.float() - a.float()).abs().max()) <= 4 * 2.0 ** -11
    assert float((lm - la).abs().max()) <= 2 * LSE_TOL


def test_rows_that_see_nothing():
    q, pool, table, n = problem(3, 5, 16, [5, 3, 0], 32, torch.float16, seed=6)  # no context; shorter than the drafts; empty
    mask = torch.tensor([[0, 1, 0b101, 0, 0b11111]] * 3)
    got, lse = check(q, pool, table, n, mask)
    assert bool((got[0, 0] == 0).all()) and bool(torch.isneginf(lse[0, 0]).all()) and bool((got[2] == 0).all())
    q, pool, table, n = problem(1, 4, 32, [4], 32, torch.float16, seed=6)
    check(q, pool, table, n, torch.zeros(1, 4, dtype=torch.int64))
    check(q, pool, table, torch.tensor([0], dtype=torch.int32), None)


def test_bits_past_the_drafts_are_ignored():
    q, pool, table, n = problem(1, 3, 16, [130], 64, torch.float16, seed=7)
    mask = torch.tensor([[1, 3, 7]])
    a, _ = check(q, pool, table, n, mask)
    b, _ = check(q, pool, table, n, mask | -8)  # every bit from 3 to 63
    assert torch.equal(a, b)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -65504.0])
def test_masked_places_may_hold_anything(bad):
    """Unwritten padded drafts, page rows past the end and pages nobody owns."""
    import ada_mla

    for lens in ([100, 257], [5, 96], [97, 131]):
        q, pool, table, n = problem(2, 5, 16, lens, 32, torch.float16, seed=8)
        mask = torch.tensor([[1, 3, 0, 0, 0], [1, 3, 5, 13, 0]])  # drafts 2.. of the first, 4 of the second are padding
        want = expect(q, pool, table, n, mask, torch.float16)
        clean, _ = check(q, pool, table, n, mask, want=want)
        flat = pool.clone().view(-1, 576)
        keep = torch.zeros(flat.shape[0], dtype=torch.bool)
        for b in range(2):
            t = torch.arange(lens[b] - (3 if b == 0 else 1))
            keep[table[b].long()[t // 32] * 32 + t % 32] = True
        flat[~keep] = bad
        got, _ = check(q, flat.view_as(pool), table, n, mask, want=want)
        assert torch.equal(got, clean)
    assert ada_mla.mla_get_device_error() == 0


def test_large_logits_and_equal_logits():
    q, pool, table, n = problem(1, 8, 16, [400], 64, torch.float16, seed=9)
    check((q * 0), pool, table, n, random_tree(1, 8, seed=2))
    q2 = q * 6  # logits to +-60: the running maximum moves by many powers of two
    w = expect(q2, pool, table, n, None, torch.float16)
    import ada_mla

    got, lse = ada_mla.mla_decode_tree(q2.cuda(), pool.cuda(), table.cuda(), n.cuda(), softmax_scale=SCALE, return_lse=True)
    # logits six times larger carry six times the fp32 error into the weights
    assert bool(((got.double().cpu() - w[0]).abs() <= 6 * w[2]).all())
    assert float((lse.cpu().double() - w[1]).abs().max()) <= 8 * LSE_TOL


@pytest.mark.parametrize("batch,k,heads,lens", [(2, 5, 128, [700, 333]), (1, 12, 128, [2000]), (3, 40, 128, [97, 1300, 5]), (1, 64, 3, [900]), (2, 64, 16, [0, 800])])
def test_bound_far_above_the_lengths(batch, k, heads, lens):
    """max_seq_len is a bound: the schedule goes by the lengths."""
    import ada_mla

    lens = [n if n == 0 else max(n, k) for n in lens]
    q, pool, table, n = problem(batch, k, heads, lens, 32, torch.float16, seed=batch + k)
    mask = random_tree(batch, k, seed=k)
    want = expect(q, pool, table, n, mask, torch.float16)
    wide = torch.full((batch, 2200), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    dev = [t.cuda() for t in (q, pool, wide, n, mask)]
    for bound in (int(n.max()), 70000):
        got, lse = ada_mla.mla_decode_tree(*dev, max_seq_len=bound, softmax_scale=SCALE, return_lse=True)
        assert ada_mla.mla_get_device_error() == 0
        diff = (got.double().cpu() - want[0]).abs()
        assert bool((diff <= want[2]).all()), float((diff / want[2].clamp(min=1e-30)).max())
        none = torch.isinf(want[1])
        assert bool((torch.isneginf(lse.cpu()) == none).all())
        assert bool(((lse.cpu().double() - want[1])[~none].abs() <= LSE_TOL).all())


def test_max_seq_len_read_from_device_and_other_stream():
    import ada_mla

    q, pool, table, n = problem(2, 3, 16, [200, 64], 64, torch.bfloat16, seed=10)
    want = expect(q, pool, table, n, None, torch.bfloat16)
    dev = [t.cuda() for t in (q, pool, table, n)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ada_mla.mla_decode_tree(*dev, softmax_scale=SCALE)
    s.synchronize()
    assert bool(((got.double().cpu() - want[0]).abs() <= want[2]).all())


def test_refusals():
    import ada_mla

    q, pool, table, n = (t.cuda() for t in problem(2, 3, 16, [70, 40], 32, torch.float16, seed=11))
    mask = torch.ones(2, 3, dtype=torch.int64, device="cuda")
    ok = dict(query=q, kv_pages=pool, block_table=table, seq_lens=n, tree_mask=mask, max_seq_len=70)
    ada_mla.mla_decode_tree(**ok)
    big = torch.zeros(1, 65, 2, 576, device="cuda").half()
    for bad in [dict(query=q.float()), dict(query=q[:, :, :, :575]), dict(query=q.bfloat16()), dict(query=q.transpose(1, 2)), dict(query=big),
                dict(query=torch.zeros(2, 3, 129, 576, device="cuda").half()), dict(kv_pages=pool.cpu()), dict(kv_pages=pool[:, :20].contiguous()),
                dict(block_table=table.long()), dict(seq_lens=n.long()), dict(seq_lens=n[:1]), dict(tree_mask=mask.int()), dict(tree_mask=mask[:1]),
                dict(tree_mask=mask.cpu()), dict(max_seq_len=1 << 20), dict(softmax_scale=0.0), dict(softmax_scale=float("nan"))]:
        with pytest.raises(RuntimeError):
            ada_mla.mla_decode_tree(**{**ok, **bad})
    with pytest.raises(ValueError):
        ada_mla.mla_decode_tree(**ok, out_dtype=torch.bfloat16)
    assert ada_mla.mla_decode_tree(q[:0], pool, table[:0], n[:0]).shape == (0, 3, 16, 512)


def test_calls_back_to_back():
    """Streams longer than the L2, 112 rows a tile, call after call: loads come in late and
    out of order, and every call gives the first one's bits."""
    import ada_mla

    g = torch.Generator().manual_seed(5)
    lens = [1000 + 97 * i for i in range(48)]
    sets = []
    for s in range(2):
        need = [-(-n // 64) for n in lens]
        perm = torch.randperm(sum(need), generator=g).to(torch.int32)
        table = torch.full((48, max(need)), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = perm[at:at + n]
            at += n
        sets.append((torch.randn(48, 7, 16, 576, generator=g).half().cuda(), torch.randn(sum(need), 64, 576, device="cuda").half(),
                     table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()))
    first = [ada_mla.mla_decode_tree(*s, max_seq_len=max(lens), softmax_scale=SCALE) for s in sets]
    for _ in range(20):
        outs = [ada_mla.mla_decode_tree(*sets[i % 2], max_seq_len=max(lens), softmax_scale=SCALE) for i in range(40)]
        assert all(torch.equal(o, first[i % 2]) for i, o in enumerate(outs))
    assert ada_mla.mla_get_device_error() == 0


@pytest.mark.parametrize("batch,k,heads,n", [(1, 8, 16, 1500), (2, 7, 16, 700), (1, 12, 128, 900), (7, 3, 16, 400), (40, 7, 16, 1700)])
def test_chained_calls_back_to_back(batch, k, heads, n):
    """Few row tiles' decode, merge and next decode are chained: a merge is resident while
    its decode writes.  Calls on inputs in turn give each input's own bits."""
    import ada_mla

    lens = [n - 40 * b for b in range(batch)]
    sets = [[t.cuda() for t in problem(batch, k, heads, lens, 64, torch.float16, seed=30 + s)] for s in range(3)]
    first = []
    for s in sets:
        first.append(ada_mla.mla_decode_tree(*s, max_seq_len=n, softmax_scale=SCALE, return_lse=True))
        torch.cuda.synchronize()
    for _ in range(20):
        outs = [ada_mla.mla_decode_tree(*sets[i % 3], max_seq_len=n, softmax_scale=SCALE, return_lse=True) for i in range(60)]
        assert all(torch.equal(o, first[i % 3][0]) and torch.equal(l, first[i % 3][1]) for i, (o, l) in enumerate(outs))
    assert ada_mla.mla_get_device_error() == 0


def uneven(batch, k, heads, lens, dtype, seed, span):
    """Latent columns of sizes 1 to 2^span within any 32 neighbours, all of one sign, so that
    no column's output averages out; the queries take the sizes out of the logits again."""
    q, pool, table, n = problem(batch, k, heads, lens, 64, dtype, seed)
    size = 2.0 ** (torch.arange(512) * 7 % (span + 1))
    pool[..., :512] = (pool[..., :512].float().abs() * size).to(dtype)
    q[..., :512] = (q[..., :512].float() / size).to(dtype)
    return q, pool, table, n


@pytest.mark.parametrize("out_dtype", [None, torch.float32])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("span", [6, 10])
@pytest.mark.parametrize("k,heads,lens", [(8, 16, [1900]), (7, 16, [1100, 300, 2000]), (12, 128, [800])])
def test_columns_of_different_sizes(k, heads, lens, span, dtype, out_dtype):
    """A column's error goes by that column's values, whatever its neighbours hold and
    whether the sequence is split or not.  For 16-bit output the split partials are fp32 cut
    to 24 bits, below 2^-15 of each value: 2^-15 A on top of the bound above."""
    import ada_mla

    q, pool, table, n = uneven(len(lens), k, heads, lens, dtype, 40 + k, span)
    mask = random_tree(len(lens), k, seed=k)
    w, wl, tol = expect(q, pool, table, n, mask, dtype, out_dtype)
    if out_dtype is None:
        tol = tol + 2.0 ** -15 * w  # (all values are positive: A is the output itself)
    for splits in (-1, 1, 3):
        got, _ = check(q, pool, table, n, mask, num_splits=splits, out_dtype=out_dtype, want=(w, wl, tol))
    assert ada_mla.mla_get_device_error() == 0


@pytest.mark.parametrize("num_splits", [-1, 1, 4])
def test_an_infinite_value_stays_in_its_column(num_splits):
    """A cached row with an infinite value whose logit is -inf: 0 x inf in that column, and
    nothing else changes."""
    import ada_mla

    q, pool, table, n = problem(1, 8, 16, [1500], 64, torch.float16, seed=50)
    q[..., 100] = -1.0
    at = int(table[0, 3]) * 64 + 5
    flat = pool.view(-1, 576)
    flat[at, 100] = float("inf")
    rows = torch.arange(1500) != 3 * 64 + 5
    c = rows_of(pool, table, 0, 1500)[rows].double()
    dev = [t.cuda() for t in (q, pool, table, n)]
    got, lse = ada_mla.mla_decode_tree(*dev, max_seq_len=1500, softmax_scale=SCALE, num_splits=num_splits, return_lse=True)
    got = got.double().cpu()
    assert bool(got[..., 100].isnan().all())
    keep = torch.arange(512) != 100
    for i in range(8):
        see = c[:1499 - 7 + i]
        p = torch.softmax(q[0, i].double() @ see.t() * SCALE, 1)
        o, a = p @ see[:, :512], p @ see[:, :512].abs()
        tol = (2.0 ** -11 + 2.0 ** -13) * a + 2.0 ** -25 * see[:, :512].abs().sum(0) + 2.0 ** -11 * o.abs() + 2.0 ** -24 + 2.0 ** -15 * a
        assert bool(((got[0, i] - o).abs() <= tol)[:, keep].all())
    assert ada_mla.mla_get_device_error() == 0


@pytest.mark.parametrize("batch,k,heads", [
    (31, 4, 16), (32, 4, 16), (480, 2, 128), (961, 2, 16), (481, 2, 128), (1030, 3, 32), (35, 32, 128)])
def test_many_row_tiles(batch, k, heads):
    """31 / 32 and 960 / 961 row tiles are where the schedule is made in another way; above
    1024 the plan kernel takes more than one round.  Lengths from zero on, a tree for each
    sequence whose last draft is padding on a row of NaN."""
    g = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, 130, (batch,), generator=g).tolist()
    lens[0], lens[batch // 2], lens[-1] = 900, 0, 700
    q, pool, table, n = problem(batch, k, heads, lens, 32, torch.float16, seed=60)
    mask = random_tree(batch, k, seed=61)
    mask[:, -1] = 0
    want = expect(q, pool, table, n, mask, torch.float16)
    flat = pool.view(-1, 576)
    for b, m in enumerate(lens):
        if m > 0:
            flat[int(table[b, (m - 1) // 32]) * 32 + (m - 1) % 32] = float("nan")
    a, la = check(q, pool, table, n, mask, want=want)
    b, lb = check(q, pool, table, n, mask, want=want)
    assert torch.equal(a, b) and torch.equal(la, lb)


def test_a_pool_past_32_bits_of_elements():
    """Pages whose elements and bytes lie beyond 2^31 and 2^32 of the pool's start."""
    rows = 4_200_000 // 64
    q, pool, table, n = problem(2, 5, 16, [500, 130], 64, torch.float16, seed=70)
    want = expect(q, pool, table, n, None, torch.float16)
    big = torch.empty(rows, 64, 576, dtype=torch.float16, device="cuda")
    first = rows - pool.shape[0]
    big[first:] = pool.cuda()
    at = torch.where(table >= 0, table + first, table)
    import ada_mla

    got, lse = ada_mla.mla_decode_tree(q.cuda(), big, at.cuda(), n.cuda(), max_seq_len=500, softmax_scale=SCALE, return_lse=True)
    assert bool(((got.double().cpu() - want[0]).abs() <= want[2]).all())
    assert bool(((lse.double().cpu() - want[1]).abs() <= LSE_TOL).all())
    assert ada_mla.mla_get_device_error() == 0
