"""Prompt attention in expanded form (mla_prefill) against the definition in 64 bits.

Bound of one output element, with u the unit roundoff of the inputs' type (2^-11 fp16,
2^-8 bf16), p the softmax row and A = sum_j p_j |v_j|: the weights go into the second
product rounded to that type (u A, and at most 2^-25 each for fp16 weights below its
normal numbers, relative to a largest weight of at least 1), the output is rounded once
(u |o|, and half a spacing of fp16's subnormal numbers), and fp32 logits and sums (192
and Lk terms) stay below 2^-13 A.  LSE: fp32 logits of size below 16: 2^-14."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SCALE = 192.0 ** -0.5
LSE_TOL = 2.0 ** -14


def problem(lens_q, lens_k, heads, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    tq, tk = sum(lens_q), sum(lens_k)
    q = torch.randn(tq, heads, 192, generator=g).to(dtype)
    kv = torch.randn(tk, heads, 256, generator=g).to(dtype)
    return q, kv, torch.randn(tk, 64, generator=g).to(dtype)


def cu(lens):
    return torch.tensor([0] + lens).cumsum(0).to(torch.int32)


def expect(q, kv, rope, lens_q, lens_k, causal, scale=SCALE):
    heads, u = q.shape[1], U[q.dtype]
    q, kv, rope = q.cuda().double(), kv.cuda().double(), rope.cuda().double()
    out = torch.zeros(q.shape[0], heads, 128, dtype=torch.float64, device="cuda")
    lse = torch.full((q.shape[0], heads), float("-inf"), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    q0 = k0 = 0
    for nq, nk in zip(lens_q, lens_k):
        seen = torch.ones(nq, nk, dtype=torch.bool, device="cuda")
        if causal:
            seen = torch.arange(nk, device="cuda") <= torch.arange(nq, device="cuda")[:, None] + nk - nq
        some = seen.any(1)
        for h in range(heads):
            if not bool(some.any()):
                break
            k = torch.cat([kv[k0:k0 + nk, h, :128], rope[k0:k0 + nk]], 1)
            x = (q[q0:q0 + nq, h] @ k.t() * scale).masked_fill(~seen, float("-inf"))[some]
            v = kv[k0:k0 + nk, h, 128:]
            p = torch.softmax(x, 1)
            rows = torch.arange(q0, q0 + nq, device="cuda")[some]
            out[rows, h] = p @ v
            lse[rows, h] = torch.logsumexp(x, 1)
            tol[rows, h] = (u + 2.0 ** -13) * (p @ v.abs()) + u * (p @ v).abs() + 2.0 ** -24 + 2.0 ** -25 * seen[some].double() @ v.abs()
        q0, k0 = q0 + nq, k0 + nk
    return out, lse, tol


def compare(got, lse, want):
    import ada_mla

    assert ada_mla.mla_get_device_error() == 0
    w, wl, tol = want
    diff = (got.double() - w).abs()
    assert bool((diff <= tol).all()), float((diff / tol.clamp(min=1e-30)).max())
    none = torch.isinf(wl)
    assert bool((torch.isneginf(lse) == none).all())
    assert bool(((lse.double() - wl)[~none].abs() <= LSE_TOL).all())


def check(lens_q, lens_k, heads, dtype, causal=True, seed=0, **kw):
    import ada_mla

    q, kv, rope = problem(lens_q, lens_k, heads, dtype, seed)
    dev = [t.cuda() for t in (q, kv, rope)]
    got, lse = ada_mla.mla_prefill(dev[0], dev[1][..., :128], dev[2], dev[1][..., 128:], cu(lens_q).cuda(), cu(lens_k).cuda(),
                                   max_seq_len_q=max(lens_q), max_seq_len_k=max(lens_k), softmax_scale=SCALE, causal=causal, return_lse=True, **kw)
    compare(got, lse, expect(q, kv, rope, lens_q, lens_k, causal))
    return got, lse


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 127, 128, 129, 255, 256, 257, 400, 640, 1000])
def test_one_prompt(n, causal, dtype):
    check([n], [n], 3, dtype, causal, seed=n)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens_q,lens_k,heads", [
    ([1], [1000], 5), ([100], [3000], 2), ([300], [301], 4), ([128, 1, 256], [129, 700, 256], 7), ([7, 0, 300, 20], [90, 50, 300, 20], 3),
    ([513, 31, 256, 700], [513, 1055, 257, 900], 8), ([17] * 40, [17] * 40, 2), ([200, 3], [1600, 128], 128)])
def test_packed_batches_over_longer_keys(lens_q, lens_k, heads, dtype):
    check(lens_q, lens_k, heads, dtype, seed=sum(lens_q))
    check(lens_q, lens_k, heads, dtype, causal=False, seed=sum(lens_q))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens_q,lens_k,heads", [
    ([1], [9000], 1), ([300], [5000], 3), ([256, 17, 130], [4096, 2000, 513], 4), ([40, 300], [0, 6000], 2), ([700, 1], [800, 8191], 1)])
def test_few_queries_over_many_keys(lens_q, lens_k, heads, dtype):
    """Fewer items than SMs: the keys are split and the shares joined."""
    check(lens_q, lens_k, heads, dtype, seed=sum(lens_k))
    check(lens_q, lens_k, heads, dtype, causal=False, seed=sum(lens_k))


def test_rows_without_keys():
    got, lse = check([300, 5], [100, 0], 3, torch.float16)   # the first 200 queries come before every key
    assert bool((got[:200] == 0).all()) and bool((got[300:] == 0).all())
    check([10, 20], [0, 0], 2, torch.bfloat16)
    check([5], [0], 2, torch.bfloat16)
    check([600, 129], [20, 1], 3, torch.bfloat16)


def test_many_items_per_block():
    """Long runs of items through every block: mixed lengths, tails in most of them."""
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(1, 400, (60,), generator=g).tolist()
    check(lens, lens, 24, torch.float16, seed=4)
    check(lens, [n + 5 for n in lens], 24, torch.bfloat16, seed=5)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -65504.0])
def test_neighbours_may_hold_anything(bad):
    """What lies behind a sequence's last key in the packed rows is another request's."""
    import ada_mla

    for lens in ([100, 30, 200], [129, 64, 65], [3, 130, 7]):
        q, kv, rope = problem(lens, lens, 4, torch.float16, 6)
        lo, hi = lens[0], lens[0] + lens[1]
        want = expect(q, kv, rope, lens, lens, True)
        for t in (q, kv, rope):
            t[lo:hi] = bad
        kv2, rope2 = torch.cat([kv, torch.full_like(kv[:200], bad)]), torch.cat([rope, torch.full_like(rope[:200], bad)])
        args = (q.cuda(), kv2.cuda()[..., :128], rope2.cuda(), kv2.cuda()[..., 128:], cu(lens).cuda(), cu(lens).cuda())
        got, lse = ada_mla.mla_prefill(*args, softmax_scale=SCALE, return_lse=True)
        keep = torch.ones(sum(lens), dtype=torch.bool, device="cuda")
        keep[lo:hi] = False
        compare(got[keep], lse[keep], tuple(t[keep] for t in want))


def test_dense_matches_packed_and_strides():
    import ada_mla

    lens = [260] * 3
    got, lse = check(lens, lens, 5, torch.bfloat16, seed=9)
    q, kv, rope = (t.cuda() for t in problem(lens, lens, 5, torch.bfloat16, 9))
    qd, kvd, rd = q.view(3, 260, 5, 192), kv.view(3, 260, 5, 256), rope.view(3, 260, 64)
    a, la = ada_mla.mla_prefill(qd, kvd[..., :128], rd, kvd[..., 128:], softmax_scale=SCALE, return_lse=True)
    assert torch.equal(a.view(-1, 5, 128), got) and torch.equal(la.view(-1, 5), lse)
    # heads outermost, wider rows, a rope key cut out of a latent row
    q2 = torch.empty(5, 780, 200, device="cuda", dtype=q.dtype)[..., 8:].permute(1, 0, 2).copy_(q)
    k2 = torch.empty(5, 780, 128, device="cuda", dtype=q.dtype).permute(1, 0, 2).copy_(kv[..., :128])
    lat = torch.randn(780, 576, device="cuda").to(q.dtype)
    lat[:, 512:] = rope
    b = ada_mla.mla_prefill(q2, k2, lat[:, 512:], kv[..., 128:], cu(lens).cuda(), cu(lens).cuda(), softmax_scale=SCALE)
    assert torch.equal(b, got)


def test_logits_that_grow_along_the_keys():
    """The running maximum rises tile by tile, so O is corrected again and again."""
    import ada_mla

    q, kv, rope = problem([300], [900], 3, torch.float16, 11)
    q[..., 0] = 8.0
    kv[..., 0] = torch.linspace(0, 60, 900)[:, None].half()
    want = expect(q, kv, rope, [300], [900], False)
    got, lse = ada_mla.mla_prefill(q.cuda(), kv.cuda()[..., :128], rope.cuda(), kv.cuda()[..., 128:], cu([300]).cuda(), cu([900]).cuda(),
                                   softmax_scale=SCALE, causal=False, return_lse=True)
    # logits up to 40 carry four times the fp32 error of the bound's into the weights
    assert bool(((got.double() - want[0]).abs() <= 4 * want[2]).all())
    assert float((lse.double() - want[1]).abs().max()) <= 4 * LSE_TOL


def test_same_result_twice_and_on_another_stream():
    import ada_mla

    lens = [300, 700, 20]
    a, la = check(lens, lens, 8, torch.float16, seed=12)
    q, kv, rope = (t.cuda() for t in problem(lens, lens, 8, torch.float16, 12))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b, lb = ada_mla.mla_prefill(q, kv[..., :128], rope, kv[..., 128:], cu(lens).cuda(), cu(lens).cuda(), softmax_scale=SCALE, return_lse=True)
    s.synchronize()
    assert torch.equal(a, b) and torch.equal(la, lb)


def test_matches_the_absorbed_decode():
    """The last token of a prompt, expanded, against the latent decode of that token."""
    import ada_mla
    from ada_mla import absorbed

    g = torch.Generator().manual_seed(13)
    heads, n = 20, 333
    lat = torch.randn(n, 576, generator=g).half()
    w_uk, w_uv = torch.randn(heads, 128, 512, generator=g) / 22.6, torch.randn(heads, 512, 128, generator=g) / 22.6
    q = torch.randn(n, heads, 192, generator=g).half().cuda()
    c = lat[:, :512].cuda()
    kn = torch.einsum("tc,hdc->thd", c.double(), w_uk.half().cuda().double()).half()
    v = torch.einsum("tc,hcd->thd", c.double(), w_uv.half().cuda().double()).half()
    got = ada_mla.mla_prefill(q[None], kn[None], lat[None, :, 512:].cuda(), v[None])[0, -1]
    one = absorbed.mla_decode_absorbed(q[-1:, :, :128].contiguous(), q[-1:, :, 128:].contiguous(), w_uk.half().cuda(), lat[None].cuda(),
                                       w_uv.half().cuda())[0]
    # both within their own roundings of the same value: keys, values, queries and
    # latent outputs rounded to fp16 on one side or the other
    assert float((got.float() - one.float()).abs().max()) <= 16 * 2.0 ** -11


def test_refusals():
    import ada_mla

    q, kv, rope = (t.cuda() for t in problem([70], [70], 4, torch.float16, 14))
    c = cu([70]).cuda()
    ok = dict(query=q, k_nope=kv[..., :128], k_rope=rope, v=kv[..., 128:], cu_seqlens_q=c, cu_seqlens_k=c)
    ada_mla.mla_prefill(**ok)
    odd = torch.zeros(70 * 4 * 128 + 4, device="cuda").half()[4:].view(70, 4, 128)
    for bad in [dict(query=q.float()), dict(query=q.cpu()), dict(query=q[..., :128]), dict(query=q[:, :3]), dict(k_nope=kv), dict(k_nope=odd),
                dict(k_nope=kv[..., :128].bfloat16()), dict(v=kv[:, :2, 128:]), dict(v=kv[:60, :, 128:]), dict(k_rope=rope[:, :32]), dict(k_rope=rope[:69]),
                dict(v=kv[..., 128:].transpose(1, 2).contiguous().transpose(1, 2)), dict(cu_seqlens_k=None), dict(cu_seqlens_q=c.long()),
                dict(cu_seqlens_k=torch.zeros(3, dtype=torch.int32, device="cuda")), dict(softmax_scale=0.0), dict(softmax_scale=float("inf"))]:
        with pytest.raises(RuntimeError):
            ada_mla.mla_prefill(**{**ok, **bad})
    assert ada_mla.mla_prefill(q[:0], kv[:0, :, :128], rope[:0], kv[:0, :, 128:], c[:1], c[:1]).shape == (0, 4, 128)


@pytest.mark.parametrize("lens_q,lens_k,heads", [([300, 20, 513], [300, 700, 600], 64), ([100], [3000], 2), ([0, 0], [40, 7], 3)])
def test_bounds_far_above_the_lengths(lens_q, lens_k, heads):
    """max_seq_len_q / _k are bounds: any that lies above the lengths gives the same bits."""
    import ada_mla

    q, kv, rope = (t.cuda() for t in problem(lens_q, lens_k, heads, torch.float16, 21))

    def call(bq, bk):
        return ada_mla.mla_prefill(q, kv[..., :128], rope, kv[..., 128:], cu(lens_q).cuda(), cu(lens_k).cuda(), max_seq_len_q=bq, max_seq_len_k=bk,
                                   softmax_scale=SCALE, return_lse=True)

    # (bounds at or above all rows are one and the same, so the keys are split alike)
    want, lse = call(sum(lens_q), sum(lens_k))
    compare(want, lse, expect(q, kv, rope, lens_q, lens_k, True))
    for bound in (1 << 20, 2 ** 31 - 128, 2 ** 31 - 127, 2 ** 31 - 1):
        got, l2 = call(bound, bound)
        assert torch.equal(got, want) and torch.equal(l2, lse), bound
    assert ada_mla.mla_get_device_error() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_dense_single_rows_of_longer_sequences(dtype):
    """The last query of each dense sequence (q[:, -1:]), and single keys, are taken where
    they lie; longer slices, whose sequences do not follow one another, are refused."""
    import ada_mla

    batch, n, heads = 5, 300, 6
    q, kv, rope = problem([n] * batch, [n] * batch, heads, dtype, 17)
    dev = [t.cuda() for t in (q, kv, rope)]
    qd, kvd, rd = (t.view(batch, n, *t.shape[1:]) for t in dev)
    got, lse = ada_mla.mla_prefill(qd[:, -1:], kvd[..., :128], rd, kvd[..., 128:], softmax_scale=SCALE, return_lse=True)
    assert got.shape == (batch, 1, heads, 128) and lse.shape == (batch, 1, heads)
    last = torch.arange(1, batch + 1) * n - 1
    compare(got[:, 0], lse[:, 0], expect(q[last], kv, rope, [1] * batch, [n] * batch, True))
    one, l1 = ada_mla.mla_prefill(qd[:, :1], kvd[:, 7:8, :, :128], rd[:, 7:8], kvd[:, 7:8, :, 128:], softmax_scale=SCALE, return_lse=True)
    at = torch.arange(batch) * n
    compare(one[:, 0], l1[:, 0], expect(q[at], kv[at + 7], rope[at + 7], [1] * batch, [1] * batch, True))
    with pytest.raises(RuntimeError):
        ada_mla.mla_prefill(qd[:, -2:], kvd[..., :128], rd, kvd[..., 128:])
    with pytest.raises(RuntimeError):
        ada_mla.mla_prefill(qd[:, -1:], kvd[:, 1:, :, :128], rd[:, 1:], kvd[:, 1:, :, 128:])


def test_a_long_prompt():
    """Up to 133 key tiles an item."""
    check([16500], [16500], 2, torch.bfloat16, seed=22)
    check([700, 9000], [17000, 9001], 1, torch.float16, seed=23)
