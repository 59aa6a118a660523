"""The tensor-core decode, call after call on inputs in turn: loads come in late and out of
order, sequences of one tile hand Q from issuer to issuer, and every call gives the bits of
that input's first one, which is checked against the definition in 64 bits.

Bound of one output element, with u the unit roundoff of the inputs' type and A = sum_j p_j
|c_j|: the weights are rounded to that type before the second product (u A, and 2^-25 each
for fp16 weights below its normal numbers), split partials once more (u A), the output once
(u |o|, and half a spacing of fp16's subnormal numbers), and fp32 logits and sums stay below
2^-13 A.  An e4m3 cache takes Q* and P in two e4m3 planes instead, 2^-8 of each: Q*'s part
moves a logit by up to 2^-8 of its terms' sizes, so there only equality is checked (parity
has tests of its own)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SCALE = 192.0 ** -0.5
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def inputs(kind, lens, heads, dtype, seed):
    """(call's arguments, packed rows) of one set."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    b, total = len(lens), sum(lens)
    q = torch.randn(b, heads, 576, generator=g, device="cuda").to(dtype)
    rows = torch.randn(total, 576, generator=g, device="cuda").to(dtype)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    if kind == "paged":
        need = [-(-n // 64) for n in lens]
        perm = torch.randperm(sum(need), generator=torch.Generator().manual_seed(seed))
        pool = torch.full((sum(need), 64, 576), float("nan"), dtype=dtype, device="cuda")
        table = torch.full((b, max(max(need), 1)), -1, dtype=torch.int32)
        at = row = 0
        for i, (n, k) in enumerate(zip(lens, need)):
            pages = perm[at:at + k]
            table[i, :k] = pages
            t = torch.arange(n)
            pool.view(-1, 576)[(pages[t // 64] * 64 + t % 64).cuda()] = rows[row:row + n]
            at, row = at + k, row + n
        return (q, pool, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), max(lens)), rows
    if kind == "fp8":
        return (q, rows.to(torch.float8_e4m3fn), cu, max(lens)), rows
    return (q, rows, cu, max(lens)), rows


def decode(kind, args):
    import ada_mla

    if kind == "paged":
        return ada_mla.mla_decode_paged(*args, softmax_scale=SCALE)
    return ada_mla.mla_decode_batched(*args, softmax_scale=SCALE)


@pytest.mark.parametrize("kind,heads,dtype,lens", [
    ("packed", 128, torch.float16, [1 + 95 * i // 399 for i in range(400)]),    # one tile each
    ("packed", 128, torch.float16, [40 + 61 * i % 211 for i in range(300)]),    # one to three tiles
    ("packed", 128, torch.bfloat16, [1000 + 97 * i for i in range(48)]),
    ("packed", 16, torch.float16, [9000]),
    ("paged", 128, torch.float16, [1 + 95 * i // 399 for i in range(400)]),
    ("paged", 128, torch.bfloat16, [1000 + 97 * i for i in range(48)]),
    ("paged", 16, torch.float16, [5000, 33, 700]),
    ("fp8", 128, torch.float16, [1 + 95 * i // 399 for i in range(400)]),
    ("fp8", 128, torch.float16, [1000 + 97 * i for i in range(48)])])
def test_calls_back_to_back(kind, heads, dtype, lens):
    import ada_mla

    sets = [inputs(kind, lens, heads, dtype, 80 + s) for s in range(2)]
    first = []
    for args, rows in sets:
        out = decode(kind, args)
        first.append(out)
        if kind == "fp8":
            continue
        at = 0
        for b, n in enumerate(lens):
            if b % max(1, len(lens) // 24) == 0:
                c = rows[at:at + n].double()
                p = torch.softmax(args[0][b].double() @ c.t() * SCALE, 1)
                o, a, u = p @ c[:, :512], p @ c[:, :512].abs(), U[dtype]
                tol = (2 * u + 2.0 ** -13) * a + u * o.abs() + 2.0 ** -24 + 2.0 ** -25 * c[:, :512].abs().sum(0)
                assert bool(((out[b].double() - o).abs() <= tol).all()), b
            at += n
    for _ in range(15):
        outs = [decode(kind, sets[i % 2][0]) for i in range(40)]
        assert all(torch.equal(o, first[i % 2]) for i, o in enumerate(outs))
    assert ada_mla.mla_get_device_error() == 0
