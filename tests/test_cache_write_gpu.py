"""Latent rows into the cache (mla_cache_write) against the formula in 64 bits.

Bound of one element: the one rounding to the cache's type (u = 2^-11 fp16, 2^-8
bf16, 2^-4 e4m3, and half a spacing of the subnormal numbers: 2^-25, 0, 2^-10), and
fp32 arithmetic before it: a 512-term sum of squares, a reciprocal root and three
products, together below 2^-18 relative; the rotation's two products cancel, so there
it is 2^-18 of |a| + |b|.  e4m3: of the value over its scale, the scale itself to 2^-18."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float16: (2.0 ** -11, 2.0 ** -25), torch.bfloat16: (2.0 ** -8, 0.0), torch.float8_e4m3fn: (2.0 ** -4, 2.0 ** -10)}
FP32 = 2.0 ** -18


def table(n, dtype=torch.float64):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    return torch.cat([a.cos(), a.sin()], 1).to(torch.float32)


def formula(x, w, eps, pos, cs, interleaved):
    """Rows in 64 bits, and for each value the size that its fp32 error goes by."""
    x = x.double()
    c, r = x[:, :512], x[:, 512:]
    if w is not None:
        c = c / torch.sqrt((c * c).mean(1, keepdim=True) + eps) * w.double()
    size = r.abs()
    if pos is not None:
        t = cs.double()[pos.long()]
        cos, sin = t[:, :32], t[:, 32:]
        a, b = (r[:, 0::2], r[:, 1::2]) if interleaved else (r[:, :32], r[:, 32:])
        y = [a * cos - b * sin, a * sin + b * cos]
        both = a.abs() + b.abs()
        r = torch.stack(y, 2).flatten(1) if interleaved else torch.cat(y, 1)
        size = torch.stack([both, both], 2).flatten(1) if interleaved else torch.cat([both, both], 1)
    return torch.cat([c, r], 1), torch.cat([c.abs(), size], 1)


@pytest.mark.parametrize("src", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dst", [torch.float16, torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("tokens,offset,norm,rope,interleaved", [
    (1, 0, True, True, True), (7, 64, True, True, False), (300, 1, True, True, True),  # 1: rows off 16 bytes
    (65, 3, True, False, True), (129, 0, False, True, False), (40, 64, False, False, True)])
def test_against_formula(src, dst, tokens, offset, norm, rope, interleaved):
    import ada_mla

    g = torch.Generator().manual_seed(tokens)
    wide = torch.randn(tokens, 576 + offset, generator=g).to(src).cuda()
    latent = wide[:, offset:]
    rows = tokens + 50
    slots = torch.randperm(rows, generator=g)[:tokens]
    slots[tokens // 2:tokens // 2 + 1] = -1 if tokens > 1 else 0
    pos = torch.randint(0, 500, (tokens,), generator=g).to(torch.int32) if rope else None
    cs = table(500) if rope else None
    w = (1 + 0.2 * torch.randn(512, generator=g)).to(src) if norm else None
    cache = torch.zeros(rows, 576).to(dst).cuda()
    scales = torch.full((rows,), -1.0, device="cuda") if dst == torch.float8_e4m3fn else None
    cuda = lambda t: None if t is None else t.cuda()  # noqa: E731
    ada_mla.mla_cache_write(latent, slots.cuda(), cache, norm_weight=cuda(w), eps=1e-5, positions=cuda(pos), cos_sin=cuda(cs),
                            interleaved=interleaved, kv_scales=scales)
    got = cache.cpu().double()
    want, size = formula(latent.cpu(), w, 1e-5, pos, cs, interleaved)
    real = slots >= 0
    u, sub = U[dst]
    s = torch.ones(tokens, 1, dtype=torch.float64)
    if scales is not None:
        s = (want.abs().amax(1) / 448)[:, None]
        sc = scales.cpu().double()
        assert bool(((sc[slots[real]] - s[real, 0]).abs() <= FP32 * 2 * s[real, 0]).all())
        left = torch.ones(rows, dtype=torch.bool)
        left[slots[real]] = False
        assert bool((sc[left] == -1).all())
    diff = (got[slots[real]] - want[real] / s[real]).abs()
    tol = u * want[real].abs() / s[real] + sub + 4 * FP32 * size[real] / s[real]
    assert bool((diff <= tol).all()), float((diff / tol).max())
    untouched = torch.ones(rows, dtype=torch.bool)
    untouched[slots[real]] = False
    assert bool((got[untouched] == 0).all())


def test_rows_that_are_not_written():
    import ada_mla

    x = torch.randn(6, 576, device="cuda").half()
    slots = torch.tensor([0, 1, 99, -1, 1 << 40, 2], device="cuda")
    pos = torch.tensor([0, 9, 0, 0, 0, -1], dtype=torch.int32, device="cuda")  # the table has 5 positions
    cache = torch.full((4, 576), 7.0, device="cuda").half()
    ada_mla.mla_cache_write(x, slots, cache, positions=pos, cos_sin=table(5).cuda())
    assert bool((cache[0] == x[0]).all()) and bool((cache[1:] == 7).all())


def test_e4m3_zeros_and_tiny_rows():
    import ada_mla

    x = torch.zeros(3, 576, device="cuda")
    x[1, 5] = 1e-38
    x[2, 575] = -3e4
    cache = torch.ones(3, 576, device="cuda").to(torch.float8_e4m3fn)
    scales = torch.zeros(3, device="cuda")
    ada_mla.mla_cache_write(x, torch.arange(3, device="cuda"), cache, kv_scales=scales)
    c, s = cache.float().cpu(), scales.cpu()
    assert float(s[0]) == 1.0 and bool((c[0] == 0).all())
    assert float(s[1]) >= 1.17549435e-38 and bool(torch.isfinite(c[1]).all())
    assert float(c[2, 575]) == -448.0 and abs(float(s[2]) - 3e4 / 448) < 1e-4


def test_page_pool_and_large_offsets():
    """A pool of more than 2^31 elements: row offsets pass 32 bits."""
    import ada_mla

    rows = (1 << 31) // 576 + 4096
    pool = torch.zeros(rows // 64, 64, 576, dtype=torch.float16, device="cuda")
    x = torch.randn(3, 576, device="cuda").half()
    last = pool.shape[0] * 64 - 1
    slots = torch.tensor([last, last - 70, 5], device="cuda")
    ada_mla.mla_cache_write(x, slots, pool)
    assert bool((pool.view(-1, 576)[slots] == x).all())
    assert float(pool[:1000].float().abs().sum()) > 0 and float(pool[1000:2000].float().abs().sum()) == 0


def test_refusals():
    import ada_mla

    x, slots = torch.randn(4, 576, device="cuda").half(), torch.arange(4, device="cuda")
    cache = torch.zeros(8, 576, device="cuda").half()
    cs, pos = table(10).cuda(), torch.zeros(4, dtype=torch.int32, device="cuda")
    ok = dict(latent=x, slots=slots, cache=cache, norm_weight=torch.ones(512, device="cuda").half(), positions=pos, cos_sin=cs)
    ada_mla.mla_cache_write(**ok)
    for bad in [dict(latent=x.cpu()), dict(latent=x.double()), dict(latent=x[:, :575]), dict(latent=x.t().contiguous().t()), dict(slots=slots[:3]),
                dict(slots=slots.int()), dict(cache=cache.float()), dict(cache=cache[:, :512]), dict(cache=cache[:, ::2]), dict(norm_weight=cs[0]),
                dict(norm_weight=torch.ones(512, device="cuda")), dict(positions=None), dict(cos_sin=None), dict(positions=pos.long()),
                dict(cos_sin=cs[:, :32]), dict(kv_scales=torch.ones(8, device="cuda")), dict(cache=cache.to(torch.float8_e4m3fn)), dict(eps=-1.0),
                dict(cache=cache.to(torch.float8_e4m3fn), kv_scales=torch.ones(7, device="cuda"))]:
        with pytest.raises(RuntimeError):
            ada_mla.mla_cache_write(**{**ok, **bad})
    ada_mla.mla_cache_write(x[:0], slots[:0], cache)
