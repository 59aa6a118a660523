"""Host-side checks, without a GPU, of the entry points around the paged cache:
arguments refused before any launch, workspace sizes, tree masks from parents."""
import pytest
import torch

import ada_mla
from ada_mla import capi


def test_tree_mask_from_parents():
    assert ada_mla.tree_mask([-1, 0, 0, 1, -1]).tolist() == [1, 3, 5, 11, 16]
    chain = ada_mla.tree_mask(torch.arange(64) - 1)
    assert chain[62].item() == (1 << 63) - 1 and chain[63].item() == -1
    assert ada_mla.tree_mask([[-1, -1], [-1, 0]]).tolist() == [[1, 2], [1, 3]]
    for bad in ([0], [-2], [-1, 1], [], list(range(-1, 64))):
        with pytest.raises(ValueError):
            ada_mla.tree_mask(bad)


def tree(**kw):
    a = dict(q=16, kv=16, bt=16, sl=16, mask=16, shared=0, batch=1, drafts=4, heads=16, pages=4, page=64, blocks=4, longest=64, scale=1.0,
             splits=0, out=32, dtype=capi.OUT_F16, lse=None, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return capi.lib().mla_b200_decode_tree_f16(*a.values())


def test_tree_arguments():
    for bad in [dict(q=None), dict(kv=None), dict(bt=None), dict(sl=None), dict(out=None), dict(out=16), dict(q=18), dict(kv=24), dict(mask=12), dict(lse=2),
                dict(batch=-1), dict(drafts=0), dict(heads=0), dict(page=0), dict(longest=-1), dict(longest=257), dict(scale=0.0),
                dict(scale=float("inf")), dict(dtype=capi.OUT_BF16), dict(dtype=9)]:
        assert tree(**bad) == capi.ERR_INVALID_ARG, bad
    for bad in [dict(drafts=65), dict(heads=129), dict(page=48, longest=0), dict(pages=1 << 30, page=64), dict(batch=70000)]:
        assert tree(**bad) == capi.ERR_UNSUPPORTED, bad
    if not torch.cuda.is_available():
        assert tree() == capi.ERR_NO_DEVICE


def test_tree_workspace():
    size = capi.lib().mla_b200_workspace_size_tree
    assert size(2, 8, 16, 1000, -1) >= capi.workspace_size(2, 128, 2000, 1000, -1)
    assert size(2, 9, 16, 1000, -1) >= capi.workspace_size(4, 80, 4000, 1000, -1)  # 9 drafts: tiles of 5 and 4
    assert size(-1, 8, 16, 10, -1) == 0 and size(70000, 1, 16, 10, -1) == 0


def test_slots_arguments():
    def call(**kw):
        a = dict(lens=16, new=16, table=16, stride=8, blocks=8, free=16, nfree=4, head=None, batch=2, page=64, tokens=2, slots=16, pos=16,
                 cu=16, out=16, nhead=16, stream=None)
        a.update(kw)
        return capi.lib().mla_b200_build_slots(*a.values())

    for bad in [dict(lens=None), dict(new=None), dict(table=None), dict(stride=7), dict(free=None), dict(batch=-1), dict(page=0),
                dict(tokens=-1), dict(slots=None), dict(pos=None), dict(cu=None), dict(out=None), dict(nhead=None), dict(slots=12),
                dict(lens=18), dict(head=2), dict(nfree=-1), dict(blocks=-1)]:
        assert call(**bad) == capi.ERR_INVALID_ARG, bad
    if not torch.cuda.is_available():
        assert call() == capi.ERR_NO_DEVICE


def test_write_arguments():
    def call(**kw):
        a = dict(latent=16, dtype=0, stride=576, slots=16, tokens=2, w=16, eps=1e-6, pos=16, cs=16, maxpos=8, inter=1, cache=16, cdtype=0,
                 rows=10, scales=None, stream=None)
        a.update(kw)
        return capi.lib().mla_b200_cache_write(*a.values())

    for bad in [dict(latent=None), dict(dtype=3), dict(dtype=7), dict(stride=-1), dict(slots=None), dict(tokens=-1), dict(eps=-1.0),
                dict(eps=float("nan")), dict(pos=None), dict(cs=None), dict(maxpos=-1), dict(cache=None), dict(cache=24), dict(cdtype=1),
                dict(cdtype=3), dict(scales=16), dict(rows=-1), dict(latent=17), dict(slots=12), dict(w=17)]:
        assert call(**bad) == capi.ERR_INVALID_ARG, bad
    if not torch.cuda.is_available():
        assert call() == capi.ERR_NO_DEVICE


def test_prefill_arguments():
    def call(**kw):
        a = dict(q=16, qs=768, qh=192, k=16, ks=1024, kh=256, r=16, rs=64, v=16, vs=1024, vh=256, cuq=16, cuk=16, batch=2, heads=4, tq=100, tk=100,
                 mq=64, mk=64, causal=1, scale=1.0, out=32, lse=None, ws=16, ws_bytes=1 << 20, stream=None)
        a.update(kw)
        return capi.lib().mla_b200_prefill_f16(*a.values())

    for bad in [dict(q=None), dict(k=None), dict(r=None), dict(v=None), dict(out=None), dict(out=16), dict(q=24), dict(qs=764), dict(kh=4), dict(rs=60),
                dict(vs=-8), dict(cuq=None), dict(cuk=None), dict(cuq=None, cuk=None), dict(batch=-1), dict(heads=0), dict(tq=-1), dict(tk=-1),
                dict(mq=-1), dict(mk=-1), dict(scale=0.0), dict(scale=float("nan")), dict(lse=2)]:
        assert call(**bad) == capi.ERR_INVALID_ARG, bad
    assert call(tq=1 << 31) == capi.ERR_UNSUPPORTED and call(tk=1 << 31) == capi.ERR_UNSUPPORTED
    if not torch.cuda.is_available():
        assert call() == capi.ERR_NO_DEVICE
    size = capi.lib().mla_b200_workspace_size_prefill
    assert size(3, 128, 1000, 500, 500) >= 8 * (1000 // 256 + 3) and size(-1, 8, 5, 5, 5) == 0
    assert size(1, 2, 100, 100, 8192) >= 16 * 100 * 2 * 129 * 4  # 2 items: the keys are split


def test_tree_workspace_does_not_grow_with_the_tiles():
    """Two partial slots a cluster hold whatever the automatic schedule splits; only the
    schedule's tables grow."""
    size = capi.lib().mla_b200_workspace_size_tree
    slots = 148 * 128 * (512 + 1) * 4  # 148 SMs, 128 rows
    for batch, drafts in ((1, 4), (256, 8), (2000, 32), (65535, 1)):
        tiles = batch * drafts  # 128 heads: a tile a draft
        assert size(batch, drafts, 128, 32767, -1) <= slots + 64 * (tiles + 148) + 4096, (batch, drafts)


@pytest.mark.parametrize("seed", range(30))
def test_partial_slots_of_the_balanced_schedule(seed):
    """The schedule's items, as its workers walk them: those of split tiles have slots of
    their own below two a worker (part_slot in csrc/mla_tree.cuh)."""
    import random

    rng = random.Random(seed)
    workers, cost = rng.choice((1, 2, 13, 74)), rng.randrange(1, 5)
    tiles = [rng.choice((0, 1, 2, rng.randrange(0, 300))) for _ in range(rng.choice((1, 3, 31, 200, 1100)))]
    base, total = [], 0
    for n in tiles:
        base.append(total + cost)
        total += n + cost if n > 0 else 0
    quota = max(1, -(-total // workers))
    taken = set()
    for v, n in enumerate(tiles):
        if n == 0:
            continue
        first, last = base[v] // quota, (base[v] + n - 1) // quota
        if first == last:
            continue
        for s, w in enumerate(range(first, last + 1)):
            ident = v + w
            slot = ident - v + (workers if s == 0 else 0)
            assert 0 <= slot < 2 * workers and slot not in taken
            taken.add(slot)
