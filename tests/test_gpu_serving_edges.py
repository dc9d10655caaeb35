"""GPU tests of the serving operators where they can go wrong: tiles without boxes, values that must not matter, values that
are not finite in places that are seen and in places that are not."""
import pytest
import torch

import serving_ref as S
from test_gpu_serving import BF, DEV, E4, FP, I8, Cache, check, cu, decode, gen, tree, tree_check, words  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    yield
    from vllm_exact import _lib
    assert _lib.device_error() == 0


@pytest.mark.parametrize("dtype", [None, I8, E4])
@pytest.mark.parametrize("H,KV,D", [(8, 2, 64), (8, 1, 128), (4, 1, 256)])
def test_tree_many_tiles_of_one_box(dtype, H, KV, D):
    """Requests of a few keys, and requests whose last block is a few keys: most producer warps have no box in such tiles."""
    T = [17, 20, 17, 30] * 40
    lens = [max(t, x) for t, x in zip(T, [17, 129, 257, 30, 130, 520, 22, 1025] * 20)]
    c = Cache(lens, 16, KV, D, dtype, seed=D)
    q = torch.randn(sum(T), H, D, generator=gen(1)).to(BF)
    made = [words(t, "chain", None) for t in T]
    got = tree(c, q, T, D ** -0.5, None)
    tree_check(c, q, T, [s for _, s in made], got, D ** -0.5, BF)


# rows a KV head: 8 and 16 are the few-row kernel's, 24 and 64 stand in the tile in copies, 68 and 132 do not
DRAFTS = [2, 4, 6, 16, 17, 33]


# ---- value rows that are not finite
@pytest.mark.parametrize("dtype", [I8, E4])
@pytest.mark.parametrize("T", DRAFTS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_tree_value_rows_written_from_numbers_that_are_not_finite(dtype, T, D, bad):
    """All value rows of one head of a request, and those of a last block that begins with the drafted tokens, were written
    from infinities or NaN: every row that sees one is NaN there, the other head and request keep their bits."""
    from vllm_exact import kv_cache as C
    H, KV = 8, 2
    lens = [100, 128 + T, 1000, 100]
    c = Cache(lens, 16, KV, D, dtype)
    q = torch.randn(len(lens) * T, H, D, generator=gen(5)).to(BF)
    clean = tree(c, q, [T] * 4, 0.1, None)
    for b, lo in ((0, 0), (1, 128), (2, 0)):
        pos = torch.arange(lo, lens[b])
        slots = c.table[b].long()[pos // 16] * 16 + pos % 16
        x = torch.randn(len(pos), KV, D, generator=gen(7)).to(BF).to(DEV)
        v = c.seq(1, b)[lo:].float().to(BF).to(DEV)
        v[:, 1, 3] = bad
        keep = [t.clone() for t in (c.dk, c.ds[0])]
        before = [c.dv.clone(), c.ds[1].clone()]
        C.cache_write(x, v, c.dk, c.dv, *c.ds, slots.to(DEV))
        c.dk.copy_(keep[0])
        c.ds[0].copy_(keep[1])
        blk, off = c.table[b].long()[pos // 16].to(DEV), (pos % 16).to(DEV)
        c.dv.view(torch.uint8)[blk, off, 0] = before[0].view(torch.uint8)[blk, off, 0]  # head 0 as it was
        c.ds[1][blk, 0, off] = before[1][blk, 0, off]
    got = tree(c, q, [T] * 4, 0.1, None)
    assert bool(torch.isnan(got[:3 * T, 4:]).all())
    assert torch.equal(got[:, :4], clean[:, :4]) and torch.equal(got[3 * T:], clean[3 * T:])
