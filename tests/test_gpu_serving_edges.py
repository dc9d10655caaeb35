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
