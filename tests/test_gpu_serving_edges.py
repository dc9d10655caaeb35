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


def close(q, k, v, seen, scale, dtype, q8):
    """(out, bound) as serving_ref.attend, but with a bound made of what the row sees and weighs alone: hidden keys, and keys
    of next to no weight, do not widen it. Element by element:
      * the output to its type (below bf16's normal numbers half of 2^-133; below float16's of 2^-24);
      * weights and sums: A (the sum of p |v|) times half a step of 16 bits, twice the scores' error and the float32 sums';
      * float16 weights below the normal numbers (q8, float16): at most half a step, 2^-25, of the reference each, on a
        code of at most Q. The reference is at most the largest weight times value scale of the row, which times Q is the
        largest weight times largest |v| of its key;
      * q8: the reference is at least 2^-126 (2^-25 2^-126 448 a key), products of weight and scale below the normal
        numbers are rounded to 2^-149 (half of it times 448)."""
    q, k, v = q.detach().cpu().double(), k.detach().cpu().double(), v.detach().cpu().double()
    T, H, D = q.shape
    G = H // k.shape[1]
    kh, vh = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    hide = ~seen.cpu()[None]
    s = (torch.einsum("thd,lhd->htl", q, kh) * scale).masked_fill(hide, -torch.inf)
    s_abs = (torch.einsum("thd,lhd->htl", q.abs(), kh.abs()) * abs(scale)).masked_fill(hide, 0.0)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m > -torch.inf, m, torch.zeros_like(m))).masked_fill(hide, 0.0)
    l = p.sum(-1, keepdim=True)
    p = torch.where(l > 0, p / l.clamp(min=1e-300), torch.zeros_like(p))
    out = torch.einsum("htl,lhd->thd", p, vh)
    A = torch.einsum("htl,lhd->thd", p, vh.abs())
    # the scores of keys with a weight that counts (2^-160 and more of the largest); of the others nothing is left
    counts = p > 2.0 ** -160
    ds = s_abs.masked_fill(~counts, 0.0).amax(-1) * ((D + 8) * 2.0 ** -23) + 2.0 ** -21
    if q8:
        kmax = kh.abs().amax(-1).T[:, None].expand_as(p).masked_fill(~counts, 0.0).amax(-1)  # (H, T)
        ds = ds + D * 2.0 ** -25 * q.abs().amax(-1).T * kmax * abs(scale) * 2
    n = seen.double().sum(-1)[:, None, None]
    half = S.HALF_STEP[FP if q8 else dtype]
    bound = S.HALF_STEP[dtype] * out.abs() + A * (half + 2 * ds.T[..., None] + (k.shape[0] + 128) * 2.0 ** -23) * 1.01
    if q8 or dtype == FP:
        heaviest = (p * vh.abs().amax(-1).T[:, None]).amax(-1).T[..., None]  # (T, H, 1)
        bound = bound + n * 2.0 ** -25 * heaviest * 1.01
    bound = bound + (2.0 ** -25 if dtype == FP else 2.0 ** -134)
    if q8:
        bound = bound + n * (2.0 ** -142 + 2.0 ** -141)
    return out, bound


def put_value(c, b, pos, codes, scale):
    """The value row of token `pos` of sequence b of an 8-bit cache, and what it then stands for."""
    blk, off = int(c.table[b, pos // c.page]), pos % c.page
    c.dv.view(torch.uint8)[blk, off] = codes.view(torch.uint8).to(DEV)
    c.ds[1][blk, :, off] = scale.to(DEV)
    c.real[1][blk, off] = S.values(codes, scale)


# ---- value scales
@pytest.mark.parametrize("dtype", [I8, E4])
@pytest.mark.parametrize("T", DRAFTS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_tree_hidden_value_scales(dtype, T, D):
    """What the value row of a drafted token holds, an ordinary row or one of 1e30, does not change a bit of the rows that do
    not see it; those that see it are right."""
    H, KV = 8, 2
    lens = [100, 700]
    c = Cache(lens, 16, KV, D, dtype)
    q = torch.randn(2 * T, H, D, generator=gen(5)).to(BF)
    w, see = words(T, "tree", gen(9))
    hidden = T // 2
    see[:, hidden] &= torch.arange(T) % 2 == hidden % 2
    w = [sum(1 << j for j in range(T) if see[i, j]) for i in range(T)]
    w = [x - (1 << 64) if x >> 63 else x for x in w]
    clean = tree(c, q, [T, T], 0.1, w * 2)
    other = torch.randn(KV, D, generator=gen(8))
    for factor in (1.0, 2.0 ** 14, 1e30):
        codes, scale = S.quantise(other, dtype)
        for b in range(2):
            put_value(c, b, lens[b] - T + hidden, codes, scale * factor)
        got = tree(c, q, [T, T], 0.1, w * 2)
        blind = (~see[:, hidden]).repeat(2).to(DEV)
        assert torch.equal(got[blind], clean[blind]), factor
        for b in range(2):
            seen = torch.cat([torch.ones(T, lens[b] - T, dtype=torch.bool), see], 1)
            want, bound = close(q[b * T:b * T + T], c.seq(0, b), c.seq(1, b), seen, 0.1, BF, True)
            check(got[b * T:b * T + T], want, bound, (factor, b))


@pytest.mark.parametrize("dtype", [I8, E4])
@pytest.mark.parametrize("T", [1, 4, 6, 33])
@pytest.mark.parametrize("bits,ratio", [(144, 14), (144, 26), (144, 100), (60, 40), (60, 60), (60, 58), (30, 40), (3, 20)])
def test_value_scales_of_keys_with_little_weight(dtype, T, bits, ratio):
    """One key with values 2^ratio times the others' and a weight of about 2^-bits: the result is the weighted sum, whichever
    of the two wins, wherever the key lies."""
    H, KV, D, lens = 8, 2, 128, [1000, 90, 300]
    scale = 0.125
    c = Cache(lens, 16, KV, D, dtype)
    u = torch.sign(torch.randn(KV, D, generator=gen(3)))
    q = torch.randn(len(lens) * T, KV, H // KV, D, generator=gen(4)) * 0.05 + u[:, None]
    q = q.reshape(-1, H, D).to(BF)
    for b, pos in enumerate((3, 50, 290 - T)):
        blk, off = int(c.table[b, pos // 16]), pos % 16
        codes, s = S.quantise(-u, dtype)  # the score of u on it: -D a scale
        s = s * (bits * 0.6931 / (D * scale))
        c.dk.view(torch.uint8)[blk, off] = codes.view(torch.uint8).to(DEV)
        c.ds[0][blk, :, off] = s.to(DEV)
        c.real[0][blk, off] = S.values(codes, s)
        codes, s = S.quantise(torch.randn(KV, D, generator=gen(6)), dtype)
        put_value(c, b, pos, codes, s * 2.0 ** ratio)
    if T == 1:
        got = decode(c, q.to(DEV), scale)
    else:
        got = tree(c, q, [T] * len(lens), scale, None)
    for b, L in enumerate(lens):
        seen = torch.ones(T, L, dtype=torch.bool).tril(L - T)
        want, bound = close(q[b * T:b * T + T], c.seq(0, b), c.seq(1, b), seen, scale, BF, True)
        check(got[b * T:b * T + T], want, bound, b)


# ---- tiny values
@pytest.mark.parametrize("dtype", [I8, E4])
@pytest.mark.parametrize("T", [1, 4, 6, 33])
@pytest.mark.parametrize("down", [100, 118, 122, 126, 132])
def test_values_next_to_the_smallest_numbers(dtype, T, down):
    """Values of 2^-down: their scales are below float32's normal numbers, what they stand for is not below bf16's."""
    H, KV, D, lens = 8, 2, 128, [300, 2600]
    c = Cache(lens, 16, KV, D, dtype, garbage=False)
    c.ds[1].mul_(2.0 ** -down)
    small = c.ds[1].cpu().double()
    c.real[1] = c.codes[1].float().double() * small.transpose(1, 2).unsqueeze(-1)
    q = torch.randn(len(lens) * T, H, D, generator=gen(4)).to(BF)
    got = decode(c, q.to(DEV), 0.1) if T == 1 else tree(c, q, [T] * len(lens), 0.1, None)
    for b, L in enumerate(lens):
        seen = torch.ones(T, L, dtype=torch.bool).tril(L - T)
        want, bound = close(q[b * T:b * T + T], c.seq(0, b), c.seq(1, b), seen, 0.1, BF, True)
        # the bound tells them from zeros (at 2^-126 and 2600 keys it is a tenth of them)
        assert down > 122 or float(want.abs().max()) > 16 * float(bound.min())
        check(got[b * T:b * T + T], want, bound, b)


def test_prompt_attention_scores_of_minus_infinity():
    """Keys whose scores are -infinity, whole blocks of them and the first ones, have no weight."""
    from vllm_exact import prompt_attn as A
    for D, real in ((64, BF), (128, BF), (128, FP), (256, BF)):
        H, KV, L, gone = 4, 2, 1100, 300
        g = gen(D)
        q = torch.randn(L, H, D, generator=g)
        q[..., 0] = q[..., 0].abs() + 0.5
        q = q.to(real)
        k, v = (torch.randn(L, KV, D, generator=g).to(real) for _ in range(2))
        k[:gone, :, 0] = -float("inf")
        got = A.prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV), cu([L]), cu([L]), 0.1)
        k[:gone, :, 0] = 0
        seen = torch.ones(L, L, dtype=torch.bool).tril()
        seen[:, :gone] = False
        want, bound = S.attend(q, k, v, seen, 0.1, real)
        check(got[gone:], want[gone:], bound[gone:], (D, real))
        k[:gone, :, 0] = -float("inf")
        for lo, hi in ((256, 420), (700, 1100)):  # and with other rows in the tiles
            assert torch.equal(A.prompt_attention(q[lo:hi].to(DEV), k[:hi].to(DEV), v[:hi].to(DEV), cu([hi - lo]), cu([hi]), 0.1)[gone - min(lo, gone):], got[max(lo, gone):hi])


def test_prompt_attention_offsets_that_are_not_followed():
    """Sequences whose offsets leave the arrays, of queries or of keys, or run backwards: their rows are left as they were."""
    from vllm_exact import prompt_attn as A
    H, KV, D = 4, 2, 64
    g = gen(1)
    q = torch.randn(400, H, D, generator=g).to(BF).to(DEV)
    k, v = (torch.randn(500, KV, D, generator=g).to(BF).to(DEV) for _ in range(2))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    alone = A.prompt_attention(q[:100], k[:120], v[:120], cu([100]), cu([120]), 0.1)
    for cq, ck in ((i32(0, 100, 350), i32(0, 120, 501)), (i32(0, 100, 350), i32(0, 120, 2 ** 31 - 1)),
                   (i32(0, 100, 401), i32(0, 120, 400)), (i32(0, 100, 350), i32(0, 120, 100)),
                   (i32(0, 100, 350), i32(0, 120, -(2 ** 31)))):
        out = torch.full_like(q, 7.0)
        A.prompt_attention(q, k, v, cq, ck, 0.1, out=out)
        assert torch.equal(out[:100], alone) and bool((out[100:] == 7.0).all()), (cq, ck)
    out = torch.full_like(q, 7.0)
    A.prompt_attention(q, k, v, i32(0, 100, 350), i32(0, 120, 120), 0.1, out=out)  # no keys: zeros
    assert torch.equal(out[:100], alone) and bool((out[100:350] == 0).all()) and bool((out[350:] == 7.0).all())
    # sequences behind such a one are served
    want = A.prompt_attention(q[100:350], k[200:500], v[200:500], cu([250]), cu([300]), 0.1)
    out = torch.full_like(q, 7.0)
    A.prompt_attention(q, k, v, i32(0, 100, 10 ** 9, 100, 350), i32(0, 120, 120, 200, 500), 0.1, out=out)
    assert torch.equal(out[:100], alone) and torch.equal(out[100:350], want) and bool((out[350:] == 7.0).all())


@pytest.mark.parametrize("dtype", [None, I8, E4])
@pytest.mark.parametrize("T", [2, 6, 33])
def test_tree_scales_that_leave_no_score(dtype, T):
    """A softmax scale of 1e-30, queries of zeros and next to zeros: every key that is seen weighs the same."""
    H, KV, D, lens = 8, 2, 128, [100, 700]
    c = Cache(lens, 16, KV, D, dtype)
    q = torch.randn(2 * T, H, D, generator=gen(5)).to(BF)
    q[0] = 0
    q[1] = q[1] * 1e-38
    q[T] = 0
    got = tree(c, q, [T, T], 1e-30, None)
    for b, L in enumerate(lens):
        seen = torch.ones(T, L, dtype=torch.bool).tril(L - T)
        want, bound = close(q[b * T:b * T + T], c.seq(0, b), c.seq(1, b), seen, 1e-30, BF, dtype is not None)
        check(got[b * T:b * T + T], want, bound, b)


@pytest.mark.parametrize("real", [BF, FP])
@pytest.mark.parametrize("T", DRAFTS + [8])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_tree_infinities_in_the_context(real, T, D):
    """An infinite value that every row sees makes its own element infinite, in every row, and no other; infinities of both
    signs, or one and a NaN, make NaN."""
    H, KV, L = 8, 2, 900
    c = Cache([L, 300], 16, KV, D, None, real=real)
    for pos in (5, 40, 70, 200, 300, 301, 700):  # a score of 0: some weight in 16 bits
        c.dk[int(c.table[0, pos // 16]), pos % 16] = 0
    q = torch.randn(2 * T, H, D, generator=gen(5)).to(real)
    clean = tree(c, q, [T, T], 0.1, None)
    inf = float("inf")

    def put(pos, head, d, x):
        c.dv[int(c.table[0, pos // 16]), pos % 16, head, d] = x

    put(5, 0, 3, inf)
    put(200, 0, 3, inf)
    put(70, 0, 9, -inf)
    put(300, 1, D - 1, inf)
    put(301, 1, D - 1, -inf)
    put(40, 1, 0, -inf)
    put(700, 1, 0, float("nan"))
    got = tree(c, q, [T, T], 0.1, None)
    bad = torch.zeros(2 * T, H, D, dtype=torch.bool, device=DEV)
    bad[:T, :4, 3] = bad[:T, :4, 9] = bad[:T, 4:, D - 1] = bad[:T, 4:, 0] = True
    assert torch.equal(got[~bad], clean[~bad])
    assert bool((got[:T, :4, 3] == inf).all()) and bool((got[:T, :4, 9] == -inf).all())
    assert bool(torch.isnan(got[:T, 4:, D - 1]).all()) and bool(torch.isnan(got[:T, 4:, 0]).all())


# ---- values that are not finite and that a row may not see
@pytest.mark.parametrize("kind", [BF, FP, E4])
@pytest.mark.parametrize("T", DRAFTS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_tree_hidden_values_that_are_not_finite_change_no_bit(kind, T, D):
    """NaN, infinities (16-bit) and NaN codes (e4m3) in a drafted token's values: element by element in the rows that see it,
    not a bit in the others. A row that sees it sees it however small its weight is."""
    H, KV = 8, 2
    lens = [100, 700]
    c = Cache(lens, 16, KV, D, E4 if kind == E4 else None, real=BF if kind == E4 else kind)
    q = torch.randn(2 * T, H, D, generator=gen(5))
    q[..., 1] = q[..., 1].abs() + 4
    q = q.to(BF if kind == E4 else kind)
    w, see = words(T, "tree", gen(9))
    bad = T // 2
    see[:, bad] &= torch.arange(T) % 2 == bad % 2
    w = [sum(1 << j for j in range(T) if see[i, j]) for i in range(T)]
    w = [x - (1 << 64) if x >> 63 else x for x in w]
    for b in range(2):  # a score of about -500: no weight at all in float32
        pos = lens[b] - T + bad
        blk, off = int(c.table[b, pos // 16]), pos % 16
        if kind == E4:
            c.dk.view(torch.uint8)[blk, off, :, 1] = 0xfe  # -448
            c.ds[0][blk, :, off] = 4.0
        else:
            c.dk[blk, off, :, 1] = -2000.0
    clean = tree(c, q, [T, T], 0.1, w * 2)
    for b in range(2):
        pos = lens[b] - T + bad
        blk, off = int(c.table[b, pos // 16]), pos % 16
        if kind == E4:
            c.dv.view(torch.uint8)[blk, off, 0, 3] = 0x7f
            c.dv.view(torch.uint8)[blk, off, 1, D - 1] = 0xff
        else:
            c.dv[blk, off, 0, 3] = float("nan")
            c.dv[blk, off, 1, D - 1] = float("inf")
            c.dv[blk, off, 1, 16] = -float("inf")
    got = tree(c, q, [T, T], 0.1, w * 2)
    hit = torch.zeros(2 * T, H, D, dtype=torch.bool, device=DEV)
    sees = see[:, bad].repeat(2).to(DEV)
    hit[sees, :4, 3] = True
    hit[sees, 4:, D - 1] = True
    if kind != E4:
        hit[sees, 4:, 16] = True
    assert torch.equal(got[~hit], clean[~hit]) and bool(torch.isfinite(clean).all())
    assert bool(torch.isnan(got[sees][:, :4, 3]).all())
    if kind == E4:
        assert bool(torch.isnan(got[sees][:, 4:, D - 1]).all())
    else:
        assert bool((got[sees][:, 4:, D - 1] == float("inf")).all()) and bool((got[sees][:, 4:, 16] == -float("inf")).all())


# ---- further calls that the documentation allows
@pytest.mark.parametrize("dtype", [None, I8, E4])
@pytest.mark.parametrize("T", [3, 6, 33])
def test_tree_pages_that_do_not_exist(dtype, T):
    """Tokens on pages outside the cache are not seen: single pages, a whole block of keys, the first page and the last."""
    H, KV, D, lens = 8, 2, 128, [90, 1200, 640]
    c = Cache(lens, 16, KV, D, dtype)
    q = torch.randn(3 * T, H, D, generator=gen(5)).to(BF)
    gone = {0: [1], 1: [3, 20] + list(range(32, 48)), 2: [0] + [39]}
    for b, pages in gone.items():
        for i, x in enumerate(pages):
            c.dt[b, x] = (-1, c.dk.shape[0], 2 ** 31 - 1, -(2 ** 31))[i % 4]
    got = tree(c, q, [T] * 3, 0.1, None)
    for b, L in enumerate(lens):
        seen = torch.ones(T, L, dtype=torch.bool).tril(L - T)
        for x in gone[b]:
            seen[:, x * 16:(x + 1) * 16] = False
        want, bound = close(q[b * T:b * T + T], c.seq(0, b), c.seq(1, b), seen, 0.1, BF, dtype is not None)
        check(got[b * T:b * T + T], want, bound, b)


@pytest.mark.parametrize("dtype", [None, I8, E4])
@pytest.mark.parametrize("T", [1, 4, 6, 33])
def test_negative_softmax_scales(dtype, T):
    H, KV, D, lens = 8, 2, 64, [90, 700, 2100]
    c = Cache(lens, 16, KV, D, dtype)
    q = torch.randn(3 * T, H, D, generator=gen(5)).to(BF)
    calls = [tree(c, q, [T] * 3, -0.1, None)]
    if dtype is not None and T == 1:
        calls.append(decode(c, q.to(DEV), -0.1))
    for got in calls:
        for b, L in enumerate(lens):
            seen = torch.ones(T, L, dtype=torch.bool).tril(L - T)
            want, bound = close(q[b * T:b * T + T], c.seq(0, b), c.seq(1, b), seen, -0.1, BF, dtype is not None)
            check(got[b * T:b * T + T], want, bound, b)


@pytest.mark.parametrize("dtype", [None, I8, E4])
@pytest.mark.parametrize("T", [1, 4, 6, 33])
@pytest.mark.parametrize("most", [0, 1, 300, 2050])
def test_requests_longer_than_max_seq_len(dtype, T, most):
    """Tokens behind max_seq_len are not seen, the drafted ones among them; the others keep their places."""
    H, KV, D, lens = 8, 2, 128, [90, 700, 2100]
    c = Cache(lens, 16, KV, D, dtype)
    q = torch.randn(3 * T, H, D, generator=gen(5)).to(BF)
    calls = [tree(c, q, [T] * 3, 0.1, None, max_seq_len=most)]
    if dtype is not None and T == 1:
        calls.append(decode(c, q.to(DEV), 0.1, max_seq_len=most))
    for got in calls:
        for b, L in enumerate(lens):
            seen = torch.ones(T, L, dtype=torch.bool).tril(L - T)
            seen[:, most:] = False
            want, bound = close(q[b * T:b * T + T], c.seq(0, b), c.seq(1, b), seen, 0.1, BF, dtype is not None)
            check(got[b * T:b * T + T], want, bound, b)


@pytest.mark.parametrize("dtype", [BF, E4])
@pytest.mark.parametrize("T", [4, 20])
def test_tree_offsets_beyond_32_bits(dtype, T):
    """Caches of more than 2^32 bytes a tensor (and, 8-bit, codes beyond 2^32 elements), a sequence in the last pages."""
    from vllm_exact import paged_attn as P
    KV, D, H, page, L = 8, 256, 32, 16, 1000
    c = Cache([L], page, KV, D, E4 if dtype == E4 else None)
    q = torch.randn(T, H, D, generator=gen(7)).to(BF).to(DEV)
    want = tree(c, q, [T], 0.1, None)
    blocks = 2 ** 32 // (KV * D * page) // (1 if dtype == E4 else 2) + 70
    wide = c.dt.shape[1]
    to = torch.arange(blocks - wide, blocks, device=DEV)
    big = []
    for x in (c.dk, c.dv):
        y = torch.zeros(blocks, page, KV, D, dtype=torch.uint8 if dtype == E4 else BF, device=DEV)
        y[to] = (x.view(torch.uint8) if dtype == E4 else x)[c.dt[0].long()]
        big.append(y.view(E4) if dtype == E4 else y)
    scales = [None, None]
    if dtype == E4:
        for i, s in enumerate(c.ds):
            scales[i] = torch.zeros(blocks, KV, page, device=DEV)
            scales[i][to] = s[c.dt[0].long()]
    out = torch.empty_like(q)
    P.tree_attention(q, *big, to.view(1, -1).to(torch.int32), c.dl, cu([T]), 0.1, out, T, key_scale=scales[0], value_scale=scales[1])
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [None, E4])
@pytest.mark.parametrize("T", [4, 6, 33])
def test_tree_lengths_around_the_segments(dtype, T):
    """Requests as long as the lengths at which the segments change, one shorter and one longer; each has its bits alone."""
    from vllm_exact import paged_attn as P
    H, KV, D = 4, 1, 64
    lens = [x + d for x in (512, 2048, 8192, 10000, 16384) for d in (-1, 0, 1)]
    c = Cache(lens, 16, KV, D, dtype)
    q = torch.randn(len(lens) * T, H, D, generator=gen(5)).to(BF)
    got = tree(c, q, [T] * len(lens), 0.1, None)
    for b, L in enumerate(lens):
        seen = torch.ones(T, L, dtype=torch.bool).tril(L - T)
        want, bound = close(q[b * T:b * T + T], c.seq(0, b), c.seq(1, b), seen, 0.1, BF, dtype is not None)
        check(got[b * T:b * T + T], want, bound, L)
        one = torch.empty(T, H, D, dtype=BF, device=DEV)
        P.tree_attention(q[b * T:b * T + T].to(DEV), c.dk, c.dv, c.dt[b:b + 1], c.dl[b:b + 1], cu([T]), 0.1, one, T,
                         key_scale=c.ds[0], value_scale=c.ds[1], max_seq_len=L)
        assert torch.equal(one, got[b * T:b * T + T]), L


@pytest.mark.parametrize("kind", [BF, E4])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_tree_notes_of_many_items_in_turn(kind, D):
    """Thirty short requests a CTA, every third with a value that is not finite: no request hears of another's, however many
    items lie between."""
    from vllm_exact import paged_attn as P
    H, KV, T, lens = 16, 1, 2, [20, 20]
    c = Cache(lens, 16, KV, D, E4 if kind == E4 else None)
    q = torch.randn(T, H, D, generator=gen(21)).to(BF).to(DEV)
    for x in (c.dk, c.dv, *c.ds):  # the same keys and values in both sequences
        if x is not None:
            y = x.view(torch.uint8) if x.element_size() == 1 else x
            y[c.dt[1].long()] = y[c.dt[0].long()]
    blk = int(c.table[1, 0])
    if kind == E4:
        c.dv.view(torch.uint8)[blk, 3, 0, 5] = 0x7f
    else:
        c.dv[blk, 3, 0, 5] = float("inf")
    n = 30 * torch.cuda.get_device_properties(0).multi_processor_count
    bad = torch.arange(n, device=DEV) % 3 == 0
    table = c.dt[bad.long()].contiguous()
    out = torch.empty(n * T, H, D, dtype=BF, device=DEV)
    P.tree_attention(q.repeat(n, 1, 1), c.dk, c.dv, table, torch.full((n,), 20, dtype=torch.int32, device=DEV), cu([T] * n), 0.1, out, T,
                     key_scale=c.ds[0], value_scale=c.ds[1])
    out = out.view(n, T, H, D)
    assert torch.equal(out[~bad], out[1].expand(n, T, H, D)[~bad]) and bool(torch.isfinite(out[1]).all())
    assert torch.equal(torch.isfinite(out[bad]), (torch.arange(D, device=DEV) != 5).expand(n, T, H, D)[bad])
