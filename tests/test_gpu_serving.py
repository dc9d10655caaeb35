"""GPU tests of the 8-bit paged cache (write, read, decode), draft-tree attention and packed prompt attention: against
64-bit implementations within bounds that count the roundings, bitwise invariance, and the calls that can go wrong."""
import itertools

import pytest
import torch

import serving_ref as S

pytestmark = pytest.mark.gpu
DEV = "cuda"
I8, E4 = torch.int8, torch.float8_e4m3fn
BF, FP = torch.bfloat16, torch.float16
HEADS = [(32, 8, 128), (16, 4, 256), (8, 1, 64), (6, 6, 128), (16, 1, 128), (12, 4, 64)]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    yield
    from vllm_exact import _lib
    assert _lib.device_error() == 0


def gen(seed):
    return torch.Generator().manual_seed(seed)


def cu(v):
    return torch.tensor([0] + list(itertools.accumulate(v)), dtype=torch.int32, device=DEV)


class Cache:
    """A paged cache with sequences of the given lengths in random pages; places of no sequence hold garbage."""

    def __init__(self, lens, page, KV, D, dtype, real=BF, seed=0, spare=3, garbage=True):
        g = gen(seed)
        wide = max(1, max((-(-x // page) for x in lens), default=1))
        n = len(lens)
        blocks = n * wide + spare
        self.lens, self.page, self.dtype = lens, page, dtype
        self.table = torch.randperm(blocks, generator=g)[:n * wide].view(n, wide).to(torch.int32)
        self.kv = [(torch.randn(blocks, page, KV, D, generator=g) * torch.where(torch.rand(KV, D, generator=g) < 0.03, 8.0, 1.0)).to(real) for _ in range(2)]
        used = torch.zeros(blocks, page, dtype=torch.bool)
        for b, x in enumerate(lens):
            for i in range(0, x, page):
                used[self.table[b, i // page], :min(page, x - i)] = True
        self.scales = None
        if dtype in S.QMAX:
            q = [S.quantise(x, dtype) for x in self.kv]
            self.real = [S.values(*x) for x in q]
            self.codes = [x[0].clone() for x in q]
            self.scales = [x[1].transpose(1, 2).contiguous() for x in q]
            if garbage:
                for c, s in zip(self.codes, self.scales):
                    c.view(torch.uint8)[~used] = 0x7f
                    s.transpose(1, 2)[~used] = float("nan")
        else:
            self.real = [x.double() for x in self.kv]
            self.codes = [x.clone() for x in self.kv]
            if garbage:
                for c in self.codes:
                    c[~used] = float("nan")
        self.to()

    def to(self):
        self.dt = self.table.to(DEV)
        self.dk, self.dv = (c.to(DEV) for c in self.codes)
        self.ds = [s.to(DEV) for s in self.scales] if self.scales else [None, None]
        self.dl = torch.tensor(self.lens, dtype=torch.int32, device=DEV)

    def seq(self, which, b):
        x = self.real[which][self.table[b].long()]
        return x.reshape(-1, *x.shape[2:])[:self.lens[b]]


def decode(c, q, scale, n=None, **kw):
    from vllm_exact import paged_attn as P
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device=DEV)
    n = len(c.lens) if n is None else n
    P.paged_decode_q8(q, c.dk, c.dv, *c.ds, c.dt, c.dl, scale, out, n, **kw)
    return out


def check(got, want, bound, what=""):
    got = got.detach().cpu().double()
    off = (got - want).abs()
    assert torch.isfinite(got).all(), what
    assert bool((off <= bound).all()), (what, float((off / bound).max()))


# ------------------------------------------------------------------------------------------------------------ cache
@pytest.mark.parametrize("dtype", [I8, E4])
@pytest.mark.parametrize("real", [BF, FP])
@pytest.mark.parametrize("T,KV,D,page", [(1, 8, 128, 16), (37, 4, 256, 528), (130, 1, 64, 24), (5, 6, 128, 1), (64, 3, 64, 7)])
def test_cache_write_is_the_rounded_formula(dtype, real, T, KV, D, page):
    from vllm_exact import kv_cache as C
    g = gen(T + D)
    x = torch.randn(T, 2, KV, D, generator=g)
    x[:, :, :, 3] *= 40
    if T > 4:
        x[0] = 0.0
        x[1, 0] = 1e-7 if real == FP else 1e-39
        x[2, 1, 0, 5] = float("inf")
        x[3, 0, 0, 1] = float("nan")
        x[4] = torch.round(x[4] * 4) * 0.5  # ties of the rounding
    x = x.to(real).to(DEV)
    blocks = -(-T // page) + 2
    kc, vc, ks, vs = C.alloc_q8_cache(blocks, page, KV, D, dtype, DEV)
    for t in (kc, vc):
        t.view(torch.uint8).fill_(0x55)
    ks.fill_(3.0)
    vs.fill_(3.0)
    slots = torch.randperm(blocks * page, generator=g)[:T]
    if T > 8:
        slots[6], slots[7], slots[8] = -1, blocks * page, -(2 ** 40)
    ko, vo = (torch.empty(T, KV, D, dtype=real, device=DEV) for _ in range(2))
    C.cache_write(x[:, 0], x[:, 1], kc, vc, ks, vs, slots.to(DEV), key_out=ko, value_out=vo)
    for i, (codes, scale, back) in enumerate(((kc, ks, ko), (vc, vs, vo))):
        q, s = S.quantise(x[:, i], dtype)
        want_c = torch.full((blocks * page, KV, D), 0x55, dtype=torch.uint8)
        want_s = torch.full((blocks * page, KV), 3.0)
        for t, w in enumerate(slots.tolist()):
            if 0 <= w < blocks * page:
                want_c[w], want_s[w] = q.view(torch.uint8)[t], s[t]
        got_c, got_s = codes.view(torch.uint8).cpu().view(-1, KV, D), scale.cpu().transpose(1, 2).reshape(-1, KV)
        # a negative zero code of e4m3 stands for the same number
        assert torch.equal(got_c.view(dtype).float(), want_c.view(dtype).float()) or torch.equal(got_c, want_c)
        assert torch.equal(got_s.view(torch.int32)[torch.isfinite(want_s)], want_s.view(torch.int32)[torch.isfinite(want_s)])
        assert torch.equal(torch.isnan(got_s), torch.isnan(want_s)) and torch.equal(torch.isinf(got_s), torch.isinf(want_s))
        want_b = (q.float() * s.unsqueeze(-1)).to(real)
        assert torch.equal(torch.nan_to_num(back.cpu().float(), nan=-1.5), torch.nan_to_num(want_b.float(), nan=-1.5))


@pytest.mark.parametrize("dtype", [I8, E4])
@pytest.mark.parametrize("real", [BF, FP])
def test_cache_write_quotients_are_those_of_the_division(dtype, real):
    """Rows of every magnitude (scales down to the subnormal numbers, where the quotient is taken another way), values
    over 2^14 below the largest, short mantissas among them, so that quotients lie on ties and next to them."""
    from vllm_exact import kv_cache as C
    g = gen(5)
    T, KV, D, page = 700, 6, 128, 16
    lo, hi = (-133, 127) if real == BF else (-24, 15)
    e = torch.randint(lo, hi + 1, (T, 2, KV, 1), generator=g) - torch.randint(0, 15, (T, 2, KV, D), generator=g)
    m = 1 + torch.randint(0, 256, (T, 2, KV, D), generator=g) / 256.0
    m = torch.where(torch.rand(T, 2, KV, D, generator=g) < 0.3, 1 + torch.randint(0, 8, m.shape, generator=g) / 8.0, m)
    x = (torch.ldexp(m.double(), e) * torch.where(torch.rand(m.shape, generator=g) < 0.5, -1.0, 1.0)).to(real)
    assert bool(torch.isfinite(x).all()) and int((x != 0).sum()) > x.numel() // 2
    kc, vc, ks, vs = C.alloc_q8_cache(T // page + 1, page, KV, D, dtype, DEV)
    x = x.to(DEV)
    C.cache_write(x[:, 0], x[:, 1], kc, vc, ks, vs, torch.arange(T, device=DEV))
    for i, (codes, scale) in enumerate(((kc, ks), (vc, vs))):
        q, s = S.quantise(x[:, i], dtype)
        assert torch.equal(codes.cpu().view(-1, KV, D)[:T].float(), q.float())
        assert torch.equal(scale.cpu().transpose(1, 2).reshape(-1, KV)[:T], s)


def test_cache_write_without_values_and_empty():
    from vllm_exact import kv_cache as C
    kc, vc, ks, vs = C.alloc_q8_cache(4, 16, 8, 128, I8, DEV)
    x = torch.randn(9, 8, 128, device=DEV, dtype=BF)
    slots = torch.arange(9, device=DEV) * 3
    C.cache_write(x, -x, kc, vc, ks, vs, slots)
    assert torch.equal(kc, -vc) and torch.equal(ks, vs) and int(kc.abs().max()) == 127
    before = kc.clone()
    C.cache_write(x[:0], x[:0], kc, vc, ks, vs, slots[:0])
    assert torch.equal(kc, before)


@pytest.mark.parametrize("dtype,real", [(I8, BF), (E4, FP), (E4, BF)])
@pytest.mark.parametrize("KV,D,page", [(8, 128, 16), (4, 256, 528), (1, 64, 24), (3, 128, 5)])
def test_cache_read(dtype, real, KV, D, page):
    from vllm_exact import kv_cache as C
    lens = [0, 1, 77, page, 0, page + 1, 130, 0]
    c = Cache(lens, page, KV, D, dtype, seed=page)
    total = sum(lens)
    ko, vo = (torch.full((total + 9, KV, D), 7.0, dtype=real, device=DEV) for _ in range(2))
    C.cache_read(c.dk, c.dv, *c.ds, c.dt, cu(lens), ko, vo)
    for i, got in enumerate((ko, vo)):
        want = torch.cat([c.seq(i, b) for b in range(len(lens))]).float().to(real)
        assert torch.equal(got[:total].cpu(), want)
        assert bool((got[total:] == 7.0).all())


def test_cache_read_many_sequences_and_bad_pages():
    """1500 sequences (three steps of the search for a row's sequence), then pages that the cache does not have."""
    from vllm_exact import kv_cache as C
    lens = [(i * 7) % 5 for i in range(1500)]
    c = Cache(lens, 8, 1, 64, I8)
    ko, vo = (torch.full((sum(lens), 1, 64), 7.0, dtype=BF, device=DEV) for _ in range(2))
    C.cache_read(c.dk, c.dv, *c.ds, c.dt, cu(lens), ko, vo)
    want = torch.cat([c.seq(1, b) for b in range(len(lens))]).float().to(BF)
    assert torch.equal(vo.cpu(), want)
    bad = c.dt.clone()
    bad[1], bad[2] = -1, 10 ** 8
    ko.fill_(7.0)
    C.cache_read(c.dk, c.dv, *c.ds, bad, cu(lens), ko, vo)
    gone = lens[0] + lens[1] + lens[2]
    assert bool((ko[:gone] == 7.0).all()) and not bool((ko[gone:] == 7.0).all())


# ----------------------------------------------------------------------------------------------------------- decode
LENS = [0, 1, 15, 16, 63, 64, 65, 255, 256, 257, 700, 2048, 2049, 4500]


@pytest.mark.parametrize("dtype", [I8, E4])
@pytest.mark.parametrize("H,KV,D", HEADS)
@pytest.mark.parametrize("page,real", [(16, BF), (24, FP), (528, BF)])
def test_decode_q8(dtype, H, KV, D, page, real):
    c = Cache(LENS, page, KV, D, dtype, seed=D + page)
    q = torch.randn(len(LENS), H, D, generator=gen(1)).to(real)
    q[3] *= 30
    q[4] *= 1e-3
    got = decode(c, q.to(DEV), D ** -0.5)
    for b, L in enumerate(LENS):
        want, bound = S.attend(q[b:b + 1], c.seq(0, b), c.seq(1, b), torch.ones(1, L, dtype=torch.bool), D ** -0.5, real, q8=True)
        check(got[b:b + 1], want, bound, L)


@pytest.mark.parametrize("dtype", [I8, E4])
def test_decode_q8_invariance(dtype):
    """A request's bits: alone, in a prefix, in another order, and with its pages elsewhere."""
    H, KV, D, page = 32, 8, 128, 16
    lens = [1000, 5, 2500, 300, 64, 1024, 0, 777]
    c = Cache(lens, page, KV, D, dtype)
    q = torch.randn(len(lens), H, D, generator=gen(2)).to(BF).to(DEV)
    full = decode(c, q, 0.1)
    part = decode(c, q, 0.1, n=3)
    assert torch.equal(part[:3], full[:3]) and bool((part[3:] == 7.0).all())
    from vllm_exact import paged_attn as P
    for b in range(len(lens)):
        one = torch.empty(1, H, D, dtype=BF, device=DEV)
        P.paged_decode_q8(q[b:b + 1], c.dk, c.dv, *c.ds, c.dt[b:b + 1], c.dl[b:b + 1], 0.1, one, 1, max_seq_len=max(lens[b], 1))
        assert torch.equal(one[0], full[b]), b
    order = torch.randperm(len(lens), generator=gen(3)).to(DEV)
    out = torch.empty_like(full)
    P.paged_decode_q8(q[order], c.dk, c.dv, *c.ds, c.dt[order], c.dl[order], 0.1, out, len(lens))
    assert torch.equal(out, full[order])
    to = torch.randperm(c.dk.shape[0], generator=gen(4)).to(DEV)
    moved = [torch.empty_like(x.view(torch.uint8) if x.element_size() == 1 else x) for x in (c.dk, c.dv, *c.ds)]
    for m, x in zip(moved, (c.dk, c.dv, *c.ds)):
        m[to] = x.view(m.dtype)
    P.paged_decode_q8(q, moved[0].view(dtype), moved[1].view(dtype), moved[2], moved[3], to[c.dt.long()].to(torch.int32), c.dl, 0.1, out, len(lens))
    assert torch.equal(out, full)


def test_decode_q8_layouts():
    """Strided queries, outputs and caches (a slice of KV heads of a fused cache) give the bits of contiguous ones."""
    from vllm_exact import paged_attn as P
    lens, page, KV, D, H = [100, 800], 16, 4, 128, 8
    c = Cache(lens, page, KV, D, E4)
    q = torch.randn(2, H, D, generator=gen(2)).to(BF).to(DEV)
    want = decode(c, q, 0.1)
    wide = torch.zeros(2, H + 5, D, dtype=BF, device=DEV)
    wide[:, 2:2 + H] = q
    out = torch.full((2, H * 3, D), 7.0, dtype=BF, device=DEV)
    both = torch.stack([c.dk.view(torch.uint8), c.dv.view(torch.uint8)], 3).view(E4)  # (blocks, page, KV, 2, D)
    pad = [torch.zeros(s.shape[0], KV + 3, page, device=DEV) for s in c.ds]
    for p, s in zip(pad, c.ds):
        p[:, 1:1 + KV] = s
    P.paged_decode_q8(wide[:, 2:2 + H], both[:, :, :, 0], both[:, :, :, 1], pad[0][:, 1:1 + KV], pad[1][:, 1:1 + KV],
                      c.dt, c.dl, 0.1, out[:, H:2 * H], 2)
    assert torch.equal(out[:, H:2 * H], want) and bool((out[:, :H] == 7.0).all()) and bool((out[:, 2 * H:] == 7.0).all())


def test_decode_q8_pages_that_do_not_exist_and_poisoned_rows():
    """Tokens on pages outside the cache are not seen; a visible row that was written with an infinity gives NaN to its
    own request and KV head only."""
    from vllm_exact import kv_cache as C
    lens, page, KV, D, H = [90, 700], 16, 2, 64, 4
    c = Cache(lens, page, KV, D, I8)
    q = torch.randn(2, H, D, generator=gen(5)).to(BF)
    c.dt[0, 1], c.dt[1, 3], c.dt[1, 20] = -1, c.dk.shape[0], 2 ** 31 - 1
    got = decode(c, q.to(DEV), 0.125)
    for b, gone in ((0, [1]), (1, [3, 20])):
        seen = torch.ones(1, lens[b], dtype=torch.bool)
        for x in gone:
            seen[:, x * page:(x + 1) * page] = False
        want, bound = S.attend(q[b:b + 1], c.seq(0, b), c.seq(1, b), seen, 0.125, BF, q8=True)
        check(got[b:b + 1], want, bound, b)
    c = Cache(lens, page, KV, D, I8)
    clean = decode(c, q.to(DEV), 0.125)
    x = torch.ones(1, KV, D, dtype=BF, device=DEV)
    x[0, 1, 7] = float("inf")
    slot = (c.dt[1, 2].long() * page + 5).view(1)
    keep = [t.clone() for t in (c.dk, *c.ds)]
    kept_v, kept_vs = c.dv.clone(), c.ds[1].clone()
    C.cache_write(x, x, c.dk, c.dv, *c.ds, slot)
    bad = decode(c, q.to(DEV), 0.125)
    assert bool(torch.isnan(bad[1, 2:]).all()) and torch.equal(bad[0], clean[0]) and bool(torch.isfinite(bad[1, :2]).all())
    # the value row alone
    c.dk.copy_(keep[0])
    c.ds[0].copy_(keep[1])
    bad = decode(c, q.to(DEV), 0.125)
    assert bool(torch.isnan(bad[1, 2:]).all()) and torch.equal(bad[0], clean[0])


def test_decode_q8_graph_stream_and_workspace():
    """Captured once and replayed with other contents; on a side stream; with a caller's workspace full of NaN."""
    from vllm_exact import paged_attn as P
    lens, page, KV, D, H = [3000, 64, 900], 16, 8, 128, 32
    a, b = Cache(lens, page, KV, D, E4, seed=1), Cache([500, 2999, 0], page, KV, D, E4, seed=1)
    q = torch.randn(3, H, D, generator=gen(6)).to(BF).to(DEV)
    want = [decode(x, q, 0.1) for x in (a, b)]
    ws = torch.full((P.rows_workspace_bytes(3, H, D, 3008) // 4,), float("nan"), device=DEV)
    out = torch.empty_like(q)
    table, sl = torch.zeros(3, 188, dtype=torch.int32, device=DEV), a.dl.clone()
    table[:, :a.dt.shape[1]] = a.dt
    args = (q, a.dk, a.dv, *a.ds, table, sl, 0.1, out, 3)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        P.paged_decode_q8(*args, workspace=ws)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, want[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        P.paged_decode_q8(*args)  # its workspace belongs to the graph
    for c, w in ((b, want[1]), (a, want[0]), (b, want[1])):
        a.dk.view(torch.uint8)[:c.dk.shape[0]] = c.dk.view(torch.uint8) if c is b else Cache(lens, page, KV, D, E4, seed=1).dk.view(torch.uint8)
        fresh = Cache(c.lens, page, KV, D, E4, seed=1)
        n = fresh.dk.shape[0]
        for dst, src in zip((a.dk, a.dv), (fresh.dk, fresh.dv)):
            dst.view(torch.uint8)[:n] = src.view(torch.uint8)
        for dst, src in zip(a.ds, fresh.ds):
            dst[:n] = src
        table[:, :fresh.dt.shape[1]] = fresh.dt
        sl.copy_(fresh.dl)
        out.fill_(5.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)
    del g


def test_decode_q8_offsets_beyond_32_bits():
    """A cache of more than 2^32 bytes per tensor, its sequences in the first and last pages."""
    from vllm_exact import kv_cache as C, paged_attn as P
    KV, D, H, page = 8, 256, 16, 16
    blocks = (2 ** 32) // (KV * D * page) + 70
    kc, vc, ks, vs = C.alloc_q8_cache(blocks, page, KV, D, E4, DEV)
    lens = [1000]
    c = Cache(lens, page, KV, D, E4)
    q = torch.randn(1, H, D, generator=gen(7)).to(BF).to(DEV)
    want = decode(c, q, 0.1)
    wide = c.dt.shape[1]
    to = torch.arange(blocks - wide, blocks, device=DEV)
    for dst, src in ((kc.view(torch.uint8), c.dk.view(torch.uint8)), (vc.view(torch.uint8), c.dv.view(torch.uint8)), (ks, c.ds[0]), (vs, c.ds[1])):
        dst[to] = src[c.dt[0].long()]
    out = torch.empty_like(q)
    P.paged_decode_q8(q, kc, vc, ks, vs, to.view(1, -1).to(torch.int32), c.dl, 0.1, out, 1)
    assert torch.equal(out, want)
    x = torch.randn(3, KV, D, generator=gen(8)).to(BF).to(DEV)
    C.cache_write(x, x, kc, vc, ks, vs, blocks * page - 1 - torch.arange(3, device=DEV))
    ko, vo = torch.empty(3, KV, D, dtype=BF, device=DEV), torch.empty(3, KV, D, dtype=BF, device=DEV)
    C.cache_read(kc, vc, ks, vs, torch.full((1, 1), blocks - 1, dtype=torch.int32, device=DEV), cu([3]), ko, vo)
    got = kc.view(torch.uint8)[blocks - 1, page - 3:].flip(0).view(E4).float()
    assert torch.equal(got.cpu(), S.quantise(x, E4)[0].float())
    del kc, vc, ks, vs


# ------------------------------------------------------------------------------------------------------------- tree
def words(T, kind, g):
    """Mask words of T drafted tokens and the (T, T) matrix they stand for."""
    see = torch.zeros(T, T, dtype=torch.bool)
    for i in range(T):
        if kind == "tree" and i:
            see[i] = see[int(torch.randint(0, i, (1,), generator=g))]
        if kind == "any":
            see[i] = torch.rand(T, generator=g) < 0.4
        elif kind == "chain":
            see[i, :i + 1] = True
        elif kind != "none":
            see[i, i] = True
    w = [sum(1 << j for j in range(T) if see[i, j]) for i in range(T)]
    return [x - (1 << 64) if x >> 63 else x for x in w], see


def tree(c, q, T, scale, mask, most=None, **kw):
    from vllm_exact import paged_attn as P
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device=DEV)
    P.tree_attention(q.to(DEV), c.dk, c.dv, c.dt, c.dl, cu(T), scale, out, max(T) if most is None else most,
                     tree_mask=None if mask is None else torch.tensor(mask, dtype=torch.int64, device=DEV),
                     key_scale=c.ds[0], value_scale=c.ds[1], **kw)
    return out


def tree_check(c, q, T, see, got, scale, real):
    at = 0
    for b, t in enumerate(T):
        L = c.lens[b]
        seen = torch.cat([torch.ones(t, L - t, dtype=torch.bool), see[b]], 1)
        want, bound = S.attend(q[at:at + t], c.seq(0, b), c.seq(1, b), seen, scale, real, q8=c.scales is not None)
        check(got[at:at + t], want, bound, (b, t, L))
        at += t


@pytest.mark.parametrize("dtype", [None, I8, E4])
@pytest.mark.parametrize("H,KV,D", HEADS)
@pytest.mark.parametrize("most,page,real", [(1, 16, BF), (3, 24, FP), (16, 16, BF), (64, 528, BF), (64, 16, FP)])
def test_tree_attention(dtype, H, KV, D, most, page, real):
    g = gen(most + D)
    T = [x for x in (0, 1, 2, 3, 8, 16, 17, 63, 64) if x <= most]
    T = (T + T)[:max(4, len(T))]
    lens = [max(t, x) for t, x in zip(T, [70, 1, 300, 64, 2100, 8, 2049, 127, 64])]
    c = Cache(lens, page, KV, D, dtype, real=real, seed=D)
    q = torch.randn(sum(T), H, D, generator=g).to(real)
    made = [words(t, ["tree", "any", "chain"][b % 3], g) for b, t in enumerate(T)]
    got = tree(c, q, T, D ** -0.5, [x for w, _ in made for x in w], most=most)
    tree_check(c, q, T, [s for _, s in made], got, D ** -0.5, real)


@pytest.mark.parametrize("dtype", [None, E4])
def test_tree_rows_that_see_nothing(dtype):
    """No context and empty words: zeros. Every other row of the batch is as it should be."""
    T, lens = [4, 5, 3], [4, 9, 3]
    c = Cache(lens, 16, 2, 64, dtype)
    q = torch.randn(sum(T), 8, 64, generator=gen(3)).to(BF)
    made = [words(4, "none", gen(1)), words(5, "none", gen(1)), words(3, "tree", gen(1))]
    made[0][0][2] = 0b0011
    made[0][1][2, :2] = True
    got = tree(c, q, T, 0.125, [x for w, _ in made for x in w])
    assert bool((got[[0, 1, 3]] == 0).all())
    tree_check(c, q, T, [s for _, s in made], got, 0.125, BF)


@pytest.mark.parametrize("dtype", [None, I8])
def test_tree_chain_is_the_default_and_bits_do_not_depend_on_the_batch(dtype):
    from vllm_exact import paged_attn as P
    H, KV, D = 32, 8, 128
    T, lens = [5, 1, 20, 64], [2600, 300, 1000, 640]
    c = Cache(lens, 16, KV, D, dtype)
    q = torch.randn(sum(T), H, D, generator=gen(4)).to(BF)
    made = [words(t, "chain", None) for t in T]
    full = tree(c, q, T, 0.1, [x for w, _ in made for x in w])
    assert torch.equal(full, tree(c, q, T, 0.1, None))
    tree_check(c, q, T, [s for _, s in made], full, 0.1, BF)
    at = 0
    for b, t in enumerate(T):
        out = torch.empty(t, H, D, dtype=BF, device=DEV)
        P.tree_attention(q[at:at + t].to(DEV), c.dk, c.dv, c.dt[b:b + 1], c.dl[b:b + 1], cu([t]), 0.1, out, t,
                         key_scale=c.ds[0], value_scale=c.ds[1], max_seq_len=lens[b])
        assert torch.equal(out, full[at:at + t]), b
        at += t
    if dtype is not None:  # one drafted token is a decode step
        one = decode(c, q[5:6].expand(4, H, D).contiguous().to(DEV), 0.1)
        assert torch.equal(one[1], full[5])


@pytest.mark.parametrize("real", [BF, FP])
def test_tree_hidden_values_that_are_not_finite(real):
    """A drafted token with infinities and NaN in its key and value reaches the rows that see it and no others."""
    H, KV, D, T = 8, 2, 128, 6
    c = Cache([100, 70], 16, KV, D, None, real=real)
    q = torch.randn(2 * T, H, D, generator=gen(5)).to(real)
    made = words(T, "tree", gen(9))
    clean = tree(c, q, [T, T], 0.1, made[0] * 2)
    for b, x in ((0, 100), (1, 70)):
        pos = x - T + 2
        blk, off = int(c.table[b, pos // 16]), pos % 16
        c.dk[blk, off, 0, 3] = float("nan")
        c.dv[blk, off, 1, 5] = float("inf")
        c.dv[blk, off, 0, 9] = float("nan")
    got = tree(c, q, [T, T], 0.1, made[0] * 2)
    for i in range(2 * T):
        sees = bool(made[1][i % T, 2])
        if not sees:
            # the block's products are made in another order, so the bits may differ by their rounding
            assert bool(torch.isfinite(got[i]).all()), i
            assert float((got[i] - clean[i]).abs().max()) <= 4 * S.HALF_STEP[real] * float(clean[i].abs().max().clamp(min=1))
        else:
            assert bool(torch.isnan(got[i, :4]).all()) and not bool(torch.isfinite(got[i, 4:, 5]).any())
            assert bool(torch.isfinite(got[i, 4:, :5]).all())


def test_tree_rows_left_untouched():
    """Requests with more rows than max_query_len, and rows of no request."""
    c = Cache([50, 60, 70], 16, 2, 64, None)
    T = [2, 9, 3]
    q = torch.randn(20, 4, 64, generator=gen(5)).to(BF).to(DEV)
    got = tree(c, q, T, 0.1, None, most=4)
    assert bool((got[2:11] == 7.0).all()) and bool((got[14:] == 7.0).all())
    assert not bool((got[:2] == 7.0).any()) and not bool((got[11:14] == 7.0).any())
    short = tree(c, q[:12], T, 0.1, None, most=9)  # the last request's rows are not all in q
    assert bool((short[11:] == 7.0).all()) and not bool((short[:11] == 7.0).any())


def test_tree_many_empty_requests_between():
    """Values that are not finite belong to their own request, however many requests without keys lie between two that have
    some (a CTA takes every so many-th item)."""
    from vllm_exact import paged_attn as P
    H, KV, D, T = 16, 1, 128, 2
    step = 8 * torch.cuda.get_device_properties(0).multi_processor_count
    n = 2 * step + 1
    c = Cache([20, 30, 40], 16, KV, D, None)
    lens = torch.zeros(n, dtype=torch.int32, device=DEV)
    table = torch.zeros(n, c.dt.shape[1], dtype=torch.int32, device=DEV)
    for i, b in enumerate((0, step, 2 * step)):
        lens[b], table[b] = c.lens[i], c.dt[i]
        c.dv[int(c.table[i, 0]), 3, 0, 5 + i] = float("inf")
    q = torch.randn(T, H, D, generator=gen(21)).to(BF).to(DEV).repeat(n, 1, 1)
    out = torch.full_like(q, 7.0)
    P.tree_attention(q, c.dk, c.dv, table, lens, cu([T] * n), 0.1, out, T)
    out = out.view(n, T, H, D)
    some = torch.tensor([0, step, 2 * step], device=DEV)
    empty = torch.ones(n, dtype=torch.bool, device=DEV)
    empty[some] = False
    assert bool((out[empty] == 0).all())
    want = torch.zeros(3, T, H, D, dtype=torch.bool, device=DEV)
    for i in range(3):
        want[i, :, :, 5 + i] = True
    assert torch.equal(out[some] == float("inf"), want) and torch.equal(~torch.isfinite(out[some]), want)


@pytest.mark.parametrize("dtype", [None, E4])
def test_tree_padded_batch(dtype):
    """Rows behind the last request (a captured step of a fixed number of rows): the requests' bits are those of the batch
    without them, the rows are left as they were."""
    H, KV, D, most = 32, 8, 128, 8
    T, lens = [1, 8, 3], [900, 2300, 40]
    c = Cache(lens, 16, KV, D, dtype)
    q = torch.randn(most * len(T), H, D, generator=gen(14)).to(BF)
    want = tree(c, q[:sum(T)], T, 0.1, None, most=most)
    got = tree(c, q, T, 0.1, None, most=most)
    assert torch.equal(got[:sum(T)], want) and bool((got[sum(T):] == 7.0).all())


# ----------------------------------------------------------------------------------------------------------- prompt
def prompt(q, k, v, Lq, Lk, scale, out=None):
    from vllm_exact import prompt_attn as A
    return A.prompt_attention(q, k, v, cu(Lq), cu(Lk), scale, out=out)


def prompt_check(q, k, v, Lq, Lk, scale, got, real, tag=""):
    i = j = 0
    for b, (x, y) in enumerate(zip(Lq, Lk)):
        seen = torch.ones(x, y, dtype=torch.bool).tril(y - x)
        want, bound = S.attend(q[i:i + x], k[j:j + y], v[j:j + y], seen, scale, real)
        check(got[i:i + x], want, bound, (tag, b, x, y))
        i, j = i + x, j + y


@pytest.mark.parametrize("real", [BF, FP])
@pytest.mark.parametrize("H,KV,D", [(4, 2, 128), (4, 1, 256), (8, 1, 64), (3, 3, 128)])
@pytest.mark.parametrize("lens", [[(1, 1)], [(1, 1), (2, 2), (63, 63), (64, 64), (65, 65)], [(127, 127), (128, 128), (129, 129)],
                                  [(300, 300), (0, 0), (5, 700), (0, 40), (1, 513)], [(255, 256), (257, 257), (90, 1000)],
                                  [(20, 7), (300, 129), (4, 0), (33, 33)]])
def test_prompt_attention(real, H, KV, D, lens):
    Lq, Lk = zip(*lens)
    g = gen(sum(Lq) + D)
    q = torch.randn(sum(Lq), H, D, generator=g).to(real)
    kv = torch.randn(max(1, sum(Lk)), 2, KV, D, generator=g).to(real)
    got = prompt(q.to(DEV), kv[:, 0].to(DEV), kv[:, 1].to(DEV), Lq, Lk, D ** -0.5)
    prompt_check(q, kv[:, 0], kv[:, 1], Lq, Lk, D ** -0.5, got, real)


def test_prompt_attention_large_scores():
    """Scores of a few hundred (one key takes nearly all weight), growing along the sequence, so that the running maximum
    moves in every block."""
    L, H, D = 700, 2, 128
    g = gen(3)
    q, k, v = (torch.randn(L, H, D, generator=g) for _ in range(3))
    k = k + torch.linspace(-4, 4, L)[:, None, None] * 2
    q = q.abs() * 2
    q, k, v = (x.to(BF) for x in (q, k, v))
    got = prompt(q.to(DEV), k.to(DEV), v.to(DEV), [L], [L], 0.2)
    prompt_check(q, k, v, [L], [L], 0.2, got, BF)


def test_prompt_attention_invariance_layout_and_untouched_rows():
    """Bits alone and in the batch; q, k, v as slices of one projection; rows of no sequence keep their contents."""
    H, KV, D = 8, 2, 128
    Lq, Lk = [300, 17, 513, 1], [300, 400, 513, 77]
    g = gen(4)
    wide = torch.randn(sum(Lk) + 4, H + 2 * KV, D, generator=g).to(BF).to(DEV)
    q = torch.randn(sum(Lq) + 5, H + 3, D, generator=g).to(BF).to(DEV)[:, 1:1 + H]
    k, v = wide[:, H:H + KV], wide[:, H + KV:]
    out = torch.full((sum(Lq) + 5, H, D), 7.0, dtype=BF, device=DEV)
    full = prompt(q, k, v, Lq, Lk, 0.1, out=out)
    assert full is out and bool((out[sum(Lq):] == 7.0).all())
    prompt_check(q, k, v, Lq, Lk, 0.1, full, BF)
    i = j = 0
    for x, y in zip(Lq, Lk):
        one = prompt(q[i:i + x].contiguous(), k[j:j + y].contiguous(), v[j:j + y].contiguous(), [x], [y], 0.1)
        assert torch.equal(one, full[i:i + x])
        i, j = i + x, j + y


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_attention_neighbours_that_are_not_finite(D):
    """NaN keys and values of the other sequences and behind the last one do not reach a sequence."""
    H, KV = 4, 2
    Lq = Lk = [70, 200, 130]
    g = gen(5)
    q = torch.randn(400, H, D, generator=g).to(BF).to(DEV)
    kv = torch.randn(450, 2, KV, D, generator=g).to(BF).to(DEV)
    clean = prompt(q, kv[:, 0], kv[:, 1], Lq, Lk, 0.1)
    kv[:70], kv[270:] = float("nan"), float("inf")
    q[:70] = float("nan")
    got = prompt(q, kv[:, 0], kv[:, 1], Lq, Lk, 0.1)
    assert torch.equal(got[70:270], clean[70:270]) and bool(torch.isnan(got[:70]).all())


@pytest.mark.parametrize("real", [BF, FP])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_attention_hidden_values_that_are_not_finite(D, real):
    """Infinities and NaN in a key and value reach the queries behind it and none before it, element by element."""
    H, KV, L, before = 4, 2, 400, 70
    g = gen(7)
    q = torch.randn(L - before, H, D, generator=g).to(real).to(DEV)
    k, v = (torch.randn(L, KV, D, generator=g).to(real).to(DEV) for _ in range(2))
    clean = prompt(q, k, v, [L - before], [L], 0.1)
    v2 = v.clone()
    v2[100, 0, 3], v2[301, 1, D - 1], v2[301, 1, 0] = float("inf"), float("nan"), float("-inf")
    k2 = k.clone()
    k2[350, 0, 2] = float("nan")
    got = prompt(q, k2, v2, [L - before], [L], 0.1)
    i = torch.arange(before, L)
    bad = torch.zeros(L - before, H, D, dtype=torch.bool)
    bad[i >= 100, :2, 3] = True
    bad[i >= 301, 2:, 0] = True
    bad[i >= 301, 2:, D - 1] = True
    bad[i >= 350, :2] = True
    bad = bad.to(DEV)
    assert torch.equal(got[~bad], clean[~bad])
    assert not bool(torch.isfinite(got[bad]).any())
    assert bool((got[31:280, :2, 3] == float("inf")).all()) and bool(torch.isnan(got[280:, :2]).all())


def test_prompt_attention_graph():
    H, KV, D = 4, 2, 128
    g0 = gen(6)
    q, k, v = (torch.randn(600, h, D, generator=g0).to(BF).to(DEV) for h in (H, KV, KV))
    cq = cu([100, 500])
    out = torch.empty_like(q)
    from vllm_exact import prompt_attn as A
    want = [A.prompt_attention(q, k, v, cu(x), cu(x), 0.1) for x in ([100, 500], [599, 1], [0, 600])]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        A.prompt_attention(q, k, v, cq, cq, 0.1, out=out)
    for x, w in zip(([100, 500], [599, 1], [0, 600]), want):
        cq.copy_(cu(x))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)
    del g


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_attention_in_pieces(D):
    """A prompt whose last queries come by themselves, over all keys so far, has the bits of the whole."""
    H, KV, L = 4, 2, 700
    g = gen(12)
    q = torch.randn(L, H, D, generator=g).to(BF).to(DEV)
    k, v = (torch.randn(L, KV, D, generator=g).to(BF).to(DEV) for _ in range(2))
    q[650] *= 30  # a row whose largest score grows late, with its neighbours'
    whole = prompt(q, k, v, [L], [L], 0.2)
    for lo, hi in ((0, 130), (130, 500), (500, 501), (501, 700)):
        assert torch.equal(prompt(q[lo:hi], k[:hi], v[:hi], [hi - lo], [hi], 0.2), whole[lo:hi]), (lo, hi)


# ---------------------------------------------------------------------------------------------------------- together
def test_calls_on_two_streams_at_once():
    """Prompt, decode and draft calls of two streams, each with its own outputs and workspaces, in flight together."""
    from vllm_exact import paged_attn as P, prompt_attn as A
    H, KV, D = 16, 4, 128
    g = gen(13)
    T, lens = [20, 3], [3000, 700]
    caches = [Cache(lens, 16, KV, D, E4), Cache(lens, 16, KV, D, None)]
    q = torch.randn(600, H, D, generator=g).to(BF).to(DEV)
    kv = torch.randn(600, 2, KV, D, generator=g).to(BF).to(DEV)
    cq, ct = cu([400, 200]), cu(T)

    def run():
        a, b, c, d = (torch.empty_like(x) for x in (q, q[:2], q[:23], q[:23]))
        A.prompt_attention(q, kv[:, 0], kv[:, 1], cq, cq, 0.1, out=a)
        P.paged_decode_q8(q[:2], caches[0].dk, caches[0].dv, *caches[0].ds, caches[0].dt, caches[0].dl, 0.1, b, 2)
        for x, o in zip(caches, (c, d)):
            P.tree_attention(q[:23], x.dk, x.dv, x.dt, x.dl, ct, 0.1, o, 20, key_scale=x.ds[0], value_scale=x.ds[1])
        return a, b, c, d

    want = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(6):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    for x in got:
        assert all(torch.equal(y, w) for y, w in zip(x, want))


def test_calls_without_work():
    from vllm_exact import kv_cache as C, paged_attn as P, prompt_attn as A
    c = Cache([20], 16, 2, 64, E4)
    q = torch.ones(3, 4, 64, dtype=BF, device=DEV)
    kv = torch.ones(3, 2, 64, dtype=BF, device=DEV)
    out = torch.full_like(q, 7.0)
    none = cu([])
    A.prompt_attention(q, kv, kv, none, none, 0.1, out=out)
    assert A.prompt_attention(q[:0], kv, kv, cu([0]), cu([3]), 0.1).shape == (0, 4, 64)
    P.paged_decode_q8(q, c.dk, c.dv, *c.ds, c.dt, c.dl, 0.1, out, 0)
    P.tree_attention(q, c.dk, c.dv, c.dt[:0], c.dl[:0], none, 0.1, out, 4, key_scale=c.ds[0], value_scale=c.ds[1])
    P.tree_attention(q, c.dk, c.dv, c.dt, c.dl, cu([0]), 0.1, out, 4, key_scale=c.ds[0], value_scale=c.ds[1])
    rows = torch.full((3, 2, 64), 7.0, dtype=BF, device=DEV)
    C.cache_read(c.dk, c.dv, *c.ds, c.dt[:0], none, rows, rows)
    C.cache_read(c.dk, c.dv, *c.ds, c.dt, cu([0]), rows, rows)
    C.cache_read(c.dk, c.dv, *c.ds, c.dt, cu([3]), rows[:0], rows[:0])
    assert bool((out == 7.0).all()) and bool((rows == 7.0).all())


@pytest.mark.parametrize("dtype", [I8, E4])
def test_a_served_conversation(dtype):
    """A prompt is cached and attended to with the numbers the cache stands for, one token is decoded, a draft is
    verified, and the conversation is continued over the cache read back: every step gives the attention over the same
    cached numbers."""
    from vllm_exact import kv_cache as C, paged_attn as P, prompt_attn as A
    H, KV, D, page, scale = 8, 2, 128, 16, 128 ** -0.5
    g = gen(11)
    lens = [150, 47]
    more = 1 + 5 + 20  # decoded, drafted, continued
    blocks = 40
    kc, vc, ks, vs = C.alloc_q8_cache(blocks, page, KV, D, dtype, DEV)
    table = torch.randperm(blocks, generator=g)[:30].view(2, 15).to(torch.int32).to(DEV)
    qkv = [torch.randn(L + more, H + 2 * KV, D, generator=g).to(BF).to(DEV) for L in lens]

    def slots(b, lo, hi):
        i = torch.arange(lo, hi, device=DEV)
        return table[b].long()[i // page] * page + i % page

    def new(lo_of, hi_of):
        x = torch.cat([qkv[b][lo_of(b):hi_of(b)] for b in range(2)])
        s = torch.cat([slots(b, lo_of(b), hi_of(b)) for b in range(2)])
        kb, vb = torch.empty(x.shape[0], KV, D, dtype=BF, device=DEV), torch.empty(x.shape[0], KV, D, dtype=BF, device=DEV)
        C.cache_write(x[:, H:H + KV], x[:, H + KV:], kc, vc, ks, vs, s, key_out=kb, value_out=vb)
        return x[:, :H], kb, vb

    stands = []
    for b in range(2):
        kv = [S.values(*S.quantise(qkv[b][:, H + KV * i:H + KV * (i + 1)], dtype)) for i in range(2)]
        stands.append(kv)

    def want(b, lo, hi, q8):
        seen = torch.ones(hi - lo, hi, dtype=torch.bool).tril(lo)
        k, v = (x[:hi] for x in stands[b])
        if not q8:
            k, v = k.float().to(BF), v.float().to(BF)
        return S.attend(qkv[b][lo:hi, :H], k, v, seen, scale, BF, q8=q8)

    q, kb, vb = new(lambda b: 0, lambda b: lens[b])
    out = A.prompt_attention(q, kb, vb, cu(lens), cu(lens), scale)
    for b, part in enumerate(out.split(lens)):
        check(part, *want(b, 0, lens[b], False), ("prompt", b))
    q, _, _ = new(lambda b: lens[b], lambda b: lens[b] + 1)
    out = P.paged_decode_q8(q, kc, vc, ks, vs, table, torch.tensor(lens, dtype=torch.int32, device=DEV) + 1, scale, torch.empty_like(q), 2)
    for b in range(2):
        check(out[b:b + 1], *want(b, lens[b], lens[b] + 1, True), ("decode", b))
    q, _, _ = new(lambda b: lens[b] + 1, lambda b: lens[b] + 6)
    out = P.tree_attention(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device=DEV) + 6, cu([5, 5]), scale,
                           torch.empty_like(q), 5, key_scale=ks, value_scale=vs)
    for b, part in enumerate(out.split([5, 5])):
        check(part, *want(b, lens[b] + 1, lens[b] + 6, True), ("tree", b))
    q, _, _ = new(lambda b: lens[b] + 6, lambda b: lens[b] + more)
    total = [L + more for L in lens]
    kb, vb = torch.empty(sum(total), KV, D, dtype=BF, device=DEV), torch.empty(sum(total), KV, D, dtype=BF, device=DEV)
    C.cache_read(kc, vc, ks, vs, table, cu(total), kb, vb)
    out = A.prompt_attention(q, kb, vb, cu([20, 20]), cu(total), scale)
    for b, part in enumerate(out.split([20, 20])):
        check(part, *want(b, lens[b] + 6, lens[b] + more, False), ("continued", b))
