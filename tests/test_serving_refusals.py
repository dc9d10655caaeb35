"""CPU tests: the refusals of the 8-bit cache, tree and prompt attention entry points, before anything is launched, and
the plain implementations that their GPU tests compare with."""
import ctypes

import pytest
import torch

import serving_ref as S

BF = torch.bfloat16


@pytest.fixture(scope="module")
def X():
    from vllm_exact import _lib
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    return _lib


P = ctypes.c_void_p(256)  # never dereferenced: every call below fails validation first


def refuse(f, base, status, **change):
    args = dict(base, **change)
    assert f(*args.values()) == status, change


WRITE = dict(key=P, sk_t=1024, sk_h=128, value=P, sv_t=1024, sv_h=128, dtype=1, code=0, kc=P, vc=P, s_block=16384,
             s_page=1024, s_head=128, ks=P, vs=P, ss_block=128, ss_head=16, nb=10, BS=16, slots=P, tokens=3, KV=8, D=128,
             ko=None, sko_t=0, sko_h=0, vo=None, svo_t=0, svo_h=0, stream=None)
READ = dict(kc=P, vc=P, code=1, s_block=16384, s_page=1024, s_head=128, ks=P, vs=P, ss_block=128, ss_head=16, nb=10, BS=16,
            bt=P, sbt=4, width=4, cu=P, n=2, rows=40, KV=8, D=128, dtype=1, ko=P, sko_t=1024, sko_h=128, vo=P, svo_t=1024,
            svo_h=128, stream=None)
DECODE = dict(q=P, sq_t=4096, sq_h=128, qd=1, kc=P, vc=P, code=0, s_block=16384, s_page=1024, s_head=128, ks=P, vs=P,
              ss_block=128, ss_head=16, nb=10, bt=P, sbt=300, width=300, sl=P, n=2, H=32, KV=8, D=128, BS=16, scale=0.1,
              max_len=4800, out=P, so_t=4096, so_h=128, ws=P, wsb=0, stream=None)
TREE = dict(list(DECODE.items())[:19] + [("qsl", P), ("mask", None), ("n", 2), ("tokens", 10), ("most", 8)] +
            list(DECODE.items())[20:])
PROMPT = dict(q=P, sq_t=4096, sq_h=128, k=P, sk_t=1024, sk_h=128, v=P, sv_t=1024, sv_h=128, dtype=1, cq=P, ck=P, n=2,
              tokens=10, keys=10, H=32, KV=8, D=128, scale=0.1, out=P, so_t=4096, so_h=128, stream=None)


def test_cache_refusals(X):
    for f, base in ((X.lib().ex_cache_write_q8, WRITE), (X.lib().ex_cache_read_q8, READ)):
        for status, change in [(X.EX_ERR_ARG, dict(code=2)), (X.EX_ERR_ARG, dict(code=-1)), (X.EX_ERR_ARG, dict(KV=0)),
                               (X.EX_ERR_ARG, dict(BS=0)), (X.EX_ERR_ARG, dict(nb=0)), (X.EX_ERR_ARG, dict(kc=None)),
                               (X.EX_ERR_ARG, dict(vs=None)), (X.EX_ERR_DTYPE, dict(dtype=0)),
                               (X.EX_ERR_UNSUPPORTED, dict(D=96)), (X.EX_ERR_ALIGN, dict(s_page=1020)),
                               (X.EX_ERR_ALIGN, dict(kc=ctypes.c_void_p(8)))]:
            refuse(f, base, status, **change)
    f = X.lib().ex_cache_write_q8
    refuse(f, WRITE, X.EX_ERR_ARG, tokens=-1)
    refuse(f, WRITE, X.EX_ERR_ARG, slots=None)
    refuse(f, WRITE, X.EX_ERR_ARG, ko=P)  # without value_out
    refuse(f, WRITE, X.EX_ERR_ALIGN, sk_t=1028)
    refuse(f, WRITE, X.EX_ERR_ALIGN, ko=P, vo=P, sko_t=4, sko_h=128, svo_t=1024, svo_h=128)
    refuse(f, WRITE, X.EX_ERR_UNSUPPORTED, tokens=2 ** 31)
    refuse(f, WRITE, X.EX_OK, tokens=0)
    f = X.lib().ex_cache_read_q8
    refuse(f, READ, X.EX_ERR_ARG, cu=None)
    refuse(f, READ, X.EX_ERR_ARG, vo=None)
    refuse(f, READ, X.EX_ERR_ALIGN, svo_h=4)
    refuse(f, READ, X.EX_OK, rows=0)
    refuse(f, READ, X.EX_OK, n=0)


def test_decode_and_tree_refusals(X):
    L = X.lib()
    for f, base in ((L.ex_paged_decode_q8, DECODE), (L.ex_tree_attention, TREE)):
        for status, change in [(X.EX_ERR_ARG, dict(H=30)), (X.EX_ERR_ARG, dict(n=-1)), (X.EX_ERR_ARG, dict(code=3)),
                               (X.EX_ERR_ARG, dict(width=-1)), (X.EX_ERR_ARG, dict(max_len=-1)),
                               (X.EX_ERR_ARG, dict(ks=None)), (X.EX_ERR_ARG, dict(out=None)),
                               (X.EX_ERR_DTYPE, dict(qd=0)), (X.EX_ERR_UNSUPPORTED, dict(D=80)),
                               (X.EX_ERR_UNSUPPORTED, dict(BS=12)), (X.EX_ERR_UNSUPPORTED, dict(H=256)),
                               (X.EX_ERR_ALIGN, dict(sq_t=4100)), (X.EX_ERR_ALIGN, dict(ss_head=6)),
                               (X.EX_ERR_ALIGN, dict(s_head=8)), (X.EX_ERR_ALIGN, dict(ks=ctypes.c_void_p(260))),
                               (X.EX_ERR_WORKSPACE, {})]:
            refuse(f, base, status, **change)
        refuse(f, base, X.EX_OK, n=0)
    refuse(L.ex_paged_decode_q8, DECODE, X.EX_ERR_ARG, code=-1)
    refuse(L.ex_tree_attention, TREE, X.EX_ERR_UNSUPPORTED, most=65)
    refuse(L.ex_tree_attention, TREE, X.EX_ERR_ARG, most=0)
    refuse(L.ex_tree_attention, TREE, X.EX_ERR_ARG, qsl=None)
    refuse(L.ex_tree_attention, TREE, X.EX_ERR_ALIGN, code=-1, s_page=1028, ks=None, vs=None)
    refuse(L.ex_tree_attention, TREE, X.EX_OK, tokens=0)
    need = L.ex_paged_rows_workspace_bytes
    assert need(2, 32, 128, 0) == 0 and need(2, 32, 128, 1) == 0 and need(0, 32, 128, 9000) == 0
    assert need(2, 32, 128, 5000) >= 2 * 32 * 130 * 4 * 2
    sizes = [need(2, 32, 128, x) for x in range(1, 20000, 37)]
    assert sizes == sorted(sizes)  # a larger bound is enough for every shorter request


def test_prompt_refusals(X):
    f = X.lib().ex_prompt_attention
    for status, change in [(X.EX_ERR_ARG, dict(n=-1)), (X.EX_ERR_ARG, dict(KV=5)), (X.EX_ERR_ARG, dict(tokens=-1)),
                           (X.EX_ERR_ARG, dict(k=None)), (X.EX_ERR_ARG, dict(ck=None)), (X.EX_ERR_DTYPE, dict(dtype=0)),
                           (X.EX_ERR_UNSUPPORTED, dict(D=192)), (X.EX_ERR_ALIGN, dict(sk_t=1028)),
                           (X.EX_ERR_ALIGN, dict(so_h=132)), (X.EX_ERR_ALIGN, dict(v=ctypes.c_void_p(264))),
                           (X.EX_OK, dict(n=0)), (X.EX_OK, dict(tokens=0))]:
        refuse(f, PROMPT, status, **change)


@pytest.mark.parametrize("scale", [0.0, float("inf"), float("nan"), 3e38])
def test_scales_that_are_refused(X, scale):
    """0 and what is not finite (3e38 times log2 e is not); prompts take positive scales only."""
    L = X.lib()
    for f, base in ((L.ex_paged_decode_q8, DECODE), (L.ex_tree_attention, TREE), (L.ex_prompt_attention, PROMPT)):
        refuse(f, base, X.EX_ERR_ARG, scale=scale)
    refuse(L.ex_prompt_attention, PROMPT, X.EX_ERR_ARG, scale=-0.1)


def test_launch_on_restores_the_current_device(X, monkeypatch):
    now = [1]
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "set_device", lambda d: now.__setitem__(0, d))
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 100 + d, raising=False)
    with X.launch_on(1) as stream:
        assert stream == 101 and now == [1]
    with pytest.raises(KeyError):
        with X.launch_on(3) as stream:
            assert stream == 103 and now == [3]
            raise KeyError
    assert now == [1]


def test_python_refusals(X):
    """CPU tensors and wrong types raise (there is no CPU path)."""
    from vllm_exact import kv_cache as C, paged_attn as A, prompt_attn as Q
    kc, vc, ks, vs = C.alloc_q8_cache(4, 16, 2, 64, torch.int8, "cpu")
    assert kc.shape == (4, 16, 2, 64) and ks.shape == (4, 2, 16) and kc.dtype == torch.int8
    x = torch.zeros(3, 2, 64, dtype=BF)
    i32 = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(TypeError):
        C.alloc_q8_cache(4, 16, 2, 64, torch.uint8, "cpu")
    with pytest.raises(ValueError, match="CUDA"):
        C.cache_write(x, x, kc, vc, ks, vs, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        C.cache_read(kc, vc, ks, vs, i32.view(1, 3), i32[:2], x, x)
    with pytest.raises(ValueError, match="CUDA"):
        A.paged_decode_q8(x, kc, vc, ks, vs, i32.view(3, 1), i32, 0.1, x, 3)
    with pytest.raises(ValueError, match="row for every request"):
        A.paged_decode_q8(x, kc, vc, ks, vs, i32.view(3, 1), i32, 0.1, x, 4)
    with pytest.raises(ValueError, match="CUDA"):
        A.tree_attention(x, kc, vc, i32.view(3, 1), i32, i32, 0.1, x, 4)
    with pytest.raises(ValueError, match="max_query_len"):
        A.tree_attention(x, kc, vc, i32.view(3, 1), i32, i32, 0.1, x, 65)
    with pytest.raises(TypeError, match="tree_mask"):
        A.tree_attention(x, kc, vc, i32.view(3, 1), i32, i32, 0.1, x, 4, tree_mask=i32)
    with pytest.raises(ValueError, match="CUDA"):
        Q.prompt_attention(x, x, x, i32, i32, 0.1)
    for bad, err in [(dict(ks=ks.half()), TypeError), (dict(vc=vc.view(torch.float8_e4m3fn)), TypeError),
                     (dict(ks=ks[:, :1]), ValueError), (dict(kc=kc[:2]), ValueError), (dict(kc=kc.float()), TypeError)]:
        t = dict(dict(kc=kc, vc=vc, ks=ks, vs=vs), **bad)
        with pytest.raises(err):
            C._check_cache(t["kc"], t["vc"], t["ks"], t["vs"], kc.device)


def test_plain_attention_matches_softmax():
    """The 64-bit comparison itself: torch's softmax where every row sees something, zeros where it sees nothing, and a
    bound that a value moved by one rounding step passes and a wrong scale does not."""
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(*s, generator=g).to(BF) for s in ((5, 4, 64), (9, 2, 64), (9, 2, 64)))
    seen = torch.ones(5, 9, dtype=torch.bool).tril(4)
    out, bound = S.attend(q, k, v, seen, 0.125, BF)
    for h in range(4):
        s = (q[:, h].double() @ k[:, h // 2].double().T * 0.125).masked_fill(~seen, -torch.inf)
        assert torch.allclose(out[:, h], torch.softmax(s, -1) @ v[:, h // 2].double(), atol=1e-12)
    assert bool(((out.float().to(BF).double() - out).abs() <= bound).all())
    wrong, _ = S.attend(q, k, v, seen, 0.15, BF)
    assert not bool(((wrong - out).abs() <= bound).all())
    seen[2] = False
    assert bool((S.attend(q, k, v, seen, 0.125, BF)[0][2] == 0).all())


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_plain_quantisation(dtype):
    x = torch.randn(50, 3, 64, generator=torch.Generator().manual_seed(1)).to(BF)
    codes, scale = S.quantise(x, dtype)
    back = S.values(codes, scale)
    step = scale.double().unsqueeze(-1) * (0.5 if dtype == torch.int8 else 2.0 ** -10) * 1.0001
    rel = 0.0 if dtype == torch.int8 else 2.0 ** -4 * 1.0001  # half a step of 3 mantissa bits, or of the smallest number
    assert bool(((back - x.double()).abs() <= step + rel * x.double().abs()).all())
    assert float(codes.float().abs().max()) == S.QMAX[dtype]
