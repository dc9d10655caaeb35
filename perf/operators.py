"""The operators of an attention layer that serves from an 8-bit or 16-bit paged cache: what is measured of them.

Five operators, as one serving step uses them:

* ``write``   new keys and values quantised into an 8-bit paged cache (int8 or e4m3 codes, one float32 scale for each
              token and head), optionally with the values that the cache now stands for;
* ``read``    whole sequences of that cache read back as packed 16-bit rows;
* ``decode``  one query token per sequence over the 8-bit cache;
* ``tree``    up to 64 drafted tokens per sequence over a 16-bit or 8-bit cache, under an ancestor mask;
* ``prompt``  causal attention of packed prompts of different lengths with grouped heads, over keys that may start
              before the queries.

``own`` selects the framework's kernels; otherwise the plain form in elementary torch operations runs.
"""
import math
import os
import sys

import torch

_PACKAGE = os.path.join(os.getcwd(), "vllm-exact_b200")  # the repository's root is the working folder
if _PACKAGE not in sys.path:
    sys.path.insert(0, _PACKAGE)

own = False

QMAX = {"int8": 127.0, "e4m3": 448.0}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
REAL = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ----------------------------------------------------------------------------------------------------------- cases
def listed():
    """Head layouts, page sizes and batches are the repository's own: 32 query heads over 8 KV heads of size 128 with
    pages of 16, 16 over 4 of size 256 with pages of 528, decode batches of 256 x 1K, 64 x 8K and 16 x 16K."""
    return [
        # one decode step of a small batch: latency of the smallest cache write
        dict(name="write decode step", op="write", code="int8", real="bf16", tokens=16, KV=8, D=128, page=16, back=False),
        # a long prompt's keys and values, with the rounded values that its own attention then reads
        dict(name="write prompt", op="write", code="e4m3", real="bf16", tokens=16000, KV=8, D=128, page=16, back=True),
        # a conversation is continued: one cached sequence comes back
        dict(name="read one", op="read", code="e4m3", real="bf16", n=1, lo=777, hi=777, KV=8, D=128, page=16),
        # a batch of conversations is continued, in the large head size and its long pages
        dict(name="read batch", op="read", code="int8", real="bf16", n=48, lo=100, hi=2100, KV=4, D=256, page=528),
        # a single user's chat: latency of one decode call
        dict(name="decode single", op="decode", code="e4m3", real="bf16", n=1, lo=1000, hi=1000, H=32, KV=8, D=128, page=16),
        # the repository's decode batches, 25 % around the nominal context
        dict(name="decode b256 1K", op="decode", code="e4m3", real="bf16", n=256, lo=768, hi=1280, H=32, KV=8, D=128, page=16),
        dict(name="decode b16 16K", op="decode", code="int8", real="bf16", n=16, lo=12288, hi=20480, H=32, KV=8, D=128, page=16),
        # a small draft tree for one user, large head size
        dict(name="tree single", op="tree", code="", real="bf16", n=1, lo=700, hi=700, draft=8, H=16, KV=4, D=256, page=528),
        # a served batch that verifies 16 drafted tokens per sequence
        dict(name="tree b64 8K", op="tree", code="", real="bf16", n=64, lo=6144, hi=10240, draft=16, H=32, KV=8, D=128, page=16),
        # the same on an 8-bit cache with deep contexts and small trees
        dict(name="tree b16 16K e4m3", op="tree", code="e4m3", real="bf16", n=16, lo=12288, hi=20480, draft=7, H=32, KV=8, D=128, page=16),
        # three packed prompts of very different lengths, one of them a single token
        dict(name="prompt short ragged", op="prompt", real="bf16", n=3, lo=1, hi=333, before=0, H=32, KV=8, D=128),
        # packed long prompts, the largest work here
        dict(name="prompt long", op="prompt", real="bf16", n=3, lo=2048, hi=8192, before=0, H=32, KV=8, D=128),
    ]


HEADS = [(32, 8, 128), (16, 4, 256), (16, 2, 128), (12, 4, 64), (8, 1, 64), (6, 6, 128), (16, 1, 128)]
PAGES = [16, 32, 528, 24]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["write", "read", "decode", "decode", "tree", "tree", "prompt", "prompt"])
    H, KV, D = rng.choice(HEADS)
    c = dict(op=op, real=rng.choice(["bf16", "bf16", "fp16"]), KV=KV, D=D)
    if op == "write":
        return dict(c, code=rng.choice(["int8", "e4m3"]), tokens=_log(rng, 1, 16000), page=rng.choice(PAGES),
                    back=rng.random() < 0.5)
    if op == "prompt":
        # at most the listed batch's products; keys may start before the queries (a continued conversation)
        n, hi = _log(rng, 1, 24), _log(rng, 1, 6000)
        before = rng.choice([0, 0, rng.randrange(1, hi // 2 + 2)])
        n = max(1, min(n, int(7.5e11 / (4 * H * D * hi * (before + hi / 2 + 1)))))
        return dict(c, n=n, lo=_log(rng, 1, hi), hi=hi, before=before, H=H)
    c["page"] = rng.choice(PAGES)
    ctx = _log(rng, 2, 16000)
    n = _log(rng, 1, max(1, min(256, 250000 * 8 * 128 // (ctx * KV * D))))
    lo, hi = max(1, ctx * 3 // 4), ctx * 5 // 4
    if op == "read":
        n = max(1, min(n, 48 * 2100 * 4 * 256 // (hi * KV * D)))
        return dict(c, code=rng.choice(["int8", "e4m3"]), n=n, lo=lo, hi=hi)
    if op == "decode":
        return dict(c, code=rng.choice(["int8", "e4m3"]), n=n, lo=lo, hi=hi, H=H)
    draft = _log(rng, 1, 64)
    n = max(1, min(n, 64 * 16 * 32 * 10240 // (draft * H * hi)))
    return dict(c, code=rng.choice(["", "int8", "e4m3"]), n=n, lo=lo, hi=hi, draft=draft, H=H)


def _lengths(c):
    """n lengths spread evenly over [lo, hi], in an order that is not sorted."""
    n, lo, hi = c["n"], c["lo"], c["hi"]
    v = [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]
    step = next(s for s in (7, 5, 3, 11, 13, 1) if math.gcd(s, n) == 1)
    return [v[(i * step) % n] for i in range(n)]


def _drafts(c):
    """Drafted tokens of each sequence: `draft` for most, fewer for every third; a draft is part of its sequence."""
    full = c["draft"]
    return [min(L, full if i % 3 else max(1, full - full // 3)) for i, L in enumerate(_lengths(c))]


# ------------------------------------------------------------------------------------------------------------ work
def work(case):
    """Each input once, each output once; attention's two products over the keys that a row sees."""
    c, op = case, case["op"]
    KV, D = c["KV"], c["D"]
    row8, row16 = KV * (D + 4) * 2, KV * D * 2 * 2  # keys and values of one token: codes with scales, 16-bit
    if op == "write":
        return {"bytes": c["tokens"] * (row16 + row8 + 8 + (row16 if c["back"] else 0)), "flops": c["tokens"] * KV * D * 2 * 3}
    L = _lengths(c)
    if op == "read":
        return {"bytes": sum(L) * (row8 + row16) + sum(-(-x // c["page"]) for x in L) * 4, "flops": sum(L) * KV * D * 2}
    H = c["H"]
    if op == "prompt":
        b = c["before"]
        pairs = sum(x * b + x * (x + 1) // 2 for x in L)
        return {"bytes": sum(L) * H * D * 2 * 2 + sum(x + b for x in L) * row16, "flops": 4 * D * H * pairs}
    T = _drafts(c) if op == "tree" else [1] * c["n"]
    per_key = row8 if c["code"] else row16
    # a drafted token sees the context and, on average, about half of the drafts before it
    pairs = sum(t * (x - t) + t * (t + 1) // 2 for x, t in zip(L, T))
    return {"bytes": sum(L) * per_key + sum(T) * (H * D * 2 * 2 + (8 if op == "tree" else 0)) + sum(-(-x // c["page"]) for x in L) * 4,
            "flops": 4 * D * H * pairs}


# --------------------------------------------------------------------------------------------------------- prepare
def _quantise(x, code):
    """Codes and scales of rows of the last dimension: scale = max|x| / QMAX, code = x / scale rounded to nearest."""
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True)
    scale = amax / torch.full_like(amax, QMAX[code])  # a tensor, so that the division is not made a product
    y = torch.where(scale > 0, x / scale, torch.zeros_like(x)).clamp(-QMAX[code], QMAX[code])
    return (y.round() if code == "int8" else y).to(CODE[code]), scale.squeeze(-1)


def _cumulative(v, dev):
    return torch.tensor([0] + list(v), device=dev).cumsum(0).to(torch.int32)


def _kv(g, dev, shape, real):
    """Keys or values as projections give them: normal, with a few channels that are ten times larger."""
    x = torch.randn(shape, generator=g, device=dev)
    gain = torch.where(torch.rand(shape[-2:], generator=g, device=dev) < 0.02, 10.0, 1.0)
    return (x * gain).to(REAL[real])


def _cache(c, g, dev, L):
    """A paged cache that holds sequences of these lengths in randomly placed pages, and its block table."""
    KV, D, P = c["KV"], c["D"], c["page"]
    wide = -(-max(L) // P)
    blocks = c["n"] * wide + 3
    s = {"table": torch.randperm(blocks, generator=g, device=dev)[: c["n"] * wide].view(c["n"], wide).to(torch.int32)}
    for k in ("key", "value"):
        x = _kv(g, dev, (blocks, P, KV, D), c["real"])
        if c["code"]:
            q, scale = _quantise(x, c["code"])
            s[k], s[k + "_scale"] = q, scale.transpose(1, 2).contiguous()  # scales are (block, KV head, place in page)
        else:
            s[k], s[k + "_scale"] = x, None
    return s


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    KV, D, real = c["KV"], c["D"], REAL[c["real"]]
    s = {"op": c["op"], "code": c.get("code", ""), "D": D, "KV": KV, "page": c.get("page", 0), "real": real,
         "scale": D ** -0.5, "n": c.get("n", 0)}
    if c["op"] == "write":
        T = c["tokens"]
        blocks = -(-T // c["page"]) + 5
        s["slots"] = torch.randperm(blocks * c["page"], generator=g, device=dev)[:T].to(torch.int64)
        if T > 4:
            s["slots"][T // 2] = -1  # a padded token of the batch: not written
        both = _kv(g, dev, (T, 2, KV, D), c["real"])  # slices of one projection's output
        s["k"], s["v"] = both[:, 0], both[:, 1]
        for k in ("key", "value"):
            s[k] = torch.zeros(blocks, c["page"], KV, D, device=dev).to(CODE[c["code"]])
            s[k + "_scale"] = torch.zeros(blocks, KV, c["page"], device=dev)
            s[k + "_back"] = torch.zeros(T, KV, D, device=dev, dtype=real) if c["back"] else None
        return s
    L = _lengths(c)
    s["most"] = max(L)
    if c["op"] == "prompt":
        b, H = c["before"], c["H"]
        s["q"] = torch.randn(sum(L), H, D, generator=g, device=dev).to(real)
        both = _kv(g, dev, (sum(L) + c["n"] * b, 2, KV, D), c["real"])
        s["k"], s["v"] = both[:, 0], both[:, 1]
        s["cu_q"], s["cu_k"] = _cumulative(L, dev), _cumulative([x + b for x in L], dev)
        s["most_k"] = s["most"] + b
        s["out"] = torch.empty_like(s["q"])
        return s
    s |= _cache(c, g, dev, L)
    s["lens"] = torch.tensor(L, device=dev, dtype=torch.int32)
    if c["op"] == "read":
        s["cu"] = _cumulative(L, dev)
        for k in ("key", "value"):
            s[k + "_back"] = torch.empty(sum(L), KV, D, device=dev, dtype=real)
        return s
    T = _drafts(c) if c["op"] == "tree" else [1] * c["n"]
    s["q"] = torch.randn(sum(T), c["H"], D, generator=g, device=dev).to(real)
    s["out"] = torch.empty_like(s["q"])
    if c["op"] == "tree":
        s["draft"] = max(T)
        s["cu"] = _cumulative(T, dev)
        # every drafted token's parent is a token before it (or the context's last one); it sees its ancestors and itself
        parent = [[-1] + [int(x) for x in (torch.rand(t - 1, generator=g, device=dev) * torch.arange(1, t, device=dev)).tolist()] if t > 1 else [-1] for t in T]
        words = []
        for p in parent:
            seen = []
            for i, j in enumerate(p):
                seen.append((seen[j] if j >= 0 else 0) | (1 << i))
            words += [w - (1 << 64) if w >> 63 else w for w in seen]
        s["mask"] = torch.tensor(words, device=dev, dtype=torch.int64)
    return s


# ------------------------------------------------------------------------------------------------------------- run
def run(state):
    s = state
    if own:
        from vllm_exact import kv_cache, paged_attn, prompt_attn
        if s["op"] == "write":
            kv_cache.cache_write(s["k"], s["v"], s["key"], s["value"], s["key_scale"], s["value_scale"], s["slots"],
                                 key_out=s["key_back"], value_out=s["value_back"])
            return _written(s)
        if s["op"] == "read":
            kv_cache.cache_read(s["key"], s["value"], s["key_scale"], s["value_scale"], s["table"], s["cu"],
                                s["key_back"], s["value_back"])
            return [s["key_back"], s["value_back"]]
        if s["op"] == "decode":
            return paged_attn.paged_decode_q8(s["q"], s["key"], s["value"], s["key_scale"], s["value_scale"],
                                              s["table"], s["lens"], s["scale"], s["out"], s["n"],
                                              max_seq_len=s["most"])
        if s["op"] == "tree":
            return paged_attn.tree_attention(s["q"], s["key"], s["value"], s["table"], s["lens"], s["cu"], s["scale"],
                                             s["out"], s["draft"], tree_mask=s["mask"], key_scale=s["key_scale"],
                                             value_scale=s["value_scale"], max_seq_len=s["most"])
        return prompt_attn.prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], s["scale"], out=s["out"])
    return {"write": _plain_write, "read": _plain_read, "decode": _plain_decode, "tree": _plain_tree,
            "prompt": _plain_prompt}[s["op"]](s)


def _written(s):
    """The cache after the call, and the values that its new rows stand for where they were asked for."""
    got = {"key": s["key"], "value": s["value"], "key_scale": s["key_scale"], "value_scale": s["value_scale"]}
    if s["key_back"] is not None:
        got |= {"key_back": s["key_back"], "value_back": s["value_back"]}
    return got


def _plain_write(s):
    """Rows of slot -1 are sent to a spare row behind the cache, which is then dropped: no choice on the host."""
    slots = s["slots"]
    total = s["key"].shape[0] * s["page"]
    to = torch.where(slots >= 0, slots, torch.full_like(slots, total))
    _plain_store(s, s["k"], "key", to, total)
    _plain_store(s, s["v"], "value", to, total)
    return _written(s)


def _plain_store(s, x, k, to, total):
    q, scale = _quantise(x, s["code"])
    rows = torch.cat([s[k].view(torch.uint8).view(total, s["KV"], -1), q[:1].view(torch.uint8)])
    rows[to] = q.view(torch.uint8)
    s[k].view(torch.uint8).copy_(rows[:total].view(s[k].shape))
    flat = torch.cat([s[k + "_scale"].transpose(1, 2).reshape(total, s["KV"]), scale[:1]])
    flat[to] = scale
    s[k + "_scale"].copy_(flat[:total].view(-1, s["page"], s["KV"]).transpose(1, 2))
    if s[k + "_back"] is not None:
        s[k + "_back"].copy_(q.float() * scale.unsqueeze(-1))


def _gathered(s, k):
    """Keys or values of every sequence, float32: (sequence, token, KV head, D), padded to whole pages."""
    t = s["table"].long()
    x = s[k]
    if s[k + "_scale"] is None:
        x = x[t].float()
    else:
        x = x.view(torch.uint8)[t].view(x.dtype).float() * s[k + "_scale"].transpose(1, 2)[t].unsqueeze(-1)
    return x.flatten(1, 2)


def _place(cu, rows):
    """Sequence and position in it of each packed row."""
    r = torch.arange(rows, device=cu.device)
    b = torch.searchsorted(cu[1:].long(), r, right=True)
    return b, r - cu.long()[b]


def _plain_read(s):
    b, i = _place(s["cu"], s["key_back"].shape[0])
    blk, i = s["table"].long()[b, i // s["page"]], i % s["page"]
    _plain_take(s, "key", blk, i)
    _plain_take(s, "value", blk, i)
    return [s["key_back"], s["value_back"]]


def _plain_take(s, k, blk, i):
    x = s[k].view(torch.uint8)[blk, i].view(s[k].dtype).float()
    s[k + "_back"].copy_(x * s[k + "_scale"][blk, :, i].unsqueeze(-1))


def _attend(q, k, v, seen, scale):
    """softmax(scale q k^T) v in float32: q (n, T, H, D), k and v (n, L, KV, D), seen (n, T, L); a row that sees no
    key gives zeros."""
    n, T, H, D = q.shape
    KV = k.shape[2]
    q = q.view(n, T, KV, H // KV, D).permute(0, 2, 3, 1, 4).reshape(n, KV, -1, D)
    s = torch.matmul(q * scale, k.permute(0, 2, 3, 1)).view(n, KV, H // KV, T, -1)
    s.masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    s.sub_(torch.where(m > -math.inf, m, torch.zeros_like(m))).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(n, KV, -1, s.shape[-1]), v.permute(0, 2, 1, 3)).view(n, KV, H // KV, T, D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.permute(0, 3, 1, 2, 4).reshape(n, T, H, D)


def _plain_decode(s):
    k, v = _gathered(s, "key"), _gathered(s, "value")
    seen = torch.arange(k.shape[1], device=k.device) < s["lens"].long()[:, None, None]
    s["out"].copy_(_attend(s["q"].float().unsqueeze(1), k, v, seen, s["scale"]).squeeze(1))
    return s["out"]


def _padded(x, cu, most):
    """Packed rows as (sequence, position, ...), and which positions are rows of the sequence."""
    i = torch.arange(most, device=x.device)
    at = cu[:-1].long()[:, None] + i
    real = at < cu[1:].long()[:, None]
    return x[at.clamp(max=x.shape[0] - 1)].float(), real


def _plain_tree(s):
    k, v = _gathered(s, "key"), _gathered(s, "value")
    q, real = _padded(s["q"], s["cu"], s["draft"])
    first = (s["lens"].long() - (s["cu"][1:] - s["cu"][:-1]).long())[:, None, None]  # the first drafted token's place
    word = s["mask"][(s["cu"][:-1].long()[:, None] + torch.arange(s["draft"], device=q.device)).clamp(max=s["mask"].shape[0] - 1)]
    at = torch.arange(k.shape[1], device=q.device)
    bit = (word[:, :, None] >> (at - first).clamp(0, 63)) & 1
    seen = (at < first) | ((at < s["lens"].long()[:, None, None]) & (bit == 1))
    o = _attend(q, k, v, seen & real[:, :, None], s["scale"])
    b, i = _place(s["cu"], s["q"].shape[0])
    s["out"].copy_(o[b, i])
    return s["out"]


def _plain_prompt(s):
    q, _ = _padded(s["q"], s["cu_q"], s["most"])
    k, real = _padded(s["k"], s["cu_k"], s["most_k"])
    v, _ = _padded(s["v"], s["cu_k"], s["most_k"])
    before = ((s["cu_k"][1:] - s["cu_k"][:-1]) - (s["cu_q"][1:] - s["cu_q"][:-1])).long()
    i = torch.arange(q.shape[1], device=q.device)[:, None]
    seen = (torch.arange(k.shape[1], device=q.device) <= before[:, None, None] + i) & real[:, None]
    o = _attend(q, k, v, seen, s["scale"])
    b, i = _place(s["cu_q"], s["q"].shape[0])
    s["out"].copy_(o[b, i])
    return s["out"]


# ----------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """The definitions in 64 bits, sequence by sequence; codes have no value between them, so none is given."""
    c, s = case, prepare(case, seed)
    if c["op"] == "write":
        got = {"key": None, "value": None}
        total, KV = s["key"].shape[0] * c["page"], c["KV"]
        for x, k in ((s["k"], "key"), (s["v"], "value")):
            x = x.double()
            scale = x.abs().amax(-1) / QMAX[c["code"]]
            flat = torch.zeros(total, KV, dtype=torch.float64, device=x.device)
            kept = s["slots"] >= 0
            flat[s["slots"][kept]] = scale[kept]
            got[k + "_scale"] = flat.view(-1, c["page"], KV).transpose(1, 2)
            if c["back"]:
                y = x / scale.unsqueeze(-1)
                # e4m3: 3 bits behind the leading one, the smallest step is 2^-9
                step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3) if c["code"] == "e4m3" else torch.ones_like(y)
                got[k + "_back"] = torch.round(y / step) * step * scale.unsqueeze(-1)
        return got
    L = _lengths(c)

    def cached(k, b):
        x = s[k][s["table"][b].long().cpu().tolist()] if not c["code"] else s[k].view(torch.uint8)[s["table"][b].long()].view(s[k].dtype)
        x = x.double()
        if c["code"]:
            x = x * s[k + "_scale"].double()[s["table"][b].long()].permute(0, 2, 1).unsqueeze(-1)
        return x.reshape(-1, c["KV"], c["D"])[: L[b]]

    if c["op"] == "read":
        return [torch.cat([cached(k, b) for b in range(c["n"])]) for k in ("key", "value")]
    G = c["H"] // c["KV"]
    rows = []
    for b in range(c["n"]):
        if c["op"] == "prompt":
            before = c["before"]
            k, v = (s[x][int(s["cu_k"][b]): int(s["cu_k"][b + 1])].double() for x in ("k", "v"))
            q = s["q"][int(s["cu_q"][b]): int(s["cu_q"][b + 1])].double()
            seen = torch.ones(q.shape[0], k.shape[0], dtype=torch.bool, device=q.device).tril(before)
        else:
            k, v = cached("key", b), cached("value", b)
            if c["op"] == "decode":
                q, seen = s["q"][b: b + 1].double(), torch.ones(1, L[b], dtype=torch.bool, device=k.device)
            else:
                lo, hi = int(s["cu"][b]), int(s["cu"][b + 1])
                q = s["q"][lo:hi].double()
                bits = torch.tensor([[(w >> j) & 1 for j in range(hi - lo)] for w in s["mask"][lo:hi].tolist()], device=k.device) == 1
                seen = torch.cat([torch.ones(hi - lo, L[b] - (hi - lo), dtype=torch.bool, device=k.device), bits], 1)
        heads = []
        for h in range(c["H"]):
            z = (q[:, h] @ k[:, h // G].T) * s["scale"]
            heads.append(torch.softmax(z.masked_fill(~seen, -math.inf), -1) @ v[:, h // G])
        rows.append(torch.stack(heads, 1))
    return torch.cat(rows)
