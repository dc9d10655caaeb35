"""Plain 64-bit implementations and error bounds for the tests of the 8-bit cache and the attention around it."""
import math

import torch

QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def quantise(x, dtype):
    """Codes and scales of rows of the last dimension, every step rounded in float32 as IEEE 754 says (on the CPU)."""
    x = x.detach().cpu().float()
    amax = x.abs().amax(-1, keepdim=True)  # propagates NaN
    scale = amax / torch.full_like(amax, QMAX[dtype])
    y = torch.where((scale > 0) & torch.isfinite(scale), x / scale, torch.zeros_like(x))
    y = torch.nan_to_num(y, nan=0.0).clamp(-QMAX[dtype], QMAX[dtype])
    return (y.round() if dtype == torch.int8 else y).to(dtype), scale.squeeze(-1)


def values(codes, scale):
    return codes.cpu().float().double() * scale.cpu().double().unsqueeze(-1)


def attend(q, k, v, seen, scale, dtype, q8=False):
    """(out, bound) in float64 of one sequence: q (T, H, D), k and v (L, KV, D) the numbers that the cache stands for,
    seen (T, L). The bound of |computed - out|, element by element, adds up what the kernels round:
      * the output to its type: half a step of |out|;
      * every weight to 16 bits: half a step of sum p|v| (A below), or 2^-25 of the largest weight times |v| where a
        float16 weight is below the normal numbers (q8: every weight is float16);
      * float32 sums over D and over the keys (2^-23 a step, truncating tensor cores included), the rescalings of the
        blocks and segments, and 2^x to 2^-22 with its argument rounded to 2^-23 of |x|; an error d of the
        scores changes a normalised weight by at most 2 d of itself (prompts: an eighth of the weights by a polynomial of
        relative error 2.7e-6; twice that is 46 steps, among the 128 that are added to the L of the sums);
      * q8: query elements below 2^-14 of their row's largest keep 2^-25 of it."""
    q, k, v = q.detach().cpu().double(), k.detach().cpu().double(), v.detach().cpu().double()
    seen = seen.cpu()
    T, H, D = q.shape
    L, KV, _ = k.shape
    if L == 0 or T == 0:
        return torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, D, dtype=torch.float64)
    G = H // KV
    kh, vh = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    s = torch.einsum("thd,lhd->htl", q, kh) * scale
    s_abs = torch.einsum("thd,lhd->htl", q.abs(), kh.abs()) * scale
    hide = ~seen[None]
    s = s.masked_fill(hide, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m > -math.inf, m, torch.zeros_like(m))).masked_fill(hide, 0.0)
    l = p.sum(-1, keepdim=True)
    p = torch.where(l > 0, p / l.clamp(min=1e-300), torch.zeros_like(p))
    out = torch.einsum("htl,lhd->thd", p, vh)
    A = torch.einsum("htl,lhd->thd", p, vh.abs())
    s_abs = s_abs.masked_fill(hide, 0.0)
    ds = s_abs.amax(-1) * ((D + 8) * 2.0 ** -23) + 2.0 ** -21
    if q8:
        ds = ds + D * 2.0 ** -25 * q.abs().amax(-1).T * kh.abs().amax((0, 2))[:, None] * scale * 2
    half = HALF_STEP[torch.float16 if q8 else dtype]
    rel = half + 2 * ds.T[..., None] + (L + 128) * 2.0 ** -23
    bound = HALF_STEP[dtype] * out.abs() + A * rel * 1.01 + 1e-30
    if q8 or dtype == torch.float16:
        # at most one unnormalised weight in 2^-25 steps per key; the largest weight is at least 1 before division by l
        low = 2.0 ** -24 * torch.einsum("tl,lhd->thd", seen.double(), vh.abs())
        if q8:
            low = 2.0 ** -24 * seen.double().sum(-1)[:, None, None] * vh.abs().amax((0, 2))[None, :, None]
        bound = bound + low / l.permute(1, 0, 2).clamp(min=1.0)
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25  # outputs below the normal numbers
    return out, bound
