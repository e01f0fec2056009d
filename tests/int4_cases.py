"""What the tests of the 4-bit cache's ranges share: requests over a shuffled pool, one call of the attention, and
attention in 64 bits with a bound that follows each token's own roundings."""

import math

import torch

import int4_reference as ref
from mla_kv_quant_b200 import int4

SM = 192**-0.5


def pool_for(lens, seed):
    """A shuffled page table for the lengths -> table [B, max_pages] (CPU), pages of the pool."""
    counts = [-(-n // 64) for n in lens]
    order = torch.randperm(sum(counts) + 2, generator=torch.Generator().manual_seed(seed)).int()
    table = torch.full((len(lens), max(max(counts), 1)), -1, dtype=torch.int32)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at : at + c]
        at += c
    return table, sum(counts) + 2


def slots_of(table, i, n):
    pos = torch.arange(n)
    return table[i].long()[pos // 64] * 64 + pos % 64


def stored(rows, pe, table, lens, pages):
    """The cache that holds rows[i] (FP32 [n, D]) and pe[i] as request i; empty elsewhere."""
    d, dr = rows[0].shape[1], pe[0].shape[1]
    codes, params = torch.zeros(pages * 64, d // 2, dtype=torch.uint8), torch.zeros(pages * 64, d // 128, 2)
    rope = torch.zeros(pages * 64, dr, dtype=torch.bfloat16)
    for i, n in enumerate(lens):
        at = slots_of(table, i, n)
        code, params[at] = ref.quantise(rows[i])
        codes[at], rope[at] = ref.pack(code), pe[i].bfloat16()
    return [codes.cuda(), params.cuda(), rope.cuda()]


def decode(q, cache, table, lens, sm_scale=SM):
    """out and lse of one call, on the CPU in 64 bits; q [B, T, H, W]."""
    view = int4.Int4View(*cache)
    b, t, h, _ = q.shape
    out = torch.full((b, t, h, view.latent_dim), 7.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((b, t, h), 7.0, device="cuda")
    ws = int4.Workspace(view, b, t, h, table.shape[1])
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    int4.decode(q.cuda(), view, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), sm_scale, out, lse, ws, err)
    assert err.item() == 0
    return out.cpu().double(), lse.cpu().double()


def attend(q, cache, table, lens, sm_scale=SM):
    """FP64 out, lse and bounds of their errors.

    A token's logit is off by up to 600 FP32 roundings of the sum of its terms' sizes (codes and zeros apart) and a
    relative 2^-22; its weight times its group's scale is held in 11 bits, or to 2^-26 of the row's largest such
    product, on codes up to 15; 2^-13 for FP32 sums.  The output's rounding to BF16 comes on top (`rounds`)."""
    codes, params, rope = (x.cpu() for x in cache)
    q = q.cpu().double()
    b, t, h, _ = q.shape
    d = codes.shape[1] * 2
    out, lse = torch.zeros(b, t, h, d, dtype=torch.float64), torch.full((b, t, h), -math.inf, dtype=torch.float64)
    tol_o, tol_l = torch.zeros_like(out), torch.zeros_like(lse)
    for i, n in enumerate(lens):
        for j in range(t):
            seen = n - t + j + 1
            if seen <= 0:
                continue
            at = slots_of(table, i, seen)
            code = ref.unpack(codes[at]).double()
            s, z = (params[at][..., k].double().repeat_interleave(128, 1) for k in (0, 1))
            v, pe = (code - z) * s, rope[at].double()
            size = (code + z.abs()) * s.abs()
            logit = q[i, j] @ torch.cat([v, pe], 1).T * sm_scale
            off = 600 * 2.0**-24 * (q[i, j].abs() @ torch.cat([size, pe.abs()], 1).T * sm_scale) + 2.0**-22 * (1 + logit.abs())
            p = torch.softmax(logit, 1)
            lse[i, j], out[i, j] = torch.logsumexp(logit, 1), p @ v
            tol_l[i, j] = torch.logsumexp(logit + off, 1) - lse[i, j] + 2.0**-20 * lse[i, j].abs()
            coded = s * (code.view(seen, -1, 128).amax(-1) > 0).repeat_interleave(128, 1)
            largest = (p[:, :, None] * coded[None]).amax(1)
            tol_o[i, j] = (p * (torch.expm1(off + tol_l[i, j][:, None]) + 2.0**-11 + 2.0**-13)) @ size + seen * 2.0**-22 * largest + 1e-30
    return out, lse, tol_o, tol_l


def rounds(out, o, tol):
    """Whether each BF16 output is the rounding of a value within tol of o (rounding keeps the order)."""
    return (out >= (o - tol).bfloat16().double()) & (out <= (o + tol).bfloat16().double())


def check(q, cache, table, lens, sm_scale=SM, rows=slice(None)):
    """The kernel's out and lse of the query tokens `rows` against 64 bits."""
    out, lse = decode(q, cache, table, lens, sm_scale)
    o, l, tol_o, tol_l = attend(q, cache, table, lens, sm_scale)
    assert ((lse - l).abs() <= tol_l)[:, rows].all(), float((lse - l).abs()[:, rows].max())
    assert rounds(out, o, tol_o)[:, rows].all(), float(((out - o).abs() / tol_o.clamp(min=1e-300))[:, rows].max())
    return out, lse
