"""Plain restatements of the 4-bit cache's operators: 64-bit attention with an error bound, the codec in
single IEEE FP32 steps, the boxes and the page choice in whole numbers."""

import math

import torch

PAGE, GROUP = 64, 128


def quantise(x):
    """FP32 rows [n, D] -> codes [n, D] (one per element), params [n, D/128, 2], each step one FP32 rounding."""
    g = x.float().reshape(x.shape[0], x.shape[1] // GROUP, GROUP)
    lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
    scale = torch.where((hi - lo).abs() <= 1e-8, torch.ones_like(lo), (hi - lo) / torch.full_like(lo, 15.0))
    code = torch.round((g - lo) / scale).clamp(0, 15).to(torch.uint8)
    return code.reshape(x.shape), torch.cat([scale, -lo / scale], -1)


def pack(code):
    return code[:, 0::2] | (code[:, 1::2] << 4)


def values32(code, params):
    g = code.float().reshape(code.shape[0], code.shape[1] // GROUP, GROUP)
    return ((g - params[..., 1:]) * params[..., :1]).reshape(code.shape)


def unpack(codes):
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2)


def random_cache(slots, d, dr, seed, device="cuda", spread=1.0):
    """Codes, params, rope of `slots` written slots; `spread`: how much the groups' scales differ."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(slots, d + dr, generator=g)
    x[:, :d] *= torch.exp(spread * torch.randn(slots, 1, generator=g)) * (0.25 + 1.5 * torch.rand(d, generator=g))
    x[:, :d] += 0.3 * torch.randn(d, generator=g)
    code, params = quantise(x[:, :d].to(torch.bfloat16))
    return [pack(code).to(device), params.contiguous().to(device), x[:, d:].to(torch.bfloat16).to(device)]


def attend(q, cache, table, lens, sm_scale):
    """FP64 result, lse and their error bounds, for q [B, T, H, W].

    Bounds: a token's weight is off by its logit's error (600 FP32 roundings of the sum of the terms' sizes, codes
    and zeros apart) and by 2^-11 where weight times scale is held in 11 bits; the output is rounded to BF16."""
    codes, params, rope = (x.cpu() for x in cache)
    q = q.cpu().double()
    b, t, h, w = q.shape
    d = codes.shape[1] * 2
    out, lse = torch.zeros(b, t, h, d, dtype=torch.float64), torch.full((b, t, h), -math.inf, dtype=torch.float64)
    tol_o, tol_l = torch.zeros_like(out), torch.zeros_like(lse)
    pool = codes.shape[0] // PAGE
    for i in range(b):
        n = int(min(lens[i], table.shape[1] * PAGE))
        pos = torch.arange(n)
        pages = table[i].cpu().long()[pos // PAGE]
        good = (pages >= 0) & (pages < pool)
        pos, at = pos[good], (pages * PAGE + pos % PAGE)[good]
        code = unpack(codes[at]).double()
        s, z = (params[at][..., k].double().repeat_interleave(GROUP, 1) for k in (0, 1))
        v, pe = (code - z) * s, rope[at].double()
        k = torch.cat([v, pe], 1)
        size = torch.cat([(code + z.abs()) * s.abs(), pe.abs()], 1)
        for j in range(t):
            ok = pos <= n - t + j
            if not bool(ok.any()):
                continue
            logit = q[i, j] @ k[ok].T * sm_scale
            lse[i, j] = torch.logsumexp(logit, 1)
            p = torch.softmax(logit, 1)
            out[i, j] = p @ v[ok]
            off = 600 * 2.0**-24 * (q[i, j].abs() @ size[ok].T * sm_scale).max(1).values + 2.0**-22 * (1 + logit.abs().max(1).values)
            tol_l[i, j] = off + 2.0**-20 * lse[i, j].abs()
            # weights at 11 bits; values 2^-25 of the largest lost; products summed in FP32
            tol_o[i, j] = 2.0**-9 * out[i, j].abs() + (2.0**-11 + 2.0**-13 + 2 * off)[:, None] * (p @ size[ok][:, :d]) + 1e-30
    return out, lse, tol_o, tol_l


def exponent(top):
    if not top > 0:
        return 0
    m, x = math.frexp(min(top, 3.402823466e38))
    return max(x - 6 if m > 127 / 128 else x - 7, -100)


def boxes(cache, page, count):
    """center, radius, exps of one page, in FP32 steps."""
    codes, params, rope = (x[page * PAGE : page * PAGE + count].cpu() for x in cache)
    v = torch.cat([values32(unpack(codes), params), rope.float()], 1)
    d = codes.shape[1] * 2
    lo, hi = v.min(0).values, v.max(0).values
    top = torch.maximum(lo.abs(), hi.abs())
    exps = [exponent(float(top[:d].max())), exponent(float(top[d:].max()))]
    unit = torch.tensor([2.0 ** -exps[0]] * d + [2.0 ** -exps[1]] * (v.shape[1] - d))
    center = torch.round((lo + hi) * 0.5 * unit)
    radius = torch.ceil(torch.maximum(hi * unit - center, center - lo * unit))
    return center.to(torch.int8), radius.to(torch.uint8), exps


def choose(q, box, table, n_tokens, budget, keep_first, keep_last):
    """The kept indexes of one request's pages, in order; q [H, W]."""
    held = -(-n_tokens // PAGE)
    if held <= budget:
        return list(range(held))
    center, radius, exps = (x.cpu() for x in box)
    q = q.cpu().double()
    d = q.shape[1] - {544: 32, 576: 64, 288: 32, 320: 64}[q.shape[1]]
    parts = (slice(0, d), slice(d, q.shape[1]))
    scores = []
    e_q = [exponent(float(q[:, p].abs().max())) for p in parts]
    q8 = [torch.round(q[:, p] * 2.0 ** -e) for p, e in zip(parts, e_q)]
    for j in range(held):
        page = int(table[j])
        if j < keep_first or j >= held - keep_last:
            scores.append(math.inf)
        elif page < 0 or page >= center.shape[0]:
            scores.append(-math.inf)
        else:
            s = 0
            for p, x, e, k in zip(parts, q8, e_q, (0, 1)):
                whole = x @ center[page, p].double() + x.abs() @ radius[page, p].double()
                s = s + (whole * 2.0 ** (e + int(exps[page, k]))).float()
            scores.append(float(s.max()))
    order = sorted(range(held), key=lambda j: (-scores[j], j))
    return sorted(order[:budget])
