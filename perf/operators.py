"""What is measured of the 4-bit latent cache: storing it, attending over it, and attending over the pages of it that
a cheap score selects.

The cache of one layer is paged, 64 slots to a page:
  codes  uint8 [slots, D/2]       two codes a byte, element 2i in the low half of byte i
  params f32   [slots, D/128, 2]  (scale, zero) of each 128 elements; an element stands for (code - zero) * scale
  rope   bf16  [slots, Dr]        the key's rotary part, unquantised
and beside it, for the page selection, one box per page (see `plain_boxes`).

`run` is the plain form (elementary torch operations in 32 bits) unless `own` is set; then it makes the calls that a
user makes of mla_kv_quant_b200.int4.
"""
import math
import random

import torch

own = False

PAGE, GROUP, LEVELS = 64, 128, 15
LOG2E = 1.4426950408889634

# (latent dim, rotary dim, heads) of the decode shapes that the framework builds
SHAPES = {"d512_h16": (512, 64, 16), "d512_h8": (512, 64, 8), "d256_h40": (256, 32, 40), "d256_h16": (256, 32, 16)}


def listed():
    return [
        # The rows that one decode step of 64 requests appends, read back: launch latency.
        {"name": "store_step", "op": "store", "shape": "d512_h16", "rows": 64, "dtype": "bf16"},
        # A prefill of 8 x 16384 tokens, stored from the strided halves of the down-projection and read back.
        {"name": "store_prefill", "op": "store", "shape": "d512_h16", "rows": 131072, "dtype": "bf16"},
        # 64 requests of about 16K tokens: the ordinary serving step.
        {"name": "attend_b64_16k", "op": "attend", "shape": "d512_h16", "batch": 64, "ctx": 16384, "ragged": 0.1, "q_len": 1, "lens_seed": 1},
        # 128 requests of 8K tokens, 40 heads over a 256-wide latent.
        {"name": "attend_b128_8k", "op": "attend", "shape": "d256_h40", "batch": 128, "ctx": 8192, "ragged": 0.0, "q_len": 1, "lens_seed": 2},
        # One request of 128K tokens: the work has to be split over its length.
        {"name": "attend_b1_128k", "op": "attend", "shape": "d512_h16", "batch": 1, "ctx": 131072, "ragged": 0.0, "q_len": 1, "lens_seed": 3},
        # A few short requests, some just begun, one without a token: latency.
        {"name": "attend_short", "op": "attend", "shape": "d512_h8", "batch": 5, "ctx": 700, "ragged": 1.0, "q_len": 1, "lens_seed": 4},
        # Four drafted tokens of each request verified at once, causal among themselves.
        {"name": "attend_verify", "op": "attend", "shape": "d512_h16", "batch": 16, "ctx": 8192, "ragged": 0.5, "q_len": 4, "lens_seed": 5},
        # The boxes of the pages that a decode step of 64 requests wrote to.
        {"name": "boxes_step", "op": "boxes", "shape": "d512_h16", "pages": 64, "full": False},
        # The boxes of a prefill of 8 x 16384 tokens.
        {"name": "boxes_prefill", "op": "boxes", "shape": "d512_h16", "pages": 2048, "full": True},
        # 64 requests of about 16K tokens, each attending to 32 of its 256 pages.
        {"name": "sparse_b64_16k", "op": "sparse", "shape": "d512_h16", "batch": 64, "ctx": 16384, "ragged": 0.1, "budget": 32, "lens_seed": 6},
        # One request of 128K tokens attending to 64 of its 2048 pages.
        {"name": "sparse_b1_128k", "op": "sparse", "shape": "d512_h16", "batch": 1, "ctx": 131072, "ragged": 0.0, "budget": 64, "lens_seed": 7},
        # 128 requests of up to 8K tokens, 40 heads, an odd budget.
        {"name": "sparse_b128_8k", "op": "sparse", "shape": "d256_h40", "batch": 128, "ctx": 8192, "ragged": 0.7, "budget": 25, "lens_seed": 8},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "attend", "attend", "attend", "boxes", "sparse", "sparse"])
    shape = rng.choice(list(SHAPES))
    if op == "store":
        return {"op": op, "shape": shape, "rows": _log_uniform(rng, 1, 131072), "dtype": rng.choice(["bf16", "bf16", "f32"])}
    if op == "boxes":
        return {"op": op, "shape": shape, "pages": _log_uniform(rng, 1, 2048), "full": rng.random() < 0.5}
    batch = _log_uniform(rng, 1, 128)
    q_len = rng.choice([1, 1, 2, 3, 4, 8]) if op == "attend" else 1
    # no more than the largest listed cases read and compute, and no request longer than 128K tokens
    most = min(131072, 64 * 16384 // (batch * q_len))
    case = {"op": op, "shape": shape, "batch": batch, "ctx": _log_uniform(rng, 1, most), "ragged": round(rng.choice([0.0, 0.1, 0.5, 1.0]), 1),
            "lens_seed": rng.randrange(1 << 20)}
    return dict(case, q_len=q_len) if op == "attend" else dict(case, budget=rng.randint(4, 80))


def lengths(case):
    """The requests' lengths, from the case alone: between (1 - ragged) * ctx and ctx; where ragged is 1 the last one is 0."""
    rng = random.Random(case["lens_seed"])
    lens = [case["ctx"] - int(case["ragged"] * rng.random() * case["ctx"]) for _ in range(case["batch"])]
    if case["ragged"] >= 1.0 and case["batch"] > 1:
        lens[-1] = 0
    return lens


# ---- inputs --------------------------------------------------------------------------------------------------------


def _latents(gen, n, w, dev, page_share=0.0):
    """n rows of w values as a latent norm gives them: channels of unequal size, the tokens of a page alike in part."""
    x = torch.randn(n, w, generator=gen, device=dev)
    if page_share:
        pages = torch.randn(-(-n // PAGE), w, generator=gen, device=dev).repeat_interleave(PAGE, 0)[:n]
        x = x.mul_(math.sqrt(1 - page_share**2)).add_(pages, alpha=page_share)
    return x.mul_(torch.rand(w, generator=gen, device=dev).mul_(1.5).add_(0.25))


def _filled_cache(gen, slots, d, dr, dev):
    """A cache of `slots` written slots, filled a part at a time."""
    codes = torch.empty(slots, d // 2, dtype=torch.uint8, device=dev)
    params = torch.empty(slots, d // GROUP, 2, dtype=torch.float32, device=dev)
    rope = torch.empty(slots, dr, dtype=torch.bfloat16, device=dev)
    for at in range(0, slots, 1 << 17):
        n = min(1 << 17, slots - at)
        x = _latents(gen, n, d + dr, dev, 0.6).to(torch.bfloat16)
        codes[at : at + n], params[at : at + n] = plain_quantise(x[:, :d].float())
        rope[at : at + n] = x[:, d:]
    return codes, params, rope


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    d, dr, heads = SHAPES[case["shape"]]
    s = {"op": case["op"], "d": d, "dr": dr}
    if case["op"] == "store":
        n = case["rows"]
        slots = -(-n // PAGE) * PAGE + 8 * PAGE
        x = _latents(gen, n, d + dr, dev).to(torch.bfloat16)
        s["c"], s["k_pe"] = x[:, :d], x[:, d:]
        if case["dtype"] == "f32":  # rows that a rotation left in 32 bits
            s["c"] = _latents(gen, n, d, dev)
        s["slots"] = torch.randperm(slots, generator=gen, device=dev)[:n].sort().values if n > 256 else torch.randperm(slots, generator=gen, device=dev)[:n]
        s["cache"] = (torch.zeros(slots, d // 2, dtype=torch.uint8, device=dev), torch.zeros(slots, d // GROUP, 2, device=dev),
                      torch.zeros(slots, dr, dtype=torch.bfloat16, device=dev))
        s["back_c"] = torch.empty(n, d, dtype=s["c"].dtype, device=dev)
        s["back_pe"] = torch.empty(n, dr, dtype=torch.bfloat16, device=dev)
    elif case["op"] == "boxes":
        n = case["pages"]
        total = n + 8
        s["cache"] = _filled_cache(gen, total * PAGE, d, dr, dev)
        s["pages"] = torch.randperm(total, generator=gen, device=dev)[:n].to(torch.int32)
        s["counts"] = torch.full((n,), PAGE, dtype=torch.int32, device=dev)
        if not case["full"]:
            s["counts"] = torch.randint(1, PAGE + 1, (n,), generator=gen, device=dev, dtype=torch.int32)
        s["boxes"] = _empty_boxes(total, d + dr, dev)
        s["lo"] = torch.empty(n, d + dr, device=dev)
        s["hi"] = torch.empty(n, d + dr, device=dev)
    else:
        lens = lengths(case)
        b, q_len = case["batch"], case.get("q_len", 1)
        counts = [-(-x // PAGE) for x in lens]
        total, width = sum(counts) + 4, max(max(counts), 1)
        s["cache"] = _filled_cache(gen, total * PAGE, d, dr, dev)
        order = torch.randperm(total, generator=gen, device=dev).to(torch.int32)
        first = torch.tensor([sum(counts[:i]) for i in range(b)], device=dev)
        col = torch.arange(width, device=dev)
        held = col[None, :] < torch.tensor(counts, device=dev)[:, None]
        s["page_table"] = torch.where(held, order[(first[:, None] + col[None, :]).clamp(max=total - 1)], -1).to(torch.int32)
        s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        s["q"] = torch.randn(b, q_len, heads, d + dr, generator=gen, device=dev).to(torch.bfloat16)
        s["sm_scale"] = 1.0 / math.sqrt(192.0 if d == 512 else 96.0)
        s["out"] = torch.empty(b, q_len, heads, d, dtype=torch.bfloat16, device=dev)
        s["lse"] = torch.empty(b, q_len, heads, device=dev)
        s["budget"] = case.get("budget", 0)
        if case["op"] == "sparse":
            s["boxes"] = plain_boxes(s["cache"], torch.arange(total, dtype=torch.int32, device=dev), torch.full((total,), PAGE, dtype=torch.int32, device=dev))
    if own:
        from mla_kv_quant_b200 import int4

        s["view"] = int4.Int4View(*s["cache"], boxes=s.get("boxes"))
        if case["op"] in ("attend", "sparse"):
            s["ws"] = int4.Workspace(s["view"], case["batch"], s["q"].shape[1], heads, s["page_table"].shape[1], budget=s["budget"])
    return s


def _empty_boxes(pages, w, dev):
    return (torch.zeros(pages, w, dtype=torch.int8, device=dev), torch.zeros(pages, w, dtype=torch.uint8, device=dev),
            torch.zeros(pages, 2, dtype=torch.int32, device=dev))


# ---- the operators -------------------------------------------------------------------------------------------------


def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "store":
        codes, params, rope = s["cache"]
        codes[s["slots"]], params[s["slots"]] = plain_quantise(s["c"].float())
        rope[s["slots"]] = s["k_pe"]
        return {"c": plain_values(codes[s["slots"]], params[s["slots"]]).to(s["c"].dtype), "k_pe": rope[s["slots"]], "params": params}
    if s["op"] == "boxes":
        center, radius, exps = plain_boxes(s["cache"], s["pages"], s["counts"])
        for held, new in zip(s["boxes"], (center, radius, exps)):
            held[s["pages"].long()] = new
        lo, hi = plain_bounds(center, radius, exps, s["d"])
        return {"lo": lo, "hi": hi, "exps": s["boxes"][2]}
    table, lens = s["page_table"], s["seq_lens"]
    got = {}
    if s["op"] == "sparse":
        table, lens = plain_select(s["q"], s["boxes"], table, lens, s["budget"], s["d"])
        got = {"sel_table": table, "sel_lens": lens}
    out, lse = plain_attend(s["q"], s["cache"], table, lens, s["sm_scale"])
    return dict(got, out=out, lse=lse)


def _run_own(s):
    from mla_kv_quant_b200 import int4

    if s["op"] == "store":
        int4.write(s["view"], s["c"], s["k_pe"], s["slots"])
        int4.read(s["view"], s["slots"], s["back_c"], s["back_pe"])
        return {"c": s["back_c"], "k_pe": s["back_pe"], "params": s["cache"][1]}
    if s["op"] == "boxes":
        int4.update_boxes(s["view"], s["pages"], s["counts"])
        int4.read_boxes(s["view"], s["pages"], s["lo"], s["hi"])
        return {"lo": s["lo"], "hi": s["hi"], "exps": s["boxes"][2]}
    if s["op"] == "attend":
        int4.decode(s["q"], s["view"], s["page_table"], s["seq_lens"], s["sm_scale"], s["out"], s["lse"], s["ws"])
        return {"out": s["out"], "lse": s["lse"]}
    int4.sparse_decode(s["q"], s["view"], s["page_table"], s["seq_lens"], s["sm_scale"], s["budget"], s["out"], s["lse"], s["ws"])
    return {"sel_table": s["ws"].sel_table, "sel_lens": s["ws"].sel_lens, "out": s["out"], "lse": s["lse"]}


def plain_quantise(x):
    """Rows of 32-bit values to codes and (scale, zero): per 128 elements scale = (max - min) / 15, or 1 where that is
    next to nothing; code = the nearest of 0..15 to (x - min) / scale, halves to even; zero = -min / scale."""
    n, d = x.shape
    g = x.reshape(n, d // GROUP, GROUP)
    lo, hi = g.amin(-1), g.amax(-1)
    scale = torch.where((hi - lo).abs() <= 1e-8, torch.ones_like(lo), (hi - lo) / torch.full_like(lo, float(LEVELS)))
    code = torch.round((g - lo[..., None]) / scale[..., None]).clamp(0, LEVELS).to(torch.uint8).reshape(n, d)
    return code[:, 0::2] | (code[:, 1::2] << 4), torch.stack([scale, -lo / scale], -1)


def plain_values(codes, params):
    """(code - zero) * scale, in 32 bits, of rows of any leading shape."""
    code = torch.stack([codes & 15, codes >> 4], -1).float().reshape(*codes.shape[:-1], params.shape[-2], GROUP)
    return ((code - params[..., 1:]) * params[..., :1]).reshape(*codes.shape[:-1], -1)


def _tokens(cache, table):
    """The key rows [B, pages * 64, D + Dr] of each request, in 32 bits; pages that it does not hold give page 0's."""
    codes, params, rope = cache
    pages = table.clamp(min=0).long()
    k = torch.empty(table.shape[0], table.shape[1] * PAGE, codes.shape[1] * 2 + rope.shape[1], device=codes.device)
    k[..., : codes.shape[1] * 2] = plain_values(codes.view(-1, PAGE, codes.shape[1])[pages].flatten(1, 2), params.view(-1, PAGE, *params.shape[1:])[pages].flatten(1, 2))
    k[..., codes.shape[1] * 2 :] = rope.view(-1, PAGE, rope.shape[1])[pages].flatten(1, 2)
    return k


def plain_attend(q, cache, table, lens, sm_scale):
    """softmax(q k^T sm_scale) over each request's tokens, times their latents: query t of q_len is the token at
    position len - q_len + t and sees itself and what came before; a row that sees nothing gives 0 and -inf."""
    b, q_len, heads, w = q.shape
    d = 2 * cache[0].shape[1]
    k = _tokens(cache, table)
    score = torch.bmm(q.reshape(b, q_len * heads, w).float(), k.transpose(1, 2)).mul_(sm_scale).view(b, q_len, heads, -1)
    seen = lens[:, None] - q_len + 1 + torch.arange(q_len, device=q.device)[None, :]
    mask = torch.arange(k.shape[1], device=q.device)[None, None, :] >= seen[..., None]
    score.masked_fill_(mask[:, :, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = torch.bmm(p.view(b, q_len * heads, -1), k[..., :d]).view(b, q_len, heads, d) / total.clamp(min=1e-30)
    return out.to(torch.bfloat16), (top + torch.log(total))[..., 0]


def _exp2(e):
    """2^e in 32 bits of whole numbers e, exactly."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _exponent(top):
    """The least whole e with top <= 127 * 2^e, at least -100; 0 where top is 0."""
    m, x = torch.frexp(top)
    e = torch.where(m > 127.0 / 128.0, x - 6, x - 7).clamp(min=-100)
    return torch.where(top > 0, e, torch.zeros_like(e)).to(torch.int32)


def plain_boxes(cache, pages, counts):
    """The box that holds the first `counts` tokens of each page: center (int8), radius (uint8) of each element, in
    units of 2^e with one e for the latent and one for the rotary part; the radius is rounded up."""
    codes, params, rope = cache
    d, n = codes.shape[1] * 2, len(pages)
    at = pages.long()
    v = torch.cat([plain_values(codes.view(-1, PAGE, codes.shape[1])[at], params.view(-1, PAGE, *params.shape[1:])[at]), rope.view(-1, PAGE, rope.shape[1])[at].float()], -1)
    out = torch.arange(PAGE, device=codes.device)[None, :, None] >= counts[:, None, None]
    lo, hi = v.masked_fill(out, math.inf).amin(1), v.masked_fill(out, -math.inf).amax(1)
    top = torch.maximum(lo.abs(), hi.abs())
    exps = _exponent(torch.stack([top[:, :d].amax(1), top[:, d:].amax(1)], 1))
    unit = _exp2(-exps).repeat_interleave(torch.tensor([d, rope.shape[1]], device=codes.device), 1, output_size=d + rope.shape[1])
    center = torch.round((lo + hi) * 0.5 * unit)
    radius = torch.ceil(torch.maximum(hi * unit - center, center - lo * unit))
    return center.to(torch.int8), radius.to(torch.uint8), exps


def plain_bounds(center, radius, exps, d):
    unit = _exp2(exps).repeat_interleave(torch.tensor([d, center.shape[1] - d], device=center.device), 1, output_size=center.shape[1])
    c, r = center.float(), radius.float()
    return (c - r) * unit, (c + r) * unit


def plain_select(q, boxes, table, lens, budget, d):
    """The pages that each request attends to: its first and its last two, and of the others those of the largest
    score, as many as the budget leaves; equal scores go by the lower index. The score of a page is the largest over
    the heads of q . center + |q| . radius, with q in 8 bits: no token of the page can score more."""
    b, _, heads, w = q.shape
    center, radius, exps = boxes
    qf = q.reshape(b, heads, w).float()
    top = torch.stack([qf[..., :d].abs().amax((1, 2)), qf[..., d:].abs().amax((1, 2))], 1)
    q_exp = _exponent(top)
    q8 = torch.round(qf * _exp2(-q_exp).repeat_interleave(torch.tensor([d, w - d], device=q.device), 1, output_size=w)[:, None, :])
    at = table.clamp(min=0).long()
    c, r = center[at].float(), radius[at].float()
    unit = _exp2(q_exp)[:, None, :] * _exp2(exps[at])
    parts = [(torch.bmm(q8[..., sl], c[..., sl].transpose(1, 2)) + torch.bmm(q8[..., sl].abs(), r[..., sl].transpose(1, 2))) * unit[:, None, :, i]
             for i, sl in enumerate((slice(0, d), slice(d, w)))]
    score = (parts[0] + parts[1]).amax(1)
    col = torch.arange(table.shape[1], device=q.device)[None, :]
    held = ((lens + PAGE - 1) // PAGE)[:, None]
    score = torch.where((col < 1) | (col >= held - 2), math.inf, score)
    score = torch.where(col < held, score, -math.inf)
    most = min(budget, table.shape[1])
    chosen = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :most]
    chosen = torch.where(torch.arange(most, device=q.device)[None, :] < held, chosen, table.shape[1]).sort(1).values
    got = torch.full((b, budget), -1, dtype=torch.int32, device=q.device)
    padded = torch.cat([table, torch.full((b, 1), -1, dtype=torch.int32, device=q.device)], 1)
    got[:, :most] = padded.gather(1, chosen)
    n = held[:, 0].clamp(max=budget)
    return got, torch.where(held[:, 0] > 0, (n - 1) * PAGE + lens - (held[:, 0] - 1) * PAGE, 0).to(torch.int32)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------


def work(case):
    d, dr, heads = SHAPES[case["shape"]]
    token = d // 2 + d // GROUP * 8 + dr * 2
    w = d + dr
    if case["op"] == "store":
        wide = d * (4 if case["dtype"] == "f32" else 2) + dr * 2
        return {"bytes": case["rows"] * (2 * wide + 2 * token + 2 * 8), "flops": case["rows"] * d * 6}
    if case["op"] == "boxes":
        tokens = case["pages"] * (PAGE if case["full"] else 33)
        return {"bytes": tokens * token + case["pages"] * (2 * (2 * w + 8) + 2 * 4 * w + 8), "flops": tokens * w * 4}
    lens, q_len = lengths(case), case.get("q_len", 1)
    rows = case["batch"] * q_len * heads
    extra = 0
    if case["op"] == "sparse":
        pages = [-(-x // PAGE) for x in lens]
        extra = sum(p * (2 * w + 8 + 4) for p in pages)
        lens = [x if p <= case["budget"] else (case["budget"] - 1) * PAGE + x - (p - 1) * PAGE for x, p in zip(lens, pages)]
        extra_flops = sum(p * heads * w * 4 for p in pages)
    tokens = sum(lens)
    table = sum(-(-x // PAGE) * 4 for x in lens)
    return {"bytes": tokens * token + rows * (w * 2 + d * 2 + 4) + table + extra,
            "flops": 2 * tokens * q_len * heads * (w + d) + (extra_flops if case["op"] == "sparse" else 0)}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    d, dr = s["d"], s["dr"]
    if case["op"] == "store":
        x = s["c"].double().reshape(-1, GROUP)
        low, span = x.amin(1, keepdim=True), x.amax(1, keepdim=True) - x.amin(1, keepdim=True)
        step = torch.where(span <= 1e-8, torch.ones_like(span), span / LEVELS)
        code = ((x - low) / step).round().clamp(0, LEVELS)
        params = s["cache"][1].double()
        params[s["slots"]] = torch.cat([step, -low / step], 1).reshape(case["rows"], -1, 2)
        return {"c": (code * step + low).reshape(-1, d), "k_pe": s["k_pe"].double(), "params": params}
    if case["op"] == "boxes":
        lo, hi = torch.empty(case["pages"], d + dr, dtype=torch.float64, device="cuda"), torch.empty(case["pages"], d + dr, dtype=torch.float64, device="cuda")
        for i, (page, n) in enumerate(zip(s["pages"].tolist(), s["counts"].tolist())):
            rows = _exact_rows(s["cache"], torch.arange(page * PAGE, page * PAGE + n, device="cuda"))
            for part in (slice(0, d), slice(d, d + dr)):
                small, big = rows[:, part].amin(0), rows[:, part].amax(0)
                unit = _exact_unit(max(abs(float(small.min())), abs(float(big.max()))))
                c = ((small + big) / (2 * unit)).round()
                r = torch.maximum(big / unit - c, c - small / unit).ceil()
                lo[i, part], hi[i, part] = (c - r) * unit, (c + r) * unit
        return {"lo": lo, "hi": hi, "exps": None}
    out, lse = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda"), torch.full(s["lse"].shape, -math.inf, dtype=torch.float64, device="cuda")
    q_len = s["q"].shape[1]
    for b, n in enumerate(lengths(case)):
        pages = s["page_table"][b, : -(-n // PAGE)].long()
        if case["op"] == "sparse" and len(pages) > s["budget"]:
            pages = pages[_exact_choice(s, b, pages)]
            n = (len(pages) - 1) * PAGE + (n - 1) % PAGE + 1
        at = (pages[:, None] * PAGE + torch.arange(PAGE, device="cuda")[None, :]).reshape(-1)[:n]
        rows = _exact_rows(s["cache"], at)
        for t in range(q_len):
            seen = n - q_len + t + 1
            if seen > 0:
                logits = s["q"][b, t].double() @ rows[:seen].T * s["sm_scale"]
                lse[b, t] = torch.logsumexp(logits, 1)
                out[b, t] = torch.softmax(logits, 1) @ rows[:seen, :d]
    return {"sel_table": None, "sel_lens": None, "out": out, "lse": lse} if case["op"] == "sparse" else {"out": out, "lse": lse}


def _exact_rows(cache, at):
    codes, params, rope = (x[at] for x in cache)
    code = torch.empty(len(at), codes.shape[1] * 2, dtype=torch.float64, device=codes.device)
    code[:, 0::2], code[:, 1::2] = (codes % 16).double(), (codes // 16).double()
    scale, zero = (params[..., i].double().repeat_interleave(GROUP, 1) for i in (0, 1))
    return torch.cat([scale * code - scale * zero, rope.double()], 1)


def _exact_unit(top):
    return 2.0 ** max(-100, math.ceil(math.log2(top / 127.0))) if top > 0 else 1.0


def _exact_choice(s, b, pages):
    """The chosen pages of one request, in order: scores in whole numbers, a page at a time of the heads."""
    d = s["d"]
    center, radius, exps = (x[pages].double() for x in s["boxes"])
    q = s["q"][b, 0].double()
    score = 0
    for i, part in enumerate((slice(0, d), slice(d, q.shape[1]))):
        unit = _exact_unit(float(q[:, part].abs().max()))
        whole = (q[:, part] / unit).round()
        score = score + (center[:, part] @ whole.T + radius[:, part] @ whole.abs().T) * unit * torch.exp2(exps[:, i : i + 1])
    score = score.amax(1).tolist()
    n = len(pages)
    forced = [0, n - 2, n - 1]
    rest = sorted((j for j in range(n) if j not in forced), key=lambda j: (-score[j], j))
    return torch.tensor(sorted(forced + rest[: s["budget"] - 3]), device=pages.device)
