"""Cases, plain forms and reference values of the paged-cache operators.

Three operators of a serving loop over a paged KV cache:

* ``pages``   block tables and slot maps from request lengths: requests take
  pages from a pool for their new tokens, every new token learns its cache
  slot, and pages beyond the kept lengths go back to the pool;
* ``append``  packed new tokens written to their slots of a 16-bit, e4m3 or
  4-bit block-scaled cache, and the cache's rows read back as values (what a
  transfer of the cache to another instance does);
* ``decode``  attention of one or a few new tokens per sequence over a 4-bit
  block-scaled paged cache.

The 4-bit cache: each KV head's row of D values is D / 16 blocks of 16 e2m1
codes (two per byte, the even element in the low half), each block with an
e4m3 scale; value = e2m1 * block scale * the KV head's fp32 scale.  Codes are
[num_blocks, page, Hkv, D / 2], block scales [num_blocks, Hkv, page, D / 16].

``own`` chooses between the plain forms (elementary torch operations) and the
framework's calls.
"""
import functools
import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one token for each of four requests: a lone user's decode step
        dict(name="pages_step_b4", op="pages", B=4, page=256, lo=1, hi=2048, new_lo=1, new_hi=1,
             share=1.0, pad=0),
        # four speculated tokens for each of 256 requests, then all rejected
        dict(name="pages_verify_b256", op="pages", B=256, page=16, lo=512, hi=8192, new_lo=4,
             new_hi=4, share=1.0, pad=0),
        # 256 prompts arrive together and later leave; the pool is a little too small for all
        dict(name="pages_prompt_b256", op="pages", B=256, page=16, lo=0, hi=0, new_lo=512,
             new_hi=8192, share=0.95, pad=4097),
        # a decode step's 64 new rows into a small 4-bit cache
        dict(name="append_step_fp4", op="append", T=64, rows=1280, Hq=32, Hkv=8, D=128, page=256,
             src="bf16", cache="fp4", fused=True, skip=0),
        # ragged prompts packed together, cut from a fused projection, some padding rows
        dict(name="append_prompt_fp4", op="append", T=58966, rows=65536, Hq=32, Hkv=8, D=128,
             page=256, src="bf16", cache="fp4", fused=True, skip=37),
        # the same path into a 16-bit cache of small pages
        dict(name="append_prompt_fp16", op="append", T=12251, rows=16000, Hq=28, Hkv=4, D=128,
             page=16, src="fp16", cache="native", fused=True, skip=5),
        # the framework's five decode workloads, over a 4-bit cache
        dict(name="decode_cfg1_b4", op="decode", B=4, sq=1, Hq=32, Hkv=8, D=128, page=256,
             q="fp16", dist="uniform", lo=1, hi=2048, causal=False),
        dict(name="decode_cfg2_b64_l4096", op="decode", B=64, sq=1, Hq=32, Hkv=8, D=128, page=256,
             q="bf16", dist="uniform", lo=4096, hi=4096, causal=False),
        dict(name="decode_cfg3_skew_b128", op="decode", B=128, sq=1, Hq=64, Hkv=8, D=128, page=256,
             q="bf16", dist="log", lo=16, hi=32768, causal=False),
        dict(name="decode_cfg4_long_b2", op="decode", B=2, sq=1, Hq=32, Hkv=8, D=128, page=256,
             q="bf16", dist="uniform", lo=262144, hi=262144, causal=False),
        dict(name="decode_cfg5_g7_b256", op="decode", B=256, sq=1, Hq=28, Hkv=4, D=128, page=16,
             q="fp16", dist="uniform", lo=512, hi=8192, causal=False),
        # four speculated tokens a sequence, checked together
        dict(name="decode_verify_b32", op="decode", B=32, sq=4, Hq=32, Hkv=8, D=128, page=16,
             q="bf16", dist="uniform", lo=1, hi=4096, causal=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["pages", "append", "decode", "decode"])
    if op == "pages":
        page = rng.choice([1, 16, 16, 64, 256])
        B = _log_int(rng, 1, 2048)
        cap = max(4, min(8192, 1000000 // B))
        if rng.random() < 0.5:  # decode steps
            hi = _log_int(rng, 1, min(8192, 60000 * page // B + 1))
            new_lo, new_hi, lo = 0, rng.randint(1, 8), 0
        else:                   # prompts
            lo = hi = 0
            new_hi = _log_int(rng, 2, min(cap, 200000 * page // B + 2))
            new_lo = rng.randint(0, new_hi)
        return dict(op="pages", B=B, page=page, lo=lo, hi=hi, new_lo=new_lo, new_hi=new_hi,
                    share=rng.choice([1.0, 1.0, round(rng.uniform(0.3, 1.0), 3)]),
                    pad=rng.randint(0, 300))
    D = rng.choice([64, 128, 128, 256])
    Hkv = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 4, 4, 5, 7, 8, 16])
    if op == "append":
        T = _log_int(rng, 1, max(2, min(60000, 58000 * 1024 // (Hkv * D))))
        return dict(op="append", T=T, rows=T + rng.randint(0, T) // 8 + 1, Hq=Hkv * group, Hkv=Hkv,
                    D=D, page=rng.choice([16, 16, 48, 64, 256]), src=rng.choice(["bf16", "fp16"]),
                    cache=rng.choice(["fp4", "fp4", "e4m3", "native"]),
                    fused=rng.random() < 0.5, skip=rng.randint(0, T // 4))
    B = _log_int(rng, 1, 256)
    sq = rng.choice([1, 1, 1, 2, 4])
    hi = _log_int(rng, 1, max(2, min(262144, 500000 * 1024 // (B * Hkv * D))))
    return dict(op="decode", B=B, sq=sq, Hq=Hkv * group, Hkv=Hkv, D=D,
                page=rng.choice([16, 16, 32, 48, 64, 128, 256]), q=rng.choice(["bf16", "fp16"]),
                dist=rng.choice(["uniform", "log"]), lo=max(1, int(hi * rng.uniform(0, 1))), hi=hi,
                causal=sq > 1 and rng.random() < 0.7)


# ------------------------------------------------------------------ inputs
def _lengths(case, g):
    B, lo, hi = case["B"], case["lo"], case["hi"]
    if case.get("dist") == "log":
        u = torch.rand((B,), generator=g, device=DEV, dtype=torch.float64)
        x = torch.exp(math.log(lo) + (math.log(hi) - math.log(lo)) * u).round().clamp(lo, hi)
        return x.to(torch.int32)
    return torch.randint(lo, hi + 1, (B,), generator=g, device=DEV, dtype=torch.int64).to(torch.int32)


def _deal_pages(lens, page, g):
    """A random permutation of just enough pages, dealt to the requests in order."""
    n = (lens.long() + page - 1) // page
    total, width = int(n.sum()), max(int(n.max()), 1)
    j = torch.arange(width, device=DEV)
    used = j[None, :] < n[:, None]
    at = (torch.cumsum(n, 0) - n)[:, None] + j[None, :]
    perm = torch.randperm(max(total, 1), generator=g, device=DEV)
    table = torch.where(used, perm[at.clamp(max=max(total, 1) - 1)], torch.full_like(at, -1))
    return table.to(torch.int32).contiguous(), max(total, 1)


def _codes(x):
    """e2m1 code of each value: the nearest of 0 .5 1 1.5 2 3 4 6, ties to the even code."""
    a = x.abs()
    c = (a > 0.25).to(torch.uint8)
    c += a >= 0.75
    c += a > 1.25
    c += a >= 1.75
    c += a > 2.5
    c += a >= 3.5
    c += a > 5.0
    return c | (torch.signbit(x).to(torch.uint8) << 3)


def _quantize_fp4(x, scale):
    """Codes [..., D / 2] and block scales [..., D / 16] of x [..., Hkv, D]; scale [Hkv]."""
    b = x.float().unflatten(-1, (-1, 16))
    g = scale[:, None]
    s8 = (b.abs().amax(-1) / (6.0 * g)).clamp(max=448.0).to(torch.float8_e4m3fn)
    s = s8.float()
    y = b / torch.where(s > 0, s * g, torch.ones_like(s))[..., None]
    y = torch.where((s > 0)[..., None], y, torch.zeros_like(y))
    c = _codes(y).flatten(-2)
    return c[..., 0::2] | (c[..., 1::2] << 4), s8


def _head_scales(Hkv, g):
    """fp32 scales of a KV head, as calibration gives them."""
    return (1.0 + torch.rand((Hkv,), generator=g, device=DEV)) / 512.0


def _fp4_cache(nb, page, Hkv, D, scale, g):
    """A filled 4-bit cache, quantised from N(0, 1) rows."""
    codes = torch.empty((nb, page, Hkv, D // 2), dtype=torch.uint8, device=DEV)
    scales = torch.empty((nb, Hkv, page, D // 16), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 26) // (page * Hkv * D))
    for i in range(0, nb, step):
        n = min(step, nb - i)
        x = torch.randn((n, page, Hkv, D), generator=g, device=DEV, dtype=torch.bfloat16)
        c, s8 = _quantize_fp4(x, scale)
        codes[i:i + n] = c
        scales[i:i + n] = s8.view(torch.uint8).permute(0, 2, 1, 3)
    return codes.view(torch.float4_e2m1fn_x2), scales.view(torch.float8_e4m3fn)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    return {"pages": _prepare_pages, "append": _prepare_append, "decode": _prepare_decode}[case["op"]](case, g)


def _prepare_pages(case, g):
    B, page = case["B"], case["page"]
    lens = _lengths(case, g)
    new = torch.randint(case["new_lo"], case["new_hi"] + 1, (B,), generator=g, device=DEV,
                        dtype=torch.int64).to(torch.int32)
    have = (lens.long() + page - 1) // page
    want = (lens.long() + new.long() + page - 1) // page
    held, more = int(have.sum()), int((want - have).sum())
    free = max(1, int(math.ceil(more * case["share"])) + (held + more) // 50)
    if case["share"] < 1.0:
        free = max(1, int(more * case["share"]))
    # a table and a pool for the longest requests; pages that are neither held nor free are others'
    width = max((case["hi"] + case["new_hi"] + page - 1) // page, 1)
    nb = case["B"] * width + 1
    free = min(free, nb - held)
    perm = torch.randperm(nb, generator=g, device=DEV).to(torch.int32)
    j = torch.arange(width, device=DEV)
    at = (torch.cumsum(have, 0) - have)[:, None] + j[None, :]
    table = torch.where(j[None, :] < have[:, None], perm[at.clamp(max=nb - 1)],
                        torch.full((), -1, dtype=torch.int32, device=DEV)).contiguous()
    pool = torch.full((nb,), -1, dtype=torch.int32, device=DEV)
    pool[:free] = perm[held:held + free]
    count = torch.tensor([free, 0], dtype=torch.int32, device=DEV)
    slots = torch.empty((B * case["new_hi"] + case["pad"] + 1,), dtype=torch.int64, device=DEV)
    return dict(op="pages", page=page, table=table, lens=lens, new=new, pool=pool, count=count, slots=slots)


def _prepare_append(case, g):
    T, Hq, Hkv, D, page = (case[k] for k in ("T", "Hq", "Hkv", "D", "page"))
    src = DTYPES[case["src"]]
    nb = (case["rows"] + page - 1) // page + 1
    H = Hq + 2 * Hkv if case["fused"] else 2 * Hkv
    rows = torch.randn((T, H, D), generator=g, device=DEV, dtype=src)
    k, v = rows[:, H - 2 * Hkv:H - Hkv], rows[:, H - Hkv:]
    if not case["fused"]:
        k, v = k.contiguous(), v.contiguous()
    # pages are whole: slots of one page follow one another
    order = torch.randperm(nb, generator=g, device=DEV)
    slots = (order[:, None] * page + torch.arange(page, device=DEV)[None, :]).reshape(-1)[:T].clone()
    if case["skip"]:
        slots[torch.randperm(T, generator=g, device=DEV)[:case["skip"]]] = -1
    s = dict(op="append", cache=case["cache"], k=k, v=v, slots=slots, src=src, page=page,
             every=torch.arange(nb * page, device=DEV), kscale=None, vscale=None, kblock=None, vblock=None)
    if case["cache"] == "native":
        s["kc"] = torch.randn((nb, page, Hkv, D), generator=g, device=DEV, dtype=src)
        s["vc"] = torch.randn((nb, page, Hkv, D), generator=g, device=DEV, dtype=src)
        return s
    s["kscale"], s["vscale"] = _head_scales(Hkv, g), _head_scales(Hkv, g)
    if case["cache"] == "e4m3":
        for n, sc in (("kc", s["kscale"]), ("vc", s["vscale"])):
            x = torch.randn((nb, page, Hkv, D), generator=g, device=DEV, dtype=src).float()
            s[n] = (x / sc[:, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
        return s
    s["kc"], s["kblock"] = _fp4_cache(nb, page, Hkv, D, s["kscale"], g)
    s["vc"], s["vblock"] = _fp4_cache(nb, page, Hkv, D, s["vscale"], g)
    return s


def _prepare_decode(case, g):
    B, sq, Hq, Hkv, D, page = (case[k] for k in ("B", "sq", "Hq", "Hkv", "D", "page"))
    lens = _lengths(case, g)
    table, nb = _deal_pages(lens, page, g)
    kscale, vscale = _head_scales(Hkv, g), _head_scales(Hkv, g)
    kc, kblock = _fp4_cache(nb, page, Hkv, D, kscale, g)
    vc, vblock = _fp4_cache(nb, page, Hkv, D, vscale, g)
    q = torch.randn((B, sq, Hq, D), generator=g, device=DEV, dtype=DTYPES[case["q"]])
    s = dict(op="decode", q=q, kc=kc, vc=vc, kblock=kblock, vblock=vblock, kscale=kscale,
             vscale=vscale, lens=lens, table=table, causal=case["causal"])
    if own:  # a serving loop binds its buffers once
        s["plan"] = _flashdecode().DecodePlan(
            q, kc, vc, lens, table, return_softmax_lse=True, causal=case["causal"], k_scale=kscale,
            v_scale=vscale, k_block_scale=kblock, v_block_scale=vblock)
    return s


# -------------------------------------------------------------------- runs
@functools.cache
def _flashdecode():
    at = os.path.join(os.getcwd(), "flashatte-hand_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import flashdecode
    return flashdecode


def run(state):
    return {"pages": _run_pages, "append": _run_append, "decode": _run_decode}[state["op"]](state)


def _run_pages(s):
    if own:
        fd = _flashdecode()
        slots, cu, after = fd.assign_pages(s["table"], s["lens"], s["new"], s["pool"], s["count"],
                                           s["page"], slot_map=s["slots"])
        fd.release_pages(s["table"], after, s["lens"], s["pool"], s["count"], s["page"])
        return dict(slots=slots, cu=cu, after=after, table=s["table"], pool=s["pool"], count=s["count"])
    page, table, pool = s["page"], s["table"], s["pool"]
    width = table.shape[1]
    lens, new = s["lens"].long().clamp(min=0), s["new"].long().clamp(min=0)
    cu = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0)])
    have = ((lens + page - 1) // page).clamp(max=width)
    fits = lens + new <= width * page
    need = torch.where(fits, (lens + new + page - 1) // page - have, torch.zeros_like(have))
    last = torch.cumsum(need, 0)
    free = s["count"][0].long()
    granted = fits & ((need == 0) | (last <= free))
    got = torch.where(granted, need, torch.zeros_like(need))
    after = torch.where(granted, lens + new, lens)
    # pages come off the top of the pool, in the order of the requests
    j = torch.arange(width, device=table.device)[None, :]
    fresh = (j >= have[:, None]) & (j < (have + got)[:, None])
    nth = (last - need)[:, None] + j - have[:, None]
    ids = pool[(free - 1 - nth).clamp(0, pool.numel() - 1)]
    taken = torch.where(fresh, ids, table)
    # slots of the packed new tokens
    t = torch.arange(s["slots"].numel(), device=table.device)
    b = torch.searchsorted(cu[1:], t, right=True).clamp(max=new.numel() - 1)
    pos = lens[b] + t - cu[b]
    ok = (t < cu[-1]) & granted[b]
    pos = torch.where(ok, pos, torch.zeros_like(pos))
    slot = taken[b, pos // page].long() * page + pos % page
    slot = torch.where(ok, slot, torch.full_like(slot, -1))
    # give back the pages beyond the kept lengths, which are the old ones
    count = free - got.sum()
    first = (lens + page - 1) // page
    back = (j >= first[:, None]) & (j < ((after + page - 1) // page)[:, None])
    order = torch.cumsum(back.flatten().long(), 0).view_as(back) - 1
    n = back.sum()
    place = torch.where(back, count + n - 1 - order, torch.full_like(order, pool.numel()))
    grown = torch.cat([pool, pool[:1]])
    grown = grown.scatter(0, place.flatten(), taken.flatten())
    left = torch.where(back, torch.full_like(taken, -1), taken)
    count = torch.stack([count + n, torch.zeros_like(n)])
    return dict(slots=slot, cu=cu.to(torch.int32), after=after.to(torch.int32), table=left,
                pool=grown[:-1], count=count.to(torch.int32))


def _values(codes, blocks, scale):
    """fp32 values [..., Hkv, D] of codes [..., Hkv, D / 2], block scales [..., Hkv, D / 16]."""
    half = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    lut = torch.cat([half, -half])
    pairs = torch.stack([lut.repeat(16), lut.repeat_interleave(16)], 1)
    x = torch.index_select(pairs, 0, codes.reshape(-1).to(torch.int32))
    x = x.view(*codes.shape[:-1], blocks.shape[-1], 16)
    x *= blocks.float()[..., None]
    x *= scale[:, None, None]
    return x.flatten(-2)


def _run_append(s):
    if own:
        fd = _flashdecode()
        extra = dict(k_scale=s["kscale"], v_scale=s["vscale"], k_block_scale=s["kblock"],
                     v_block_scale=s["vblock"])
        fd.append_kv_slots(s["k"], s["v"], s["kc"], s["vc"], s["slots"], **extra)
        if s["cache"] == "native":
            return dict(k=s["kc"], v=s["vc"])
        k, v = fd.gather_kv(s["kc"], s["vc"], s["every"], out_dtype=s["src"], **extra)
        return dict(k=k, v=v)
    slots = s["slots"]
    live = slots >= 0
    # rows without a slot go to a row of their own behind the cache
    nrows = s["kc"].shape[0] * s["page"]
    at = torch.where(live, slots, torch.full_like(slots, nrows))

    def put(cache, rows):
        flat = cache.reshape(nrows, *cache.shape[2:])
        flat = torch.cat([flat, flat[:1]])
        flat[at] = rows
        return flat[:-1]

    out = {}
    for n, x, sc in (("k", s["k"], s["kscale"]), ("v", s["v"], s["vscale"])):
        cache = s[n + "c"]
        if s["cache"] == "native":
            out[n] = put(cache, x).view_as(cache)
        elif s["cache"] == "e4m3":
            rows = (x.float() / sc[:, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
            both = put(cache.view(torch.uint8), rows.view(torch.uint8)).view(torch.float8_e4m3fn)
            out[n] = (both.float() * sc[:, None]).to(s["src"])
        else:
            codes, s8 = _quantize_fp4(x, sc)
            blocks = s[n + "block"].view(torch.uint8).permute(0, 2, 1, 3)
            codes = put(cache.view(torch.uint8), codes)
            blocks = put(blocks, s8.view(torch.uint8)).view(torch.float8_e4m3fn)
            out[n] = _values(codes, blocks, sc).to(s["src"])
    return out


def _run_decode(s):
    if own:
        out, lse = s["plan"]()
        return dict(out=out, lse=lse)
    q, lens, table = s["q"], s["lens"].long(), s["table"].long().clamp(min=0)
    B, sq, Hq, D = q.shape
    page, Hkv = s["kc"].shape[1:3]
    S = table.shape[1] * page
    G = Hq // Hkv

    def gathered(codes, blocks, scale):
        c = codes.view(torch.uint8)[table].view(B, S, Hkv, D // 2)
        e = blocks.view(torch.uint8)[table].permute(0, 1, 3, 2, 4).reshape(B, S, Hkv, D // 16)
        return _values(c, e.view(torch.float8_e4m3fn), scale).permute(0, 2, 1, 3)  # [B, Hkv, S, D]

    x = q.float().view(B, sq, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, sq * G, D)
    logits = torch.matmul(x, gathered(s["kc"], s["kblock"], s["kscale"]).transpose(2, 3)) / math.sqrt(D)
    logits = logits.view(B, Hkv, sq, G, S)
    i = torch.arange(sq, device=q.device)
    seen = lens[:, None] - (sq - 1 - i)[None, :] if s["causal"] else lens[:, None].expand(B, sq)
    masked = torch.arange(S, device=q.device)[None, None, :] >= seen[:, :, None]
    logits = logits.masked_fill(masked[:, None, :, None, :], -math.inf)
    m = logits.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    p = torch.exp(logits - m)
    total = p.sum(-1, keepdim=True)
    v = gathered(s["vc"], s["vblock"], s["vscale"])
    o = torch.matmul(p.reshape(B, Hkv, sq * G, S), v).view(B, Hkv, sq, G, D)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    lse = (m + torch.log(total))[..., 0]  # [B, Hkv, sq, G]
    out = o.permute(0, 2, 1, 3, 4).reshape(B, sq, Hq, D).to(q.dtype)
    lse = lse.permute(0, 1, 3, 2).reshape(B, Hq, sq)
    return dict(out=out, lse=lse[..., 0].contiguous() if sq == 1 else lse)


# -------------------------------------------------------------------- work
def _row_bytes(case):
    """Bytes of one KV head's row of K or V in the cache."""
    D = case["D"]
    return {"fp4": D // 2 + D // 16, "e4m3": D, "native": 2 * D}[case.get("cache", "fp4")]


def work(case):
    if case["op"] == "pages":
        B, page = case["B"], case["page"]
        tokens = B * (case["new_lo"] + case["new_hi"]) / 2
        if case["lo"] == case["hi"] == 0:
            pages = B * ((case["new_lo"] + case["new_hi"]) / 2 + (page - 1) / 2) / page
        else:
            pages = min(tokens, tokens / page)
        # lengths in and out, the slot map, each page's pool entry and table entry both ways
        return {"bytes": 16 * B + 8 * (B * case["new_hi"] + case["pad"] + 1) + 16 * pages, "flops": 0}
    if case["op"] == "append":
        T, Hkv, D, row = case["T"] - case["skip"], case["Hkv"], case["D"], _row_bytes(case)
        b = 2 * Hkv * T * (2 * D + row) + 8 * case["T"]
        if case["cache"] != "native":  # every row of the pool read back
            rows = ((case["rows"] + case["page"] - 1) // case["page"] + 1) * case["page"]
            b += 2 * Hkv * rows * (row + 2 * D) + 8 * rows
        return {"bytes": b, "flops": 0}
    lo, hi = case["lo"], case["hi"]
    if case["dist"] == "log" and hi > lo:
        mean = (hi - lo) / math.log(hi / lo)
    else:
        mean = (lo + hi) / 2
    tokens = case["B"] * mean
    rows = case["B"] * case["sq"] * case["Hq"]
    return {"bytes": 2 * tokens * case["Hkv"] * _row_bytes(case) + rows * (4 * case["D"] + 4)
            + 4 * tokens / case["page"] + 4 * case["B"],
            "flops": 4 * tokens * case["sq"] * case["Hq"] * case["D"]}


# ------------------------------------------------------------ exact values
def exact(case, seed):
    s = prepare(case, seed)
    return {"pages": _exact_pages, "append": _exact_append, "decode": _exact_decode}[case["op"]](s)


def _exact_pages(s):
    page, table = s["page"], s["table"].tolist()
    pool, count = s["pool"].tolist(), int(s["count"][0])
    width = len(table[0])
    slots, cu, after, open_ = [], [0], [], True
    for b, (n, a) in enumerate(zip(s["lens"].tolist(), s["new"].tolist())):
        cu.append(cu[-1] + a)
        pages = -(-(n + a) // page) - -(-n // page)
        if n + a > width * page or (pages and (pages > count or not open_)):
            open_ = open_ and n + a > width * page
            after.append(n)
            slots += [-1] * a
            continue
        first = -(-n // page)
        for j in range(pages):
            count -= 1
            table[b][first + j] = pool[count]
        after.append(n + a)
        slots += [table[b][p // page] * page + p % page for p in range(n, n + a)]
    slots += [-1] * (s["slots"].numel() - len(slots))
    back = []
    for b, (n, m) in enumerate(zip(s["lens"].tolist(), after)):
        for j in range(-(-n // page), -(-m // page)):
            back.append(table[b][j])
            table[b][j] = -1
    for x in reversed(back):
        pool[count] = x
        count += 1
    i32 = torch.int32
    return dict(slots=torch.tensor(slots, dtype=torch.int64), cu=torch.tensor(cu, dtype=i32),
                after=torch.tensor(after, dtype=i32), table=torch.tensor(table, dtype=i32),
                pool=torch.tensor(pool, dtype=i32), count=torch.tensor([count, 0], dtype=i32))


def _nearest(x, mant, emin, top):
    """x rounded to `mant` fraction bits, smallest exponent emin, ties to even, at most `top`."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -300))).clamp(min=emin)
    step = torch.exp2(e - mant)
    return (torch.round(x / step) * step).clamp(-top, top)


def _code_values(codes):
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    e, m = (c >> 1) & 3, (c & 1).double()
    mag = torch.where(e == 0, m / 2, (1 + m / 2) * torch.exp2(e.double() - 1))
    return torch.where(c >= 8, -mag, mag)


def _exact_append(s):
    out = {}
    live = (s["slots"] >= 0).nonzero()[:, 0]
    at = s["slots"][live]
    pg, row = at // s["page"], at % s["page"]
    for n in ("k", "v"):
        x = s[n][live].double()
        cache = s[n + "c"]
        if s["cache"] == "native":
            y = cache.double()
            y[pg, row] = x
        else:
            g = s[n + "scale"].double()[:, None]
            if s["cache"] == "e4m3":
                y = cache.float().double() * g
                y[pg, row] = _nearest(x / g, 3, -6, 448.0) * g
            else:
                b = x.unflatten(-1, (-1, 16))
                sb = _nearest(b.abs().amax(-1) / 6 / g, 3, -6, 448.0)
                d = (sb * g)[..., None]
                z = torch.where(d > 0, _nearest(b / d.clamp(min=1e-300), 1, 0, 6.0) * d, torch.zeros_like(b))
                e = s[n + "block"].float().double().permute(0, 2, 1, 3).repeat_interleave(16, -1)
                y = _code_values(cache.view(torch.uint8)) * e * g
                y[pg, row] = z.flatten(-2)
            y = y.flatten(0, 1)
        out[n] = y
    return out


def _exact_decode(s):
    q, causal = s["q"].double(), s["causal"]
    B, sq, Hq, D = q.shape
    page, Hkv = s["kc"].shape[1:3]
    out = torch.zeros((B, sq, Hq, D), dtype=torch.float64, device=q.device)
    lse = torch.full((B, Hq, sq), -math.inf, dtype=torch.float64, device=q.device)

    def rows(n, ids, L):
        c = _code_values(s[n + "c"].view(torch.uint8)[ids])
        e = s[n + "block"].float()[ids].double().permute(0, 2, 1, 3).repeat_interleave(16, -1)
        return (c * e * s[n + "scale"].double()[:, None]).flatten(0, 1)[:L]

    for b, L in enumerate(s["lens"].tolist()):
        ids = s["table"][b, :-(-L // page)].long()
        K, V = rows("k", ids, L), rows("v", ids, L)
        for i in range(sq):
            n = L - (sq - 1 - i) if causal else L
            if n <= 0:
                continue
            z = torch.einsum("hgd,thd->hgt", q[b, i].view(Hkv, -1, D), K[:n]) / math.sqrt(D)
            lse[b, :, i] = torch.logsumexp(z, -1).flatten()
            out[b, i] = torch.einsum("hgt,thd->hgd", torch.softmax(z, -1), V[:n]).reshape(Hq, D)
    return dict(out=out, lse=lse[..., 0] if sq == 1 else lse)
