"""Decode over the 4-bit block-scaled cache against a plain implementation in
64 bits on the dequantised cache.

Tolerance, from the arithmetic of the operator (eps/2 of a type is its half
step).  K and V dequantise to f16 exactly and products accumulate in fp32, so
a logit is off by at most E = (D + 8) 2^-24 max_t sum_d |q_d k_td| scale (D
additions and a few factors).  That changes every weight by a factor within
e^(+-2E); the weights are also rounded to f16 (2^-11, absolute 2^-25 of the
row's largest weight), and exp2 and the joining of partial sums cost a few
2^-22.  With A = sum_t p_t |v_t| (the row's output for |V|):
  |O - O64|   <= (2^-11 + 2 E + 2^-19) A + L 2^-25 max|v| + eps/2 |O64|
  |LSE - LSE64| <= E + 2^-19 (1 + |LSE64|)
"""
import math

import pytest
import torch

import flashdecode
from flashdecode import cases
from oracle.decode_ref import dequantize_fp4, quantize_fp4

pytestmark = pytest.mark.gpu

FD_ERR_BAD_PAGE = 6
FP4, E4M3 = torch.float4_e2m1fn_x2, torch.float8_e4m3fn


def make(seqlens, Hq, Hkv, D=128, page=256, sq=1, dtype=torch.bfloat16, seed=0, pool_extra=0, extra_len=0,
         q_std=1.0):
    """A case whose cache holds random codes and block scales everywhere; the
    rows behind each sequence's end hold NaN scales."""
    c = cases.custom_case("fp4", dtype, [max(n, 0) + extra_len for n in seqlens], Hq, Hkv, D=D, page=page,
                          seed=seed, pool_extra=pool_extra)
    g = torch.Generator().manual_seed(seed + 1)
    nb = c.num_blocks
    t = dict(lens=torch.tensor(seqlens, dtype=torch.int32), bt=c.block_table)
    t["q"] = (torch.randn((c.B, sq, Hq, D), generator=g) * q_std).to(dtype)
    t["ks"] = (1 + torch.rand(Hkv, generator=g)) / 512
    t["vs"] = (1 + torch.rand(Hkv, generator=g)) / 512
    live = torch.zeros((nb, page), dtype=torch.bool)
    for b, L in enumerate(seqlens):
        for j in range(-(-max(L, 0) // page)):
            live[int(c.block_table[b, j]), :max(L, 0) - j * page] = True
    for n in ("k", "v"):
        x = torch.randn((nb, page, Hkv, D), generator=g)
        codes, blocks = quantize_fp4(x, t[n + "s"])
        blocks[~live] = 0x7F          # NaN
        t[n] = codes
        t[n + "b"] = blocks.permute(0, 2, 1, 3).contiguous()
    return t


def on_gpu(t):
    d = {n: x.cuda() for n, x in t.items()}
    for n in ("k", "v"):
        d[n] = d[n].view(FP4)
        d[n + "b"] = d[n + "b"].view(E4M3)
    return d


def call(d, **kw):
    return flashdecode.flash_decode(d["q"], d["k"], d["v"], d["lens"], d["bt"], return_softmax_lse=True,
                                    k_scale=d["ks"], v_scale=d["vs"], k_block_scale=d["kb"],
                                    v_block_scale=d["vb"], **kw)


def reference(t, causal=False, scale=None, lens=None):
    """(O, LSE, A, E) in 64 bits; lens as in `t` unless given."""
    q, bt = t["q"].double(), t["bt"].long()
    B, sq, Hq, D = q.shape
    nb, page, Hkv, _ = t["k"].shape
    scale = 1 / math.sqrt(D) if scale is None else scale
    K = dequantize_fp4(t["k"].view(torch.uint8), t["kb"].view(torch.uint8), t["ks"])
    V = dequantize_fp4(t["v"].view(torch.uint8), t["vb"].view(torch.uint8), t["vs"])
    out = torch.zeros((B, sq, Hq, D), dtype=torch.float64)
    A, E = torch.zeros_like(out), torch.zeros((B, Hq, sq), dtype=torch.float64)
    lse = torch.full((B, Hq, sq), -math.inf, dtype=torch.float64)
    W = torch.zeros_like(out)
    for b, L in enumerate((t["lens"] if lens is None else lens).tolist()):
        L = min(max(L, 0), bt.shape[1] * page)
        ids = bt[b, :-(-L // page)]
        bad = (ids < 0) | (ids >= nb)
        kb, vb = K[ids.clamp(0, nb - 1)], V[ids.clamp(0, nb - 1)]
        kb[bad], vb[bad] = 0, 0
        kb, vb = kb.flatten(0, 1)[:L], vb.flatten(0, 1)[:L]
        for i in range(sq):
            n = L - (sq - 1 - i) if causal else L
            if n <= 0:
                continue
            x = q[b, i].view(Hkv, -1, D)
            z = torch.einsum("hgd,thd->hgt", x, kb[:n]) * scale
            p = torch.softmax(z, -1)
            lse[b, :, i] = torch.logsumexp(z, -1).flatten()
            out[b, i] = torch.einsum("hgt,thd->hgd", p, vb[:n]).reshape(Hq, D)
            A[b, i] = torch.einsum("hgt,thd->hgd", p, vb[:n].abs()).reshape(Hq, D)
            W[b, i] = n * 2.0 ** -25 * vb[:n].abs().amax()
            mass = torch.einsum("hgd,thd->hgt", x.abs(), kb[:n].abs()).amax(-1) * abs(scale)
            E[b, :, i] = ((D + 8) * 2.0 ** -24 * mass).flatten()
    return out, lse, A, E, W


def check(out, lse, ref):
    O, LSE, A, E, W = ref
    sq = O.shape[1]
    e = E.permute(0, 2, 1)[..., None]
    tol = (2.0 ** -11 + 2 * e + 2.0 ** -19) * A + W + torch.finfo(out.dtype).eps / 2 * O.abs()
    err = (out.cpu().double() - O).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} elements off, max err {float(err.max()):.3e}"
    got = lse.cpu().double().view_as(LSE) if sq > 1 else lse.cpu().double()[..., None]
    some = torch.isfinite(LSE)
    assert torch.equal(some, torch.isfinite(got)) and bool((got[~some] == -math.inf).all())
    off = (got - LSE)[some].abs()
    assert bool((off <= (E + 2.0 ** -19 * (1 + LSE.abs()))[some]).all()), float(off.max())


RAGGED = [1, 0, 31, 32, 33, 127, 128, 129, 300, 2049]


@pytest.mark.parametrize("page", [16, 48, 64, 256])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_lengths_pages_and_head_dims(page, D):
    t = make(RAGGED, 8, 2, D=D, page=page, seed=page + D)
    out, lse = call(on_gpu(t))
    torch.cuda.synchronize()
    check(out, lse, reference(t))
    assert flashdecode.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("out_dtype", [None, torch.float32])
@pytest.mark.parametrize("Hq,Hkv", [(8, 8), (32, 8), (28, 4), (16, 1), (5, 1), (48, 2)])
def test_types_and_groups(dtype, out_dtype, Hq, Hkv):
    """Groups of 1 .. 24: one pass of 8 rows, one of 16, and two of 16."""
    t = make([700, 1, 65, 0, 1500], Hq, Hkv, dtype=dtype, page=64, seed=Hq)
    out, lse = call(on_gpu(t), out_dtype=out_dtype)
    torch.cuda.synchronize()
    assert out.dtype == (out_dtype or dtype)
    check(out, lse, reference(t))


@pytest.mark.parametrize("sq,causal", [(2, True), (4, True), (3, False), (9, True), (1, True)])
@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 128), (14, 2, 64), (4, 1, 256)])
def test_several_query_tokens(sq, causal, Hq, Hkv, D):
    """Speculated tokens; lengths below sq leave rows that see no key."""
    t = make([1, 2, 0, 130, 257, 1000, 7], Hq, Hkv, D=D, page=16, sq=sq, seed=sq)
    out, lse = call(on_gpu(t), causal=causal)
    torch.cuda.synchronize()
    check(out, lse, reference(t, causal=causal))


@pytest.mark.parametrize("seqlens,Hq,Hkv", [
    ([70000], 32, 8), ([40000, 3, 17, 9000], 8, 1), ([16 * i * i for i in range(1, 41)], 16, 4),
])
def test_long_and_skewed(seqlens, Hq, Hkv):
    """Pairs cut over many CTAs and joined, beside short ones."""
    t = make(seqlens, Hq, Hkv, page=256, seed=len(seqlens))
    d = on_gpu(t)
    ref = reference(t)
    first = None
    for _ in range(3):
        out, lse = call(d)
        torch.cuda.synchronize()
        check(out, lse, ref)
        first = (out, lse) if first is None else first
        assert torch.equal(first[0], out) and torch.equal(first[1], lse)   # the same bits every time


def test_more_sequences_than_a_launch_takes():
    t = make([(7 * i) % 61 for i in range(1100)], 4, 2, page=16, seed=9)
    out, lse = call(on_gpu(t))
    torch.cuda.synchronize()
    check(out, lse, reference(t))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_query_magnitudes(dtype):
    """Rows of very large, very small and zero queries (bf16 rows are brought
    into f16's range by a power of two)."""
    t = make([300] * 5, 8, 2, dtype=dtype, page=16, seed=4)
    f = [1e4, 1e-4, 0.0, 30.0, 1e-6] if dtype == torch.float16 else [1e30, 1e-30, 0.0, 300.0, 1e-38]
    t["q"] = (t["q"].float() * torch.tensor(f)[:, None, None, None]).to(dtype)
    for scale in (None, -0.05):
        s = scale
        out, lse = call(on_gpu(t), softmax_scale=s)
        torch.cuda.synchronize()
        keep = [1, 2, 3, 4] if dtype == torch.bfloat16 else [0, 1, 2, 3, 4]
        ref = reference(t, scale=s)
        check(out[keep], lse[keep], tuple(x[keep] for x in ref))
        assert torch.isfinite(out).all()


def test_nan_and_infinity_travel_only_in_their_rows():
    t = make([200, 200, 200], 8, 2, page=16, seed=6)
    t["q"][1, 0, 3, 5] = float("nan")
    t["q"][2, 0, 1, 7] = float("inf")
    t["vb"][int(t["bt"][0, 2]), 0, 3, 1] = 0x7F       # a NaN scale inside sequence 0, KV head 0
    out, _ = call(on_gpu(t))
    torch.cuda.synchronize()
    nan = torch.isnan(out.cpu())
    assert nan[1, 0, 3].all() and not nan[1, 0, [0, 1, 2, 4, 5, 6, 7]].any()
    assert nan[2, 0, 1].all() and not nan[2, 0, [0, 2, 3]].any()
    assert nan[0, 0, :4, 16:32].all() and not nan[0, 0, :4, 32:].any() and not nan[0, 0, 4:].any()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (6, 1)])
def test_nan_scales_stay_behind_the_causal_mask(D, Hq, Hkv):
    """A speculated token with NaN block scales (of K, of V) reaches the rows
    that see it, as the formula has it, and no row before it."""
    sq, seqlens, first_bad = 4, [4, 63, 130, 2], {0: 3, 1: 62, 2: 128}
    t = make(seqlens, Hq, Hkv, D=D, page=16, sq=sq, seed=D)
    clean = {n: x.clone() for n, x in t.items()}
    for b, at in first_bad.items():
        pg, row = int(t["bt"][b, at // 16]), at % 16
        t["vb"][pg, 0, row, 1] = 0xFF                 # dims 16 .. 31 of KV head 0
        if b == 2:
            t["kb"][pg, 0, row + 1, 0] = 0x7F         # and all dims from the next token on
    out, lse = call(on_gpu(t), causal=True)
    torch.cuda.synchronize()
    ref = reference(clean, causal=True)
    nan = torch.isnan(out.cpu())
    want = torch.zeros_like(nan)
    G = Hq // Hkv
    for b, at in first_bad.items():
        for i in range(sq):
            seen = seqlens[b] - (sq - 1 - i)
            want[b, i, :G, 16:32] = seen > at
            if b == 2 and seen > at + 1:
                want[b, i, :G] = True
    assert torch.equal(nan, want)
    lse = torch.where(torch.isnan(lse.cpu()), ref[1].float(), lse.cpu())
    check(torch.where(nan, ref[0].to(out.dtype), out.cpu()), lse, ref)


def test_bad_pages_read_as_zeros():
    for bad in (-1, 10 ** 6):
        t = make([500, 100], 8, 2, page=16, seed=8)
        d = on_gpu(t)
        d["bt"][0, 3] = bad
        t["bt"] = t["bt"].clone()
        t["bt"][0, 3] = bad
        out, lse = call(d)
        torch.cuda.synchronize()
        check(out, lse, reference(t))
        assert flashdecode.device_status() == FD_ERR_BAD_PAGE


def test_length_past_the_table_is_cut():
    t = make([100, 64], 8, 2, page=16, seed=3)
    d = on_gpu(t)
    d["lens"] = torch.tensor([5000, 64], dtype=torch.int32, device="cuda")
    out, lse = call(d)
    torch.cuda.synchronize()
    t["kb"] = torch.where(t["kb"] == 0x7F, 0, t["kb"])   # sequence 0 now reaches its page's end
    t["vb"] = torch.where(t["vb"] == 0x7F, 0, t["vb"])
    width = t["bt"].shape[1] * 16
    d2 = on_gpu(t)
    d2["lens"] = d["lens"]
    out, lse = call(d2)
    torch.cuda.synchronize()
    check(out, lse, reference(t, lens=torch.tensor([width, 64])))


@pytest.mark.parametrize("sq", [1, 3])
def test_fused_append(sq):
    """k / v given: quantised into the cache, then attended; cache_seqlens
    unchanged, the rest of the pool too."""
    seqlens = [0, 15, 16, 700, 255]
    t = make(seqlens, 8, 2, page=16, sq=sq, seed=sq, extra_len=sq)
    g = torch.Generator().manual_seed(5)
    kn, vn = (torch.randn((5, sq, 2, 128), generator=g).bfloat16() for _ in range(2))
    d = on_gpu(t)
    out, lse = call(d, causal=True, k=kn.cuda(), v=vn.cuda())
    torch.cuda.synchronize()
    for n, new in (("k", kn), ("v", vn)):
        codes, blocks = quantize_fp4(new, t[n + "s"])
        for b, L in enumerate(seqlens):
            for i in range(sq):
                pg, row = int(t["bt"][b, (L + i) // 16]), (L + i) % 16
                t[n][pg, row] = codes[b, i]
                t[n + "b"][pg, :, row] = blocks[b, i]
        assert torch.equal(d[n].view(torch.uint8).cpu(), t[n])
        assert torch.equal(d[n + "b"].view(torch.uint8).cpu(), t[n + "b"])
    assert d["lens"].tolist() == seqlens
    check(out, lse, reference(t, causal=True, lens=t["lens"] + sq))


def test_plan_graph_streams_and_workspace():
    """The same bits from the eager call, a plan, a captured and replayed
    plan, another stream and a caller's workspace, also after a 16-bit call
    used the same stream's scratch."""
    t = make([5000, 17, 0, 3000], 32, 8, seed=2)
    d = on_gpu(t)
    out, lse = call(d)
    torch.cuda.synchronize()
    check(out, lse, reference(t))
    kw = dict(return_softmax_lse=True, k_scale=d["ks"], v_scale=d["vs"], k_block_scale=d["kb"], v_block_scale=d["vb"])
    plan = flashdecode.DecodePlan(d["q"], d["k"], d["v"], d["lens"], d["bt"], **kw)
    c16 = cases.custom_case("n", torch.bfloat16, [4000, 900, 5], 32, 8, seed=1)
    t16 = cases.materialize(c16, "cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            flashdecode.flash_decode(t16["q"], t16["k_cache"], t16["v_cache"], t16["cache_seqlens"], t16["block_table"])
            o, s = plan()
            side.synchronize()
            assert torch.equal(o, out) and torch.equal(s, lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan()
    for _ in range(3):
        plan.out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(plan.out, out) and torch.equal(plan.lse, lse)
    n = flashdecode.load_library().fd_decode_workspace_size_fp4(4, 1, 32, 8, 128)
    ws = torch.zeros((n,), dtype=torch.uint8, device="cuda")
    for _ in range(2):
        o, s = call(d, workspace=ws)
        torch.cuda.synchronize()
        assert torch.equal(o, out) and torch.equal(s, lse)
    with pytest.raises(flashdecode.FlashDecodeError):
        call(d, workspace=ws[:n - 256])
    assert flashdecode.device_status() == 0


def test_captured_append_and_decode():
    """The fused append captured with its decode: replays write the rows in
    the bound buffers and attend them; lengths advance between replays."""
    seqlens = [0, 30, 700]
    t = make(seqlens, 8, 2, page=16, seed=13, extra_len=6)
    d = on_gpu(t)
    kn, vn = (torch.zeros((3, 1, 2, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    plan = flashdecode.DecodePlan(d["q"], d["k"], d["v"], d["lens"], d["bt"], return_softmax_lse=True, k=kn, v=vn,
                                  k_scale=d["ks"], v_scale=d["vs"], k_block_scale=d["kb"], v_block_scale=d["vb"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan()
    g = torch.Generator().manual_seed(1)
    for step in range(6):
        new = [torch.randn((3, 1, 2, 128), generator=g).bfloat16() for _ in range(2)]
        kn.copy_(new[0])
        vn.copy_(new[1])
        graph.replay()
        torch.cuda.synchronize()
        for n, x in zip("kv", new):
            codes, blocks = quantize_fp4(x, t[n + "s"])
            for b, L in enumerate(seqlens):
                pg, row = int(t["bt"][b, (L + step) // 16]), (L + step) % 16
                t[n][pg, row] = codes[b, 0]
                t[n + "b"][pg, :, row] = blocks[b, 0]
        check(plan.out, plan.lse, reference(t, lens=t["lens"] + step + 1))
        d["lens"] += 1
    assert flashdecode.device_status() == 0


def test_two_streams_at_once():
    """Calls on two streams overlap, each with its stream's scratch."""
    ts = [make([6000, 40, 3000], 32, 8, seed=s) for s in (1, 2)]
    ds = [on_gpu(t) for t in ts]
    want = [call(d) for d in ds]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ds]
    for _ in range(5):
        got = []
        for d, st in zip(ds, streams):
            with torch.cuda.stream(st):
                got.append(call(d))
        torch.cuda.synchronize()
        for (o, l), (wo, wl) in zip(got, want):
            assert torch.equal(o, wo) and torch.equal(l, wl)
    for t, (o, l) in zip(ts, want):
        check(o, l, reference(t))


def test_offsets_beyond_32_bits():
    """A pool of more than 4 GiB of codes: the pages in use lie at its ends."""
    page, Hkv, D, nb = 256, 8, 128, 40000
    L = [600, 500]
    ids = torch.tensor([[nb - 1, 0, nb - 2], [nb - 3, 39000, -1]], dtype=torch.int32)
    g = torch.Generator().manual_seed(2)
    t = dict(q=torch.randn((2, 1, 32, D), generator=g).bfloat16(), lens=torch.tensor(L, dtype=torch.int32),
             ks=torch.full((Hkv,), 1 / 256), vs=torch.full((Hkv,), 1 / 300))
    d = {n: x.cuda() for n, x in t.items()}
    d["bt"] = ids.cuda()
    for n in ("k", "v"):
        d[n] = torch.zeros((nb, page, Hkv, D // 2), dtype=torch.uint8, device="cuda").view(FP4)
        d[n + "b"] = torch.zeros((nb, Hkv, page, D // 16), dtype=torch.uint8, device="cuda").view(E4M3)
    rows = [torch.randn((sum(L), Hkv, D), generator=g).bfloat16() for _ in range(2)]
    pos = torch.cat([torch.arange(n) for n in L])
    owner = torch.cat([torch.full((n,), b) for b, n in enumerate(L)])
    slots = ids[owner, pos // page].long() * page + pos % page
    flashdecode.append_kv_slots(rows[0].cuda(), rows[1].cuda(), d["k"], d["v"], slots.cuda(), k_scale=d["ks"],
                                v_scale=d["vs"], k_block_scale=d["kb"], v_block_scale=d["vb"])
    out, lse = call(d)
    torch.cuda.synchronize()
    t["bt"] = torch.arange(2)[:, None]     # the reference: one page a request
    for n, x in zip("kv", rows):
        wide = torch.zeros((2, max(L), Hkv, D), dtype=torch.bfloat16)
        wide[owner, pos] = x
        t[n], blocks = quantize_fp4(wide, t[n + "s"])
        t[n + "b"] = blocks.permute(0, 2, 1, 3).contiguous()
    check(out, lse, reference(t))
    assert flashdecode.device_status() == 0


def test_workload_materialised_through_the_append():
    c = cases.custom_case("m", torch.bfloat16, [40, 300, 7], 8, 2, page=16, seed=3)
    t = cases.materialize_fp4(c, "cuda", seed=3)
    t16 = cases.materialize(c, "cuda", seed=3)
    for n in ("k", "v"):
        codes, blocks = quantize_fp4(t16[n + "_cache"], t[n + "_scale"])
        assert torch.equal(t[n + "_cache"].view(torch.uint8).cpu(), codes)
        assert torch.equal(t[n + "_block_scale"].view(torch.uint8).cpu(), blocks.permute(0, 2, 1, 3))


def test_serving_steps_together():
    """Prompts arrive, get pages and slots, are appended and attended; then
    decode steps with growing lengths; one request leaves and its pages go to
    a newcomer.  The cache is checked through the attention's results against
    a reference that keeps each request's quantised rows in plain lists."""
    page, Hq, Hkv, D, nb = 16, 8, 2, 128, 40
    g = torch.Generator().manual_seed(11)
    t = make([0, 0, 0], Hq, Hkv, page=page, seed=1, pool_extra=nb)
    d = on_gpu(t)
    assert d["k"].shape[0] >= nb
    nb = d["k"].shape[0]
    table = torch.full((3, 12), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros((3,), dtype=torch.int32, device="cuda")
    pool, count = torch.arange(nb, dtype=torch.int32, device="cuda"), torch.tensor([nb, 0], dtype=torch.int32, device="cuda")
    kw = dict(k_scale=d["ks"], v_scale=d["vs"], k_block_scale=d["kb"], v_block_scale=d["vb"])
    held = [([], []) for _ in range(3)]
    steps = [[37, 100, 0], [1, 1, 0], [1, 1, 50], [2, 0, 1], "leave 1", [1, 120, 1], [1, 1, 1]]
    for new in steps:
        if new == "leave 1":
            keep = lens.clone()
            keep[1] = 0
            flashdecode.release_pages(table, lens, keep, pool, count, page)
            lens.copy_(keep)
            held[1] = ([], [])
            continue
        T = sum(new)
        n = torch.tensor(new, dtype=torch.int32, device="cuda")
        slots, cu, _ = flashdecode.assign_pages(table, lens, n, pool, count, page, num_slots=T + 2, seqlens_out=lens)
        k, v = (torch.randn((T + 2, Hkv, D), generator=g).bfloat16() for _ in range(2))
        flashdecode.append_kv_slots(k.cuda(), v.cuda(), d["k"], d["v"], slots, **kw)
        cu = cu.tolist()
        for b in range(3):
            held[b][0].append(k[cu[b]:cu[b + 1]])
            held[b][1].append(v[cu[b]:cu[b + 1]])
        q = torch.randn((3, 1, Hq, D), generator=g).bfloat16()
        out, lse = flashdecode.flash_decode(q.cuda(), d["k"], d["v"], lens, table, return_softmax_lse=True, **kw)
        torch.cuda.synchronize()
        # the reference: contiguous caches of one page a request
        L = [sum(x.shape[0] for x in h[0]) for h in held]
        assert lens.tolist() == L
        ref = dict(q=q, lens=torch.tensor(L), bt=torch.arange(3)[:, None], ks=t["ks"], vs=t["vs"])
        wide = max(L)
        for name, i in (("k", 0), ("v", 1)):
            rows = torch.zeros((3, wide, Hkv, D), dtype=torch.bfloat16)
            for b in range(3):
                rows[b, :L[b]] = torch.cat(held[b][i]) if held[b][i] else 0
            ref[name], blocks = quantize_fp4(rows, t[name + "s"])
            ref[name + "b"] = blocks.permute(0, 2, 1, 3).contiguous()
        check(out, lse, reference(ref))
    assert int(count[0]) == nb - sum(-(-n // page) for n in L)
    assert flashdecode.device_status() == 0


def test_refusals():
    t = make([100, 20], 8, 2, page=16)
    d = on_gpu(t)

    def bad(err, **over):
        x = {**d, **{k: v for k, v in over.items() if k in d}}
        with pytest.raises(err):
            call(x, **{k: v for k, v in over.items() if k not in d})

    bad(ValueError, kb=None)
    bad(ValueError, vb=d["vb"].view(torch.uint8))
    bad(ValueError, kb=d["kb"].transpose(1, 2))
    bad(ValueError, ks=None)
    bad(ValueError, q=d["q"].float())
    bad(ValueError, q=d["q"][..., :64].contiguous())
    bad(ValueError, v=d["v"].view(torch.uint8).view(E4M3))

    bad(flashdecode.FlashDecodeError, out_dtype=torch.float16)
    bad(flashdecode.FlashDecodeError, softmax_scale=float("nan"))
    for D, page in ((96, 16), (128, 8), (32, 16)):
        u = on_gpu(make([20], 4, 2, D=D, page=page))
        with pytest.raises(flashdecode.FlashDecodeError):
            call(u)
    with pytest.raises(ValueError):        # block scales with a cache that has none
        c16 = cases.custom_case("n", torch.bfloat16, [40], 8, 2, seed=1)
        t16 = cases.materialize(c16, "cuda")
        flashdecode.flash_decode(t16["q"], t16["k_cache"], t16["v_cache"], t16["cache_seqlens"],
                                 t16["block_table"], k_block_scale=d["kb"])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("out_dtype", [None, torch.float32])
@pytest.mark.parametrize("Hq,Hkv,sq", [(16, 1, 1), (8, 2, 1), (6, 3, 1), (8, 2, 3), (24, 2, 2)])
def test_many_partials_of_a_pair(D, out_dtype, Hq, Hkv, sq):
    """One long sequence over all CTAs, at every head dim: rows and partials
    shared by the warps of the joining, rows of more than one pass."""
    t = make([30000, 5], Hq, Hkv, D=D, page=64, sq=sq, seed=D + Hq, dtype=torch.float16)
    out, lse = call(on_gpu(t), causal=sq > 1, out_dtype=out_dtype)
    torch.cuda.synchronize()
    check(out, lse, reference(t, causal=sq > 1))


@pytest.mark.parametrize("D,Hq,Hkv", [(128, 8, 2), (64, 6, 3), (256, 2, 1)])
def test_many_query_tokens(D, Hq, Hkv):
    """A prompt's worth of causal query tokens: many passes over the rows, most
    of them of rows that do not see the last keys, or any."""
    t = make([70, 33, 900, 0], Hq, Hkv, D=D, page=16, sq=70, seed=D)
    out, lse = call(on_gpu(t), causal=True)
    torch.cuda.synchronize()
    check(out, lse, reference(t, causal=True))


def test_workspace_size_of_the_cache_type():
    lib = flashdecode.load_library()
    assert flashdecode.workspace_size(4, 32, 8, 128, 2, kv_dtype=FP4) == \
        lib.fd_decode_workspace_size_fp4(4, 2, 32, 8, 128) > 0
    assert flashdecode.workspace_size(4, 32, 8) == lib.fd_decode_workspace_size_mq(4, 1, 32, 8, 128)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hkv,sq", [(8, 2, 1), (16, 1, 1), (6, 3, 3)])
def test_fp32_outputs_are_worth_their_bits(D, dtype, Hq, Hkv, sq):
    """The weights enter the product with V in two f16 parts: 2^-24 of each
    weight, and 2^-32 of the row's largest.  Small queries keep E below 2^-17,
    and up to 160 tokens are at most 8 products a warp, each adding 16 tokens in
    the accumulator (17 roundings of 2^-24 at most: 2^-17 in all); with exp2, the
    division and the joining below 2^-18 the rest is 2^-16 of A.  One f16 part
    alone is off by up to 2^-12."""
    t = make([2, 3, 4, 5, 8, 17, 40, 160], Hq, Hkv, D=D, page=16, sq=sq, dtype=dtype, seed=D + sq, q_std=1 / 32)
    out, _ = call(on_gpu(t), out_dtype=torch.float32, causal=sq > 1)
    O, _, A, E, W = reference(t, causal=sq > 1)          # W: L 2^-25 max|v|
    tol = (2 * E.permute(0, 2, 1)[..., None] + 2.0 ** -16) * A + 2.0 ** -7 * W + 2.0 ** -24 * O.abs()
    err = (out.cpu().double() - O).abs()
    assert bool((err <= tol).all()), float((err / tol.clamp(min=1e-300)).max())


@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (3, 1), (16, 1)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_nan_of_a_partial_without_weight(D, Hq, Hkv):
    """Block scales of V that are NaN at tokens of no weight, around one that
    takes all of it: 0 * NaN is NaN, wherever the sequence is cut."""
    L, peak = 30000, 15000
    t = make([L], Hq, Hkv, D=D, page=16, seed=D)
    t["q"][:] = 8.0
    pg, row = int(t["bt"][0, peak // 16]), peak % 16
    t["k"][pg, row] = 0x77           # every code 6, every block scale 448
    t["kb"][pg, :, row] = 0x7E
    at = [peak + s * n * 90 for n in range(1, 1 + D // 32) for s in (-1, 1)]   # one token a block
    for block, tok in enumerate(at):
        t["vb"][int(t["bt"][0, tok // 16]), 0, tok % 16, block] = 0x7F
    out, lse = call(on_gpu(t))
    assert torch.isfinite(lse).all()
    nan = torch.isnan(out.cpu())
    want = torch.zeros_like(nan)
    want[0, 0, :Hq // Hkv] = True
    assert torch.equal(nan, want), int(nan.sum())


def test_logit_factors_below_the_smallest_number():
    """Rows near bf16's smallest numbers times tiny head scales: the factor of
    the scaled products is below fp32's range, the logits are 0 to any
    precision, and the masked keys of the last tile stay masked."""
    t = make([300, 45, 1, 129, 0], 8, 2, page=16, seed=4)
    t["q"] = (t["q"].float() * 4e-38).bfloat16()
    t["ks"][:] = 1e-12
    out, lse = call(on_gpu(t))
    check(out, lse, reference(t))


def reference_of_many_rows(t, causal):
    """reference() of a case whose sequences have many query tokens, all rows at
    once; same formulas."""
    q = t["q"].double()
    B, sq, Hq, D = q.shape
    nb, page, Hkv, _ = t["k"].shape
    G, scale = Hq // Hkv, 1 / math.sqrt(D)
    K, V = (dequantize_fp4(t[n].view(torch.uint8), t[n + "b"].view(torch.uint8), t[n + "s"]) for n in ("k", "v"))
    out, A, W = (torch.zeros((B, sq, Hq, D), dtype=torch.float64) for _ in range(3))
    E, lse = torch.zeros((B, Hq, sq), dtype=torch.float64), torch.full((B, Hq, sq), -math.inf, dtype=torch.float64)
    for b, L in enumerate(t["lens"].tolist()):
        ids = t["bt"][b, :-(-L // page)].long()
        kb, vb = K[ids].flatten(0, 1)[:L], V[ids].flatten(0, 1)[:L]
        seen = L - (sq - 1 - torch.arange(sq)) if causal else torch.full((sq,), L)
        hidden = torch.arange(L)[None, :] >= seen[:, None]
        for h in range(Hq):
            k, v, x = kb[:, h // G], vb[:, h // G], q[b, :, h]
            z = (x @ k.T * scale).masked_fill(hidden, -math.inf)
            lse[b, h] = torch.logsumexp(z, -1)
            p = torch.where(hidden, 0.0, torch.exp(z - lse[b, h].clamp(min=-1e300)[:, None]))
            out[b, :, h], A[b, :, h] = p @ v, p @ v.abs()
            E[b, h] = (D + 8) * 2.0 ** -24 * (x.abs() @ k.abs().T * scale).amax(-1)
        W[b] = L * 2.0 ** -25 * vb.abs().amax()
    return out, lse, A, E, W


@pytest.mark.parametrize("lens,sq,Hq,Hkv,D,table_tokens,causal", [
    ([300], 4096, 32, 8, 128, 16384, False),
    ([300, 5], 256, 64, 8, 128, 131072, True),
    ([300], 4096, 32, 8, 128, 131072, True),       # the passes of a sequence in several launches
    ([40, 200, 7], 500, 14, 2, 64, 4194304, False),
    ([130, 90], 210, 3, 1, 256, 8388608, True),
])
def test_many_query_tokens_under_a_wide_table(lens, sq, Hq, Hkv, D, table_tokens, causal):
    """The bound of a launch goes by the table's width: rows that one launch
    cannot take go to the next."""
    t = make(lens, Hq, Hkv, D=D, page=256, sq=sq, seed=sq)
    d = on_gpu(t)
    d["bt"] = torch.full((len(lens), table_tokens // 256), -1, dtype=torch.int32, device="cuda")
    d["bt"][:, :t["bt"].shape[1]] = t["bt"].cuda()
    out, lse = call(d, causal=causal)
    check(out, lse, reference_of_many_rows(t, causal))
    assert flashdecode.device_status() == 0


def test_partials_of_another_shape_are_no_counters():
    """The workspace's arrival counters (from byte 128; the launch epoch in the
    first word) may hold what a launch of another shape left there as partials:
    (x, 0), whose upper bits are the epoch and whose lower ones a count."""
    t = make([5000, 17, 9000, 0, 300, 2049], 32, 8, seed=5)
    d = on_gpu(t)
    want = call(d)
    check(*want, reference(t))
    n = flashdecode.workspace_size(6, 32, 8, 128, kv_dtype=FP4)
    ws = torch.zeros((n,), dtype=torch.uint8, device="cuda")
    for x in (1.0 + 2.0 ** -23, 0.7 + 3 * 2.0 ** -24, 1e-30):
        stale = torch.tensor([x, 0.0], dtype=torch.float32, device="cuda").repeat(6 * 8)
        ws[:8].view(torch.int64)[0] = int(stale[0].view(torch.int32)) >> 12
        ws[128:128 + 8 * 6 * 8].view(torch.float32).copy_(stale)
        out, lse = call(d, workspace=ws)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_whole_step_captured():
    """Pages, slots, append, decode over the new lengths, the step's rows read
    back, and the release of what is not kept: one graph on fixed buffers,
    replayed with other lengths, rows, queries and numbers of tokens kept."""
    page, B, Hq, Hkv, D, room, sq = 16, 4, 8, 2, 128, 70, 1
    t = make([0] * B, Hq, Hkv, page=page, seed=21, pool_extra=60)
    d = on_gpu(t)
    nb = d["k"].shape[0]
    i32 = dict(dtype=torch.int32, device="cuda")
    table, lens, after = torch.full((B, 12), -1, **i32), torch.zeros(B, **i32), torch.zeros(B, **i32)
    new, keep, cu = torch.zeros(B, **i32), torch.zeros(B, **i32), torch.zeros(B + 1, **i32)
    pool, count = torch.arange(nb, **i32), torch.tensor([nb, 0], **i32)
    slots = torch.zeros(room, dtype=torch.int64, device="cuda")
    k, v = (torch.zeros((room, Hkv, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    back = [torch.zeros((room, Hkv, D), device="cuda") for _ in range(2)]
    kw = dict(k_scale=d["ks"], v_scale=d["vs"], k_block_scale=d["kb"], v_block_scale=d["vb"])
    q = torch.zeros((B, sq, Hq, D), dtype=torch.bfloat16, device="cuda")
    plan = flashdecode.DecodePlan(q, d["k"], d["v"], after, table, return_softmax_lse=True, **kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        flashdecode.assign_pages(table, lens, new, pool, count, page, slot_map=slots, cu_new_lens=cu,
                                 seqlens_out=after)
        flashdecode.append_kv_slots(k, v, d["k"], d["v"], slots, **kw)
        plan()
        flashdecode.gather_kv(d["k"], d["v"], slots, out_dtype=torch.float32, k_out=back[0], v_out=back[1], **kw)
        flashdecode.release_pages(table, after, keep, pool, count, page)
        lens.copy_(keep)
    g = torch.Generator().manual_seed(3)
    held = [[[], []] for _ in range(B)]
    for step, (add, kept) in enumerate([([30, 0, 5, 16], [30, 0, 5, 16]), ([1, 1, 1, 1], [1, 1, 1, 1]),
                                        ([4, 4, 4, 4], [4, 1, 0, 3]), ([4, 20, 4, 4], [0, 20, 2, 4]),
                                        ([1, 1, 40, 1], [1, None, 40, 1]), ([1, 60, 1, 1], [1, 60, 1, 1])]):
        x = [torch.randn((room, Hkv, D), generator=g).bfloat16() for _ in range(2)]
        qs = torch.randn(q.shape, generator=g).bfloat16()
        before = [len(h[0]) for h in held]
        stay = [0 if n is None else m + n for m, n in zip(before, kept)]       # None: the request leaves
        for dst, src in ((k, x[0]), (v, x[1]), (q, qs), (new, torch.tensor(add, dtype=torch.int32)),
                         (keep, torch.tensor(stay, dtype=torch.int32))):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert cu.tolist() == [sum(add[:b]) for b in range(B + 1)]
        for b in range(B):
            for i in range(2):
                held[b][i] += list(x[i][int(cu[b]):int(cu[b + 1])])
        L = [len(h[0]) for h in held]
        assert after.tolist() == L
        ref = dict(q=qs, lens=torch.tensor(L), bt=torch.arange(B)[:, None], ks=t["ks"], vs=t["vs"])
        for i, name in enumerate("kv"):
            rows = torch.zeros((B, max(L), Hkv, D), dtype=torch.bfloat16)
            for b in range(B):
                for j, row in enumerate(held[b][i]):
                    rows[b, j] = row
            ref[name], blocks = quantize_fp4(rows, t[name + "s"])
            ref[name + "b"] = blocks.permute(0, 2, 1, 3).contiguous()
            codes, blocks = quantize_fp4(x[i], t[name + "s"])
            want = dequantize_fp4(codes[:, None], blocks[:, None].transpose(1, 2), t[name + "s"], torch.float32)[:, 0]
            want[sum(add):] = 0                                                # slots -1
            assert torch.equal(back[i].cpu(), want)
        check(plan.out, plan.lse, reference(ref))
        for b in range(B):
            held[b] = [h[:stay[b]] for h in held[b]]
        assert lens.tolist() == stay and count.tolist() == [nb - sum(-(-n // page) for n in stay), 0]
        assert [(row >= 0).sum().item() for row in table] == [-(-n // page) for n in stay]
    assert flashdecode.device_status() == 0


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv,sq", [(2, 2, 4), (3, 3, 3), (4, 2, 2), (2, 1, 2)])
def test_few_rows_of_several_query_tokens(D, Hq, Hkv, sq):
    """Up to four rows in all, twice in a tile's columns: causal masks inside a
    page, a NaN of V that only the last rows see, a sequence over many CTAs."""
    seqlens = [sq, 1, 0, 63, 130, 20000]
    t = make(seqlens, Hq, Hkv, D=D, page=16, sq=sq, seed=D + sq, dtype=torch.float16)
    clean = {n: x.clone() for n, x in t.items()}
    at = 129
    t["vb"][int(t["bt"][4, at // 16]), 0, at % 16, 1] = 0x7F
    for out_dtype in (None, torch.float32):
        out, lse = call(on_gpu(t), causal=True, out_dtype=out_dtype)
        ref = reference(clean, causal=True)
        nan = torch.isnan(out.cpu())
        want = torch.zeros_like(nan)
        want[4, sq - 1, :Hq // Hkv, 16:32] = True
        assert torch.equal(nan, want)
        check(torch.where(nan, ref[0].to(out.dtype), out.cpu()), lse, ref)
