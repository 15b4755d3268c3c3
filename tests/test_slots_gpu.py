"""Rows into the cache by slot and back: bytes of the cache compared exactly
with the oracle's quantisation, every other byte of the pool unchanged."""
import pytest
import torch

import flashdecode
from oracle.decode_ref import dequantize_fp4, quantize_e4m3, quantize_fp4

pytestmark = pytest.mark.gpu

FD_ERR_BAD_PAGE = 6
FP4 = torch.float4_e2m1fn_x2
E4M3 = torch.float8_e4m3fn


def make_cache(kind, nb, page, Hkv, D, src, seed=0):
    """A pool of random bytes (finite values) of one kind, with its scales."""
    g = torch.Generator().manual_seed(seed)
    c = {}
    ks = ((1 + torch.rand(Hkv, generator=g)) / 64).cuda()
    vs = ((1 + torch.rand(Hkv, generator=g)) / 64).cuda()
    for n in ("k", "v"):
        if kind == "native":
            c[n] = torch.randn((nb, page, Hkv, D), generator=g).to(src).cuda()
        elif kind == "e4m3":
            c[n] = torch.randint(0, 127, (nb, page, Hkv, D), generator=g, dtype=torch.uint8).cuda().view(E4M3)
        else:
            c[n] = torch.randint(0, 256, (nb, page, Hkv, D // 2), generator=g, dtype=torch.uint8).cuda().view(FP4)
            c[n + "b"] = torch.randint(0, 127, (nb, Hkv, page, D // 16), generator=g,
                                       dtype=torch.uint8).cuda().view(E4M3)
    kw = {} if kind == "native" else dict(k_scale=ks, v_scale=vs)
    if kind == "fp4":
        kw.update(k_block_scale=c["kb"], v_block_scale=c["vb"])
    return c, kw


def expect(kind, cache, blocks, rows, slots, scale):
    """The pool (and block scales) after the append, in plain loops over rows."""
    cache, blocks = raw(cache).cpu().clone(), None if blocks is None else raw(blocks).cpu().clone()
    nb, page = cache.shape[:2]
    if kind == "native":
        q = rows.cpu().view(torch.int16)
    elif kind == "e4m3":
        q = quantize_e4m3(rows, scale).view(torch.uint8)
    else:
        q, s8 = quantize_fp4(rows, scale)
    for t, slot in enumerate(slots.tolist()):
        if 0 <= slot < nb * page:
            cache[slot // page, slot % page] = q[t]
            if kind == "fp4":
                blocks[slot // page, :, slot % page] = s8[t]
    return cache, blocks


def raw(x):
    return x.view(torch.int16) if x.dtype in (torch.bfloat16, torch.float16) else x.view(torch.uint8)


def check(kind, c, kw, before, k, v, slots):
    for n, rows in (("k", k), ("v", v)):
        want, want_b = expect(kind, before[n], before.get(n + "b"), rows, slots, kw.get(n + "_scale"))
        assert torch.equal(raw(c[n]).cpu(), want), n
        if kind == "fp4":
            assert torch.equal(raw(c[n + "b"]).cpu(), want_b), n + " block scales"


def clone(c):
    return {n: raw(x).clone().view(x.dtype) for n, x in c.items()}


@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["native", "e4m3", "fp4"])
@pytest.mark.parametrize("T,Hkv,D,page", [(1, 8, 128, 256), (77, 8, 128, 16), (33, 1, 64, 48), (40, 3, 256, 16),
                                          (9, 2, 16, 1), (5, 40, 128, 64)])
def test_append(src, kind, T, Hkv, D, page):
    nb = (T + 20) // page + 2
    c, kw = make_cache(kind, nb, page, Hkv, D, src, seed=T)
    g = torch.Generator().manual_seed(T + 1)
    slots = torch.randperm(nb * page, generator=g)[:T]
    slots[torch.arange(T) % 7 == 3] = -1
    slots = slots.cuda()
    # a slice of a fused projection, and rows of their own
    fused = (3 * torch.randn((T, 2 + 2 * Hkv, D), generator=g)).to(src).cuda()
    for k, v in ((fused[:, 2:2 + Hkv], fused[:, 2 + Hkv:]),
                 (fused[:, 2:2 + Hkv].contiguous(), fused[:, 2 + Hkv:].contiguous())):
        before = clone(c)
        flashdecode.append_kv_slots(k, v, c["k"], c["v"], slots, **kw)
        torch.cuda.synchronize()
        check(kind, c, kw, before, k, v, slots)
    assert flashdecode.device_status() == 0


def test_block_extremes():
    """Blocks of zeros, of one value, of the type's largest and smallest
    values, of infinities, ties between codes, negative zeros; a NaN makes
    its block's scale NaN."""
    D, page = 128, 16
    for src in (torch.bfloat16, torch.float16):
        c, kw = make_cache("fp4", 4, page, 1, D, src)
        kw["k_scale"].fill_(2.0 ** -9)
        kw["v_scale"].fill_(3.0 * 2.0 ** -7)
        fi = torch.finfo(src)
        rows = torch.zeros((12, 1, D))
        rows[1] = 1.0
        rows[2, 0, ::16] = fi.max
        rows[3] = -fi.max
        rows[4] = fi.smallest_normal
        rows[5] = fi.tiny / 4
        rows[6, 0, ::2] = float("inf")
        rows[7, 0, 1::16] = -float("inf")
        rows[8] = -0.0
        ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0]) * 2.0 ** -9 * 4
        rows[9, 0] = torch.cat([ties, -ties]).repeat(D // 16)
        rows[10, 0] = torch.linspace(-7, 7, D)
        rows[11, 0] = torch.logspace(-8, 4, D)
        rows = rows.to(src).cuda()
        slots = torch.arange(12, device="cuda") * 5
        before = clone(c)
        flashdecode.append_kv_slots(rows, rows, c["k"], c["v"], slots, **kw)
        torch.cuda.synchronize()
        check("fp4", c, kw, before, rows, rows, slots)
        nan = rows.clone()
        nan[1, 0, 17] = float("nan")
        flashdecode.append_kv_slots(nan, nan, c["k"], c["v"], slots, **kw)
        k, _ = flashdecode.gather_kv(c["k"], c["v"], slots[1:2], out_dtype=torch.float32, **kw)
        assert torch.isnan(k[0, 0, 16:32]).all() and torch.isfinite(k[0, 0, :16]).all()
        assert torch.isfinite(k[0, 0, 32:]).all()


@pytest.mark.parametrize("kind", ["native", "e4m3", "fp4"])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("Hkv,D,page", [(8, 128, 256), (3, 64, 16), (1, 256, 48), (5, 16, 1)])
def test_gather(kind, out, Hkv, D, page):
    nb, src = 60 // page + 2, torch.bfloat16
    c, kw = make_cache(kind, nb, page, Hkv, D, src, seed=3)
    g = torch.Generator().manual_seed(4)
    slots = torch.randint(-1, nb * page, (70,), generator=g).cuda()   # repeats are fine
    k, v = flashdecode.gather_kv(c["k"], c["v"], slots, out_dtype=out, **kw)
    torch.cuda.synchronize()
    for n, got in (("k", k), ("v", v)):
        if kind == "native":
            val = c[n].cpu().double()
        elif kind == "e4m3":
            val = c[n].cpu().float().double() * kw[n + "_scale"].cpu().double()[:, None]
        else:
            val = dequantize_fp4(raw(c[n]), raw(c[n + "b"]), kw[n + "_scale"])
        want = val.flatten(0, 1)[slots.cpu().clamp(min=0)]
        want[slots.cpu() < 0] = 0
        # e2m1 * e4m3 is exact; the product with the head scale rounds once in
        # fp32 (2^-24) and once to the output type
        tol = (2.0 ** -24 + torch.finfo(out).eps / 2) * want.abs() + torch.finfo(out).smallest_normal * torch.finfo(out).eps
        assert got.dtype == out and bool(((got.cpu().double() - want).abs() <= tol).all())


def test_round_trip_reads_what_was_written():
    """Appended rows read back within half a step of the 4-bit grid: relative
    to s g the largest gap of e2m1 is 2 (4 to 6) below 6; a value saturated
    because s was rounded down by at most 2^-4 is off by at most 6 / 16."""
    c, kw = make_cache("fp4", 9, 16, 8, 128, torch.bfloat16)
    g = torch.Generator().manual_seed(1)
    k = torch.randn((100, 8, 128), generator=g).bfloat16().cuda()
    slots = torch.randperm(9 * 16, generator=g)[:100].cuda()
    flashdecode.append_kv_slots(k, -k, c["k"], c["v"], slots, **kw)
    got, neg = flashdecode.gather_kv(c["k"], c["v"], slots, out_dtype=torch.float32, **kw)
    step = got.abs().unflatten(-1, (-1, 16)).amax(-1, keepdim=True) / 6
    err = (got - k.float()).unflatten(-1, (-1, 16)).abs()
    assert bool((err <= step * 1.01).all())
    assert torch.isfinite(neg).all()


@pytest.mark.parametrize("kind", ["native", "fp4"])
def test_slots_past_the_pool_are_skipped_and_reported(kind):
    c, kw = make_cache(kind, 3, 16, 2, 64, torch.bfloat16)
    k = torch.randn((4, 2, 64), device="cuda").bfloat16()
    slots = torch.tensor([48, 5, 1 << 40, -9], device="cuda")
    before = clone(c)
    flashdecode.append_kv_slots(k, k, c["k"], c["v"], slots, **kw)
    torch.cuda.synchronize()
    check(kind, c, kw, before, k, k, slots)
    assert flashdecode.device_status() == FD_ERR_BAD_PAGE
    out, _ = flashdecode.gather_kv(c["k"], c["v"], slots, **kw)
    assert not out[0].any() and not out[2].any() and not out[3].any()
    assert flashdecode.device_status() == FD_ERR_BAD_PAGE


def test_slots_beyond_32_bits():
    """A pool of more than 2^31 rows' worth of slots: small rows, so that it
    fits; the last page is written and read through 64-bit offsets."""
    page, nb = 1 << 22, 513
    codes = torch.zeros((nb, page, 1, 8), dtype=torch.uint8, device="cuda")
    blocks = torch.zeros((nb, 1, page, 1), dtype=torch.uint8, device="cuda")
    c, b = codes.view(FP4), blocks.view(E4M3)
    sc = torch.full((1,), 0.25, device="cuda")
    k = torch.randn((3, 1, 16), device="cuda").bfloat16()
    slots = torch.tensor([nb * page - 1, (1 << 31) + 5, 7], device="cuda")
    kw = dict(k_scale=sc, v_scale=sc, k_block_scale=b, v_block_scale=b)
    flashdecode.append_kv_slots(k, k, c, c, slots, **kw)
    got, _ = flashdecode.gather_kv(c, c, slots, out_dtype=torch.float32, **kw)
    q, s8 = quantize_fp4(k, sc)
    want = dequantize_fp4(q[:, None], s8[:, None], sc, torch.float32)[:, 0]
    assert torch.equal(got.cpu(), want)
    assert int((codes.view(-1, 8) != 0).any(1).sum()) == 3
    assert flashdecode.device_status() == 0


def test_unaligned_16_bit_rows():
    """Rows at an odd element offset take the narrow copy."""
    for D, Hkv in ((20, 3), (128, 2)):
        c, kw = make_cache("native", 4, 16, Hkv, D, torch.float16)
        flat = torch.randn((11 * 2 * Hkv * D + 1,), device="cuda").half()
        rows = flat[1:].view(11, 2 * Hkv, D)
        k, v = rows[:, :Hkv], rows[:, Hkv:]
        slots = torch.randperm(64, device="cuda")[:11]
        before = clone(c)
        flashdecode.append_kv_slots(k, v, c["k"], c["v"], slots)
        torch.cuda.synchronize()
        check("native", c, kw, before, k, v, slots)


def test_empty_call_and_refusals():
    c, kw = make_cache("fp4", 3, 16, 2, 64, torch.bfloat16)
    before = clone(c)
    none = torch.empty((0, 2, 64), dtype=torch.bfloat16, device="cuda")
    s0 = torch.empty((0,), dtype=torch.int64, device="cuda")
    flashdecode.append_kv_slots(none, none, c["k"], c["v"], s0, **kw)
    k, v = flashdecode.gather_kv(c["k"], c["v"], s0, **kw)
    assert k.shape == (0, 2, 64)
    k = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device="cuda")
    s = torch.arange(2, device="cuda")

    def bad(err, k=k, v=k, slots=s, kc=c["k"], **over):
        with pytest.raises(err):
            flashdecode.append_kv_slots(k, v, kc, c["v"], slots, **{**kw, **over})

    bad(ValueError, slots=s.int())
    bad(ValueError, slots=s[:1])
    bad(ValueError, k=k.float())
    bad(ValueError, k=k.transpose(1, 2))
    bad(ValueError, k=k.half())
    bad(ValueError, k_block_scale=None)
    bad(ValueError, k_block_scale=kw["k_block_scale"].transpose(1, 2))
    bad(ValueError, k_scale=None)
    bad(ValueError, k_scale=kw["k_scale"].double())
    bad(ValueError, kc=c["k"][:, :8])
    flat = torch.zeros((2 * 2 * 64 + 1,), dtype=torch.bfloat16, device="cuda")
    bad(flashdecode.FlashDecodeError, k=flat[1:].view(2, 2, 64))   # rows not 16-byte aligned
    with pytest.raises(ValueError):
        flashdecode.gather_kv(c["k"], c["v"], s, out_dtype=torch.float64, **kw)
    with pytest.raises(ValueError):
        flashdecode.gather_kv(c["k"], c["v"], s, k_out=torch.empty((2, 2, 64), device="cuda"),
                              out_dtype=torch.bfloat16, **kw)
    torch.cuda.synchronize()
    for n in c:
        assert torch.equal(raw(c[n]), raw(before[n]))


@pytest.mark.parametrize("page", [16, 256])
def test_dense_append_matches_the_slot_append(page):
    """append_kv into a 4-bit cache: rows at cache_seqlens[b] + t of each
    sequence, rows without a page skipped."""
    B, sn, Hkv, D = 5, 3, 8, 128
    lens = torch.tensor([0, 14, 15, 30, -1], dtype=torch.int32)
    width = -(-(30 + sn) // page)
    bt = torch.randperm(B * width).to(torch.int32).view(B, width)
    c, kw = make_cache("fp4", B * width, page, Hkv, D, torch.bfloat16)
    k, v = (torch.randn((B, sn, Hkv, D), device="cuda").bfloat16() for _ in range(2))
    before = clone(c)
    flashdecode.append_kv(k, v, c["k"], c["v"], lens.cuda(), bt.cuda(), **kw)
    torch.cuda.synchronize()
    pos = lens.clamp(min=0)[:, None] + torch.arange(sn)
    slots = bt.gather(1, (pos // page).long()).long() * page + pos % page
    check("fp4", c, kw, before, k.flatten(0, 1), v.flatten(0, 1), slots.flatten())
    short = bt[:, :1].contiguous()
    before = clone(c)
    flashdecode.append_kv(k, v, c["k"], c["v"], lens.cuda(), short.cuda(), **kw)
    torch.cuda.synchronize()
    slots = torch.where(pos // page < 1, short.long() * page + pos % page, -1)
    check("fp4", c, kw, before, k.flatten(0, 1), v.flatten(0, 1), slots.flatten())
    assert flashdecode.device_status() == 0


@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
def test_zeros_keep_their_sign_among_other_values(src):
    c, kw = make_cache("fp4", 4, 16, 2, 64, src)
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn((20, 2, 64), generator=g) for _ in range(2))
    for x in (k, v):
        x[torch.rand(x.shape, generator=g) < 0.3] = -0.0
        x[torch.rand(x.shape, generator=g) < 0.2] = 0.0
    k, v = k.to(src).cuda(), v.to(src).cuda()
    slots = torch.randperm(64, generator=g)[:20].cuda()
    before = clone(c)
    flashdecode.append_kv_slots(k, v, c["k"], c["v"], slots, **kw)
    torch.cuda.synchronize()
    check("fp4", c, kw, before, k, v, slots)
    val, _ = flashdecode.gather_kv(c["k"], c["v"], slots, out_dtype=torch.float32, **kw)
    zero = k == 0
    assert torch.equal(torch.signbit(val)[zero], torch.signbit(k)[zero])
