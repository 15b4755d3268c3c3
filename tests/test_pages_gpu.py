"""Block tables and slot maps on the GPU against plain loops: all whole
numbers, compared exactly."""
import os
import subprocess
import sys

import pytest
import torch

import flashdecode
from oracle.decode_ref import assign_pages_reference, release_pages_reference

pytestmark = pytest.mark.gpu

FD_ERR_BAD_PAGE, FD_ERR_NO_PAGES = 6, 7


def make(lens, new, page, free, width=None, seed=0, spare=3):
    """Requests holding pages of a pool, with `free` more on the stack."""
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    have = [-(-max(n, 0) // page) for n in lens]
    want = [-(-(max(n, 0) + max(a, 0)) // page) for n, a in zip(lens, new)]
    width = max(want + have + [1]) if width is None else width
    nb = sum(have) + free + spare
    perm = torch.randperm(nb, generator=g).to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b in range(B):
        table[b, :have[b]] = perm[at:at + have[b]]
        at += have[b]
    pool = torch.full((nb,), -7, dtype=torch.int32)
    pool[:free] = perm[at:at + free]
    i32 = dict(dtype=torch.int32)
    s = dict(table=table, lens=torch.tensor(lens, **i32), new=torch.tensor(new, **i32), pool=pool,
             count=torch.tensor([free, 0], **i32))
    return {k: v.cuda() for k, v in s.items()}


def assign_and_check(s, page, num_slots, in_place=False):
    before = {k: v.cpu().clone() for k, v in s.items()}
    table, slots, cu, after, left = assign_pages_reference(
        before["table"], before["lens"], before["new"], before["pool"], before["count"], page, num_slots)
    buf = torch.full((num_slots,), 99, dtype=torch.int64, device="cuda")
    got, got_cu, got_after = flashdecode.assign_pages(
        s["table"], s["lens"], s["new"], s["pool"], s["count"], page, slot_map=buf,
        seqlens_out=s["lens"] if in_place else None)
    torch.cuda.synchronize()
    assert got.data_ptr() == buf.data_ptr()
    assert torch.equal(s["table"].cpu(), table)
    assert torch.equal(got.cpu(), slots)
    assert torch.equal(got_cu.cpu(), cu)
    assert torch.equal(got_after.cpu(), after)
    assert s["count"].tolist() == [left, 0]
    assert torch.equal(s["pool"].cpu(), before["pool"])
    if not in_place:
        assert torch.equal(s["lens"].cpu(), before["lens"])
    return got, got_cu, got_after


def release_and_check(s, lens, keep, page):
    table, pool, left = release_pages_reference(s["table"].cpu(), lens.cpu(), keep.cpu(), s["pool"].cpu(),
                                                s["count"].cpu(), page)
    flashdecode.release_pages(s["table"], lens, keep, s["pool"], s["count"], page)
    torch.cuda.synchronize()
    assert torch.equal(s["table"].cpu(), table)
    assert s["count"].tolist() == [left, 0]
    assert torch.equal(s["pool"][:left].cpu(), pool[:left])   # past the count nothing is defined


@pytest.mark.parametrize("page", [1, 16, 48, 256])
@pytest.mark.parametrize("lens,new", [
    ([0], [1]), ([0], [0]), ([15, 16, 17, 0, 255, 256], [1, 1, 1, 1, 1, 1]),
    ([5, 0, 300, -2, 1000], [700, 1, 0, 33, -4]),
])
def test_small_steps(page, lens, new):
    s = make(lens, new, page, free=2000)
    n = sum(max(a, 0) for a in new)
    for extra in (0, 5):
        t = {k: v.clone() for k, v in s.items()}
        _, _, after = assign_and_check(t, page, n + extra)
        release_and_check(t, after, t["lens"], page)
        assert torch.equal(t["count"], s["count"]) and torch.equal(t["pool"], s["pool"])
    assert flashdecode.device_status() == 0


@pytest.mark.parametrize("B,hi,new_hi,page", [
    (256, 8192, 8, 16), (1000, 400, 3, 16), (37, 0, 9000, 16), (64, 0, 4096, 256), (8192, 20, 2, 1),
    (3, 100000, 50000, 64),
])
def test_many_requests(B, hi, new_hi, page):
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, hi + 1, (B,), generator=g).tolist()
    new = torch.randint(0, new_hi + 1, (B,), generator=g).tolist()
    s = make(lens, new, page, free=sum(-(-a // page) + 1 for a in new))
    _, _, after = assign_and_check(s, page, sum(new) + 11)
    # some finish, some keep a part, the rest keep everything
    keep = torch.where(torch.arange(B) % 3 == 0, 0, torch.where(torch.arange(B) % 3 == 1, after.cpu() // 2,
                                                                after.cpu())).to(torch.int32).cuda()
    release_and_check(s, after, keep, page)
    assert flashdecode.device_status() == 0


def test_lengths_in_place_over_a_run():
    """A decode loop: lengths updated in place, one token a step, then all leave."""
    s = make([15, 16, 0, 31], [1, 1, 1, 1], 16, free=40, width=8)
    pool0 = s["pool"].clone()
    for _ in range(40):
        assign_and_check(s, 16, 4, in_place=True)
    assert s["lens"].tolist() == [55, 56, 40, 71]
    release_and_check(s, s["lens"], torch.zeros_like(s["lens"]), 16)
    assert int(s["count"][0]) == 40 + 4 and not torch.equal(s["pool"], pool0)
    assert flashdecode.device_status() == 0


@pytest.mark.parametrize("free", [0, 1, 5, 6])
def test_pool_too_small(free):
    """First come, first served: the first request that does not fit stops the rest."""
    lens, new = [16, 3, 0, 40, 8], [16, 5, 80, 1, 30]   # need 1, 0, 5, 0, 2 pages
    s = make(lens, new, 16, free=free, width=10)
    assign_and_check(s, 16, sum(new))
    assert flashdecode.device_status() == FD_ERR_NO_PAGES
    assert flashdecode.device_status() == 0


def test_row_or_slot_map_too_short():
    s = make([16, 10, 0], [17, 3, 5], 16, free=10, width=2)
    assign_and_check(s, 16, 25)      # request 0 outgrows its two pages
    assert flashdecode.device_status() == FD_ERR_NO_PAGES
    s = make([16, 10, 0], [16, 3, 5], 16, free=10, width=2)
    assign_and_check(s, 16, 7)       # seven slots for 24 tokens
    assert flashdecode.device_status() == FD_ERR_NO_PAGES
    s = make([16, 4], [1, 1], 16, free=10, width=2)
    s["lens"][0] = 2147483647
    got, _, after = flashdecode.assign_pages(s["table"], s["lens"], s["new"], s["pool"], s["count"], 16,
                                             num_slots=2)
    assert after.tolist() == [2147483647, 5] and got[0] == -1 and got[1] >= 0
    assert flashdecode.device_status() == FD_ERR_NO_PAGES


def test_ids_outside_the_pool():
    s = make([10, 16], [1, 1], 16, free=5)
    s["table"][0, 0] = 10 ** 6        # under a partly filled page
    got, _, _ = flashdecode.assign_pages(s["table"], s["lens"], s["new"], s["pool"], s["count"], 16, num_slots=2)
    assert got[0] == -1 and got[1] >= 0
    assert flashdecode.device_status() == FD_ERR_BAD_PAGE
    s = make([16, 16], [1, 1], 16, free=5)
    s["pool"][4] = -3                 # on the stack
    got, _, _ = flashdecode.assign_pages(s["table"], s["lens"], s["new"], s["pool"], s["count"], 16, num_slots=2)
    assert got[0] == -1 and got[1] >= 0
    assert flashdecode.device_status() == FD_ERR_BAD_PAGE
    s = make([100, 50], [0, 0], 16, free=5)
    s["table"][0, 3] = 10 ** 6
    release_and_check(s, s["lens"], torch.zeros_like(s["lens"]), 16)
    assert flashdecode.device_status() == FD_ERR_BAD_PAGE


def test_a_page_released_twice_does_not_overflow_the_stack():
    s = make([64, 64], [0, 0], 16, free=2, spare=0)
    twice = s["table"].clone()
    zero = torch.zeros_like(s["lens"])
    release_and_check(s, s["lens"], zero, 16)
    assert s["count"].tolist() == [10, 0]
    s["table"].copy_(twice)
    release_and_check(s, s["lens"], zero, 16)
    assert s["count"].tolist() == [10, 0]
    assert flashdecode.device_status() == FD_ERR_BAD_PAGE


def test_captured_step_and_other_stream():
    """One step captured and replayed on growing lengths; the stack and the
    table advance as in eager calls."""
    s = make([15, 30, 0], [1, 2, 3], 16, free=30, width=8)
    slots = torch.empty((8,), dtype=torch.int64, device="cuda")
    cu = torch.empty((4,), dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ref = {k: v.cpu().clone() for k, v in s.items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        flashdecode.assign_pages(s["table"], s["lens"], s["new"], s["pool"], s["count"], 16, slot_map=slots,
                                 cu_new_lens=cu, seqlens_out=s["lens"])
    for _ in range(12):
        graph.replay()
        torch.cuda.synchronize()
        table, want, want_cu, after, left = assign_pages_reference(ref["table"], ref["lens"], ref["new"],
                                                                   ref["pool"], ref["count"], 16, 8)
        assert torch.equal(slots.cpu(), want) and torch.equal(cu.cpu(), want_cu)
        assert torch.equal(s["table"].cpu(), table) and torch.equal(s["lens"].cpu(), after)
        ref.update(table=table, lens=after, count=torch.tensor([left, 0], dtype=torch.int32))
    assert flashdecode.device_status() == 0


def test_refusals():
    s = make([1, 2], [1, 1], 16, free=5)
    call = lambda **kw: flashdecode.assign_pages(  # noqa: E731
        *[kw.get(n, s[n]) for n in ("table", "lens", "new", "pool", "count")], kw.get("page", 16),
        num_slots=kw.get("num_slots", 2), slot_map=kw.get("slot_map"))
    for bad in (dict(table=s["table"].long()), dict(lens=s["lens"][:1]), dict(new=s["new"].cpu()),
                dict(count=s["count"][:1]), dict(pool=s["pool"][::2]), dict(num_slots=None),
                dict(slot_map=torch.empty(2, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(flashdecode.FlashDecodeError):
        call(page=0)
    big = make([0] * 8193, [1] * 8193, 16, free=10, width=1)
    with pytest.raises(flashdecode.FlashDecodeError):
        flashdecode.assign_pages(big["table"], big["lens"], big["new"], big["pool"], big["count"], 16, num_slots=1)
    with pytest.raises(ValueError):
        flashdecode.release_pages(s["table"], s["lens"], s["lens"].long(), s["pool"], s["count"], 16)
    assert s["count"].tolist() == [5, 0]


REQUESTS_AROUND_48_KB = """
import sys
import torch
sys.path[:0] = [{root!r}, {root!r} + "/flashatte-hand_b200"]
import flashdecode
i32 = dict(dtype=torch.int32, device="cuda")
for what, B in {calls}:
    table, lens = torch.arange(B, **i32)[:, None].contiguous(), torch.ones(B, **i32)
    pool, count = torch.zeros(B, **i32), torch.zeros(2, **i32)
    if what == "assign":
        slots, cu, after = flashdecode.assign_pages(table, lens, lens, pool, count, 16, num_slots=B)
        assert torch.equal(slots, torch.arange(B, device="cuda") * 16 + 1) and bool((after == 2).all())
    else:
        flashdecode.release_pages(table, lens, torch.zeros_like(lens), pool, count, 16)
        assert count.tolist() == [B, 0] and bool((table == -1).all())
        assert torch.equal(pool, torch.arange(B, **i32).flip(0))
"""


@pytest.mark.parametrize("calls", [
    [("assign", b) for b in (4083, 4084, 4085, 4095, 4096, 8192, 1)],
    [("release", b) for b in (6110, 6111, 6112, 6143, 6144, 8192, 1)],
])
def test_requests_around_the_default_limit_of_shared_memory(calls):
    """12 B + 8 and 8 B + 4 bytes of dynamic shared memory, which with the
    kernels' static arrays pass 48 KB a little before the dynamic part does; in
    a process of its own, in which no larger call came before."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", REQUESTS_AROUND_48_KB.format(root=root, calls=calls)],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
