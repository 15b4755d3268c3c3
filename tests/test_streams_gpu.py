"""Calls on a stream that is not the current one: what they allocate belongs to
that stream, so that it is no block which work queued on the current stream
still reads for its last owner."""
import pytest
import torch

import flashdecode
from flashdecode import cases

pytestmark = pytest.mark.gpu


def calls():
    c = cases.custom_case("s", torch.bfloat16, [700, 33], 8, 2, page=16, seed=1)
    t, t4 = cases.materialize(c, "cuda", seed=1), cases.materialize_fp4(c, "cuda", seed=1)
    kw4 = {n: t4[n] for n in t4 if n.endswith("_scale")}
    i32 = dict(dtype=torch.int32, device="cuda")
    slots = torch.arange(300, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    part_o = torch.randn((3, 128, 40), generator=g, device="cuda").transpose(1, 2)     # copied first
    part_lse = torch.randn((40, 3), generator=g, device="cuda").t()

    def assign(stream):
        table, pool = torch.full((50, 4), -1, **i32), torch.arange(200, **i32)
        lens, new, count = torch.zeros(50, **i32), torch.full((50,), 20, **i32), torch.tensor([200, 0], **i32)
        torch.cuda.synchronize()
        return flashdecode.assign_pages(table, lens, new, pool, count, 16, num_slots=1000, stream=stream)

    return {
        "flash_decode": lambda stream: flashdecode.flash_decode(
            t["q"], t["k_cache"], t["v_cache"], t["cache_seqlens"], t["block_table"], return_softmax_lse=True,
            stream=stream),
        "flash_decode_4bit": lambda stream: flashdecode.flash_decode(
            t4["q"], t4["k_cache"], t4["v_cache"], t4["cache_seqlens"], t4["block_table"], return_softmax_lse=True,
            stream=stream, **kw4),
        "gather_kv": lambda stream: flashdecode.gather_kv(t4["k_cache"], t4["v_cache"], slots, stream=stream, **kw4),
        "assign_pages": assign,
        "combine_lse": lambda stream: flashdecode.combine_lse(part_o, part_lse, return_lse=True, stream=stream),
    }


@pytest.mark.parametrize("name", ["flash_decode", "flash_decode_4bit", "gather_kv", "assign_pages", "combine_lse"])
def test_outputs_of_a_call_on_another_stream(name):
    call = calls()[name]
    want = call(None)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    # blocks of the outputs' sizes go back to the current stream's pool
    freed = [x.clone() for x in want for _ in range(3)]
    blocks = {x.untyped_storage().data_ptr() for x in freed}
    del freed
    torch.cuda.synchronize()
    got = call(side)
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)
        assert x.untyped_storage().data_ptr() not in blocks


@pytest.mark.parametrize("name", ["flash_decode", "gather_kv", "combine_lse"])
def test_a_stream_by_its_handle(name):
    """Any object with a cuda_stream serves, the current stream among them."""
    class Handle:
        def __init__(self, stream):
            self.cuda_stream = stream.cuda_stream

    call = calls()[name]
    want = call(None)
    torch.cuda.synchronize()
    for stream in (torch.cuda.Stream(), torch.cuda.current_stream()):
        got = call(Handle(stream))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
