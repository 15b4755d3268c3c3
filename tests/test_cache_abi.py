"""CPU checks of the paged-cache entry points' refusals: every bad argument
returns its status and a message before any device is touched."""
import flashdecode
import pytest

P = 4096          # a non-null, aligned "pointer" that is never followed
BF16, FP16, FP32, E4M3, E2M1 = range(5)
INVALID, UNSUPPORTED = 1, 2


def decode_args(**kw):
    a = dict(q=P, k=P, v=P, kb=P, vb=P, ks=P, vs=P, kn=None, vn=None, new=0, out=P, lse=None, sl=P, bt=P,
             stride=4, B=2, sq=1, Hq=8, Hkv=2, D=128, page=16, nb=8, dt=BF16, odt=BF16, scale=0.1, causal=0,
             maxk=0, ws=None, wsn=0, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(sl=None), INVALID), (dict(bt=None), INVALID),
    (dict(k=None), INVALID), (dict(kb=None), INVALID), (dict(vs=None), INVALID), (dict(kn=P), INVALID),
    (dict(kn=P, vn=P, new=0), INVALID), (dict(kn=P, vn=P, new=70000), INVALID), (dict(B=0), INVALID),
    (dict(sq=0), INVALID), (dict(Hkv=3), INVALID), (dict(page=0), INVALID), (dict(nb=0), INVALID),
    (dict(dt=FP32), INVALID), (dict(odt=FP16), INVALID), (dict(scale=float("inf")), INVALID),
    (dict(stride=0), INVALID), (dict(D=96), UNSUPPORTED), (dict(D=32), UNSUPPORTED), (dict(page=8), UNSUPPORTED),
    (dict(page=24), UNSUPPORTED), (dict(q=P + 8), UNSUPPORTED), (dict(kb=P + 4), UNSUPPORTED),
    (dict(B=1 << 31), UNSUPPORTED), (dict(nb=1 << 31), UNSUPPORTED), (dict(Hq=1 << 17, Hkv=1 << 17), UNSUPPORTED),
])
def test_decode_fp4(lib, kw, code):
    assert lib.fd_decode_paged_fp4(*decode_args(**kw)) == code
    assert flashdecode.last_error()[0] == code and flashdecode.last_error()[1]


@pytest.mark.parametrize("args", [(0, 1, 8, 2, 128), (2, 0, 8, 2, 128), (2, 1, 8, 3, 128), (2, 1, 8, 2, 96)])
def test_workspace_size_of_unsupported_shapes_is_zero(lib, args):
    assert lib.fd_decode_workspace_size_fp4(*args) == 0


def append_args(**kw):
    a = dict(k=P, kst=256, v=P, vst=256, kc=P, vc=P, kb=P, vb=P, ks=P, vs=P, slots=P, T=4, Hkv=2, D=128, page=16,
             nb=8, dt=BF16, cdt=E2M1, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(k=None), INVALID), (dict(slots=None), INVALID), (dict(kc=None), INVALID), (dict(kb=None), INVALID),
    (dict(cdt=E4M3, ks=None), INVALID), (dict(dt=FP32), INVALID), (dict(cdt=FP32), INVALID),
    (dict(cdt=FP16), INVALID), (dict(kst=255), INVALID), (dict(vst=0), INVALID), (dict(T=-1), INVALID),
    (dict(page=0), INVALID), (dict(Hkv=0), INVALID), (dict(nb=1 << 31), UNSUPPORTED),
    (dict(Hkv=65535, D=65535, kst=1 << 40, vst=1 << 40), UNSUPPORTED),
])
def test_append_slots(lib, kw, code):
    assert lib.fd_append_kv_slots(*append_args(**kw)) == code


def test_no_rows_is_no_call(lib):
    assert lib.fd_append_kv_slots(*append_args(T=0, k=None, v=None, slots=None)) == 0


@pytest.mark.parametrize("kw,code", [
    (dict(out=None), INVALID), (dict(slots=None), INVALID), (dict(odt=E4M3), INVALID), (dict(T=-1), INVALID),
    (dict(D=24), UNSUPPORTED), (dict(out=P + 2), UNSUPPORTED), (dict(cdt=7), INVALID),
])
def test_gather_slots(lib, kw, code):
    a = dict(kc=P, vc=P, kb=P, vb=P, ks=P, vs=P, slots=P, T=4, out=P, vout=P, Hkv=2, D=128, page=16, nb=8, cdt=E2M1,
             odt=BF16, stream=None)
    a.update(kw)
    assert lib.fd_gather_kv_slots(*a.values()) == code


@pytest.mark.parametrize("kw,code", [
    (dict(kn=None), INVALID), (dict(sl=None), INVALID), (dict(B=0), INVALID), (dict(new=0), INVALID),
    (dict(dt=FP32), INVALID), (dict(new=70000), UNSUPPORTED), (dict(B=1 << 20, new=1 << 14), UNSUPPORTED),
])
def test_append_paged_fp4(lib, kw, code):
    a = dict(kn=P, vn=P, kc=P, vc=P, kb=P, vb=P, ks=P, vs=P, sl=P, bt=P, stride=4, B=2, new=1, Hkv=2, D=128, page=16,
             nb=8, dt=BF16, stream=None)
    a.update(kw)
    assert lib.fd_append_kv_paged_fp4(*a.values()) == code


@pytest.mark.parametrize("kw,code", [
    (dict(bt=None), INVALID), (dict(count=None), INVALID), (dict(slots=None), INVALID), (dict(B=0), INVALID),
    (dict(page=0), INVALID), (dict(n=-1), INVALID), (dict(stride=0), INVALID), (dict(B=8193), UNSUPPORTED),
    (dict(nb=1 << 31), UNSUPPORTED), (dict(n=1 << 31), UNSUPPORTED),
])
def test_assign_pages(lib, kw, code):
    a = dict(bt=P, stride=4, sl=P, new=P, pool=P, count=P, B=2, page=16, nb=8, after=P, cu=P, slots=P, n=8, stream=None)
    a.update(kw)
    assert lib.fd_assign_pages(*a.values()) == code


@pytest.mark.parametrize("kw,code", [
    (dict(bt=None), INVALID), (dict(keep=None), INVALID), (dict(B=0), INVALID), (dict(page=0), INVALID),
    (dict(B=8193), UNSUPPORTED),
])
def test_release_pages(lib, kw, code):
    a = dict(bt=P, stride=4, sl=P, keep=P, pool=P, count=P, B=2, page=16, nb=8, stream=None)
    a.update(kw)
    assert lib.fd_release_pages(*a.values()) == code


def test_python_calls_refuse_cpu_tensors():
    import torch
    i32 = dict(dtype=torch.int32)
    with pytest.raises(ValueError):
        flashdecode.assign_pages(torch.zeros((1, 2), **i32), torch.zeros(1, **i32), torch.zeros(1, **i32),
                                 torch.zeros(4, **i32), torch.zeros(2, **i32), 16, num_slots=1)
    with pytest.raises(ValueError):
        flashdecode.release_pages(torch.zeros((1, 2), **i32), torch.zeros(1, **i32), torch.zeros(1, **i32),
                                  torch.zeros(4, **i32), torch.zeros(2, **i32), 16)
    c = torch.zeros((2, 16, 1, 32), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        flashdecode.append_kv_slots(c[0], c[0], c, c, torch.zeros(16, dtype=torch.int64))
    with pytest.raises(ValueError):
        flashdecode.gather_kv(c, c, torch.zeros(16, dtype=torch.int64))


def test_status_string(lib):
    assert lib.fd_error_string(7) == b"not enough pages or slots for the step"


@pytest.mark.parametrize("kw", [dict(out=P + 2), dict(odt=FP32, out=P + 4)])
def test_decode_fp4_output_alignment(lib, kw):
    assert lib.fd_decode_paged_fp4(*decode_args(**kw)) == UNSUPPORTED


def test_tensors_of_several_devices_are_refused():
    class OnDevice:
        def __init__(self, index):
            self.index = index

        def get_device(self):
            return self.index

    from flashdecode import ops
    ops._require_device(OnDevice(1), OnDevice(1), None, OnDevice(1))
    with pytest.raises(ValueError, match="one device"):
        ops._require_device(OnDevice(0), OnDevice(0), None, OnDevice(1))
    with pytest.raises(ValueError, match="CUDA tensors only"):
        ops._require_device(OnDevice(-1), OnDevice(-1))


def test_workspace_size_by_cache_type(lib):
    import torch
    assert flashdecode.workspace_size(2, 8, 2, 96, kv_dtype=torch.float4_e2m1fn_x2) == 0   # not a head dim it has
