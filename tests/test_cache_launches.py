"""The launches of the paged-cache entry points, on the CPU: their host code
compiled with stand-ins for the device and the launchers (cache_api_host.cpp)."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent
CSRC = HERE.parent / "flashatte-hand_b200" / "csrc"


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    from flashdecode.build import nvcc_path
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    include = Path(nvcc_path()).resolve().parent.parent / "include"
    exe = tmp_path_factory.mktemp("host") / "cache_api_host"
    subprocess.run([gxx, "-std=c++17", "-O1", "-I", str(include), "-o", str(exe), str(HERE / "cache_api_host.cpp"),
                    "-x", "c++", str(CSRC / "fd_cache_api.cu"), "-ldl"], check=True)

    def run(sms, *args):
        out = subprocess.run([str(exe), str(sms), *map(str, args)], capture_output=True, text=True, timeout=60)
        assert out.returncode == 0, (out.returncode, out.stderr)
        lines = out.stdout.split("\n")[:-1]
        return int(lines[-1].split()[1]), lines[:-1]
    return run


def decode_launches(host, B, sq, Hq, Hkv, D, page, width):
    """Checks that the launches cover every row of every sequence once and that
    each one's cost line fits the kernel's 32-bit divisions; returns them."""
    status, lines = host(148, "decode", B, sq, Hq, Hkv, D, page, width)
    assert status == 0, lines
    qrows = sq * (Hq // Hkv)
    seen = {}
    for line in lines:
        seq, batch, t0, nt, rows, heads, grid, tile, seg, align = map(int, re.findall(r"-?\d+", line))
        for b in range(seq, seq + batch):
            assert seen.get(b, 0) == t0         # tile after tile
            seen[b] = t0 + nt
        length = min(width * page, 0x1fffffff)
        cut = seg + -(-length * heads // 128) * (8 + tile)
        whole = heads * (seg + align * (8 + tile) + 1)
        assert batch * nt * Hkv // heads * max(cut, whole) * (grid + 1) < 2 ** 32
        assert batch * max(cut, whole) < 2 ** 31 and 0 < batch <= 512 and nt > 0
    assert seen == {b: -(-qrows // rows) for b in range(B)}
    return lines


@pytest.mark.parametrize("B,sq,Hq,Hkv,D,page,width,launches", [
    (64, 1, 32, 8, 128, 256, 16, 1),
    (1, 4096, 32, 8, 128, 256, 64, 1),          # a prompt over a table of 16384 tokens
    (2, 256, 64, 8, 128, 256, 512, 2),          # 16 passes over a table of 131072
    (256, 1, 32, 8, 128, 256, 512, 2),          # short sequences under a wide table
    (1, 4096, 32, 8, 128, 256, 512, None),      # its passes in several launches
    (3, 1000, 28, 4, 64, 16, 16384, None),
    (1, 300, 5, 5, 256, 64, 4096, None),
    (700, 1, 8, 1, 128, 16, 2, 2),
])
def test_launches_cover_every_row(host, B, sq, Hq, Hkv, D, page, width, launches):
    lines = decode_launches(host, B, sq, Hq, Hkv, D, page, width)
    assert launches is None or len(lines) == launches, lines


def test_a_table_too_wide_for_one_pass_is_refused(host):
    status, lines = host(148, "decode", 1, 1, 512, 512, 128, 256, 1 << 21)
    assert status == 2 and "too wide" in lines[0]


@pytest.mark.parametrize("call", ["append", "append_paged", "gather"])
def test_no_count_of_the_sms_is_an_error(host, call):
    """The launchers divide by it."""
    status, lines = host(0, call)
    assert status == 4 and lines == ["cannot query SM count"]
    status, lines = host(148, call)
    assert status == 0 and lines[0].endswith("sms 148")
