"""How the 8-bit product is cut, without a GPU: the parts that the kernels leave lie in the workspace that the library asks for, for every form it may pick."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def cuts(tmp_path_factory):
    exe = tmp_path_factory.mktemp("fp8_cut") / "check"
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", str(ROOT / "eke_hive_b200" / "csrc"), str(ROOT / "tests" / "fp8_cut_check.cpp"), "-o", str(exe)], check=True)

    def run(*products):
        r = subprocess.run([str(exe), *(str(v) for p in products for v in p)], capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stdout
        return [tuple(int(v) for v in line.split()) for line in r.stdout.splitlines()]
    return run


def test_parts_lie_in_the_workspace_and_steps_are_done_once(cuts):
    assert cuts() == []


def test_the_workspace_is_the_librarys(cuts):
    from eke_hive_b200 import _lib
    L = _lib.load()
    ps = [(M, N, K) for M in (1, 16, 17, 32, 33, 64, 127, 128, 129, 333, 4096) for N in (1, 256, 640, 5120) for K in (16, 4096, 16384, 17408, 1 << 20)]
    for (M, N, K), (rows, room, _) in zip(ps, cuts(*ps), strict=True):
        assert L.hb_fp8_gemm_ws_bytes(M, N, K) == room, (M, N, K, rows)


def test_tiles_of_a_pair_are_for_more_rows_than_one_cta_takes(cuts):
    """Up to 128 rows the second CTA of a pair would have no row at all."""
    ps = [(M, N, K) for M in (33, 64, 128) for N, K in ((256, 16384), (640, 17408), (7168, 2048), (2048, 2048), (4096, 1536), (256, 1 << 20))]
    assert all(rows == 128 for rows, _, _ in cuts(*ps))
    assert [rows for rows, _, _ in cuts((4096, 17408, 5120), (512, 5120, 17408))] == [256, 256]
