"""CPU-side checks of the 8-bit operators' boundary: record layout, workspace sizes, refusals that need no device, and the 64-bit forms the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

import fp8_ref as R


@pytest.fixture(scope="module")
def lib():
    from eke_hive_b200 import _lib
    return _lib


@pytest.mark.parametrize("H,I", [(128, 128), (2048, 512), (4096, 1536), (7168, 2048), (384, 640)])
def test_record_layout(lib, H, I):
    r = lib.Fp8RecLayout()
    assert lib.load().hb_fp8_rec_layout_make(H, I, C.byref(r)) == 0
    sc = (H // 128) * (I // 128) * 4
    assert (r.w1, r.w3, r.w2, r.s1, r.s3, r.s2) == (0, H * I, 2 * H * I, 3 * H * I, 3 * H * I + sc, 3 * H * I + 2 * sc)
    assert r.total % 4096 == 0 and 0 <= r.total - (r.s2 + sc) < 4096


def test_refusals_without_a_device(lib):
    L = lib.load()
    r = lib.Fp8RecLayout()
    for H, I in ((0, 128), (128, 0), (192, 128), (128, 64), (-128, 128)):
        assert L.hb_fp8_rec_layout_make(H, I, C.byref(r)) < 0
        assert L.hb_moe_fp8_ws_bytes(4, 2, 8, H, I) == 0
    assert L.hb_fp8_rec_layout_make(128, 128, None) < 0
    assert L.hb_moe_fp8_ws_bytes(0, 2, 8, 128, 128) == 0 and L.hb_moe_fp8_ws_bytes(4, 0, 8, 128, 128) == 0
    assert L.hb_fp8_gemm_ws_bytes(0, 128, 128) == 0
    assert L.hb_fp8_gemm(None, None, None, 0, None, 0, 1, None, None, 0, None, None) < 0
    assert L.hb_fp8_quant_rows(None, None, 0, 1, 16, None, 16, None, 1, None) < 0
    assert L.hb_fp8_quantize(None, None, 0, 1, 16, None, None, None) < 0
    assert L.hb_moe_fp8(None, None, None, 1, 1, None, 0, 1, None, 128, 128, 0.0, None, None, None, None) < 0
    assert L.hb_route_grouped_topk(None, None, 1, 1, 1, 1, 1, 1, 1, 0, None, 0, 1.0, None, None, None) < 0


def test_shapes_beyond_the_range(lib):
    L = lib.load()
    r = lib.Fp8RecLayout()
    assert L.hb_fp8_rec_layout_make(1 << 20, 128, C.byref(r)) == 0 and r.w3 == 128 << 20
    for H, I in (((1 << 20) + 128, 128), (128, (1 << 20) + 128), (2 ** 31 - 128, 128)):
        assert L.hb_fp8_rec_layout_make(H, I, C.byref(r)) < 0 and L.hb_moe_fp8_ws_bytes(1, 1, 1, H, I) == 0


def test_workspaces_grow_with_the_call(lib):
    L = lib.load()
    last = 0
    for M in (1, 2, 16, 64, 65, 1000, 8192):
        ws = L.hb_moe_fp8_ws_bytes(M, 8, 256, 2048, 512)
        assert ws % 256 == 0 and ws > last and ws >= M * 8 * (2048 + 512)
        last = ws
        assert L.hb_fp8_gemm_ws_bytes(M, 5120, 2048) > 0


def test_nearest_e4m3_is_torchs_rounding():
    import torch
    v = torch.cat([torch.arange(0, 449, 0.125, dtype=torch.float64), torch.arange(0, 4096, dtype=torch.float64) * 2.0 ** -13, torch.rand(10000, dtype=torch.float64) * 448])
    assert torch.equal(R.nearest_e4m3(v), v.float().to(torch.float8_e4m3fn).double())
    assert torch.equal(R.nearest_e4m3(-v), -R.nearest_e4m3(v))
    # a value just off a border may take the code on its other side, and no further
    step = R.border(v, 1e-9)
    for d in (1 - 1e-10, 1 + 1e-10):
        assert ((R.nearest_e4m3((v * d).clamp(max=448)) - R.nearest_e4m3(v)).abs() <= step).all()


def test_route_definition():
    lg = np.array([[0.0, 2.0, 1.0, 1.0, 3.0, -1.0, -1.0, 2.9]], np.float32)
    ids, w = R.route(lg, None, 2, 4, 2, 2, "softmax", True, 1.0)         # group values by sums: (0,2) (1,1) (3,-1) (-1,2.9): groups 2 and 3 have the best pair
    assert ids.tolist() == [[4, 7]] and abs(w.sum() - 1) < 1e-12
    ids, _ = R.route(lg, np.array([0, 0, 5, 0, 0, 0, 0, 0], np.float32), 2, 4, 1, 1, "sigmoid", False, 1.0)
    assert ids.tolist() == [[2, 3]]


def test_a_wait_that_gave_up_names_its_kernel(tmp_path):
    """The 8-bit products' waits share bits with other kernels': a bit of their own tells them apart, in every wait, and the message says so."""
    import re
    import subprocess
    from pathlib import Path
    csrc = Path(__file__).resolve().parent.parent / "eke_hive_b200" / "csrc"
    (tmp_path / "text.cpp").write_text(r"""#include "device_error.h"
#include <cstdlib>
#include <initializer_list>
int main(int argc, char** argv) {
  for (uint32_t v : {kErrFp8Stage, kErrFp8AccFree, kErrFp8Loads, kErrFp8Mma, kErrFp8Acc, kErrFp8ScaleFree}) printf("%x\n", v);
  for (int i = 1; i < argc; ++i) { char s[512]; hb_device_error_text(strtoul(argv[i], nullptr, 16), s, sizeof s); printf("%s\n", s); }
}
""")
    subprocess.run(["g++", "-std=c++17", "-I", str(csrc), str(tmp_path / "text.cpp"), "-o", str(tmp_path / "text")], check=True)
    out = subprocess.run([str(tmp_path / "text"), "800400", "400", "c00000", "40000"], capture_output=True, text=True, check=True).stdout.splitlines()
    sites, text = [int(v, 16) for v in out[:6]], out[6:]
    assert len(set(sites)) == 6 and all(v & 0x800000 and bin(v).count("1") == 2 for v in sites)
    assert "0x800400" in text[0] and "8-bit product" in text[0] and "decode layer" not in text[0]
    assert "decode layer" in text[1] and "8-bit" not in text[1]
    assert "8-bit product" in text[2] and "not 16-byte aligned" in text[2]
    assert "rows of another rank" in text[3] and all(len(t) < 511 for t in text)
    for f in ("fp8_gemm.cuh", "fp8_pair.cuh"):
        waits = re.findall(r"mbar_wait\([^;]*?a\.err, (\w+)\)", (csrc / f).read_text())
        assert len(waits) >= 5 and all(w.startswith("kErrFp8") for w in waits), (f, waits)
