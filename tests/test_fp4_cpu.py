"""CPU: the 4-bit oracle against torch's own conversions, and every refusal of
the 4-bit entry points (host checks: nothing reaches a device)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import fp4_oracle as f4
from taomate_hd_b200 import capi as capi_mod


def test_e4m3_table_is_the_format():
    codes = torch.arange(127, dtype=torch.uint8)
    np.testing.assert_array_equal(f4.E4M3, codes.view(torch.float8_e4m3fn).double().numpy())


def test_nearest_code_is_rounding_to_nearest_even():
    """Against torch's conversion to e4m3 (values fp32 holds exactly), and the
    e2m1 ties by hand."""
    v = torch.cat((torch.rand(4000, generator=torch.Generator().manual_seed(0)) * 500,
                   torch.tensor(f4.E4M3[1:] + f4.E4M3[:-1]).float() / 2)).clamp(max=448.0)
    want = v.to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    got = f4.nearest_code(v.double().numpy(), np.ones(len(v)), f4.E4M3)
    np.testing.assert_array_equal(got, want)
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0])
    got = f4.E2M1[f4.nearest_code(ties, np.ones(8), f4.E2M1)]
    np.testing.assert_array_equal(got, [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0])


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_oracle_round_trip_and_padding(fmt):
    x = torch.randn(130, 96, generator=torch.Generator().manual_seed(1)).bfloat16()
    x[5] = 0.0
    packed, tiles, row = f4.quantise(x, fmt)
    value = f4.stored_values(packed, tiles, fmt)
    if row is not None:
        value = value * row.astype(np.float64)[:, None]
    # e2m1 keeps one fraction bit and the scale at most 1/16 of rounding: an element is off by a
    # quarter of itself or of the block's smallest step; at most a third of the block maximum
    block = np.abs(x.double().numpy()).reshape(130, -1, f4.BLOCK[fmt]).max(-1)
    err = np.abs(value - x.double().numpy()).reshape(130, -1, f4.BLOCK[fmt]).max(-1)
    assert (err <= block / 3 + 1e-30).all()
    # every byte that no (row, block) owns is 0
    owned = np.zeros(tiles.size, dtype=bool)
    owned[f4.tile_offsets(130, 96 // f4.BLOCK[fmt])] = True
    assert not tiles.reshape(-1)[~owned].any() and owned.sum() == 130 * 96 // f4.BLOCK[fmt]


def _lib():
    from taomate_hd_b200 import _native

    return _native.capi()


P = ctypes.c_void_p(1 << 20)  # never dereferenced: every call below is refused first
ODD = ctypes.c_void_p((1 << 20) + 8)


def test_block_scales_size():
    lib, n = _lib(), ctypes.c_uint64()
    for rows, cols, fmt, want in ((1, 32, 0, 512), (128, 64, 0, 512), (129, 64, 0, 1024),
                                  (128, 96, 0, 1024), (128, 128, 1, 512), (200, 160, 1, 2048),
                                  (0, 64, 0, 0)):
        assert lib.tm_fp4_block_scales_size(rows, cols, fmt, ctypes.byref(n)) == 0 and n.value == want
    assert lib.tm_fp4_block_scales_size(1, 48, 0, ctypes.byref(n)) == capi_mod.TM_ERR_SHAPE
    assert lib.tm_fp4_block_scales_size(1, 64, 2, ctypes.byref(n)) == capi_mod.TM_ERR_UNSUPPORTED
    assert lib.tm_fp4_block_scales_size(1, 64, 0, None) == capi_mod.TM_ERR_NULL_POINTER


@pytest.mark.parametrize("change,status", [
    (dict(format=3), "UNSUPPORTED"), (dict(rows=-1), "SHAPE"), (dict(cols=0), "SHAPE"),
    (dict(cols=48), "SHAPE"), (dict(ld=32), "SHAPE"), (dict(dtype=7), "DTYPE"),
    (dict(q=None), "NULL_POINTER"), (dict(blocks=None), "NULL_POINTER"),
    (dict(x=None), "NULL_POINTER"), (dict(scales=None), "NULL_POINTER"),
    (dict(given=P), "NULL_POINTER"),  # both scales
    (dict(format=1), "UNSUPPORTED"),  # mxfp4 takes no fp32 scale
    (dict(q=ODD), "ALIGNMENT"), (dict(cols=(1 << 30) + 32, ld=(1 << 30) + 32), "TOO_LARGE"),
    (dict(rows=0, q=None), "OK"),
])
def test_quant_refusals(change, status):
    a = dict(q=P, blocks=P, scales=P, given=None, x=P, dtype=0, format=0, rows=4, cols=64, ld=64)
    a.update(change)
    rc = _lib().tm_scaled_fp4_quant(a["q"], a["blocks"], a["scales"], a["given"], a["x"], a["dtype"],
                                    a["format"], a["rows"], a["cols"], a["ld"], None)
    assert rc == (0 if status == "OK" else getattr(capi_mod, "TM_ERR_" + status))


@pytest.mark.parametrize("change,status", [
    (dict(format=3), "UNSUPPORTED"), (dict(cols=40), "SHAPE"), (dict(numel=3), "SHAPE"),
    (dict(dtype=9), "DTYPE"), (dict(out=None), "NULL_POINTER"), (dict(out=ODD), "ALIGNMENT"),
    (dict(q=ODD), "ALIGNMENT"), (dict(rows=0), "OK"),
])
def test_dequant_refusals(change, status):
    a = dict(out=P, dtype=0, q=P, blocks=P, scales=P, numel=4, format=0, rows=4, cols=64)
    a.update(change)
    if a["rows"] == 0:
        a["numel"] = 1
    rc = _lib().tm_dequantize_fp4(a["out"], a["dtype"], a["q"], a["blocks"], a["scales"], a["numel"],
                                  a["format"], a["rows"], a["cols"], None)
    assert rc == (0 if status == "OK" else getattr(capi_mod, "TM_ERR_" + status))


def test_producer_refusals():
    lib = _lib()
    mod, rms = lib.tm_modulate_fp4_quant, lib.tm_rms_norm_modulate_fp4_quant
    res = lib.tm_residual_gate_rms_norm_modulate_fp4_quant
    #          q  b  s  hid   x  sh sc idx  stride fmt rows cols
    assert mod(P, P, P, None, P, P, P, None, 64, 0, 4, 48, None) == capi_mod.TM_ERR_SHAPE
    assert mod(P, P, P, None, P, P, P, None, 32, 0, 4, 64, None) == capi_mod.TM_ERR_SHAPE
    assert mod(P, P, P, None, P, P, P, None, 68, 0, 4, 64, None) == capi_mod.TM_ERR_ALIGNMENT
    assert mod(P, P, None, None, P, P, P, None, 64, 0, 4, 64, None) == capi_mod.TM_ERR_NULL_POINTER
    assert mod(P, P, P, None, ODD, P, P, None, 64, 0, 4, 64, None) == capi_mod.TM_ERR_ALIGNMENT
    assert mod(P, P, P, ODD, P, P, P, None, 64, 0, 4, 64, None) == capi_mod.TM_ERR_ALIGNMENT
    assert mod(P, P, P, None, P, P, P, None, 64, 5, 4, 64, None) == capi_mod.TM_ERR_UNSUPPORTED
    assert mod(P, P, P, None, P, P, P, None, 65536, 0, 4, 65536, None) == capi_mod.TM_ERR_TOO_LARGE
    assert mod(P, P, P, None, P, P, P, None, 64, 0, 0, 64, None) == capi_mod.TM_OK
    assert rms(P, P, P, None, P, None, 1e-6, P, P, None, 64, 0, 4, 64, None) == capi_mod.TM_ERR_NULL_POINTER
    assert rms(P, P, P, None, P, ODD, 1e-6, P, P, None, 64, 0, 4, 64, None) == capi_mod.TM_ERR_ALIGNMENT
    assert res(P, P, P, P, None, P, None, P, P, 1e-6, P, P, None, 64, 0, 4, 64,
               None) == capi_mod.TM_ERR_NULL_POINTER
    assert res(P, P, P, ODD, None, P, P, P, P, 1e-6, P, P, None, 64, 0, 4, 64,
               None) == capi_mod.TM_ERR_ALIGNMENT


@pytest.mark.parametrize("change,status", [
    (dict(format=2), "UNSUPPORTED"), (dict(k=48), "SHAPE"), (dict(n=252), "SHAPE"),
    (dict(m=-1), "SHAPE"), (dict(lda=128), "SHAPE"), (dict(ldb=128), "SHAPE"),
    (dict(ldo=248), "SHAPE"), (dict(epi=4), "UNSUPPORTED"), (dict(epi=3), "UNSUPPORTED"),
    (dict(epi=2, n=224, ldo=224), "SHAPE"), (dict(dtype=2), "DTYPE"), (dict(out=None), "NULL_POINTER"),
    (dict(ba=None), "NULL_POINTER"), (dict(sa=None), "NULL_POINTER"), (dict(na=7), "SHAPE"),
    (dict(nb=7), "SHAPE"), (dict(format=1), "UNSUPPORTED"), (dict(lda=264), "ALIGNMENT"),
    (dict(a=ODD), "ALIGNMENT"), (dict(bb=ODD), "ALIGNMENT"), (dict(out=ODD), "ALIGNMENT"),
    (dict(ldo=260), "ALIGNMENT"), (dict(k=(1 << 30) + 32, lda=1 << 30, ldb=1 << 30), "TOO_LARGE"),
    (dict(n=0x7fffff80 + 64, nb=1, ldo=1 << 31), "TOO_LARGE"), (dict(m=0), "OK"),
])
def test_mm_refusals(change, status):
    a = dict(out=P, dtype=0, a=P, b=P, ba=P, bb=P, sa=P, na=128, sb=P, nb=256, bias=None, format=0,
             m=128, n=256, k=512, lda=256, ldb=256, ldo=256, epi=0)
    a.update(change)
    rc = _lib().tm_scaled_mm_fp4(*a.values(), None)
    assert rc == (0 if status == "OK" else getattr(capi_mod, "TM_ERR_" + status))


def test_python_refusals():
    from taomate_hd_b200 import ops

    x = torch.randn(4, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.scaled_fp4_quant(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.dequantize_fp4(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(128, 4))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.scaled_mm_fp4(torch.zeros(4, 32, dtype=torch.uint8),
                          torch.zeros(32, 8, dtype=torch.uint8), torch.zeros(128, 4),
                          torch.zeros(128, 4))
    with pytest.raises(ValueError, match="block_format"):
        ops._is_mx("fp4")
    with pytest.raises(NotImplementedError):  # no CPU implementation is registered
        torch.ops.taomate_w8a8.scaled_fp4_quant_new(x, None, False)


@pytest.mark.parametrize("name", ["quant_fp4.cu", "gemm_fp4.cu"])
def test_reads_stay_behind_the_wait_for_the_previous_grid(name):
    """The kernels start while the grid before them runs, so no load of its results may
    be one that the compiler can move ahead of griddep_wait: a kernel with read-only
    loads takes its thread index, on which every address depends, from behind the wait,
    and the load helpers' assembly is volatile."""
    import re
    from pathlib import Path

    csrc = Path(capi_mod.__file__).parent / "csrc"
    source = (csrc / name).read_text()
    for part in source.split("__global__"):
        if re.search(r"__ldg\(|ld_cached16\(|ld_nc16\(", part):
            assert part.count("threadIdx") == 1
            assert part.index("griddep_wait();") < part.index("behind_wait(static_cast<int>(threadIdx.x))")
    text = source + "".join((csrc / h).read_text() for h in ("ptx.cuh", "rows.cuh"))
    for helper in set(re.findall(r"\b(ld_\w+|prefetch_\w+)\(", source)):
        body = re.search(rf"\b{helper}\([^)]*\)\s*{{(.*?)\n}}", text, re.S)
        assert body and not re.search(r"asm\(", body[1]), helper


def test_device_numbers_are_kept_only_once_known(tmp_path):
    """known_per_device (the resident pairs of the 4-bit product): a failed query is
    asked again, a found number is kept for its device, other devices and numbers out of
    range do not touch it, and host threads may ask at once (thread sanitiser)."""
    import shutil
    import subprocess
    from pathlib import Path

    from taomate_hd_b200 import build

    csrc = Path(capi_mod.__file__).parent / "csrc"
    source = (csrc / "gemm_fp4.cu").read_text()
    body = source[source.index("int max_fp4_pairs("):]
    assert "known_per_device(" in body[:body.index("\n}\n")] and "static int cache" not in source
    (tmp_path / "t.cpp").write_text(f"""
#include <cassert>
#include <thread>
#include <vector>
#include "{csrc / 'common.h'}"
int main() {{
  static std::atomic<int> known[64] = {{}};
  int asked = 0;
  auto fails = [&] {{ ++asked; return 0; }};
  assert(tmw::known_per_device(known, 3, fails) == 0);
  assert(tmw::known_per_device(known, 3, fails) == 0 && asked == 2);
  auto seven = [&] {{ ++asked; return 7; }};
  assert(tmw::known_per_device(known, 3, seven) == 7 && asked == 3);
  assert(tmw::known_per_device(known, 3, fails) == 7 && asked == 3);
  assert(tmw::known_per_device(known, 4, fails) == 0 && asked == 4);
  assert(tmw::known_per_device(known, -1, seven) == 0 && tmw::known_per_device(known, 64, seven) == 0);
  std::vector<std::thread> all;
  for (int i = 0; i < 8; ++i)
    all.emplace_back([&] {{
      for (int d = 0; d < 64; ++d)
        assert(tmw::known_per_device(known, d, [&] {{ return 7; }}) == 7);
    }});
  for (auto& t : all) t.join();
}}
""")
    compiler = shutil.which("g++")
    assert compiler
    command = [compiler, "-std=c++17", "-O1", f"-I{build._cuda_home() / 'include'}", "-pthread",
               str(tmp_path / "t.cpp"), "-o", str(tmp_path / "t")]
    sanitised = subprocess.run([*command, "-fsanitize=thread"], capture_output=True, text=True)
    if sanitised.returncode:  # no sanitiser runtime on this machine
        subprocess.run(command, check=True)
    subprocess.run([str(tmp_path / "t")], check=True, timeout=120)
