"""Microscaling formats without a GPU: the plain implementation's own numbers, and what the operators refuse."""

import math
import os
import re
import subprocess

import numpy as np
import pytest
import torch

import plain_mx
from liyab_amd.csrc import build
from liyab_amd.errors import KernelError
from liyab_amd.kernels import mx


def test_numbers_of_the_formats():
    assert plain_mx.E4M3[-1] == 448 and plain_mx.E4M3[1] == 2.0 ** -9 and len(plain_mx.E4M3) == 127
    t = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(t, plain_mx.E4M3)


@pytest.mark.parametrize("amax,e4m3,e2m1", [(448.0, 127, 133), (448.0000001, 128, 134), (1.75, 119, 125), (1.0, 119, 125), (7.0, 121, 127), (7.001, 122, 128),
                                            (0.0, 0, 0), (2.0 ** -149, 0, 0), (math.inf, 255, 255), (3.4e38, 247, 253)])
def test_scale_of_a_group(amax, e4m3, e2m1):
    assert plain_mx.scale_byte(amax, 8) == e4m3 and plain_mx.scale_byte(amax, 2) == e2m1


def test_rounding_of_the_plain_implementation():
    """Ties go to the even code; e4m3 agrees with torch's conversion where nothing is cut off."""
    v = np.array([0.25, 0.75, 1.25, 2.5, 3.5, 5.0, 6.9, -1.25])
    assert plain_mx.E2M1[plain_mx.nearest(v, plain_mx.E2M1)].tolist() == [0.0, 1.0, 1.0, 2.0, 4.0, 4.0, 6.0, 1.0]
    x = torch.randn(4096, generator=torch.Generator().manual_seed(1)) * torch.logspace(-4, 2, 4096)
    x = x.clamp(-448, 448)
    assert np.array_equal(plain_mx.E4M3[plain_mx.nearest(x.double().numpy(), plain_mx.E4M3)], x.abs().to(torch.float8_e4m3fn).double().numpy())


def test_operands_on_the_host_are_refused():
    rows = torch.zeros(2, 64)
    with pytest.raises(KernelError):
        mx.Mxfp4Matrix.quantize(rows)
    with pytest.raises(KernelError):
        mx.Mxfp4Matrix.pack(torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8), 64)
    with pytest.raises(KernelError):
        mx.Mxfp8Rows.empty(2, 64, device="cpu")
    with pytest.raises(KernelError):
        mx.Mxfp8Rows.pack(torch.zeros(2, 64, dtype=torch.float8_e4m3fn), torch.zeros(2, 2, dtype=torch.uint8))


@pytest.mark.parametrize("rows,width", [(0, 64), (4, 0), (-1, 64)])
def test_matrices_of_no_size_are_refused(rows, width):
    with pytest.raises(KernelError):
        mx.Mxfp4Matrix(torch.zeros(1, 1, mx.BLOCK_BYTES, dtype=torch.uint8), rows, width)


@pytest.mark.parametrize("width,codes,scales", [(1, 128, 16), (128, 128, 16), (129, 256, 16), (512, 512, 16), (513, 640, 32), (1600, 1664, 64)])
def test_places_of_rows(width, codes, scales):
    """Rows of codes are whole chunks of 128, rows of scales whole pieces of 16 bytes that hold a byte for each group of the chunks."""
    assert mx._round_up(width, mx.CHUNK) == codes and mx.Mxfp8Rows.scale_width(width) == scales and scales >= codes // 32


@pytest.mark.parametrize("source", ["mx_product.hip", "mx_tiles.hip"])
def test_the_products_waits_are_counted(source, tmp_path):
    """Both products keep loads in flight across their waits. A spilled register would be a load that the counts do not know of; and the tiles' loop waits for
    no load but the stage that it needs next, whatever the compiler makes of its reads from LDS."""
    hipcc = build.hipcc_path()
    if hipcc is None:
        pytest.skip("hipcc was not found")
    out = tmp_path / "kernels.s"
    r = subprocess.run([hipcc, *build.FLAGS, *build.FILE_FLAGS.get(source, []), "-I", build.CSRC, "--cuda-device-only", "-Rpass-analysis=kernel-resource-usage", "-S",
                        os.path.join(build.CSRC, source), "-o", str(out)], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    kernels = re.split(r"Function Name: ", r.stderr)[1:]
    assert kernels
    for k in kernels:
        spilled, scratch = (int(re.search(what + r": (\d+)", k)[1]) for what in ("VGPRs Spill", r"ScratchSize \[bytes/lane\]"))
        assert spilled == 0 and scratch == 0, f"{k.split()[0]}: {spilled} registers spilled, {scratch} bytes of scratch a lane"
    if source == "mx_tiles.hip":
        tiles = re.findall(r"(?ms)^_ZN5liyab14mx_tile_kernel\S*:.*?^\.Lfunc_end", out.read_text())
        assert len(tiles) == 72
        for t in tiles:
            # from the first product to the last; a stage's loads are the rows', the blocks' and one of scales
            loop = t[t.index("v_mfma"):t.rindex("v_mfma")]
            counts = {int(n) for n in re.findall(r"vmcnt\((\d+)\)", loop)}
            stage = re.match(r"_ZN5liyab14mx_tile_kernelILi(\d)ELi(\d)ELi(\d)ELi(\d)ELi(\d)E", t)
            mx_rows, wm, wn, tm, tn = int(stage[1]) == 2, *(int(stage[i]) for i in range(2, 6))
            loads = wm * tm * 16 // 8 // (wm * wn) + wn * tn * (1024 if mx_rows else 512) // 1024 // (wm * wn) + 1
            assert counts == {loads}, f"{t.split(':')[0]}: waits until {sorted(counts)} loads are left, a stage has {loads}"


def kernel_parameters(source, kernel, tmp_path):
    """The parameters of every instantiation of a kernel, as the compiler's intermediate form declares them."""
    hipcc = build.hipcc_path()
    if hipcc is None:
        pytest.skip("hipcc was not found")
    out = tmp_path / "kernels.ll"
    r = subprocess.run([hipcc, *build.FLAGS, *build.FILE_FLAGS.get(source, []), "-I", build.CSRC, "--cuda-device-only", "-emit-llvm", "-S", os.path.join(build.CSRC, source), "-o", str(out)],
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    found = re.findall(rf"(?m)^define [^@]*amdgpu_kernel void @_ZN5liyab\d+{kernel}I[^(]*\((.*)\) local_unnamed_addr", out.read_text())
    assert found
    return [re.split(r", (?=ptr|i\d|float|double)", f) for f in found]


@pytest.mark.parametrize("kernel", ["mx_norm_kernel", "mx_norm_long_kernel"])
def test_the_norms_stream_may_be_their_input(kernel, tmp_path):
    """`norm_mx` takes stream=x: the compiler is told nothing that the call breaks. (codes and scales are nobody else's: there it is told.)"""
    for p in kernel_parameters("mx_rows.hip", kernel, tmp_path):
        assert "noalias" in p[0] and "noalias" in p[2]
        assert not any("noalias" in p[i] for i in (4, 5, 6)), f"{kernel}: x, add or stream are declared to be nobody else's: {p[4:7]}"


def test_what_loads_behind_a_row_read_is_aligned_as_they_read(tmp_path):
    """Loads into LDS take 16 bytes: the zeros' own type says that they start on such a boundary."""
    hipcc = build.hipcc_path()
    if hipcc is None:
        pytest.skip("hipcc was not found")
    source = tmp_path / "zeros.hip"
    source.write_text('#include "mx_product.h"\nusing namespace liyab;\nstatic_assert(alignof(decltype(*mx_zeros())) >= 16 && sizeof(*mx_zeros()) == 16, "a load\'s 16 bytes");\n')
    r = subprocess.run([hipcc, *build.FLAGS, "-I", build.CSRC, "--cuda-device-only", "-fsyntax-only", str(source)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
