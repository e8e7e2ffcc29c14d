"""The layer operators at the edges of their arguments, without a GPU."""
import importlib
import importlib.util
import os
import re
import shutil
import subprocess

import pytest
import torch

import w4_cases

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, E4M3, E5M2 = 0, 2, 3
INVALID = 2
P = 4096  # an aligned address that is never dereferenced


@pytest.mark.parametrize("out", [E4M3, E5M2])
def test_norm_of_no_rows(pkg, out):
    """An empty array of row scales may be NULL; one scale of the tensor, or a given one, may not."""
    lib = pkg.load_library()

    def call(mode, scale):
        return lib.gg_rms_norm(BF16, BF16, out, mode, 0, 128, 1e-6, None, 128, None, 0, P, None, 0, None, None, scale, P, None)

    assert call(2, None) == 0 and call(2, P) == 0 and call(3, P) == 0
    for mode in (1, 3):
        assert call(mode, None) == INVALID and "scale is null" in lib.gg_layer_last_error().decode()


@pytest.mark.parametrize("at", [(0, 0, 0), (1, 23, 127), (1, 5, 64)])
def test_pack_w4_refuses_what_is_no_nibble(pkg, at):
    q = torch.full((2, 24, 128), 15, dtype=torch.uint8)
    s = torch.ones(2, 24, 2, dtype=torch.bfloat16)
    pkg.pack_w4(q, s)
    q[at] = 16
    with pytest.raises(ValueError, match="0..15"):
        pkg.pack_w4(q, s)


def test_example_quantizes_an_expert_of_zeros(pkg):
    w = torch.randn(3, 16, 32, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    w[1] = 0
    q, scale = importlib.import_module(pkg.__name__ + ".moe_example")._to_fp8(w)
    assert bool(q.float().isfinite().all()) and bool((q[1].float() == 0).all()) and bool((scale > 0).all())
    back = q.float() * scale[:, None, None]  # e4m3: 2^-4 of a value, 2^-10 of the scale at least
    assert bool(((back - w.float()).abs() <= 2.0**-4 * w.float().abs() + 2.0**-10 * scale[:, None, None]).all())


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_4_bit_sizes_reach_the_kernels_they_are_for(tmp_path):
    """A threshold that moves must take the GPU tests' sizes with it."""
    cases = w4_cases.CHOICES + w4_cases.TRIPS
    exe = tmp_path / "w4_choice"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-I", os.path.join(ROOT, "groupgemm-cktile-optimized_amd", "csrc"),
                    os.path.join(ROOT, "tests", "w4_choice.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)] + [str(v) for c in cases for v in c[1:]], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.split() == [c[0] for c in cases]


@pytest.mark.skipif(shutil.which("nm") is None, reason="needs nm")
def test_the_library_keeps_nothing_of_a_call(pkg):
    """No variable of the layer operators outlives a call but the thread's last message: what one device's call found
    would else be used on another."""
    r = subprocess.run(["nm", "-C", pkg.LIB_PATH], capture_output=True, text=True, timeout=120)
    names = [line for line in r.stdout.splitlines() if "gg::layer::" in line]
    assert r.returncode == 0 and any("g_error" in n for n in names)
    # data and its guards (local, initialized, unique or weak), but for the kernels' handles, which have parameters
    kept = [n for n in names if n.split(maxsplit=2)[1] in "bBdDuvV" and not n.endswith(")") and "g_error" not in n]
    assert not kept, kept[:3]


def _spill_check():
    spec = importlib.util.spec_from_file_location("acc", os.path.join(ROOT, "groupgemm-cktile-optimized_amd", "csrc",
                                                                      "check_mfma_acc_hazard.py"))
    acc = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(acc)
    return acc


def test_spill_check_of_short_loops():
    """The check sees a K loop of few MFMAs where it is told of it, and allows no more lane operations than told."""
    acc = _spill_check()
    mfma = "    v_mfma_f32_16x16x32_bf16 a[0:3], v[0:3], v[8:11], a[0:3]\n"
    lane = "    v_readlane_b32 s4, v185, 12\n"

    def spills(lanes, mfmas, **options):
        return acc.scan_text("\n_Zk:\n.LBB0_3:\n" + lane * lanes + mfma * mfmas + "\n.Lfunc_end0:\n", **options)[1]

    assert not spills(1, 20) and spills(1, 20, loop=8) and not spills(1, 7, loop=8)
    assert not spills(4, 20, loop=8, allow=4) and spills(5, 20, loop=8, allow=4)


def test_layer_kernels_spill_no_vector_registers():
    """The compiler's report of every kernel of the layer operators: no vector register spilled, no scratch."""
    path = os.path.join(ROOT, "groupgemm-cktile-optimized_amd", "lib", "resource_usage.txt")
    if not os.path.exists(path):
        pytest.skip("library not built")
    seen, bad, name = 0, [], None
    with open(path, errors="replace") as f:
        for line in f:
            m = re.search(r"Function Name: (\S+)", line)
            if m:
                name = m.group(1) if "2gg5layer" in m.group(1) else None
                seen += name is not None
            m = re.search(r"\s(VGPRs Spill|ScratchSize \[bytes/lane\]): (\d+)", line)
            if m and name and int(m.group(2)) != 0:
                bad.append((name, m.group(1), int(m.group(2))))
    assert seen >= 200 and not bad, (seen, bad)


def test_backward_workgroups_fit_the_gpu(pkg):
    """The RMS norm's gradient takes no more workgroups than 256 CUs hold at once, by the compiler's report of each
    instance's waves for each of a CU's four SIMDs: the numbers are written down, as the workspace's size needs them."""
    path = os.path.join(ROOT, "groupgemm-cktile-optimized_amd", "lib", "resource_usage.txt")
    if not os.path.exists(path):
        pytest.skip("library not built")
    waves, name = {}, None
    with open(path, errors="replace") as f:
        for line in f:
            m = re.search(r"Function Name: (\S+)", line)
            if m:  # <type, waves of a row, pieces, with the sums>
                name = re.search(r"norm_back_kernelINS0_\w+?ELi(\d+)ELi(\d+)ELb1E", m.group(1))
            m = re.search(r"Occupancy \[waves/SIMD\]: (\d+)", line)
            if m and name:
                key = int(name.group(1)), int(name.group(2))
                waves[key] = min(waves.get(key, 8), int(m.group(1)))
    assert len(waves) >= 9
    for hidden in (8, 512, 520, 1024, 1032, 2048, 2056, 4096, 4104, 6144, 6152, 8192, 8200, 12288, 12296, 16384, 16392, 32768):
        wpr = 1 if hidden <= 1024 else 4 if hidden <= 16384 else 16
        pieces = min(p for w, p in waves if w == wpr and p * 512 * w >= hidden)
        of_block = 16 if wpr == 16 else 4
        blocks = pkg.load_library().gg_rms_norm_backward_workspace(1 << 20, hidden) // (4 * hidden)
        assert 256 <= blocks <= 256 * (waves[wpr, pieces] * 4 // of_block), (hidden, blocks, waves[wpr, pieces])
