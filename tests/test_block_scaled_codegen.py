"""Properties of the compiled kernels of the block-scaled cache that their speed rests on, checked on the
generated gfx950 code (no GPU needed)."""

import os
import re
import subprocess

from tests.test_kernel_codegen import CSRC, FLAGS, _functions, hipcc  # noqa: F401  (hipcc is a fixture)


def test_no_scratch_and_two_waves_a_simd(hipcc, tmp_path):  # noqa: F811
    """Nothing is parked in memory, and the two-wave workgroups stay at 256 registers: two waves a SIMD."""
    sources = {"fca_attend_block.hip": (4, 512), "fca_attend_block_wide.hip": (6, 256), "fca_merge_long.hip": (3, 256), "fca_cache_block.hip": (6, 256)}
    jobs = {
        src: subprocess.Popen(
            [hipcc, *FLAGS, "-c", "-Rpass-analysis=kernel-resource-usage", os.path.join(CSRC, src), "-o", str(tmp_path / (src + ".o"))],
            stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, cwd=CSRC,
        )
        for src in sources
    }
    for src, job in jobs.items():
        _, stderr = job.communicate()
        assert job.returncode == 0, stderr[-2000:]
        names = re.findall(r"Function Name: (\S+)", stderr)
        scratch = [int(n) for n in re.findall(r"ScratchSize \[bytes/lane\]: (\d+)", stderr)]
        vgprs = [int(n) for n in re.findall(r" VGPRs: (\d+)", stderr)]
        agprs = [int(n) for n in re.findall(r" AGPRs: (\d+)", stderr)]
        count, most = sources[src]
        assert len(names) == len(scratch) == len(vgprs) == len(agprs), (src, names)
        assert len(names) == count, (src, names)
        for name, s, v, a in zip(names, scratch, vgprs, agprs):
            assert s == 0 and v + a <= most, (name, s, v, a)


def test_tile_loops_wait_for_counted_loads(hipcc, tmp_path):  # noqa: F811
    """Between the barriers of the wide kernel's tile loops every wait for memory leaves the tiles further ahead
    in flight: a wait for everything would stop the ring."""
    out = tmp_path / "wide.s"
    res = subprocess.run([hipcc, *FLAGS, "-S", os.path.join(CSRC, "fca_attend_block_wide.hip"), "-o", str(out)], capture_output=True, text=True, cwd=CSRC)
    assert res.returncode == 0, res.stderr[-2000:]
    kernels = {n: b for n, b in _functions(out.read_text()).items() if "attend_block_wide" in n}
    assert len(kernels) == 6
    for name, body in kernels.items():
        # (requests of a wave and tile: D / 32; tiles left in flight behind the one waited for: 2, at head size 256 one)
        d = int(re.search(r"ILi(\d+)E", name).group(1))
        left = (1 if d == 256 else 2) * d // 32
        loops, label, inside = 0, "", {}
        for line in body.splitlines():
            if re.match(r"\.LBB", line):
                label = line
                inside[label] = []
            elif label:
                inside[label].append(line)
        for label, lines in inside.items():
            text = "\n".join([label, *lines])
            if "Depth=2" not in text.split("\n\t")[0] and "Depth=2" not in label:
                continue
            waits = [int(n) for n in re.findall(r"s_waitcnt [^\n]*vmcnt\((\d+)\)", text)]
            if "s_barrier" in text:
                assert waits and min(waits) == left, (name, label, waits)
                loops += 1
            else:
                assert all(w >= left for w in waits), (name, label, waits)
        assert loops == 2, (name, loops)  # full tiles, and the last one
