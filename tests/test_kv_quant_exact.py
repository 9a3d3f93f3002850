"""The cache writer's quotients, checked exhaustively on the CPU: quant8b's sequence (quant_exact_check.c) under the
writer's scales, fl(amax * fl(1 / 127)), against the IEEE divide, for every bf16 amax with a scale in [2^-100, 2^126] and
every bf16 value up to it.  A scale that has grown is such a scale times a power of two, which changes no rounding."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_quotient_exact_every_bf16(tmp_path):
    with open(os.path.join(HERE, "quant_exact_check.c")) as f:
        text = f.read()
    mine = text.replace("const float sc = amax / 127.0f;", "const float sc = amax * (1.0f / 127.0f);")
    assert mine != text
    src, exe = str(tmp_path / "chk.c"), str(tmp_path / "chk")
    with open(src, "w") as f:
        f.write(mine)
    subprocess.run(["gcc", "-O2", "-std=c11", "-ffp-contract=off", "-fno-fast-math", "-frounding-math", "-o", exe, src, "-lm"], check=True)
    cuts = [1, 0x3C00, 0x4080, 0x4300, 0x4600, 0x4C00, 0x5400, 0x6000, 0x7F80]
    procs = [subprocess.Popen([exe, hex(a), hex(b)], stdout=subprocess.PIPE, text=True) for a, b in zip(cuts, cuts[1:])]
    pairs = 0
    for p in procs:
        out, _ = p.communicate(timeout=600)
        assert p.returncode == 0, out
        pairs += int(out.split("pairs ")[1].split()[0])
    assert pairs == 523237695
