"""The attention kernels' assembly, compiled here: what the compiler cannot be told of the loads
that are written by hand."""

from __future__ import annotations

import importlib.util
import re
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def _build():
    path = ROOT / "custom-3dgs-cuda_amd" / "build.py"
    spec = importlib.util.spec_from_file_location("gsr_build", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def _outside(text: str) -> str:
    """The assembly that the compiler wrote."""
    return re.sub(r"#ASMSTART.*?#ASMEND", "", text, flags=re.S)


def test_what_is_taken_as_written_by_hand():
    text = "\ts_mov_b32 m0, s1\n\t;;#ASMSTART\n\ts_mov_b32 m0, s0\n\t;;#ASMEND\n\ts_endpgm\n"
    assert _outside(text).count("m0") == 1 and "s_endpgm" in _outside(text)


@pytest.mark.parametrize("source", ["gsd_attention_fwd.hip", "gsd_attention_bwd.hip"])
def test_m0_is_the_hand_written_loads_alone(source, tmp_path):
    """They write m0, which is reserved and cannot be named as changed: no instruction of the
    compiler's own may count on it.  And no packed fp32 instruction is there."""
    mod = _build()
    out = tmp_path / "kernels.s"
    subprocess.run([mod.HIPCC, *mod.HIP_FLAGS, "-w", "--cuda-device-only", "-S", str(mod.DECODER / source),
                    "-o", str(out)], check=True, capture_output=True, timeout=300)
    text = out.read_text()
    assert text.count("s_mov_b32 m0") > 100 and text.count("s_endpgm") > 5
    assert not re.findall(r"^.*\bm0\b.*$", _outside(text), flags=re.M)
    assert not re.findall(r"\bv_pk_(?:add|mul|fma)_f32\b", text)
