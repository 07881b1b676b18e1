"""Launchers of the mixture-of-experts kernels and of the 8-bit checkpoints report a launch that was refused (no GPU needed: without one
every launch is refused)."""

import ctypes
import re
from pathlib import Path

import pytest
import torch

from torchure_b200 import ops

CSRC = Path(__file__).resolve().parent.parent / "torchure_b200" / "csrc"
ROWS = {      # launcher: (linker name, arguments; pointers are null, the sizes those of a small matrix)
    "quantize8": ("_ZN2tb9quantize8EPK13__nv_bfloat16lPaPfliP11CUstream_st", "plpplip", (0, 64, 0, 0, 4, 64, 0)),
    "dequantize8": ("_ZN2tb11dequantize8EPKaPKfP13__nv_bfloat16liP11CUstream_st", "ppplip", (0, 0, 0, 4, 64, 0)),
    "swiglu8_fwd": ("_ZN2tb11swiglu8_fwdEPK13__nv_bfloat16lPS0_PaPfliP11CUstream_st", "plppplip", (0, 128, 0, 0, 0, 4, 64, 0)),
    "swiglu8_bwd": ("_ZN2tb11swiglu8_bwdEPK13__nv_bfloat16lPKaPKfPS0_liP11CUstream_st", "plppplip", (0, 64, 0, 0, 0, 4, 64, 0)),
    "expert_swiglu_bwd": ("_ZN2tb17expert_swiglu_bwdEPK13__nv_bfloat16S2_PKaPKfS6_PKiS8_PS0_S9_PfiiiP11CUstream_st", "ppppppppppiiip",
                          (0,) * 10 + (4, 2, 64, 0)),
    "rows_gather": ("_ZN2tb11rows_gatherEPKvblPKiP13__nv_bfloat16iiiiP11CUstream_st", "pblppiiiip", (0, 1, 64, 0, 0, 4, 2, 8, 64, 0)),
    "rows_combine": ("_ZN2tb12rows_combineEPKvbPKfPKiPvbiiiiP11CUstream_st", "pbpppbiiiip", (0, 1, 0, 0, 0, 1, 4, 2, 8, 64, 0)),
    "rows_combine_bwd": ("_ZN2tb16rows_combine_bwdEPKvblPK13__nv_bfloat16PKfPKiS8_PS2_PfiiiiP11CUstream_st", "pblppppppiiiip",
                         (0, 1, 64, 0, 0, 0, 0, 0, 0, 4, 2, 4, 64, 0)),
}
KINDS = {"p": ctypes.c_void_p, "l": ctypes.c_int64, "i": ctypes.c_int, "b": ctypes.c_bool}


@pytest.mark.skipif(ops.ext() is None, reason="the CUDA extension is not built")
@pytest.mark.skipif(torch.cuda.is_available(), reason="there is a GPU: launches are not refused")
@pytest.mark.parametrize("name", ROWS)
def test_refused_launches_are_reported(name):
    symbol, kinds, values = ROWS[name]
    launch = getattr(ctypes.CDLL(ops.ext().__file__), symbol)
    launch.restype, launch.argtypes = ctypes.c_int, [KINDS[k] for k in kinds]
    assert launch(*values) == -21


def test_every_launcher_returns_a_code_that_callers_look_at():
    header = re.sub(r"//[^\n]*", "", (CSRC / "moe_api.h").read_text())
    assert not re.search(r"\bvoid \w+\(", header)
    launchers = re.findall(r"\[\[nodiscard\]\] int (\w+)\(", header)
    assert set(ROWS) < set(launchers) and len(launchers) == len(re.findall(r"cudaStream_t stream\)", header))
    calls = re.sub(r"//[^\n]*", "", (CSRC / "moe_bindings.cpp").read_text())
    for m in re.finditer(rf"\btb::({'|'.join(launchers)})\(", calls):
        head = calls[:m.start()].rstrip()
        assert head.endswith("rc =") or re.search(r"\bdone\(\"[\w /]+\",$", head), m.group()


def test_launchers_keep_nothing_in_plain_globals():
    """Forward and backward passes launch from different threads: what a launcher finds out once stands behind a lock, by kernel and device."""
    for name in ("grouped_gemm_sm100.cu", "moe_route.cu", "moe_rows.cu", "moe_token.cu", "act8.cu"):
        text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
        assert not re.search(r"^(?:static )?(?:int|bool|int64_t) g?_?\w+ = [^;]*;", text, re.M), name
