"""Device error codes are told by one number in the C header, the kernels and the Python messages."""

import re
from pathlib import Path

import flash_next_rtxpro6000_b200 as fx
from flash_next_rtxpro6000_b200 import _lib

ROOT = Path(fx.__file__).resolve().parents[1]


def test_codes_agree():
    header = {int(n): name for name, n in re.findall(r"#define FNX_DEVERR_(\w+) (\d+)", (ROOT / "include/fnx_gemv.h").read_text())}
    kernels = re.search(r"enum ErrCode[^{]*{(.*?)}", (ROOT / "flash_next_rtxpro6000_b200/csrc/fnx_common.cuh").read_text(), re.S)[1]
    kernels = {int(n): name for name, n in re.findall(r"ERR_(\w+) = (\d+)", kernels)}
    for code, text in _lib.DEVICE_ERRORS.items():
        assert text.startswith(kernels[code] + ":") and header[code] == kernels[code]
    assert set(kernels) - {0} == set(_lib.DEVICE_ERRORS) == set(header) - {0}


def test_sums_of_probabilities_are_arguments():
    message = str(fx.DeviceWaitError([("a", 19)]))
    assert "PROBS" in message and "out of bounds" in message and "wait" not in message
