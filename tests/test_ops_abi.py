"""The entry points of include/qgops.h without a device: NULL handles are
refused, the binding covers the header, and the cache's layout gives every
position and element a byte of its own."""
from __future__ import annotations

import ctypes
import pathlib
import re
from unittest import mock

import pytest

ROOT = pathlib.Path(__file__).resolve().parent.parent


def test_null_handles(rinf):
    lib, h, n = rinf.load_library(), ctypes.c_void_p(), ctypes.c_size_t()
    assert lib.qg_kv8_create(None, 1, 1, 64, 32, ctypes.byref(h)) == 1
    assert lib.qg_kv8_free(None, None) == 1
    assert lib.qg_kv8_info(None, None, None, None, None, None) == 1
    assert lib.qg_kv8_write_dev(None, None, None, None, None, None) == 1
    assert lib.qg_kv8_read_dev(None, None, 0, 0, 0, 0, None, None, None) == 1
    assert lib.qg_kv8_attention_dev(None, None, None, 1, None, 1.0, 0, None, None, 0, None) == 1
    assert lib.qg_kv8_attention_work(None, None, 1, 1, ctypes.byref(n)) == 1
    assert lib.qg_logprobs_work(None, 1, 1, 1, ctypes.byref(n)) == 1
    assert lib.qg_logprobs_dev(None, None, 0, 1, 1, 1, None, 0, None, None, 0, None, None, None, 0, None) == 1


def test_constants_match_the_header(rinf):
    text = (ROOT / "include" / "qgops.h").read_text()
    assert int(re.search(r"QG_KV8_BLOCK = (\d+)", text).group(1)) == rinf.KV8_BLOCK
    assert int(re.search(r"QG_LOGPROBS_MAX_TOP = (\d+)", text).group(1)) == rinf.LOGPROBS_MAX_TOP
    assert int(re.search(r"QG_TOKEN_NONE (0x[0-9A-F]+)u", text).group(1), 16) == rinf.TOKEN_NONE
    assert ctypes.sizeof(rinf.Rows) == 32 and ctypes.sizeof(rinf.Batch) == 24


def _function(name):
    """key_at / value_at of csrc/qg_kv8.h as Python (one C expression of integers)."""
    text = (ROOT / "rust-inference_amd" / "csrc" / "qg_kv8.h").read_text()
    args, body = re.search(name + r"\(([^)]*)\)\s*\{\s*return (.*?);", text, re.S).groups()
    names = [a.split()[-1] for a in args.split(",")]
    return eval(f"lambda {', '.join(names)}: {' '.join(re.sub(r'(?<=[0-9])u', '', body).split())}")


@pytest.mark.parametrize("dp", [64, 128, 192, 256])
def test_layout_is_one_to_one(dp):
    key, value = _function("key_at"), _function("value_at")
    for f in (lambda t, d: key(t, d, dp), value):
        assert sorted(f(t, d) for t in range(32) for d in range(dp)) == list(range(32 * dp))


def test_tensors_of_another_device(rinf):
    """Host tensors are refused before their addresses reach the library."""
    import torch

    class Context:                                # no device, and a library that is not to be called
        device, h, lib = 0, None, mock.MagicMock()
        logprobs_dev = rinf.GpuContext.logprobs_dev

    cache = rinf.Kv8Cache(Context(), None, 1, 1, 64, 32)
    x, lens = torch.zeros(1, 1, 64), torch.ones(1, dtype=torch.int32)
    for call in (lambda: cache.write_dev(x, x, lens), lambda: cache.attention_dev(x, x, lens),
                 lambda: cache.read_dev(0, 1, 0, 1, x, x),
                 lambda: Context().logprobs_dev(x[0], lens.view(1, 1), x[0, :, :1])):
        with pytest.raises(rinf.QgemvError, match="device"):
            call()
    for f in ("qg_kv8_write_dev", "qg_kv8_attention_dev", "qg_kv8_read_dev", "qg_logprobs_dev"):
        assert not getattr(Context.lib, f).called
