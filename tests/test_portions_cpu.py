"""What the operators for portions refuse before anything is launched, their plans, and the frequencies of stretched contexts."""
import ctypes
import math
import os
import subprocess
import sys

import pytest
import torch

from axono_b200 import _capi, ops

FAKE = 1 << 20  # an address that nothing follows: every call here is refused on the host


def turn(**kw):
    a = dict(q=FAKE, q_ld=256, k=FAKE + 64, k_ld=128, qw=None, kw=None, eps=1e-6, pos=FAKE, freq=FAKE, rot=64, inter=0, factor=1.0, mrope=0, h=0,
             w=0, qo=FAKE, ko=FAKE + 4096, rows=4, hq=4, hkv=2, d=64, dtype=_capi.FLOAT16, stream=None)
    a.update(kw)
    return _capi.lib().axb200_qk_norm_rope(*a.values())


def append(**kw):
    a = dict(qkv=FAKE, ld=512, qw=None, kw=None, eps=1e-6, qo=FAKE + 4096, k=FAKE, v=FAKE, table=FAKE, lens=FAKE, start=FAKE, pos=None, freq=FAKE, rot=64,
             inter=0, factor=1.0, mrope=0, h=0, w=0, rows=4, batch=2, hq=4, hkv=2, d=64, page=64, blocks=4, pages=8, dtype=_capi.FLOAT16,
             advance=1, stream=None)
    a.update(kw)
    return _capi.lib().axb200_qkv_norm_rope_append_portions(*a.values())


def attend(**kw):
    a = dict(q=FAKE, out=FAKE + 4096, k=FAKE, v=FAKE, table=FAKE, lens=FAKE, start=FAKE, rows=4, batch=2, hq=4, hkv=2, d=64, page=64, blocks=4, pages=8,
             max_len=200, window=0, dtype=_capi.FLOAT16, ws=FAKE, bytes=1 << 40, stream=None)
    a.update(kw)
    return _capi.lib().axb200_gqa_attention_portions_paged(*a.values())


INVALID, MEMORY, TYPE, SHAPE, POINTER = 1, 2, 3, 4, 7


def test_turn_refuses():
    for kw, status in ((dict(dtype=_capi.INT32), TYPE), (dict(rot=3), INVALID), (dict(rot=66), INVALID), (dict(rot=-2), INVALID),
                       (dict(d=257), INVALID), (dict(d=0), INVALID), (dict(rows=-1), INVALID), (dict(hq=0, hkv=0), INVALID),
                       (dict(q=None), POINTER), (dict(ko=None), POINTER), (dict(pos=None), POINTER), (dict(freq=None), POINTER),
                       (dict(q_ld=255), SHAPE), (dict(k_ld=127), SHAPE), (dict(q_ld=300), SHAPE), (dict(rows=0), 0), (dict(h=-1), INVALID)):
        assert turn(**kw) == status, kw


def test_append_refuses():
    for kw, status in ((dict(dtype=_capi.BFLOAT16), TYPE), (dict(rot=65), INVALID), (dict(batch=0), INVALID), (dict(page=32), INVALID),
                       (dict(page=0), INVALID), (dict(blocks=0), INVALID), (dict(pages=0), INVALID), (dict(hkv=0), INVALID),
                       (dict(hq=0), INVALID), (dict(ld=511), SHAPE), (dict(start=None), POINTER), (dict(lens=None), POINTER),
                       (dict(freq=None), POINTER), (dict(qkv=None), POINTER), (dict(d=300, rot=0), INVALID), (dict(qo=FAKE), INVALID),
                       (dict(blocks=1 << 26), INVALID), (dict(rows=0), 0)):
        assert append(**kw) == status, kw


def test_attention_refuses():
    for kw, status in ((dict(dtype=_capi.BFLOAT16), TYPE), (dict(d=257), INVALID), (dict(hkv=3), SHAPE), (dict(page=96), INVALID),
                       (dict(max_len=0), INVALID), (dict(max_len=1 << 31), INVALID), (dict(window=-1), INVALID), (dict(batch=0), INVALID),
                       (dict(rows=-1), INVALID), (dict(out=None), POINTER), (dict(out=FAKE), INVALID), (dict(table=None), POINTER), (dict(rows=0), 0),
                       (dict(blocks=1 << 26), INVALID), (dict(max_len=1 << 20, blocks=1 << 14, ws=None), MEMORY),
                       (dict(max_len=1 << 20, blocks=1 << 14, bytes=16), MEMORY), (dict(max_len=1 << 20, blocks=1 << 14, ws=FAKE + 4), POINTER)):
        assert attend(**kw) == status, kw


def test_workspace_is_for_few_rows_over_many_keys():
    size = lambda rows, batch, max_len, hkv=8, window=0: _capi.lib().axb200_gqa_attention_portions_workspace_bytes(  # noqa: E731
        rows, batch, 16, hkv, 128, 64, 1 << 14, max_len, window, 1, _capi.FLOAT16)
    assert size(8, 1, 32768) > 0
    assert size(8, 1, 64) == 0
    assert size(8, 1, 32768, window=64) == 0
    assert size(8192, 1, 8192) == 0
    assert size(8, 1, 32768) < 64 << 20
    assert size(0, 1, 32768) == 0


def test_operators_want_cuda_tensors():
    x = torch.zeros((2, 4, 64), dtype=torch.float16)
    for call in (lambda: ops.qk_norm_rope(x, None, torch.zeros(2, dtype=torch.int64), torch.ones(32, dtype=torch.float64)),
                 lambda: ops.gqa_attention_portions_paged(x, x, x, x, x, x, 10),
                 lambda: ops.qkv_norm_rope_append_portions(x[0], 2, None, None, 1e-6, x, x, x, x, x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(RuntimeError):
        ops.qk_norm_rope(None, None, None, None)


def test_frequencies():
    base, one = ops.rope_frequencies(64, 1e4, device="cpu")
    assert base.dtype == torch.float64 and one == 1.0
    for i in range(32):
        assert math.isclose(float(base[i]), 1e4 ** (-i / 32), rel_tol=1e-14)
    half, one = ops.rope_frequencies(64, 1e4, dict(kind="linear", factor=2.0), device="cpu")
    assert one == 1.0 and torch.allclose(half * 2, base, rtol=1e-14, atol=0)
    ntk, _ = ops.rope_frequencies(64, 1e4, dict(kind="ntk", factor=4.0), device="cpu")
    assert float(ntk[0]) == 1.0 and math.isclose(float(ntk[-1]) * 4, float(base[-1]), rel_tol=1e-12)
    smooth, one = ops.rope_frequencies(128, 5e5, dict(kind="smooth", factor=8.0, original=8192), device="cpu")
    plain, _ = ops.rope_frequencies(128, 5e5, device="cpu")
    assert one == 1.0
    for f, p in zip(smooth.tolist(), plain.tolist()):
        turns = 8192 * p / (2 * math.pi)
        want = p if turns > 4 else p / 8 if turns < 1 else p * ((turns - 1) / 3) + p / 8 * (1 - (turns - 1) / 3)
        assert math.isclose(f, want, rel_tol=1e-12)
    yarn, factor = ops.rope_frequencies(128, 1e4, dict(kind="yarn", factor=16.0, original=4096), device="cpu")
    plain, _ = ops.rope_frequencies(128, 1e4, device="cpu")
    assert math.isclose(factor, 0.1 * math.log(16) + 1)
    ratio = plain / yarn
    assert float(ratio[0]) == 1.0 and math.isclose(float(ratio[-1]), 16.0, rel_tol=1e-12) and (ratio.diff() >= -1e-12).all()
    # 32 turns in 4096 tokens: pair 128 ln(4096 / (64 pi)) / (2 ln 1e4) = 20.9; one turn: 45.03
    assert float(ratio[20]) == 1.0 and float(ratio[21]) > 1.0 and float(ratio[45]) < 16.0 and math.isclose(float(ratio[46]), 16.0, rel_tol=1e-12)
    assert ops.rope_frequencies(128, 1e4, dict(kind="yarn", factor=16.0, original=4096, attention_factor=1.0), device="cpu")[1] == 1.0
    for bad in (dict(kind="other", factor=2.0), dict(kind="linear"), dict(kind="linear", factor=0.5), dict(kind="yarn", factor=2.0),
                dict(kind="smooth", factor=2.0, original=10, low=4.0, high=1.0)):
        with pytest.raises(RuntimeError):
            ops.rope_frequencies(64, 1e4, bad, device="cpu")
    for rot in (0, 3, -2):
        with pytest.raises(RuntimeError):
            ops.rope_frequencies(rot, device="cpu")


def test_signatures_hold_what_the_header_declares():
    for name, args in (("axb200_qk_norm_rope", 23), ("axb200_qkv_norm_rope_append_portions", 30),
                       ("axb200_gqa_attention_portions_workspace_bytes", 11), ("axb200_gqa_attention_portions_paged", 21)):
        assert len(_capi.SIGNATURES[name][1]) == args
    assert _capi.SIGNATURES["axb200_gqa_attention_portions_workspace_bytes"][0] is ctypes.c_size_t


def test_the_form_with_slots_refuses_what_the_other_does():
    for kw, status in ((dict(dtype=_capi.BFLOAT16), TYPE), (dict(batch=0), INVALID), (dict(ld=511), SHAPE), (dict(lens=None), POINTER), (dict(rows=0), 0)):
        a = dict(qkv=FAKE, ld=512, qw=None, kw=None, eps=1e-6, qo=FAKE + 4096, k=FAKE, v=FAKE, table=FAKE, lens=FAKE, start=FAKE, pos=None, freq=FAKE,
                 rot=64, inter=0, factor=1.0, mrope=0, h=0, w=0, rows=4, batch=2, hq=4, hkv=2, d=64, page=64, blocks=4, pages=8,
                 dtype=_capi.FLOAT16, advance=1, slots=FAKE, stream=None)
        a.update(kw)
        assert _capi.lib().axb200_qkv_norm_rope_append_portions_at(*a.values()) == status, kw


def test_the_operators_import_where_torch_lacks_cuda_bindings():
    """A torch built without CUDA has neither of the two names that calls take device and stream from."""
    code = ("import torch\n"
            "for name in ('_cuda_getDevice', '_cuda_getCurrentRawStream'):\n"
            "    if hasattr(torch._C, name): delattr(torch._C, name)\n"
            "from axono_b200 import ops\n"
            "assert ops._device_now is torch.cuda.current_device and callable(ops._stream_now)\n")
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def test_outputs_that_share_memory_with_inputs_are_refused():
    """Wherever the output begins in or runs into what is read - but not between the rows of a strided input."""
    q_bytes = 4 * 4 * 64 * 2
    for off in (2, 128, q_bytes - 2, -2, 2 - q_bytes):
        assert attend(out=FAKE + off) == INVALID, off
        assert turn(k=None, hkv=0, ko=None, qo=FAKE + off) == INVALID, off
        assert turn(q=None, hq=0, qo=None, k=FAKE, k_ld=256, hkv=4, ko=FAKE + off) == INVALID, off
    for off in (2, 4 * 512 * 2 - 2, 2 - q_bytes):
        assert append(qo=FAKE + off) == INVALID, off
    # rows of 1024 bytes, 8192 apart: from the gap behind one into the next
    for off in (8192 - 512, 3 * 8192 - 512, 3 * 8192 + 1022, 2 - q_bytes):
        assert append(ld=4096, qo=FAKE + off) == INVALID, off
