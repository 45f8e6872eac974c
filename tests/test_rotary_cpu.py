"""What the rotating append, the 4-bit cache and its decode refuse, without a GPU."""
import ctypes as C
import re
from pathlib import Path

import pytest
import torch

from loopfuse_b200 import _native
from loopfuse_b200 import functional as F

INVALID, UNSUPPORTED, ALIGNMENT, WORKSPACE, TOO_LARGE = -1, -2, -3, -4, -7
HEADER = Path(__file__).resolve().parents[1] / "include" / "lf_sm100.h"


def fill(a, **change):
    for name, value in change.items():
        if isinstance(value, tuple):
            for i, x in enumerate(value):
                getattr(a, name)[i] = x
        else:
            setattr(a, name, value)
    return a


def rotary_args(**change):
    a = _native.LfRotaryArgs()
    for name in ("q", "k", "q_out", "k_out", "positions", "table"):
        setattr(a, name, 0x1000)
    fill(a, T=4, Hq=4, Hkv=2, D=64, rot=64, n_positions=8, table_stride=64, eps=1e-6, q_stride=(256, 64),
         k_stride=(128, 64), qo_stride=(256, 64), ko_stride=(128, 64))
    return fill(a, **change)


def append_args(**change):
    a = rotary_args(k_out=None, v=0x1000, k_pool=0x1000, v_pool=0x1000, slots=0x1000, page_size=16, n_pages=8,
                    bits=4, v_stride=(128, 64), kp_stride=(1280, 40, 640), vp_stride=(1280, 40, 640))
    return fill(a, **change)


def test_rotary_refusals(native_lib):
    call = lambda a: native_lib.lf_rotary_bf16(C.byref(a), None)  # noqa: E731
    assert call(_native.LfRotaryArgs()) == INVALID
    for code, change in [
            (INVALID, dict(k=None)), (INVALID, dict(table=None)), (INVALID, dict(positions=None)),
            (INVALID, dict(k_out=None)), (INVALID, dict(q_out=None)), (INVALID, dict(T=-1)),
            (INVALID, dict(Hkv=0)), (INVALID, dict(Hq=0)), (INVALID, dict(n_positions=0)),
            (INVALID, dict(eps=-1.0)), (INVALID, dict(eps=float("nan"))),
            (UNSUPPORTED, dict(D=96)), (UNSUPPORTED, dict(rot=0)), (UNSUPPORTED, dict(rot=24)),
            (UNSUPPORTED, dict(rot=80)),
            (ALIGNMENT, dict(q=0x1008)), (ALIGNMENT, dict(q_out=0x1002)), (ALIGNMENT, dict(table=0x1004)),
            (ALIGNMENT, dict(q_weight=0x1002)), (ALIGNMENT, dict(table_stride=66)),
            (ALIGNMENT, dict(k_stride=(124, 64))), (ALIGNMENT, dict(qo_stride=(256, 60))),
            (0, dict(T=0))]:
        assert call(rotary_args(**change)) == code, change
    for code, change in [
            (INVALID, dict(slots=None)), (INVALID, dict(v=None)), (INVALID, dict(v_pool=None)),
            (INVALID, dict(page_size=0)), (INVALID, dict(n_pages=0)), (UNSUPPORTED, dict(bits=8)),
            (ALIGNMENT, dict(k_pool=0x1004)), (ALIGNMENT, dict(vp_stride=(1280, 44, 640))),
            (ALIGNMENT, dict(v_stride=(128, 60))), (ALIGNMENT, dict(bits=16, kp_stride=(1280, 44, 640))),
            (TOO_LARGE, dict(n_pages=1 << 28)), (0, dict(T=0)), (0, dict(T=0, q=None, Hq=0))]:
        assert call(append_args(**change)) == code, change


def test_gather_refusals(native_lib):
    call = lambda a: native_lib.lf_kv_gather_4bit(C.byref(a), None)  # noqa: E731
    assert call(_native.LfGather4Args()) == INVALID
    for code, change in [
            (INVALID, dict(B=0)), (INVALID, dict(T=-1)), (INVALID, dict(bt_blocks=0)), (INVALID, dict(cu_k=None)),
            (INVALID, dict(page_size=0)), (UNSUPPORTED, dict(D=32)), (TOO_LARGE, dict(T=(1 << 30) + 1)),
            (ALIGNMENT, dict(k_pool=0x1004)), (ALIGNMENT, dict(kp_stride=(1280, 20, 640))),
            (ALIGNMENT, dict(v_out=0x1008)), (ALIGNMENT, dict(ko_stride=(128, 60))), (0, dict(T=0))]:
        a = _native.LfGather4Args()
        for name in ("k_pool", "v_pool", "k_out", "v_out", "block_table", "cu_k"):
            setattr(a, name, 0x1000)
        fill(a, B=2, T=8, Hkv=2, D=64, page_size=16, n_pages=8, bt_blocks=4, bt_stride=4,
             kp_stride=(1280, 40, 640), vp_stride=(1280, 40, 640), ko_stride=(128, 64), vo_stride=(128, 64))
        assert call(fill(a, **change)) == code, change


def test_decode_refusals(native_lib):
    call = lambda a: native_lib.lf_decode_4bit(C.byref(a), None)  # noqa: E731
    assert call(_native.LfDecode4Args()) == INVALID
    for code, change in [
            (UNSUPPORTED, dict(D=32)), (UNSUPPORTED, dict(G=129)), (INVALID, dict(max_seq_len=1025)),
            (INVALID, dict(window=-1)), (INVALID, dict(B=0)), (TOO_LARGE, dict(B=65536)),
            (ALIGNMENT, dict(k=0x1002)), (ALIGNMENT, dict(k_stride=(640, 20, 320))),
            (ALIGNMENT, dict(q_stride=(384, 192, 60))), (ALIGNMENT, dict(o_stride=(384, 192, 62))),
            (UNSUPPORTED, dict(scale=-0.5)), (UNSUPPORTED, dict(n_mod=1, mod_op=(4,))), (WORKSPACE, dict()),
            (ALIGNMENT, dict(workspace=0x1004, workspace_bytes=1 << 30))]:
        a = _native.LfDecode4Args()
        for name in ("q", "k", "v", "out", "block_table", "seq_lens"):
            setattr(a, name, 0x1000)
        fill(a, B=4, Hkv=2, G=3, D=64, bt_blocks=64, page_size=16, n_pages=64, max_seq_len=1024, scale=0.125,
             q_stride=(384, 192, 64), o_stride=(384, 192, 64), k_stride=(1280, 40, 640), v_stride=(1280, 40, 640))
        assert call(fill(a, **change)) == code, change


def test_workspace_holds_a_part_for_every_warp_and_unit(native_lib):
    size = native_lib.lf_decode_4bit_workspace_bytes
    assert size(4, 8, 4, 128, 0, 0) == 0
    assert size(4, 8, 129, 128, 0, 64) == 0
    assert size(4, 8, 4, 128, 0, 500) == 0               # few short units: their CTAs join them
    for B, Hkv, G, D, window, longest in ((1, 1, 1, 64, 0, 1000), (64, 8, 4, 128, 0, 500), (37, 5, 3, 64, 100, 1500),
                                          (3, 2, 17, 128, 0, 700)):
        units = B * Hkv * -(-G // 8)
        assert size(B, Hkv, G, D, window, longest) >= (units + 4) * 8 * (D + 2) * 4 + units * 8


def test_records_of_the_binding_have_the_fields_of_the_header():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    for name in ("LfRotaryArgs", "LfGather4Args", "LfDecode4Args"):
        body = re.search(r"typedef struct \{([^{}]*)\} " + name + ";", text).group(1)
        want = [re.sub(r"[\s*]|\[.*?\]", "", x.split()[-1]) for line in body.split(";") if line.strip()
                for x in line.split(",")]
        assert [f[0] for f in getattr(_native, name)._fields_] == want


def test_cache_has_the_records_of_its_head_dim():
    k, v = F.kv_cache_4bit(3, 16, 2, 128, device="cpu")
    assert k.shape == v.shape == (3, 16, 2, 80) and k.dtype == torch.uint8 and k.stride() == (2560, 80, 1280, 1)
    assert F.kv_cache_4bit(3, 16, 2, 64, device="cpu")[0].shape == (3, 16, 2, 40)
    with pytest.raises(ValueError, match="head_dim"):
        F.kv_cache_4bit(3, 16, 2, 96, device="cpu")


def test_tensor_functions_refuse_cpu_tensors():
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    k_pool, v_pool = F.kv_cache_4bit(4, 4, 2, 64, device="cpu")
    table = torch.zeros(8, 64)
    blocks = torch.zeros(1, 2, dtype=torch.int32)
    for call in (lambda: F.qk_norm_rotary(bf(1, 4, 64), bf(1, 2, 64), i32(0), table),
                 lambda: F.kv_append_rotary(bf(1, 2, 64), bf(1, 2, 64), k_pool, v_pool, i32(0), i32(0), table),
                 lambda: F.kv_gather_4bit(k_pool, v_pool, blocks, i32(0, 4), 4),
                 lambda: F.decode_attention_4bit(bf(1, 2, 2, 64), k_pool, v_pool, blocks, i32(4))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
