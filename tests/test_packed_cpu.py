"""What the entry points for requests of different lengths refuse, without a GPU: the C ABI by status
before any CUDA work, the tensor functions by exception."""
import ctypes as C
import gc

import pytest
import torch

from loopfuse_b200 import _native
from loopfuse_b200 import functional as F

INVALID, UNSUPPORTED, ALIGNMENT, WORKSPACE, TOO_LARGE = -1, -2, -3, -4, -7


@pytest.fixture(autouse=True, scope="module")
def _no_garbage():
    """Tensors that cycles keep (exceptions and their frames, modules) go with the module that made them, not
    in the middle of a later test that counts allocated bytes."""
    yield
    gc.collect()


def test_plan_pages_refusals(native_lib):
    call = lambda a: native_lib.lf_plan_pages(C.byref(a), None)  # noqa: E731
    a = _native.LfPagePlanArgs()
    assert call(a) == INVALID
    for name in ("kv_lens", "new_lens", "free_pages", "block_table", "cu_seqlens", "seq_lens", "slots",
                 "positions", "pages_used"):
        setattr(a, name, 0x1000)
    a.B, a.n_free, a.bt_blocks, a.page_size, a.num_tokens = 4, 8, 2, 0, 16
    assert call(a) == INVALID                      # page size
    a.page_size, a.num_tokens = 16, -1
    assert call(a) == INVALID
    a.num_tokens, a.B = 16, 16385
    assert call(a) == TOO_LARGE
    a.B, a.slots = 4, None
    assert call(a) == INVALID


def test_append_refusals(native_lib):
    call = lambda a: native_lib.lf_kv_append_packed_bf16(C.byref(a), None)  # noqa: E731
    a = _native.LfKvAppendPackedArgs()
    assert call(a) == INVALID
    for name in ("k_new", "v_new", "k_pool", "v_pool", "slots"):
        setattr(a, name, 0x1000)
    a.T, a.Hkv, a.D, a.page_size, a.n_pages = 4, 2, 96, 16, 8
    assert call(a) == UNSUPPORTED                  # head dim
    a.D, a.k_new = 64, 0x1008
    assert call(a) == ALIGNMENT
    a.k_new = 0x1000
    a.vn_stride[0] = 4
    assert call(a) == ALIGNMENT
    a.vn_stride[0], a.n_pages = 128, 1 << 30
    assert call(a) == TOO_LARGE                    # slots past 31 bits
    a.T = 0
    assert call(a) == 0                            # nothing to store


def packed_args():
    a = _native.LfPackedArgs()
    for name in ("q", "k", "v", "out", "cu_q", "cu_k"):
        setattr(a, name, 0x1000)
    a.B, a.T, a.Tk, a.Hq, a.Hkv, a.D = 2, 64, 64, 4, 2, 64
    for i, s in enumerate((256, 64)):
        a.q_stride[i] = a.o_stride[i] = s
        a.k_stride[i] = a.v_stride[i] = s
    a.scale, a.mask_kind = 0.125, 1
    return a


def test_packed_prefill_refusals(native_lib):
    call = lambda a: native_lib.lf_packed_prefill_bf16(C.byref(a), None)  # noqa: E731
    assert call(_native.LfPackedArgs()) == INVALID

    def refused(code, **change):
        a = packed_args()
        for name, value in change.items():
            setattr(a, name, value)
        assert call(a) == code, change

    refused(INVALID, Hkv=3)
    refused(UNSUPPORTED, D=80)
    refused(UNSUPPORTED, Hq=258, Hkv=2)            # 129 query heads per kv head
    refused(INVALID, mask_kind=3)
    refused(INVALID, mask_kind=2, window=0)
    refused(INVALID, cu_k=None)
    refused(INVALID, block_table=0x1000)           # a table without its page geometry
    refused(TOO_LARGE, Tk=(1 << 30) + 1)
    refused(ALIGNMENT, q=0x1008)
    refused(ALIGNMENT, out=0x1004)
    refused(UNSUPPORTED, scale=-1.0)               # scores times a negative factor
    refused(UNSUPPORTED, scale=float("nan"))
    refused(INVALID, n_mod=9)
    for ops in ((4,), (3, 3), (3, 2), (2,)):       # exp; tanh twice; tanh, add; add
        a = packed_args()
        a.n_mod = len(ops)
        for i, op in enumerate(ops):
            a.mod_op[i], a.mod_arg[i] = op, 1.0
        assert call(a) == UNSUPPORTED, ops
    a = packed_args()
    a.o_stride[0] = 4
    assert call(a) == ALIGNMENT
    a = packed_args()
    a.T = 0
    assert call(a) == 0


def test_shared_prefix_refusals(native_lib):
    call = lambda a: native_lib.lf_shared_prefix_decode_bf16(C.byref(a), None)  # noqa: E731
    assert call(_native.LfSharedPrefixArgs()) == INVALID

    def refused(code, **change):
        a = _native.LfSharedPrefixArgs()
        for name in ("q", "k", "v", "out", "block_table", "seq_lens"):
            setattr(a, name, 0x1000)
        a.B, a.Hkv, a.G, a.D = 4, 2, 3, 64
        a.bt_blocks, a.page_size, a.n_pages = 8, 16, 64
        a.prefix_len, a.max_seq_len, a.scale = 64, 128, 0.125
        for name, value in change.items():
            setattr(a, name, value)
        assert call(a) == code, change

    refused(UNSUPPORTED, D=32)
    refused(UNSUPPORTED, G=129)
    refused(INVALID, prefix_len=129)               # more than the table holds
    refused(INVALID, max_seq_len=129)
    refused(INVALID, prefix_len=-1)
    refused(TOO_LARGE, B=65536)
    refused(ALIGNMENT, k=0x1002)
    refused(UNSUPPORTED, scale=-0.5)
    refused(WORKSPACE)                             # none given


def test_tensor_functions_refuse_cpu_tensors():
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    with pytest.raises(RuntimeError, match="no CPU path"):
        F.plan_pages(i32(0), i32(4), i32(1), torch.zeros(1, 2, dtype=torch.int32), page_size=4, num_tokens=4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        F.kv_append_packed(bf(1, 2, 64), bf(1, 2, 64), bf(4, 4, 2, 64), bf(4, 4, 2, 64), i32(0))
    with pytest.raises(RuntimeError, match="no CPU path"):
        F.packed_prefill_attention(bf(4, 2, 64), bf(4, 2, 64), bf(4, 2, 64), i32(0, 4))
    with pytest.raises(RuntimeError, match="no CPU path"):
        F.shared_prefix_decode_attention(bf(1, 2, 2, 64), bf(4, 4, 2, 64), bf(4, 4, 2, 64),
                                         torch.zeros(1, 2, dtype=torch.int32), i32(4), 0)


@pytest.mark.gpu
def test_tensor_functions_refuse_what_does_not_fit():
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    pool, q, q4 = bf(4, 4, 2, 64), bf(4, 4, 64), bf(1, 2, 2, 64)
    bad = [
        (TypeError, lambda: F.plan_pages(i32(0).long(), i32(4), i32(1), table, page_size=4, num_tokens=4)),
        (TypeError, lambda: F.plan_pages(i32(0), i32(4), i32(1), table.long(), page_size=4, num_tokens=4)),
        (ValueError, lambda: F.plan_pages(i32(0), i32(4, 1), i32(1), table, page_size=4, num_tokens=4)),
        (ValueError, lambda: F.plan_pages(i32(0), i32(4), i32(1), table.t(), page_size=4, num_tokens=4)),
        (ValueError, lambda: F.plan_pages(i32(0), i32(4), i32(1), table, page_size=0, num_tokens=4)),
        (ValueError, lambda: F.plan_pages(i32(0), i32(4), i32(1), table, page_size=4, num_tokens=-1)),
        (ValueError, lambda: F.kv_append_packed(bf(3, 2, 64), bf(3, 2, 64), pool, pool, i32(0))),
        (ValueError, lambda: F.kv_append_packed(bf(1, 1, 64), bf(1, 1, 64), pool, pool, i32(0))),
        (TypeError, lambda: F.kv_append_packed(bf(1, 2, 64).float(), bf(1, 2, 64), pool, pool, i32(0))),
        (ValueError, lambda: F.packed_prefill_attention(q, bf(4, 3, 64), bf(4, 3, 64), i32(0, 4))),
        (ValueError, lambda: F.packed_prefill_attention(q, bf(5, 2, 64), bf(5, 2, 64), i32(0, 4))),
        (ValueError, lambda: F.packed_prefill_attention(q, pool, pool, i32(0, 4), block_table=table)),
        (ValueError, lambda: F.packed_prefill_attention(q, pool, pool, i32(0, 4), block_table=table,
                                                        seq_lens=i32(4), cu_seqlens_k=i32(0, 4))),
        (ValueError, lambda: F.packed_prefill_attention(q, q, q, i32(4))),
        (ValueError, lambda: F.packed_prefill_attention(q, q, q, i32(0, 4), out=bf(5, 4, 64))),
        (_native.LfError, lambda: F.packed_prefill_attention(q, q, q, i32(0, 4), scale=-1.0)),
        (ValueError, lambda: F.shared_prefix_decode_attention(q4, pool, pool, table, i32(4), 9)),
        (ValueError, lambda: F.shared_prefix_decode_attention(q4, pool, pool, table, i32(4), 0, max_seq_len=9)),
        (ValueError, lambda: F.shared_prefix_decode_attention(q4, pool, pool, table, i32(4, 4), 0)),
        (ValueError, lambda: F.shared_prefix_decode_attention(bf(1, 1, 2, 64), pool, pool, table, i32(4), 0)),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()
