"""Refusals of the long-context operators beyond those of test_longctx_cpu.py,
without a GPU."""
import ctypes as C

import pytest

from inferno_b200._lib import InfernoAttention, InfernoRope, lib

A = 0x10000            # addresses that are checked, never read
STEP = 0x1000000


def _refused(rc, word):
    assert rc == -1, rc
    msg = lib().inferno_last_error().decode()
    assert word in msg, msg


@pytest.mark.parametrize("kw", [dict(type=0), dict(batch=2), dict(prefix_len=0), dict(batch=0)])
def test_attention_timeout_check_needs_a_kernel_that_waits(kw):
    """fp32, few query rows and no prefix take kernels without bounded waits."""
    a = InfernoAttention(**{**dict(type=30, batch=40, n_tokens=1, n_heads=8, n_kv_heads=2, head_dim=64, prefix_len=10000,
                                   q_stride=512, out_stride=512, q=A, out=A + STEP, prefix_k=A + 2 * STEP,
                                   prefix_v=A + 3 * STEP), **kw})
    rc = lib().inferno_debug_attention_timeout(C.byref(a), C.c_void_p(A), 1 << 40, None)
    if kw.get("batch") == 0:
        assert rc == 0
    else:
        _refused(rc, "bounded waits")


@pytest.mark.parametrize("field", ["positions", "slots", "freq_factors"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_rope_refuses_misaligned_indices(field, off):
    a = InfernoRope(type=30, n_tokens=4, n_heads=8, n_kv_heads=2, head_dim=64, rope_dim=32, theta=1e4, positions=A,
                    slots=A, n_rows=4, freq_factors=A, q=A + STEP, k=A + 2 * STEP, q_out=A + 3 * STEP, k_out=A + 4 * STEP,
                    q_stride=512, k_stride=128, q_out_stride=512, k_out_stride=128)
    setattr(a, field, A + off)
    _refused(lib().inferno_rope(C.byref(a), None), "aligned")
