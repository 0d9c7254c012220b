"""Refusals and host logic of the long-context operators, without a GPU: every
bad argument is turned into a status and a message before any device work."""
import ctypes as C
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

from inferno_b200._lib import InfernoAttention, InfernoEvict, InfernoRope, lib

HEADER = Path(__file__).resolve().parent.parent / "include" / "inferno_b200.h"
A = 0x10000            # addresses that are checked, never read
STEP = 0x1000000


def _rope(**kw):
    a = dict(type=30, n_tokens=4, n_heads=8, n_kv_heads=2, head_dim=64, rope_dim=32, theta=1e4, positions=A,
             q=A + STEP, k=A + 2 * STEP, q_out=A + 3 * STEP, k_out=A + 4 * STEP, q_stride=512, k_stride=128,
             q_out_stride=512, k_out_stride=128)
    a.update(kw)
    return InfernoRope(**a)


def _attn(**kw):
    a = dict(type=30, batch=2, n_tokens=1, n_heads=8, n_kv_heads=2, head_dim=64, prefix_len=100, max_len=50,
             q_stride=512, out_stride=512, seq_stride=50 * 128, score_stride=50, q=A, out=A + STEP,
             prefix_k=A + 2 * STEP, prefix_v=A + 3 * STEP, k_cache=A + 4 * STEP, v_cache=A + 5 * STEP,
             lens=A + 6 * STEP, scores=A + 7 * STEP)
    a.update(kw)
    return InfernoAttention(**a)


def _evict(**kw):
    a = dict(type=30, batch=2, n_kv_heads=2, head_dim=64, max_len=50, budget=20, n_sink=2, n_recent=4,
             seq_stride=50 * 128, score_stride=50, k_cache=A, v_cache=A + STEP, scores=A + 2 * STEP,
             slot_pos=A + 3 * STEP, lens=A + 4 * STEP, next_pos=A + 5 * STEP, scores_out=A + 6 * STEP,
             slot_pos_out=A + 7 * STEP, lens_out=A + 8 * STEP)
    a.update(kw)
    return InfernoEvict(**a)


def _refused(rc, word):
    assert rc == -1, rc
    msg = lib().inferno_last_error().decode()
    assert word in msg, msg


@pytest.mark.parametrize("kw,word", [
    (dict(type=2), "type"), (dict(n_tokens=-1), "sizes"), (dict(head_dim=0), "sizes"), (dict(rope_dim=31), "rope_dim"),
    (dict(rope_dim=66), "rope_dim"), (dict(rope_dim=0), "rope_dim"), (dict(head_dim=2048, rope_dim=1024), "rope_dim"),
    (dict(layout=2), "layout"), (dict(scaling=3), "scaling"), (dict(inverse=2), "inverse"), (dict(theta=1.0), "theta"),
    (dict(theta=float("nan")), "theta"), (dict(scaling=1, factor=0.0), "factor"), (dict(scaling=2, factor=4.0), "orig_ctx"),
    (dict(scaling=2, factor=4.0, orig_ctx=100, beta_slow=-1.0), "beta"), (dict(mscale=-1.0), "mscale"),
    (dict(positions=None), "positions"), (dict(q=None), "q or q_out"), (dict(k_out=None), "k_out"),
    (dict(v=A + 5 * STEP, v_out=A + 6 * STEP, v_stride=128, v_out_stride=128), "slots"),
    (dict(slots=A, n_rows=-1), "n_rows"), (dict(q_stride=511), "stride"), (dict(k_out_stride=-128), "stride"),
    (dict(q=A + STEP + 1), "aligned"), (dict(n_heads=1 << 20), "heads"),
    # an output over an input of other strides, over another output, a shifted copy of itself, a cache over its source
    (dict(q_out=A + STEP, q_out_stride=1024), "overlaps"), (dict(k_out=A + 3 * STEP), "overlaps"),
    (dict(q_out=A + STEP + 64), "overlaps"), (dict(k_out=A + STEP, k_out_stride=512), "overlaps"),
    (dict(slots=A, n_rows=4, k_out=A + 2 * STEP), "overlaps"),
])
def test_rope_refuses(kw, word):
    _refused(lib().inferno_rope(C.byref(_rope(**kw)), None), word)


def test_rope_struct_size_null_and_empty():
    _refused(lib().inferno_rope(None, None), "null")
    a = _rope()
    a.struct_size -= 8
    _refused(lib().inferno_rope(C.byref(a), None), "struct_size")
    assert lib().inferno_rope(C.byref(_rope(n_tokens=0, positions=None)), None) == 0
    assert lib().inferno_rope(C.byref(_rope(n_heads=0, k=None)), None) == 0


ATTN_SIZES = [
    (dict(type=8), "type"), (dict(head_dim=96), "head_dim"), (dict(batch=-1), "sizes"), (dict(n_tokens=0), "sizes"),
    (dict(n_heads=7), "sizes"), (dict(n_kv_heads=0), "sizes"), (dict(prefix_len=-1), "prefix_len"),
    (dict(max_len=-5), "max_len"), (dict(batch=1 << 20, n_tokens=1 << 10), "query rows"),
    (dict(scale=float("inf")), "scale"),
]


@pytest.mark.parametrize("kw,word", ATTN_SIZES + [
    (dict(q=None), "q or out"), (dict(out=None), "q or out"), (dict(prefix_v=None), "prefix"), (dict(lens=None), "lens"),
    (dict(k_cache=None), "k_cache"), (dict(q_stride=511), "q_stride"), (dict(out_stride=0), "out_stride"),
    (dict(seq_stride=49 * 128), "seq_stride"), (dict(score_stride=49), "score_stride"), (dict(q=A + 8), "16 bytes"),
    (dict(q_stride=516), "16 bytes"), (dict(prefix_k=A + 2), "16 bytes"), (dict(seq_stride=50 * 128 + 4), "16 bytes"),
    (dict(lens=A + 2), "4 bytes"), (dict(scores=A + 1), "4 bytes"),
])
def test_attention_refuses(kw, word):
    _refused(lib().inferno_attention_cached(C.byref(_attn(**kw)), C.c_void_p(A), 1 << 40, None), word)


@pytest.mark.parametrize("kw,word", ATTN_SIZES)
def test_attention_workspace_refuses(kw, word):
    _refused(lib().inferno_attention_cached_workspace(C.byref(_attn(**kw))), word)


def test_attention_workspace_checked():
    a = _attn()
    n = lib().inferno_attention_cached_workspace(C.byref(a))
    assert n > 0 and n % 256 == 0
    for ws, size in ((A, n - 1), (None, n), (A + 128, n)):
        _refused(lib().inferno_attention_cached(C.byref(a), C.c_void_p(ws), size, None), "workspace")
    assert lib().inferno_attention_cached(C.byref(_attn(batch=0)), None, 0, None) == 0
    # the gathered weights need the logits of the own rows
    assert lib().inferno_attention_cached_workspace(C.byref(_attn(scores=None))) < n


EVICT_SIZES = [
    (dict(type=12), "type"), (dict(batch=-1), "sizes"), (dict(n_kv_heads=0), "sizes"), (dict(batch=40000), "sizes"),
    (dict(max_len=-1), "sizes"), (dict(max_len=1000001, seq_stride=1 << 40, score_stride=1 << 30), "max_len"), (dict(head_dim=65), "head_dim"), (dict(head_dim=16384), "head_dim"),
    (dict(budget=0), "budget"), (dict(n_sink=17), "budget"), (dict(n_recent=-1), "budget"), (dict(reserved=1), "reserved"),
]


@pytest.mark.parametrize("kw,word", EVICT_SIZES + [
    (dict(scores_out=None), "null"), (dict(next_pos=None), "null"), (dict(seq_stride=49 * 128), "seq_stride"),
    (dict(score_stride=49), "score_stride"), (dict(k_cache=A + 8), "16 bytes"), (dict(lens_out=A + 2), "4 bytes"),
])
def test_evict_refuses(kw, word):
    _refused(lib().inferno_cache_evict(C.byref(_evict(**kw)), C.c_void_p(A), 1 << 40, None), word)


@pytest.mark.parametrize("kw,word", EVICT_SIZES)
def test_evict_workspace_refuses(kw, word):
    _refused(lib().inferno_cache_evict_workspace(C.byref(_evict(**kw))), word)


@pytest.mark.parametrize("kw", [dict(), dict(type=0, head_dim=256), dict(prefix_len=0), dict(prefix_len=1 << 20),
                                dict(n_tokens=1 << 30, n_heads=8, n_kv_heads=2)])
def test_attention_workspace_of_an_empty_batch(kw):
    # a status or a size: an empty batch has no rows to cut the prefix for
    code = ("import ctypes as C\n"
            "from inferno_b200._lib import InfernoAttention, lib\n"
            f"a = InfernoAttention(**{dict(dict(type=30, batch=0, n_tokens=1, n_heads=8, n_kv_heads=2, head_dim=64, prefix_len=100, max_len=50), **kw)!r})\n"
            "print(lib().inferno_attention_cached_workspace(C.byref(a)))\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True,
                       cwd=HEADER.parent.parent / "inferno.jl_b200", timeout=120)
    assert r.returncode == 0 and int(r.stdout) >= 0, (r.returncode, r.stderr)


def test_evict_workspace_checked():
    a = _evict()
    n = lib().inferno_cache_evict_workspace(C.byref(a))
    assert n > 0
    for ws, size in ((A, n - 1), (None, n), (A + 4, n)):
        _refused(lib().inferno_cache_evict(C.byref(a), C.c_void_p(ws), size, None), "workspace")
    assert lib().inferno_cache_evict(C.byref(_evict(batch=0)), None, 0, None) == 0


def test_struct_layouts_match_the_c_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "inferno_b200.h"', 'int main(void) {']
    structs = (InfernoRope, InfernoAttention, InfernoEvict)
    for s in structs:
        lines.append(f'printf("%zu\\n", sizeof({s.__name__}));')
        lines += [f'printf("%zu\\n", offsetof({s.__name__}, {f}));' for f, _ in s._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run([cc, "-I", str(HEADER.parent), str(src), "-o", str(tmp_path / "layout")], check=True)
    got = list(map(int, subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True).stdout.split()))
    want = []
    for s in structs:
        want += [C.sizeof(s)] + [getattr(s, f).offset for f, _ in s._fields_]
    assert got == want
