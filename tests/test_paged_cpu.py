"""The paged-cache and scoring entry points without a GPU: the C ABI's argument
checks, the wrappers' refusals, the op's report and the custom ops' shapes."""

from __future__ import annotations

import ctypes

import pytest
import torch

from repercep_runtime_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    from repercep_runtime_b200 import build

    build.build()  # no-op when up to date; nvcc cross-compiles without a GPU
    return _lib.load()


DUMMY = 1 << 20  # an aligned address that no check reads through


def kv(**changes):
    fields = dict(k=DUMMY, v=DUMMY, k_scales=DUMMY, v_scales=DUMMY, strides=(2 * 16 * 128, 16 * 128, 128),
                  dtype=_lib.RP_KV_BF16, num_pages=4, heads=2, page_size=16, head_dim=128)
    fields.update(changes)
    return ctypes.byref(_lib.PagedKVStruct(**{k: (ctypes.c_int64 * 3)(*v) if k == "strides" else v for k, v in fields.items()}))


def append(lib, pool=None, **changes):
    a = dict(k=DUMMY, v=DUMMY, strides=(256, 128, 256, 128), dtype=0, tokens=2, starts=None, table=DUMMY, stride=3,
             pages=3, lengths=DUMMY, B=2, weights=None, w_strides=None, cols=0, out=DUMMY)
    a.update(changes)
    return lib.rp_paged_append(pool or kv(), a["k"], a["v"], _lib.i64_array(a["strides"]), a["dtype"], a["tokens"],
                               a["starts"], a["table"], a["stride"], a["pages"], a["lengths"], a["B"], a["weights"],
                               a["w_strides"], a["cols"], a["out"], None)


def decode(lib, pool=None, **changes):
    a = dict(q=DUMMY, q_strides=(512, 128), dtype=0, B=2, Hq=4, table=DUMMY, stride=3, pages=3, lengths=DUMMY,
             scale=0.0, out=DUMMY, o_strides=(512, 128), weights=None, w_strides=None, cols=0, ws=DUMMY, bytes=1 << 40)
    a.update(changes)
    return lib.rp_paged_decode(pool or kv(), a["q"], _lib.i64_array(a["q_strides"]), a["dtype"], a["B"], a["Hq"],
                               a["table"], a["stride"], a["pages"], a["lengths"], a["scale"], a["out"],
                               _lib.i64_array(a["o_strides"]), None, a["weights"], a["w_strides"], a["cols"], a["ws"],
                               a["bytes"], None)


def evict(lib, pool=None, **changes):
    a = dict(table=DUMMY, stride=3, pages=3, lengths=DUMMY, B=2, weights=DUMMY, w_strides=(96, 48), cols=48,
             out_table=DUMMY, out_stride=2, out_pages=2, budget=20, recent=4, kept=DUMMY, out=DUMMY, w_out=DUMMY)
    a.update(changes)
    return lib.rp_paged_evict(pool or kv(), a["table"], a["stride"], a["pages"], a["lengths"], a["B"], a["weights"],
                              _lib.i64_array(a["w_strides"]), a["cols"], a["out_table"], a["out_stride"],
                              a["out_pages"], a["budget"], a["recent"], a["kept"], a["out"], a["w_out"], None)


def scores(lib, **changes):
    a = dict(logits=DUMMY, stride=100, dtype=0, rows=2, vocab=100, tokens=DUMMY, top=3, lp=DUMMY, en=DUMMY, tl=DUMMY, ti=DUMMY)
    a.update(changes)
    return lib.rp_token_logprobs(a["logits"], a["stride"], a["dtype"], a["rows"], a["vocab"], a["tokens"], a["top"],
                                 a["lp"], a["en"], a["tl"], a["ti"], None)


POOLS = [
    (dict(dtype=3), -2, b"dtype"),
    (dict(head_dim=96), -2, b"head_dim"),
    (dict(num_pages=0), -1, b"positive"),
    (dict(heads=70000), -2, b"heads"),
    (dict(k=None), -1, b"null"),
    (dict(v=DUMMY + 8), -3, b"16-byte"),
    (dict(dtype=2, v_scales=None), -1, b"scales"),
    (dict(strides=(4096, 2048, 100)), -3, b"stride"),
    (dict(strides=(-4096, 2048, 128)), -3, b"stride"),
    (dict(dtype=2, strides=(4096, 2048, 136)), -3, b"stride"),
]


@pytest.mark.parametrize("call", [append, decode, evict])
@pytest.mark.parametrize("changes, rc, words", POOLS)
def test_pools_are_checked(lib, call, changes, rc, words):
    assert call(lib, kv(**changes)) == rc and words in lib.rp_last_error()


@pytest.mark.parametrize("call, changes, rc, words", [
    (append, dict(B=-1), -1, b"negative"),
    (append, dict(B=70000), -2, b"sequences"),
    (append, dict(lengths=None), -1, b"null"),
    (append, dict(stride=2), -1, b"page_table"),
    (append, dict(pages=1 << 28, stride=1 << 28), -2, b"2^31"),
    (append, dict(dtype=2), -2, b"dtype"),
    (append, dict(dtype=1), -1, b"share a dtype"),
    (append, dict(tokens=3), -1, b"without starts"),
    (append, dict(tokens=-1), -1, b"negative"),
    (append, dict(tokens=1 << 30, starts=DUMMY), -2, b"2^31"),
    (append, dict(strides=(256, 128, 256, 130)), -3, b"strides"),
    (append, dict(k=DUMMY + 2), -3, b"aligned"),
    (append, dict(out=None), -1, b"lengths_out"),
    (append, dict(weights=DUMMY, w_strides=_lib.i64_array((96, 48)), cols=47), -1, b"positions"),
    (append, dict(weights=DUMMY, cols=48), -1, b"strides"),
    (decode, dict(Hq=3), -1, b"multiple"),
    (decode, dict(Hq=0), -1, b"multiple"),
    (decode, dict(dtype=1), -1, b"share a dtype"),
    (decode, dict(dtype=2), -2, b"dtype"),
    (decode, dict(scale=float("nan")), -1, b"finite"),
    (decode, dict(q=None), -1, b"null"),
    (decode, dict(q_strides=(512, 100)), -3, b"16-byte"),
    (decode, dict(ws=None), -6, b"workspace"),
    (decode, dict(bytes=16), -6, b"workspace"),
    (evict, dict(budget=0), -1, b"budget"),
    (evict, dict(recent=21), -1, b"recent"),
    (evict, dict(budget=33), -1, b"out_table"),
    (evict, dict(weights=None), -1, b"weights"),
    (evict, dict(kept=None), -1, b"null"),
    (scores, dict(dtype=3), -2, b"dtype"),
    (scores, dict(vocab=0), -1, b"vocab"),
    (scores, dict(top=65), -1, b"top"),
    (scores, dict(vocab=2), -1, b"top"),
    (scores, dict(tokens=None), -1, b"null"),
    (scores, dict(dtype=2, logits=DUMMY + 2), -3, b"aligned"),
    (scores, dict(stride=-100), -1, b"stride"),
])
def test_arguments_are_checked(lib, call, changes, rc, words):
    assert call(lib, **changes) == rc and words in lib.rp_last_error(), lib.rp_last_error()


def test_pools_of_odd_strides_and_terabytes_are_refused(lib):
    far = kv(num_pages=1 << 30, strides=((1 << 12) + 8, 2048, 128))
    assert decode(lib, far) == -2 and b"strides" in lib.rp_last_error()


def test_nothing_to_do_is_no_error(lib):
    assert append(lib, B=0, tokens=0) == 0
    assert decode(lib, B=0) == 0
    assert evict(lib, B=0) == 0
    assert scores(lib, rows=0) == 0


def test_workspace_bytes_grow_with_weights_only(lib):
    n, w, one = ctypes.c_size_t(), ctypes.c_size_t(), ctypes.c_size_t()
    assert lib.rp_paged_decode_workspace_bytes(kv(), 8, 4, 100, 0, ctypes.byref(n)) == 0
    assert lib.rp_paged_decode_workspace_bytes(kv(), 1, 4, 1, 0, ctypes.byref(one)) == 0
    assert lib.rp_paged_decode_workspace_bytes(kv(), 8, 4, 100, 1, ctypes.byref(w)) == 0
    assert n.value == one.value > 0
    assert w.value - n.value >= 8 * 4 * 1600 * 4
    assert lib.rp_paged_decode_workspace_bytes(kv(head_dim=5), 8, 4, 100, 1, ctypes.byref(w)) == -2


def test_wrappers_refuse_cpu_tensors():
    from repercep_runtime_b200 import paged, scoring

    with pytest.raises(ValueError, match="CUDA"):
        paged.alloc(2, 2, 16, 64, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        scoring.token_logprobs(torch.zeros((2, 8)), torch.zeros(2, dtype=torch.int64))


def test_op_reports_itself():
    from repercep_runtime_b200.attention import PagedDecode

    op = PagedDecode()
    assert PagedDecode.name == "b200-paged-decode"
    if not torch.cuda.is_available():
        assert not op.available and not op.supports(32, 8, 128)
        with pytest.raises(RuntimeError, match="not available"):
            op(None, None, None, None)


def test_custom_ops_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from repercep_runtime_b200 import ops  # noqa: F401

    with FakeTensorMode():
        q, k = torch.empty((3, 8, 64), dtype=torch.bfloat16), torch.empty((5, 2, 16, 64), dtype=torch.bfloat16)
        table, n = torch.empty((3, 2), dtype=torch.int32), torch.empty(3, dtype=torch.int32)
        out, lse = torch.ops.repercep_b200.paged_decode(q, k, k, table, n)
        assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (3, 8) and lse.dtype == torch.float32
        got = torch.ops.repercep_b200.token_logprobs(torch.empty((4, 100)), torch.empty(4, dtype=torch.int64), 6)
        assert [tuple(t.shape) for t in got] == [(4,), (4,), (4, 6), (4, 6)] and got[3].dtype == torch.int64
