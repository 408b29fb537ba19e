"""What the token table and 8-bit floating point entry points refuse, checked without a GPU."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

from accera_b200 import runtime as rt

torch = pytest.importorskip("torch")


def _f8(*shape, kind=None):
    return torch.zeros(*shape).to(kind or torch.float8_e4m3fn)


def _c(fn, *args):
    lib = rt.lib()
    rc = getattr(lib, fn)(*args)
    return rc, lib.accb_last_error().decode()


def test_embedding_arguments():
    t, ids, out = torch.zeros(9, 8), torch.zeros(3, dtype=torch.int64), torch.zeros(3, 8)
    bad = [
        ((t[0], ids, out), ValueError, "rank 2"), ((t, ids, out[:2]), ValueError, "shape mismatch"), ((t, ids.float(), out), TypeError, "ids"),
        ((t.int(), ids, out), TypeError, "table"), ((t, ids, out.double()), TypeError, "float64"), ((torch.zeros(8, 9).t(), ids, out), ValueError, "contiguous"),
        ((t, torch.zeros(6, dtype=torch.int64)[::2], out), ValueError, "ids must be contiguous"), ((t, ids, torch.zeros(1, 8).expand(3, 8)), ValueError, "overlap"),
        ((t, torch.zeros(2, 2, dtype=torch.int64), torch.zeros(2, 3, 8)[:, :2]), ValueError, "evenly spaced"), ((t, [1, 2, 3], out), TypeError, "numpy array or a torch tensor"),
    ]
    for args, kind, text in bad:
        with pytest.raises(kind, match=text):
            rt.embedding(*args)
        with pytest.raises(kind):
            rt.embedding_grad(args[2], args[1], args[0])
    with pytest.raises(ValueError, match="padding_id"):
        rt.embedding_grad(out, ids, t, padding_id=-1)
    with pytest.raises(TypeError, match="not bfloat16"):
        rt.embedding(t, ids, out, table_kind="bfloat16")


def test_packed_descriptors_have_the_structures_layout():
    for pack, kind, values in [(rt._pack_embedding, rt.EmbeddingDesc, (1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11.0, 12.0)),
                               (rt._pack_quantize, rt.QuantizeFp8Desc, (1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11)),
                               (rt._pack_gemm, rt.GemmDesc, (1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14.0, 15.0, 16, 17)),
                               (rt._pack_scales, rt.Fp8Scales, (1, 2, 3, 4, 5, 6))]:
        d = kind.from_buffer_copy(pack(*values))
        flat = []
        for name, _ in kind._fields_:
            v = getattr(d, name)
            flat += list(v) if isinstance(v, ctypes.Array) else [v]
        assert tuple(flat) == values and len(pack(*values)) == ctypes.sizeof(kind)


def test_embedding_descriptor():
    p = ctypes.c_void_p(64)
    good = dict(tokens=3, vocab=9, dim=8, table_type=rt.F32, rows_type=rt.BF16, id_bytes=8, reserved=0, table_stride=8, rows_stride=8, padding_id=-1, scale=1.0, beta=0.0)
    for change, text in [(dict(tokens=-1), "negative"), (dict(vocab=1 << 31), "too large"), (dict(tokens=(1 << 30) + 1), "too large"), (dict(dim=(1 << 20) + 1), "2^20"), (dict(table_type=rt.S32), "fp32, fp16 or bf16"),
                         (dict(rows_type=rt.E4M3), "fp32, fp16 or bf16"), (dict(id_bytes=2), "id_bytes"), (dict(reserved=1), "reserved"), (dict(table_stride=7), "at least dim"),
                         (dict(rows_stride=0), "at least dim")]:
        d = rt.EmbeddingDesc(**{**good, **change})
        for fn in ("accb_embedding", "accb_embedding_grad"):
            rc, msg = _c(fn, ctypes.byref(d), p, p, p)
            assert rc == rt.ERR_ARG and text in msg and msg.startswith(fn + ":"), (change, msg)
    d = rt.EmbeddingDesc(**good)
    assert _c("accb_embedding", None, p, p, p)[0] == rt.ERR_ARG
    assert _c("accb_embedding", ctypes.byref(d), None, p, p)[0] == rt.ERR_ARG
    assert _c("accb_embedding_grad", ctypes.byref(d), p, None, p)[0] == rt.ERR_ARG
    for empty in (dict(tokens=0), dict(dim=0)):                            # nothing to do: no device needed
        assert _c("accb_embedding", ctypes.byref(rt.EmbeddingDesc(**{**good, **empty})), None, None, None)[0] == 0
    assert _c("accb_embedding_grad", ctypes.byref(rt.EmbeddingDesc(**{**good, "vocab": 0})), None, None, None)[0] == 0


def test_quantize_arguments():
    x, q, s = torch.zeros(200, 300), _f8(200, 300), torch.zeros(200, 3)
    bad = [
        ((x[0], q, s), ValueError, "shape"), ((x, q[:100], s), ValueError, "shape"), ((x, q, s[:, :2]), ValueError, "columns"), ((x, q, s[:3]), ValueError, "3 scales for 200"),
        ((x, q.t().contiguous().t(), s), ValueError, "rows must be contiguous"), ((x, x, s), TypeError, "q"), ((x, q, s.half()), TypeError, "scales"),
        ((x.double(), q, s), TypeError, "float64"), ((x[:1].expand(200, 300), q, s), ValueError, "positive"), ((x.numpy(), np.zeros((200, 300), np.uint8), s.numpy()), TypeError, "q"),
    ]
    for args, kind, text in bad:
        with pytest.raises(kind, match=text):
            rt.quantize_fp8(*args)
    p = ctypes.c_void_p(64)
    for change, text in [(dict(rows=-1), "negative"), (dict(cols=1 << 31), "too large"), (dict(x_type=rt.S8), "fp32, fp16 or bf16"), (dict(q_type=rt.F16), "E4M3"),
                         (dict(block_rows=64), "1 or 128"), (dict(q_stride=299), "q_stride"), (dict(reserved=3), "reserved")]:
        d = rt.QuantizeFp8Desc(**{**dict(rows=200, cols=300, x_type=rt.F32, q_type=rt.E4M3, block_rows=1, reserved=0, q_stride=300), **change})
        d.x_stride[:], d.scale_stride[:] = (300, 1), (3, 1)
        rc, msg = _c("accb_quantize_fp8", ctypes.byref(d), p, p, p)
        assert rc == rt.ERR_ARG and text in msg, (change, msg)


def test_gemm_arguments():
    A, B, C = _f8(40, 300), _f8(300, 260), torch.zeros(40, 260)
    sa, sb = torch.zeros(40, 3), torch.zeros(3, 3)
    bad = [
        ((A, B[:200], C, sa, sb), ValueError, "shape mismatch"), ((A, B, C[:, :5], sa, sb), ValueError, "shape mismatch"), ((A, B, C, sa[:, :2], sb), ValueError, "blocks of K"),
        ((A, B, C, sa[:7], sb), ValueError, "a_scales"), ((A, B, C, sa, sb[:, :2]), ValueError, "b_scales"), ((C, B, C, sa, sb), TypeError, "A"),
        ((A, B, _f8(40, 260), sa, sb), TypeError, "C"), ((A, B, C, sa.double(), sb), TypeError, "a_scales"), ((A[0], B, C, sa, sb), ValueError, "rank 2"),
        ((A[:1].expand(40, 300), B, C, sa, sb), ValueError, "positive"),
    ]
    for args, kind, text in bad:
        with pytest.raises(kind, match=text):
            rt.gemm_fp8(*args)
    with pytest.raises(ValueError, match="bias"):
        rt.gemm_fp8(A, B, C, sa, sb, bias=torch.zeros(259))
    with pytest.raises(rt.AccbError, match="compute"):
        rt.gemm_fp8(A, B, C, sa, sb, compute="tensor_2sm")
    with pytest.raises(TypeError):                                         # the other GEMMs take no 8-bit floating point operands
        rt.gemm(A, B, C)
    p = ctypes.c_void_p(64)
    s = rt.Fp8Scales(1, 128)
    s.a_stride[:], s.b_stride[:] = (3, 1), (3, 1)
    for change, text in [(dict(m=-1), "negative"), (dict(k=1 << 31), "too large"), (dict(a_type=rt.S8), "E4M3"), (dict(c_type=rt.S32), "fp32, fp16 or bf16"),
                         (dict(epilogue=7), "epilogue"), (dict(max_ctas=-1), "max_ctas"), (dict(compute=3), "compute")]:
        d = rt.GemmDesc(**{**dict(m=40, n=260, k=300, a_type=rt.E4M3, b_type=rt.E5M2, c_type=rt.F32, compute=0), **change})
        d.a_stride[:], d.b_stride[:], d.c_stride[:] = (300, 1), (260, 1), (260, 1)
        rc, msg = _c("accb_gemm_fp8", ctypes.byref(d), ctypes.byref(s), p, p, p, p, p, None)
        assert rc == rt.ERR_ARG and text in msg, (change, msg)
    d = rt.GemmDesc(40, 260, 300, rt.E4M3, rt.E4M3, rt.F32, 0)
    d.a_stride[:], d.b_stride[:], d.c_stride[:] = (300, 1), (260, 1), (260, 1)
    for blocks in ((2, 128), (1, 64)):
        t = rt.Fp8Scales(*blocks)
        t.a_stride[:], t.b_stride[:] = (3, 1), (3, 1)
        assert _c("accb_gemm_fp8", ctypes.byref(d), ctypes.byref(t), p, p, p, p, p, None)[0] == rt.ERR_ARG
    assert _c("accb_gemm_fp8", ctypes.byref(d), ctypes.byref(s), None, p, p, p, p, None)[0] == rt.ERR_ARG
    d.m = 0
    assert _c("accb_gemm_fp8", ctypes.byref(d), ctypes.byref(s), None, None, None, None, None, None)[0] == 0


def test_options_of_the_8_bit_gemm():
    for name, value in (("gemm_fp8.kernel", 3), ("gemm_fp8.slices", 3), ("gemm_fp8.slices", -1)):
        with pytest.raises(rt.AccbError, match=name):
            rt.set_option(name, value)
    with rt.options(**{"gemm_fp8.kernel": 2, "gemm_fp8.slices": 8}):
        pass


def test_valid_host_calls_need_a_gpu():
    if rt.device_count():
        pytest.skip("a GPU is there")
    with pytest.raises(rt.AccbError) as e:
        rt.embedding(np.zeros((4, 8), np.float32), np.zeros((2, 1), np.int32), np.zeros((2, 1, 8), np.float32))
    assert e.value.code == rt.ERR_CUDA
    with pytest.raises(rt.AccbError) as e:
        rt.quantize_fp8(np.zeros((4, 8), np.uint16), np.zeros((4, 8), np.uint8), np.zeros((4, 1), np.float32), kind="bfloat16", q_kind="float8_e5m2")
    assert e.value.code == rt.ERR_CUDA


def test_bad_token_ids_are_attributed_to_the_launch_that_had_them():
    ALL, GATHER, EMBED = 0, 2, 3
    words = [0, 0, 0, 0, 0, 0, 4, 12]
    code, msg = rt.decode_status(words, EMBED, 12)
    assert code == rt.ERR_INDEX and "4 token id(s)" in msg
    assert rt.decode_status(words, EMBED, 13) == (0, "") and rt.decode_status(words, GATHER, 12) == (0, "")
    assert rt.decode_status(words, ALL)[0] == rt.ERR_INDEX


def test_a_wait_for_scales_is_named():
    code, msg = rt.decode_status([0, (6 << 24) | 5, 8, 77, 2, 0, 0, 0])
    assert code == rt.ERR_TIMEOUT and "epilogue waiting for scales, block 5, step 8" in msg
    with rt.options(**{"gemm_fp8.test_drop_scales": 1}):
        pass


_SUBCLASS = """
import torch
from accera_b200 import runtime as rt

class Marked(torch.Tensor):
    pass

make = lambda *shape: torch.zeros(*shape).as_subclass(Marked)
{first}
"""


@pytest.mark.parametrize("first,text", [
    ("rt.embedding(make(9), make(3), make(3, 8))", "ids: unsupported tensor dtype"),
    ("rt.quantize_fp8(make(4, 8), make(4, 8), make(4, 1))", "q: unsupported tensor dtype"),
    ("rt.gemm_fp8(make(4, 8), make(8, 4), make(4, 4), make(4, 1), make(1, 1))", "A: unsupported tensor dtype"),
    ("rt.gemm(make(4, 8), make(7, 4), make(4, 4))", "shape mismatch"),
])
def test_a_tensor_subclass_may_be_the_first_argument_of_a_process(first, text):
    r = subprocess.run([sys.executable, "-c", _SUBCLASS.format(first=first)], capture_output=True, text=True, timeout=300,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode != 0 and text in r.stderr, r.stderr


def test_results_are_not_written_to_read_only_arrays():
    f, q = lambda *shape: np.zeros(shape, np.float32), lambda *shape: np.zeros(shape, np.uint8)
    ids = np.zeros(3, np.int64)

    def fixed(x):
        x.flags.writeable = False
        return x

    kinds = dict(a_kind="float8_e4m3", b_kind="float8_e4m3")
    for call, name in [(lambda: rt.embedding(f(9, 8), ids, fixed(f(3, 8))), "rows"), (lambda: rt.embedding_grad(f(3, 8), ids, fixed(f(9, 8))), "table"),
                       (lambda: rt.quantize_fp8(f(4, 8), fixed(q(4, 8)), f(4, 1), q_kind="float8_e4m3"), "q"),
                       (lambda: rt.quantize_fp8(f(4, 8), q(4, 8), fixed(f(4, 1)), q_kind="float8_e4m3"), "scales"),
                       (lambda: rt.gemm_fp8(q(4, 8), q(8, 6), fixed(f(4, 6)), f(4, 1), f(1, 1), **kinds), "C")]:
        with pytest.raises(ValueError, match=f"{name}: the array is read-only"):
            call()
    if not rt.device_count():                                              # what is only read may be read-only
        with pytest.raises(rt.AccbError):
            rt.embedding(fixed(f(9, 8)), fixed(ids.copy()), f(3, 8))
