"""A call on host arrays reports its own launches' failures, whatever launches on device pointers have recorded and nobody has collected
yet, and leaves those for the next synchronize."""
import numpy as np
import pytest

from accera_b200 import runtime as rt

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def _leave_a_bad_id():
    out = torch.empty(3, 8, device="cuda")
    rt.embedding(torch.ones(4, 8, device="cuda"), torch.tensor([4, -1, 9], device="cuda"), out)


def test_token_ids():
    rt.synchronize()
    table, out = np.ones((4, 8), np.float32), np.zeros((2, 8), np.float32)
    _leave_a_bad_id()
    rt.embedding(table, np.array([0, 3]), out)                       # good ids: not this call's failure
    with pytest.raises(rt.AccbError, match=r"embedding: 1 token id"):
        rt.embedding(table, np.array([0, 7]), out)
    with pytest.raises(rt.AccbError, match=r"embedding: 2 token id"):
        rt.embedding_grad(out, np.array([-3, 7]), table)
    rt.embedding(table, np.array([0, 3]), out)
    with pytest.raises(rt.AccbError, match=r"embedding: 3 token id"):
        rt.synchronize()
    rt.synchronize()


def test_gather_indices():
    rt.synchronize()
    data, out = np.ones((4, 8), np.float32), np.zeros((2, 1, 8), np.float32)
    got = torch.empty(3, 1, 8, device="cuda")
    rt.gather_rank2(torch.ones(4, 8, device="cuda"), torch.tensor([[4], [-9], [0]], device="cuda"), got)
    rt.gather_rank2(data, np.array([[0], [3]]), out)
    with pytest.raises(rt.AccbError, match=r"gather: 1 index"):
        rt.gather_rank2(data, np.array([[0], [7]]), out)
    with pytest.raises(rt.AccbError, match=r"gather: 2 index"):
        rt.synchronize()
    rt.synchronize()


def _fp8_call(k=256):
    a, b = np.full((20, k), 0x38, np.uint8), np.full((30, k), 0x38, np.uint8)        # ones in e4m3
    sa, sb = np.ones((20, k // 128), np.float32), np.ones((1, k // 128), np.float32)
    c = np.zeros((20, 30), np.float32)
    kinds = dict(a_kind="float8_e4m3", b_kind="float8_e4m3")

    def host():
        rt.gemm_fp8(a, b.T, c, sa, sb.T, beta=0.0, **kinds)
        return c

    dev = [torch.from_numpy(x).cuda() for x in (a, b, c, sa, sb)]
    f8 = [x.view(torch.float8_e4m3fn) for x in dev[:2]]
    return host, lambda: rt.gemm_fp8(f8[0], f8[1].t(), dev[2], dev[3], dev[4].t(), beta=0.0)


def _bf16_call(k=256):
    a, b = np.full((200, k), 0x3F80, np.uint16), np.full((k, 256), 0x3F80, np.uint16)
    c = np.zeros((200, 256), np.float32)

    def host():
        rt.gemm(a, b, c, beta=0.0, kind="bfloat16", compute="tensor")
        return c

    dev = [torch.ones(200, k, device="cuda").to(torch.bfloat16), torch.ones(k, 256, device="cuda").to(torch.bfloat16), torch.zeros(200, 256, device="cuda")]
    return host, lambda: rt.gemm(*dev, beta=0.0, compute="tensor")


@pytest.mark.parametrize("make", [_fp8_call, _bf16_call])
def test_waits_that_run_out(make):
    rt.synchronize()
    host, on_device = make()
    drop = {"gemm.test_drop_commit": 1, "gemm.wait_limit_us": 2000}
    with rt.options(**drop):
        on_device()
    assert (host() == 256).all()                                     # not this call's failure
    with rt.options(**drop):
        with pytest.raises(rt.AccbError) as e:
            host()
        assert e.value.code == rt.ERR_TIMEOUT
    assert (host() == 256).all()
    with pytest.raises(rt.AccbError) as e:
        rt.synchronize()
    assert e.value.code == rt.ERR_TIMEOUT
    rt.synchronize()
