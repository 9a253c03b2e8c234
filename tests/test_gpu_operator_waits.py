"""Waits of the norms' and the 8-bit product's kernels that run out, without faulting or hanging the GPU.

st_check_device_wait runs the norms' ring of rows with one row that comes and
one that never does (kind 16), and a scaling warp of the 8-bit product that
has begun to read its accumulator and whose scales never come (kinds 17 and
18).  Each gives up after its limit, waits for what it has under way, records
its code and returns; the operators work on as before."""
import ctypes

import pytest
import torch

import sptiles_b200 as st
from sptiles_b200 import _native as N

DEV = "cuda:0"
CODES = {16: 0x201, 17: 0x103, 18: 0x103}


def check_wait(ctx, kind, limit_us, flags):
    ex = N.StExec(None, 0, flags, 10000, None, 0)
    return N.lib().st_check_device_wait(ctx, kind, limit_us, ctypes.byref(ex))


def step():
    g = torch.Generator(device=DEV).manual_seed(1)
    x, r, w = (torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16) for s in [(700, 1024), (700, 1024), (1024,)])
    q, s = st.quantize_fp8(torch.randn(300, 1024, generator=g, device=DEV))
    f = st.residual_norm(x, r, w, None, w, quantize=True)
    return [f.residual, f.scale, st.matmul_fp8(f.normed, q.t(), f.scale, s.t())]


def test_kinds_outside_the_range_are_refused():
    for kind in (15, 19):
        assert check_wait(None, kind, 1000, 0) == N.ST_ERR_INVALID_ARGUMENT
        assert "st_check_device_wait: kind" in N.last_error()
    assert check_wait(None, 16, 0, 0) == N.ST_ERR_INVALID_ARGUMENT
    assert "limit_us" in N.last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(CODES))
def test_wait_that_runs_out_is_reported_and_the_operators_work_on(kind):
    want = step()
    assert check_wait(st.context(0), kind, 2000, N.ST_EXEC_SYNC) == N.ST_ERR_DEVICE_ABORT
    assert f"(code {CODES[kind]})" in N.last_error()
    st.sync(0)  # the report cleared the word
    assert check_wait(st.context(0), kind, 1000, 0) == N.ST_OK  # queued, not waited for
    with pytest.raises(st.DeviceAbort, match=f"code {CODES[kind]}"):
        st.sync(0)
    assert all(torch.equal(a, b) for a, b in zip(want, step()))
