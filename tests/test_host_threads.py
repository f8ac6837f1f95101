"""C entries called from two host threads at once, with sizes that want different amounts of
shared memory (ctypes lets both run): every call is launched, and results are those of
calls on their own."""
import ctypes as C
import threading

import pytest
import torch

from bozo_b200 import _capi

gpu = pytest.mark.gpu
BF16 = torch.bfloat16


def view(x):
    """``x [B, T, H, HD]`` as the ABI's strided view."""
    t = _capi.Tensor4()
    t.ptr, t.dtype = x.data_ptr(), {torch.float32: _capi.DT_F32, BF16: _capi.DT_BF16}[x.dtype]
    t.stride[:] = x.stride()
    return t


def decode(capacity, HD):
    """A global decode step over a ring of `capacity` keys (τ of them in shared memory)."""
    a = _capi.DecodeArgs()
    q, k, v = (torch.randn(1, 1, 2, HD, device="cuda", dtype=BF16) for _ in range(3))
    kc, vc = (torch.randn(1, capacity, 2, HD, device="cuda", dtype=BF16) for _ in "kv")
    pos = torch.full((1,), 700, dtype=torch.int32, device="cuda")
    out = torch.empty(1, 2, HD, device="cuda", dtype=BF16)
    a.B, a.H, a.HD, a.mode, a.normalize, a.capacity, a.scale = 1, 2, HD, _capi.MODE_GLOBAL, _capi.NORM_MASS, capacity, 8.0
    a.q, a.k, a.v, a.pos = view(q), view(k), view(v), pos.data_ptr()
    a.k_cache, a.v_cache, a.out = kc.data_ptr(), vc.data_ptr(), out.data_ptr()
    a.k_cache_dtype = a.v_cache_dtype = a.out_dtype = _capi.DT_BF16
    return _capi.lib().bozo_tension_decode, a, out, (q, k, v, kc, vc, pos)


def forward(window, T):
    """A local forward on the tensor cores."""
    a = _capi.FwdArgs()
    q, k, v = (torch.randn(1, T, 2, 64, device="cuda", dtype=BF16) for _ in range(3))
    out = torch.empty(1, T, 2, 64, device="cuda", dtype=BF16)
    a.B, a.T, a.H, a.HD, a.mode, a.window, a.normalize, a.scale = 1, T, 2, 64, _capi.MODE_LOCAL, window, _capi.NORM_MASS, 8.0
    a.q, a.k, a.v, a.out, a.out_dtype, a.path = view(q), view(k), view(v), out.data_ptr(), _capi.DT_BF16, _capi.PATH_TCGEN05
    return _capi.lib().bozo_tension_fwd, a, out, (q, k, v)


def projected_norm(width, rows):
    """The projection with the add and the norm in its epilogue."""
    a = _capi.WoAddRMSNormArgs()
    msg, x = (torch.randn(rows, width, device="cuda", dtype=BF16) for _ in range(2))
    wo = torch.randn(width, width, device="cuda", dtype=BF16) * width ** -0.5
    scale, out = torch.ones(width, device="cuda", dtype=BF16), torch.empty(rows, width, device="cuda", dtype=BF16)
    a.rows, a.width, a.eps, a.x_dtype = rows, width, 1e-6, _capi.DT_BF16
    a.msg, a.wo, a.x, a.scale, a.out = (t.data_ptr() for t in (msg, wo, x, scale, out))
    return _capi.lib().bozo_wo_add_rmsnorm_fwd, a, out, (msg, wo, x, scale)


@gpu
@pytest.mark.parametrize("calls", [
    lambda: (decode(14000, 64), decode(30000, 64)), lambda: (decode(16000, 48), decode(40000, 48)),
    lambda: (forward(16, 300), forward(128, 200)), lambda: (projected_norm(64, 200), projected_norm(768, 130))],
    ids=["decode", "decode, any width", "forward", "projection and norm"])
def test_two_threads_with_different_sizes(calls):
    torch.manual_seed(0)
    pair = calls()
    want = []
    for call, a, out, _ in pair:
        assert call(C.byref(a), torch.cuda.current_stream().cuda_stream) == 0
        want.append(out.clone())
        out.zero_()
    status = [set(), set()]

    def run(i):
        call, a, _, _ = pair[i]
        stream = torch.cuda.Stream()
        for _ in range(4000):
            status[i].add(call(C.byref(a), stream.cuda_stream))
        stream.synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert status == [{0}, {0}]
    for (_, _, out, _), ref in zip(pair, want):
        assert torch.equal(out, ref) and float(out.float().abs().sum()) > 0
