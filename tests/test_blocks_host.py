"""What the launchers of layer norm, the gated recurrence and the experts refuse before
anything is launched, and the sizes of their workspaces (host logic, no GPU)."""
import ctypes

import pytest

from pico_amd import kernels as K
from pico_amd._lib import hip_lib

PTR = ctypes.c_void_p(256)  # never read: every call here is refused on its arguments
EINVAL = -1


@pytest.fixture(scope="module")
def L():
    return hip_lib()


def _refused(L, status, word):
    assert status == EINVAL
    assert word in L.pk_last_error().decode()


def test_layernorm(L):
    fwd, bwd = L.pk_layernorm_fwd_f32, L.pk_layernorm_bwd_f32
    for R, C in ((-1, 4), (4, 0), (1 << 31, 4)):
        _refused(L, fwd(R, C, 1e-5, PTR, PTR, PTR, PTR, PTR, PTR, None), "R")
        _refused(L, bwd(R, C, PTR, PTR, PTR, PTR, PTR, None, PTR, PTR, PTR, 0, PTR, 1 << 40, None), "R")
    for k in (0, 1, 3):
        a = [PTR] * 6
        a[k] = None
        _refused(L, fwd(4, 4, 1e-5, *a, None), "NULL")
    for k in range(5):
        a = [PTR] * 5
        a[k] = None
        _refused(L, bwd(4, 4, *a, None, PTR, PTR, PTR, 0, PTR, 1 << 40, None), "NULL")
    need = K.layernorm_bwd_workspace(1000, 96)
    assert need >= 2 * 96 * 4
    for ws, size in ((None, need), (PTR, need - 1)):
        _refused(L, bwd(1000, 96, PTR, PTR, PTR, PTR, PTR, None, PTR, PTR, None, 0, ws, size, None), "workspace")
    assert K.layernorm_bwd_workspace(0, 4) == 0
    # no larger than 1/16 of x beyond a few hundred rows
    assert K.layernorm_bwd_workspace(8192, 4096) <= 8192 * 4096 * 4 // 8


def test_gated_scan(L):
    fwd, bwd = L.pk_gated_scan_fwd_f32, L.pk_gated_scan_bwd_f32
    for B, T, C in ((-1, 1, 1), (1, -1, 1), (1, 1, -1), (1 << 20, 1 << 20, 1), (1 << 31, 1, 1)):
        _refused(L, fwd(B, T, C, PTR, 1 << 40, PTR, 1 << 40, None, PTR, PTR, 1 << 40, None), "")
        _refused(L, bwd(B, T, C, PTR, 1 << 40, PTR, 1 << 40, None, PTR, PTR, PTR, 1 << 40, PTR, 1 << 40, None, 0,
                        PTR, 1 << 40, None), "")
    for f, ldf, x, ldx, h in ((None, 8, PTR, 8, PTR), (PTR, 8, None, 8, PTR), (PTR, 7, PTR, 8, PTR),
                              (PTR, 8, PTR, 7, PTR), (PTR, 8, PTR, 8, None)):
        _refused(L, fwd(2, 3, 8, f, ldf, x, ldx, None, h, PTR, 1 << 40, None), "pk_gated_scan")
        _refused(L, bwd(2, 3, 8, f, ldf, x, ldx, None, h, PTR, PTR, 8, PTR, 8, None, 0, PTR, 1 << 40, None),
                 "pk_gated_scan")
    for dh, lddf, lddx in ((None, 8, 8), (PTR, 7, 8), (PTR, 8, 7)):
        _refused(L, bwd(2, 3, 8, PTR, 8, PTR, 8, None, PTR, dh, PTR, lddf, PTR, lddx, None, 0, PTR, 1 << 40, None),
                 "pk_gated_scan")
    for shape in ((1, 1, 1), (64, 1, 768), (0, 5, 5), (5, 0, 5), (5, 5, 0)):
        assert K.gated_scan_workspace(*shape) == 0
    need = K.gated_scan_workspace(1, 65536, 512)
    # a small part of what the recurrence itself reads
    assert need <= 65536 * 512 * 8 // 32
    if need:
        for ws, size in ((None, need), (PTR, need - 1)):
            _refused(L, fwd(1, 65536, 512, PTR, 512, PTR, 512, None, PTR, ws, size, None), "workspace")
            _refused(L, bwd(1, 65536, 512, PTR, 512, PTR, 512, None, PTR, PTR, PTR, 512, PTR, 512, None, 0, ws, size,
                            None), "workspace")


def test_router_and_plan(L):
    for R, E, k in ((-1, 4, 1), (4, 0, 1), (4, 1025, 1), (4, 4, 0), (4, 4, 5), (4, 100, 65), (1 << 30, 64, 2)):
        _refused(L, L.pk_route_topk_f32(R, E, k, PTR, 2000, PTR, PTR, None), "pk_route_topk")
        _refused(L, L.pk_route_topk_bwd_f32(R, E, k, PTR, PTR, PTR, PTR, 2000, 0, None), "pk_route_topk")
    for a in ((None, 8, PTR, PTR), (PTR, 7, PTR, PTR), (PTR, 8, None, PTR), (PTR, 8, PTR, None)):
        _refused(L, L.pk_route_topk_f32(4, 8, 2, *a, None), "NULL")
    for k in range(4):
        a = [PTR] * 4
        a[k] = None
        _refused(L, L.pk_route_topk_bwd_f32(4, 8, 2, *a, 8, 0, None), "NULL")
    _refused(L, L.pk_route_topk_bwd_f32(4, 8, 2, PTR, PTR, PTR, PTR, 7, 0, None), "stride")
    for n, E in ((-1, 4), (1 << 31, 4), (4, 0), (4, 1025)):
        _refused(L, L.pk_expert_plan(n, E, PTR, PTR, PTR, PTR, PTR, 1 << 40, None), "pk_expert_plan")
        assert K.expert_plan_workspace(n, E) == 0
    for k in range(4):
        a = [PTR] * 4
        a[k] = None
        _refused(L, L.pk_expert_plan(8, 4, *a, PTR, 1 << 40, None), "NULL")
    need = K.expert_plan_workspace(100000, 64)
    assert need > 0 and need % (65 * 4) == 0
    for ws, size in ((None, need), (PTR, need - 1)):
        _refused(L, L.pk_expert_plan(100000, 64, PTR, PTR, PTR, PTR, ws, size, None), "workspace")
    # the count a chunk is bounded, however many slots
    assert K.expert_plan_workspace((1 << 31) - 1, 64) <= 256 * 65 * 4


def test_rows(L):
    g, c, b = L.pk_expert_gather_f32, L.pk_expert_combine_f32, L.pk_expert_combine_bwd_f32
    for n, d, k, E in ((-2, 4, 2, 4), (8, 0, 2, 4), (8, 4, 0, 4), (8, 4, 65, 4), (8, 4, 3, 4), (8, 4, 2, 0),
                       (1 << 31, 4, 2, 4)):
        _refused(L, g(n, d, k, E, PTR, PTR, PTR, 8, PTR, 8, None), "pk_expert_gather")
    for a in ((None, PTR, PTR, 8, PTR, 8), (PTR, None, PTR, 8, PTR, 8), (PTR, PTR, None, 8, PTR, 8),
              (PTR, PTR, PTR, 3, PTR, 8), (PTR, PTR, PTR, 8, None, 8), (PTR, PTR, PTR, 8, PTR, 3)):
        _refused(L, g(8, 4, 2, 4, *a, None), "NULL")
    for R, d, k in ((-1, 4, 2), (4, 0, 2), (4, 4, 0), (4, 4, 65), (1 << 30, 4, 4)):
        _refused(L, c(R, d, k, PTR, PTR, PTR, 8, PTR, 8, PTR, 8, None), "pk_expert_combine")
        _refused(L, b(R, d, k, 4, PTR, PTR, PTR, PTR, 8, PTR, 8, PTR, 8, PTR, 0, None), "pk_expert_combine_bwd")
    for a in ((None, PTR, PTR, 8, PTR, 8, PTR, 8), (PTR, PTR, None, 8, PTR, 8, PTR, 8),
              (PTR, PTR, PTR, 3, PTR, 8, PTR, 8), (PTR, PTR, PTR, 8, PTR, 3, PTR, 8),
              (PTR, PTR, PTR, 8, PTR, 8, None, 8), (PTR, PTR, PTR, 8, PTR, 8, PTR, 3)):
        _refused(L, c(4, 4, 2, *a, None), "NULL")
    for a in ((None, PTR, PTR, PTR, 8, PTR, 8, PTR, 8, PTR), (PTR, None, PTR, PTR, 8, PTR, 8, PTR, 8, PTR),
              (PTR, PTR, None, PTR, 8, PTR, 8, PTR, 8, PTR), (PTR, PTR, PTR, None, 8, PTR, 8, PTR, 8, PTR),
              (PTR, PTR, PTR, PTR, 3, PTR, 8, PTR, 8, PTR), (PTR, PTR, PTR, PTR, 8, None, 8, PTR, 8, PTR),
              (PTR, PTR, PTR, PTR, 8, PTR, 3, PTR, 8, PTR), (PTR, PTR, PTR, PTR, 8, PTR, 8, PTR, 3, PTR)):
        _refused(L, b(4, 4, 2, 4, *a, 0, None), "NULL")
    _refused(L, b(4, 4, 2, 0, PTR, PTR, PTR, PTR, 8, PTR, 8, PTR, 8, PTR, 0, None), "E")


def test_products(L):
    y, w = L.pk_gemm_experts_f32, L.pk_gemm_experts_dw_f32
    ok = dict(n=8, N=12, K=4, E=2)

    def fwd(tb=b"N", X=PTR, ldx=12, W=PTR, ldw=12, sw=48, Y=PTR, ldy=12, offsets=PTR, precision=0, **kw):
        s = {**ok, **kw}
        return y(tb, s["n"], s["N"], s["K"], s["E"], offsets, X, ldx, W, ldw, sw, Y, ldy, 0, precision, None)

    def dw(X=PTR, ldx=12, dY=PTR, ldy=12, dW=PTR, ldw=12, sw=48, offsets=PTR, precision=0, ws=PTR, **kw):
        s = {**ok, **kw}
        return w(s["n"], s["K"], s["N"], s["E"], offsets, X, ldx, dY, ldy, dW, ldw, sw, 0, precision, ws, 1 << 40,
                 None)

    for bad in (dict(n=-1), dict(N=-1), dict(K=-1), dict(E=0), dict(E=1025), dict(n=(1 << 30) + 1),
                dict(offsets=None), dict(precision=-1), dict(precision=3)):
        _refused(L, fwd(**bad), "pk_gemm_experts_f32")
        _refused(L, dw(**bad), "pk_gemm_experts_dw_f32")
    for bad in (dict(tb=b"X"), dict(X=None), dict(W=None), dict(Y=None), dict(ldx=3), dict(ldw=11), dict(ldy=11),
                dict(sw=-1), dict(tb=b"T", ldw=3), dict(ldx=1 << 22), dict(tb=b"T", ldw=1 << 22),
                dict(ldw=1 << 25), dict(n=1 << 30, N=1 << 17, ldw=1 << 17, ldy=1 << 17)):
        _refused(L, fwd(**bad), "pk_gemm_experts_f32")
    for bad in (dict(X=None), dict(dY=None), dict(dW=None), dict(ldx=3), dict(ldy=11), dict(ldw=11), dict(sw=47),
                dict(ldx=1 << 25), dict(ldy=1 << 25)):
        _refused(L, dw(**bad), "pk_gemm_experts_dw_f32")


def test_more_threads_than_a_launch_has(L):
    """sizes whose launch would have 2^32 threads or more"""
    for C in ((1 << 26) + 1, 1 << 40):
        _refused(L, L.pk_layernorm_fwd_f32(1, C, 1e-5, PTR, PTR, None, PTR, None, None, None), "2^26")
        _refused(L, L.pk_layernorm_bwd_f32(1, C, PTR, PTR, PTR, PTR, PTR, None, PTR, None, None, 0, None, 0, None),
                 "2^26")
    for C, R in ((3, 1 << 26), (20000, 1 << 22)):
        _refused(L, L.pk_layernorm_fwd_f32(R, C, 1e-5, PTR, PTR, None, PTR, None, None, None), "rows")
        _refused(L, L.pk_layernorm_bwd_f32(R, C, PTR, PTR, PTR, PTR, PTR, None, PTR, None, None, 0, None, 0, None),
                 "rows")
    for B, T, C in (((1 << 31) - 1, 1, 3), (1 << 24, 41, 4), (1 << 28, 2, 64)):
        _refused(L, L.pk_gated_scan_fwd_f32(B, T, C, PTR, 64, PTR, 64, None, PTR, PTR, 1 << 60, None), "channels")
    _refused(L, L.pk_route_topk_f32((1 << 25) + 1, 64, 1, PTR, 64, PTR, PTR, None), "2^25")
    _refused(L, L.pk_expert_gather_f32(1 << 26, 4, 2, 4, PTR, PTR, PTR, 8, PTR, 8, None), "2^25")
    _refused(L, L.pk_expert_combine_f32(1 << 25, 4, 2, PTR, PTR, PTR, 8, None, 8, PTR, 8, None), "2^25")
    # 32768 rows of 1024 experts: more tiles than a launch has, streamed or not
    _refused(L, L.pk_gemm_experts_f32(b"N", 32768, 1 << 24, 4, 1024, PTR, PTR, 4, PTR, 1 << 24, 1 << 26, PTR, 1 << 24,
                                      0, 0, None), "too large")
    _refused(L, L.pk_gemm_experts_f32(b"T", (1 << 21) * 64, 64, 64, 1, PTR, PTR, 64, PTR, 64, 0, PTR, 64, 0, 1, None),
             "too large")
    _refused(L, L.pk_gemm_experts_dw_f32(32768, 1 << 12, 1 << 20, 1024, PTR, PTR, 1 << 12, PTR, 1 << 20, PTR, 1 << 20,
                                         1 << 32, 0, 0, None, 0, None), "too large")
