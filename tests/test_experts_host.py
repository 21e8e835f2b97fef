"""The refusals of the C entry points around the experts: every check happens on the host before a launch, so it runs
without a GPU.  The pointers are addresses nobody reads."""
from __future__ import annotations

import pytest
import torch

from terrace import _hip

P = 1 << 20            # stands for a device address on any boundary; refused calls never look there
OK, EINVAL, ENOSPC = _hip.OK, _hip.EINVAL, _hip.ENOSPC


def call(name, *args):
    return getattr(_hip.load(), name)(*args)


def sort_args(x=P, idx=P, T=4, row=64, k=2, n=8, rows=P, where=P, counts=P, offsets=P, ws=P, ws_bytes=1 << 20):
    return (x, idx, T, row, k, n, rows, where, counts, offsets, None, ws, ws_bytes, None)


@pytest.mark.parametrize("bad", [
    dict(T=-1), dict(k=0), dict(k=-3), dict(n=0), dict(n=2049), dict(row=-1), dict(counts=None), dict(offsets=None),
    dict(idx=None), dict(where=None), dict(x=None), dict(rows=None), dict(T=1 << 31, k=2), dict(T=1 << 62, k=8),
    dict(row=100 | (64 << 32)), dict(row=64 | (1000 << 32)), dict(row=64 | (1024 << 32), x=P + 8), dict(T=5000, ws=None),
])
def test_expert_sort_refusals(bad):
    assert call("terrace_expert_sort", *sort_args(**bad)) == EINVAL


def test_expert_sort_workspace():
    assert _hip.query("terrace_expert_sort_workspace", 256, 8, 2048) == 256           # one launch, none needed
    need = _hip.query("terrace_expert_sort_workspace", 16384, 8, 256)
    assert need > 131072 * 4
    assert call("terrace_expert_sort", *sort_args(T=16384, k=8, n=256, ws_bytes=need - 1)) == ENOSPC
    for T, k, n in ((-1, 2, 8), (4, 0, 8), (1 << 40, 1 << 20, 8), (5000, 2, 0), (5000, 2, 4096)):
        assert _hip.query("terrace_expert_sort_workspace", T, k, n) == 256


def grad_args(rows=P, rd=1, dy=P, dd=1, where=P, w=P, wd=1, T=4, k=2, H=64, n=8, live=P, d_rows=P, d_w=P):
    return (rows, rd, dy, dd, where, w, wd, T, k, H, n, live, d_rows, d_w, None)


@pytest.mark.parametrize("bad", [
    dict(rd=3), dict(dd=3), dict(wd=-1), dict(T=-1), dict(k=0), dict(H=-1), dict(n=-1), dict(where=None), dict(dy=None),
    dict(rows=None), dict(live=None), dict(T=1 << 31, k=2), dict(T=1 << 24),
])
def test_expert_unsort_grad_refusals(bad):
    assert call("terrace_expert_unsort_grad", *grad_args(**bad)) == EINVAL


def test_expert_unsort_grad_with_nothing_to_do():
    assert call("terrace_expert_unsort_grad", *grad_args(d_rows=None, d_w=None)) == OK
    assert call("terrace_expert_unsort_grad", *grad_args(T=0, n=0)) == OK


def test_w4_sizes_and_refusals():
    size = lambda *a: _hip.query("terrace_w4_packed_bytes", *a)
    assert size(2, 17, 160, 32, 0) == 2 * 32 * 2 * 64 and size(2, 17, 160, 32, 1) == 2 * 32 * 8 * 2
    assert size(2, 17, 160, 32, 2) == 2 * 32 * 8
    for bad in ((0, 16, 64, 32, 0), (1, 0, 64, 32, 0), (1, 16, 0, 32, 0), (1, 16, 64, 16, 0), (1, 16, 96, 64, 0), (1, 16, 64, 32, 3),
                (1, 16, 64, 32, -1), (1, 1 << 24, 1 << 24, 128, 0), (1 << 21, 16, 64, 32, 0)):
        assert size(*bad) == 0, bad

    def pack(codes=P, scales=P, zeros=None, dtype=1, E=2, N=16, K=64, g=32, pc=P, ps=P, pz=None):
        return call("terrace_w4_pack", codes, scales, zeros, dtype, E, N, K, g, pc, ps, pz, None)
    for bad in (dict(codes=None), dict(scales=None), dict(pc=None), dict(ps=None), dict(zeros=P), dict(pz=P), dict(dtype=0),
                dict(g=48), dict(K=80), dict(E=0), dict(pc=P + 8), dict(scales=P + 1)):
        assert pack(**bad) == EINVAL, bad

    def linear(x=P, dtype=1, rows=4, counts=P, codes=P, scales=P, zeros=None, E=2, N=16, K=64, g=32, swiglu=0, out=P):
        return call("terrace_w4_linear", x, dtype, rows, counts, codes, scales, zeros, E, N, K, g, swiglu, out, None)
    assert linear(rows=0) == OK
    for bad in (dict(x=None), dict(counts=None), dict(codes=None), dict(scales=None), dict(out=None), dict(dtype=0), dict(rows=-1),
                dict(x=P + 8), dict(codes=P + 4), dict(scales=P + 2), dict(zeros=P + 4), dict(out=P + 1), dict(g=96), dict(K=65),
                dict(N=17, swiglu=1), dict(rows=(1 << 30) + 1), dict(rows=1 << 30, N=4096)):
        assert linear(**bad) == EINVAL, bad


def norm_args(y=P, yd=1, r=P, rd=1, wp=P, wpd=1, g=None, gd=1, kind=0, wn=P, wnd=1, T=4, H=64, h=P, n=P):
    return (y, yd, r, rd, wp, wpd, g, gd, kind, wn, wnd, 1.0, 1e-6, T, H, h, n, None, None)


NORM_BAD = [dict(T=-1), dict(H=0), dict(H=16385), dict(yd=3), dict(rd=2), dict(rd=3), dict(wpd=4), dict(wnd=-1), dict(kind=3),
            dict(kind=-1), dict(kind=1), dict(g=P), dict(g=P, kind=1, gd=3), dict(y=None), dict(r=None)]


@pytest.mark.parametrize("bad", NORM_BAD + [dict(h=None), dict(n=None)])
def test_block_norm_refusals(bad):
    assert call("terrace_block_norm", *norm_args(**bad)) == EINVAL


def norm_grad(stats=P, dh=P, dn=P, dy=P, dr=P, dwp=P, dg=None, dwn=P, ws=P, ws_bytes=1 << 24, **kw):
    return call("terrace_block_norm_grad", *norm_args(**kw)[:15], stats, dh, dn, dy, dr, dwp, dg, dwn, ws, ws_bytes, None)


@pytest.mark.parametrize("bad", NORM_BAD + [dict(stats=None), dict(ws=None), dict(ws=P + 4), dict(dg=P), dict(wp=None), dict(wn=None)])
def test_block_norm_grad_refusals(bad):
    assert norm_grad(**bad) == EINVAL


def test_block_norm_grad_workspace():
    assert _hip.query("terrace_block_norm_grad_workspace", 1000, 64) == 2 * 256 * 64 * 4
    assert _hip.query("terrace_block_norm_grad_workspace", 3, 64) == 2 * 3 * 64 * 4
    assert norm_grad(T=1000, ws_bytes=2 * 256 * 64 * 4 - 1) == ENOSPC


def test_the_python_layer_refuses_host_tensors():
    import terrace.ops as tops
    x, idx = torch.zeros(4, 32), torch.zeros(4, 2, dtype=torch.int64)
    for f in (lambda: tops.expert_sort(x, idx, 4), lambda: tops.block_norm(x, x), lambda: tops.w4_pack(x.byte(), x.half())):
        with pytest.raises(RuntimeError, match="ROCm device"):
            f()


def test_the_experts_of_one_layer_must_fit_each_other():
    from terrace.ops import W4Weights
    from terrace.ta2a_fwd import w4_experts
    w = lambda E, N, K, dt=torch.bfloat16: W4Weights(torch.zeros(1), None, None, E, N, K, 32, dt)
    w4_experts(w(4, 64, 128), w(4, 128, 32))
    for a, b in ((w(4, 63, 128), w(4, 128, 32)), (w(4, 64, 128), w(4, 128, 64)), (w(4, 64, 128), w(3, 128, 32)),
                 (w(4, 64, 128), w(4, 128, 32, torch.float16))):
        with pytest.raises(RuntimeError, match="cannot feed"):
            w4_experts(a, b)


def test_a_forward_mode_tangent_is_refused():
    import torch.autograd.forward_ad as fwAD
    import terrace.ops as tops
    x, idx = torch.zeros(4, 32), torch.zeros(4, 2, dtype=torch.int64)
    plan = tops.ExpertPlan(torch.zeros(8 + 8 + 3, dtype=torch.int64), 4, 2, 4)
    weights = tops.W4Weights(torch.zeros(1, dtype=torch.uint8), None, None, 1, 32, 32, 32, torch.float32)
    with fwAD.dual_level():
        d = fwAD.make_dual(x, torch.ones_like(x))
        rows, w = (fwAD.make_dual(t, torch.ones_like(t)) for t in (torch.zeros(8, 32), torch.zeros(4, 2)))
        calls = [lambda: tops.expert_sort(d, idx, 4), lambda: tops.expert_unsort(rows, None, plan),
                 lambda: tops.expert_unsort(torch.zeros(8, 32), w, plan), lambda: tops.block_norm(d, x),
                 lambda: tops.block_norm(x, d), lambda: tops.block_norm(x, x, d[0]), lambda: tops.block_norm(x, x, None, d[0]),
                 lambda: tops.block_norm(None, x, pre_weight=d[0]), lambda: tops.expert_linear_w4(d, None, weights)]
        for f in calls:
            with pytest.raises(RuntimeError, match="forward-mode"):
                f()
        with pytest.raises(RuntimeError, match="ROCm device"):          # a level alone is no tangent
            tops.block_norm(x, x)
        with torch.inference_mode(), pytest.raises(RuntimeError, match="ROCm device"):
            tops.block_norm(d, x)


def test_a_forward_mode_tangent_is_refused_by_the_operators_of_the_path_that_carry_gradients():
    import torch.autograd.forward_ad as fwAD
    import terrace.ops as tops
    from terrace.ops.k2_ref import k2_pack_ref
    from terrace.ta2a_dispatch import ta2a_permute, ta2a_unpermute
    x, idx, gates, probs = torch.zeros(4, 32), torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2), torch.zeros(4, 8)
    with fwAD.dual_level():
        dx, dg = (fwAD.make_dual(t, torch.ones_like(t)) for t in (x, gates))
        dp = fwAD.make_dual(probs, torch.ones_like(probs))
        geometry = dict(world=4, rank=0, rpn=2, n_experts=8)
        calls = [lambda: tops.k1_arrival(dx, idx, gates, 2, 2, 2), lambda: tops.k1_arrival(x, idx, dg, 2, 2, 2),
                 lambda: tops.k2_pack(dx, idx, gates, 4, 8, 2, 2), lambda: tops.k2_pack(x, idx, dg, 4, 8, 2, 2),
                 lambda: k2_pack_ref(dx, idx, gates, 4, 8, 2, 2), lambda: ta2a_permute(dx, probs, probs > 0, **geometry),
                 lambda: ta2a_permute(x, dp, probs > 0, **geometry), lambda: ta2a_unpermute(dx, None, x)]
        for f in calls:
            with pytest.raises(RuntimeError, match="forward-mode"):
                f()


def test_planes_that_do_not_fit_the_sizes_are_refused():
    """A product reads what the sizes say, so a handle built by hand is checked before its first one."""
    import terrace.ops as tops
    E, N, K, g = 2, 40, 160, 32                              # 3 column tiles, 2 blocks of k

    def planes(dtype=torch.bfloat16):
        return (torch.zeros(E * 48 * 2 * 64, dtype=torch.uint8), torch.zeros(E * 48 * 8, dtype=dtype),
                torch.zeros(E * 48 * 8, dtype=torch.uint8))

    c, s, z = planes()
    good = tops.W4Weights(c, s, z, E, N, K, g, torch.bfloat16)
    good.check()
    tops.W4Weights(c, s, None, E, N, K, g, torch.bfloat16).check()
    tops.W4Weights(c.view(E, 3, 2, 64, 16), s.view(E, -1), z, E, N, K, g, torch.bfloat16).check()
    odd = torch.zeros(c.numel() + 1, dtype=torch.uint8)[1:]
    for bad in ((c[:-1], s, z, E, N, K, g, torch.bfloat16), (c, s[:-8], z, E, N, K, g, torch.bfloat16),
                (c, s, z[:-8], E, N, K, g, torch.bfloat16), (c, s, z, E + 1, N, K, g, torch.bfloat16),
                (c, s, z, E, N + 16, K, g, torch.bfloat16), (c, s, z, E, N, K + 128, g, torch.bfloat16),
                (c, s, z, E, N, K, 64, torch.bfloat16), (c, s, z, E, N, 1 << 40, g, torch.bfloat16),
                (c, s, z, E, N, K, g, torch.float16), (c, s.float(), z, E, N, K, g, torch.float32),
                (c, None, z, E, N, K, g, torch.bfloat16), (c.view(torch.int8), s, z, E, N, K, g, torch.bfloat16),
                (c.repeat_interleave(2)[::2], s, z, E, N, K, g, torch.bfloat16), (odd, s, z, E, N, K, g, torch.bfloat16),
                (c, s.to("meta"), z, E, N, K, g, torch.bfloat16), (c, s, z, -1, N, K, g, torch.bfloat16)):
        with pytest.raises(RuntimeError, match="W4Weights"):
            tops.W4Weights(*bad).check()
    assert good._sound
    good.N = 56                                              # a handle that was sound is looked at again after a change
    assert not good._sound
    with pytest.raises(RuntimeError, match="W4Weights"):
        good.check()
