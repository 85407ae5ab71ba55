"""CPU: what the gated delta rule, the paged cache in 8 bits and the page tables refuse, by the C ABI and by the Python operators."""
import ctypes

import pytest
import torch

from rwkv_cuda_amd import _lib, gated_delta, page_tables, paged_attention8

P = 0x1000          # never dereferenced: every call below fails validation first
gpu = pytest.mark.gpu


def _delta(**change):
    a = dict(dtype=0, B=1, T=4, H=2, Hk=1, N=64, scale=0.1, q=P, k=P, v=P, q_sb=256, q_st=64, q_sh=64, k_sb=256, k_st=64, k_sh=64, v_sb=512, v_st=128, v_sh=64, g=P, beta=P, g_sb=8, g_st=2, beta_sb=8,
             beta_st=2, y=P, sT=P, saved=P, saved_bytes=1 << 40, dy=P, dq=P, dk=P, dv=P, dg=P, dbeta=P, workspace=P, workspace_bytes=1 << 40)
    a.update(change)
    return ctypes.byref(_lib.DeltaArgs(**a))


def _cache(**change):
    a = dict(dtype=0, n=3, Hk=2, N=64, P=5, page=16, k=P, v=P, k_st=128, k_sh=64, v_st=128, v_sh=64, k_pages=P, v_pages=P, kp_sp=2048, kp_st=128, kp_sh=64, vp_sp=2048, vp_st=128, vp_sh=64, k_scales=P,
             v_scales=P, slots=P)
    a.update(change)
    return ctypes.byref(_lib.Cache8Args(**a))


def _paged8(**change):
    a = dict(dtype=0, B=1, H=2, Hk=1, N=64, P=3, page=16, M=2, scale=0.1, cap=0.0, q=P, k_pages=P, v_pages=P, k_sp=1024, k_st=64, k_sh=64, v_sp=1024, v_st=64, v_sh=64, k_scales=P, v_scales=P, table=P,
             lens=P, y=P, workspace=P, workspace_bytes=1 << 40)
    a.update(change)
    return ctypes.byref(_lib.Paged8Args(**a))


def _tables(**change):
    a = dict(B=2, M=4, F=9, page=16, n=5, lens=P, more=P, table=P, pool=P, taken=P, slots=P, starts=P, held=P, taken_out=P)
    a.update(change)
    return ctypes.byref(_lib.TablesArgs(**a))


@pytest.mark.parametrize("change,status", [
    (dict(dtype=2), -1), (dict(B=0), -1), (dict(T=0), -1), (dict(H=3, Hk=2), -1), (dict(Hk=0), -1), (dict(N=0), -1), (dict(N=12), -1), (dict(N=136), -1), (dict(B=65536), -1), (dict(H=65536), -1),
    (dict(T=(1 << 31) - 1), -1), (dict(scale=0.0), -1), (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(q_st=4), -3), (dict(k_sb=1), -3), (dict(v_sh=12), -3), (dict(q=None), -2),
    (dict(k=P + 8), -3), (dict(v=None), -2), (dict(g=None), -2), (dict(beta=None), -2), (dict(g=P + 1), -3), (dict(beta=P + 1), -3), (dict(doc=P + 2), -3)])
def test_delta_entry_points(lib, change, status):
    assert lib.rwkv_delta_forward(None, _delta(**change)) == status
    assert lib.rwkv_delta_backward(None, _delta(**change)) == status


def test_delta_entry_points_of_one_direction(lib):
    assert lib.rwkv_delta_forward(None, None) == -2 and lib.rwkv_delta_backward(None, None) == -2
    for change, status in ((dict(y=None), -2), (dict(sT=None), -2), (dict(y=P + 8), -3), (dict(sT=P + 4), -3), (dict(s0=P + 8), -3), (dict(saved=P + 8), -3), (dict(saved_bytes=16), -4)):
        assert lib.rwkv_delta_forward(None, _delta(**change)) == status, change
    for change, status in ((dict(saved=None), -2), (dict(dq=None), -2), (dict(dk=P + 2), -3), (dict(dv=None), -2), (dict(dg=None), -2), (dict(dbeta=None), -2), (dict(dg=P + 1), -3), (dict(dy=P + 8), -3),
                           (dict(dsT=P + 8), -3), (dict(ds0=P + 8), -3), (dict(saved_bytes=16), -4), (dict(workspace=None), -4), (dict(workspace=P + 8), -4), (dict(workspace_bytes=16), -4)):
        assert lib.rwkv_delta_backward(None, _delta(**change)) == status, change
    assert lib.rwkv_delta_saved_bytes(1, 4, 2, 1, 64) > 16 and lib.rwkv_delta_workspace_bytes(1, 4, 2, 1, 64, 1) > 16
    for size in ((0, 4, 2, 1, 64), (1, 0, 2, 1, 64), (1, 4, 3, 2, 64), (1, 4, 2, 0, 64), (1, 4, 2, 1, 60), (1, 4, 2, 1, 136), (1 << 30, 1 << 30, 1 << 30, 1 << 30, 64)):
        assert lib.rwkv_delta_saved_bytes(*size) == 0 and lib.rwkv_delta_workspace_bytes(*size, 1) == 0 and lib.rwkv_delta_workspace_bytes(*size, 0) == 0


@pytest.mark.parametrize("change,status", [
    (dict(dtype=2), -1), (dict(n=0), -1), (dict(n=(1 << 31) - 1), -1), (dict(Hk=0), -1), (dict(Hk=65536), -1), (dict(N=8), -1), (dict(N=72), -1), (dict(N=144), -1), (dict(P=0), -1), (dict(page=12), -1),
    (dict(page=0), -1), (dict(k_st=4), -3), (dict(v_sh=2), -3), (dict(kp_sp=8), -3), (dict(vp_st=24), -3), (dict(k=None), -2), (dict(v=P + 8), -3), (dict(k_pages=P + 8), -3), (dict(v_pages=None), -2),
    (dict(k_scales=None), -2), (dict(v_scales=P + 2), -3), (dict(slots=None), -2), (dict(slots=P + 1), -3)])
def test_cache_entry_point(lib, change, status):
    assert lib.rwkv_cache8_write(None, _cache(**change)) == status
    assert lib.rwkv_cache8_write(None, None) == -2


@pytest.mark.parametrize("change,status", [
    (dict(dtype=2), -1), (dict(B=0), -1), (dict(H=3, Hk=2), -1), (dict(Hk=0), -1), (dict(N=8), -1), (dict(N=136), -1), (dict(P=0), -1), (dict(M=0), -1), (dict(page=3), -1), (dict(page=1 << 20, M=1 << 12), -1),
    (dict(B=65536), -1), (dict(scale=0.0), -1), (dict(cap=1e-9), -1), (dict(cap=float("nan")), -1), (dict(k_sp=8), -3), (dict(v_sh=24), -3), (dict(q=None), -2), (dict(k_pages=P + 8), -3), (dict(y=None), -2),
    (dict(table=None), -2), (dict(lens=None), -2), (dict(k_scales=None), -2), (dict(v_scales=P + 2), -3), (dict(slopes=P + 1), -3), (dict(M=4096, workspace=None), -4), (dict(M=4096, workspace=P + 8), -4),
    (dict(M=4096, workspace_bytes=16), -4)])
def test_attention_entry_point(lib, change, status):
    assert lib.rwkv_paged8_attn(None, _paged8(**change)) == status
    assert lib.rwkv_paged8_attn(None, None) == -2
    assert lib.rwkv_paged8_workspace_bytes(1, 2, 1, 64, 16, 4096) > 16 and lib.rwkv_paged8_workspace_bytes(1, 2, 1, 64, 16, 2) == 0 and lib.rwkv_paged8_workspace_bytes(1, 3, 2, 64, 16, 4096) == 0


@pytest.mark.parametrize("change,status", [
    (dict(B=0), -1), (dict(M=0), -1), (dict(F=0), -1), (dict(n=-1), -1), (dict(page=0), -1), (dict(page=24), -1), (dict(M=1 << 16, page=1 << 16), -1), (dict(B=1 << 20, M=1 << 12), -1), (dict(lens=None), -2),
    (dict(more=P + 2), -3), (dict(table=None), -2), (dict(pool=P + 1), -3), (dict(taken=None), -2), (dict(slots=None), -2), (dict(slots=P + 2), -3), (dict(starts=None), -2), (dict(held=P + 1), -3),
    (dict(taken_out=None), -2)])
def test_tables_entry_point(lib, change, status):
    assert lib.rwkv_tables_extend(None, _tables(**change)) == status
    assert lib.rwkv_tables_extend(None, None) == -2


def test_tensors_elsewhere_are_refused(lib):
    bf = torch.bfloat16
    q, g, s = torch.zeros(1, 4, 2, 64, dtype=bf), torch.zeros(1, 4, 2, dtype=bf), torch.zeros(1, 2, 64, 64)
    i32 = lambda *z: torch.zeros(*z, dtype=torch.int32)
    pages, scales = torch.zeros(3, 16, 2, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.ones(3, 2)
    for call in (lambda: gated_delta.RUN_CUDA(q, q, q, g, g), lambda: gated_delta.STEP(q[:, 0], q[:, 0], q[:, 0], g[:, 0], g[:, 0], s), lambda: paged_attention8.WRITE(q[0], q[0], pages, pages, scales, scales, i32(4)),
                 lambda: paged_attention8.RUN_CUDA(q[:, 0], pages, pages, scales, scales, i32(1, 1), i32(1)), lambda: page_tables.EXTEND(i32(2), i32(2), i32(2, 3), i32(5), i32(1), 16, 4)):
        with pytest.raises(AssertionError):
            call()


@gpu
def test_delta_refusals_on_the_device(lib):
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, device="cuda", dtype=dt)
    q, v, g, s = z(2, 4, 2, 64), z(2, 4, 4, 64), z(2, 4, 4), z(2, 4, 64, 64, dt=torch.float32)
    doc = z(2, 4, dt=torch.int32)
    R, S = gated_delta.RUN_CUDA, gated_delta.STEP
    for call in (lambda: R(q.float(), q.float(), v.float(), g.float(), g.float()), lambda: R(q, q.half(), v, g, g), lambda: R(q, q[:, :3], v, g, g), lambda: R(q, q, v[:, :, :3], g, g), lambda: R(q, q, v, g[..., :2], g),
                 lambda: R(q, q, v, g.float(), g), lambda: R(q[..., :60], q[..., :60], v[..., :60], g, g), lambda: R(q, q, v, g, g, s[:1]), lambda: R(q, q, v, g, g, s.bfloat16()), lambda: R(q, q, v, g, g, s.cpu()),
                 lambda: R(q, q, v, g, g, s, doc.long()), lambda: R(q, q, v, g, g, s, doc[:, :3]), lambda: R(q, q, v, g, g, scale=0.0), lambda: R(q, q, v, g, g, scale=float("inf")), lambda: R(q[0], q, v, g, g),
                 lambda: R(q.transpose(2, 3), q.transpose(2, 3), v, g, g), lambda: S(q, q, v, g, g, s), lambda: S(q[:, 0], q[:, 0], v[:, 0].clone().requires_grad_(True), g[:, 0], g[:, 0], s)):
        with pytest.raises(AssertionError):
            call()
    for call in (lambda: R(q[:, :0], q[:, :0], v[:, :0], g[:, :0], g[:, :0]), lambda: R(z(2, 4, 2, 68)[..., 4:], q, v, g, g)):
        with pytest.raises(_lib.RwkvHipError):
            call()
    two = z(3, 4, 64, 64, dt=torch.float32)
    with pytest.raises(AssertionError, match="memory"):
        S(q[:, 0], q[:, 0], v[:, 0], g[:, 0], g[:, 0], two[:2], out=two[1:])
    leaf = v.clone().requires_grad_(True)
    with pytest.raises(_lib.RwkvHipError, match="second derivatives"):
        torch.autograd.grad(R(q, q, leaf, g, g)[0].float().sum(), leaf, create_graph=True)
    with torch.inference_mode():
        frozen = torch.zeros(2, 4, 64, 64, device="cuda")
        S(q[:, 0], q[:, 0], v[:, 0], g[:, 0], g[:, 0], frozen)
    with pytest.raises(AssertionError, match="inference"):
        S(q[:, 0], q[:, 0], v[:, 0], g[:, 0], g[:, 0], frozen)


@gpu
def test_cache_refusals_on_the_device(lib):
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, device="cuda", dtype=dt)
    i32 = lambda *s: z(*s, dt=torch.int32)
    k, q, pages, sc = z(5, 2, 64), z(2, 4, 64), z(3, 16, 2, 64, dt=torch.uint8).view(torch.float8_e4m3fn), z(3, 2, dt=torch.float32)
    W, R = paged_attention8.WRITE, paged_attention8.RUN_CUDA
    for call in (lambda: W(k.float(), k.float(), pages, pages, sc, sc, i32(5)), lambda: W(k, k.half(), pages, pages, sc, sc, i32(5)), lambda: W(k, k[:4], pages, pages, sc, sc, i32(5)),
                 lambda: W(k, k, pages.view(torch.uint8), pages.view(torch.uint8), sc, sc, i32(5)), lambda: W(k, k, pages, pages[:2], sc, sc, i32(5)), lambda: W(k, k, pages, pages, sc[:2], sc, i32(5)),
                 lambda: W(k, k, pages, pages, sc, sc.half(), i32(5)), lambda: W(k, k, pages, pages, sc, sc, i32(4)), lambda: W(k, k, pages, pages, sc, sc, i32(5).long()), lambda: W(k[:, :1], k[:, :1], pages, pages, sc, sc, i32(5)),
                 lambda: W(k[..., :32], k[..., :32], pages, pages, sc, sc, i32(5)), lambda: W(k, k, pages[:, :12], pages[:, :12], sc, sc, i32(5)), lambda: W(k.clone().requires_grad_(True), k, pages, pages, sc, sc, i32(5)),
                 lambda: R(q.float(), pages, pages, sc, sc, i32(2, 2), i32(2)), lambda: R(q[..., :32], pages, pages, sc, sc, i32(2, 2), i32(2)), lambda: R(q[:, :3], pages, pages, sc, sc, i32(2, 2), i32(2)),
                 lambda: R(q, pages, pages, sc, sc, i32(3, 2), i32(2)), lambda: R(q, pages, pages, sc, sc, i32(2, 2).long(), i32(2)), lambda: R(q, pages, pages, sc, sc, i32(2, 2), i32(3)),
                 lambda: R(q, pages, pages, sc[:2], sc, i32(2, 2), i32(2)), lambda: R(q, pages, pages, sc, sc, i32(2, 2), i32(2), cap=-1.0), lambda: R(q, pages, pages, sc, sc, i32(2, 2), i32(2), scale=0.0),
                 lambda: R(q.clone().requires_grad_(True), pages, pages, sc, sc, i32(2, 2), i32(2)), lambda: R(q, pages, pages, sc, sc, i32(2, 2), i32(2), slopes=z(3, dt=torch.float32))):
        with pytest.raises(AssertionError):
            call()
    for call in (lambda: W(k, k, pages[:0], pages[:0], sc[:0], sc[:0], i32(5)), lambda: R(q, pages, pages, sc, sc, i32(2, 0), i32(2)), lambda: W(z(5, 2, 68)[..., 4:], k, pages, pages.clone(), sc, sc.clone(), i32(5))):
        with pytest.raises(_lib.RwkvHipError):
            call()
    # what two waves would write at once, or one while another reads it
    vp, vs = pages.clone(), sc.clone()
    W(k, k, pages, vp, sc, vs, i32(5))
    wide, whole = pages[:1].expand(3, 16, 2, 64), z(3, 2, 16, 2, 64, dt=torch.uint8).view(torch.float8_e4m3fn)
    for call, what in ((lambda: W(k, k, pages, pages, sc, vs, i32(5)), "of their own"), (lambda: W(k, k, pages, vp, sc, sc, i32(5)), "of their own"), (lambda: W(k, k, wide, vp, sc, vs, i32(5)), "expanded"),
                       (lambda: W(k, k, pages, vp[:, :1].expand(3, 16, 2, 64), sc, vs, i32(5)), "expanded"), (lambda: W(k, k, pages, vp, sc, vs, sc.view(torch.int32).flatten()[:5]), "share no memory"),
                       (lambda: W(pages.view(torch.bfloat16).flatten()[:640].view(5, 2, 64), k, pages, vp, sc, vs, i32(5)), "share no memory")):
        with pytest.raises(AssertionError, match=what):
            call()
    W(k, k, whole[:, 0], whole[:, 1], sc, vs, i32(5))            # (side by side they may lie)


@gpu
def test_tables_refusals_on_the_device(lib):
    i32 = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.int32)
    E = page_tables.EXTEND
    a, t, pool, one = i32(3), i32(3, 4), i32(9), i32(1)
    for call in (lambda: E(a.long(), a, t, pool, one, 16, 5), lambda: E(a, a[:2], t, pool, one, 16, 5), lambda: E(a, a, t[:2], pool, one, 16, 5), lambda: E(a, a, t, pool, i32(2), 16, 5), lambda: E(a, a, t, pool, one, 12, 5),
                 lambda: E(a, a, t, pool, one, 0, 5), lambda: E(a, a, t, pool, one, 16, -1), lambda: E(a, a, t, t[0], one, 16, 5), lambda: E(a, a, t.cpu(), pool, one, 16, 5), lambda: E(t[:, 0], a, t, pool, one, 16, 5)):
        with pytest.raises(AssertionError):
            call()
    for call in (lambda: E(a[:0], a[:0], t[:0], pool, one, 16, 5), lambda: E(a, a, t, pool[:0], one, 16, 5), lambda: E(a, a, t, pool, one, 1 << 30, 5)):
        with pytest.raises(_lib.RwkvHipError):
            call()
