"""CPU: what the gated recurrence, attention and paged attention refuse, by the C ABI and by the Python operators."""
import ctypes

import pytest
import torch

from rwkv_cuda_amd import _lib, attention, gated_recurrence, paged_attention

P = 0x1000          # never dereferenced: every call below fails validation first


def _grec(**change):
    n = 2 * 8 * 4 * 4
    a = dict(dtype=0, gate=0, tied=1, B=2, T=8, C=4, w=P, w_sb=32, w_st=4, x=P, x_sb=32, x_st=4, y=P, hT=P, saved=None, saved_bytes=0, dy=P, dw=P, dx=P, workspace=P, workspace_bytes=1 << 40)
    a.update(change)
    return ctypes.byref(_lib.GrecArgs(**a))


def _attn(**change):
    a = dict(dtype=0, causal=1, B=1, Tq=4, Tk=4, H=2, Hk=1, N=64, scale=0.1, cap=0.0, q=P, k=P, v=P, q_sb=512, q_st=128, q_sh=64, k_sb=256, k_st=64, k_sh=64, v_sb=256, v_st=64, v_sh=64,
             y=P, y_rest=P, lse=P, dy=P, dq=P, dk=P, dv=P, workspace=P, workspace_bytes=1 << 40)
    a.update(change)
    return ctypes.byref(_lib.AttnArgs(**a))


def _paged(**change):
    a = dict(dtype=0, B=1, H=2, Hk=1, N=64, P=3, page=16, M=2, scale=0.1, cap=0.0, q=P, k_pages=P, v_pages=P, k_sp=1024, k_st=64, k_sh=64, v_sp=1024, v_st=64, v_sh=64, table=P, lens=P, y=P,
             workspace=P, workspace_bytes=1 << 40)
    a.update(change)
    return ctypes.byref(_lib.PagedArgs(**a))


@pytest.mark.parametrize("change,status", [
    (dict(dtype=3), -1), (dict(dtype=-1), -1), (dict(gate=2), -1), (dict(B=0), -1), (dict(T=0), -1), (dict(C=-4), -1), (dict(B=65536), -1), (dict(w=None), -2), (dict(x=None), -2),
    (dict(T=(1 << 31) - 1), -1), (dict(w=P + 1), -3), (dict(dtype=2, x=P + 2), -3), (dict(h0=P + 2), -3), (dict(doc=P + 1), -3)])
def test_recurrence_entry_points(lib, change, status):
    assert lib.rwkv_grec_forward(None, _grec(**change)) == status
    need = lib.rwkv_grec_saved_bytes(2, 8, 4)
    assert lib.rwkv_grec_backward(None, _grec(saved=P, saved_bytes=need, **change)) == status


def test_recurrence_entry_points_of_one_direction(lib):
    assert lib.rwkv_grec_forward(None, None) == -2 and lib.rwkv_grec_backward(None, None) == -2
    assert lib.rwkv_grec_forward(None, _grec(y=None)) == -2 and lib.rwkv_grec_forward(None, _grec(hT=None)) == -2
    need = lib.rwkv_grec_saved_bytes(2, 8, 4)
    assert need > 0 and lib.rwkv_grec_saved_bytes(0, 8, 4) == 0
    assert lib.rwkv_grec_forward(None, _grec(saved=P, saved_bytes=need - 1)) == -4
    assert lib.rwkv_grec_forward(None, _grec(saved=P + 4, saved_bytes=need)) == -3
    assert lib.rwkv_grec_backward(None, _grec(saved=None)) == -2 and lib.rwkv_grec_backward(None, _grec(saved=P, saved_bytes=need, dw=None)) == -2
    T = 1 << 16                                                       # long enough for a workspace
    n = lib.rwkv_grec_workspace_bytes(1, T, 64)
    if n > 0:
        for ws in (dict(workspace=None), dict(workspace=P + 8), dict(workspace_bytes=n - 1)):
            assert lib.rwkv_grec_forward(None, _grec(B=1, T=T, C=64, **ws)) == -4


@pytest.mark.parametrize("change,status", [
    (dict(dtype=2), -1), (dict(B=0), -1), (dict(Tq=0), -1), (dict(Tk=3), -1), (dict(H=3, Hk=2), -1), (dict(Hk=0), -1), (dict(N=132), -1), (dict(N=12), -1), (dict(N=136), -1),
    (dict(scale=0.0), -1), (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(cap=1e-9), -1), (dict(cap=4097.0), -1), (dict(Tk=(1 << 31) - 1), -1),
    (dict(Tk=(1 << 24) + 1, slopes=P), -1), (dict(q_st=1 << 24), -1), (dict(v_st=-64), -1), (dict(cap=-1.0), -1), (dict(cap=float("nan")), -1), (dict(prefix=P, causal=0), -1), (dict(B=65536), -1), (dict(q_st=130), -3), (dict(k_sb=4), -3),
    (dict(v_sh=1), -3), (dict(q=None), -2), (dict(k=P + 8), -3), (dict(y=None), -2), (dict(doc=P + 2), -3), (dict(slopes=P + 1), -3), (dict(prefix=P + 2), -3), (dict(lse=P + 1), -3)])
def test_attention_entry_points(lib, change, status):
    assert lib.rwkv_attn_forward(None, _attn(**change)) == status
    assert lib.rwkv_attn_backward(None, _attn(**change)) == status


def test_attention_entry_points_of_one_direction(lib):
    assert lib.rwkv_attn_forward(None, None) == -2 and lib.rwkv_attn_forward(None, _attn(y_rest=P + 2)) == -3
    size = lambda *a: lib.rwkv_attn_workspace_bytes(1, a[0], a[1], 2, 1, 64, a[2], a[3])
    need = size(4, 4, 0, 1)
    assert need > 0 and size(4, 4, 0, 0) == 0 and size(5, 4, 1, 1) == 0
    with_doc = size(4, 4, 1, 0)
    assert with_doc > 0 and size(4, 4, 1, 1) > need
    parts = size(4, 70000, 0, 0)                                    # few queries, many keys: in parts
    assert parts > 0 and lib.rwkv_attn_forward(None, _attn(Tk=70000, workspace_bytes=parts - 1)) == -4
    for change in (dict(workspace=None), dict(workspace=P + 8), dict(workspace_bytes=with_doc - 1)):
        assert lib.rwkv_attn_forward(None, _attn(doc=P, **change)) == -4, change
    for change, status in ((dict(dy=None), -2), (dict(dq=P + 2), -3), (dict(lse=None), -2), (dict(y_rest=None), -2), (dict(workspace=None), -4), (dict(workspace=P + 8), -4),
                           (dict(workspace_bytes=need - 1), -4)):
        assert lib.rwkv_attn_backward(None, _attn(**change)) == status, change


@pytest.mark.parametrize("change,status", [
    (dict(dtype=2), -1), (dict(B=0), -1), (dict(H=3, Hk=2), -1), (dict(N=12), -1), (dict(N=136), -1), (dict(P=0), -1), (dict(M=0), -1), (dict(page=0), -1), (dict(page=24), -1), (dict(page=-16), -1),
    (dict(scale=-1.0), -1), (dict(cap=float("nan")), -1), (dict(cap=1e-9), -1), (dict(cap=4097.0), -1), (dict(M=1 << 27), -1), (dict(k_sp=1028), -3), (dict(v_st=4), -3), (dict(q=None), -2), (dict(k_pages=None), -2), (dict(v_pages=P + 8), -3), (dict(table=None), -2),
    (dict(lens=None), -2), (dict(lens=P + 2), -3), (dict(k=P), -2), (dict(k=P, v=P + 8), -3), (dict(y=None), -2), (dict(slopes=P + 2), -3)])
def test_paged_entry_point(lib, change, status):
    assert lib.rwkv_paged_attn(None, _paged(**change)) == status
    assert lib.rwkv_paged_attn(None, None) == -2


def test_paged_workspace(lib):
    n = lib.rwkv_paged_workspace_bytes(1, 2, 1, 64, 16, 4096)
    if n > 0:
        for ws in (dict(workspace=None), dict(workspace=P + 8), dict(workspace_bytes=n - 1)):
            assert lib.rwkv_paged_attn(None, _paged(M=4096, **ws)) == -4


def test_python_operators_refuse_cpu_tensors_and_wrong_arguments():
    w = torch.zeros(1, 4, 8)
    q = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: gated_recurrence.RUN_CUDA(w, w), lambda: gated_recurrence.RUN_CUDA(w, w[:, :3]), lambda: gated_recurrence.STEP(w[:, 0], w[:, 0], torch.zeros(1, 8)),
                 lambda: attention.RUN_CUDA(q, q, q), lambda: attention.RUN_CUDA(q[0], q, q), lambda: attention.RUN_CUDA(q, q[:, :3], q),
                 lambda: paged_attention.RUN_CUDA(q[:, 0], q, q, torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32))):
        with pytest.raises(AssertionError):
            call()
    with pytest.raises(ValueError):
        gated_recurrence.RUN_CUDA(w, w, gate="tanh")


gpu = pytest.mark.gpu


@gpu
def test_recurrence_refusals_on_the_device(lib):
    w, x, h = (torch.zeros(*s, device="cuda") for s in ((2, 4, 8), (2, 4, 8), (2, 8)))
    doc = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    R = gated_recurrence.RUN_CUDA
    for call in (lambda: R(w, x.half()), lambda: R(w.double(), x.double()), lambda: R(w, x, h.half()), lambda: R(w, x, h[:1]), lambda: R(w, x, h, doc.long()), lambda: R(w, x, h, doc[:, :3]),
                 lambda: R(w, x, h.cpu()), lambda: R(w.transpose(1, 2), x.transpose(1, 2)), lambda: R(w, x, torch.zeros(2, 16, device="cuda")[:, ::2]), lambda: R(w[0], x[0])):
        with pytest.raises(AssertionError):
            call()
    with pytest.raises(_lib.RwkvHipError):
        R(w[:, :0], x[:, :0])
    with pytest.raises(AssertionError):
        gated_recurrence.STEP(w[:, 0].requires_grad_(True), x[:, 0], h)
    w, two = w.detach(), torch.zeros(3, 8, device="cuda")             # an `out` that shares memory with the other arguments, but is not h
    for call in (lambda: gated_recurrence.STEP(w[:, 0], x[:, 0], two[:2], out=two[1:]), lambda: gated_recurrence.STEP(two[:2], x[:, 0], h, out=two[1:]),
                 lambda: gated_recurrence.STEP(w[:, 0], two[1:], two[1:])):
        with pytest.raises(AssertionError, match="memory"):
            call()
    leaf = w.detach().requires_grad_(True)
    with pytest.raises(_lib.RwkvHipError, match="second derivatives"):
        torch.autograd.grad(R(leaf, x)[0].sum(), leaf, create_graph=True)


@gpu
def test_attention_refusals_on_the_device(lib):
    bf = torch.bfloat16
    q, k = torch.zeros(2, 4, 4, 64, device="cuda", dtype=bf), torch.zeros(2, 6, 2, 64, device="cuda", dtype=bf)
    R = attention.RUN_CUDA
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    slopes = torch.zeros(4, device="cuda")
    for call in (lambda: R(q.float(), k.float(), k.float()), lambda: R(q, k.half(), k), lambda: R(q, k[:, :3], k[:, :3]), lambda: R(q[:, :, :3], k, k), lambda: R(q, k[..., :32], k[..., :32]),
                 lambda: R(q[..., :60], k[..., :60], k[..., :60]), lambda: R(q, k, k, doc=i32(2, 4)), lambda: R(q, k, k, doc=i32(2, 6).long()), lambda: R(q, k, k, prefix=i32(3)),
                 lambda: R(q, k, k, prefix=i32(2), causal=False), lambda: R(q, k, k, slopes=slopes[:2]), lambda: R(q, k, k, cap=-1.0), lambda: R(q, k, k, scale=0.0), lambda: R(q, k, k, cap=float("inf")), lambda: R(q, k, k, cap=1e-9), lambda: R(q, k, k, cap=5000.0),
                 lambda: R(q, k, k, slopes=slopes.clone().requires_grad_(True)), lambda: R(q.transpose(2, 3), k, k)):
        with pytest.raises(AssertionError):
            call()
    with pytest.raises(_lib.RwkvHipError):
        R(q[:, :0], k, k)
    odd = torch.zeros(2 * 4 * 4 * 64 + 4, device="cuda", dtype=bf)[4:].view(2, 4, 4, 64)
    with pytest.raises(_lib.RwkvHipError, match="align"):
        R(odd, k, k)
    leaf = q.clone().requires_grad_(True)
    with pytest.raises(_lib.RwkvHipError, match="second derivatives"):
        torch.autograd.grad(R(leaf, k, k).float().sum(), leaf, create_graph=True)


@gpu
def test_paged_refusals_on_the_device(lib):
    bf = torch.bfloat16
    q, kp = torch.zeros(2, 4, 64, device="cuda", dtype=bf), torch.zeros(5, 16, 2, 64, device="cuda", dtype=bf)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    R = paged_attention.RUN_CUDA
    new = torch.zeros(2, 2, 64, device="cuda", dtype=bf)
    for call in (lambda: R(q, kp, kp[:4], i32(2, 2), i32(2)), lambda: R(q, kp, kp.half(), i32(2, 2), i32(2)), lambda: R(q, kp, kp, i32(2, 2).long(), i32(2)), lambda: R(q, kp, kp, i32(3, 2), i32(2)),
                 lambda: R(q, kp, kp, i32(2, 2), i32(3)), lambda: R(q, kp, kp, i32(4), i32(2)), lambda: R(q, kp[:, :12], kp[:, :12], i32(2, 2), i32(2)), lambda: R(q[:, :3], kp, kp, i32(2, 2), i32(2)),
                 lambda: R(q, kp, kp, i32(2, 2), i32(2), k=new), lambda: R(q, kp, kp, i32(2, 2), i32(2), k=new, v=new[:1]), lambda: R(q, kp, kp, i32(2, 2), i32(2), cap=-2.0),
                 lambda: R(q.clone().requires_grad_(True), kp, kp, i32(2, 2), i32(2)), lambda: R(q, kp, kp, i32(2, 2), i32(2), scale=-1.0)):
        with pytest.raises(AssertionError):
            call()
    with pytest.raises(_lib.RwkvHipError):
        R(q, kp[:0], kp[:0], i32(2, 2), i32(2))


def test_sizes_of_workspaces_for_heads_that_do_not_fit(lib):
    """More key heads than heads, or heads that are no multiple of them: no size, as for any call that is refused."""
    assert lib.rwkv_paged_workspace_bytes(1, 1, 2, 64, 16, 4096) == 0
    assert lib.rwkv_paged_workspace_bytes(1, 3, 2, 64, 16, 4096) == 0
    assert lib.rwkv_paged_workspace_bytes(1, 2, 1, 136, 16, 4096) == 0
    assert lib.rwkv_attn_workspace_bytes(1, 4, 4, 1, 2, 64, 0, 1) == 0
    many = 1 << 30                                                  # (as many workgroups are 0 modulo 2^64)
    assert lib.rwkv_attn_workspace_bytes(many, 2048, 2048, many, many, 64, 0, 1) == 0 and lib.rwkv_paged_workspace_bytes(many, many, many, 64, 16, 4096) == 0


def test_slopes_and_the_smallest_scale(lib):
    """Biases are divided by the scale: below 2^-60 they would be infinities."""
    for call in (lib.rwkv_attn_forward, lib.rwkv_attn_backward):
        assert call(None, _attn(slopes=P, scale=2.0 ** -61)) == -1 and call(None, _attn(slopes=P, scale=1e-45)) == -1
        assert call(None, _attn(slopes=P, scale=2.0 ** -60, q=None)) == -2 and call(None, _attn(scale=2.0 ** -61, q=None)) == -2


def test_calls_that_need_a_workspace_have_one(lib):
    """The sizes for which a small or missing workspace is refused are sizes above 0, and short calls need none."""
    n, m = lib.rwkv_grec_workspace_bytes(1, 1 << 16, 64), lib.rwkv_paged_workspace_bytes(1, 2, 1, 64, 16, 4096)
    assert n > 0 and m > 0 and lib.rwkv_grec_workspace_bytes(2, 8, 4) == 0 and lib.rwkv_paged_workspace_bytes(1, 2, 1, 64, 16, 2) == 0
    for ws in (dict(workspace=None), dict(workspace=P + 8)):
        assert lib.rwkv_grec_forward(None, _grec(B=1, T=1 << 16, C=64, **ws)) == -4 and lib.rwkv_paged_attn(None, _paged(M=4096, **ws)) == -4
    assert lib.rwkv_grec_forward(None, _grec(B=1, T=1 << 16, C=64, workspace_bytes=n - 1)) == -4 and lib.rwkv_paged_attn(None, _paged(M=4096, workspace_bytes=m - 1)) == -4
