"""zs_ce_loss_grad with gradients in rows of longer rows: what Python's calls make
(bit for bit), and nothing beside it."""
import ctypes as C

import pytest
import torch

from tests.test_gpu_head import TYPES, inputs

pytestmark = pytest.mark.gpu


def call(h, W, labels, g, dh, dw):
    """The C entry; dh and dw are views of any row stride."""
    from tests.gpu_util import ctx
    from zllm_amd._lib import Ce, lib
    from zllm_amd.beam import DTYPES
    (N, D), V, size = h.shape, W.shape[0], h.element_size()
    want = 3 | (4 if W.data_ptr() % 16 or D * size % 16 or W.stride(0) * size % 16 else 0)
    need = C.c_uint64()
    assert lib().zs_ce_work(N, V, D, DTYPES[h.dtype], want, C.byref(need)) == 0
    work = torch.empty(max(1, need.value), dtype=torch.uint8, device="cuda")
    loss, lse = torch.empty(max(1, N), device="cuda"), torch.empty(max(1, N), device="cuda")
    a = Ce(N=N, V=V, D=D, dtype=DTYPES[h.dtype], ld_hidden=max(D, h.stride(0)), ld_weight=W.stride(0), d_hidden=h.data_ptr(), d_weight=W.data_ptr(),
           d_labels=labels.data_ptr(), ignore_index=-100, z_weight=0.0, d_loss=loss.data_ptr(), d_lse=lse.data_ptr(), d_row_grad=g.data_ptr(),
           row_grad_stride=1, d_dhidden=dh.data_ptr(), d_dweight=dw.data_ptr(), ld_dhidden=dh.stride(0), ld_dweight=dw.stride(0),
           d_work=work.data_ptr(), work_bytes=need.value)
    rc = lib().zs_ce_loss_grad(ctx().h, C.byref(a), torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    return loss[:N]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shift,pad", [(0, 8), (1, 3), (8, 0), (4, 4)])
@pytest.mark.parametrize("N,V,D", [(1, 33, 8), (40, 300, 99), (70, 260, 64), (130, 513, 100), (300, 700, 136), (300, 257, 7), (65400, 70, 20)])
def test_gradients_in_longer_rows(N, V, D, shift, pad, dtype):
    from tests.gpu_util import ctx
    from zllm_amd.head import head_loss_grad
    print(f"[case] strides N={N} V={V} D={D} {dtype} {shift} {pad}", flush=True)
    h, W, labels, g = inputs(N, V, D, dtype, seed=N + D, ignored=0.2)
    want = head_loss_grad(ctx(), h, W, labels, g)
    bufs = [torch.full((n + 2, shift + D + pad), -7.0, dtype=TYPES[dtype], device="cuda") for n in (N, V)]
    dh, dw = (b[1:-1, shift:shift + D] for b in bufs)
    loss = call(h, W, labels, g, dh, dw)
    for x, y in zip((loss, dh, dw), want):
        assert torch.equal(x, y)
    dh.fill_(-7.0)
    dw.fill_(-7.0)
    assert all(bool((b == -7.0).all()) for b in bufs)


def test_no_rows():
    W = torch.ones((30, 20), device="cuda")
    buf = torch.full((32, 27), -7.0, device="cuda")
    dw = buf[1:-1, 3:23]
    call(W[:0], W, torch.empty(0, dtype=torch.int64, device="cuda"), torch.empty(0, device="cuda"), torch.empty((1, 20), device="cuda"), dw)
    assert not dw.any()
    dw.fill_(-7.0)
    assert bool((buf == -7.0).all())
