"""Kernels that larger calls around a learned head take, by shape, with and without lists:
the wide workgroups of sampling, gradients that read a row twice and in segments, and
outputs that leave what lies around them alone.  test_host_head_kernels.py holds each
shape to the kernel that it is meant for."""
import head_reference as ref
import pytest
import torch
from conftest import log_case
from test_gpu_head import _cuda, _distill_inputs, _gen, _row_kw, _strided

import thrml_hip as th

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32

# rows, q, history, bias, mask: a workgroup of 1024 for a row
WIDE = [(150, 9001, 0, 0, "none"), (150, 9001, 300, 12, "rows"), (200, 20000, 0, 0, "shared"), (200, 20000, 2000, 0, "none"),
        (129, 8200, 40, 300, "rows")]
# rows, q, k of gradients that read the row twice, by type
TWICE = {F32: [(65, 65543, 40), (70, 65537, 1)], F16: [(65, 131081, 40), (66, 131073, 300)], BF16: [(65, 131081, 40), (66, 140001, 3)]}
# rows, q, k of losses alone: 8 and 16 waves
LOSS = [(300, 9001, 33), (256, 20003, 64), (3, 65543, 300)]
# rows, q, k of gradients with the row in the registers of 4, 8 and 16 waves (16 bits; in f32
# the first two)
KEPT = [(70, 32768, 9), (70, 32769, 9), (70, 65536, 9), (70, 65537, 9), (65, 131072, 9)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,q,history,bias,mask", WIDE)
def test_wide_samples(device, rows, q, history, bias, mask, dtype):
    log_case(f"wide samples {rows} {q} {history} {bias} {mask} {dtype}")
    g = _gen(rows + q + history)
    z = (2.5 * torch.randn(rows, q, generator=g)).to(dtype)
    u = torch.rand(rows, q, generator=g)
    kw = _row_kw(g, rows, q, history, bias, mask)
    for uniforms in (u, None):
        want, lp, bound = ref.sampled(z, uniforms, **kw)
        index, logprob = th.sample_logits(device, _strided(z, 3, 1), _strided(uniforms, 5) if uniforms is not None else None,
                                          **_cuda(kw))
        assert index.cpu().tolist() == want.tolist()
        ref.close(logprob, lp, bound, "logprob")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("i", [0, 1])
def test_gradients_that_read_twice(device, i, dtype):
    rows, q, k = TWICE[dtype][i]
    log_case(f"read twice {rows} {q} {k} {dtype}")
    z, ids, teacher, weight = _distill_inputs(rows, q, k, dtype, q)
    loss, lb, grad, gb = ref.distilled(z, ids, teacher, weight, 1.5)
    got_loss, got_grad = th.distill_grad(device, _strided(z, 5, 3), ids.cuda(), teacher.cuda(), weight.cuda(), 1.5)
    ref.close(got_loss, loss, lb, "loss")
    ref.close(got_grad, grad, gb, "grad")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,q,k", KEPT)
def test_gradients_in_registers(device, rows, q, k, dtype):
    log_case(f"registers {rows} {q} {k} {dtype}")
    z, ids, teacher, weight = _distill_inputs(rows, q, k, dtype, q + 1)
    loss, lb, grad, gb = ref.distilled(z, ids, teacher, weight)
    got_loss, got_grad = th.distill_grad(device, z.cuda(), ids.cuda(), teacher.cuda(), weight.cuda())
    ref.close(got_loss, loss, lb, "loss")
    ref.close(got_grad, grad, gb, "grad")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,q,k", LOSS)
def test_losses_alone(device, rows, q, k, dtype):
    log_case(f"loss alone {rows} {q} {k} {dtype}")
    z, ids, teacher, _ = _distill_inputs(rows, q, k, dtype, q + 2)
    loss, lb, _, _ = ref.distilled(z, ids, teacher, None, 0.8)
    ref.close(th.distill_loss(device, _strided(z, 1, 1), ids.cuda(), teacher.cuda(), 0.8), loss, lb, "loss")


def _guarded(rows, q, pad, dtype):
    """(the whole buffer, a view of it with `pad` elements before, between and after rows)"""
    whole = torch.full((rows + 2, q + pad), 7.0, dtype=dtype, device="cuda")
    return whole, whole[1:-1, :q]


def _untouched(whole, q):
    return bool((whole[0] == 7.0).all() and (whole[-1] == 7.0).all() and (whole[:, q:] == 7.0).all())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,q,pad", [(3, 1, 1), (5, 33, 3), (40, 4099, 1), (600, 131, 5), (9, 65537, 7), (70, 8190, 9)])
def test_outputs_within_their_rows(device, rows, q, pad, dtype):
    """(a gradient in segments, from registers, read twice; processed logits by 8 and 16)"""
    log_case(f"within rows {rows} {q} {pad} {dtype}")
    z, ids, teacher, weight = _distill_inputs(rows, q, 3, dtype, rows + q)
    args = (device, z.cuda(), ids.cuda(), teacher.cuda(), weight.cuda())
    whole, view = _guarded(rows, q, pad, dtype)
    _, grad = th.distill_grad(*args, out=view)
    assert grad is view and _untouched(whole, q)
    assert torch.equal(view, th.distill_grad(*args)[1])
    kw = _cuda(_row_kw(_gen(q), rows, q, 20, 4, "rows"))
    for out in (dtype, F32):
        whole, view = _guarded(rows, q, pad, out)
        th.process_logits(device, z.cuda(), out=view, out_dtype=out, **kw)
        assert _untouched(whole, q)
        assert torch.equal(view, th.process_logits(device, z.cuda(), out_dtype=out, **kw))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gradients_read_twice_within_their_rows(device, dtype):
    rows, q, _ = TWICE[dtype][0]
    log_case(f"read twice within rows {rows} {q} {dtype}")
    z, ids, teacher, weight = _distill_inputs(rows, q, 3, dtype, 1)
    whole, view = _guarded(rows, q, 5, dtype)
    th.distill_grad(device, z.cuda(), ids.cuda(), teacher.cuda(), weight.cuda(), out=view)
    assert _untouched(whole, q)
