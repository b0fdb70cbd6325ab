"""The operators around a learned head against their definitions in 64 bits
(head_reference.py): types, sizes from one category on, odd sizes and strides, masks
that leave nothing, infinities and NaN in masked places, histories and lists with
entries that do not count, other streams, graphs."""
import head_reference as ref
import numpy as np
import pytest
import torch
from conftest import log_case

import thrml_hip as th

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _strided(t, pad, shift=0):
    """t on the device as rows of a wider buffer, from element `shift` on"""
    rows, q = t.shape
    wide = torch.full((rows * (q + pad) + shift + 1,), 7.0).to(t.dtype).cuda()
    view = wide[shift:shift + rows * (q + pad)].view(rows, q + pad)[:, :q]
    view.copy_(t)
    return view


def _cuda(kw):
    return {k: v.cuda() if v is not None else None for k, v in kw.items()}


def _row_kw(g, rows, q, history=0, bias=0, mask="none", temperature=True):
    kw = {}
    if history:
        kw["history"] = (torch.rand(rows, history, generator=g)**3 * q).to(torch.int32)
        kw["history"][:, ::7] = torch.randint(-3, q + 3, kw["history"][:, ::7].shape, generator=g, dtype=torch.int32)
        kw["lengths"] = torch.randint(-1, history + 3, (rows,), generator=g, dtype=torch.int32)
        kw["prompt_lengths"] = torch.randint(-1, history + 2, (rows,), generator=g, dtype=torch.int32)
        kw["repetition"] = 0.8 + 0.6 * torch.rand(rows, generator=g)
        kw["presence"] = torch.randn(rows, generator=g)
        kw["frequency"] = 0.3 * torch.randn(rows, generator=g)
    if bias:
        # ids that do not count, and ids named several times
        kw["bias_ids"] = torch.randint(-2, q + 2, (rows, bias), generator=g, dtype=torch.int32)
        kw["bias_ids"][:, bias // 2:] = kw["bias_ids"][:, :bias - bias // 2]
        kw["bias_values"] = torch.randn(rows, bias, generator=g)
    if temperature:
        t = 0.25 + 1.5 * torch.rand(rows, generator=g)
        kw["temperature"] = torch.where(torch.rand(rows, generator=g) < 0.25, torch.zeros(()), t)
    if mask != "none":
        n = 1 if mask == "shared" else rows
        kw["mask"] = torch.randint(-2**31, 2**31, (n, (q + 31) // 32), generator=g).to(torch.int32)
    return kw


ROWS = [
    # rows, q, history, bias, mask, pad
    (1, 1, 0, 0, "none", 0), (3, 1, 5, 2, "none", 1), (2, 7, 3, 1, "rows", 0), (5, 33, 40, 6, "shared", 3),
    (1, 4096, 0, 0, "shared", 0), (4, 4097, 100, 0, "rows", 5), (2, 8191, 0, 17, "none", 1),
    (3, 12289, 700, 33, "rows", 7), (1, 50001, 2000, 300, "shared", 0), (2, 131072, 9000, 40, "rows", 0),
]


@pytest.mark.parametrize("out", [None, F32])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,q,history,bias,mask,pad", ROWS)
def test_process(device, rows, q, history, bias, mask, pad, dtype, out):
    log_case(f"process {rows} {q} {history} {bias} {mask} {pad} {dtype} {out}")
    g = _gen(rows * 1000 + q)
    z = (2.5 * torch.randn(rows, q, generator=g)).to(dtype)
    kw = _row_kw(g, rows, q, history, bias, mask)
    want, size = ref.processed(torch.float64, z, **kw)
    got = th.process_logits(device, _strided(z, pad, pad), out_dtype=out, **_cuda(kw))
    assert got.dtype == (out or dtype)
    # at most 6 roundings to f32, each of at most `size`
    ref.close(got, want, 6 * ref.EPS * size, "process")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,q,history,bias,mask,pad", ROWS)
def test_sample(device, rows, q, history, bias, mask, pad, dtype):
    log_case(f"sample {rows} {q} {history} {bias} {mask} {pad} {dtype}")
    g = _gen(rows * 2000 + q)
    z = (2.5 * torch.randn(rows, q, generator=g)).to(dtype)
    u = torch.rand(rows, q, generator=g)
    kw = _row_kw(g, rows, q, history, bias, mask)
    for uniforms in (u, None):
        want, lp, bound = ref.sampled(z, uniforms, **kw)
        index, logprob = th.sample_logits(device, _strided(z, pad, pad),
                                          _strided(uniforms, pad + 1) if uniforms is not None else None, **_cuda(kw))
        assert index.dtype == torch.int32 and index.cpu().tolist() == want.tolist()
        ref.close(logprob, lp, bound, "logprob")


def test_sample_many_rows(device):
    """More rows than compute units, every one by itself; rows that share an expanded
    buffer."""
    g = _gen(5)
    z = (3.0 * torch.randn(1, 700, generator=g)).to(BF16).expand(1500, 700)
    u = torch.rand(1500, 700, generator=g)
    log_case("sample 1500 x 700 expanded")
    index, logprob = th.sample_logits(device, z[:1].cuda().expand(1500, 700), u.cuda())
    want, lp, bound = ref.sampled(z, u)
    assert index.cpu().tolist() == want.tolist()
    ref.close(logprob, lp, bound, "logprob")


def test_sample_near_ties(device):
    """Uniforms that differ in their last place, or not at all: the pick is the first
    maximum of the scores in 64 bits."""
    log_case("near ties")
    g = _gen(11)
    rows, q = 64, 20000
    z = torch.randint(-2, 3, (rows, q), generator=g).float()
    base = torch.full((rows, q), 0.5)
    base[:, ::3] = float(np.nextafter(np.float32(0.5), np.float32(1)))
    z[:, torch.randint(0, q, (5,), generator=g)] = 2.0
    index, _ = th.sample_logits(device, z.cuda(), base.cuda(), temperature=torch.full((rows,), 0.7).cuda())
    want, _, _ = ref.sampled(z, base, temperature=torch.full((rows,), 0.7))
    assert index.cpu().tolist() == want.tolist()
    # all alike: the first category, in segments and workgroups of any kind
    for q in (5, 4096, 131072):
        flat = torch.zeros(2, q, device="cuda")
        log_case(f"all alike {q}")
        index, logprob = th.sample_logits(device, flat, torch.full((2, q), 0.25, device="cuda"))
        assert index.tolist() == [0, 0]
        index, logprob = th.sample_logits(device, flat)
        assert index.tolist() == [0, 0]
        assert (logprob.cpu().double() + np.log(q)).abs().max() < ref.EPS * (64 + 2 * q / 4096 + 4 * np.log(q + 1))


def test_sample_uniforms_at_the_ends(device):
    """u = 0 only where there is no other, subnormal u by its own score, u = 1 first."""
    log_case("uniform ends")
    inf = float("inf")
    z = torch.tensor([[0.0, 0.0, -inf, 0.0], [5.0, 1.0, 0.0, 0.0], [0.0, 0.0, 0.0, 0.0], [0.0, 0.05, 0.0, -inf]])
    u = torch.tensor([[0.0, 0.0, 0.5, 0.0], [0.0, 1e-30, 0.0, 0.0], [0.5, 1.0, 0.3, 1.0], [1e-45, 1e-40, 0.0, 0.9]])
    index, _ = th.sample_logits(device, z.cuda(), u.cuda())
    assert index.tolist() == [0, 1, 1, 1]
    want, _, _ = ref.sampled(z, u)
    assert index.tolist() == want.tolist()


@pytest.mark.parametrize("q", [40, 5000, 70000])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows_without_a_distribution(device, dtype, q):
    log_case(f"rows without a distribution {dtype} {q}")
    inf, nan = float("inf"), float("nan")
    low = torch.finfo(dtype).min
    z = torch.zeros(7, q)
    mask = torch.full((7, (q + 31) // 32), -1, dtype=torch.int32)
    mask[0] = 0                                  # nothing allowed
    z[1] = -inf                                  # the same by the logits
    z[2, q - 3] = nan                            # a NaN that counts
    z[3, 11] = inf
    z[4] = nan                                   # NaN and infinities in masked places alone
    z[4, 32:64:2] = inf
    mask[4] = 0
    mask[4, 0] = 1 << 9
    z[4, 9] = 1.5
    z[5] = low                                   # the type's lowest value is a logit like another
    z[6] = low
    z[6, 17] = 0.0
    z = z.to(dtype)
    u = torch.rand(7, q, generator=_gen(3)) * 0.9 + 0.05
    kw = {"mask": mask}
    got = th.process_logits(device, z.cuda(), **_cuda(kw)).cpu()
    want, _ = ref.processed(F32, z, **kw)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.to(dtype).nan_to_num())
    for uniforms in (u, None):
        index, logprob = th.sample_logits(device, z.cuda(), uniforms.cuda() if uniforms is not None else None,
                                          **_cuda(kw))
        assert index[:5].tolist() == [-1, -1, -1, -1, 9] and logprob[:4].isnan().all() and logprob[4] == 0.0
        want, lp, bound = ref.sampled(z, uniforms, **kw)
        assert index.cpu().tolist() == want.tolist()
        assert abs(float(logprob[5]) + np.log(q)) < ref.EPS * (64 + 2 * q / 4096 + 4 * np.log(q)) and logprob[6] == 0.0


@pytest.mark.parametrize("rows,q,history,bias", [(3, 40000, 8192, 0), (300, 9000, 8192, 300), (2, 9000, 30000, 5000),
                                                (1, 300000, 20000, 3000), (40, 5000, 300, 4000)])
def test_long_lists(device, rows, q, history, bias):
    """Histories and bias lists that a workgroup's LDS holds for parts of a row alone; the
    same bits from every call."""
    log_case(f"long lists {rows} {q} {history} {bias}")
    g = _gen(rows + q + history)
    z = 2.5 * torch.randn(rows, q, generator=g)
    u = torch.rand(rows, q, generator=g)
    kw = _row_kw(g, rows, q, history, bias, "rows")
    if rows > 5:  # (the reference takes a while for each row)
        z, u = z[:5].repeat(rows // 5, 1), u[:5].repeat(rows // 5, 1)
        kw = {k: v[:5].repeat(rows // 5, 1) if v.dim() == 2 else v[:5].repeat(rows // 5) for k, v in kw.items()}
    few = {k: v[:5] for k, v in kw.items()}
    times = max(1, rows // 5) if rows > 5 else 1
    want, size = ref.processed(torch.float64, z[:5], **few)
    got = th.process_logits(device, z.cuda(), **_cuda(kw))
    ref.close(got, want.repeat(times, 1), (6 * ref.EPS * size).repeat(times, 1), "process")
    want, lp, bound = ref.sampled(z[:5], u[:5], **few)
    index, logprob = th.sample_logits(device, z.cuda(), u.cuda(), **_cuda(kw))
    assert index.cpu().tolist() == want.tolist() * times
    ref.close(logprob, lp.repeat(times), bound.repeat(times), "logprob")
    for _ in range(3):
        again, logprob_again = th.sample_logits(device, z.cuda(), u.cuda(), **_cuda(kw))
        assert torch.equal(again, index) and torch.equal(logprob_again, logprob)


def test_rows_past_32_bits(device):
    """Rows that begin beyond 2^32 elements of their buffer."""
    log_case("offsets past 2^32 elements")
    rows, q = 70000, 65536
    z = torch.zeros(rows, q, dtype=BF16, device="cuda")
    g = _gen(21)
    at = [0, 65535, 65536, rows - 1]
    for r in at:
        z[r] = (2.0 * torch.randn(q, generator=g)).to(BF16).cuda()
    index, logprob = th.sample_logits(device, z)
    ids = torch.full((rows, 1), 7, dtype=torch.int32, device="cuda")
    loss = th.distill_loss(device, z, ids, torch.zeros(rows, 1, device="cuda"))
    part = z[at].cpu()
    want, lp, bound = ref.sampled(part)
    assert index[at].cpu().tolist() == want.tolist() and int(index[at[1] - 1]) == 0
    ref.close(logprob[at], lp, bound, "logprob")
    want, lb, _, _ = ref.distilled(part, ids[at].cpu(), torch.zeros(len(at), 1))
    ref.close(loss[at], want, lb, "loss")
    assert th.process_logits(device, z, out=z, temperature=torch.full((rows,), 0.5, device="cuda")) is z
    assert torch.equal(z[at].cpu(), (2.0 * part.float()).to(BF16)) and not z[65537].any()
    del z


def test_history_edges(device):
    """One category named thousands of times, lengths of zero, past the end and
    negative, a history of no entries."""
    log_case("history edges")
    z = torch.ones(4, 100)
    h = torch.full((4, 6000), 42, dtype=torch.int32)
    kw = {"history": h, "lengths": torch.tensor([0, 6000, 99999, -5], dtype=torch.int32),
          "prompt_lengths": torch.tensor([0, 1, 7000, 0], dtype=torch.int32),
          "repetition": torch.full((4,), 2.0), "presence": torch.full((4,), 0.25), "frequency": torch.full((4,), 0.125)}
    got = th.process_logits(device, z.cuda(), **_cuda(kw)).cpu()
    want = torch.ones(4, 100)
    want[1, 42] = 0.5 - 0.125 * 5999 - 0.25
    want[2, 42] = 0.5
    assert torch.equal(got, want)
    kw["history"] = h[:, :0]
    assert torch.equal(th.process_logits(device, z.cuda(), **_cuda(kw)).cpu(), z)


def test_in_place_and_out(device):
    log_case("process in place")
    g = _gen(8)
    z = torch.randn(6, 5001, generator=g).to(BF16)
    kw = _row_kw(g, 6, 5001, 60, 9, "rows")
    want = th.process_logits(device, z.cuda(), **_cuda(kw))
    view = _strided(z, 3)
    assert th.process_logits(device, view, out=view, **_cuda(kw)) is view
    assert torch.equal(view, want)


def test_transposed_and_empty(device):
    log_case("transposed logits, no rows")
    g = _gen(9)
    z = torch.randn(300, 5, generator=g)
    want, size = ref.processed(torch.float64, z.t())
    ref.close(th.process_logits(device, z.cuda().t()), want, size * 0, "transposed")
    assert th.process_logits(device, torch.zeros(0, 9, device="cuda")).shape == (0, 9)
    index, logprob = th.sample_logits(device, torch.zeros(0, 9, device="cuda"))
    assert index.shape == (0,) and logprob.shape == (0,)
    e = torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    loss, grad = th.distill_grad(device, torch.zeros(0, 9, device="cuda"), e, e.float(), torch.zeros(0, device="cuda"))
    assert loss.shape == (0,) and grad.shape == (0, 9)
    y = th.linear_i8(device, torch.zeros(0, 9, device="cuda"), torch.zeros(4, 9, dtype=torch.int8, device="cuda"),
                     torch.ones(4, device="cuda"))
    assert y.shape == (0, 4)


# ---------------------------------------------------------------------------
DISTILL = [
    # rows, q, k, tau, pad
    (1, 1, 1, 1.0, 0), (3, 2, 4, 0.5, 1), (5, 37, 1, 2.0, 3), (7, 1000, 8, 1.0, 0), (4, 4097, 33, 2.0, 5),
    (3, 16385, 64, 1.0, 1), (2, 50001, 300, 0.7, 0), (2, 65536, 256, 1.0, 8), (1, 131072, 1000, 1.0, 0),
    (2, 131073, 5, 3.0, 0), (1, 262145, 4096, 1.0, 0), (1300, 64, 3, 1.0, 0), (9, 9000, 0, 1.0, 0),
    (20, 65537, 40, 1.5, 3), (70, 33000, 12, 1.0, 0),
]


def _distill_inputs(rows, q, k, dtype, seed):
    g = _gen(seed)
    z = (2.5 * torch.randn(rows, q, generator=g)).to(dtype)
    ids = torch.randint(0, q, (rows, k), generator=g, dtype=torch.int32)  # an id may come twice
    drop = torch.rand(rows, k, generator=g)
    ids = torch.where(drop < 0.1, -1, torch.where(drop > 0.95, q + 2, ids))
    if rows > 2:
        ids[1] = -1
    teacher = 3.0 * torch.randn(rows, k, generator=g)
    if k > 3:
        teacher[0, 3] = -float("inf")
    return z, ids, teacher, torch.randn(rows, generator=g)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,q,k,tau,pad", DISTILL)
def test_distill(device, rows, q, k, tau, pad, dtype):
    log_case(f"distill {rows} {q} {k} {tau} {pad} {dtype}")
    z, ids, teacher, weight = _distill_inputs(rows, q, k, dtype, rows + q + k)
    loss, lb, grad, gb = ref.distilled(z, ids, teacher, weight, tau)
    zd = _strided(z, pad, pad)
    got = th.distill_loss(device, zd, ids.cuda(), teacher.cuda(), tau)
    ref.close(got, loss, lb, "loss alone")
    got_loss, got_grad = th.distill_grad(device, zd, ids.cuda(), teacher.cuda(), weight.cuda(), tau)
    assert got_grad.dtype == dtype
    ref.close(got_loss, loss, lb, "loss")
    ref.close(got_grad, grad, gb, "grad")


def test_distill_differences(device):
    """The gradient against differences of the loss: d of 2^-6 in one logit moves the
    loss by d grad + d^2 / 2 softmax (1 - softmax) + ...; symmetric differences leave
    d^2 / 6 times a third derivative of at most 1, and the two losses' roundings."""
    log_case("distill differences")
    z, ids, teacher, _ = _distill_inputs(1, 40, 6, F32, 77)
    z, ids, teacher = z.cuda(), ids.cuda(), teacher.cuda()
    _, grad = th.distill_grad(device, z, ids, teacher, torch.ones(1, device="cuda"))
    d = 2.0**-6
    e = torch.eye(40, device="cuda") * d
    up = th.distill_loss(device, z + e, ids.expand(40, -1), teacher.expand(40, -1)).double()
    down = th.distill_loss(device, z - e, ids.expand(40, -1), teacher.expand(40, -1)).double()
    _, lb, _, _ = ref.distilled(z.cpu(), ids.cpu(), teacher.cpu())
    assert ((up - down) / (2 * d) - grad[0].double()).abs().max() < d * d / 6 + 2 * float(lb[0]) / (2 * d)


@pytest.mark.parametrize("k,names", [(2, 1), (31, 7), (32, 31), (33, 1), (64, 63), (65, 20), (1000, 3), (4096, 2000), (4096, 1)])
@pytest.mark.parametrize("q,rows", [(40, 300), (5001, 3), (70000, 2)])
def test_distill_repeats(device, k, names, q, rows):
    """Lists that name few categories many times; each sum of m probabilities adds m
    roundings of itself to the bound (70000 categories: the rows in segments)."""
    log_case(f"distill repeats {k} {names} {q} {rows}")
    rows = rows if k < 1000 else 2
    z, _, teacher, weight = _distill_inputs(rows, q, k, F32, q + k + names)
    g = _gen(k)
    pool = torch.stack([torch.randperm(q, generator=g)[:names] for _ in range(rows)])
    pick = torch.randint(0, pool.shape[1], (rows, k), generator=g)
    ids = torch.gather(pool, 1, pick).int()
    ids[0, k // 2] = -1
    loss, lb, grad, gb = ref.distilled(z, ids, teacher, weight)
    p = torch.softmax(torch.where(ids < 0, -float("inf"), teacher.double()), 1)
    total, times = torch.zeros_like(grad), torch.zeros_like(grad)
    total.scatter_add_(1, ids.clamp(min=0).long(), p)
    times.scatter_add_(1, ids.clamp(min=0).long(), torch.ones_like(p))
    gb = gb + weight.abs().double()[:, None] * ref.EPS * times * total
    args = (device, z.cuda(), ids.cuda(), teacher.cuda(), weight.cuda())
    got_loss, got_grad = th.distill_grad(*args)
    ref.close(got_loss, loss, lb, "loss")
    ref.close(got_grad, grad, gb, "grad")
    assert torch.equal(got_grad, th.distill_grad(*args)[1])


@pytest.mark.parametrize("q", [50, 70000])
def test_distill_edges(device, q):
    """(70000 categories: the rows in segments)"""
    log_case(f"distill edges {q}")
    inf, nan = float("inf"), float("nan")
    z = torch.zeros(6, q)
    z[0, 7] = -inf                     # a logit without probability that the teacher wants
    z[1, 7] = -inf                     # one that it does not
    z[2] = nan                         # no entry: nothing of the row counts
    z[3, 4] = nan
    z[4] = torch.finfo(F32).min        # a row of the lowest value is uniform
    ids = torch.tensor([[7, 8], [3, 3], [-1, q + 9], [1, 2], [1, 1], [4, 5]], dtype=torch.int32)
    teacher = torch.tensor([[1.0, 1.0], [0.0, 2.0], [0.0, 0.0], [0.0, 1.0], [0.0, 0.0], [-inf, -inf]])
    loss, grad = th.distill_grad(device, z.cuda(), ids.cuda(), teacher.cuda(), torch.ones(6, device="cuda"))
    loss, grad = loss.cpu(), grad.cpu()
    assert loss[0] == inf and grad[0].isfinite().all() and abs(float(grad[0, 7]) + 0.5) < 4 * ref.EPS
    p = np.exp([0.0, 2.0] - np.logaddexp(0.0, 2.0))  # both of one id
    want = np.log(q - 1) + (p * np.log(p)).sum()
    assert abs(float(loss[1]) - want) < (64 + 2 * q / 4096) * ref.EPS * 16 and grad[1, 7] == 0.0
    assert loss[2] == 0.0 and (grad[2] == 0.0).all()
    assert loss[3].isnan() and grad[3].isnan().all()
    share = 1 / q
    assert abs(float(grad[4, 0]) - share) < (64 + 2 * q / 4096) * ref.EPS * share
    assert abs(float(grad[4, 1]) + 1 - share) < 16 * ref.EPS
    assert loss[5] == 0.0 and (grad[5] == 0.0).all()


# ---------------------------------------------------------------------------
LINEAR = [
    # rows, k, q
    (1, 1, 1), (1, 64, 32), (1, 4096, 500), (2, 100, 33), (3, 1000, 700), (5, 17, 65), (8, 512, 130),
    (16, 1001, 257), (17, 128, 1000), (31, 63, 31), (33, 1000, 1001), (64, 192, 64), (65, 333, 513),
    (100, 2048, 300), (128, 65, 128), (129, 256, 129), (200, 1007, 1030), (300, 640, 777), (513, 64, 2049),
    (1030, 320, 515),
]


def _linear_inputs(rows, k, q, dtype, seed):
    g = _gen(seed)
    x = torch.randn(rows, k, generator=g) * (1.0 + 20.0 * (torch.rand(k, generator=g) < 0.02))
    w = torch.randint(-128, 128, (q, k), generator=g).to(torch.int8)
    return x.to(dtype), w, (0.5 + torch.rand(q, generator=g)) * 1e-3, torch.randn(q, generator=g)


@pytest.mark.parametrize("dtype,out", [(BF16, BF16), (F16, F32), (F32, F32), (F32, F16), (BF16, F32)])
@pytest.mark.parametrize("rows,k,q", LINEAR)
def test_linear(device, rows, k, q, dtype, out):
    log_case(f"linear {rows} {k} {q} {dtype} {out}")
    x, w, s, b = _linear_inputs(rows, k, q, dtype, rows + k + q)
    for bias in (b, None):
        want, bound = ref.product(x, w, s, bias)
        got = th.linear_i8(device, x.cuda(), w.cuda(), s.cuda(), None if bias is None else bias.cuda(), out)
        assert got.dtype == out
        ref.close(got, want, bound, "linear")


@pytest.mark.parametrize("rows,k,q,xpad,wpad,shift", [(4, 96, 200, 3, 5, 1), (40, 256, 300, 0, 16, 0), (40, 256, 300, 8, 0, 7),
                                                    (300, 512, 600, 1, 3, 2), (300, 512, 600, 0, 48, 16)])
def test_linear_strides(device, rows, k, q, xpad, wpad, shift):
    """Rows of wider buffers, weights from any byte on."""
    log_case(f"linear strides {rows} {k} {q} {xpad} {wpad} {shift}")
    x, w, s, _ = _linear_inputs(rows, k, q, BF16, 3)
    want, bound = ref.product(x, w, s)
    got = th.linear_i8(device, _strided(x, xpad, xpad), _strided(w, wpad, shift), s.cuda(), out_dtype=F32)
    ref.close(got, want, bound, "linear")


@pytest.mark.parametrize("rows", [1, 6, 40, 300])
def test_linear_special_rows(device, rows):
    """A row of zeros, rows with infinities or NaN, the largest values, the weight -128."""
    log_case(f"linear special rows {rows}")
    k, q = 200, 90
    inf, nan = float("inf"), float("nan")
    for i, v in enumerate((0.0, inf, nan, 3e38)):
        x = torch.randn(rows, k, generator=_gen(i))
        x[rows - 1] = 0.0
        x[rows - 1, 33] = v
        w = torch.full((q, k), -128, dtype=torch.int8)
        got = th.linear_i8(device, x.cuda(), w.cuda(), torch.full((q,), 1e-3, device="cuda"))
        if v == 0.0:
            assert (got[rows - 1] == 0.0).all()
        elif v == 3e38:
            assert ((got[rows - 1].double() + 128e-3 * 3e38).abs() < 4 * ref.EPS * 128e-3 * 3e38).all()
        else:
            assert got[rows - 1].isnan().all()
        assert got[:rows - 1].isfinite().all()


def test_linear_longest_sum(device):
    """127 * 128 * 131072 just fits 32 bits."""
    log_case("linear k 131072")
    x = torch.ones(2, 131072, device="cuda")
    w = torch.full((3, 131072), -128, dtype=torch.int8, device="cuda")
    got = th.linear_i8(device, x, w, torch.ones(3, device="cuda")).cpu().double()
    want = -128.0 * 131072
    assert (got - want).abs().max() <= 4 * ref.EPS * abs(want)


# ---------------------------------------------------------------------------
def _all_operators(dev, a):
    """A head's product, its next categories, and the gradient of its logits."""
    y = th.linear_i8(dev, a["x"], a["w"], a["s"])
    index, logprob = th.sample_logits(dev, y, a["u"], history=a["history"], repetition=a["rep"])
    p = th.process_logits(dev, y, history=a["history"], repetition=a["rep"], out_dtype=F32)
    loss, grad = th.distill_grad(dev, y, a["ids"], a["t"], a["wt"])
    return [y, index, logprob, p, loss, grad]


def _operator_inputs(rows, k, q):
    g = _gen(rows + k + q)
    x, w, s, _ = _linear_inputs(rows, k, q, BF16, 4)
    a = {"x": x, "w": w, "s": s, "u": torch.rand(rows, q, generator=g),
         "history": torch.randint(0, q, (rows, 50), generator=g, dtype=torch.int32),
         "rep": torch.full((rows,), 1.3), "ids": torch.randint(0, q, (rows, 9), generator=g, dtype=torch.int32),
         "t": torch.randn(rows, 9, generator=g), "wt": torch.randn(rows, generator=g)}
    return {k_: v.cuda() for k_, v in a.items()}


SIZES = [(1, 128, 20000), (3, 100, 5000), (40, 256, 700), (300, 128, 1500)]


@pytest.mark.parametrize("rows,k,q", SIZES)
def test_streams(device, rows, k, q):
    """On the device's own stream, and on one of torch's, with work queued before and
    after on the current one; the same inputs give the same bits."""
    a = _operator_inputs(rows, k, q)
    want = [t.clone() for t in _all_operators(device, a)]
    log_case(f"streams {rows} {k} {q}")
    dev = th.Device(0)
    side = torch.cuda.Stream()
    try:
        for stream in (None, side.cuda_stream, torch.cuda.current_stream().cuda_stream):
            if stream is not None:
                dev.set_stream(stream)
            late = torch.zeros_like(a["x"])
            for _ in range(20):
                late.add_(1.0)
            late.copy_(a["x"])
            got = _all_operators(dev, {**a, "x": late})
            late.zero_()
            for x, y in zip(got, want):
                assert torch.equal(x, y)
        with torch.cuda.stream(side):
            got = _all_operators(dev, a)
        side.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)
    finally:
        torch.cuda.synchronize()
        dev.close()


@pytest.mark.parametrize("rows,k,q", SIZES)
def test_graph(device, rows, k, q):
    """Captured once and replayed with other inputs, eager calls between the replays."""
    a = _operator_inputs(rows, k, q)
    dev = th.Device(0)
    side = torch.cuda.Stream()
    dev.set_stream(side.cuda_stream)
    try:
        with torch.cuda.stream(side):
            _all_operators(dev, a)
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            log_case(f"graph {rows} {k} {q}")
            with torch.cuda.graph(graph, stream=side):
                got = _all_operators(dev, a)
            for i in range(4):
                a["x"].copy_(torch.randn(a["x"].shape, generator=_gen(100 + i)).to(BF16))
                want = [t.clone() for t in _all_operators(dev, a)]
                graph.replay()
                side.synchronize()
                for x, y in zip(got, want):
                    assert torch.equal(x, y), i
    finally:
        torch.cuda.synchronize()
        dev.close()
