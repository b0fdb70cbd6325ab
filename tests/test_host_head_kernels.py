"""Which kernels calls around a learned head launch, against a stand-in of the HIP runtime
(hostrun.py): the shapes of the GPU tests reach the kernels that they are meant for."""
import hostrun
import test_gpu_head_dispatch as dispatch
import test_gpu_linear_tiles as tiles
import torch
from test_host_head import P, _c_calls, _distill, _linear, _sample

CODES = {torch.float32: 1, torch.bfloat16: 2, torch.float16: 3}


def _kernel(name, dtype, *numbers):
    """A kernel of one type and numbers as the runtime names it (16-bit types: mangled)."""
    if dtype == torch.float32:
        return f"{name}<{','.join(['float', *map(str, numbers)])}>"
    return f"{len(name)}{name}I{'DF16b' if dtype == torch.bfloat16 else 'DF16_'}{''.join(f'Li{n}E' for n in numbers)}E"


def _launched(calls):
    """The names of the kernels that each call launches."""
    got = hostrun.call(_c_calls, calls)
    assert all(rc == 0 for rc, _, _ in got), got
    return [" ".join(names).replace(" ", "") for _, _, names in got]


def test_products():
    calls = [_linear(rows=rows, k=k, xs=k, w=P + shift, q=q, ws=k + pad, ys=q, n=1 << 40)
             for _, rows, q, k, pad, shift in tiles.CASES]
    for (kind, rows, q, k, pad, shift), names in zip(tiles.CASES, _launched(calls)):
        if kind == "few":
            odd = (k + pad) % 4 != 0 or shift % 4 != 0
            want = f"linear_few_kernel<float,float,0,{str(odd).lower()}>"
        else:
            want = f"linear_tile_kernel<thrml::{kind},float,{str(tiles._direct(k, pad, shift)).lower()}>"
        assert want in names, (kind, rows, q, k, pad, shift, names)


def test_samples():
    shapes = [(c, d) for c in dispatch.WIDE for d in CODES]
    calls = [_sample(dict(rows=rows, q=q, logits_stride=q, dtype=CODES[d], history=P if h else None, history_len=h,
                          history_stride=h, bias_ids=P if b else None, bias_values=P if b else None, n_bias=b,
                          bias_stride=b), us=q) for (rows, q, h, b, _), d in shapes]
    for (c, d), names in zip(shapes, _launched(calls)):
        assert _kernel("sample_kernel", d, 1024) in names and "join" not in names, (c, d, names)


def test_distillation():
    calls, wants = [], []

    def add(rows, q, k, d, *numbers, **kw):
        calls.append(_distill(rows=rows, q=q, zs=q, gs=q, k=k, ts=k, dtype=CODES[d], **kw))
        wants.append(_kernel("distill_kernel", d, *numbers))

    for d, shapes in dispatch.TWICE.items():
        for rows, q, k in shapes:
            add(rows, q, k, d, 1024, 0)
    for (rows, q, k), block in zip(dispatch.LOSS, (512, 1024, 1024)):
        for d in CODES:
            add(rows, q, k, d, block, 0, weight=None)
    for (rows, q, k), block in zip(dispatch.KEPT, (256, 512, 512, 1024, 1024)):
        add(rows, q, k, torch.bfloat16, block, 16)
    for (rows, q, k), block in zip(dispatch.KEPT, (512, 1024, 1024)):
        add(rows, q, k, torch.float32, block, 8)
    for want, names, call in zip(wants, _launched(calls), calls):
        assert want in names, (want, names, call)
