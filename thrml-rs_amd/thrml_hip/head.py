"""Operators around a learned head over q categories, on torch tensors of the
device (no counterpart in the reference):

  process_logits   penalties, biases, temperature and mask on rows of logits
  sample_logits    the same, and a category for each row with its log-probability
  distill_loss     loss of logits against a teacher's top candidates
  distill_grad     that loss, and its gradient in the logits
  linear_i8        the head's product in 8-bit integers

Every call queues its kernels on the device's stream and returns tensors.  Where
that is another stream than torch's current one, the kernels wait for what torch
has queued there, and what torch queues there afterwards waits for them.  Calls
may be captured into a graph.

torch's gradients do not go through these calls: but for distill_grad, which returns the
gradient, they refuse tensors that require one unless gradients are off.
"""
import struct

from . import _lib
from ._lib import ThrmlError, check, load

torch = None  # the module, from the first call on (the package works without it)
_TYPES = {}
_raw_stream = None  # of a device's index, torch's current stream as an address
_FLOATS = _INT32 = _FLOAT32 = _INT8 = _WORDS = ()
_PACK = struct.Struct("@PiIQqPqIPPPPPPPqIPPq").pack  # thrml_logits


def _setup():
    global torch, _raw_stream, _FLOATS, _INT32, _FLOAT32, _INT8, _WORDS
    import torch as t

    # (without the stream object that torch.cuda.current_stream makes: 1 us of a call's 11)
    _raw_stream = getattr(t._C, "_cuda_getCurrentRawStream", None) or (
        lambda index: t.cuda.current_stream(index).cuda_stream)

    _TYPES.update({t.float32: _lib.DTYPE_F32, t.bfloat16: _lib.DTYPE_BF16, t.float16: _lib.DTYPE_F16})
    _FLOATS, _INT32, _FLOAT32, _INT8 = tuple(_TYPES), (t.int32,), (t.float32,), (t.int8,)
    _WORDS = (t.int32, t.uint32)
    torch = t  # last: with it a call, from any thread, takes the rest to be there


def _refuse(msg):
    raise ThrmlError(_lib.THRML_EINVAL, msg)


# The checks read few attributes of a tensor: a call's time on the host is what small
# calls cost (each attribute is about 0.1 us).
def _matrix(name, t, dtypes, rows=None, cols=None):
    """(t, a [rows, cols] tensor, with contiguous rows; its rows' stride)"""
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
        _refuse(f"{name} must be a {' or '.join(str(d)[6:] for d in dtypes)} tensor")
    s = t.shape
    if len(s) != 2 or (rows is not None and s[0] != rows) or (cols is not None and s[1] != cols):
        _refuse(f"{name} must have shape [{'rows' if rows is None else rows}, "
                f"{'n' if cols is None else cols}], got {list(s)}")
    stride = t.stride()
    if stride[1] == 1 or s[1] <= 1:
        return t, stride[0]
    t = t.contiguous()
    return t, t.stride(0)


def _vector(name, t, n, dtypes):
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes or t.shape != (n,):
        _refuse(f"{name} must be a {str(dtypes[0])[6:]} tensor of shape [{n}]")
    return t if t.is_contiguous() else t.contiguous()


def _type(name, d):
    if d not in _TYPES:
        _refuse(f"{name} must be float32, bfloat16 or float16")
    return _TYPES[d]


def _out(name, t, rows, q, dtype):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.shape != (rows, q) or (t.stride(1) != 1 and q > 1):
        _refuse(f"{name} must be a {str(dtype)[6:]} tensor of shape [{rows}, {q}] with contiguous rows")
    return t


def _on_device(device, names, tensors, differentiable=True):
    ordinal = device.ordinal
    for t in tensors:
        if t is not None and (t.requires_grad or t.get_device() != ordinal):
            _check_tensors(ordinal, names, tensors, differentiable)
            return


def _check_tensors(ordinal, names, tensors, differentiable):
    """differentiable: torch's gradients would have to go through the call, and do not"""
    given = [(n, t) for n, t in zip(names, tensors) if t is not None]
    for name, t in given:
        if differentiable and t.requires_grad and torch.is_grad_enabled():
            _refuse(f"{name} requires a gradient, which this call does not carry on: detach it, or call under "
                    "torch.no_grad() (distill_grad gives the gradient of the logits itself)")
    for name, t in given:
        if t.get_device() != ordinal:
            _refuse(f"{name} is on {t.device}, the device is cuda:{ordinal}")


def _run(device, fn, *args):
    """fn on the device's stream, ordered with torch's current one."""
    mine = device.stream or 0
    if _raw_stream(device.ordinal) == mine:
        check(fn(device.handle, *args))
        return
    current = torch.cuda.current_stream(device.ordinal)
    stream = torch.cuda.ExternalStream(mine, device=device.ordinal)
    stream.wait_stream(current)
    check(fn(device.handle, *args))
    current.wait_stream(stream)


_ROW_NAMES = ("logits", "history", "lengths", "prompt_lengths", "repetition", "presence", "frequency", "bias_ids",
              "bias_values", "temperature", "mask")
_SAMPLE_NAMES = _ROW_NAMES + ("u",)


def _rows(logits, history, lengths, prompt_lengths, repetition, presence, frequency, bias_ids, bias_values,
          temperature, mask):
    """(the C descriptor, the tensors that it points into, rows, q)"""
    if torch is None:
        _setup()
    z, zs = _matrix("logits", logits, _FLOATS)
    rows, q = z.shape
    if q == 0:
        _refuse("logits must have at least one category")
    hp = hs = hn = lp = pp = rp = np_ = fp = bp = vp = bs = bn = tp = mp = ms = 0
    if history is not None:
        history, hs = _matrix("history", history, _INT32, rows)
        hp, hn = history.data_ptr(), history.shape[1]
        if lengths is not None:
            lengths = _vector("lengths", lengths, rows, _INT32)
            lp = lengths.data_ptr()
        if prompt_lengths is not None:
            prompt_lengths = _vector("prompt_lengths", prompt_lengths, rows, _INT32)
            pp = prompt_lengths.data_ptr()
        if repetition is not None:
            repetition = _vector("repetition", repetition, rows, _FLOAT32)
            rp = repetition.data_ptr()
        if presence is not None:
            presence = _vector("presence", presence, rows, _FLOAT32)
            np_ = presence.data_ptr()
        if frequency is not None:
            frequency = _vector("frequency", frequency, rows, _FLOAT32)
            fp = frequency.data_ptr()
    else:
        for name, t in zip(_ROW_NAMES[2:7], (lengths, prompt_lengths, repetition, presence, frequency)):
            if t is not None:
                _refuse(f"{name} needs a history")
    if bias_ids is not None and bias_values is not None:
        bias_ids, bs = _matrix("bias_ids", bias_ids, _INT32, rows)
        bn = bias_ids.shape[1]
        bias_values, vs = _matrix("bias_values", bias_values, _FLOAT32, rows, bn)
        if rows > 1 and bs != vs:
            bias_ids, bias_values, bs = bias_ids.contiguous(), bias_values.contiguous(), bn
        bp, vp = bias_ids.data_ptr(), bias_values.data_ptr()
    elif bias_ids is not None or bias_values is not None:
        _refuse("bias_ids and bias_values go together")
    if temperature is not None:
        temperature = _vector("temperature", temperature, rows, _FLOAT32)
        tp = temperature.data_ptr()
    if mask is not None:
        mask, ms = _matrix("mask", mask, _WORDS, None, (q + 31) // 32)
        n = mask.shape[0]
        if n != 1 and n != rows:
            _refuse(f"mask must have 1 or {rows} rows, got {n}")
        mp, ms = mask.data_ptr(), ms if n > 1 else 0
    d = _PACK(z.data_ptr(), _TYPES[z.dtype], q, rows, zs if rows > 1 else q, hp, hs, hn, lp, pp, rp, np_, fp,
              bp, vp, bs, bn, tp, mp, ms)
    return d, (z, history, lengths, prompt_lengths, repetition, presence, frequency, bias_ids, bias_values,
               temperature, mask), rows, q


def process_logits(device, logits, *, history=None, lengths=None, prompt_lengths=None, repetition=None,
                   presence=None, frequency=None, bias_ids=None, bias_values=None, temperature=None, mask=None,
                   out_dtype=None, out=None):
    """Processed logits [rows, q] in out_dtype (default: the logits'), the steps in
    f32 in this order, those whose argument is None left out:

      history [rows, h] int32   the categories of each row so far, the first
          lengths[row] of them (default: all), of which the first
          prompt_lengths[row] (default: none) are a prompt; entries outside
          0 .. q-1 do not count
      repetition [rows]   a category that occurs in the history: z / repetition
          where z > 0, else z * repetition
      frequency [rows]    less frequency times its occurrences after the prompt
      presence [rows]     less presence where it occurs after the prompt
      bias_ids, bias_values [rows, n]   plus the value at the category (ids
          outside 0 .. q-1 do not count; several for one category are added)
      temperature [rows]  divided by it where it is above 0
      mask [1 or rows, ceil(q / 32)] int32   -inf where bit c % 32 of word
          c // 32 is clear, whatever the logit

    out: a tensor for the result; it may be the logits themselves."""
    d, keep, rows, q = _rows(logits, history, lengths, prompt_lengths, repetition, presence, frequency, bias_ids,
                             bias_values, temperature, mask)
    z = keep[0]
    dtype = out_dtype or z.dtype
    code = _TYPES.get(dtype) or _type("out_dtype", dtype)
    stride = q
    if out is None:
        _on_device(device, _ROW_NAMES, keep)
        out = torch.empty((rows, q), dtype=dtype, device=z.device)
    else:
        if out is logits and z is not logits:
            _refuse("out may be the logits only where their rows are contiguous")
        _on_device(device, _ROW_NAMES + ("out",), keep + (_out("out", out, rows, q, dtype),))
        if rows > 1:
            stride = out.stride(0)
    _run(device, load().thrml_process_logits, d, out.data_ptr(), code, stride)
    return out


def sample_logits(device, logits, u=None, *, history=None, lengths=None, prompt_lengths=None, repetition=None,
                  presence=None, frequency=None, bias_ids=None, bias_values=None, temperature=None, mask=None):
    """(index [rows] int32, logprob [rows] float32): a category for each row from
    its processed logits x (process_logits), the first argmax of x - log(-log u)
    over the allowed ones with scores in 64 bits, u [rows, q] float32 uniforms in
    [0, 1); of x itself where u is None or the row's temperature is not above 0.
    The same inputs give the same category.  logprob is x less log sum exp x.  A
    row without a distribution (nothing allowed; a NaN or +inf among the allowed
    logits) gets index -1 and logprob NaN."""
    d, keep, rows, q = _rows(logits, history, lengths, prompt_lengths, repetition, presence, frequency, bias_ids,
                             bias_values, temperature, mask)
    us = q
    if u is not None:
        u, us = _matrix("u", u, _FLOAT32, rows, q)
    _on_device(device, _SAMPLE_NAMES, keep + (u,))
    where = keep[0].device
    index = torch.empty(rows, dtype=torch.int32, device=where)
    logprob = torch.empty(rows, dtype=torch.float32, device=where)
    lib = load()
    n = lib.thrml_sample_logits_work(device.handle, rows, q)
    work = torch.empty(n, dtype=torch.uint8, device=where) if n else None
    _run(device, lib.thrml_sample_logits, d, u.data_ptr() if u is not None else 0,
         us if rows > 1 else q, index.data_ptr(), logprob.data_ptr(),
         work.data_ptr() if n else 0, n)
    return index, logprob


def _distill(device, logits, ids, teacher, weight, tau, grad):
    """weight None: the loss alone; grad: a tensor for the gradient, or None"""
    if torch is None:
        _setup()
    z, zs = _matrix("logits", logits, _FLOATS)
    rows, q = z.shape
    if q == 0:
        _refuse("logits must have at least one category")
    ids, ids_stride = _matrix("ids", ids, _INT32, rows)
    k = ids.shape[1]
    teacher, teacher_stride = _matrix("teacher", teacher, _FLOAT32, rows, k)
    if weight is not None:
        weight = _vector("weight", weight, rows, _FLOAT32)
        if grad is not None:
            _out("out", grad, rows, q, z.dtype)
    _on_device(device, ("logits", "ids", "teacher", "weight", "out"), (z, ids, teacher, weight, grad), weight is None)
    where = z.device
    loss = torch.empty(rows, dtype=torch.float32, device=where)
    lib = load()
    dtype, n, wp, gp, gs = _TYPES[z.dtype], 0, 0, 0, q
    if weight is not None:
        if grad is None:
            grad = torch.empty((rows, q), dtype=z.dtype, device=where)
        elif rows > 1:
            gs = grad.stride(0)
        wp, gp = weight.data_ptr(), grad.data_ptr()
        n = lib.thrml_distill_work(device.handle, dtype, rows, q)
        work = torch.empty(n, dtype=torch.uint8, device=where) if n else None
    _run(device, lib.thrml_distill, z.data_ptr(), dtype, rows, q, zs if rows > 1 else q, ids.data_ptr(),
         ids_stride if rows > 1 else k, teacher.data_ptr(), teacher_stride if rows > 1 else k, k,
         float(tau), wp, loss.data_ptr(), gp, gs, work.data_ptr() if n else 0, n)
    return loss, grad


def distill_loss(device, logits, ids, teacher, tau=1.0):
    """Loss [rows] float32 of logits [rows, q] against a teacher's k top candidates:
    ids [rows, k] int32 (those outside 0 .. q-1 fill up shorter rows) with their
    logits teacher [rows, k] float32.  With p = softmax(teacher / tau) over the
    row's candidates, tau^2 sum_i p_i (log p_i - log softmax(logits / tau)[ids_i]);
    0 for a row without candidates.  k is at most 4096, tau positive, finite and not
    subnormal."""
    return _distill(device, logits, ids, teacher, None, tau, None)[0]


def distill_grad(device, logits, ids, teacher, weight, tau=1.0, out=None):
    """(loss, grad): distill_loss and the gradient of sum(weight * loss) in the
    logits, [rows, q] in their type: weight tau (softmax(logits / tau) - p), 0 in a
    row without candidates.  weight [rows] float32 carries the mean over the rows,
    what follows the loss, and a loss scale.  out: a tensor for the gradient, other
    than the logits."""
    if weight is None:
        _refuse("weight is needed")
    return _distill(device, logits, ids, teacher, weight, tau, out)


def linear_i8(device, x, w, w_scale, bias=None, out_dtype=None):
    """y [rows, q] = (a @ w.T) * s * w_scale + bias in out_dtype (default: x's): w
    [q, k] int8 weights with a scale w_scale [q] float32 for each output channel, x
    [rows, k] activations that the call quantises row by row, s = max |x| * (1 /
    127) in f32 (a subnormal s is rounded up: |a| is at most 127), a = x / s rounded to
    integers (ties to even).  The sum is exact in integers, the rest is in f32.  A row of x with an infinity or a NaN gives NaN.  k is at most
    131072."""
    if torch is None:
        _setup()
    x, xs = _matrix("x", x, _FLOATS)
    rows, k = x.shape
    w, ws = _matrix("w", w, _INT8, None, k)
    q = w.shape[0]
    if k == 0 or q == 0:
        _refuse("w must have at least one row and column")
    if w_scale is None:
        _refuse("w_scale is needed")
    w_scale = _vector("w_scale", w_scale, q, _FLOAT32)
    if bias is not None:
        bias = _vector("bias", bias, q, _FLOAT32)
    dtype = out_dtype or x.dtype
    code = _type("out_dtype", dtype)
    _on_device(device, ("x", "w", "w_scale", "bias"), (x, w, w_scale, bias))
    where = x.device
    y = torch.empty((rows, q), dtype=dtype, device=where)
    lib = load()
    n = lib.thrml_linear_i8_work(device.handle, rows, k, q)
    work = torch.empty(n, dtype=torch.uint8, device=where) if n else None
    _run(device, lib.thrml_linear_i8, x.data_ptr(), _TYPES[x.dtype], rows, k, xs if rows > 1 else k,
         w.data_ptr(), q, ws if q > 1 else k, w_scale.data_ptr(), bias.data_ptr() if bias is not None else 0,
         y.data_ptr(), code, q, work.data_ptr() if n else 0, n)
    return y
