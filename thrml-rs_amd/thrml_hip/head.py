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
"""
import ctypes

from . import _lib
from ._lib import ThrmlError, check, load


def _refuse(msg):
    raise ThrmlError(_lib.THRML_EINVAL, msg)


def _types():
    import torch

    return {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


class _Call:
    """The tensors of one call: checks them, and orders the device's stream with
    torch's current one around the launches."""

    def __init__(self, device):
        import torch

        self.torch = torch
        self.device = device
        self.types = _types()
        self.where = []  # (name, tensor), to be on the device

    def floats(self, name, t):
        if not isinstance(t, self.torch.Tensor) or t.dtype not in self.types:
            _refuse(f"{name} must be a float32, bfloat16 or float16 tensor")
        return t

    def matrix(self, name, t, dtypes=None, rows=None, cols=None):
        """A [rows, cols] tensor whose rows are contiguous."""
        if dtypes is None:
            self.floats(name, t)
        elif not isinstance(t, self.torch.Tensor) or t.dtype not in dtypes:
            _refuse(f"{name} must be a {' or '.join(str(d)[6:] for d in dtypes)} tensor")
        if t.dim() != 2 or (rows is not None and t.shape[0] != rows) or (cols is not None and t.shape[1] != cols):
            _refuse(f"{name} must have shape [{'rows' if rows is None else rows}, "
                    f"{'n' if cols is None else cols}], got {list(t.shape)}")
        self.where.append((name, t))
        return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()

    def vector(self, name, t, n, dtype):
        if t is None:
            return None
        if not isinstance(t, self.torch.Tensor) or t.dtype != dtype or t.dim() != 1 or t.shape[0] != n:
            _refuse(f"{name} must be a {str(dtype)[6:]} tensor of shape [{n}]")
        self.where.append((name, t))
        return t.contiguous()

    def dtype(self, name, d):
        if d not in self.types:
            _refuse(f"{name} must be float32, bfloat16 or float16")
        return self.types[d]

    def out(self, name, t, rows, q, dtype, like):
        if t is None:
            return self.torch.empty(rows, q, dtype=dtype, device=like.device)
        if not isinstance(t, self.torch.Tensor) or t.dtype != dtype or tuple(t.shape) != (rows, q) or (
                t.stride(1) != 1 and q > 1):
            _refuse(f"{name} must be a {str(dtype)[6:]} tensor of shape [{rows}, {q}] with contiguous rows")
        self.where.append((name, t))
        return t

    def work(self, n, like):
        return self.torch.empty(n, dtype=self.torch.uint8, device=like.device) if n else None

    def on_device(self):
        for name, t in self.where:
            if t.device.type != "cuda" or t.device.index != self.device.ordinal:
                _refuse(f"{name} is on {t.device}, the device is cuda:{self.device.ordinal}")

    def run(self, fn, *args):
        torch = self.torch
        mine = self.device.stream or 0
        current = torch.cuda.current_stream(self.device.ordinal)
        if current.cuda_stream == mine:
            check(fn(self.device.handle, *args))
            return
        stream = torch.cuda.ExternalStream(mine, device=self.device.ordinal)
        stream.wait_stream(current)
        check(fn(self.device.handle, *args))
        current.wait_stream(stream)


def _stride(t):
    return t.stride(0) if t is not None and t.shape[0] > 1 else (t.shape[1] if t is not None else 0)


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _rows(call, logits, history, lengths, prompt_lengths, repetition, presence, frequency, bias_ids, bias_values,
          temperature, mask):
    """(the C descriptor, the tensors that it points into)"""
    torch = call.torch
    logits = call.matrix("logits", logits)
    rows, q = logits.shape
    if q == 0:
        _refuse("logits must have at least one category")
    i32, f32 = (torch.int32,), (torch.float32,)
    if history is None:
        for name, t in (("lengths", lengths), ("prompt_lengths", prompt_lengths), ("repetition", repetition),
                        ("presence", presence), ("frequency", frequency)):
            if t is not None:
                _refuse(f"{name} needs a history")
    else:
        history = call.matrix("history", history, i32, rows)
    if (bias_ids is None) != (bias_values is None):
        _refuse("bias_ids and bias_values go together")
    if bias_ids is not None:
        bias_ids = call.matrix("bias_ids", bias_ids, i32, rows)
        n = bias_ids.shape[1]
        bias_values = call.matrix("bias_values", bias_values, f32, rows, n)
        if rows > 1 and bias_ids.stride(0) != bias_values.stride(0):
            bias_ids, bias_values = bias_ids.contiguous(), bias_values.contiguous()
    if mask is not None:
        words = (q + 31) // 32
        mask = call.matrix("mask", mask, (torch.int32, getattr(torch, "uint32", torch.int32)), None, words)
        if mask.shape[0] not in (1, rows):
            _refuse(f"mask must have 1 or {rows} rows, got {mask.shape[0]}")
    vec = {name: call.vector(name, t, rows, dtype) for name, t, dtype in (
        ("lengths", lengths, torch.int32), ("prompt_lengths", prompt_lengths, torch.int32),
        ("repetition", repetition, torch.float32), ("presence", presence, torch.float32),
        ("frequency", frequency, torch.float32), ("temperature", temperature, torch.float32))}
    d = _lib.Logits(
        _ptr(logits), call.types[logits.dtype], q, rows, _stride(logits), _ptr(history), _stride(history),
        history.shape[1] if history is not None else 0, _ptr(vec["lengths"]), _ptr(vec["prompt_lengths"]),
        _ptr(vec["repetition"]), _ptr(vec["presence"]), _ptr(vec["frequency"]), _ptr(bias_ids), _ptr(bias_values),
        _stride(bias_ids), bias_ids.shape[1] if bias_ids is not None else 0, _ptr(vec["temperature"]), _ptr(mask),
        _stride(mask) if mask is not None and mask.shape[0] > 1 else 0)
    return d, logits, (logits, history, bias_ids, bias_values, mask, vec)


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
    call = _Call(device)
    d, z, keep = _rows(call, logits, history, lengths, prompt_lengths, repetition, presence, frequency, bias_ids,
                       bias_values, temperature, mask)
    dt = call.dtype("out_dtype", out_dtype or z.dtype)
    if out is logits and z is not logits:
        _refuse("out may be the logits only where their rows are contiguous")
    out = call.out("out", out, d.rows, d.q, out_dtype or z.dtype, z)
    call.on_device()
    call.run(load().thrml_process_logits, ctypes.byref(d), out.data_ptr(), dt, _stride(out))
    del keep
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
    call = _Call(device)
    torch = call.torch
    d, z, keep = _rows(call, logits, history, lengths, prompt_lengths, repetition, presence, frequency, bias_ids,
                       bias_values, temperature, mask)
    if u is not None:
        u = call.matrix("u", u, (torch.float32,), d.rows, d.q)
    call.on_device()
    index = torch.empty(d.rows, dtype=torch.int32, device=z.device)
    logprob = torch.empty(d.rows, dtype=torch.float32, device=z.device)
    lib = load()
    n = lib.thrml_sample_logits_work(device.handle, d.rows, d.q)
    work = call.work(n, z)
    call.run(lib.thrml_sample_logits, ctypes.byref(d), _ptr(u), _stride(u), index.data_ptr(), logprob.data_ptr(),
             _ptr(work), n)
    del keep
    return index, logprob


def _distill(device, logits, ids, teacher, weight, tau, out):
    call = _Call(device)
    torch = call.torch
    z = call.matrix("logits", logits)
    rows, q = z.shape
    if q == 0:
        _refuse("logits must have at least one category")
    ids = call.matrix("ids", ids, (torch.int32,), rows)
    teacher = call.matrix("teacher", teacher, (torch.float32,), rows, ids.shape[1])
    grad = None
    if weight is not None:
        weight = call.vector("weight", weight, rows, torch.float32)
        grad = call.out("out", out, rows, q, z.dtype, z)
    call.on_device()
    loss = torch.empty(rows, dtype=torch.float32, device=z.device)
    lib = load()
    n = lib.thrml_distill_work(device.handle, rows, q, ids.shape[1])
    work = call.work(n, z)
    call.run(lib.thrml_distill, _ptr(z), call.types[z.dtype], rows, q, _stride(z), _ptr(ids), _stride(ids),
             _ptr(teacher), _stride(teacher), ids.shape[1], float(tau), _ptr(weight), _ptr(loss), _ptr(grad),
             _stride(grad), _ptr(work), n)
    return loss, grad


def distill_loss(device, logits, ids, teacher, tau=1.0):
    """Loss [rows] float32 of logits [rows, q] against a teacher's k top candidates:
    ids [rows, k] int32 (those outside 0 .. q-1 fill up shorter rows) with their
    logits teacher [rows, k] float32.  With p = softmax(teacher / tau) over the
    row's candidates, tau^2 sum_i p_i (log p_i - log softmax(logits / tau)[ids_i]);
    0 for a row without candidates.  k is at most 4096."""
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
    [rows, k] activations that the call quantises row by row, s = max |x| / 127, a
    = x / s rounded to integers (ties to even).  The sum is exact in integers, the
    rest is in f32.  A row of x with an infinity or a NaN gives NaN.  k is at most
    131072."""
    call = _Call(device)
    torch = call.torch
    x = call.matrix("x", x)
    rows, k = x.shape
    w = call.matrix("w", w, (torch.int8,), None, k)
    q = w.shape[0]
    if k == 0 or q == 0:
        _refuse("w must have at least one row and column")
    w_scale = call.vector("w_scale", w_scale, q, torch.float32)
    if w_scale is None:
        _refuse("w_scale is needed")
    bias = call.vector("bias", bias, q, torch.float32)
    dt = call.dtype("out_dtype", out_dtype or x.dtype)
    call.on_device()
    y = torch.empty(rows, q, dtype=out_dtype or x.dtype, device=x.device)
    lib = load()
    n = lib.thrml_linear_i8_work(device.handle, rows, k, q)
    work = call.work(n, x)
    call.run(lib.thrml_linear_i8, _ptr(x), call.types[x.dtype], rows, k, _stride(x), _ptr(w), q, _stride(w),
             _ptr(w_scale), _ptr(bias), _ptr(y), dt, _stride(y), _ptr(work), n)
    return y
