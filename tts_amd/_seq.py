"""Argument checks shared by the sequence operators (`recurrence`, `adapters`)."""
import torch

from . import _lib

DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


# What torch.cuda.current_stream() and torch.cuda.device() wrap: a call of the smallest size is bound by the host.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_functions = {}


def call(name, device, *args):
    """The entry point `name` with `args` and the current stream of `device`, run on that device."""
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(_lib.load(), name)
    index = device.index
    if torch.cuda.current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc != _lib.OK:
        _lib.check(rc, name)


def are_tensors(what, *named):
    for name, t in named:
        if not isinstance(t, torch.Tensor):
            raise ValueError("%s: %s must be a tensor, got %s" % (what, name, type(t).__name__))


def on_device(what, *named):
    """All on one GPU, none part of an autograd graph (None stands for an argument left out)."""
    if torch.is_grad_enabled():
        for _, t in named:
            if t is not None and t.requires_grad:
                raise ValueError("%s records no autograd graph: call it under torch.no_grad(); gradients are a call of "
                                 "their own" % what)
    dev = None
    for name, t in named:
        if t is None:
            continue
        if not t.is_cuda:
            raise _lib.TtsxError("%s runs on the GPU only: %s is on %s (there is no CPU path)" % (what, name, t.device))
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError("%s: %s is on %s, the others are on %s" % (what, name, t.device, dev))
    return dev


def pointer(t):
    return None if t is None else t.data_ptr()


def rows(t, furthest=None):
    """t with a contiguous last axis; other strides stay, up to `furthest` between rows."""
    strides = t.stride()
    if (strides[-1] != 1 and t.shape[-1] > 1) or (furthest is not None and strides[-2] > furthest):
        return t.contiguous()
    return t


def lengths_on(what, lengths, B, T, device):
    """Lengths as int32 on the device.  On the device already, they are clamped there by the kernels; on the host they
    are checked here."""
    if lengths is None:
        return None
    if not isinstance(lengths, torch.Tensor):
        lengths = torch.as_tensor(lengths)
    if lengths.shape != (B,) or lengths.dtype not in (torch.int32, torch.int64):
        raise ValueError("%s: lengths must be int32 or int64 [%d], got %s %s"
                         % (what, B, lengths.dtype, tuple(lengths.shape)))
    if not lengths.is_cuda:
        if B and (int(lengths.min()) < 0 or int(lengths.max()) > T):
            raise ValueError("%s: lengths must lie in 0..%d" % (what, T))
    elif lengths.device != device:
        raise ValueError("%s: lengths is on %s, the others are on %s" % (what, lengths.device, device))
    elif lengths.dtype == torch.int32 and lengths.is_contiguous():
        return lengths
    return lengths.clamp(0, T).to(device=device, dtype=torch.int32).contiguous()


def _span(t):
    last = 1
    for n, stride in zip(t.shape, t.stride()):
        if n == 0:
            return None
        last += (n - 1) * stride
    first = t.data_ptr()
    return first, first + last * t.element_size()


def overlaps(a, b):
    """Whether the two tensors' memory ranges meet (strided tensors may interleave and still count)."""
    a, b = _span(a), _span(b)
    return a is not None and b is not None and a[0] < b[1] and b[0] < a[1]


def same_place(a, b):
    return a.data_ptr() == b.data_ptr() and a.shape == b.shape and a.stride() == b.stride()


def columns_apart(a, b):
    """Whether two [B,T,n] tensors are different columns of the same rows (slices of one buffer)."""
    if a.stride()[:2] != b.stride()[:2] or a.shape[:2] != b.shape[:2] or a.element_size() != b.element_size():
        return False
    d = (b.data_ptr() - a.data_ptr()) // a.element_size()
    first, second = (a.shape[2], b.shape[2]) if d >= 0 else (b.shape[2], a.shape[2])
    pitch = min([s for s, n in zip(a.stride()[:2], a.shape[:2]) if n > 1] or [abs(d) + second])
    return first <= abs(d) and abs(d) + second <= pitch


def writable_rows(what, name, t):
    """Refuses an output [B,T,n] whose rows are not contiguous or share memory."""
    if t.stride(2) != 1 and t.shape[2] > 1:
        raise ValueError("%s: the last axis of %s must be contiguous" % (what, name))
    need = t.shape[2]
    for stride, n in sorted((s, n) for s, n in zip(t.stride()[:2], t.shape[:2]) if n > 1):
        if stride < need:
            raise ValueError("%s: rows of %s share memory" % (what, name))
        need = stride * (n - 1) + need
