"""Array-family handling: NumPy in -> NumPy out, device tensor in -> device
tensor out (the reference's type policy, ozaki_jax/matmul.py:803-821).

Device arrays are torch CUDA tensors (the plumbing this build uses for device
memory and streams).  Staging of NumPy inputs goes through pinned host
buffers so the copies run as DMA.
"""

import numpy as np
import torch


def is_device_array(x):
    return isinstance(x, torch.Tensor)


def same_family(A, B):
    return is_device_array(A) == is_device_array(B)


def device_of(*xs):
    for x in xs:
        if is_device_array(x) and x.is_cuda:
            return x.device
    if not torch.cuda.is_available():
        raise RuntimeError("ozaki_jax_b200 needs a CUDA device; none is visible")
    return torch.device("cuda", torch.cuda.current_device())


def ndim(x):
    return x.dim() if is_device_array(x) else np.ndim(x)


def shape(x):
    return tuple(x.shape) if is_device_array(x) else np.shape(x)


def to_device_f64(x, device):
    """A contiguous float64 CUDA tensor with the values of x (copied only when
    needed)."""
    if is_device_array(x):
        t = x.to(device=device, dtype=torch.float64)
        return t.contiguous()
    a = np.ascontiguousarray(x, dtype=np.float64)
    host = torch.from_numpy(a)
    if a.nbytes >= (1 << 20) and not host.is_pinned():
        # pageable: the library's page-locked staging with host memcpy threads
        from . import _lib as L
        out = torch.empty(a.shape, dtype=torch.float64, device=device)
        with torch.cuda.device(device):
            L.check(L.load().ozk_memcpy_staged(out.data_ptr(), a.ctypes.data, a.nbytes,
                                               stream_handle(device)))
        return out
    return host.to(device, non_blocking=True)


def host_empty_f64(shape):
    """Uninitialised float64 NumPy array; page-locked (from torch's pinned host
    pool) when large, so device-to-host copies into it run as DMA."""
    n = int(np.prod(shape)) if len(shape) else 1
    if n >= (1 << 17) and torch.cuda.is_available():
        return torch.empty(tuple(shape), dtype=torch.float64, pin_memory=True).numpy()
    return np.empty(shape, dtype=np.float64)


def to_host_f64(t):
    """NumPy float64 array with the values of the CUDA tensor t (blocking)."""
    if t.numel() >= (1 << 17):
        out = torch.empty(t.shape, dtype=torch.float64, pin_memory=True)
        out.copy_(t, non_blocking=True)
        torch.cuda.current_stream(t.device).synchronize()
        return out.numpy()
    return t.cpu().numpy()


# The raw handle without a Stream object around it, where torch has the call.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_handle(device):
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


_status = {}


def status_word(device):
    """Address of the device's status word for calls that do not wait for
    their kernels: page-locked host memory that a kernel whose bounded wait
    ran out writes to.  A word that is set raises here, in the next call."""
    word = _status.get(device.index)
    if word is None:
        import ctypes

        from . import _lib as L
        address = ctypes.c_void_p()
        with on_device(device):
            L.check(L.load().ozk_status_word(ctypes.byref(address)))
        word = _status[device.index] = ctypes.c_int32.from_address(address.value)
        word.address = address.value
    if word.value:
        from . import _lib as L
        flags, word.value = word.value, 0
        raise L.OzakiError(L.OZK_ERR_TIMEOUT,
                           f"an earlier call's kernel gave up a wait (flags {flags:#x}); its "
                           "results are not valid")
    return word.address


class _Here:
    """No change of device."""

    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_HERE = _Here()


_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def on_device(device):
    """Context in which `device`, that of a CUDA tensor, is the current one."""
    if device.index == _current_device():
        return _HERE
    return torch.cuda.device(device)
