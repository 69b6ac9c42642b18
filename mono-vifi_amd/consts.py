"""Small constant device tensors, created once per (values, device, dtype).

``torch.tensor([...], device="cuda")`` inside a step is a pageable host-to-device copy per
call: a hidden synchronisation point in eager mode and not permitted while a HIP graph is being
captured (``Trainer --hip_graph``).  The first (eager warm-up) use creates the tensor; later
uses -- including the capture -- find it here.  Callers must not modify the result in place."""
import torch

_CACHE = {}


def device_of(device):
    """``device`` with the index that a bare "cuda" means now: what a key names has to be where its tensor is."""
    device = torch.device(device)
    return torch.device("cuda", torch.cuda.current_device()) if device.type == "cuda" and device.index is None else device


def cached(key, make):
    """The tensor ``make()`` returned the first time ``key`` came up.  An ordinary tensor also if that was under
    ``torch.inference_mode``: later calls may save it for a backward."""
    t = _CACHE.get(key)
    if t is None:
        with torch.inference_mode(False):
            t = _CACHE[key] = make()
    return t


def const_tensor(values, device, dtype=torch.float32):
    device = device_of(device)
    return cached((tuple(float(v) for v in values), str(device), dtype),
                  lambda: torch.tensor([float(v) for v in values], dtype=dtype, device=device))
