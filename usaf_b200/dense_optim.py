"""AdamW over many tensors at once, states in 32 or 8 bits, on the device.

Beside :class:`usaf_b200.sparse_optim.SparseAdam`, which steps the selected
coordinates of the experts: :class:`AdamW` steps whole tensors (norms,
embedding, routers) with decoupled weight decay, all of them in one launch per
parameter type (and count of steps, where some had no gradient at times).
:func:`adamw_step` is the step itself over tensors and state buffers that the
caller keeps.

States lie in flat buffers shared by the tensors, each tensor from a multiple
of 256 values on (:func:`state_layout`).  With 8-bit states the first moment m
and the root of the second, sqrt(v), are e4m3 values times one fp32 scale per
256 values: 2.03 bytes a value instead of 8.  Codes lie 6 to 12 % apart, more than
a late step moves a value, so from about the tenth step on a value takes the upper
of its two neighbouring codes as often as its place between them asks for (by
the step's number and the value's place in its tensor, nothing random): m and v
follow the betas in the mean, each sqrt(v) within about 25 % of its 32-bit value.

Every operation of the step is rounded by itself in fp32, in a fixed order; with
8-bit states the update's quotient may be off by one in its last place.
"""
from __future__ import annotations

from array import array
from bisect import bisect_left
from itertools import accumulate
from operator import gt
from typing import Dict, Iterable, List, Optional, Sequence, Tuple, Union

import torch

from . import _lib
from ._lib import call_on, ptr

BLOCK = 256

Packed = Tuple[torch.Tensor, torch.Tensor]


def state_layout(numels: Iterable[int]) -> Tuple[List[int], int]:
    """Where the states of tensors of these sizes start, and the size of the
    flat buffers that hold them."""
    places = list(accumulate([(int(n) + BLOCK - 1) // BLOCK * BLOCK for n in numels], initial=0))
    return places[:-1], places[-1]


def _check_flat(name: str, t: torch.Tensor, n: int, dtype: torch.dtype, index: int) -> int:
    """The address of a state buffer."""
    if t.numel() != n or t.dtype is not dtype or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name}: expected {n} contiguous {dtype} values on CUDA device {index}, got {t.numel()} "
                         f"{t.dtype} on {t.device}")
    a = t.data_ptr()
    if a % 16:
        raise ValueError(f"{name}: must start on a 16-byte boundary")
    return a


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], m: Union[torch.Tensor, Packed],
               v: Union[torch.Tensor, Packed], *, step: int, lr: float, betas: Tuple[float, float] = (0.9, 0.999),
               eps: float = 1e-8, weight_decay: Union[float, Sequence[float]] = 0.0,
               masters: Optional[torch.Tensor] = None, grad_div: float = 1.0,
               starts: Optional[Sequence[int]] = None) -> None:
    """One AdamW step in place over ``params`` (one type, contiguous) with
    ``grads`` (the parameters' type or fp32).

    ``m`` and ``v`` are flat fp32 buffers in :func:`state_layout`'s order, or
    for states in 8 bits the pairs ``(values, scales)`` of flat float8_e4m3fn
    values (of m and of sqrt(v)) and one fp32 scale per 256 of them.
    ``masters``: flat fp32 weights that the step updates and ``params`` are
    rounded from.  ``weight_decay``: one value, or one for each tensor.
    ``grad_div`` divides the gradients first.  ``starts`` gives the tensors'
    places when they are not all that the buffers hold.  A captured call repeats
    its step number: the bias corrections, and the roundings of 8-bit codes.

    Parameters, states and masters that share memory are refused; gradients
    must not lie in any of them either."""
    _launch(_checked(params, grads, m, v, step, lr, betas, eps, weight_decay, masters, grad_div, starts))


def _launch(call: Optional[tuple]) -> None:
    if call is not None:
        index, args, _, written = call
        call_on(index, "usaf_adamw", *args)
        torch.autograd.graph.increment_version(written)      # a graph that saved them finds them changed


def _checked(params, grads, m, v, step, lr, betas, eps, weight_decay, masters, grad_div, starts) -> Optional[tuple]:
    """The arguments of :func:`adamw_step`, refused or made ready: the device, the
    entry point's arguments, the host arrays that they point into and the tensors
    that the step writes (None: nothing to do)."""
    n = len(params)
    if len(grads) != n:
        raise ValueError(f"{len(grads)} gradients for {n} parameters")
    if not 1 <= step < 1 << 31:
        raise ValueError(f"step: expected 1 to 2^31 - 1, got {step}")
    if grad_div == 0:
        raise ValueError("grad_div must not be 0")
    if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1 and eps >= 0):
        raise ValueError(f"betas {betas} outside [0, 1), or eps {eps} below 0")
    eight = not isinstance(m, torch.Tensor)
    if eight == isinstance(v, torch.Tensor):
        raise TypeError("m and v: both flat tensors, or both (values, scales) pairs")
    if n == 0:
        return None
    dev, dtype, g_dtype = params[0].device, params[0].dtype, grads[0].dtype
    if g_dtype is not dtype and g_dtype is not torch.float32:
        raise TypeError(f"gradients: expected {dtype} or torch.float32, got {g_dtype}")
    ptr(params[0])      # on a CUDA device, and so are the others
    index = params[0].get_device()
    size = params[0].element_size()
    numels = list(map(torch.Tensor.numel, params))
    for i, (p, g, k) in enumerate(zip(params, grads, numels)):
        if p.dtype is not dtype or g.dtype is not g_dtype:
            raise TypeError(f"tensor {i}: {p.dtype} with a gradient of {g.dtype}, the first has {dtype} and {g_dtype}")
        if p.get_device() != index or g.get_device() != index:
            raise ValueError(f"tensor {i}: expected on {dev}")
        if g.numel() != k or not p.is_contiguous() or not g.is_contiguous():
            raise ValueError(f"tensor {i}: the parameter and a gradient of its size must be contiguous")
    at, grads_at = list(map(torch.Tensor.data_ptr, params)), list(map(torch.Tensor.data_ptr, grads))
    # apart: each one has ended where the next begins (an empty one's address is 0)
    begins, ends = sorted(at), sorted([a + k * size for a, k in zip(at, numels)])
    if any(map(gt, ends, begins[1:])):
        raise ValueError("a parameter is listed twice, or two share memory")
    if starts is None:
        places, total = state_layout(numels)
    else:
        places = [int(a) for a in starts]
        total = (m[0] if eight else m).numel()
        end = 0
        for a, k in sorted(zip(places, numels)):
            if a % BLOCK or a < end:
                end = -1
                break
            end = a + -(-k // BLOCK) * BLOCK
        if len(places) != n or not 0 <= end <= total:
            raise ValueError("starts: one multiple of 256 for each tensor, within the states, none overlapping")
    decays = [float(weight_decay)] * n if isinstance(weight_decay, (int, float)) else list(map(float, weight_decay))
    if len(decays) != n:
        raise ValueError(f"{len(decays)} weight decays for {n} parameters")
    # one host array of each, read before the call returns
    tab = (array("Q", at), array("Q", grads_at), array("q", numels), array("q", places),
           array("d", decays))
    f32, e4m3, blocks = torch.float32, torch.float8_e4m3fn, total // BLOCK
    if eight:
        (m, ms), (v, vs) = m, v
        written = [m, v, ms, vs]
        states = [_check_flat("m", m, total, e4m3, index), _check_flat("v", v, total, e4m3, index),
                  _check_flat("m scales", ms, blocks, f32, index), _check_flat("v scales", vs, blocks, f32, index)]
        sizes = [total, total, 4 * blocks, 4 * blocks]
    else:
        written = [m, v]
        states = [_check_flat("m", m, total, f32, index), _check_flat("v", v, total, f32, index), None, None]
        sizes = [4 * total, 4 * total]
    held, master_at = list(zip(states, sizes)), None
    if masters is not None:
        written.append(masters)
        master_at = _check_flat("masters", masters, total, f32, index)
        held.append((master_at, 4 * total))
    if total:
        held.sort()
        end = 0
        for a, size in held:
            i = bisect_left(begins, a + size)       # so many parameters begin below the buffer's end
            if a < end or (i and ends[i - 1] > a):
                raise ValueError("m, v, their scales and the masters must not share memory, nor with a parameter")
            end = a + size
    return index, (n, *[a.buffer_info()[0] for a in tab], _lib.dtype_code(dtype), _lib.dtype_code(g_dtype), master_at,
                   8 if eight else 32, *states, float(grad_div), int(step), float(lr), float(betas[0]), float(betas[1]),
                   float(eps)), tab, [*params, *written]


class _Group:
    """The tensors of one type and their flat states."""

    def __init__(self, names: List[str], params: List[torch.Tensor], bits: int, masters: bool):
        dev = params[0].device
        self.names = names
        self.starts, self.total = state_layout(p.numel() for p in params)
        self.place = dict(zip(names, self.starts))
        f32 = dict(dtype=torch.float32, device=dev)
        if bits == 8:
            self.m, self.v = ((torch.zeros(self.total, dtype=torch.float8_e4m3fn, device=dev),
                               torch.zeros(self.total // BLOCK, **f32)) for _ in range(2))
        else:
            self.m, self.v = torch.zeros(self.total, **f32), torch.zeros(self.total, **f32)
        self.masters = torch.zeros(self.total, **f32) if masters else None

    def parts(self, name: str, numel: int) -> Dict[str, torch.Tensor]:
        """Views of one tensor's states in the flat buffers."""
        a = self.place[name]
        b = slice(a // BLOCK, a // BLOCK + -(-numel // BLOCK))
        out = {}
        for k, t in (("m", self.m), ("v", self.v)):
            if isinstance(t, tuple):
                out[k], out[f"{k}_scale"] = t[0][a:a + numel], t[1][b]
            else:
                out[k] = t[a:a + numel]
        if self.masters is not None:
            out["master"] = self.masters[a:a + numel]
        return out


class AdamW:
    """AdamW over named tensors; the step of one call covers all of them.

    ``state_bits``: 32, or 8 for m and sqrt(v) as e4m3 values with block
    scales.  ``master_weights``: fp32 copies of 16-bit parameters, from which
    they are rounded after each step (default: for every parameter that is
    not fp32).  ``no_decay``: names that ``weight_decay`` leaves alone."""

    def __init__(self, named_params: Dict[str, torch.nn.Parameter], lr: float = 1e-4, betas: tuple = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 0.01, no_decay: Iterable[str] = (), state_bits: int = 32,
                 master_weights: bool = True):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        self.lr, self.betas, self.eps, self.weight_decay = lr, betas, eps, weight_decay
        self.state_bits = state_bits
        self._named = dict(named_params)
        self.no_decay = frozenset(no_decay)
        unknown = self.no_decay - self._named.keys()
        if unknown:
            raise ValueError(f"no_decay: no parameter named {sorted(unknown)}")
        self._step = 0                              # calls of step()
        self._steps = dict.fromkeys(self._named, 0)     # of them, those with a gradient of the parameter
        by_type: Dict[tuple, List[str]] = {}
        for name, p in self._named.items():
            if not p.is_cuda:
                raise TypeError("usaf_b200 AdamW keeps its state on the parameter's CUDA device")
            _lib.dtype_code(p.dtype)
            if not p.is_contiguous():
                raise ValueError(f"{name}: must be contiguous")
            by_type.setdefault((p.dtype, p.device), []).append(name)
        self._groups = [_Group(names, [self._named[n] for n in names], state_bits,
                               master_weights and dt != torch.float32) for (dt, _), names in by_type.items()]
        self._group_of = {n: g for g in self._groups for n in g.names}
        self.refresh_masters()

    def refresh_masters(self) -> None:
        """Take the masters from the parameters again (after loading weights)."""
        for g in self._groups:
            if g.masters is not None:
                for name in g.names:
                    p = self._named[name]
                    g.parts(name, p.numel())["master"].copy_(p.detach().reshape(-1))

    def zero_grad(self, set_to_none: bool = True):
        for p in self._named.values():
            if p.grad is not None:
                if set_to_none:
                    p.grad = None
                else:
                    p.grad.zero_()

    def step(self, grads: Optional[Dict[str, torch.Tensor]] = None, grad_div: float = 1.0):
        """One step with ``grads`` by name (default: the parameters' ``.grad``);
        a parameter without a gradient stays as it is and does not count the
        step: bias corrections follow the steps that it took.  ``grad_div`` divides
        the gradients first, as in :meth:`SparseAdam.step`.  A call that is
        refused changes nothing."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW.step counts its steps on the host; a captured one would repeat the same step")
        work = []
        for g in self._groups:
            alike: Dict[tuple, list] = {}       # one launch for each type of gradient and count of steps
            for name, start in zip(g.names, g.starts):
                p = self._named[name]
                d = p.grad if grads is None else grads.get(name)
                if d is not None:
                    alike.setdefault((d.dtype, self._steps[name]), []).append(
                        (p, d if d.is_contiguous() else d.detach().contiguous(), start,
                         0.0 if name in self.no_decay else self.weight_decay, name))
            work += [(g, taken + 1, *map(list, zip(*rows))) for (_, taken), rows in alike.items()]
        # all of them are checked before the first one moves
        calls = [_checked(params, ds, g.m, g.v, step, self.lr, self.betas, self.eps, decays, g.masters, grad_div,
                          starts) for g, step, params, ds, starts, decays, _ in work]
        for call in calls:
            _launch(call)
        for _, step, *_, names in work:
            self._steps.update(dict.fromkeys(names, step))
        self._step += 1

    def state(self, name: str) -> Dict[str, torch.Tensor]:
        """fp32 m and v of one parameter as the step reads them (and its
        master), in the parameter's shape."""
        p = self._named[name]
        s = self._group_of[name].parts(name, p.numel())
        out = {}
        for k in ("m", "v"):
            t = s[k].float()
            if self.state_bits == 8:
                t = t * s[f"{k}_scale"].repeat_interleave(BLOCK)[:t.numel()]
                t = t * t if k == "v" else t
            out[k] = t.view(p.shape)
        if "master" in s:
            out["master"] = s["master"].view(p.shape)
        return out

    def state_dict(self) -> dict:
        """CPU tensors by name; 8-bit states as their bytes and scales."""
        out: dict = {"step": self._step, "steps": dict(self._steps), "state_bits": self.state_bits}
        for name, p in self._named.items():
            for k, t in self._group_of[name].parts(name, p.numel()).items():
                t = t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
                out.setdefault(k, {})[name] = t.detach().cpu().clone()
        return out

    def load_state_dict(self, sd: dict) -> None:
        """Refuses states of another width or size (``ValueError``) before any
        of them is taken over.  Without ``steps``, every parameter took ``step``."""
        if int(sd["state_bits"]) != self.state_bits:
            raise ValueError(f"states of {sd['state_bits']} bits for an AdamW of {self.state_bits}")
        todo = []
        for name, p in self._named.items():
            for k, t in self._group_of[name].parts(name, p.numel()).items():
                new = sd.get(k, {}).get(name)
                held = t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
                if new is None or new.numel() != t.numel() or new.dtype != held.dtype:
                    raise ValueError(f"{name}: no {k} of {t.numel()} {held.dtype} values in the state")
                todo.append((held, new))
        steps = sd.get("steps", dict.fromkeys(self._named, sd["step"]))
        if not self._named.keys() <= steps.keys():
            raise ValueError(f"no count of steps of {sorted(self._named.keys() - steps.keys())} in the state")
        for held, new in todo:
            held.copy_(new.reshape(-1))
        self._step, self._steps = int(sd["step"]), {n: int(steps[n]) for n in self._named}

    @property
    def optimizer_memory_mb(self) -> float:
        n = 0
        for g in self._groups:
            for t in (*(g.m if isinstance(g.m, tuple) else (g.m,)), *(g.v if isinstance(g.v, tuple) else (g.v,)),
                      g.masters):
                n += 0 if t is None else t.numel() * t.element_size()
        return n / (1024 * 1024)
