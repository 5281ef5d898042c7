"""AdamW over many tensors at once, the updater of the full-vocabulary training path.

The moments are held in fp32 or in 8 bits (codes of one byte, one scale for 256 elements); one
kernel launch reads and writes every tensor once.  PyTorch supplies memory and streams only.
"""
from __future__ import annotations

import ctypes as C
import dataclasses
import warnings
from array import array
from bisect import bisect_right

import torch

from . import _lib
from .cumach import cuda_error_string

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def check(err: int, what: str):
    if err:
        raise RuntimeError(f"{what} error " + ("1: arguments refused" if err == 1 else cuda_error_string(err)))


class on_device:
    """Makes ``device`` current, at no cost where it is already."""

    def __init__(self, device: torch.device):
        self._guard = None if torch.cuda.current_device() == device.index else torch.cuda.device(device)

    def __enter__(self):
        if self._guard is not None:
            self._guard.__enter__()

    def __exit__(self, *exc):
        if self._guard is not None:
            self._guard.__exit__(*exc)


def stream_of(device: torch.device) -> int:
    """Handle of the device's current stream."""
    return _raw_stream(device.index)


# the handle without a Stream object around it, where torch offers that
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


@dataclasses.dataclass
class Opts:
    """``lrate`` and the usual constants; ``bits``: 32 or 8 for the moments.

    ``rounding`` of 8-bit moments: ``"random"``, for training, rounds a code up or down so that the stored moments
    are right in the mean (random bits from ``seed``, the step and the element: equal runs give equal
    bits).  ``"nearest"`` is for a few steps, or for comparing with one: the codes of sqrt(v) are 3 to 6 %
    apart and a step with ``beta2`` 0.999 lowers it by 0.05 %, so a moment rounded to nearest never falls and
    hardly rises.  None is ``"nearest"`` with a warning.  Either way 8 bits span 16 octaves: beside the largest of its
    256 elements, an ``m`` below 2^-16 is held as zero and a sqrt(v) as the smallest code."""
    lrate: float = 1e-3
    beta1: float = 0.9
    beta2: float = 0.999
    eps: float = 1e-8
    wdecay: float = 0.01
    bits: int = 32
    rounding: str | None = None
    seed: int = 0


class AdamW:
    """``step(grads)`` applies, to every tensor of ``params`` in place,

        m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2,
        p = p (1 - lrate wdecay) - lrate m / (1 - beta1^t) / (sqrt(v / (1 - beta2^t)) + eps)

    ``params``: contiguous CUDA tensors of one device, fp32, bf16 or fp16, none overlapping another.
    ``state``, when given, is the state to go on from (its tensors are used in place): ``t`` steps
    done, and lists ``m`` and ``v`` like the parameters: fp32, or for 8 bits uint8 of as many
    elements, with lists ``mscale`` and ``vscale`` of fp32, one for every 256 elements, none overlapping
    another or a parameter.  Without it
    the moments start at zero.  The arithmetic is fp32; a 16-bit parameter is rounded to nearest
    once a step, so a step smaller than half of its last place leaves it as it is.

    A parameter may be given other memory between steps (``p.data = ...``); a captured step keeps the addresses
    that it was captured with.

    The step count lives on the device: a captured step counts its replays."""

    Opts = Opts

    def __init__(self, params, opts: Opts | None = None, state: dict | None = None):
        self.params = list(params)
        self.opts = opts or Opts()
        o = self.opts
        if o.bits not in (8, 32):
            raise ValueError("bits must be 32 or 8")
        if not (0 <= o.beta1 < 1 and 0 <= o.beta2 < 1 and o.eps > 0 and o.wdecay >= 0):
            raise ValueError("need 0 <= beta1, beta2 < 1, eps > 0, wdecay >= 0")
        if o.rounding not in (None, "nearest", "random"):
            raise ValueError("rounding is 'random' or 'nearest'")
        if o.bits == 8 and o.rounding is None:
            warnings.warn("8-bit moments rounded to nearest do not follow their gradients over many steps: "
                          "give rounding='random' for training, or 'nearest'", stacklevel=2)
        if not self.params:
            raise ValueError("AdamW needs at least one tensor")
        self._check_params()
        self.device = self.params[0].device
        if any(p.device != self.device for p in self.params):
            raise ValueError("parameters on more than one device")
        self.m, self.v, self.mscale, self.vscale, t = self._state(state)
        n = len(self.params)
        self._sizes = [p.numel() for p in self.params]
        self._types = [p.dtype for p in self.params]
        self._pointers = C.c_void_p * n
        self._kinds = (C.c_int * n)(*[TYPES[t] for t in self._types])
        self._table = (_lib.W2VAdamwTensor * n)()
        self._fill()
        self._clock = torch.zeros(4, dtype=torch.float64, device=self.device)
        self._clock_at = self._clock.data_ptr()
        with on_device(self.device):
            check(_lib.load().w2v_adamw_clock(self._clock_at, o.beta1, o.beta2, t, stream_of(self.device)),
                  "w2v_adamw_clock")

    def _check_params(self):
        for p in self.params:
            if not isinstance(p, torch.Tensor) or p.dtype not in TYPES:
                raise ValueError("parameters are fp32, bf16 or fp16 tensors")
            if not p.is_contiguous():
                raise ValueError("parameters have to be contiguous")
        self._apart(self.params, "two parameters overlap")
        if any(not p.is_cuda for p in self.params):
            raise ValueError("AdamW expects CUDA tensors")

    def _fill(self):
        """The table of addresses.  Aliases of the parameters are kept beside it, so that the memory it names
        stays theirs until it is filled again."""
        spans = self._apart([*self.params, *self.m, *self.v, *(self.mscale or ()), *(self.vscale or ())],
                            "a tensor of the state overlaps another or a parameter")
        self._held = [p.detach() for p in self.params]
        self._begins, self._ends = [a for a, _ in spans], [b for _, b in spans]
        self._seen = set()      # addresses that have passed `_foreign`
        self._at = list(map(torch.Tensor.data_ptr, self.params))
        for i, p in enumerate(self.params):
            self._table[i] = _lib.W2VAdamwTensor(
                self._at[i], self.m[i].data_ptr(), self.v[i].data_ptr(),
                self.mscale[i].data_ptr() if self.mscale else 0, self.vscale[i].data_ptr() if self.vscale else 0,
                self._sizes[i], TYPES[p.dtype])

    def _foreign(self, tensors, key, what):
        """Refuses tensors that share memory with a parameter or the state.  `key` is what the answer hangs on,
        the tensors' addresses and types: those that have passed need no second look."""
        if key in self._seen:
            return
        for x in tensors:
            a, n = x.data_ptr(), x.numel()
            i = bisect_right(self._begins, a)
            if n and (i and self._ends[i - 1] > a or i < len(self._begins) and self._begins[i] < a + n * x.element_size()):
                raise ValueError(what)
        if len(self._seen) >= 64:
            self._seen.clear()
        self._seen.add(key)

    def _moved(self):
        """Parameters whose memory is another now (``p.data = ...``, ``p.set_``, ``p.resize_``)."""
        self._check_params()
        if list(map(torch.Tensor.numel, self.params)) != self._sizes or [p.dtype for p in self.params] != self._types \
                or any(p.device != self.device for p in self.params):
            raise ValueError("a parameter has changed its size, type or device")
        self._fill()

    def _state(self, state):
        bits = self.opts.bits
        dtype = torch.float32 if bits == 32 else torch.uint8
        blocks = [(p.numel() + 255) // 256 for p in self.params]

        def fresh(sizes, dt):
            return [torch.zeros(n, dtype=dt, device=self.device) for n in sizes]

        sizes = [p.numel() for p in self.params]
        if state is None:
            scales = (fresh(blocks, torch.float32), fresh(blocks, torch.float32)) if bits == 8 else (None, None)
            return fresh(sizes, dtype), fresh(sizes, dtype), *scales, 0

        def given(name, want, dt):
            got = list(state[name])
            if len(got) != len(want):
                raise ValueError(f"state[{name!r}] has {len(got)} tensors for {len(want)} parameters")
            for x, n in zip(got, want):
                if x.dtype != dt or x.numel() != n or x.device != self.device or not x.is_contiguous():
                    raise ValueError(f"state[{name!r}] wants contiguous {dt} tensors of {self.device}, "
                                     "as many elements as it describes")
            return [x.detach() for x in got]      # aliases of our own: they stay where the state is now

        if int(state["t"]) < 0:
            raise ValueError("state['t'] is negative")
        scales = (given("mscale", blocks, torch.float32), given("vscale", blocks, torch.float32)) if bits == 8 \
            else (None, None)
        return given("m", sizes, dtype), given("v", sizes, dtype), *scales, int(state["t"])

    @staticmethod
    def _apart(tensors, what):
        """Refuses tensors that share memory; returns the begin and end of each, in order."""
        spans = sorted((at, at + n * x.element_size()) for x in tensors if (n := x.numel()) for at in (x.data_ptr(),))
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError(what)
        return spans

    def _like(self, tensors, sizes, what):
        """Refuses tensors that are not contiguous ones of this device and these sizes (in few passes:
        a model may have hundreds)."""
        if list(map(torch.Tensor.numel, tensors)) != sizes or not all(map(torch.Tensor.is_contiguous, tensors)) \
                or set(map(torch.Tensor.get_device, tensors)) != {self.device.index}:
            raise ValueError(what)

    def step(self, grads, lrate: "float | torch.Tensor | None" = None):
        """One step.  ``grads``: a tensor for each parameter, same number of elements, contiguous, fp32
        or the parameter's type, in memory of its own (one tensor may serve several parameters).
        ``lrate`` replaces the option's: a number, or a one-element fp32 tensor of the device, read when
        the step runs."""
        n = len(self._sizes)
        if len(grads) != n:
            raise ValueError(f"{len(grads)} gradients for {n} parameters")
        dev = self.device
        if list(map(torch.Tensor.data_ptr, self.params)) != self._at:
            self._moved()
        self._like(grads, self._sizes, "a gradient has its parameter's device and size and is contiguous")
        types = [g.dtype for g in grads]
        if types == self._types:
            kinds = self._kinds
        elif all(t is torch.float32 or t is p for t, p in zip(types, self._types)):
            kinds = (C.c_int * n)(*[TYPES[t] for t in types])
        else:
            raise ValueError("a gradient is fp32 or of its parameter's type")
        o = self.opts
        rate, rate_ptr = o.lrate, None
        if isinstance(lrate, torch.Tensor):
            if lrate.dtype != torch.float32 or lrate.numel() != 1 or lrate.device != dev:
                raise ValueError("lrate: a number or a one-element fp32 tensor of the parameters' device")
            rate_ptr = lrate.data_ptr()
        elif lrate is not None:
            rate = float(lrate)
        at = array("Q", map(torch.Tensor.data_ptr, grads))
        self._foreign(grads, (at.tobytes(), bytes(kinds)), "a gradient shares memory with a parameter or the state")
        opts = _lib.W2VAdamwOpts(rate, o.beta1, o.beta2, o.eps, o.wdecay)
        with on_device(dev):
            pointers = self._pointers.from_buffer(at)
            if o.bits == 8 and o.rounding == "random":
                check(_lib.load().w2v_adamw_step_random(self._table, pointers, kinds, n, C.byref(opts), rate_ptr,
                                                        o.seed & (2 ** 64 - 1), self._clock_at, stream_of(dev)),
                      "w2v_adamw_step_random")
            else:
                check(_lib.load().w2v_adamw_step(self._table, pointers, kinds, n, o.bits, C.byref(opts), rate_ptr,
                                                 self._clock_at, stream_of(dev)), "w2v_adamw_step")

    def moments(self, mout=None, vout=None):
        """Both moments as fp32 values: lists (m, v).  With 32 bits these are the state itself; with 8
        the codes are decoded into new tensors or into the lists ``mout`` and ``vout``, whose tensors
        overlap neither each other nor the state nor a parameter."""
        if self.opts.bits == 32:
            if mout is not None or vout is not None:
                raise ValueError("32-bit moments are not copied: mout and vout are for 8 bits")
            return self.m, self.v
        if list(map(torch.Tensor.data_ptr, self.params)) != self._at:
            self._moved()
        n = len(self._sizes)
        if mout is None:
            mout = [torch.empty(k, dtype=torch.float32, device=self.device) for k in self._sizes]
        if vout is None:
            vout = [torch.empty(k, dtype=torch.float32, device=self.device) for k in self._sizes]
        if len(mout) != n or len(vout) != n:
            raise ValueError("mout and vout have a tensor for each parameter")
        dev = self.device
        what = "mout and vout: contiguous fp32 tensors of the parameters' device and sizes"
        both = [*mout, *vout]
        self._like(both, self._sizes * 2, what)
        if any(x.dtype is not torch.float32 for x in both):
            raise ValueError(what)
        at = array("Q", map(torch.Tensor.data_ptr, both))
        key = at.tobytes()
        if key not in self._seen:
            self._apart(both, "two tensors of mout and vout overlap")
            self._foreign(both, key, "mout or vout shares memory with a parameter or the state")
        with on_device(dev):
            check(_lib.load().w2v_adamw_moments(self._table, self._pointers.from_buffer(at),
                                                self._pointers.from_buffer(at, 8 * n), n, stream_of(dev)),
                  "w2v_adamw_moments")
        return mout, vout
