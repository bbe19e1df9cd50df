"""Gradient clip + Adam step with true weight decay for a model with flat parameters, as two launches (vc_clip_adamw).

Reference: tools/train_utils/train_utils.py:50-51 runs ``clip_grad_norm_(model.parameters(), GRAD_NORM_CLIP)`` and then
``optimizer.step()``; the optimizer (tools/train_utils/optimization/__init__.py:19-32, ``adam_onecycle``) is torch Adam with betas
(0.9, 0.99) inside fastai's ``OptimWrapper`` with ``true_wd=True, bn_wd=True``, whose step (fastai_optim.py:132-149) multiplies every
parameter by ``1 - wd * lr`` and then runs Adam without weight decay -- the arithmetic of ``torch.optim.AdamW``.

``ClipAdamW`` is a ``torch.optim.Optimizer``: ``param_groups[0]["lr"]`` / ``["betas"]`` are read at every step, so a one-cycle scheduler
that rewrites them per iteration (fastai's ``OneCycle``, ``torch.optim.lr_scheduler.OneCycleLR``) drives it unchanged, and its state
(``step``, ``exp_avg``, ``exp_avg_sq`` per parameter) has the keys and shapes of ``torch.optim.AdamW``'s, so optimizer checkpoints move
between the two.  It wants what ``feature_pass.flatten_parameters`` returns: a few contiguous fp32 tensors on the GPU (at most 16).
There is no CPU path: without the HIP library the constructor raises.

``AdamW`` takes a model as it is -- any number of fp32, fp16 or bf16 parameters, any number of groups -- and keeps the moments in 32 or in
8 bits (vc_adamw): one launch per 88 or 76 tensors, no clip inside.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import _lib, ops

from ._lib import ADAM_MAX_TENSORS as MAX_TENSORS, AdamTensor


_written = torch.autograd.graph.increment_version
"""Memory that a kernel wrote through a pointer: autograd's saved tensors, and caches keyed on a version (SparseBEVStem's packed weight), see it by that."""


def supports(params) -> bool:
    """Can ClipAdamW take this parameter list?  (a few contiguous fp32 CUDA tensors: the flat parameters of a flattened model)"""
    params = list(params)
    return (0 < len(params) <= MAX_TENSORS and all(p.is_cuda and p.dtype == torch.float32 and p.is_contiguous() for p in params)
            and len({p.device for p in params}) == 1)


class ClipAdamW(torch.optim.Optimizer):
    """``clip_grad_norm_(params, max_norm)`` + ``AdamW.step()`` in two kernel launches.  One parameter group.

    ``step()`` returns the total gradient norm (0-dim tensor on the device, what ``clip_grad_norm_`` returns) without a host read.
    ``max_norm`` None or <= 0: no clipping.  ``scale_grads=True`` also leaves the clipped gradients in ``.grad`` as
    ``clip_grad_norm_`` does (nothing on the training path reads them, so the default skips that write)."""

    clips = True   # a training loop that sees this attribute skips its own clip_grad_norm_ (bench.train_step)

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.01, max_norm=10.0, scale_grads=False):
        defaults = dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, max_norm=max_norm, scale_grads=scale_grads)
        super().__init__(params, defaults)
        if len(self.param_groups) != 1:
            raise ValueError("ClipAdamW: one parameter group (the clip is over all parameters at once)")
        ps = self.param_groups[0]["params"]
        if not supports(ps):
            raise ValueError(f"ClipAdamW: wants 1..{MAX_TENSORS} contiguous float32 CUDA tensors on one device "
                             f"(feature_pass.flatten_parameters(model)), got {len(ps)} parameter(s)")
        self._lib = ops.get_backend().lib    # raises without libvirconv_hip.so
        self._device = ps[0].device
        if self._device.index is None:
            self._device = torch.device("cuda", torch.cuda.current_device())
        self._ws = None
        self._norm = None

    def _state_of(self, p):
        st = self.state[p]
        if not st:
            st["step"] = torch.tensor(0.0, dtype=torch.float32)          # as torch.optim.AdamW keeps it (capturable=False)
            st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
            st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
        return st

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        g = self.param_groups[0]
        live = [p for p in g["params"] if p.grad is not None]
        arr = (AdamTensor * MAX_TENSORS)()
        steps = set()
        for i, p in enumerate(live):
            grad = p.grad
            if grad.dtype != torch.float32 or not grad.is_contiguous() or grad.is_sparse or grad.device != p.device:
                raise ValueError("ClipAdamW: gradients must be dense contiguous float32 tensors on the parameter's device")
            st = self._state_of(p)
            if not torch.is_tensor(st["step"]):            # a checkpoint of an old torch: a Python number
                st["step"] = torch.tensor(float(st["step"]), dtype=torch.float32)
            elif st["step"].is_cuda:                       # a checkpoint of torch.optim.AdamW(fused=True): the counter lives on the device there;
                st["step"] = st["step"].cpu()              # here the host needs it (one read, once)
            st["step"] += 1
            steps.add(int(st["step"]))
            arr[i] = AdamTensor(p.data_ptr(), grad.data_ptr(), st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr(), p.numel())
        if self._norm is None:
            self._norm = torch.zeros((), dtype=torch.float32, device=self._device)
        if not live:
            self._norm.zero_()
            return self._norm if loss is None else loss
        if len(steps) != 1:
            raise ValueError(f"ClipAdamW: the parameters are at different steps {sorted(steps)} (one bias correction per call)")
        n_ws = self._lib.vc_clip_adamw_workspace_bytes(len(live))
        if self._ws is None or self._ws.numel() < n_ws:
            self._ws = torch.empty((n_ws,), dtype=torch.uint8, device=self._device)
        max_norm = g["max_norm"]
        b1, b2 = g["betas"]
        _lib.check(self._lib.vc_clip_adamw(C.cast(arr, C.c_void_p), len(live), float(g["lr"]), float(b1), float(b2), float(g["eps"]),
                                           float(g["weight_decay"]), steps.pop(), float(max_norm) if max_norm else 0.0,
                                           int(bool(g["scale_grads"])), self._norm.data_ptr(), self._ws.data_ptr(), n_ws,
                                           torch._C._cuda_getCurrentRawStream(self._device.index)), "vc_clip_adamw")
        _written([self._norm, *live, *(self.state[p][k] for p in live for k in ("exp_avg", "exp_avg_sq")),
                  *((p.grad for p in live) if g["scale_grads"] else ())])
        return self._norm if loss is None else loss

    @property
    def total_norm(self):
        """The gradient norm of the last step (device tensor; None before the first step)."""
        return self._norm


STATE_BLOCK = 128    # elements that share an exponent in the 8-bit states


def _dense(t: torch.Tensor) -> bool:
    """Do the elements of t fill one stretch of memory, each once (in any order of its axes)?"""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != want:
            return False
        want *= size
    return True


def _order(t: torch.Tensor):
    """What tells the order of t's elements in memory: the strides of its axes, those of one element apart."""
    return [s for s, n in zip(t.stride(), t.shape) if n != 1]


def _decode(codes: torch.Tensor, exponents: torch.Tensor) -> torch.Tensor:
    """The values of an 8-bit moment, fp32, of its shape and order in memory."""
    n = codes.numel()
    scale = torch.exp2(exponents.float() - 7).repeat_interleave(STATE_BLOCK, 0)[:n]
    out = torch.empty_like(codes, dtype=torch.float32, memory_format=torch.preserve_format)
    torch.as_strided(out, (n,), (1,)).copy_(torch.as_strided(codes.view(torch.uint8), (n,), (1,)).view(torch.float8_e4m3fn).float() * scale)
    return out


class AdamW(torch.optim.Optimizer):
    """AdamW (torch.optim.AdamW's arithmetic: true weight decay, bias correction) over all parameters of a group in a few launches.

    Parameters: fp32, fp16 or bf16 tensors on one GPU, dense in any order of their axes; gradients of the same type.  The step computes in
    fp32 and rounds a parameter once.  ``state_bits=32``: the moments are fp32, with the keys and shapes of torch.optim.AdamW's state (a
    checkpoint of either loads into the other, unless it asks for amsgrad or maximize).  ``state_bits=8``: 2 bytes an element instead of 8 -- ``exp_avg`` and ``exp_avg_rms`` (the
    square root of the second moment) are float8_e4m3fn values over a power of two for every 128 elements (``exponents``, int8), rounded up or
    down at random in proportion so that a moment follows changes smaller than its resolution.  The second moment gains the rounding's variance
    by it: under steady gradients it settles about 4 per cent (3 to 6) above its 32-bit value, so steps are 1 to 2 per cent shorter.  The
    random numbers follow from ``seed``, the step and the element's place: a run repeats, and resumes from a checkpoint, bit for bit.
    ``decoded_state(p)`` gives the moments as fp32 tensors.  The 128 elements of an exponent are neighbours in memory, so a checkpoint has to
    keep its tensors' strides (torch.save does); loaded into a parameter of another order of its axes the moments are rounded once more, to
    the nearest.  A step counts on the host, so it cannot be captured into a graph."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.01, state_bits=32, seed=0):
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: states in {state_bits} bits (8 or 32)")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))
        self.state_bits, self.seed = int(state_bits), int(seed)
        self._attach()
        for g in self.param_groups:
            self._check_group(g)

    def __setstate__(self, state):
        super().__setstate__(state)
        self._attach()

    def _attach(self):
        be = ops.get_backend()               # raises without libvirconv_hip.so
        self._lib, self._host = be.lib, be.host
        self._order, self._lists = [], {}

    def __getstate__(self):
        return {**super().__getstate__(), "state_bits": self.state_bits, "seed": self.seed}

    def add_param_group(self, group):
        super().add_param_group(group)
        if hasattr(self, "_lib"):
            self._check_group(self.param_groups[-1])

    def _check_group(self, g):
        b1, b2 = g["betas"]
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"AdamW: betas {g['betas']} outside [0, 1)")
        if not (g["lr"] >= 0.0 and g["eps"] >= 0.0 and g["weight_decay"] >= 0.0):
            raise ValueError(f"AdamW: lr {g['lr']}, eps {g['eps']}, weight_decay {g['weight_decay']} have to be 0 or more")
        device = next((p.device for group in self.param_groups for p in group["params"]), None)
        for p in g["params"]:
            if not p.is_cuda or p.device != device:
                raise ValueError(f"AdamW: parameters have to be on one GPU, got {p.device} beside {device} (there is no CPU path)")
            if p.dtype not in _PARAM_DTYPES or not _dense(p):
                raise ValueError(f"AdamW: wants dense float32, float16 or bfloat16 parameters, got {p.dtype} of strides {p.stride()}")

    def _new_state(self, p):
        st = self.state[p]
        st["step"] = 0
        if self.state_bits == 32:
            st["exp_avg"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
            st["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
        else:
            zero = torch.zeros_like(p, dtype=torch.uint8, memory_format=torch.preserve_format)
            st["exp_avg"], st["exp_avg_rms"] = zero.view(torch.float8_e4m3fn), zero.clone().view(torch.float8_e4m3fn)
            st["exponents"] = torch.zeros((-(-p.numel() // STATE_BLOCK), 2), dtype=torch.int8, device=p.device)
        return st

    def _check_state(self, p, st):
        """The state's tensors as the kernel takes them: types, sizes, order of elements and device (what a checkpoint may have changed)."""
        second, dtype = ("exp_avg_sq", torch.float32) if self.state_bits == 32 else ("exp_avg_rms", torch.float8_e4m3fn)
        if second not in st or (self.state_bits == 8 and "exponents" not in st):
            raise ValueError(f"AdamW: a state without {second!r}: was it saved with other state_bits than {self.state_bits}?")
        for k in ("exp_avg", second):
            t = st[k]
            if t.dtype != dtype or t.shape != p.shape or t.device != p.device or t.stride() != p.stride():
                raise ValueError(f"AdamW: state {k!r} is {t.dtype} {tuple(t.shape)} {t.stride()} on {t.device}, the parameter wants {dtype} "
                                 f"{tuple(p.shape)} {p.stride()} on {p.device}")
        if self.state_bits == 8:
            e = st["exponents"]
            if e.dtype != torch.int8 or e.shape != (-(-p.numel() // STATE_BLOCK), 2) or not e.is_contiguous() or e.device != p.device:
                raise ValueError(f"AdamW: state 'exponents' is {e.dtype} {tuple(e.shape)} on {e.device}")

    def load_state_dict(self, state_dict):
        for g in state_dict["param_groups"]:
            # what another optimizer's checkpoint may ask of a step, which this one does not do
            for option in ("amsgrad", "maximize"):
                if g.get(option):
                    raise ValueError(f"AdamW: a state saved with {option}=True: there is no such step here")
            if not g.get("decoupled_weight_decay", True) and g.get("weight_decay"):
                raise ValueError("AdamW: a state saved by an optimizer that adds its weight decay to the gradient")
        # torch casts every floating-point state to the parameter's type: the moments keep their own here
        super().load_state_dict(state_dict)
        saved = state_dict["state"]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, params):
            if i not in saved:
                continue
            st = self.state[p]
            for k, v in saved[i].items():
                if k != "step" and torch.is_tensor(v):
                    like = k != "exponents" and v.shape == p.shape
                    t = torch.empty_strided(p.shape, p.stride(), dtype=v.dtype, device=p.device) if like else torch.empty(v.shape, dtype=v.dtype, device=p.device)
                    st[k] = t.copy_(v)
            if self.state_bits == 8 and "exponents" in st:
                for column, k in enumerate(("exp_avg", "exp_avg_rms")):
                    v = saved[i].get(k)
                    if v is not None and v.dtype == st[k].dtype and v.shape == p.shape and _order(v) != _order(p):
                        # its elements lie in another order in memory than p's, so other ones share an exponent now
                        if not _dense(v):
                            raise ValueError(f"AdamW: state {k!r} of strides {v.stride()} is not dense: which of its elements share an exponent is not known")
                        self._encode(p, st, column, k, _decode(v.to(p.device), saved[i]["exponents"].to(p.device)[:, column]))
            if self.state_bits == 32 and "exp_avg" in st:
                for k in ("exp_avg", "exp_avg_sq"):
                    if k in st:
                        st[k] = st[k].float()
            st["step"] = int(saved[i]["step"])
            self._check_state(p, st)

    @staticmethod
    def _encode(p, st, column, k, values):
        """`values` (fp32, p's shape) as the 8-bit moment k of p, to the nearest; a root that is not zero does not become zero (it divides)."""
        n = p.numel()
        flat = torch.as_strided(torch.empty_strided(p.shape, p.stride(), dtype=torch.float32, device=p.device).copy_(values), (n,), (1,))
        blocks = torch.nn.functional.pad(flat, (0, -n % STATE_BLOCK)).view(-1, STATE_BLOCK)
        top = torch.where(blocks.isfinite(), blocks.abs(), 0).amax(1)
        exponents = ((top.view(torch.int32) >> 23) - 127).clamp(min=-119)
        scaled = (blocks * torch.exp2(7.0 - exponents.float())[:, None])
        if column == 1:
            scaled = torch.where((scaled > 0) & (scaled < 2.0 ** -9), 2.0 ** -9, scaled)
        codes = scaled.to(torch.float8_e4m3fn).view(torch.uint8).reshape(-1)[:n]
        torch.as_strided(st[k].view(torch.uint8), (n,), (1,)).copy_(codes)
        st["exponents"][:, column] = exponents

    def decoded_state(self, p):
        """The two moments of parameter p as fp32 tensors of its shape: (exp_avg, exp_avg_sq)."""
        st = self.state[p]
        if self.state_bits == 32:
            return st["exp_avg"].clone(), st["exp_avg_sq"].clone()
        m, r = (_decode(st[k], st["exponents"][:, column]) for column, k in enumerate(("exp_avg", "exp_avg_rms")))
        return m, r * r

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        place = 0
        for k, g in enumerate(self.param_groups):
            ps = g["params"]
            b1, b2 = g["betas"]
            if self._host.adamw(ps, self._states_of(k, ps), place, self.state_bits, float(g["lr"]), float(b1), float(b2), float(g["eps"]),
                                float(g["weight_decay"]), self.seed & 0xffffffff) < 0:
                # the first step, parameters that joined later or have other orders of their axes, or something to refuse
                live = [k for k, p in enumerate(ps) if p.grad is not None]
                with torch.no_grad():
                    self._step_tensors(g, [ps[k] for k in live], [ps[k].grad for k in live], [place + k for k in live])
            place += len(ps)
        return loss

    def _states_of(self, k, ps):
        """The state dicts of group k's parameters, in order, None for one that has none.  The list is kept as long as self.state holds the same
        dicts for the same parameters and the group the same parameters."""
        if not self._host.same_items(self.state, self._order):
            self._order, self._lists = [x for item in self.state.items() for x in item], {}
        known = self._lists.get(k)
        if known is None or not self._host.same_objects(ps, known[0]):
            known = self._lists[k] = (list(ps), [self.state[p] if p in self.state else None for p in ps])
        return known[1]

    def _step_tensors(self, g, ps, grads, places):
        if not ps:
            return
        first = ps[0]
        with torch.cuda.device(first.device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(self._host.ADAMW_CAPTURED)
        index = first.get_device()
        state = self.state
        states = [state[p] if p in state else self._new_state(p) for p in ps]
        second = "exp_avg_sq" if self.state_bits == 32 else "exp_avg_rms"
        for p, st in zip(ps, states):
            self._check_state(p, st)
        steps = {st["step"] for st in states}
        dtypes = {p.dtype for p in ps}
        if len(steps) != 1 or len(dtypes) != 1 or not all(type(s) is int for s in steps):
            # parameters that joined later, or of several types: a call for each
            for st in states:
                if type(st["step"]) is not int:
                    st["step"] = int(st["step"])
            sets = {}
            for k, (p, st) in enumerate(zip(ps, states)):
                sets.setdefault((st["step"], p.dtype), []).append(k)
            if len(sets) > 1:
                for ks in sets.values():
                    self._step_tensors(g, [ps[k] for k in ks], [grads[k] for k in ks], [places[k] for k in ks])
                return
        dtype, step = first.dtype, states[0]["step"] + 1
        if not (all(map(torch.Tensor.is_contiguous, grads)) and all(map(torch.Tensor.is_contiguous, ps))):
            grads = [x if not x.is_sparse and x.stride() == p.stride() else self._like(p, x) for p, x in zip(ps, grads)]
        if {x.dtype for x in grads} != dtypes or {x.get_device() for x in grads} != {index} or {p.get_device() for p in ps} != {index}:
            raise ValueError(f"AdamW: parameters and gradients have to be {dtype} on {first.device}")
        moments = [st["exp_avg"] for st in states], [st[second] for st in states], [st.get("exponents") for st in states]
        sizes = [p.numel() for p in ps]
        table = np.zeros((len(ps), 7), np.int64)
        table[:, 0] = [p.data_ptr() for p in ps]
        table[:, 1] = [x.data_ptr() for x in grads]
        table[:, 2] = [t.data_ptr() for t in moments[0]]
        table[:, 3] = [t.data_ptr() for t in moments[1]]
        if self.state_bits == 8:
            table[:, 4] = [t.data_ptr() for t in moments[2]]
        table[:, 5] = sizes
        table[:, 6] = places
        b1, b2 = g["betas"]
        with torch.cuda.device(index):
            _lib.check(self._lib.vc_adamw(table.ctypes.data, len(ps), _PARAM_DTYPES[dtype], self.state_bits, float(g["lr"]), float(b1), float(b2),
                                          float(g["eps"]), float(g["weight_decay"]), step, self.seed & 0xffffffff,
                                          torch._C._cuda_getCurrentRawStream(index)), "vc_adamw")
        _written([*ps, *(t for ts in moments for t in ts if t is not None)])
        for st in states:
            st["step"] = step

    @staticmethod
    def _like(p, grad):
        if grad.is_sparse:
            raise ValueError("AdamW: gradients have to be dense")
        return torch.empty_like(p, memory_format=torch.preserve_format).copy_(grad)


_PARAM_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}   # vc_dtype
