"""Newton-Schulz orthogonalisation and the Muon optimizer on the MI355X matrix cores.

``newton_schulz(x)`` replaces a matrix by (nearly) its orthogonal factor: with
``X = x / max(|x|_F, eps)``, ``steps`` times ``X = a X + (b S + c S^2) X``, ``S = X X^T``.
``Muon`` is a drop-in for ``torch.optim.Muon``: the same constructor, ``param_groups`` and
state (``momentum_buffer``; checkpoints interchange).  It steps the matrices of the hidden
layers (mini-megatron's qkv, o, fc1 and fc2 weights, model/transformer.py:22-23,42-43);
embeddings, layer norms and the head stay with ``FusedAdamW``.  A step of many matrices of
any sizes runs as one sequence of launches over all of them.

Precision.  ``"half"``: fp16 products with fp32 sums, the iterate in two fp16 terms and the
square factors' diagonals in fp32.  Against the iteration in 64 bits (relative, in the 2-norm of
its entries) the result is 3e-4 to 7e-4 off on gradients' spectra and full ranks, below what a bf16
result rounds, up to 2e-3 on matrices of low rank and 4e-3 on those of a handful of nonzero
entries; the same iteration in bf16 is 1e-2 off, and more than 0.1 on low ranks.  ``"single"``:
fp32's error, at three products for one.  Matrices with a side up to 128 always run in single: their
products take no time.  Up to 64 x 512 and 128 x 128 a matrix is one workgroup's, in one launch.
"""
from __future__ import annotations

import ctypes
import functools
import math

import numpy as np
import torch
from torch.optim import Optimizer

from . import _lib
from .norm import refuse_records
from .optimizer import _ROW_DTYPE, _upload

NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}
_PRECISIONS = {"half": _lib.NS_HALF, "single": _lib.NS_SINGLE}
_SMALL = 128                   # sides up to here run in single precision
_WORKSPACE = 1 << 30           # bytes of workspace that a batch of matrices may take
_LAUNCH = (1 << 23) - 1        # matrices that a launch of a workgroup each may take
_MATRIX_DTYPE = np.dtype([("workspace", "<i8"), ("rows", "<i4"), ("cols", "<i4"),
                          ("lr_ratio", "<f4"), ("reserved", "<i4")])
assert _MATRIX_DTYPE.itemsize == ctypes.sizeof(_lib.Matrix)


def _options(coefficients, eps: float, steps: int, precision: int) -> _lib.NsOptions:
    """The checked options of a call, or ValueError."""
    if type(steps) is not int:
        raise ValueError(f"Number of steps must be a positive integer, got {steps}")
    return _checked_options(tuple(coefficients), float(eps), steps, precision)


@functools.lru_cache(maxsize=64)
def _checked_options(coefficients: tuple, eps: float, steps: int,
                     precision: int) -> _lib.NsOptions:
    if len(coefficients) != 3:
        raise ValueError("Coefficients must be a tuple of exactly 3 values")
    if steps < 1:
        raise ValueError(f"Number of steps must be a positive integer, got {steps}")
    if steps >= 100:
        raise ValueError("Number of steps must be less than 100 for computational efficiency")
    if not (0 <= eps <= _lib.FP32_MAX):
        raise ValueError(f"eps should be >= 0 and finite in fp32 but is: {eps}")
    o = _lib.NsOptions(*(float(c) for c in coefficients), eps, steps, precision)
    if _lib.load().mi_adamw_ns_check(ctypes.byref(o)) != _lib.OK:
        raise ValueError(f"Newton-Schulz coefficients {tuple(coefficients)} let singular values "
                         "grow past the range the kernels hold")
    return o


def _precision(name, rows: int, cols: int, dtype: torch.dtype) -> int:
    if name is not None and name not in _PRECISIONS:
        raise ValueError(f'precision must be None, "half" or "single", got {name!r}')
    if min(rows, cols) <= _SMALL:
        return _lib.NS_SINGLE
    if name is None:
        return _lib.NS_SINGLE if dtype == torch.float32 else _lib.NS_HALF
    return _PRECISIONS[name]


def _rows_dense(t: torch.Tensor) -> bool:
    """Whether the matrices of a 3-D tensor lie row by row, rows at any distance."""
    return ((t.shape[2] == 1 or t.stride(2) == 1) and
            (t.shape[1] == 1 or t.stride(1) >= t.shape[2]))


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(1) if t.shape[1] > 1 else t.shape[2]


def _overlap(x: torch.Tensor, out: torch.Tensor) -> bool:
    """Whether writing a matrix of a 3-D out may change another one of x before it is read: out
    shares memory with x and is not the same view.  (Each matrix is read before it is written.)"""
    if x.shape[0] == 1 or (x.data_ptr() == out.data_ptr() and x.stride() == out.stride()):
        return False
    ends = [t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in
                                                       zip(t.shape, t.stride()))) for t in (x, out)]
    return x.data_ptr() < ends[1] and out.data_ptr() < ends[0]


@torch.no_grad()
def newton_schulz(x: torch.Tensor, *, steps: int = 5, coefficients=NS_COEFFICIENTS,
                  eps: float = 1e-7, precision: str | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Orthogonalise a matrix, or each matrix of a 3-D batch, by Newton-Schulz products.

    x:          fp32 or bf16 on a ROCm GPU, 2-D or 3-D; rows or columns dense at any stride
                (other layouts are copied first).  The result carries no gradient, and a
                forward-mode tangent is refused.
    precision:  "half", "single", or None: single for fp32, half for bf16.
    out:        where the result goes (same shape, dtype and device; may be x itself or share
                memory with it).
    """
    if torch.compiler.is_compiling():
        return _untraced(x, steps=steps, coefficients=coefficients, eps=eps, precision=precision,
                         out=out)
    if x.dim() not in (2, 3):
        raise ValueError(f"newton_schulz takes a matrix or a batch of them, got {x.dim()} "
                         "dimensions")
    if x.dtype not in _DTYPES:
        raise NotImplementedError(f"newton_schulz: dtype {x.dtype} is not supported (fp32 and "
                                  "bf16 are)")
    o = _options(coefficients, eps, steps, _precision(precision, *x.shape[-2:], x.dtype))
    if x.device.type != "cuda":
        raise RuntimeError(f"newton_schulz runs on a ROCm GPU only; got a {x.device.type} tensor")
    if out is not None and (out.shape != x.shape or out.dtype != x.dtype
                            or out.device != x.device):
        raise ValueError("newton_schulz: out needs x's shape, dtype and device")
    refuse_records("newton_schulz", x, out)
    given = out is not None
    if not given:
        out = torch.empty_like(x)
    if x.numel() == 0:
        return out
    x3, o3 = (x, out) if x.dim() == 3 else (x.unsqueeze(0), out.unsqueeze(0))
    if not _rows_dense(x3) or not _rows_dense(o3):
        xt, ot = x3.transpose(1, 2), o3.transpose(1, 2)
        if _rows_dense(xt) and _rows_dense(ot):
            x3, o3 = xt, ot         # the iteration commutes with the transposition
        else:
            x3 = x3 if _rows_dense(x3) else x3.contiguous()
    to = o3
    if not _rows_dense(o3) or _overlap(x3, o3) or (
            o3.shape[0] > 1 and
            o3.stride(0) < (o3.shape[1] - 1) * _row_stride(o3) + o3.shape[2]):
        to = torch.empty(o3.shape, dtype=o3.dtype, device=o3.device)
    batch, rows, cols = x3.shape
    lib = _lib.load()
    per = lib.mi_adamw_ns_workspace(rows, cols, o.precision)
    if per < 0:
        raise NotImplementedError(f"newton_schulz: a {rows} x {cols} matrix is too large")
    index = x.device.index
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(index):
            return newton_schulz(x, steps=steps, coefficients=coefficients, eps=eps,
                                 precision=precision, out=out)
    at_once = max(1, min(batch, _WORKSPACE // per if per else _LAUNCH))
    ws = torch.empty(at_once * per, dtype=torch.uint8, device=x.device) if per else None
    size = x.element_size()
    stream = torch._C._cuda_getCurrentRawStream(index)
    for b in range(0, batch, at_once):
        _lib.check(lib.mi_adamw_newton_schulz(
            x3.data_ptr() + b * x3.stride(0) * size, x3.stride(0), _row_stride(x3),
            to.data_ptr() + b * to.stride(0) * size, to.stride(0), _row_stride(to),
            min(at_once, batch - b), rows, cols, _DTYPES[x.dtype], ctypes.addressof(o),
            None if ws is None else ws.data_ptr(), at_once * per, stream),
            "mi_adamw_newton_schulz")
    if to is not o3:
        o3.copy_(to)
    elif given:
        torch.autograd.graph.increment_version(out)     # as an operator that writes it in place
    return out


# torch.compile ends its graph here: it cannot trace the library's calls
_untraced = torch._disable_dynamo(newton_schulz)


class _Batch:
    """The device tables of matrices that are stepped by one sequence of launches."""

    __slots__ = ("params", "rows", "host_rows", "matrices", "items", "tables", "options",
                 "workspace", "stream", "rows_stream", "recorded", "kept", "__weakref__")

    def __init__(self, entries, options: _lib.NsOptions, adjust, copies, device, stream: int):
        """entries: (parameter, gradient, momentum) triples; stream: the current one."""
        lib = _lib.load()
        self.params = [p for p, _, _ in entries]
        self.options = options
        self.stream = self.rows_stream = stream     # where the tables and the rows were allocated
        # What graphs read, once a step was recorded: their end is not announced, so it stays.
        # `recorded`: the present rows are among it, and then never change.
        self.kept: list = []
        self.recorded = False
        n = len(entries)
        rows = np.zeros(n, dtype=_ROW_DTYPE)
        rows["param"] = [p.data_ptr() for p in self.params]
        rows["grad"] = [g.data_ptr() for _, g, _ in entries]
        rows["exp_avg"] = [m.data_ptr() for _, _, m in entries]
        if copies is not None:
            rows["param_copy"] = [copies[id(p)].data_ptr() for p in self.params]
        rows["numel"] = [p.numel() for p in self.params]
        mats = np.zeros(n, dtype=_MATRIX_DTYPE)
        mats["rows"] = [p.shape[0] for p in self.params]
        mats["cols"] = [p.shape[1] for p in self.params]
        mats["lr_ratio"] = [adjust(*p.shape) for p in self.params]
        sizes = [lib.mi_adamw_ns_workspace(*p.shape, options.precision) for p in self.params]
        mats["workspace"] = np.cumsum([0] + sizes[:-1])
        self.workspace = sum(sizes)
        self.host_rows = rows
        self.rows = _upload(rows, device)
        self.matrices = _upload(mats, device)
        self.tables = _lib.MuonTables()
        self.items = []
        self.tables.whole = lib.mi_adamw_ns_whole(*self.params[0].shape)
        _lib.check(lib.mi_adamw_muon_cut(mats.ctypes.data, n, options.precision,
                                         ctypes.addressof(self.tables)), "mi_adamw_muon_cut")
        for kind in range(5):
            if (kind == _lib.NS_WHOLE) != bool(self.tables.whole):
                self.items.append(None)
                continue
            tile = self.tables.pair_tile if kind == _lib.NS_PAIRS else self.tables.tile
            args = (mats.ctypes.data, n, kind, tile, self.tables.split)
            count = lib.mi_adamw_muon_items(*args, None, 0)
            _lib.check(int(min(count, 0)), "mi_adamw_muon_items")
            items = np.empty(2 * count, dtype=np.int32)
            lib.mi_adamw_muon_items(*args, items.ctypes.data, count)
            self.items.append(_upload(items, device))
            self.tables.items[kind] = self.items[-1].data_ptr()
            self.tables.n_items[kind] = count

    def used_on(self, stream: int, device: torch.device) -> None:
        """An eager launch on `stream` reads the tables.  A program orders the steps of the same
        parameters on different streams, and so the tables' contents; their memory has to outlast
        what is queued on streams other than the one it was allocated on."""
        if device.type != "cuda" or stream == self.stream == self.rows_stream:
            return
        current = torch.cuda.current_stream(device)
        for t, home in ((self.rows, self.rows_stream), (self.matrices, self.stream),
                        *((t, self.stream) for t in self.items)):
            if t is not None and home != stream:
                t.record_stream(current)

    def record(self, entries) -> None:
        """A graph's launches take these tables, and with them the tensors whose addresses
        they hold: parameter, gradient, momentum and copy of each entry."""
        if not self.recorded:
            self.recorded = True
            self.kept.append((self.rows, entries))

    def grads(self) -> np.ndarray:
        """The addresses of the gradients now."""
        return np.fromiter((p.grad.data_ptr() for p in self.params), dtype=np.uint64,
                           count=len(self.params))

    def move_grads(self, grads: np.ndarray, device: torch.device, stream: int) -> None:
        """The gradients lie elsewhere: their addresses go to the device as kernel arguments,
        or in new rows where a graph reads the old ones."""
        idx = np.flatnonzero(grads != self.host_rows["grad"]).astype(np.int32)
        if not len(idx):
            return
        if self.recorded:
            self.recorded = False
            self.host_rows["grad"] = grads
            self.rows, self.rows_stream = _upload(self.host_rows, device), stream
            return
        moved = np.ascontiguousarray(grads[idx])
        vec = np.zeros(len(idx), dtype=np.uint8)
        code = _lib.load().mi_adamw_set_grads(self.rows.data_ptr(), len(self.host_rows), len(idx),
                                              idx.ctypes.data, moved.ctypes.data,
                                              vec.ctypes.data, stream)
        self.host_rows["grad"] = grads if code == _lib.OK else 0
        _lib.check(code, "mi_adamw_set_grads")


def _original(rows: int, cols: int) -> float:
    return math.sqrt(max(1.0, rows / cols))


def _match_rms_adamw(rows: int, cols: int) -> float:
    return 0.2 * math.sqrt(max(rows, cols))


_ADJUST = {None: _original, "original": _original, "match_rms_adamw": _match_rms_adamw}


class Muon(Optimizer):
    """torch.optim.Muon with every matrix's step in hand-written MI355X kernels: momentum,
    orthogonalisation and weight update of all matrices in one sequence of launches.

    The constructor takes torch.optim.Muon's arguments with its defaults and checks; a step is

        buf = lerp(buf, grad, 1 - momentum);  u = lerp(grad, buf, momentum) if nesterov else buf
        p = p (1 - lr weight_decay) - lr ratio newton_schulz(u)

    with ratio sqrt(max(1, rows / cols)) (adjust_lr_fn None or "original") or
    0.2 sqrt(max(rows, cols)) ("match_rms_adamw").  Keyword-only:

    ns_precision: "half" (default) or "single", see the module.
    bf16_copy:    keep a bf16 copy of every parameter, written by the step, for
                  ``mi_adamw.bf16_weights``.

    Parameters are 2-D, contiguous, fp32 and on one ROCm GPU, as are their gradients.  A step
    may be recorded into a HIP graph, on any stream, once an eager one has built its tables
    with the gradients in place; the learning rate is recorded as its value.
    """

    def __init__(self, params, lr: float | torch.Tensor = 1e-3, weight_decay: float = 0.1,
                 momentum: float = 0.95, nesterov: bool = True,
                 ns_coefficients: tuple[float, float, float] = NS_COEFFICIENTS,
                 eps: float = 1e-7, ns_steps: int = 5, adjust_lr_fn: str | None = None, *,
                 ns_precision: str = "half", bf16_copy: bool = False) -> None:
        if isinstance(lr, torch.Tensor) and lr.numel() != 1:
            raise ValueError("Tensor lr must be 1-element")
        if not 0.0 <= lr:
            raise ValueError(f"Learning rate should be >= 0 but is: {lr}")
        if not 0.0 <= momentum:
            raise ValueError(f"momentum should be >= 0 but is: {momentum}")
        if not 0.0 <= weight_decay:
            raise ValueError(f"weight decay should be >= 0 but is: {weight_decay}")
        if adjust_lr_fn not in _ADJUST:
            raise ValueError(f"Adjust learning rate function {adjust_lr_fn} is not supported")
        if ns_precision not in _PRECISIONS:
            raise ValueError(f'ns_precision must be "half" or "single", got {ns_precision!r}')
        _options(ns_coefficients, eps, ns_steps, _PRECISIONS[ns_precision])
        self.ns_precision = ns_precision
        self.bf16_copy = bool(bf16_copy)
        self._reset_bookkeeping()
        super().__init__(params, dict(
            lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov,
            ns_coefficients=ns_coefficients, eps=eps, ns_steps=ns_steps,
            adjust_lr_fn=adjust_lr_fn))
        self.register_load_state_dict_post_hook(Muon._after_load_state_dict)

    def _reset_bookkeeping(self) -> None:
        self._copies: dict[int, torch.Tensor] = {}
        self._copy_sync: dict[int, tuple[int, int]] | None = None
        self._batches: list[list[_Batch]] = []
        self._kept: list = []
        self._key = None

    def __getstate__(self):
        state = super().__getstate__()
        state["mi_adamw_options"] = {"ns_precision": self.ns_precision,
                                     "bf16_copy": self.bf16_copy}
        return state

    def __setstate__(self, state) -> None:
        options = state.pop("mi_adamw_options", None)
        super().__setstate__(state)
        if options is None:                 # load_state_dict
            self._key = None
            return
        self.__dict__.update(options)
        self._reset_bookkeeping()
        self.register_load_state_dict_post_hook(Muon._after_load_state_dict)
        for group in self.param_groups:
            self._make_copies(group["params"])

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        for p in group["params"]:
            if p.dim() != 2:
                self.param_groups.pop()
                raise ValueError("Muon only supports 2D parameters whereas we found a parameter "
                                 f"with size: {p.size()}")
        self._make_copies(group["params"])

    def _make_copies(self, params) -> None:
        if self.bf16_copy:
            for p in params:
                self._refresh_copy(p)

    def _after_load_state_dict(self: "Muon") -> None:
        self._key = None
        if self.bf16_copy:
            self.refresh_bf16_copies()

    # ------------------------------------------------------------ bf16 copies

    def bf16_param(self, p: torch.Tensor) -> torch.Tensor:
        if not self.bf16_copy:
            raise RuntimeError("Muon was built without bf16_copy=True")
        return self._copies[id(p)]

    def bf16_params(self) -> list[torch.Tensor]:
        """The bf16 model copies, in param_groups order (bf16_copy=True)."""
        return [self.bf16_param(p) for g in self.param_groups for p in g["params"]]

    @torch.no_grad()
    def refresh_bf16_copies(self) -> None:
        """Rewrite every bf16 copy from its fp32 master (after the masters were changed
        outside the optimizer, e.g. through ``p.data``)."""
        if not self.bf16_copy:
            raise RuntimeError("Muon was built without bf16_copy=True")
        for g in self.param_groups:
            for p in g["params"]:
                self._refresh_copy(p)

    def _refresh_copy(self, p: torch.Tensor) -> None:
        c = self._copies.get(id(p))
        if c is None or c.shape != p.shape or c.device != p.device:
            self._copies[id(p)] = p.detach().to(torch.bfloat16,
                                                memory_format=torch.contiguous_format)
            self._key = None
        else:
            c.copy_(p.detach())
        if self._copy_sync is not None:
            self._copy_sync[id(p)] = (p._version, p.data_ptr())

    def _track_copies(self) -> None:
        """First use of bf16_weights: every copy is rewritten once, then each step records the
        masters it wrote."""
        if self._copy_sync is None:
            self._copy_sync = {}
            self.refresh_bf16_copies()

    def _current_copies(self, masters: list) -> list:
        """The masters' copies, rewritten first where the master changed since."""
        stale = [p for p in masters
                 if self._copy_sync.get(id(p)) != (p._version, p.data_ptr())]
        if stale:
            with torch.no_grad():
                for p in stale:
                    self._refresh_copy(p)
        return [self._copies[id(p)] for p in masters]

    # ------------------------------------------------------------ step

    def _entry(self, p: torch.Tensor):
        """(parameter, gradient, momentum) of a parameter to step, checked."""
        g = p.grad
        if g.is_sparse:
            raise RuntimeError("Muon does not support sparse gradients")
        if torch.is_complex(p):
            raise RuntimeError("Muon does not support complex parameters")
        if p.device.type != "cuda":
            raise RuntimeError(f"Muon steps parameters on a ROCm GPU only; got a {p.device.type} "
                               "parameter")
        if p.dtype != torch.float32:
            raise NotImplementedError(f"Muon: parameter dtype {p.dtype} is not supported (fp32 "
                                      "master parameters only)")
        if p.dim() != 2:
            raise ValueError("Muon only supports 2D parameters whereas we found a parameter "
                             f"with size: {p.size()}")
        if g.dtype != p.dtype or g.shape != p.shape or g.device != p.device:
            raise RuntimeError("Muon: gradient dtype/shape/device differs from its parameter")
        if not (p.is_contiguous() and g.is_contiguous()):
            raise NotImplementedError("Muon: parameters and gradients must be contiguous")
        st = self.state[p]
        m = st.get("momentum_buffer")
        if m is None:
            if torch.cuda.is_current_stream_capturing():
                self._refuse_capture()      # its zeros would only be recorded
            m = st["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
        if m.dtype != torch.float32 or m.shape != p.shape or m.device != p.device:
            raise RuntimeError("Muon: momentum_buffer dtype/shape/device differs from its "
                               "parameter")
        if not m.is_contiguous():
            m = st["momentum_buffer"] = m.contiguous()
        return p, g, m

    @staticmethod
    def _refuse_capture() -> None:
        raise RuntimeError("Muon: step() under graph capture, but its tables are not those of "
                           "the last eager step; run one eager step with the same parameters, "
                           "gradient tensors, state and options before capturing")

    def _build(self, groups, device, stream: int) -> list[list[_Batch]]:
        """Each group's matrices, by precision, in batches whose workspace stays bounded."""
        lib = _lib.load()
        built = []
        for group, entries in zip(self.param_groups, groups):
            adjust = _ADJUST[group["adjust_lr_fn"]]
            built.append([])
            # matrices that one workgroup works on, by the kernel that does; the others by
            # precision
            classes: dict[tuple, list] = {}
            for e in entries:
                shape = e[0].shape
                precision = _precision(self.ns_precision, *shape, torch.float32)
                classes.setdefault((lib.mi_adamw_ns_whole(*shape), precision), []).append(e)
            for (_, precision), members in sorted(classes.items(), key=lambda c: c[0]):
                # the longest sums first: two layers of 2048 x 8192 4.99 ms so, 5.27 as they come
                members.sort(key=lambda e: -max(e[0].shape))
                options = _options(group["ns_coefficients"], group["eps"], group["ns_steps"],
                                   precision)
                batch, size = [], 0
                for e in members:
                    need = lib.mi_adamw_ns_workspace(*e[0].shape, precision)
                    if need < 0:
                        raise NotImplementedError("Muon: a matrix of size "
                                                  f"{tuple(e[0].shape)} is too large")
                    if batch and size + need > _WORKSPACE:
                        built[-1].append(_Batch(batch, options, adjust, self._copies_or_none(),
                                                device, stream))
                        batch, size = [], 0
                    batch.append(e)
                    size += need
                built[-1].append(_Batch(batch, options, adjust, self._copies_or_none(), device,
                                        stream))
        return built

    def _copies_or_none(self):
        return self._copies if self.bf16_copy else None

    @torch.no_grad()
    def step(self, closure=None):
        """One optimizer step.  Returns closure's loss."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        groups = [[self._entry(p) for p in g["params"] if p.grad is not None and p.numel()]
                  for g in self.param_groups]
        device = next((e[0].device for entries in groups for e in entries), None)
        if device is None:
            return loss
        if any(e[0].device != device for entries in groups for e in entries):
            raise RuntimeError("Muon: every parameter must be on one ROCm GPU")
        if torch._C._cuda_getDevice() != device.index:
            with torch.cuda.device(device.index):
                self._launch(groups, device)
        else:
            self._launch(groups, device)
        return loss

    def _launch(self, groups, device) -> None:
        capturing = torch.cuda.is_current_stream_capturing()
        if self.bf16_copy:
            for entries in groups:
                for p, _, _ in entries:
                    c = self._copies.get(id(p))
                    if c is None or c.shape != p.shape or c.device != device:
                        if capturing:
                            self._refuse_capture()
                        self._refresh_copy(p)
        stream = torch._C._cuda_getCurrentRawStream(device.index)
        key = (self.ns_precision,
               [(g["adjust_lr_fn"], tuple(g["ns_coefficients"]), g["eps"], g["ns_steps"])
                for g in self.param_groups],
               [[(p.data_ptr(), m.data_ptr(), p.shape) for p, _, m in entries]
                for entries in groups])
        if capturing and (key != self._key or any(
                not np.array_equal(b.grads(), b.host_rows["grad"])
                for batches in self._batches for b in batches)):
            self._refuse_capture()
        if key != self._key:
            self._key = None
            new = self._build(groups, device, stream)
            self._kept += [b for batches in self._batches for b in batches if b.kept]
            self._batches = new
            self._key = key
        lib = _lib.load()
        most = max(b.workspace for batches in self._batches for b in batches)
        ws = torch.empty(most, dtype=torch.uint8, device=device)
        flags = _lib.F_BF16_COPY if self.bf16_copy else 0
        for group, batches in zip(self.param_groups, self._batches):
            lr, momentum = float(group["lr"]), float(group["momentum"])
            hyper = _lib.MuonHyper(1 - momentum, momentum, bool(group["nesterov"]),
                                   1 - lr * group["weight_decay"], -lr)
            for b in batches:
                if capturing:
                    b.record([(p.detach(), p.grad, self.state[p]["momentum_buffer"],
                               self._copies.get(id(p))) for p in b.params])
                else:
                    b.move_grads(b.grads(), device, stream)
                    b.used_on(stream, device)
                _lib.check(lib.mi_adamw_muon_step(
                    b.rows.data_ptr(), b.matrices.data_ptr(), ctypes.addressof(b.tables),
                    ctypes.addressof(hyper), ctypes.addressof(b.options), flags, ws.data_ptr(),
                    stream), "mi_adamw_muon_step")
        for entries in groups:
            for p, _, m in entries:
                copy = (self._copies[id(p)],) if self.bf16_copy else ()
                torch.autograd.graph.increment_version((p, m, *copy))
                if self._copy_sync is not None:
                    self._copy_sync[id(p)] = (p._version, p.data_ptr())
